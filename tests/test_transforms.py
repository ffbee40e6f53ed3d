"""The few-token layer and linear / grouped_linear under what records calls instead of running them,
on the host (no GPU): fake tensors and make_fx."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import moe_ops_b200 as M
from moe_ops_b200.moe_layer import MoELayer

BF = torch.bfloat16


def fake(*shape, dtype=BF):
    return torch.empty(*shape, device="cuda", dtype=dtype)


def recorded(f, *args):
    """Names of the library's ops in the graph of f."""
    g = make_fx(f)(*args).graph
    return [str(n.target) for n in g.nodes if "moeb200" in str(n.target)]


@pytest.mark.parametrize("k,n", [(64, 40), (4097, 4099)])  # the second has rows of no 16-byte multiple
def test_linear(k, n):
    with FakeTensorMode():
        x, w, b, r = fake(3, 2, k), fake(n, k), fake(n), fake(3, 2, n)
        y = M.linear(x, w, bias=b, activation="gelu", residual=r)
        assert y.shape == (3, 2, n) and y.dtype == BF
        assert recorded(lambda a: M.linear(a, w, bias=b), x) == ["moeb200.linear_fwd.default"]
        A, B, off = fake(90, k), fake(5, n, k), fake(6, dtype=torch.int32)
        assert M.grouped_linear(A, B, off).shape == (90, n)
        assert recorded(lambda a: M.grouped_linear(a, B, off, activation="relu"), A) == \
            ["moeb200.linear_fwd.default"]


def test_few_tokens():
    with FakeTensorMode(), torch.no_grad():
        x, wr, wg, wd = fake(3, 64), fake(8, 64), fake(8, 48, 64), fake(8, 64, 48)
        assert M.moe_few_tokens(x, wr, wg, wg, wd, 2).shape == (3, 64)
        assert recorded(lambda a: M.moe_few_tokens(a, wr, wg, wg, wd, 2), x) == \
            ["moeb200.few_tokens.default"]
        w, i = fake(3, 2, dtype=torch.float32), fake(3, 2, dtype=torch.int32)
        assert M.moe_few_experts(x, w, i, wg, wg, wd).shape == (3, 64)
        assert recorded(lambda a: M.moe_few_experts(a, w, i, wg, wg, wd), x) == \
            ["moeb200.few_experts.default"]


def test_layer():
    with FakeTensorMode(), torch.no_grad():
        m = MoELayer(64, 8, 2, 48, device="cuda", dtype=BF, shared_hidden=32)
        m.few_tokens = 16
        ops = recorded(lambda a: m(a), fake(5, 64))
        assert ops == ["moeb200.few_tokens.default"] + ["moeb200.linear_fwd.default"] * 2


def test_registered_ops_give_the_real_shapes():
    """Shapes and dtypes of the four ops' fake forms."""
    ops, f32 = torch.ops.moeb200, torch.float32
    with FakeTensorMode():
        x, w, B, off, dy = fake(7, 64), fake(24, 64), fake(3, 64, 24), fake(4, dtype=torch.int32), fake(7, 24)
        wr, wg, wd = fake(8, 64), fake(8, 48, 64), fake(8, 64, 48)
        got = {
            "linear_fwd": ops.linear_fwd(x, w, None, None, None, 4, True, True),
            "linear_fwd, no z": ops.linear_fwd(x, B, None, None, off, 0, False, False),
            "linear_bwd": ops.linear_bwd(dy, x, w, dy, None, 4, True, True, True, True),
            "linear_bwd, grouped": ops.linear_bwd(dy, x, B, None, off, 0, False, False, True, True),
            "few_tokens": (ops.few_tokens(x, wr, wg, wg, wd, 2, None),),
            "few_experts": (ops.few_experts(x, fake(7, 2, dtype=f32), fake(7, 2, dtype=torch.int32), wg, wg, wd),),
        }
    want = {
        "linear_fwd": [(7, 24), (7, 24)], "linear_fwd, no z": [(7, 24), (0,)],
        "linear_bwd": [(7, 64), (24, 64), (24,)], "linear_bwd, grouped": [(0,), (3, 64, 24), (3, 24)],
        "few_tokens": [(7, 64)], "few_experts": [(7, 64)],
    }
    for name, out in got.items():
        assert [tuple(t.shape) for t in out] == want[name] and all(t.dtype == BF for t in out), name
