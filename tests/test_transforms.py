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
