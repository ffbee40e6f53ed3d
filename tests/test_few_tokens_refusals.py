"""What the few-token layer refuses, on the host (no GPU)."""
import pytest
import torch

import moe_ops_b200 as M
from moe_ops_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _call(lib, T=4, d=64, H=64, E=8, K=2, dtype=2, ws=1 << 40, given=False, p=16):
    fn = lib.moe_few_experts_fwd if given else lib.moe_few_tokens_fwd
    st = fn(p, p, p, p, p, p, dtype, T, d, H, E, K, p, p, ws, None)
    return st, lib.moe_last_error_string()


def test_c_abi_refusals(lib):
    assert lib.moe_few_tokens_workspace_bytes(0, 64, 64, 8, 2, 2) == 0
    need = lib.moe_few_tokens_workspace_bytes(4, 64, 64, 8, 2, 2)
    assert need >= 4 * 8 * 4
    st, msg = _call(lib, ws=need - 1)
    assert st == 4 and b"workspace" in msg
    for kw, word in ((dict(T=129), b"num_tokens"), (dict(T=-1), b"num_tokens"), (dict(E=0), b"E"),
                     (dict(E=1025), b"E"), (dict(K=0), b"K"), (dict(K=9), b"K"),
                     (dict(K=17, E=32), b"K"), (dict(K=17, E=32, given=True), b"K"),
                     (dict(dtype=7), b"dtype"), (dict(d=-8), b"sizes"), (dict(H=-1), b"sizes"),
                     (dict(p=None), b"NULL")):
        st, msg = _call(lib, **kw)
        assert st == 1 and word in msg, (kw, st, msg)
    assert _call(lib, T=0)[0] == 0


def test_python_refusals():
    x, wr = torch.zeros(2, 8), torch.zeros(4, 8)
    wg, wu, wd = torch.zeros(4, 6, 8), torch.zeros(4, 6, 8), torch.zeros(4, 8, 6)
    with pytest.raises(RuntimeError, match="CUDA"):
        M.moe_few_tokens(x, wr, wg, wu, wd, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        M.moe_few_experts(x, torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int32), wg, wu, wd)


@pytest.mark.gpu
def test_python_refusals_on_device(cuda_dev):
    def z(*s, dtype=torch.bfloat16):
        return torch.zeros(*s, device=cuda_dev, dtype=dtype)

    x, wr, wg, wu, wd = z(2, 8), z(4, 8), z(4, 6, 8), z(4, 6, 8), z(4, 8, 6)
    i2 = z(2, 2, dtype=torch.int32)
    bad = [
        lambda: M.moe_few_tokens(z(2, 9), wr, wg, wu, wd, 2),
        lambda: M.moe_few_tokens(x[0], wr, wg, wu, wd, 2),
        lambda: M.moe_few_tokens(x, wr, wg, z(4, 5, 8), wd, 2),
        lambda: M.moe_few_tokens(x, wr, wg, wu, z(4, 6, 8), 2),
        lambda: M.moe_few_tokens(x, z(3, 8), wg, wu, wd, 2),
        lambda: M.moe_few_tokens(x, wr.float(), wg, wu, wd, 2),
        lambda: M.moe_few_tokens(x.half(), wr, wg, wu, wd, 2),
        lambda: M.moe_few_tokens(x, wr, wg, wu, wd, 0),
        lambda: M.moe_few_tokens(x, wr, wg, wu, wd, 5),
        lambda: M.moe_few_tokens(z(129, 8), wr, wg, wu, wd, 2),
        lambda: M.moe_few_tokens(x, wr, wg, wu, wd, 2, router_bias=z(3)),
        lambda: M.moe_few_experts(x, z(2, 3), i2, wg, wu, wd),
        lambda: M.moe_few_experts(x, z(3, 2), z(3, 2, dtype=torch.int32), wg, wu, wd),
        lambda: M.moe_few_experts(x, z(2, 2), z(2, 2), wg, wu, wd),
        lambda: M.moe_few_experts(x, z(2, 17), z(2, 17, dtype=torch.int32), wg, wu, wd),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        M.moe_few_tokens(*(t.double() for t in (x, wr, wg, wu, wd)), 2)
    wg.requires_grad_(True)
    with pytest.raises(RuntimeError, match="backward"):
        M.moe_few_tokens(x, wr, wg, wu, wd, 2)
    with torch.no_grad():
        assert M.moe_few_tokens(x, wr, wg, wu, wd, 2).shape == (2, 8)
