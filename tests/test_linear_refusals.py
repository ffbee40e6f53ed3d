"""What linear / grouped_linear refuse, on the host (no GPU)."""
import pytest
import torch

import moe_ops_b200 as M
from moe_ops_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_c_abi_refusals(lib):
    p = 16

    def fwd(m=4, n=8, k=8, E=1, act=0, dtype=2, num_offsets=0, off=None, a=p, ws=1 << 40):
        st = lib.moe_linear_fwd(a, p, p, p, p, None, off, num_offsets, m, n, k, E, 1, act, dtype, p, ws, None)
        return st, lib.moe_last_error_string()

    for kw, word in ((dict(act=5), b"activation"), (dict(act=-1), b"activation"),
                     (dict(dtype=3), b"dtype"), (dict(m=-1), b"negative"), (dict(k=-8), b"negative"),
                     (dict(E=2), b"num_offsets"), (dict(num_offsets=3, off=p, E=4), b"num_offsets"),
                     (dict(num_offsets=4, E=4), b"offsets"), (dict(a=None), b"NULL")):
        st, msg = fwd(**kw)
        assert st == 1 and word in msg, (kw, st, msg)
    assert fwd(m=0)[0] == 0
    ws = lib.moe_linear_workspace_bytes(4, 8, 8, 1, 1, 2)
    assert ws > 0 and lib.moe_linear_workspace_bytes(100000, 8, 8, 1, 1, 2) == 0
    st, msg = fwd(ws=ws - 1)
    assert st == 4 and b"workspace" in msg
    need = lib.moe_linear_bwd_workspace_bytes(300, 64, 3, 4, 2)
    assert need >= 300 * 64 * 2 + 3 * 64 * 4

    def bwd(z=p, b=p, off=None, num=0, E=1, act=4, ws=need, dtype=2, k=8):
        st = lib.moe_linear_bwd(p, p, b, z, p, p, p, off, num, 300, 64, k, E, 1, act, dtype, p, ws, None)
        return st, lib.moe_last_error_string()

    for kw, status, word in ((dict(ws=8), 4, b"workspace"), (dict(z=None), 1, b"preact"),
                             (dict(b=None), 1, b"NULL"), (dict(act=9), 1, b"activation"),
                             (dict(dtype=5), 1, b"dtype"), (dict(E=3), 1, b"num_offsets"),
                             (dict(k=-1), 1, b"negative")):
        st, msg = bwd(**kw)
        assert st == status and word in msg, (kw, st, msg)


def test_python_refusals():
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        M.linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        M.grouped_linear(x, torch.zeros(2, 5, 8), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        M.linear(x, torch.zeros(5, 9))
    with pytest.raises(ValueError):
        M.linear(x, torch.zeros(2, 5, 8))


@pytest.mark.gpu
def test_python_refusals_on_device(cuda_dev):
    def z(*s, dtype=torch.bfloat16):
        return torch.zeros(*s, device=cuda_dev, dtype=dtype)

    x, w, B, off = z(3, 8), z(5, 8), z(2, 5, 8), z(3, dtype=torch.int32)
    for f in (lambda: M.linear(x, w, activation="tanh"), lambda: M.linear(x, w, bias=z(4)),
              lambda: M.linear(x, w, bias=z(5, dtype=torch.float32)), lambda: M.linear(x, w.float()),
              lambda: M.linear(x, w, residual=z(3, 4)), lambda: M.linear(x, w, residual=z(1, 5)),
              lambda: M.linear(x, z(5, 8, dtype=torch.float16)),
              lambda: M.grouped_linear(x, B, z(5, dtype=torch.int32)),
              lambda: M.grouped_linear(x, B, off, bias=z(5)),
              lambda: M.grouped_linear(x, B, off, residual=z(3, 8)),
              lambda: M.grouped_linear(x, B, off, trans_b=False),
              lambda: M.grouped_linear(x, w, off)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        M.linear(x.double(), w.double())
