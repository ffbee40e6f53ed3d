"""What one block stores and another reads inside a launch: h between the two phases of the
few-token layer, and the parts of a cut product.  Every workspace holds NaN before the call, so
a value read before it was written shows."""
import math

import pytest
import torch

import moe_ops_b200 as M
from moe_ops_b200 import _lib

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
CODE = {BF: 2, FP: 1}


def poison(dev, nbytes):
    """Leaves a block of that size filled with NaN patterns for the next allocation."""
    if nbytes:
        torch.empty(nbytes, device=dev, dtype=torch.uint8).fill_(0xFF)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T,d,E,K,H", [(1, 1024, 16, 2, 4096), (13, 512, 24, 4, 1096), (64, 256, 8, 3, 520)])
def test_layer(cuda_dev, T, d, E, K, H, dtype):
    g = torch.Generator(device=cuda_dev).manual_seed(T)
    rnd = lambda *s: torch.randn(*s, device=cuda_dev, generator=g)  # noqa: E731
    x, wr = rnd(T, d).to(dtype), rnd(E, d).div(math.sqrt(d)).to(dtype)
    wg, wu = (rnd(E, H, d).div(math.sqrt(d)).to(dtype) for _ in range(2))
    wd = rnd(E, d, H).div(math.sqrt(H)).to(dtype)
    logits = x.double() @ wr.double().t()
    top = torch.sort(logits, dim=1, descending=True, stable=True)
    p, idx = torch.softmax(top.values[:, :K], 1), top.indices[:, :K]
    X = x.double()
    want, mag = torch.zeros_like(X), torch.zeros_like(X)
    for e in range(E):
        t, k = torch.nonzero(idx == e, as_tuple=True)
        gate = X[t] @ wg[e].double().t()
        h = gate * torch.sigmoid(gate) * (X[t] @ wu[e].double().t())
        want.index_add_(0, t, h @ wd[e].double().t() * p[t, k][:, None])
        mag.index_add_(0, t, h.abs() @ wd[e].double().abs().t() * p[t, k][:, None])
    # h and y are rounded to the dtype (half a step each; fp16 below 2^-14 by 2^-25); fp32 sums of
    # n terms, at most n / 32 + 10 roundings deep, the magnitudes of gate and up about sqrt(d)
    # times their values.
    half = torch.finfo(dtype).eps / 2
    tol = half * (want.abs() + mag) + 4 * (max(d, H) / 32 + 10) * 2.0 ** -24 * (1 + math.sqrt(d)) * mag
    tol = tol + 2.0 ** -24 * math.sqrt(H)
    ws = _lib.load().moe_few_tokens_workspace_bytes(T, d, H, E, K, CODE[dtype])
    first = None
    for _ in range(40):
        poison(cuda_dev, ws)
        y = M.moe_few_tokens(x, wr, wg, wu, wd, K)
        first = y if first is None else first
        assert torch.equal(y, first)
    assert ((first.double() - want).abs() <= tol).all()
    assert _lib.read_device_error() == 0


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,k,n", [(1, 8192, 264), (37, 7168, 1000), (130, 4096, 520)])
def test_cut_product(cuda_dev, m, k, n, dtype):
    g = torch.Generator(device=cuda_dev).manual_seed(m)
    x = torch.randn(m, k, device=cuda_dev, generator=g).to(dtype)
    w = torch.randn(n, k, device=cuda_dev, generator=g).div(math.sqrt(k)).to(dtype)
    ws = _lib.load().moe_linear_workspace_bytes(m, n, k, 1, 1, CODE[dtype])
    assert ws > m * n * 4, "the contraction is not cut"
    want = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    first = None
    for _ in range(40):
        poison(cuda_dev, ws)
        y = M.linear(x, w)
        first = y if first is None else first
        assert torch.equal(y, first)
    # one rounding to the dtype, and fp32 sums: k roundings at most, whatever the order
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (k + 2) * 2.0 ** -24 * mag + 2.0 ** -25
    assert ((first.double() - want).abs() <= tol).all()
    assert _lib.read_device_error() == 0
