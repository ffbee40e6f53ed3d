"""linear / grouped_linear for a few rows over large weights that the tensor cores cannot read in
place: fp32, rows of no 16-byte multiple, weights off a boundary."""
import math

import pytest
import torch

import moe_ops_b200 as M
import test_linear_gpu

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def make(dev, m, k, n, dtype, E=0, trans_b=True):
    g = torch.Generator(device=dev).manual_seed(m + k)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    lead = (E,) if E else ()
    w = rnd(*lead, *((n, k) if trans_b else (k, n))).div(math.sqrt(k)).to(dtype)
    return rnd(m, k).to(dtype), w, rnd(*lead, n).to(dtype)


def check(y, x, w, b, dtype):
    """y = x w^T + b in 64 bits; one rounding to the dtype and k + 1 of fp32 in any order."""
    want = x.double() @ w.double().t() + b.double()
    mag = x.double().abs() @ w.double().abs().t() + b.double().abs()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (x.shape[1] + 2) * 2.0 ** -24 * mag
    assert ((y.double() - want).abs() <= tol).all()


def peak(f):
    """Bytes that a call holds at its peak beside what was there before."""
    f()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    f()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m", [1, 3, 8, 21])
@pytest.mark.parametrize("k,n", [(7168, 5504), (4097, 4099), (2048, 8193)])
def test_values(cuda_dev, m, k, n, dtype):
    x, w, b = make(cuda_dev, m, k, n, dtype)
    check(M.linear(x, w, bias=b), x, w, b, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("m", [2, 40, 300])
def test_grouped_values(cuda_dev, m, trans_b, dtype):
    E, k, n = 9, 1001, 1203
    x, w, b = make(cuda_dev, m, k, n, dtype, E, trans_b)
    cuts = torch.sort(torch.randint(0, m + 1, (E - 1,), generator=torch.Generator().manual_seed(m))).values
    ends = [0] + cuts.tolist() + [m]
    off = torch.tensor(ends, device=cuda_dev, dtype=torch.int32)
    y = M.grouped_linear(x, w, off, bias=b, trans_b=trans_b)
    for e in range(E):
        s = slice(ends[e], ends[e + 1])
        check(y[s], x[s], w[e] if trans_b else w[e].t(), b[e], dtype)


def test_no_copy_of_weights_that_few_rows_read_once(cuda_dev):
    x, w, b = make(cuda_dev, 1, 4097, 4099, BF)
    assert peak(lambda: M.linear(x, w, bias=b)) < w.numel()  # half the weight's bytes
    flat = torch.empty(4096 * 4096 + 1, device=cuda_dev, dtype=BF)
    w = flat[1:].view(4096, 4096).normal_(generator=torch.Generator(device=cuda_dev).manual_seed(1)).div_(64)
    x = torch.ones(2, 4096, device=cuda_dev, dtype=BF)
    assert peak(lambda: M.linear(x, w)) < w.numel()
    check(M.linear(x, w), x, w, torch.zeros(4096, device=cuda_dev), BF)
    E, m = 32, 20
    x, w, b = make(cuda_dev, m, 1001, 1003, BF, E)
    off = torch.tensor([m] * E, device=cuda_dev, dtype=torch.int32)
    assert peak(lambda: M.grouped_linear(x, w, off, bias=b)) < w.numel()
    check(M.grouped_linear(x, w, off, bias=b), x, w[0], b[0], BF)


@pytest.mark.parametrize("dtype", [BF, torch.float16])
@pytest.mark.parametrize("m,k,n,E", [(3, 1563, 4951, 0), (4, 2001, 2104, 0), (6, 985, 4908, 2), (47, 3898, 187, 13)])
def test_gradients_of_odd_rows(cuda_dev, m, k, n, E, dtype):
    """Rows too few for a copy of the weights in the forward: the same values with and without gradients,
    and the formula's gradients."""
    x, w, b, r, dy = test_linear_gpu.make(cuda_dev, m, k, n, dtype, m + k, E=E)
    g = torch.Generator().manual_seed(m)
    cuts = torch.sort(torch.randint(0, m + 1, (max(0, E - 1),), generator=g)).values.tolist()
    off = torch.tensor([0] + cuts + [m], device=cuda_dev, dtype=torch.int32) if E else None
    for act in ("none", "silu"):
        test_linear_gpu.run_case(x, w, b, r, dy, act, dtype, offsets=off)
