"""The activations of linear and their derivatives over the range of their argument, relative to
their own value: z is exact here (one product by 1), so only the activation and one rounding count."""
import math

import pytest
import torch

import moe_ops_b200 as M

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
ACTS = ["gelu", "gelu_tanh", "silu"]
A = math.sqrt(2 / math.pi)


def truth(z, act):
    """(act, act', magnitude of act's derivative's terms, argument of the exponential, factor beside the
    exponential in act') in 64 bits, with no difference of close numbers."""
    if act == "gelu":
        cdf, arg = torch.special.erfc(-z / math.sqrt(2)) / 2, z * z / 2
        slope, factor = z * torch.exp(-arg) / math.sqrt(2 * math.pi), z.abs()
    else:
        arg = z if act == "silu" else 2 * A * (z + 0.044715 * z ** 3)
        inner = 1 if act == "silu" else 2 * A * (1 + 3 * 0.044715 * z * z)
        e = torch.exp(-arg.abs())
        cdf = torch.where(arg < 0, e, torch.ones_like(e)) / (1 + e)
        slope, factor = z * inner * e / (1 + e) ** 2, z.abs() * inner
    return z * cdf, cdf + slope, cdf + slope.abs(), arg.abs(), factor


def bars(value, scale, arg, factor, dtype):
    """Half a step of the rounding to the dtype, and the fp32 evaluation: the exponential's argument
    passes at most 5 roundings of 2^-24 relative, which move it by 5 |arg| 2^-24 absolutely; 20 more
    roundings stand for the other operations and CUDA's functions (5 units of 2^-23 at most); the
    16-bit results' normal distribution is fitted to 2^-17.  Below the normal numbers half a
    subnormal step of the dtype; and an exponential below 2^-126 is a multiple of 2^-149, so off by up to
    that, which `factor` (|z| for act, for act' what stands beside the exponential: |z| times the
    argument's derivative, 278 at z = -10.7 for gelu_tanh) multiplies; products of it are rounded to
    multiples of 2^-149 again, hence twice that and one more."""
    half = torch.finfo(dtype).eps / 2
    rel = (5 * arg.clamp(max=160) + 20) * 2.0 ** -24 + (2.0 ** -17 if dtype != F32 else 0)
    tiny = torch.finfo(dtype).smallest_normal * half
    return half * value.abs() + rel * scale * (1 + half) + tiny + (factor + 1) * 2.0 ** -148


def grid(dev, dtype):
    """Every value of a 16-bit dtype (fp32: a sample) with 2^-10 <= |z| <= 128, and 0."""
    if dtype == F32:
        g = torch.Generator(device=dev).manual_seed(1)
        z = torch.exp2(torch.rand(20000, device=dev, generator=g) * 17 - 10)
    else:
        bits = torch.arange(0, 1 << 15, device=dev, dtype=torch.int32).to(torch.int16)
        z = bits.view(dtype).float()
        z = z[(z >= 2.0 ** -10) & (z <= 128)]
    return torch.cat([z, -z, z.new_zeros(1)]).to(dtype)


def check(got, want, tol, z, what):
    err = (got.double() - want).abs()
    worst = (err / tol).argmax()
    assert (err <= tol).all(), (what, z[worst].item(), got[worst].item(), want[worst].item(),
                                (err / tol)[worst].item())


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("k", [8, 7])  # 7: rows of no 16-byte multiple
def test_many_rows(cuda_dev, k, dtype, act):
    z = grid(cuda_dev, dtype)
    x = torch.zeros(z.numel(), k, device=cuda_dev, dtype=dtype)
    x[:, 0] = z
    w = torch.zeros(8, k, device=cuda_dev, dtype=dtype)
    w[0, 0] = 1
    x.requires_grad_(True)
    y = M.linear(x, w, activation=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    zd = z.double()
    want, slope, mag, arg, factor = truth(zd, act)
    check(y.detach()[:, 0], want, bars(want, want.abs(), arg, zd.abs(), dtype), z, act)
    check(dx[:, 0], slope, bars(slope, mag, arg, factor, dtype), z, act + "'")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("m", [1, 20])
def test_few_rows(cuda_dev, m, dtype, act):
    z = grid(cuda_dev, dtype)
    z = z[:z.numel() // 8 * 8]
    w = torch.zeros(z.numel(), 8, device=cuda_dev, dtype=dtype)
    w[:, 0] = z
    x = torch.zeros(m, 8, device=cuda_dev, dtype=dtype)
    x[:, 0] = 1
    y = M.linear(x, w, activation=act)
    zd = z.double()
    want, _, _, arg, _ = truth(zd, act)
    for r in (0, m - 1):
        check(y[r], want, bars(want, want.abs(), arg, zd.abs(), dtype), z, act)


@pytest.mark.parametrize("act", ["none", "relu"] + ACTS)
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("m", [1, 130])
def test_infinities_nan_and_largest_values(cuda_dev, m, dtype, act):
    """Through the bias.  Infinite z: the limit for +, for - as z * 0 (NaN) except for relu; the
    derivative is its limit."""
    big = torch.finfo(dtype).max
    b = torch.tensor([math.inf, -math.inf, math.nan, big, -big, 1.0, 0.0, -1.0], device=cuda_dev, dtype=dtype)
    b.requires_grad_(True)
    x, w = (torch.zeros(s, 8, device=cuda_dev, dtype=dtype) for s in (m, 8))
    y = M.linear(x, w, bias=b, activation=act)
    dy = torch.zeros_like(y)
    dy[0] = 1
    db, = torch.autograd.grad(y, b, dy)
    lo = -math.inf if act == "none" else 0.0 if act == "relu" else math.nan
    want = torch.tensor([math.inf, lo, math.nan, big, -big if act == "none" else 0.0], device=cuda_dev)
    for r in (0, m - 1):
        got = y.detach()[r, :5].float()
        assert torch.equal(got.isnan(), want.isnan()), got
        assert torch.equal(got.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0),
                           want.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0)), got
    left = 1.0 if act == "none" else 0.0
    slope = torch.tensor([1.0, left, 1.0 if act == "none" else math.nan, 1.0, left], device=cuda_dev)
    got = db[:5].float()
    assert torch.equal(got.isnan(), slope.isnan()) and torch.equal(got.nan_to_num(7.0), slope.nan_to_num(7.0)), got
    assert torch.isfinite(y[:, 5:]).all() and torch.isfinite(db[5:]).all()
