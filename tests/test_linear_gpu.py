"""linear / grouped_linear against a 64-bit evaluation of their definition, values and
gradients."""
import math

import pytest
import torch
import torch.nn.functional as F

import moe_ops_b200 as M
from moe_ops_b200 import _lib

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
ACT64 = {"none": lambda z: z, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu,
         "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}
MAX_SLOPE, MAX_CURVE = 1.14, 1.1  # |act'| and |act''| of every activation (relu's kink aside)


def ends_of(offsets, E):
    o = offsets.tolist()
    return o if len(o) == E + 1 else [0] + o


def truth(x, w, b, r, dy, act, offsets=None, trans_b=True):
    """Values and gradients in 64 bits, and the magnitudes that rounding errors scale with."""
    leaf = [None if t is None else t.double().requires_grad_(True) for t in (x, w, b, r)]
    X, W, B, R = leaf
    f = ACT64[act]
    if offsets is None:
        z = X @ W.t()
        z = z if B is None else z + B
        live = torch.ones(x.shape[0], dtype=torch.bool, device=x.device)
    else:
        E = w.shape[0]
        ends = ends_of(offsets, E)
        parts = []
        for e in range(E):
            ze = X[ends[e]:ends[e + 1]] @ (W[e].t() if trans_b else W[e])
            parts.append(ze if B is None else ze + B[e])
        n_tail = x.shape[0] - ends[-1]
        n = w.shape[1 if trans_b else 2]
        z = torch.cat(parts + [X.new_zeros(n_tail, n)])
        live = torch.arange(x.shape[0], device=x.device) < ends[-1]
    y = torch.where(live[:, None], f(z), torch.zeros_like(z))
    y = y if R is None else y + R
    grads = torch.autograd.grad(y, [t for t in leaf if t is not None], dy.double(), allow_unused=True)
    zd = z.detach().requires_grad_(True)
    slope = torch.autograd.grad(f(zd).sum(), zd)[0]
    it = iter(grads)
    g = [None if t is None else next(it) for t in leaf]
    return y.detach(), g, z.detach(), slope * live[:, None]


def abs_products(x, w, dzmag, offsets, trans_b):
    """|dz| . |W| and |dz|^T . |x| per group: what errors in dz and in the sums scale with."""
    X, W = x.double().abs(), w.double().abs()
    if offsets is None:
        return dzmag @ W, dzmag.t() @ X
    E = w.shape[0]
    ends = ends_of(offsets, E)
    dx, dw = torch.zeros_like(X), torch.zeros_like(W)
    for e in range(E):
        s = slice(ends[e], ends[e + 1])
        We = W[e] if trans_b else W[e].t()
        dx[s] = dzmag[s] @ We
        d = dzmag[s].t() @ X[s]
        dw[e] = d if trans_b else d.t()
    return dx, dw


def close(got, want, tol, what):
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{what}: {((got.double() - want).abs() / tol).max().item():.3g} of the tolerance"


def run_case(x, w, b, r, dy, act, dtype, offsets=None, trans_b=True, call=None):
    leaf = [None if t is None else t.clone().requires_grad_(True) for t in (x, w, b, r)]
    if offsets is None:
        y = M.linear(leaf[0], leaf[1], bias=leaf[2], activation=act, residual=leaf[3])
        y0 = M.linear(x, w, bias=b, activation=act, residual=r)
    else:
        y = M.grouped_linear(leaf[0], leaf[1], offsets, bias=leaf[2], activation=act,
                             residual=leaf[3], trans_b=trans_b)
        y0 = M.grouped_linear(x, w, offsets, bias=b, activation=act, residual=r, trans_b=trans_b)
    grads = torch.autograd.grad(y, [t for t in leaf if t is not None], dy)
    again = torch.autograd.grad(
        M.linear(leaf[0], leaf[1], bias=leaf[2], activation=act, residual=leaf[3]) if offsets is None
        else M.grouped_linear(leaf[0], leaf[1], offsets, bias=leaf[2], activation=act,
                              residual=leaf[3], trans_b=trans_b),
        [t for t in leaf if t is not None], dy)
    assert torch.equal(y.detach(), y0), "the forward differs with and without gradients"
    assert all(torch.equal(a, c) for a, c in zip(grads, again)), "two backward passes differ"

    y64, g64, z, slope = truth(x, w, b, r, dy, act, offsets, trans_b)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half * 2  # half a subnormal step
    K, m = x.shape[1], x.shape[0]
    # fp32 sums of n products: off by at most n * 2^-24 of the sum of their magnitudes in any
    # order; the act functions add a few steps of fp32 relative to |z|.
    fp = 2.0 ** -24
    if offsets is None:
        zmag = x.double().abs() @ w.double().abs().t()
    else:
        zmag = torch.zeros_like(z)
        ends = ends_of(offsets, w.shape[0])
        for e in range(w.shape[0]):
            s = slice(ends[e], ends[e + 1])
            We = w[e].double().abs()
            zmag[s] = x[s].double().abs() @ (We.t() if trans_b else We)
    zerr = fp * (K + 2) * zmag + 8 * fp * z.abs() + fp * 4
    rmag = 0 if r is None else r.double().abs()
    close(y, y64, half * y64.abs() + MAX_SLOPE * zerr + 2 * fp * rmag + tiny, "y")
    # dz: the stored z is off by half a step of it, which moves act' by |act''| times that; then
    # dz is rounded once.  relu's slope changes only where |z| is within its error of 0.
    d = dy.double().abs()
    if act == "none":
        dzerr = torch.zeros_like(d)
    elif act == "relu":
        dzerr = d * (z.abs() <= zerr + tiny) + half * d * slope.abs()
    else:
        dzerr = d * (MAX_CURVE * (half * z.abs() + zerr + tiny) + half * slope.abs() + 8 * fp) + tiny
    dzmag = d * slope.abs() + dzerr
    ex, ew = abs_products(x, w, dzerr, offsets, trans_b)
    mx, mw = abs_products(x, w, dzmag, offsets, trans_b)
    N = dy.shape[1]
    got = iter(grads)
    gx, gw = next(got), next(got)
    close(gx, g64[0], half * g64[0].abs() + ex + fp * (N + 2) * mx + tiny, "dx")
    close(gw, g64[1], half * g64[1].abs() + ew + fp * (m + 2) * mw + tiny, "dw")
    if b is not None:
        gb = next(got)
        if offsets is None:
            eb, mb = dzerr.sum(0), dzmag.sum(0)
        else:
            ends = ends_of(offsets, w.shape[0])
            eb = torch.stack([dzerr[ends[e]:ends[e + 1]].sum(0) for e in range(w.shape[0])])
            mb = torch.stack([dzmag[ends[e]:ends[e + 1]].sum(0) for e in range(w.shape[0])])
        close(gb, g64[2], half * g64[2].abs() + eb + fp * (m + 2) * mb + tiny, "db")
    if r is not None:
        assert torch.equal(next(got), dy)


def make(dev, m, k, n, dtype, seed, E=0, trans_b=True, bias=True, residual=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    lead = (E,) if E else ()
    shape = lead + ((n, k) if trans_b else (k, n))
    return (rnd(m, k).to(dtype), rnd(*shape).div(math.sqrt(max(1, k))).to(dtype),
            rnd(*lead, n).to(dtype) if bias else None, rnd(m, n).to(dtype) if residual else None,
            rnd(m, n).to(dtype))


DENSE = [  # m, k, n
    (1, 64, 8), (1, 512, 1000), (2, 72, 264), (16, 256, 136), (17, 1024, 520), (64, 2048, 256),
    (65, 200, 328), (130, 136, 64), (257, 320, 776), (1025, 128, 512), (2100, 192, 320),
]
ODD = [(1, 1, 1), (1, 469, 160), (5, 263, 531), (33, 257, 130), (70, 64, 63), (129, 7, 256)]


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("m,k,n", DENSE + ODD)
def test_dense(cuda_dev, m, k, n, dtype):
    act = ["gelu", "silu", "none", "relu", "gelu_tanh"][(m + k + n) % 5]
    x, w, b, r, dy = make(cuda_dev, m, k, n, dtype, m + k)
    run_case(x, w, b, r, dy, act, dtype)


@pytest.mark.parametrize("act", list(ACT64))
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m", [3, 150])
def test_activations_and_optional_inputs(cuda_dev, act, bias, residual, m):
    x, w, b, r, dy = make(cuda_dev, m, 128, 200, BF, 7, bias=bias, residual=residual)
    run_case(x, w, b, r, dy, act, BF)


GROUPED = [  # sizes, tail rows, k, n
    ([5, 0, 17, 300, 129, 128, 1, 0, 64, 96], 0, 192, 200),
    ([0, 0, 3], 5, 64, 72),
    ([1] * 40, 0, 256, 264),
    ([0] * 7, 9, 64, 64),
    ([1200, 1500], 33, 128, 256),
    ([2, 0, 1, 4], 0, 33, 19),
    ([70, 0, 9], 3, 130, 41),
]


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("sizes,tail,k,n", GROUPED)
def test_grouped(cuda_dev, sizes, tail, k, n, trans_b, dtype):
    E, m = len(sizes), sum(sizes) + tail
    act = ["silu", "gelu", "relu", "none", "gelu_tanh"][(E + k) % 5]
    x, w, b, r, dy = make(cuda_dev, m, k, n, dtype, m + k, E=E, trans_b=trans_b)
    off = torch.tensor([0] + sizes, device=cuda_dev).cumsum(0).to(torch.int32)
    run_case(x, w, b, r, dy, act, dtype, offsets=off, trans_b=trans_b)
    ends_only = M.grouped_linear(x, w, off[1:], bias=b, activation=act, residual=r, trans_b=trans_b)
    assert torch.equal(ends_only, M.grouped_linear(x, w, off, bias=b, activation=act, residual=r,
                                                   trans_b=trans_b))


def test_poison_behind_the_last_group_stays_out(cuda_dev):
    """NaN rows behind the last offset reach no other row and no gradient."""
    x, w, b, r, dy = make(cuda_dev, 40, 64, 72, BF, 1, E=3)
    off = torch.tensor([0, 10, 10, 25], device=cuda_dev, dtype=torch.int32)
    x[25:] = math.nan
    dy[25:] = math.nan
    leaf = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = M.grouped_linear(leaf[0], leaf[1], off, bias=leaf[2], activation="silu")
    gx, gw, gb = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(y[25:], torch.zeros_like(y[25:]))
    assert torch.equal(gx[25:], torch.zeros_like(gx[25:]))
    assert all(torch.isfinite(t).all() for t in (y, gx, gw, gb))
    assert torch.equal(gw[1], torch.zeros_like(gw[1])) and torch.equal(gb[1], torch.zeros_like(gb[1]))


def test_gradient_against_differences(cuda_dev):
    """fp32, central differences of the operator itself along random directions."""
    x, w, b, r, dy = make(cuda_dev, 9, 40, 24, F32, 2)
    for act in ACT64:
        leaf = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        f = lambda a: (M.linear(a[0], a[1], bias=a[2], activation=act,  # noqa: E731
                                residual=a[3]).double() * dy.double()).sum()
        grads = torch.autograd.grad(M.linear(leaf[0], leaf[1], bias=leaf[2], activation=act,
                                             residual=leaf[3]), leaf, dy)
        h = 2.0 ** -7
        for i in range(4):
            v = torch.randn_like(leaf[i])
            v /= v.norm()
            hi = [t.detach() + (h * v if j == i else 0) for j, t in enumerate(leaf)]
            lo = [t.detach() - (h * v if j == i else 0) for j, t in enumerate(leaf)]
            want = ((f(hi) - f(lo)) / (2 * h)).item()
            got = (grads[i].double() * v.double()).sum().item()
            # third derivatives (h^2 / 6 of them) and the fp32 rounding of 216 outputs of size
            # ~3 over 2h
            scale = dy.double().abs().sum().item()
            tol = scale * (2 * h * h) + 216 * 3 * 2.0 ** -24 / h
            if act == "relu":
                # z is linear along the direction, z +- h c: the quotient of relu is s * c with
                # s in [0, 1], the gradient 0 * c or 1 * c; they are equal unless the kink lies
                # inside the step, |z| <= h |c|, and then differ by at most |c|.
                z = [a[0].double() @ a[1].double().t() + a[2].double() for a in (hi, lo)]
                c, mid = (z[0] - z[1]) / (2 * h), (z[0] + z[1]) / 2
                tol += (dy.double() * c).abs()[mid.abs() <= h * c.abs() + 1e-5].sum().item()
            assert abs(got - want) <= tol, (act, i, got, want, tol)


def test_shapes_strides_and_empty(cuda_dev):
    x, w, b, r, dy = make(cuda_dev, 24, 64, 40, BF, 3)
    want = M.linear(x, w, bias=b, activation="gelu", residual=r)
    y = M.linear(x.view(2, 3, 4, 64), w, bias=b, activation="gelu", residual=r.view(2, 3, 4, 40))
    assert y.shape == (2, 3, 4, 40) and torch.equal(y.view(24, 40), want)
    assert torch.equal(M.linear(x[0], w, bias=b, activation="gelu", residual=r[0]),
                       M.linear(x[:1], w, bias=b, activation="gelu", residual=r[:1])[0])
    xs = x.t().contiguous().t()
    ws = w.t().contiguous().t()
    wide = torch.zeros(24, 80, device=cuda_dev, dtype=BF)
    wide[:, ::2] = r
    assert torch.equal(M.linear(xs, ws, bias=b, activation="gelu", residual=wide[:, ::2]), want)
    # off a 16-byte boundary: the CUDA-core path, same definition
    flat = torch.empty(24 * 64 + 1, device=cuda_dev, dtype=BF)
    xo = flat[1:].view(24, 64)
    xo.copy_(x)
    run_case(xo, w, b, r, dy, "gelu", BF)
    assert M.linear(x[:0], w, bias=b).shape == (0, 40)
    assert M.linear(x, w[:0]).shape == (24, 0)
    y = M.linear(x[:, :0], w[:, :0], bias=b, activation="silu", residual=r)
    assert torch.allclose(y.float(), (F.silu(b.float()) + r.float()).to(BF).float(), rtol=2 ** -7)
    e = x[:0].clone().requires_grad_(True)
    we = w.clone().requires_grad_(True)
    be = b.clone().requires_grad_(True)
    M.linear(e, we, bias=be, activation="silu").sum().backward()
    assert e.grad.shape == (0, 64)
    assert torch.equal(we.grad, torch.zeros_like(w)) and torch.equal(be.grad, torch.zeros_like(b))


@pytest.mark.parametrize("E,trans_b", [(0, True), (3, True), (3, False)])
def test_large_unaligned_products_are_padded(cuda_dev, E, trans_b):
    """16-bit rows that are no 16-byte multiples, large enough for the padded path."""
    m, k, n = 140, 401, 333
    x, w, b, r, dy = make(cuda_dev, m, k, n, BF, 8, E=E, trans_b=trans_b)
    off = torch.tensor([0, 50, 50, 131], device=cuda_dev, dtype=torch.int32) if E else None
    run_case(x, w, b, r, dy, "silu", BF, offsets=off, trans_b=trans_b)


def test_large_products_off_a_boundary(cuda_dev):
    m, k, n = 140, 400, 336
    x, w, b, r, dy = make(cuda_dev, m, k, n, FP, 9)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, device=cuda_dev, dtype=t.dtype)
        v = flat[1:].view(t.shape)
        v.copy_(t)
        return v

    got = M.linear(shifted(x), shifted(w), bias=shifted(b), activation="gelu", residual=shifted(r))
    assert torch.equal(got, M.linear(x, w, bias=b, activation="gelu", residual=r))


def test_no_experts_and_no_rows(cuda_dev):
    x, w, b, r, dy = make(cuda_dev, 6, 64, 72, BF, 10, E=2)
    none = torch.zeros(1, device=cuda_dev, dtype=torch.int32)
    leaf = x.clone().requires_grad_(True)
    y = M.grouped_linear(leaf, w[:0], none, bias=b[:0], activation="silu", residual=r)
    assert torch.equal(y.detach(), r)
    y.sum().backward()
    assert torch.equal(leaf.grad, torch.zeros_like(x))
    off = torch.zeros(3, device=cuda_dev, dtype=torch.int32)
    leaf = [t.clone().requires_grad_(True) for t in (w, b)]
    y = M.grouped_linear(x[:0], leaf[0], off, bias=leaf[1], activation="silu")
    y.sum().backward()
    assert y.shape == (0, 72) and all(torch.equal(t.grad, torch.zeros_like(t)) for t in leaf)


def test_a_cut_few_row_product(cuda_dev):
    """Rows, columns and depth for which the contraction is cut: the parts' order is fixed."""
    for m, k, n in ((37, 4160, 256), (64, 8192, 1000), (130, 4096, 520), (16, 4160, 8)):
        x, w, b, r, dy = make(cuda_dev, m, k, n, BF, m)
        run_case(x, w, b, r, dy, "silu", BF)


def test_partial_gradients(cuda_dev):
    """Each subset of the inputs that require a gradient gives the same gradients."""
    x, w, b, r, dy = make(cuda_dev, 140, 72, 96, BF, 4)
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(M.linear(full[0], full[1], bias=full[2], activation="silu",
                                        residual=full[3]), full, dy)
    for mask in range(1, 16):
        leaf = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b, r))]
        need = [t for t in leaf if t.requires_grad]
        got = torch.autograd.grad(M.linear(leaf[0], leaf[1], bias=leaf[2], activation="silu",
                                           residual=leaf[3]), need, dy)
        assert all(torch.equal(a, want[i]) for a, i in
                   zip(got, [i for i in range(4) if mask >> i & 1]))


def test_shared_and_strided_gradients(cuda_dev):
    """One bias leaf used by two calls, an expanded output gradient, a broadcast residual."""
    x, w, b, r, dy = make(cuda_dev, 12, 64, 64, F32, 5)
    bl = b.clone().requires_grad_(True)
    row = r[:1].clone().requires_grad_(True)
    y = M.linear(M.linear(x, w, bias=bl, activation="silu"), w, bias=bl,
                 residual=row.expand(12, 64))
    y.sum().backward()  # the gradient arrives expanded (stride 0)
    bd, rd = b.double().requires_grad_(True), r[:1].double().requires_grad_(True)
    yd = F.silu(x.double() @ w.double().t() + bd) @ w.double().t() + bd + rd
    yd.sum().backward()
    assert torch.allclose(bl.grad.double(), bd.grad, rtol=1e-5, atol=1e-4)
    assert torch.equal(row.grad.double(), rd.grad)


def test_side_stream_and_graph(cuda_dev):
    x, w, b, r, dy = make(cuda_dev, 48, 256, 384, BF, 6)
    want = M.linear(x, w, bias=b, activation="silu", residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = M.linear(x, w, bias=b, activation="silu", residual=r)
    s.synchronize()
    assert torch.equal(side, want)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    leaf = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ref = torch.autograd.grad(M.linear(leaf[0], leaf[1], bias=leaf[2], activation="silu"), leaf, dy)
    torch.cuda.synchronize()
    with torch.cuda.graph(g1):
        y1 = M.linear(x, w, bias=b, activation="silu", residual=r)
    with torch.cuda.graph(g2):
        y2 = M.linear(leaf[0], leaf[1], bias=leaf[2], activation="silu")
        grads = torch.autograd.grad(y2, leaf, dy)
    for _ in range(3):
        with torch.cuda.stream(s):
            g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y1, want)
        assert all(torch.equal(a, c) for a, c in zip(grads, ref))
    assert _lib.read_device_error() == 0
