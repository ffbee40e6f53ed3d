"""The few-token MoE layer against a 64-bit evaluation of its definition."""
import math

import pytest
import torch

import moe_ops_b200 as M
from moe_ops_b200 import _lib

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def make(dev, T, d, E, H, dtype, seed=0, scale=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    scale = scale or 1.0 / math.sqrt(d)
    return dict(x=rnd(T, d).to(dtype), w_router=rnd(E, d).mul(scale).to(dtype),
                w_gate=rnd(E, H, d).mul(scale).to(dtype), w_up=rnd(E, H, d).mul(scale).to(dtype),
                w_down=rnd(E, d, H).mul(1.0 / math.sqrt(H)).to(dtype))


def route64(p, K, bias=None):
    logits = p["x"].double() @ p["w_router"].double().t()
    if bias is not None:
        logits = logits + bias.double()
    top = torch.sort(logits, dim=1, descending=True, stable=True)
    v, idx = top.values[:, :K], top.indices[:, :K]
    live = v > -math.inf
    ex = torch.where(live, torch.exp(v - v[:, :1]), torch.zeros_like(v))
    ex = torch.where(live.any(1, keepdim=True), ex, torch.zeros_like(ex))
    w = ex / ex.sum(1, keepdim=True).clamp(min=1e-300)
    return w, idx


def layer64(p, w, idx):
    """(y, sum_k |p| * |h| . |Wd|) in 64 bits: the second bounds what rounding h may change."""
    x = p["x"].double()
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    E = p["w_gate"].shape[0]
    for e in sorted(set(idx.flatten().tolist())):
        if not 0 <= e < E:
            continue
        t, k = torch.nonzero(idx == e, as_tuple=True)
        g = x[t] @ p["w_gate"][e].double().t()
        u = x[t] @ p["w_up"][e].double().t()
        h = g * torch.sigmoid(g) * u
        wk = w[t, k][:, None].double()
        live = wk[:, 0] != 0
        t, wk, h = t[live], wk[live], h[live]
        y.index_add_(0, t, (h @ p["w_down"][e].double().t()) * wk)
        mag.index_add_(0, t, (h.abs() @ p["w_down"][e].double().abs().t()) * wk.abs())
    return y, mag


def check(y, y64, mag, dtype, d, H):
    # Half a step for each rounding to the dtype: h (weighted by the sum of its magnitudes) and
    # y.  The products' fp32 sums: a sum of n terms in any tree of depth >= log2(n) and at most
    # n/32 serial steps per lane is off by at most (n/32 + 10) * 2^-24 of its magnitude sum; the
    # magnitude sums of gate and up exceed their values by about sqrt(d), which
    # 1 + sqrt(d) absorbs for these normal inputs with a factor of 4 to spare.
    half = torch.finfo(dtype).eps / 2
    sums = (max(d, H) / 32 + 10) * 2.0 ** -24
    tol = half * (y64.abs() + mag) + 4 * sums * (1 + math.sqrt(d)) * mag
    if dtype == FP:
        tol = tol + 2.0 ** -24 * math.sqrt(H)  # subnormal h and y
    bad = (y.double() - y64).abs() > tol
    assert not bad.any(), ((y.double() - y64).abs() / tol).max().item()


CASES = [  # T, d, E, K, H
    (1, 512, 8, 2, 1024),
    (1, 64, 1, 1, 8),
    (3, 200, 5, 5, 136),
    (16, 1024, 64, 2, 512),
    (17, 768, 16, 4, 1000),
    (33, 256, 40, 8, 264),
    (64, 512, 8, 2, 768),
    (65, 320, 4, 1, 640),
    (128, 192, 3, 3, 200),
    (128, 128, 300, 16, 72),
]
ODD = [(1, 7, 3, 2, 5), (5, 129, 9, 3, 67), (19, 250, 1000, 4, 33)]


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("T,d,E,K,H", CASES + ODD)
def test_whole_layer(cuda_dev, T, d, E, K, H, dtype):
    p = make(cuda_dev, T, d, E, H, dtype, seed=T * 7 + E)
    y = M.moe_few_tokens(**p, top_k=K)
    w, idx = route64(p, K)
    y64, mag = layer64(p, w, idx)
    assert y.shape == (T, d) and y.dtype == dtype
    check(y, y64, mag, dtype, d, H)
    again = M.moe_few_tokens(**p, top_k=K)
    assert torch.equal(y, again), "two runs differ"


@pytest.mark.parametrize("dtype", [BF, F32])
def test_router_bias_masks_and_empty_rows(cuda_dev, dtype):
    T, d, E, K, H = 9, 256, 12, 4, 128
    p = make(cuda_dev, T, d, E, H, dtype, seed=3)
    bias = torch.randn(E, device=cuda_dev)
    bias[2] = -math.inf
    w, idx = route64(p, K, bias)
    y64, mag = layer64(p, w, idx)
    check(M.moe_few_tokens(**p, top_k=K, router_bias=bias), y64, mag, dtype, d, H)
    # fewer unmasked experts than K: the masked slots weigh nothing, and masked experts'
    # weights are not read (NaN there must not show)
    bias[:] = -math.inf
    bias[5] = 0.25
    q = dict(p)
    for n in ("w_gate", "w_up", "w_down"):
        q[n] = p[n].clone()
        q[n][torch.arange(E, device=cuda_dev) != 5] = math.nan
    w, idx = route64(p, K, bias)
    y64, mag = layer64(p, w, idx)
    check(M.moe_few_tokens(**q, top_k=K, router_bias=bias), y64, mag, dtype, d, H)
    # every expert masked: zeros
    bias[:] = -math.inf
    assert torch.equal(M.moe_few_tokens(**q, top_k=K, router_bias=bias), torch.zeros_like(p["x"]))
    # the lowest finite value is a logit like any other
    low = torch.full((E,), torch.finfo(F32).min, device=cuda_dev)
    y = M.moe_few_tokens(**p, top_k=K, router_bias=low)
    assert torch.isfinite(y).all() and (y != 0).any()


def test_ties_go_to_the_lower_expert(cuda_dev):
    T, d, E, K, H = 4, 64, 37, 3, 64
    p = make(cuda_dev, T, d, E, H, F32, seed=4)
    p["w_router"].zero_()
    bias = torch.zeros(E, device=cuda_dev)
    bias[[3, 11, 20, 30]] = 1.0
    w = torch.full((T, K), 1 / 3, device=cuda_dev, dtype=torch.float64)
    idx = torch.tensor([3, 11, 20], device=cuda_dev).expand(T, K)
    y64, mag = layer64(p, w, idx)
    check(M.moe_few_tokens(**p, top_k=K, router_bias=bias), y64, mag, F32, d, H)


def test_nan_and_inf_tokens_stay_in_their_rows(cuda_dev):
    T, d, E, K, H = 6, 128, 8, 2, 128
    p = make(cuda_dev, T, d, E, H, BF, seed=5)
    clean = M.moe_few_tokens(**p, top_k=K)
    q = dict(p, x=p["x"].clone())
    q["x"][2, 5] = math.nan
    q["x"][4, 0] = math.inf
    y = M.moe_few_tokens(**q, top_k=K)
    rows = [0, 1, 3, 5]
    assert torch.equal(y[rows], clean[rows])
    assert torch.isnan(y[2]).all()
    assert not torch.isfinite(y[4]).any()


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("T,d,E,K,H", [(1, 512, 8, 2, 1024), (11, 1000, 20, 3, 1416),
                                       (40, 256, 3, 6, 136), (128, 128, 2, 16, 64), (7, 33, 5, 3, 19)])
def test_given_routing(cuda_dev, T, d, E, K, H, dtype):
    """Random picks with repeats (K may exceed E), some zero weights, int32 and int64."""
    p = make(cuda_dev, T, d, E, H, dtype, seed=T + d)
    g = torch.Generator(device=cuda_dev).manual_seed(T)
    idx = torch.randint(0, E, (T, K), device=cuda_dev, generator=g)
    w = torch.randn(T, K, device=cuda_dev, generator=g)
    w[torch.rand(T, K, device=cuda_dev, generator=g) < 0.2] = 0
    ex = {k: v for k, v in p.items() if k != "w_router"}
    x = ex.pop("x")
    y = M.moe_few_experts(x, w, idx, **ex)
    y64, mag = layer64(p, w, idx)
    check(y, y64, mag, dtype, d, H)
    assert torch.equal(y, M.moe_few_experts(x, w, idx.int(), **ex))


def test_out_of_range_index_is_dropped_and_reported(cuda_dev):
    p = make(cuda_dev, 3, 128, 4, 128, BF)
    ex = {k: v for k, v in p.items() if k not in ("w_router", "x")}
    idx = torch.tensor([[0, 4], [-1, 2], [1, 3]], device=cuda_dev)
    w = torch.ones(3, 2, device=cuda_dev)
    _lib.read_device_error()
    y = M.moe_few_experts(p["x"], w, idx, **ex)
    assert _lib.read_device_error() == 2
    y64, mag = layer64(p, w, idx)
    check(y, y64, mag, BF, 128, 128)


def test_no_tokens(cuda_dev):
    p = make(cuda_dev, 0, 128, 4, 128, BF)
    assert M.moe_few_tokens(**p, top_k=2).shape == (0, 128)


def test_strided_inputs(cuda_dev):
    T, d, E, K, H = 5, 256, 6, 2, 192
    p = make(cuda_dev, T, d, E, H, BF, seed=9)
    want = M.moe_few_tokens(**p, top_k=K)
    wide = torch.zeros(T, 2 * d, device=cuda_dev, dtype=BF)
    wide[:, 1::2] = p["x"]
    q = {k: v.transpose(-1, -2).contiguous().transpose(-1, -2) for k, v in p.items()}
    q["x"] = wide[:, 1::2]
    assert not q["x"].is_contiguous() and not q["w_gate"].is_contiguous()
    assert torch.equal(M.moe_few_tokens(**q, top_k=K), want)
    # rows that start off a 16-byte boundary
    flat = torch.empty(T * d + 1, device=cuda_dev, dtype=BF)
    off = flat[1:].view(T, d)
    off.copy_(p["x"])
    w, idx = route64(p, K)
    y64, mag = layer64(p, w, idx)
    check(M.moe_few_tokens(**dict(p, x=off), top_k=K), y64, mag, BF, d, H)


def test_side_stream_and_graph_replay(cuda_dev):
    """Two captured graphs and eager calls on another stream, with inputs that change."""
    T, d, E, K, H = 4, 512, 16, 2, 256
    p = make(cuda_dev, T, d, E, H, BF, seed=11)
    q = make(cuda_dev, 12, d, E, H, BF, seed=12)
    want_p, want_q = M.moe_few_tokens(**p, top_k=K), M.moe_few_tokens(**q, top_k=3)
    torch.cuda.synchronize()
    graphs = []
    for a, k in ((p, K), (q, 3)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = M.moe_few_tokens(**a, top_k=k)
        graphs.append((g, y))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            graphs[0][0].replay()
            eager = M.moe_few_tokens(**q, top_k=3)
        with torch.cuda.stream(s2):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want_p) and torch.equal(graphs[1][1], want_q)
        assert torch.equal(eager, want_q)
    p["x"].copy_(p["x"].flip(0))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want_p.flip(0))
    assert _lib.read_device_error() == 0


def test_two_streams_at_once(cuda_dev):
    """Eager calls that overlap on two streams, both persistent over all SMs."""
    a = make(cuda_dev, 9, 1024, 32, 1024, BF, seed=21)
    b = make(cuda_dev, 3, 512, 8, 2048, BF, seed=22)
    want_a, want_b = M.moe_few_tokens(**a, top_k=4), M.moe_few_tokens(**b, top_k=2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            got.append((M.moe_few_tokens(**a, top_k=4), want_a))
        with torch.cuda.stream(s2):
            got.append((M.moe_few_tokens(**b, top_k=2), want_b))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for y, w in got)
    assert _lib.read_device_error() == 0


def test_a_row_does_not_depend_on_its_batch(cuda_dev):
    """The same token alone and among others, with the sizes' split held (same T): other rows'
    values change nothing."""
    p = make(cuda_dev, 8, 512, 16, 512, BF, seed=23)
    y = M.moe_few_tokens(**p, top_k=2)
    q = dict(p, x=p["x"].clone())
    q["x"][1:] = torch.randn_like(q["x"][1:])
    assert torch.equal(M.moe_few_tokens(**q, top_k=2)[0], y[0])
