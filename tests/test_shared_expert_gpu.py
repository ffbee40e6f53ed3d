"""MoELayer with a shared expert and the few-token path: the new operators together, as the
layer runs them."""
import math

import pytest
import torch
import torch.nn.functional as F

from moe_ops_b200 import _lib
from moe_ops_b200.moe_layer import MoELayer

pytestmark = pytest.mark.gpu


def layer(dev, dtype, shared=96, d=128, E=8, K=2, H=192):
    g = torch.Generator(device=dev).manual_seed(5)
    m = MoELayer(d, E, K, H, fp32_routing=True, device=dev, dtype=dtype, shared_hidden=shared)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape, device=dev, generator=g) / math.sqrt(p.shape[-1]))
    return m


def reference(m, x, logits):
    """The layer in 64 bits, its experts picked by the given logits."""
    top = torch.sort(logits, dim=1, descending=True, stable=True)
    idx, w = top.indices[:, :m.top_k], torch.softmax(top.values[:, :m.top_k].double(), 1)
    X = x.double()
    y = torch.zeros_like(X)
    for e in range(m.num_experts):
        t, k = torch.nonzero(idx == e, as_tuple=True)
        h = F.silu(X[t] @ m.w_gate[e].double().t()) * (X[t] @ m.w_up[e].double().t())
        y = y.index_add(0, t, h @ m.w_down[e].double().t() * w[t, k][:, None])
    s = F.silu(X @ m.w_shared_in.double().t() + m.b_shared_in.double())
    return y + s @ m.w_shared_out.double().t() + m.b_shared_out.double()


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def test_training_step(cuda_dev):
    """bf16, 300 tokens: output and every gradient against automatic differentiation in 64 bits.

    The bars count roundings of 2^-8 (relative, at most half a step each): the output passes four
    in a row (h, expert output, combine, epilogue), an input gradient seven.  Each is at most
    2^-8 of its value, and norms of independent errors add up more slowly than linearly.
    """
    m = layer(cuda_dev, torch.bfloat16)
    x = torch.randn(300, 128, device=cuda_dev, dtype=torch.bfloat16).requires_grad_(True)
    dy = torch.randn(300, 128, device=cuda_dev, dtype=torch.bfloat16)
    y = m(x)
    logits = (x.detach() @ m.w_router.detach().t()).float()
    y.backward(dy)
    r = layer(cuda_dev, torch.bfloat16).double()
    xr = x.detach().double().requires_grad_(True)
    # routing weights as the layer's router rounds them, constant here
    want = reference(r, xr, logits)
    want.backward(dy.double())
    assert rel(y, want.detach()) < 4 * 2.0 ** -8
    for n in ("w_gate", "w_up", "w_down", "w_shared_in", "b_shared_in", "w_shared_out", "b_shared_out"):
        assert rel(getattr(m, n).grad, getattr(r, n).grad) < 7 * 2.0 ** -8, n
    # the x gradient also holds the router's part, which the reference leaves out
    assert torch.isfinite(x.grad).all() and m.w_router.grad is not None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T", [1, 7, 64])
def test_decoding(cuda_dev, T, dtype):
    m = layer(cuda_dev, dtype)
    m.few_tokens = 64
    x = torch.randn(T, 128, device=cuda_dev, dtype=dtype)
    with torch.no_grad():
        before = _lib.launch_count
        y = m(x)
        assert _lib.launch_count - before == 4  # router + experts, and the two projections
        want = reference(m, x, x.double() @ m.w_router.double().t())
        # h, the shared expert's h and the routed output are rounded to the dtype, then y
        bar = 4 * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 1e-5
        assert rel(y, want) < bar
        # one more token than the limit runs the assembled layer
        before = _lib.launch_count
        m(torch.randn(65, 128, device=cuda_dev, dtype=dtype))
        assert _lib.launch_count - before > 4


def test_decoding_path_is_not_taken_with_gradients(cuda_dev):
    m = layer(cuda_dev, torch.bfloat16)
    m.few_tokens = 64
    y = m(torch.randn(3, 128, device=cuda_dev, dtype=torch.bfloat16))
    y.sum().backward()
    assert all(p.grad is not None for p in m.parameters())


def test_captured_decoding_step(cuda_dev):
    m = layer(cuda_dev, torch.bfloat16)
    m.few_tokens = 16
    x = torch.randn(4, 128, device=cuda_dev, dtype=torch.bfloat16)
    with torch.no_grad():
        want = m(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = m(x)
        for _ in range(3):
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
        x.copy_(x.flip(0))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want.flip(0))
