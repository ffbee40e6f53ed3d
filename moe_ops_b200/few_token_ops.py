"""The SwiGLU MoE layer for a few tokens (serving).

The layer the reference assembles from its ops (tests/test_moe.py:68-87; ``MoELayer`` here)
runs a router GEMM, a top-k, a permute, two grouped GEMMs and an unpermute, whose tiles hold
128 rows.  When every expert sees one row or a few, the layer is a single stream over the
picked experts' weights instead:

    moe_few_tokens(x, w_router, w_gate, w_up, w_down, top_k, router_bias=None) -> y
    moe_few_experts(x, weights, indices, w_gate, w_up, w_down) -> y

Two ways it differs from the assembled layer, both towards fewer roundings: the router's
logits stay in fp32 (the assembled layer rounds them to x's dtype, so close logits may rank
differently), and gate, up and the experts' outputs are never rounded to 16 bits.

Forward only: the calls refuse inputs that require a gradient while grad mode is on, and inputs
with a forward-mode tangent.  Eager calls go to the C ABI at once, because at one token the host's
part of a call is of the order of the kernel's time; under torch's tracers and torch.compile they go
through the registered ops ``moeb200::few_tokens`` and ``moeb200::few_experts``.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib

MAX_TOKENS = 128  # tokens of a call
MAX_TOPK = 16


def _check_experts(x, w_gate, w_up, w_down) -> tuple[int, int, int, int]:
    _lib.require_cuda(x, w_gate, w_up, w_down)
    if x.dim() != 2 or w_gate.dim() != 3 or w_down.dim() != 3:
        raise ValueError("x must be [T, d] and the expert weights 3-D")
    T, d = x.shape
    E, H, _ = w_gate.shape
    if w_gate.shape != (E, H, d) or w_up.shape != (E, H, d) or w_down.shape != (E, d, H):
        raise ValueError(
            f"expected w_gate / w_up [E, H, {d}] and w_down [E, {d}, H]; got {tuple(w_gate.shape)}, "
            f"{tuple(w_up.shape)}, {tuple(w_down.shape)}")
    if not (x.dtype == w_gate.dtype == w_up.dtype == w_down.dtype):
        raise ValueError("x and the weights must share one dtype")
    if not (x.device == w_gate.device == w_up.device == w_down.device):
        raise ValueError("x and the weights must be on one device")
    if T > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} tokens (got {T}); use the assembled layer")
    return T, d, E, H


def _no_grad_only(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the few-token layer has no backward; call it under torch.no_grad() "
                           "or use MoELayer / moe_layer_forward")


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(T: int, d: int, H: int, E: int, K: int, code: int) -> int:
    return _lib.load().moe_few_tokens_workspace_bytes(T, d, H, E, K, code)


def _run(x, route, w_gate, w_up, w_down, dims, K: int, given: bool) -> torch.Tensor:
    T, d, E, H = dims
    code = _lib.dtype_code(x.dtype)
    x, w_gate, w_up, w_down = (x.contiguous(), w_gate.contiguous(), w_up.contiguous(),
                               w_down.contiguous())
    lib = _lib.load()
    y = x.new_empty((T, d))
    fn = lib.moe_few_experts_fwd if given else lib.moe_few_tokens_fwd
    with _lib.on_device(x):
        ws_bytes = _workspace_bytes(T, d, H, E, K, code)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
        st = fn(x.data_ptr(), _lib.ptr(route[0]), _lib.ptr(route[1]), w_gate.data_ptr(),
                w_up.data_ptr(), w_down.data_ptr(), code, T, d, H, E, K, y.data_ptr(),
                ws.data_ptr(), ws_bytes, _lib.raw_stream(x))
    _lib.check(st, "moe_few_experts" if given else "moe_few_tokens")
    _lib.count_launches(2)
    return y


@torch.library.custom_op("moeb200::few_tokens", mutates_args=())
def few_tokens(x: torch.Tensor, w_router: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
               w_down: torch.Tensor, top_k: int, router_bias: Optional[torch.Tensor]) -> torch.Tensor:
    """moe_few_tokens for checked arguments; router_bias in fp32."""
    route = (w_router.contiguous(), None if router_bias is None else router_bias.contiguous())
    E, H, d = w_gate.shape
    return _run(x, route, w_gate, w_up, w_down, (x.shape[0], d, E, H), top_k, False)


@torch.library.custom_op("moeb200::few_experts", mutates_args=())
def few_experts(x: torch.Tensor, weights: torch.Tensor, indices: torch.Tensor, w_gate: torch.Tensor,
                w_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """moe_few_experts for checked arguments; weights in fp32, indices in int32."""
    E, H, d = w_gate.shape
    return _run(x, (weights.contiguous(), indices.contiguous()), w_gate, w_up, w_down,
                (x.shape[0], d, E, H), weights.shape[1], True)


@few_tokens.register_fake
def _(x, w_router, w_gate, w_up, w_down, top_k, router_bias):
    return x.new_empty(x.shape)


@few_experts.register_fake
def _(x, weights, indices, w_gate, w_up, w_down):
    return x.new_empty(x.shape)


def moe_few_tokens(x: torch.Tensor, w_router: torch.Tensor, w_gate: torch.Tensor,
                   w_up: torch.Tensor, w_down: torch.Tensor, top_k: int,
                   router_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The whole layer for x [T, d], T <= 128: y[t] = sum_k p[t,k] expert_{idx[t,k]}(x[t]).

    Args:
        w_router: [E, d]; the logits are x . w_router^T (+ router_bias [E]) in fp32.
        w_gate, w_up: [E, H, d];  w_down: [E, d, H].
        top_k: picks per token, at most min(E, 16); ties go to the lower expert index.
        router_bias: optional; -inf masks an expert (it is never weighted nor read).  A token
            whose experts are all masked gets zeros.

    Returns:
        y [T, d] in x's dtype.
    """
    T, d, E, H = dims = _check_experts(x, w_gate, w_up, w_down)
    _lib.require_cuda(w_router, router_bias)
    if w_router.shape != (E, d) or w_router.dtype != x.dtype or w_router.device != x.device:
        raise ValueError(f"w_router must be [{E}, {d}] of x's dtype and device")
    if not 0 < top_k <= min(E, MAX_TOPK):
        raise ValueError(f"top_k must be in [1, {min(E, MAX_TOPK)}] (got {top_k})")
    if router_bias is not None:
        if router_bias.shape != (E,) or router_bias.device != x.device:
            raise ValueError(f"router_bias must be [{E}] on x's device")
    _no_grad_only(x, w_router, w_gate, w_up, w_down, router_bias)
    if T == 0:
        return torch.empty_like(x)
    direct = _lib.direct(x, w_router, w_gate, w_up, w_down, router_bias)
    if not direct:
        _lib.refuse_tangents("moe_few_tokens", x, w_router, w_gate, w_up, w_down, router_bias)
    if router_bias is not None:
        router_bias = router_bias.detach().float().contiguous()
    if not direct:
        return torch.ops.moeb200.few_tokens(x, w_router, w_gate, w_up, w_down, top_k, router_bias)
    return _run(x, (w_router.contiguous(), router_bias), w_gate, w_up, w_down, dims, top_k, False)


def moe_few_experts(x: torch.Tensor, weights: torch.Tensor, indices: torch.Tensor,
                    w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """The experts' part with the routing given: y[t] = sum_k weights[t,k] expert_{indices[t,k]}(x[t]).

    weights [T, K] (used in fp32), indices [T, K] (int32), K <= 16.  An expert may appear more
    than once for a token.  An index outside [0, E) adds nothing and sets the device error
    word (code 2), as in ``permute``.
    """
    T, d, E, H = dims = _check_experts(x, w_gate, w_up, w_down)
    _lib.require_cuda(weights, indices)
    if weights.dim() != 2 or weights.shape != indices.shape or weights.shape[0] != T:
        raise ValueError(f"weights and indices must both be [{T}, K]")
    K = weights.shape[1]
    if not 0 < K <= MAX_TOPK:
        raise ValueError(f"K must be in [1, {MAX_TOPK}] (got {K})")
    if weights.device != x.device or indices.device != x.device:
        raise ValueError("weights and indices must be on x's device")
    if indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"indices must be int32 or int64 (got {indices.dtype})")
    _no_grad_only(x, weights, w_gate, w_up, w_down)
    if T == 0:
        return torch.empty_like(x)
    if indices.dtype == torch.int64:
        # out-of-range values stay out of range in 32 bits
        indices = indices.clamp(-1, E).to(torch.int32)
    if not _lib.direct(x, weights, indices, w_gate, w_up, w_down):
        _lib.refuse_tangents("moe_few_experts", x, weights, w_gate, w_up, w_down)
        return torch.ops.moeb200.few_experts(x, weights.float(), indices, w_gate, w_up, w_down)
    route = (weights.float().contiguous(), indices.contiguous())
    return _run(x, route, w_gate, w_up, w_down, dims, K, True)


__all__ = ["moe_few_tokens", "moe_few_experts"]
