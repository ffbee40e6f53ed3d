"""Matrix product with bias, activation and residual in its epilogue, dense and per expert.

    linear(x, weight, bias=None, activation="none", residual=None) -> y
    grouped_linear(A, B, offsets, bias=None, activation="none", residual=None, trans_b=True) -> C

        z = x . W^T + bias            (per expert row range for grouped_linear)
        y = act(z) + residual

``grouped_linear`` stands beside ``grouped_gemm`` (same A, B, offsets and trans_b) for experts
with biases or an activation of their own; ``linear`` is the dense product next to the routed
experts (a shared expert, a projection).  The sum, the bias, the activation and the residual are in
fp32 inside the product's kernel and y is rounded once.  (A cut few-row product launches one more
kernel, which zeroes its counters, and a grouped call one more for the rows behind the last group.)

Both are differentiable in every tensor argument.  With an activation the forward also writes z
(rounded to the dtype) when a gradient will be needed; the backward is one elementwise pass
(dz = dy * act'(z), and the bias gradient from the unrounded dz), then the library's dgrad and
wgrad GEMMs.  The residual's gradient is dy itself.

Activations: "none", "relu", "gelu" (erf), "gelu_tanh", "silu".

Eager calls go to the C ABI at once: for one row the host's part of a call is of the order of the
kernel's time.  Under torch's tracers, torch.compile and functorch they go through the
registered ops ``moeb200::linear_fwd`` and ``moeb200::linear_bwd``.  There is no forward-mode
derivative; a dual input raises.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
import torch.nn.functional as F

from . import _lib

MAX_GROUPS = 1024
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _check(x, w, bias, residual, out_shape, bias_shape, activation) -> int:
    _lib.require_cuda(x, w, bias, residual)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)} (got {activation!r})")
    dtype, device = x.dtype, x.device
    _lib.dtype_code(dtype)
    if w.dtype != dtype or w.device != device:
        raise ValueError("weight must have the input's dtype and device")
    if bias is not None and (bias.dtype != dtype or bias.device != device or bias.shape != bias_shape):
        raise ValueError(f"bias must be {list(bias_shape)} of the input's dtype and device")
    if residual is not None and (residual.dtype != dtype or residual.device != device
                                 or residual.shape != out_shape):
        raise ValueError(f"residual must be {list(out_shape)} of the input's dtype and device")
    return act


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(m: int, n: int, k: int, E: int, trans_b: int, code: int) -> int:
    return _lib.load().moe_linear_workspace_bytes(m, n, k, E, trans_b, code)


def _forward(x, w, bias, residual, offsets, act: int, trans_b: bool, E: int, n: int, want_z: bool):
    """x [m, k], w [E, n, k] or [E, k, n] (2-D when dense), contiguous; returns (y, z or None)."""
    m, k = x.shape
    px, pw, pb, pr = x.data_ptr(), w.data_ptr(), _lib.ptr(bias), _lib.ptr(residual)
    if (px | pw | (pb or 0) | (pr or 0)) & 15:
        x, w, bias, residual = _on_boundary(m, n, k, E, trans_b, x, w, bias, residual)
        px, pw, pb, pr = x.data_ptr(), w.data_ptr(), _lib.ptr(bias), _lib.ptr(residual)
    y = x.new_empty((m, n))
    z = torch.empty_like(y) if want_z else None
    lib = _lib.load()
    code = _lib.dtype_code(x.dtype)
    with _lib.on_device(x):
        ws_bytes = _workspace_bytes(m, n, k, E, int(trans_b), code)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
        st = lib.moe_linear_fwd(
            px, pw, pb, pr, y.data_ptr(), _lib.ptr(z), _lib.ptr(offsets),
            0 if offsets is None else offsets.numel(), m, n, k, E, int(trans_b), act, code,
            _lib.ptr(ws), ws_bytes, _lib.raw_stream(x))
    _lib.check(st, "moe_linear_fwd")
    _lib.count_launches(1)
    return y, z


@functools.lru_cache(maxsize=4096)
def _bwd_workspace_bytes(m: int, n: int, E: int, act: int, code: int) -> int:
    return _lib.load().moe_linear_bwd_workspace_bytes(m, n, E, act, code)


def _backward(dy, x, w, z, offsets, act: int, trans_b: bool, E: int, n: int, bias_shape, wanted):
    """(dx, dw, dbias), None where not wanted."""
    m, k = x.shape
    if (n % 8 or k % 8) and x.dtype != torch.float32 and m * n * k >= _PAD_FROM and _copy_pays(m, n, E, False):
        return _backward_padded(dy, x, w, z, offsets, act, trans_b, E, n, bias_shape, wanted)
    if (x.data_ptr() | w.data_ptr() | dy.data_ptr()) & 15:
        x, w, dy = _on_boundary(m, n, k, E, False, x, w, dy)
    dx = torch.empty_like(x) if wanted[0] else None
    dw = torch.empty_like(w) if wanted[1] else None
    db = x.new_empty(bias_shape) if wanted[2] else None
    code = _lib.dtype_code(x.dtype)
    lib = _lib.load()
    with _lib.on_device(x):
        ws_bytes = _bwd_workspace_bytes(m, n, E, act, code) if act or wanted[2] else 0
        ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
        st = lib.moe_linear_bwd(
            dy.data_ptr(), x.data_ptr(), w.data_ptr(), _lib.ptr(z), _lib.ptr(dx), _lib.ptr(dw),
            _lib.ptr(db), _lib.ptr(offsets), 0 if offsets is None else offsets.numel(), m, n, k, E,
            int(trans_b), act, code, _lib.ptr(ws), ws_bytes, _lib.raw_stream(x))
    _lib.check(st, "moe_linear_bwd")
    _lib.count_launches(sum(wanted) + int(act != 0))
    return dx, dw, db


def _sizes(w, trans_b: bool) -> tuple[int, int]:
    """(E, n) of a weight [n, k] (E = 1), [E, n, k] or [E, k, n]."""
    return (1, w.shape[0]) if w.dim() == 2 else (w.shape[0], w.shape[1 if trans_b else 2])


@torch.library.custom_op("moeb200::linear_fwd", mutates_args=())
def linear_fwd(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor],
               residual: Optional[torch.Tensor], offsets: Optional[torch.Tensor], act: int,
               trans_b: bool, want_z: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, z): y = act(z) + residual, z = x . w^T + bias per row range; z is empty unless wanted."""
    E, n = _sizes(w, trans_b)
    x, w, bias, residual, offsets = (t if t is None else t.contiguous()
                                     for t in (x, w, bias, residual, offsets))
    y, z = _forward(x, w, bias, residual, offsets, act, trans_b, E, n, want_z)
    return y, x.new_empty(0) if z is None else z


@linear_fwd.register_fake
def _(x, w, bias, residual, offsets, act, trans_b, want_z):
    shape = (x.shape[0], _sizes(w, trans_b)[1])
    return x.new_empty(shape), x.new_empty(shape if want_z else (0,))


@torch.library.custom_op("moeb200::linear_bwd", mutates_args=())
def linear_bwd(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, z: Optional[torch.Tensor],
               offsets: Optional[torch.Tensor], act: int, trans_b: bool, want_x: bool, want_w: bool,
               want_bias: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw, dbias) of linear_fwd from its z (not read without an activation); empty where not
    wanted."""
    E, n = _sizes(w, trans_b)
    dy, x, w, z, offsets = (t if t is None else t.contiguous() for t in (dy, x, w, z, offsets))
    got = _backward(dy, x, w, z, offsets, act, trans_b, E, n, (n,) if w.dim() == 2 else (E, n),
                    (want_x, want_w, want_bias))
    return tuple(x.new_empty(0) if t is None else t for t in got)


@linear_bwd.register_fake
def _(dy, x, w, z, offsets, act, trans_b, want_x, want_w, want_bias):
    E, n = _sizes(w, trans_b)
    bias = (n,) if w.dim() == 2 else (E, n)
    return (x.new_empty(x.shape if want_x else (0,)), w.new_empty(w.shape if want_w else (0,)),
            x.new_empty(bias if want_bias else (0,)))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, offsets, act, trans_b, E, n, direct):
        want_z = act != 0 and any(ctx.needs_input_grad[:3])
        if direct:
            y, z = _forward(x, w, bias, residual, offsets, act, trans_b, E, n, want_z)
        else:
            y, z = torch.ops.moeb200.linear_fwd(x, w, bias, residual, offsets, act, trans_b, want_z)
            z = z if want_z else None
        ctx.save_for_backward(x, w, z, offsets)
        ctx.cfg = (act, trans_b, E, n, None if bias is None else bias.shape, direct)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, z, offsets = ctx.saved_tensors
        act, trans_b, E, n, bias_shape, direct = ctx.cfg
        wanted = ctx.needs_input_grad[:3]
        dx = dw = db = None
        if True in wanted:
            if direct and _lib.direct(dy):
                dx, dw, db = _backward(dy.contiguous(), x, w, z, offsets, act, trans_b, E, n, bias_shape, wanted)
            else:
                _lib.refuse_tangents("the backward of linear", dy)
                got = torch.ops.moeb200.linear_bwd(dy, x, w, z, offsets, act, trans_b, *wanted)
                dx, dw, db = (t if on else None for t, on in zip(got, wanted))
        return dx, dw, db, dy if ctx.needs_input_grad[3] else None, *([None] * 6)


# 16-bit operands whose rows are not 16-byte multiples, or that start off a 16-byte boundary: from
# this many multiplications on, and if _copy_pays, they are copied into rows that are (zeros behind)
# for the tensor cores; otherwise the CUDA cores take them as they are.
_PAD_FROM = 1 << 24


def _copy_pays(m: int, n: int, E: int, trans_b: bool) -> bool:
    """Whether m rows over E groups amortise a copy of every group's weights.  (The backward asks
    without trans_b: its dgrad reads the weights as such a product does.)

    Measured, bf16, CUDA cores / copy and tensor cores in us (rows, K -> N):
        4 x 4097 -> 4097        72 / 85     8: 114 / 85     64: 475 / 95
        2 x 7167 -> 11007       211 / 269   4: 275 / 269    16: 712 / 273
        8 groups 1999 -> 2001   32: 132 / 140   64: 214 / 138
        64 groups 999 -> 1001   16: 52 / 224    256: 247 / 245   512: 390 / 247
    Without trans_b the CUDA cores have only 64 x 64 tiles, whose time follows K and how many there
    are, while a copy's follows E * N * K:
        1 x 4097 -> 4097        468 / 98
        8 groups 1999 -> 2001   1: 231 / 133    64: 276 / 139
        32 groups 999 -> 1001   1: 121 / 125    16: 159 / 133
        64 groups 999 -> 1001   32: 165 / 229   64: 310 / 240
    """
    return m > 4 * E if trans_b else (E * n <= 40000 or m >= E)


def _on_boundary(m, n, k, E, trans_b, x, w, *others):
    """The operands, those off a 16-byte boundary copied where that lets the tensor cores take them."""
    off = [t is not None and t.data_ptr() & 15 != 0 for t in (x, w, *others)]
    if (x.dtype == torch.float32 or n % 8 or k % 8 or m * n * k < _PAD_FROM
            or (off[1] and not _copy_pays(m, n, E, trans_b))):
        return x, w, *others
    return tuple(t.clone() if o else t for t, o in zip((x, w, *others), off))


def _pad_weight(w, trans_b, dn, dk):
    return F.pad(w, (0, dk, 0, dn) if trans_b else (0, dn, 0, dk))


def _padded(x, w, bias, residual, offsets, act, trans_b, E, n):
    k = x.shape[1]
    dn, dk = -n % 8, -k % 8
    w = _pad_weight(w, trans_b, dn, dk)
    y = _apply(F.pad(x, (0, dk)), w, None if bias is None else F.pad(bias, (0, dn)),
               None if residual is None else F.pad(residual, (0, dn)), offsets, act, trans_b, E, n + dn)
    return y[:, :n].contiguous()


def _backward_padded(dy, x, w, z, offsets, act, trans_b, E, n, bias_shape, wanted):
    """_backward through 16-byte rows, where the forward's rows were too few for a copy."""
    k = x.shape[1]
    dn, dk = -n % 8, -k % 8
    dx, dw, db = _backward(F.pad(dy, (0, dn)), F.pad(x, (0, dk)), _pad_weight(w, trans_b, dn, dk),
                           None if z is None else F.pad(z, (0, dn)), offsets, act, trans_b, E, n + dn,
                           None if bias_shape is None else (*bias_shape[:-1], n + dn), wanted)
    if dx is not None:
        dx = dx[:, :k].contiguous()
    if dw is not None:
        dw = (dw[..., :n, :k] if trans_b else dw[..., :k, :n]).contiguous()
    return dx, dw, None if db is None else db[..., :n].contiguous()


def _apply(x, w, bias, residual, offsets, act, trans_b, E, n):
    m, k = x.shape
    if (n % 8 or k % 8) and x.dtype != torch.float32 and m * n * k >= _PAD_FROM and _copy_pays(m, n, E, trans_b):
        return _padded(x, w, bias, residual, offsets, act, trans_b, E, n)
    grads = torch.is_grad_enabled() and (
        x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)
        or (residual is not None and residual.requires_grad))
    direct = _lib.direct(x, w, bias, residual, offsets)
    # The autograd Function refuses what it cannot differentiate (forward mode, functorch).
    if grads or not direct:
        return _Linear.apply(x, w, bias, residual, offsets, act, trans_b, E, n, direct)
    return _forward(x, w, bias, residual, offsets, act, trans_b, E, n, False)[0]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           activation: str = "none", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x . weight^T + bias) + residual, in the product's kernel.

    Args:
        x: [..., K].
        weight: [N, K].
        bias: [N], or None.
        activation: "none", "relu", "gelu", "gelu_tanh" or "silu".
        residual: [..., N] (the output's shape), or None.

    Returns:
        [..., N] in x's dtype.
    """
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x [..., K] and weight [N, K] do not match: {list(x.shape)}, {list(weight.shape)}")
    n, k = weight.shape
    if x.dim() == 2:
        x2, out_shape = x, (x.shape[0], n)
    else:
        out_shape = x.shape[:-1] + (n,)
        x2 = x.reshape(out_shape[:-1].numel(), k)
    act = _check(x, weight, bias, residual, out_shape, (n,), activation)
    r2 = None if residual is None else residual.reshape(x2.shape[0], n).contiguous()
    y = _apply(x2.contiguous(), weight.contiguous(), None if bias is None else bias.contiguous(), r2,
               None, act, True, 1, n)
    return y if x.dim() == 2 else y.view(out_shape)


def grouped_linear(A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, activation: str = "none",
                   residual: Optional[torch.Tensor] = None, trans_b: bool = True) -> torch.Tensor:
    """``grouped_gemm`` with a bias per expert, an activation and a residual in its epilogue.

    Args:
        A: [total_tokens, K], the experts' rows stacked.
        B: [E, N, K] if trans_b else [E, K, N].
        offsets: int32 [E+1] (starting at 0) or [E] end rows, as in ``grouped_gemm``.
        bias: [E, N], or None.
        activation, residual: as in ``linear``; residual [total_tokens, N].

    At most 1024 experts.  A backward pass can be captured into a CUDA graph once every eager
    output of the same leaves is released (autograd otherwise waits for the stream those used, which
    invalidates the capture).

    Returns:
        [total_tokens, N].  Rows behind the last offset get the residual (zero without one), and
        their input gradient is zero.
    """
    if A.dim() != 2 or B.dim() != 3 or B.shape[2 if trans_b else 1] != A.shape[1]:
        raise ValueError(f"A [M, K] and B do not match: {list(A.shape)}, {list(B.shape)}, trans_b={trans_b}")
    E, n = B.shape[0], B.shape[1 if trans_b else 2]
    if E > MAX_GROUPS:
        raise ValueError(f"at most {MAX_GROUPS} experts (got {E})")
    act = _check(A, B, bias, residual, (A.shape[0], n), (E, n), activation)
    _lib.require_cuda(offsets)
    if offsets.numel() not in (E, E + 1) or offsets.numel() == 0 or offsets.device != A.device:
        raise ValueError(f"offsets must have E ({E}) or E+1 entries on A's device, got {offsets.numel()}")
    if offsets.dtype != torch.int32:
        offsets = offsets.to(torch.int32)
    return _apply(A.contiguous(), B.contiguous(), None if bias is None else bias.contiguous(),
                  None if residual is None else residual.contiguous(), offsets.contiguous(), act,
                  bool(trans_b), E, n)


__all__ = ["linear", "grouped_linear"]
