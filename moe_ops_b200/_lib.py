"""ctypes binding of libmoe_b200.so (the C ABI declared in include/moe_b200.h).

The library is loaded from this package directory.  There is no fallback: if the
shared library is missing or a call fails, a RuntimeError is raised.
"""
from __future__ import annotations

import ctypes
import os
import threading

import torch
from torch.autograd import forward_ad

LIB_NAME = "libmoe_b200.so"
LIB_PATH = os.environ.get("MOE_B200_LIB") or os.path.join(
    os.path.dirname(os.path.abspath(__file__)), LIB_NAME)

MOE_F32, MOE_F16, MOE_BF16 = 0, 1, 2
_DTYPE_CODE = {torch.float32: MOE_F32, torch.float16: MOE_F16, torch.bfloat16: MOE_BF16}

_c_i32 = ctypes.c_int32
_c_i64 = ctypes.c_int64
_c_int = ctypes.c_int
_c_ptr = ctypes.c_void_p
_c_size = ctypes.c_size_t

# name -> (restype, argtypes); must match include/moe_b200.h.
SIGNATURES = {
    "moe_version": (ctypes.c_char_p, []),
    "moe_last_error_string": (ctypes.c_char_p, []),
    "moe_read_device_error": (_c_int, [ctypes.POINTER(_c_int)]),
    "moe_peek_device_error": (_c_int, [_c_ptr, _c_ptr]),
    "moe_selftest_bounded_wait": (_c_int, [ctypes.c_uint64, _c_ptr, _c_ptr]),
    "moe_write_probe": (_c_int, [_c_ptr, ctypes.c_size_t, _c_ptr]),
    "moe_ipc_malloc": (_c_int, [ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p), _c_ptr]),
    "moe_ipc_open": (_c_int, [_c_ptr, ctypes.POINTER(ctypes.c_void_p)]),
    "moe_ipc_close": (_c_int, [_c_ptr]),
    "moe_ipc_free": (_c_int, [_c_ptr]),
    "moe_ep_slot_map": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_i64, _c_i32, _c_i32, _c_i32, _c_i32,
                                 _c_i64, _c_ptr, _c_ptr, _c_ptr]),
    "moe_ep_dispatch": (_c_int, [_c_ptr, _c_int, _c_ptr, _c_ptr, _c_ptr, _c_i64, _c_i32, _c_i64,
                                 _c_ptr, _c_ptr]),
    "moe_ep_combine": (_c_int, [_c_ptr, _c_int, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_i64, _c_i32,
                                _c_i64, _c_ptr, _c_ptr, _c_ptr]),
    "moe_ep_combine_bwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_int, _c_ptr, _c_ptr, _c_ptr, _c_int,
                                    _c_i64, _c_i32, _c_i64, _c_ptr, _c_ptr, _c_ptr]),
    "moe_add_rows": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_i64, _c_i64, _c_int, _c_ptr]),
    "moe_ep_barrier": (_c_int, [_c_ptr, _c_i32, _c_i32, _c_ptr, ctypes.c_uint64, _c_ptr, _c_ptr]),
    "moe_ep_put_counts": (_c_int, [_c_ptr, _c_i32, _c_ptr, _c_i32, _c_i32, _c_ptr]),
    "moe_topk_softmax_fwd": (_c_int, [_c_ptr, _c_int, _c_i64, _c_i32, _c_i32, _c_ptr, _c_ptr, _c_ptr]),
    "moe_topk_softmax_bwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_int, _c_i64, _c_i32, _c_i32, _c_ptr, _c_ptr]),
    "moe_permute_workspace_bytes": (_c_size, [_c_i64, _c_i32, _c_i32]),
    "moe_permute": (_c_int, [_c_ptr, _c_int, _c_ptr, _c_i64, _c_i32, _c_i64, _c_i32, _c_i64,
                             _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_size, _c_ptr]),
    "moe_permute_capacity": (_c_int, [_c_ptr, _c_int, _c_ptr, _c_i64, _c_i32, _c_i64, _c_i32,
                                      _c_i32, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_size,
                                      _c_ptr]),
    "moe_permute_index": (_c_int, [_c_ptr, _c_i64, _c_i32, _c_i32, _c_ptr, _c_ptr, _c_ptr, _c_ptr,
                                   _c_size, _c_ptr]),
    "moe_gmm_fwd_gather": (_c_int, [_c_ptr, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_i32, _c_i64,
                                    _c_i64, _c_i64, _c_i32, _c_int, _c_int, _c_ptr]),
    "moe_gmm_gate_up_fwd_gather": (_c_int, [_c_ptr, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr,
                                            _c_ptr, _c_ptr, _c_i32, _c_i64, _c_i64, _c_i64, _c_i32,
                                            _c_int, _c_int, _c_ptr]),
    "moe_gmm_wgrad_gather": (_c_int, [_c_ptr, _c_ptr, _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_i32, _c_i64,
                                      _c_i64, _c_i64, _c_i32, _c_int, _c_int, _c_ptr]),
    "moe_permute_noalloc": (_c_int, [_c_ptr, _c_int, _c_ptr, _c_i64, _c_i32, _c_i64, _c_i32,
                                     _c_i64, _c_ptr, _c_ptr, _c_ptr, _c_ptr]),
    "moe_permute_noalloc_max_slots": (_c_size, [_c_i32]),
    "moe_swiglu_fwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_i64, _c_int, _c_ptr]),
    "moe_swiglu_bwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i64, _c_int, _c_ptr]),
    "moe_scatter_rows": (_c_int, [_c_ptr, _c_int, _c_ptr, _c_i64, _c_i32, _c_i64, _c_ptr, _c_ptr]),
    "moe_unpermute_fwd": (_c_int, [_c_ptr, _c_int, _c_ptr, _c_ptr, _c_int, _c_i64, _c_i32, _c_i64,
                                   _c_ptr, _c_ptr]),
    "moe_unpermute_bwd": (_c_int, [_c_ptr, _c_ptr, _c_int, _c_ptr, _c_ptr, _c_int, _c_i64, _c_i32,
                                   _c_i64, _c_ptr, _c_ptr, _c_ptr]),
    "moe_gmm_fwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i32, _c_i64, _c_i64, _c_i64, _c_i32,
                             _c_int, _c_int, _c_ptr]),
    "moe_gmm_gate_up_fwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i32,
                                     _c_i64, _c_i64, _c_i64, _c_i32, _c_int, _c_int, _c_ptr]),
    "moe_gmm_dgrad_swiglu_bwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr,
                                          _c_i32, _c_i64, _c_i64, _c_i64, _c_i32, _c_int, _c_int,
                                          _c_ptr]),
    "moe_gmm_dgrad": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i32, _c_i64, _c_i64, _c_i64, _c_i32,
                               _c_int, _c_int, _c_ptr]),
    "moe_gmm_dgrad_dual": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i32, _c_i64,
                                    _c_i64, _c_i64, _c_i64, _c_i32, _c_int, _c_int, _c_ptr]),
    "moe_gmm_wgrad": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i32, _c_i64, _c_i64, _c_i64, _c_i32,
                               _c_int, _c_int, _c_ptr]),
    "moe_linear_fwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i32, _c_i64,
                                _c_i64, _c_i64, _c_i32, _c_int, _c_int, _c_int, _c_ptr, _c_size, _c_ptr]),
    "moe_linear_workspace_bytes": (_c_size, [_c_i64, _c_i64, _c_i64, _c_i32, _c_int, _c_int]),
    "moe_linear_bwd_workspace_bytes": (_c_size, [_c_i64, _c_i64, _c_i32, _c_int, _c_int]),
    "moe_linear_bwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_i32,
                                _c_i64, _c_i64, _c_i64, _c_i32, _c_int, _c_int, _c_int, _c_ptr,
                                _c_size, _c_ptr]),
    "moe_few_tokens_workspace_bytes": (_c_size, [_c_i64, _c_i64, _c_i64, _c_i32, _c_i32, _c_int]),
    "moe_few_tokens_fwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_i64,
                                    _c_i64, _c_i64, _c_i32, _c_i32, _c_ptr, _c_ptr, _c_size, _c_ptr]),
    "moe_few_experts_fwd": (_c_int, [_c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_ptr, _c_int, _c_i64,
                                     _c_i64, _c_i64, _c_i32, _c_i32, _c_ptr, _c_ptr, _c_size, _c_ptr]),
}

_lib = None
_lock = threading.Lock()

# Instrumentation used by bench.py: number of library kernels launched so far (the main kernels
# of each call: zeroed counters, rows behind the last group, the bias gradient's second pass
# and the CUDA cores' extra launches of the few-token layer are not counted), and an optional list that collects (name, start_event, end_event, flops) around every grouped
# GEMM call (CUDA events on the launching stream).
launch_count = 0
gemm_timing: list | None = None


def count_launches(n: int) -> None:
    global launch_count
    launch_count += n


def load() -> ctypes.CDLL:
    """Loads the shared library once; raises RuntimeError if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"{LIB_NAME} is not built ({LIB_PATH} missing); run "
                    "`python -m moe_ops_b200.build` (nvcc, sm_100a)")
            lib = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16") from None


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream_of(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


class _Here:
    """A context that changes nothing."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_device(t: torch.Tensor):
    """torch.cuda.device(t.device), without its cost when that device is current already."""
    index = t.device.index
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def raw_stream(t: torch.Tensor) -> int:
    """stream_of without building a Stream object."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


_PLAIN = (torch.Tensor, torch.nn.Parameter)
_compiling = torch.compiler.is_compiling
_tracing = torch._C._get_tracing_state
_modes = torch._C._len_torch_dispatch_stack
_functorch = torch._C._functorch.peek_interpreter_stack


def direct(*tensors: torch.Tensor | None) -> bool:
    """Whether a call on these tensors may go to the library at once.

    False while something records or transforms calls (jit.trace, make_fx and other dispatch
    modes, torch.compile, functorch, forward-mode differentiation) or a tensor is of another
    class (fake, distributed, ...): such a call goes through the registered op, which those
    see.  About half a microsecond, a tenth of a registered op's own cost.
    """
    if _compiling() or _tracing() is not None or _modes() or _functorch() is not None:
        return False
    if forward_ad._current_level >= 0:
        return False
    for t in tensors:
        if t is not None and type(t) not in _PLAIN:
            return False
    return True


def refuse_tangents(what: str, *tensors: torch.Tensor | None) -> None:
    """Raises where an input carries a forward-mode tangent, which the kernels would drop."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")


def check(status: int, what: str) -> None:
    if status != 0:
        msg = load().moe_last_error_string().decode(errors="replace")
        raise RuntimeError(f"{what} failed (status {status}): {msg}")


def require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(
                "moe_ops_b200 runs on CUDA tensors only (sm_100a kernels); got a tensor on "
                f"{t.device}")


def read_device_error() -> int:
    """Reads and clears the library's device-side error word (synchronises)."""
    code = _c_int(0)
    check(load().moe_read_device_error(ctypes.byref(code)), "moe_read_device_error")
    return code.value
