"""ctypes binding of the C ABI declared in include/bitween_b200.h.

This is the only place the Python host code crosses into native code.  There is no
fallback of any kind: if the shared library is missing (and cannot be built because nvcc
is absent) or no CUDA device is present, the calls raise.
"""
import contextlib
import ctypes
import importlib.util
import os
import sys
import threading
import warnings

import torch
import torch.autograd.forward_ad as fwad
from torch.utils import _python_dispatch

F32, F16, BF16, I32 = 0, 1, 2, 3
RTN_UPCAST_F32 = 1
RTN_TMA_STREAM = 2
ERR_WORKSPACE = 7

_DTYPE_CODE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.int32: I32}

_PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(_PKG, "_C", "libbitween_b200.so")

_lib = None
_lock = threading.Lock()


class BitweenKernelError(RuntimeError):
    """A C-ABI call returned a non-zero bw_status."""

    def __init__(self, status, text):
        super().__init__(f"libbitween_b200: {text} (status {status})")
        self.status = status


def dtype_code(dt):
    try:
        return _DTYPE_CODE[dt]
    except KeyError:
        raise TypeError(f"bitween_b200: unsupported dtype {dt}") from None


ACT_NONE, ACT_RELU, ACT_SILU_MUL = 0, 1, 2


class Epilogue(ctypes.Structure):
    """bw_epilogue of include/bitween_b200.h."""
    _fields_ = [("activation", ctypes.c_int), ("residual", ctypes.c_void_p)]


class Rotary(ctypes.Structure):
    """bw_rotary of include/bitween_b200.h."""
    _fields_ = [("table", ctypes.c_void_p), ("max_positions", ctypes.c_int64), ("rotary_dim", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("num_axes", ctypes.c_int), ("axes", ctypes.c_char_p), ("positions", ctypes.c_void_p), ("axis_stride", ctypes.c_int64)]


class RtnJob(ctypes.Structure):
    """bw_rtn_job of include/bitween_b200.h."""
    _fields_ = [("w", ctypes.c_void_p), ("qweight", ctypes.c_void_p), ("scale", ctypes.c_void_p),
                ("zero_point", ctypes.c_void_p), ("N", ctypes.c_int64), ("K", ctypes.c_int64)]


def _declare(L):
    i64, i32, vp, u32, sz = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_uint, ctypes.c_size_t
    L.bw_rtn_quantize_pack.argtypes = [vp, i32, i64, i64, i32, i32, vp, vp, i32, vp, i32, u32, vp]
    L.bw_rtn_quantize_pack.restype = i32
    L.bw_rtn_batch_table_bytes.argtypes = [i32]
    L.bw_rtn_batch_table_bytes.restype = sz
    L.bw_rtn_quantize_pack_batch.argtypes = [ctypes.POINTER(RtnJob), i32, i32, i32, i32, i32, i32, u32, vp, sz, vp]
    L.bw_rtn_quantize_pack_batch.restype = i32
    L.bw_peer_alloc.argtypes = [sz, ctypes.POINTER(vp), ctypes.c_char_p]
    L.bw_peer_alloc.restype = i32
    L.bw_peer_open.argtypes = [ctypes.c_char_p, ctypes.POINTER(vp)]
    L.bw_peer_open.restype = i32
    L.bw_peer_close.argtypes = [vp]
    L.bw_peer_close.restype = i32
    L.bw_peer_free.argtypes = [vp]
    L.bw_peer_free.restype = i32
    L.bw_peer_flag_bytes.restype = sz
    L.bw_peer_state_bytes.restype = sz
    L.bw_peer_allreduce_f16.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(vp), i32, i32, vp, i64, vp, vp]
    L.bw_peer_allreduce_f16.restype = i32
    L.bw_peer_allreduce2_f16.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(vp), ctypes.POINTER(vp), i32, i32, vp, i64, vp, vp]
    L.bw_peer_allreduce2_f16.restype = i32
    L.bw_fake_quant.argtypes = [vp, i32, i64, i64, i32, i32, vp, vp, vp, i32, vp, vp, vp]
    L.bw_fake_quant.restype = i32
    L.bw_fake_quant_native16.argtypes = [vp, i32, i64, i64, i32, i32, vp, vp, vp, vp, vp, vp]
    L.bw_fake_quant_native16.restype = i32
    L.bw_fake_quant_backward.argtypes = [vp, i32, i64, i64, i32, i32, vp, vp, vp, i32, vp, vp, vp, vp]
    L.bw_fake_quant_backward.restype = i32
    L.bw_group_params.argtypes = [vp, vp, i32, vp, vp, i64, i32, vp, vp, vp, vp]
    L.bw_group_params.restype = i32
    L.bw_group_params_backward.argtypes = [vp, vp, i32, vp, vp, vp, i64, i32, vp, vp, vp, vp, vp]
    L.bw_group_params_backward.restype = i32
    f32 = ctypes.c_float
    L.bw_kv_append.argtypes = [vp, vp, i32, i64, i64, i64, i64, i64, vp, i32, i32, i32, i64, i32, vp, vp, vp, vp]
    L.bw_kv_append.restype = i32
    L.bw_kv_read.argtypes = [vp, vp, vp, i32, i32, i32, i64, i32, vp, i64, vp, vp, i32, vp]
    L.bw_kv_read.restype = i32
    L.bw_kv_attend_workspace_bytes.argtypes = [i64, i32, i32, i32, i32, i64]
    L.bw_kv_attend_workspace_bytes.restype = sz
    L.bw_kv_attend.argtypes = [vp, i32, i64, i32, i64, i64, vp, vp, vp, i32, i64, i32, i32, i32, vp, i64, i64, vp, f32, vp, vp, sz, vp]
    L.bw_kv_attend.restype = i32
    L.bw_kv_attend_window_workspace_bytes.argtypes = [i64, i32, i32, i32, i32, i64, i64, i64]
    L.bw_kv_attend_window_workspace_bytes.restype = sz
    L.bw_kv_attend_window.argtypes = [vp, i32, i64, i32, i64, i64, vp, vp, vp, i32, i64, i32, i32, i32, vp, i64, i64, vp, i64, i64, f32, vp, vp, sz, vp]
    L.bw_kv_attend_window.restype = i32
    rotary = ctypes.POINTER(Rotary)
    L.bw_rotate.argtypes = [rotary, i64, i32, i32, i32, vp, i32, i64, i64, vp, vp, i32, i64, i64, vp, vp]
    L.bw_rotate.restype = i32
    L.bw_kv_append_rotated.argtypes = [rotary, vp, i32, i64, i64, vp, vp, vp, i32, i64, i64, i64, i64, i64, vp, i32, i32, i32, i64, i32, vp, vp, vp, vp]
    L.bw_kv_append_rotated.restype = i32
    L.bw_token_log_probs.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, i32, vp, vp, vp, vp]
    L.bw_token_log_probs.restype = i32
    L.bw_token_log_probs_grad.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, vp, i32, vp, vp, vp, vp]
    L.bw_token_log_probs_grad.restype = i32
    L.bw_adapter_hidden_bytes.argtypes = [i64, i32]
    L.bw_adapter_hidden_bytes.restype = sz
    L.bw_adapter_forward.argtypes = [vp, i32, i64, i64, i64, vp, vp, i32, i32, vp, vp, vp, vp, vp, sz, vp]
    L.bw_adapter_forward.restype = i32
    L.bw_adapter_backward.argtypes = [vp, i32, vp, i64, i64, i64, vp, vp, i32, i32, vp, vp, vp, sz, vp, vp, vp, vp, sz, vp]
    L.bw_adapter_backward.restype = i32
    L.bw_dequantize.argtypes = [vp, vp, i32, vp, i32, i64, i64, i32, i32, vp, i32, vp]
    L.bw_dequantize.restype = i32
    L.bw_qmatmul_workspace_bytes.argtypes = [i64, i64, i64, i32, i32]
    L.bw_qmatmul_workspace_bytes.restype = sz
    L.bw_qmatmul_workspace_bytes_for.argtypes = [i64, i64, i64, i32, i32, i32, i32]
    L.bw_qmatmul_workspace_bytes_for.restype = sz
    L.bw_qmatmul.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, vp, vp, i32, i32, i32, vp, sz, vp]
    L.bw_qmatmul.restype = i32
    L.bw_qmatmul_fused.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, vp, vp, i32, i32, i32, ctypes.POINTER(Epilogue), vp, sz, vp]
    L.bw_qmatmul_fused.restype = i32
    L.bw_qmatmul_noalloc.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, vp, vp, i32, i32, i32, vp]
    L.bw_qmatmul_noalloc.restype = i32
    L.bw_qmatmul_noalloc_max_scratch_bytes.argtypes = []
    L.bw_qmatmul_noalloc_max_scratch_bytes.restype = sz
    L.bw_qmatmul_host.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, vp, vp, i32, i32, i32, vp, vp, vp,
                                  sz, vp]
    L.bw_qmatmul_host.restype = i32
    L.bw_qmatmul_grad_input.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, vp, i32, i32, vp]
    L.bw_qmatmul_grad_input.restype = i32
    L.bw_status_string.argtypes = [i32]
    L.bw_status_string.restype = ctypes.c_char_p
    L.bw_last_cuda_error.argtypes = []
    L.bw_last_cuda_error.restype = ctypes.c_char_p
    L.bw_last_qmatmul_kernel.argtypes = []
    L.bw_last_qmatmul_kernel.restype = ctypes.c_char_p
    L.bw_last_kernel.argtypes = []
    L.bw_last_kernel.restype = ctypes.c_char_p
    L.bw_version.argtypes = []
    L.bw_version.restype = i32
    L.bw_device_status.argtypes = []
    L.bw_device_status.restype = i32
    L.bw_selftest_division.argtypes = [ctypes.c_ulonglong, ctypes.c_ulonglong]
    L.bw_selftest_division.restype = ctypes.c_longlong


def lib():
    """Loads (building first if the .so is absent and nvcc is present) the native library."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    try:
                        from ..csrc.build import build
                        build()
                    except Exception as e:  # noqa: BLE001
                        raise RuntimeError(
                            "bitween_b200: the CUDA extension libbitween_b200.so is not built and could "
                            f"not be built here ({e}). Run `python -m bitween_b200.csrc.build`. "
                            "There is no CPU fallback.") from e
                L = ctypes.CDLL(LIB_PATH)
                _declare(L)
                _lib = L
    return _lib


def _takes_no_call(*args):
    return None


class _NoOperators:
    """Stands for the native host side of the operators where there is none: it takes no call."""
    kv_append = kv_read = kv_attend = adapter_matmul = rotate = kv_append_rotated = token_log_probs = staticmethod(_takes_no_call)


_host = None
_operators = None
# (compiled against torch's C++ interfaces: one for each Python and torch)
HOST_LIB_PATH = os.path.join(_PKG, "_C", f"_host_forward.{sys.implementation.cache_tag}.torch-{torch.__version__}.so")


def host_forward():
    """The native host side of a layer's forward (csrc/host_forward.cpp), loaded with the library and built with it.
    Where it can be neither loaded nor built (no g++, no torch headers), that is reported once, and what is returned
    takes no call: each goes through the autograd function, to the same kernels."""
    global _host, _operators
    if _host is None:
        L = lib()
        with _lock:
            if _host is None:
                try:
                    if not os.path.exists(HOST_LIB_PATH):
                        from ..csrc.build import build_host
                        build_host()
                    spec = importlib.util.spec_from_file_location("_host_forward", HOST_LIB_PATH)
                    module = importlib.util.module_from_spec(spec)
                    spec.loader.exec_module(module)
                    module.set_entry(ctypes.cast(L.bw_qmatmul, ctypes.c_void_p).value, _workspaces)
                    module.set_operators(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
                        L.bw_kv_append, L.bw_kv_read, L.bw_kv_attend, L.bw_kv_attend_workspace_bytes, L.bw_adapter_hidden_bytes,
                        L.bw_adapter_forward, L.bw_adapter_backward, L.bw_kv_attend_window, L.bw_kv_attend_window_workspace_bytes, L.bw_rotate,
                        L.bw_kv_append_rotated, L.bw_token_log_probs, L.bw_token_log_probs_grad)))
                    _operators = module
                    _host = module.forward
                except Exception as e:  # noqa: BLE001
                    warnings.warn(f"bitween_b200: forwards run without the native host side ({e})", stacklevel=2)
                    _operators = _NoOperators
                    _host = _takes_no_call
    return _host


def host_operators():
    """The native host side of the operators beside the linears (cache, rotary positions, adapters, log probabilities), from the same
    module: each takes plain calls and answers None to the others."""
    if _operators is None:
        host_forward()
    return _operators


def refuse_capture(name):
    """For backward passes of the Python path: which stream a gradient's consumer was recorded on is not known here, and where that is the default
    stream (a graph of the same leaves that still lives) torch does not survive handing it a captured gradient."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name}: this backward pass cannot be captured without the native host side of the operators, or of tensors that it does not take")


# (not public: where a torch build has no such function, recorders are not told from other modes)
_dispatch_modes = getattr(_python_dispatch, "_get_current_dispatch_mode_stack", tuple)


def any_tangent(*tensors):
    """Whether one of them has a forward-mode tangent.  (Only asked where a level of such is open.)"""
    return getattr(fwad, "_current_level", 0) >= 0 and any(t is not None and fwad.unpack_dual(t).tangent is not None for t in tensors)


def for_autograd(*tensors):
    """Whether a call that the native side has left is one for the operator's autograd function: recorded, traced, or with a tangent.  (Others are spared it.)"""
    return torch.jit.is_tracing() or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or any_tangent(*tensors)


def refuse_recorders(name, traced=False):
    """For the Python path of the operators, whose kernels are foreign calls: whoever writes torch operations down to run them again (make_fx, fake tensors) would keep the
    allocation of an output and nothing that fills it.  `traced`: so would torch.jit.trace, which keeps an autograd function, where there is one, whole."""
    if (traced and torch.jit.is_tracing()) or any(getattr(mode, "_mode_key", None) is not None for mode in _dispatch_modes()):
        raise RuntimeError(f"{name}: calls of this library cannot be recorded as torch operations")


def check(status):
    if status != 0:
        L = lib()
        text = L.bw_status_string(status).decode()
        if status == 8:
            text += ": " + L.bw_last_cuda_error().decode()
        raise BitweenKernelError(status, text)


def require_cuda(t, name):
    if not t.is_cuda:
        raise RuntimeError(f"bitween_b200: `{name}` must be a CUDA tensor; this library has no CPU path")
    return t


def stream_ptr(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# (not public: where a torch build has no such function, the public way, 1 us a call slower, is used)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def raw_stream(device):
    """The current stream of `device` as an integer handle."""
    return _raw_stream(device.index) if _raw_stream else torch.cuda.current_stream(device).cuda_stream


_NO_GUARD = contextlib.nullcontext()


def on_device(device):
    """Context in which `device` is the current one; nothing is switched when it already is."""
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


_workspaces = {}


def _capturing(raw_stream):
    # (the default stream, handle 0, cannot be captured)
    return raw_stream != 0 and torch.cuda.is_current_stream_capturing()


def workspace(device, nbytes):
    """Scratch for one bw_qmatmul call on the current stream of `device` (the current device).

    Outside captures it is cached per (device, stream) and only grows: calls that may overlap on the GPU must not
    share scratch, and calls on one stream are ordered.  A captured call takes scratch of its own from the graph's
    memory pool instead: torch captures every graph on the same stream, but graphs are replayed on any."""
    if nbytes == 0:
        return None
    stream = raw_stream(device)
    if _capturing(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, stream)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 21), dtype=torch.uint8, device=device)
        _workspaces[key] = buf
    return buf


def current_workspace(device, raw_stream):
    """The scratch `workspace` would return on this stream if it is large enough; None before the first call
    and inside a capture."""
    return None if _capturing(raw_stream) else _workspaces.get((device.index, raw_stream))


def last_qmatmul_kernel():
    return lib().bw_last_qmatmul_kernel().decode()


def last_kernel():
    return lib().bw_last_kernel().decode()
