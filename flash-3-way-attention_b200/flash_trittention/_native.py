"""ctypes binding of ``libtritt_sm100.so`` (declared in ``include/tritt.h``).

The library is the only compute path: if it is missing, loading raises and every entry
point of the package fails loudly.  There is no PyTorch or CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import functools
import importlib
import os
import threading
import warnings

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libtritt_sm100.so")

F32, F16, BF16 = 0, 1, 2
OP_TDP_FWD, OP_TDP_BWD, OP_DPS_FWD, OP_DPS_BWD = 0, 1, 2, 3
OP_TDP_DECODE, OP_DPS_APPEND, OP_DPS_DECODE = 4, 5, 6
CODES = {torch.float16: 0, torch.float8_e4m3fn: 1, torch.int8: 2}  # what a cached element is held in
FLAG_FORCE_SIMT, FLAG_BWD_PARTIAL, FLAG_WIDE_OPERANDS, FLAG_BWD_CTA_PAIRS = 1, 2, 4, 8
PATH_SIMT, PATH_TCGEN05 = 0, 1

_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}

# every symbol include/tritt.h declares
SYMBOLS = (
    "tritt_version", "tritt_kernel_launches", "tritt_last_error", "tritt_workspace_bytes", "tritt_workspace_bytes_flags",
    "tritt_tdp_fwd_workspace", "tritt_tdp_fwd_min_workspace", "tritt_tdp_path", "tritt_dps_path", "tritt_tdp_fwd",
    "tritt_tdp_bwd", "tritt_tdp_bwd_finalize", "tritt_tdp_bwd_partials_offset", "tritt_dps_fwd",
    "tritt_dps_bwd", "tritt_dps_bwd_saved", "tritt_selftest_umma", "tritt_selftest_wait_expiry", "tritt_tdp_fwd_noalloc",
    "tritt_noalloc_scratch_bytes", "tritt_selftest_bwd_registers",
    "tritt_tdp_bwd_plan", "tritt_qk_norm_rotary_fwd", "tritt_qk_norm_rotary_bwd", "tritt_qk_norm_rotary_workspace",
    "tritt_qk_norm_rotary_axes_fwd", "tritt_qk_norm_rotary_axes_bwd",
    "tritt_cache_write", "tritt_cache_read", "tritt_tdp_decode", "tritt_dps_append", "tritt_dps_decode", "tritt_decode_workspace",
    "tritt_decode_path", "tritt_tdp_weigh", "tritt_tdp_weigh_workspace", "tritt_dps_weigh", "tritt_cache_evict",
)

_lib = None
_host = None  # the extension module, once lib() has loaded it
_lock = threading.Lock()
_status = {}  # device index -> pinned int32 status word (created under _lock)
_status_np = {}  # device index -> numpy view of the same word (a host read without any tensor machinery)
_status_ptr = {}  # device index -> address of the same word
launches = 0  # kernels-enqueuing library calls made by this process (bench bookkeeping)


class TrittError(RuntimeError):
    pass


class Rows(C.Structure):
    """``tritt_rows_t``: rows of a [B, N, T, D] tensor by its strides."""

    _fields_ = [("p", C.c_void_p), ("stride_b", C.c_longlong), ("stride_n", C.c_longlong), ("stride_t", C.c_longlong)]


class NormRotary(C.Structure):
    """``tritt_norm_rotary_t``."""

    _fields_ = [("x", Rows * 3), ("y", Rows * 3), ("dx", Rows * 3), ("w", C.c_void_p * 3), ("dw", C.c_void_p * 3),
                ("cos", C.c_void_p), ("sin", C.c_void_p), ("positions", C.c_void_p), ("position_stride_b", C.c_longlong),
                ("position_stride_t", C.c_longlong), ("positions64", C.c_int), ("table", C.c_int), ("rot", C.c_int),
                ("interleaved", C.c_int), ("weight_heads", C.c_int), ("weight_dtype", C.c_int), ("B", C.c_int), ("N", C.c_int),
                ("T", C.c_int), ("D", C.c_int), ("dtype", C.c_int), ("eps", C.c_float)]


class Axes(C.Structure):
    """``tritt_axes_t``."""

    _fields_ = [("position_stride", C.c_longlong), ("count", C.c_int), ("of", C.c_ubyte * 32)]


class Cache(C.Structure):
    """``tritt_cache_t``."""

    _fields_ = [("codes", C.c_void_p), ("exponents", C.c_void_p), ("lse", C.c_void_p), ("pages", C.c_int), ("page_size", C.c_int),
                ("N", C.c_int), ("D", C.c_int), ("code", C.c_int), ("table", C.c_void_p), ("table_stride", C.c_longlong),
                ("table_pages", C.c_int), ("context", C.c_void_p), ("counts", C.c_void_p), ("ancestors", C.c_void_p), ("B", C.c_int),
                ("n", C.c_int)]


class Weights(C.Structure):
    """``tritt_weights_t``."""

    _fields_ = [("before", C.c_void_p), ("after", C.c_void_p), ("before_stride_b", C.c_longlong), ("before_stride_n", C.c_longlong),
                ("after_stride_b", C.c_longlong), ("after_stride_n", C.c_longlong), ("before_length", C.c_int), ("after_length", C.c_int),
                ("decay", C.c_float)]


def host_forward(*args):
    """A whole forward call by the native extension, ``csrc/host/tritt_host.cpp`` (whose function takes this one's place once
    ``lib()`` has loaded it), or ``None``: the call is one for the Python code."""


def host_backward(*args):
    """The same for a backward call."""


def host_norm_rotary(*args):
    """The same for ``qk_norm_rotary``, ..."""


def host_norm_rotary_backward(*args):
    """... its backward,"""


def host_cache_write(*args):
    """``cache_write``,"""


def host_cache_read(*args):
    """``cache_read``,"""


def host_decode(*args):
    """``tdp_decode``, ``dps_append`` and ``dps_decode``,"""


def host_weigh(*args):
    """``tdp_weigh`` and ``dps_weigh``,"""


def host_evict(*args):
    """``cache_evict``."""


def _load_host(L):
    global _host, host_forward, host_backward, host_norm_rotary, host_norm_rotary_backward, host_cache_write, host_cache_read, host_decode
    global host_weigh, host_evict
    try:
        host = importlib.import_module("._host", __package__)
        built_for = getattr(host, "torch_version", "another version")
        if built_for != torch.__version__:
            raise ImportError(f"built for PyTorch {built_for}, not {torch.__version__}")
    except ImportError as e:
        warnings.warn(f"the host extension of flash_trittention cannot be loaded ({e}): short calls take twice as long; build it "
                      "with `python flash-3-way-attention_b200/build.py`", stacklevel=3)
        return
    _host = host
    # (the order is that of the extension's own list)
    _host.init(*(C.cast(getattr(L, "tritt_" + name), C.c_void_p).value for name in (
        "tdp_fwd", "tdp_bwd", "dps_fwd", "dps_bwd", "dps_bwd_saved", "workspace_bytes_flags", "tdp_fwd_workspace", "qk_norm_rotary_fwd",
        "qk_norm_rotary_bwd", "qk_norm_rotary_workspace", "cache_write", "cache_read", "tdp_decode", "dps_append", "dps_decode",
        "decode_workspace", "qk_norm_rotary_axes_fwd", "qk_norm_rotary_axes_bwd", "tdp_weigh", "tdp_weigh_workspace", "dps_weigh", "cache_evict")))
    for device, address in _status_ptr.items():
        _host.set_status(device, address)
    host_forward, host_backward = _host.forward, _host.backward
    host_norm_rotary, host_norm_rotary_backward = _host.norm_rotary, _host.norm_rotary_backward
    host_cache_write, host_cache_read, host_decode = _host.cache_write, _host.cache_read, _host.decode
    host_weigh, host_evict = _host.weigh, _host.cache_evict


def lib():
    """Loads the shared library on first use."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    raise TrittError(
                        f"{LIB_PATH} not found: build it with `python flash-3-way-attention_b200/build.py` "
                        "(there is no fallback path)")
                L = C.CDLL(LIB_PATH)
                vp, i, f, sz = C.c_void_p, C.c_int, C.c_float, C.c_size_t
                L.tritt_version.restype = i
                L.tritt_kernel_launches.restype = C.c_ulonglong
                L.tritt_last_error.restype = C.c_char_p
                L.tritt_workspace_bytes.restype = sz
                L.tritt_workspace_bytes.argtypes = [i] * 6
                L.tritt_workspace_bytes_flags.restype = sz
                L.tritt_workspace_bytes_flags.argtypes = [i] * 7
                L.tritt_tdp_fwd_workspace.restype = sz
                L.tritt_tdp_fwd_workspace.argtypes = [i] * 12
                L.tritt_tdp_fwd_min_workspace.restype = sz
                L.tritt_tdp_fwd_min_workspace.argtypes = [i] * 11
                L.tritt_tdp_path.restype = i
                L.tritt_tdp_path.argtypes = [i] * 10
                L.tritt_dps_path.restype = i
                L.tritt_dps_path.argtypes = [i] * 5
                L.tritt_tdp_bwd_partials_offset.restype = sz
                L.tritt_tdp_bwd_partials_offset.argtypes = [i] * 5
                L.tritt_tdp_fwd.restype = i
                L.tritt_tdp_fwd.argtypes = [vp] * 7 + [i] * 5 + [f] + [i] * 7 + [vp, sz, vp, i, vp]
                L.tritt_tdp_bwd.restype = i
                L.tritt_tdp_bwd.argtypes = [vp] * 13 + [i] * 5 + [f] + [i] * 7 + [vp, sz, vp, i, vp]
                L.tritt_tdp_bwd_finalize.restype = i
                L.tritt_tdp_bwd_finalize.argtypes = [vp] * 5 + [i] * 5 + [vp, sz, vp]
                L.tritt_dps_fwd.restype = i
                L.tritt_dps_fwd.argtypes = [vp] * 7 + [i] * 5 + [f] + [i] * 2 + [vp, sz, vp, i, vp]
                L.tritt_dps_bwd.restype = i
                L.tritt_dps_bwd.argtypes = [vp] * 13 + [i] * 5 + [f] + [i] * 2 + [vp, sz, vp, i, vp]
                L.tritt_dps_bwd_saved.restype = i
                L.tritt_dps_bwd_saved.argtypes = [vp] * 13 + [i] * 5 + [f] + [i] * 2 + [vp, sz, vp, sz, vp, i, vp]
                L.tritt_tdp_fwd_noalloc.restype = i
                L.tritt_tdp_fwd_noalloc.argtypes = [vp] * 7 + [i] * 5 + [f] + [i] * 5 + [vp, i, vp]
                L.tritt_noalloc_scratch_bytes.restype = sz
                L.tritt_selftest_bwd_registers.restype = i
                L.tritt_selftest_bwd_registers.argtypes = [i]
                L.tritt_tdp_bwd_plan.restype = i
                L.tritt_tdp_bwd_plan.argtypes = [i] * 11 + [vp]
                L.tritt_selftest_umma.restype = i
                L.tritt_selftest_umma.argtypes = [vp] * 5 + [i, vp, vp]
                L.tritt_selftest_wait_expiry.restype = i
                L.tritt_selftest_wait_expiry.argtypes = [i, C.c_longlong, vp, vp]
                norm, cache, rows = C.POINTER(NormRotary), C.POINTER(Cache), C.POINTER(Rows)
                L.tritt_qk_norm_rotary_fwd.argtypes = [norm, vp, vp]
                L.tritt_qk_norm_rotary_bwd.argtypes = [norm, vp, sz, vp, vp]
                L.tritt_qk_norm_rotary_axes_fwd.argtypes = [norm, C.POINTER(Axes), vp, vp]
                L.tritt_qk_norm_rotary_axes_bwd.argtypes = [norm, C.POINTER(Axes), vp, sz, vp, vp]
                L.tritt_qk_norm_rotary_workspace.argtypes = [norm]
                L.tritt_qk_norm_rotary_workspace.restype = sz
                L.tritt_cache_write.argtypes = [cache, rows, i, vp, vp]
                L.tritt_cache_read.argtypes = [cache, vp, vp, i, vp, vp]
                L.tritt_tdp_decode.argtypes = [cache, rows, vp, vp, i, f] + [i] * 4 + [vp, sz, vp, i, vp]
                L.tritt_dps_append.argtypes = [cache, rows, i, f, i, vp, sz, vp, i, vp]
                L.tritt_dps_decode.argtypes = [cache, rows, vp, vp, i, f, vp, sz, vp, i, vp]
                L.tritt_decode_workspace.argtypes = [i, cache] + [i] * 4
                L.tritt_decode_workspace.restype = sz
                L.tritt_decode_path.argtypes = [i] * 4
                weights = C.POINTER(Weights)
                L.tritt_tdp_weigh.argtypes = [cache, weights, rows, vp, i, f] + [i] * 4 + [vp, sz, vp, vp]
                L.tritt_tdp_weigh_workspace.argtypes = [cache, i, i]
                L.tritt_tdp_weigh_workspace.restype = sz
                L.tritt_dps_weigh.argtypes = [cache, weights, rows, rows, vp, i, f, i, vp, vp]
                L.tritt_cache_evict.argtypes = [cache, weights, vp, C.c_longlong] + [i] * 4 + [vp] * 4
                for name in ("tdp_weigh", "dps_weigh", "cache_evict", "qk_norm_rotary_fwd", "qk_norm_rotary_bwd", "qk_norm_rotary_axes_fwd", "qk_norm_rotary_axes_bwd", "cache_write", "cache_read", "tdp_decode", "dps_append", "dps_decode",
                             "decode_path"):
                    getattr(L, "tritt_" + name).restype = i
                _load_host(L)
                _lib = L
    return _lib


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPES[dt]
    except KeyError:
        raise ValueError(f"unsupported dtype {dt}: expected float32, float16 or bfloat16") from None


def host_result(out, what: str):
    """What a call of the extension returned, its tensors or 0; an error code is raised."""
    global launches
    if out.__class__ is int and out:
        _check(out, what)
    launches += 1
    return out


def _check(rc: int, what: str):
    if rc != 0:
        msg = lib().tritt_last_error().decode("utf-8", "replace")
        if rc < 0:
            raise ValueError(f"{what}: {msg} (code {rc})")
        raise TrittError(f"{what}: {msg} (CUDA error {rc})")


STATUS_BITS = {1: "self-test kernel", 2: "triple-dot-product forward", 4: "triple-dot-product backward",
               8: "shared memory of a tensor-core kernel was not 1024-byte aligned",
               16: "soft-max attention forward (dot-product-sum)", 32: "soft-max attention backward (dot-product-sum)",
               64: "an input element beyond the fp16 operand range (65504) in an fp32 / wide-operand call",
               128: "wait-expiry self-test", 256: "a rotation whose position its tables do not have",
               512: "a token without a place in its cache", 1024: "triple-dot-product attention over a cache (or more new tokens times cached ones than it can count)"}


def _device_index(device) -> int:
    d = torch.device(device)
    return torch.cuda.current_device() if d.index is None else d.index


def status_word(device) -> torch.Tensor:
    """Per-device int32 that kernels OR a code into when a bounded barrier wait ran out.

    The word lives in page-locked host memory, which the GPU addresses directly (unified addressing): only a
    kernel that gives up ever writes it, and the host can look at it without a copy or a synchronisation."""
    key = _device_index(device)
    t = _status.get(key)
    if t is None:
        with _lock:
            t = _status.get(key)
            if t is None:
                t = torch.zeros(1, dtype=torch.int32).pin_memory()
                _status_np[key] = t.numpy()
                _status_ptr[key] = t.data_ptr()
                _status[key] = t
                if _host is not None:
                    _host.set_status(key, t.data_ptr())
    return t


def _status_address(device: torch.device) -> int:
    """Address of ``status_word(device)`` (the word is never freed)."""
    ptr = _status_ptr.get(device.index)
    return status_word(device).data_ptr() if ptr is None else ptr


def _describe(v: int) -> str:
    return ", ".join(name for bit, name in STATUS_BITS.items() if v & bit) or f"code {v}"


def read_status(device) -> int:
    """Synchronises the device and returns (then clears) its kernel status word."""
    torch.cuda.synchronize(torch.device("cuda", _device_index(device)))
    t = status_word(device)
    v = int(t[0])
    if v:
        t.zero_()
    return v


def check_status(device=None, synchronize: bool = True) -> None:
    """Raises ``TrittError`` if a kernel enqueued earlier on ``device`` gave up on a bounded wait (its results are
    then invalid).  With ``synchronize=False`` only kernels that have already finished are seen; every compute
    entry point of this module makes that cheap check on entry, so a time-out surfaces at the latest on the next
    call after the failed kernel has retired."""
    if not synchronize:
        # the per-call check: one host read of the pinned word
        idx = device.index if isinstance(device, torch.device) else None
        arr = _status_np.get(idx) if idx is not None else None
        if arr is not None and arr[0] == 0:
            return
    dev = _device_index(torch.cuda.current_device() if device is None else device)
    if synchronize:
        v = read_status(dev)
    else:
        t = status_word(dev)
        v = int(t[0])
        if v:
            t.zero_()
    if v:
        raise TrittError(f"a kernel of an earlier call on cuda:{dev} reported a failure: gave up waiting on a barrier "
                         f"after its time limit, or met unusable input ({_describe(v)}); the results of that call "
                         "are invalid")


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(op: int, B: int, N: int, T: int, D: int, dtype: int, flags: int) -> int:
    return max(int(lib().tritt_workspace_bytes_flags(op, B, N, T, D, dtype, flags)), 256)


@functools.lru_cache(maxsize=1024)
def _tdp_fwd_workspace_bytes(*args) -> int:
    return max(int(lib().tritt_tdp_fwd_workspace(*args)), 256)


def tdp_fwd_workspace(B: int, N: int, T: int, D: int, dtype: int, causal, k1w, k2w, kkl, kkr, device, q_mod: int = 1,
                      flags: int = 0) -> torch.Tensor:
    """What a forward with these windows makes use of (``workspace`` holds the most that any mask does)."""
    n = _tdp_fwd_workspace_bytes(B, N, T, D, dtype, int(bool(causal)), _win(k1w, T), _win(k2w, T), _win(kkl, T), _win(kkr, T), q_mod,
                                 flags)
    return torch.empty(n, dtype=torch.uint8, device=device)


def workspace(op: int, B: int, N: int, T: int, D: int, dtype: int, device, flags: int = 0) -> torch.Tensor:
    return torch.empty(_workspace_bytes(op, B, N, T, D, dtype, flags), dtype=torch.uint8, device=device)


def aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` made contiguous and, if its storage offset leaves it off a 16-byte boundary (a view into a larger
    buffer), copied: the library's vector and TMA accesses require that alignment and reject other pointers."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def strided(t: torch.Tensor) -> torch.Tensor:
    """``t`` ([B, N, T, D]) itself if its rows are contiguous and start on 16-byte boundaries, whatever its other strides; else
    a contiguous copy."""
    unit = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(st % unit == 0 or size == 1 for st, size in zip(t.stride()[:3], t.shape)):
        return t
    return aligned(t.contiguous())


def rows(t: torch.Tensor) -> Rows:
    """The rows of a tensor that ``strided`` has returned."""
    b, n, tt = (st if size > 1 else 0 for st, size in zip(t.stride()[:3], t.shape))
    return Rows(t.data_ptr(), b, n, tt)


# The current stream's handle and the current device without the Python objects around them (a call of a short sequence
# takes as long to enqueue as to run: the stream object alone is 1-2 us of ~45).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream(dev: torch.device) -> int:
    return _raw_stream(dev.index) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


class _on_device:
    """``torch.cuda.device(dev)`` only when ``dev`` is not already the current device (the common case costs one
    query instead of a get / set / restore)."""

    __slots__ = ("ctx",)

    def __init__(self, dev: torch.device):
        self.ctx = None if dev.index == _current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            return self.ctx.__exit__(*exc)
        return False


def _win(w, T):
    return T if w is None else int(w)


def tdp_path(op, T, D, dtype, causal, k1w, k2w, kkl, kkr, flags=0) -> int:
    return lib().tritt_tdp_path(op, T, D, dtype, int(bool(causal)), _win(k1w, T), _win(k2w, T), _win(kkl, T),
                                _win(kkr, T), flags)


def dps_path(T, D, dtype, k_diff, flags=0) -> int:
    return lib().tritt_dps_path(T, D, dtype, int(k_diff), flags)


def tdp_fwd(q, k1, k2, v1, v2, o, lse, alpha, causal, k1w, k2w, kkl, kkr, q_mod=1, q_rem=0, flags=0, ws=None):
    """``ws``: a caller-provided workspace (uint8 tensor) instead of one of ``tritt_tdp_fwd_workspace`` bytes."""
    global launches
    B, N, T, D = q.shape
    dt = dtype_code(q.dtype)
    check_status(q.device, synchronize=False)
    with _on_device(q.device):
        if ws is None:
            ws = tdp_fwd_workspace(B, N, T, D, dt, causal, k1w, k2w, kkl, kkr, q.device, q_mod, flags)
        rc = lib().tritt_tdp_fwd(q.data_ptr(), k1.data_ptr(), k2.data_ptr(), v1.data_ptr(), v2.data_ptr(),
                                 o.data_ptr(), lse.data_ptr(), B, N, T, D, dt, float(alpha), int(bool(causal)),
                                 _win(k1w, T), _win(k2w, T), _win(kkl, T), _win(kkr, T), q_mod, q_rem,
                                 ws.data_ptr(), ws.numel(), _status_address(q.device), flags, _stream(q.device))
    _check(rc, "tritt_tdp_fwd")
    launches += 1


def tdp_bwd(q, k1, k2, v1, v2, o, do, lse, dq, dk1, dk2, dv1, dv2, alpha, causal, k1w, k2w, kkl, kkr,
            q_mod=1, q_rem=0, flags=0, ws=None):
    """Returns the workspace tensor (holds the fp32 partial sums when FLAG_BWD_PARTIAL is set)."""
    global launches
    B, N, T, D = q.shape
    dt = dtype_code(q.dtype)
    ptr = lambda t: 0 if t is None else t.data_ptr()
    check_status(q.device, synchronize=False)
    with _on_device(q.device):
        if ws is None:
            ws = workspace(OP_TDP_BWD, B, N, T, D, dt, q.device, flags)
        rc = lib().tritt_tdp_bwd(q.data_ptr(), k1.data_ptr(), k2.data_ptr(), v1.data_ptr(), v2.data_ptr(),
                                 o.data_ptr(), do.data_ptr(), lse.data_ptr(), dq.data_ptr(), ptr(dk1), ptr(dk2),
                                 ptr(dv1), ptr(dv2), B, N, T, D, dt, float(alpha), int(bool(causal)),
                                 _win(k1w, T), _win(k2w, T), _win(kkl, T), _win(kkr, T), q_mod, q_rem,
                                 ws.data_ptr(), ws.numel(), _status_address(q.device), flags, _stream(q.device))
    _check(rc, "tritt_tdp_bwd")
    launches += 1
    return ws


def tdp_bwd_plan(T, D, dtype, causal, k1w, k2w, kkl, kkr, q_mod=1, q_rem=0, flags=0):
    """(query rows in exact fp32, cells executed on the tensor cores, by the kernel that steps over queries) of one head of a
    backward call."""
    out = (C.c_longlong * 3)()
    _check(lib().tritt_tdp_bwd_plan(T, D, dtype, int(bool(causal)), _win(k1w, T), _win(k2w, T), _win(kkl, T), _win(kkr, T),
                                    q_mod, q_rem, flags, out), "tritt_tdp_bwd_plan")
    return tuple(out)


def tdp_bwd_finalize(v1, dk1, dk2, dv1, dv2, ws):
    global launches
    B, N, T, D = v1.shape
    check_status(v1.device, synchronize=False)
    with _on_device(v1.device):
        rc = lib().tritt_tdp_bwd_finalize(v1.data_ptr(), dk1.data_ptr(), dk2.data_ptr(), dv1.data_ptr(),
                                          dv2.data_ptr(), B, N, T, D, dtype_code(v1.dtype), ws.data_ptr(),
                                          ws.numel(), _stream(v1.device))
    _check(rc, "tritt_tdp_bwd_finalize")
    launches += 1


def dps_fwd(q, k1, k2, v1, v2, o, m, alpha, causal, k_diff, flags=0):
    """Returns the workspace tensor: handed to ``dps_bwd(..., fwd_ws=...)`` it spares the backward the inner
    attention's recomputation (keep it untouched until then)."""
    global launches
    B, N, T, D = q.shape
    dt = dtype_code(q.dtype)
    check_status(q.device, synchronize=False)
    with _on_device(q.device):
        ws = workspace(OP_DPS_FWD, B, N, T, D, dt, q.device)
        rc = lib().tritt_dps_fwd(q.data_ptr(), k1.data_ptr(), k2.data_ptr(), v1.data_ptr(), v2.data_ptr(),
                                 o.data_ptr(), m.data_ptr(), B, N, T, D, dt, float(alpha), int(bool(causal)),
                                 int(k_diff), ws.data_ptr(), ws.numel(), _status_address(q.device), flags,
                                 _stream(q.device))
    _check(rc, "tritt_dps_fwd")
    launches += 1
    return ws


def dps_bwd(q, k1, k2, v1, v2, o, do, m, dq, dk1, dk2, dv1, dv2, alpha, causal, k_diff, flags=0, fwd_ws=None):
    """``fwd_ws``: the tensor ``dps_fwd`` returned for the same inputs, if it was kept untouched."""
    global launches
    B, N, T, D = q.shape
    dt = dtype_code(q.dtype)
    check_status(q.device, synchronize=False)
    with _on_device(q.device):
        ws = workspace(OP_DPS_BWD, B, N, T, D, dt, q.device)
        args = (q.data_ptr(), k1.data_ptr(), k2.data_ptr(), v1.data_ptr(), v2.data_ptr(), o.data_ptr(), do.data_ptr(),
                m.data_ptr(), dq.data_ptr(), dk1.data_ptr(), dk2.data_ptr(), dv1.data_ptr(), dv2.data_ptr(), B, N, T, D,
                dt, float(alpha), int(bool(causal)), int(k_diff), ws.data_ptr(), ws.numel())
        if fwd_ws is None:
            rc = lib().tritt_dps_bwd(*args, _status_address(q.device), flags, _stream(q.device))
        else:
            rc = lib().tritt_dps_bwd_saved(*args, fwd_ws.data_ptr(), fwd_ws.numel(), _status_address(q.device),
                                           flags, _stream(q.device))
    _check(rc, "tritt_dps_bwd")
    launches += 1


def tdp_fwd_noalloc(q, k1, k2, v1, v2, o, lse, alpha, causal, k1w, k2w, kkl, kkr, flags=0):
    """Forward through ``tritt_tdp_fwd_noalloc``: no workspace is passed; the library uses the scratch
    array built into its device image (for callers that are not allowed to allocate device memory).
    Calls on one GPU must not overlap in time."""
    global launches
    B, N, T, D = q.shape
    check_status(q.device, synchronize=False)
    with _on_device(q.device):
        rc = lib().tritt_tdp_fwd_noalloc(q.data_ptr(), k1.data_ptr(), k2.data_ptr(), v1.data_ptr(), v2.data_ptr(),
                                         o.data_ptr(), lse.data_ptr(), B, N, T, D, dtype_code(q.dtype), float(alpha),
                                         int(bool(causal)), _win(k1w, T), _win(k2w, T), _win(kkl, T), _win(kkr, T),
                                         _status_address(q.device), flags, _stream(q.device))
    _check(rc, "tritt_tdp_fwd_noalloc")
    launches += 1


def norm_rotary(a: NormRotary, dev: torch.device, backward: bool = False, axes: Axes | None = None):
    global launches
    check_status(dev, synchronize=False)
    L = lib()
    with _on_device(dev):
        if backward:
            n = int(L.tritt_qk_norm_rotary_workspace(C.byref(a)))
            ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
            rest = (0 if ws is None else ws.data_ptr(), n, _status_address(dev), _stream(dev))
        else:
            rest = (_status_address(dev), _stream(dev))
        if axes is not None:
            rc = (L.tritt_qk_norm_rotary_axes_bwd if backward else L.tritt_qk_norm_rotary_axes_fwd)(C.byref(a), C.byref(axes), *rest)
        else:
            rc = (L.tritt_qk_norm_rotary_bwd if backward else L.tritt_qk_norm_rotary_fwd)(C.byref(a), *rest)
    _check(rc, "tritt_qk_norm_rotary")
    launches += 1


def cache_write(c: Cache, new, dtype: int, dev: torch.device):
    global launches
    check_status(dev, synchronize=False)
    with _on_device(dev):
        rc = lib().tritt_cache_write(C.byref(c), (Rows * 4)(*(rows(t) for t in new)), dtype, _status_address(dev), _stream(dev))
    _check(rc, "tritt_cache_write")
    launches += 1


def cache_read(c: Cache, parts, lse, dtype: int, dev: torch.device):
    global launches
    check_status(dev, synchronize=False)
    with _on_device(dev):
        rc = lib().tritt_cache_read(C.byref(c), (C.c_void_p * 4)(*(t.data_ptr() for t in parts)), 0 if lse is None else lse.data_ptr(),
                                    dtype, _status_address(dev), _stream(dev))
    _check(rc, "tritt_cache_read")
    launches += 1


def _decode_scratch(op, c, dtype, k1w, k2w, flags, dev):
    return torch.empty(max(int(lib().tritt_decode_workspace(op, C.byref(c), dtype, k1w, k2w, flags)), 256), dtype=torch.uint8, device=dev)


def tdp_decode(c: Cache, q, o, lse, alpha, k1w, k2w, kkl, kkr, flags=0):
    global launches
    dev, dt = q.device, dtype_code(q.dtype)
    check_status(dev, synchronize=False)
    with _on_device(dev):
        ws = _decode_scratch(OP_TDP_DECODE, c, dt, k1w, k2w, flags, dev)
        rc = lib().tritt_tdp_decode(C.byref(c), C.byref(rows(q)), o.data_ptr(), 0 if lse is None else lse.data_ptr(), dt, alpha, k1w, k2w,
                                    kkl, kkr, ws.data_ptr(), ws.numel(), _status_address(dev), flags, _stream(dev))
    _check(rc, "tritt_tdp_decode")
    launches += 1


def dps_append(c: Cache, new, alpha, k_diff, flags=0):
    global launches
    dev, dt = new[0].device, dtype_code(new[0].dtype)
    check_status(dev, synchronize=False)
    with _on_device(dev):
        ws = _decode_scratch(OP_DPS_APPEND, c, dt, 0, 0, flags, dev)
        rc = lib().tritt_dps_append(C.byref(c), (Rows * 4)(*(rows(t) for t in new)), dt, alpha, k_diff, ws.data_ptr(), ws.numel(),
                                    _status_address(dev), flags, _stream(dev))
    _check(rc, "tritt_dps_append")
    launches += 1


def dps_decode(c: Cache, q, o, m, alpha, flags=0):
    global launches
    dev, dt = q.device, dtype_code(q.dtype)
    check_status(dev, synchronize=False)
    with _on_device(dev):
        ws = _decode_scratch(OP_DPS_DECODE, c, dt, 0, 0, flags, dev)
        rc = lib().tritt_dps_decode(C.byref(c), C.byref(rows(q)), o.data_ptr(), 0 if m is None else m.data_ptr(), dt, alpha, ws.data_ptr(),
                                    ws.numel(), _status_address(dev), flags, _stream(dev))
    _check(rc, "tritt_dps_decode")
    launches += 1


def decode_path(op, D, dtype, flags=0) -> int:
    return lib().tritt_decode_path(op, D, dtype, flags)


def tdp_weigh(c: Cache, w: Weights, q, lse, alpha, k1w, k2w, kkl, kkr):
    global launches
    dev = q.device
    check_status(dev, synchronize=False)
    with _on_device(dev):
        ws = torch.empty(max(int(lib().tritt_tdp_weigh_workspace(C.byref(c), k1w, k2w)), 256), dtype=torch.uint8, device=dev)
        rc = lib().tritt_tdp_weigh(C.byref(c), C.byref(w), C.byref(rows(q)), lse.data_ptr(), dtype_code(q.dtype), alpha, k1w, k2w, kkl, kkr,
                                   ws.data_ptr(), ws.numel(), _status_address(dev), _stream(dev))
    _check(rc, "tritt_tdp_weigh")
    launches += 1


def dps_weigh(c: Cache, w: Weights, q, k2, m, alpha, k_diff):
    global launches
    dev = q.device
    check_status(dev, synchronize=False)
    with _on_device(dev):
        rc = lib().tritt_dps_weigh(C.byref(c), C.byref(w), C.byref(rows(q)), C.byref(rows(k2)), m.data_ptr(), dtype_code(q.dtype), alpha, k_diff,
                                   _status_address(dev), _stream(dev))
    _check(rc, "tritt_dps_weigh")
    launches += 1


def cache_evict(c: Cache, w: Weights, table_out, keep, first, recent, context_out, kept):
    global launches
    dev = kept.device
    check_status(dev, synchronize=False)
    where = (0, 0, 0) if table_out is None else (table_out.data_ptr(), table_out.stride(0), table_out.shape[1])
    with _on_device(dev):
        rc = lib().tritt_cache_evict(C.byref(c), C.byref(w), *where, keep, first, recent, context_out.data_ptr(), kept.data_ptr(), _status_address(dev),
                                     _stream(dev))
    _check(rc, "tritt_cache_evict")
    launches += 1
