"""ctypes view of the C ABI in include/mfa_b200.h (libmfa_b200.so).

This is the boundary a non-Python host binds; the tests use it to call the kernels exactly
as such a host would: raw device pointers, sizes and a stream handle.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libmfa_b200.so"

# Every symbol declared in include/mfa_b200.h.
EXPORTED_SYMBOLS = (
    "mfa_fwd_f16",
    "mfa_fwd_simple_f16",
    "mfa_fwd_f16_noalloc",
    "mfa_fwd",
    "mfa_fwd_rows",
    "mfa_fwd_lse",
    "mfa_bwd",
    "mfa_fwd_window",
    "mfa_bwd_window",
    "mfa_fwd_window_rest",
    "mfa_bwd_window_rest",
    "mfa_extend_block_tables",
    "mfa_append_kv",
    "mfa_paged_attention",
    "mfa_shared_prefix_attention",
    "mfa_paged_workspace_bytes",
    "mfa_fwd_workspace_bytes",
    "mfa_last_error_string",
    "mfa_device_status",
    "mfa_set_watchdog_ns",
    "mfa_watchdog_selftest",
    "mfa_version",
)

MFA_OK = 0
MFA_ERR_INVALID_ARGUMENT = 1
MFA_ERR_HEAD_DIM = 2
MFA_ERR_SEQ_LEN = 3
MFA_ERR_CAUSAL = 4
MFA_ERR_CUDA = 5
MFA_ERR_DEVICE = 6
STATUS_TIMEOUT_BASE = 0x100
STATUS_BAD_PAGE = 0x200
NOALLOC_SCRATCH_BYTES = 20971520  # MFA_NOALLOC_SCRATCH_BYTES
DTYPE_FP16, DTYPE_BF16 = 0, 1
LAYOUT_BHND, LAYOUT_BNHD = 0, 1

_LIB: ctypes.CDLL | None = None


class MfaError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


def load(path: str | Path | None = None) -> ctypes.CDLL:
    """Load libmfa_b200.so (once) and declare the C signatures."""
    global _LIB
    if _LIB is not None and path is None:
        return _LIB
    lib = ctypes.CDLL(str(path or LIB_PATH), mode=ctypes.RTLD_GLOBAL)
    fwd_args = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_float, ctypes.c_int32,
                ctypes.c_void_p]
    for name in ("mfa_fwd_f16", "mfa_fwd_simple_f16", "mfa_fwd_f16_noalloc"):
        fn = getattr(lib, name)
        fn.argtypes = fwd_args
        fn.restype = ctypes.c_int
    lib.mfa_fwd.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
                                                    ctypes.c_int32, ctypes.c_float, ctypes.c_int32,
                                                    ctypes.c_int32, ctypes.c_int32,
                                                    ctypes.c_void_p]
    lib.mfa_fwd.restype = ctypes.c_int
    lib.mfa_fwd_rows.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_int64] * 5 + [
        ctypes.c_int32, ctypes.c_float, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
        ctypes.c_void_p]
    lib.mfa_fwd_rows.restype = ctypes.c_int
    lib.mfa_fwd_lse.argtypes = [ctypes.c_void_p] * 5 + [ctypes.c_int64, ctypes.c_int64,
                                                        ctypes.c_int64, ctypes.c_int32,
                                                        ctypes.c_float, ctypes.c_int32,
                                                        ctypes.c_int32, ctypes.c_int32,
                                                        ctypes.c_void_p]
    lib.mfa_fwd_lse.restype = ctypes.c_int
    lib.mfa_bwd.argtypes = [ctypes.c_void_p] * 9 + [ctypes.c_int64, ctypes.c_int64,
                                                    ctypes.c_int64, ctypes.c_int32, ctypes.c_float,
                                                    ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                                    ctypes.c_void_p]
    lib.mfa_bwd.restype = ctypes.c_int
    window_args = [ctypes.c_int64] * 4 + [ctypes.c_int32, ctypes.c_int64, ctypes.c_int64,
                                          ctypes.c_float, ctypes.c_int32, ctypes.c_int32,
                                          ctypes.POINTER(ctypes.c_int64), ctypes.c_void_p]
    lib.mfa_fwd_window.argtypes = [ctypes.c_void_p] * 6 + window_args
    lib.mfa_fwd_window.restype = ctypes.c_int
    lib.mfa_bwd_window.argtypes = [ctypes.c_void_p] * 10 + window_args
    lib.mfa_bwd_window.restype = ctypes.c_int
    ptr, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    lib.mfa_fwd_window_rest.argtypes = [ptr] * 6 + [i64] + window_args
    lib.mfa_fwd_window_rest.restype = ctypes.c_int
    lib.mfa_bwd_window_rest.argtypes = [ptr] * 7 + [i64] + [ptr] * 3 + window_args
    lib.mfa_bwd_window_rest.restype = ctypes.c_int
    lib.mfa_extend_block_tables.argtypes = [ptr] * 7 + [i64] * 5 + [ptr]
    lib.mfa_append_kv.argtypes = [ptr] * 5 + [i64] * 9 + [ptr]
    lib.mfa_paged_attention.argtypes = [ptr] * 7 + [ctypes.c_uint64] + [i64] * 3 + [
        i32, *[i64] * 7, ctypes.c_float, i32, ptr]
    lib.mfa_shared_prefix_attention.argtypes = [ptr] * 4 + [i64] + [ptr] * 4 + [
        ctypes.c_uint64, *[i64] * 3, i32, *[i64] * 5, ctypes.c_float, i32, ptr]
    lib.mfa_paged_workspace_bytes.argtypes = [i64] * 3 + [i32] + [i64] * 3 + [
        ctypes.POINTER(ctypes.c_uint64)]
    for name in ("mfa_extend_block_tables", "mfa_append_kv", "mfa_paged_attention",
                 "mfa_shared_prefix_attention", "mfa_paged_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_int
    lib.mfa_last_error_string.argtypes = []
    lib.mfa_last_error_string.restype = ctypes.c_char_p
    lib.mfa_device_status.argtypes = [ctypes.c_int, ctypes.POINTER(ctypes.c_int), ctypes.c_int]
    lib.mfa_device_status.restype = ctypes.c_int
    lib.mfa_set_watchdog_ns.argtypes = [ctypes.c_uint64]
    lib.mfa_set_watchdog_ns.restype = ctypes.c_int
    lib.mfa_watchdog_selftest.argtypes = [ctypes.c_void_p, ctypes.c_uint64,
                                          ctypes.POINTER(ctypes.c_int)]
    lib.mfa_watchdog_selftest.restype = ctypes.c_int
    lib.mfa_version.argtypes = []
    lib.mfa_version.restype = ctypes.c_char_p
    lib.mfa_fwd_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
                                            ctypes.c_int32, ctypes.c_int32,
                                            ctypes.POINTER(ctypes.c_uint64)]
    lib.mfa_fwd_workspace_bytes.restype = ctypes.c_int
    if path is None:
        _LIB = lib
    return lib


def last_error() -> str:
    return load().mfa_last_error_string().decode()


def _check(rc: int) -> None:
    if rc != MFA_OK:
        raise MfaError(rc, last_error())


def fwd(q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, bh: int, n: int, d: int,
        scale: float, causal: bool = False, stream: int = 0, simple: bool = False) -> None:
    """Launch mfa_fwd_f16 (or mfa_fwd_simple_f16) on raw device pointers; raises MfaError."""
    lib = load()
    fn = lib.mfa_fwd_simple_f16 if simple else lib.mfa_fwd_f16
    _check(fn(q_ptr, k_ptr, v_ptr, out_ptr, bh, n, d, scale, int(causal), stream))


def fwd_noalloc(q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, bh: int, n: int, d: int,
                scale: float, causal: bool = False, stream: int = 0) -> None:
    """Launch mfa_fwd_f16_noalloc (no device allocation; static scratch shared by all calls
    on a device, so calls must not overlap on the GPU); raises MfaError."""
    _check(load().mfa_fwd_f16_noalloc(q_ptr, k_ptr, v_ptr, out_ptr, bh, n, d, scale,
                                       int(causal), stream))


def fwd_general(q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, batch: int, heads: int,
                n: int, d: int, scale: float, causal: bool = False, dtype: int = DTYPE_FP16,
                layout: int = LAYOUT_BHND, stream: int = 0) -> None:
    """Launch mfa_fwd (dtype and layout selectable); raises MfaError."""
    _check(load().mfa_fwd(q_ptr, k_ptr, v_ptr, out_ptr, batch, heads, n, d, scale, int(causal),
                          dtype, layout, stream))


def fwd_rows(q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, batch: int, heads: int,
             n: int, q_begin: int, q_end: int, d: int, scale: float, causal: bool = False,
             dtype: int = DTYPE_FP16, layout: int = LAYOUT_BHND, stream: int = 0) -> None:
    """Launch mfa_fwd_rows (query rows [q_begin, q_end) of every head); raises MfaError."""
    _check(load().mfa_fwd_rows(q_ptr, k_ptr, v_ptr, out_ptr, batch, heads, n, q_begin, q_end, d,
                               scale, int(causal), dtype, layout, stream))


def bwd(q_ptr: int, k_ptr: int, v_ptr: int, o_ptr: int, do_ptr: int, lse_ptr: int, dq_ptr: int,
        dk_ptr: int, dv_ptr: int, batch: int, heads: int, n: int, d: int, scale: float,
        causal: bool = False, dtype: int = DTYPE_FP16, layout: int = LAYOUT_BHND,
        stream: int = 0) -> None:
    """Launch mfa_bwd; raises MfaError."""
    _check(load().mfa_bwd(q_ptr, k_ptr, v_ptr, o_ptr, do_ptr, lse_ptr, dq_ptr, dk_ptr, dv_ptr,
                          batch, heads, n, d, scale, int(causal), dtype, layout, stream))


def _nine(strides):
    return None if strides is None else (ctypes.c_int64 * 9)(*strides)


def fwd_window(q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, lse_ptr: int, batch: int,
               heads: int, kv_heads: int, n: int, d: int, window: int, sinks: int, scale: float,
               dtype: int = DTYPE_FP16, layout: int = LAYOUT_BHND, stream: int = 0,
               strides: tuple[int, ...] | None = None, rest_ptr: int = 0,
               rest_rows: int | None = None) -> None:
    """Launch mfa_fwd_window (lse_ptr, rest_ptr 0: not written; strides: the nine (batch, head,
    token) element strides of q, k and v) or, with rest_rows, mfa_fwd_window_rest; raises
    MfaError."""
    tail = (batch, heads, kv_heads, n, d, window, sinks, scale, dtype, layout, _nine(strides),
            stream)
    if rest_rows is None:
        _check(load().mfa_fwd_window(q_ptr, k_ptr, v_ptr, out_ptr, lse_ptr, rest_ptr, *tail))
    else:
        _check(load().mfa_fwd_window_rest(q_ptr, k_ptr, v_ptr, out_ptr, lse_ptr, rest_ptr,
                                          rest_rows, *tail))


def bwd_window(q_ptr: int, k_ptr: int, v_ptr: int, o_ptr: int, do_ptr: int, lse_ptr: int,
               dq_ptr: int, dk_ptr: int, dv_ptr: int, batch: int, heads: int, kv_heads: int,
               n: int, d: int, window: int, sinks: int, scale: float, dtype: int = DTYPE_FP16,
               layout: int = LAYOUT_BHND, stream: int = 0,
               strides: tuple[int, ...] | None = None, rest_ptr: int = 0,
               rest_rows: int | None = None) -> None:
    """Launch mfa_bwd_window (strides as for fwd_window, rest_ptr 0: none) or, with rest_rows,
    mfa_bwd_window_rest; raises MfaError."""
    tail = (dq_ptr, dk_ptr, dv_ptr, batch, heads, kv_heads, n, d, window, sinks, scale, dtype,
            layout, _nine(strides), stream)
    head = (q_ptr, k_ptr, v_ptr, o_ptr, do_ptr, lse_ptr, rest_ptr)
    if rest_rows is None:
        _check(load().mfa_bwd_window(*head, *tail))
    else:
        _check(load().mfa_bwd_window_rest(*head, rest_rows, *tail))


def extend_block_tables(table_ptr: int, cached_ptr: int, added_ptr: int, free_ptr: int,
                        slots_ptr: int, starts_ptr: int, used_ptr: int, batch: int, columns: int,
                        free_count: int, page_size: int, capacity: int, stream: int = 0) -> None:
    """Launch mfa_extend_block_tables; raises MfaError."""
    _check(load().mfa_extend_block_tables(table_ptr, cached_ptr, added_ptr, free_ptr, slots_ptr,
                                          starts_ptr, used_ptr, batch, columns, free_count,
                                          page_size, capacity, stream))


def append_kv(k_ptr: int, v_ptr: int, k_cache_ptr: int, v_cache_ptr: int, slots_ptr: int,
              tokens: int, kv_heads: int, d: int, k_strides: tuple[int, int],
              v_strides: tuple[int, int], pages: int, page_size: int, stream: int = 0) -> None:
    """Launch mfa_append_kv ((token, head) strides in elements); raises MfaError."""
    _check(load().mfa_append_kv(k_ptr, v_ptr, k_cache_ptr, v_cache_ptr, slots_ptr, tokens,
                                kv_heads, d, *k_strides, *v_strides, pages, page_size, stream))


def paged_attention(q_ptr: int, k_cache_ptr: int, v_cache_ptr: int, table_ptr: int,
                    lengths_ptr: int, out_ptr: int, workspace_ptr: int, workspace_bytes: int,
                    batch: int, heads: int, kv_heads: int, d: int, pages: int, page_size: int,
                    columns: int, scale: float, window: int = 0, sinks: int = 0,
                    dtype: int = DTYPE_FP16, stream: int = 0,
                    q_strides: tuple[int, int] | None = None) -> None:
    """Launch mfa_paged_attention (q_strides: (batch, head) element strides of q, contiguous if
    None); raises MfaError."""
    _check(load().mfa_paged_attention(q_ptr, k_cache_ptr, v_cache_ptr, table_ptr, lengths_ptr,
                                      out_ptr, workspace_ptr, workspace_bytes, batch, heads,
                                      kv_heads, d, *(q_strides or (heads * d, d)), pages,
                                      page_size, columns, window, sinks, scale, dtype, stream))


def shared_prefix_attention(q_ptr: int, k_cache_ptr: int, v_cache_ptr: int, prefix_ptr: int,
                            prefix_length: int, table_ptr: int, lengths_ptr: int, out_ptr: int,
                            workspace_ptr: int, workspace_bytes: int, batch: int, heads: int,
                            kv_heads: int, d: int, pages: int, page_size: int, columns: int,
                            scale: float, dtype: int = DTYPE_FP16, stream: int = 0,
                            q_strides: tuple[int, int] | None = None) -> None:
    """Launch mfa_shared_prefix_attention (q_strides as for paged_attention); raises MfaError."""
    _check(load().mfa_shared_prefix_attention(
        q_ptr, k_cache_ptr, v_cache_ptr, prefix_ptr, prefix_length, table_ptr, lengths_ptr,
        out_ptr, workspace_ptr, workspace_bytes, batch, heads, kv_heads, d,
        *(q_strides or (heads * d, d)), pages, page_size, columns, scale, dtype, stream))


def paged_workspace_bytes(batch: int, heads: int, kv_heads: int, d: int, page_size: int,
                          columns: int, prefix_length: int = 0) -> int:
    """Workspace bytes of paged_attention (or, with a prefix_length, shared_prefix_attention) on
    the current device. Raises MfaError."""
    out = ctypes.c_uint64(0)
    _check(load().mfa_paged_workspace_bytes(batch, heads, kv_heads, d, page_size, columns,
                                            prefix_length, ctypes.byref(out)))
    return out.value


def fwd_workspace_bytes(batch: int, heads: int, n: int, d: int = 64,
                        causal: bool = False) -> int:
    """Device scratch bytes one forward call takes on the current device (0 unless the
    key dimension is split); nothing is launched or allocated. Raises MfaError."""
    out = ctypes.c_uint64(0)
    _check(load().mfa_fwd_workspace_bytes(batch, heads, n, d, int(causal), ctypes.byref(out)))
    return out.value


def device_status(device: int = 0, reset: bool = True) -> int:
    st = ctypes.c_int(0)
    _check(load().mfa_device_status(device, ctypes.byref(st), int(reset)))
    return st.value


def set_watchdog_ns(ns: int) -> None:
    _check(load().mfa_set_watchdog_ns(ns))


def watchdog_selftest(timeout_ns: int, stream: int = 0) -> int:
    st = ctypes.c_int(-1)
    _check(load().mfa_watchdog_selftest(stream, timeout_ns, ctypes.byref(st)))
    return st.value


def version() -> str:
    return load().mfa_version().decode()
