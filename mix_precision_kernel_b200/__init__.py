"""B200 (sm_100a) MXFP8 x BF16 GEMM, MXFP8 codec, int8 products and products grouped by expert.

Python binding of ``libmpk.so`` (C ABI in ``include/mpk.h``) through ctypes.
The function names follow the reference project's C++ API
(chcoliang/mix_precision_kernel ``include/gemm_kernels.h:12-16`` and
``include/mxfp8_utils.h:34-47``) with the same argument order and meaning:

    gemm_fp8_tensorcore(A_data, A_scales, B, C_data, C_scales, D_data, D_scales, M, N, K, stream)
    mxfp8_quantize_gpu(input, data, scales, M, K, stream)
    mxfp8_dequantize_gpu(data, scales, output, M, K, stream)
    mxfp8_quantize_host(input, data, scales, M, K)
    mxfp8_dequantize_host(data, scales, output, M, K)

The int8 products (``gemm_int8``, ``linear_int8``), the products grouped by expert
(``gemm_grouped``, ``gemm_grouped_int8``, ``gemm_grouped_mxfp8``, ``gemm_grouped_wgrad``) and the
int8 quantizers (``quantize_int8``, ``quantize_int8_cols``) have no counterpart there.

Arguments are torch CUDA tensors (or raw device addresses as ints) for the GPU
functions and numpy arrays for the host functions.  Where the reference calls
``exit()`` on a CUDA error, these raise :class:`MpkError`.  There is no CPU
fallback: if ``libmpk.so`` is missing the import of any GPU function fails.
"""
from __future__ import annotations

import ctypes
import os
import threading

__all__ = [
    "MpkError", "lib", "library_path",
    "gemm_fp8_tensorcore", "mxfp8_quantize_gpu", "mxfp8_dequantize_gpu",
    "mxfp8_quantize_host", "mxfp8_dequantize_host",
    "gemm_fp8_tensorcore_ws", "gemm_workspace_size", "release_workspace_pool",
    "mxfp8_dequantize_bf16_gpu", "mxfp8_quantize_bf16_gpu", "gemm_fp8_tensorcore_gather", "peer_barrier",
    "mxfp8_quantize_cols_gpu", "mxfp8_quantize_bf16_cols_gpu", "quantize_cols",
    "ipc_export", "ipc_import", "ipc_close",
    "gemm_fp8_tensorcore_noalloc", "NOALLOC_SCRATCH_BYTES",
    "gemm", "quantize", "dequantize", "device_status", "set_wait_timeout_ns", "wait_selftest",
    "set_gemm_schedule", "gemm_schedule", "gemm_plan", "SCHEDULE_AUTO", "SCHEDULE_TILES", "SCHEDULE_STREAM_K",
    "gemm_path", "PATH_PREPASS", "PATH_ONCHIP",
    "int8_quantize_rows_gpu", "int8_quantize_cols_gpu", "gemm_int8_gpu", "linear_int8_gpu",
    "gemm_grouped_gpu", "gemm_grouped_int8_gpu", "gemm_grouped_mxfp8_gpu", "gemm_grouped_wgrad_gpu",
    "quantize_int8", "quantize_int8_cols", "gemm_int8", "linear_int8",
    "gemm_grouped", "gemm_grouped_int8", "gemm_grouped_mxfp8", "gemm_grouped_wgrad",
    "TYPE_F32", "TYPE_BF16", "TYPE_F16", "B_KN", "B_NK", "MAX_GROUPS",
    "MX_BLOCK", "nblk",
]

MX_BLOCK = 32
_PKG = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_PKG, "_lib", "libmpk.so")
_lock = threading.Lock()
_lib = None

MPK_SUCCESS = 0
MPK_ERR_INVALID_VALUE = 1001
MPK_ERR_UNSUPPORTED = 1002
MPK_ERR_MISALIGNED = 1003
MPK_ERR_DEVICE_TIMEOUT = 1004
MPK_ERR_ARCH = 1005
MPK_ERR_DRIVER = 1006

# GEMM work schedules (MPK_SCHEDULE_* in include/mpk.h)
SCHEDULE_AUTO = 0
SCHEDULE_TILES = 1
SCHEDULE_STREAM_K = 2
# Kernel paths of the default GEMM entry point (MPK_PATH_* in include/mpk.h)
PATH_PREPASS = 0
PATH_ONCHIP = 1
# Element types and layouts of B of the int8 and expert-grouped entry points
# (MPK_TYPE_*, MPK_B_* in include/mpk.h)
TYPE_F32 = 0
TYPE_BF16 = 1
TYPE_F16 = 2
B_KN = 0
B_NK = 1
MAX_GROUPS = 1024


class MpkError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"mpk status {status}: {message}")
        self.status = status


def nblk(cols: int) -> int:
    return (cols + MX_BLOCK - 1) // MX_BLOCK


def library_path() -> str:
    return _LIB_PATH


def lib() -> ctypes.CDLL:
    """Load libmpk.so (built in-tree by ``mix_precision_kernel_b200.build``)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(_LIB_PATH):
                raise ImportError(
                    f"{_LIB_PATH} is missing: build it with `python -m mix_precision_kernel_b200.build`")
            L = ctypes.CDLL(_LIB_PATH)
            vp, ci, u8p = ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p
            L.mpk_gemm_mxfp8_bf16.argtypes = [vp, vp, vp, vp, vp, vp, vp, ci, ci, ci, vp]
            L.mpk_gemm_mxfp8_bf16_ws.argtypes = [vp, vp, vp, vp, vp, vp, vp, ci, ci, ci, vp,
                                                 ctypes.c_size_t, vp]
            L.mpk_gemm_workspace_size.argtypes = [ci, ci, ci, ctypes.POINTER(ctypes.c_size_t)]
            L.mpk_release_workspace_pool.argtypes = []
            L.mpk_gemm_mxfp8_bf16_noalloc.argtypes = [vp, vp, vp, vp, vp, vp, vp, ci, ci, ci, vp]
            L.mpk_mxfp8_quantize.argtypes = [vp, vp, vp, ci, ci, vp]
            L.mpk_mxfp8_dequantize.argtypes = [vp, vp, vp, ci, ci, vp]
            L.mpk_mxfp8_dequantize_bf16.argtypes = [vp, vp, vp, ci, ci, vp]
            L.mpk_mxfp8_quantize_bf16.argtypes = [vp, vp, vp, ci, ci, vp]
            L.mpk_mxfp8_quantize_cols.argtypes = [vp, vp, vp, ci, ci, vp]
            L.mpk_mxfp8_quantize_bf16_cols.argtypes = [vp, vp, vp, ci, ci, vp]
            L.mpk_gemm_mxfp8_bf16_gather.argtypes = [vp, vp, vp, vp, vp, ci, ci, ci, ctypes.c_int64,
                                                     ctypes.c_int64, ci, ci, vp, vp, ci, vp, ctypes.c_size_t,
                                                     vp]
            L.mpk_peer_barrier.argtypes = [vp, ci, ci, ctypes.c_uint32, vp]
            L.mpk_ipc_export.argtypes = [vp, vp, ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(ctypes.c_uint64)]
            L.mpk_ipc_import.argtypes = [vp, ctypes.c_uint64, ctypes.c_uint64, ctypes.POINTER(ctypes.c_void_p)]
            L.mpk_ipc_close.argtypes = [vp]
            L.mpk_mxfp8_quantize_host.argtypes = [vp, u8p, u8p, ci, ci]
            L.mpk_mxfp8_dequantize_host.argtypes = [u8p, u8p, vp, ci, ci]
            L.mpk_device_status.argtypes = [ctypes.POINTER(ci)]
            L.mpk_set_wait_timeout_ns.argtypes = [ctypes.c_uint64]
            L.mpk_wait_selftest.argtypes = [ctypes.c_uint64, vp]
            L.mpk_status_string.argtypes = [ci]
            L.mpk_status_string.restype = ctypes.c_char_p
            L.mpk_last_error.argtypes = []
            L.mpk_last_error.restype = ctypes.c_char_p
            L.mpk_last_error_string.argtypes = []
            L.mpk_last_error_string.restype = ctypes.c_char_p
            L.mpk_set_gemm_schedule.argtypes = [ci]
            L.mpk_gemm_schedule.argtypes = []
            ip = ctypes.POINTER(ci)
            L.mpk_gemm_plan.argtypes = [ci, ci, ci, ip, ip, ip]
            L.mpk_gemm_path.argtypes = [vp, vp, ci, ci, ci, ip]
            i64 = ctypes.c_int64
            L.mpk_int8_quantize_rows.argtypes = [vp, ci, i64, vp, i64, vp, ci, ci, vp]
            L.mpk_int8_quantize_cols.argtypes = [vp, ci, i64, vp, i64, vp, ci, ci, ci, vp]
            L.mpk_gemm_int8.argtypes = [vp, i64, vp, vp, i64, ci, vp, vp, vp, ci, i64, ci, ci, ci, vp]
            L.mpk_linear_int8.argtypes = [vp, ci, i64, vp, i64, ci, vp, vp, vp, ci, i64, ci, ci, ci, vp]
            L.mpk_gemm_grouped.argtypes = [vp, i64, vp, i64, ci, ci, vp, ci, i64, vp, ci, ci, ci, ci, vp]
            L.mpk_gemm_grouped_int8.argtypes = [vp, i64, vp, vp, i64, ci, vp, vp, ci, i64, vp, ci, ci, ci, ci, vp]
            L.mpk_gemm_grouped_mxfp8.argtypes = [vp, vp, vp, i64, vp, vp, vp, ci, ci, ci, ci, vp]
            L.mpk_gemm_grouped_wgrad.argtypes = [vp, i64, vp, i64, ci, vp, ci, i64, vp, ci, ci, ci, ci, vp]
            for f in ("mpk_int8_quantize_rows", "mpk_int8_quantize_cols", "mpk_gemm_int8", "mpk_linear_int8",
                      "mpk_gemm_grouped", "mpk_gemm_grouped_int8", "mpk_gemm_grouped_mxfp8",
                      "mpk_gemm_grouped_wgrad"):
                getattr(L, f).restype = ci
            for f in ("mpk_gemm_mxfp8_bf16", "mpk_gemm_mxfp8_bf16_ws", "mpk_gemm_workspace_size",
                      "mpk_release_workspace_pool", "mpk_mxfp8_quantize", "mpk_mxfp8_dequantize",
                      "mpk_mxfp8_dequantize_bf16", "mpk_gemm_mxfp8_bf16_noalloc",
                      "mpk_mxfp8_quantize_bf16", "mpk_gemm_mxfp8_bf16_gather", "mpk_peer_barrier",
                      "mpk_mxfp8_quantize_cols", "mpk_mxfp8_quantize_bf16_cols",
                      "mpk_ipc_export", "mpk_ipc_import", "mpk_ipc_close",
                      "mpk_mxfp8_quantize_host", "mpk_mxfp8_dequantize_host", "mpk_device_status",
                      "mpk_set_wait_timeout_ns", "mpk_wait_selftest", "mpk_version",
                      "mpk_set_gemm_schedule", "mpk_gemm_schedule", "mpk_gemm_plan", "mpk_gemm_path"):
                getattr(L, f).restype = ci
            _lib = L
    return _lib


def _check(status: int) -> None:
    if status != MPK_SUCCESS:
        L = lib()
        detail = (L.mpk_last_error_string() or b"").decode(errors="replace")
        msg = L.mpk_status_string(status).decode(errors="replace")
        raise MpkError(status, f"{msg}; {detail}" if detail else msg)


def _addr(t) -> int | None:
    """Device address of a torch tensor, an int address, or None."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def _stream(stream, *tensors) -> int | None:
    if stream is None:
        for t in tensors:
            if t is not None and not isinstance(t, int) and getattr(t, "is_cuda", False):
                import torch
                return torch.cuda.current_stream(t.device).cuda_stream
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _np_ptr(a):
    import numpy as np
    assert isinstance(a, np.ndarray) and a.flags["C_CONTIGUOUS"]
    return a.ctypes.data


# ---------------------------------------------------------------------------
# Reference-named entry points
# ---------------------------------------------------------------------------

def gemm_fp8_tensorcore(A_data, A_scales, B, C_data, C_scales, D_data, D_scales,
                        M: int, N: int, K: int, stream=None) -> None:
    """D = A*B + C (MXFP8 A, BF16 B [K][N], MXFP8 C/D along N).  C may be None."""
    s = _stream(stream, A_data, D_data)
    _check(lib().mpk_gemm_mxfp8_bf16(_addr(A_data), _addr(A_scales), _addr(B), _addr(C_data),
                                     _addr(C_scales), _addr(D_data), _addr(D_scales), M, N, K, s))


def gemm_workspace_size(M: int, N: int, K: int) -> int:
    n = ctypes.c_size_t(0)
    _check(lib().mpk_gemm_workspace_size(M, N, K, ctypes.byref(n)))
    return n.value


def _nbytes(buf, nbytes):
    """Size of a workspace given as a tensor, or as a raw address plus its size."""
    if buf is None:
        return 0
    if isinstance(buf, int):
        if nbytes is None:
            raise ValueError("a workspace given as a raw address needs workspace_bytes")
        return int(nbytes)
    return buf.numel() * buf.element_size()


def gemm_fp8_tensorcore_ws(A_data, A_scales, B, C_data, C_scales, D_data, D_scales,
                           M: int, N: int, K: int, workspace, stream=None,
                           workspace_bytes: int | None = None) -> None:
    """gemm_fp8_tensorcore with the A operand dequantized into a caller workspace
    (a uint8 CUDA tensor of at least gemm_workspace_size(M, N, K) bytes, or a raw
    device address with workspace_bytes), or, with workspace=None, converted on chip
    by the GEMM kernel itself."""
    s = _stream(stream, A_data, D_data)
    nbytes = _nbytes(workspace, workspace_bytes)
    _check(lib().mpk_gemm_mxfp8_bf16_ws(_addr(A_data), _addr(A_scales), _addr(B), _addr(C_data),
                                        _addr(C_scales), _addr(D_data), _addr(D_scales), M, N, K,
                                        _addr(workspace), nbytes, s))


NOALLOC_SCRATCH_BYTES = 32 * 1024 * 1024  # MPK_NOALLOC_SCRATCH_BYTES in include/mpk.h


def gemm_fp8_tensorcore_noalloc(A_data, A_scales, B, C_data, C_scales, D_data, D_scales,
                                M: int, N: int, K: int, stream=None) -> None:
    """gemm_fp8_tensorcore for callers that may not allocate device memory: the A
    workspace is the library's fixed per-device array (M*K*2 <= NOALLOC_SCRATCH_BYTES).
    Calls that can overlap on one device share that array and race; issue them on
    one stream or order them."""
    s = _stream(stream, A_data, D_data)
    _check(lib().mpk_gemm_mxfp8_bf16_noalloc(_addr(A_data), _addr(A_scales), _addr(B), _addr(C_data),
                                             _addr(C_scales), _addr(D_data), _addr(D_scales), M, N, K, s))


def gemm_fp8_tensorcore_gather(A_data, A_scales, B, C_data, C_scales, M: int, N: int, K: int,
                               row_offset: int, M_total: int, D_dest, Ds_dest, workspace,
                               stream=None, workspace_bytes: int | None = None,
                               col_offset: int = 0, N_total: int | None = None) -> None:
    """Fused GEMM + all-gather: element (r, c) of this slab's D goes to
    (row_offset + r, col_offset + c) of every destination (device addresses;
    D_dest[0] is this GPU's full M_total x N_total D).  The other GPUs' parts are
    present after peer_barrier on every GPU."""
    n = len(D_dest)
    assert n == len(Ds_dest) and 1 <= n <= 8
    dd = (ctypes.c_void_p * n)(*[_addr(x) for x in D_dest])
    ds = (ctypes.c_void_p * n)(*[_addr(x) for x in Ds_dest])
    s = _stream(stream, A_data)
    nbytes = _nbytes(workspace, workspace_bytes)
    _check(lib().mpk_gemm_mxfp8_bf16_gather(_addr(A_data), _addr(A_scales), _addr(B), _addr(C_data),
                                            _addr(C_scales), M, N, K, row_offset, col_offset, M_total,
                                            N if N_total is None else N_total, dd, ds, n,
                                            _addr(workspace), nbytes, s))


def peer_barrier(flags, rank: int, world: int, epoch: int, stream=None) -> None:
    """Stream-ordered barrier over the GPUs' flag arrays (device addresses, rank order)."""
    arr = (ctypes.c_void_p * world)(*[_addr(x) for x in flags])
    _check(lib().mpk_peer_barrier(arr, rank, world, epoch, _stream(stream)))


def ipc_export(t) -> tuple[bytes, int, int]:
    """(handle, offset, allocation bytes) describing the device allocation of t."""
    h = ctypes.create_string_buffer(64)
    off, size = ctypes.c_uint64(0), ctypes.c_uint64(0)
    _check(lib().mpk_ipc_export(_addr(t), h, ctypes.byref(off), ctypes.byref(size)))
    return h.raw, off.value, size.value


def ipc_import(handle: bytes, offset: int, alloc_bytes: int) -> int:
    """Map another process's exported buffer for the current device; returns its address."""
    p = ctypes.c_void_p(0)
    _check(lib().mpk_ipc_import(ctypes.c_char_p(handle), offset, alloc_bytes, ctypes.byref(p)))
    return p.value


def ipc_close(addr: int) -> None:
    _check(lib().mpk_ipc_close(addr))


def release_workspace_pool() -> None:
    """Return the current device's pooled GEMM workspace to the driver."""
    _check(lib().mpk_release_workspace_pool())


def mxfp8_quantize_gpu(input, data, scales, M: int, K: int, stream=None) -> None:
    s = _stream(stream, input, data)
    _check(lib().mpk_mxfp8_quantize(_addr(input), _addr(data), _addr(scales), M, K, s))


def mxfp8_dequantize_gpu(data, scales, output, M: int, K: int, stream=None) -> None:
    s = _stream(stream, data, output)
    _check(lib().mpk_mxfp8_dequantize(_addr(data), _addr(scales), _addr(output), M, K, s))


def mxfp8_quantize_bf16_gpu(input, data, scales, M: int, K: int, stream=None) -> None:
    """BF16 [M, K] -> MXFP8 along K (each value widened exactly to FP32 first)."""
    s = _stream(stream, input, data)
    _check(lib().mpk_mxfp8_quantize_bf16(_addr(input), _addr(data), _addr(scales), M, K, s))


def mxfp8_quantize_cols_gpu(input, data, scales, M: int, K: int, stream=None) -> None:
    """float32 [M, K] -> MXFP8 with blocks of 32 rows per column: data [M, K], scales
    [ceil(M/32), K]."""
    s = _stream(stream, input, data)
    _check(lib().mpk_mxfp8_quantize_cols(_addr(input), _addr(data), _addr(scales), M, K, s))


def mxfp8_quantize_bf16_cols_gpu(input, data, scales, M: int, K: int, stream=None) -> None:
    """BF16 [M, K] -> MXFP8 with blocks of 32 rows per column (values widened exactly)."""
    s = _stream(stream, input, data)
    _check(lib().mpk_mxfp8_quantize_bf16_cols(_addr(input), _addr(data), _addr(scales), M, K, s))


def quantize_cols(x, stream=None):
    """float32 or bfloat16 CUDA tensor [M, K] -> (codes uint8 [M, K], scales uint8
    [ceil(M/32), K]), blocks of 32 rows per column."""
    import torch
    assert x.is_cuda and x.dim() == 2 and x.is_contiguous() and x.dtype in (torch.float32, torch.bfloat16)
    M, K = x.shape
    d = torch.empty((M, K), dtype=torch.uint8, device=x.device)
    s = torch.empty((nblk(M), K), dtype=torch.uint8, device=x.device)
    (mxfp8_quantize_cols_gpu if x.dtype == torch.float32 else mxfp8_quantize_bf16_cols_gpu)(x, d, s, M, K, stream)
    return d, s


def mxfp8_dequantize_bf16_gpu(data, scales, output, M: int, K: int, stream=None) -> None:
    """MXFP8 -> BF16 (the GEMM's A pre-pass); output is a bfloat16 CUDA tensor [M, K]."""
    s = _stream(stream, data, output)
    _check(lib().mpk_mxfp8_dequantize_bf16(_addr(data), _addr(scales), _addr(output), M, K, s))


def mxfp8_quantize_host(input, data, scales, M: int, K: int) -> None:
    _check(lib().mpk_mxfp8_quantize_host(_np_ptr(input), _np_ptr(data), _np_ptr(scales), M, K))


def mxfp8_dequantize_host(data, scales, output, M: int, K: int) -> None:
    _check(lib().mpk_mxfp8_dequantize_host(_np_ptr(data), _np_ptr(scales), _np_ptr(output), M, K))


def device_status() -> int:
    """Synchronize the current device, then read and clear its device status word."""
    v = ctypes.c_int(0)
    st = lib().mpk_device_status(ctypes.byref(v))
    if st not in (MPK_SUCCESS, MPK_ERR_DEVICE_TIMEOUT):
        _check(st)
    return v.value


def set_wait_timeout_ns(ns: int) -> None:
    _check(lib().mpk_set_wait_timeout_ns(int(ns)))


def wait_selftest(timeout_ns: int, stream=None) -> None:
    _check(lib().mpk_wait_selftest(int(timeout_ns), _stream(stream)))


def set_gemm_schedule(schedule: int) -> int:
    """Sets the process-wide GEMM work schedule (SCHEDULE_AUTO, SCHEDULE_TILES or
    SCHEDULE_STREAM_K); returns the previous one."""
    L = lib()
    prev = L.mpk_gemm_schedule()
    _check(L.mpk_set_gemm_schedule(int(schedule)))
    return prev


def gemm_schedule() -> int:
    return lib().mpk_gemm_schedule()


def gemm_path(A_data, B, M: int, N: int, K: int) -> int:
    """PATH_PREPASS or PATH_ONCHIP: the kernel path gemm_fp8_tensorcore takes for these
    operands (tensors or device addresses) under the current schedule."""
    path = ctypes.c_int(-1)
    _check(lib().mpk_gemm_path(_addr(A_data), _addr(B), M, N, K, ctypes.byref(path)))
    return path.value


def gemm_plan(M: int, N: int, K: int) -> tuple[int, int, int]:
    """(tiles, stream-K tiles, stream-K SM pairs) of an M x N x K product on the
    current device under the current schedule."""
    t, st, sp = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
    _check(lib().mpk_gemm_plan(M, N, K, ctypes.byref(t), ctypes.byref(st), ctypes.byref(sp)))
    return t.value, st.value, sp.value


# ---------------------------------------------------------------------------
# int8 and expert-grouped products (tensors or device addresses; see include/mpk.h)
# ---------------------------------------------------------------------------

def _sizes(*sizes):
    """The C entry points take sizes as 32-bit integers; ctypes would cut larger ones off."""
    if max(sizes) > 0x7FFFFFFF or min(sizes) < -0x80000000:
        raise ValueError(f"sizes must fit 32-bit integers, got {sizes}")


def int8_quantize_rows_gpu(input, input_type: int, ld_input: int, codes, ld_codes: int, scales, M: int, K: int,
                           stream=None) -> None:
    """int8 codes of input [M, K] and one FP32 scale per row; row strides in elements."""
    _sizes(M, K)
    s = _stream(stream, input, codes)
    _check(lib().mpk_int8_quantize_rows(_addr(input), input_type, ld_input, _addr(codes), ld_codes, _addr(scales),
                                        M, K, s))


def int8_quantize_cols_gpu(input, input_type: int, ld_input: int, codes, ld_codes: int, scales, E: int, K: int,
                           N: int, stream=None) -> None:
    """int8 codes of input [E, K, N] and one FP32 scale per matrix and column."""
    _sizes(E, N, K)
    s = _stream(stream, input, codes)
    _check(lib().mpk_int8_quantize_cols(_addr(input), input_type, ld_input, _addr(codes), ld_codes, _addr(scales),
                                        E, K, N, s))


def gemm_int8_gpu(A, lda: int, A_scales, B, ldb: int, b_layout: int, B_scales, bias, D, d_type: int, ldd: int,
                  M: int, N: int, K: int, stream=None) -> None:
    """D = (A*B) * A_scales[row] * B_scales[column] + bias (int8 A and B; bias may be None)."""
    _sizes(M, N, K)
    s = _stream(stream, A, D)
    _check(lib().mpk_gemm_int8(_addr(A), lda, _addr(A_scales), _addr(B), ldb, b_layout, _addr(B_scales),
                               _addr(bias), _addr(D), d_type, ldd, M, N, K, s))


def linear_int8_gpu(x, x_type: int, ldx: int, B, ldb: int, b_layout: int, B_scales, bias, D, d_type: int, ldd: int,
                    M: int, N: int, K: int, stream=None) -> None:
    """gemm_int8_gpu of x quantized per row on the way."""
    _sizes(M, N, K)
    s = _stream(stream, x, D)
    _check(lib().mpk_linear_int8(_addr(x), x_type, ldx, _addr(B), ldb, b_layout, _addr(B_scales), _addr(bias),
                                 _addr(D), d_type, ldd, M, N, K, s))


def gemm_grouped_gpu(A, lda: int, B, ldb: int, b_layout: int, ab_type: int, D, d_type: int, ldd: int, offsets,
                     E: int, M: int, N: int, K: int, stream=None) -> None:
    """Rows offsets[e]..offsets[e + 1] of D = the same rows of A times B[e] (16-bit types)."""
    _sizes(E, M, N, K)
    s = _stream(stream, A, D)
    _check(lib().mpk_gemm_grouped(_addr(A), lda, _addr(B), ldb, b_layout, ab_type, _addr(D), d_type, ldd,
                                  _addr(offsets), E, M, N, K, s))


def gemm_grouped_int8_gpu(A, lda: int, A_scales, B, ldb: int, b_layout: int, B_scales, D, d_type: int, ldd: int,
                          offsets, E: int, M: int, N: int, K: int, stream=None) -> None:
    """gemm_grouped_gpu of int8 codes with row scales [M] and column scales [E, N]."""
    _sizes(E, M, N, K)
    s = _stream(stream, A, D)
    _check(lib().mpk_gemm_grouped_int8(_addr(A), lda, _addr(A_scales), _addr(B), ldb, b_layout, _addr(B_scales),
                                       _addr(D), d_type, ldd, _addr(offsets), E, M, N, K, s))


def gemm_grouped_mxfp8_gpu(A_data, A_scales, B, ldb: int, D_data, D_scales, offsets, E: int, M: int, N: int, K: int,
                           stream=None) -> None:
    """gemm_grouped_gpu with A and D in MXFP8 and B in BF16."""
    _sizes(E, M, N, K)
    s = _stream(stream, A_data, D_data)
    _check(lib().mpk_gemm_grouped_mxfp8(_addr(A_data), _addr(A_scales), _addr(B), ldb, _addr(D_data),
                                        _addr(D_scales), _addr(offsets), E, M, N, K, s))


def gemm_grouped_wgrad_gpu(A, lda: int, dD, ldg: int, ab_type: int, dB, d_type: int, ldd: int, offsets, E: int,
                           M: int, N: int, K: int, stream=None) -> None:
    """dB[e] [K, N] = A[rows of e]^T * dD[rows of e]; zeros for an empty group."""
    _sizes(E, M, N, K)
    s = _stream(stream, A, dB)
    _check(lib().mpk_gemm_grouped_wgrad(_addr(A), lda, _addr(dD), ldg, ab_type, _addr(dB), d_type, ldd,
                                        _addr(offsets), E, M, N, K, s))


# ---------------------------------------------------------------------------
# Allocating conveniences (torch tensors)
# ---------------------------------------------------------------------------

def quantize(x, stream=None):
    """float32 CUDA tensor [M, K] -> (codes uint8 [M, K], scales uint8 [M, ceil(K/32)])."""
    import torch
    assert x.dtype == torch.float32 and x.is_cuda and x.dim() == 2 and x.is_contiguous()
    M, K = x.shape
    d = torch.empty((M, K), dtype=torch.uint8, device=x.device)
    s = torch.empty((M, nblk(K)), dtype=torch.uint8, device=x.device)
    mxfp8_quantize_gpu(x, d, s, M, K, stream)
    return d, s


def dequantize(d, s, stream=None):
    import torch
    assert d.dtype == torch.uint8 and d.is_cuda and d.dim() == 2 and d.is_contiguous()
    M, K = d.shape
    out = torch.empty((M, K), dtype=torch.float32, device=d.device)
    mxfp8_dequantize_gpu(d, s, out, M, K, stream)
    return out


def gemm(A_data, A_scales, B, C_data=None, C_scales=None, stream=None):
    """Allocating form of :func:`gemm_fp8_tensorcore`; B is a bf16 CUDA tensor [K, N]."""
    import torch
    M, K = A_data.shape
    K2, N = B.shape
    assert K == K2 and B.dtype == torch.bfloat16 and B.is_contiguous()
    D = torch.empty((M, N), dtype=torch.uint8, device=A_data.device)
    Ds = torch.empty((M, nblk(N)), dtype=torch.uint8, device=A_data.device)
    gemm_fp8_tensorcore(A_data, A_scales, B, C_data, C_scales, D, Ds, M, N, K, stream)
    return D, Ds


# Allocating forms of the int8 and expert-grouped products.  They take CUDA tensors whose
# last dimension is contiguous (rows may be strided), check types, shapes and devices,
# and run on the current stream of the tensors' device.  A decoding step makes many such
# calls of a few microseconds each, so the checks are written out as plain comparisons
# (`_want` and `_vector` run on the way to an error only).

_torch = None
_types: dict = {}


def _init_torch():
    global _torch
    import torch
    _types.update({torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16})
    _torch = torch
    return torch


def _type_code(dtype, what: str, allowed=(TYPE_F32, TYPE_BF16, TYPE_F16)) -> int:
    code = _types.get(dtype)
    if code not in allowed:
        raise ValueError(f"{what}: type {dtype} is not supported")
    return code


def _row_stride(t, what: str) -> int:
    """Elements between the rows of t [.., rows, columns], matrices back to back."""
    shape, st = t.shape, t.stride()
    rows, cols, ld = shape[-2], shape[-1], st[-2]
    if rows <= 1 and ld < cols:
        ld = cols
    if (cols > 1 and st[-1] != 1) or ld < cols:
        raise ValueError(f"{what}: the last dimension must be contiguous, got strides {tuple(st)}")
    if len(st) == 3 and shape[0] > 1 and st[0] != rows * ld and t.numel() > 0:
        if rows == 1 and st[0] >= cols:
            return st[0]
        raise ValueError(f"{what}: the matrices must lie back to back, got strides {tuple(st)}")
    return ld


def _want(t, what: str, dim: int, dtype=None, shape=None, like=None):
    if not t.is_cuda or t.dim() != dim or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{what}: expected a {dim}-dimensional CUDA tensor"
                         f"{'' if dtype is None else f' of {dtype}'}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{what} is on {t.device}, not on {like.device}")


def _matrix(t, what: str, dim: int, dtype, like=None):
    """t's shape: a `dim`-dimensional CUDA tensor of dtype (None: any) on like's device."""
    shape = t.shape
    if (len(shape) != dim or (dtype is not None and t.dtype is not dtype) or not t.is_cuda
            or (like is not None and t.get_device() != like.get_device())):
        _want(t, what, dim, dtype, None, like)
    if max(shape) > 0x7FFFFFFF:
        _sizes(*shape)
    return shape


def _vector(t, what: str, dtype, shape: tuple, like):
    if (t.dtype is not dtype or t.shape != shape or t.get_device() != like.get_device() or not t.is_contiguous()):
        _want(t, what, len(shape), dtype, shape, like)
        raise ValueError(f"{what} must be contiguous")


def _result(out, shape: tuple, dtype, like):
    """(out, or a new contiguous tensor; its row stride)."""
    if out is None:
        cols = shape[-1]
        strides = (cols, 1) if len(shape) == 2 else (shape[1] * cols, cols, 1)
        return _torch.empty_strided(shape, strides, dtype=dtype, device=like.device), cols
    if out.shape != shape or out.dtype is not dtype or out.get_device() != like.get_device():
        _want(out, "out", len(shape), dtype, shape, like)
    return out, _row_stride(out, "out")


def _raw_stream(index: int) -> int:
    get = getattr(_torch._C, "_cuda_getCurrentRawStream", None)
    return get(index) if get is not None else _torch.cuda.current_stream(index).cuda_stream


def _launch(fn, like, *args):
    """Call a C entry point on the current stream of like's device."""
    index = like.get_device()
    if _torch.cuda.current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with _torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status != MPK_SUCCESS:
        _check(status)


def _padded_codes(shape, like):
    """int8 codes whose rows start on 16-byte boundaries (read in place by the products), and
    their row stride."""
    ld = (shape[-1] + 15) // 16 * 16
    strides = (ld, 1) if len(shape) == 2 else (shape[1] * ld, ld, 1)
    return _torch.empty_strided(tuple(shape), strides, dtype=_torch.int8, device=like.device), ld


def _scales(shape: tuple, like):
    strides = (1,) if len(shape) == 1 else (shape[1], 1)
    return _torch.empty_strided(shape, strides, dtype=_torch.float32, device=like.device)


def quantize_int8(x):
    """float32, bfloat16 or float16 [M, K] -> (codes int8 [M, K], scales float32 [M]): one
    scale per row.  The codes' rows are padded to a multiple of 16 bytes."""
    if _torch is None:
        _init_torch()
    M, K = _matrix(x, "x", 2, None)
    t = _type_code(x.dtype, "x")
    ldx = _row_stride(x, "x")
    codes, ld = _padded_codes((M, K), x)
    scales = _scales((M,), x)
    _launch(lib().mpk_int8_quantize_rows, x, x.data_ptr(), t, ldx, codes.data_ptr(), ld, scales.data_ptr(), M, K)
    return codes, scales


def quantize_int8_cols(w):
    """float32, bfloat16 or float16 [K, N] or [E, K, N] -> (codes int8 of the same shape,
    scales float32 [N] or [E, N]): one scale per column.  The codes' rows are padded to a
    multiple of 16 bytes."""
    if _torch is None:
        _init_torch()
    shape = _matrix(w, "w", 3 if w.dim() == 3 else 2, None)
    t = _type_code(w.dtype, "w")
    E = shape[0] if len(shape) == 3 else 1
    K, N = shape[-2:]
    ldw = _row_stride(w, "w")
    codes, ld = _padded_codes(shape, w)
    scales = _scales((N,) if len(shape) == 2 else (E, N), w)
    _launch(lib().mpk_int8_quantize_cols, w, w.data_ptr(), t, ldw, codes.data_ptr(), ld, scales.data_ptr(), E, K, N)
    return codes, scales


def _b_sizes(shape, b_layout: int, K: int) -> int:
    """N of B [.., K, N] (B_KN) or [.., N, K] (B_NK)."""
    if b_layout == B_KN:
        k, n = shape[-2], shape[-1]
    elif b_layout == B_NK:
        n, k = shape[-2], shape[-1]
    else:
        raise ValueError(f"unknown layout of B {b_layout}")
    if k != K:
        raise ValueError(f"B {tuple(shape)} does not fit a reduction of {K}")
    return n


def gemm_int8(A, A_scales, B, B_scales, bias=None, out_dtype=None, b_layout: int = B_KN, out=None):
    """D [M, N] = (A*B) * A_scales[row] * B_scales[column] + bias: int8 A [M, K] and B [K, N]
    (or [N, K] with b_layout=B_NK), float32 scales and bias; D in out_dtype (default bfloat16)."""
    torch = _torch or _init_torch()
    M, K = _matrix(A, "A", 2, torch.int8)
    N = _b_sizes(_matrix(B, "B", 2, torch.int8, A), b_layout, K)
    _vector(A_scales, "A_scales", torch.float32, (M,), A)
    _vector(B_scales, "B_scales", torch.float32, (N,), A)
    if bias is not None:
        _vector(bias, "bias", torch.float32, (N,), A)
    dtype = out_dtype or (torch.bfloat16 if out is None else out.dtype)
    d = _type_code(dtype, "D")
    D, ldd = _result(out, (M, N), dtype, A)
    _launch(lib().mpk_gemm_int8, A, A.data_ptr(), _row_stride(A, "A"), A_scales.data_ptr(), B.data_ptr(),
            _row_stride(B, "B"), b_layout, B_scales.data_ptr(), None if bias is None else bias.data_ptr(),
            D.data_ptr(), d, ldd, M, N, K)
    return D


def linear_int8(x, B, B_scales, bias=None, out_dtype=None, b_layout: int = B_KN, out=None):
    """gemm_int8 of x [M, K] (float32, bfloat16 or float16) quantized per row on the way; D in
    out_dtype (default x's type).  out may lie in x's place."""
    torch = _torch or _init_torch()
    M, K = _matrix(x, "x", 2, None)
    t = _type_code(x.dtype, "x")
    N = _b_sizes(_matrix(B, "B", 2, torch.int8, x), b_layout, K)
    _vector(B_scales, "B_scales", torch.float32, (N,), x)
    if bias is not None:
        _vector(bias, "bias", torch.float32, (N,), x)
    dtype = out_dtype or (x.dtype if out is None else out.dtype)
    d = _type_code(dtype, "D")
    D, ldd = _result(out, (M, N), dtype, x)
    _launch(lib().mpk_linear_int8, x, x.data_ptr(), t, _row_stride(x, "x"), B.data_ptr(), _row_stride(B, "B"),
            b_layout, B_scales.data_ptr(), None if bias is None else bias.data_ptr(), D.data_ptr(), d,
            ldd, M, N, K)
    return D


def gemm_grouped(A, B, offsets, out_dtype=None, b_layout: int = B_KN, out=None):
    """Rows offsets[e]:offsets[e + 1] of D [M, N] = the same rows of A [M, K] times B[e]; B
    [E, K, N] (or [E, N, K] with b_layout=B_NK) of A's type (bfloat16 or float16), offsets
    int32 [E + 1] on the device.  Rows outside every group keep out's values (and are
    undefined without out).  The gradient of A is gemm_grouped(dD, B, offsets) with the
    other b_layout, that of B is gemm_grouped_wgrad(A, dD, offsets)."""
    torch = _torch or _init_torch()
    M, K = _matrix(A, "A", 2, None)
    t = _type_code(A.dtype, "A", (TYPE_BF16, TYPE_F16))
    b_shape = _matrix(B, "B", 3, A.dtype, A)
    N = _b_sizes(b_shape, b_layout, K)
    E = b_shape[0]
    _vector(offsets, "offsets", torch.int32, (E + 1,), A)
    dtype = out_dtype or (A.dtype if out is None else out.dtype)
    d = _type_code(dtype, "D")
    D, ldd = _result(out, (M, N), dtype, A)
    _launch(lib().mpk_gemm_grouped, A, A.data_ptr(), _row_stride(A, "A"), B.data_ptr(), _row_stride(B, "B"),
            b_layout, t, D.data_ptr(), d, ldd, offsets.data_ptr(), E, M, N, K)
    return D


def gemm_grouped_int8(A, A_scales, B, B_scales, offsets, out_dtype=None, b_layout: int = B_KN, out=None):
    """gemm_grouped of int8 codes: row scales A_scales [M], column scales B_scales [E, N]; D
    in out_dtype (default bfloat16)."""
    torch = _torch or _init_torch()
    M, K = _matrix(A, "A", 2, torch.int8)
    b_shape = _matrix(B, "B", 3, torch.int8, A)
    N = _b_sizes(b_shape, b_layout, K)
    E = b_shape[0]
    _vector(A_scales, "A_scales", torch.float32, (M,), A)
    _vector(B_scales, "B_scales", torch.float32, (E, N), A)
    _vector(offsets, "offsets", torch.int32, (E + 1,), A)
    dtype = out_dtype or (torch.bfloat16 if out is None else out.dtype)
    d = _type_code(dtype, "D")
    D, ldd = _result(out, (M, N), dtype, A)
    _launch(lib().mpk_gemm_grouped_int8, A, A.data_ptr(), _row_stride(A, "A"), A_scales.data_ptr(), B.data_ptr(),
            _row_stride(B, "B"), b_layout, B_scales.data_ptr(), D.data_ptr(), d, ldd,
            offsets.data_ptr(), E, M, N, K)
    return D


def gemm_grouped_mxfp8(A_data, A_scales, B, offsets, out=None):
    """gemm_grouped with A in MXFP8 (codes [M, K], scales [M, ceil(K/32)]) and bfloat16 B
    [E, K, N]; returns D in MXFP8 along N (codes [M, N], scales [M, ceil(N/32)])."""
    torch = _torch or _init_torch()
    M, K = _matrix(A_data, "A_data", 2, torch.uint8)
    b_shape = _matrix(B, "B", 3, torch.bfloat16, A_data)
    N = _b_sizes(b_shape, B_KN, K)
    E = b_shape[0]
    _vector(A_data, "A_data", torch.uint8, (M, K), A_data)
    _vector(A_scales, "A_scales", torch.uint8, (M, nblk(K)), A_data)
    _vector(offsets, "offsets", torch.int32, (E + 1,), A_data)
    D, Ds = out if out is not None else (None, None)
    D, _ = _result(D, (M, N), torch.uint8, A_data)
    Ds, _ = _result(Ds, (M, nblk(N)), torch.uint8, A_data)
    if not D.is_contiguous() or not Ds.is_contiguous():
        raise ValueError("out must be contiguous")
    _launch(lib().mpk_gemm_grouped_mxfp8, A_data, A_data.data_ptr(), A_scales.data_ptr(), B.data_ptr(),
            _row_stride(B, "B"), D.data_ptr(), Ds.data_ptr(), offsets.data_ptr(), E, M, N, K)
    return D, Ds


def gemm_grouped_wgrad(A, dD, offsets, out_dtype=None, out=None):
    """Gradient of gemm_grouped's B [E, K, N]: dB[e] = A[rows of e]^T * dD[rows of e] (zeros
    for an empty group), in out_dtype (default A's type)."""
    torch = _torch or _init_torch()
    M, K = _matrix(A, "A", 2, None)
    t = _type_code(A.dtype, "A", (TYPE_BF16, TYPE_F16))
    rows, N = _matrix(dD, "dD", 2, A.dtype, A)
    if rows != M:
        raise ValueError(f"dD has {rows} rows, A has {M}")
    E = _matrix(offsets, "offsets", 1, torch.int32, A)[0] - 1
    if E < 0:
        raise ValueError("offsets must hold at least one value")
    _vector(offsets, "offsets", torch.int32, (E + 1,), A)
    dtype = out_dtype or (A.dtype if out is None else out.dtype)
    d = _type_code(dtype, "dB")
    dB, ldd = _result(out, (E, K, N), dtype, A)
    _launch(lib().mpk_gemm_grouped_wgrad, A, A.data_ptr(), _row_stride(A, "A"), dD.data_ptr(), _row_stride(dD, "dD"),
            t, dB.data_ptr(), d, ldd, offsets.data_ptr(), E, M, N, K)
    return dB
