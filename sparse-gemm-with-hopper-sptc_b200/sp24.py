"""ctypes binding of the sp24 C ABI (include/sp24.h) for tests and the bench.

The product is the C-ABI shared library ``lib/libsp24.so`` built from
``csrc/`` for sm_100a.  This module only marshals torch CUDA tensors into the
plain pointers/sizes that ABI takes; every computation runs in the library's
CUDA kernels.  There is no CPU path: if the library or a GPU is missing, the
calls raise.

Reference interfaces mirrored (codes1gn/sparse-gemm-with-hopper-sptc):
  gemm()      wgmma_sp_raw_kernel<Element,BlockN>, wgmma_sp_raw_common.hpp:955-1030
  compress()  compress_structured_sparse_a, wgmma_sp_raw_common.hpp:140-205
"""
from __future__ import annotations

import ctypes
import os
import struct
from ctypes import (POINTER, Structure, c_char_p, c_float, c_int, c_int64, c_longlong,
                    c_size_t, c_uint8, c_ulonglong, c_void_p)

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libsp24.so")
PEAK_LIB_PATH = os.path.join(HERE, "lib", "libsp24_peak.so")

F16, BF16, E4M3 = 0, 1, 2
# Mixed fp8: A's format first, B's second (kind::f8f6f4 formats may differ).
E5M2_E4M3, E4M3_E5M2, E5M2 = 3, 4, 5
# Rows and products of the MLP block: 8-bit integers, fp32 output.
I8, F32 = 6, 7
META_REF, META_TC, META_K16 = 0, 1, 2

STATUS = {
    0: "SP24_OK", 1: "SP24_ERR_SHAPE", 2: "SP24_ERR_ALIGN", 3: "SP24_ERR_NOT_2OF4",
    4: "SP24_ERR_ARCH", 5: "SP24_ERR_CUDA", 6: "SP24_ERR_TIMEOUT", 7: "SP24_ERR_NCCL",
    8: "SP24_ERR_ARG", 9: "SP24_ERR_WORKSPACE", 10: "SP24_ERR_SCRATCH_LIMIT",
}

# Every symbol include/sp24.h declares.
EXPORTS = [
    "sp24_version", "sp24_status_string", "sp24_check_device", "sp24_meta_tc_bytes",
    "sp24_gemm_workspace_bytes", "sp24_compress", "sp24_prune_2of4", "sp24_repack_meta",
    "sp24_gemm", "sp24_last_kernel_status", "sp24_selftest_timeout", "sp24_amax_f32",
    "sp24_quantize_e4m3", "sp24_shard_columns", "sp24_unshard_columns_f32",
    "sp24_gemm_noalloc", "sp24_quantize_e5m2", "sp24_gemm_fused", "sp24_repack_meta_k16",
    "sp24_gemm_allgather", "sp24_ipc_get_handle", "sp24_ipc_open_handle", "sp24_ipc_close",
    "sp24_set_launch_hints", "sp24_get_launch_hints", "sp24_reload_tuning",
    "sp24_gemm_multi", "sp24_replicate", "sp24_gemm_multi_workspace_bytes",
    "sp24_rmsnorm_quant", "sp24_swiglu_quant", "sp24_quantize_rows", "sp24_gemm_scaled",
    "sp24_ffn_forward", "sp24_ffn_backward", "sp24_ffn_saved_bytes", "sp24_ffn_workspace_bytes",
]
MAX_PEERS = 7
HINT_NONE, HINT_STATIC_WEIGHTS = 0, 1

ACT_NONE, ACT_SILU = 0, 1
ACT_GELU_TANH = 2   # ffn_gated only


class Sp24Error(RuntimeError):
    def __init__(self, code: int, where: str):
        self.code = code
        super().__init__(f"{where}: {STATUS.get(code, code)}")


class GemmDesc(Structure):
    _fields_ = [
        ("dtype", c_int), ("m", c_int), ("n", c_int), ("k", c_int),
        ("a_c", c_void_p), ("lda_c", c_int64),
        ("meta", c_void_p), ("meta_format", c_int),
        ("b", c_void_p), ("ldb", c_int64),
        ("c_f32", c_void_p), ("c_bf16", c_void_p), ("ldc", c_int64),
        ("alpha", c_float), ("tile_n", c_int),
        ("workspace", c_void_p), ("workspace_bytes", c_size_t),
        ("status_dev", c_void_p),
    ]


class Epilogue(Structure):
    _fields_ = [
        ("bias", c_void_p), ("act", c_int),
        ("a_c_up", c_void_p), ("lda_c_up", c_int64), ("meta_up", c_void_p),
        ("alpha_up", c_float), ("bias_up", c_void_p),
    ]


class PeerOut(Structure):
    _fields_ = [("n_peers", c_int), ("c_f32", c_void_p * 7), ("c_bf16", c_void_p * 7)]


MAX_GPUS = 8
MULTI_FULL, MULTI_SHARD = 0, 1


class MultiDesc(Structure):
    _fields_ = [
        ("gemm", GemmDesc), ("ngpu", c_int), ("devices", c_int * MAX_GPUS),
        ("streams", c_void_p * MAX_GPUS), ("a_c", c_void_p * MAX_GPUS),
        ("meta", c_void_p * MAX_GPUS), ("b", c_void_p * MAX_GPUS), ("b_layout", c_int),
        ("c_f32", c_void_p * MAX_GPUS), ("c_bf16", c_void_p * MAX_GPUS), ("c_layout", c_int),
        ("workspace", c_void_p * MAX_GPUS), ("workspace_bytes", c_size_t),
    ]


class RowQuantDesc(Structure):
    _fields_ = [
        ("dtype", c_int), ("qdtype", c_int), ("rows", c_int), ("cols", c_int),
        ("x", c_void_p), ("ldx", c_int64), ("up", c_void_p), ("ld_up", c_int64),
        ("residual", c_void_p), ("ld_residual", c_int64),
        ("residual_out", c_void_p), ("ld_residual_out", c_int64),
        ("weight", c_void_p), ("eps", c_float), ("q", c_void_p), ("ldq", c_int64),
        ("scale", c_void_p),
    ]


class ScaledDesc(Structure):
    _fields_ = [
        ("dtype", c_int), ("cdtype", c_int), ("m", c_int), ("n", c_int), ("k", c_int),
        ("a_c", c_void_p), ("lda_c", c_int64), ("meta", c_void_p),
        ("x", c_void_p), ("ldx", c_int64),
        ("scale_m", c_void_p), ("scale_n", c_void_p), ("bias", c_void_p),
        ("c", c_void_p), ("ldc", c_int64), ("status_dev", c_void_p),
    ]


class FfnDesc(Structure):
    _fields_ = [
        ("dtype", c_int), ("t", c_int), ("h", c_int), ("f", c_int), ("act", c_int),
        ("x", c_void_p), ("ldx", c_int64), ("w_gate", c_void_p), ("ld_gate", c_int64),
        ("w_up", c_void_p), ("ld_up", c_int64),
        ("saved", c_void_p), ("saved_bytes", c_size_t), ("status_dev", c_void_p),
    ]


class FfnGrads(Structure):
    _fields_ = [
        ("d_out", c_void_p), ("ld_d_out", c_int64), ("dx", c_void_p), ("ld_dx", c_int64),
        ("dw_gate", c_void_p), ("ld_dgate", c_int64), ("dw_up", c_void_p), ("ld_dup", c_int64),
        ("workspace", c_void_p), ("workspace_bytes", c_size_t),
    ]


_lib = None


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the shared library (raises if it was not built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} missing: run __graft_entry__.build() first")
    lib = ctypes.CDLL(path)
    lib.sp24_version.restype = c_char_p
    lib.sp24_status_string.restype = c_char_p
    lib.sp24_status_string.argtypes = [c_int]
    lib.sp24_check_device.argtypes = [c_int]
    lib.sp24_meta_tc_bytes.restype = c_size_t
    lib.sp24_meta_tc_bytes.argtypes = [c_int, c_int]
    lib.sp24_gemm_workspace_bytes.restype = c_size_t
    lib.sp24_gemm_workspace_bytes.argtypes = [POINTER(GemmDesc)]
    lib.sp24_gemm.argtypes = [POINTER(GemmDesc), c_void_p]
    lib.sp24_gemm_noalloc.argtypes = [POINTER(GemmDesc), c_void_p]
    lib.sp24_gemm_fused.argtypes = [POINTER(GemmDesc), POINTER(Epilogue), c_void_p]
    lib.sp24_gemm_allgather.argtypes = [POINTER(GemmDesc), POINTER(PeerOut), c_void_p]
    lib.sp24_gemm_multi.argtypes = [POINTER(MultiDesc), c_int]
    lib.sp24_gemm_multi_workspace_bytes.argtypes = [POINTER(MultiDesc)]
    lib.sp24_gemm_multi_workspace_bytes.restype = c_size_t
    lib.sp24_replicate.argtypes = [c_void_p, c_int, c_size_t, c_int, POINTER(c_int),
                                   POINTER(c_void_p), POINTER(c_void_p)]
    lib.sp24_ipc_get_handle.argtypes = [c_void_p, c_void_p, POINTER(c_size_t)]
    lib.sp24_ipc_open_handle.argtypes = [c_void_p, POINTER(c_void_p)]
    lib.sp24_ipc_close.argtypes = [c_void_p]
    lib.sp24_selftest_timeout.argtypes = [POINTER(GemmDesc), c_ulonglong, c_void_p]
    lib.sp24_last_kernel_status.argtypes = [c_void_p]
    lib.sp24_set_launch_hints.argtypes = [ctypes.c_uint]
    lib.sp24_set_launch_hints.restype = None
    lib.sp24_get_launch_hints.restype = ctypes.c_uint
    lib.sp24_reload_tuning.restype = None
    lib.sp24_reload_tuning.argtypes = []
    lib.sp24_compress.argtypes = [c_int, c_void_p, c_int, c_int, c_int64, c_void_p, c_int64,
                                  c_void_p, c_void_p, POINTER(c_longlong), c_void_p]
    lib.sp24_prune_2of4.argtypes = [c_int, c_void_p, c_int, c_int, c_int64, c_void_p, c_int64,
                                    c_void_p]
    lib.sp24_repack_meta.argtypes = [c_int, c_void_p, c_int, c_int, c_void_p, c_void_p]
    lib.sp24_repack_meta_k16.argtypes = [c_int, c_void_p, c_int, c_int, c_void_p, c_void_p]
    lib.sp24_amax_f32.argtypes = [c_void_p, c_size_t, c_void_p, c_void_p]
    lib.sp24_quantize_e4m3.argtypes = [c_void_p, c_size_t, c_void_p, c_void_p, c_void_p,
                                       c_void_p]
    lib.sp24_quantize_e5m2.argtypes = [c_void_p, c_size_t, c_void_p, c_void_p, c_void_p,
                                       c_void_p]
    lib.sp24_shard_columns.restype = None
    lib.sp24_shard_columns.argtypes = [c_int, c_int, c_int, c_int, POINTER(c_int),
                                       POINTER(c_int)]
    lib.sp24_unshard_columns_f32.argtypes = [c_void_p, c_void_p, c_int, c_int, c_int, c_int,
                                             c_void_p]
    for name in ("sp24_rmsnorm_quant", "sp24_swiglu_quant", "sp24_quantize_rows"):
        getattr(lib, name).argtypes = [c_void_p, c_void_p]   # descriptors: byref(...) or packed bytes
        getattr(lib, name).restype = c_int
    lib.sp24_gemm_scaled.argtypes = [c_void_p, c_void_p]
    lib.sp24_ffn_forward.argtypes = [c_void_p, c_void_p, c_int64, c_void_p]
    lib.sp24_ffn_backward.argtypes = [c_void_p, c_void_p, c_void_p]
    lib.sp24_ffn_saved_bytes.argtypes = [c_int, c_int]
    lib.sp24_ffn_workspace_bytes.argtypes = [c_int, c_int, c_int]
    for name in ("sp24_ffn_saved_bytes", "sp24_ffn_workspace_bytes"):
        getattr(lib, name).restype = c_size_t
    for name in ("sp24_gemm_scaled", "sp24_ffn_forward", "sp24_ffn_backward",
                 "sp24_gemm", "sp24_gemm_noalloc", "sp24_gemm_fused", "sp24_gemm_allgather",
                 "sp24_gemm_multi", "sp24_replicate",
                 "sp24_ipc_get_handle", "sp24_ipc_open_handle", "sp24_ipc_close",
                 "sp24_selftest_timeout",
                 "sp24_last_kernel_status",
                 "sp24_compress", "sp24_prune_2of4", "sp24_repack_meta", "sp24_repack_meta_k16",
                 "sp24_amax_f32",
                 "sp24_quantize_e4m3", "sp24_quantize_e5m2", "sp24_unshard_columns_f32",
                 "sp24_check_device"):
        getattr(lib, name).restype = c_int
    _lib = lib
    return lib


def _check(code: int, where: str) -> None:
    if code != 0:
        raise Sp24Error(code, where)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _stream(stream) -> int:
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
    return stream.cuda_stream


def dtype_code(tdtype) -> int:
    """Library dtype of a torch dtype (uint8 = e4m3 bits); ints pass through
    (the mixed fp8 codes cannot be told from one tensor)."""
    import torch
    if isinstance(tdtype, int):
        return tdtype
    if tdtype == torch.float8_e5m2:
        return E5M2
    if tdtype == torch.float16:
        return F16
    if tdtype == torch.bfloat16:
        return BF16
    if tdtype in (torch.float8_e4m3fn, torch.uint8):
        return E4M3
    raise ValueError(f"unsupported dtype {tdtype}")


def meta_tc_bytes(m: int, k: int) -> int:
    return int(load().sp24_meta_tc_bytes(m, k))


def compress(a_dense, stream=None, dtype=None):
    """Dense 2:4 A (m x k, CUDA) -> (A_c m x k/2, reference metadata m x k/8 uint8).
    dtype: library dtype code when the tensor's own dtype does not say it
    (fp8 bits held as uint8)."""
    import torch
    lib = load()
    m, k = a_dense.shape
    a_c = torch.empty((m, k // 2), dtype=a_dense.dtype, device=a_dense.device)
    meta = torch.empty((m, k // 8), dtype=torch.uint8, device=a_dense.device)
    bad_dev = torch.empty(1, dtype=torch.int64, device=a_dense.device)
    bad = c_longlong(-1)
    code = lib.sp24_compress(dtype_code(dtype if dtype is not None else a_dense.dtype),
                             _ptr(a_dense), m, k, a_dense.stride(0),
                             _ptr(a_c), a_c.stride(0), _ptr(meta), _ptr(bad_dev),
                             ctypes.byref(bad), _stream(stream))
    if code == 3:
        err = Sp24Error(code, f"sp24_compress (first bad group {bad.value})")
        err.bad_group = bad.value
        raise err
    _check(code, "sp24_compress")
    return a_c, meta


def prune_2of4(a, stream=None, dtype=None):
    import torch
    lib = load()
    m, k = a.shape
    out = torch.empty_like(a)
    code = dtype_code(dtype if dtype is not None else a.dtype)
    _check(lib.sp24_prune_2of4(code, _ptr(a), m, k, a.stride(0), _ptr(out),
                               out.stride(0), _stream(stream)), "sp24_prune_2of4")
    return out


def repack_meta(meta_ref, m: int, k: int, dtype, stream=None):
    import torch
    lib = load()
    out = torch.empty(meta_tc_bytes(m, k), dtype=torch.uint8, device=meta_ref.device)
    _check(lib.sp24_repack_meta(dtype_code(dtype), _ptr(meta_ref), m, k, _ptr(out),
                                _stream(stream)), "sp24_repack_meta")
    return out


def repack_meta_k16(meta_k16, m: int, k: int, dtype, stream=None):
    """tcgen05 image from metadata in the reference's m16n8k16 layout."""
    import torch
    lib = load()
    out = torch.empty(meta_tc_bytes(m, k), dtype=torch.uint8, device=meta_k16.device)
    _check(lib.sp24_repack_meta_k16(dtype_code(dtype), _ptr(meta_k16), m, k, _ptr(out),
                                    _stream(stream)), "sp24_repack_meta_k16")
    return out


def make_desc(a_c, meta, b, m, n, k, *, meta_format=META_REF, c_f32=None, c_bf16=None,
              alpha=1.0, tile_n=0, workspace=None, status=None, dtype=None) -> GemmDesc:
    d = GemmDesc()
    d.dtype = dtype_code(dtype if dtype is not None else a_c.dtype)
    d.m, d.n, d.k = m, n, k
    d.a_c, d.lda_c = _ptr(a_c), a_c.stride(0)
    d.meta, d.meta_format = _ptr(meta), meta_format
    d.b, d.ldb = _ptr(b), b.stride(0)
    d.c_f32, d.c_bf16 = _ptr(c_f32), _ptr(c_bf16)
    ref = c_f32 if c_f32 is not None else c_bf16
    d.ldc = ref.stride(0)
    d.alpha = alpha
    d.tile_n = tile_n
    d.workspace = _ptr(workspace)
    d.workspace_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    d.status_dev = _ptr(status)
    return d


def workspace_bytes(desc: GemmDesc) -> int:
    return int(load().sp24_gemm_workspace_bytes(ctypes.byref(desc)))


def gemm(a_c, meta, b, m, n, k, *, meta_format=META_REF, out_f32=True, out_bf16=False,
         alpha=1.0, tile_n=0, workspace=None, c_f32=None, c_bf16=None, stream=None,
         dtype=None):
    """C = alpha * decompress(A_c, meta) @ B through sp24_gemm.  Returns (c_f32, c_bf16)."""
    import torch
    lib = load()
    dev = a_c.device
    if out_f32 and c_f32 is None:
        c_f32 = torch.empty((m, n), dtype=torch.float32, device=dev)
    if out_bf16 and c_bf16 is None:
        c_bf16 = torch.empty((m, n), dtype=torch.bfloat16, device=dev)
    d = make_desc(a_c, meta, b, m, n, k, meta_format=meta_format, c_f32=c_f32, c_bf16=c_bf16,
                  alpha=alpha, tile_n=tile_n, workspace=workspace, dtype=dtype)
    need = workspace_bytes(d)
    if need and (workspace is None or d.workspace_bytes < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        d.workspace, d.workspace_bytes = workspace.data_ptr(), need
    _check(lib.sp24_gemm(ctypes.byref(d), _stream(stream)), "sp24_gemm")
    return c_f32, c_bf16


def gemm_fused(a_c, meta, b, m, n, k, *, bias=None, act=ACT_NONE, a_c_up=None, meta_up=None,
               alpha_up=1.0, bias_up=None, meta_format=META_TC, out_f32=True, out_bf16=False,
               alpha=1.0, tile_n=0, c_f32=None, c_bf16=None, stream=None, dtype=None):
    """sp24_gemm_fused: C = act(alpha A B + bias) [* (alpha_up A_up B + bias_up)]."""
    import torch
    lib = load()
    dev = a_c.device
    if out_f32 and c_f32 is None:
        c_f32 = torch.empty((m, n), dtype=torch.float32, device=dev)
    if out_bf16 and c_bf16 is None:
        c_bf16 = torch.empty((m, n), dtype=torch.bfloat16, device=dev)
    d = make_desc(a_c, meta, b, m, n, k, meta_format=meta_format, c_f32=c_f32, c_bf16=c_bf16,
                  alpha=alpha, tile_n=tile_n, dtype=dtype)
    need = workspace_bytes(d)
    ws = None
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        d.workspace, d.workspace_bytes = ws.data_ptr(), need
    e = Epilogue()
    e.bias, e.act = _ptr(bias), act
    e.a_c_up = _ptr(a_c_up)
    e.lda_c_up = 0 if a_c_up is None else a_c_up.stride(0)
    e.meta_up, e.alpha_up, e.bias_up = _ptr(meta_up), alpha_up, _ptr(bias_up)
    _check(lib.sp24_gemm_fused(ctypes.byref(d), ctypes.byref(e), _stream(stream)),
           "sp24_gemm_fused")
    return c_f32, c_bf16


# ------------------------------------------------------------------ the MLP block
# Activations are token-major: one row per token, its features contiguous.
# These calls serve single tokens, where the host's time is what counts: shapes
# and strides are read once, and descriptors are packed in one go (fields and
# padding as in the structures above).
_PACK_ROWS = struct.Struct("@4iQqQqQqQqQfQqQ").pack
_PACK_SCALED = struct.Struct("@5iQqQQqQQQQqQ").pack
_PACK_FFN = struct.Struct("@5iQqQqQqQNQ").pack
_PACK_GRADS = struct.Struct("@QqQqQqQqQN").pack

def _rows2d(t, what, cols=None, rows=None):
    """(t, row stride) of a matrix whose rows are contiguous, any row stride;
    others are copied.  A single row's stride says nothing: 0."""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{what}: a 2-D tensor is wanted")
    r, c = shape
    if (cols is not None and c != cols) or (rows is not None and r != rows):
        raise ValueError(f"{what}: shape {tuple(shape)}, expected "
                         f"({'any' if rows is None else rows}, {'any' if cols is None else cols})")
    ld, step = t.stride()
    if r > 1 and ld < c or c > 1 and step != 1:
        t = t.contiguous()
        ld = c
    return t, (ld if r > 1 else 0)


def _tma_rows(t, what, cols=None, rows=None):
    """_rows2d whose rows also start on 16-byte boundaries (TMA operands):
    others are copied into padded rows first."""
    t, ld = _rows2d(t, what, cols, rows)
    size = t.element_size()
    if (t.data_ptr() | (ld or t.shape[1]) * size) & 15 == 0:
        return t, ld
    unit = 16 // size
    ld = (t.shape[1] + unit - 1) // unit * unit
    padded = t.new_empty((t.shape[0], ld))[:, :t.shape[1]]
    padded.copy_(t)
    return padded, ld


def _after_copies(lib, call, *args):
    """call(*args) where a weight operand was copied on the stream just now:
    whatever the caller says of its own weights, this launch may not load them
    before the work ahead of it is done.  The hint is the calling thread's own."""
    hints = lib.sp24_get_launch_hints()
    lib.sp24_set_launch_hints(hints & ~HINT_STATIC_WEIGHTS)
    try:
        return call(*args)
    finally:
        lib.sp24_set_launch_hints(hints)


def _same_device(first, *rest):
    """Index of the CUDA device that holds all of them."""
    index = first.get_device()
    if index < 0:
        raise ValueError(f"CUDA tensors are wanted, not {first.device}")
    for t in rest:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on several devices: {first.device}, {t.device}")
    return index


def _on(index, stream, call, *args):
    """call(raw stream, *args) with the tensors' device current and `stream`
    (None: the current one) torch's current stream, so that copies and outputs
    made on the way are ordered with the kernels.  Inputs used on a stream that
    was named are recorded with it: their memory outlives the call there."""
    import torch
    if stream is None and torch._C._cuda_getDevice() == index:
        return call(torch._C._cuda_getCurrentRawStream(index), *args)
    if stream is not None and stream.device_index != index:
        raise ValueError(f"a stream of cuda:{stream.device_index} for tensors on cuda:{index}")
    with torch.cuda.device(index), torch.cuda.stream(stream):
        if stream is not None:
            for t in args:
                if isinstance(t, torch.Tensor):
                    t.record_stream(stream)
        return call(torch._C._cuda_getCurrentRawStream(index), *args)


_codes = {}


def _code_tables():
    """Torch dtype -> library code, by use.  Published whole: another thread sees
    no table or all of them."""
    global _codes
    import torch
    _codes = {
        "16": {torch.float16: F16, torch.bfloat16: BF16},
        "8": {torch.int8: I8, torch.float8_e4m3fn: E4M3},
        "out": {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32},
        "of_8": {I8: torch.int8, E4M3: torch.float8_e4m3fn},
    }
    return _codes


def _rows_quant(s, entry, x, qdtype, up, weight, residual, eps):
    import torch
    tables = _codes or _code_tables()
    dt, q_torch = tables["16"].get(x.dtype), tables["of_8"].get(qdtype)
    if dt is None:
        raise ValueError(f"{entry}: float16 or bfloat16 rows, not {x.dtype}")
    if q_torch is None:
        raise ValueError(f"{entry}: qdtype {qdtype}, not I8 or E4M3")
    for t in (up, weight, residual):
        if t is not None and t.dtype != x.dtype:
            raise ValueError(f"{entry}: {t.dtype} beside {x.dtype}")
    x, ldx = _rows2d(x, "x")
    rows, cols = x.shape
    total = None
    ld_up = ld_res = p_up = p_res = p_total = p_weight = 0
    if up is not None:
        up, ld_up = _rows2d(up, "up", cols, rows)
        p_up = up.data_ptr()
    if weight is not None:
        if weight.shape != (cols,):
            raise ValueError(f"weight: shape {tuple(weight.shape)}, expected ({cols},)")
        weight = weight.contiguous()
        p_weight = weight.data_ptr()
    plain = x.is_contiguous()
    if residual is not None:
        residual, ld_res = _rows2d(residual, "residual", cols, rows)
        total = torch.empty_like(x) if plain else x.new_empty((rows, cols))
        p_res, p_total = residual.data_ptr(), total.data_ptr()
    q = torch.empty_like(x, dtype=q_torch) if plain else x.new_empty((rows, cols), dtype=q_torch)
    scale = x.new_empty((rows,), dtype=torch.float32)
    d = _PACK_ROWS(dt, qdtype, rows, cols, x.data_ptr(), ldx, p_up, ld_up, p_res, ld_res,
                   p_total, 0, p_weight, eps, q.data_ptr(), 0, scale.data_ptr())
    _check(getattr(_lib or load(), entry)(d, s), entry)
    return (q, scale) if total is None else (q, scale, total)


def rmsnorm_quant(x, weight, residual=None, *, eps=1e-6, qdtype=I8, stream=None):
    """sp24_rmsnorm_quant: 8-bit rows of rmsnorm(x [+ residual]) * weight.
    Returns (q, scale), or (q, scale, x + residual) when a residual is given;
    a row's values are q * scale."""
    return _on(_same_device(x, weight, residual), stream, _rows_quant, "sp24_rmsnorm_quant", x,
               qdtype, None, weight, residual, eps)


def swiglu_quant(gate, up, *, qdtype=I8, stream=None):
    """sp24_swiglu_quant: 8-bit rows of silu(gate) * up -> (q, scale)."""
    return _on(_same_device(gate, up), stream, _rows_quant, "sp24_swiglu_quant", gate, qdtype, up,
               None, None, 0.0)


def quantize_rows(x, *, qdtype=I8, stream=None):
    """sp24_quantize_rows: 8-bit rows of x -> (q, scale).  Applied to a 16-bit
    A_c it gives the 8-bit weights of gemm_scaled and their channel scales."""
    return _on(_same_device(x), stream, _rows_quant, "sp24_quantize_rows", x, qdtype, None, None,
               None, 0.0)


def _vector_f32(t, size, what):
    """(tensor to keep, pointer) of an optional vector of `size` floats."""
    import torch
    if t is None:
        return None, 0
    if t.dtype != torch.float32 or t.numel() != size:
        raise ValueError(f"{what}: {size} float32 values are wanted")
    if not t.is_contiguous():
        t = t.contiguous()
    return t, t.data_ptr()


def _gemm_scaled(s, a_c, meta_tc, x, scale_w, scale_x, bias, out_dtype):
    import torch
    lib = _lib or load()
    tables = _codes or _code_tables()
    code, out = tables["8"].get(x.dtype), tables["out"].get(out_dtype or torch.bfloat16)
    if code is None or a_c.dtype != x.dtype:
        raise ValueError(f"gemm_scaled: {x.dtype} tokens and {a_c.dtype} weights; both int8 or "
                         "both float8_e4m3fn are wanted")
    if out is None:
        raise ValueError(f"gemm_scaled: out_dtype {out_dtype}")
    given, copied = a_c, False
    a_c, lda = _tma_rows(a_c, "a_c")
    m, k = a_c.shape[0], 2 * a_c.shape[1]
    x, ldx = _tma_rows(x, "x", k)
    n = x.shape[0]
    image = (m + 255) // 256 * ((k + 127) // 128) * 4096      # sp24_meta_tc_bytes
    if meta_tc.nbytes != image:
        raise ValueError(f"meta_tc: {meta_tc.nbytes} bytes, {image} expected")
    if not meta_tc.is_contiguous():
        meta_tc, copied = meta_tc.contiguous(), True
    scale_w, p_w = _vector_f32(scale_w, m, "scale_w")
    scale_x, p_x = _vector_f32(scale_x, n, "scale_x")
    bias, p_b = _vector_f32(bias, m, "bias")
    c = x.new_empty((n, m), dtype=out_dtype or torch.bfloat16)
    d = _PACK_SCALED(code, out, m, n, k, a_c.data_ptr(), lda, meta_tc.data_ptr(), x.data_ptr(), ldx,
                     p_w, p_x, p_b, c.data_ptr(), 0, 0)
    if copied or a_c is not given:
        code = _after_copies(lib, lib.sp24_gemm_scaled, d, s)
    else:
        code = lib.sp24_gemm_scaled(d, s)
    _check(code, "sp24_gemm_scaled")
    return c


def gemm_scaled(a_c, meta_tc, x, scale_w=None, scale_x=None, *, bias=None, out_dtype=None,
                stream=None):
    """sp24_gemm_scaled: tokens x [n, k] (int8 or e4m3) times the 2:4 weights
    (a_c [m, k/2] of the same type, tcgen05 metadata image) with a scale for
    each channel (scale_w [m]) and each token (scale_x [n]) -> [n, m] of
    out_dtype (bfloat16, float16 or float32; default bfloat16)."""
    return _on(_same_device(x, a_c, meta_tc, scale_w, scale_x, bias), stream, _gemm_scaled, a_c,
               meta_tc, x, scale_w, scale_x, bias, out_dtype)


def _ffn_args(x, w_gate, w_up, act):
    """The leading fields of a descriptor, and the tensors they point to."""
    dt = (_codes or _code_tables())["16"].get(x.dtype)
    if dt is None or w_gate.dtype != x.dtype or w_up.dtype != x.dtype:
        raise ValueError(f"ffn_gated: {x.dtype}, {w_gate.dtype}, {w_up.dtype}; one of float16 and "
                         "bfloat16 for all is wanted")
    x, ldx = _tma_rows(x, "x")
    t, h = x.shape
    w_gate, ldg = _tma_rows(w_gate, "w_gate", h)
    f = w_gate.shape[0]
    w_up, ldu = _tma_rows(w_up, "w_up", h, f)
    return (dt, t, h, f, act, x.data_ptr(), ldx, w_gate.data_ptr(), ldg, w_up.data_ptr(), ldu), \
        (x, w_gate, w_up)


def _ffn_forward(s, x, w_gate, w_up, act, save):
    import torch
    lib = _lib or load()
    args, keep = _ffn_args(x, w_gate, w_up, act)
    t, f = args[1], args[3]
    out = x.new_empty((t, f))
    saved, p_saved, n_saved = None, 0, 0
    if save:
        n_saved = lib.sp24_ffn_saved_bytes(t, f)
        saved = x.new_empty((n_saved,), dtype=torch.uint8)
        p_saved = saved.data_ptr()
    call = _PACK_FFN(*args, p_saved, n_saved, 0), out.data_ptr(), 0, s
    if keep[1] is not w_gate or keep[2] is not w_up:
        code = _after_copies(lib, lib.sp24_ffn_forward, *call)
    else:
        code = lib.sp24_ffn_forward(*call)
    _check(code, "sp24_ffn_forward")
    del keep
    return (out, saved) if save else out


def ffn_gated(x, w_gate, w_up, *, act=ACT_SILU, save=False, stream=None):
    """sp24_ffn_forward: act(x w_gate^T) * (x w_up^T) -> [t, f], act one of
    ACT_SILU, ACT_GELU_TANH and ACT_NONE; with save=True also the opaque buffer
    that ffn_gated_backward takes.  No autograd graph is recorded, not for inputs
    that require gradients either: they come from ffn_gated_backward."""
    return _on(_same_device(x, w_gate, w_up), stream, _ffn_forward, x, w_gate, w_up, act, save)


def _ffn_backward(s, d_out, x, w_gate, w_up, saved, act, need_dx, need_dw):
    import torch
    lib = _lib or load()
    if d_out.dtype != x.dtype:
        raise ValueError(f"ffn_gated_backward: {d_out.dtype} beside {x.dtype}")
    args, keep = _ffn_args(x, w_gate, w_up, act)
    _, t, h, f = args[:4]
    d_out, ldd = _rows2d(d_out, "d_out", f, t)
    if not saved.is_contiguous():
        saved = saved.contiguous()
    dx = x.new_empty((t, h)) if need_dx else None
    dw_gate = dw_up = None
    if need_dw:
        dw_gate, dw_up = x.new_empty((f, h)), x.new_empty((f, h))
    ws = x.new_empty((lib.sp24_ffn_workspace_bytes(t, h, f),), dtype=torch.uint8)
    d = _PACK_FFN(*args, saved.data_ptr(), saved.nbytes, 0)
    g = _PACK_GRADS(d_out.data_ptr(), ldd, _ptr(dx), 0, _ptr(dw_gate), 0, _ptr(dw_up), 0,
                    ws.data_ptr(), ws.nbytes)
    _check(lib.sp24_ffn_backward(d, g, s), "sp24_ffn_backward")
    del keep
    return dx, dw_gate, dw_up


def ffn_gated_backward(d_out, x, w_gate, w_up, saved, *, act=ACT_SILU, need_dx=True,
                       need_dw=True, stream=None):
    """sp24_ffn_backward: (dx, dw_gate, dw_up) from dL/dout and what
    ffn_gated(save=True) kept (None for gradients that are not wanted)."""
    return _on(_same_device(x, d_out, w_gate, w_up, saved), stream, _ffn_backward, d_out, x,
               w_gate, w_up, saved, act, need_dx, need_dw)


def ipc_handle(t):
    """(64-byte handle, byte offset) of the CUDA allocation holding tensor t."""
    h = ctypes.create_string_buffer(64)
    off = c_size_t(0)
    _check(load().sp24_ipc_get_handle(_ptr(t), h, ctypes.byref(off)), "sp24_ipc_get_handle")
    return h.raw, off.value


def ipc_open(handle: bytes) -> int:
    """Map a peer's allocation into this process; returns its base address."""
    base = c_void_p(0)
    buf = ctypes.create_string_buffer(handle, 64)
    _check(load().sp24_ipc_open_handle(buf, ctypes.byref(base)), "sp24_ipc_open_handle")
    return base.value


def ipc_close(base: int) -> None:
    _check(load().sp24_ipc_close(c_void_p(base)), "sp24_ipc_close")


def gemm_allgather(desc: GemmDesc, peer_f32=(), peer_bf16=(), stream=None) -> None:
    """sp24_gemm_allgather with peer element addresses (ints) for each output."""
    po = PeerOut()
    po.n_peers = max(len(peer_f32), len(peer_bf16))
    for i, a in enumerate(peer_f32):
        po.c_f32[i] = a
    for i, a in enumerate(peer_bf16):
        po.c_bf16[i] = a
    _check(load().sp24_gemm_allgather(ctypes.byref(desc), ctypes.byref(po), _stream(stream)),
           "sp24_gemm_allgather")


def replicate(src, dsts, streams=None) -> None:
    """sp24_replicate: copy tensor src into each tensor of dsts (one per
    device, same size), enqueued on each destination device's stream."""
    n = len(dsts)
    devs = (c_int * n)(*[t.device.index for t in dsts])
    ptrs = (c_void_p * n)(*[t.data_ptr() for t in dsts])
    strs = (c_void_p * n)(*[(s.cuda_stream if s is not None else None) for s in
                            (streams or [None] * n)])
    _check(load().sp24_replicate(src.data_ptr(), src.device.index,
                                 src.numel() * src.element_size(), n, devs, ptrs, strs),
           "sp24_replicate")


def make_multi_desc(m, n, k, dtype, a_c, meta, b, *, c_f32=None, c_bf16=None,
                    meta_format=META_TC, b_layout=MULTI_FULL, c_layout=MULTI_FULL, ldb=0, ldc=0,
                    alpha=1.0, workspaces=None, streams=None) -> MultiDesc:
    """A sp24_multi_desc from per-device tensors (lists, one per GPU, in
    device order)."""
    md = MultiDesc()
    g = md.gemm
    g.dtype, g.m, g.n, g.k = dtype_code(dtype), m, n, k
    g.meta_format, g.ldb, g.ldc, g.alpha = meta_format, ldb, ldc, alpha
    md.ngpu = len(a_c)
    for i, t in enumerate(a_c):
        md.devices[i] = t.device.index
        md.a_c[i], md.meta[i], md.b[i] = t.data_ptr(), meta[i].data_ptr(), b[i].data_ptr()
        md.c_f32[i] = _ptr(c_f32[i]) if c_f32 is not None else None
        md.c_bf16[i] = _ptr(c_bf16[i]) if c_bf16 is not None else None
        md.streams[i] = streams[i].cuda_stream if streams is not None else None
        if workspaces is not None and workspaces[i] is not None:
            md.workspace[i] = workspaces[i].data_ptr()
    if workspaces is not None:
        md.workspace_bytes = min(w.numel() for w in workspaces if w is not None)
    md.b_layout, md.c_layout = b_layout, c_layout
    g.lda_c = a_c[0].stride(0)
    return md


def multi_workspace_bytes(md: MultiDesc) -> int:
    return int(load().sp24_gemm_multi_workspace_bytes(ctypes.byref(md)))


def gemm_multi(md: MultiDesc, allgather_c: bool = False) -> list:
    """sp24_gemm_multi; when md carries no workspaces and the problem needs
    them, allocates one per device first.  Returns the workspaces (keep them
    alive until the streams are done)."""
    import torch
    keep = []
    need = multi_workspace_bytes(md)
    if need and not any(md.workspace[i] for i in range(md.ngpu)):
        for i in range(md.ngpu):
            w = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", md.devices[i]))
            md.workspace[i] = w.data_ptr()
            keep.append(w)
        md.workspace_bytes = need
    _check(load().sp24_gemm_multi(ctypes.byref(md), 1 if allgather_c else 0), "sp24_gemm_multi")
    return keep


def set_launch_hints(hints: int) -> None:
    """sp24_set_launch_hints for later GEMM calls of this thread
    (HINT_STATIC_WEIGHTS: A_c / metadata images are not written by in-flight work)."""
    load().sp24_set_launch_hints(hints)


def get_launch_hints() -> int:
    return load().sp24_get_launch_hints()


def reload_tuning() -> None:
    """sp24_reload_tuning: the library reads its SP24_* tuning variables once;
    call this after changing them in os.environ."""
    load().sp24_reload_tuning()


class tuning_env:
    """Context manager: set SP24_* tuning variables for the calls inside it
    (and re-read them in the library), restoring the old values on exit."""

    def __init__(self, env: dict):
        self.env = {k: str(v) for k, v in env.items()}

    def __enter__(self):
        self.old = {k: os.environ.get(k) for k in self.env}
        os.environ.update(self.env)
        reload_tuning()
        return self

    def __exit__(self, *exc):
        for k, v in self.old.items():
            if v is None:
                os.environ.pop(k, None)
            else:
                os.environ[k] = v
        reload_tuning()


def last_kernel_status(stream=None) -> int:
    return int(load().sp24_last_kernel_status(_stream(stream)))


def amax_quantize_e4m3(x, stream=None, e5m2=False):
    """fp32 CUDA tensor -> (fp8 bits as uint8, scale tensor[1]) with scale =
    448/amax (e4m3) or 57344/amax (e5m2)."""
    import torch
    lib = load()
    amax = torch.empty(1, dtype=torch.float32, device=x.device)
    scale = torch.empty(1, dtype=torch.float32, device=x.device)
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    s = _stream(stream)
    _check(lib.sp24_amax_f32(_ptr(x), x.numel(), _ptr(amax), s), "sp24_amax_f32")
    fn = lib.sp24_quantize_e5m2 if e5m2 else lib.sp24_quantize_e4m3
    _check(fn(_ptr(x), x.numel(), _ptr(amax), _ptr(scale), _ptr(q), s),
           "sp24_quantize_e5m2" if e5m2 else "sp24_quantize_e4m3")
    return q, scale


def amax_quantize_e5m2(x, stream=None):
    return amax_quantize_e4m3(x, stream, e5m2=True)


def shard_columns(n: int, world: int, rank: int, align: int):
    a, b = c_int(0), c_int(0)
    load().sp24_shard_columns(n, world, rank, align, ctypes.byref(a), ctypes.byref(b))
    return a.value, b.value


def unshard_columns_f32(src, m: int, n: int, world: int, align: int, stream=None):
    import torch
    dst = torch.empty((m, n), dtype=torch.float32, device=src.device)
    _check(load().sp24_unshard_columns_f32(_ptr(src), _ptr(dst), m, n, world, align,
                                           _stream(stream)), "sp24_unshard_columns_f32")
    return dst


_peak = None


def probe_mma_rate(dtype: int, sparse: bool, iters: int = 4096, reps: int = 5, stream=None):
    """Tensor-core rate of the CTA-pair MMA shape with operands resident in
    shared memory (lib/libsp24_peak.so, measurement only): returns
    (dense-equivalent TFLOP/s, ms per launch).  dtype: F16, BF16 or E4M3."""
    global _peak
    import torch
    if _peak is None:
        if not os.path.exists(PEAK_LIB_PATH):
            raise FileNotFoundError(f"{PEAK_LIB_PATH} missing: run __graft_entry__.build() first")
        _peak = ctypes.CDLL(PEAK_LIB_PATH)
        _peak.sp24_probe_mma_rate.restype = c_int
        _peak.sp24_probe_mma_rate.argtypes = [c_int, c_int, c_int, c_int, POINTER(c_float),
                                              POINTER(ctypes.c_double), c_void_p, c_void_p]
    ms, flops = c_float(0.0), ctypes.c_double(0.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check(_peak.sp24_probe_mma_rate(dtype, 1 if sparse else 0, iters, reps, ctypes.byref(ms),
                                     ctypes.byref(flops), _ptr(status), _stream(stream)),
           "sp24_probe_mma_rate")
    torch.cuda.synchronize()
    if status.item() != 0:
        raise Sp24Error(6, "sp24_probe_mma_rate")
    return flops.value / (ms.value * 1e-3) / 1e12, ms.value
