"""ctypes binding of libmoss_hip.so (C ABI declared in include/moss_hip.h).

The library is the product: if it is missing this module raises instead of
falling back to anything else.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PKG_DIR, "libmoss_hip.so")

OK, EINVAL, EDEVICE, EFORMAT, EUNSUPPORTED, ESTATE = 0, 1, 2, 3, 4, 5
F32, F16, I8, E4M3 = 0, 1, 2, 3

# Quantiser capture (moss_hip_llm_capture): kinds and the per-step float offsets of a decode
# capture, as include/moss_hip.h declares them (name -> (offset, length)).
CAP_GLOBAL, CAP_LOCAL, CAP_PREFILL = 0, 1, 2
CAP_STEP = 17088
CAP = {"xin": (0, 768), "ln1": (768, 768), "ln1_q": (1536, 768), "ln1_d": (2304, 24), "qkv": (2328, 2304),
       "att": (4632, 768), "att_q": (5400, 768), "att_d": (6168, 24), "xm": (6192, 768), "ln2": (6960, 768),
       "ln2_q": (7728, 768), "ln2_d": (8496, 24), "h": (8520, 3072), "h_q": (11592, 3072), "h_d": (14664, 96),
       "xout": (14760, 768), "lnf": (15528, 768), "lnf_q": (16296, 768), "lnf_d": (17064, 24)}

EXPORTED = [
    "moss_hip_last_error", "moss_hip_abi_version",
    "moss_hip_llm_create", "moss_hip_llm_create_from_file", "moss_hip_llm_destroy", "moss_hip_llm_reset",
    "moss_hip_llm_position", "moss_hip_llm_get_hidden", "moss_hip_llm_set_hidden", "moss_hip_llm_prefill",
    "moss_hip_llm_global_step", "moss_hip_llm_generate", "moss_hip_llm_set_cancel_flag",
    "moss_hip_llm_snapshot_prefix", "moss_hip_llm_restore_prefix", "moss_hip_llm_prefix_pos",
    "moss_hip_llm_gate_rows", "moss_hip_llm_fallbacks", "moss_hip_fallbacks_total",
    "moss_hip_llm_kv_export", "moss_hip_llm_kv_import", "moss_hip_llm_capture", "moss_hip_llm_capture_read",
    "moss_hip_batch_create", "moss_hip_batch_destroy", "moss_hip_batch_set_stream", "moss_hip_batch_admit", "moss_hip_batch_get_hidden",
    "moss_hip_batch_position", "moss_hip_batch_kv_export", "moss_hip_batch_global_step", "moss_hip_batch_generate",
    "moss_hip_batch_capture", "moss_hip_batch_capture_read",
    "moss_hip_gemv_q8x4", "moss_hip_gemm_q8x4", "moss_hip_dequant_rows_q8x4", "moss_hip_attn_decode",
    "moss_hip_attn_decode_noalloc", "moss_hip_attn_paged",
    "moss_hip_quantize_rows", "moss_hip_gemm_q8x4_w8a8", "moss_hip_gemv_q8x4_w8a8",
    "moss_hip_rope_freqs", "moss_hip_rope_rows", "moss_hip_kv_write", "moss_hip_kv_read",
    "moss_hip_attn_tree", "moss_hip_attn_tree_workspace",
    "moss_hip_token_logprobs", "moss_hip_token_logprobs_workspace",
    "moss_hip_codec_create", "moss_hip_codec_create_from_file", "moss_hip_codec_destroy",
    "moss_hip_codec_samples_per_frame", "moss_hip_codec_reset_stream", "moss_hip_codec_decode_chunk",
    "moss_hip_codec_decode", "moss_hip_codec_last_ms", "moss_hip_codec_stage_ms",
]


class MossHipError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


class Options(C.Structure):
    _fields_ = [("device", C.c_int), ("max_ctx", C.c_int), ("kv_dtype", C.c_int), ("use_graphs", C.c_int),
                ("prefill_a16", C.c_int), ("decode_kernels", C.c_int), ("decode_a8", C.c_int)]


class CodecOptions(C.Structure):
    """moss_hip_codec_options."""
    _fields_ = [("device", C.c_int), ("max_chunk_frames", C.c_int), ("contexts", C.c_int * 4), ("eager", C.c_int)]


class SampleParams(C.Structure):
    """moss_hip_sample_params == SampleParams (csrc/include/moss/sampler.h:8-22)."""
    _fields_ = [("greedy", C.c_int), ("temperature", C.c_float), ("top_k", C.c_int), ("top_p", C.c_float),
                ("repetition_penalty", C.c_float), ("end_greedy", C.c_int), ("min_frames", C.c_int),
                ("greedy_frames", C.c_int)]

    @classmethod
    def make(cls, greedy=True, temperature=1.0, top_k=0, top_p=1.0, repetition_penalty=1.0, end_greedy=True,
             min_frames=0, greedy_frames=0):
        return cls(int(greedy), temperature, top_k, top_p, repetition_penalty, int(end_greedy), min_frames,
                   greedy_frames)


class RopeParams(C.Structure):
    """moss_hip_rope_params."""
    _fields_ = [("rot_dim", C.c_int), ("scaling", C.c_int), ("base", C.c_double), ("factor", C.c_double),
                ("orig_ctx", C.c_int), ("beta_fast", C.c_double), ("beta_slow", C.c_double)]


class RopeStruct(C.Structure):
    """moss_hip_rope."""
    _fields_ = [("freqs", C.c_void_p), ("rot_dim", C.c_int), ("halves", C.c_int), ("mscale", C.c_float)]


class KVCacheStruct(C.Structure):
    """moss_hip_kv_cache."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("kv_dtype", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int), ("page_size", C.c_int),
                ("n_pages", C.c_int), ("page_table", C.c_void_p), ("table_stride", C.c_int), ("streams", C.c_int)]


FRAME_CB = C.CFUNCTYPE(None, C.c_void_p, C.c_int, C.POINTER(C.c_int32))

_lib = None


def load(path: str = LIB_PATH) -> C.CDLL:
    """Load libmoss_hip.so (once).  Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing: build it with `make -C dsh-moss-tts_amd` (or __graft_entry__.build())")
    L = C.CDLL(path)
    vp, i32, f32p = C.c_void_p, C.c_int, C.POINTER(C.c_float)
    L.moss_hip_last_error.restype = C.c_char_p
    L.moss_hip_abi_version.restype = C.c_int
    L.moss_hip_llm_create.argtypes = [vp, C.c_size_t, C.POINTER(Options), C.POINTER(vp)]
    L.moss_hip_llm_create_from_file.argtypes = [C.c_char_p, C.POINTER(Options), C.POINTER(vp)]
    L.moss_hip_llm_destroy.argtypes = [vp]
    L.moss_hip_llm_destroy.restype = None
    for n in ("moss_hip_llm_reset", "moss_hip_llm_snapshot_prefix", "moss_hip_llm_restore_prefix"):
        getattr(L, n).argtypes = [vp]
    L.moss_hip_llm_position.argtypes = [vp]
    L.moss_hip_llm_prefix_pos.argtypes = [vp]
    L.moss_hip_llm_gate_rows.argtypes = [vp]
    L.moss_hip_llm_fallbacks.argtypes = [vp]
    L.moss_hip_llm_get_hidden.argtypes = [vp, vp]
    L.moss_hip_llm_set_hidden.argtypes = [vp, vp]
    L.moss_hip_llm_prefill.argtypes = [vp, vp, i32, i32]
    L.moss_hip_llm_global_step.argtypes = [vp, vp]
    L.moss_hip_llm_generate.argtypes = [vp, i32, C.POINTER(SampleParams), C.c_uint64, vp, i32, vp, C.POINTER(i32),
                                        vp, vp, vp, FRAME_CB, vp]
    L.moss_hip_llm_set_cancel_flag.argtypes = [vp, vp]
    L.moss_hip_llm_kv_export.argtypes = [vp, i32, vp, vp]
    L.moss_hip_llm_kv_import.argtypes = [vp, i32, vp, vp, vp]
    L.moss_hip_llm_capture.argtypes = [vp, i32]
    L.moss_hip_llm_capture_read.argtypes = [vp, i32, vp, C.c_size_t, C.POINTER(C.c_size_t)]
    L.moss_hip_gemv_q8x4.argtypes = [vp, i32, i32, vp, i32, vp, i32, vp]
    L.moss_hip_gemv_q8x4_w8a8.argtypes = [vp, i32, i32, vp, vp, vp]
    L.moss_hip_gemm_q8x4.argtypes = [vp, i32, i32, vp, i32, vp, vp]
    L.moss_hip_quantize_rows.argtypes = [vp, i32, i32, vp, vp, vp]
    L.moss_hip_gemm_q8x4_w8a8.argtypes = [vp, i32, i32, vp, vp, i32, vp, vp]
    L.moss_hip_batch_create.argtypes = [vp, i32, i32, i32, C.POINTER(vp)]
    L.moss_hip_batch_destroy.argtypes = [vp]
    L.moss_hip_batch_destroy.restype = None
    L.moss_hip_batch_set_stream.argtypes = [vp, i32, i32, vp, vp, vp]
    L.moss_hip_batch_admit.argtypes = [vp, i32, vp]
    L.moss_hip_batch_capture.argtypes = [vp, i32]
    L.moss_hip_batch_capture_read.argtypes = [vp, vp, C.c_size_t, C.POINTER(C.c_size_t)]
    L.moss_hip_batch_get_hidden.argtypes = [vp, i32, vp]
    L.moss_hip_batch_position.argtypes = [vp, i32]
    L.moss_hip_batch_kv_export.argtypes = [vp, i32, i32, vp, vp]
    L.moss_hip_batch_global_step.argtypes = [vp, i32, vp]
    L.moss_hip_batch_generate.argtypes = [vp, i32, i32, C.POINTER(SampleParams), vp, vp, vp, C.POINTER(C.c_double)]
    L.moss_hip_dequant_rows_q8x4.argtypes = [vp, i32, i32, vp, i32, vp, vp]
    L.moss_hip_attn_decode.argtypes = [vp, vp, vp, i32, i32, i32, i32, vp, i32, vp]
    L.moss_hip_attn_decode_noalloc.argtypes = [vp, vp, vp, i32, i32, i32, i32, vp, i32, vp]
    L.moss_hip_attn_paged.argtypes = [vp, vp, vp, i32, i32, vp, i32, i32, i32, vp, vp, i32, vp, i32, vp]
    i64, f32, sz = C.c_int64, C.c_float, C.c_size_t
    L.moss_hip_rope_freqs.argtypes = [C.POINTER(RopeParams), vp, C.POINTER(f32)]
    L.moss_hip_rope_rows.argtypes = [vp, i64, i64, vp, i64, i64, i32, i32, i32, i32, vp, vp, vp]
    L.moss_hip_kv_write.argtypes = [vp, vp, i64, vp, i64, i32, i32, vp, vp, vp, vp, vp]
    L.moss_hip_kv_read.argtypes = [vp, vp, vp, i32, vp, i64, vp, i64, i32, vp]
    L.moss_hip_attn_tree.argtypes = [vp, i64, i32, i32, vp, vp, vp, vp, i32, i32, i32, f32, vp, i64, i32, vp, vp, sz, vp]
    L.moss_hip_attn_tree_workspace.argtypes = [vp, i32, i32, i32, i32, C.POINTER(sz)]
    L.moss_hip_token_logprobs.argtypes = [vp, i64, i32, i32, i32, vp, f32, vp, vp, i32, vp, vp, vp, sz, vp]
    L.moss_hip_token_logprobs_workspace.argtypes = [i32, i32, i32, C.POINTER(sz)]
    L.moss_hip_codec_create.argtypes = [vp, C.c_size_t, C.POINTER(CodecOptions), C.POINTER(vp)]
    L.moss_hip_codec_create_from_file.argtypes = [C.c_char_p, C.POINTER(CodecOptions), C.POINTER(vp)]
    L.moss_hip_codec_destroy.argtypes = [vp]
    L.moss_hip_codec_destroy.restype = None
    L.moss_hip_codec_samples_per_frame.argtypes = [vp]
    L.moss_hip_codec_reset_stream.argtypes = [vp]
    L.moss_hip_codec_decode_chunk.argtypes = [vp, vp, i32, vp]
    L.moss_hip_codec_decode.argtypes = [vp, vp, i32, vp]
    L.moss_hip_codec_last_ms.argtypes = [vp]
    L.moss_hip_codec_last_ms.restype = C.c_double
    L.moss_hip_codec_stage_ms.argtypes = [vp, C.POINTER(C.c_double)]
    _lib = L
    return L


def check(rc: int) -> None:
    if rc != OK:
        raise MossHipError(rc, load().moss_hip_last_error().decode(errors="replace"))


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


# ---------------------------------------------------------------- operators (torch device tensors)

def _stream(stream):
    if stream is not None:
        return C.c_void_p(stream)
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def gemv_q8x4(w, rows: int, cols: int, x, y, stream=None) -> None:
    """y = W x on the device.  w: uint8 tensor (Q8_0_4X4), x/y: float32 or float16 tensors."""
    import torch
    dt = {torch.float32: F32, torch.float16: F16}
    check(load().moss_hip_gemv_q8x4(C.c_void_p(w.data_ptr()), rows, cols, C.c_void_p(x.data_ptr()), dt[x.dtype],
                                    C.c_void_p(y.data_ptr()), dt[y.dtype], _stream(stream)))


def gemv_q8x4_w8a8(w, rows: int, cols: int, x, y, stream=None) -> None:
    """y = W x with x quantised per 32-block (the reference's W8A8 gemv_par); x, y fp32."""
    check(load().moss_hip_gemv_q8x4_w8a8(C.c_void_p(w.data_ptr()), rows, cols, C.c_void_p(x.data_ptr()),
                                         C.c_void_p(y.data_ptr()), _stream(stream)))


def gemm_q8x4(w, rows: int, cols: int, x, m: int, y, stream=None) -> None:
    """Y[m][rows] = X[m][cols] W^T on the matrix cores (fp32 x / y device tensors)."""
    check(load().moss_hip_gemm_q8x4(C.c_void_p(w.data_ptr()), rows, cols, C.c_void_p(x.data_ptr()), m,
                                    C.c_void_p(y.data_ptr()), _stream(stream)))


def quantize_rows(x, m: int, cols: int, q, d, stream=None) -> None:
    """W8A8 activation quantisation: q[m][cols] int8, d[m][cols/32] fp32 (device tensors)."""
    check(load().moss_hip_quantize_rows(C.c_void_p(x.data_ptr()), m, cols, C.c_void_p(q.data_ptr()),
                                        C.c_void_p(d.data_ptr()), _stream(stream)))


def gemm_q8x4_w8a8(w, rows: int, cols: int, q, d, m: int, y, stream=None) -> None:
    """Y[m][rows] from int8 activations q and block scales d on the int8 matrix cores."""
    check(load().moss_hip_gemm_q8x4_w8a8(C.c_void_p(w.data_ptr()), rows, cols, C.c_void_p(q.data_ptr()),
                                         C.c_void_p(d.data_ptr()), m, C.c_void_p(y.data_ptr()), _stream(stream)))


def dequant_rows_q8x4(w, mat_rows: int, cols: int, rows_idx, out, stream=None) -> None:
    check(load().moss_hip_dequant_rows_q8x4(C.c_void_p(w.data_ptr()), mat_rows, cols, C.c_void_p(rows_idx.data_ptr()),
                                            rows_idx.numel(), C.c_void_p(out.data_ptr()), _stream(stream)))


def attn_decode(q, k_cache, v_cache, heads: int, ctx_stride: int, n_keys: int, out, stream=None,
                noalloc: bool = False) -> None:
    """moss_hip_attn_decode, or with noalloc=True moss_hip_attn_decode_noalloc (static scratch)."""
    import torch
    dt = {torch.float32: F32, torch.float16: F16}
    L = load()
    fn = L.moss_hip_attn_decode_noalloc if noalloc else L.moss_hip_attn_decode
    check(fn(C.c_void_p(q.data_ptr()), C.c_void_p(k_cache.data_ptr()), C.c_void_p(v_cache.data_ptr()),
             dt[k_cache.dtype], heads, ctx_stride, n_keys, C.c_void_p(out.data_ptr()), dt[out.dtype], _stream(stream)))


def attn_paged(q, k_pool, v_pool, heads: int, page_table, table_stride: int, page_size: int, row_pos, max_keys: int,
               out, row_stream=None, stream=None) -> None:
    """moss_hip_attn_paged: row r (stream row_stream[r], or r) attends its keys 0 .. row_pos[r]."""
    import torch
    dt = {torch.float32: F32, torch.float16: F16}
    L = load()
    rows = q.shape[0]
    check(L.moss_hip_attn_paged(C.c_void_p(q.data_ptr()), C.c_void_p(k_pool.data_ptr()), C.c_void_p(v_pool.data_ptr()),
                                dt[k_pool.dtype], heads, C.c_void_p(page_table.data_ptr()), table_stride, page_size,
                                rows, C.c_void_p(row_stream.data_ptr()) if row_stream is not None else None,
                                C.c_void_p(row_pos.data_ptr()), max_keys, C.c_void_p(out.data_ptr()), dt[out.dtype],
                                _stream(stream)))


# ---------------------------------------------------------------- a caller's own decoding loop

ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


# These calls are a few microseconds long, so their Python is kept short: torch is looked up once, devices are
# compared as numbers, and a stream is asked for as its handle.
_torch = None


def _t():
    global _torch
    if _torch is None:
        import torch
        _torch = torch
    return _torch


def _types(t):
    """Element type of a tensor of rows."""
    torch, d = _t(), t.dtype
    if d is torch.float32:
        return F32
    if d is torch.float16:
        return F16
    raise TypeError(f"float32 or float16 rows are wanted, not {d}")


def _whole(name, t, dtype, shape, device, optional=False):
    """The address of a contiguous tensor of this type and shape on this device's number (None: NULL)."""
    if t is None and optional:
        return None
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name}: a contiguous {dtype} tensor of shape {tuple(shape)} on device {device} is wanted, "
                     f"not {t.dtype} {tuple(t.shape)} on {t.device}")


def _on(device, stream):
    """The stream to launch on: the caller's handle, or torch's current one.  The calls launch on the current device:
    tensors of another one are refused."""
    torch = _t()
    if device < 0:
        raise ValueError("tensors on the GPU are wanted")
    if device != torch.cuda.current_device():
        raise ValueError(f"the tensors are on cuda:{device}, the current device is cuda:{torch.cuda.current_device()}")
    if stream is not None:
        return stream
    # (torch.cuda.current_stream() makes an object first: 2.9 us, where the handle takes 0.1)
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream().cuda_stream


def _rows(name, t, heads, dim, device):
    """(address, row stride) of rows [rows][heads][dim] (or [rows][heads * dim]) whose rows are contiguous."""
    shape, st = t.shape, t.stride()
    if len(shape) == 3:
        fits, whole = shape[1] == heads and shape[2] == dim, st[2] == 1 and (st[1] == dim or heads == 1)
    else:
        fits, whole = len(shape) == 2 and shape[1] == heads * dim, st[-1] == 1
    if not fits or t.get_device() != device:
        raise ValueError(f"{name}: [rows][{heads}][{dim}] on device {device} is wanted, not {tuple(shape)} on {t.device}")
    if not whole:
        raise ValueError(f"{name}: the heads of a row must be contiguous")
    return t.data_ptr(), st[0]


def _workspace(given, size_of, device, stream):
    """(address, bytes): the caller's (the call checks that it is large enough), or a new one from torch's allocator,
    which is safe on torch's current stream."""
    torch = _t()
    if given is None:
        size = size_of()
        if size == 0:
            return None, 0
        if stream is not None and stream != torch.cuda.current_stream().cuda_stream:
            raise ValueError("on a stream other than torch's current one, pass a workspace")
        given = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", device))
    elif given.get_device() != device or not given.is_contiguous():
        raise ValueError(f"workspace: a contiguous tensor on device {device} is wanted")
    return given.data_ptr(), given.numel() * given.element_size()


def rope_freqs(rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, orig_ctx: int = 0,
               beta_fast: float = 0.0, beta_slow: float = 0.0):
    """moss_hip_rope_freqs: (angles per position [rot_dim / 2] float64, the factor of sine and cosine)."""
    p = RopeParams(rot_dim, ROPE_SCALING[scaling], base, factor, orig_ctx, beta_fast, beta_slow)
    f, m = np.empty(max(rot_dim // 2, 1), np.float64), C.c_float(1.0)
    check(load().moss_hip_rope_freqs(C.byref(p), _ptr(f), C.byref(m)))
    return f, m.value


class Rope:
    """A rotation a program keeps: its angles per position on the device (moss_hip_rope).

    Rope(rot_dim, ...) takes the arguments of rope_freqs; Rope(freqs=tensor) takes float64 angles of the
    caller's own, where they are, and no scaling.  halves: pairs (i, i + rot_dim / 2) rather than (2i, 2i + 1);
    mscale: the factor of sine and cosine, by default what the scaling asks for."""

    def __init__(self, rot_dim: int | None = None, halves: bool = False, freqs=None, mscale: float | None = None, device=None, **scaling):
        import torch
        if freqs is None:
            f, m = rope_freqs(64 if rot_dim is None else rot_dim, **scaling)
            freqs = torch.from_numpy(f).to("cuda" if device is None else device)
            mscale = m if mscale is None else mscale
        elif scaling or rot_dim not in (None, 2 * freqs.numel()):
            raise ValueError("freqs say the angles and their number: no scaling or other rot_dim besides")
        elif device is not None and torch.empty(0, device=device).device != freqs.device:
            raise ValueError(f"freqs are on {freqs.device}, not {device}")
        mscale = 1.0 if mscale is None else mscale
        self.freqs, self.device = freqs, freqs.get_device()
        _whole("freqs", freqs, torch.float64, (freqs.numel(),), self.device)
        self.struct = RopeStruct(freqs.data_ptr(), 2 * freqs.numel(), int(halves), mscale)
        self.ref = C.addressof(self.struct)


class KVCache:
    """One layer's paged cache as the calls take it (moss_hip_kv_cache): pools [n_pages][kv_heads][page_size][head_dim]
    (float32, float16, int8 or float8_e4m3fn; the 8-bit ones with float32 scales [n_pages][kv_heads][page_size])
    and the block table [streams][pages of a stream] (int32).  Keeps the tensors, owns nothing else."""

    def __init__(self, k, v, page_table, k_scale=None, v_scale=None):
        import torch
        kinds = {torch.float32: F32, torch.float16: F16, torch.int8: I8, torch.float8_e4m3fn: E4M3}
        if k.dim() != 4 or k.dtype not in kinds or page_table.dim() != 2:
            raise ValueError("pools [n_pages][kv_heads][page_size][head_dim] and a table [streams][pages] are wanted")
        self.tensors, self.device = (k, v, page_table, k_scale, v_scale), k.get_device()
        n, h, size, dim = k.shape
        self.kv_heads, self.head_dim, self.streams = h, dim, page_table.shape[0]
        self.struct = KVCacheStruct(
            _whole("k", k, k.dtype, (n, h, size, dim), self.device), _whole("v", v, k.dtype, (n, h, size, dim), self.device),
            _whole("k_scale", k_scale, torch.float32, (n, h, size), self.device, optional=True),
            _whole("v_scale", v_scale, torch.float32, (n, h, size), self.device, optional=True),
            kinds[k.dtype], h, dim, size, n,
            _whole("page_table", page_table, torch.int32, tuple(page_table.shape), self.device), page_table.shape[1],
            page_table.shape[0])
        self.ref = C.addressof(self.struct)


def rope_rows(x, pos, rope: Rope, out=None, stream=None):
    """moss_hip_rope_rows on x [rows][heads][head_dim] (any row and head strides) at positions pos [rows] int32, into
    out (x itself by default); returns out."""
    out = x if out is None else out
    dev, shape = x.get_device(), x.shape
    on = _on(dev, stream)
    if len(shape) != 3 or out.shape != shape or out.dtype is not x.dtype or out.get_device() != dev or rope.device != dev:
        raise ValueError("x and out must be [rows][heads][head_dim] of one type, on one device with the rotation")
    rows, heads, dim = shape
    if rows * heads * dim == 0:
        return out
    xs, os_ = x.stride(), out.stride()
    if xs[2] != 1 or os_[2] != 1:
        raise ValueError("the elements of a head must be contiguous")
    check(load().moss_hip_rope_rows(x.data_ptr(), xs[0], xs[1], out.data_ptr(), os_[0], os_[1], _types(x), rows, heads, dim,
                                    _whole("pos", pos, _torch.int32, (rows,), dev), rope.ref, on))
    return out


def kv_write(cache: KVCache, k, v, row_stream, row_pos, rope: Rope | None = None, rope_pos=None, stream=None) -> None:
    """moss_hip_kv_write: rows k, v [rows][kv_heads][head_dim] to position row_pos[r] of stream row_stream[r], keys turned
    by `rope` at rope_pos (row_pos by default)."""
    dev, n = cache.device, k.shape[0]
    on = _on(dev, stream)
    if v.shape[0] != n or v.dtype is not k.dtype or (rope is not None and rope.device != dev):
        raise ValueError("k and v must have the same rows and type, and the rotation their device")
    if n == 0:
        return
    kp, ks = _rows("k", k, cache.kv_heads, cache.head_dim, dev)
    vp, vs = _rows("v", v, cache.kv_heads, cache.head_dim, dev)
    check(load().moss_hip_kv_write(cache.ref, kp, ks, vp, vs, _types(k), n,
                                   _whole("row_stream", row_stream, _torch.int32, (n,), dev),
                                   _whole("row_pos", row_pos, _torch.int32, (n,), dev),
                                   None if rope is None else rope.ref,
                                   _whole("rope_pos", rope_pos, _torch.int32, (n,), dev, optional=True), on))


def kv_read(cache: KVCache, row_stream, row_pos, k, v, stream=None) -> None:
    """moss_hip_kv_read: those rows back, into k, v [rows][kv_heads][head_dim]."""
    dev, n = cache.device, k.shape[0]
    on = _on(dev, stream)
    if v.shape[0] != n or v.dtype is not k.dtype:
        raise ValueError("k and v must have the same rows and type")
    if n == 0:
        return
    kp, ks = _rows("k", k, cache.kv_heads, cache.head_dim, dev)
    vp, vs = _rows("v", v, cache.kv_heads, cache.head_dim, dev)
    check(load().moss_hip_kv_read(cache.ref, _whole("row_stream", row_stream, _torch.int32, (n,), dev),
                                  _whole("row_pos", row_pos, _torch.int32, (n,), dev), n, kp, ks, vp, vs, _types(k), on))


def attn_tree_workspace(cache: KVCache, heads: int, rows: int, max_rows: int, max_keys: int) -> int:
    """Bytes of workspace attn_tree takes for `rows` rows in all, max_rows of one stream, max_keys keys."""
    n = C.c_size_t(0)
    check(load().moss_hip_attn_tree_workspace(cache.ref, heads, rows, max_rows, max_keys, C.byref(n)))
    return n.value


def attn_tree(q, cache: KVCache, row_start, ctx_len, out, max_rows: int, max_keys: int, row_mask=None, scale: float | None = None,
              lse=None, workspace=None, stream=None) -> None:
    """moss_hip_attn_tree: q [rows][heads][head_dim] against the cache, into out (float32 or float16).

    row_start [streams + 1] and ctx_len [streams] int32; row_mask [rows] int64 (bit j: drafted row j of the
    stream), None: a chain; scale: head_dim ** -0.5 by default; lse [rows][heads] float32 or None."""
    dev, dim = cache.device, cache.head_dim
    on = _on(dev, stream)
    rows = q.shape[0]
    heads = q.shape[1] if q.dim() == 3 else q.shape[1] // dim
    if out.shape[0] != rows:
        raise ValueError("q and out must have the same rows")
    if rows == 0:
        return
    qp, qs = _rows("q", q, heads, dim, dev)
    op, os_ = _rows("out", out, heads, dim, dev)
    wp, wb = _workspace(workspace, lambda: attn_tree_workspace(cache, heads, rows, max_rows, max_keys), dev, stream)
    check(load().moss_hip_attn_tree(qp, qs, _types(q), heads, cache.ref,
                                    _whole("row_start", row_start, _torch.int32, (cache.streams + 1,), dev),
                                    _whole("ctx_len", ctx_len, _torch.int32, (cache.streams,), dev),
                                    _whole("row_mask", row_mask, _torch.int64, (rows,), dev, optional=True), rows, max_rows,
                                    max_keys, dim ** -0.5 if scale is None else scale, op, os_, _types(out),
                                    _whole("lse", lse, _torch.float32, (rows, heads), dev, optional=True), wp, wb, on))


def token_logprobs_workspace(rows: int, vocab: int, top_k: int) -> int:
    """Bytes of workspace token_logprobs takes."""
    n = C.c_size_t(0)
    check(load().moss_hip_token_logprobs_workspace(rows, vocab, top_k, C.byref(n)))
    return n.value


def token_logprobs(logits, tokens, logprob, entropy=None, top_ids=None, top_logprobs=None, inv_temperature: float = 1.0,
                   workspace=None, stream=None) -> None:
    """moss_hip_token_logprobs: of tokens [rows] int32 under logits [rows][vocab] (float32 or float16, any row stride), into
    logprob and entropy [rows] and the alternatives top_ids (int32), top_logprobs [rows][top_k]."""
    dev, shape = logits.get_device(), logits.shape
    on = _on(dev, stream)
    if len(shape) != 2:
        raise ValueError("logits [rows][vocab] are wanted")
    rows, vocab = shape
    k = 0 if top_ids is None else top_ids.shape[1]
    if (top_ids is None) != (top_logprobs is None):
        raise ValueError("top_ids and top_logprobs come together")
    if rows == 0:
        return
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("the logits of a row must be contiguous")
    wp, wb = _workspace(workspace, lambda: token_logprobs_workspace(rows, vocab, k), dev, stream)
    check(load().moss_hip_token_logprobs(logits.data_ptr(), logits.stride(0), _types(logits), rows, vocab,
                                         _whole("tokens", tokens, _torch.int32, (rows,), dev), inv_temperature,
                                         _whole("logprob", logprob, _torch.float32, (rows,), dev),
                                         _whole("entropy", entropy, _torch.float32, (rows,), dev, optional=True), k,
                                         _whole("top_ids", top_ids, _torch.int32, (rows, k), dev, optional=True),
                                         _whole("top_logprobs", top_logprobs, _torch.float32, (rows, k), dev, optional=True),
                                         wp, wb, on))


# ---------------------------------------------------------------- model

class HipLLM:
    """Python view of the GPU LlmModel (moss_hip_llm_*)."""

    def __init__(self, blob: bytes, device: int = 0, max_ctx: int = 0, kv_fp32: bool = False, graphs: bool = True,
                 prefill_a16: bool = False, per_op: bool = False, decode_a8: bool = False):
        L = self.L = load()
        self._h = C.c_void_p()
        buf = np.frombuffer(blob, dtype=np.uint8)
        opt = Options(device, max_ctx, 1 if kv_fp32 else 0, 1 if graphs else 0, 1 if prefill_a16 else 0,
                      1 if per_op else 0, 1 if decode_a8 else 0)
        check(L.moss_hip_llm_create(_ptr(buf), buf.size, C.byref(opt), C.byref(self._h)))

    def close(self):
        if getattr(self, "_h", None) and self._h.value:
            self.L.moss_hip_llm_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        self.close()

    @property
    def position(self) -> int:
        return self.L.moss_hip_llm_position(self._h)

    @property
    def prefix_pos(self) -> int:
        return self.L.moss_hip_llm_prefix_pos(self._h)

    @property
    def fallbacks(self) -> int:
        """Fused decode launches redone on the per-operator path (moss_hip_llm_fallbacks)."""
        return self.L.moss_hip_llm_fallbacks(self._h)

    def reset(self):
        check(self.L.moss_hip_llm_reset(self._h))

    def hidden(self) -> np.ndarray:
        out = np.empty(768, np.float32)
        check(self.L.moss_hip_llm_get_hidden(self._h, _ptr(out)))
        return out

    def set_hidden(self, h):
        h = np.ascontiguousarray(h, np.float32)
        check(self.L.moss_hip_llm_set_hidden(self._h, _ptr(h)))

    def prefill(self, rows, start: int = 0):
        rows = np.ascontiguousarray(rows, np.int32).reshape(-1, 17)
        check(self.L.moss_hip_llm_prefill(self._h, _ptr(rows), rows.shape[0], start))

    def global_step(self, row):
        row = np.ascontiguousarray(row, np.int32).reshape(17)
        check(self.L.moss_hip_llm_global_step(self._h, _ptr(row)))

    def generate(self, max_frames: int, params: SampleParams | None = None, seed: int = 0, forced=None,
                 timing: bool = False, logits: bool = False, gate: bool = False, on_frame=None):
        params = params or SampleParams.make()
        out = np.zeros((max(max_frames, 1), 17), np.int32)
        fa = np.ascontiguousarray(forced, np.int32).reshape(-1, 17) if forced is not None else None
        t = np.zeros((max(max_frames, 1), 2), np.float64) if timing else None
        ld = np.zeros((max(max_frames, 1), 16, 1024), np.float32) if logits else None
        gd = np.zeros((max(max_frames, 1), 4), np.float32) if gate else None
        n = C.c_int(0)
        cb = FRAME_CB(lambda u, f, row: on_frame(f, np.ctypeslib.as_array(row, (17,)).copy())) if on_frame \
            else FRAME_CB()
        check(self.L.moss_hip_llm_generate(self._h, max_frames, C.byref(params), seed,
                                           _ptr(fa) if fa is not None else None, 0 if fa is None else fa.shape[0],
                                           _ptr(out), C.byref(n), _ptr(t) if t is not None else None,
                                           _ptr(ld) if ld is not None else None, _ptr(gd) if gd is not None else None,
                                           cb, None))
        res = {"rows": out[:n.value]}
        if timing:
            res["timing"] = t[:n.value]
        if logits:
            res["logits"] = ld[:n.value]
        if gate:
            res["gate"] = gd[:self.L.moss_hip_llm_gate_rows(self._h)]
        return res

    def set_cancel_flag(self, flag_array: np.ndarray | None):
        """flag_array: a 1-element uint8 numpy array kept alive by the caller (or None)."""
        self._cancel = flag_array
        check(self.L.moss_hip_llm_set_cancel_flag(self._h, _ptr(flag_array) if flag_array is not None else None))

    def snapshot_prefix(self):
        check(self.L.moss_hip_llm_snapshot_prefix(self._h))

    def restore_prefix(self):
        check(self.L.moss_hip_llm_restore_prefix(self._h))

    def capture(self, on: bool = True):
        """Quantiser capture (tests): W8A8 quantisers record their inputs and outputs."""
        check(self.L.moss_hip_llm_capture(self._h, 1 if on else 0))

    def capture_read(self, what: int) -> np.ndarray:
        """Raw bytes of the last capture of `what` (CAP_GLOBAL / CAP_LOCAL / CAP_PREFILL)."""
        n = C.c_size_t(0)
        check(self.L.moss_hip_llm_capture_read(self._h, what, None, 0, C.byref(n)))
        out = np.empty(n.value, np.uint8)
        check(self.L.moss_hip_llm_capture_read(self._h, what, _ptr(out), out.size, None))
        return out

    def capture_steps(self, what: int) -> list:
        """A decode capture as one dict per step (block or local position) of named float arrays."""
        raw = self.capture_read(what).view(np.float32).reshape(-1, CAP_STEP)
        return [{k: step[o:o + n].copy() for k, (o, n) in CAP.items()} for step in raw]

    def kv_export(self, n_pos: int):
        k = np.empty((12, n_pos, 768), np.float32)
        v = np.empty((12, n_pos, 768), np.float32)
        check(self.L.moss_hip_llm_kv_export(self._h, n_pos, _ptr(k), _ptr(v)))
        return k, v

    def kv_import(self, k, v, hidden=None):
        k = np.ascontiguousarray(k, np.float32)
        v = np.ascontiguousarray(v, np.float32)
        h = np.ascontiguousarray(hidden, np.float32) if hidden is not None else None
        check(self.L.moss_hip_llm_kv_import(self._h, k.shape[1], _ptr(k), _ptr(v), _ptr(h) if h is not None else None))


class HipBatch:
    """Python view of a moss_hip_batch (many streams decoded in lock-step)."""

    def __init__(self, model: HipLLM, max_streams: int, capacity: int, kv_fp32: bool = False):
        self.L = load()
        self.model = model  # keeps the weights alive
        self._h = C.c_void_p()
        check(self.L.moss_hip_batch_create(model._h, max_streams, capacity, 1 if kv_fp32 else 0, C.byref(self._h)))

    def close(self):
        if getattr(self, "_h", None) and self._h.value:
            self.L.moss_hip_batch_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        self.close()

    def set_stream(self, s: int, k, v, hidden):
        k = np.ascontiguousarray(k, np.float32)
        v = np.ascontiguousarray(v, np.float32)
        h = np.ascontiguousarray(hidden, np.float32)
        check(self.L.moss_hip_batch_set_stream(self._h, s, k.shape[1], _ptr(k), _ptr(v), _ptr(h)))

    def capture(self, on: bool = True):
        """Attention capture of a W8A8 batch (tests)."""
        check(self.L.moss_hip_batch_capture(self._h, 1 if on else 0))

    def capture_attention(self, max_streams: int) -> list:
        """The last frame's attention records: 29 dicts (12 global layers, local positions 0..16)
        of out [max_streams][768] fp32 and the raw int8 / scale operand (matrix-core order)."""
        n = C.c_size_t(0)
        check(self.L.moss_hip_batch_capture_read(self._h, None, 0, C.byref(n)))
        raw = np.empty(n.value, np.uint8)
        check(self.L.moss_hip_batch_capture_read(self._h, _ptr(raw), raw.size, None))
        s16 = (max_streams + 15) // 16 * 16
        per = 4 * max_streams * 768 + s16 * 768 + 4 * s16 * 24
        assert raw.size == 29 * per
        out = []
        for e in range(29):
            b = e * per
            out.append({"out": raw[b:b + 4 * max_streams * 768].view(np.float32).reshape(max_streams, 768),
                        "q": raw[b + 4 * max_streams * 768: b + 4 * max_streams * 768 + s16 * 768],
                        "d": raw[b + 4 * max_streams * 768 + s16 * 768: b + per]})
        return out

    def admit(self, s: int, model: HipLLM):
        """Stream s takes `model`'s state (K/V, hidden, position) device to device."""
        check(self.L.moss_hip_batch_admit(self._h, s, model._h))

    def position(self, s: int) -> int:
        return self.L.moss_hip_batch_position(self._h, s)

    def hidden(self, s: int) -> np.ndarray:
        out = np.empty(768, np.float32)
        check(self.L.moss_hip_batch_get_hidden(self._h, s, _ptr(out)))
        return out

    def kv_export(self, s: int, n_pos: int):
        k = np.empty((12, n_pos, 768), np.float32)
        v = np.empty((12, n_pos, 768), np.float32)
        check(self.L.moss_hip_batch_kv_export(self._h, s, n_pos, _ptr(k), _ptr(v)))
        return k, v

    def global_step(self, rows):
        rows = np.ascontiguousarray(rows, np.int32).reshape(-1, 17)
        check(self.L.moss_hip_batch_global_step(self._h, rows.shape[0], _ptr(rows)))

    def generate(self, n_streams: int, frames: int, params: SampleParams | None = None, seeds=None):
        params = params or SampleParams.make()
        out = np.zeros((max(frames, 1), n_streams, 17), np.int32)
        nf = np.zeros(n_streams, np.int32)
        ms = C.c_double(0.0)
        sd = None if seeds is None else np.ascontiguousarray(seeds, np.uint64).reshape(n_streams)
        check(self.L.moss_hip_batch_generate(self._h, n_streams, frames, C.byref(params),
                                             None if sd is None else _ptr(sd), _ptr(out), _ptr(nf), C.byref(ms)))
        return {"rows": out[:frames], "frames": nf, "ms": ms.value}


class HipCodec:
    """The GPU audio codec decoder (moss::AudioDecoder, csrc/include/moss/decoder.h:14-83).

    codes: int array [16][frames] (quantizer-major) in [0, 1024); results are float32 arrays
    of frames * samples_per_frame interleaved stereo samples."""

    def __init__(self, blob: bytes, max_chunk_frames: int = 0, contexts=(0, 0, 0, 0), eager: bool = False,
                 device: int = 0):
        L = load()
        o = CodecOptions(device, max_chunk_frames, (C.c_int * 4)(*contexts), int(eager))
        h = C.c_void_p()
        self._blob = np.frombuffer(blob, dtype=np.uint8)
        check(L.moss_hip_codec_create(_ptr(self._blob), len(blob), C.byref(o), C.byref(h)))
        self._h = h
        self.samples_per_frame = L.moss_hip_codec_samples_per_frame(h)

    def close(self):
        if getattr(self, "_h", None):
            load().moss_hip_codec_destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()

    def _run(self, fn, codes):
        c = np.ascontiguousarray(codes, dtype=np.int32)
        if c.ndim != 2 or c.shape[0] != 16:
            raise ValueError("codes must be [16][frames]")
        out = np.empty(c.shape[1] * self.samples_per_frame, np.float32)
        check(fn(self._h, _ptr(c), c.shape[1], _ptr(out)))
        return out

    def reset_stream(self) -> None:
        check(load().moss_hip_codec_reset_stream(self._h))

    def decode_chunk(self, codes) -> np.ndarray:
        return self._run(load().moss_hip_codec_decode_chunk, codes)

    def decode(self, codes) -> np.ndarray:
        return self._run(load().moss_hip_codec_decode, codes)

    @property
    def last_ms(self) -> float:
        return load().moss_hip_codec_last_ms(self._h)

    @property
    def stage_ms(self):
        out = (C.c_double * 4)()
        check(load().moss_hip_codec_stage_ms(self._h, out))
        return list(out)
