"""ctypes binding of libqa_b200.so (the C ABI in include/qa_b200.h and
include/qa_b200_kernels.h).

The library is built in-tree by ``make`` in this directory (see
``__graft_entry__.build``).  There is no fallback: if the shared object is
missing, :func:`lib` raises, so a product path can never silently run on the
CPU.
"""
from __future__ import annotations

import ctypes
import os
import struct
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libqa_b200.so")

QA_OK = 0
QA_ERR_SHAPE = 1
QA_ERR_CAP = 2
QA_ERR_CUDA = 3
QA_ERR_OOM = 4
QA_ERR_TIMEOUT = 5
QA_ERR_STATE = 6
QA_ERR_WEIGHTS = 7
QA_ERR_ARG = 8

ERR_NAMES = {
    QA_ERR_SHAPE: "QA_ERR_SHAPE",
    QA_ERR_CAP: "QA_ERR_CAP",
    QA_ERR_CUDA: "QA_ERR_CUDA",
    QA_ERR_OOM: "QA_ERR_OOM",
    QA_ERR_TIMEOUT: "QA_ERR_TIMEOUT",
    QA_ERR_STATE: "QA_ERR_STATE",
    QA_ERR_WEIGHTS: "QA_ERR_WEIGHTS",
    QA_ERR_ARG: "QA_ERR_ARG",
}

QA_HALF_F16 = 0
QA_HALF_BF16 = 1
QA_DTYPE_F32 = 0
QA_DTYPE_F16 = 1
QA_DTYPE_BF16 = 2

EPI_STORE16 = 0
EPI_RESID16 = 1
EPI_RESID32 = 2
EPI_SWIGLU16 = 3
EPI_STORE32 = 4
EPI_ARGMAX = 5
ACT_NONE = 0
ACT_GELU = 1

# Every symbol the two public headers declare; tests check each is exported.
EXPORTED = [
    "qa_open", "qa_load", "qa_close", "qa_last_error", "qa_set_timeout_ms", "qa_half",
    "qa_get_timings", "qa_mel", "qa_audio_embeds", "qa_ensure_capacity", "qa_text_hidden",
    "qa_head", "qa_align_batch", "qa_batch_stage", "qa_batch_run", "qa_batch_fetch",
    "qa_set_stream", "qa_set_profile", "qa_get_profile", "qa_fix_timestamps",
    "qa_decode_wav", "qa_resampled_length", "qa_resample",
    "qa_head_noalloc", "qa_probe_timeout", "qa_local_head_load", "qa_set_local_head_enabled",
    "qa_local_head_enabled", "qa_local_head_refine",
    "qa_k_gemm", "qa_k_conv3x3s2", "qa_k_causal_attention", "qa_k_window_attention",
    "qa_k_conv1", "qa_k_gemm_qkv_rope", "qa_k_kv_append", "qa_k_cache_attention",
    "qa_k_cache_attention_workspace", "qa_k_w4_linear", "qa_k_kv_append_v",
    "qa_k_cache_attention_v", "qa_k_w4_linear_v",
]

c_void_p = ctypes.c_void_p
c_int = ctypes.c_int
c_ll = ctypes.c_longlong


class QaTensor(ctypes.Structure):
    """qa_tensor (include/qa_b200.h)."""
    _fields_ = [("name", ctypes.c_char_p), ("dtype", c_int), ("ndim", c_int),
                ("shape", ctypes.c_int64 * 4), ("data", c_void_p)]


class QaCfg(ctypes.Structure):
    """qa_cfg (include/qa_b200.h)."""
    _fields_ = [(n, c_int) for n in (
        "d_model", "encoder_layers", "encoder_heads", "encoder_ffn_dim", "num_mel_bins",
        "downsample_hidden", "max_source_positions", "n_window", "n_window_infer", "output_dim",
        "vocab_size", "hidden_size", "intermediate_size", "num_layers", "num_heads",
        "num_kv_heads", "head_dim")] + [("rms_norm_eps", ctypes.c_double),
                                       ("rope_theta", ctypes.c_double)] + [
        (n, c_int) for n in ("num_labels", "timestamp_token_id", "audio_token_id")] + [
        ("timestamp_segment_time_ms", ctypes.c_double), ("max_seq", c_int)]


class QaTimings(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in (
        "h2d_ms", "mel_ms", "enc_ms", "gather_ms", "prefill_ms", "head_ms", "d2h_ms",
        "total_ms")] + [("gpu_launches", ctypes.c_int64), ("h2d_bytes", ctypes.c_int64),
                        ("d2h_bytes", ctypes.c_int64), ("local_ms", ctypes.c_double)]


class QaKernelStat(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 32), ("launches", ctypes.c_int64),
                ("total_ms", ctypes.c_double), ("flops", ctypes.c_double),
                ("bytes", ctypes.c_double)]


class QaClip(ctypes.Structure):
    _fields_ = [("samples", c_void_p), ("n_samples", ctypes.c_int64), ("input_ids", c_void_p),
                ("seq_len", c_int)]


class QaResult(ctypes.Structure):
    _fields_ = [("raw_ms", c_void_p), ("n_ts", c_int), ("logits", c_void_p),
                ("normed", c_void_p), ("intervals", c_void_p)]


def make_cfg(mc) -> QaCfg:
    """QaCfg from a synth.ModelConfig-like object."""
    c = QaCfg()
    for name, _ in QaCfg._fields_:
        setattr(c, name, getattr(mc, name))
    return c


def make_tensors(weights: dict):
    """(QaTensor array, keepalive) from name -> (dtype, np array) or bf16 bits."""
    import numpy as np
    items = []
    for name, v in weights.items():
        if isinstance(v, tuple):
            dt, arr = v
        else:
            dt, arr = "BF16", v
        code = {"BF16": QA_DTYPE_BF16, "F16": QA_DTYPE_F16, "F32": QA_DTYPE_F32}[dt]
        arr = np.ascontiguousarray(arr)
        items.append((name.encode(), code, arr))
    arr_t = (QaTensor * len(items))()
    for i, (nm, code, a) in enumerate(items):
        arr_t[i].name = nm
        arr_t[i].dtype = code
        arr_t[i].ndim = a.ndim
        for d in range(a.ndim):
            arr_t[i].shape[d] = a.shape[d]
        arr_t[i].data = a.ctypes.data
    return arr_t, items


class QaError(RuntimeError):
    """A non-zero status from the C ABI."""

    def __init__(self, code: int, msg: str = ""):
        self.code = code
        super().__init__(f"{ERR_NAMES.get(code, code)}: {msg}")


_lock = threading.Lock()
_lib = None


def lib_exists() -> bool:
    return os.path.exists(LIB_PATH)


def lib() -> ctypes.CDLL:
    """Load (once) and return the shared library; raise if it was not built."""
    global _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"{LIB_PATH} is missing: build it with `make` in {_HERE} "
                    "(or __graft_entry__.build()); there is no CPU fallback")
            L = ctypes.CDLL(LIB_PATH)
            _declare(L)
            _lib = L
        return _lib


def _declare(L: ctypes.CDLL) -> None:
    L.qa_k_gemm.argtypes = [c_void_p, c_ll, c_void_p, c_ll, c_int, c_int, c_int, c_int, c_int,
                            c_int, c_void_p, c_ll, c_void_p, c_void_p, c_void_p, c_int, c_void_p,
                            c_void_p, c_int, c_void_p]
    L.qa_k_gemm.restype = c_int
    L.qa_k_conv3x3s2.argtypes = [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int,
                                 c_int, c_int, c_int, c_void_p, c_ll, c_void_p, c_void_p, c_void_p]
    L.qa_k_gemm_qkv_rope.argtypes = [c_void_p, c_ll, c_void_p, c_ll, c_int, c_int, c_int, c_int,
                                     c_void_p, c_ll, c_void_p, c_void_p, c_void_p, c_int,
                                     c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                     ctypes.c_float, c_int, c_int, c_void_p, c_int, c_void_p]
    L.qa_k_conv1.argtypes = [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p,
                             c_int, c_void_p]
    L.qa_k_causal_attention.argtypes = [c_void_p, c_ll, c_ll, c_int, c_int, c_void_p, c_int,
                                        c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p,
                                        c_int, c_void_p, c_void_p]
    L.qa_k_window_attention.argtypes = [c_void_p, c_ll, c_int, c_int, c_void_p, c_int, c_int,
                                        c_void_p, c_int, c_void_p, c_void_p]
    L.qa_k_kv_append.argtypes = [c_void_p, c_ll, c_void_p, c_ll, c_void_p, c_ll, c_void_p, c_ll,
                                 c_ll, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_int,
                                 c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                 c_void_p, c_void_p, c_int, c_void_p, c_ll, c_int, c_void_p,
                                 c_void_p, c_void_p, ctypes.c_float, c_int, c_void_p, c_void_p]
    L.qa_k_cache_attention.argtypes = [c_void_p, c_ll, c_ll, c_int, c_int, c_int, c_void_p,
                                       c_void_p, c_int, c_int, c_int, c_void_p, c_int, c_void_p,
                                       c_void_p, c_int, c_void_p, c_void_p, ctypes.c_float, c_int,
                                       c_void_p, c_ll, c_void_p, c_void_p, c_ll, c_int, c_void_p,
                                       c_void_p]
    L.qa_k_cache_attention_workspace.argtypes = [c_int] * 6
    L.qa_k_cache_attention_workspace.restype = ctypes.c_int64
    L.qa_k_w4_linear.argtypes = [c_void_p, c_ll, c_int, c_int, c_void_p, c_ll, c_int, c_int,
                                 c_void_p, c_void_p, c_void_p, c_void_p, c_ll, c_int, c_void_p]
    L.qa_k_kv_append_v.argtypes = [ctypes.c_char_p, ctypes.c_float]
    L.qa_k_cache_attention_v.argtypes = [ctypes.c_char_p, ctypes.c_float]
    L.qa_k_w4_linear_v.argtypes = [ctypes.c_char_p]
    if hasattr(L, "qa_open"):
        L.qa_open.argtypes = [c_int, c_int, ctypes.POINTER(c_void_p)]
        L.qa_load.argtypes = [c_void_p, c_void_p, c_int, c_void_p]
        L.qa_close.argtypes = [c_void_p]
        L.qa_last_error.argtypes = [c_void_p]
        L.qa_last_error.restype = ctypes.c_char_p
        L.qa_set_timeout_ms.argtypes = [c_void_p, c_int]
        L.qa_half.argtypes = [c_void_p]
        L.qa_get_timings.argtypes = [c_void_p, c_void_p]
        L.qa_mel.argtypes = [c_void_p, c_void_p, ctypes.c_int64, c_void_p, ctypes.c_int64,
                             ctypes.POINTER(c_int)]
        L.qa_audio_embeds.argtypes = [c_void_p, c_void_p, c_int, c_int, c_void_p, ctypes.c_int64]
        L.qa_ensure_capacity.argtypes = [c_void_p, c_int, ctypes.POINTER(c_int)]
        L.qa_text_hidden.argtypes = [c_void_p, c_void_p, c_int, c_void_p]
        L.qa_head.argtypes = [c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p,
                              c_void_p]
        L.qa_align_batch.argtypes = [c_void_p, c_void_p, c_int, c_void_p]
        L.qa_batch_stage.argtypes = [c_void_p, c_void_p, c_int, c_void_p]
        L.qa_fix_timestamps.argtypes = [c_void_p, c_int, c_void_p]
        L.qa_decode_wav.argtypes = [c_void_p, ctypes.c_int64, c_void_p, ctypes.c_int64,
                                    ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(c_int),
                                    ctypes.POINTER(c_int)]
        L.qa_resampled_length.argtypes = [ctypes.c_int64, c_int, c_int]
        L.qa_resampled_length.restype = ctypes.c_int64
        L.qa_resample.argtypes = [c_void_p, ctypes.c_int64, c_int, c_int, c_void_p,
                                  ctypes.c_int64]
        L.qa_head_noalloc.argtypes = [c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p,
                                      c_void_p]
        L.qa_probe_timeout.argtypes = [c_void_p, c_int]
        L.qa_batch_run.argtypes = [c_void_p]
        L.qa_batch_fetch.argtypes = [c_void_p, c_void_p]
        L.qa_set_stream.argtypes = [c_void_p, c_void_p]
        L.qa_set_profile.argtypes = [c_void_p, c_int]
        L.qa_get_profile.argtypes = [c_void_p, c_void_p, c_int, ctypes.POINTER(c_int)]
        L.qa_local_head_load.argtypes = [c_void_p, c_void_p, c_int, c_void_p, c_void_p]
        L.qa_set_local_head_enabled.argtypes = [c_void_p, c_int]
        L.qa_local_head_enabled.argtypes = [c_void_p]
        L.qa_local_head_refine.argtypes = [c_void_p, c_void_p, ctypes.c_int64, c_int, c_void_p,
                                           c_int, c_void_p, c_int, c_void_p, c_void_p, c_void_p,
                                           c_void_p]


def check(rc: int, ctx=None) -> None:
    if rc != QA_OK:
        msg = ""
        if ctx is not None:
            m = lib().qa_last_error(ctx)
            msg = m.decode() if m else ""
        raise QaError(rc, msg)


def fix_timestamps(raw) -> list:
    """qa_fix_timestamps over an int64 sequence (the compiled LIS repair)."""
    import numpy as np
    a = np.ascontiguousarray(raw, np.int64)
    out = np.empty_like(a)
    if len(a):
        check(lib().qa_fix_timestamps(a.ctypes.data, len(a), out.ctypes.data))
    return out.tolist()


def ptr(t) -> int:
    """Device/host address of a torch tensor (0 for None)."""
    return 0 if t is None else int(t.data_ptr())


def gemm(A, B, out, mode=EPI_STORE16, act=ACT_NONE, bias=None, row_map=None, pe=None,
         pe_period=1, keys=None, status=None, force_bn=0, stream=None):
    """Run the tcgen05 GEMM on torch CUDA tensors: A [M, K], B [N, K]."""
    import torch
    M, K = A.shape
    N = B.shape[0]
    assert B.shape[1] == K and A.dtype == B.dtype
    bf16 = 1 if A.dtype == torch.bfloat16 else 0
    s = stream if stream is not None else torch.cuda.current_stream().cuda_stream
    rc = lib().qa_k_gemm(ptr(A), A.stride(0), ptr(B), B.stride(0), M, N, K, bf16, mode, act,
                         ptr(out), out.stride(0) if out is not None else 0, ptr(bias),
                         ptr(row_map), ptr(pe), pe_period, ptr(keys), ptr(status), force_bn, s)
    check(rc)


def conv3x3s2(x, wt, out, time_major=False, mode=EPI_STORE16, act=ACT_NONE, bias=None,
              status=None, stream=None):
    """Implicit-GEMM conv on torch CUDA tensors: x [n, h, w, c] NHWC, wt [c_out, 9c]."""
    import torch
    n, h, w, c = x.shape
    bf16 = 1 if x.dtype == torch.bfloat16 else 0
    s = stream if stream is not None else torch.cuda.current_stream().cuda_stream
    rc = lib().qa_k_conv3x3s2(ptr(x), n, h, w, c, ptr(wt), wt.shape[0], 1 if time_major else 0,
                              bf16, mode, act, ptr(out), out.stride(0), ptr(bias), ptr(status), s)
    check(rc)


def causal_attention(qkv, nqh, nkvh, tiles, block_tab, kpool, vpool, out, status=None,
                     stream=None, validate=True):
    """Paged causal attention on torch CUDA tensors.

    qkv [T, ldq] 16-bit, tiles int32 [n, 4] (clip, q0, tok0, len), block_tab
    int32 [clips, max_pages], kpool/vpool [pages, nkvh, 64, 128], out [T, nqh*128].
    """
    import torch
    if validate:  # copies tiles and block_tab to the host
        check_attention_args(qkv, nqh, nkvh, tiles, block_tab, kpool, vpool, out)
    bf16 = 1 if qkv.dtype == torch.bfloat16 else 0
    s = stream if stream is not None else torch.cuda.current_stream().cuda_stream
    rc = lib().qa_k_causal_attention(ptr(qkv), qkv.stride(0), qkv.shape[0], nqh, nkvh,
                                     ptr(tiles), tiles.shape[0], ptr(block_tab),
                                     block_tab.shape[1], ptr(kpool), ptr(vpool), kpool.shape[0],
                                     ptr(out), bf16, ptr(status), s)
    check(rc)


def window_attention(qkv, nh, windows, out, status=None, stream=None, max_window=None):
    """Windowed attention on torch CUDA tensors: qkv [T, 3*64*nh] 16-bit,
    windows int32 [n, 2] (first token, length), out [T, 64*nh].  The windows
    are range-checked on the host (a copy to the host) unless `max_window`
    (the longest window) is given, which a caller that checked them passes."""
    import torch
    T = qkv.shape[0]
    dm = 64 * nh
    if (qkv.dim() != 2 or qkv.shape[1] != 3 * dm or tuple(out.shape) != (T, dm)
            or qkv.dtype != out.dtype or windows.dtype != torch.int32 or windows.dim() != 2
            or windows.shape[1] != 2):
        raise ValueError("qkv [T, 3*64*nh], out [T, 64*nh] of one dtype, windows int32 [n, 2]")
    if max_window is None:
        w = windows.cpu()
        if w.numel() and (int(w[:, 0].min()) < 0 or int(w[:, 1].min()) < 1
                          or int((w[:, 0] + w[:, 1]).max()) > T or int(w[:, 1].max()) > 128):
            raise ValueError("window (start, len) out of range")
        max_window = int(w[:, 1].max()) if w.numel() else 1
    bf16 = 1 if qkv.dtype == torch.bfloat16 else 0
    s = stream if stream is not None else torch.cuda.current_stream().cuda_stream
    check(lib().qa_k_window_attention(ptr(qkv), T, dm, nh, ptr(windows), windows.shape[0],
                                      max_window, ptr(out), bf16, ptr(status), s))


def check_attention_args(qkv, nqh, nkvh, tiles, block_tab, kpool, vpool, out) -> None:
    """Host-side shape and range checks for causal_attention (ValueError on failure)."""
    import torch
    T = qkv.shape[0]
    if (tiles.dim() != 2 or tiles.shape[1] != 4 or tiles.dtype != torch.int32
            or block_tab.dim() != 2 or block_tab.dtype != torch.int32):
        raise ValueError("tiles must be int32 [n, 4] and block_tab int32 [clips, max_pages]")
    if tuple(kpool.shape[1:]) != (nkvh, 64, 128) or kpool.shape != vpool.shape:
        raise ValueError("kpool/vpool must be [pages, nkvh, 64, 128]")
    if qkv.dim() != 2 or qkv.shape[1] < (nqh + 2 * nkvh) * 128 or tuple(out.shape) != (
            T, nqh * 128) or not (qkv.dtype == kpool.dtype == vpool.dtype == out.dtype):
        raise ValueError("qkv [T, >= (nqh + 2 nkvh) 128], out [T, nqh 128], one 16-bit dtype")
    t = tiles.cpu()
    bt = block_tab.cpu()
    if t.numel() and (int(t[:, 0].min()) < 0 or int(t[:, 0].max()) >= bt.shape[0]
                      or int(t[:, 1].min()) < 0 or int((t[:, 1] - t[:, 3]).max()) >= 0
                      or int((t[:, 2] + t[:, 3]).max()) > T
                      or int(t[:, 3].max()) > 64 * bt.shape[1]):
        raise ValueError("tile (clip, q0, tok0, len) out of range")
    if bt.numel() and (int(bt.min()) < 0 or int(bt.max()) >= kpool.shape[0]):
        raise ValueError("block_tab names a page outside the pools")


def conv1(mel, wt, bias, out, stream=None):
    """conv1 + bias + GELU on torch CUDA tensors: mel [n, h, w] f32 -> out [n*ho*wo, c_out]."""
    import torch
    n, h, w = mel.shape
    bf16 = 1 if out.dtype == torch.bfloat16 else 0
    s = stream if stream is not None else torch.cuda.current_stream().cuda_stream
    check(lib().qa_k_conv1(ptr(mel), n, h, w, ptr(wt), ptr(bias), wt.shape[0], ptr(out), bf16, s))


def gemm_qkv_rope(A, B, q_out, pos_of, clip_of, block_tab, kc, vc, cos_t, sin_t, qn, kn, eps,
                  nq, nkv, status=None, force_bn=0, stream=None):
    """The fused decoder QKV GEMM on torch CUDA tensors (see qa_k_gemm_qkv_rope)."""
    import torch
    M, K = A.shape
    N = B.shape[0]
    bf16 = 1 if A.dtype == torch.bfloat16 else 0
    s = stream if stream is not None else torch.cuda.current_stream().cuda_stream
    check(lib().qa_k_gemm_qkv_rope(ptr(A), A.stride(0), ptr(B), B.stride(0), M, N, K, bf16,
                                   ptr(q_out), q_out.stride(0), ptr(pos_of), ptr(clip_of),
                                   ptr(block_tab), block_tab.shape[1], ptr(kc), ptr(vc),
                                   ptr(cos_t), ptr(sin_t), ptr(qn), ptr(kn), eps, nq, nkv,
                                   ptr(status), force_bn, s))


# ---------------------------------------------------------------- growing sessions
# A decoding step calls these once a layer, so their checks read each attribute of a
# tensor once and build a message only when something is wrong, and the arguments go
# to the library as one array (qa_k_*_v).
_pack35, _pack27, _pack15 = (struct.Struct(f"{n}q").pack for n in (35, 27, 15))

_F16 = _BF16 = _F32 = _I32 = _U8 = _E4M3 = _cuda = None


def _types():
    global _F16, _BF16, _F32, _I32, _U8, _E4M3, _cuda
    import torch
    _cuda = torch.cuda
    _F16, _BF16, _F32, _I32, _U8, _E4M3 = (torch.float16, torch.bfloat16, torch.float32, torch.int32,
                                           torch.uint8, torch.float8_e4m3fn)
    return _F16


def _rows(t, T, width, dt, name) -> int:
    """Row stride of t, which is [T, width] of 16-bit `dt` with adjacent columns."""
    if t.shape == (T, width) and t.dtype is dt:
        ld, one = t.stride()
        if T < 2:
            ld = width
        if (one == 1 or width == 1) and ld >= width:
            return ld
    raise ValueError(f"{name}: [{T}, {width}] of {dt} with adjacent columns")


def _flat(t, shape, dt, what) -> None:
    """t is a contiguous tensor of that shape and type."""
    if t.dtype is not dt or t.shape != shape or not t.is_contiguous():
        raise ValueError(what)


def _seq_args(q_start, kv_len, block_tab, kpool, vpool, max_q) -> tuple:
    """Shapes of the sequence maps and pools; (n_seqs, max_pages, pages, nkv, hd)."""
    if (kv_len.dim() != 1 or block_tab.dim() != 2 or kpool.dim() != 4):
        raise ValueError("kv_len [n], block_tab [n, max_pages], pools [pages, heads, 64, hd]")
    n = kv_len.shape[0]
    bt = block_tab.shape
    what = "q_start int32 [n + 1], kv_len int32 [n], block_tab int32 [n, max_pages], contiguous"
    _flat(q_start, (n + 1,), _I32, what)
    _flat(kv_len, (n,), _I32, what)
    _flat(block_tab, (n, bt[1]), _I32, what)
    ps = kpool.shape
    pages, nkv, page, hd = ps
    if (page != 64 or (hd != 64 and hd != 128) or pages == 0 or nkv == 0 or bt[1] == 0
            or vpool.shape != ps or vpool.dtype is not kpool.dtype
            or not kpool.is_contiguous() or not vpool.is_contiguous()):
        raise ValueError("kpool / vpool [pages, heads, 64, 64 or 128], contiguous, of one type, and max_pages > 0")
    if max_q < 0:
        raise ValueError("max_q >= 0")
    return n, bt[1], pages, nkv, hd


def check_sequences(T, q_start, kv_len, block_tab, pages, max_q, appending) -> None:
    """Host-side range checks of the sequence maps (copies them to the host;
    ValueError on failure): what the kernels would otherwise report in *status."""
    import torch

    def need(ok, what):
        if not ok:
            raise ValueError(what)

    qs, kl, bt = q_start.cpu().long(), kv_len.cpu().long(), block_tab.cpu().long()
    n = qs.diff()
    if n.numel() == 0:
        return
    need(int(qs[0]) >= 0 and int(n.min()) >= 0 and int(qs[-1]) <= T, "q_start out of range")
    need(int(n.max()) <= max_q, "a sequence has more than max_q new tokens")
    need(int(kl.min()) >= 0 and int(kl.max()) <= 64 * bt.shape[1], "kv_len out of range")
    need(not appending or bool((kl >= n).all()), "kv_len counts the new tokens")
    used = torch.arange(bt.shape[1])[None] < ((kl + 63) // 64)[:, None]
    ids = bt[used]
    need(ids.numel() == 0 or (int(ids.min()) >= 0 and int(ids.max()) < pages),
         "block_tab names a page outside the pools")
    if appending:
        first = ((kl - n) // 64)[:, None]
        written = bt[used & (torch.arange(bt.shape[1])[None] >= first) & (n > 0)[:, None]]
        need(written.unique().numel() == written.numel(), "two sequences append to one page")


def _stream(dev, stream):
    return _cuda.current_stream(dev).cuda_stream if stream is None else stream


def _launch(dev, entry, *args) -> None:
    """Calls a C entry with the tensors' device `dev` current: it launches there, and a
    default stream's handle names no device."""
    if _cuda.current_device() == dev:
        rc = entry(*args)
    else:
        with _cuda.device(dev):
            rc = entry(*args)
    if rc:
        check(rc)


def _elsewhere():
    raise ValueError("all tensors on one CUDA device")


def kv_append(q, k, v, q_out, q_start, kv_len, block_tab, kpool, vpool, *, max_q, kscale=None,
              vscale=None, cos=None, sin=None, pos=None, axis_of=None, qn=None, kn=None, eps=1e-6,
              status=None, stream=None, validate=True):
    """Rotate queries and append keys and values to a paged cache (qa_k_kv_append).

    q [T, nq * hd], k and v [T, nkv * hd] 16-bit (rows may be slices of one
    packed projection), q_out like q (or q itself); q_start int32 [n + 1],
    kv_len int32 [n] (the new tokens counted), block_tab int32 [n, max_pages].
    Pools [pages, nkv, 64, hd]: float8_e4m3fn with kscale / vscale f32 [pages,
    nkv], or q's type without.  cos / sin f32 [rows, hd / 2]; pos int32 [T] or
    [axes, T] (None: the cache index) with axis_of int32 [hd / 2] when there are
    several axes; qn / kn f32 [hd].  `validate` copies the maps and the positions
    to the host to check them; without it, what is malformed sets bit 2 of
    `status` (int32 [1]) and is skipped.
    """
    if _F16 is None:
        _types()
    n, max_pages, pages, nkv, hd = _seq_args(q_start, kv_len, block_tab, kpool, vpool, max_q)
    dt = q.dtype
    if q.dim() != 2 or (dt is not _F16 and dt is not _BF16):
        raise ValueError("q [T, heads * hd] float16 or bfloat16")
    T, width = q.shape
    nq = width // hd
    if nq == 0 or nq % nkv or nq * hd != width:
        raise ValueError("q has a multiple of the cache's heads")
    max_q = min(max_q, T)  # no sequence has more
    kw = nkv * hd
    ldq, ldqo = _rows(q, T, width, dt, "q"), _rows(q_out, T, width, dt, "q_out")
    ldk, ldv = _rows(k, T, kw, dt, "k"), _rows(v, T, kw, dt, "v")
    dev = q.get_device()
    if dev < 0 or not (k.get_device() == v.get_device() == q_out.get_device() == q_start.get_device()
                       == kv_len.get_device() == block_tab.get_device() == kpool.get_device()
                       == vpool.get_device() == dev):
        here = False
    else:
        here = True
    ks = vs = cs = sn = ps = ax = gq = gk = st = 0
    if kscale is None:
        if vscale is not None or kpool.dtype is not dt:
            raise ValueError("pools of q's type, or e4m3 with both scales")
    else:
        if vscale is None or kpool.dtype is not _E4M3:
            raise ValueError("e4m3 pools with kscale and vscale f32 [pages, heads]")
        _flat(kscale, (pages, nkv), _F32, "kscale f32 [pages, heads]")
        _flat(vscale, (pages, nkv), _F32, "vscale f32 [pages, heads]")
        ks, vs = kscale.data_ptr(), vscale.data_ptr()
        here = here and kscale.get_device() == dev and vscale.get_device() == dev
    rows, axes, stride = 0, 1, 0
    if cos is not None:
        if sin is None or cos.dim() != 2 or cos.shape[0] == 0:
            raise ValueError("cos and sin f32 [rows, hd / 2]")
        rows = cos.shape[0]
        _flat(cos, (rows, hd // 2), _F32, "cos f32 [rows, hd / 2]")
        _flat(sin, (rows, hd // 2), _F32, "sin f32 [rows, hd / 2]")
        cs, sn = cos.data_ptr(), sin.data_ptr()
        here = here and cos.get_device() == dev and sin.get_device() == dev
        if pos is not None:
            d = pos.dim()
            if (pos.dtype is not _I32 or d not in (1, 2) or pos.shape[-1] != T
                    or (T > 1 and pos.stride(-1) != 1)):
                raise ValueError("pos int32 [T] or [axes, T]")
            if d == 2:
                axes, stride = pos.shape[0], pos.stride(0)
            if not 1 <= axes <= 4:
                raise ValueError("one to four axes")
            ps = pos.data_ptr()
            here = here and pos.get_device() == dev
            if axes > 1:
                if axis_of is None:
                    raise ValueError("axis_of int32 [hd / 2] for several axes")
                _flat(axis_of, (hd // 2,), _I32, "axis_of int32 [hd / 2]")
                ax = axis_of.data_ptr()
                here = here and axis_of.get_device() == dev
    elif sin is not None or pos is not None:
        raise ValueError("sin and pos go with cos")
    if qn is not None or kn is not None:
        if qn is None or kn is None:
            raise ValueError("qn and kn go together")
        _flat(qn, (hd,), _F32, "qn f32 [hd]")
        _flat(kn, (hd,), _F32, "kn f32 [hd]")
        gq, gk = qn.data_ptr(), kn.data_ptr()
        here = here and qn.get_device() == dev and kn.get_device() == dev
    if status is not None:
        if status.dtype is not _I32 or status.numel() == 0:
            raise ValueError("status int32 [1]")
        st = status.data_ptr()
        here = here and status.get_device() == dev
    if validate:
        check_sequences(T, q_start, kv_len, block_tab, pages, max_q, True)
        if axes > 1:
            a = axis_of.cpu()
            if int(a.min()) < 0 or int(a.max()) >= axes:
                raise ValueError("axis_of out of range")
        if pos is not None:
            if T and (int(pos.min()) < 0 or int(pos.max()) >= rows):
                raise ValueError("pos outside the tables")
        elif cos is not None and n and int(kv_len.max()) > rows:
            raise ValueError("kv_len outside the tables")
    if not here:
        _elsewhere()
    _launch(dev, _fn_kv_append(), _pack35(
        q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, q_out.data_ptr(), ldqo, T, nq, nkv,
        hd, q_start.data_ptr(), kv_len.data_ptr(), n, max_q, block_tab.data_ptr(), max_pages,
        kpool.data_ptr(), vpool.data_ptr(), pages, ks, vs, cs, sn, rows, ps, stride, axes, ax, gq, gk,
        1 if dt is _BF16 else 0, st, _stream(dev, stream)), eps)


def _workspace(need, device, stream):
    """`need` bytes that belong to the stream of the launch, so that whoever gets
    them next is behind it; under graph capture they come from the graph's pool."""
    import torch
    if stream is None:
        return torch.empty(need, dtype=_U8, device=device)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
        return torch.empty(need, dtype=_U8, device=device)


def cache_attention(q, q_start, kv_len, block_tab, kpool, vpool, kscale, vscale, out, *, max_q,
                    max_kv, causal=True, scale=None, lse=None, status=None, stream=None,
                    validate=True):
    """Attention over the e4m3 paged cache (qa_k_cache_attention).

    q and out [T, nq * hd] 16-bit; the maps, pools and scales as for kv_append;
    lse f32 [T, nq] optional; scale defaults to 1 / sqrt(hd).  max_q and max_kv
    bound the sequences' new and cached tokens.  `validate` copies the maps to
    the host to check them.  The workspace is torch's, taken and given back in the
    order of the launch stream; a graph that captures the call has its own.
    """
    if _F16 is None:
        _types()
    n, max_pages, pages, nkv, hd = _seq_args(q_start, kv_len, block_tab, kpool, vpool, max_q)
    dt = q.dtype
    if q.dim() != 2 or (dt is not _F16 and dt is not _BF16):
        raise ValueError("q [T, heads * hd] float16 or bfloat16")
    if kpool.dtype is not _E4M3:
        raise ValueError("e4m3 pools")
    _flat(kscale, (pages, nkv), _F32, "kscale f32 [pages, heads]")
    _flat(vscale, (pages, nkv), _F32, "vscale f32 [pages, heads]")
    T, width = q.shape
    nq = width // hd
    if nq == 0 or nq % nkv or nq * hd != width:
        raise ValueError("q has a multiple of the cache's heads")
    ldq, ldo = _rows(q, T, width, dt, "q"), _rows(out, T, width, dt, "out")
    if max_kv < 0:
        raise ValueError("max_kv >= 0")
    max_q, max_kv = min(max_q, T), min(max_kv, 64 * max_pages)  # no sequence has more
    ls = st = 0
    dev = q.get_device()
    here = dev >= 0 and (out.get_device() == q_start.get_device() == kv_len.get_device()
                         == block_tab.get_device() == kpool.get_device() == vpool.get_device()
                         == kscale.get_device() == vscale.get_device() == dev)
    if lse is not None:
        _flat(lse, (T, nq), _F32, "lse f32 [T, heads]")
        ls = lse.data_ptr()
        here = here and lse.get_device() == dev
    if status is not None:
        if status.dtype is not _I32 or status.numel() == 0:
            raise ValueError("status int32 [1]")
        st = status.data_ptr()
        here = here and status.get_device() == dev
    if validate:
        check_sequences(T, q_start, kv_len, block_tab, pages, max_q, False)
        if n and int(kv_len.max()) > max_kv:
            raise ValueError("a cache is longer than max_kv")
    if not here:
        _elsewhere()
    s = _stream(dev, stream)
    call, size = _fn_cache_attention()
    need = size(nq, nkv, hd, n, max_q, max_kv)
    ws = 0
    if need:
        buf = _workspace(need, q.device, stream)
        ws = buf.data_ptr()
    _launch(dev, call, _pack27(
        q.data_ptr(), ldq, T, nq, nkv, hd, q_start.data_ptr(), kv_len.data_ptr(), n, max_q,
        max_kv, block_tab.data_ptr(), max_pages, kpool.data_ptr(), vpool.data_ptr(), pages,
        kscale.data_ptr(), vscale.data_ptr(), 1 if causal else 0, out.data_ptr(), ldo, ls, ws, need,
        1 if dt is _BF16 else 0, st, s), hd ** -0.5 if scale is None else scale)


def w4_linear(x, wq, scales, out, *, zeros=None, bias=None, stream=None):
    """out [M, N] = x [M, K] . W^T + bias, W in 4 bits (qa_k_w4_linear).

    wq uint8 [N, K / 2], low nibble first; scales [N, K / group] of x's type with
    group 32, 64 or 128 (told by the shapes); zeros uint8 like scales, any value (None: 8);
    bias f32 [N].
    """
    if _F16 is None:
        _types()
    dt = x.dtype
    if x.dim() != 2 or wq.dim() != 2 or scales.dim() != 2 or (dt is not _F16 and dt is not _BF16):
        raise ValueError("x [M, K] float16 or bfloat16, wq [N, K / 2], scales [N, K / group]")
    M, K = x.shape
    N, half = wq.shape
    ldw, one = wq.stride()
    if N < 2:
        ldw = half
    if wq.dtype is not _U8 or 2 * half != K or (one != 1 and half > 1) or ldw < half:
        raise ValueError("wq uint8 [N, K / 2]")
    groups = scales.shape[1]
    _flat(scales, (N, groups), dt, "scales [N, K / group] of x's type")
    group = K // groups if groups else 0
    if group not in (32, 64, 128) or group * groups != K:
        raise ValueError("group 32, 64 or 128")
    ldx, ldo = _rows(x, M, K, dt, "x"), _rows(out, M, N, dt, "out")
    dev = x.get_device()
    here = dev >= 0 and wq.get_device() == scales.get_device() == out.get_device() == dev
    z = b = 0
    if zeros is not None:
        _flat(zeros, (N, groups), _U8, "zeros uint8 [N, K / group]")
        z = zeros.data_ptr()
        here = here and zeros.get_device() == dev
    if bias is not None:
        _flat(bias, (N,), _F32, "bias f32 [N]")
        b = bias.data_ptr()
        here = here and bias.get_device() == dev
    if not here:
        _elsewhere()
    _launch(dev, _fn_w4_linear(), _pack15(
        x.data_ptr(), ldx, M, K, wq.data_ptr(), ldw, N, group, scales.data_ptr(), z, b,
        out.data_ptr(), ldo, 1 if dt is _BF16 else 0, _stream(dev, stream)))


# The C functions, looked up once: lib() takes a lock.
_fns: dict = {}


def _fn_kv_append():
    return _fns.get("append") or _fns.setdefault("append", lib().qa_k_kv_append_v)


def _fn_cache_attention():
    return _fns.get("attend") or _fns.setdefault(
        "attend", (lib().qa_k_cache_attention_v, lib().qa_k_cache_attention_workspace))


def _fn_w4_linear():
    return _fns.get("w4") or _fns.setdefault("w4", lib().qa_k_w4_linear_v)
