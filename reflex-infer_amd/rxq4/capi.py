"""ctypes binding of the C ABI in include/rxq4.h, plus torch-tensor helpers.

Every helper takes device tensors, passes raw pointers, launches on the given
stream (default: torch's current stream) and raises :class:`rxq4.RxQ4Error`
on a non-success status.
"""
from __future__ import annotations

import ctypes

import torch

from . import DTYPE_BF16, DTYPE_F16, DTYPE_F32, GGML_TYPE_Q4_K, SUCCESS, RxQ4Error, load

c_void_p, c_int, c_int64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64


class Rows(ctypes.Structure):
    """rxq4_rows: one output range of a multi-matrix GEMV."""
    _fields_ = [("y", c_void_p), ("w", c_void_p), ("ggml_type", c_int), ("M", c_int)]


class PagedKVStruct(ctypes.Structure):
    """rxq4_paged_kv: a paged KV cache."""
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("k_scales", c_void_p), ("v_scales", c_void_p),
                ("page_table", c_void_p), ("page_stride", c_int64), ("table_stride", c_int), ("n_pages", c_int),
                ("page_size", c_int), ("n_kv_heads", c_int), ("head_dim", c_int), ("kv_int8", c_int)]


class SeqBatchStruct(ctypes.Structure):
    """rxq4_seq_batch: the new tokens of a batch of sequences."""
    _fields_ = [("q_starts", c_void_p), ("seq_lens", c_void_p), ("n_seqs", c_int), ("n_tokens", c_int),
                ("max_new", c_int), ("max_len", c_int)]


# name -> (restype, argtypes); every name is declared in include/rxq4.h.
SIGNATURES = {
    "rxq4_gemv_f16": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p]),
    "rxq4_gemv_add_f16": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int, c_int,
                                  c_void_p]),
    "rxq4_gemv_multi_f16": (c_int, [ctypes.POINTER(Rows), c_int, c_void_p, c_int, c_void_p]),
    "rxq4_gemv_f32": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p]),
    "rxq4_gemm_f16": (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_int,
                              c_void_p]),
    "rxq4_embed_row_f16": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]),
    "rxq4_gemm": (c_int, [c_void_p, c_int, c_void_p, c_int, c_void_p, c_int, c_int, c_int,
                          c_int, c_void_p]),
    "rxq4_embed_rows_f16": (c_int, [c_void_p, c_void_p, c_int, c_int64, c_void_p, c_int, c_int,
                                    c_void_p]),
    "rxq4_gemm_noalloc": (c_int, [c_void_p, c_int, c_void_p, c_int, c_void_p, c_int, c_int, c_int,
                                  c_int, c_void_p]),
    "rxq4_quantize_q4k": (c_int, [c_void_p, c_void_p, c_int64, c_int, c_void_p]),
    "rxq4_quantize": (c_int, [c_void_p, c_int, c_void_p, c_int64, c_int, c_void_p]),
    "rxq4_attention_decode_f16": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int,
                                          c_int, c_int, ctypes.c_float, c_int, c_void_p,
                                          c_void_p, c_void_p]),
    "rxq4_attention_prefill_f16": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int,
                                           c_int, c_int, c_int, ctypes.c_float, c_int, c_void_p,
                                           c_void_p, c_void_p]),
    "rxq4_qk_norm_rope": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int64, c_int64, c_int, c_void_p,
                                  c_void_p, ctypes.c_float, c_void_p, c_int, c_int,
                                  ctypes.POINTER(SeqBatchStruct), ctypes.POINTER(PagedKVStruct), c_void_p]),
    "rxq4_attention_paged_f16": (c_int, [c_void_p, c_void_p, c_int, ctypes.c_float, ctypes.POINTER(SeqBatchStruct),
                                         ctypes.POINTER(PagedKVStruct), c_void_p]),
    "rxq4_sample_f32": (c_int, [c_void_p, c_void_p, c_int64, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p,
                                c_void_p, c_void_p]),
    "rxq4_host_gemv": (c_int, [c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p, c_int,
                               c_int]),
    "rxq4_host_gemv_calls": (ctypes.c_longlong, []),
    "rxq4_reserve_workspace": (c_int, [c_void_p]),
    "rxq4_release_workspace": (c_int, [c_void_p]),
    "rxq4_resolve_weights": (c_void_p, [c_void_p, c_void_p]),
    "rxq4_version": (ctypes.c_char_p, []),
    "rxq4_last_error": (ctypes.c_char_p, []),
}

_L = None


def _bind(lib: ctypes.CDLL) -> None:
    global _L
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _L = lib


def lib() -> ctypes.CDLL:
    if _L is None:
        load()
    return _L


def last_error() -> str:
    return lib().rxq4_last_error().decode()


def _check(status: int, what: str) -> int:
    if status != SUCCESS:
        raise RxQ4Error(status, f"{what} ({last_error()})")
    return status


# torch's current stream as a raw handle, without the Stream object that
# torch.cuda.current_stream() builds on every call (7.2 -> 4.1 us for a
# gemv_f32 call; the smallest kernels take 2.6 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream(stream) -> int:
    if stream is None:
        if _raw_stream is not None and _device is not None and torch.cuda.is_initialized():
            return _raw_stream(_device())
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _dtype_code(t: torch.Tensor) -> int:
    return {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}[t.dtype]


def gemv_f16(y, w, x, M, K, stream=None, ggml_type=GGML_TYPE_Q4_K):
    return _check(lib().rxq4_gemv_f16(_ptr(y), _ptr(w), ggml_type, _ptr(x), M, K,
                                      _stream(stream)), "rxq4_gemv_f16")


def gemv_f32(y, w, x, M, K, stream=None, ggml_type=GGML_TYPE_Q4_K):
    return _check(lib().rxq4_gemv_f32(_ptr(y), _ptr(w), ggml_type, _ptr(x), M, K,
                                      _stream(stream)), "rxq4_gemv_f32")


def gemv_add_f16(y, w, x, residual, M, K, stream=None, ggml_type=GGML_TYPE_Q4_K):
    return _check(lib().rxq4_gemv_add_f16(_ptr(y), _ptr(w), ggml_type, _ptr(x), _ptr(residual),
                                          M, K, _stream(stream)), "rxq4_gemv_add_f16")


def gemv_multi_f16(ranges, x, K, stream=None):
    """ranges: list of (y, w, M) or (y, w, M, ggml_type)."""
    arr = (Rows * len(ranges))()
    for i, r in enumerate(ranges):
        y, w, M = r[0], r[1], r[2]
        t = r[3] if len(r) > 3 else GGML_TYPE_Q4_K
        arr[i] = Rows(_ptr(y), _ptr(w), t, M)
    return _check(lib().rxq4_gemv_multi_f16(arr, len(ranges), _ptr(x), K, _stream(stream)),
                  "rxq4_gemv_multi_f16")


def gemm_f16(y, w, x, M, N, K, stream=None, ggml_type=GGML_TYPE_Q4_K):
    return _check(lib().rxq4_gemm_f16(_ptr(y), _ptr(w), ggml_type, _ptr(x), M, N, K,
                                      _stream(stream)), "rxq4_gemm_f16")


def gemm(y, w, x, M, N, K, stream=None, ggml_type=GGML_TYPE_Q4_K):
    """Typed GEMM: dtypes taken from the tensors (x fp16|bf16, y fp32|fp16|bf16)."""
    return _check(lib().rxq4_gemm(_ptr(y), _dtype_code(y), _ptr(w), ggml_type, _ptr(x),
                                  _dtype_code(x), M, N, K, _stream(stream)), "rxq4_gemm")


def gemm_noalloc(y, w, x, M, N, K, stream=None, ggml_type=GGML_TYPE_Q4_K):
    """rxq4_gemm with its split partials in the library's fixed device array
    (allocates nothing)."""
    return _check(lib().rxq4_gemm_noalloc(_ptr(y), _dtype_code(y), _ptr(w), ggml_type, _ptr(x),
                                          _dtype_code(x), M, N, K, _stream(stream)),
                  "rxq4_gemm_noalloc")


def embed_row_f16(dst, w, token_id, hidden, stream=None, ggml_type=GGML_TYPE_Q4_K):
    return _check(lib().rxq4_embed_row_f16(_ptr(dst), _ptr(w), ggml_type, token_id, hidden,
                                           _stream(stream)), "rxq4_embed_row_f16")


def embed_rows_f16(dst, w, n_vocab, ids, hidden, stream=None, ggml_type=GGML_TYPE_Q4_K):
    return _check(lib().rxq4_embed_rows_f16(_ptr(dst), _ptr(w), ggml_type, n_vocab, _ptr(ids),
                                            ids.numel(), hidden, _stream(stream)),
                  "rxq4_embed_rows_f16")


def quantize_q4k(dst, src, n_rows, K, stream=None):
    return _check(lib().rxq4_quantize_q4k(_ptr(dst), _ptr(src), n_rows, K, _stream(stream)),
                  "rxq4_quantize_q4k")


def quantize(src: torch.Tensor, stream=None) -> torch.Tensor:
    """Quantise a device fp32 [rows, K] tensor to a uint8 [rows, K/256*144] tensor."""
    rows, K = src.shape
    dst = torch.empty((rows, (K // 256) * 144), dtype=torch.uint8, device=src.device)
    quantize_q4k(dst, src.contiguous(), rows, K, stream)
    return dst


_TYPE_BYTES = {12: 144, 13: 176, 14: 210}


def quantize_ggml(src: torch.Tensor, ggml_type: int = GGML_TYPE_Q4_K, stream=None) -> torch.Tensor:
    """ggml's reference quantiser on the GPU: device fp32 [rows, K] -> uint8
    [rows, K/256 * block bytes] of ggml_type 12, 13 or 14."""
    rows, K = src.shape
    dst = torch.empty((rows, (K // 256) * _TYPE_BYTES.get(ggml_type, 144)), dtype=torch.uint8,
                      device=src.device)
    _check(lib().rxq4_quantize(_ptr(dst), ggml_type, _ptr(src.contiguous()), rows, K,
                               _stream(stream)), "rxq4_quantize")
    return dst


def attention_decode_f16(out, q, k, v, n_heads, n_kv_heads, head_dim, seq_len, scale,
                         kv_int8=False, k_scales=None, v_scales=None, stream=None):
    return _check(lib().rxq4_attention_decode_f16(
        _ptr(out), _ptr(q), _ptr(k), _ptr(v), n_heads, n_kv_heads, head_dim, seq_len, scale,
        int(kv_int8), _ptr(k_scales), _ptr(v_scales), _stream(stream)), "rxq4_attention_decode_f16")


def attention_prefill_f16(out, q, k, v, n_heads, n_kv_heads, head_dim, N, start_pos, scale,
                          kv_int8=False, k_scales=None, v_scales=None, stream=None):
    return _check(lib().rxq4_attention_prefill_f16(
        _ptr(out), _ptr(q), _ptr(k), _ptr(v), n_heads, n_kv_heads, head_dim, N, start_pos, scale,
        int(kv_int8), _ptr(k_scales), _ptr(v_scales), _stream(stream)),
        "rxq4_attention_prefill_f16")


def _int32(t, what):
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor")
    return t


def _same_device(name, first, *others):
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"{name}: tensors on {device} and {t.device}")


def _on_current_device(name, t):
    if not t.is_cuda or t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name}: tensors on {t.device}, which is not the current GPU")


class PagedKV:
    """A layer's paged KV cache, built once beside its tensors: k, v
    [n_pages, page_size, n_kv_heads, head_dim] fp16 or int8 (the pages may lie
    apart in memory, each dense in itself), int8 scales [n_pages, page_size,
    n_kv_heads] fp32, page_table int32 [n_seqs, pages] (None: one sequence whose
    pages are in order).  Holds the tensors."""

    def __init__(self, k, v, page_table=None, k_scales=None, v_scales=None):
        n_pages, page_size, n_kv, hd = k.shape
        if v.shape != k.shape or v.dtype != k.dtype or k.dtype not in (torch.float16, torch.int8):
            raise ValueError("PagedKV: k and v must be alike, fp16 or int8")
        stride = k.stride(0) if n_pages > 1 else page_size * n_kv * hd
        for t in (k, v):
            if t.stride()[1:] != (n_kv * hd, hd, 1) or (n_pages > 1 and t.stride(0) != stride):
                raise ValueError("PagedKV: a page must be dense, and K and V pages lie alike")
        if stride < page_size * n_kv * hd:
            raise ValueError("PagedKV: pages must not share memory")
        for t in (k_scales, v_scales):
            if t is not None and (t.dtype != torch.float32 or t.shape != k.shape[:3] or not t.is_contiguous()):
                raise ValueError("PagedKV: scales must be contiguous fp32 [n_pages, page_size, n_kv_heads]")
        if page_table is not None and (page_table.dim() != 2 or page_table.dtype != torch.int32 or
                                       (page_table.shape[1] > 1 and page_table.stride(1) != 1)):
            raise ValueError("PagedKV: page_table must be int32 [n_seqs, pages], its rows dense")
        _same_device("PagedKV", k, v, page_table, k_scales, v_scales)
        # (a table of no entries needs an address too: none at all means a contiguous cache)
        self._table = page_table.new_empty(1) if page_table is not None and page_table.numel() == 0 else page_table
        self.tensors = (k, v, page_table, k_scales, v_scales)
        self.n_seqs = 1 if page_table is None else page_table.shape[0]
        self.n_kv_heads, self.head_dim = n_kv, hd
        pages = 0 if page_table is None else page_table.shape[1]
        if pages > 0 and self.n_seqs > 1 and page_table.stride(0) != pages:
            raise ValueError("PagedKV: page_table must be dense")
        self.struct = PagedKVStruct(_ptr(k), _ptr(v), _ptr(k_scales), _ptr(v_scales),
                                    _ptr(self._table), stride, pages,
                                    n_pages, page_size, n_kv, hd, int(k.dtype == torch.int8))
        self.ref = ctypes.byref(self.struct)


class SeqBatch:
    """The new tokens of a batch (rxq4_seq_batch): q_starts int32 [n_seqs + 1],
    seq_lens int32 [n_seqs] on the device, and their limits.  Holds the tensors,
    whose values may change between calls (and replays) within the limits."""

    def __init__(self, q_starts, seq_lens, n_tokens, max_new, max_len):
        self.tensors = (_int32(q_starts, "q_starts"), _int32(seq_lens, "seq_lens"))
        self.n_seqs, self.n_tokens = seq_lens.numel(), n_tokens
        if q_starts.numel() != self.n_seqs + 1:
            raise ValueError("SeqBatch: q_starts must have one value more than seq_lens")
        _same_device("SeqBatch", q_starts, seq_lens)
        self.struct = SeqBatchStruct(_ptr(q_starts), _ptr(seq_lens), self.n_seqs, n_tokens, max_new, max_len)
        self.ref = ctypes.byref(self.struct)


def _fits(name, batch, cache):
    if batch.n_seqs > cache.n_seqs:
        raise ValueError(f"{name}: {batch.n_seqs} sequences, page_table has {cache.n_seqs}")
    _same_device(name, batch.tensors[0], cache.tensors[0])


def qk_norm_rope(q_out, q, k, v, batch, cache, inv_freq, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                 stream=None):
    """q [n_tokens, n_heads, head_dim] and k, v [n_tokens, n_kv_heads, head_dim]
    (fp16, bf16 or fp32, e.g. slices of one fused projection): head norms,
    rotation by position * inv_freq, queries to q_out, keys and values into the
    cache's pages."""
    _fits("qk_norm_rope", batch, cache)
    n, heads, hd = q.shape
    want = (batch.n_tokens, cache.n_kv_heads, cache.head_dim)
    if (n, hd) != (want[0], want[2]) or k.shape != want or v.shape != want or q_out.shape != q.shape:
        raise ValueError(f"qk_norm_rope: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, q_out "
                         f"{tuple(q_out.shape)} for {want[0]} tokens, {want[1]} KV heads of {want[2]}")
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    if sq[1:] != (hd, 1) or sk[1:] != (hd, 1) or sv[1:] != (hd, 1) or (sk[0] != sv[0] and n > 1) or \
            q.dtype != k.dtype or q.dtype != v.dtype or q_out.dtype != torch.float16 or not q_out.is_contiguous():
        raise ValueError("qk_norm_rope: rows must be dense, k and v rows equally far apart, q, k, v of one type, "
                         "q_out contiguous fp16")
    for t in (inv_freq, q_weight, k_weight):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError("qk_norm_rope: inv_freq and weights must be contiguous fp32")
    for t in (q_weight, k_weight):
        if t is not None and t.numel() != hd:
            raise ValueError(f"qk_norm_rope: weights must have head_dim={hd} values")
    _same_device("qk_norm_rope", cache.tensors[0], q_out, q, k, v, inv_freq, q_weight, k_weight)
    _on_current_device("qk_norm_rope", q)
    return _check(lib().rxq4_qk_norm_rope(
        _ptr(q_out), _ptr(q), _ptr(k), _ptr(v), _dtype_code(q), sq[0] if n > 1 else heads * hd,
        sk[0] if n > 1 else want[1] * hd, heads, _ptr(q_weight), _ptr(k_weight), eps, _ptr(inv_freq),
        0 if inv_freq is None else 2 * inv_freq.numel(), int(interleaved), batch.ref, cache.ref, _stream(stream)),
        "rxq4_qk_norm_rope")


def attention_paged_f16(out, q, batch, cache, scale, stream=None):
    """out, q fp16 [n_tokens, n_heads, head_dim]: each sequence's new tokens over
    its pages, causal."""
    _fits("attention_paged_f16", batch, cache)
    if q.dim() != 3 or q.shape[0] != batch.n_tokens or q.shape[2] != cache.head_dim or out.shape != q.shape or \
            q.dtype != torch.float16 or out.dtype != torch.float16 or not q.is_contiguous() or not out.is_contiguous():
        raise ValueError(f"attention_paged_f16: q and out must be contiguous fp16 [{batch.n_tokens}, n_heads, "
                         f"{cache.head_dim}]")
    _same_device("attention_paged_f16", cache.tensors[0], out, q)
    _on_current_device("attention_paged_f16", q)
    return _check(lib().rxq4_attention_paged_f16(_ptr(out), _ptr(q), q.shape[1], scale, batch.ref, cache.ref,
                                                 _stream(stream)), "rxq4_attention_paged_f16")


def sample_f32(ids, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, stream=None):
    """ids int32 [n] = the next token of each row of logits fp32 [n, vocab] from u
    fp32 [n] in [0, 1); the parameters are per-row tensors or None."""
    n, vocab = logits.shape
    for t, dtype in ((ids, torch.int32), (u, torch.float32), (temperature, torch.float32), (top_k, torch.int32),
                     (top_p, torch.float32), (min_p, torch.float32)):
        if t is not None and (t.dtype != dtype or t.numel() != n or not t.is_contiguous()):
            raise ValueError(f"sample_f32: every parameter must have one value for each of {n} rows (fp32; ids and "
                             "top_k int32)")
    if logits.dtype != torch.float32 or (vocab > 1 and logits.stride(1) != 1):
        raise ValueError("sample_f32: logits must be fp32 with dense rows")
    _same_device("sample_f32", logits, ids, u, temperature, top_k, top_p, min_p)
    _on_current_device("sample_f32", logits)
    return _check(lib().rxq4_sample_f32(_ptr(ids), _ptr(logits), logits.stride(0) if n > 1 else vocab, n, vocab,
                                        _ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p), _ptr(u),
                                        _stream(stream)), "rxq4_sample_f32")


def host_gemv(w, x, M: int, K: int, ggml_type: int = GGML_TYPE_Q4_K, out: str = "f32",
              residual=None):
    """The host GEMV (rxq4_host_gemv) on numpy arrays: w uint8 blocks, x fp16
    bits (uint16); out "f32" -> float32 [M], "f16" -> uint16 fp16 bits [M];
    residual (uint16 fp16 bits [M]) gives the add variant."""
    import numpy as np
    w = np.ascontiguousarray(w)
    x = np.ascontiguousarray(x, dtype=np.uint16)
    y = np.empty(M, dtype=np.float32 if out == "f32" else np.uint16)
    res = None if residual is None else np.ascontiguousarray(residual, dtype=np.uint16)
    _check(lib().rxq4_host_gemv(y.ctypes.data, DTYPE_F32 if out == "f32" else DTYPE_F16,
                                w.ctypes.data, ggml_type, x.ctypes.data,
                                None if res is None else res.ctypes.data, M, K),
           "rxq4_host_gemv")
    return y


def host_gemv_calls() -> int:
    """Computations made by the host GEMV in this process so far."""
    return int(lib().rxq4_host_gemv_calls())


def reserve_workspace(stream=None):
    return _check(lib().rxq4_reserve_workspace(_stream(stream)), "rxq4_reserve_workspace")


def release_workspace(stream=None):
    return _check(lib().rxq4_release_workspace(_stream(stream)), "rxq4_release_workspace")
