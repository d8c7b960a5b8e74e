"""Rotary positions, a paged key-value cache and its attention, on torch device tensors.

The calls are asynchronous on `stream` (a raw hipStream_t; None: torch's current stream of
the tensors' device). Tensors a call works on belong to one device and stay
alive, and unchanged by others, until the stream has run it.
"""
import ctypes as C

import torch

from . import _lib
from ._lib import OPTS_PACK, ROWS_PACK, PagedCacheC, check, load

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
SCALING = {"none": 0, "linear": 1, "base": 2, "parts": 3}


# The checks below run before every launch, which takes a few us itself: each reads
# a tensor's attributes once, and builds a message only to raise it.

def _rows(t, name, shape, index):
    """uocr_hip_rows of a tensor [rows, heads, head_dim] on GPU `index` whose last dim is contiguous."""
    st = t.stride()
    if t.shape != shape or (st[2] != 1 and shape[2] > 1):
        raise ValueError(f"{name} must be [rows, heads, head_dim] = {tuple(shape)} with contiguous dims of a head, got "
                         f"{tuple(t.shape)} with strides {tuple(st)}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on GPU {index}")
    dt = _DTYPE.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name} must be f32, bf16 or f16")
    return ROWS_PACK(t.data_ptr(), dt, st[0], st[1])


def _shape(t, name, index):
    """[rows, heads, head_dim] of a call's first tensor."""
    if index < 0:
        raise ValueError("tensors must be on a GPU")
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name} must be [rows, heads, head_dim], got {tuple(shape)}")
    return shape


def _vector(t, name, n, index, dtype=torch.int32):
    """Device address of a contiguous vector of n entries (None: 0)."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != index or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} entries on GPU {index}")
    return t.data_ptr()


def _call(fn, index, stream, *args):
    """fn(*args, stream) with GPU `index` current."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _call(fn, index, stream, *args)
    rc = fn(*args, torch._C._cuda_getCurrentRawStream(index) if stream is None else stream)
    if rc:
        check(rc)


def rope_frequencies(rotary_dim, base=10000.0, scaling="none", factor_len=1.0, original_len=0, fast=32.0, slow=1.0):
    """(inv_freq, factor): the f32 CPU tensor of rotary frequencies [rotary_dim / 2] and the factor
    on cos and sin. `scaling`: "none", "linear" (positions divided by factor_len), "base" (a
    larger base) or "parts" (each frequency by its turns over original_len positions)."""
    if scaling not in SCALING:
        raise ValueError(f"scaling must be one of {sorted(SCALING)}")
    f = torch.empty(max(rotary_dim // 2, 1), dtype=torch.float32)
    m = C.c_float(0.0)
    check(load().uocr_hip_rope_frequencies(rotary_dim, float(base), SCALING[scaling], float(factor_len),
                                           original_len, float(fast), float(slow), f.data_ptr(), C.byref(m)))
    return f, m.value


class PagedKVCache:
    """A paged key-value cache over the caller's tensors: k_pages and v_pages
    [n_pages, page_size, kv_heads, head_dim] (any strides that both share, the dims of a head
    contiguous) and page_table int32 [n_seqs, max_pages] (entries contiguous), whose entries may change
    between calls. Holds the tensors."""

    def __init__(self, k_pages, v_pages, page_table):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride() or \
                k_pages.dtype != v_pages.dtype:
            raise ValueError("k_pages and v_pages must be [n_pages, page_size, kv_heads, head_dim] of one type and layout")
        if k_pages.dtype not in _DTYPE:
            raise TypeError("pages must be f32, bf16 or f16")
        if k_pages.stride(3) != 1:
            raise ValueError("the dims of a head must be contiguous")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.stride(1) != 1:
            raise ValueError("page_table must be int32 [n_seqs, max_pages] with contiguous rows")
        self.device, self.index = k_pages.device, k_pages.get_device()
        if self.index < 0:
            raise ValueError("tensors must be on a GPU")
        if v_pages.device != self.device or page_table.device != self.device:
            raise ValueError("k_pages, v_pages and page_table must be on one GPU")
        self.k_pages, self.v_pages, self.page_table = k_pages, v_pages, page_table
        self.n_pages, self.page_size, self.kv_heads, self.head_dim = k_pages.shape
        self.n_seqs, self.max_pages = page_table.shape
        self.dtype = k_pages.dtype
        st = k_pages.stride()
        self.desc = PagedCacheC(k_pages.data_ptr(), v_pages.data_ptr(), _DTYPE[self.dtype], self.n_pages, self.page_size,
                                self.kv_heads, self.head_dim, st[0], st[1], st[2], page_table.data_ptr(), self.n_seqs,
                                self.max_pages, page_table.stride(0))
        self.address = C.addressof(self.desc)


def rope(q, k, positions, inv_freq, q_out, k_out, interleaved=False, factor=1.0, stream=None):
    """q_out, k_out = q, k [rows, heads, head_dim] with the first 2 * len(inv_freq) dims of every
    head turned by positions[row] * inv_freq[i]. k and k_out may be None; q_out may be q, k_out k."""
    g = q.get_device()
    shape = _shape(q, "q", g)
    n, h, d = shape
    if (k is None) != (k_out is None):
        raise ValueError("k and k_out go together")
    hk, ki, ko = 0, None, None
    if k is not None:
        ks = _shape(k, "k", g)
        hk = ks[1]
        ks = torch.Size((n, hk, d))
        ki, ko = _rows(k, "k", ks, g), _rows(k_out, "k_out", ks, g)
    half = inv_freq.numel()
    _call(load().uocr_hip_rope, g, stream, _rows(q, "q", shape, g), ki, n, h, hk, d, _vector(positions, "positions", n, g),
          _vector(inv_freq, "inv_freq", half, g, torch.float32), 2 * half, interleaved, factor,
          _rows(q_out, "q_out", shape, g), ko)


def rope_append(q, k, v, positions, inv_freq, cache, seqs, rows, q_out, interleaved=False, factor=1.0, stream=None):
    """rope() of q into q_out, and of k with v into the cache: row t becomes row rows[t] of sequence
    seqs[t] (outside the table's sequences: padding, left alone). q_out has the cache's
    type; inv_freq None (or empty) appends without rotation."""
    g = cache.index
    shape = _shape(q, "q", g)
    n, h, d = shape
    ks = torch.Size((n, cache.kv_heads, cache.head_dim))
    half = inv_freq.numel() if inv_freq is not None else 0
    if d != cache.head_dim:
        raise ValueError(f"q has head_dim {d}, the cache {cache.head_dim}")
    _call(load().uocr_hip_rope_append_paged, g, stream, _rows(q, "q", shape, g), _rows(k, "k", ks, g), _rows(v, "v", ks, g),
          n, h, _vector(positions, "positions", n, g) if half else 0,
          _vector(inv_freq, "inv_freq", half, g, torch.float32) if half else 0, 2 * half, interleaved, factor,
          cache.address, _vector(seqs, "seqs", n, g), _vector(rows, "rows", n, g), _rows(q_out, "q_out", shape, g))


def attention_workspace(cache, heads, rows):
    """A workspace for the attention calls of up to `rows` query rows, set up on torch's current stream.
    Calls that overlap in time need one each."""
    n = load().uocr_hip_paged_attention_workspace_size(cache.address, heads, rows)
    if n == 0 and rows > 0:
        raise _lib.HipError(_lib.EINVAL, load().uocr_hip_last_error().decode())
    ws = torch.empty(n, dtype=torch.uint8, device=cache.device)
    if n:
        _call(load().uocr_hip_paged_attention_workspace_init, cache.index, None, ws.data_ptr(), n)
    return ws


def _attention(fn, cache, q, out, kv_len, seqs, batch, scale, softcap, slopes, causal, window, prefix_len, both_ways, key_begin,
               key_end, max_kv_len, workspace, stream, *rows):
    g = cache.index
    shape = _shape(q, "q", g)
    n, h, d = shape
    if d != cache.head_dim:
        raise ValueError(f"q has head_dim {d}, the cache {cache.head_dim}")
    s = cache.n_seqs
    opts = OPTS_PACK(h, scale or 0.0, softcap, _vector(slopes, "slopes", h, g, torch.float32), causal, window,
                     _vector(prefix_len, "prefix_len", s, g), both_ways, _vector(key_begin, "key_begin", n, g),
                     _vector(key_end, "key_end", n, g))
    ws = size = 0
    if workspace is not None:
        ws, size = workspace.data_ptr(), workspace.nbytes
        if workspace.get_device() != g or not workspace.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on GPU {g}")
    _call(fn, g, stream, cache.address, opts, _rows(q, "q", shape, g), *rows, _vector(seqs, "seqs", batch, g),
          _vector(kv_len, "kv_len", s, g), max_kv_len, _rows(out, "out", shape, g), ws, size)


def attention_decode(q, cache, kv_len, out, seqs=None, scale=None, softcap=0.0, slopes=None, window=0, prefix_len=None,
                     key_begin=None, key_end=None, max_kv_len=0, workspace=None, stream=None):
    """Attention of one new token per sequence: row b of q and out [batch, heads, head_dim] is the
    last position of sequence seqs[b] (b if None), its K and V in the cache already. kv_len and
    prefix_len [n_seqs] int32; see uocr_hip_attention_opts for the scores and masks.
    max_kv_len (0: the table's room) only chooses the split."""
    n = q.size(0)
    _attention(load().uocr_hip_paged_attention_decode, cache, q, out, kv_len, seqs, n, scale, softcap, slopes, True, window,
               prefix_len, False, key_begin, key_end, max_kv_len, workspace, stream, n)


def attention_prefill(q, cache, q_start, kv_len, out, seqs=None, causal=True, scale=None, softcap=0.0, slopes=None, window=0,
                      prefix_len=None, prefix_both_ways=False, key_begin=None, key_end=None, max_kv_len=0,
                      workspace=None, stream=None):
    """Attention of many rows per sequence: rows q_start[b] .. q_start[b + 1] - 1 of q and out
    [rows, heads, head_dim] are the last positions of sequence seqs[b] (b if None). See attention_decode."""
    batch = q_start.numel() - 1
    if batch < 0:
        raise ValueError("q_start needs batch + 1 entries")
    _attention(load().uocr_hip_paged_attention_prefill, cache, q, out, kv_len, seqs, batch, scale, softcap, slopes, causal,
               window, prefix_len, prefix_both_ways, key_begin, key_end, max_kv_len, workspace, stream, q.size(0), batch,
               _vector(q_start, "q_start", batch + 1, cache.index))
