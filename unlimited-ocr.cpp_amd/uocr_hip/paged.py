"""Rotary positions, a paged key-value cache and its attention, on torch device tensors.

The calls are asynchronous on `stream` (a raw hipStream_t; None: torch's current stream of
the tensors' device). Tensors a call works on belong to one device and stay
alive, and unchanged by others, until the stream has run it.
"""
import ctypes as C

import torch

from . import _lib
from ._lib import AttentionOptsC, PagedCacheC, RowsC, check, load

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
SCALING = {"none": 0, "linear": 1, "base": 2, "parts": 3}


def _rows(t, name, heads=None, head_dim=None, rows=None):
    """uocr_hip_rows of a tensor [rows, heads, head_dim] whose last dim is contiguous."""
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or (st[2] != 1 and shape[2] > 1):
        raise ValueError(f"{name} must be [rows, heads, head_dim] with contiguous dims of a head")
    if (rows is not None and shape[0] != rows) or (heads is not None and shape[1] != heads) or \
            (head_dim is not None and shape[2] != head_dim):
        raise ValueError(f"{name} has shape {tuple(shape)}")
    dt = _DTYPE.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name} must be f32, bf16 or f16")
    return RowsC(t.data_ptr(), dt, st[0], st[1])


def _ints(t, name, n, device):
    """Device pointer of an int32 vector of n entries (None: NULL)."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on {device}")
    return t.data_ptr()


def _floats(t, name, n, device):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.device != device or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{name} must be a contiguous f32 tensor" + (f" of {n} entries" if n is not None else "") + f" on {device}")
    return t.data_ptr()


def _same_device(device, **tensors):
    if device.type != "cuda":
        raise ValueError("tensors must be on a GPU")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _call(fn, device, stream, *args):
    """fn(*args, stream) with `device` current."""
    if torch.cuda.current_device() == device.index:
        check(fn(*args, stream if stream is not None else torch._C._cuda_getCurrentRawStream(device.index)))
    else:
        with torch.cuda.device(device):
            check(fn(*args, stream if stream is not None else torch._C._cuda_getCurrentRawStream(device.index)))


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
        self.device = k_pages.device
        _same_device(self.device, v_pages=v_pages, page_table=page_table)
        self.k_pages, self.v_pages, self.page_table = k_pages, v_pages, page_table
        self.n_pages, self.page_size, self.kv_heads, self.head_dim = k_pages.shape
        self.n_seqs, self.max_pages = page_table.shape
        self.dtype = k_pages.dtype
        st = k_pages.stride()
        self.desc = PagedCacheC(k_pages.data_ptr(), v_pages.data_ptr(), _DTYPE[self.dtype], self.n_pages, self.page_size,
                                self.kv_heads, self.head_dim, st[0], st[1], st[2], page_table.data_ptr(), self.n_seqs,
                                self.max_pages, page_table.stride(0))
        self.ref = C.byref(self.desc)


def rope(q, k, positions, inv_freq, q_out, k_out, interleaved=False, factor=1.0, stream=None):
    """q_out, k_out = q, k [rows, heads, head_dim] with the first 2 * len(inv_freq) dims of every
    head turned by positions[row] * inv_freq[i]. k and k_out may be None; q_out may be q, k_out k."""
    n, h, d = q.shape
    dev = q.device
    _same_device(dev, k=k, q_out=q_out, k_out=k_out)
    if (k is None) != (k_out is None):
        raise ValueError("k and k_out go together")
    a, b = _rows(q, "q"), _rows(q_out, "q_out", h, d, n)
    e = g = None
    hk = 0
    if k is not None:
        hk = k.shape[1]
        e, g = C.byref(_rows(k, "k", None, d, n)), C.byref(_rows(k_out, "k_out", hk, d, n))
    _call(load().uocr_hip_rope, dev, stream, C.byref(a), e, n, h, hk, d, _ints(positions, "positions", n, dev),
          _floats(inv_freq, "inv_freq", None, dev), 2 * inv_freq.numel(), int(interleaved), float(factor), C.byref(b), g)


def rope_append(q, k, v, positions, inv_freq, cache, seqs, rows, q_out, interleaved=False, factor=1.0, stream=None):
    """rope() of q into q_out, and of k with v into the cache: row t becomes row rows[t] of sequence
    seqs[t] (outside the table's sequences: padding, left alone). q_out has the cache's
    type; inv_freq None (or empty) appends without rotation."""
    n, h, d = q.shape
    dev = cache.device
    _same_device(dev, q=q, k=k, v=v, q_out=q_out)
    a, b = _rows(q, "q", None, cache.head_dim), _rows(q_out, "q_out", h, d, n)
    e, f = _rows(k, "k", cache.kv_heads, d, n), _rows(v, "v", cache.kv_heads, d, n)
    turn = inv_freq is not None and inv_freq.numel() > 0
    _call(load().uocr_hip_rope_append_paged, dev, stream, C.byref(a), C.byref(e), C.byref(f), n, h,
          _ints(positions, "positions", n, dev) if turn else None,
          _floats(inv_freq, "inv_freq", None, dev) if turn else None, 2 * inv_freq.numel() if turn else 0,
          int(interleaved), float(factor), cache.ref, _ints(seqs, "seqs", n, dev), _ints(rows, "rows", n, dev), C.byref(b))


def attention_workspace(cache, heads, rows):
    """A workspace for the attention calls of up to `rows` query rows. Calls
    that overlap in time need one each."""
    n = load().uocr_hip_paged_attention_workspace_size(cache.ref, heads, rows)
    if n == 0 and rows > 0:
        raise _lib.HipError(_lib.EINVAL, load().uocr_hip_last_error().decode())
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


def _opts(cache, heads, rows, scale, softcap, slopes, causal, window, prefix_len, both_ways, key_begin, key_end):
    dev = cache.device
    return AttentionOptsC(heads, scale or 0.0, softcap, _floats(slopes, "slopes", heads, dev), int(causal), window,
                          _ints(prefix_len, "prefix_len", cache.n_seqs, dev), int(both_ways),
                          _ints(key_begin, "key_begin", rows, dev), _ints(key_end, "key_end", rows, dev))


def _space(workspace, dev):
    if workspace is None:
        return None, 0
    if workspace.device != dev or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor on the cache's device")
    return workspace.data_ptr(), workspace.numel()


def attention_decode(q, cache, kv_len, out, seqs=None, scale=None, softcap=0.0, slopes=None, window=0, prefix_len=None,
                     key_begin=None, key_end=None, max_kv_len=0, workspace=None, stream=None):
    """Attention of one new token per sequence: row b of q and out [batch, heads, head_dim] is the
    last position of sequence seqs[b] (b if None), its K and V in the cache already. kv_len and
    prefix_len [n_seqs] int32; see uocr_hip_attention_opts for the scores and masks.
    max_kv_len (0: the table's room) only chooses the split."""
    n, h, d = q.shape
    dev = cache.device
    _same_device(dev, q=q, out=out)
    a, b = _rows(q, "q", None, cache.head_dim), _rows(out, "out", h, d, n)
    o = _opts(cache, h, n, scale, softcap, slopes, True, window, prefix_len, False, key_begin, key_end)
    ws, size = _space(workspace, dev)
    _call(load().uocr_hip_paged_attention_decode, dev, stream, cache.ref, C.byref(o), C.byref(a), n,
          _ints(seqs, "seqs", n, dev), _ints(kv_len, "kv_len", cache.n_seqs, dev), max_kv_len, C.byref(b), ws, size)


def attention_prefill(q, cache, q_start, kv_len, out, seqs=None, causal=True, scale=None, softcap=0.0, slopes=None, window=0,
                      prefix_len=None, prefix_both_ways=False, key_begin=None, key_end=None, max_kv_len=0,
                      workspace=None, stream=None):
    """Attention of many rows per sequence: rows q_start[b] .. q_start[b + 1] - 1 of q and out
    [rows, heads, head_dim] are the last positions of sequence seqs[b] (b if None). See attention_decode."""
    n, h, d = q.shape
    dev = cache.device
    _same_device(dev, q=q, out=out)
    batch = q_start.numel() - 1
    if batch < 0:
        raise ValueError("q_start needs batch + 1 entries")
    a, b = _rows(q, "q", None, cache.head_dim), _rows(out, "out", h, d, n)
    o = _opts(cache, h, n, scale, softcap, slopes, causal, window, prefix_len, prefix_both_ways, key_begin, key_end)
    ws, size = _space(workspace, dev)
    _call(load().uocr_hip_paged_attention_prefill, dev, stream, cache.ref, C.byref(o), C.byref(a), n, batch,
          _ints(q_start, "q_start", batch + 1, dev), _ints(seqs, "seqs", batch, dev),
          _ints(kv_len, "kv_len", cache.n_seqs, dev), max_kv_len, C.byref(b), ws, size)
