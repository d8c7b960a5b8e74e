"""Rotary positions, a paged key-value cache and its attention, on torch device tensors.

The calls are asynchronous on `stream` (a raw hipStream_t; None: torch's current stream of
the tensors' device). Tensors a call works on belong to one device and stay
alive, and unchanged by others, until the stream has run it.
"""
import ctypes as C
import importlib.machinery
import importlib.util
import os

import torch

from . import _lib
from ._lib import PagedCacheC, check, load

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
SCALING = {"none": 0, "linear": 1, "base": 2, "parts": 3}


def _native():
    """The native binding (csrc/torch_binding.cpp), on the entry points of the loaded library."""
    lib = load()
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lib", "_uocr_torch.so")
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is missing: build it first (python -c 'import __graft_entry__ as g; g.build()')")
    spec = importlib.util.spec_from_file_location("_uocr_torch", path,
                                                  loader=importlib.machinery.ExtensionFileLoader("_uocr_torch", path))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.bind(*(C.cast(getattr(lib, "uocr_hip_" + n), C.c_void_p).value
             for n in ("rope", "rope_append_paged", "paged_attention_decode", "paged_attention_prefill")))
    return m


_n = _native()
_current_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream


def _call(fn, index, stream, args):
    """fn(*args, stream) with GPU `index` current."""
    if index >= 0 and _current_device() != index:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index) if stream is None else stream)
    else:
        rc = fn(*args, stream if stream is not None or index < 0 else _raw_stream(index))
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
    _call(_n.rope, q.get_device(), stream, (q, k, positions, inv_freq, q_out, k_out, interleaved, factor))


def rope_append(q, k, v, positions, inv_freq, cache, seqs, rows, q_out, interleaved=False, factor=1.0, stream=None):
    """rope() of q into q_out, and of k with v into the cache: row t becomes row rows[t] of sequence
    seqs[t] (outside the table's sequences: padding, left alone). q_out has the cache's
    type; inv_freq None (or empty) appends without rotation."""
    _call(_n.rope_append, cache.index, stream,
          (q, k, v, positions, inv_freq, cache.address, cache.index, seqs, rows, q_out, interleaved, factor))


def attention_workspace(cache, heads, rows):
    """A workspace for the attention calls of up to `rows` query rows, set up on torch's current stream.
    Calls that overlap in time need one each."""
    n = load().uocr_hip_paged_attention_workspace_size(cache.address, heads, rows)
    if n == 0 and rows > 0:
        raise _lib.HipError(_lib.EINVAL, load().uocr_hip_last_error().decode())
    ws = torch.empty(n, dtype=torch.uint8, device=cache.device)
    if n:
        _call(load().uocr_hip_paged_attention_workspace_init, cache.index, None, (ws.data_ptr(), n))
    return ws


def attention_decode(q, cache, kv_len, out, seqs=None, scale=None, softcap=0.0, slopes=None, window=0, prefix_len=None,
                     key_begin=None, key_end=None, max_kv_len=0, workspace=None, stream=None):
    """Attention of one new token per sequence: row b of q and out [batch, heads, head_dim] is the
    last position of sequence seqs[b] (b if None), its K and V in the cache already. kv_len and
    prefix_len [n_seqs] int32; see uocr_hip_attention_opts for the scores and masks.
    max_kv_len (0: the table's room) only chooses the split. workspace: from attention_workspace, for as
    many rows; without one, calls that are split are refused."""
    _call(_n.attention, cache.index, stream,
          (q, cache.address, cache.index, None, kv_len, out, seqs, True, scale, softcap, slopes, window, prefix_len, False,
           key_begin, key_end, max_kv_len, workspace))


def attention_prefill(q, cache, q_start, kv_len, out, seqs=None, causal=True, scale=None, softcap=0.0, slopes=None, window=0,
                      prefix_len=None, prefix_both_ways=False, key_begin=None, key_end=None, max_kv_len=0,
                      workspace=None, stream=None):
    """Attention of many rows per sequence: rows q_start[b] .. q_start[b + 1] - 1 of q and out
    [rows, heads, head_dim] are the last positions of sequence seqs[b] (b if None). See attention_decode."""
    if q_start is None:
        raise ValueError("q_start is missing")
    _call(_n.attention, cache.index, stream,
          (q, cache.address, cache.index, q_start, kv_len, out, seqs, causal, scale, softcap, slopes, window, prefix_len,
           prefix_both_ways, key_begin, key_end, max_kv_len, workspace))
