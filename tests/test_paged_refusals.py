"""What the rotary and paged-attention entry points refuse, before any device work: run on the
CPU with addresses that nothing reads."""
import ctypes as C

import numpy as np
import pytest

from uocr_hip import _lib
from uocr_hip._lib import EINVAL, EUNSUPPORTED, EWORKSPACE, OK, AttentionOptsC, PagedCacheC, RowsC

A = 1 << 20  # a 16-byte aligned address


def rows(**kw):
    return RowsC(**{**dict(data=A, dtype=1, row_stride=512, head_stride=128), **kw})


def cache(**kw):
    return PagedCacheC(**{**dict(k=A, v=A, dtype=1, n_pages=8, page_size=16, kv_heads=2, head_dim=128, page_stride=4096,
                                 row_stride=256, head_stride=128, page_table=A, n_seqs=3, max_pages=4, table_stride=4), **kw})


def opts(**kw):
    return AttentionOptsC(**{**dict(heads=4, causal=1), **kw})


def ref(x):
    return None if x is None else C.byref(x)


def decode(c=None, o=None, q=None, out=None, batch=3, seqs=None, kv_len=A, hint=0, ws=None, size=0):
    lib = _lib.load()
    return lib.uocr_hip_paged_attention_decode(ref(c or cache()), ref(o or opts()), ref(q or rows()), batch, seqs, kv_len, hint,
                                               ref(out or rows()), ws, size, None)


def prefill(c=None, o=None, q=None, out=None, n=20, batch=3, start=A, seqs=None, kv_len=A, hint=0, ws=None, size=0):
    lib = _lib.load()
    return lib.uocr_hip_paged_attention_prefill(ref(c or cache()), ref(o or opts()), ref(q or rows()), n, batch, start, seqs,
                                                kv_len, hint, ref(out or rows()), ws, size, None)


BAD_CACHES = [
    (dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(page_table=None), EINVAL), (dict(dtype=7), EINVAL),
    (dict(n_pages=0), EINVAL), (dict(page_size=0), EINVAL), (dict(page_size=-16), EINVAL), (dict(kv_heads=0), EINVAL),
    (dict(n_seqs=0), EINVAL), (dict(max_pages=0), EINVAL), (dict(head_dim=0), EUNSUPPORTED), (dict(head_dim=12), EUNSUPPORTED),
    (dict(head_dim=264), EUNSUPPORTED), (dict(page_stride=-8), EINVAL), (dict(row_stride=-8), EINVAL),
    (dict(head_stride=4), EUNSUPPORTED), (dict(row_stride=132), EUNSUPPORTED), (dict(page_stride=4100), EUNSUPPORTED),
    (dict(k=A + 8), EUNSUPPORTED), (dict(v=A + 2), EUNSUPPORTED), (dict(table_stride=3), EINVAL), (dict(table_stride=-4), EINVAL),
    (dict(page_table=A + 2), EINVAL), (dict(page_size=(1 << 30) + 1), EUNSUPPORTED), (dict(page_stride=2**62), EINVAL),
    (dict(dtype=0, head_stride=130), EUNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_caches(kw, code):
    lib = _lib.load()
    bad = cache(**kw)
    assert decode(c=bad) == code and lib.uocr_hip_last_error()
    assert prefill(c=bad) == code
    assert lib.uocr_hip_paged_attention_workspace_size(C.byref(bad), 4, 10) == 0 and lib.uocr_hip_last_error()
    r = rows()
    assert lib.uocr_hip_rope_append_paged(C.byref(r), C.byref(r), C.byref(r), 2, 4, A, A, 128, 0, 1.0, C.byref(bad), A, A,
                                          C.byref(r), None) == code
    assert lib.uocr_hip_paged_attention_decode(None, None, None, 1, None, None, 0, None, None, 0, None) == EINVAL


@pytest.mark.parametrize("call", [decode, prefill])
@pytest.mark.parametrize("kw,code", [
    (dict(o=opts(heads=0)), EINVAL), (dict(o=opts(heads=3)), EINVAL), (dict(o=opts(heads=-2)), EINVAL),
    (dict(o=opts(scale=float("nan"))), EINVAL), (dict(o=opts(scale=float("inf"))), EINVAL), (dict(o=opts(softcap=-1.0)), EINVAL),
    (dict(o=opts(softcap=float("nan"))), EINVAL), (dict(o=opts(softcap=1e-30)), EUNSUPPORTED), (dict(o=opts(scale=1e30)), EUNSUPPORTED), (dict(o=opts(window=-1)), EINVAL), (dict(batch=-1), EINVAL),
    (dict(hint=-1), EINVAL), (dict(q=rows(data=None)), EINVAL), (dict(out=rows(data=None)), EINVAL),
    (dict(q=rows(dtype=0)), EINVAL), (dict(q=rows(dtype=3)), EINVAL), (dict(out=rows(dtype=2)), EINVAL),
    (dict(q=rows(data=A + 4)), EUNSUPPORTED), (dict(q=rows(row_stride=513)), EUNSUPPORTED),
    (dict(q=rows(head_stride=-128)), EINVAL), (dict(out=rows(data=A + 1)), EINVAL), (dict(kv_len=None), EINVAL),
    (dict(batch=4), EINVAL),  # more sequences than the cache has, and no d_seqs
    (dict(q=rows(row_stride=2**61)), EINVAL)])
def test_attention_arguments(call, kw, code):
    assert call(**kw) == code and _lib.load().uocr_hip_last_error()


def test_attention_workspace_and_the_rest():
    big = cache(max_pages=4096, table_stride=4096)
    need = _lib.load().uocr_hip_paged_attention_workspace_size(C.byref(big), 4, 3)
    assert need > 0
    assert decode(c=big) == EWORKSPACE and decode(c=big, ws=A, size=64) == EWORKSPACE
    assert decode(c=big, ws=A + 4, size=need) == EINVAL
    assert _lib.load().uocr_hip_paged_attention_workspace_size(C.byref(big), 3, 3) == 0
    assert _lib.load().uocr_hip_paged_attention_workspace_size(C.byref(big), 4, -1) == 0
    init = _lib.load().uocr_hip_paged_attention_workspace_init
    assert init(None, need, None) == EINVAL and init(A + 8, need, None) == EINVAL and init(A, 1024, None) == EWORKSPACE
    assert prefill(start=None) == EINVAL and prefill(n=-1) == EINVAL
    assert prefill(o=opts(window=4, causal=0)) == EINVAL
    assert prefill(n=2**30, o=opts(heads=4)) == EUNSUPPORTED
    # nothing to do
    assert decode(batch=0) == OK and prefill(n=0) == OK and prefill(batch=0) == OK


def rope(q=None, k=None, n=2, heads=4, kv=2, d=128, pos=A, freq=A, rot=128, factor=1.0, qo=None, ko=None):
    lib = _lib.load()
    return lib.uocr_hip_rope(ref(q or rows()), ref(k or rows()), n, heads, kv, d, pos, freq, rot, 0, factor, ref(qo or rows()),
                             ref(ko or rows()), None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), EINVAL), (dict(heads=-1), EINVAL), (dict(kv=-1), EINVAL), (dict(d=0), EUNSUPPORTED), (dict(d=257), EUNSUPPORTED),
    (dict(rot=3), EINVAL), (dict(rot=-2), EINVAL), (dict(rot=130), EINVAL), (dict(pos=None), EINVAL), (dict(freq=None), EINVAL),
    (dict(factor=float("nan")), EINVAL), (dict(q=rows(data=None)), EINVAL), (dict(ko=rows(data=None)), EINVAL),
    (dict(k=rows(dtype=0)), EINVAL), (dict(ko=rows(dtype=0)), EINVAL), (dict(q=rows(dtype=9)), EINVAL),
    (dict(q=rows(data=A + 1)), EINVAL), (dict(heads=2**30, d=256), EUNSUPPORTED)])
def test_rope_arguments(kw, code):
    assert rope(**kw) == code and _lib.load().uocr_hip_last_error()


def test_rope_nothing_to_do():
    assert rope(n=0) == OK and rope(heads=0, kv=0) == OK and rope(n=0, pos=None) == OK


def append(c=None, q=None, k=None, v=None, qo=None, n=2, heads=4, rot=128, seqs=A, at=A, pos=A):
    lib = _lib.load()
    return lib.uocr_hip_rope_append_paged(ref(q or rows()), ref(k or rows()), ref(v or rows()), n, heads, pos, A, rot, 0, 1.0,
                                          ref(c or cache()), seqs, at, ref(qo or rows()), None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), EINVAL), (dict(rot=256), EINVAL), (dict(seqs=None), EINVAL), (dict(at=None), EINVAL), (dict(pos=None), EINVAL),
    (dict(k=rows(data=None)), EINVAL), (dict(v=rows(data=None)), EINVAL), (dict(v=rows(dtype=0)), EINVAL),
    (dict(q=rows(dtype=0)), EINVAL), (dict(qo=rows(dtype=0)), EINVAL), (dict(qo=rows(data=None)), EINVAL)])
def test_append_arguments(kw, code):
    assert append(**kw) == code and _lib.load().uocr_hip_last_error()


def freqs(n=64, base=10000.0, kind=0, factor=1.0, length=0, fast=32.0, slow=1.0):
    out = np.zeros(max(n // 2, 1), np.float32)
    m = C.c_float(0)
    rc = _lib.load().uocr_hip_rope_frequencies(n, base, kind, factor, length, fast, slow, out.ctypes.data, C.byref(m))
    return rc, out, m.value


@pytest.mark.parametrize("kw", [
    dict(n=0), dict(n=3), dict(n=258), dict(base=1.0), dict(base=float("nan")), dict(base=float("inf")), dict(kind=4), dict(kind=-1),
    dict(kind=1, factor=0.5), dict(kind=1, factor=float("nan")), dict(kind=2, n=2, factor=2.0), dict(kind=3, factor=2.0),
    dict(kind=3, factor=2.0, length=100, slow=0.0), dict(kind=3, factor=2.0, length=100, fast=1.0, slow=1.0)])
def test_frequency_arguments(kw):
    assert freqs(**kw)[0] == EINVAL


def test_frequencies():
    """Against the formulas; each value rounded once to f32 (64-bit pow is good to a few 2^-53)."""
    i = np.arange(32)
    f = 10000.0 ** (-2.0 * i / 64)
    assert np.array_equal(freqs()[1], f.astype(np.float32)) and freqs()[2] == 1.0
    assert np.array_equal(freqs(kind=1, factor=4.0)[1], (f / 4).astype(np.float32))
    g = (10000.0 * 4.0 ** (64 / 62)) ** (-2.0 * i / 64)
    assert (np.abs(freqs(kind=2, factor=4.0)[1] - g) <= 2.0**-24 * g + 1e-13 * g).all()
    rc, h, m = freqs(kind=3, factor=8.0, length=4096)
    turns = 4096 * f / (2 * np.pi)
    assert rc == OK and m == np.float32(0.1 * np.log(8.0) + 1.0)
    kept, div = turns >= 32, turns <= 1
    assert kept.any() and div.any()
    # the ramp's ends are whole indices: one index of leeway beyond the turn limits
    assert np.array_equal(h[kept], f[kept].astype(np.float32)) and np.array_equal(h[div][1:], (f[div] / 8).astype(np.float32)[1:])
    assert (np.diff(h / f.astype(np.float32)) <= 1e-6).all()


def test_python_refuses_before_the_library():
    torch = pytest.importorskip("torch")
    from uocr_hip import paged
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    t = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        paged.PagedKVCache(k, k, t)
    for a, b, c in ((k, k.float(), t), (k, k[:3], t), (k, k.transpose(0, 1).contiguous().transpose(0, 1), t), (k[0], k[0], t),
                    (k, k, t.long()), (k, k, t[0]), (k[..., ::2], k[..., ::2], t)):
        with pytest.raises(ValueError):
            paged.PagedKVCache(a, b, c)
    with pytest.raises(TypeError):
        paged.PagedKVCache(k.double(), k.double(), t)
    q = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="GPU"):
        paged.rope(q, None, t[0, :2], torch.zeros(32), q, None)
    with pytest.raises(TypeError, match="tensor"):
        paged._n.rope([], None, None, None, None, None, 0, 1.0, 0)
    with pytest.raises(TypeError, match="9 arguments"):
        paged._n.rope(q)
    with pytest.raises(ValueError, match="scaling"):
        paged.rope_frequencies(64, scaling="dynamic")
    f, m = paged.rope_frequencies(64, scaling="parts", factor_len=8.0, original_len=4096)
    assert f.shape == (32,) and m > 1.2
