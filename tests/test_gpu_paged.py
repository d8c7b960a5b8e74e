"""Rotary positions, the append to a paged cache and single-token attention over it, against
plain implementations in 64 bits. Tolerances: see paged_ref.py."""
import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
# weights of the decode kernel: two halves of the type
P_ERR = {"f32": 0.0, "bf16": 2.0**-15, "f16": 2.0**-20}


def paged():
    from uocr_hip import paged as m
    return m


def i32(v, dev):
    return torch.tensor(list(v), dtype=torch.int32, device=dev)


def rand(rng, *shape, std=1.0):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * std)


# ---- rotary positions --------------------------------------------------------

def check_turned(got, want, x, rotary, interleaved, factor, dtype):
    """Within half a step of the result and of the f32 arithmetic: each of the two products and
    their sum rounds once in f32, the sine and the cosine (and factor) to 2^-22."""
    a = np.abs(x.double().numpy())
    if rotary:
        f, s = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
        both = (a[..., f] + a[..., s]) * factor
        err = np.zeros_like(a)
        err[..., f] = err[..., s] = both * (2.0**-21 if factor else 0)
    else:
        err = np.zeros_like(a)
    R.close(got, want, R.HALF[dtype] * (np.abs(want) + err) + err + R.TINY[dtype])


@pytest.mark.parametrize("xt,ot", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("heads,kv_heads,d,rotary,interleaved", [
    (10, 10, 128, 128, False), (8, 2, 64, 64, True), (3, 1, 96, 64, False), (3, 1, 96, 64, True),
    (4, 4, 256, 256, False), (5, 5, 80, 20, False), (2, 1, 18, 6, True), (1, 1, 8, 0, False), (2, 2, 128, 2, True)])
def test_rope(dev, xt, ot, heads, kv_heads, d, rotary, interleaved):
    rng = np.random.default_rng(heads * d + rotary)
    n = 13
    x = rand(rng, n, (heads + kv_heads) * d + 8).to(R.DT[xt])
    q, k = (t.unflatten(1, (-1, d)) for t in (x[:, :heads * d], x[:, heads * d:(heads + kv_heads) * d]))
    xd = x.to(dev)
    qd, kd = (t.unflatten(1, (-1, d)) for t in (xd[:, :heads * d], xd[:, heads * d:(heads + kv_heads) * d]))
    pos = np.concatenate([[0, 1, 2, -5, 2**31 - 1, 1048575, 999999], rng.integers(0, 200000, n - 7)])
    freq, factor = (paged().rope_frequencies(rotary, 10000.0, "parts", 8.0, 4096) if rotary
                    else (torch.empty(0), 1.0))
    qo, ko = (torch.empty(t.shape, dtype=R.DT[ot], device=dev) for t in (q, k))
    paged().rope(qd, kd, i32(pos, dev), freq.to(dev), qo, ko, interleaved=interleaved, factor=factor)
    for got, t in ((qo, q), (ko, k)):
        want = R.turned(t.double().numpy(), pos, freq.numpy(), rotary, interleaved, factor)
        check_turned(got, want, t, rotary, interleaved, factor, ot)
    if xt == ot:  # in place, and without k
        paged().rope(qd, None, i32(pos, dev), freq.to(dev), qd, None, interleaved=interleaved, factor=factor)
        assert torch.equal(qd, qo)
        assert torch.equal(xd[:, heads * d:].cpu(), x[:, heads * d:])


def test_rope_unaligned_rows(dev):
    """Rows that start off a 16-byte boundary take the element-wise kernel: the same bits."""
    rng = np.random.default_rng(5)
    n, h, d = 9, 3, 64
    x = rand(rng, n, h * d + 1).to(torch.bfloat16).to(dev)
    odd = x[:, 1:].unflatten(1, (h, d))
    freq, factor = paged().rope_frequencies(64)
    pos = i32(rng.integers(0, 5000, n), dev)
    a, b = torch.empty(n, h, d, dtype=x.dtype, device=dev), torch.empty(n, h, d, dtype=x.dtype, device=dev)
    paged().rope(odd, None, pos, freq.to(dev), a, None)
    paged().rope(odd.contiguous(), None, pos, freq.to(dev), b, None)
    assert torch.equal(a, b)


@pytest.mark.parametrize("xt,ct,layout,page", [("f32", "bf16", "nhd", 16), ("bf16", "bf16", "hnd", 5), ("f16", "f16", "kv", 1),
                                               ("f32", "f32", "nhd", 24), ("bf16", "f16", "hnd", 64)])
@pytest.mark.parametrize("rotary", [64, 0])
def test_append(dev, xt, ct, layout, page, rotary):
    """Rows land where the table says, padding and rows without a page leave the cache (and, for
    padding, q_out) as they were."""
    rng = np.random.default_rng(page)
    hk, h, d, lens = 2, 6, 64, [37, 1, 70]
    pool = R.Pool(rng, lens, hk, d, page, ct, dev, layout)
    cache = pool.cache()
    before = [cache.k_pages.clone(), cache.v_pages.clone()]
    seqs = [0, 2, 2, 1, -1, 3, 0, 2, 2**31 - 1, 0]
    rows = [36, 0, 69, 0, 4, 0, -1, 70 + 3 * page, 0, 40 * 1000]  # the last ones outside the table, or the sequences
    ok = [0, 1, 2, 3]
    n = len(seqs)
    pos = rng.integers(0, 100000, n)
    qkv = rand(rng, n, (h + 2 * hk) * d).to(R.DT[xt])
    freq, factor = paged().rope_frequencies(64, scaling="linear", factor_len=4.0)
    freq = freq[:rotary // 2]
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], 1))
    qd, kd, vd = (t.unflatten(1, (-1, d)) for t in qkv.to(dev).split([h * d, hk * d, hk * d], 1))
    qo = torch.full((n, h, d), 7.0, dtype=R.DT[ct], device=dev)
    paged().rope_append(qd, kd, vd, i32(pos, dev), freq.to(dev), cache, i32(seqs, dev), i32(rows, dev), qo, factor=factor)
    live = [t for t in range(n) if 0 <= seqs[t] < 3]
    dead = [t for t in range(n) if t not in live]
    turn = lambda t: R.turned(t.double().numpy(), pos, freq.numpy(), rotary, False, factor)  # noqa: E731
    check_turned(qo[live], turn(q)[live], q[live], rotary, False, factor, ct)
    assert torch.equal(qo[dead].cpu(), torch.full((len(dead), h, d), 7.0, dtype=R.DT[ct]))
    wk = turn(k)
    touched = []
    for t in ok:
        p, r = int(pool.table[seqs[t], rows[t] // page]), rows[t] % page
        touched.append((p, r))
        check_turned(cache.k_pages[p, r][None], wk[t:t + 1], k[t:t + 1], rotary, False, factor, ct)
        assert torch.equal(cache.v_pages[p, r].cpu(), v[t].to(R.DT[ct]))
        before[0][p, r], before[1][p, r] = cache.k_pages[p, r], cache.v_pages[p, r]
    for a, b in zip(before, (cache.k_pages, cache.v_pages)):
        assert torch.equal(torch.nan_to_num(a.float(), 99.0), torch.nan_to_num(b.float(), 99.0))


def test_rope_many_rows_and_none(dev):
    freq, _ = paged().rope_frequencies(16)
    e = torch.empty(0, 2, 16, device=dev)
    paged().rope(e, None, i32([], dev), freq.to(dev), e, None)
    n = 70001
    x = torch.ones(n, 1, 16, device=dev)
    paged().rope(x, None, torch.arange(n, dtype=torch.int32, device=dev), freq.to(dev), x, None)
    want = R.turned(np.ones((3, 1, 16)), [0, 65536, 70000], freq.numpy(), 16, False, 1.0)
    R.close(x[[0, 65536, 70000]], want, np.full(want.shape, 2.0**-20))


def test_rope_more_rows_than_one_grid(dev):
    """Beyond 2^22 rows a workgroup takes several: the same results at both ends."""
    n = (1 << 22) + 300
    freq, _ = paged().rope_frequencies(8)
    x = torch.ones(n, 1, 8, dtype=torch.float16, device=dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    paged().rope(x, None, pos, freq.to(dev), x, None)
    rows = [0, 299, 300, 1 << 22, n - 1]
    want = R.turned(np.ones((len(rows), 1, 8)), rows, freq.numpy(), 8, False, 1.0)
    R.close(x[rows], want, R.HALF["f16"] * np.abs(want) + 2.0**-20)


# ---- attention of one new token ------------------------------------------------

def run_decode(dev, rng, pool, heads, out_dtype=None, seqs=None, spread=1.5, strided=False, **kw):
    """Decode over every sequence (or `seqs`) of the pool, checked against 64 bits."""
    cache = pool.cache()
    d = cache.head_dim
    rows = list(range(len(pool.lens))) if seqs is None else list(seqs)
    n = len(rows)
    out_dtype = out_dtype or pool.dtype
    wide = rand(rng, n, heads + 1, d + 8, std=spread).to(R.DT[pool.dtype])
    q = wide[:, 1:, :d] if strided else wide[:, 1:, :d].contiguous()
    qd = wide.to(dev)[:, 1:, :d] if strided else q.to(dev)
    out = torch.full((n, heads, d), 7.0, dtype=R.DT[out_dtype], device=dev)
    arg = dict(kw)
    host = {}
    for name in ("prefix_len", "key_begin", "key_end"):
        if arg.get(name) is not None:
            host[name] = list(arg[name])
            arg[name] = i32(arg[name], dev)
    if arg.get("slopes") is not None:
        arg["slopes"] = torch.tensor(arg["slopes"], dtype=torch.float32, device=dev)
    ws = paged().attention_workspace(cache, heads, n)
    paged().attention_decode(qd, cache, pool.kv_len, out, seqs=None if seqs is None else i32(seqs, dev), workspace=ws, **arg)
    for i, b in enumerate(rows):
        if not 0 <= b < len(pool.lens):
            assert (out[i].float() == 7.0).all()
            continue
        mask = dict(window=kw.get("window", 0), prefix=host["prefix_len"][b] if "prefix_len" in host else 0,
                    begin=host["key_begin"][i] if "key_begin" in host else 0,
                    end=host["key_end"][i] if "key_end" in host else None)
        want, bound = R.attend(q[i], pool.k[b], pool.v[b], pool.lens[b] - 1, out_dtype, pool.dtype, P_ERR[pool.dtype],
                               scale=kw.get("scale"), softcap=kw.get("softcap", 0.0), fast_cap=pool.dtype != "f32",
                               slopes=arg["slopes"].cpu().numpy() if arg.get("slopes") is not None else None, **mask)
        R.close(out[i], want, bound)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [
    (10, 10, 128, 16), (8, 2, 64, 32), (4, 1, 256, 24), (6, 2, 96, 1), (5, 5, 80, 7), (20, 1, 128, 64), (2, 1, 8, 16),
    (3, 3, 192, 256), (40, 2, 32, 8)])
def test_decode(dev, dtype, heads, kv_heads, d, page):
    print(f"[decode] {dtype} {heads}/{kv_heads}x{d} page {page}", flush=True)
    rng = np.random.default_rng(heads * d + page)
    pool = R.Pool(rng, [1, 2, 15, 16, 17, 31, 32, 33, 63, 127, 128, 129, 0, 300], kv_heads, d, page, dtype, dev)
    run_decode(dev, rng, pool, heads)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["hnd", "kv"])
def test_decode_layouts_and_types(dev, dtype, layout):
    rng = np.random.default_rng(3)
    pool = R.Pool(rng, [5, 200, 77], 2, 64, 16, dtype, dev, layout)
    run_decode(dev, rng, pool, 6, out_dtype="f32", strided=True)
    run_decode(dev, rng, pool, 6, strided=True, scale=0.3)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kw", [
    dict(window=1), dict(window=100), dict(window=5, prefix_len=[3, 40, 0, 700, 1]), dict(prefix_len=[1, 2, 3, 4, 5]),
    dict(window=40, prefix_len=[0, 33, 64, 31, 200]), dict(key_begin=[0, 10, 98, 300, 500]),
    dict(key_begin=[1, 0, 50, 10**9, -4], key_end=[1, 70, 20, 50, 2**31 - 1]),  # rows 0, 2, 3 see nothing
    dict(softcap=5.0), dict(slopes=[0.5, 0.01, 1.0, 0.0]), dict(softcap=30.0, slopes=[0.1, 0.2, 0.3, 2.0], window=64),
    dict(scale=-0.2), dict(softcap=0.01)])
def test_decode_masks(dev, dtype, kw):
    rng = np.random.default_rng(11)
    pool = R.Pool(rng, [1, 70, 99, 260, 515], 2, 128, 16, dtype, dev)
    run_decode(dev, rng, pool, 4, **kw)


@pytest.mark.parametrize("hint", [0, 1, 64, 3001, 10**9])
def test_decode_split(dev, hint):
    """One long sequence beside short ones: split and joined, whatever length the host expects."""
    rng = np.random.default_rng(17)
    pool = R.Pool(rng, [3001, 1, 0, 640], 1, 128, 16, "bf16", dev)
    a = run_decode(dev, rng, pool, 4, max_kv_len=hint)
    b = run_decode(dev, np.random.default_rng(17), R.Pool(np.random.default_rng(17), [3001, 1, 0, 640], 1, 128, 16, "bf16", dev),
                   4, max_kv_len=hint)
    assert a.shape == b.shape


def test_decode_split_f32_large_scores(dev):
    """Scores of some hundreds: one key takes it all, in whichever split it is."""
    rng = np.random.default_rng(23)
    pool = R.Pool(rng, [2500, 900], 2, 64, 32, "f32", dev, std=3.0)
    run_decode(dev, rng, pool, 2, spread=40.0)


@pytest.mark.parametrize("heads,kv_heads,d,lens,hint", [
    (4, 1, 64, [9000], 0), (32, 2, 128, [2500, 2500, 1, 0, 40], 2500), (3, 3, 96, [1200] * 9, 0), (16, 1, 256, [1500, 700], 0),
    (18, 1, 64, [800] * 40, 0), (2, 2, 128, [30] * 300, 2000),
    (1, 1, 64, [700] + [9] * 1100, 0)])
def test_decode_shares(dev, heads, kv_heads, d, lens, hint):
    """Many shares of one sequence (joined by a kernel of its own), a few of each, several sequences in one; on one
    workspace in turn, so that each call leaves it as the next needs it."""
    rng = np.random.default_rng(len(lens))
    pool = R.Pool(rng, lens, kv_heads, d, 16, "bf16", dev)
    first = run_decode(dev, np.random.default_rng(1), pool, heads, max_kv_len=hint)
    cache = pool.cache()
    ws = paged().attention_workspace(cache, heads, len(lens))
    q = rand(np.random.default_rng(1), len(lens), heads + 1, d + 8, std=1.5).to(torch.bfloat16)[:, 1:, :d].contiguous().to(dev)
    for _ in range(4):
        out = torch.zeros_like(q)
        paged().attention_decode(q, cache, pool.kv_len, out, max_kv_len=hint, workspace=ws)
        assert torch.equal(out, first)
        few = torch.zeros_like(q[:1])
        paged().attention_decode(q[:1], cache, pool.kv_len, few, max_kv_len=0, workspace=ws)
        assert torch.isfinite(few).all()


def test_decode_workspace_that_was_not_set_up(dev):
    """NaN, not something that looks like a result."""
    rng = np.random.default_rng(3)
    pool = R.Pool(rng, [2000, 700], 1, 64, 16, "bf16", dev)
    cache = pool.cache()
    q = rand(rng, 2, 2, 64).to(torch.bfloat16).to(dev)
    out = torch.zeros_like(q)
    ws = torch.zeros_like(paged().attention_workspace(cache, 2, 2))
    paged().attention_decode(q, cache, pool.kv_len, out, workspace=ws)
    assert torch.isnan(out).all()


def test_decode_padding_and_order(dev):
    rng = np.random.default_rng(29)
    pool = R.Pool(rng, [40, 90, 10], 2, 64, 16, "bf16", dev)
    run_decode(dev, rng, pool, 4, seqs=[2, -1, 0, 3, 2, 1, 2**31 - 1])  # (the same sequence twice)


def test_decode_equal_calls_equal_bits(dev):
    rng = np.random.default_rng(31)
    pool = R.Pool(rng, [2000, 5, 333], 2, 128, 16, "bf16", dev)
    a = run_decode(dev, np.random.default_rng(1), pool, 8)
    b = run_decode(dev, np.random.default_rng(1), pool, 8)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_values_that_are_not_finite(dev, dtype):
    """What a row does not see changes nothing; what it sees and is not finite shows."""
    rng = np.random.default_rng(37)
    pool = R.Pool(rng, [100, 100, 300], 1, 64, 16, dtype, dev)
    for j in (0, 17, 49):
        pool.poison(0, j)
        pool.poison(2, j)
    run_decode(dev, rng, pool, 2, window=50, prefix_len=[0, 10, 0])
    cache = pool.cache()
    q = rand(rng, 3, 2, 64).to(R.DT[dtype]).to(dev)
    out = torch.empty_like(q)
    ws = paged().attention_workspace(cache, 2, 3)
    p, r = int(pool.table[1, 2]), 3
    pool.v_pages[p, r, 0, 5] = float("inf")
    pool.v_pages[p, r, 0, 6] = float("-inf")
    pool.v_pages[p, r, 0, 7] = float("nan")
    paged().attention_decode(q, cache, pool.kv_len, out, workspace=ws)
    assert torch.isnan(out[0]).all() and torch.isnan(out[2]).all()
    o = out[1].float().cpu()
    assert (o[:, 5] == float("inf")).all() and (o[:, 6] == float("-inf")).all() and torch.isnan(o[:, 7]).all()
    assert torch.isfinite(o[:, :5]).all() and torch.isfinite(o[:, 8:]).all()


def test_decode_bad_pages_and_lengths(dev):
    """A seen key without a page, or more keys than the table has room for: NaN, there alone."""
    rng = np.random.default_rng(41)
    pool = R.Pool(rng, [100, 100, 100, 64], 1, 64, 16, "bf16", dev, extra_cols=0)
    for bad in (-1, pool.k_pages.shape[0], -2**31):
        pool.table[0, 3] = bad
        pool.kv_len[:] = i32([100, 100, 7 * 16 + 1, 2**31 - 1], dev)
        cache = pool.cache()
        q = rand(rng, 4, 2, 64).to(torch.bfloat16).to(dev)
        out = torch.empty_like(q)
        paged().attention_decode(q, cache, pool.kv_len, out, workspace=paged().attention_workspace(cache, 2, 4))
        assert torch.isnan(out[[0, 2, 3]]).all() and torch.isfinite(out[1]).all()
    # a window that does not reach the page: not read
    pool.kv_len[:] = i32([100, 100, 100, 64], dev)
    run_decode(dev, rng, pool, 2, window=30)
    pool.kv_len[:] = i32([-3, 0, -2**31, 1], dev)
    out.fill_(5.0)
    paged().attention_decode(q, cache, pool.kv_len, out, workspace=paged().attention_workspace(cache, 2, 4))
    assert (out[:3] == 0).all() and torch.isfinite(out[3]).all()


def test_decode_far_offsets(dev):
    """Pages beyond 4 GiB of one another: offsets pass 32 bits."""
    rng = np.random.default_rng(43)
    small = R.Pool(rng, [70, 33], 1, 64, 16, "bf16", dev)
    n = small.k_pages.shape[0]
    far = 340000  # rows of 64 x 16 bf16 values between pages: 700 MB
    big = torch.empty(2, (n - 1) * far + 1, 16, 1, 64, dtype=torch.bfloat16, device=dev)
    assert big[0].numel() * 2 > 2**32
    for p in range(n):
        big[0, p * far], big[1, p * far] = small.k_pages[p], small.v_pages[p]
    small.k_pages, small.v_pages = big[0, ::far], big[1, ::far]
    run_decode(dev, rng, small, 4)


def test_decode_captured(dev):
    """A captured call follows the device's lengths and pages; eager calls run between its replays."""
    rng = np.random.default_rng(47)
    pool = R.Pool(rng, [900, 40, 333], 2, 64, 16, "bf16", dev)
    cache = pool.cache()
    q = rand(rng, 3, 4, 64).to(torch.bfloat16).to(dev)
    out, eager = torch.empty_like(q), torch.empty_like(q)
    ws, ws2 = (paged().attention_workspace(cache, 4, 3) for _ in range(2))
    kv = pool.kv_len.clone()
    call = lambda o, w: paged().attention_decode(q, cache, kv, o, workspace=w)  # noqa: E731
    call(out, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out, ws)
    for lens in ([900, 40, 333], [1, 0, 333], [500, 39, 2], [899, 40, 64]):
        kv.copy_(i32(lens, dev))
        out.fill_(9.0)
        g.replay()
        call(eager, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens


def test_decode_on_another_stream(dev):
    rng = np.random.default_rng(53)
    pool = R.Pool(rng, [600, 40], 2, 64, 16, "bf16", dev)
    cache = pool.cache()
    q = rand(rng, 2, 4, 64).to(torch.bfloat16).to(dev)
    a, b = torch.empty_like(q), torch.empty_like(q)
    ws = paged().attention_workspace(cache, 4, 2)
    paged().attention_decode(q, cache, pool.kv_len, a, workspace=ws)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    paged().attention_decode(q, cache, pool.kv_len, b, workspace=ws, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(a, b)
    with torch.cuda.stream(s):
        b.zero_()
        paged().attention_decode(q, cache, pool.kv_len, b, workspace=ws)
    s.synchronize()
    assert torch.equal(a, b)
    paged().attention_decode(q, cache, pool.kv_len, q, workspace=ws)  # out may be q
    assert torch.equal(q, a)
