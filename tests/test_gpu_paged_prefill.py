"""Attention of many query rows over a paged cache against the plain implementation in 64
bits, row by row and head by head. Tolerances: see paged_ref.py."""
import numpy as np
import pytest
import torch

import paged_ref as R
from test_gpu_paged import i32, paged, rand

pytestmark = pytest.mark.gpu
# weights of the prefill kernel: rounded to the type
P_ERR = {"f32": 0.0, "bf16": 2.0**-8, "f16": 2.0**-11}


def run_prefill(dev, rng, pool, q_rows, heads, out_dtype=None, seqs=None, spread=1.5, strided=False, behind=3, check=None,
                q_start=None, **kw):
    """q_rows[b] rows of each entry (and `behind` rows of none), checked row by row."""
    cache = pool.cache()
    d, n = cache.head_dim, sum(q_rows) + behind
    out_dtype = out_dtype or pool.dtype
    wide = rand(rng, n, heads + 1, d + 8, std=spread).to(R.DT[pool.dtype])
    q = wide[:, 1:, :d]
    qd = wide.to(dev)[:, 1:, :d] if strided else q.contiguous().to(dev)
    if strided:
        out = torch.full((n, heads + 2, d), 7.0, dtype=R.DT[out_dtype], device=dev)[:, :heads]
    else:
        out = torch.full((n, heads, d), 7.0, dtype=R.DT[out_dtype], device=dev)
    starts = np.concatenate([[0], np.cumsum(q_rows)])
    arg, host = dict(kw), {}
    for name in ("prefix_len", "key_begin", "key_end"):
        if arg.get(name) is not None:
            host[name] = list(arg[name])
            arg[name] = i32(list(arg[name]) + ([0] * behind if name != "prefix_len" else []), dev)
    if arg.get("slopes") is not None:
        arg["slopes"] = torch.tensor(arg["slopes"], dtype=torch.float32, device=dev)
    ws = paged().attention_workspace(cache, heads, n)
    paged().attention_prefill(qd, cache, i32(starts, dev), pool.kv_len, out, seqs=None if seqs is None else i32(seqs, dev),
                              workspace=ws, **arg)
    res = out.cpu()
    assert (res[starts[-1]:].float() == 7.0).all()
    for b in range(len(q_rows)):
        s = b if seqs is None else seqs[b]
        if not 0 <= s < len(pool.lens):
            assert (res[starts[b]:starts[b + 1]].float() == 7.0).all()
            continue
        for i in range(q_rows[b]):
            t = starts[b] + i
            if check is not None and t not in check:
                continue
            mask = dict(causal=kw.get("causal", True), window=kw.get("window", 0), both_ways=kw.get("prefix_both_ways", False),
                        prefix=host["prefix_len"][s] if "prefix_len" in host else 0,
                        begin=host["key_begin"][t] if "key_begin" in host else 0,
                        end=host["key_end"][t] if "key_end" in host else None)
            want, bound = R.attend(q[t], pool.k[s], pool.v[s], pool.lens[s] - q_rows[b] + i, out_dtype, pool.dtype,
                                   P_ERR[pool.dtype], scale=kw.get("scale"), softcap=kw.get("softcap", 0.0), fast_cap=True,
                                   slopes=arg["slopes"].cpu().numpy() if arg.get("slopes") is not None else None, **mask)
            R.close(res[t], want, bound)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,d,page", [
    (10, 10, 128, 16), (8, 2, 64, 32), (4, 1, 256, 24), (6, 2, 96, 1), (5, 5, 80, 7), (20, 1, 128, 64), (2, 1, 8, 16),
    (3, 3, 192, 256), (14, 2, 32, 8)])
def test_prefill(dev, dtype, heads, kv_heads, d, page):
    print(f"[prefill] {dtype} {heads}/{kv_heads}x{d} page {page}", flush=True)
    rng = np.random.default_rng(heads * d + page)
    lens, q = [1, 33, 64, 65, 200, 0, 50, 129], [1, 33, 60, 2, 70, 0, 0, 129]
    pool = R.Pool(rng, lens, kv_heads, d, page, dtype, dev)
    run_prefill(dev, rng, pool, q, heads)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["hnd", "kv"])
def test_prefill_layouts_and_types(dev, dtype, layout):
    rng = np.random.default_rng(3)
    pool = R.Pool(rng, [5, 150, 77], 2, 64, 16, dtype, dev, layout)
    run_prefill(dev, rng, pool, [5, 40, 77], 6, out_dtype="f32", strided=True)
    run_prefill(dev, rng, pool, [2, 150, 1], 6, strided=True, scale=0.3)


MASKS = [
    dict(window=1), dict(window=50), dict(window=5, prefix_len=[3, 40, 300]), dict(prefix_len=[7, 31, 64]),
    dict(window=20, prefix_len=[1, 90, 129], prefix_both_ways=True), dict(prefix_len=[9, 100, 500], prefix_both_ways=True),
    dict(causal=False), dict(causal=False, docs=24), dict(docs=24), dict(docs=50, softcap=5.0), dict(softcap=0.01),
    dict(slopes=[0.5, 0.01, 1.0, 0.0]), dict(softcap=30.0, slopes=[0.1, 0.2, 0.3, 2.0], window=64, prefix_len=[0, 70, 64],
                                             prefix_both_ways=True),
    dict(causal=False, slopes=[0.3, 0.2, 0.1, 0.05]), dict(scale=-0.2), dict(none=True)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", range(len(MASKS)))
def test_prefill_masks(dev, dtype, case):
    kw = dict(MASKS[case])
    rng = np.random.default_rng(case)
    lens, q = [9, 170, 131], [9, 100, 131]
    pool = R.Pool(rng, lens, 2, 128, 16, dtype, dev)
    pos = [n - r + i for n, r in zip(lens, q) for i in range(r)]
    doc = kw.pop("docs", 0)
    if doc:
        kw["key_begin"] = [p // doc * doc for p in pos]
        if not kw.get("causal", True):
            kw["key_end"] = [p // doc * doc + doc for p in pos]
    if kw.pop("none", False):  # some rows see nothing, others one key
        kw["key_begin"] = [p + 1 - p % 2 if p % 3 else 10**9 for p in pos]
        kw["key_end"] = [p + 1 for p in pos]
    run_prefill(dev, rng, pool, q, 4, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefill_more_rows_than_keys(dev, dtype):
    """Rows before position 0 see nothing under the causal mask; all keys without it."""
    rng = np.random.default_rng(2)
    pool = R.Pool(rng, [5, 0, 40], 1, 64, 16, dtype, dev)
    run_prefill(dev, rng, pool, [9, 3, 41], 2)
    run_prefill(dev, rng, pool, [9, 3, 41], 2, causal=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 4, 1), (3, 8, 2), (17, 2, 1), (130, 4, 2)])
def test_prefill_few_rows_on_a_long_cache(dev, dtype, rows, heads, kv_heads):
    """Split over the keys and joined."""
    rng = np.random.default_rng(rows)
    pool = R.Pool(rng, [2100, 700], kv_heads, 64, 16, dtype, dev)
    check = {0, 1, rows - 1, rows, rows + rows // 2}
    for hint in (0, 2100, 1):
        run_prefill(dev, rng, pool, [rows, max(1, rows // 2)], heads, check=check, max_kv_len=hint)
    run_prefill(dev, rng, pool, [rows, max(1, rows // 2)], heads, check=check, window=300, prefix_len=[500, 100])


@pytest.mark.parametrize("dtype,rows,heads,kv_heads,d", [
    ("bf16", 900, 72, 72, 64), ("f16", 1030, 130, 65, 32), ("f32", 2050, 66, 66, 32), ("bf16", 300, 12, 3, 200), ("f32", 300, 4, 2, 256)])
@pytest.mark.parametrize("kw", [dict(), dict(window=200, prefix_len=[100, 40]), dict(docs=130, softcap=8.0), dict(causal=False)])
def test_prefill_whole_chip(dev, dtype, rows, heads, kv_heads, d, kw):
    """Enough workgroups of 128 (row, head) pairs for the chip, and heads above 128: over many tiles of keys."""
    kw = dict(kw)
    rng = np.random.default_rng(rows)
    lens, q = [rows + 70, 150], [rows, 150]
    pool = R.Pool(rng, lens, kv_heads, d // 8 * 8, 16, dtype, dev)
    doc = kw.pop("docs", 0)
    if doc:
        kw["key_begin"] = [p // doc * doc for n, r in zip(lens, q) for p in range(n - r, n)]
    run_prefill(dev, rng, pool, q, heads, check={0, 1, 63, 127, 128, rows // 2, rows - 1, rows, rows + 149}, **kw)


def test_prefill_sequences_by_slot(dev):
    rng = np.random.default_rng(7)
    pool = R.Pool(rng, [40, 90, 10], 2, 64, 16, "bf16", dev)
    run_prefill(dev, rng, pool, [10, 5, 33, 4, 20], 4, seqs=[2, -1, 0, 3, 1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefill_values_that_are_not_finite(dev, dtype):
    """Rows that do not see a key with NaN or infinities keep their results; those that do show it."""
    rng = np.random.default_rng(9)
    pool = R.Pool(rng, [100, 150], 2, 64, 16, dtype, dev)
    q = rand(rng, 250, 4, 64, std=1.5).to(R.DT[dtype])
    begin = [p // 40 * 40 for n in (100, 150) for p in range(n)]
    clean, dirty = (torch.zeros(250, 4, 64, dtype=R.DT[dtype], device=dev) for _ in range(2))
    for out in (clean, dirty):
        cache = pool.cache()
        paged().attention_prefill(q.to(dev), cache, i32([0, 100, 250], dev), pool.kv_len, out, key_begin=i32(begin, dev),
                                  workspace=paged().attention_workspace(cache, 4, 250))
        pool.poison(0, 50)  # document 1 of sequence 0: rows 50..79 see it
        pool.poison(1, 149)
    sees = list(range(50, 80)) + [249]
    rest = [t for t in range(250) if t not in sees]
    assert torch.isnan(dirty[sees]).all() and torch.isfinite(dirty[rest]).all()
    for t in rest[::7] + [49, 80, 248]:
        s, p = (0, t) if t < 100 else (1, t - 100)
        want, bound = R.attend(q[t], pool.k[s], pool.v[s], p, dtype, dtype, P_ERR[dtype], begin=begin[t])
        R.close(dirty[t], want, bound)
    # an infinite value in V: infinite where it is seen
    pool = R.Pool(np.random.default_rng(9), [100, 150], 2, 64, 16, dtype, dev)
    pool.v_pages[int(pool.table[0, 2]), 5, 1, 3] = float("inf")  # row 37
    cache = pool.cache()
    paged().attention_prefill(q.to(dev), cache, i32([0, 100, 250], dev), pool.kv_len, dirty, key_begin=i32(begin, dev),
                              workspace=paged().attention_workspace(cache, 4, 250))
    assert (dirty[37:40, 2:, 3].float() == float("inf")).all()
    dirty[37:40, 2:, 3] = clean[37:40, 2:, 3]
    assert torch.isfinite(dirty).all()
    tol = {"bf16": 3 * 2.0**-7, "f32": 1e-5}[dtype]  # (those rows may take another order of sums)
    assert ((dirty.float() - clean.float()).abs() <= tol * (1 + clean.float().abs())).all()


def test_prefill_bad_pages_and_lengths(dev):
    rng = np.random.default_rng(13)
    pool = R.Pool(rng, [100, 100, 100, 30], 1, 64, 16, "bf16", dev, extra_cols=0)
    pool.table[0, 3] = -1  # rows 48..63 of sequence 0
    pool.kv_len[:] = i32([100, 100, 113, -5], dev)
    cache = pool.cache()
    q = rand(rng, 170, 2, 64).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, 7.0)
    starts = i32([0, 100, 140, 160, 165], dev)
    paged().attention_prefill(q, cache, starts, pool.kv_len, out, workspace=paged().attention_workspace(cache, 2, 170))
    assert torch.isfinite(out[:48]).all() and torch.isnan(out[48:100]).all()
    assert torch.isfinite(out[100:140]).all() and torch.isnan(out[140:160]).all()
    assert (out[160:165] == 0).all() and (out[165:] == 7.0).all()


def test_prefill_captured_and_on_another_stream(dev):
    rng = np.random.default_rng(15)
    pool = R.Pool(rng, [900, 40, 333], 2, 64, 16, "bf16", dev)
    cache = pool.cache()
    q = rand(rng, 60, 4, 64).to(torch.bfloat16).to(dev)
    out, eager = torch.zeros_like(q), torch.zeros_like(q)
    ws, ws2 = (paged().attention_workspace(cache, 4, 60) for _ in range(2))
    kv, starts = pool.kv_len.clone(), i32([0, 20, 40, 60], dev)
    call = lambda o, w: paged().attention_prefill(q, cache, starts, kv, o, workspace=w)  # noqa: E731
    call(out, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out, ws)
    for lens, at in (([900, 40, 333], [0, 20, 40, 60]), ([30, 0, 333], [0, 1, 2, 60]), ([500, 39, 2], [0, 50, 58, 60])):
        kv.copy_(i32(lens, dev))
        starts.copy_(i32(at, dev))
        out.fill_(9.0)
        g.replay()
        call(eager, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens
    s = torch.cuda.Stream()
    out.zero_()
    torch.cuda.synchronize()
    paged().attention_prefill(q, cache, starts, kv, out, workspace=ws, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, eager)
    paged().attention_prefill(q, cache, starts, kv, q, workspace=ws)  # out may be q
    assert torch.equal(q, eager)


@pytest.mark.parametrize("dtype,rows,heads,d", [("bf16", 1, 1, 64), ("f32", 3, 2, 40), ("bf16", 2, 2, 256)])
def test_prefill_many_splits(dev, dtype, rows, heads, d):
    """Few rows over tens of thousands of keys: more splits than a wave has lanes, some of them without a key
    that the row sees; values that are not finite in hidden places, and an infinite one that all see."""
    print(f"[prefill splits] {dtype} {rows}x{heads}x{d}", flush=True)
    n, rng = 120001 if d <= 64 else 33001, np.random.default_rng(d)
    pool = R.Pool(rng, [n, 20], 1, d, 64, dtype, dev)
    q = [rows, rows]
    run_prefill(dev, rng, pool, q, heads)
    run_prefill(dev, rng, pool, q, heads, window=700, prefix_len=[130, 4])
    run_prefill(dev, rng, pool, q, heads, key_begin=[20000] * rows + [30] * rows, softcap=20.0)  # (the second sees nothing)
    pool.poison(0, 19999)
    pool.table[0, 3] = -1
    run_prefill(dev, rng, pool, q, heads, key_begin=[20000] * rows + [5] * rows)
    pool.v_pages[int(pool.table[0, 400]), 0, 0, 1] = float("inf")
    cache = pool.cache()
    qd = rand(rng, 2 * rows, heads, d).to(R.DT[dtype]).to(dev)
    out = torch.zeros_like(qd)
    paged().attention_prefill(qd, cache, i32([0, rows, 2 * rows], dev), pool.kv_len, out, key_begin=i32([20000] * 2 * rows, dev),
                              workspace=paged().attention_workspace(cache, heads, 2 * rows))
    assert (out[:rows, :, 1].float() == float("inf")).all() and (out[rows:] == 0).all()
    out[:rows, :, 1] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype,heads,kv_heads,d", [("bf16", 2, 1, 256), ("f32", 1, 1, 136), ("bf16", 6, 3, 64)])
def test_prefill_splits_of_a_full_chip(dev, dtype, heads, kv_heads, d):
    """More entries than the chip takes at once, three of them long: split in rounds, most splits empty."""
    print(f"[prefill full] {dtype} {heads}/{kv_heads}x{d}", flush=True)
    rng = np.random.default_rng(heads + d)
    lens = [int(x) for x in rng.integers(0, 40, 270)]
    for b, n in ((0, 6000), (130, 5003), (269, 6000)):
        lens[b] = n
    q = [1 + b % 3 for b in range(270)]
    at = np.concatenate([[0], np.cumsum(q)])
    pool = R.Pool(rng, lens, kv_heads, d, 16, dtype, dev)
    check = {int(at[b]) + i for b in (0, 1, 2, 64, 129, 130, 131, 200, 268, 269) for i in range(q[b])}
    for kw in (dict(), dict(window=3000), dict(causal=False)):
        run_prefill(dev, rng, pool, q, heads, check=check, max_kv_len=6000, **kw)


def test_prefill_split_captured(dev):
    """A captured call that splits its keys, replayed between others on the same workspace and with other lengths."""
    rng = np.random.default_rng(3)
    pool = R.Pool(rng, [5000, 4000], 2, 64, 16, "bf16", dev)
    cache = pool.cache()
    q = rand(rng, 12, 4, 64, std=1.5).to(torch.bfloat16).to(dev)
    start, out, ws = i32([0, 5, 12], dev), torch.zeros_like(q), paged().attention_workspace(cache, 4, 12)

    def call(o):
        paged().attention_prefill(q, cache, start, pool.kv_len, o, max_kv_len=5000, workspace=ws)

    call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for lens in ([5000, 4000], [9, 3999], [5, 7], [4999, 0], [5000, 4000]):
        pool.kv_len.copy_(i32(lens, dev))
        want = torch.zeros_like(q)
        call(want)
        paged().attention_decode(q[:2], cache, pool.kv_len, torch.zeros_like(q[:2]), max_kv_len=5000, workspace=ws)
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
