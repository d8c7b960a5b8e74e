"""Plain 64-bit implementations of the paged attention and rotary operators, and bounds on
what rounding may change, for the tests.

Bound of an attention output against 64 bits, per element:
  half a step of the output's type, plus
  (2 d + e) * sum p |v|, where
    d  the largest error of a score: a chain of head_dim products and sums in f32 gives at most
       (head_dim + 8) 2^-24 sum |q k| scale, the cap, bias and change of base 6 roundings of 2^-23 |terms|
       (twice: it enters the weights and their sum), and 2^-20 absolute where the cap runs on the
       fast exponential (16-bit prefill: 2^-22 of the cap);
    e  the rounding of the weights (half a step of their type; 2^-15 where they are held in two
       halves of bf16, 2^-20 of f16, f32: 0) and 2^-18 for the sums over keys, the exponentials and the joins.
"""
import numpy as np
import torch

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}
TINY = {"f32": 2.0**-149, "bf16": 2.0**-134, "f16": 2.0**-25}  # half a step of the smallest values


class Pool:
    """Sequences' K and V rows in 64 bits, and the paged cache that holds them: pages in
    random order, everything that belongs to no row NaN, unused table entries out of range."""

    def __init__(self, rng, lens, kv_heads, head_dim, page, dtype, dev, layout="nhd", extra_cols=2, std=1.0):
        self.lens, self.page, self.dev, self.dtype = list(lens), page, dev, dtype
        dt = DT[dtype]
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + 2
        order = rng.permutation(n_pages)
        cols = max(need + [0]) + extra_cols
        table = rng.choice([-1, -7, n_pages, 2**31 - 1], size=(len(lens), cols)).astype(np.int32)
        k = torch.full((n_pages, page, kv_heads, head_dim), float("nan"), dtype=dt)
        v = k.clone()
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(lens):
            kb, vb = (torch.from_numpy(rng.standard_normal((n, kv_heads, head_dim)).astype(np.float32) * std).to(dt)
                      for _ in range(2))
            self.k.append(kb)
            self.v.append(vb)
            for j in range(need[b]):
                p = int(order[at])
                at += 1
                table[b, j] = p
                rows = min(page, n - j * page)
                k[p, :rows] = kb[j * page:j * page + rows]
                v[p, :rows] = vb[j * page:j * page + rows]
        if layout == "nhd":
            self.k_pages, self.v_pages = k.to(dev), v.to(dev)
        elif layout == "hnd":  # heads outside the rows of a page
            self.k_pages, self.v_pages = (x.permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3) for x in (k, v))
        else:  # "kv": K and V of a page side by side
            kv = torch.stack((k, v), 1).to(dev)
            self.k_pages, self.v_pages = kv[:, 0], kv[:, 1]
        self.table = torch.from_numpy(table).to(dev)
        self.kv_len = torch.tensor(lens, dtype=torch.int32, device=dev)

    def cache(self):
        from uocr_hip import paged
        return paged.PagedKVCache(self.k_pages, self.v_pages, self.table)

    def poison(self, b, j):
        """Row j of sequence b becomes NaN in the cache (not in .k / .v)."""
        p = int(self.table[b, j // self.page])
        self.k_pages[p, j % self.page] = float("nan")
        self.v_pages[p, j % self.page] = float("inf")


def visible(pos, n, causal=True, window=0, prefix=0, both_ways=False, begin=0, end=None):
    j = np.arange(n)
    seen = (j <= pos) if causal else np.ones(n, bool)
    if window:
        seen &= j > pos - window
    seen |= (j < prefix) & (np.ones(n, bool) if both_ways or not causal else j <= pos)
    seen &= j >= begin
    if end is not None:
        seen &= j < end
    return np.nonzero(seen)[0]


def attend(q, k, v, pos, out_dtype, dtype, p_err, scale=None, softcap=0.0, slopes=None, fast_cap=False, **mask):
    """One row: q [heads, d], k / v [n, kv_heads, d] (tensors) -> (out, bound) f64 [heads, d]."""
    q = q.double().numpy()
    h, d = q.shape
    hk = k.shape[1]
    scale = scale or 1.0 / np.sqrt(np.float64(d))
    seen = visible(pos, k.shape[0], **mask)
    out, bound = np.zeros((h, d)), np.zeros((h, d))
    if len(seen) == 0:
        return out, bound
    ks, vs = k[seen].double().numpy(), v[seen].double().numpy()
    for i in range(h):
        kk, vv = ks[:, i // (h // hk)], vs[:, i // (h // hk)]
        s = kk @ q[i] * scale
        err = (d + 8) * 2.0**-24 * (np.abs(kk) @ np.abs(q[i])) * abs(scale)
        if softcap:
            s = softcap * np.tanh(s / softcap)
            err = err + 4 * 2.0**-23 * np.abs(s) + (softcap * 2.0**-22 if fast_cap else 0.0)
        if slopes is not None:
            b = float(slopes[i]) * np.abs(pos - seen)
            s = s - b
            err = err + 2 * 2.0**-23 * b
        err = err + 6 * 2.0**-23 * np.abs(s) + 2 * 2.0**-23 * np.abs(s - s.max())
        w = np.exp(s - s.max())
        w /= w.sum()
        out[i] = w @ vv
        # (a score's error moves its own weight; the sum of the weights by their mean)
        bound[i] = (w * np.expm1(err)) @ np.abs(vv) + (w @ np.expm1(err)) * np.abs(out[i])
        bound[i] += (p_err + 2.0**-18) * (w @ np.abs(vv))
    return out, bound + HALF[out_dtype] * (np.abs(out) + bound) + TINY[out_dtype]


def close(got, want, bound):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4], bound[bad][:4])


def turned(x, positions, freq, rotary, interleaved, factor):
    """Rotary positions in 64 bits: x [rows, heads, d] f64 numpy."""
    y = x.copy()
    if rotary:
        z = factor * np.exp(1j * np.asarray(positions, np.float64)[:, None] * np.asarray(freq, np.float64)[None])[:, None]
        a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
        w = (x[..., a] + 1j * x[..., b]) * z
        y[..., a], y[..., b] = w.real, w.imag
    return y
