"""The attention half of a decoder layer on a paged key-value cache.

Three families, each through a public entry point of ``uocr_hip.paged``:

* ``rope``     rotary positions of q and k, alone or together with the append of
               K and V into the cache's pages.
* ``decode``   attention of one new token per sequence over its pages.
* ``prefill``  attention of many rows per sequence (a prompt, or a chunk of one).

``own`` chooses between the framework's calls and the plain form in torch.
Lengths are a function of the case alone, so that ``work`` knows them; contents,
page order and positions come from the seed.
"""
import math
import os
import sys
import types

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _paged():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unlimited-ocr.cpp_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    from uocr_hip import paged
    return paged


# ---- cases ------------------------------------------------------------------

def _rope(name, **kw):
    c = dict(name=name, kind="rope", seqs=1, tokens=16, context=0, heads=10, kv_heads=10, head_dim=128, rotary=128,
             interleaved=False, scaling="none", x="bf16", cache="bf16", page=16)
    c.update(kw)
    return c


def _decode(name, **kw):
    c = dict(name=name, kind="decode", batch=1, shortest=1, longest=700, heads=10, kv_heads=10, head_dim=128,
             dtype="bf16", page=16, softcap=0.0, bias=False, window=0, prefix=0, docs=False)
    c.update(kw)
    return c


def _prefill(name, **kw):
    c = dict(name=name, kind="prefill", batch=1, rows=283, context=0, heads=10, kv_heads=10, head_dim=128,
             dtype="bf16", page=16, softcap=0.0, bias=False, window=0, prefix=0, both_ways=False, doc=0)
    c.update(kw)
    return c


def listed():
    return [
        # 16 requests, each appending its new token: f32 activations into a bf16
        # cache, the decoder's 10 heads of 128; latency counts
        _rope("rope_append_decode_16", seqs=16, tokens=16, context=1100, x="f32"),
        # two long prompts, grouped heads, frequencies scaled for a long context
        _rope("rope_append_prompt_8192", seqs=2, tokens=8192, context=100000, heads=32, kv_heads=8, scaling="parts",
              page=64),
        # rotation alone, no cache: f32, pairs side by side, two thirds of the
        # head, far positions
        _rope("rope_f32_part_1111", seqs=3, tokens=1111, context=900000, heads=12, kv_heads=4, head_dim=96, rotary=64,
              interleaved=True, scaling="linear", x="f32", cache="none"),
        # one request decoding a page: the smallest attention call
        _decode("decode_1", longest=700),
        # 16 requests in the reference's scheme: the prompt's rows and a window
        # of 128 decoded ones, f32 as the contiguous cache has it
        _decode("decode_16_rswa", batch=16, shortest=600, longest=4000, dtype="f32", window=128, prefix=1000),
        # a large batch with grouped heads and very different lengths
        _decode("decode_64_grouped", batch=64, shortest=500, longest=8192, heads=32, kv_heads=8, page=64),
        # one sequence with a very long cache
        _decode("decode_1_long", longest=262144, shortest=262144, heads=32, kv_heads=8, dtype="f16", page=256),
        # capped scores and a distance bias, narrow heads, odd pages and lengths
        _decode("decode_33_capped", batch=33, longest=5001, heads=16, kv_heads=2, head_dim=64, page=24, softcap=30.0,
                bias=True),
        # one page's prompt: the 273 visual tokens and a few words
        _prefill("prefill_283"),
        # four ragged prompts of packed documents in f32
        _prefill("prefill_4_docs_f32", batch=4, rows=1000, dtype="f32", doc=300),
        # a long prompt, grouped heads: the largest call
        _prefill("prefill_8192", rows=8192, heads=32, kv_heads=8, page=64),
        # chunks of prompts on cached context: capped scores, a sliding window
        # beside a prefix that sees itself both ways, wide heads
        _prefill("prefill_3_chunks", batch=3, rows=700, context=20000, heads=16, kv_heads=4, head_dim=256, dtype="f16",
                 page=48, softcap=50.0, window=4096, prefix=1500, both_ways=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    kind = rng.choice(["rope", "decode", "decode", "prefill", "prefill"])
    heads, kv_heads = rng.choice([(10, 10), (32, 8), (16, 2), (12, 4), (7, 1), (24, 24), (40, 8), (20, 1)])
    head_dim = rng.choice([64, 128, 128, 96, 256, 80, 32, 192])
    page = rng.choice([16, 16, 32, 64, 256, 8, 24, 48, 1])
    if kind == "rope":
        rotary = rng.choice([head_dim, head_dim, head_dim // 2, 16])
        x = rng.choice(["f32", "bf16", "f16"])
        tokens = _log(rng, 1, 8000)
        return _rope("", seqs=rng.randint(1, min(16, tokens)), tokens=tokens, context=_log(rng, 1, 1000000),
                     heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary,
                     interleaved=rng.random() < 0.4, scaling=rng.choice(["none", "linear", "parts"]), x=x,
                     cache=rng.choice(["none", "bf16", "f16", "f32"]), page=page)
    mods = dict(softcap=rng.choice([0.0, 0.0, 30.0, 5.0]), bias=rng.random() < 0.3,
                window=rng.choice([0, 0, _log(rng, 1, 4096)]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "decode":
        batch = _log(rng, 1, 128)
        most = 5e8 / (batch * kv_heads * head_dim * 2 * SIZE[dtype])
        longest = _log(rng, 1, max(2, min(200000, int(most))))
        return _decode("", batch=batch, shortest=_log(rng, 1, max(1, longest)), longest=longest, heads=heads,
                       kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, page=page,
                       prefix=rng.choice([0, _log(rng, 1, longest)]), docs=rng.random() < 0.2, **mods)
    batch = rng.choice([1, 1, 2, 3, 5, 8])
    rows = _log(rng, 2, 4000 if dtype != "f32" else 1500)
    room = 1.0e9 * min(1.0, 128 / head_dim) / (batch * heads * rows)
    context = 0 if rng.random() < 0.4 else _log(rng, 1, 30000)
    room = min(room, 5e8 / (batch * kv_heads * head_dim * SIZE[dtype]))  # a cache of a GB at most
    context = int(min(context, max(0, room - rows)))
    if batch * heads * rows * (rows + context) > 2.0e9:
        batch = 1
    return _prefill("", batch=batch, rows=rows, context=context, heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, dtype=dtype, page=page, prefix=rng.choice([0, _log(rng, 1, rows + context)]),
                    both_ways=rng.random() < 0.5, doc=rng.choice([0, 0, _log(rng, 1, rows)]), **mods)


# ---- lengths, from the case alone --------------------------------------------

def _spread(lo, hi, n):
    """n whole numbers in [lo, hi], the first hi, the others spread evenly but out of order."""
    return [hi] + [lo + int((hi - lo + 1) * ((i * 0.6180339887) % 1.0)) for i in range(1, n)]


def _lengths(case):
    """(query rows, cache length) of each sequence."""
    if case["kind"] == "rope":
        n, b = case["tokens"], case["seqs"]
        rows = [n // b + (1 if i < n % b else 0) for i in range(b)]
        return rows, [r + c for r, c in zip(rows, _spread(case["context"] // 2, case["context"], b))]
    if case["kind"] == "decode":
        ls = _spread(min(case["shortest"], case["longest"]), case["longest"], case["batch"])
        return [1] * len(ls), ls
    rows = _spread(max(1, case["rows"] // 3), case["rows"], case["batch"])
    return rows, [r + c for r, c in zip(rows, _spread(case["context"] // 2, case["context"], case["batch"]))]


def _doc_starts(case):
    """First key that each row may see: the start of its document (None: no such mask)."""
    rows, lens = _lengths(case)
    if case["kind"] == "decode":
        return [n // 3 for n in lens] if case["docs"] else None
    if not case["doc"]:
        return None
    return [(n - r + i) // case["doc"] * case["doc"] for r, n in zip(rows, lens) for i in range(r)]


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def frequencies(case):
    """Rotary frequencies [rotary / 2] in f64 and the factor on cos and sin: base 10000,
    divided by 8 ("linear"), or by 8 only where the original 4096 positions hold less than one turn,
    not at all above 32 turns and in between by a ramp ("parts")."""
    n = case["rotary"]
    f = 10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if case["scaling"] == "linear":
        return f / 8, 1.0
    if case["scaling"] == "parts":
        at = lambda turns: n * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
        lo, hi = max(0, math.floor(at(32))), min(n - 1, math.ceil(at(1)))
        ramp = ((torch.arange(n // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / 8 * ramp + f * (1 - ramp), 0.1 * math.log(8) + 1.0
    return f, 1.0


def _pages(s, g, case, lens, dtype, fill):
    """K and V pages of sequences of these lengths, in random order, and the page table."""
    ps = case["page"]
    need = [-(-n // ps) for n in lens]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    wide = torch.arange(max(need), device="cuda")[None, :]
    first = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)[:, None]
    used = wide < torch.tensor(need, device="cuda")[:, None]
    s.table = torch.where(used, order[(first + wide).clamp(max=n_pages - 1)], -1).contiguous()
    shape = (n_pages, ps, case["kv_heads"], case["head_dim"])
    s.k_pages, s.v_pages = ((_randn(g, *shape) if fill else torch.zeros(shape, device="cuda")).to(dtype)
                            for _ in range(2))
    if own:
        s.cache = _paged().PagedKVCache(s.k_pages, s.v_pages, s.table)


def _prepare_rope(case, g):
    s = types.SimpleNamespace(case=case)
    rows, lens = _lengths(case)
    t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    # q, k and v are columns of one projection's output
    qkv = _randn(g, t, (h + 2 * hk) * d).to(DT[case["x"]])
    s.q = qkv[:, :h * d].view(t, h, d)
    s.k = qkv[:, h * d:(h + hk) * d].view(t, hk, d)
    s.v = qkv[:, (h + hk) * d:].view(t, hk, d)
    f, s.factor = frequencies(case)
    s.freq = f.float().cuda()
    s.positions = _i32([n - r + i for r, n in zip(rows, lens) for i in range(r)])
    if case["cache"] != "none":
        # the rows before the new ones are taken as written: the cache holds the
        # last page or two of them
        back = [(n - r) % 7 for r, n in zip(rows, lens)]
        s.seqs = _i32([b for b, r in enumerate(rows) for _ in range(r)])
        s.rows = _i32([o + i for r, o in zip(rows, back) for i in range(r)])
        _pages(s, g, case, [r + o for r, o in zip(rows, back)], DT[case["cache"]], False)
    return s


def _prepare_attention(case, g):
    s = types.SimpleNamespace(case=case)
    rows, lens = _lengths(case)
    dt = DT[case["dtype"]]
    s.q = _randn(g, sum(rows), case["heads"], case["head_dim"]).mul_(1.5).to(dt)
    s.kv_len = _i32(lens)
    s.q_start = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    _pages(s, g, case, lens, dt, True)
    s.longest, s.max_rows = max(lens), max(rows)
    h = case["heads"]
    s.slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["bias"] else None
    s.prefix = _i32([min(n, case["prefix"]) for n in lens]) if case["prefix"] else None
    starts = _doc_starts(case)
    s.begin = _i32(starts) if starts is not None else None
    s.out = torch.empty_like(s.q)
    if own:
        s.workspace = _paged().attention_workspace(s.cache, h, s.q.shape[0])
    return s


def prepare(case, seed):
    g = _gen(seed)
    return _prepare_rope(case, g) if case["kind"] == "rope" else _prepare_attention(case, g)


# ---- one pass ----------------------------------------------------------------

def _rotate(x, cos, sin, n, interleaved):
    x = x.float()
    r, rest = x[..., :n], x[..., n:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :n // 2], r[..., n // 2:])
    u, w = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((r, rest), -1)


def _plain_rope(s):
    c = s.case
    angle = s.positions.double()[:, None, None] * s.freq.double()
    cos, sin = angle.cos().float() * s.factor, angle.sin().float() * s.factor
    q, k = (_rotate(x, cos, sin, c["rotary"], c["interleaved"]) for x in (s.q, s.k))
    if c["cache"] == "none":
        return {"q": q.to(s.q.dtype), "k": k.to(s.k.dtype)}
    dt = DT[c["cache"]]
    page, at = s.table[s.seqs.long(), (s.rows // c["page"]).long()].long(), (s.rows % c["page"]).long()
    s.k_pages[page, at] = k.to(dt)
    s.v_pages[page, at] = s.v.to(dt)
    return {"q": q.to(dt), "k_pages": s.k_pages, "v_pages": s.v_pages}


def _plain_attention(s):
    c = s.case
    n, h, d = s.q.shape
    hk, b = c["kv_heads"], s.table.shape[0]
    table = s.table.clamp(min=0).long()
    k, v = (p[table].float().view(b, -1, hk, d).permute(0, 2, 1, 3) for p in (s.k_pages, s.v_pages))
    # rows of each sequence side by side: [sequence, longest row count]
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(s.q_start[1:].long(), row, right=True)
    at = row - s.q_start[seq]
    q = torch.zeros(b, s.max_rows, h, d, device="cuda")
    q[seq, at] = s.q.float()
    q = q.view(b, s.max_rows, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(b, hk, -1, d), k.transpose(-1, -2)).view(b, hk, h // hk, s.max_rows, -1)
    x *= 1.0 / math.sqrt(d)
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    # what a row sees
    key = torch.arange(x.shape[-1], device="cuda")[None, None, :]
    lens = s.kv_len.long()[:, None, None]
    pos = lens - (s.q_start[1:] - s.q_start[:-1])[:, None, None] + torch.arange(s.max_rows, device="cuda")[None, :, None]
    seen = key <= pos
    if c["window"]:
        seen = seen & (key > pos - c["window"])
    if s.prefix is not None:
        first = key < s.prefix[:, None, None]
        seen = seen | (first if c.get("both_ways") else first & (key <= pos))
    seen = seen & (key < lens)
    if s.begin is not None:
        begin = torch.zeros(b, s.max_rows, dtype=torch.int32, device="cuda")
        begin[seq, at] = s.begin
        seen = seen & (key >= begin[:, :, None])
    if s.slopes is not None:
        x -= s.slopes.view(hk, -1, 1, 1) * (pos - key).abs().float()[:, None, None]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hk, -1, x.shape[-1]), v).view(b, hk, h // hk, s.max_rows, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(b, s.max_rows, h, d)
    return o[seq, at].to(s.q.dtype)


def run(state):
    s, c = state, state.case
    if not own:
        return _plain_rope(s) if c["kind"] == "rope" else _plain_attention(s)
    paged = _paged()
    if c["kind"] == "rope":
        turn = dict(interleaved=c["interleaved"], factor=s.factor)
        if c["cache"] == "none":
            q, k = torch.empty(s.q.shape, dtype=s.q.dtype, device="cuda"), torch.empty(s.k.shape, dtype=s.k.dtype, device="cuda")
            paged.rope(s.q, s.k, s.positions, s.freq, q, k, **turn)
            return {"q": q, "k": k}
        q = torch.empty(s.q.shape, dtype=DT[c["cache"]], device="cuda")
        paged.rope_append(s.q, s.k, s.v, s.positions, s.freq, s.cache, s.seqs, s.rows, q, **turn)
        return {"q": q, "k_pages": s.k_pages, "v_pages": s.v_pages}
    mask = dict(softcap=c["softcap"], slopes=s.slopes, window=c["window"], prefix_len=s.prefix, key_begin=s.begin,
                max_kv_len=s.longest, workspace=s.workspace)
    if c["kind"] == "decode":
        paged.attention_decode(s.q, s.cache, s.kv_len, s.out, **mask)
    else:
        paged.attention_prefill(s.q, s.cache, s.q_start, s.kv_len, s.out, prefix_both_ways=c["both_ways"], **mask)
    return s.out


# ---- the definition in 64 bits, one sequence and one head at a time -----------

def _exact_rope(case, s):
    f = torch.polar(torch.full((), s.factor, dtype=torch.float64, device="cuda"),
                    torch.outer(s.positions.double(), s.freq.double()))[:, None]
    n = case["rotary"]

    def turned(x):
        y = x.double().clone()
        first, second = (slice(0, n, 2), slice(1, n, 2)) if case["interleaved"] else (slice(0, n // 2), slice(n // 2, n))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * f
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turned(s.q), turned(s.k)
    if case["cache"] == "none":
        return {"q": q, "k": k}
    kp, vp = s.k_pages.double(), s.v_pages.double()
    rows, wide = s.rows.long(), s.table.shape[1]
    place = s.table.reshape(-1).long()[s.seqs.long() * wide + rows // case["page"]] * case["page"] + rows % case["page"]
    kp.view(-1, *kp.shape[2:])[place] = k
    vp.view(-1, *vp.shape[2:])[place] = s.v.double()
    return {"q": q, "k_pages": kp, "v_pages": vp}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, s)
    rows, lens = _lengths(case)
    starts = _doc_starts(case)
    group = case["heads"] // case["kv_heads"]
    out, t = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda"), 0
    for b, (r, n) in enumerate(zip(rows, lens)):
        where = s.table[b, torch.arange(n, device="cuda") // case["page"]].long()
        inside = torch.arange(n, device="cuda") % case["page"]
        j = torch.arange(n, device="cuda")
        p = torch.arange(n - r, n, device="cuda")
        far = p[:, None] - j[None, :]
        hidden = far < 0
        if case["window"]:
            hidden |= far >= case["window"]
        if case["prefix"]:
            early = (j < case["prefix"])[None, :]
            hidden &= ~(early if case.get("both_ways") else early & (far >= 0))
        if starts is not None:
            hidden |= j[None, :] < torch.tensor(starts[t:t + r], device="cuda")[:, None]
        for head in range(case["heads"]):
            k = s.k_pages[where, inside, head // group].double()
            v = s.v_pages[where, inside, head // group].double()
            x = s.q[t:t + r, head].double() @ k.T / math.sqrt(case["head_dim"])
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            if case["bias"]:
                x = x - float(s.slopes[head]) * far.abs()
            w = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[t:t + r, head] = torch.nan_to_num(w) @ v
        t += r
    return out


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    rows, lens = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rope":
        t, size = case["tokens"], SIZE[case["x"]]
        if case["cache"] == "none":
            return {"bytes": 2 * t * (h + hk) * d * size + 4 * t, "flops": 3 * t * (h + hk) * case["rotary"]}
        return {"bytes": t * (h + 2 * hk) * d * (size + SIZE[case["cache"]]) + 12 * t,
                "flops": 3 * t * (h + hk) * case["rotary"]}
    size, starts = SIZE[case["dtype"]], _doc_starts(case)
    pairs = keys = t = 0
    for r, n in zip(rows, lens):
        lowest, prefix = n, min(n, case["prefix"])
        for i in range(r):
            p = n - r + i
            begin = starts[t] if starts is not None else 0
            lo = max(begin, p + 1 - case["window"] if case["window"] else 0)
            seen = prefix if case.get("both_ways") else min(prefix, p + 1)  # keys of the prefix that this row may see
            pairs += p + 1 - min(p + 1, max(lo, seen)) + max(0, seen - begin)
            lowest = min(lowest, max(lo, prefix))
            t += 1
        first = min(starts[t - r:t]) if starts is not None else 0
        keys += n - lowest + max(0, min(prefix, lowest) - first)
    return {"bytes": 2 * sum(rows) * h * d * size + 2 * keys * hk * d * size + 4 * sum(-(-n // case["page"]) for n in lens),
            "flops": 4 * pairs * h * d}
