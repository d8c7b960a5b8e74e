"""The attention half of a decoder layer on a paged cache, as a program runs it: projection, rotary
positions with the append, attention, projection back and the MoE block, through prefill and decoding with a
prefix and a window (the R-SWA set of keys). The reference is this library's contiguous R-SWA cache
(uocr_hip_rswa_*) on the same projections: f32 on both sides, each within 2^-17 of the exact
result at these sizes (chains of 128 f32 products of unit scale, at most 100 keys; 1e-5 is
over 8 times that)."""
import numpy as np
import pytest
import torch

from test_gpu_paged import i32, paged

pytestmark = pytest.mark.gpu
H, HEADS, D, P, W, B, STEPS = 1280, 10, 128, 57, 32, 2, 40


def lib():
    from uocr_hip import _lib
    return _lib.load()


def ok(rc):
    from uocr_hip._lib import check
    check(rc)


class Request:
    """B requests' projections, rotary table and both caches."""

    def __init__(self, dev, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
        self.dev = dev
        self.wqkv = (rand(3 * H, H) * H**-0.5).to(torch.bfloat16)
        self.wo = (rand(H, H) * H**-0.5).to(torch.bfloat16)
        self.x = rand(B * (P + STEPS), H)  # hidden states, step by step: all prompts, then a row per request
        freq, self.factor = paged().rope_frequencies(D, scaling="parts", factor_len=4.0, original_len=64)
        self.freq = freq.to(dev)
        page, n = 16, -(-(P + STEPS) // 16)
        order = torch.randperm(B * n, generator=g, device=dev).to(torch.int32)
        pages = [torch.full((B * n, page, HEADS, D), float("nan"), device=dev) for _ in range(2)]
        self.cache = paged().PagedKVCache(*pages, order.view(B, n).contiguous())
        self.ws = paged().attention_workspace(self.cache, HEADS, B * P)
        self.kc, self.vc = (torch.zeros(B, P + W, HEADS, D, device=dev) for _ in range(2))
        self.slots, self.plen = i32(range(B), dev), i32([P] * B, dev)
        self.ring_len, self.ring = i32([P] * B, dev), i32([0] * B, dev)

    def project(self, x):
        from uocr_hip import ops
        out = torch.empty(x.shape[0], 3 * H, device=self.dev)
        ops.matmul_t_bf16(x, self.wqkv.view(torch.int16), out)
        return [t.unflatten(1, (HEADS, D)) for t in out.split(H, 1)]


def test_layer_matches_the_contiguous_cache(dev):
    from uocr_hip import MoELayerInt4, ops, synth
    r = Request(dev)
    # prefill, both requests in one ragged call
    q, k, v = r.project(r.x[:B * P])
    pos, seq = i32(list(range(P)) * B, dev), i32([b for b in range(B) for _ in range(P)], dev)
    qr, kr, out, want = (torch.empty(B * P, HEADS, D, device=dev) for _ in range(4))
    paged().rope_append(q, k, v, pos, r.freq, r.cache, seq, pos, qr, factor=r.factor)
    paged().attention_prefill(qr, r.cache, i32([0, P, 2 * P], dev), r.plen, out, window=W, prefix_len=r.plen, workspace=r.ws)
    paged().rope(k, None, pos, r.freq, kr, None, factor=r.factor)
    vd = v.contiguous()
    ok(lib().uocr_hip_rswa_write_prefill_ragged(kr.data_ptr(), vd.data_ptr(), r.kc.data_ptr(), r.vc.data_ptr(), seq.data_ptr(),
                                                pos.data_ptr(), B * P, P + W, HEADS, D, None))
    ok(lib().uocr_hip_rswa_attention_ragged(qr.data_ptr(), r.kc.data_ptr(), r.vc.data_ptr(), seq.data_ptr(), pos.data_ptr(), B * P,
                                            P + W, HEADS, HEADS, D, want.data_ptr(), None))
    assert (out - want).abs().max().item() <= 1e-5
    # decoding: the prompt's rows and the last W tokens
    L = synth.random_layer(seed=7, n_experts=8, group=32)
    moe, mws = MoELayerInt4(L), None
    mws = moe.alloc_workspace(B, dev)
    for step in range(STEPS):
        x = r.x[B * (P + step):B * (P + step + 1)]
        q, k, v = r.project(x)
        pos = i32([P + step] * B, dev)
        kv_len = i32([P + step + 1] * B, dev)
        qr, kr, out, want = (torch.empty(B, HEADS, D, device=dev) for _ in range(4))
        paged().rope_append(q, k, v, pos, r.freq, r.cache, r.slots, pos, qr, factor=r.factor)
        paged().attention_decode(qr, r.cache, kv_len, out, window=W, prefix_len=r.plen, workspace=r.ws)
        paged().rope(k, None, pos, r.freq, kr, None, factor=r.factor)
        vd = v.contiguous()
        ok(lib().uocr_hip_rswa_append_decode_batch(kr.data_ptr(), vd.data_ptr(), r.kc.data_ptr(), r.vc.data_ptr(),
                                                   r.ring_len.data_ptr(), r.ring.data_ptr(), r.plen.data_ptr(), r.slots.data_ptr(),
                                                   B, P + W, W, HEADS, D, None))
        ok(lib().uocr_hip_rswa_attention_batch(qr.data_ptr(), r.kc.data_ptr(), r.vc.data_ptr(), r.ring_len.data_ptr(),
                                               r.slots.data_ptr(), B, P + W, HEADS, HEADS, D, want.data_ptr(), None))
        assert (out - want).abs().max().item() <= 1e-5, step
        if step % 10 == 0:  # the rest of the layer on what attention gave
            h = torch.empty(B, H, device=dev)
            ops.matmul_t_bf16(out.view(B, H), r.wo.view(torch.int16), h)
            y = torch.empty_like(h)
            moe.forward(h, y, mws)
            assert torch.isfinite(y).all()
    moe.close()


def test_decode_step_captured(dev):
    """One captured step (projection, append, attention, lengths moved on the device) replayed token by
    token gives the eager run's bits."""
    runs = []
    for captured in (False, True):
        r = Request(dev, 3)
        q, k, v = r.project(r.x[:B * P])
        pos, seq = i32(list(range(P)) * B, dev), i32([b for b in range(B) for _ in range(P)], dev)
        qr = torch.empty(B * P, HEADS, D, device=dev)
        paged().rope_append(q, k, v, pos, r.freq, r.cache, seq, pos, qr, factor=r.factor)
        at, kv_len = i32([P] * B, dev), i32([P + 1] * B, dev)
        x, out, qs = r.x[:B].clone(), torch.empty(B, HEADS, D, device=dev), torch.empty(B, HEADS, D, device=dev)

        def step():
            q, k, v = r.project(x)
            paged().rope_append(q, k, v, at, r.freq, r.cache, r.slots, at, qs, factor=r.factor)
            paged().attention_decode(qs, r.cache, kv_len, out, window=W, prefix_len=r.plen, workspace=r.ws)
            at.add_(1)
            kv_len.add_(1)

        results = []
        if captured:
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step()
            at.fill_(P)
            kv_len.fill_(P + 1)
        for i in range(STEPS):
            x.copy_(r.x[B * (P + i):B * (P + i + 1)])
            g.replay() if captured else step()
            results.append(out.clone())
            if i % 7 == 0:
                torch.cuda.synchronize()
        runs.append(torch.stack(results))
    assert torch.isfinite(runs[0]).all() and torch.equal(*runs)
