// Attention of many query rows over a paged KV cache, tiled on MFMA
// (instantiated per type in paged_prefill_{bf16,f16,f32}.hip).
//
// out = softmax(s) V row by row, s = scale q.k with cap, bias and mask; one pass over the
// keys with a running maximum and sum per row. 4 head_dim operations per visible pair and head
// on the matrix cores, beside which a score costs some 4 vector instructions (scale, exponential,
// sum, rounding). 8192 rows of 32 heads of 128 over 8, causal, bf16: 655 us, 839 TFLOP/s; the matrix cores
// are busy for 39% of the cycles, the vector units for 47, LDS for 35, bank conflicts below 1. f32, 4096 rows of 10 heads: 470 us, 91 TFLOP/s.
//
// A workgroup of 4 waves takes 128 query rows of one KV head (64 or 32 in small calls, the waves
// then also taking turns at the tiles of keys): the `group` query heads that
// share it side by side for each token, so that K and V tiles serve all of them. 16-bit heads above 128
// take 8 waves, two per SIMD, in two turns at the keys, where they fill the chip. Tiles of 64 keys (32 for f32 and for heads above 128) go
// through registers into LDS, the next one in flight during the current one's products; registers (and not a
// direct load) because pages may start anywhere and rows are padded. Each wave has 32 rows:
//   * S^T = K Q^T on v_mfma_f32_32x32x16: lane (i, h) = (lane % 32, lane / 32) holds row i's
//     scores of keys 8 (r / 4) + 4 h + r % 4, so a row's maximum and sum need one exchange between
//     the halves of the wave, and ...
//   * ... O^T = V^T P^T takes the probabilities where they are: a 16-key step's slots (h, e) are
//     keys 4 h + e and 4 h + 8 + e - 4. V's transposed operand comes from LDS by
//     ds_read_b64_tr_b16 (4 keys x 16 dims per 16 lanes); f32 reads it directly.
// LDS rows are padded so that these reads cover all banks: K rows to an odd multiple
// of 16 bytes, V rows to 64 bytes more or less than a multiple of 256 (f32: 32 bytes more).
// The running maximum is raised only where a score passes it by 2^8 (probabilities up to 256 are as
// exact as those up to 1), so sums are rarely rescaled.
// Rows whose result is not finite, or that saw a key without a page, are done again by row_attention:
// NaN and infinities of keys that only other rows of the tile see do not reach them.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>

#include "launch.hpp"
#include "paged_device.hpp"
#include "paged_host.hpp"

namespace uocr_hip {

// RW: waves along the rows; KW groups of them take turns at the tiles of keys
template <typename T, int DP, int RW, int KW>
struct PreShape {
    static constexpr int ES = sizeof(T), WAVES = RW * KW;
    static constexpr int ROWS = RW * 32;  // packed query rows per workgroup
    static constexpr int KEYS = ES == 4 || DP > 128 ? 32 : 64;  // per tile
    static constexpr int KSTR = DP * ES + 16;
    static constexpr int VPAD = ES == 4 ? 32 : (DP * 2 % 256 == 64 || DP * 2 % 256 == 192) ? 0 : 64;
    static constexpr int VSTR = DP * ES + VPAD;
    static constexpr int TILE = KEYS * (KSTR + VSTR);
    static constexpr int BUFS = KW == 1 ? 2 : 1;
    // 8 waves: the query operand waits in LDS (heads of 256: 64 registers; in them 4096 rows of 16 heads take 301 us, not 219)
    static constexpr bool QLDS = WAVES == 8;
    static constexpr int QAT = TILE * KW * BUFS, TILES = QAT + (QLDS ? ROWS * KSTR : 0);
    static constexpr int OUT = ROWS * (DP * 4 + 16);                                    // a workgroup's rows on their way out
    static constexpr int SUMS = KW == 1 ? 0 : (DP / 32 * 4 + 1) * 1024 * (WAVES / 2);  // half the waves' sums
    static constexpr int LDS = TILES > OUT ? (TILES > SUMS ? TILES : SUMS) : OUT > SUMS ? OUT : SUMS;
    // waves per SIMD that registers and LDS allow
    static constexpr int PER_SIMD = WAVES == 8 ? 2 : DP > 128 || KW == 4 ? 1 : 2;
};

// Row range of sequence entry b in [0, rows]
__device__ __forceinline__ int pre_start(const PagedAttnArgs& a, int b) { return imin(imax(a.q_start[b], 0), a.rows); }

// Entry b, its sequence and cache length, and the tile within it, of tile index t (tiles of entry after
// entry); -1: none. A lane holds an entry, so that nothing is loaded one after the other.
template <int ROWS>
__device__ __forceinline__ int pre_find(const PagedAttnArgs& a, int t, int& tile, int& seq, int& kv) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = b0 + lane;
        int n = 0, my_seq = -1, my_kv = 0;
        if (b < a.batch) {
            my_seq = a.seqs ? a.seqs[b] : b;
            if ((uint32_t)my_seq < (uint32_t)a.c.n_seqs) my_kv = a.kv_len[my_seq];
            else my_seq = -1;
            n = (imax(pre_start(a, b + 1) - pre_start(a, b), 0) * a.group + ROWS - 1) / ROWS;
        }
        int sum = n;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
            const int y = __shfl_up(sum, x, 64);
            if (lane >= x) sum += y;
        }
        const uint64_t hit = __ballot(before + sum > t);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            tile = t - before - (__builtin_amdgcn_readlane(sum, src) - __builtin_amdgcn_readlane(n, src));
            seq = __builtin_amdgcn_readlane(my_seq, src);
            kv = __builtin_amdgcn_readlane(my_kv, src);
            return b0 + src;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int x = 1; x < 64; x *= 2) v = imin(v, __shfl_xor(v, x, 64));
    return v;
}
__device__ __forceinline__ int wave_max(int v) { return -wave_min(-v); }

// max over the two halves of a wave
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// bits [b, e) of a 64-bit word, any ints
__device__ __forceinline__ uint64_t bits(int b, int e) {
    b = imin(imax(b, 0), 64);
    e = imin(imax(e, 0), 64);
    if (b >= e) return 0;
    return (e == 64 ? ~0ull : (1ull << e) - 1) & ~(b == 64 ? ~0ull : (1ull << b) - 1);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ s16x4 lds_tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(__attribute__((address_space(3))) void*)(void*)p);
}

template <typename T, int DP, bool CAP, bool BIAS, int RW, int KW>
__global__ __launch_bounds__(RW * KW * 64, (PreShape<T, DP, RW, KW>::PER_SIMD)) void paged_prefill_kernel(PagedAttnArgs a) {
    typedef PreShape<T, DP, RW, KW> P;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int ES = sizeof(T), BN = P::KEYS, KB = BN / 32, CH = DP * ES / 16, GT = RW * 64, NL = BN * CH / GT;
    static_assert(BN * CH % GT == 0, "whole 16-byte units per thread");
    constexpr int KSTR = P::KSTR, VSTR = P::VSTR;
    constexpr int NF = F32 ? DP / 8 : DP / 16;  // 16-byte pieces of a query row per lane
    constexpr int DB = DP / 32;
    typedef typename Vec8<T>::type vec_t;
    extern __shared__ __attribute__((aligned(16))) char s_buf[];  // tiles: K rows, then V rows
    __shared__ int s_range[P::WAVES][4];
    __shared__ int s_lost;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 31, h = lane >> 5;
    const int rw = wave % RW, kg = wave / RW, gtid = tid % GT;
    // Last tiles first: they see the most keys under a causal mask. The KV heads of a tile side by
    // side: workgroup b runs on XCD b % 8, so 8 of them leave each XCD's L2 one head's K and V, and other
    // numbers of heads share every XCD's evenly (4096 rows of 10 heads, 128 pairs to a workgroup: runs of
    // one head per XCD 158 us, this way 126).
    const int per = a.n_tiles * a.kv_heads, split = blockIdx.x / per, item = blockIdx.x % per;
    const int kvh = item % a.kv_heads;
    int tile, seq, kv;
    const int entry = pre_find<P::ROWS>(a, a.n_tiles - 1 - item / a.kv_heads, tile, seq, kv);
    if (entry < 0 || seq < 0) return;
    const int start = pre_start(a, entry), n = imax(pre_start(a, entry + 1) - start, 0);
    const bool gone = kv > a.c.capacity();  // more keys than the table has room for
    const int len = gone ? 0 : imax(kv, 0);

    // this lane's query row
    const int packed = tile * P::ROWS + rw * 32 + i;
    const bool live = packed < n * a.group;
    const int token = packed / a.group, row = start + imin(token, n - 1), head = kvh * a.group + packed % a.group;
    const int pos = len - n + token;
    const int prefix = a.mask.prefix_len ? a.mask.prefix_len[seq] : 0;
    Span span{0, 0, 0, 0};
    if (live)
        span = row_span(a.mask.causal, a.mask.window, a.mask.both_ways, pos, len, prefix,
                        a.mask.key_begin ? a.mask.key_begin[row] : 0, a.mask.key_end ? a.mask.key_end[row] : len);
    // keys that some row sees: two ranges. Rows without limits of their own: the first and last
    // row's say it (the window moves on with the row, and so does the end).
    int lo0, hi0, lo1, hi1;
    if (!a.mask.key_begin && !a.mask.key_end) {
        const int last = imin((tile + 1) * P::ROWS, n * a.group) - 1;
        tile_range(a.mask.causal, a.mask.window, a.mask.both_ways, len - n + tile * P::ROWS / a.group,
                   len - n + last / a.group, len, prefix, lo0, hi0, lo1, hi1);
    } else {
        constexpr int kFar = 0x7fffffff;
        const bool in0 = span.e0 > span.b0, in1 = span.e1 > span.b1;
        const int r0 = wave_min(in0 ? span.b0 : kFar), r1 = wave_max(in0 ? span.e0 : 0);
        const int r2 = wave_min(in1 ? span.b1 : kFar), r3 = wave_max(in1 ? span.e1 : 0);
        if (lane == 0) {
            s_range[wave][0] = r0;
            s_range[wave][1] = r1;
            s_range[wave][2] = r2;
            s_range[wave][3] = r3;
        }
        __syncthreads();
        lo0 = lo1 = kFar;
        hi0 = hi1 = 0;
#pragma unroll
        for (int w = 0; w < P::WAVES; ++w) {
            lo0 = imin(lo0, s_range[w][0]);
            hi0 = imax(hi0, s_range[w][1]);
            lo1 = imin(lo1, s_range[w][2]);
            hi1 = imax(hi1, s_range[w][3]);
        }
        lo0 = __builtin_amdgcn_readfirstlane(lo0);
        hi0 = __builtin_amdgcn_readfirstlane(hi0);
        lo1 = __builtin_amdgcn_readfirstlane(lo1);
        hi1 = __builtin_amdgcn_readfirstlane(hi1);
    }
    if (tid == 0) s_lost = 0;
    bool lost = false;  // a key of this lane's tiles has no page
    // as tiles; one range where a tile would be in both
    int t0 = hi0 ? lo0 / BN : 0, n0 = hi0 ? (hi0 - 1) / BN + 1 - t0 : 0;
    int t1 = hi1 ? lo1 / BN : 0, n1 = hi1 ? (hi1 - 1) / BN + 1 - t1 : 0;
    if (n0 && n1 && t0 < t1 + n1 && t1 < t0 + n0) {
        const int e = imax(t0 + n0, t1 + n1);
        t0 = imin(t0, t1);
        n0 = e - t0;
        n1 = 0;
        lo0 = imin(lo0, lo1);
        hi0 = imax(hi0, hi1);
    }
    const int tiles = n0 + n1, share = (tiles + a.n_splits - 1) / a.n_splits;
    const int t_begin = imin(split * share, tiles), t_end = imin(t_begin + share, tiles);

    // query operand: dims 16 f + 8 h .. + 7 (f32: 8 f + 4 h .. + 3) of row i
    vec_t q[P::QLDS ? 1 : NF];
    char* const q_lds = s_buf + P::QAT + (rw * 32 + i) * KSTR + h * 16;
    if (!P::QLDS || kg == 0) {
        const char* qp = a.q.p + row * a.q.row_bytes + head * a.q.head_bytes;
        // a negative scale is moved into q: the maximum is taken before the scale
        const uint32_t flip = a.sc.negative ? (F32 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int d = (2 * f + h) * (16 / ES);
            const bool in = live && d < a.head_dim;
            u32x4 w = {0, 0, 0, 0};
            if (in) w = *reinterpret_cast<const u32x4*>(qp + d * ES);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] ^= flip;
            if constexpr (P::QLDS) *reinterpret_cast<u32x4*>(q_lds + f * 32) = w;
            else q[f] = as_vec<vec_t>(w);
        }
    }
    PagedScores sc = a.sc;
    sc.scale2 = fabsf(sc.scale2);
    sc.in = fabsf(sc.in);
    sc.in2 = fabsf(sc.in2);
    const float scale2 = sc.scale2;
    float slope2 = 0.0f;
    if constexpr (BIAS) slope2 = a.sc.slopes[head] * kLog2e;

    // tile t of the block's ranges: K and V to registers, then to LDS
    const char* kbase = a.c.k + kvh * a.c.head_bytes;
    const char* vbase = a.c.v + kvh * a.c.head_bytes;
    u32x4 kw[NL], vw[NL];
    auto tile_base = [&](int t) { return (t < n0 ? t0 + t : t1 + t - n0) * BN; };
    auto place = [&](int t) {  // of key `lane` (mod BN); keys outside the range: those at its ends
        const int lo = t < n0 ? lo0 : lo1, hi = t < n0 ? hi0 : hi1;
        long long off = a.c.offset(seq, imin(imax(tile_base(t) + (lane & (BN - 1)), lo), hi - 1));
        lost |= off < 0;
        return off < 0 ? 0 : off;
    };
    auto load = [&](long long off) {
#pragma unroll
        for (int e = 0; e < NL; ++e) {
            const int u = e * GT + gtid, r = u / CH, c = u % CH;
            const long long at = shfl64(off, r) + imin(c, a.head_dim * ES / 16 - 1) * 16;
            kw[e] = *reinterpret_cast<const u32x4*>(kbase + at);
            vw[e] = *reinterpret_cast<const u32x4*>(vbase + at);
        }
    };
    auto store = [&](char* buf) {
        if (a.head_dim < DP) {  // 0 past the head
#pragma unroll
            for (int e = 0; e < NL; ++e)
                if ((e * GT + gtid) % CH * (16 / ES) >= a.head_dim) kw[e] = vw[e] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int e = 0; e < NL; ++e) {
            const int u = e * GT + gtid, r = u / CH, c = u % CH;
            *reinterpret_cast<u32x4*>(buf + r * KSTR + c * 16) = kw[e];
            *reinterpret_cast<u32x4*>(buf + BN * KSTR + r * VSTR + c * 16) = vw[e];
        }
    };

    float m = -INFINITY, l = 0.0f;  // of row i (l: over this lane's keys), in log 2
    f32x16 o[DB] = {};
    const int rounds = (t_end - t_begin + KW - 1) / KW;  // (the same for every wave: barriers)
    if (rounds) {
        // group kg: tiles t_begin + kg, + KW, ..
        int t = t_begin + kg;
        char* const own = s_buf + kg * P::TILE;
        if (t < t_end) load(place(t));
        long long next = t + KW < t_end ? place(t + KW) : 0;
        if (t < t_end) store(own);
        for (int round = 0; round < rounds; ++round, t += KW) {
            // one wave per group: its tile is its own, and LDS accesses of a wave stay in order
            if constexpr (RW > 1) __syncthreads();
            const char* buf = own + (P::BUFS == 2 ? (round & 1) * P::TILE : 0);
            if (t + KW < t_end) load(next);
            if (t + 2 * KW < t_end) next = place(t + 2 * KW);
            if (t < t_end) {
                const int base = tile_base(t);
            const uint64_t seen = bits(span.b0 - base, span.e0 - base) | bits(span.b1 - base, span.e1 - base);
            constexpr uint64_t kAll = BN == 64 ? ~0ull : (1ull << BN) - 1;
            if (__any((seen & kAll) != 0)) {
                f32x16 s[KB];
#pragma unroll
                for (int b = 0; b < KB; ++b) s[b] = f32x16{};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    vec_t qf;
                    if constexpr (P::QLDS) qf = *reinterpret_cast<const vec_t*>(q_lds + f * 32);
                    else qf = q[f];
#pragma unroll
                    for (int b = 0; b < KB; ++b) {
                        const vec_t k = *reinterpret_cast<const vec_t*>(buf + (b * 32 + i) * KSTR + h * 16 + f * 32);
                        if constexpr (F32) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[b] = mfma_32x32x2(k[e], qf[e], s[b]);
                        } else {
                            s[b] = mfma_32x32x16(k, qf, s[b]);
                        }
                    }
                }
                const bool whole = __all((seen & kAll) == kAll);
                if constexpr (CAP || BIAS) {
                    const float dist0 = (float)(pos - base - 4 * h);
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[b][r] = score2<CAP, BIAS, F32>(s[b][r], sc, slope2, dist0 - (float)(b * 32 + 8 * (r >> 2) + (r & 3)));
                }
                constexpr bool kScaled = CAP || BIAS;
                if (!whole) {
                    uint64_t mine = seen >> (4 * h);
                    // (a branch: as selects it would be a third of the loop's vector instructions)
                    asm volatile("" : "+v"(mine));
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[b][r] = (uint32_t)(mine >> (32 * b)) >> (8 * (r >> 2) + (r & 3)) & 1 ? s[b][r] : -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
                top = half_max(top);
                if constexpr (!kScaled) top *= scale2;
                if (__any(top > m + 8.0f)) {
                    const float up = fmaxf(m, top), ref = up == -INFINITY ? 0.0f : up;
                    const float alpha = __builtin_amdgcn_exp2f(m - ref);
                    m = up;
                    l *= alpha;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                float sum[4] = {};
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        s[b][r] = __builtin_amdgcn_exp2f(kScaled ? s[b][r] - ref : fmaf(s[b][r], scale2, -ref));
                        sum[r & 3] += s[b][r];
                    }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                const char* vp = buf + BN * KSTR;
                if constexpr (F32) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
#pragma unroll
                        for (int d = 0; d < DB; ++d)
                            o[d] = mfma_32x32x2(*reinterpret_cast<const float*>(vp + (8 * (r >> 2) + (r & 3) + 4 * h) * VSTR + (d * 32 + i) * 4),
                                                s[0][r], o[d]);
                } else {
                    vp += (4 * h + (lane >> 2 & 3)) * VSTR + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
#pragma unroll
                    for (int st = 0; st < KB * 2; ++st) {
                        vec_t p;
#pragma unroll
                        for (int e = 0; e < 8; ++e) p[e] = (T)s[st >> 1][8 * (st & 1) + e];
#pragma unroll
                        for (int d = 0; d < DB; ++d) {
                            s16x4 v[2];
                            v[0] = lds_tr(vp + st * 16 * VSTR + d * 64);
                            v[1] = lds_tr(vp + (st * 16 + 8) * VSTR + d * 64);
                            vec_t vv;
                            __builtin_memcpy(&vv, v, 16);
                            o[d] = mfma_32x32x16(vv, p, o[d]);
                        }
                    }
                }
            }
            }
            if constexpr (RW > 1 && P::BUFS == 1) __syncthreads();
            if (t + KW < t_end) store(own + (P::BUFS == 2 ? (round + 1 & 1) * P::TILE : 0));
        }
    }
    __syncthreads();
    if (lost) s_lost = 1;
    __syncthreads();
    // the groups' sums of the same rows, by halves
#pragma unroll
    for (int half = KW / 2; half >= 1; half /= 2) {
        f32x4* at = reinterpret_cast<f32x4*>(s_buf) + (size_t)(kg % half * RW + rw) * (DB * 4 + 1) * 64 + lane;
        if (kg >= half && kg < 2 * half) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) at[(d * 4 + r / 4) * 64] = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
            at[DB * 4 * 64] = f32x4{m, l, 0.0f, 0.0f};
        }
        __syncthreads();
        if (kg < half) {
            const f32x4 ml = at[DB * 4 * 64];
            const float up = fmaxf(m, ml[0]), ref = up == -INFINITY ? 0.0f : up;
            const float f1 = __builtin_amdgcn_exp2f(m - ref), f2 = __builtin_amdgcn_exp2f(ml[0] - ref);
            m = up;
            l = l * f1 + ml[1] * f2;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x4 v = at[(d * 4 + r / 4) * 64];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][r + e] = o[d][r + e] * f1 + v[e] * f2;
                }
        }
        __syncthreads();
    }
    if (kg) return;
    l += __shfl_xor(l, 32, 64);
    if (a.n_splits > 1) {
        if (live) {
            const size_t rec = ((size_t)row * a.heads + head) * a.n_splits + split;
            if (h == 0) {
                a.part_ml[2 * rec] = m;
                a.part_ml[2 * rec + 1] = s_lost ? NAN : l;  // (the join does such a row again)
            }
            if (m != -INFINITY || l != 0.0f) {
                float* p = a.part + rec * a.head_dim;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const int d0 = d * 32 + 2 * r + 4 * h;
                        if (d0 < a.head_dim)
                            *reinterpret_cast<f32x4*>(p + d0) = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
                    }
            }
        }
        return;
    }
    const float inv = 1.0f / l;
    bool bad = s_lost || !(l > 0.0f && l < INFINITY);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[d][r] *= inv;
            bad |= !(fabsf(o[d][r]) < INFINITY);
        }
    if (span.count() == 0) {
        bad = false;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = gone ? NAN : 0.0f;
    }
    uint64_t again = __ballot(bad && live);
    again = (again | again >> 32) & 0xffffffffu;
    const uint64_t keep = __ballot(live) & ~again;
    // rows through LDS, so that a row leaves in 16-byte pieces side by side (8-byte pieces of
    // 32 rows per store: 6 us for 64 rows of 32 heads instead of 1)
    const bool wide = (((uintptr_t)a.out.p | a.out.row_bytes | a.out.head_bytes) & 15) == 0;
    const long long out_at = row * a.out.row_bytes + head * a.out.head_bytes;
    const auto put = [&](auto type) {
        typedef decltype(type) O;
        constexpr int OES = sizeof(O), OSTR = DP * OES + 16, PIECES = DP * OES / 16;
        char* so = s_buf + rw * 32 * OSTR;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                O t[4] = {(O)o[d][r], (O)o[d][r + 1], (O)o[d][r + 2], (O)o[d][r + 3]};
                __builtin_memcpy(__builtin_assume_aligned(so + i * OSTR + (d * 32 + 2 * r + 4 * h) * OES, 4 * OES), t, 4 * OES);
            }
#pragma unroll 4
        for (int u = lane; u < 32 * PIECES; u += 64) {
            const int r = u / PIECES, c = u % PIECES;
            char* p = a.out.p + shfl64(out_at, r) + c * 16;
            if (c * (16 / OES) >= a.head_dim || !(keep >> r & 1)) continue;
            const u32x4 v = *reinterpret_cast<const u32x4*>(so + r * OSTR + c * 16);
            if (wide) {
                *reinterpret_cast<u32x4*>(p) = v;
            } else {
                for (int e = 0; e < 16 / OES; ++e) {
                    if constexpr (OES == 4) reinterpret_cast<uint32_t*>(p)[e] = v[e];
                    else reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
                }
            }
        }
    };
    if (F32 || a.out_f32) put(0.0f);
    else put((T)0.0f);
    for (; again; again &= again - 1) {
        const int src = __builtin_ctzll(again);
        row_attention<T>(a, seq, __shfl(row, src, 64), __shfl(head, src, 64), __shfl(pos, src, 64), len, gone);
    }
}

// Joins the splits of each (row, head), in their order: one wave each.
template <typename T>
__global__ __launch_bounds__(256) void paged_prefill_join_kernel(PagedAttnArgs a) {
    const int lane = threadIdx.x & 63;
    const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= (long long)a.rows * a.heads) return;
    const int row = (int)(u / a.heads), head = (int)(u % a.heads);
    // the entry whose rows include it
    int lo = 0, hi = a.batch;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.q_start[mid + 1] > row) hi = mid;
        else lo = mid + 1;
    }
    if (lo >= a.batch || a.q_start[lo] > row) return;
    const int seq = a.seqs ? a.seqs[lo] : lo;
    if ((uint32_t)seq >= (uint32_t)a.c.n_seqs) return;
    const int kv = a.kv_len[seq];
    const bool gone = kv > a.c.capacity();
    const int len = gone ? 0 : imax(kv, 0), start = pre_start(a, lo), n = pre_start(a, lo + 1) - start;
    const size_t rec = (size_t)u * a.n_splits;
    // lane s: maximum, factor and sum of splits s and 64 + s
    static_assert(kPagedMaxSplits <= 128, "two splits per lane");
    float ms[2], f[2], M = -INFINITY, L = 0.0f, o[4] = {};
    bool there[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int s = lane + 64 * k;
        ms[k] = -INFINITY;
        f[k] = 0.0f;
        if (s < a.n_splits) {
            ms[k] = a.part_ml[2 * (rec + s)];
            f[k] = a.part_ml[2 * (rec + s) + 1];
        }
        there[k] = ms[k] != -INFINITY || f[k] != 0.0f;  // (else no sums were written)
        M = fmaxf(M, ms[k]);
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x, 64));
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float w = there[k] ? __builtin_amdgcn_exp2f(ms[k] - ref) : 0.0f;
        L = fmaf(f[k], w, L);
        f[k] = w;
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) L += __shfl_xor(L, x, 64);
    const uint64_t has[2] = {__ballot(there[0]), __ballot(there[1])};
    // 4 splits' sums in flight (64 rows of 32 heads on 16000 keys in 16 splits: 57 us, one after the other, now 46)
    for (int s0 = 0; s0 < a.n_splits; s0 += 4) {
        const float fs = s0 < 64 ? f[0] : f[1];
        const uint64_t in = (s0 < 64 ? has[0] : has[1]) >> (s0 & 63);
        float v[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = imin(lane + 64 * e, a.head_dim - 1);
                v[k][e] = 64 * e < a.head_dim ? a.part[(rec + imin(s0 + k, a.n_splits - 1)) * a.head_dim + d] : 0.0f;
            }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = __shfl(fs, (s0 & 63) + k, 64);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(in >> k & 1 ? v[k][e] : 0.0f, w, o[e]);
        }
    }
    bool bad = !(L > 0.0f && L < INFINITY);
    const float inv = 1.0f / L;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        o[e] *= inv;
        bad |= !(fabsf(o[e]) < INFINITY) && lane + 64 * e < a.head_dim;
    }
    if (__any(bad)) {  // (rows that see nothing, too)
        row_attention<T>(a, seq, row, head, len - n + (row - start), len, gone);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < a.head_dim) store_out(a, (const T*)nullptr, row, head, lane + 64 * e, o[e]);
}

// A launch of more than the 64 KiB of LDS that a kernel has by default; asked for once per device
template <auto KERNEL>
int launch_lds(const PagedAttnArgs& a, dim3 grid, dim3 block, uint32_t lds, hipStream_t st) {
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (e == hipSuccess && !(ready.load(std::memory_order_relaxed) & bit)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e == hipSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != hipSuccess) return set_error(UOCR_HIP_EHIP, std::string("paged prefill LDS: ") + hipGetErrorString(e));
    launch_k(KERNEL, grid, block, lds, st, a);
    return UOCR_HIP_OK;
}

template <typename T, int DP, int RW, int KW>
int launch_prefill_shape(const PagedAttnArgs& a, hipStream_t st) {
    typedef PreShape<T, DP, RW, KW> P;
    const dim3 grid((unsigned)((long long)a.n_tiles * a.kv_heads * a.n_splits)), block(P::WAVES * 64);
    const bool cap = a.sc.cap2 > 0.0f, bias = a.sc.slopes != nullptr;
    if (cap && bias) return launch_lds<paged_prefill_kernel<T, DP, true, true, RW, KW>>(a, grid, block, P::LDS, st);
    if (cap) return launch_lds<paged_prefill_kernel<T, DP, true, false, RW, KW>>(a, grid, block, P::LDS, st);
    if (bias) return launch_lds<paged_prefill_kernel<T, DP, false, true, RW, KW>>(a, grid, block, P::LDS, st);
    return launch_lds<paged_prefill_kernel<T, DP, false, false, RW, KW>>(a, grid, block, P::LDS, st);
}
template <typename T, int DP>
int launch_prefill_dp(const PagedAttnArgs& a, int rw, hipStream_t st) {
    constexpr bool F32 = sizeof(T) == 4;
    if constexpr (F32 && DP <= 128)
        if (rw == 1) return launch_prefill_shape<T, DP, 1, 4>(a, st);
    if constexpr (F32 || DP <= 128 || DP > 192)
        if (rw == 2) return launch_prefill_shape<T, DP, 2, 2>(a, st);
    if constexpr (!F32 && DP > 128) return launch_prefill_shape<T, DP, 4, 2>(a, st);
    else if constexpr (!F32 || DP > 128) return launch_prefill_shape<T, DP, 4, 1>(a, st);
    else return set_error(UOCR_HIP_EINVAL, "attention: no such shape");  // (f32 up to 128 plans 1 or 2)
}

template <typename T>
int launch_prefill_t(const PagedAttnArgs& a, int rw, hipStream_t st) {
    int rc;
    if (a.head_dim <= 64) rc = launch_prefill_dp<T, 64>(a, rw, st);
    else if (a.head_dim <= 96) rc = launch_prefill_dp<T, 96>(a, rw, st);
    else if (a.head_dim <= 128) rc = launch_prefill_dp<T, 128>(a, rw, st);
    else if (a.head_dim <= 192) rc = launch_prefill_dp<T, 192>(a, rw, st);
    else rc = launch_prefill_dp<T, 256>(a, rw, st);
    if (rc) return rc;
    if (a.n_splits > 1)
        launch_k(paged_prefill_join_kernel<T>, dim3((unsigned)(((long long)a.rows * a.heads + 3) / 4)), dim3(256), 0, st, a);
    return UOCR_HIP_OK;
}

int launch_prefill_f32(const PagedAttnArgs& a, int rw, hipStream_t st);
int launch_prefill_bf16(const PagedAttnArgs& a, int rw, hipStream_t st);
int launch_prefill_f16(const PagedAttnArgs& a, int rw, hipStream_t st);

}  // namespace uocr_hip
