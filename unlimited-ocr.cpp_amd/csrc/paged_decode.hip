// Attention of one new token per sequence over a paged KV cache, split over the
// cache's length and joined.
//
// For query head h over the visible keys j: p_j = exp2(s_j - max s), out = sum p_j v_j /
// sum p_j. Every visible K and V row is read once per group of query heads
// that share it (up to 16), so the call is bound by HBM.
//
// A wave walks tiles of 32 keys (16 for f32) with a running maximum and sum. The
// products run on MFMA with up to 16 query heads as one side, also for a single head: at 16 KiB
// per tile the matrix cores are busy for about a tenth of the time that the tile's bytes
// take, and nothing moves between lanes:
//   * S = K Q^T: lane (i, g) = (lane % 16, lane / 16) holds 8 dims of key i, straight from
//     its page, and of head i. D has head i, keys 4g .. 4g + 3 of each 16.
//   * O^T = V^T P^T: those keys are taken as the k-slots of group g, so the
//     probabilities are an operand where they are. Lane (i, g) loads V rows of its
//     group's 8 keys, 8 dims each (16 lanes: one row), and transposes the 8 x 8 block in its
//     registers (32 v_perm_b32): MFMA e takes dims 8i + e.
// The next tile's K is loaded as soon as this one's scores are done, its V after this one's
// sums, so every wave keeps 8 to 16 KiB in flight without further registers.
// 16-bit probabilities go in as two halves (p and its rounding error), since the matrix cores
// have room for it: the result is as exact as with f32 probabilities. A rounding error of 0 makes
// NaN of an infinite V, so a wave whose sums hold a NaN goes over its keys again without that half.
//
// Two ways to share the work, with workgroups of 8 waves that take a sequence's tiles in turn
// and are combined in LDS:
//   * short caches: a workgroup per (sequence, KV head), of one wave where there are many;
//   * else all sequences' tiles are one line, cut into equal shares whatever the
//     lengths: a workgroup per (share, KV head), its KV heads' neighbours beside it (their rows are
//     side by side in memory). Of a sequence that several shares cut, each leaves its sums (at most
//     two such sequences per share, its first and its last), and the workgroup that is last to do so
//     joins them, found by a counter: no second launch, which costs 3.5 us before it begins and 5 us
//     itself. Sums and counters move past the XCDs' own L2s (sc1). Where a sequence has so many
//     sums that one workgroup would take longer than that, a second kernel joins them.
#include <hip/hip_runtime.h>

#include "launch.hpp"
#include "paged_device.hpp"
#include "paged_host.hpp"

namespace uocr_hip {
namespace {

template <int DP>
constexpr int kDecWaves = DP > 128 ? 4 : 8;  // (heads of 256: 8 waves' registers do not fit)
constexpr int kDecCols = 16;  // query heads per workgroup

template <typename T>
constexpr int kDecKeys = sizeof(T) == 4 ? 16 : 32;  // keys per tile

struct DecodeRow {
    int seq, len;
    bool gone;  // kv_len is beyond the table's room
    Span span;
    TileWalk walk;
};

template <int KT>
__device__ __forceinline__ DecodeRow decode_row(const PagedAttnArgs& a, int b) {
    DecodeRow r;
    r.seq = a.seqs ? a.seqs[b] : b;
    r.len = 0;
    r.gone = false;
    r.span = Span{0, 0, 0, 0};
    r.walk = TileWalk{0, 0, 0, 0};
    if ((uint32_t)r.seq >= (uint32_t)a.c.n_seqs) {
        r.seq = -1;
        return r;
    }
    const int kv = a.kv_len[r.seq];
    r.gone = kv > a.c.capacity();
    r.len = r.gone ? 0 : imax(kv, 0);
    r.span = row_span(1, a.mask.window, 0, r.len - 1, r.len, a.mask.prefix_len ? a.mask.prefix_len[r.seq] : 0,
                      a.mask.key_begin ? a.mask.key_begin[b] : 0, a.mask.key_end ? a.mask.key_end[b] : r.len);
    r.walk = tile_walk<KT>(r.span);
    return r;
}

// The row that lane `b` holds, for the whole wave
__device__ __forceinline__ DecodeRow row_of_lane(const DecodeRow& r, int b) {
    const auto at = [&](int v) { return __builtin_amdgcn_readlane(v, b); };
    return DecodeRow{at(r.seq), at(r.len), at(r.gone) != 0, {at(r.span.b0), at(r.span.e0), at(r.span.b1), at(r.span.e1)},
                     {at(r.walk.t0), at(r.walk.n0), at(r.walk.t1), at(r.walk.n1)}};
}

// A row's result from its sums; NaN where they or its pages are not fit for one
__device__ __forceinline__ float finish(float acc, float l, bool gone, bool empty) {
    if (gone) return NAN;
    if (l > 0.0f) return acc / l;
    return l == 0.0f && empty ? 0.0f : NAN;
}

// One wave's query heads and its sums over some tiles of one sequence
template <typename T, int DP, bool CAP, bool BIAS>
struct DecodeWave {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int KT = kDecKeys<T>, KB = KT / 16;
    static constexpr int VEC = DP == 64 || F32 ? 4 : 8;  // dims of a V row per lane and load
    static constexpr int NC = DP / (16 * VEC);           // such loads
    static constexpr int KS = F32 ? DP / 16 : DP / 32;   // 16-byte loads of a K row per lane
    static constexpr int KD = F32 ? 4 : 8;               // dims in each
    static constexpr int VR = KT / 4;                    // V rows per lane
    static constexpr uint32_t kAll = (uint32_t)((1ull << KT) - 1);
    typedef typename Vec8<T>::type vec_t;

    int col, g, cols, head0, head;
    vec_t q[KS];
    float slope2;
    const char* kbase;
    const char* vbase;
    float m, l;
    f32x4 acc[NC][VEC];

    // heads of (KV head, block of 16) number kb of row b
    __device__ __forceinline__ void begin(const PagedAttnArgs& a, int b, int kb) {
        const int blocks = (a.group + kDecCols - 1) / kDecCols, kvh = kb / blocks, hb = kb % blocks;
        col = threadIdx.x & 15;
        g = (threadIdx.x & 63) >> 4;
        cols = imin(kDecCols, a.group - hb * kDecCols);
        head0 = kvh * a.group + hb * kDecCols;
        head = head0 + imin(col, cols - 1);
        const char* qp = a.q.p + b * a.q.row_bytes + head * a.q.head_bytes;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * (4 * KD) + g * KD;
            const bool in = d < a.head_dim && col < cols;
            const u32x4 w = *reinterpret_cast<const u32x4*>(qp + (in ? d : 0) * sizeof(T));
            q[s] = as_vec<vec_t>(in ? w : u32x4{0, 0, 0, 0});
        }
        slope2 = 0.0f;
        if constexpr (BIAS) slope2 = a.sc.slopes[head] * kLog2e;
        kbase = a.c.k + kvh * a.c.head_bytes;
        vbase = a.c.v + kvh * a.c.head_bytes;
    }

    __device__ __forceinline__ void load_k(const PagedAttnArgs& a, long long off, u32x4 (&kw)[KB][KS]) {
#pragma unroll
        for (int h = 0; h < KB; ++h) {
            const char* kp = kbase + shfl64(off, h * 16 + col);
#pragma unroll
            for (int s = 0; s < KS; ++s)
                kw[h][s] = *reinterpret_cast<const u32x4*>(kp + imin(s * (4 * KD) + g * KD, a.head_dim - KD) * sizeof(T));
        }
    }
    __device__ __forceinline__ int v_key(int e) const { return F32 ? g * 4 + e : (e >> 2) * 16 + g * 4 + (e & 3); }
    __device__ __forceinline__ void load_v(const PagedAttnArgs& a, long long off, uint32_t (&vw)[NC][VR][VEC * sizeof(T) / 4]) {
#pragma unroll
        for (int e = 0; e < VR; ++e) {
            const char* vp = vbase + shfl64(off, v_key(e));
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = imin(c * 16 * VEC + col * VEC, a.head_dim - VEC);
                __builtin_memcpy(vw[c][e], __builtin_assume_aligned(vp + d * sizeof(T), VEC * sizeof(T)), VEC * sizeof(T));
            }
        }
    }

    // tiles t, t + step, .. below t_end of row r
    __device__ __forceinline__ void walk(const PagedAttnArgs& a, const DecodeRow& r, int t_begin, int t_end, int step) {
        for (bool halves = true;; halves = false) {
            tiles(a, r, t_begin, t_end, step, halves);
            if (F32 || !halves) break;
            bool nan = false;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) nan |= acc[c][i][j] != acc[c][i][j];
            if (!__any(nan)) break;
        }
    }

    __device__ __forceinline__ void tiles(const PagedAttnArgs& a, const DecodeRow& r, int t_begin, int t_end, int step,
                                          bool halves) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[c][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (t_begin >= t_end) return;
        // a tile's places are looked up one tile ahead; lane: key lane % KT
        bool in;
        long long at;
        int base;
        const auto place = [&](int t) {
            const bool first = t < r.walk.n0;
            base = (first ? r.walk.t0 + t : r.walk.t1 + t - r.walk.n0) * KT;
            const int my = base + (threadIdx.x & (KT - 1));
            in = my >= (first ? r.span.b0 : r.span.b1) && my < (first ? r.span.e0 : r.span.e1);
            at = in ? a.c.offset(r.seq, my) : 0;
        };
        u32x4 kw[KB][KS];
        uint32_t vw[NC][VR][VEC * sizeof(T) / 4];
        place(t_begin);
        load_k(a, at < 0 ? 0 : at, kw);
        load_v(a, at < 0 ? 0 : at, vw);
        for (int t = t_begin; t < t_end; t += step) {
            const uint32_t seen = (uint32_t)__ballot(in) & kAll, lost = (uint32_t)__ballot(at < 0) & kAll;
            const float dist0 = (float)(r.len - 1 - base);
            const bool more = t + step < t_end;
            if (more) place(t + step);
            // scores: keys h * 16 + g * 4 + i of head col
            f32x4 s[KB];
#pragma unroll
            for (int h = 0; h < KB; ++h) {
                s[h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    u32x4 w = kw[h][k];
                    if (k * (4 * KD) + g * KD >= a.head_dim) w = u32x4{0, 0, 0, 0};  // (past the head: 0 on both sides)
                    const vec_t kv = as_vec<vec_t>(w);
                    if constexpr (F32) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[h] = mfma_16x16x4(kv[e], q[k][e], s[h]);
                    } else {
                        s[h] = mfma_16x16x32(kv, q[k], s[h]);
                    }
                }
            }
            if (more) load_k(a, at < 0 ? 0 : at, kw);
            float p[KB][4], top = m;
#pragma unroll
            for (int h = 0; h < KB; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = h * 16 + g * 4 + i;
                    float x = score2<CAP, BIAS, F32>(s[h][i], a.sc, slope2, dist0 - (float)key);
                    if (lost >> key & 1) x = NAN;
                    p[h][i] = seen >> key & 1 ? x : -INFINITY;
                    top = fmaxf(top, p[h][i]);
                }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float ref = top == -INFINITY ? 0.0f : top;
            const float alpha = __builtin_amdgcn_exp2f(m - ref);
            m = top;
            float sum = 0.0f;
#pragma unroll
            for (int h = 0; h < KB; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[h][i] = __builtin_amdgcn_exp2f(p[h][i] - ref);
                    sum += p[h][i];
                }
            l = fmaf(l, alpha, sum);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] *= alpha;
            // V of keys that the row does not see must not meet their weight of 0
            if (seen != kAll) {
#pragma unroll
                for (int e = 0; e < VR; ++e) {
                    const bool keep = seen >> v_key(e) & 1;
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int i = 0; i < (int)(VEC * sizeof(T) / 4); ++i) vw[c][e][i] = keep ? vw[c][e][i] : 0;
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < VR; ++e)
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int i = 0; i < VEC; ++i)
                            acc[c][i] = mfma_16x16x4(__uint_as_float(vw[c][e][i]), p[0][e], acc[c][i]);
            } else {
                vec_t hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = p[e >> 2][e & 3];
                    hi[e] = (T)x;
                    lo[e] = (T)(x - (float)hi[e]);
                }
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        u32x4 w;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = __builtin_amdgcn_perm(vw[c][2 * e + 1][i / 2], vw[c][2 * e][i / 2],
                                                         i & 1 ? 0x07060302u : 0x05040100u);
                        const vec_t v = as_vec<vec_t>(w);
                        acc[c][i] = mfma_16x16x32(v, hi, acc[c][i]);
                        if (halves) acc[c][i] = mfma_16x16x32(v, lo, acc[c][i]);
                    }
            }
            if (more) load_v(a, at < 0 ? 0 : at, vw);
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
    }

    // first of the VEC dims that acc[c][0 .. VEC - 1][j] hold
    __device__ __forceinline__ int dim(int c, int j) const { return c * 16 * VEC + (g * 4 + j) * VEC; }
};

// LDS of a workgroup's results
template <int UW>
struct DecodeLds {
    float m[UW][kDecCols], l[UW][kDecCols];
};

// The waves' sums into LDS: o [waves][cols][DP + 4]
template <typename W, int UW, int DP>
__device__ __forceinline__ void leave_sums(const W& w, int wave, DecodeLds<UW>& s, float* o) {
    if (w.g == 0) {
        s.m[wave][w.col] = w.m;
        s.l[wave][w.col] = w.l;
    }
    if (w.col < w.cols) {
#pragma unroll
        for (int c = 0; c < W::NC; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < W::VEC; i += 4)
                    *reinterpret_cast<f32x4*>(&o[(wave * w.cols + w.col) * (DP + 4) + w.dim(c, j) + i]) =
                        f32x4{w.acc[c][i][j], w.acc[c][i + 1][j], w.acc[c][i + 2][j], w.acc[c][i + 3][j]};
    }
}

// Dims d .. d + 3 of head c over the waves, with their maximum and sum
template <int UW, int DP>
__device__ __forceinline__ f32x4 combine(const DecodeLds<UW>& s, const float* o, int cols, int c, int d, float& M, float& L) {
    M = -INFINITY;
    L = 0.0f;
#pragma unroll
    for (int v = 0; v < UW; ++v) M = fmaxf(M, s.m[v][c]);
    const float ref = M == -INFINITY ? 0.0f : M;
    f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int v = 0; v < UW; ++v) {
        const float f = __builtin_amdgcn_exp2f(s.m[v][c] - ref);
        L = fmaf(s.l[v][c], f, L);
        const f32x4 x = *reinterpret_cast<const f32x4*>(&o[(v * cols + c) * (DP + 4) + d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = fmaf(x[i], f, r[i]);
    }
    return r;
}

// One (sequence, KV head, 16 query heads) per workgroup of UW waves
template <typename T, int DP, bool CAP, bool BIAS, int UW>
__global__ __launch_bounds__(UW * 64) void paged_decode_unit_kernel(PagedAttnArgs a) {
    typedef DecodeWave<T, DP, CAP, BIAS> W;
    __shared__ DecodeLds<UW> s_w;
    extern __shared__ __attribute__((aligned(16))) float s_o[];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvb = a.kv_heads * ((a.group + kDecCols - 1) / kDecCols), b = blockIdx.x / kvb;
    const DecodeRow r = decode_row<W::KT>(a, b);
    if (r.seq < 0) return;
    W w;
    w.begin(a, b, blockIdx.x % kvb);
    w.walk(a, r, wave, r.walk.count(), UW);
    leave_sums<W, UW, DP>(w, wave, s_w, s_o);
    __syncthreads();
    const int quads = a.head_dim / 4;
    for (int u = tid; u < w.cols * quads; u += UW * 64) {
        const int c = u / quads, d = (u - c * quads) * 4;
        float M, L;
        const f32x4 o = combine<UW, DP>(s_w, s_o, w.cols, c, d, M, L);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            store_out(a, (const T*)nullptr, b, w.head0 + c, d + i, finish(o[i], L, r.gone, r.span.count() == 0));
    }
}

// A line of tiles cut into shares of q + 1 (the first `rem`) and q tiles
struct Shares {
    int n, q, rem;
    __device__ __forceinline__ Shares(int tiles, int shares) : n(shares), q(tiles / shares), rem(tiles % shares) {}
    __device__ __forceinline__ int begin(int s) const { return s * q + imin(s, rem); }
    __device__ __forceinline__ int of(int t) const {  // (q > 0)
        const int cut = rem * (q + 1);
        return t < cut ? t / (q + 1) : rem + (t - cut) / q;
    }
};

// Sums that waves on other XCDs read: written through to, and read from, where they all meet (sc1)
struct PartBuffer {
    __amdgpu_buffer_rsrc_t rs;
    __device__ __forceinline__ explicit PartBuffer(float* p) : rs(__builtin_amdgcn_make_buffer_rsrc(p, 0, 0x7fffffff, 0x00020000)) {}
    __device__ __forceinline__ void store(int i, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rs, i * 4, 0, 16);
    }
    __device__ __forceinline__ void store2(int i, float x, float y) const {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(x), __float_as_uint(y)}, rs, i * 4, 0, 16);
    }
    __device__ __forceinline__ f32x4 load(int i) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, i * 4, 0, 16));
    }
    __device__ __forceinline__ void load2(int i, float& x, float& y) const {
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, i * 4, 0, 16));
        x = __uint_as_float(v[0]);
        y = __uint_as_float(v[1]);
    }
};

// A workgroup joins the n shares from s0 on of row b's query heads head0 .. + live - 1, in a fixed
// order. o: its LDS of at least THREADS * 4 floats.
template <typename T, int THREADS>
__device__ __forceinline__ void join_row(const PagedAttnArgs& a, const PartBuffer& part, const PartBuffer& ml, int b, int head0,
                                         int live, int cols, int s0, int kvb, int kb, int n, float* o) {
    __shared__ float s_M[kDecCols], s_L[kDecCols];
    const int tid = threadIdx.x;
    const auto record = [&](int s, int c) { return (((s0 + s) * kvb + kb) * 2 + (s == 0)) * cols + c; };
    // maximum and sum of each head: 16 lanes of it, a share each
    for (int c = tid / 16; c < live; c += THREADS / 16) {
        float M = -INFINITY, L = 0.0f;
        for (int s = tid % 16; s < n; s += 16) {
            float m, l;
            ml.load2(2 * record(s, c), m, l);
            const float up = fmaxf(M, m), ref = up == -INFINITY ? 0.0f : up;
            L = L * __builtin_amdgcn_exp2f(M - ref) + l * __builtin_amdgcn_exp2f(m - ref);
            M = up;
        }
#pragma unroll
        for (int x = 1; x < 16; x *= 2) {
            const float m2 = __shfl_xor(M, x, 64), l2 = __shfl_xor(L, x, 64);
            const float up = fmaxf(M, m2), ref = up == -INFINITY ? 0.0f : up;
            L = L * __builtin_amdgcn_exp2f(M - ref) + l2 * __builtin_amdgcn_exp2f(m2 - ref);
            M = up;
        }
        if (tid % 16 == 0) {
            s_M[c] = M;
            s_L[c] = L;
        }
    }
    // 16 bytes of a record per thread; the groups of threads that hold one are dealt out over the
    // heads, then each head's over its shares, 4 in flight
    const int quads = a.head_dim / 4, groups = THREADS / quads, mine = tid / quads, d = (tid % quads) * 4;
    const int per = imax(1, groups / live);  // groups per head
    for (int c0 = 0; c0 < live; c0 += groups) {
        const int c = c0 + (per > 1 ? mine / per : mine), k0 = per > 1 ? mine % per : 0;
        const bool in = c < live && mine < groups && (per > 1 ? mine < per * live : true);
        f32x4 v[4];
        float m[4], l;
        const auto load = [&](int s) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int rec = record(imin(s + k * per, n - 1), c);
                v[k] = part.load(rec * a.head_dim + d);
                ml.load2(2 * rec, m[k], l);
            }
        };
        if (in) load(k0);
        __syncthreads();  // s_M, s_L; o is free
        if (in) {
            const float ref = s_M[c] == -INFINITY ? 0.0f : s_M[c];
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int s = k0; s < n; s += 4 * per) {
                if (s != k0) load(s);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (s + k * per < n) {
                        const float f = __builtin_amdgcn_exp2f(m[k] - ref);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum[i] = fmaf(v[k][i], f, sum[i]);
                    }
            }
            *reinterpret_cast<f32x4*>(&o[tid * 4]) = sum;
        }
        __syncthreads();
        if (in && k0 == 0) {
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int k = 0; k < imin(per, n); ++k) sum += *reinterpret_cast<const f32x4*>(&o[(tid + k * quads) * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i) store_out(a, (const T*)nullptr, b, head0 + c, d + i, finish(sum[i], s_L[c], false, false));
        }
    }
    __syncthreads();
}

// The shares of a call: all rows' tiles in a line (a row without any counts as one, so that a
// share meets it and writes its result)
template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(kDecWaves<DP> * 64) void paged_decode_share_kernel(PagedAttnArgs a) {
    constexpr int UW = kDecWaves<DP>, THREADS = UW * 64;
    typedef DecodeWave<T, DP, CAP, BIAS> W;
    __shared__ DecodeLds<UW> s_w;
    __shared__ int s_end[kPagedShareRows];  // tiles of rows 0 .. b
    __shared__ int s_sum[UW], s_last;
    extern __shared__ __attribute__((aligned(16))) float s_o[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // up to 64 rows: each wave holds one per lane (a reload costs 0.5 us before the first key)
    const bool few = a.batch <= 64;
    DecodeRow mine{-1, 0, false, {0, 0, 0, 0}, {0, 0, 0, 0}};
    int mine_end = 0;
    int total = 0;  // (the launcher sees to it that it fits)
    const auto scan = [&](int v) {  // inclusive, over the wave
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
            const int y = __shfl_up(v, x, 64);
            if (lane >= x) v += y;
        }
        return v;
    };
    if (few) {
        if (lane < a.batch) mine = decode_row<W::KT>(a, lane);
        mine_end = scan(lane < a.batch ? imax(mine.walk.count(), 1) : 0);
        total = __builtin_amdgcn_readlane(mine_end, 63);
    } else {
        constexpr int N = kPagedShareRows / THREADS;
        int n[N], sum = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {  // thread: rows N * tid .. + N - 1
            const int b = N * tid + k;
            n[k] = 0;
            if (b < a.batch) n[k] = imax(decode_row<W::KT>(a, b).walk.count(), 1);
            sum += n[k];
        }
        const int up = scan(sum);
        if (lane == 63) s_sum[wave] = up;
        __syncthreads();
        int before = up - sum;
#pragma unroll
        for (int w = 0; w < UW; ++w) before += w < wave ? s_sum[w] : 0;
#pragma unroll
        for (int w = 0; w < UW; ++w) total += __builtin_amdgcn_readfirstlane(s_sum[w]);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            before += n[k];
            if (N * tid + k < a.batch) s_end[N * tid + k] = before;
        }
        __syncthreads();
    }
    const auto row_end = [&](int b) {  // tiles of rows 0 .. b
        return b < 0 ? 0 : few ? __builtin_amdgcn_readlane(mine_end, b) : __builtin_amdgcn_readfirstlane(s_end[b]);
    };
    const int kvb = a.kv_heads * ((a.group + kDecCols - 1) / kDecCols);
    const int worker = blockIdx.x, share = worker / kvb, kb = worker % kvb;
    // 4 tiles in a share at least: a CU alone reads some 60 KB per us, so few keys are spread wide
    // (700 keys of 10 heads: 2 tiles 11.6 us, 4 11.2, 8 12.2)
    const Shares cut(total, imin((total + 3) / 4, a.n_splits));
    if (share >= cut.n) return;
    int at = cut.begin(share);
    const int end = cut.begin(share + 1);
    // the row that tile `at` belongs to
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (row_end(mid) > at) hi = mid;
        else lo = mid + 1;
    }
    // a workspace that was never set up has no counters to go by: NaN
    const bool unfit = a.counters && a.counters[-1] != kPagedMagic;
    const PartBuffer part(a.part), ml(a.part_ml);
    const int quads = a.head_dim / 4;
    W w;
    for (int b = lo; at < end; ++b) {
        const int b_begin = row_end(b - 1), b_end = row_end(b), stop = imin(end, b_end);
        const DecodeRow r = few ? row_of_lane(mine, b) : decode_row<W::KT>(a, b);
        const bool whole = (at == b_begin && stop == b_end) || unfit;
        int s0 = -1, n = 0;
        if (!whole) {
            s0 = cut.of(b_begin);
            n = cut.of(b_end - 1) - s0 + 1;
        }
        if (!a.counters && kb == 0 && tid == 0 && at == b_begin) {  // for the join kernel (-1: nothing to join)
            a.part_rows[2 * b] = r.seq < 0 ? -1 : s0;
            a.part_rows[2 * b + 1] = s0 + n - 1;
        }
        if (r.seq >= 0) {
            w.begin(a, b, kb);
            w.walk(a, r, at - b_begin + wave, imin(stop - b_begin, r.walk.count()), UW);
            leave_sums<W, UW, DP>(w, wave, s_w, s_o);
            __syncthreads();
            // whole: the result; else this share's sums: its first row's (begun by an earlier
            // share) or its last's (a later one goes on)
            const int cols = imin(a.group, kDecCols), rec0 = (worker * 2 + (at == b_begin)) * cols;
            for (int u = tid; u < w.cols * quads; u += THREADS) {
                const int c = u / quads, d = (u - c * quads) * 4;
                float M, L;
                const f32x4 o = combine<UW, DP>(s_w, s_o, w.cols, c, d, M, L);
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        store_out(a, (const T*)nullptr, b, w.head0 + c, d + i,
                                  finish(o[i], L, r.gone || unfit, r.span.count() == 0));
                } else {
                    part.store((rec0 + c) * a.head_dim + d, o);
                    if (d == 0) ml.store2(2 * (rec0 + c), M, L);
                }
            }
            if (!whole && a.counters) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the sums are where the other XCDs see them
                __syncthreads();
                int* counter = a.counters + b * kvb + kb;
                if (tid == 0) {
                    const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    if (before == n - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    s_last = before == n - 1;
                }
                __syncthreads();
                if (s_last) join_row<T, THREADS>(a, part, ml, b, w.head0, w.cols, cols, s0, kvb, kb, n, s_o);
            } else {
                __syncthreads();  // s_w, s_o are free
            }
        }
        at = stop;
    }
}

// Joins the shares of each (row, head) that more than one has tiles of: 16 bytes of a record per
// thread, as many records side by side as there are threads for, 4 of each in flight; the
// shares in a fixed order.
constexpr int kJoinThreads = 256;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void paged_decode_join_kernel(PagedAttnArgs a) {
    __shared__ __attribute__((aligned(16))) float s_o[kJoinThreads * 4];
    const int head = blockIdx.x % a.heads, b = blockIdx.x / a.heads, tid = threadIdx.x, lane = tid & 63;
    const int first = a.part_rows[2 * b], n = a.part_rows[2 * b + 1] - first + 1;
    if (first < 0) return;
    const int blocks = (a.group + kDecCols - 1) / kDecCols, kvb = a.kv_heads * blocks;
    const int kvh = head / a.group, in_group = head % a.group;
    const int kb = kvh * blocks + in_group / kDecCols, cols = imin(a.group, kDecCols), col = in_group % kDecCols;
    const auto record = [&](int s) { return ((size_t)((first + s) * kvb + kb) * 2 + (s == 0)) * cols + col; };
    const int quads = a.head_dim / 4, side = kJoinThreads / quads, mine = tid / quads, d = (tid % quads) * 4;
    constexpr int F = 4;
    f32x4 v[F];
    float vm[F];
    const auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < F; ++k) {
            const size_t rec = record(imin(s0 + k * side, n - 1));
            v[k] = *reinterpret_cast<const f32x4*>(a.part + rec * a.head_dim + d);
            vm[k] = a.part_ml[2 * rec];
        }
    };
    load(mine);
    float M = -INFINITY, L = 0.0f;
    for (int s = lane; s < n; s += 64) M = fmaxf(M, a.part_ml[2 * record(s)]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x, 64));
    const float ref = M == -INFINITY ? 0.0f : M;
    for (int s = lane; s < n; s += 64) L = fmaf(a.part_ml[2 * record(s) + 1], __builtin_amdgcn_exp2f(a.part_ml[2 * record(s)] - ref), L);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) L += __shfl_xor(L, x, 64);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine < side) {
        for (int s0 = mine; s0 < n; s0 += F * side) {
            if (s0 != mine) load(s0);
#pragma unroll
            for (int k = 0; k < F; ++k)
                if (s0 + k * side < n) {
                    const float w = __builtin_amdgcn_exp2f(vm[k] - ref);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = fmaf(v[k][i], w, o[i]);
                }
        }
        *reinterpret_cast<f32x4*>(&s_o[mine * a.head_dim + d]) = o;
    }
    __syncthreads();
    if (tid < a.head_dim) {
        float sum = 0.0f;
        for (int k = 0; k < imin(side, n); ++k) sum += s_o[k * a.head_dim + tid];
        store_out(a, (const T*)nullptr, b, head, tid, finish(sum, L, false, false));
    }
}

template <typename T, int DP, int UW>
void launch_unit(const PagedAttnArgs& a, hipStream_t st) {
    const bool cap = a.sc.cap2 > 0.0f, bias = a.sc.slopes != nullptr;
    const dim3 grid((unsigned)a.batch * a.kv_heads * ((a.group + kDecCols - 1) / kDecCols)), block(UW * 64);
    const uint32_t lds = UW * std::min(a.group, kDecCols) * (DP + 4) * sizeof(float);
    if (cap && bias) launch_k(paged_decode_unit_kernel<T, DP, true, true, UW>, grid, block, lds, st, a);
    else if (cap) launch_k(paged_decode_unit_kernel<T, DP, true, false, UW>, grid, block, lds, st, a);
    else if (bias) launch_k(paged_decode_unit_kernel<T, DP, false, true, UW>, grid, block, lds, st, a);
    else launch_k(paged_decode_unit_kernel<T, DP, false, false, UW>, grid, block, lds, st, a);
}

template <typename T, int DP>
void launch_dp(const PagedAttnArgs& a, hipStream_t st) {
    const int kvb = a.kv_heads * ((a.group + kDecCols - 1) / kDecCols);
    const bool cap = a.sc.cap2 > 0.0f, bias = a.sc.slopes != nullptr;
    const dim3 block(kDecWaves<DP> * 64);
    // (the join takes 16 bytes per thread)
    const uint32_t lds = std::max<uint32_t>(kDecWaves<DP> * std::min(a.group, kDecCols) * (DP + 4) * sizeof(float), block.x * 16);
    if (!a.n_splits) {
        if (a.unit_waves == 1) launch_unit<T, DP, 1>(a, st);
        else launch_unit<T, DP, kDecWaves<DP>>(a, st);
        return;
    }
    const dim3 grid((unsigned)a.n_splits * kvb);
    if (cap && bias) launch_k(paged_decode_share_kernel<T, DP, true, true>, grid, block, lds, st, a);
    else if (cap) launch_k(paged_decode_share_kernel<T, DP, true, false>, grid, block, lds, st, a);
    else if (bias) launch_k(paged_decode_share_kernel<T, DP, false, true>, grid, block, lds, st, a);
    else launch_k(paged_decode_share_kernel<T, DP, false, false>, grid, block, lds, st, a);
    if (!a.counters) launch_k(paged_decode_join_kernel<T>, dim3((unsigned)a.batch * a.heads), dim3(kJoinThreads), 0, st, a);
}

template <typename T>
void launch_decode(const PagedAttnArgs& a, hipStream_t st) {
    if (a.head_dim <= 64) launch_dp<T, 64>(a, st);
    else if (a.head_dim <= 128) launch_dp<T, 128>(a, st);
    else launch_dp<T, 256>(a, st);
}

}  // namespace

int launch_paged_decode(PagedAttnArgs a, int dtype, long long max_keys, void* ws, size_t ws_bytes, hipStream_t st) {
    const DecodePlan p = paged_decode_plan(a.batch, a.heads, a.kv_heads, dtype == UOCR_HIP_DTYPE_F32 ? 16 : 32, max_keys,
                                           std::min<long long>(a.c.capacity(), INT_MAX));
    a.n_splits = p.shares;
    a.unit_waves = p.unit_waves;
    if ((long long)a.batch * a.kv_heads * p.blocks >= 1 << 23)  // (a launch has fewer than 2^32 threads)
        return set_error(UOCR_HIP_EUNSUPPORTED, "attention: batch too large");
    if (p.shares)
        if (int rc = paged_take_workspace(a, p.records, a.batch, ws, ws_bytes)) return rc;
    // a workgroup joins up to 256 KiB in less time than a launch takes
    if ((long long)(p.shares / a.batch + 2) * std::min(a.group, kDecCols) * a.head_dim * 4 > 256 << 10) a.counters = nullptr;
    if (dtype == UOCR_HIP_DTYPE_F32) launch_decode<float>(a, st);
    else if (dtype == UOCR_HIP_DTYPE_BF16) launch_decode<bf16>(a, st);
    else launch_decode<f16>(a, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UOCR_HIP_OK
                           : set_error(UOCR_HIP_EHIP, std::string("paged decode launch: ") + hipGetErrorString(e));
}

}  // namespace uocr_hip
