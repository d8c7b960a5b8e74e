// Attention of one new token per sequence over a paged KV cache, split over the
// cache's length and joined.
//
// For query head h over the visible keys j: p_j = exp2(s_j - max s), out = sum p_j v_j /
// sum p_j. Every visible K and V row is read once per group of query heads
// that share it (up to 16), so the call is bound by HBM.
//
// A workgroup of 4 waves takes one (sequence, KV head, split); its waves take
// the split's tiles of 32 keys (16 for f32) in turn, each with a running
// maximum and sum, and are combined in LDS. The products run on MFMA
// with up to 16 query heads as one side, also for a single head: at 16 KiB per tile the
// matrix cores are busy for about a tenth of the time that the tile's bytes take, and nothing
// moves between lanes:
//   * S = K Q^T: lane (i, g) = (lane % 16, lane / 16) holds 8 dims of key i, straight from
//     its page, and of head i. D has head i, keys 4g .. 4g + 3 of each 16.
//   * O^T = V^T P^T: those keys are taken as the k-slots of group g, so the
//     probabilities are an operand where they are. Lane (i, g) loads V rows of its
//     group's 8 keys, 8 dims each (16 lanes: one row), and transposes the 8 x 8 block in its
//     registers (32 v_perm_b32): MFMA e takes dims 8i + e.
// 16-bit probabilities go in as two halves (p and its rounding error), since the matrix cores
// have room for it: the result is as exact as with f32 probabilities.
#include <hip/hip_runtime.h>

#include "launch.hpp"
#include "paged_device.hpp"
#include "paged_host.hpp"

namespace uocr_hip {
namespace {

constexpr int kDecWaves = 4;
constexpr int kDecCols = 16;  // query heads per workgroup

template <typename T>
constexpr int kDecKeys = sizeof(T) == 4 ? 16 : 32;  // keys per tile

// One row's split: which keys, how many splits of them there are
struct DecodeRow {
    int seq, len;
    bool lost;  // kv_len is beyond the table's room
    Span span;
    TileWalk walk;
    int splits, chunk;  // tiles in each
};

template <int KT>
__device__ __forceinline__ DecodeRow decode_row(const PagedAttnArgs& a, int b) {
    DecodeRow r;
    r.seq = a.seqs ? a.seqs[b] : b;
    if ((uint32_t)r.seq >= (uint32_t)a.c.n_seqs) {
        r.seq = -1;
        return r;
    }
    r.len = a.kv_len[r.seq];
    r.lost = r.len > a.c.capacity();
    const int len = r.lost ? 0 : imax(r.len, 0);
    r.span = row_span(1, a.mask.window, 0, len - 1, len, a.mask.prefix_len ? a.mask.prefix_len[r.seq] : 0,
                      a.mask.key_begin ? a.mask.key_begin[b] : 0, a.mask.key_end ? a.mask.key_end[b] : len);
    r.walk = tile_walk<KT>(r.span);
    // (more keys than the launcher was told of: larger splits)
    r.chunk = imax(a.chunk, (r.walk.count() + a.n_splits - 1) / a.n_splits);
    r.splits = imax(1, (r.walk.count() + r.chunk - 1) / r.chunk);
    return r;
}

// What a row's result is where its weights sum to 0 or it has none to look at
__device__ __forceinline__ float finish(float acc, float l, const DecodeRow& r) {
    if (r.lost) return NAN;
    if (l > 0.0f) return acc / l;
    return l == 0.0f && r.span.count() == 0 ? 0.0f : NAN;
}

template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(kDecWaves * 64) void paged_decode_kernel(PagedAttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int KT = kDecKeys<T>, KB = KT / 16;
    constexpr int VEC = DP == 64 || F32 ? 4 : 8;     // dims of a V row per lane and load
    constexpr int NC = DP / (16 * VEC);              // such loads
    constexpr int KS = F32 ? DP / 16 : DP / 32;      // 16-byte loads of a K row per lane
    constexpr int KD = F32 ? 4 : 8;                  // dims in each
    constexpr int VR = KT / 4;                       // V rows per lane
    typedef typename Vec8<T>::type vec_t;
    __shared__ float s_m[kDecWaves][kDecCols], s_l[kDecWaves][kDecCols];
    __shared__ __attribute__((aligned(16))) float s_o[kDecWaves][kDecCols][DP + 4];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int blocks = (a.group + kDecCols - 1) / kDecCols;  // blocks of heads per KV head
    int idx = blockIdx.x;
    const int hb = idx % blocks;
    idx /= blocks;
    const int kvh = idx % a.kv_heads;
    idx /= a.kv_heads;
    const int split = idx % a.n_splits, b = idx / a.n_splits;
    const DecodeRow r = decode_row<KT>(a, b);
    if (r.seq < 0 || split >= r.splits) return;
    const int cols = imin(kDecCols, a.group - hb * kDecCols), head0 = kvh * a.group + hb * kDecCols;
    const int head = head0 + imin(col, cols - 1);
    const int n = r.walk.count();
    const int t_begin = split * r.chunk, t_end = imin(n, t_begin + r.chunk);

    vec_t q[KS];
    {
        const char* qp = a.q.p + b * a.q.row_bytes + head * a.q.head_bytes;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * (4 * KD) + g * KD;
            const bool in = d < a.head_dim && col < cols;
            const u32x4 w = *reinterpret_cast<const u32x4*>(qp + (in ? d : 0) * sizeof(T));
            q[s] = as_vec<vec_t>(in ? w : u32x4{0, 0, 0, 0});
        }
    }
    float slope2 = 0.0f;
    if constexpr (BIAS) slope2 = a.sc.slopes[head] * kLog2e;

    float m, l;
    f32x4 acc[NC][VEC];
    const char* kbase = a.c.k + kvh * a.c.head_bytes;
    const char* vbase = a.c.v + kvh * a.c.head_bytes;
    for (bool halves = true;; halves = false) {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[c][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int t = t_begin + wave; t < t_end; t += kDecWaves) {
        const bool first = t < r.walk.n0;
        const int base = (first ? r.walk.t0 + t : r.walk.t1 + t - r.walk.n0) * KT;
        const int kb = first ? r.span.b0 : r.span.b1, ke = first ? r.span.e0 : r.span.e1;
        const int my = base + (lane & (KT - 1));
        const bool in = my >= kb && my < ke;
        const long long at = in ? a.c.offset(r.seq, my) : 0;
        const uint32_t seen = (uint32_t)__ballot(in) & (uint32_t)((1ull << KT) - 1);
        const uint32_t lost = (uint32_t)__ballot(at < 0) & (uint32_t)((1ull << KT) - 1);
        const long long off = at < 0 ? 0 : at;
        // K rows, then V rows, all in flight together
        u32x4 kw[KB][KS];
        uint32_t vw[NC][VR][VEC * sizeof(T) / 4];
#pragma unroll
        for (int h = 0; h < KB; ++h) {
            const char* kp = kbase + shfl64(off, h * 16 + col);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = s * (4 * KD) + g * KD;
                kw[h][s] = *reinterpret_cast<const u32x4*>(kp + (DP == 64 || d < a.head_dim ? imin(d, a.head_dim - KD) : 0) * sizeof(T));
            }
        }
#pragma unroll
        for (int e = 0; e < VR; ++e) {
            const int key = F32 ? g * 4 + e : (e >> 2) * 16 + g * 4 + (e & 3);
            const char* vp = vbase + shfl64(off, key);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = c * 16 * VEC + col * VEC;
                __builtin_memcpy(vw[c][e], __builtin_assume_aligned(vp + imin(d, a.head_dim - VEC) * sizeof(T), VEC * sizeof(T)), VEC * sizeof(T));
            }
        }
        // scores: keys h * 16 + g * 4 + r of head col
        float p[KB][4];
        float top = m;
#pragma unroll
        for (int h = 0; h < KB; ++h) {
            f32x4 s = {};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                u32x4 w = kw[h][k];
                if (k * (4 * KD) + g * KD >= a.head_dim) w = u32x4{0, 0, 0, 0};  // (past the head: 0 on both sides)
                const vec_t kv = as_vec<vec_t>(w);
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s = mfma_16x16x4(kv[e], q[k][e], s);
                } else {
                    s = mfma_16x16x32(kv, q[k], s);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = h * 16 + g * 4 + i;
                float x = score2<CAP, BIAS, true>(s[i], a.sc, slope2, r.len - 1 - (base + key));
                if (lost >> key & 1) x = NAN;
                p[h][i] = seen >> key & 1 ? x : -INFINITY;
                top = fmaxf(top, p[h][i]);
            }
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
        if (seen != (uint32_t)((1ull << KT) - 1)) {
#pragma unroll
            for (int e = 0; e < VR; ++e) {
                const int key = F32 ? g * 4 + e : (e >> 2) * 16 + g * 4 + (e & 3);
                const bool keep = seen >> key & 1;
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
    }
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

    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
        s_m[wave][col] = m;
        s_l[wave][col] = l;
    }
    if (col < cols) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < VEC; i += 4)
                    *reinterpret_cast<f32x4*>(&s_o[wave][col][c * 16 * VEC + (g * 4 + j) * VEC + i]) =
                        f32x4{acc[c][i][j], acc[c][i + 1][j], acc[c][i + 2][j], acc[c][i + 3][j]};
    }
    __syncthreads();
    const bool alone = r.splits == 1;
    for (int u = tid; u < cols * a.head_dim; u += kDecWaves * 64) {
        const int c = u / a.head_dim, d = u - c * a.head_dim;
        float M = -INFINITY, L = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecWaves; ++w) M = fmaxf(M, s_m[w][c]);
        const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < kDecWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][c] - ref);
            L = fmaf(s_l[w][c], f, L);
            o = fmaf(s_o[w][c][d], f, o);
        }
        if (alone) {
            store_out(a, (const T*)nullptr, b, head0 + c, d, finish(o, L, r));
        } else {
            const size_t rec = ((size_t)b * a.heads + head0 + c) * a.n_splits + split;
            a.part[rec * a.head_dim + d] = o;
            if (d == 0) {
                a.part_ml[2 * rec] = M;
                a.part_ml[2 * rec + 1] = L;
            }
        }
    }
}

// Joins the splits of each (row, head), in their order.
template <typename T>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(PagedAttnArgs a) {
    const int head = blockIdx.x % a.heads, b = blockIdx.x / a.heads;
    const DecodeRow r = decode_row<kDecKeys<T>>(a, b);
    if (r.seq < 0 || r.splits == 1) return;
    const size_t rec = ((size_t)b * a.heads + head) * a.n_splits;
    float M = -INFINITY;
    for (int s = 0; s < r.splits; ++s) M = fmaxf(M, a.part_ml[2 * (rec + s)]);
    const float ref = M == -INFINITY ? 0.0f : M;
    for (int d = threadIdx.x; d < a.head_dim; d += blockDim.x) {
        float L = 0.0f, o = 0.0f;
        for (int s = 0; s < r.splits; ++s) {
            const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * (rec + s)] - ref);
            L = fmaf(a.part_ml[2 * (rec + s) + 1], f, L);
            o = fmaf(a.part[(rec + s) * a.head_dim + d], f, o);
        }
        store_out(a, (const T*)nullptr, b, head, d, finish(o, L, r));
    }
}

template <typename T, int DP>
void launch_dp(const PagedAttnArgs& a, dim3 grid, hipStream_t st) {
    const dim3 block(kDecWaves * 64);
    const bool cap = a.sc.softcap > 0.0f, bias = a.sc.slopes != nullptr;
    if (cap && bias) launch_k(paged_decode_kernel<T, DP, true, true>, grid, block, 0, st, a);
    else if (cap) launch_k(paged_decode_kernel<T, DP, true, false>, grid, block, 0, st, a);
    else if (bias) launch_k(paged_decode_kernel<T, DP, false, true>, grid, block, 0, st, a);
    else launch_k(paged_decode_kernel<T, DP, false, false>, grid, block, 0, st, a);
}

template <typename T>
void launch_decode(const PagedAttnArgs& a, hipStream_t st) {
    const int blocks = (a.group + kDecCols - 1) / kDecCols;
    const dim3 grid((unsigned)((long long)a.batch * a.n_splits * a.kv_heads * blocks));
    if (a.head_dim <= 64) launch_dp<T, 64>(a, grid, st);
    else if (a.head_dim <= 128) launch_dp<T, 128>(a, grid, st);
    else launch_dp<T, 256>(a, grid, st);
    if (a.n_splits > 1)
        launch_k(paged_decode_join_kernel<T>, dim3((unsigned)a.batch * a.heads), dim3((a.head_dim + 63) / 64 * 64), 0,
                 st, a);
}

}  // namespace

int launch_paged_decode(PagedAttnArgs a, int dtype, long long max_keys, void* ws, size_t ws_bytes, hipStream_t st) {
    const int blocks = (a.group + kDecCols - 1) / kDecCols;
    const long long units = (long long)a.batch * a.kv_heads * blocks;
    const int kt = dtype == UOCR_HIP_DTYPE_F32 ? 16 : 32;
    const long long tiles = std::max(1ll, (max_keys + kt - 1) / kt);
    a.n_splits = paged_splits(units, tiles);
    a.chunk = (int)((tiles + a.n_splits - 1) / a.n_splits);
    if (int rc = paged_take_workspace(a, a.batch, ws, ws_bytes)) return rc;
    if (units * a.n_splits > INT_MAX) return set_error(UOCR_HIP_EUNSUPPORTED, "attention: batch too large");
    if (dtype == UOCR_HIP_DTYPE_F32) launch_decode<float>(a, st);
    else if (dtype == UOCR_HIP_DTYPE_BF16) launch_decode<bf16>(a, st);
    else launch_decode<f16>(a, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UOCR_HIP_OK
                           : set_error(UOCR_HIP_EHIP, std::string("paged decode launch: ") + hipGetErrorString(e));
}

}  // namespace uocr_hip
