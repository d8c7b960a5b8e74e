// Device pieces and argument blocks of the paged attention kernels.
#pragma once
#include <hip/hip_runtime.h>

#include "common.hpp"
#include "paged.hpp"

namespace uocr_hip {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;

// Rows of heads; strides in bytes
struct PagedRows {
    char* p;
    long long row_bytes, head_bytes;
};

// Scores in units of log 2 (the softmax runs on exp2), with log2(e) folded into the constants
struct PagedScores {
    float scale2;   // scale log2(e)
    float cap2;     // softcap log2(e); 0: no cap
    float in, in2;  // scale / softcap, and 2 log2(e) of that
    const float* slopes;  // [heads] or null
    int negative;   // scale < 0
};

struct PagedAttnArgs {
    PagedCache c;
    PagedRows q, out;
    int out_f32;
    int rows, batch, heads, kv_heads, head_dim, group;
    const int* q_start;  // (prefill) [batch + 1]
    const int* seqs;     // [batch] or null
    const int* kv_len;   // [n_seqs]
    PagedScores sc;
    MaskArgs mask;
    int n_splits;  // prefill: splits of the keys; decode: shares (0: one workgroup per unit)
    float* part;   // partial results: sums of p v [records][head_dim], then
    float* part_ml;  // [records][2]: maximum and sum, then
    int* counters;   // (decode) [batch][KV heads x blocks of 16 heads]: sums that are there (0 between calls);
                     // the workspace's first word before them. Null: joined by a kernel of its own
    int* part_rows;  // (decode) [batch][2]: first and last share with tiles of a row
    int unit_waves;  // (decode) waves of such a workgroup: 1, or as many as there are
    int n_tiles;   // (prefill) query tiles that the grid has room for
};

__device__ __forceinline__ f32x4 mfma_16x16x32(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_16x16x32(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_16x16x4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_32x32x16(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_32x32x16(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_32x32x2(float a, float b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

template <typename T> struct Vec8;
template <> struct Vec8<f16> { typedef f16x8 type; };
template <> struct Vec8<bf16> { typedef bf16x8 type; };
template <> struct Vec8<float> { typedef f32x4 type; };  // (16 bytes of it)

template <typename V>
__device__ __forceinline__ V as_vec(u32x4 w) {
    V v;
    __builtin_memcpy(&v, &w, 16);
    return v;
}

__device__ __forceinline__ long long shfl64(long long v, int src) {
    const int lo = __shfl((int)(uint32_t)v, src, 64), hi = __shfl((int)(v >> 32), src, 64);
    return (long long)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

// Score of a visible pair; dist: positions between query and key (for the bias)
template <bool CAP, bool BIAS, bool EXACT>
__device__ __forceinline__ float score2(float qk, const PagedScores& sc, float slope2, float dist) {
    float s;
    if constexpr (!CAP) s = qk * sc.scale2;
    else if constexpr (EXACT) s = sc.cap2 * tanhf(qk * sc.in);
    // tanh x = 1 - 2 / (e^2x + 1): absolute error below 2^-22, a step of f16 scores of 1024
    else s = fmaf(-2.0f * sc.cap2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(qk * sc.in2) + 1.0f), sc.cap2);
    if constexpr (BIAS) s = fmaf(-slope2, fabsf(dist), s);
    return s;
}

__device__ __forceinline__ void store_out(const PagedAttnArgs& a, const bf16*, int row, int head, int d, float v) {
    char* p = a.out.p + row * a.out.row_bytes + head * a.out.head_bytes;
    if (a.out_f32) reinterpret_cast<float*>(p)[d] = v;
    else reinterpret_cast<bf16*>(p)[d] = (bf16)v;
}
__device__ __forceinline__ void store_out(const PagedAttnArgs& a, const f16*, int row, int head, int d, float v) {
    char* p = a.out.p + row * a.out.row_bytes + head * a.out.head_bytes;
    if (a.out_f32) reinterpret_cast<float*>(p)[d] = v;
    else reinterpret_cast<f16*>(p)[d] = (f16)v;
}
__device__ __forceinline__ void store_out(const PagedAttnArgs& a, const float*, int row, int head, int d, float v) {
    reinterpret_cast<float*>(a.out.p + row * a.out.row_bytes + head * a.out.head_bytes)[d] = v;
}

// One (row, head) by one wave, straight from the definition: 64 keys at a time,
// a key per lane for the scores, dims over the lanes for the sums. f32
// throughout; nothing that the row does not see is read.
template <typename T>
__device__ void row_attention(const PagedAttnArgs& a, int seq, int row, int head, int pos, int len, bool lost) {
    const int lane = threadIdx.x & 63, D = a.head_dim, kvh = head / a.group;
    const Span span = row_span(a.mask.causal, a.mask.window, a.mask.both_ways, pos, len,
                               a.mask.prefix_len ? a.mask.prefix_len[seq] : 0, a.mask.key_begin ? a.mask.key_begin[row] : 0,
                               a.mask.key_end ? a.mask.key_end[row] : len);
    const T* q = reinterpret_cast<const T*>(a.q.p + row * a.q.row_bytes + head * a.q.head_bytes);
    const char* kbase = a.c.k + kvh * a.c.head_bytes;
    const char* vbase = a.c.v + kvh * a.c.head_bytes;
    const float slope2 = a.sc.slopes ? a.sc.slopes[head] * kLog2e : 0.0f;
    const TileWalk w = tile_walk<64>(span);
    float m = -INFINITY, l = 0.0f, acc[4] = {};
    for (int t = 0; t < w.count(); ++t) {
        const bool first = t < w.n0;
        const int j = (first ? w.t0 + t : w.t1 + t - w.n0) * 64 + lane;
        const bool in = j >= (first ? span.b0 : span.b1) && j < (first ? span.e0 : span.e1);
        const long long off = in ? a.c.offset(seq, j) : -1;
        float s = -INFINITY;
        if (in) {
            s = NAN;
            if (off >= 0) {
                const T* k = reinterpret_cast<const T*>(kbase + off);
                float x = 0.0f;
                for (int d = 0; d < D; ++d) x = fmaf((float)q[d], (float)k[d], x);
                const float dist = (float)(pos - j);
                s = a.sc.cap2 > 0.0f ? score2<true, true, true>(x, a.sc, slope2, dist)
                                        : score2<false, true, true>(x, a.sc, slope2, dist);
            }
        }
        float top = fmaxf(m, s);
#pragma unroll
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
        const float ref = top == -INFINITY ? 0.0f : top;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = top;
        const float p = in ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
        l = fmaf(l, alpha, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= alpha;
        for (uint64_t left = __ballot(in && off >= 0); left; left &= left - 1) {
            const int src = __builtin_ctzll(left);
            const T* v = reinterpret_cast<const T*>(vbase + shfl64(off, src));
            const float pj = __shfl(p, src, 64);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < D) acc[i] = fmaf(pj, (float)v[lane + 64 * i], acc[i]);
        }
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x, 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float o = acc[i] / l;
        if (l == 0.0f) o = span.count() == 0 ? 0.0f : NAN;
        // (l is NaN where a key has no page; a sum may be NaN on its own)
        if (lane + 64 * i < D) store_out(a, (const T*)nullptr, row, head, lane + 64 * i, lost ? NAN : o);
    }
}

}  // namespace uocr_hip
