// Rotary positions of q and k, alone or with the append of K and V to a paged cache.
//
// A pair (a, b) of row t turns by positions[t] * inv_freq[i]. The angle is
// reduced to a fraction of a turn in 64 bits (an f32 product is off by up to
// 0.03 rad at position 10^6), sine and cosine of that are f32. Bound by the bytes: each
// element is read and written once; the sines of a row are computed once in LDS for all
// heads. One workgroup per row: 8 elements (16-byte accesses for 16-bit types) per thread and
// step, the rotated half and its partner in one thread, so q_out may be q. 8192 rows of 48 heads of
// 128: bf16 32 us, 6.2 TB/s read and written; f32 79 us, 5.1. Stores past the caches (nontemporal) take calls of
// more than 32 MB from 48 to 41 us, but the attention that follows then reads q and K from memory: 3000 rows of 32 heads
// over 8 together 145 us instead of 132, 8192 rows 701 instead of 697.
#include <hip/hip_runtime.h>

#include <initializer_list>

#include "paged_host.hpp"

namespace uocr_hip {
namespace {

constexpr int kRopeThreads = 256;

struct RopeArgs {
    PagedRows q, k, v, qo, ko;  // (append: ko unused)
    int rows, heads, kv_heads, head_dim;
    const int* positions;
    const float* freq;
    int rotary, interleaved;
    float factor;
    int append;
    PagedCache c;
    const int* seqs;
    const int* at;
};

template <typename T, int N>
__device__ __forceinline__ void load_n(const char* p, float (&x)[N]) {
    T t[N];
    __builtin_memcpy(t, N == 1 ? p : (const char*)__builtin_assume_aligned(p, 16), N * sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)t[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_n(char* p, const float (&x)[N]) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)x[i];
    __builtin_memcpy(N == 1 ? p : (char*)__builtin_assume_aligned(p, 16), t, N * sizeof(T));
}

// One row. TI, TO: types in and out; N: elements per access (8, or 1 where alignment or sizes ask for it)
template <typename TI, typename TO, int N>
__device__ __forceinline__ void rope_row(const RopeArgs& a, int t, float* s_cos, float* s_sin) {
    const int tid = threadIdx.x, half = a.rotary / 2, D = a.head_dim;
    long long page = -1;
    if (a.append) {
        const int seq = a.seqs[t];
        if ((uint32_t)seq >= (uint32_t)a.c.n_seqs) return;  // padding
        const int at = a.at[t];
        if (at >= 0 && at < a.c.capacity()) page = a.c.offset(seq, at);
    }
    if (half) {
        const double pos = (double)a.positions[t];
        for (int i = tid; i < half; i += kRopeThreads) {
            const double turns = pos * (double)a.freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
            const float f = (float)(turns - rint(turns));
            float sn, cs;
            sincospif(2.0f * f, &sn, &cs);
            s_cos[i] = cs * a.factor;
            s_sin[i] = sn * a.factor;
        }
        __syncthreads();
    }
    // work per head: `half / N` units of pairs (interleaved: 2N elements side by
    // side), then (D - rotary) / N units to copy; V heads: D / N units
    const int pairs = half / N, units = pairs + (D - a.rotary) / N;
    const int n_qk = (a.heads + a.kv_heads) * units, n_v = a.append ? a.kv_heads * (D / N) : 0;
    for (int u = tid; u < n_qk + n_v; u += kRopeThreads) {
        if (u >= n_qk) {
            const int h = (u - n_qk) / (D / N), d = ((u - n_qk) - h * (D / N)) * N;
            if (page < 0) continue;
            float x[N];
            load_n<TI, N>(a.v.p + t * a.v.row_bytes + h * a.v.head_bytes + d * sizeof(TI), x);
            store_n<TO, N>(a.c.v + page + h * a.c.head_bytes + d * sizeof(TO), x);
            continue;
        }
        const int h = u / units, j = u - h * units;
        const bool is_q = h < a.heads;
        const int hk = h - a.heads;
        const char* src = is_q ? a.q.p + t * a.q.row_bytes + h * a.q.head_bytes : a.k.p + t * a.k.row_bytes + hk * a.k.head_bytes;
        char* dst;
        if (is_q) dst = a.qo.p + t * a.qo.row_bytes + h * a.qo.head_bytes;
        else if (a.append) {
            if (page < 0) continue;
            dst = a.c.k + page + hk * a.c.head_bytes;
        } else dst = a.ko.p + t * a.ko.row_bytes + hk * a.ko.head_bytes;
        if (j >= pairs) {
            const int d = a.rotary + (j - pairs) * N;
            float x[N];
            load_n<TI, N>(src + d * sizeof(TI), x);
            store_n<TO, N>(dst + d * sizeof(TO), x);
        } else {
            const int i0 = j * N;
            const int d0 = a.interleaved ? 2 * i0 : i0, d1 = a.interleaved ? 2 * i0 + N : i0 + half;
            float x[N], y[N];
            load_n<TI, N>(src + d0 * sizeof(TI), x);
            load_n<TI, N>(src + d1 * sizeof(TI), y);
            if (a.interleaved && N > 1) {
                // pairs 2e, 2e + 1 of x, then of y
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const float c0 = s_cos[i0 + e], n0 = s_sin[i0 + e], c1 = s_cos[i0 + N / 2 + e], n1 = s_sin[i0 + N / 2 + e];
                    const float p0 = x[2 * e], p1 = x[2 * e + 1], r0 = y[2 * e], r1 = y[2 * e + 1];
                    x[2 * e] = p0 * c0 - p1 * n0;
                    x[2 * e + 1] = p1 * c0 + p0 * n0;
                    y[2 * e] = r0 * c1 - r1 * n1;
                    y[2 * e + 1] = r1 * c1 + r0 * n1;
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float c0 = s_cos[i0 + e], n0 = s_sin[i0 + e], p0 = x[e], p1 = y[e];
                    x[e] = p0 * c0 - p1 * n0;
                    y[e] = p1 * c0 + p0 * n0;
                }
            }
            store_n<TO, N>(dst + d0 * sizeof(TO), x);
            store_n<TO, N>(dst + d1 * sizeof(TO), y);
        }
    }
}

template <typename TI, typename TO, int N>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
    __shared__ float s_cos[128], s_sin[128];
    for (long long t = blockIdx.x; t < a.rows; t += gridDim.x) {
        if (t != blockIdx.x) __syncthreads();  // (the last row's sines are read)
        rope_row<TI, TO, N>(a, (int)t, s_cos, s_sin);
    }
}

template <typename TI, typename TO>
void launch_n(const RopeArgs& a, bool vec, hipStream_t st) {
    const dim3 grid(std::min(a.rows, 1 << 22)), block(kRopeThreads);  // (a launch has fewer than 2^32 threads)
    if (vec) launch_k(rope_kernel<TI, TO, 8>, grid, block, 0, st, a);
    else launch_k(rope_kernel<TI, TO, 1>, grid, block, 0, st, a);
}
template <typename TI>
void launch_to(const RopeArgs& a, int to, bool vec, hipStream_t st) {
    if (to == UOCR_HIP_DTYPE_F32) launch_n<TI, float>(a, vec, st);
    else if (to == UOCR_HIP_DTYPE_BF16) launch_n<TI, bf16>(a, vec, st);
    else launch_n<TI, f16>(a, vec, st);
}

bool aligned16(const PagedRows& r) { return !((uintptr_t)r.p % 16 || r.row_bytes % 16 || r.head_bytes % 16); }

int launch_rope(const RopeArgs& a, int from, int to, bool vec, hipStream_t st) {
    // 8 elements at a time where the pairs divide and every place is 16-byte aligned
    // (8192 rows of 48 heads of 128: bf16 32 us, 61 one at a time; f32 79 and 94)
    const int half = a.rotary / 2;
    vec = vec && a.head_dim % 8 == 0 && half % 8 == 0;
    if (from == UOCR_HIP_DTYPE_F32) launch_to<float>(a, to, vec, st);
    else if (from == UOCR_HIP_DTYPE_BF16) launch_to<bf16>(a, to, vec, st);
    else launch_to<f16>(a, to, vec, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UOCR_HIP_OK : set_error(UOCR_HIP_EHIP, std::string("rope launch: ") + hipGetErrorString(e));
}

int check_rotation(int rows, int heads, int kv_heads, int head_dim, const int* positions, const float* inv_freq,
                   int rotary_dim, float factor) {
    if (rows < 0 || heads < 0 || kv_heads < 0) return set_error(UOCR_HIP_EINVAL, "rope: negative size");
    if (head_dim <= 0 || head_dim > 256) return set_error(UOCR_HIP_EUNSUPPORTED, "rope: head_dim must be in [1, 256]");
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
        return set_error(UOCR_HIP_EINVAL, "rope: rotary_dim must be even, in [0, head_dim]");
    if (rows && rotary_dim && (!positions || !inv_freq)) return set_error(UOCR_HIP_EINVAL, "rope: null positions or inv_freq");
    if (!std::isfinite(factor)) return set_error(UOCR_HIP_EINVAL, "rope: factor must be finite");
    if (((long long)heads + kv_heads) * head_dim > INT_MAX / 4) return set_error(UOCR_HIP_EUNSUPPORTED, "rope: too many heads");
    return UOCR_HIP_OK;
}

}  // namespace
}  // namespace uocr_hip

using namespace uocr_hip;

extern "C" {

int uocr_hip_rope_frequencies(int rotary_dim, double base, int scaling, double factor_len, int original_len,
                              double fast, double slow, float* inv_freq, float* factor) {
    if (!inv_freq || !factor) return set_error(UOCR_HIP_EINVAL, "rope_frequencies: null output");
    if (rotary_dim <= 0 || rotary_dim > 256 || rotary_dim % 2)
        return set_error(UOCR_HIP_EINVAL, "rope_frequencies: rotary_dim must be even, in [2, 256]");
    if (!(base > 1.0) || !std::isfinite(base)) return set_error(UOCR_HIP_EINVAL, "rope_frequencies: base must be finite, > 1");
    if (scaling < UOCR_HIP_ROPE_NONE || scaling > UOCR_HIP_ROPE_PARTS)
        return set_error(UOCR_HIP_EINVAL, "rope_frequencies: unknown scaling");
    if (scaling != UOCR_HIP_ROPE_NONE && (!(factor_len >= 1.0) || !std::isfinite(factor_len)))
        return set_error(UOCR_HIP_EINVAL, "rope_frequencies: factor_len must be finite, >= 1");
    if (scaling == UOCR_HIP_ROPE_BASE && rotary_dim < 4)
        return set_error(UOCR_HIP_EINVAL, "rope_frequencies: a scaled base needs rotary_dim >= 4");
    const double two_pi = 6.283185307179586477, n = rotary_dim;
    double lo = 0.0, span = 1.0;
    if (scaling == UOCR_HIP_ROPE_PARTS) {
        if (original_len <= 0 || !(slow > 0.0) || !(fast > slow) || !std::isfinite(fast))
            return set_error(UOCR_HIP_EINVAL, "rope_frequencies: original_len > 0 and fast > slow > 0 are needed");
        // the index whose frequency makes r turns over original_len positions
        const auto at = [&](double r) { return n * std::log(original_len / (r * two_pi)) / (2.0 * std::log(base)); };
        lo = std::max(0.0, std::floor(at(fast)));
        span = std::max(0.001, std::min(n - 1.0, std::ceil(at(slow))) - lo);
    }
    if (scaling == UOCR_HIP_ROPE_BASE) base *= std::pow(factor_len, n / (n - 2.0));
    *factor = scaling == UOCR_HIP_ROPE_PARTS ? (float)(0.1 * std::log(factor_len) + 1.0) : 1.0f;
    for (int i = 0; i < rotary_dim / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / n);
        double g = f;
        if (scaling == UOCR_HIP_ROPE_LINEAR) g = f / factor_len;
        if (scaling == UOCR_HIP_ROPE_PARTS) {
            const double ramp = std::min(1.0, std::max(0.0, (i - lo) / span));
            g = f / factor_len * ramp + f * (1.0 - ramp);
        }
        inv_freq[i] = (float)g;
    }
    return UOCR_HIP_OK;
}

int uocr_hip_rope(const uocr_hip_rows* q, const uocr_hip_rows* k, int rows, int heads, int kv_heads, int head_dim,
                  const int* positions, const float* inv_freq, int rotary_dim, int interleaved, float factor,
                  const uocr_hip_rows* q_out, const uocr_hip_rows* k_out, void* stream) {
    if (int rc = check_rotation(rows, heads, kv_heads, head_dim, positions, inv_freq, rotary_dim, factor)) return rc;
    if (heads + kv_heads == 0 || rows == 0) return UOCR_HIP_OK;
    RopeArgs a{};
    const uocr_hip_rows *in = heads ? q : k, *out = heads ? q_out : k_out;
    if (heads) {
        if (int rc = paged_rows("q", q, false, &a.q)) return rc;
        if (int rc = paged_rows("q_out", q_out, false, &a.qo)) return rc;
    }
    if (kv_heads) {
        if (int rc = paged_rows("k", k, false, &a.k)) return rc;
        if (int rc = paged_rows("k_out", k_out, false, &a.ko)) return rc;
        if (k->dtype != in->dtype || k_out->dtype != out->dtype)
            return set_error(UOCR_HIP_EINVAL, "rope: q and k, q_out and k_out must have the same dtype");
    }
    a.rows = rows;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.positions = positions;
    a.freq = inv_freq;
    a.rotary = rotary_dim;
    a.interleaved = interleaved != 0;
    a.factor = factor;
    const bool vec = (!heads || (aligned16(a.q) && aligned16(a.qo))) && (!kv_heads || (aligned16(a.k) && aligned16(a.ko)));
    return launch_rope(a, in->dtype, out->dtype, vec, (hipStream_t)stream);
}

int uocr_hip_rope_append_paged(const uocr_hip_rows* q, const uocr_hip_rows* k, const uocr_hip_rows* v, int rows,
                               int heads, const int* positions, const float* inv_freq, int rotary_dim,
                               int interleaved, float factor, const uocr_hip_paged_cache* cache, const int* d_seqs,
                               const int* d_rows, const uocr_hip_rows* q_out, void* stream) {
    RopeArgs a{};
    if (int rc = paged_cache(cache, &a.c)) return rc;
    if (int rc = check_rotation(rows, heads, cache->kv_heads, cache->head_dim, positions, inv_freq, rotary_dim, factor))
        return rc;
    if (rows == 0) return UOCR_HIP_OK;
    if (int rc = paged_rows("k", k, false, &a.k)) return rc;
    if (int rc = paged_rows("v", v, false, &a.v)) return rc;
    if (v->dtype != k->dtype) return set_error(UOCR_HIP_EINVAL, "rope: k and v must have the same dtype");
    if (heads) {
        if (int rc = paged_rows("q", q, false, &a.q)) return rc;
        if (int rc = paged_rows("q_out", q_out, false, &a.qo)) return rc;
        if (q->dtype != k->dtype) return set_error(UOCR_HIP_EINVAL, "rope: q and k must have the same dtype");
        if (q_out->dtype != cache->dtype) return set_error(UOCR_HIP_EINVAL, "rope: q_out must have the cache's dtype");
    }
    if (!d_seqs || !d_rows) return set_error(UOCR_HIP_EINVAL, "rope: null d_seqs or d_rows");
    a.rows = rows;
    a.heads = heads;
    a.kv_heads = cache->kv_heads;
    a.head_dim = cache->head_dim;
    a.positions = positions;
    a.freq = inv_freq;
    a.rotary = rotary_dim;
    a.interleaved = interleaved != 0;
    a.factor = factor;
    a.append = 1;
    a.seqs = d_seqs;
    a.at = d_rows;
    const bool vec = aligned16(a.k) && aligned16(a.v) && (!heads || (aligned16(a.q) && aligned16(a.qo)));
    return launch_rope(a, k->dtype, cache->dtype, vec, (hipStream_t)stream);
}

}  // extern "C"
