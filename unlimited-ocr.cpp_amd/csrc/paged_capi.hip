// Entry points of the paged attention: argument checks, kernel arguments.
#include "paged_host.hpp"

namespace uocr_hip {

int paged_cache(const uocr_hip_paged_cache* c, PagedCache* out) {
    if (!c || !c->k || !c->v || !c->page_table) return set_error(UOCR_HIP_EINVAL, "paged cache: null pointer");
    const int es = dtype_bytes(c->dtype);
    if (!es) return set_error(UOCR_HIP_EINVAL, "paged cache: unknown dtype");
    if (c->n_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->n_seqs <= 0 || c->max_pages <= 0)
        return set_error(UOCR_HIP_EINVAL, "paged cache: n_pages, page_size, kv_heads, n_seqs and max_pages must be > 0");
    if (c->page_size > (1 << 30)) return set_error(UOCR_HIP_EUNSUPPORTED, "paged cache: page_size above 2^30");
    if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim % 8)
        return set_error(UOCR_HIP_EUNSUPPORTED, "paged cache: head_dim must be a multiple of 8 in [8, 256]");
    if (c->page_stride < 0 || c->row_stride < 0 || c->head_stride < 0 || c->table_stride < 0)
        return set_error(UOCR_HIP_EINVAL, "paged cache: negative stride");
    constexpr long long kMost = LLONG_MAX / 8;
    if (c->page_stride > kMost / c->n_pages || c->row_stride > kMost / c->page_size ||
        c->head_stride > kMost / c->kv_heads || c->table_stride > kMost / c->n_seqs)
        return set_error(UOCR_HIP_EINVAL, "paged cache: stride too large");
    const long long per16 = 16 / es;
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || c->page_stride % per16 || c->row_stride % per16 ||
        c->head_stride % per16)
        return set_error(UOCR_HIP_EUNSUPPORTED, "paged cache: k, v and the strides must be multiples of 16 bytes");
    if ((uintptr_t)c->page_table % 4) return set_error(UOCR_HIP_EINVAL, "paged cache: page_table must be 4-byte aligned");
    if (c->n_seqs > 1 && c->table_stride < c->max_pages)
        return set_error(UOCR_HIP_EINVAL, "paged cache: table_stride is below max_pages");
    *out = PagedCache{(char*)c->k, (char*)c->v, c->page_table, c->page_stride * es, c->row_stride * es,
                      c->head_stride * es, c->table_stride, c->n_pages, c->n_seqs, c->max_pages,
                      fast_div((uint32_t)c->page_size)};
    return UOCR_HIP_OK;
}

int paged_rows(const char* what, const uocr_hip_rows* r, bool vec, PagedRows* out) {
    if (!r || !r->data) return set_error(UOCR_HIP_EINVAL, std::string(what) + ": null pointer");
    const int es = dtype_bytes(r->dtype);
    if (!es) return set_error(UOCR_HIP_EINVAL, std::string(what) + ": unknown dtype");
    if (r->row_stride < 0 || r->head_stride < 0)
        return set_error(UOCR_HIP_EINVAL, std::string(what) + ": negative stride");
    if (r->row_stride > LLONG_MAX / 8 / INT_MAX || r->head_stride > LLONG_MAX / 8 / INT_MAX)
        return set_error(UOCR_HIP_EINVAL, std::string(what) + ": stride too large");
    const uintptr_t align = vec ? 16 : es;
    if ((uintptr_t)r->data % align || r->row_stride * es % align || r->head_stride * es % align)
        return set_error(vec ? UOCR_HIP_EUNSUPPORTED : UOCR_HIP_EINVAL,
                         std::string(what) + (vec ? ": data and strides must be multiples of 16 bytes" : ": misaligned"));
    *out = PagedRows{(char*)r->data, r->row_stride * es, r->head_stride * es};
    return UOCR_HIP_OK;
}

int paged_take_workspace(PagedAttnArgs& a, size_t records, int rows, void* ws, size_t ws_bytes) {
    const size_t need = kPagedHead + records * (a.head_dim + 2) * sizeof(float) + rows * 2 * sizeof(int);
    if (!ws || ws_bytes < need)
        return set_error(UOCR_HIP_EWORKSPACE, "attention: workspace of " + std::to_string(ws ? ws_bytes : 0) + " bytes, " +
                                                  std::to_string(need) + " needed");
    if ((uintptr_t)ws % 16) return set_error(UOCR_HIP_EINVAL, "attention: workspace must be 16-byte aligned");
    // one word before the counters, on their cache line
    a.counters = static_cast<int*>(ws) + 1;
    a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + kPagedHead);
    a.part_ml = a.part + records * a.head_dim;
    a.part_rows = reinterpret_cast<int*>(a.part_ml + 2 * records);
    return UOCR_HIP_OK;
}

namespace {

__global__ __launch_bounds__(256) void paged_workspace_kernel(int* ws) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < kPagedHead / 4) ws[i] = i ? 0 : kPagedMagic;
}

int attn_args(const uocr_hip_paged_cache* cache, const uocr_hip_attention_opts* o, const uocr_hip_rows* q,
              const uocr_hip_rows* out, int rows, int batch, const int* d_seqs, const int* d_kv_len, int max_kv_len,
              PagedAttnArgs* a) {
    *a = PagedAttnArgs{};
    if (int rc = paged_cache(cache, &a->c)) return rc;
    if (!o) return set_error(UOCR_HIP_EINVAL, "attention: null options");
    if (o->heads <= 0 || o->heads % cache->kv_heads)
        return set_error(UOCR_HIP_EINVAL, "attention: heads must be a positive multiple of kv_heads");
    if (rows < 0 || batch < 0 || max_kv_len < 0)
        return set_error(UOCR_HIP_EINVAL, "attention: rows, batch and max_kv_len must be >= 0");
    if (!std::isfinite(o->scale) || !std::isfinite(o->softcap) || o->softcap < 0.0f)
        return set_error(UOCR_HIP_EINVAL, "attention: scale and softcap must be finite, softcap >= 0");
    if ((o->scale != 0.0f && !(std::fabs(o->scale) >= 1e-15f && std::fabs(o->scale) <= 1e15f)) ||
        (o->softcap != 0.0f && !(o->softcap >= 1e-15f && o->softcap <= 1e15f)))
        return set_error(UOCR_HIP_EUNSUPPORTED, "attention: |scale| and softcap, if not 0, must be in [1e-15, 1e15]");
    if (o->window < 0) return set_error(UOCR_HIP_EINVAL, "attention: window must be >= 0");
    if ((long long)rows * o->heads > INT_MAX)
        return set_error(UOCR_HIP_EUNSUPPORTED, "attention: more than 2^31 - 1 (row, head) pairs");
    if (rows > 0 && batch > 0) {
        if (int rc = paged_rows("q", q, true, &a->q)) return rc;
        if (int rc = paged_rows("out", out, false, &a->out)) return rc;
        if (q->dtype != cache->dtype) return set_error(UOCR_HIP_EINVAL, "attention: q must have the cache's dtype");
        if (out->dtype != q->dtype && out->dtype != UOCR_HIP_DTYPE_F32)
            return set_error(UOCR_HIP_EINVAL, "attention: out must be f32 or have q's dtype");
        if (!d_kv_len) return set_error(UOCR_HIP_EINVAL, "attention: null d_kv_len");
        if (!d_seqs && batch > cache->n_seqs)
            return set_error(UOCR_HIP_EINVAL, "attention: batch exceeds the cache's n_seqs (and no d_seqs is given)");
        a->out_f32 = out->dtype == UOCR_HIP_DTYPE_F32;
    }
    a->rows = rows;
    a->batch = batch;
    a->heads = o->heads;
    a->kv_heads = cache->kv_heads;
    a->head_dim = cache->head_dim;
    a->group = o->heads / cache->kv_heads;
    a->seqs = d_seqs;
    a->kv_len = d_kv_len;
    const double log2e = 1.4426950408889634, scale = o->scale != 0.0f ? o->scale : 1.0 / std::sqrt((double)cache->head_dim);
    const double in = o->softcap > 0.0f ? scale / o->softcap : 0.0;
    a->sc = PagedScores{(float)(scale * log2e), (float)(o->softcap * log2e), (float)in, (float)(2.0 * log2e * in), o->slopes,
                        scale < 0.0};
    a->mask = MaskArgs{o->causal != 0, o->window, o->prefix_both_ways != 0, o->prefix_len, o->key_begin, o->key_end};
    return UOCR_HIP_OK;
}

// keys that `rows` rows side by side may see, as far as the host knows
long long most_keys(const PagedAttnArgs& a, int max_kv_len, int rows) {
    long long n = std::min<long long>(a.c.capacity(), INT_MAX);
    if (max_kv_len > 0) n = std::min<long long>(n, max_kv_len);
    if (a.mask.window > 0 && !a.mask.prefix_len) n = std::min<long long>(n, (long long)a.mask.window + rows - 1);
    return std::max(n, 1ll);
}

}  // namespace
}  // namespace uocr_hip

using namespace uocr_hip;

extern "C" {

size_t uocr_hip_paged_attention_workspace_size(const uocr_hip_paged_cache* cache, int heads, int rows) {
    PagedCache c;
    if (paged_cache(cache, &c)) return 0;
    if (heads <= 0 || heads % cache->kv_heads || rows < 0) {
        set_error(UOCR_HIP_EINVAL, "workspace: heads must be a positive multiple of kv_heads, rows >= 0");
        return 0;
    }
    return kPagedHead + paged_workspace_records(rows, heads, cache->kv_heads) * (cache->head_dim + 2) * sizeof(float) +
           std::min(rows, kPagedShareRows) * 2 * sizeof(int);
}

int uocr_hip_paged_attention_workspace_init(void* workspace, size_t workspace_bytes, void* stream) {
    if (!workspace || (uintptr_t)workspace % 16)
        return set_error(UOCR_HIP_EINVAL, "workspace: null or not 16-byte aligned");
    if (workspace_bytes < kPagedHead) return set_error(UOCR_HIP_EWORKSPACE, "workspace: too small");
    launch_k(paged_workspace_kernel, dim3(kPagedHead / 4 / 256 + 1), dim3(256), 0, (hipStream_t)stream,
             static_cast<int*>(workspace));
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UOCR_HIP_OK
                           : set_error(UOCR_HIP_EHIP, std::string("workspace launch: ") + hipGetErrorString(e));
}

int uocr_hip_paged_attention_decode(const uocr_hip_paged_cache* cache, const uocr_hip_attention_opts* opts,
                                    const uocr_hip_rows* q, int batch, const int* d_seqs, const int* d_kv_len,
                                    int max_kv_len, const uocr_hip_rows* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    PagedAttnArgs a;
    if (int rc = attn_args(cache, opts, q, out, batch, batch, d_seqs, d_kv_len, max_kv_len, &a)) return rc;
    if (batch == 0) return UOCR_HIP_OK;
    a.mask.causal = 1;
    return launch_paged_decode(a, cache->dtype, most_keys(a, max_kv_len, 1), workspace, workspace_bytes,
                               (hipStream_t)stream);
}

int uocr_hip_paged_attention_prefill(const uocr_hip_paged_cache* cache, const uocr_hip_attention_opts* opts,
                                     const uocr_hip_rows* q, int rows, int batch, const int* d_q_start,
                                     const int* d_seqs, const int* d_kv_len, int max_kv_len, const uocr_hip_rows* out,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    PagedAttnArgs a;
    if (int rc = attn_args(cache, opts, q, out, rows, batch, d_seqs, d_kv_len, max_kv_len, &a)) return rc;
    if (rows == 0 || batch == 0) return UOCR_HIP_OK;
    if (!d_q_start) return set_error(UOCR_HIP_EINVAL, "attention: null d_q_start");
    if (opts->window > 0 && !opts->causal) return set_error(UOCR_HIP_EINVAL, "attention: a window needs causal");
    a.q_start = d_q_start;
    const long long most = most_keys(a, max_kv_len, std::min(rows, 128 / a.group + 2));
    // the first of an entry's rows, of entries of equal length
    long long least = most_keys(a, max_kv_len, INT_MAX) - (opts->causal ? rows / batch : 0);
    least = std::max(std::min(least, most), 0ll);
    return launch_paged_prefill(a, cache->dtype, most, least, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
