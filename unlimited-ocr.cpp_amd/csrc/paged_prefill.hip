// Launch of the paged prefill attention: tiles and splits.
#include "paged_prefill.hpp"

namespace uocr_hip {

int launch_paged_prefill(PagedAttnArgs a, int dtype, long long max_keys, long long min_keys, void* ws, size_t ws_bytes,
                         hipStream_t st) {
    const PrefillPlan p = paged_prefill_plan(a.rows, a.batch, a.heads, a.kv_heads, a.head_dim, dtype == UOCR_HIP_DTYPE_F32,
                                             max_keys, min_keys);
    if (p.tiles * a.kv_heads * p.splits >= 1 << 23)  // (a launch has fewer than 2^32 threads)
        return set_error(UOCR_HIP_EUNSUPPORTED, "attention: too many rows or entries");
    a.n_tiles = (int)p.tiles;
    a.n_splits = p.splits;
    if (a.n_splits > 1)
        if (int rc = paged_take_workspace(a, (size_t)a.rows * a.heads * a.n_splits, 0, ws, ws_bytes)) return rc;
    const int rc = dtype == UOCR_HIP_DTYPE_F32    ? launch_prefill_f32(a, p.row_waves, st)
                   : dtype == UOCR_HIP_DTYPE_BF16 ? launch_prefill_bf16(a, p.row_waves, st)
                                                  : launch_prefill_f16(a, p.row_waves, st);
    if (rc) return rc;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UOCR_HIP_OK
                           : set_error(UOCR_HIP_EHIP, std::string("paged prefill launch: ") + hipGetErrorString(e));
}

}  // namespace uocr_hip
