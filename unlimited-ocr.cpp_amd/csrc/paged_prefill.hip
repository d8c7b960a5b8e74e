// Launch of the paged prefill attention: tiles and splits.
#include "paged_prefill.hpp"

namespace uocr_hip {

int launch_paged_prefill(PagedAttnArgs a, int dtype, long long max_keys, void* ws, size_t ws_bytes, hipStream_t st) {
    const int bn = dtype == UOCR_HIP_DTYPE_F32 ? 32 : 64;
    const long long tiles = (long long)a.rows * a.group / kPreRows + a.batch;  // (each entry rounds up by less than one)
    if (tiles * a.kv_heads > INT_MAX / kPagedMaxSplits / 2) return set_error(UOCR_HIP_EUNSUPPORTED, "attention: too many rows or entries");
    a.n_tiles = (int)tiles;
    a.n_splits = paged_prefill_splits(tiles * a.kv_heads, (max_keys + bn - 1) / bn);
    if (a.n_splits > 1)
        if (int rc = paged_take_workspace(a, (size_t)a.rows * a.heads * a.n_splits, 0, ws, ws_bytes)) return rc;
    const dim3 grid((unsigned)((tiles * a.kv_heads + kXcds - 1) / kXcds * kXcds * a.n_splits));
    const int rc = dtype == UOCR_HIP_DTYPE_F32    ? launch_prefill_f32(a, grid, st)
                   : dtype == UOCR_HIP_DTYPE_BF16 ? launch_prefill_bf16(a, grid, st)
                                                  : launch_prefill_f16(a, grid, st);
    if (rc) return rc;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UOCR_HIP_OK
                           : set_error(UOCR_HIP_EHIP, std::string("paged prefill launch: ") + hipGetErrorString(e));
}

}  // namespace uocr_hip
