// Checks of the paged cache's descriptors and the launchers behind its entry points.
#pragma once
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "launch.hpp"
#include "paged_device.hpp"
#include "uocr_hip/moe_capi.h"

namespace uocr_hip {

inline int dtype_bytes(int dtype) {
    return dtype == UOCR_HIP_DTYPE_F32 ? 4 : dtype == UOCR_HIP_DTYPE_BF16 || dtype == UOCR_HIP_DTYPE_F16 ? 2 : 0;
}

// A cache descriptor checked and in the kernels' form
int paged_cache(const uocr_hip_paged_cache* c, PagedCache* out);  // paged_capi.hip
// Rows of `heads` heads, checked; `vec`: 16-byte alignment needed
int paged_rows(const char* what, const uocr_hip_rows* r, bool vec, PagedRows* out);

// max_keys: what a row may see, min_keys: what the rows of an entry that fills many tiles all see, as far as the host knows. UOCR_HIP_OK or a code with its message.
int launch_paged_decode(PagedAttnArgs a, int dtype, long long max_keys, void* ws, size_t ws_bytes, hipStream_t st);
int launch_paged_prefill(PagedAttnArgs a, int dtype, long long max_keys, long long min_keys, void* ws, size_t ws_bytes, hipStream_t st);

// Gives a call its place for `records` partial results and (decode) `rows` entries about rows
int paged_take_workspace(PagedAttnArgs& a, size_t records, int rows, void* ws, size_t ws_bytes);

}  // namespace uocr_hip
