// Attention of many query rows over a paged KV cache.
#include <hip/hip_runtime.h>

#include "launch.hpp"
#include "paged_device.hpp"
#include "paged_host.hpp"

namespace uocr_hip {
namespace {

// One wave per (row, head)
template <typename T>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedAttnArgs a) {
    const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= (long long)a.rows * a.heads) return;
    const int row = (int)(u / a.heads), head = (int)(u % a.heads);
    // the sequence whose rows include it: the last start at or before the row
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
    const bool lost = kv > a.c.capacity();
    const int len = lost ? 0 : imax(kv, 0), n = a.q_start[lo + 1] - a.q_start[lo];
    row_attention<T>(a, seq, row, head, len - n + (row - a.q_start[lo]), len, lost);
}

}  // namespace

int launch_paged_prefill(PagedAttnArgs a, int dtype, long long max_keys, void* ws, size_t ws_bytes, hipStream_t st) {
    const long long blocks = ((long long)a.rows * a.heads + 3) / 4;
    const dim3 grid((unsigned)blocks), block(256);
    if (dtype == UOCR_HIP_DTYPE_F32) launch_k(paged_rows_kernel<float>, grid, block, 0, st, a);
    else if (dtype == UOCR_HIP_DTYPE_BF16) launch_k(paged_rows_kernel<bf16>, grid, block, 0, st, a);
    else launch_k(paged_rows_kernel<f16>, grid, block, 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UOCR_HIP_OK
                           : set_error(UOCR_HIP_EHIP, std::string("paged prefill launch: ") + hipGetErrorString(e));
}

}  // namespace uocr_hip
