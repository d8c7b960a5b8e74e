// Instances of the paged prefill kernel for bf16 caches.
#include "paged_prefill.hpp"

namespace uocr_hip {

int launch_prefill_bf16(const PagedAttnArgs& a, int rw, hipStream_t st) { return launch_prefill_t<bf16>(a, rw, st); }

}  // namespace uocr_hip
