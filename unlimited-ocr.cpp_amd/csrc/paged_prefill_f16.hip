// Instances of the paged prefill kernel for f16 caches.
#include "paged_prefill.hpp"

namespace uocr_hip {

int launch_prefill_f16(const PagedAttnArgs& a, int rw, hipStream_t st) { return launch_prefill_t<f16>(a, rw, st); }

}  // namespace uocr_hip
