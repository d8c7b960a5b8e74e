// Instances of the paged prefill kernel for f32 caches.
#include "paged_prefill.hpp"

namespace uocr_hip {

int launch_prefill_f32(const PagedAttnArgs& a, int rw, hipStream_t st) { return launch_prefill_t<float>(a, rw, st); }

}  // namespace uocr_hip
