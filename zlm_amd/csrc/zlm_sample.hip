// zlm_sample.hip -- CDNA4 (gfx950) kernels that draw a token from each row of
// logits by temperature, top-k, top-p and min-p with a given uniform number
// (sample_impl.h).  Built as a device-only code object (hipcc --genco) and loaded by
// the host library.
#include "sample_impl.h"

extern "C" __global__ void __launch_bounds__(256, 8) zlm_sample_hist(Args a) { slice_hist<256>(a, blockIdx.y); }
extern "C" __global__ void __launch_bounds__(1024) zlm_sample_hist_wide(Args a) { slice_hist<1024>(a, blockIdx.y); }
extern "C" __global__ void __launch_bounds__(512) zlm_sample_pick(Args a) {
    zlm::SampleCut none;
    pick<true>(a, blockIdx.x, none);
}
