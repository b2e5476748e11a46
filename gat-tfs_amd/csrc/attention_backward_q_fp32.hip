// Segment attention, backward over query rows, FP32 storage (attention_backward.hpp).
#include "attention_backward.hpp"

namespace gatgpu {
hipError_t launch_attention_backward_q_fp32(const AttnArgs& a, int waves, hipStream_t s) {
    return backward_q<float>(a, waves, s);
}
size_t attention_backward_lds_fp32(int pass, int dim, int waves, int bias, int group, int buckets) {
    return backward_lds<float>(pass, dim, waves, bias, group, buckets);
}
}  // namespace gatgpu
