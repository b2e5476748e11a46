// Segment attention of short segments, FP32 storage (attention_small.hpp).
#include "attention_small.hpp"

namespace gatgpu {
hipError_t launch_attention_small_forward_fp32(const AttnArgs& a, int blocks, hipStream_t s) {
    return small_forward<float>(a, blocks, s);
}
hipError_t launch_attention_small_backward_fp32(const AttnArgs& a, int waves, hipStream_t s) {
    return small_backward<float>(a, waves, s);
}
size_t attention_small_backward_lds_fp32(int dim, int waves, int bias, int group, int buckets) {
    return small_backward_lds<float>(dim, waves, bias, group, buckets);
}
}  // namespace gatgpu
