// Segment attention of short segments, bf16 storage (attention_small.hpp).
#include "attention_small.hpp"

namespace gatgpu {
hipError_t launch_attention_small_forward_bf16(const AttnArgs& a, int blocks, hipStream_t s) {
    return small_forward<uint16_t>(a, blocks, s);
}
hipError_t launch_attention_small_backward_bf16(const AttnArgs& a, int waves, hipStream_t s) {
    return small_backward<uint16_t>(a, waves, s);
}
size_t attention_small_backward_lds_bf16(int dim, int waves, int bias, int group, int buckets) {
    return small_backward_lds<uint16_t>(dim, waves, bias, group, buckets);
}
}  // namespace gatgpu
