// Segment attention, backward over query rows, bf16 storage (attention_backward.hpp).
#include "attention_backward.hpp"

namespace gatgpu {
hipError_t launch_attention_backward_q_bf16(const AttnArgs& a, int waves, hipStream_t s) {
    return backward_q<uint16_t>(a, waves, s);
}
size_t attention_backward_lds_bf16(int pass, int dim, int waves, int bias, int group, int buckets) {
    return backward_lds<uint16_t>(pass, dim, waves, bias, group, buckets);
}
}  // namespace gatgpu
