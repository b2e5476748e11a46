// Segment attention, backward over keys, FP32 storage (attention_backward.hpp).
#include "attention_backward.hpp"

namespace gatgpu {
hipError_t launch_attention_backward_kv_fp32(const AttnArgs& a, int waves, hipStream_t s) {
    return backward_kv<float>(a, waves, s);
}
}  // namespace gatgpu
