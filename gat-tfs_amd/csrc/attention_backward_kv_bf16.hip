// Segment attention, backward over keys, bf16 storage (attention_backward.hpp).
#include "attention_backward.hpp"

namespace gatgpu {
hipError_t launch_attention_backward_kv_bf16(const AttnArgs& a, int waves, hipStream_t s) {
    return backward_kv<uint16_t>(a, waves, s);
}
}  // namespace gatgpu
