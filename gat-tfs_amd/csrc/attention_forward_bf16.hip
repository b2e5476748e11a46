// Segment attention, forward, bf16 storage (attention_forward.hpp).
#include "attention_forward.hpp"

namespace gatgpu {
hipError_t launch_attention_forward_bf16(const AttnArgs& a, int waves, hipStream_t s) { return forward<uint16_t>(a, waves, s); }
}  // namespace gatgpu
