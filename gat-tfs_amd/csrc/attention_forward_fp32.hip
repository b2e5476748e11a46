// Segment attention, forward, FP32 storage (attention_forward.hpp).
#include "attention_forward.hpp"

namespace gatgpu {
hipError_t launch_attention_forward_fp32(const AttnArgs& a, int waves, hipStream_t s) { return forward<float>(a, waves, s); }
}  // namespace gatgpu
