// Segment attention, forward, bf16 storage (attention_forward.hpp).
#include "attention_forward.hpp"

namespace gatgpu {
hipError_t launch_attention_forward_bf16(const AttnArgs& a, int waves, hipStream_t s) { return forward<uint16_t>(a, waves, s); }
hipError_t launch_attention_forward_cut_bf16(const AttnArgs& a, hipStream_t s) { return forward_cut<uint16_t>(a, s); }
size_t attention_forward_cut_lds_bf16(int dim, int bias, int group) { return forward_cut_lds<uint16_t>(dim, bias, group); }
}  // namespace gatgpu
