// Segment attention, forward, FP32 storage (attention_forward.hpp).
#include "attention_forward.hpp"

namespace gatgpu {
hipError_t launch_attention_forward_fp32(const AttnArgs& a, int waves, hipStream_t s) { return forward<float>(a, waves, s); }
hipError_t launch_attention_forward_cut_fp32(const AttnArgs& a, hipStream_t s) { return forward_cut<float>(a, s); }
size_t attention_forward_cut_lds_fp32(int dim, int bias, int group) { return forward_cut_lds<float>(dim, bias, group); }
}  // namespace gatgpu
