// Attention among queries in fp32: a file for each type, which compile side by side.
#include "query_attention_kernels.hpp"

namespace dcn {

hipError_t attn_forward_fp32(const AttnLaunch &p, hipStream_t stream, size_t *bytes) { return forward_t<F32>(p, stream, bytes); }
hipError_t attn_backward_fp32(const AttnLaunch &p, hipStream_t stream, size_t *bytes) { return backward_t<F32>(p, stream, bytes); }

}  // namespace dcn
