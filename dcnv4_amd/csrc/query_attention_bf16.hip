// Attention among queries in bf16: a file for each type, which compile side by side.
#include "query_attention_kernels.hpp"

namespace dcn {

hipError_t attn_forward_bf16(const AttnLaunch &p, hipStream_t stream, size_t *bytes) { return forward_t<BF16>(p, stream, bytes); }
hipError_t attn_backward_bf16(const AttnLaunch &p, hipStream_t stream, size_t *bytes) { return backward_t<BF16>(p, stream, bytes); }

}  // namespace dcn
