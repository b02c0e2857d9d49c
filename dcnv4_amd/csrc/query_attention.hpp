// Launch struct of the attention among queries (query_attention.hip); beside the C ABI, for the extension.
#pragma once
#include <hip/hip_runtime.h>

#include <stddef.h>

namespace dcn {

// A (batch, tokens, heads, width) tensor: elements between neighbours; the width is dense, its rows start on 16 bytes.
struct AttnRows {
  const void *base;
  long long batch, token, head;
};

struct AttnLaunch {
  AttnRows q, k, v;
  int batch, nq, nk, heads, kv_heads, width;      // width: a multiple of 8, at most kMaxAttnWidth
  float scale, cap;                               // cap 0: scores as they are
  const int *q_segments, *k_segments;             // (batch, tokens); no k_segments: all see all; no q_segments: zeros
  const float *q_points, *k_points, *slopes;      // (batch, tokens, 2), (heads,): all or none
  void *out;                                      // dense (batch, nq, heads, width)
  void *out_rest;                                 // like out: what rounding took from it, for the backward of 16-bit types; or null
  float *lse;                                     // (batch, heads, nq): base-2 log of a row's sum; infinite where it sees nothing
  // backward; gradients are dense and of the tensors' type
  AttnRows grad_out;
  void *grad_q, *grad_k, *grad_v;                 // null where not wanted
  float *grad_slopes;                             // (heads,) or null
  void *workspace;
};

constexpr int kMaxAttnWidth = 128;
// Scratch of a call, 256-byte aligned; destroyed.
size_t attn_forward_workspace_bytes(int dtype, const AttnLaunch &p);
size_t attn_backward_workspace_bytes(int dtype, const AttnLaunch &p);
hipError_t launch_attn_forward(int dtype, const AttnLaunch &p, hipStream_t stream);
// Wants out, out_rest and lse of the forward.
hipError_t launch_attn_backward(int dtype, const AttnLaunch &p, hipStream_t stream);

// A type's own (query_attention_*.hip): the launch, or where `bytes` is not null the scratch it wants and no launch.
hipError_t attn_forward_fp32(const AttnLaunch &p, hipStream_t stream, size_t *bytes);
hipError_t attn_forward_fp16(const AttnLaunch &p, hipStream_t stream, size_t *bytes);
hipError_t attn_forward_bf16(const AttnLaunch &p, hipStream_t stream, size_t *bytes);
hipError_t attn_backward_fp32(const AttnLaunch &p, hipStream_t stream, size_t *bytes);
hipError_t attn_backward_fp16(const AttnLaunch &p, hipStream_t stream, size_t *bytes);
hipError_t attn_backward_bf16(const AttnLaunch &p, hipStream_t stream, size_t *bytes);
// grad[head] = sum over batch and parts of part[batch][heads][parts]
hipError_t launch_slope_grad(const float *part, float *grad, int batch, int heads, int parts, hipStream_t stream);

}  // namespace dcn
