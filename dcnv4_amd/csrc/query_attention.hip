// Attention among queries: by type, and the sums of the slopes' parts (the kernels: query_attention_kernels.hpp).
#include "query_attention.hpp"

#include "common.hpp"

namespace dcn {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;

// Sums of the slopes' parts of a head, [batch][heads][parts], in a fixed order.
__global__ void __launch_bounds__(kThreads) attn_slope_grad_kernel(const float *part, float *grad, int batch, int heads, int parts) {
  __shared__ float s_sum[kWaves];
  const int head = blockIdx.x, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  float sum = 0.f;
  for (int b = 0; b < batch; ++b)
    for (int i = threadIdx.x; i < parts; i += kThreads) sum += part[((size_t)b * heads + head) * parts + i];
  sum = cluster_sum(sum, kWave);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) grad[head] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

hipError_t forward(int dtype, const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  switch (dtype) {
    case F32::kCode: return attn_forward_fp32(p, stream, bytes);
    case F16::kCode: return attn_forward_fp16(p, stream, bytes);
    case BF16::kCode: return attn_forward_bf16(p, stream, bytes);
  }
  return hipErrorInvalidValue;
}
hipError_t backward(int dtype, const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  switch (dtype) {
    case F32::kCode: return attn_backward_fp32(p, stream, bytes);
    case F16::kCode: return attn_backward_fp16(p, stream, bytes);
    case BF16::kCode: return attn_backward_bf16(p, stream, bytes);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_slope_grad(const float *part, float *grad, int batch, int heads, int parts, hipStream_t stream) {
  hipLaunchKernelGGL(attn_slope_grad_kernel, dim3(heads), dim3(kThreads), 0, stream, part, grad, batch, heads, parts);
  return hipGetLastError();
}

size_t attn_forward_workspace_bytes(int dtype, const AttnLaunch &p) {
  size_t bytes = 0;
  if (forward(dtype, p, nullptr, &bytes) != hipSuccess) return 0;      // the launch says why
  return bytes;
}
size_t attn_backward_workspace_bytes(int dtype, const AttnLaunch &p) {
  size_t bytes = 0;
  if (backward(dtype, p, nullptr, &bytes) != hipSuccess) return 0;
  return bytes;
}

hipError_t launch_attn_forward(int dtype, const AttnLaunch &p, hipStream_t stream) { return forward(dtype, p, stream, nullptr); }
hipError_t launch_attn_backward(int dtype, const AttnLaunch &p, hipStream_t stream) { return backward(dtype, p, stream, nullptr); }

}  // namespace dcn
