// Attention among queries, the dense attention beside the sampling one of a deformable decoder.  Per sequence and head
//   x_ij = scale q_i . k_j,   s_ij = cap tanh(x_ij / cap) - slope |p_i - p_j|   (the cap and the distance where there are any)
//   out_i = sum_j P_ij v_j,   P = softmax over the keys that i sees;  a row that sees none is zeros
// where i sees j if i's segment number is not negative and j's is the same or 0.  Backward, with delta_i = dO_i . out_i:
//   dV = P^T dO,  dS = P (dO V^T - delta),  dslope = -sum dS |p_i - p_j|,  dX = dS (1 - tanh^2),  dQ = scale dX K,  dK = scale dX^T Q
// Heads that share a key head add up in its gradient.
//
// A wave owns a row: of 64 keys at a time (queries, for the gradients of a key) each lane forms the score of its own, the
// lanes then take a column of the result each and walk the 64.  What a row does not see is skipped, not multiplied by zero, so
// infinities and NaN there go nowhere.
#include "query_attention.hpp"

#include "common.hpp"
#include "mfma.hpp"

namespace dcn {
namespace {

constexpr int kRowThreads = 256, kRowWaves = kRowThreads / kWave;
constexpr float kInf = __builtin_inff();

__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) { return cluster_sum(v, kWave); }

template <typename Tag>
__device__ __forceinline__ const char *row_of(const AttnRows &t, int b, int token, int head) {
  return static_cast<const char *>(t.base) + (b * t.batch + token * t.token + head * t.head) * (long long)Tag::kBytes;
}

// Dot product of a row in memory with one in LDS.
template <typename Tag>
__device__ __forceinline__ float dot_row(const char *row, const float *other, int width) {
  float sum = 0.f;
  for (int d = 0; d < width; d += 8) {
    float f[8];
    load8<Tag>(row, d, f);
#pragma unroll
    for (int c = 0; c < 8; ++c) sum = fmaf(f[c], other[d + c], sum);
  }
  return sum;
}

struct Score {
  float s, slope_factor, bent;      // the score; the distance; 1 - tanh^2
};
__device__ __forceinline__ Score finish_score(const AttnLaunch &p, float dot, int b, int head, int i, int j) {
  Score r;
  r.s = dot * p.scale;
  r.bent = 1.f;
  if (p.cap > 0.f) {
    const float t = tanhf(r.s / p.cap);
    r.s = p.cap * t;
    r.bent = fmaf(-t, t, 1.f);
  }
  r.slope_factor = 0.f;
  if (p.slopes != nullptr) {
    const float *a = p.q_points + ((long long)b * p.nq + i) * 2, *c = p.k_points + ((long long)b * p.nk + j) * 2;
    const float dx = a[0] - c[0], dy = a[1] - c[1];
    r.slope_factor = sqrtf(fmaf(dx, dx, dy * dy));
    r.s = fmaf(-p.slopes[head], r.slope_factor, r.s);
  }
  return r;
}
__device__ __forceinline__ bool sees(const AttnLaunch &p, int b, int i, int j) {
  if (p.k_segments == nullptr) return true;
  const int mine = p.q_segments != nullptr ? p.q_segments[(long long)b * p.nq + i] : 0, theirs = p.k_segments[(long long)b * p.nk + j];
  return mine >= 0 && (theirs == mine || theirs == 0);
}

// A row of a tensor into a wave's LDS.
template <typename Tag>
__device__ __forceinline__ void park_row(float *dst, const char *row, int width, int lane) {
  if (lane * 8 < width) {
    float f[8];
    load8<Tag>(row, lane * 8, f);
#pragma unroll
    for (int c = 0; c < 8; ++c) dst[lane * 8 + c] = f[c];
  }
}
// acc[u] += weight of lane l's row times its elements at lane and lane + 64, over all lanes; rows of weight 0 are not read.
template <typename Tag, typename RowAt>
__device__ __forceinline__ void add_rows(float (&acc)[2], float weight, int width, int lane, RowAt row_at) {
  uint64_t left = __ballot(weight != 0.f);
  while (left != 0) {
    const int l = __builtin_ctzll(left);
    left &= left - 1;
    const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), l));
    const char *row = row_at(l);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int d = lane + u * 64;
      if (d < width) {
        float f[1];
        Pack<Tag, 1>::decode(reinterpret_cast<const typename RawWord<Tag::kBytes>::type *>(row)[d], f);
        acc[u] = fmaf(w, f[0], acc[u]);
      }
    }
  }
}
template <typename Tag>
__device__ __forceinline__ void write_row(void *base, long long row, const float (&acc)[2], float factor, int width, int lane) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int d = lane + u * 64;
    const float f[1] = {acc[u] * factor};
    if (d < width) reinterpret_cast<typename RawWord<Tag::kBytes>::type *>(base)[row * width + d] = Pack<Tag, 1>::encode(f);
  }
}

template <typename Tag>
__global__ void __launch_bounds__(kRowThreads) attn_rows_forward_kernel(const AttnLaunch p) {
  __shared__ float s_row[kRowWaves][kMaxAttnWidth];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const long long row = (long long)blockIdx.x * kRowWaves + wave;
  if (row >= (long long)p.batch * p.nq * p.heads) return;
  const int head = (int)(row % p.heads), i = (int)(row / p.heads % p.nq), b = (int)(row / p.heads / p.nq);
  const int kv = head / (p.heads / p.kv_heads);
  float *mine = s_row[wave];
  park_row<Tag>(mine, row_of<Tag>(p.q, b, i, head), p.width, lane);
  float top = -kInf, sum = 0.f, acc[2] = {0.f, 0.f};
  for (int j0 = 0; j0 < p.nk; j0 += kWave) {
    const int j = j0 + lane;
    float s = -kInf;
    if (j < p.nk && sees(p, b, i, j)) s = finish_score(p, dot_row<Tag>(row_of<Tag>(p.k, b, j, kv), mine, p.width), b, head, i, j).s;
    const float now = fmaxf(top, wave_max(s));
    if (now == -kInf) continue;
    const float w = expf(s - now), keep = expf(top - now);
    sum = fmaf(sum, keep, wave_sum(w));
    acc[0] *= keep;
    acc[1] *= keep;
    top = now;
    add_rows<Tag>(acc, w, p.width, lane, [&](int l) { return row_of<Tag>(p.v, b, j0 + l, kv); });
  }
  const bool empty = sum == 0.f;
  write_row<Tag>(p.out, row, acc, empty ? 0.f : 1.f / sum, p.width, lane);
  if (p.lse != nullptr && lane == 0) p.lse[((long long)b * p.heads + head) * p.nq + i] = empty ? kInf : top + logf(sum);
}

// grad_q, the rows' delta and their part of the slopes' gradient
template <typename Tag>
__global__ void __launch_bounds__(kRowThreads) attn_rows_grad_q_kernel(const AttnLaunch p, float *delta_out, float *slope_part) {
  __shared__ float s_row[kRowWaves][2][kMaxAttnWidth];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const long long row = (long long)blockIdx.x * kRowWaves + wave;
  if (row >= (long long)p.batch * p.nq * p.heads) return;
  const int head = (int)(row % p.heads), i = (int)(row / p.heads % p.nq), b = (int)(row / p.heads / p.nq);
  const int kv = head / (p.heads / p.kv_heads);
  float *query = s_row[wave][0], *grad = s_row[wave][1];
  park_row<Tag>(query, row_of<Tag>(p.q, b, i, head), p.width, lane);
  park_row<Tag>(grad, row_of<Tag>(p.grad_out, b, i, head), p.width, lane);
  const long long at = ((long long)b * p.heads + head) * p.nq + i;
  const float delta = dot_row<Tag>(static_cast<const char *>(p.out) + row * p.width * Tag::kBytes, grad, p.width), lse = p.lse[at];
  float acc[2] = {0.f, 0.f}, slope = 0.f;
  for (int j0 = 0; j0 < p.nk; j0 += kWave) {
    const int j = j0 + lane;
    float dx = 0.f;
    if (j < p.nk && sees(p, b, i, j)) {
      const Score s = finish_score(p, dot_row<Tag>(row_of<Tag>(p.k, b, j, kv), query, p.width), b, head, i, j);
      const float ds = expf(s.s - lse) * (dot_row<Tag>(row_of<Tag>(p.v, b, j, kv), grad, p.width) - delta);
      slope = fmaf(-ds, s.slope_factor, slope);
      dx = ds * s.bent;
    }
    add_rows<Tag>(acc, dx, p.width, lane, [&](int l) { return row_of<Tag>(p.k, b, j0 + l, kv); });
  }
  if (p.grad_q != nullptr) write_row<Tag>(p.grad_q, row, acc, p.scale, p.width, lane);
  slope = wave_sum(slope);
  if (lane == 0) {
    delta_out[at] = delta;
    if (slope_part != nullptr) slope_part[at] = slope;
  }
}

template <typename Tag>
__global__ void __launch_bounds__(kRowThreads) attn_rows_grad_kv_kernel(const AttnLaunch p, const float *delta) {
  __shared__ float s_row[kRowWaves][2][kMaxAttnWidth];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const long long row = (long long)blockIdx.x * kRowWaves + wave;
  if (row >= (long long)p.batch * p.nk * p.kv_heads) return;
  const int kv = (int)(row % p.kv_heads), j = (int)(row / p.kv_heads % p.nk), b = (int)(row / p.kv_heads / p.nk);
  const int share = p.heads / p.kv_heads;
  float *key = s_row[wave][0], *value = s_row[wave][1];
  park_row<Tag>(key, row_of<Tag>(p.k, b, j, kv), p.width, lane);
  park_row<Tag>(value, row_of<Tag>(p.v, b, j, kv), p.width, lane);
  float dk[2] = {0.f, 0.f}, dv[2] = {0.f, 0.f};
  for (int head = kv * share; head < (kv + 1) * share; ++head)
    for (int i0 = 0; i0 < p.nq; i0 += kWave) {
      const int i = i0 + lane;
      float weight = 0.f, dx = 0.f;
      if (i < p.nq && sees(p, b, i, j)) {
        const long long at = ((long long)b * p.heads + head) * p.nq + i;
        const Score s = finish_score(p, dot_row<Tag>(row_of<Tag>(p.q, b, i, head), key, p.width), b, head, i, j);
        weight = expf(s.s - p.lse[at]);
        dx = weight * (dot_row<Tag>(row_of<Tag>(p.grad_out, b, i, head), value, p.width) - delta[at]) * s.bent;
      }
      add_rows<Tag>(dv, weight, p.width, lane, [&](int l) { return row_of<Tag>(p.grad_out, b, i0 + l, head); });
      add_rows<Tag>(dk, dx, p.width, lane, [&](int l) { return row_of<Tag>(p.q, b, i0 + l, head); });
    }
  if (p.grad_k != nullptr) write_row<Tag>(p.grad_k, row, dk, p.scale, p.width, lane);
  if (p.grad_v != nullptr) write_row<Tag>(p.grad_v, row, dv, 1.f, p.width, lane);
}

// Sums of the slopes' parts of a head, [batch][heads][parts], in a fixed order.
__global__ void __launch_bounds__(kRowThreads) attn_slope_grad_kernel(const float *part, float *grad, int batch, int heads, int parts) {
  __shared__ float s_sum[kRowWaves];
  const int head = blockIdx.x, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  float sum = 0.f;
  for (int b = 0; b < batch; ++b)
    for (int i = threadIdx.x; i < parts; i += kRowThreads) sum += part[((long long)b * heads + head) * parts + i];
  sum = wave_sum(sum);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) grad[head] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

unsigned row_blocks(long long rows) { return (unsigned)((rows + kRowWaves - 1) / kRowWaves); }
size_t rows_bytes(const AttnLaunch &p) { return ((size_t)p.batch * p.heads * p.nq * sizeof(float) + 255) / 256 * 256; }

template <typename Tag>
hipError_t forward_t(const AttnLaunch &p, hipStream_t stream) {
  hipLaunchKernelGGL((attn_rows_forward_kernel<Tag>), dim3(row_blocks((long long)p.batch * p.nq * p.heads)), dim3(kRowThreads), 0, stream, p);
  return hipGetLastError();
}

template <typename Tag>
hipError_t backward_t(const AttnLaunch &p, hipStream_t stream) {
  float *delta = static_cast<float *>(p.workspace);
  float *slope_part = p.grad_slopes != nullptr ? reinterpret_cast<float *>(static_cast<char *>(p.workspace) + rows_bytes(p)) : nullptr;
  hipLaunchKernelGGL((attn_rows_grad_q_kernel<Tag>), dim3(row_blocks((long long)p.batch * p.nq * p.heads)), dim3(kRowThreads), 0, stream, p, delta, slope_part);
  if (hipError_t e = hipGetLastError()) return e;
  if (slope_part != nullptr) {
    hipLaunchKernelGGL(attn_slope_grad_kernel, dim3(p.heads), dim3(kRowThreads), 0, stream, slope_part, p.grad_slopes, p.batch, p.heads, p.nq);
    if (hipError_t e = hipGetLastError()) return e;
  }
  hipLaunchKernelGGL((attn_rows_grad_kv_kernel<Tag>), dim3(row_blocks((long long)p.batch * p.nk * p.kv_heads)), dim3(kRowThreads), 0, stream, p, delta);
  return hipGetLastError();
}

}  // namespace

size_t attn_forward_workspace_bytes(int, const AttnLaunch &) { return 0; }
size_t attn_backward_workspace_bytes(int, const AttnLaunch &p) { return rows_bytes(p) * (p.slopes != nullptr ? 2 : 1); }

hipError_t launch_attn_forward(int dtype, const AttnLaunch &p, hipStream_t stream) {
  switch (dtype) {
    case F32::kCode: return forward_t<F32>(p, stream);
    case F16::kCode: return forward_t<F16>(p, stream);
    case BF16::kCode: return forward_t<BF16>(p, stream);
  }
  return hipErrorInvalidValue;
}
hipError_t launch_attn_backward(int dtype, const AttnLaunch &p, hipStream_t stream) {
  switch (dtype) {
    case F32::kCode: return backward_t<F32>(p, stream);
    case F16::kCode: return backward_t<F16>(p, stream);
    case BF16::kCode: return backward_t<BF16>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace dcn
