// Layer normalisation of a sum, out = (z - mean) / sqrt(var + eps) * weight + bias with z = x + residual: what stands between
// the layers of a transformer, after the sum (post-norm) or with the sum kept as the stream (pre-norm).  Backward, with
// xhat = (z - mean) * rstd and a = grad_out * weight,
//   dz = rstd (a - mean(a) - xhat mean(a xhat)) + grad_sum,   dweight = sum over rows of grad_out xhat,   dbias = sum of grad_out
//
// HBM-bound: each tensor is read or written once.  A team of lanes (a power of two, up to a whole workgroup of 512) owns a row, a
// lane eight or twice eight elements of it, which stay in registers as fp32 from the sum to the result: the sum is not rounded
// before it is normalised.  The mean and the deviations about it are two reductions over the team; both are kept for the
// backward, 8 bytes a row, which then reduces once.  A workgroup walks a slab of rows with the parameters in registers and the next
// row's loads under way.  A row may start at any element and have any width: the loads are unaligned ones, the last
// elements of a width that is no multiple of eight are read and written one by one.
//
// The parameters' gradients are summed in registers down a workgroup's slab, over its teams through LDS, and over the workgroups by a
// second kernel, always in the same order.
#include "add_norm.hpp"

#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace dcn {
namespace {

struct None {};
constexpr int kVec = 8;

struct __attribute__((packed, aligned(2))) Unaligned { u32x4 v; };
struct Raw { u32x4 w[2]; };      // eight elements; of a 16-bit type in w[0]

template <typename Tag>
__device__ __forceinline__ void load_vec(const char *at, int live, Raw &r) {
  if (live == kVec) {
#pragma unroll
    for (int i = 0; i < Tag::kBytes / 2; ++i) r.w[i] = reinterpret_cast<const Unaligned *>(at)[i].v;
    return;
  }
  if constexpr (Tag::kBytes == 4) {
#pragma unroll
    for (int c = 0; c < kVec; ++c)
      if (c < live) r.w[c / 4][c % 4] = reinterpret_cast<const uint32_t *>(at)[c];
  } else {
#pragma unroll
    for (int c = 0; c < kVec; ++c)
      if (c < live) r.w[0][c / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(at)[c] << (c % 2 * 16);
  }
}
template <typename Tag>
__device__ __forceinline__ void decode_vec(const Raw &r, float (&f)[kVec]) {
  if constexpr (Tag::kBytes == 4) {
    float a[4], b[4];
    Pack<Tag, 4>::decode(r.w[0], a);
    Pack<Tag, 4>::decode(r.w[1], b);
#pragma unroll
    for (int c = 0; c < 4; ++c) { f[c] = a[c]; f[4 + c] = b[c]; }
  } else {
    Pack<Tag, 8>::decode(r.w[0], f);
  }
}
template <typename Tag>
__device__ __forceinline__ void store_vec(char *at, int live, const float (&f)[kVec]) {
  if (live == kVec) {
    if constexpr (Tag::kBytes == 4) {
      const float a[4] = {f[0], f[1], f[2], f[3]}, b[4] = {f[4], f[5], f[6], f[7]};
      reinterpret_cast<Unaligned *>(at)[0].v = Pack<Tag, 4>::encode(a);
      reinterpret_cast<Unaligned *>(at)[1].v = Pack<Tag, 4>::encode(b);
    } else {
      reinterpret_cast<Unaligned *>(at)->v = Pack<Tag, 8>::encode(f);
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < kVec; ++c)
    if (c < live) {
      const float one[1] = {f[c]};
      reinterpret_cast<typename RawWord<Tag::kBytes>::type *>(at)[c] = Pack<Tag, 1>::encode(one);
    }
}
// Parameters go by their type's code, one for all lanes.
__device__ __forceinline__ int bytes_of(int dtype) { return dtype == F32::kCode ? 4 : 2; }
__device__ __forceinline__ void load_params(const AddNormLaunch &p, const void *v, float none, int column, int live, float (&f)[kVec]) {
#pragma unroll
  for (int c = 0; c < kVec; ++c) f[c] = none;
  if (v == nullptr || live == 0) return;
  const char *at = static_cast<const char *>(v) + (long long)column * bytes_of(p.param_dtype);
  Raw r = {};
  if (p.param_dtype == F32::kCode) {
    load_vec<F32>(at, live, r);
    decode_vec<F32>(r, f);
  } else {
    load_vec<F16>(at, live, r);
    if (p.param_dtype == F16::kCode) decode_vec<F16>(r, f);
    else decode_vec<BF16>(r, f);
  }
}
template <typename Tag>
__device__ __forceinline__ char *element(const void *base, long long i) { return static_cast<char *>(const_cast<void *>(base)) + i * Tag::kBytes; }

// Sums over a team of lanes.  A team that is a whole workgroup of several waves meets in LDS; two sets of slots in turn, so one
// barrier a sum is enough.
constexpr int kMostWaves = 8;
template <int N>
__device__ __forceinline__ void team_sum(float (&v)[N], int team, float (*slots)[kMostWaves][2], int &turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = cluster_sum(v[i], team < kWave ? team : kWave);
  if (team <= kWave) return;
  const int wave = threadIdx.x / kWave, waves = team / kWave;
  if (threadIdx.x % kWave == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) slots[turn][wave][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int w = 0; w < waves; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += slots[turn][w][i];
  turn ^= 1;
}

struct Geometry {
  int team;             // lanes a row
  int threads;          // of a workgroup; == team where that is more than a wave
  long long slab;       // rows a workgroup, a multiple of its teams
  unsigned blocks;
};

// X, R: the summands' types (R may be None); the sum has the wider one's, the result as well or, WIDE, fp32.  V: vectors a lane.
template <typename X_, typename R_, bool WIDE, int V_>
struct Types {
  typedef X_ X;
  typedef R_ R;
  static constexpr bool kSum = !std::is_same_v<R, None>;
  typedef std::conditional_t<std::is_same_v<R, F32>, F32, X> Sum;
  typedef std::conditional_t<WIDE, F32, Sum> Out;
  static constexpr int V = V_;
};

// What a lane reads of a row: x and, where there is one, the residual.
template <typename T>
struct RowLoads {
  Raw x[T::V], r[T::V];
  __device__ __forceinline__ void request(const AddNormLaunch &p, long long row, const int (&column)[T::V], const int (&live)[T::V]) {
#pragma unroll
    for (int u = 0; u < T::V; ++u) {
      x[u] = {};
      r[u] = {};
      if (live[u] == 0) continue;
      load_vec<typename T::X>(element<typename T::X>(p.x.base, row * p.x.pitch + column[u]), live[u], x[u]);
      if constexpr (T::kSum) load_vec<typename T::R>(element<typename T::R>(p.residual.base, row * p.residual.pitch + column[u]), live[u], r[u]);
    }
  }
  __device__ __forceinline__ void sum(float (&z)[T::V][kVec]) const {
#pragma unroll
    for (int u = 0; u < T::V; ++u) {
      decode_vec<typename T::X>(x[u], z[u]);
      if constexpr (T::kSum) {
        float f[kVec];
        decode_vec<typename T::R>(r[u], f);
#pragma unroll
        for (int c = 0; c < kVec; ++c) z[u][c] += f[c];
      }
    }
  }
};

constexpr int kMostThreads = kMostWaves * kWave;
template <typename T>
__global__ void __launch_bounds__(kMostThreads) add_norm_forward_kernel(const AddNormLaunch p, const Geometry g) {
  constexpr int V = T::V;
  __shared__ float s_slots[2][kMostWaves][2];
  int turn = 0;
  const int teams = (int)blockDim.x / g.team, mine = threadIdx.x / g.team;
  int column[V], width_live[V], none[V];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    column[u] = ((threadIdx.x & (g.team - 1)) + u * g.team) * kVec;
    width_live[u] = min(kVec, max(0, p.width - column[u]));
    none[u] = 0;
  }
  const float inv = 1.f / (float)p.width;
  const long long begin = blockIdx.x * g.slab, end = min(begin + g.slab, p.rows);
  RowLoads<T> next;
  next.request(p, begin + mine, column, begin + mine < end ? width_live : none);
  float w[V][kVec], b[V][kVec];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    load_params(p, p.weight, 1.f, column[u], width_live[u], w[u]);
    load_params(p, p.bias, 0.f, column[u], width_live[u], b[u]);
  }
  for (long long row0 = begin; row0 < end; row0 += teams) {
    const long long row = row0 + mine;
    float z[V][kVec];
    next.sum(z);
    next.request(p, row + teams, column, row + teams < end ? width_live : none);
    float sum[1] = {0.f};
#pragma unroll
    for (int u = 0; u < V; ++u)
#pragma unroll
      for (int c = 0; c < kVec; ++c) sum[0] += z[u][c];      // zeros beyond the width
    team_sum(sum, g.team, s_slots, turn);
    const float mean = sum[0] * inv;
    float squares[1] = {0.f};
#pragma unroll
    for (int u = 0; u < V; ++u)
#pragma unroll
      for (int c = 0; c < kVec; ++c) squares[0] = c < width_live[u] ? fmaf(z[u][c] - mean, z[u][c] - mean, squares[0]) : squares[0];
    team_sum(squares, g.team, s_slots, turn);
    const float rstd = 1.f / sqrtf(fmaf(squares[0], inv, p.eps));
    if (row >= end) continue;
    if (p.stats != nullptr && column[0] == 0) reinterpret_cast<f32x2 *>(p.stats)[row] = f32x2{mean, rstd};
#pragma unroll
    for (int u = 0; u < V; ++u) {
      if (width_live[u] == 0) continue;
      const long long at = row * p.width + column[u];
      if (p.sum != nullptr) store_vec<typename T::Sum>(element<typename T::Sum>(p.sum, at), width_live[u], z[u]);
#pragma unroll
      for (int c = 0; c < kVec; ++c) z[u][c] = fmaf((z[u][c] - mean) * rstd, w[u][c], b[u][c]);
      store_vec<typename T::Out>(element<typename T::Out>(p.out, at), width_live[u], z[u]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kMostThreads) add_norm_backward_kernel(const AddNormLaunch p, const Geometry g) {
  constexpr int V = T::V;
  typedef typename T::Out Out;
  typedef typename T::Sum Sum;
  extern __shared__ float s_columns[];      // [teams][vectors * 8]
  __shared__ float s_slots[2][kMostWaves][2];
  int turn = 0;
  const int teams = (int)blockDim.x / g.team, mine = threadIdx.x / g.team;
  int column[V], width_live[V], none[V];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    column[u] = ((threadIdx.x & (g.team - 1)) + u * g.team) * kVec;
    width_live[u] = min(kVec, max(0, p.width - column[u]));
    none[u] = 0;
  }
  const float inv = 1.f / (float)p.width;
  const long long begin = blockIdx.x * g.slab, end = min(begin + g.slab, p.rows);
  RowLoads<T> next;
  Raw next_g[V], next_s[V];
  f32x2 next_stats;
  auto request = [&](long long row) {
    next.request(p, row, column, row < end ? width_live : none);
    next_stats = f32x2{0.f, 0.f};
    if (row < end) next_stats = reinterpret_cast<const f32x2 *>(p.stats)[row];
#pragma unroll
    for (int u = 0; u < V; ++u) {
      next_g[u] = {};
      next_s[u] = {};
      if (row >= end || width_live[u] == 0) continue;
      const long long at = row * p.width + column[u];
      load_vec<Out>(element<Out>(p.grad_out, at), width_live[u], next_g[u]);
      if (p.grad_sum != nullptr) load_vec<Sum>(element<Sum>(p.grad_sum, at), width_live[u], next_s[u]);
    }
  };
  request(begin + mine);
  float w[V][kVec], dw[V][kVec], db[V][kVec];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    load_params(p, p.weight, 1.f, column[u], width_live[u], w[u]);
#pragma unroll
    for (int c = 0; c < kVec; ++c) dw[u][c] = db[u][c] = 0.f;
  }
  for (long long row0 = begin; row0 < end; row0 += teams) {
    const long long row = row0 + mine;
    float z[V][kVec], a[V][kVec], around[V][kVec];
    next.sum(z);
#pragma unroll
    for (int u = 0; u < V; ++u) {
      decode_vec<Out>(next_g[u], a[u]);
      decode_vec<Sum>(next_s[u], around[u]);
    }
    const float rstd = next_stats.y, shift = -next_stats.x * rstd;
    request(row + teams);
    float sums[2] = {0.f, 0.f};
    // beyond the width and the rows the gradients are zeros, and so is all that is added up
#pragma unroll
    for (int u = 0; u < V; ++u)
#pragma unroll
      for (int c = 0; c < kVec; ++c) {
        z[u][c] = fmaf(z[u][c], rstd, shift);
        dw[u][c] = fmaf(a[u][c], z[u][c], dw[u][c]);
        db[u][c] += a[u][c];
        a[u][c] *= w[u][c];
        sums[0] += a[u][c];
        sums[1] = fmaf(a[u][c], z[u][c], sums[1]);
      }
    team_sum(sums, g.team, s_slots, turn);
    if (row >= end) continue;
    const float m1 = sums[0] * inv, m2 = sums[1] * inv;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      if (width_live[u] == 0) continue;
      const long long at = row * p.width + column[u];
#pragma unroll
      for (int c = 0; c < kVec; ++c) a[u][c] = fmaf(rstd, a[u][c] - m1 - z[u][c] * m2, around[u][c]);
      if (p.grad_x != nullptr) store_vec<typename T::X>(element<typename T::X>(p.grad_x, at), width_live[u], a[u]);
      if constexpr (T::kSum)
        if (p.grad_residual != nullptr) store_vec<typename T::R>(element<typename T::R>(p.grad_residual, at), width_live[u], a[u]);
    }
  }
  if (p.grad_weight == nullptr && p.grad_bias == nullptr) return;
  const int padded = (p.width + kVec - 1) / kVec * kVec;
  float *part = static_cast<float *>(p.workspace) + (size_t)blockIdx.x * 2 * padded;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < V; ++u)
      if (width_live[u] > 0)
#pragma unroll
        for (int c = 0; c < kVec; ++c) s_columns[(size_t)mine * padded + column[u] + c] = q == 0 ? dw[u][c] : db[u][c];
    __syncthreads();
    for (int c = threadIdx.x; c < padded; c += blockDim.x) {
      float sum = 0.f;
      for (int t = 0; t < teams; ++t) sum += s_columns[(size_t)t * padded + c];
      part[(size_t)q * padded + c] = sum;
    }
  }
}

// The workgroups' sums [blocks][2][padded width]: a workgroup takes 32 columns, 32 lanes each, four loads a lane under way; the lanes'
// sums meet in LDS in their order.
constexpr int kGradColumns = 32, kGradLanes = 32;
__global__ void __launch_bounds__(kGradColumns * kGradLanes) add_norm_param_grad_kernel(const AddNormLaunch p, unsigned blocks) {
  __shared__ float s_part[kGradLanes][kGradColumns + 1];
  const int padded = (p.width + kVec - 1) / kVec * kVec;
  const int c = threadIdx.x % kGradColumns, lane = threadIdx.x / kGradColumns, index = blockIdx.x * kGradColumns + c;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (index < 2 * padded) {
    const float *from = static_cast<const float *>(p.workspace) + index;
    const size_t step = (size_t)2 * padded;
    unsigned i = lane;
    for (; i + 3 * kGradLanes < blocks; i += 4 * kGradLanes)
#pragma unroll
      for (int u = 0; u < 4; ++u) sum[u] += from[(i + u * kGradLanes) * step];
    for (; i < blocks; i += kGradLanes) sum[0] += from[i * step];
  }
  s_part[lane][c] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (lane != 0 || index >= 2 * padded) return;
  const int column = index < padded ? index : index - padded;
  void *to = index < padded ? p.grad_weight : p.grad_bias;
  if (to == nullptr || column >= p.width) return;
  float total[kVec] = {};
#pragma unroll
  for (int l = 0; l < kGradLanes; ++l) total[0] += s_part[l][c];
  char *at = static_cast<char *>(to) + (long long)column * bytes_of(p.param_dtype);
  if (p.param_dtype == F32::kCode) store_vec<F32>(at, 1, total);
  else if (p.param_dtype == F16::kCode) store_vec<F16>(at, 1, total);
  else store_vec<BF16>(at, 1, total);
}

// A lane has two vectors of rows of more than 64, so that a wave holds a row of up to 1024 channels and meets no barrier.
int vectors_of(const AddNormLaunch &p) { return (p.width + kVec - 1) / kVec; }
bool two_a_lane(const AddNormLaunch &p) { return vectors_of(p) > kWave; }
// Parameters in registers pay over several rows; workgroups enough to fill the chip come first.
Geometry geometry(const AddNormLaunch &p, long long most_blocks) {
  Geometry g;
  const int vectors = (vectors_of(p) + two_a_lane(p)) / (two_a_lane(p) ? 2 : 1);
  g.team = 1;
  while (g.team < vectors) g.team *= 2;
  g.threads = std::max(g.team, 64);
  if (g.team <= kWave && p.rows * g.team >= 256ll * 1024) g.threads = 256;
  const long long teams = g.threads / g.team, passes = (p.rows + teams - 1) / teams;
  const long long blocks = std::min(passes, most_blocks);
  g.slab = (passes + blocks - 1) / blocks * teams;
  g.blocks = (unsigned)((p.rows + g.slab - 1) / g.slab);
  return g;
}
Geometry forward_geometry(const AddNormLaunch &p) { return geometry(p, 4096); }
Geometry backward_geometry(const AddNormLaunch &p) {
  // partial sums stay below 32 MB
  const long long columns = (long long)vectors_of(p) * kVec;
  return geometry(p, std::max<long long>(1, std::min<long long>(1024, (32ll << 20) / (8 * columns))));
}

template <typename T>
hipError_t run(const AddNormLaunch &p, hipStream_t stream, bool backward) {
  if (!backward) {
    const Geometry g = forward_geometry(p);
    hipLaunchKernelGGL((add_norm_forward_kernel<T>), dim3(g.blocks), dim3(g.threads), 0, stream, p, g);
    return hipGetLastError();
  }
  const Geometry g = backward_geometry(p);
  const int padded = vectors_of(p) * kVec;
  const size_t lds = (size_t)(g.threads / g.team) * padded * sizeof(float);
  hipLaunchKernelGGL((add_norm_backward_kernel<T>), dim3(g.blocks), dim3(g.threads), lds, stream, p, g);
  if (hipError_t e = hipGetLastError()) return e;
  if (p.grad_weight == nullptr && p.grad_bias == nullptr) return hipSuccess;
  hipLaunchKernelGGL(add_norm_param_grad_kernel, dim3((2 * padded + kGradColumns - 1) / kGradColumns), dim3(kGradColumns * kGradLanes), 0, stream, p, g.blocks);
  return hipGetLastError();
}
template <typename X, typename R, bool WIDE>
hipError_t with_types(const AddNormLaunch &p, hipStream_t stream, bool backward) {
  return two_a_lane(p) ? run<Types<X, R, WIDE, 2>>(p, stream, backward) : run<Types<X, R, WIDE, 1>>(p, stream, backward);
}
template <typename X>
hipError_t with_residual(const AddNormLaunch &p, hipStream_t stream, bool backward) {
  const bool none = p.residual.base == nullptr;
  if constexpr (X::kCode == F32::kCode) {
    if (none) return with_types<X, None, false>(p, stream, backward);
    return p.residual.dtype == X::kCode ? with_types<X, X, false>(p, stream, backward) : hipErrorInvalidValue;
  } else {
    if (none) return p.wide ? with_types<X, None, true>(p, stream, backward) : with_types<X, None, false>(p, stream, backward);
    if (p.residual.dtype == F32::kCode) return with_types<X, F32, false>(p, stream, backward);
    if (p.residual.dtype != X::kCode) return hipErrorInvalidValue;
    return p.wide ? with_types<X, X, true>(p, stream, backward) : with_types<X, X, false>(p, stream, backward);
  }
}
hipError_t launch(const AddNormLaunch &p, hipStream_t stream, bool backward) {
  if (p.rows <= 0 || p.width <= 0 || p.width > kMaxNormWidth) return hipErrorInvalidValue;
  switch (p.x.dtype) {
    case F32::kCode: return with_residual<F32>(p, stream, backward);
    case F16::kCode: return with_residual<F16>(p, stream, backward);
    case BF16::kCode: return with_residual<BF16>(p, stream, backward);
  }
  return hipErrorInvalidValue;
}

}  // namespace

size_t add_norm_backward_workspace_bytes(const AddNormLaunch &p) {
  if (p.grad_weight == nullptr && p.grad_bias == nullptr) return 0;
  return (size_t)backward_geometry(p).blocks * 2 * vectors_of(p) * kVec * sizeof(float);
}
hipError_t launch_add_norm_forward(const AddNormLaunch &p, hipStream_t stream) { return launch(p, stream, false); }
hipError_t launch_add_norm_backward(const AddNormLaunch &p, hipStream_t stream) { return launch(p, stream, true); }

}  // namespace dcn
