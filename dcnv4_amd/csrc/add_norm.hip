// Layer normalisation of a sum, out = (z - mean) / sqrt(var + eps) * weight + bias with z = x + residual: what stands between
// the layers of a transformer, after the sum (post-norm) or with the sum kept as the stream (pre-norm).  Backward, with
// xhat = (z - mean) * rstd and a = grad_out * weight,
//   dz = rstd (a - mean(a) - xhat mean(a xhat)) + grad_sum,   dweight = sum over rows of grad_out xhat,   dbias = sum of grad_out
//
// HBM-bound: each tensor is read or written once.  A team of lanes (a power of two, up to a whole workgroup of 512) owns a row, a
// lane eight or sixteen elements of it, which stay in registers as fp32 from the sum to the result: the sum is not rounded
// before it is normalised.  The mean and the deviations about it are two reductions over the team; both are kept for the
// backward, 8 bytes a row, which then reduces once.  A workgroup walks a slab of rows with the parameters in registers and the loads of the
// next under way.
//
// Rows that all start on 16 bytes go in vectors of eight elements.  Others (an odd width, an odd offset) go element by element, neighbours
// in neighbouring lanes: a 16-byte access that crosses its alignment costs twice (100000 x 1023, 16 bits, forward 283 us and backward 589
// in unaligned vectors, 195 and 251 so; 1024 channels 147 and 222, all on one machine; on another 164 and 233, and 121 and 179).  The backward
// reads up to four tensors for the one it writes: 4.5 to 4.7 TB/s of the 5.0 to 5.3 that a plain stream of that mix reaches; loads two rows ahead
// were slower (401408 x 112: 112 us for 98).
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

// One access: G consecutive elements, eight or one.
template <typename Tag, int G> struct Access {
  static constexpr int kWords = G * Tag::kBytes > 16 ? 2 : 1;
  typedef Pack<Tag, G / kWords> pack_t;
  struct raw_t { typename pack_t::raw_t w[kWords]; };
  static __device__ __forceinline__ raw_t load(const char *at) { return *reinterpret_cast<const raw_t *>(at); }
  static __device__ __forceinline__ void decode(const raw_t &r, float (&f)[G]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      float part[G / kWords];
      pack_t::decode(r.w[i], part);
#pragma unroll
      for (int c = 0; c < G / kWords; ++c) f[i * (G / kWords) + c] = part[c];
    }
  }
  static __device__ __forceinline__ void store(char *at, const float (&f)[G]) {
    raw_t r;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      float part[G / kWords];
#pragma unroll
      for (int c = 0; c < G / kWords; ++c) part[c] = f[i * (G / kWords) + c];
      r.w[i] = pack_t::encode(part);
    }
    *reinterpret_cast<raw_t *>(at) = r;
  }
};
// Parameters go by their type's code, one for all lanes.
__device__ __forceinline__ int bytes_of(int dtype) { return dtype == F32::kCode ? 4 : 2; }
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

// X, R: the summands' types (R may be None); the sum has the wider one's, the result as well or, WIDE, fp32.  A lane makes N accesses
// of G elements a row.
template <typename X_, typename R_, bool WIDE, int G_, int N_>
struct Types {
  typedef X_ X;
  typedef R_ R;
  static constexpr bool kSum = !std::is_same_v<R, None>;
  typedef std::conditional_t<std::is_same_v<R, F32>, F32, X> Sum;
  typedef std::conditional_t<WIDE, F32, Sum> Out;
  static constexpr int G = G_, N = N_;
};

// The columns of a lane.
template <typename T>
struct Columns {
  int at[T::N];
  bool live[T::N];
  __device__ __forceinline__ Columns(int team, int width) {
#pragma unroll
    for (int n = 0; n < T::N; ++n) {
      at[n] = ((threadIdx.x & (team - 1)) + n * team) * T::G;
      live[n] = at[n] < width;
    }
  }
};

// What a lane reads of a row: x and, where there is one, the residual.
template <typename T>
struct RowLoads {
  typedef Access<typename T::X, T::G> ax;
  typedef Access<std::conditional_t<T::kSum, typename T::R, typename T::X>, T::G> ar;
  typename ax::raw_t x[T::N];
  typename ar::raw_t r[T::N];
  __device__ __forceinline__ void request(const AddNormLaunch &p, long long row, const Columns<T> &c, bool there) {
#pragma unroll
    for (int n = 0; n < T::N; ++n) {
      x[n] = {};
      r[n] = {};
      if (!there || !c.live[n]) continue;
      x[n] = ax::load(element<typename T::X>(p.x.base, row * p.x.pitch + c.at[n]));
      if constexpr (T::kSum) r[n] = ar::load(element<typename T::R>(p.residual.base, row * p.residual.pitch + c.at[n]));
    }
  }
  __device__ __forceinline__ void sum(float (&z)[T::N][T::G]) const {
#pragma unroll
    for (int n = 0; n < T::N; ++n) {
      ax::decode(x[n], z[n]);
      if constexpr (T::kSum) {
        float f[T::G];
        ar::decode(r[n], f);
#pragma unroll
        for (int c = 0; c < T::G; ++c) z[n][c] += f[c];
      }
    }
  }
};

template <typename T, typename Tag>
__device__ __forceinline__ void load_params(const void *v, const Columns<T> &column, float (&f)[T::N][T::G]) {
  typename Access<Tag, T::G>::raw_t r[T::N];
#pragma unroll
  for (int n = 0; n < T::N; ++n)
    if (column.live[n]) r[n] = Access<Tag, T::G>::load(element<Tag>(v, column.at[n]));
#pragma unroll
  for (int n = 0; n < T::N; ++n)
    if (column.live[n]) Access<Tag, T::G>::decode(r[n], f[n]);
}
template <typename T>
__device__ __forceinline__ void load_params(const AddNormLaunch &p, const void *v, float none, const Columns<T> &column, float (&f)[T::N][T::G]) {
#pragma unroll
  for (int n = 0; n < T::N; ++n)
#pragma unroll
    for (int c = 0; c < T::G; ++c) f[n][c] = none;
  if (v == nullptr) return;
  if (p.param_dtype == F32::kCode) load_params<T, F32>(v, column, f);
  else if (p.param_dtype == F16::kCode) load_params<T, F16>(v, column, f);
  else load_params<T, BF16>(v, column, f);
}

constexpr int kMostThreads = kMostWaves * kWave;
template <typename T>
__global__ void __launch_bounds__(kMostThreads) add_norm_forward_kernel(const AddNormLaunch p, const Geometry g) {
  constexpr int N = T::N, G = T::G;
  __shared__ float s_slots[2][kMostWaves][2];
  int turn = 0;
  const int teams = (int)blockDim.x / g.team, mine = threadIdx.x / g.team;
  const Columns<T> column(g.team, p.width);
  const float inv = 1.f / (float)p.width;
  const long long begin = blockIdx.x * g.slab, end = min(begin + g.slab, p.rows);
  RowLoads<T> next;
  next.request(p, begin + mine, column, begin + mine < end);
  float w[N][G], b[N][G];
  load_params<T>(p, p.weight, 1.f, column, w);
  load_params<T>(p, p.bias, 0.f, column, b);
  for (long long row0 = begin; row0 < end; row0 += teams) {
    const long long row = row0 + mine;
    float z[N][G];
    next.sum(z);
    next.request(p, row + teams, column, row + teams < end);
    float sum[1] = {0.f};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int c = 0; c < G; ++c) sum[0] += z[n][c];      // zeros beyond the width
    team_sum(sum, g.team, s_slots, turn);
    const float mean = sum[0] * inv;
    float squares[1] = {0.f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float own = squares[0];
#pragma unroll
      for (int c = 0; c < G; ++c) own = fmaf(z[n][c] - mean, z[n][c] - mean, own);
      squares[0] = column.live[n] ? own : squares[0];
    }
    team_sum(squares, g.team, s_slots, turn);
    const float rstd = 1.f / sqrtf(fmaf(squares[0], inv, p.eps));
    if (row >= end) continue;
    if (p.stats != nullptr && column.at[0] == 0) reinterpret_cast<f32x2 *>(p.stats)[row] = f32x2{mean, rstd};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!column.live[n]) continue;
      const long long at = row * p.width + column.at[n];
      if (p.sum != nullptr) Access<typename T::Sum, G>::store(element<typename T::Sum>(p.sum, at), z[n]);
#pragma unroll
      for (int c = 0; c < G; ++c) z[n][c] = fmaf((z[n][c] - mean) * rstd, w[n][c], b[n][c]);
      Access<typename T::Out, G>::store(element<typename T::Out>(p.out, at), z[n]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kMostThreads) add_norm_backward_kernel(const AddNormLaunch p, const Geometry g) {
  constexpr int N = T::N, G = T::G;
  typedef typename T::Out Out;
  typedef typename T::Sum Sum;
  extern __shared__ float s_columns[];      // [teams][width]
  __shared__ float s_slots[2][kMostWaves][2];
  int turn = 0;
  const int teams = (int)blockDim.x / g.team, mine = threadIdx.x / g.team;
  const Columns<T> column(g.team, p.width);
  const float inv = 1.f / (float)p.width;
  const long long begin = blockIdx.x * g.slab, end = min(begin + g.slab, p.rows);
  RowLoads<T> next;
  typename Access<Out, G>::raw_t next_g[N];
  typename Access<Sum, G>::raw_t next_s[N];
  f32x2 next_stats;
  auto request = [&](long long row) {
    const bool there = row < end;
    next.request(p, row, column, there);
    next_stats = f32x2{0.f, 0.f};
    if (there) next_stats = reinterpret_cast<const f32x2 *>(p.stats)[row];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      next_g[n] = {};
      next_s[n] = {};
      if (!there || !column.live[n]) continue;
      const long long at = row * p.width + column.at[n];
      next_g[n] = Access<Out, G>::load(element<Out>(p.grad_out, at));
      if (p.grad_sum != nullptr) next_s[n] = Access<Sum, G>::load(element<Sum>(p.grad_sum, at));
    }
  };
  request(begin + mine);
  float w[N][G], dw[N][G], db[N][G];
  load_params<T>(p, p.weight, 1.f, column, w);
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int c = 0; c < G; ++c) dw[n][c] = db[n][c] = 0.f;
  for (long long row0 = begin; row0 < end; row0 += teams) {
    const long long row = row0 + mine;
    float z[N][G], a[N][G], around[N][G];
    next.sum(z);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      Access<Out, G>::decode(next_g[n], a[n]);
      Access<Sum, G>::decode(next_s[n], around[n]);
    }
    const float mean = next_stats.x, rstd = next_stats.y;
    request(row + teams);
    float sums[2] = {0.f, 0.f};
    // beyond the width and the rows the gradients are zeros, and so is all that is added up
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int c = 0; c < G; ++c) {
        z[n][c] = (z[n][c] - mean) * rstd;      // as the forward: z rstd - mean rstd would lose what is small beside the mean
        dw[n][c] = fmaf(a[n][c], z[n][c], dw[n][c]);
        db[n][c] += a[n][c];
        a[n][c] *= w[n][c];
        sums[0] += a[n][c];
        sums[1] = fmaf(a[n][c], z[n][c], sums[1]);
      }
    team_sum(sums, g.team, s_slots, turn);
    if (row >= end) continue;
    const float m1 = sums[0] * inv, m2 = sums[1] * inv;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!column.live[n]) continue;
      const long long at = row * p.width + column.at[n];
#pragma unroll
      for (int c = 0; c < G; ++c) a[n][c] = fmaf(rstd, a[n][c] - m1 - z[n][c] * m2, around[n][c]);
      if (p.grad_x != nullptr) Access<typename T::X, G>::store(element<typename T::X>(p.grad_x, at), a[n]);
      if constexpr (T::kSum)
        if (p.grad_residual != nullptr) Access<typename T::R, G>::store(element<typename T::R>(p.grad_residual, at), a[n]);
    }
  }
  if (p.grad_weight == nullptr && p.grad_bias == nullptr) return;
  float *part = static_cast<float *>(p.workspace) + (size_t)blockIdx.x * 2 * p.width;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (column.live[n])
#pragma unroll
        for (int c = 0; c < G; ++c) s_columns[(size_t)mine * p.width + column.at[n] + c] = q == 0 ? dw[n][c] : db[n][c];
    __syncthreads();
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      float sum = 0.f;
      for (int t = 0; t < teams; ++t) sum += s_columns[(size_t)t * p.width + c];
      part[(size_t)q * p.width + c] = sum;
    }
  }
}

// The workgroups' sums [blocks][2][width]: a workgroup takes 32 columns, 32 lanes each, four loads a lane under way; the lanes'
// sums meet in LDS in their order.
constexpr int kGradColumns = 32, kGradLanes = 32;
__global__ void __launch_bounds__(kGradColumns * kGradLanes) add_norm_param_grad_kernel(const AddNormLaunch p, unsigned blocks) {
  __shared__ float s_part[kGradLanes][kGradColumns + 1];
  const int c = threadIdx.x % kGradColumns, lane = threadIdx.x / kGradColumns, index = blockIdx.x * kGradColumns + c;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (index < 2 * p.width) {
    const float *from = static_cast<const float *>(p.workspace) + index;
    const size_t step = (size_t)2 * p.width;
    unsigned i = lane;
    for (; i + 3 * kGradLanes < blocks; i += 4 * kGradLanes)
#pragma unroll
      for (int u = 0; u < 4; ++u) sum[u] += from[(i + u * kGradLanes) * step];
    for (; i < blocks; i += kGradLanes) sum[0] += from[i * step];
  }
  s_part[lane][c] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (lane != 0 || index >= 2 * p.width) return;
  void *to = index < p.width ? p.grad_weight : p.grad_bias;
  if (to == nullptr) return;
  float total[1] = {0.f};
#pragma unroll
  for (int l = 0; l < kGradLanes; ++l) total[0] += s_part[l][c];
  char *at = static_cast<char *>(to) + (long long)(index < p.width ? index : index - p.width) * bytes_of(p.param_dtype);
  if (p.param_dtype == F32::kCode) Access<F32, 1>::store(at, total);
  else if (p.param_dtype == F16::kCode) Access<F16, 1>::store(at, total);
  else Access<BF16, 1>::store(at, total);
}

// Whether every row of every tensor starts on 16 bytes and is whole vectors.
bool in_vectors(const AddNormLaunch &p) {
  auto fits = [](const void *base, long long bytes) { return reinterpret_cast<uintptr_t>(base) % 16 == 0 && bytes % 16 == 0; };
  auto row_fits = [&](const NormRows &t) { return t.base == nullptr || fits(t.base, t.pitch * (t.dtype == F32::kCode ? 4 : 2)); };
  return p.width % 8 == 0 && row_fits(p.x) && row_fits(p.residual) && fits(p.weight, 0) && fits(p.bias, 0) && fits(p.out, 0) && fits(p.sum, 0) &&
         fits(p.grad_out, 0) && fits(p.grad_sum, 0) && fits(p.grad_x, 0) && fits(p.grad_residual, 0);
}
// Elements a lane: eight, and sixteen where a row needs more than 512 lanes of eight.  Sixteen also for many rows of 513 to 1024
// channels: a wave then holds a row and meets no barrier, which pays once the waves are many (768 channels, 16 bits, 8 and 16: forward
// of 5003 rows 10.4 and 10.3 us, of 40000 49.7 and 43.5; backward 14.6 and 17.8, 81 and 60).  The forward of rows that go element
// by element stays at eight (20000 x 1001: 42 us and 68).
int lane_elements(const AddNormLaunch &p, bool backward) {
  if (p.width > 4096) return 16;
  return p.width > 512 && p.width <= 1024 && p.rows > 16384 && (backward || in_vectors(p)) ? 16 : 8;
}
// Parameters in registers pay over several rows; workgroups enough to fill the chip come first.
Geometry geometry(const AddNormLaunch &p, int elements, long long most_blocks) {
  Geometry g;
  g.team = 1;
  while (g.team * elements < p.width) g.team *= 2;
  g.threads = std::max(g.team, 64);
  if (g.team <= kWave && p.rows * g.team >= 256ll * 1024) g.threads = 256;
  const long long teams = g.threads / g.team, passes = (p.rows + teams - 1) / teams;
  const long long blocks = std::min(passes, most_blocks);
  g.slab = (passes + blocks - 1) / blocks * teams;
  g.blocks = (unsigned)((p.rows + g.slab - 1) / g.slab);
  return g;
}
Geometry forward_geometry(const AddNormLaunch &p) { return geometry(p, lane_elements(p, false), 4096); }
Geometry backward_geometry(const AddNormLaunch &p) {
  // partial sums stay below 32 MB
  return geometry(p, lane_elements(p, true), std::max<long long>(1, std::min<long long>(1024, (32ll << 20) / (8ll * p.width))));
}

template <typename T>
hipError_t run(const AddNormLaunch &p, hipStream_t stream, bool backward) {
  if (!backward) {
    const Geometry g = forward_geometry(p);
    hipLaunchKernelGGL((add_norm_forward_kernel<T>), dim3(g.blocks), dim3(g.threads), 0, stream, p, g);
    return hipGetLastError();
  }
  const Geometry g = backward_geometry(p);
  const size_t lds = (size_t)(g.threads / g.team) * p.width * sizeof(float);
  hipLaunchKernelGGL((add_norm_backward_kernel<T>), dim3(g.blocks), dim3(g.threads), lds, stream, p, g);
  if (hipError_t e = hipGetLastError()) return e;
  if (p.grad_weight == nullptr && p.grad_bias == nullptr) return hipSuccess;
  hipLaunchKernelGGL(add_norm_param_grad_kernel, dim3((2 * p.width + kGradColumns - 1) / kGradColumns), dim3(kGradColumns * kGradLanes), 0, stream, p, g.blocks);
  return hipGetLastError();
}
template <typename X, typename R, bool WIDE>
hipError_t with_types(const AddNormLaunch &p, hipStream_t stream, bool backward) {
  const int elements = lane_elements(p, backward);
  if (in_vectors(p)) return elements == 8 ? run<Types<X, R, WIDE, 8, 1>>(p, stream, backward) : run<Types<X, R, WIDE, 8, 2>>(p, stream, backward);
  return elements == 8 ? run<Types<X, R, WIDE, 1, 8>>(p, stream, backward) : run<Types<X, R, WIDE, 1, 16>>(p, stream, backward);
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
  return (size_t)backward_geometry(p).blocks * 2 * p.width * sizeof(float);
}
hipError_t launch_add_norm_forward(const AddNormLaunch &p, hipStream_t stream) { return launch(p, stream, false); }
hipError_t launch_add_norm_backward(const AddNormLaunch &p, hipStream_t stream) { return launch(p, stream, true); }

}  // namespace dcn
