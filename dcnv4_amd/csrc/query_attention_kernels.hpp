#pragma once
// Attention among queries, the dense attention beside the sampling one of a deformable decoder.  Per sequence and head
//   x_ij = scale q_i . k_j,   s_ij = cap tanh(x_ij / cap) - slope |p_i - p_j|   (the cap and the distance where there are any)
//   out_i = sum_j P_ij v_j,   P = softmax over the keys that i sees;  a row that sees none is zeros
// where i sees j if i's segment number is not negative and j's is the same or 0.  Backward, with delta_i = dO_i . out_i:
//   dV = P^T dO,  dS = P (dO V^T - delta),  dslope = -sum dS |p_i - p_j|,  dX = dS (1 - tanh^2),  dQ = scale dX K,  dK = scale dX^T Q
// Heads that share a key head add up in its gradient.
//
// One scheme for the three kernels (forward, dQ, dK and dV).  A workgroup owns *columns* - queries, queries, keys - whose operands
// lie in registers, and walks *rows* - keys, keys, queries - in tiles that come through LDS.  A matrix instruction forms 16 rows x 16
// columns of scores with the rows first: lane (g, c) then holds rows 4 g .. + 3 of column c, which is how the next instruction
// wants the weights, as its second operand with the rows as depth, so weights never leave the registers.  Its first operand is
// the tile again with rows and width exchanged: 16-bit types are turned by the transposing LDS read, fp32 needs one element a lane.
// Everything that belongs to a column (maximum, sum, logarithm, delta, scales) is one register a lane.
//
// The scores of a tile are 16 instructions' issue slots or more a lane against few matrix clocks at widths of 32 and 64, so it is the
// vector instructions that are counted there: the running maximum moves only when a score passes it by 2^8, and the row sums of 16-bit
// types are a product with ones.
#include "query_attention.hpp"

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "mfma.hpp"

namespace dcn {
namespace {

constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / kWave;
constexpr float kInf = __builtin_inff(), kLog2e = 1.44269504088896340736f;
constexpr int kHiddenColumn = -2;      // the segment of a column or query row that sees nothing; -1 is a padded key's

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Rounding of P and dX to fp16 next to its subnormals would cost what bf16 and fp32 never lose: exponents are moved up, and
// back in the results.  Forward: weights against a maximum that is up to 2^8 behind stay below 2^12.
template <typename Tag> constexpr float kForwardShift = Tag::kCode == F16::kCode ? 4.f : 0.f;
// Backward: weights of at most 1; a row of a million keys still has normal ones.
template <typename Tag> constexpr float kBackwardShift = Tag::kCode == F16::kCode ? 12.f : 0.f;

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// A value that is the same in all lanes, in a scalar register.
__device__ __forceinline__ float wave_uniform(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); }
// Over the four lanes that share a column.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// What goes into a kernel's scores: a cap, distances or a factor that is not positive; the products alone; a cap above kQuickCap, in 16-bit types.
enum ScoreKind { kAnyScores, kPlainScores, kHighCap };
// A kernel's shape.  KIND: a ScoreKind; W: the width, zeros behind the tensors' own; RT: rows of a tile; RW: waves that share the columns and divide
// a tile's rows, the others divide the columns; CF: sixteens of columns a wave; WAVES: of a workgroup.
template <typename Tag_, int KIND_, int W_, int RT_, int RW_, int CF_, int WAVES_>
struct Shape {
  typedef Tag_ Tag;
  static constexpr int kKind = KIND_;
  static constexpr bool kPlain = KIND_ == kPlainScores;
  static constexpr int W = W_, RT = RT_, RW = RW_, CF = CF_, kWaves = WAVES_, kThreads = kWaves * kWave;
  static constexpr int kSlices = W * Tag::kBytes / 64, kWidthBlocks = W / 16;
  static constexpr int kColumnWaves = kWaves / RW, kColumns = 16 * CF * kColumnWaves;
  static constexpr int kRowBlocks = RT / RW / 16;                // of a wave in a tile, to work on
  static constexpr int kCarried = RT / 16 / kWaves;              // and to bring into LDS
  static constexpr int kTensorBytes = RT * W * Tag::kBytes;
  // two tensors, then by row: segment, poison, position (2), logarithm, delta
  static constexpr int kSegments = 2 * kTensorBytes, kPoison = kSegments + RT * 4, kPoints = kPoison + RT * 4, kLse = kPoints + RT * 8,
                       kDelta = kLse + RT * 4, kTileBytes = kDelta + RT * 4;
  // sums of the waves that divide the rows: of the results, and four values a column
  static constexpr int kMergeStats = kWaves * 16 * CF * (W + 4) * 4, kMergeBytes = RW > 1 ? kMergeStats + kWaves * 16 * CF * 16 : 0;
  // two waves a SIMD at least, which also keeps the matrix instructions' results out of the accumulation registers and their copies;
  // the largest tiles leave room for one
  static constexpr int kWavesPerSimd = W * Tag::kBytes > 256 ? 1 : 2;
  // narrow heads by 64 columns: three where that costs next to no scratch memory.  32 channels, bf16: forward of 32 heads, 2500 queries 92 -> 83
  // us, with distances 122 -> 112; dK and dV of bf16 96 -> 87 (fp16, with its scales a column, or distances: spills, 32 -> 40).  What is kept
  // in scratch memory: 20 to 44 bytes a lane there, 36 in the 16-bit forward of 128 channels by 128 columns with caps or distances, 12 to 36 in
  // fp16's dK and dV of 64 channels by 128 columns with them and by 32
  static constexpr bool kNarrow = W * Tag::kBytes <= 64 && RW == 2;
  static constexpr int kForwardWaves = kNarrow ? 3 : kWavesPerSimd, kGradKvWaves = kNarrow && kPlain && Tag::kCode == BF16::kCode ? 3 : kWavesPerSimd;
  static constexpr int kLdsBytes = std::max(2 * kTileBytes, kMergeBytes);
  static_assert(kRowBlocks % 2 == 0 && kCarried * kWaves * 16 == RT && kLdsBytes <= 156 * 1024);
};

// ---------------------------------------------------------------- a tile's way into LDS
// Rows in slices of 64 bytes, 16 to a block of 1 KB, a row's vectors at vector ^ (row / 4 & 3) (fragment_offset): both the fragment
// reads and the transposing ones then spread over the banks.  A wave carries sixteens of rows, four lanes a row.
__device__ __forceinline__ int turned_by(int r4) { return -r4 & 3; }      // of rows 4 r4 .. + 3 of sixteen
__device__ __forceinline__ uint32_t fragment_at(int r16, int kb) { return (uint32_t)(r16 * 64 + (kb ^ turned_by(r16 >> 2)) * 16); }

struct HeadRows {
  const char *base;
  long long pitch;      // bytes
};
template <typename Tag>
__device__ __forceinline__ HeadRows head_rows(const AttnRows &t, int b, int head) {
  return {static_cast<const char *>(t.base) + (b * t.batch + head * t.head) * (long long)Tag::kBytes, t.token * (long long)Tag::kBytes};
}

template <typename S>
struct TileLoads {
  u32x4 v[S::kCarried][S::kSlices];

  __device__ __forceinline__ void request(const HeadRows &t, int row0, int rows, int width_bytes, int wave, int lane) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(t.base + row0 * t.pitch, 0x7fffffffu);
    const int vec = (lane & 3) ^ turned_by(lane >> 4);
#pragma unroll
    for (int u = 0; u < S::kCarried; ++u) {
      const int row = (wave + S::kWaves * u) * 16 + lane / 4;
      const uint32_t at = (uint32_t)row * (uint32_t)t.pitch + (uint32_t)vec * 16;
#pragma unroll
      for (int s = 0; s < S::kSlices; ++s)
        v[u][s] = buffer_load<16>(r, row0 + row < rows && s * 64 + vec * 16 < width_bytes ? at + s * 64 : kDropOffset);
    }
  }
  __device__ __forceinline__ void put(char *tensor, int wave, int lane) const {
#pragma unroll
    for (int u = 0; u < S::kCarried; ++u)
#pragma unroll
      for (int s = 0; s < S::kSlices; ++s)
        *reinterpret_cast<u32x4 *>(tensor + s * S::RT * 64 + (wave + S::kWaves * u) * 1024 + lane * 16) = v[u][s];
  }
  // Clears vectors that hold an infinity or NaN; whether the lane's row u had one.
  __device__ __forceinline__ bool clear_bad(int u) {
    constexpr uint32_t top = S::Tag::kCode == F32::kCode ? 0x7f800000u : S::Tag::kCode == F16::kCode ? 0x7c00u : 0x7f80u;
    bool row = false;
#pragma unroll
    for (int s = 0; s < S::kSlices; ++s) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bad = bad || (v[u][s][i] & top) == top;
        if constexpr (S::Tag::kBytes == 2) bad = bad || (v[u][s][i] & top << 16) == top << 16;
      }
      if (bad) v[u][s] = u32x4{0, 0, 0, 0};
      row = row || bad;
    }
    return row;
  }
};
// A row that holds an infinity or NaN, in a tile of which some columns do not see all: zeros in the products (0 times either would
// reach every column), and this added to its scores, so that the columns that do see it get NaN.
template <typename S>
__device__ __forceinline__ void put_poison(char *tile, int u, bool bad, int wave, int lane) {
  const uint64_t all = __ballot(bad);
  if ((lane & 3) == 0)
    reinterpret_cast<float *>(tile + S::kPoison)[(wave + S::kWaves * u) * 16 + lane / 4] = (all >> lane & 15) != 0 ? __builtin_nanf("") : 0.f;
}

template <typename S>
__device__ __forceinline__ u32x4 fragment(const char *tensor, int block, int slice, int lane) {
  return *reinterpret_cast<const u32x4 *>(tensor + slice * S::RT * 64 + block * 1024 + fragment_at(lane & 15, lane >> 4));
}
// Weights of 32 rows as the second operand of a product; 16-bit types round them, rest() is what that took.
template <typename S>
struct Weights {
  typedef typename S::Tag Tag;
  static constexpr bool kHalf = Tag::kBytes == 2;
  u32x4 half[kHalf ? S::CF : 1];
  f32x4 full[kHalf ? 1 : 2][kHalf ? 1 : S::CF];
  __device__ __forceinline__ explicit Weights(const f32x4 (&p)[2][S::CF]) {
#pragma unroll
    for (int f = 0; f < S::CF; ++f) {
      if constexpr (kHalf) {
        const float v[8] = {p[0][f].x, p[0][f].y, p[0][f].z, p[0][f].w, p[1][f].x, p[1][f].y, p[1][f].z, p[1][f].w};
        half[f] = Pack<Tag, 8>::encode(v);
      } else {
        full[0][f] = p[0][f];
        full[1][f] = p[1][f];
      }
    }
  }
  __device__ __forceinline__ Weights rest(const f32x4 (&p)[2][S::CF]) const {
    f32x4 left[2][S::CF];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int f = 0; f < S::CF; ++f)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const uint32_t pair = half[f][h * 2 + r / 2];
          left[h][f][r] = -plus_half<Tag, 0>(pair, -p[h][f][r]);
          left[h][f][r + 1] = -plus_half<Tag, 1>(pair, -p[h][f][r + 1]);
        }
    return Weights(left);
  }
};
// Rows 16 block .. + 31 of a tensor with rows and width exchanged, sixteens d of the width: a lane's first operand.
template <typename S>
struct Turned {
  static constexpr bool kHalf = S::Tag::kBytes == 2;
  u32x4 half;
  float full[kHalf ? 1 : 2][4];
  __device__ __forceinline__ void read(const char *tensor, int block, int d, int lane) {
    const int g = lane >> 4, c = lane & 15;
    if constexpr (kHalf) {
      const char *at = tensor + d / 2 * S::RT * 64 + block * 1024 + (4 * g + (c >> 2)) * 64 + (((d & 1) * 2 + ((c & 3) >> 1)) ^ turned_by(g)) * 16 + (c & 1) * 8;
      typedef __attribute__((address_space(3))) s16x4 lds_words;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_words *)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_words *)(at + 1024));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
      half = u32x4{a.x, a.y, b.x, b.y};
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char *at = tensor + d * S::RT * 64 + (block + h) * 1024 + 4 * g * 64 + ((c >> 2) ^ turned_by(g)) * 16 + (c & 3) * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) full[h][r] = *reinterpret_cast<const float *>(at + r * 64);
      }
    }
  }
};
// acc[d][f] += those rows times the weights, and where SETS is 2 times more weights
template <typename S, int SETS = 1>
__device__ __forceinline__ void add_product(f32x4 (&acc)[S::kWidthBlocks][S::CF], const char *tensor, int block, const Weights<S> &w, const Weights<S> &more, int lane) {
  typedef typename S::Tag Tag;
  Turned<S> t[2];
  t[0].read(tensor, block, 0, lane);
#pragma unroll
  for (int d = 0; d < S::kWidthBlocks; ++d) {
    if (d + 1 < S::kWidthBlocks) {
      t[(d + 1) & 1].read(tensor, block, d + 1, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (Tag::kBytes == 2) {
#pragma unroll
      for (int f = 0; f < S::CF; ++f) {
        acc[d][f] = mfma_64_bytes<Tag>(t[d & 1].half, w.half[f], acc[d][f]);
        if constexpr (SETS == 2) acc[d][f] = mfma_64_bytes<Tag>(t[d & 1].half, more.half[f], acc[d][f]);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int f = 0; f < S::CF; ++f) acc[d][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(t[d & 1].full[h][r], w.full[h][f][r], acc[d][f], 0, 0, 0);
    }
  }
}
template <typename S>
__device__ __forceinline__ void add_product(f32x4 (&acc)[S::kWidthBlocks][S::CF], const char *tensor, int block, const f32x4 (&p)[2][S::CF], int lane) {
  const Weights<S> w(p);
  add_product<S>(acc, tensor, block, w, w, lane);
}

// A column's operand, straight from memory: the second operand of the score products.
template <typename S>
__device__ __forceinline__ void load_columns(u32x4 (&to)[S::CF][S::kSlices], const HeadRows &t, int column0, int columns, int width_bytes, int lane) {
  const __amdgpu_buffer_rsrc_t r = make_rsrc(t.base + column0 * t.pitch, 0x7fffffffu);
  const int kb = lane >> 4;
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    const int column = 16 * f + (lane & 15);
#pragma unroll
    for (int s = 0; s < S::kSlices; ++s)
      to[f][s] = buffer_load<16>(r, column0 + column < columns && s * 64 + kb * 16 < width_bytes ? (uint32_t)column * (uint32_t)t.pitch + s * 64 + kb * 16 : kDropOffset);
  }
}
template <typename Tag>
__device__ __forceinline__ float dot_16_bytes(u32x4 a, u32x4 b, float sum) {
  constexpr int N = 16 / Tag::kBytes;
  float x[N], y[N];
  Pack<Tag, N>::decode(a, x);
  Pack<Tag, N>::decode(b, y);
#pragma unroll
  for (int i = 0; i < N; ++i) sum = fmaf(x[i], y[i], sum);
  return sum;
}

// Products of 32 rows of two tensors of a tile with the columns' operands, on top of what is in s and t.  Fragments are read two slices
// ahead of their products.
template <typename S>
__device__ __forceinline__ void two_products(const char *first, const char *second, int block, const u32x4 (&x)[S::CF][S::kSlices], const u32x4 (&y)[S::CF][S::kSlices],
                                             f32x4 (&s)[2][S::CF], f32x4 (&t)[2][S::CF], int lane) {
  typedef typename S::Tag Tag;
  constexpr int kStep = S::kSlices > 1 ? 2 : 1, kSteps = 2 * S::kSlices / kStep;
  u32x4 a[2][kStep], b[2][kStep];
  auto read = [&](int k) {
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      const int at = k * kStep + i;
      a[k & 1][i] = fragment<S>(first, block + at / S::kSlices, at % S::kSlices, lane);
      b[k & 1][i] = fragment<S>(second, block + at / S::kSlices, at % S::kSlices, lane);
    }
  };
  read(0);
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    if (k + 1 < kSteps) {
      read(k + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      const int h = (k * kStep + i) / S::kSlices, sl = (k * kStep + i) % S::kSlices;
#pragma unroll
      for (int f = 0; f < S::CF; ++f) {
        s[h][f] = mfma_64_bytes<Tag>(a[k & 1][i], x[f][sl], s[h][f]);
        t[h][f] = mfma_64_bytes<Tag>(b[k & 1][i], y[f][sl], t[h][f]);
      }
    }
  }
}

// ---------------------------------------------------------------- scores
// 16-bit types form cap tanh(x / cap) as cap - 2 cap / (exp(2 x / cap) + 1), four instructions whose error is that of numbers of the cap's size:
// at most 2^-20 cap (a last bit of exponential and reciprocal each, the sum's half), which the weights show.  At 256 that is half a rounding
// of fp16's weights; higher caps take a form that is exact for small x / cap, in kernels of their own: as a branch of the others it cost every
// call with a cap 2 %.
constexpr float kQuickCap = 256.f;
// To a relative 2^-21: a series whose next term is 3e-7 at 1/4, and beyond it (1 - e) / (1 + e) with e = exp(-2 |x|), which loses no digits there.
// fp32 results see the last bits, which tanhf has; it takes more registers.
template <typename Tag>
__device__ __forceinline__ float exact_tanh(float x) {
  if constexpr (Tag::kBytes == 4) return tanhf(x);
  const float e = __builtin_amdgcn_exp2f(fabsf(x) * (-2.f * kLog2e)), z = x * x;
  const float near = fmaf(fmaf(fmaf(z, -17.f / 315.f, 2.f / 15.f), z, -1.f / 3.f), z * x, x);
  return fabsf(x) < 0.25f ? near : copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
}
// Scores go into exp2, so they are in units of its exponent.  Without cap and distance that is one factor, which rides along where
// the maximum is taken off.
template <int KIND>
struct Scores {
  float tanh_scale, factor, slope;
  static constexpr bool high = KIND == kHighCap;
  bool bent, apart, scaled;      // there is a cap; a distance; neither, but a factor that cannot ride along
  __device__ __forceinline__ Scores(const AttnLaunch &p, int head) : bent(high || p.cap > 0.f), apart(p.slopes != nullptr) {
    tanh_scale = bent ? p.scale / p.cap : 0.f;
    factor = (bent ? p.cap : p.scale) * kLog2e;
    slope = apart ? p.slopes[head] * kLog2e : 0.f;
    scaled = !bent;
  }
};
// Nothing but a positive factor: the products stand for the scores, in the order of their size.  Kernels of their own, which have
// registers for more waves.
template <>
struct Scores<kPlainScores> {
  float factor;
  static constexpr float tanh_scale = 0.f, slope = 0.f;
  static constexpr bool bent = false, high = false, apart = false, scaled = false;
  __device__ __forceinline__ Scores(const AttnLaunch &p, int) : factor(p.scale * kLog2e) {}
};
// tanh(x) = 1 - 2 r with r = 1 / (exp(2 x) + 1), whose derivative is 4 (r - r^2): 16-bit types carry r - r^2 and the factor at the end.
template <typename Tag> constexpr float kBendFactor = Tag::kBytes == 4 ? 1.f : 4.f;
__device__ __forceinline__ float distance(f32x2 a, f32x2 b) {
  const float x = a.x - b.x, y = a.y - b.y;
  return __builtin_amdgcn_sqrtf(fmaf(x, x, y * y));
}

// Scores of N blocks of 16 rows, from the products in s.  What a call has is the same for all lanes: a loop for each, not a question
// for each score.  Forward; where `by_slope` says so the scores are left in units of the slope, `ratio` being the product's factor in them.
// Positions are subtracted as they come, which is exact for near points, and in the backward too.
template <typename Tag, int KIND, int N, int CF, typename Points>
__device__ __forceinline__ void finish_scores(const Scores<KIND> &scores, bool by_slope, float ratio, f32x4 (&s)[N][CF], const f32x2 (&point)[CF], Points point_of) {
  if (scores.bent) {
    const float rate = scores.tanh_scale * (2.f * kLog2e), twice = -2.f * scores.factor;
    if constexpr (Tag::kBytes == 4 || Scores<KIND>::high) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int f = 0; f < CF; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[n][f][r] = exact_tanh<Tag>(s[n][f][r] * scores.tanh_scale) * scores.factor;
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int f = 0; f < CF; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[n][f][r] = fmaf(twice, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[n][f][r] * rate) + 1.f), scores.factor);
    }
  }
  if (by_slope) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x2 there = point_of(n, r);
#pragma unroll
        for (int f = 0; f < CF; ++f) s[n][f][r] = fmaf(s[n][f][r], ratio, -distance(point[f], there));
      }
    return;
  }
  if (scores.scaled)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int f = 0; f < CF; ++f) s[n][f] *= scores.factor;
  if (scores.apart)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x2 there = point_of(n, r);
#pragma unroll
        for (int f = 0; f < CF; ++f) s[n][f][r] = fmaf(-scores.slope, distance(point[f], there), s[n][f][r]);
      }
}
// Backward: weights of 32 rows without what is not seen, from the products in s and the rows' or columns' logarithms; the distances,
// and the tanh's derivative over kBendFactor.  seen(): masks s in place, before the exponential.
template <typename Tag, int KIND, int CF, typename Points, typename Lse, typename Seen>
__device__ __forceinline__ void form_weights(const Scores<KIND> &scores, f32x4 (&s)[2][CF], f32x4 (&far)[2][CF], f32x4 (&bend)[2][CF], const f32x2 (&point)[CF],
                                             Points point_of, Lse lse, Seen seen) {
  if constexpr (KIND == kPlainScores) {
    seen();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int f = 0; f < CF; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[h][f][r] = __builtin_amdgcn_exp2f(fmaf(s[h][f][r], scores.factor, -lse(h, r, f)));
    return;
  }
  if (scores.bent) {
    const float rate = scores.tanh_scale * (2.f * kLog2e), twice = -2.f * scores.factor;
    if constexpr (Tag::kBytes == 4 || Scores<KIND>::high) {
      constexpr float bend0 = 1.f / kBendFactor<Tag>;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < CF; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float t = exact_tanh<Tag>(s[h][f][r] * scores.tanh_scale);
            bend[h][f][r] = fmaf(t * -bend0, t, bend0);
            s[h][f][r] = fmaf(t, scores.factor, -lse(h, r, f));
          }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < CF; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float t = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[h][f][r] * rate) + 1.f);
            bend[h][f][r] = fmaf(-t, t, t);
            s[h][f][r] = fmaf(twice, t, scores.factor - lse(h, r, f));
          }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int f = 0; f < CF; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[h][f][r] = fmaf(s[h][f][r], scores.factor, -lse(h, r, f));
  }
  if (scores.apart)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x2 there = point_of(h, r);
#pragma unroll
        for (int f = 0; f < CF; ++f) {
          far[h][f][r] = distance(point[f], there);
          s[h][f][r] = fmaf(-scores.slope, far[h][f][r], s[h][f][r]);
        }
      }
  seen();
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int f = 0; f < CF; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[h][f][r] = __builtin_amdgcn_exp2f(s[h][f][r]);
}

// ---------------------------------------------------------------- which tiles
// What the segment numbers of a workgroup's columns leave of a tile: whether any pair sees each other and whether all do.
struct ColumnRange {
  int lo, hi;              // of the numbers that count
  bool shared, hidden;     // a key column of segment 0; a column that sees or shows nothing
};
template <bool KEYS>
__device__ __forceinline__ ColumnRange column_range(const int *segments, int column0, int columns, int count, int lane) {
  ColumnRange r = {0x7fffffff, -1, false, false};
  bool shared = false, hidden = false;
  for (int i = lane; i < count; i += kWave)
    if (column0 + i < columns) {
      const int v = segments != nullptr ? segments[column0 + i] : 0;
      if (v < 0) hidden = true;
      else if (KEYS && v == 0) shared = true;
      else { r.lo = min(r.lo, v); r.hi = max(r.hi, v); }
    }
  for (int o = 32; o > 0; o >>= 1) {
    r.lo = min(r.lo, __shfl_xor(r.lo, o, kWave));
    r.hi = max(r.hi, __shfl_xor(r.hi, o, kWave));
  }
  r.shared = __ballot(shared) != 0;
  r.hidden = __ballot(hidden) != 0;
  return r;
}
// By a row's number: whether some column sees it (shows itself to it), and whether all do.
template <bool KEYS>
__device__ __forceinline__ bool some_pair(const ColumnRange &c, int row) {
  const bool within = row >= c.lo && row <= c.hi;
  return KEYS ? row >= 0 && (c.shared || within) : c.hi >= 0 && (row == 0 || within);
}
template <bool KEYS>
__device__ __forceinline__ bool every_pair(const ColumnRange &c, int row) {
  if (c.hidden) return false;
  return KEYS ? row >= 0 && (c.hi < 0 || (c.lo == row && c.hi == row)) : row == 0 || (c.lo == row && c.hi == row);
}

struct TileMasks {
  uint64_t some, every;      // bit t: tile t of up to 64
};
// Rows first .. last - 1; all waves together.  flags: 64 bytes of LDS, free again behind the next barrier.
template <int RT, int WAVES, bool KEYS>
__device__ __forceinline__ TileMasks tile_masks(const int *row_segments, bool masked, const ColumnRange &c, int first, int last, char *flags, int wave, int lane) {
  const int tiles = min(64, (last - first + RT - 1) / RT);
  if (!masked) {
    TileMasks m;
    m.some = tiles == 64 ? ~0ull : (1ull << tiles) - 1;
    m.every = first + tiles * RT <= last ? m.some : m.some >> 1;
    return m;
  }
  // a wave's tiles all at once: their loads are one wait
  constexpr int kMine = 64 / WAVES, kParts = RT / 64;
  int v[kMine][kParts];
#pragma unroll
  for (int i = 0; i < kMine; ++i)
#pragma unroll
    for (int u = 0; u < kParts; ++u) {
      const int row = first + (wave + i * WAVES) * RT + u * 64 + lane;
      v[i][u] = row < last ? (row_segments != nullptr ? row_segments[row] : 0) : kHiddenColumn;
    }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int t = wave + i * WAVES;
    if (t >= tiles) break;
    bool some = false, every = true;
#pragma unroll
    for (int u = 0; u < kParts; ++u) {
      some = some || some_pair<KEYS>(c, v[i][u]);
      every = every && first + t * RT + u * 64 + lane < last && every_pair<KEYS>(c, v[i][u]);
    }
    const uint64_t has = __ballot(some), all = __ballot(every);
    if (lane == 0) flags[t] = (char)((has != 0) | (all == ~0ull) << 1);
  }
  __syncthreads();
  const int mine = lane < tiles ? flags[lane] : 0;
  return {__ballot(mine & 1), __ballot(mine & 2)};
}

// What a thread carries of a row beside the tensors.
struct RowLoads {
  int segment;
  f32x2 point;
  float lse, delta;
};

// Walks the tiles: request(row0) starts the loads of a tile, put(tile, every) brings what came into LDS, work(tile, every) computes.
// A tile's loads are under way while the one before is worked on (two ahead gained nothing); two tiles of LDS in turn, one barrier a tile.
template <typename S, bool KEYS, typename Request, typename Put, typename Work>
__device__ __forceinline__ void walk_tiles(const int *row_segments, bool masked, const ColumnRange &c, int first, int last, char *lds, char *flags, int wave,
                                           int lane, Request request, Put put, Work work) {
  for (int window = first; window < last; window += 64 * S::RT) {
    TileMasks m = tile_masks<S::RT, S::kWaves, KEYS>(row_segments, masked, c, window, last, flags, wave, lane);
    if (m.some != 0) {
      bool every = false;
      auto next = [&] {
        const int t = __builtin_ctzll(m.some);
        m.some &= m.some - 1;
        every = m.every >> t & 1;
        request(window + t * S::RT);
      };
      next();
      for (int turn = 0;; turn ^= 1) {
        char *tile = lds + turn * S::kTileBytes;
        const bool whole = every, more = m.some != 0;
        put(tile, whole);
        __syncthreads();
        if (more) next();
        work(tile, whole);
        if (!more) break;
      }
    }
    __syncthreads();
  }
}

// Where a workgroup stands: [batch][head][column tile][chunk], neighbours on one XCD.
struct Place {
  int b, head, tile, chunk;
  __device__ __forceinline__ Place(int heads, int tiles, int chunks) {
    int id = (int)xcd_contiguous_block(blockIdx.x, gridDim.x);
    chunk = id % chunks; id /= chunks;
    tile = id % tiles; id /= tiles;
    head = id % heads;
    b = id / heads;
  }
};

// Sums of a column tile over the waves that divided the rows, through LDS: acc of wave (RW index) 0 .. RW - 1 times its factor.
// Afterwards wave w holds the sums of the width blocks w, w + RW, ... and `mine` says so.
template <typename S>
__device__ __forceinline__ void merge_rows(f32x4 (&acc)[S::kWidthBlocks][S::CF], char *lds, int row_wave, int column_wave, int lane) {
  if constexpr (S::RW > 1) {
    constexpr int pitch = S::W + 4;
    float *s = reinterpret_cast<float *>(lds);
    const int g = lane >> 4, c = lane & 15;
    __syncthreads();
#pragma unroll
    for (int f = 0; f < S::CF; ++f)
#pragma unroll
      for (int d = 0; d < S::kWidthBlocks; ++d)
        *reinterpret_cast<f32x4 *>(s + (size_t)(((row_wave * S::kColumnWaves + column_wave) * S::CF + f) * 16 + c) * pitch + d * 16 + g * 4) = acc[d][f];
    __syncthreads();
#pragma unroll
    for (int f = 0; f < S::CF; ++f)
#pragma unroll
      for (int d = 0; d < S::kWidthBlocks; ++d) {
        if (d % S::RW != row_wave) continue;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < S::RW; ++w)
          sum += *reinterpret_cast<const f32x4 *>(s + (size_t)(((w * S::kColumnWaves + column_wave) * S::CF + f) * 16 + c) * pitch + d * 16 + g * 4);
        acc[d][f] = sum;
      }
  }
}
template <typename S>
__device__ __forceinline__ bool holds(int width_block, int row_wave) { return S::RW == 1 || width_block % S::RW == row_wave; }

template <typename Tag>
__device__ __forceinline__ void store4(void *base, size_t element, f32x4 v) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  reinterpret_cast<typename RawWord<4 * Tag::kBytes>::type *>(base)[element / 4] = Pack<Tag, 4>::encode(f);
}
// What rounding took from v, in the type.
template <typename Tag>
__device__ __forceinline__ f32x4 rounded_off(f32x4 v) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  float r[4];
  Pack<Tag, 4>::decode(Pack<Tag, 4>::encode(f), r);
  return f32x4{f[0] - r[0], f[1] - r[1], f[2] - r[2], f[3] - r[3]};
}

// ---------------------------------------------------------------- forward
struct Split {
  int tiles, chunks, chunk_rows;      // column tiles of a head; parts of the rows, a whole number of tiles each
  float *part, *stats;                // [chunk][batch][query][head][width], [..][2]: unnormalised sums; maximum and sum
};

// What the backward forms a row's weights from again: infinite, so zeros, where it sees nothing.  A weight is then off by half a last bit of the
// logarithm and of its score: 1e-4 of it for scores of 1000 (in units of exp2), some hundredths at 2^20.  Beyond that what comes out has lost its
// size, of a single key's weight too (2^8 for one at 1e8): no number rather than a wrong one.
template <typename Tag>
__device__ __forceinline__ float row_logarithm(float top, float sum) {
  if (sum == 0.f) return kInf;
  return fabsf(top) > 0x1p20f ? __builtin_nanf("") : top - kForwardShift<Tag> + __builtin_amdgcn_logf(sum);
}

// TRAIN: a backward follows (16-bit types; fp32 ones have nothing to round).
template <typename S, bool TRAIN>
__global__ void __launch_bounds__(S::kThreads, S::kForwardWaves) attn_forward_kernel(const AttnLaunch p, const Split split) {
  typedef typename S::Tag Tag;
  extern __shared__ __align__(16) char lds[];
  __shared__ char s_flags[64];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, g = lane >> 4, c = lane & 15;
  const int row_wave = wave / S::kColumnWaves, column_wave = wave % S::kColumnWaves;
  const Place at(p.heads, split.tiles, split.chunks);
  const int kv = at.head / (p.heads / p.kv_heads), width_bytes = p.width * Tag::kBytes;
  const int column0 = at.tile * S::kColumns, mine0 = column0 + column_wave * 16 * S::CF;
  const int first = at.chunk * split.chunk_rows, last = min(p.nk, first + split.chunk_rows);
  const HeadRows keys = head_rows<Tag>(p.k, at.b, kv), values = head_rows<Tag>(p.v, at.b, kv);
  const Scores<S::kKind> scores(p, at.head);
  const bool masked = p.k_segments != nullptr;
  // without a cap the product's factor and the distance are one operation in units of a positive slope, which rides along where the
  // maximum is taken off; a slope within 2^20 of the factor, so that no score leaves the range of fp32 in its units.  (The ratio in a scalar
  // register leaves others a vector register: 2 x 7744 queries of 8 heads of 64, bf16, with a cap and distances 873 us, 856 so; the slope in
  // one as well, 5 % longer.)
  const float ratio = wave_uniform(scores.apart ? scores.factor / scores.slope : 0.f);
  const bool by_slope = scores.apart && !scores.bent && scores.slope > 0.f && fabsf(ratio) >= 0x1p-20f && fabsf(ratio) <= 0x1p20f;
  const float factor = S::kPlain ? scores.factor : (by_slope ? scores.slope : 1.f);

  u32x4 q[S::CF][S::kSlices];
  load_columns<S>(q, head_rows<Tag>(p.q, at.b, at.head), mine0, p.nq, width_bytes, lane);
  const int *q_segments = p.q_segments != nullptr ? p.q_segments + (long long)at.b * p.nq : nullptr;
  const int *k_segments = masked ? p.k_segments + (long long)at.b * p.nk : nullptr;
  int segment[S::CF];
  f32x2 point[S::CF];
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    const int i = mine0 + 16 * f + c;
    segment[f] = i < p.nq ? (q_segments != nullptr ? q_segments[i] : 0) : kHiddenColumn;
    if (segment[f] < 0) segment[f] = kHiddenColumn;
    point[f] = f32x2{0.f, 0.f};
    // (columns behind the last query stand where it stands: when a wave's maxima move does not depend on the points' origin)
    if (scores.apart) point[f] = reinterpret_cast<const f32x2 *>(p.q_points)[(long long)at.b * p.nq + min(i, p.nq - 1)];
  }
  const ColumnRange range = masked ? column_range<false>(q_segments, column0, p.nq, S::kColumns, lane) : ColumnRange{};

  // total: sums of the weights as the product takes them.  In 16-bit types that is rounded; where a backward follows, what rounding took
  // goes through the products as well: delta, and the logarithm from which the weights are formed again, then belong to the weights
  // themselves (with delta of rounded ones dQ was off by 1.5 of its own roundings, with those of 1.4).  Without a backward the rounding stays:
  // results are off by 2.6e-4 to 2.8e-4 in fp16 and 2.2e-3 in bf16, root mean square, where one rounding of the result alone is 2.1e-4 and
  // 1.7e-3, and the rests would cost half as much again (2 x 4096 tokens, 8 heads of 64, bf16: 100 us, with them 145).
  f32x4 acc[S::kWidthBlocks][S::CF], total[S::CF];
  float top[S::CF];
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    top[f] = -kInf;
    total[f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < S::kWidthBlocks; ++d) acc[d][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  TileLoads<S> next_k, next_v;
  RowLoads next = {};
  auto request = [&](int row0) {
    next_k.request(keys, row0, last, width_bytes, wave, lane);
    next_v.request(values, row0, last, width_bytes, wave, lane);
    const int row = row0 + (int)threadIdx.x;
    if ((int)threadIdx.x < S::RT) {
      next.segment = row < last ? (masked ? k_segments[row] : 0) : -1;
      if (scores.apart) next.point = row < last ? reinterpret_cast<const f32x2 *>(p.k_points)[(long long)at.b * p.nk + row] : f32x2{0.f, 0.f};
    }
  };
  auto put = [&](char *tile, bool every) {
    if (!every)
#pragma unroll
      for (int u = 0; u < S::kCarried; ++u) put_poison<S>(tile, u, next_v.clear_bad(u), wave, lane);
    next_k.put(tile, wave, lane);
    next_v.put(tile + S::kTensorBytes, wave, lane);
    if ((int)threadIdx.x < S::RT) {
      reinterpret_cast<int *>(tile + S::kSegments)[threadIdx.x] = next.segment;
      if (scores.apart) reinterpret_cast<f32x2 *>(tile + S::kPoints)[threadIdx.x] = next.point;
    }
  };
  auto work = [&](const char *tile, bool every) {
    const int block0 = row_wave * S::kRowBlocks;
    // a block's fragments are read while the one before is multiplied; said so, for the compiler reads each where it is used and waits
    f32x4 s[S::kRowBlocks][S::CF];
    u32x4 a[2][S::kSlices];
#pragma unroll
    for (int sl = 0; sl < S::kSlices; ++sl) a[0][sl] = fragment<S>(tile, block0, sl, lane);
#pragma unroll
    for (int n = 0; n < S::kRowBlocks; ++n) {
      if (n + 1 < S::kRowBlocks) {
#pragma unroll
        for (int sl = 0; sl < S::kSlices; ++sl) a[(n + 1) & 1][sl] = fragment<S>(tile, block0 + n + 1, sl, lane);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int f = 0; f < S::CF; ++f) s[n][f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int sl = 0; sl < S::kSlices; ++sl)
#pragma unroll
        for (int f = 0; f < S::CF; ++f) s[n][f] = mfma_64_bytes<Tag>(a[n & 1][sl], q[f][sl], s[n][f]);
    }
    const f32x2 *points = reinterpret_cast<const f32x2 *>(tile + S::kPoints) + block0 * 16 + 4 * g;
    finish_scores<Tag, S::kKind, S::kRowBlocks, S::CF>(scores, by_slope, ratio, s, point, [&](int n, int r) { return points[n * 16 + r]; });
    if (!every)
#pragma unroll
      for (int n = 0; n < S::kRowBlocks; ++n) {
        const int *segments = reinterpret_cast<const int *>(tile + S::kSegments) + (block0 + n) * 16 + 4 * g;
        const float *poison = reinterpret_cast<const float *>(tile + S::kPoison) + (block0 + n) * 16 + 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int f = 0; f < S::CF; ++f) s[n][f][r] = segments[r] == 0 || segments[r] == segment[f] ? s[n][f][r] + poison[r] : -kInf;
      }
    // the maximum moves where a score passes it by 2^8
    float high[S::CF];
    bool passed = false;
#pragma unroll
    for (int f = 0; f < S::CF; ++f) {
      high[f] = fmaxf(fmaxf(s[0][f][0], s[0][f][1]), fmaxf(s[0][f][2], s[0][f][3]));
#pragma unroll
      for (int n = 1; n < S::kRowBlocks; ++n) high[f] = max3(max3(high[f], s[n][f][0], s[n][f][1]), s[n][f][2], s[n][f][3]);
      passed = passed || high[f] * factor > top[f] + 8.f;
    }
    if (__ballot(passed) != 0)
#pragma unroll
      for (int f = 0; f < S::CF; ++f) {
        const float now = fmaxf(top[f], column_max(high[f]) * factor);
        const float keep = __builtin_amdgcn_exp2f(top[f] - (now == -kInf ? 0.f : now));
        top[f] = now;
#pragma unroll
        for (int d = 0; d < S::kWidthBlocks; ++d) acc[d][f] *= keep;
        total[f] *= keep;
      }
#pragma unroll
    for (int f = 0; f < S::CF; ++f) {
      const float off = kForwardShift<Tag> - (top[f] == -kInf ? 0.f : top[f]);
#pragma unroll
      for (int n = 0; n < S::kRowBlocks; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[n][f][r] = __builtin_amdgcn_exp2f(fmaf(s[n][f][r], factor, off));
    }
    if constexpr (Tag::kBytes == 4)
#pragma unroll
      for (int f = 0; f < S::CF; ++f)
#pragma unroll
        for (int n = 0; n < S::kRowBlocks; ++n) total[f] += s[n][f];
#pragma unroll
    for (int n = 0; n < S::kRowBlocks; n += 2) {
      f32x4 p32[2][S::CF];
#pragma unroll
      for (int f = 0; f < S::CF; ++f) {
        p32[0][f] = s[n][f];
        p32[1][f] = s[n + 1][f];
      }
      const Weights<S> w(p32);
      auto count = [&](const Weights<S> &v) {
        constexpr uint32_t one = Tag::kCode == F16::kCode ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
        for (int f = 0; f < S::CF; ++f) total[f] = mfma_64_bytes<Tag>(u32x4{one, one, one, one}, v.half[f], total[f]);
      };
      if constexpr (Tag::kBytes == 2) {
        count(w);
      }
      if constexpr (TRAIN) {
        const Weights<S> left = w.rest(p32);
        count(left);
        add_product<S, 2>(acc, tile + S::kTensorBytes, block0 + n, w, left, lane);
      } else {
        add_product<S>(acc, tile + S::kTensorBytes, block0 + n, w, w, lane);
      }
    }
  };
  walk_tiles<S, false>(k_segments, masked, range, first, last, lds, s_flags, wave, lane, request, put, work);

  float sum[S::CF];
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    sum[f] = Tag::kBytes == 4 ? column_sum((total[f].x + total[f].y) + (total[f].z + total[f].w)) : total[f].x;
    if (segment[f] < 0) {      // sees nothing
      sum[f] = 0.f;
      top[f] = -kInf;
#pragma unroll
      for (int d = 0; d < S::kWidthBlocks; ++d) acc[d][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  if constexpr (S::RW > 1) {
    f32x2 *s_stats = reinterpret_cast<f32x2 *>(lds + S::kMergeStats);
    auto slot = [&](int w, int f) { return ((w * S::kColumnWaves + column_wave) * S::CF + f) * 16 + c; };
#pragma unroll
    for (int f = 0; f < S::CF; ++f)
      if (g == 0) s_stats[slot(row_wave, f)] = f32x2{top[f], sum[f]};
    __syncthreads();
#pragma unroll
    for (int f = 0; f < S::CF; ++f) {
      const float was = top[f];
      float now = -kInf;
#pragma unroll
      for (int w = 0; w < S::RW; ++w) now = fmaxf(now, s_stats[slot(w, f)].x);
      const float base = now == -kInf ? 0.f : now;
      sum[f] = 0.f;
#pragma unroll
      for (int w = 0; w < S::RW; ++w) sum[f] = fmaf(s_stats[slot(w, f)].y, __builtin_amdgcn_exp2f(s_stats[slot(w, f)].x - base), sum[f]);
      const float keep = __builtin_amdgcn_exp2f(was - base);
      top[f] = now;
#pragma unroll
      for (int d = 0; d < S::kWidthBlocks; ++d) acc[d][f] *= keep;
    }
    merge_rows<S>(acc, lds, row_wave, column_wave, lane);
  }
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    const int i = mine0 + 16 * f + c;
    if (i >= p.nq) continue;
    const size_t row = ((size_t)at.b * p.nq + i) * p.heads + at.head;
    const bool split_rows = split.chunks > 1;
    const size_t part_row = ((size_t)at.chunk * p.batch * p.nq * p.heads + row);
    const float inv = sum[f] == 0.f ? 0.f : 1.f / sum[f];
#pragma unroll
    for (int d = 0; d < S::kWidthBlocks; ++d) {
      const int column = d * 16 + g * 4;
      if (!holds<S>(d, row_wave) || column >= p.width) continue;
      if (split_rows) {
        *reinterpret_cast<f32x4 *>(split.part + part_row * p.width + column) = acc[d][f];
      } else {
        const f32x4 v = acc[d][f] * inv;
        store4<Tag>(p.out, row * p.width + column, v);
        if (p.out_rest != nullptr) store4<Tag>(p.out_rest, row * p.width + column, rounded_off<Tag>(v));
      }
    }
    if (g != 0 || row_wave != 0) continue;
    if (split_rows) reinterpret_cast<f32x2 *>(split.stats)[part_row] = f32x2{top[f], sum[f]};
    else if (p.lse != nullptr)
      p.lse[((size_t)at.b * p.heads + at.head) * p.nq + i] = row_logarithm<Tag>(top[f], sum[f]);
  }
}

// The chunks of a row: a wave each, a lane four elements of every (64 / lanes)th chunk.  Lanes a row: a power of two.
template <typename Tag>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const AttnLaunch p, const Split split, int lanes) {
  const int lane = threadIdx.x % kWave, teams = kWave / lanes, team = lane / lanes, column = lane % lanes * 4;
  const long long rows = (long long)p.batch * p.nq * p.heads, row = (long long)blockIdx.x * kJoinWaves + threadIdx.x / kWave;
  if (row >= rows) return;
  const f32x2 *stats = reinterpret_cast<const f32x2 *>(split.stats);
  float top = -kInf;
  for (int k = lane; k < split.chunks; k += kWave) top = fmaxf(top, stats[k * rows + row].x);
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
  const float base = top == -kInf ? 0.f : top;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int k = team; k < split.chunks; k += teams) {
    const f32x2 s = stats[k * rows + row];
    const float w = __builtin_amdgcn_exp2f(s.x - base);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (column < p.width) v = *reinterpret_cast<const f32x4 *>(split.part + (k * rows + row) * p.width + column);
    sum = fmaf(w, s.y, sum);
    acc += v * w;
  }
  for (int o = lanes; o < kWave; o <<= 1) {
    sum += __shfl_xor(sum, o, kWave);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o, kWave);
  }
  if (team != 0 || column >= p.width) return;
  acc *= sum == 0.f ? 0.f : 1.f / sum;
  store4<Tag>(p.out, row * p.width + column, acc);
  if (p.out_rest != nullptr) store4<Tag>(p.out_rest, row * p.width + column, rounded_off<Tag>(acc));
  if (p.lse != nullptr && column == 0) {
    const long long head = row % p.heads, i = row / p.heads % p.nq, b = row / p.heads / p.nq;
    p.lse[(b * p.heads + head) * p.nq + i] = row_logarithm<Tag>(top, sum);
  }
}

// ---------------------------------------------------------------- backward
// 16-bit types round the weights and dX for their products: gradients are off by 3.0e-4 in fp16 and 2.4e-3 in bf16, root mean square, one rounding
// of them alone being 2.1e-4 and 1.7e-3.  Rests as in the forward would double three of the products.
// dX in fp16: a column's values are kept in the type's normal range by a power of two of its own, chosen when one first leaves it
// (the largest goes to 2^13), and the sums follow.  Gradients of loss-scaled or averaged losses and weights of thousands of keys
// would round to subnormals otherwise.
template <typename S>
struct ColumnScale {
  static constexpr bool kNeeded = S::Tag::kCode == F16::kCode;
  float by[S::CF];
  __device__ __forceinline__ ColumnScale() {
#pragma unroll
    for (int f = 0; f < S::CF; ++f) by[f] = kNeeded ? 0x1p100f : 1.f;
  }
  __device__ __forceinline__ void apply(f32x4 (&v)[2][S::CF], f32x4 (&acc)[S::kWidthBlocks][S::CF]) {
    if constexpr (kNeeded) {
      float high[S::CF];
      bool passed = false;
#pragma unroll
      for (int f = 0; f < S::CF; ++f) {
        high[f] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) high[f] = max3(max3(high[f], fabsf(v[h][f].x), fabsf(v[h][f].y)), fabsf(v[h][f].z), fabsf(v[h][f].w));
        passed = passed || high[f] * by[f] > 32768.f;
      }
      if (__ballot(passed) != 0)
#pragma unroll
        for (int f = 0; f < S::CF; ++f) {
          const float most = column_max(high[f]);
          if (most * by[f] > 32768.f) {
            const int e = 267 - (int)(__builtin_bit_cast(uint32_t, most) >> 23);
            const float now = __builtin_bit_cast(float, (uint32_t)max(1, min(e, 227)) << 23);
            const float ratio = now / by[f];
            by[f] = now;
#pragma unroll
            for (int d = 0; d < S::kWidthBlocks; ++d) acc[d][f] *= ratio;
          }
        }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < S::CF; ++f) v[h][f] *= by[f];
    }
  }
};

struct BackwardParts {
  float *delta, *slopes;      // (batch, heads, queries); (batch, heads, column tiles)
  int tiles;                  // column tiles of a head
  // Few columns: the rows, and heads that share a key head, are divided among workgroups; parts [chunk][token][head][width] in fp32 are
  // added behind.
  int chunks, chunk_rows, head_parts;
  float *part;
};
// Where a chunk's results go.
template <typename Tag>
__device__ __forceinline__ void store_grad(void *grad, float *part, size_t chunk_rows_before, size_t row, int width, int column, f32x4 v) {
  if (part != nullptr) *reinterpret_cast<f32x4 *>(part + (chunk_rows_before + row) * width + column) = v;
  else if (grad != nullptr) store4<Tag>(grad, row * width + column, v);
}

// dQ, delta and the slopes' parts: columns are queries, rows keys.
template <typename S>
__global__ void __launch_bounds__(S::kThreads, S::kWavesPerSimd) attn_grad_q_kernel(const AttnLaunch p, const BackwardParts parts) {
  typedef typename S::Tag Tag;
  extern __shared__ __align__(16) char lds[];
  __shared__ char s_flags[64];
  __shared__ float s_slopes[S::kWaves];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, g = lane >> 4, c = lane & 15;
  const int row_wave = wave / S::kColumnWaves, column_wave = wave % S::kColumnWaves;
  const Place at(p.heads, parts.tiles, parts.chunks);
  const int kv = at.head / (p.heads / p.kv_heads), width_bytes = p.width * Tag::kBytes;
  const int column0 = at.tile * S::kColumns, mine0 = column0 + column_wave * 16 * S::CF;
  const int first = at.chunk * parts.chunk_rows, last = min(p.nk, first + parts.chunk_rows);
  const HeadRows keys = head_rows<Tag>(p.k, at.b, kv), values = head_rows<Tag>(p.v, at.b, kv);
  const Scores<S::kKind> scores(p, at.head);
  const bool masked = p.k_segments != nullptr;

  u32x4 q[S::CF][S::kSlices], go[S::CF][S::kSlices];
  load_columns<S>(q, head_rows<Tag>(p.q, at.b, at.head), mine0, p.nq, width_bytes, lane);
  load_columns<S>(go, head_rows<Tag>(p.grad_out, at.b, at.head), mine0, p.nq, width_bytes, lane);
  float delta[S::CF];
  {
    const long long token = (long long)p.heads * p.width;
    u32x4 o[S::CF][S::kSlices];
    load_columns<S>(o, head_rows<Tag>(AttnRows{p.out, token * p.nq, token, p.width}, at.b, at.head), mine0, p.nq, width_bytes, lane);
#pragma unroll
    for (int f = 0; f < S::CF; ++f) {
      delta[f] = 0.f;
#pragma unroll
      for (int s = 0; s < S::kSlices; ++s) delta[f] = dot_16_bytes<Tag>(go[f][s], o[f][s], delta[f]);
    }
    if (p.out_rest != nullptr) {
      load_columns<S>(o, head_rows<Tag>(AttnRows{p.out_rest, token * p.nq, token, p.width}, at.b, at.head), mine0, p.nq, width_bytes, lane);
#pragma unroll
      for (int f = 0; f < S::CF; ++f)
#pragma unroll
        for (int s = 0; s < S::kSlices; ++s) delta[f] = dot_16_bytes<Tag>(go[f][s], o[f][s], delta[f]);
    }
  }
  const int *q_segments = p.q_segments != nullptr ? p.q_segments + (long long)at.b * p.nq : nullptr;
  const int *k_segments = masked ? p.k_segments + (long long)at.b * p.nk : nullptr;
  int segment[S::CF];
  f32x2 point[S::CF];
  float lse[S::CF];
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    const int i = mine0 + 16 * f + c;
    const long long stat = ((long long)at.b * p.heads + at.head) * p.nq + i;
    segment[f] = i < p.nq ? (q_segments != nullptr ? q_segments[i] : 0) : kHiddenColumn;
    if (segment[f] < 0) segment[f] = kHiddenColumn;
    point[f] = f32x2{0.f, 0.f};
    if (scores.apart && i < p.nq) point[f] = reinterpret_cast<const f32x2 *>(p.q_points)[(long long)at.b * p.nq + i];
    lse[f] = i < p.nq ? p.lse[stat] : kInf;
    delta[f] = column_sum(delta[f]);
    if (i < p.nq && g == 0 && row_wave == 0 && at.chunk == 0) parts.delta[stat] = delta[f];
  }
  const ColumnRange range = masked ? column_range<false>(q_segments, column0, p.nq, S::kColumns, lane) : ColumnRange{};

  f32x4 acc[S::kWidthBlocks][S::CF];
#pragma unroll
  for (int f = 0; f < S::CF; ++f)
#pragma unroll
    for (int d = 0; d < S::kWidthBlocks; ++d) acc[d][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  ColumnScale<S> up;
  // The slopes' gradient is fp32 and a sum of terms that nearly cancel in each row: delta, which is as exact as the forward's weights
  // were rounded, would show.  A row adds -sum dS distance with dS = w (t - delta), less delta's error sum dS times sum w distance
  // (the weights add up to 1): sums of dS, w distance, dS distance.
  const bool want_slopes = parts.slopes != nullptr;
  float moment[S::CF][3];
  f32x4 minus_delta[S::CF];      // what the product dO V^T starts from
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    moment[f][0] = moment[f][1] = moment[f][2] = 0.f;
    minus_delta[f] = f32x4{-delta[f], -delta[f], -delta[f], -delta[f]};
  }

  TileLoads<S> next_k, next_v;
  RowLoads next = {};
  auto request = [&](int row0) {
    next_k.request(keys, row0, last, width_bytes, wave, lane);
    next_v.request(values, row0, last, width_bytes, wave, lane);
    const int row = row0 + (int)threadIdx.x;
    if ((int)threadIdx.x < S::RT) {
      next.segment = row < last ? (masked ? k_segments[row] : 0) : -1;
      if (scores.apart) next.point = row < last ? reinterpret_cast<const f32x2 *>(p.k_points)[(long long)at.b * p.nk + row] : f32x2{0.f, 0.f};
    }
  };
  auto put = [&](char *tile, bool every) {
    if (!every)
#pragma unroll
      for (int u = 0; u < S::kCarried; ++u) put_poison<S>(tile, u, next_k.clear_bad(u), wave, lane);
    next_k.put(tile, wave, lane);
    next_v.put(tile + S::kTensorBytes, wave, lane);
    if ((int)threadIdx.x < S::RT) {
      reinterpret_cast<int *>(tile + S::kSegments)[threadIdx.x] = next.segment;
      if (scores.apart) reinterpret_cast<f32x2 *>(tile + S::kPoints)[threadIdx.x] = next.point;
    }
  };
  auto work = [&](const char *tile, bool every) {
#pragma unroll 1
    for (int n = 0; n < S::kRowBlocks; n += 2) {
      const int block = row_wave * S::kRowBlocks + n;
      f32x4 s[2][S::CF], t[2][S::CF], far[2][S::CF], bend[2][S::CF];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < S::CF; ++f) {
          s[h][f] = f32x4{0.f, 0.f, 0.f, 0.f};
          t[h][f] = minus_delta[f];
        }
      two_products<S>(tile, tile + S::kTensorBytes, block, q, go, s, t, lane);
      const f32x2 *points = reinterpret_cast<const f32x2 *>(tile + S::kPoints) + block * 16 + 4 * g;
      const int *segments = reinterpret_cast<const int *>(tile + S::kSegments) + block * 16 + 4 * g;
      const float *poison = reinterpret_cast<const float *>(tile + S::kPoison) + block * 16 + 4 * g;
      form_weights<Tag, S::kKind, S::CF>(scores, s, far, bend, point, [&](int h, int r) { return points[h * 16 + r]; }, [&](int, int, int f) { return lse[f]; }, [&] {
        if (every) return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int f = 0; f < S::CF; ++f) {
              const bool seen = segments[h * 16 + r] == 0 || segments[h * 16 + r] == segment[f];
              s[h][f][r] = seen ? s[h][f][r] + poison[h * 16 + r] : -kInf;
              // what else there is of a pair that is not seen may be anything
              t[h][f][r] = seen ? t[h][f][r] : 0.f;
              if (scores.apart) far[h][f][r] = seen ? far[h][f][r] : 0.f;
              if (scores.bent) bend[h][f][r] = seen ? bend[h][f][r] : 0.f;
            }
      });
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < S::CF; ++f) t[h][f] *= s[h][f];
      if (want_slopes)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int f = 0; f < S::CF; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              moment[f][0] += t[h][f][r];
              moment[f][1] = fmaf(s[h][f][r], far[h][f][r], moment[f][1]);
              moment[f][2] = fmaf(t[h][f][r], far[h][f][r], moment[f][2]);
            }
      if (scores.bent)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int f = 0; f < S::CF; ++f) t[h][f] *= bend[h][f];
      up.apply(t, acc);
      add_product<S>(acc, tile, block, t, lane);
    }
  };
  walk_tiles<S, false>(k_segments, masked, range, first, last, lds, s_flags, wave, lane, request, put, work);

#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    const float by = p.scale * (scores.bent ? kBendFactor<Tag> : 1.f) / up.by[f];
    const bool sees = segment[f] >= 0;
#pragma unroll
    for (int d = 0; d < S::kWidthBlocks; ++d) acc[d][f] = sees ? acc[d][f] * by : f32x4{0.f, 0.f, 0.f, 0.f};
    if (!sees) moment[f][0] = moment[f][1] = moment[f][2] = 0.f;
  }
  merge_rows<S>(acc, lds, row_wave, column_wave, lane);
  const size_t rows_before = (size_t)at.chunk * p.batch * p.nq * p.heads;
  if (p.grad_q != nullptr)
#pragma unroll
    for (int f = 0; f < S::CF; ++f) {
      const int i = mine0 + 16 * f + c;
      if (i >= p.nq) continue;
      const size_t row = ((size_t)at.b * p.nq + i) * p.heads + at.head;
#pragma unroll
      for (int d = 0; d < S::kWidthBlocks; ++d)
        if (holds<S>(d, row_wave) && d * 16 + g * 4 < p.width)
          store_grad<Tag>(p.grad_q, parts.part, rows_before, row, p.width, d * 16 + g * 4, acc[d][f]);
    }
  if (want_slopes) {
#pragma unroll
    for (int f = 0; f < S::CF; ++f)
#pragma unroll
      for (int e = 0; e < 3; ++e) moment[f][e] = column_sum(moment[f][e]);
    if constexpr (S::RW > 1) {
      f32x4 *s_stats = reinterpret_cast<f32x4 *>(lds + S::kMergeStats);
      auto slot = [&](int w, int f) { return ((w * S::kColumnWaves + column_wave) * S::CF + f) * 16 + c; };
#pragma unroll
      for (int f = 0; f < S::CF; ++f)
        if (g == 0) s_stats[slot(row_wave, f)] = f32x4{moment[f][0], moment[f][1], moment[f][2], 0.f};
      __syncthreads();
#pragma unroll
      for (int f = 0; f < S::CF; ++f) {
        f32x4 all = s_stats[slot(0, f)];
#pragma unroll
        for (int w = 1; w < S::RW; ++w) all += s_stats[slot(w, f)];
        moment[f][0] = all.x; moment[f][1] = all.y; moment[f][2] = all.z;
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int f = 0; f < S::CF; ++f)
      if (g == 0 && row_wave == 0 && mine0 + 16 * f + c < p.nq) sum -= moment[f][2] - moment[f][0] * moment[f][1];
    sum = cluster_sum(sum, kWave);
    if (lane == 0) s_slopes[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      sum = s_slopes[0];
#pragma unroll
      for (int w = 1; w < S::kWaves; ++w) sum += s_slopes[w];
      parts.slopes[((size_t)at.b * p.heads + at.head) * parts.tiles + at.tile] = sum;
    }
  }
}

// dK and dV: columns are keys, rows the queries of every head that shares the key head.
template <typename S>
__global__ void __launch_bounds__(S::kThreads, S::kGradKvWaves) attn_grad_kv_kernel(const AttnLaunch p, const BackwardParts parts) {
  typedef typename S::Tag Tag;
  extern __shared__ __align__(16) char lds[];
  __shared__ char s_flags[64];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, g = lane >> 4, c = lane & 15;
  const int row_wave = wave / S::kColumnWaves, column_wave = wave % S::kColumnWaves;
  const Place at(p.kv_heads, parts.tiles, parts.chunks);
  const int share = p.heads / p.kv_heads, heads_here = share / parts.head_parts, head0 = at.head * share + at.chunk % parts.head_parts * heads_here;
  const int first = at.chunk / parts.head_parts * parts.chunk_rows, last = min(p.nq, first + parts.chunk_rows);
  const int width_bytes = p.width * Tag::kBytes;
  const int column0 = at.tile * S::kColumns, mine0 = column0 + column_wave * 16 * S::CF;
  const bool masked = p.k_segments != nullptr;

  u32x4 k[S::CF][S::kSlices], v[S::CF][S::kSlices];
  load_columns<S>(k, head_rows<Tag>(p.k, at.b, at.head), mine0, p.nk, width_bytes, lane);
  load_columns<S>(v, head_rows<Tag>(p.v, at.b, at.head), mine0, p.nk, width_bytes, lane);
  const int *q_segments = p.q_segments != nullptr ? p.q_segments + (long long)at.b * p.nq : nullptr;
  const int *k_segments = masked ? p.k_segments + (long long)at.b * p.nk : nullptr;
  // queries low .. low + span see a key: its own segment's, or all that are not negative
  int low[S::CF];
  uint32_t span[S::CF];
  f32x2 point[S::CF];
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    const int j = mine0 + 16 * f + c, segment = j < p.nk ? (masked ? k_segments[j] : 0) : -1;
    low[f] = max(segment, -1);
    span[f] = segment == 0 ? 0x7fffffffu : 0u;
    point[f] = f32x2{0.f, 0.f};
    if (p.slopes != nullptr && j < p.nk) point[f] = reinterpret_cast<const f32x2 *>(p.k_points)[(long long)at.b * p.nk + j];
  }
  const ColumnRange range = masked ? column_range<true>(k_segments, column0, p.nk, S::kColumns, lane) : ColumnRange{};

  f32x4 dk[S::kWidthBlocks][S::CF], dv[S::kWidthBlocks][S::CF];
#pragma unroll
  for (int f = 0; f < S::CF; ++f)
#pragma unroll
    for (int d = 0; d < S::kWidthBlocks; ++d) dk[d][f] = dv[d][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  ColumnScale<S> up;

  for (int head = head0; head < head0 + heads_here; ++head) {
    const HeadRows queries = head_rows<Tag>(p.q, at.b, head), grads = head_rows<Tag>(p.grad_out, at.b, head);
    const Scores<S::kKind> scores(p, head);
    TileLoads<S> next_q, next_g;
    RowLoads next = {};
    auto request = [&](int row0) {
      next_q.request(queries, row0, last, width_bytes, wave, lane);
      next_g.request(grads, row0, last, width_bytes, wave, lane);
      const int row = row0 + (int)threadIdx.x;
      if ((int)threadIdx.x < S::RT) {
        const bool there = row < last;
        const long long stat = ((long long)at.b * p.heads + head) * p.nq + row;
        next.segment = there ? (q_segments != nullptr ? q_segments[row] : 0) : kHiddenColumn;
        next.lse = there ? p.lse[stat] : kInf;
        next.delta = there ? parts.delta[stat] : 0.f;
        if (scores.apart) next.point = there ? reinterpret_cast<const f32x2 *>(p.q_points)[(long long)at.b * p.nq + row] : f32x2{0.f, 0.f};
      }
    };
    auto put = [&](char *tile, bool every) {
      if (!every)
#pragma unroll
        for (int u = 0; u < S::kCarried; ++u) {
          const bool bad_q = next_q.clear_bad(u), bad_g = next_g.clear_bad(u);
          put_poison<S>(tile, u, bad_q || bad_g, wave, lane);
        }
      next_q.put(tile, wave, lane);
      next_g.put(tile + S::kTensorBytes, wave, lane);
      if ((int)threadIdx.x < S::RT) {
        reinterpret_cast<int *>(tile + S::kSegments)[threadIdx.x] = max(next.segment, kHiddenColumn) == -1 ? kHiddenColumn : max(next.segment, kHiddenColumn);
        reinterpret_cast<float *>(tile + S::kLse)[threadIdx.x] = next.lse - kBackwardShift<Tag>;
        reinterpret_cast<float *>(tile + S::kDelta)[threadIdx.x] = -next.delta;      // what the product dO V^T starts from
        if (scores.apart) reinterpret_cast<f32x2 *>(tile + S::kPoints)[threadIdx.x] = next.point;
      }
    };
    auto work = [&](const char *tile, bool every) {
#pragma unroll 1
      for (int n = 0; n < S::kRowBlocks; n += 2) {
        const int block = row_wave * S::kRowBlocks + n;
        f32x4 s[2][S::CF], t[2][S::CF], far[2][S::CF], bend[2][S::CF];
        const f32x4 *minus_delta = reinterpret_cast<const f32x4 *>(tile + S::kDelta) + block * 4 + g;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int f = 0; f < S::CF; ++f) {
            s[h][f] = f32x4{0.f, 0.f, 0.f, 0.f};
            t[h][f] = minus_delta[h * 4];
          }
        two_products<S>(tile, tile + S::kTensorBytes, block, k, v, s, t, lane);
        const f32x2 *points = reinterpret_cast<const f32x2 *>(tile + S::kPoints) + block * 16 + 4 * g;
        const int *segments = reinterpret_cast<const int *>(tile + S::kSegments) + block * 16 + 4 * g;
        const float *poison = reinterpret_cast<const float *>(tile + S::kPoison) + block * 16 + 4 * g;
        const float *lse = reinterpret_cast<const float *>(tile + S::kLse) + block * 16 + 4 * g;
        form_weights<Tag, S::kKind, S::CF>(scores, s, far, bend, point, [&](int h, int r) { return points[h * 16 + r]; }, [&](int h, int r, int) { return lse[h * 16 + r]; },
                                 [&] {
                                   if (every) return;
#pragma unroll
                                   for (int h = 0; h < 2; ++h)
#pragma unroll
                                     for (int f = 0; f < S::CF; ++f)
#pragma unroll
                                       for (int r = 0; r < 4; ++r) s[h][f][r] += poison[h * 16 + r];
                                 });
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int f = 0; f < S::CF; ++f) {
            t[h][f] *= s[h][f];
            if (scores.bent) t[h][f] *= bend[h][f];
          }
        if (!every)      // whatever there is of a pair that is not seen
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int f = 0; f < S::CF; ++f) {
                const bool seen = (uint32_t)segments[h * 16 + r] - (uint32_t)low[f] <= span[f];
                s[h][f][r] = seen ? s[h][f][r] : 0.f;
                t[h][f][r] = seen ? t[h][f][r] : 0.f;
              }
        add_product<S>(dv, tile + S::kTensorBytes, block, s, lane);
        up.apply(t, dk);
        add_product<S>(dk, tile, block, t, lane);
      }
    };
    walk_tiles<S, true>(q_segments, masked, range, first, last, lds, s_flags, wave, lane, request, put, work);
  }

  const float down = __builtin_amdgcn_exp2f(-kBackwardShift<Tag>);
#pragma unroll
  for (int f = 0; f < S::CF; ++f)
#pragma unroll
    for (int d = 0; d < S::kWidthBlocks; ++d) {
      dk[d][f] *= p.scale * (p.cap > 0.f ? kBendFactor<Tag> : 1.f) * down / up.by[f];
      dv[d][f] *= down;
    }
  merge_rows<S>(dk, lds, row_wave, column_wave, lane);
  merge_rows<S>(dv, lds, row_wave, column_wave, lane);
#pragma unroll
  for (int f = 0; f < S::CF; ++f) {
    const int j = mine0 + 16 * f + c;
    if (j >= p.nk) continue;
    const size_t rows = (size_t)p.batch * p.nk * p.kv_heads, row = ((size_t)at.b * p.nk + j) * p.kv_heads + at.head;
#pragma unroll
    for (int d = 0; d < S::kWidthBlocks; ++d) {
      if (!holds<S>(d, row_wave) || d * 16 + g * 4 >= p.width) continue;
      store_grad<Tag>(p.grad_k, parts.part, 2 * at.chunk * rows, row, p.width, d * 16 + g * 4, dk[d][f]);
      store_grad<Tag>(p.grad_v, parts.part, (2 * at.chunk + 1) * rows, row, p.width, d * 16 + g * 4, dv[d][f]);
    }
  }
}

// The chunks' parts, [chunk][tensors][elements], added in order and rounded: a lane takes four elements of one of the tensors.
template <typename Tag>
__global__ void __launch_bounds__(kJoinThreads) attn_join_grads_kernel(const float *part, int chunks, long long elements, void *first, void *second) {
  const int tensors = gridDim.y;
  const long long at = ((long long)blockIdx.x * kJoinThreads + threadIdx.x) * 4;
  void *to = blockIdx.y == 0 ? first : second;
  if (at >= elements || to == nullptr) return;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < chunks; ++k) sum += *reinterpret_cast<const f32x4 *>(part + ((long long)k * tensors + blockIdx.y) * elements + at);
  store4<Tag>(to, at, sum);
}

// ---------------------------------------------------------------- host
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Lanes that hold a row in fours, a power of two.
int row_lanes(const AttnLaunch &p) {
  int lanes = 2;
  while (lanes * 4 < p.width) lanes *= 2;
  return lanes;
}

// Columns a workgroup: many share the loads of a tile, few make workgroups for all CUs.  The most of which each CU gets one; with 16
// the four waves divide the rows, as they do in part with 64 and 32.  us of the forward kernel with 128 / 64 / 32 / 16 columns, heads of 32, 16
// bits: 8 heads x 300 queries 12.1 / 13.1 / 9.8 / 7.6; 16 x 1100 20.9 / 19.2 / 25.8 / 29.7; 32 x 1100 28.7 / 31.0 / 38.8 / 49.5; 32 x 2500
// 82 / 85 / 113 / 165.  The gradients' kernels go the same way: dK and dV 16.8 / 11.4 / 9.9 / 7.9 and 33.9 / 28.6 / 34.7 / 42.0 for the first two.
enum Mode { kColumns128, kColumns64, kColumns32, kColumns16 };
Mode column_mode(long long heads, int columns, bool masked, bool even) {
  // sequences that end within a tile cost the whole of it, and make workgroups of unequal work: 16 heads of 128, 5003 queries in sequences of
  // some hundred, forward with 128 columns 216 us, with 64 164
  // two workgroups a CU should come out even, but for plain scores of heads above 64 channels, whose tiles cost more to bring in: forward and
  // dQ of 8 heads, bf16, with distances, 32 channels, 2 x 2500 queries: 320 workgroups of 128 columns 95 and 103 us, 640 of 64 92 and 98;
  // 7744 queries 488 for 276 and 299, 968 for 320 and 313; plain, 5000 queries 320 for 124 and 101, 632 for 112 and 81; of 128 channels 227
  // for 232
  const long long blocks = heads * ceil_div(columns, 128), places = (blocks + 511) / 512 * 512;
  if (blocks >= (masked ? 1024 : 256) && (!even || 4 * blocks >= 3 * places)) return kColumns128;
  if (heads * ceil_div(columns, 64) >= 256) return kColumns64;
  return heads * ceil_div(columns, 32) >= 256 ? kColumns32 : kColumns16;
}
// Rows of a tile and sixteens of columns a wave, by the bytes of a row: narrow rows make long tiles; a wave with two sixteens reads half as
// much LDS, but backward it has no room for rows of 256 bytes (the gradients' kernels, 16 heads of 128, 4096 queries, 16 bits: 1560 us for 857).
template <typename Tag, int KIND, int W>
struct ForwardModes {
  static constexpr int kBytes = W * Tag::kBytes, kTwo = kBytes > 256 ? 1 : 2;
  typedef Shape<Tag, KIND, W, (kBytes > 64 ? 64 : 128), 1, kTwo, 4> Columns128;
  typedef Shape<Tag, KIND, W, (kBytes > 128 ? 64 : 128), (kBytes > 256 ? 1 : 2), kTwo, 4> Columns64;
  typedef Shape<Tag, KIND, W, (kBytes > 128 ? 64 : kBytes > 64 ? 128 : 256), (kBytes > 128 ? 2 : 4), (kBytes > 128 ? 1 : 2), 4> Columns32;
  typedef Shape<Tag, KIND, W, (kBytes > 128 ? 64 : 128), (kBytes > 128 ? 2 : 4), 1, 4> Columns16;
};
template <typename Tag, int KIND, int W>
struct BackwardModes {
  static constexpr int kBytes = W * Tag::kBytes, kTwo = kBytes > 128 ? 1 : 2;
  typedef Shape<Tag, KIND, W, (kBytes > 64 ? 64 : 128), 1, kTwo, 4> Columns128;
  typedef Shape<Tag, KIND, W, (kBytes > 64 ? 64 : 128), (kBytes > 128 ? 1 : 2), kTwo, 4> Columns64;
  typedef Shape<Tag, KIND, W, (kBytes > 128 ? 64 : 128), (kBytes > 128 ? 2 : 4), kTwo, 4> Columns32;
  typedef Shape<Tag, KIND, W, (kBytes > 128 ? 64 : 128), (kBytes > 128 ? 2 : 4), 1, 4> Columns16;
};

template <typename S, typename... A>
hipError_t run(void (*kernel)(A...), long long blocks, hipStream_t stream, A... args) {
  if (blocks * S::kThreads > 0xffffffffll) return hipErrorInvalidConfiguration;
  if (S::kLdsBytes > (int)kMaxDynamicLds)
    if (hipError_t e = ensure_dynamic_lds_limit(reinterpret_cast<const void *>(kernel), S::kLdsBytes)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(S::kThreads), S::kLdsBytes, stream, args...);
  return hipGetLastError();
}

// Few columns: the rows of a head are divided among workgroups too, four tiles or more each, and joined behind: two or three
// workgroups a compute unit, whose loads hide one another.  2 x 1 queries over 22223 rows, 8 heads of 32 in half precision:
// 11.0 us and 4.6 to join with 704 workgroups, 15.5 with 512 of twice the tile.
template <typename S>
Split plan_forward(const AttnLaunch &p) {
  Split s = {};
  s.tiles = ceil_div(p.nq, S::kColumns);
  s.chunks = 1;
  const long long blocks = (long long)p.batch * p.heads * s.tiles;
  const int row_tiles = std::max(1, ceil_div(p.nk, S::RT));
  int per_chunk = row_tiles;
  if (S::RW > 1 && blocks < 256 && row_tiles >= 8) {
    per_chunk = std::max(4, ceil_div(row_tiles, std::max(1ll, 768 / blocks)));
    s.chunks = ceil_div(row_tiles, per_chunk);
  }
  s.chunk_rows = per_chunk * S::RT;
  return s;
}
size_t part_bytes(const AttnLaunch &p, const Split &s) {
  return s.chunks > 1 ? padded((size_t)s.chunks * p.batch * p.nq * p.heads * p.width * sizeof(float)) : 0;
}
size_t forward_bytes(const AttnLaunch &p, const Split &s) {
  return s.chunks > 1 ? part_bytes(p, s) + padded((size_t)s.chunks * p.batch * p.nq * p.heads * 2 * sizeof(float)) : 0;
}

template <typename S>
hipError_t forward_shape(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  typedef typename S::Tag Tag;
  Split s = plan_forward<S>(p);
  if (bytes != nullptr) {
    *bytes = forward_bytes(p, s);
    return hipSuccess;
  }
  s.part = static_cast<float *>(p.workspace);
  s.stats = reinterpret_cast<float *>(static_cast<char *>(p.workspace) + part_bytes(p, s));
  const long long blocks = (long long)p.batch * p.heads * s.tiles * s.chunks;
  constexpr bool half = Tag::kBytes == 2;
  const bool train = half && p.lse != nullptr;
  if (hipError_t e = train ? run<S>(attn_forward_kernel<S, half>, blocks, stream, p, s) : run<S>(attn_forward_kernel<S, false>, blocks, stream, p, s)) return e;
  if (s.chunks == 1) return hipSuccess;
  hipLaunchKernelGGL((attn_join_kernel<Tag>), dim3((unsigned)ceil_div((long long)p.batch * p.nq * p.heads, kJoinWaves)), dim3(kJoinThreads), 0, stream, p, s,
                     row_lanes(p));
  return hipGetLastError();
}

// Chunks of the rows, where the columns' workgroups leave much of the chip free; each has some tiles of work.
template <typename S>
void divide_rows(BackwardParts *parts, long long blocks, int rows, int head_parts) {
  const int row_tiles = std::max(1, ceil_div(rows, S::RT));
  int per_chunk = row_tiles;
  if (blocks * head_parts < 192) per_chunk = ceil_div(row_tiles, std::max(1, (int)std::min<long long>(512 / (blocks * head_parts), row_tiles / 4)));
  parts->chunk_rows = per_chunk * S::RT;
  parts->head_parts = head_parts;
  parts->chunks = ceil_div(row_tiles, per_chunk) * head_parts;
}
template <typename S>
BackwardParts plan_grad_q(const AttnLaunch &p) {
  BackwardParts parts = {};
  parts.tiles = ceil_div(p.nq, S::kColumns);
  const long long blocks = (long long)p.batch * p.heads * parts.tiles;
  // (the slopes' sums are of whole rows)
  divide_rows<S>(&parts, p.slopes != nullptr ? 512 : blocks, p.nk, 1);
  return parts;
}
template <typename S>
BackwardParts plan_grad_kv(const AttnLaunch &p) {
  BackwardParts parts = {};
  parts.tiles = ceil_div(p.nk, S::kColumns);
  const long long blocks = (long long)p.batch * p.kv_heads * parts.tiles;
  // heads that share a key head in as many parts, all alike, as make 1024 workgroups: 64 heads of 64 over one, 5000 tokens, 16 bits, the whole
  // backward 2848 us, with 512 3433, with 2048 2892, with a head each 4244; 24 over 2, 8 x 1000 279, 273, 318, 316
  const int share = p.heads / p.kv_heads;
  int head_parts = 1;
  while (head_parts < share && (blocks * head_parts < 1024 || share % head_parts != 0)) ++head_parts;
  divide_rows<S>(&parts, blocks, p.nq, head_parts);
  return parts;
}
size_t delta_bytes(const AttnLaunch &p) { return padded((size_t)p.batch * p.heads * p.nq * sizeof(float)); }
size_t slope_bytes(const AttnLaunch &p) {      // of 16 columns or more each
  return p.slopes != nullptr ? padded((size_t)p.batch * p.heads * ceil_div(p.nq, 16) * sizeof(float)) : 0;
}
size_t query_elements(const AttnLaunch &p) { return (size_t)p.batch * p.nq * p.heads * p.width; }
size_t key_elements(const AttnLaunch &p) { return (size_t)p.batch * p.nk * p.kv_heads * p.width; }

// delta, the slopes' parts, then the chunks of the kernel at work
template <typename S>
hipError_t grad_q_shape(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  typedef typename S::Tag Tag;
  BackwardParts parts = plan_grad_q<S>(p);
  if (bytes != nullptr) {
    *bytes = parts.chunks > 1 ? padded(parts.chunks * query_elements(p) * sizeof(float)) : 0;
    return hipSuccess;
  }
  char *ws = static_cast<char *>(p.workspace);
  parts.delta = reinterpret_cast<float *>(ws);
  if (p.grad_slopes != nullptr) parts.slopes = reinterpret_cast<float *>(ws + delta_bytes(p));
  if (parts.chunks > 1) parts.part = reinterpret_cast<float *>(ws + delta_bytes(p) + slope_bytes(p));
  if (hipError_t e = run<S>(attn_grad_q_kernel<S>, (long long)p.batch * p.heads * parts.tiles * parts.chunks, stream, p, parts)) return e;
  if (parts.slopes != nullptr) {
    if (hipError_t e = launch_slope_grad(parts.slopes, p.grad_slopes, p.batch, p.heads, parts.tiles, stream)) return e;
  }
  if (parts.chunks == 1 || p.grad_q == nullptr) return hipSuccess;
  const long long n = (long long)query_elements(p);
  hipLaunchKernelGGL((attn_join_grads_kernel<Tag>), dim3(ceil_div(n, 4 * kJoinThreads)), dim3(kJoinThreads), 0, stream, parts.part, parts.chunks, n, p.grad_q,
                     (void *)nullptr);
  return hipGetLastError();
}
template <typename S>
hipError_t grad_kv_shape(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  typedef typename S::Tag Tag;
  BackwardParts parts = plan_grad_kv<S>(p);
  if (bytes != nullptr) {
    *bytes = parts.chunks > 1 ? padded(2 * parts.chunks * key_elements(p) * sizeof(float)) : 0;
    return hipSuccess;
  }
  char *ws = static_cast<char *>(p.workspace);
  parts.delta = reinterpret_cast<float *>(ws);
  if (parts.chunks > 1) parts.part = reinterpret_cast<float *>(ws + delta_bytes(p) + slope_bytes(p));
  if (hipError_t e = run<S>(attn_grad_kv_kernel<S>, (long long)p.batch * p.kv_heads * parts.tiles * parts.chunks, stream, p, parts)) return e;
  if (parts.chunks == 1) return hipSuccess;
  const long long n = (long long)key_elements(p);
  hipLaunchKernelGGL((attn_join_grads_kernel<Tag>), dim3(ceil_div(n, 4 * kJoinThreads), 2), dim3(kJoinThreads), 0, stream, parts.part, parts.chunks, n, p.grad_k,
                     p.grad_v);
  return hipGetLastError();
}

template <typename Tag, int KIND, int W>
hipError_t forward_width(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  typedef ForwardModes<Tag, KIND, W> M;
  switch (column_mode((long long)p.batch * p.heads, p.nq, p.k_segments != nullptr, KIND != kPlainScores || W <= 64)) {
    case kColumns128: return forward_shape<typename M::Columns128>(p, stream, bytes);
    case kColumns64: return forward_shape<typename M::Columns64>(p, stream, bytes);
    case kColumns32: return forward_shape<typename M::Columns32>(p, stream, bytes);
    default: return forward_shape<typename M::Columns16>(p, stream, bytes);
  }
}

template <typename Tag, int KIND, int W>
hipError_t backward_width(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  typedef BackwardModes<Tag, KIND, W> M;
  const bool keys = bytes != nullptr || p.grad_k != nullptr || p.grad_v != nullptr;
  size_t q_bytes = 0, kv_bytes = 0;
  hipError_t e = hipSuccess;
  switch (column_mode((long long)p.batch * p.heads, p.nq, p.k_segments != nullptr, KIND != kPlainScores || W <= 64)) {
    case kColumns128: e = grad_q_shape<typename M::Columns128>(p, stream, bytes ? &q_bytes : nullptr); break;
    case kColumns64: e = grad_q_shape<typename M::Columns64>(p, stream, bytes ? &q_bytes : nullptr); break;
    case kColumns32: e = grad_q_shape<typename M::Columns32>(p, stream, bytes ? &q_bytes : nullptr); break;
    default: e = grad_q_shape<typename M::Columns16>(p, stream, bytes ? &q_bytes : nullptr);
  }
  if (e != hipSuccess || !keys) return e;
  switch (column_mode((long long)p.batch * p.kv_heads, p.nk, p.k_segments != nullptr, KIND != kPlainScores || W <= 64)) {
    case kColumns128: e = grad_kv_shape<typename M::Columns128>(p, stream, bytes ? &kv_bytes : nullptr); break;
    case kColumns64: e = grad_kv_shape<typename M::Columns64>(p, stream, bytes ? &kv_bytes : nullptr); break;
    case kColumns32: e = grad_kv_shape<typename M::Columns32>(p, stream, bytes ? &kv_bytes : nullptr); break;
    default: e = grad_kv_shape<typename M::Columns16>(p, stream, bytes ? &kv_bytes : nullptr);
  }
  if (bytes != nullptr) *bytes = delta_bytes(p) + slope_bytes(p) + std::max(q_bytes, kv_bytes);
  return e;
}

bool plain_scores(const AttnLaunch &p) { return p.cap == 0.f && p.slopes == nullptr && p.scale > 0.f; }

template <typename Tag, int KIND>
hipError_t forward_scores(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  if (p.width <= 32) return forward_width<Tag, KIND, 32>(p, stream, bytes);
  return p.width <= 64 ? forward_width<Tag, KIND, 64>(p, stream, bytes) : forward_width<Tag, KIND, 128>(p, stream, bytes);
}
template <typename Tag>
hipError_t forward_t(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  if (plain_scores(p)) return forward_scores<Tag, kPlainScores>(p, stream, bytes);
  if constexpr (Tag::kBytes == 2)
    if (p.cap > kQuickCap) return forward_scores<Tag, kHighCap>(p, stream, bytes);
  return forward_scores<Tag, kAnyScores>(p, stream, bytes);
}
template <typename Tag, int KIND>
hipError_t backward_scores(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  if (p.width <= 32) return backward_width<Tag, KIND, 32>(p, stream, bytes);
  return p.width <= 64 ? backward_width<Tag, KIND, 64>(p, stream, bytes) : backward_width<Tag, KIND, 128>(p, stream, bytes);
}
template <typename Tag>
hipError_t backward_t(const AttnLaunch &p, hipStream_t stream, size_t *bytes) {
  if (plain_scores(p)) return backward_scores<Tag, kPlainScores>(p, stream, bytes);
  if constexpr (Tag::kBytes == 2)
    if (p.cap > kQuickCap) return backward_scores<Tag, kHighCap>(p, stream, bytes);
  return backward_scores<Tag, kAnyScores>(p, stream, bytes);
}

}  // namespace
}  // namespace dcn
