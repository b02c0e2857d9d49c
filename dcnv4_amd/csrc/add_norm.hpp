// Launch struct of the normalised sum (add_norm.hip); beside the C ABI, for the extension.
#pragma once
#include <hip/hip_runtime.h>

#include <stddef.h>

namespace dcn {

// A matrix of rows: its type's code and the elements between rows; rows need only their elements' alignment.
struct NormRows {
  const void *base;
  int dtype;
  long long pitch;
};

// out = LayerNorm(x + residual) over rows of `width`, and the sum itself.
struct AddNormLaunch {
  NormRows x, residual;           // residual may be null; of x's type or fp32
  const void *weight, *bias;      // of type param_dtype, or null: ones and zeros
  int param_dtype;
  long long rows;
  int width;
  float eps;
  bool wide;                      // a result in fp32 whatever the summands
  void *out, *sum;                // dense; the sum, of the summands' wider type, may be null
  float *stats;                   // (rows, 2): mean and 1 / deviation; the forward writes them where they are wanted
  // backward: x, residual, stats and
  const void *grad_out, *grad_sum;                  // dense, of the outputs' types; grad_sum may be null
  void *grad_x, *grad_residual;                     // dense, of the summands' types; each may be null
  void *grad_weight, *grad_bias;                    // each may be null
  void *workspace;
};

constexpr int kMaxNormWidth = 8192;
size_t add_norm_backward_workspace_bytes(const AddNormLaunch &p);
hipError_t launch_add_norm_forward(const AddNormLaunch &p, hipStream_t stream);
hipError_t launch_add_norm_backward(const AddNormLaunch &p, hipStream_t stream);

}  // namespace dcn
