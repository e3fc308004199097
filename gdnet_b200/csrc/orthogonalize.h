// Host-visible interface of the Newton-Schulz products (orthogonalize.cu).
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace gd {

constexpr int NS_MAX_BATCH = 64;       // matrices of one shape per call: their addresses travel in the kernel arguments
constexpr int NS_NORM_BLOCKS = 256;    // partial sums of a matrix's norm

// Element-wise ends of a call: what the matrices are made from and where the result goes.
struct NsEnds {
  int batch, rows, cols;
  int ld;                              // row pitch of the workspace planes (elements)
  int64_t plane;                       // elements of one workspace plane
  const void* grad[NS_MAX_BATCH];      // input, or the (task) gradient
  const void* info[NS_MAX_BATCH];      // information gradient, may be null
  void* moment[NS_MAX_BATCH];          // fp32 momentum, updated in place (momentum != 0)
  void* out[NS_MAX_BATCH];             // result, or the parameter, updated in place
  int grad_dtype, out_dtype;           // ElemType
  int64_t grad_ld;                     // row pitch of the input without momentum
  const float* scalars;                // {projection coefficient, gradient scale} on the device, may be null
  float beta, mu, eps, decay, step;
  int momentum, nesterov;
  float* u;
  double* partial;
  __half* x_hi;
  __half* x_lo;
  int tpr_log2;                        // threads per row (log2)
  uint32_t* done;                      // tile counts, cleared by the first kernel of a call
  uint32_t* next_item;
};

// All products of a call (see ns_chain_body). Tensor maps [buffer][hi, lo], of the symmetric factors [hi, lo][K-major, MN-major].
struct NsPlan {
  CUtensorMap x_gram[2][2], x_apply[2][2], x_box[2][2];
  CUtensorMap a_load[2][2], b_load[2][2], a_box[2], b_box[2];
  int batch, steps, rows, cols, tall;
  int k, wide;                         // smaller and larger side
  int tiles_sym, tiles_x, tiles_xm;    // tiles of a symmetric product, of X, row blocks of X
  int items;
  float a, b, c;
  uint32_t* done;                      // [batch] finished tiles, counted in epilogue warps
  uint32_t* next_item;
};

// A call whose matrices stay in one cluster each (see ns_small_kernel).
struct NsSmall {
  int k, wide, tall, steps;
  int ctas, slice;                     // CTAs per matrix, columns of X per CTA
  float a, b, c;
};

struct NsCall {
  NsEnds ends;
  void* workspace;                     // ns_workspace_bytes(), 256-byte aligned
  int steps, pairs;
  float c[3];                          // coefficients a, b, c of the step
};

int64_t ns_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int steps, int pairs);
const char* launch_orthogonalize(const NsCall& call, Status* status, cudaStream_t st);

}  // namespace gd
