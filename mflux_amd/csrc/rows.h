// What abi.hip hands to the kernels of rms_norm.hip and int8_matmul.hip.
#pragma once

#include "common.h"

namespace mfq {

// Rows through the norm, into codes, or back.  Strides are of rows, in elements; what has none is densely packed.
struct RowsCall {
  const void *x, *residual, *weight;  // backward: x is what was normalised
  const void *dy, *dsum;
  void *y, *sum, *dx, *dweight;
  int8_t* codes;   // forward: these and the scales, or y
  float* scales;
  float* parts;    // backward: partial sums of the weight's gradient, one row a workgroup
  int64_t rows, columns;
  int64_t x_stride, residual_stride, dy_stride, dsum_stride, code_stride;
  float eps;
  bool norm;
};

// wide: every array is 16-byte aligned, its rows too, and they are whole 16 bytes long (codes: half as much)
int launch_rows(int dtype, const RowsCall& c, bool wide, bool backward, hipStream_t stream);
size_t rows_workspace_bytes(int64_t rows, int64_t columns);  // of the backward pass with a weight's gradient
int launch_rows_values(const int8_t* codes, int64_t stride, const float* scales, int64_t rows, int64_t columns, int dtype, void* out,
                       hipStream_t stream);

// y = x_scales[m] w_scales[n] sum_k x[m][k] w[n][k] + bias[n]
struct Int8Call {
  const int8_t *x, *w;
  const float *x_scales, *w_scales;
  const void* bias;  // of y's type, or nullptr
  void* y;           // [M, N], rows of y_stride
  int64_t M, N, K, y_stride;
  int64_t x_stride, w_stride;  // of rows, whole 16 bytes
};

// The kernel a call takes and how it is cut
struct Int8Tiles {
  int rows, columns;  // of a workgroup's tile
  int places;         // of workgroups on a compute unit
};
struct Int8Plan {
  int kernel;   // MFQ_INT8_*
  int splits;   // ranges of K
  Int8Tiles tiles;
  int64_t first;   // columns of y that these tiles have, 0: all
  Int8Tiles rest;  // of the others
};
Int8Plan int8_plan(int dtype, int64_t M, int64_t N, int64_t K);
size_t int8_workspace_bytes(const Int8Plan& p, int64_t M, int64_t N);
int launch_int8_matmul(int dtype, const Int8Call& c, const Int8Plan& p, void* workspace, hipStream_t stream);

}  // namespace mfq
