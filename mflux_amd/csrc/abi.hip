// C ABI of libmfq.so: argument validation and dispatch.  No kernel is
// launched unless every check has passed, so a caller's mistake is an error
// code and never a device fault.
#include "attention.h"
#include "common.h"
#include "rows.h"

#include <cmath>
#include <limits>

namespace {

int check_common(int gs, int bits) {
  if (gs != 32 && gs != 64 && gs != 128) return MFQ_EGROUP;
  if (bits != 3 && bits != 4 && bits != 5 && bits != 6 && bits != 8) return MFQ_EBITS;
  return MFQ_OK;
}

bool is16(int dtype) { return dtype == MFQ_BF16 || dtype == MFQ_F16; }
bool known(int dtype) { return dtype == MFQ_F32 || is16(dtype); }

// The float32 planes of mfq_qmm_t_static's K split.  Every device the library
// runs on holds its own copy of this array, at its own address, until the
// process ends; the name below is only the host's handle for it, the address
// on the current device comes from hipGetSymbolAddress (scratch_on_device).
constexpr size_t kScratchBytes = MFQ_STATIC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];
std::atomic<void*> scratch_ptr[mfq::kMaxDevices];

// Address of `scratch` on the current device, looked up once per device.
int scratch_on_device(void** out) {
  const int dev = mfq::device_index();
  if (dev < 0) return MFQ_ELAUNCH;
  void* p = scratch_ptr[dev].load(std::memory_order_acquire);
  if (!p) {
    if (hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)) != hipSuccess || !p) return MFQ_ELAUNCH;
    scratch_ptr[dev].store(p, std::memory_order_release);
  }
  *out = p;
  return MFQ_OK;
}

}  // namespace

extern "C" {

int mfq_version(void) { return 100; }

const char* mfq_strerror(int status) {
  switch (status) {
    case MFQ_OK: return "ok";
    case MFQ_EDTYPE: return "unsupported dtype";
    case MFQ_EGROUP: return "group_size must be 32, 64 or 128";
    case MFQ_EBITS: return "bits must be 3, 4, 5, 6 or 8";
    case MFQ_ESHAPE: return "bad shape: sizes must be positive and K a multiple of group_size";
    case MFQ_ENULL: return "null pointer";
    case MFQ_EALIGN: return "buffers must be 16-byte aligned";
    case MFQ_ELAUNCH: return "HIP launch failed";
    case MFQ_EUNSUPPORTED: return "no kernel for this combination";
    case MFQ_ESCRATCH: return "the shape needs more scratch than the library's built-in buffer holds";
    default: return "unknown status";
  }
}

int mfq_quantize_affine(const void* w, int dtype, int64_t rows, int64_t K, int group_size, int bits, uint32_t* wq,
                        void* scales, void* biases, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (!known(dtype)) return MFQ_EDTYPE;
  if (rows <= 0 || K <= 0 || K % group_size) return MFQ_ESHAPE;
  if (!w || !wq || !scales || !biases) return MFQ_ENULL;
  if (!mfq::aligned16(w) || !mfq::aligned16(wq)) return MFQ_EALIGN;
  return mfq::launch_quantize(w, dtype, rows, K, group_size, bits, wq, scales, biases, (hipStream_t)stream);
}

int mfq_dequantize_affine(const uint32_t* wq, const void* scales, const void* biases, int sb_dtype, int64_t rows,
                          int64_t K, int group_size, int bits, void* out, int out_dtype, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (!known(sb_dtype) || !known(out_dtype)) return MFQ_EDTYPE;
  if (rows <= 0 || K <= 0 || K % group_size) return MFQ_ESHAPE;
  if (!wq || !scales || !biases || !out) return MFQ_ENULL;
  if (!mfq::aligned16(wq) || !mfq::aligned16(out)) return MFQ_EALIGN;
  return mfq::launch_dequantize(wq, scales, biases, sb_dtype, rows, K, group_size, bits, out, out_dtype,
                                (hipStream_t)stream);
}

int mfq_dequantize_rows(const uint32_t* wq, const void* scales, const void* biases, int sb_dtype, const int64_t* indices,
                        int64_t n_indices, int64_t n_rows, int64_t K, int group_size, int bits, void* out,
                        int out_dtype, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (!known(sb_dtype) || !known(out_dtype)) return MFQ_EDTYPE;
  if (n_indices <= 0 || n_rows <= 0 || K <= 0 || K % group_size) return MFQ_ESHAPE;
  if (n_indices > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  if (!wq || !scales || !biases || !indices || !out) return MFQ_ENULL;
  if (!mfq::aligned16(wq) || !mfq::aligned16(out)) return MFQ_EALIGN;
  return mfq::launch_dequantize_rows(wq, scales, biases, sb_dtype, indices, n_indices, n_rows, K, group_size, bits,
                                     out, out_dtype, (hipStream_t)stream);
}

// the kernel of a call and what else is asked for, planned once: a plan is a good part of a small call's host time
static int route_of(int64_t M, int64_t K, int64_t N, int group_size, int bits,
                    mfq::QmmRoute (*plan)(int64_t M, int64_t N, int64_t K, int gs, int bits), mfq::QmmRoute* route) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (M <= 0 || N <= 0 || K <= 0 || K % group_size || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  const bool odd_bits = bits != 4 && bits != 8;
  if (odd_bits && M == 1 && K > 8192) return MFQ_EUNSUPPORTED;  // (a GEMM without the workspace that qmm_route() counts on)
  *route = mfq::QmmRoute{MFQ_KERNEL_MATVEC, 1, 0, 0};
  if (M > (odd_bits ? 1 : 16)) *route = plan(M, N, K, group_size, bits);
  return route->kernel;
}

int mfq_qmm_t_kernel(int64_t M, int64_t K, int64_t N, int group_size, int bits, int* k_ranges) {
  mfq::QmmRoute route;
  const int kernel = route_of(M, K, N, group_size, bits, mfq::qmm_route, &route);
  if (kernel > 0 && k_ranges) *k_ranges = route.ranges;
  return kernel;
}

size_t mfq_qmm_t_workspace_bytes(int64_t M, int64_t K, int64_t N, int group_size, int bits) {
  if (check_common(group_size, bits) != MFQ_OK) return 0;
  if (N <= 0 || K <= 0 || K % group_size || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return 0;
  if (M <= (bits == 4 || bits == 8 ? 16 : 1)) return 0;
  const mfq::QmmRoute route = mfq::qmm_route(M, N, K, group_size, bits);
  return route.copy + route.planes;
}

int mfq_qmm_t_plan(int64_t M, int64_t K, int64_t N, int group_size, int bits, int epilogue, int* k_ranges, int* tile_rows,
                   int* tile_columns, size_t* workspace_bytes) {
  if (workspace_bytes) *workspace_bytes = 0;
  if (epilogue < 0 || epilogue > MFQ_EPILOGUE_SWIGLU) return MFQ_ESHAPE;
  mfq::QmmRoute route;
  const int kernel = route_of(M, K, N, group_size, bits, epilogue ? mfq::qmm_epilogue_route : mfq::qmm_linear_route, &route);
  if (kernel < 0) return kernel;
  if (epilogue && (M <= 16 || N % 8)) return MFQ_EUNSUPPORTED;
  if (epilogue == MFQ_EPILOGUE_SWIGLU && N % 64) return MFQ_ESHAPE;
  if (k_ranges) *k_ranges = route.ranges;
  if (workspace_bytes) *workspace_bytes = route.copy + route.planes;
  if (tile_rows && tile_columns) mfq::qmm_route_tile(route, M, N, K, group_size, bits, !epilogue, tile_rows, tile_columns);
  return route.kernel;
}

int mfq_qmm_t(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq, const void* scales,
              const void* biases, int sb_dtype, const void* bias, int64_t N, int group_size, int bits, void* y,
              int y_dtype, void* stream) {
  return mfq_qmm_t_ws(x, x_dtype, M, K, wq, scales, biases, sb_dtype, bias, N, group_size, bits, y, y_dtype, nullptr, 0,
                      stream);
}

int mfq_qmm_t_ws(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq, const void* scales,
                 const void* biases, int sb_dtype, const void* bias, int64_t N, int group_size, int bits, void* y,
                 int y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return mfq_qmm_t_low_rank(x, x_dtype, M, K, wq, scales, biases, sb_dtype, bias, N, group_size, bits, nullptr, nullptr,
                            0, y, y_dtype, workspace, workspace_bytes, stream);
}

int mfq_qmm_t_static(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq, const void* scales,
                     const void* biases, int sb_dtype, const void* bias, int64_t N, int group_size, int bits, void* y,
                     int y_dtype, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  size_t need = mfq_qmm_t_workspace_bytes(M, K, N, group_size, bits);
  // a scratch copy of the weights that does not fit is done without (the fused kernel); the planes of a K split are not
  if (need > kScratchBytes && (bits == 4 || bits == 8) && M > 16) need = mfq::qmm_route(M, N, K, group_size, bits).planes;
  if (need > kScratchBytes) return MFQ_ESCRATCH;
  void* ws = nullptr;
  if (need) {
    if (int rc = scratch_on_device(&ws)) return rc;
  }
  return mfq_qmm_t_low_rank(x, x_dtype, M, K, wq, scales, biases, sb_dtype, bias, N, group_size, bits, nullptr, nullptr,
                            0, y, y_dtype, ws, need, stream);
}

size_t mfq_qmm_t_prepared_bytes(int64_t N, int64_t K, int bits) {
  if (N <= 0 || K <= 0 || N > INT32_MAX || K > INT32_MAX || !mfq::qmm_frag_shape_ok(1, N, K, bits)) return 0;
  return mfq::qmm_frag_copy_bytes(N, K);
}

int mfq_qmm_t_prepare(const uint32_t* wq, const void* scales, const void* biases, int sb_dtype, int64_t N, int64_t K,
                      int group_size, int bits, void* prepared, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (!is16(sb_dtype)) return MFQ_EDTYPE;
  if (N <= 0 || K <= 0 || K % group_size || N > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  if (!wq || !scales || !biases || !prepared) return MFQ_ENULL;
  if (!mfq::aligned16(wq) || !mfq::aligned16(prepared)) return MFQ_EALIGN;
  return mfq::launch_qmm_frag_copy(sb_dtype, wq, scales, biases, N, K, group_size, bits, prepared, (hipStream_t)stream);
}

size_t mfq_qmm_t_prepared_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return 0;
  if (!mfq::qmm_frag_shape_ok(M, N, K, 4)) return 0;
  return mfq::qmm_prepared_workspace_bytes(M, N, K);
}

int mfq_qmm_t_prepared(const void* x, int dtype, int64_t M, int64_t K, const void* prepared, const void* bias, int64_t N,
                       void* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (!is16(dtype)) return MFQ_EDTYPE;
  if (M <= 0 || N <= 0 || K <= 0) return MFQ_ESHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  if (!x || !prepared || !y) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(prepared) || !mfq::aligned16(y)) return MFQ_EALIGN;
  return mfq::launch_qmm_prepared(x, dtype, M, K, prepared, bias, N, y, workspace, workspace_bytes, (hipStream_t)stream);
}

int mfq_qmm_t_low_rank(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq, const void* scales,
                       const void* biases, int sb_dtype, const void* bias, int64_t N, int group_size, int bits,
                       const void* t, const void* bs, int64_t rank, void* y, int y_dtype, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (rank < 0 || rank > 1024 || rank % 16) return MFQ_ESHAPE;
  if (rank && (!t || !bs)) return MFQ_ENULL;
  if (rank && (!mfq::aligned16(t) || !mfq::aligned16(bs))) return MFQ_EALIGN;
  mfq::LowRank low_rank;
  if (rank) {
    low_rank.t = t;
    low_rank.bs = bs;
    low_rank.R = (int)rank;
  }
  const bool odd_bits = bits != 4 && bits != 8;
  if (!is16(x_dtype) || x_dtype != sb_dtype) return MFQ_EDTYPE;
  if (y_dtype != sb_dtype && y_dtype != MFQ_F32) return MFQ_EDTYPE;
  if (M <= 0 || N <= 0 || K <= 0 || K % group_size) return MFQ_ESHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  if (!x || !wq || !scales || !biases || !y) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(wq)) return MFQ_EALIGN;
  if (M > 16 && !mfq::aligned16(y)) return MFQ_EALIGN;  // the GEMM writes y in 16-byte pieces
  if (odd_bits) {
    // 3, 5, 6 bits: the one-row kernel for the rows it takes, the sliced or the 128-column-tile GEMM for everything else
    if (M == 1) {
      const int rc = mfq::launch_qmv_odd(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                                         (hipStream_t)stream);
      if (rc != MFQ_EUNSUPPORTED)
        return rc ? rc : mfq::launch_low_rank_add(x_dtype, low_rank, M, N, y, y_dtype, (hipStream_t)stream);
    }
    if (!mfq::aligned16(y)) return MFQ_EALIGN;
    // many rows and room for the scratch copy: the two-kernel path of the 4- and 8-bit weights
    if (M > 16 && K % 64 == 0 && (y_dtype == x_dtype || !rank) && workspace && mfq::aligned16(workspace) &&
        mfq::qmm_frag_shape_ok(M, N, K, bits) && workspace_bytes >= mfq::qmm_frag_copy_bytes(N, K) &&
        mfq::prefer_frag_path(M, N, K, group_size, bits))
      return mfq::launch_qmm(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype, workspace,
                             workspace_bytes, (hipStream_t)stream, low_rank);
    return mfq::launch_qmm_mid_stream(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                                      workspace, workspace_bytes, (hipStream_t)stream, low_rank);
  }
  if (M <= 16) {
    const int rc = mfq::launch_qmv(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                                   (hipStream_t)stream);
    return rc ? rc : mfq::launch_low_rank_add(x_dtype, low_rank, M, N, y, y_dtype, (hipStream_t)stream);
  }
  if (K % 64)  // group size 32 with K an odd multiple of it: the 128-column-tile GEMM pads the last k step with zeros
    return mfq::launch_qmm_mid(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype, nullptr, 0,
                               (hipStream_t)stream, low_rank);
  return mfq::launch_qmm(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype, workspace,
                         workspace_bytes, (hipStream_t)stream, low_rank);
}

int mfq_qmm_t_epilogue(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq, const void* scales,
                       const void* biases, int sb_dtype, const void* bias, int64_t N, int group_size, int bits,
                       int epilogue, const void* gate, const void* residual, int64_t act_from, void* y, int y_dtype,
                       void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (epilogue != MFQ_EPILOGUE_GELU && epilogue != MFQ_EPILOGUE_GATE_RESIDUAL && epilogue != MFQ_EPILOGUE_SWIGLU)
    return MFQ_ESHAPE;
  if (!is16(x_dtype) || x_dtype != sb_dtype || y_dtype != sb_dtype) return MFQ_EDTYPE;
  if (M <= 0 || N <= 0 || K <= 0 || K % group_size) return MFQ_ESHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  if (!x || !wq || !scales || !biases || !y) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(wq) || !mfq::aligned16(y)) return MFQ_EALIGN;
  mfq::Epilogue epi;
  epi.kind = epilogue;
  if (epilogue == MFQ_EPILOGUE_GELU) {
    if (act_from < 0 || act_from > N || act_from % 8) return MFQ_ESHAPE;
    epi.act_from = (int)act_from;
  } else if (epilogue == MFQ_EPILOGUE_GATE_RESIDUAL) {
    if (!gate || !residual) return MFQ_ENULL;
    if (!mfq::aligned16(gate) || !mfq::aligned16(residual)) return MFQ_EALIGN;
    epi.gate = static_cast<const uint16_t*>(gate);
    epi.residual = static_cast<const uint16_t*>(residual);
  } else if (N % 64) {
    return MFQ_ESHAPE;  // gate and up projections alternate in blocks of 32 rows
  }
  // the matvec kernels (M <= 16) have no epilogue, nor have rows that are not whole 16-byte pieces
  if (M <= 16 || N % 8) return MFQ_EUNSUPPORTED;
  if (bits != 4 && bits != 8)
    return mfq::launch_qmm_mid_stream(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                                      workspace, workspace_bytes, (hipStream_t)stream, mfq::LowRank(), epi);
  if (K % 64)
    return mfq::launch_qmm_mid(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype, nullptr, 0,
                               (hipStream_t)stream, mfq::LowRank(), epi);
  return mfq::launch_qmm(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype, workspace,
                         workspace_bytes, (hipStream_t)stream, mfq::LowRank(), epi);
}

int mfq_qmm_n(const void* x, int x_dtype, int64_t M, int64_t N, const uint32_t* wq, const void* scales,
              const void* biases, int sb_dtype, int64_t K, int group_size, int bits, void* y, int y_dtype, void* stream) {
  return mfq_qmm_n_ws(x, x_dtype, M, N, wq, scales, biases, sb_dtype, K, group_size, bits, y, y_dtype, nullptr, 0, stream);
}

size_t mfq_qmm_n_workspace_bytes(int64_t M, int64_t N, int64_t K, int group_size, int bits) {
  if (check_common(group_size, bits) != MFQ_OK) return 0;
  if (M <= 0 || N <= 0 || K <= 0 || K % group_size || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return 0;
  return mfq::qmm_n_workspace_bytes(M, N, K, group_size, bits);
}

int mfq_qmm_n_ws(const void* x, int x_dtype, int64_t M, int64_t N, const uint32_t* wq, const void* scales,
                 const void* biases, int sb_dtype, int64_t K, int group_size, int bits, void* y, int y_dtype,
                 void* workspace, size_t workspace_bytes, void* stream) {
  return mfq_qmm_n_low_rank(x, x_dtype, M, N, wq, scales, biases, sb_dtype, K, group_size, bits, nullptr, nullptr, 0, y,
                            y_dtype, workspace, workspace_bytes, stream);
}

int mfq_qmm_n_low_rank(const void* x, int x_dtype, int64_t M, int64_t N, const uint32_t* wq, const void* scales,
                       const void* biases, int sb_dtype, int64_t K, int group_size, int bits, const void* t,
                       const void* bs, int64_t rank, void* y, int y_dtype, void* workspace, size_t workspace_bytes,
                       void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (rank < 0 || rank > 1024 || rank % 16) return MFQ_ESHAPE;
  if (rank && (!t || !bs)) return MFQ_ENULL;
  if (rank && (!mfq::aligned16(t) || !mfq::aligned16(bs))) return MFQ_EALIGN;
  mfq::LowRank low_rank;
  if (rank) {
    low_rank.t = t;
    low_rank.bs = bs;
    low_rank.R = (int)rank;
  }
  if (!is16(x_dtype) || x_dtype != sb_dtype) return MFQ_EDTYPE;
  if (y_dtype != sb_dtype && y_dtype != MFQ_F32) return MFQ_EDTYPE;
  if (M <= 0 || N <= 0 || K <= 0 || K % group_size) return MFQ_ESHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX || N * (K * bits / 32) >= (int64_t)1 << 31) return MFQ_ESHAPE;
  if (!x || !wq || !scales || !biases || !y) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(wq) || !mfq::aligned16(y)) return MFQ_EALIGN;
  return mfq::launch_qmm_n_ws(x, x_dtype, M, N, wq, scales, biases, K, group_size, bits, y, y_dtype, workspace,
                              workspace_bytes, (hipStream_t)stream, low_rank);
}

int mfq_qmv_silu(const void* x, int x_dtype, int64_t M, int64_t K, const uint32_t* wq, const void* scales,
                 const void* biases, int sb_dtype, const void* bias, int64_t N, int group_size, int bits, void* y,
                 int y_dtype, void* stream) {
  if (int rc = check_common(group_size, bits)) return rc;
  if (!is16(x_dtype) || x_dtype != sb_dtype) return MFQ_EDTYPE;
  if (y_dtype != sb_dtype && y_dtype != MFQ_F32) return MFQ_EDTYPE;
  if (M <= 0 || N <= 0 || K <= 0 || K % group_size) return MFQ_ESHAPE;
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  if (!x || !wq || !scales || !biases || !y) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(wq)) return MFQ_EALIGN;
  if (bits != 4 && bits != 8) return MFQ_EUNSUPPORTED;
#ifndef MFQ_NO_OCT
  if (mfq::qmv_oct_covers(M, K, N, group_size, bits, x, scales, biases))
    return mfq::launch_qmv_oct(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                               (hipStream_t)stream, true);
  if (mfq::qmv_oct4_covers(M, K, N, group_size, bits, x, scales, biases))
    return mfq::launch_qmv_oct4(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                                (hipStream_t)stream, true);
#endif
  if (mfq::qmv_dot_covers(M, K, bits))
    return mfq::launch_qmv_dot(x, x_dtype, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                               (hipStream_t)stream, true);
  if (M >= 2 && M <= 4 && mfq::qmv_quad_covers(M, K, N, group_size, bits, scales, biases, bias, y, y_dtype))
    return mfq::launch_qmv_quad(x, x_dtype, M, K, wq, scales, biases, bias, N, group_size, bits, y, y_dtype,
                                (hipStream_t)stream, true);
  return MFQ_EUNSUPPORTED;
}

int mfq_silu(const void* x, int dtype, int64_t n, void* y, void* stream) {
  if (!is16(dtype)) return MFQ_EDTYPE;
  if (n <= 0 || n > INT32_MAX) return MFQ_ESHAPE;
  if (!x || !y) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(y)) return MFQ_EALIGN;
  return mfq::launch_silu(x, dtype, n, y, (hipStream_t)stream);
}

int mfq_round(const float* x, int64_t n, int dtype, void* y, void* stream) {
  if (!is16(dtype)) return MFQ_EDTYPE;
  if (n <= 0 || n > (int64_t)1 << 40) return MFQ_ESHAPE;
  if (!x || !y) return MFQ_ENULL;
  if (!mfq::aligned16(y)) return MFQ_EALIGN;
  return mfq::launch_round(x, n, dtype, y, (hipStream_t)stream);
}

int mfq_layer_norm_modulate(const void* x, int dtype, int64_t M, int64_t K, const void* scale, const void* shift,
                            int64_t rows_per_vector, float eps, void* y, void* stream) {
  if (!is16(dtype)) return MFQ_EDTYPE;
  if (M <= 0 || K <= 0 || M > INT32_MAX || K > INT32_MAX) return MFQ_ESHAPE;
  if (!x || !y || (scale == nullptr) != (shift == nullptr)) return MFQ_ENULL;
  if (scale && (rows_per_vector <= 0 || M % rows_per_vector)) return MFQ_ESHAPE;
  if (!(eps >= 0.f)) return MFQ_ESHAPE;
  if (!mfq::aligned16(x) || !mfq::aligned16(y) || !mfq::aligned16(scale) || !mfq::aligned16(shift)) return MFQ_EALIGN;
  return mfq::launch_layer_norm_modulate(x, dtype, M, K, scale, shift, scale ? rows_per_vector : M, eps, y,
                                         (hipStream_t)stream);
}

int mfq_low_rank_down(const void* x, const void* at, int dtype, int64_t M, int64_t K, int64_t rank, void* t,
                      void* stream) {
  if (!is16(dtype)) return MFQ_EDTYPE;
  if (M <= 0 || K <= 0 || M > INT32_MAX || K > INT32_MAX || K % 32) return MFQ_ESHAPE;
  if (rank <= 0 || rank > 1024 || rank % 16) return MFQ_ESHAPE;
  if (M * K >= (int64_t)1 << 40) return MFQ_ESHAPE;
  if (!x || !at || !t) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(at) || !mfq::aligned16(t)) return MFQ_EALIGN;
  return mfq::launch_low_rank_down(x, dtype, M, K, at, rank, t, (hipStream_t)stream);
}

static int check_training(int dtype, int64_t rows, int64_t columns, int64_t rank, int64_t R) {
  if (!is16(dtype)) return MFQ_EDTYPE;
  if (rank <= 0 || rank > R || (R != 16 && R != 32)) return MFQ_ESHAPE;
  if (rows <= 0 || columns <= 0 || columns % 32 || rows > INT32_MAX - 64 || columns > (1 << 24)) return MFQ_ESHAPE;
  return rows * columns < (int64_t)1 << 40 ? MFQ_OK : MFQ_ESHAPE;
}

int mfq_low_rank_pack(const void* lora_a, const void* lora_b, int dtype, int64_t K, int64_t N, int64_t rank, int64_t R,
                      float scale, void* af, void* bf, void* bs, void* ap, void* stream) {
  if (int rc = check_training(dtype, 1, K, rank, R)) return rc;
  if (int rc = check_training(dtype, 1, N, rank, R)) return rc;
  if (!lora_a || !lora_b || !af || !bf || !bs) return MFQ_ENULL;
  if (!mfq::aligned16(af) || !mfq::aligned16(bf) || !mfq::aligned16(bs) || !mfq::aligned16(ap)) return MFQ_EALIGN;
  return mfq::launch_low_rank_pack(lora_a, lora_b, dtype, K, N, (int)rank, (int)R, scale, af, bf, bs, ap, (hipStream_t)stream);
}

int mfq_low_rank_forward(const void* x, const void* af, int dtype, int64_t M, int64_t K, int64_t rank, int64_t R, void* t,
                         void* tf, void* stream) {
  if (int rc = check_training(dtype, M, K, rank, R)) return rc;
  if (!x || !af || !t || !tf) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(af) || !mfq::aligned16(t) || !mfq::aligned16(tf)) return MFQ_EALIGN;
  return mfq::launch_low_rank_forward(x, dtype, M, K, af, (int)rank, (int)R, t, tf, (hipStream_t)stream);
}

int mfq_low_rank_gradient(const void* g, const void* bf, const void* tf, int dtype, int64_t M, int64_t N, int64_t rank,
                          int64_t R, float scale, void* gt, void* gtf, void* db, void* stream) {
  if (int rc = check_training(dtype, M, N, rank, R)) return rc;
  if (!g || (gt == nullptr) != (gtf == nullptr) || (gt && !bf) || (db && !tf) || (!gt && !db)) return MFQ_ENULL;
  if (!mfq::aligned16(g) || !mfq::aligned16(bf) || !mfq::aligned16(tf) || !mfq::aligned16(gt) || !mfq::aligned16(gtf) ||
      !mfq::aligned16(db))
    return MFQ_EALIGN;
  return mfq::launch_low_rank_gradient(g, dtype, M, N, bf, tf, (int)rank, (int)R, scale, gt, gtf, db, (hipStream_t)stream);
}

int mfq_low_rank_up(const void* x, const void* tf, int dtype, int64_t M, int64_t K, int64_t rank, int64_t R, void* out,
                    void* stream) {
  if (int rc = check_training(dtype, M, K, rank, R)) return rc;
  if (!x || !tf || !out) return MFQ_ENULL;
  if (!mfq::aligned16(x) || !mfq::aligned16(tf) || !mfq::aligned16(out)) return MFQ_EALIGN;
  return mfq::launch_low_rank_up(x, dtype, M, K, tf, (int)rank, (int)R, out, (hipStream_t)stream);
}

int mfq_low_rank_add(const void* t, const void* bs, int dtype, int64_t M, int64_t N, int64_t rank, void* y, int y_dtype,
                     void* stream) {
  if (!is16(dtype)) return MFQ_EDTYPE;
  if (y_dtype != dtype && y_dtype != MFQ_F32) return MFQ_EDTYPE;
  if (M <= 0 || N <= 0 || M > INT32_MAX || N > INT32_MAX) return MFQ_ESHAPE;
  if (rank <= 0 || rank > 1024 || rank % 16) return MFQ_ESHAPE;
  if (!t || !bs || !y) return MFQ_ENULL;
  if (!mfq::aligned16(t) || !mfq::aligned16(bs)) return MFQ_EALIGN;
  mfq::LowRank low_rank;
  low_rank.t = t;
  low_rank.bs = bs;
  low_rank.R = (int)rank;
  return mfq::launch_low_rank_add(dtype, low_rank, M, N, y, y_dtype, (hipStream_t)stream);
}

int mfq_rotary_tables(const int32_t* positions, int64_t n, int axes, int pairs, const double* frequencies, const uint8_t* axis, float factor,
                      float* cos, float* sin, void* stream) {
  if (n <= 0 || axes <= 0 || axes > 255 || pairs <= 0 || pairs > MFQ_ROTARY_MAX_PAIRS || n > ((int64_t)1 << 31)) return MFQ_ESHAPE;
  if (n * pairs > ((int64_t)1 << 38)) return MFQ_ESHAPE;
  if (!positions || !frequencies || !axis || !cos || !sin) return MFQ_ENULL;
  if (!(std::fabs(factor) <= std::numeric_limits<float>::max())) return MFQ_ESHAPE;
  for (int i = 0; i < pairs; ++i)
    if (axis[i] >= axes || !(std::fabs(frequencies[i]) <= 4.0)) return MFQ_ESHAPE;
  return mfq::launch_rotary_tables(positions, n, axes, pairs, frequencies, axis, factor, cos, sin, (hipStream_t)stream);
}

static int check_rotary(const mfq_rotary_args* a, bool backward, bool* wide) {
  if (!a) return MFQ_ENULL;
  if (!known(a->dtype)) return MFQ_EDTYPE;
  if (a->layout != MFQ_ROTARY_HALF && a->layout != MFQ_ROTARY_INTERLEAVED) return MFQ_ESHAPE;
  if (a->dim <= 0 || a->dim > 512 || a->dim % 2 || a->rotated < 0 || a->rotated > a->dim || a->rotated % 2) return MFQ_ESHAPE;
  if (a->batch <= 0 || a->tokens <= 0 || a->batch > INT32_MAX || a->tokens > INT32_MAX || a->batch * a->tokens > ((int64_t)1 << 40)) return MFQ_ESHAPE;
  if (a->table_rows <= 0 || a->table_rows > INT32_MAX || a->position_batch < 0) return MFQ_ESHAPE;
  if (a->q.heads <= 0 || a->k.heads < 0 || a->q.heads > 65536 || a->k.heads > 65536) return MFQ_ESHAPE;
  if (a->batch * a->tokens * a->q.heads >= INT32_MAX || a->batch * a->tokens * a->k.heads >= INT32_MAX) return MFQ_ESHAPE;
  if (!(a->eps >= 0.f)) return MFQ_ESHAPE;
  if (a->rotated && (!a->cos || !a->sin)) return MFQ_ENULL;
  const int64_t per16 = a->dtype == MFQ_F32 ? 4 : 8;
  *wide = mfq::aligned16(a->cos) && mfq::aligned16(a->sin);
  for (const mfq_rotary_tensor* t : {&a->q, &a->k}) {
    if (!t->heads) {
      if (backward && t->dweight) return MFQ_ESHAPE;  // no rows to sum over
      continue;
    }
    if ((!backward || t->weight) && !t->x) return MFQ_ENULL;
    if (!backward && !t->out) return MFQ_ENULL;
    if (backward && !t->dy) return MFQ_ENULL;
    if (t->dweight && !t->weight) return MFQ_ENULL;
    for (int i = 0; i < 3; ++i) {
      if (t->x_stride[i] < 0 || t->dy_stride[i] < 0) return MFQ_ESHAPE;
      *wide = *wide && t->x_stride[i] % per16 == 0 && (!backward || t->dy_stride[i] % per16 == 0);
    }
    *wide = *wide && mfq::aligned16(t->x) && mfq::aligned16(t->out) && mfq::aligned16(t->weight) && (!backward || mfq::aligned16(t->dy));
    *wide = *wide && a->dim % per16 == 0;  // rows of the result
  }
  return MFQ_OK;
}

size_t mfq_rotary_workspace_bytes(const mfq_rotary_args* args) { return args ? mfq::rotary_workspace_bytes(*args) : 0; }

int mfq_rotary(const mfq_rotary_args* args, void* stream) {
  bool wide = false;
  if (int rc = check_rotary(args, false, &wide)) return rc;
  return mfq::launch_rotary(*args, wide, false, nullptr, (hipStream_t)stream);
}

int mfq_rotary_backward(const mfq_rotary_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  bool wide = false;
  if (int rc = check_rotary(args, true, &wide)) return rc;
  const size_t need = mfq::rotary_workspace_bytes(*args);
  if (need && !workspace) return MFQ_ENULL;
  if (need > workspace_bytes) return MFQ_ESCRATCH;
  if (need && !mfq::aligned16(workspace)) return MFQ_EALIGN;
  return mfq::launch_rotary(*args, wide, true, static_cast<float*>(workspace), (hipStream_t)stream);
}

static int attention_call(const mfq_attention_args* a, bool backward, mfq::AttentionCall* c) {
  if (!a) return MFQ_ENULL;
  if (!is16(a->dtype)) return MFQ_EDTYPE;
  if (a->dim <= 0 || a->dim > 256 || a->dim % 8) return MFQ_ESHAPE;
  if (a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads || a->heads > 65536) return MFQ_ESHAPE;
  if (a->batch <= 0 || a->q_tokens <= 0 || a->k_tokens <= 0 || a->batch > (1 << 24)) return MFQ_ESHAPE;
  if (a->q_tokens > (1 << 30) || a->k_tokens > (1 << 30) || a->q_tokens * a->heads > (1 << 30)) return MFQ_ESHAPE;
  if (!(a->scale > 0.f) || a->scale > 1e30f) return MFQ_ESHAPE;
  if ((a->q_offsets == nullptr) != (a->k_offsets == nullptr)) return MFQ_ENULL;
  if (a->q_offsets && (a->q_lengths || a->k_lengths)) return MFQ_EUNSUPPORTED;
  struct In {
    const mfq_attention_tensor* t;
    mfq::AttentionTensor* to;
  } in[] = {{&a->q, &c->q}, {&a->k, &c->k}, {&a->v, &c->v}, {&a->y, &c->y}, {&a->dy, &c->dy}};
  for (int i = 0; i < (backward ? 5 : 3); ++i) {
    const mfq_attention_tensor& t = *in[i].t;
    if (!t.p) return MFQ_ENULL;
    if (!mfq::aligned16(t.p)) return MFQ_EALIGN;
    for (int64_t s : t.stride)
      if (s < 0) return MFQ_ESHAPE;
      else if (s % 8) return MFQ_EALIGN;
    if (t.stride[1] >= (1 << 24)) return MFQ_ESHAPE;
    *in[i].to = {static_cast<const uint16_t*>(t.p), t.stride[0], t.stride[1], t.stride[2]};
  }
  if (!backward && !a->out) return MFQ_ENULL;
  if (backward && (!a->lse || !a->delta || (!a->dq && !a->dk && !a->dv))) return MFQ_ENULL;
  for (const void* p : {(const void*)a->out, (const void*)a->rest, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
    if (!mfq::aligned16(p)) return MFQ_EALIGN;
  c->out = static_cast<uint16_t*>(a->out);
  c->rest = static_cast<uint16_t*>(a->rest);
  c->dq = static_cast<uint16_t*>(a->dq);
  c->dk = static_cast<uint16_t*>(a->dk);
  c->dv = static_cast<uint16_t*>(a->dv);
  c->lse = a->lse;
  c->delta = a->delta;
  c->q_offsets = a->q_offsets;
  c->k_offsets = a->k_offsets;
  c->q_lengths = a->q_lengths;
  c->k_lengths = a->k_lengths;
  c->batch = (int)a->batch;
  c->heads = (int)a->heads;
  c->kv_heads = (int)a->kv_heads;
  c->dim = a->dim;
  c->q_tokens = (int)a->q_tokens;
  c->k_tokens = (int)a->k_tokens;
  c->causal = a->causal != 0;
  c->scale = a->scale;
  return MFQ_OK;
}

size_t mfq_attention_workspace_bytes(const mfq_attention_args* args) {
  mfq::AttentionCall c;
  if (attention_call(args, false, &c) != MFQ_OK) return 0;
  return mfq::attention_split_bytes(c, mfq::attention_splits(c));
}

int mfq_attention_ranges(const mfq_attention_args* args) {
  mfq::AttentionCall c;
  if (int rc = attention_call(args, false, &c)) return rc;
  return mfq::attention_splits(c);
}

size_t mfq_attention_backward_workspace_bytes(const mfq_attention_args* args) {
  mfq::AttentionCall c;
  if (attention_call(args, true, &c) != MFQ_OK) return 0;
  return mfq::attention_backward_bytes(c, mfq::attention_backward_parts(c));
}

int mfq_attention(const mfq_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  mfq::AttentionCall c;
  if (int rc = attention_call(args, false, &c)) return rc;
  const int splits = mfq::attention_splits(c);
  if (!splits) return mfq::launch_attention(args->dtype, c, (hipStream_t)stream);
  const size_t need = mfq::attention_split_bytes(c, splits);
  if (need && !workspace) return MFQ_ENULL;
  if (need > workspace_bytes) return MFQ_ESCRATCH;
  if (need && !mfq::aligned16(workspace)) return MFQ_EALIGN;
  return mfq::launch_attention_split(args->dtype, c, splits, workspace, (hipStream_t)stream);
}

int mfq_attention_backward(const mfq_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  mfq::AttentionCall c;
  if (int rc = attention_call(args, true, &c)) return rc;
  const int parts = mfq::attention_backward_parts(c);
  const size_t need = mfq::attention_backward_bytes(c, parts);
  if (need && !workspace) return MFQ_ENULL;
  if (need > workspace_bytes) return MFQ_ESCRATCH;
  if (need && !mfq::aligned16(workspace)) return MFQ_EALIGN;
  return mfq::launch_attention_backward(args->dtype, c, parts, workspace, (hipStream_t)stream);
}

// Rows of `count` x `columns` at `stride`, and whether a call loads them 16 bytes at a time
static int check_rows(const void* p, int64_t stride, int64_t rows, int64_t columns, int64_t per16, bool* wide) {
  if (!p) return MFQ_ENULL;
  if (stride < 0 || (rows > 1 && stride > ((int64_t)1 << 40))) return MFQ_ESHAPE;
  *wide = *wide && mfq::aligned16(p) && columns % per16 == 0 && (rows == 1 || stride % per16 == 0);
  return MFQ_OK;
}

static int rms_norm_call(const mfq_rms_norm_args* a, bool backward, bool norm, mfq::RowsCall* c, bool* wide) {
  if (!a) return MFQ_ENULL;
  if (!known(a->dtype)) return MFQ_EDTYPE;
  if (a->rows <= 0 || a->columns <= 0 || a->rows > INT32_MAX || a->columns > (1 << 28) || a->rows * a->columns > ((int64_t)1 << 46)) return MFQ_ESHAPE;
  if (norm && !(a->eps >= 0.f && a->eps <= std::numeric_limits<float>::max())) return MFQ_ESHAPE;
  const int64_t per16 = a->dtype == MFQ_F32 ? 4 : 8;
  *wide = mfq::aligned16(a->weight);
  if (int rc = check_rows(a->x, a->x_stride, a->rows, a->columns, per16, wide)) return rc;
  if (backward) {
    if (int rc = check_rows(a->dy, a->dy_stride, a->rows, a->columns, per16, wide)) return rc;
    if (a->dsum)
      if (int rc = check_rows(a->dsum, a->dsum_stride, a->rows, a->columns, per16, wide)) return rc;
    if (!a->dx && !a->dweight) return MFQ_ENULL;
    if (a->dweight && !a->weight) return MFQ_ENULL;
    *wide = *wide && mfq::aligned16(a->dx);
  } else {
    if (a->residual) {
      if (int rc = check_rows(a->residual, a->residual_stride, a->rows, a->columns, per16, wide)) return rc;
      if (!a->sum) return MFQ_ENULL;
      *wide = *wide && mfq::aligned16(a->sum);
    }
    if (a->codes) {
      if (a->y) return MFQ_EUNSUPPORTED;  // one of the two
      if (!a->scales) return MFQ_ENULL;
      if (a->rows > 1 && a->code_stride < a->columns) return MFQ_ESHAPE;
      *wide = *wide && reinterpret_cast<uintptr_t>(a->codes) % per16 == 0 && (a->rows == 1 || a->code_stride % per16 == 0);
    } else {
      if (!a->y) return MFQ_ENULL;
      *wide = *wide && mfq::aligned16(a->y);
    }
  }
  *c = {};
  c->x = a->x;
  c->residual = a->residual;
  c->weight = a->weight;
  c->dy = a->dy;
  c->dsum = a->dsum;
  c->y = a->y;
  c->sum = a->sum;
  c->dx = a->dx;
  c->dweight = a->dweight;
  c->codes = backward ? nullptr : a->codes;
  c->scales = a->scales;
  c->rows = a->rows;
  c->columns = a->columns;
  c->x_stride = a->x_stride;
  c->residual_stride = a->residual_stride;
  c->dy_stride = a->dy_stride;
  c->dsum_stride = a->dsum_stride;
  c->code_stride = a->code_stride;
  c->eps = a->eps;
  c->norm = norm;
  return MFQ_OK;
}

size_t mfq_rms_norm_workspace_bytes(const mfq_rms_norm_args* args) {
  if (!args || !args->dweight || args->rows <= 0 || args->columns <= 0) return 0;
  return mfq::rows_workspace_bytes(args->rows, args->columns);
}

int mfq_rms_norm(const mfq_rms_norm_args* args, void* stream) {
  mfq::RowsCall c;
  bool wide = false;
  if (int rc = rms_norm_call(args, false, true, &c, &wide)) return rc;
  return mfq::launch_rows(args->dtype, c, wide, false, (hipStream_t)stream);
}

int mfq_rms_norm_backward(const mfq_rms_norm_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  mfq::RowsCall c;
  bool wide = false;
  if (int rc = rms_norm_call(args, true, true, &c, &wide)) return rc;
  const size_t need = mfq_rms_norm_workspace_bytes(args);
  if (need && !workspace) return MFQ_ENULL;
  if (need > workspace_bytes) return MFQ_ESCRATCH;
  if (need && !mfq::aligned16(workspace)) return MFQ_EALIGN;
  c.parts = need ? static_cast<float*>(workspace) : nullptr;
  return mfq::launch_rows(args->dtype, c, wide, true, (hipStream_t)stream);
}

int mfq_int8_quantize(const void* x, int dtype, int64_t rows, int64_t columns, int64_t x_stride, int8_t* codes, int64_t code_stride,
                      float* scales, void* stream) {
  if (!codes) return known(dtype) ? MFQ_ENULL : MFQ_EDTYPE;
  mfq_rms_norm_args a = {};
  a.dtype = dtype;
  a.rows = rows;
  a.columns = columns;
  a.x = x;
  a.x_stride = x_stride;
  a.codes = codes;
  a.code_stride = code_stride;
  a.scales = scales;
  mfq::RowsCall c;
  bool wide = false;
  if (int rc = rms_norm_call(&a, false, false, &c, &wide)) return rc;
  return mfq::launch_rows(dtype, c, wide, false, (hipStream_t)stream);
}

int mfq_int8_dequantize(const int8_t* codes, int64_t code_stride, const float* scales, int64_t rows, int64_t columns, void* out, int dtype,
                        void* stream) {
  if (!known(dtype)) return MFQ_EDTYPE;
  if (rows <= 0 || columns <= 0 || rows > INT32_MAX || columns > (1 << 28) || rows * columns > ((int64_t)1 << 46)) return MFQ_ESHAPE;
  if (!codes || !scales || !out) return MFQ_ENULL;
  if (code_stride < 0 || (rows > 1 && code_stride > ((int64_t)1 << 40))) return MFQ_ESHAPE;
  return mfq::launch_rows_values(codes, code_stride, scales, rows, columns, dtype, out, (hipStream_t)stream);
}

static int check_int8(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 || K >= (1 << 17) || M > (1 << 30) || N > (1 << 30)) return MFQ_ESHAPE;
  if (M * N > ((int64_t)1 << 42)) return MFQ_ESHAPE;
  return MFQ_OK;
}

int mfq_int8_matmul_plan(int64_t M, int64_t N, int64_t K, int dtype, int* k_ranges, int* tile_rows, int* tile_columns) {
  if (!known(dtype)) return MFQ_EDTYPE;
  if (int rc = check_int8(M, N, K)) return rc;
  const mfq::Int8Plan p = mfq::int8_plan(dtype, M, N, K);
  if (k_ranges) *k_ranges = p.splits;
  if (tile_rows) *tile_rows = p.tiles.rows;
  if (tile_columns) *tile_columns = p.tiles.columns;
  return p.kernel;
}

size_t mfq_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
  if (!known(dtype) || check_int8(M, N, K) != MFQ_OK) return 0;
  return mfq::int8_workspace_bytes(mfq::int8_plan(dtype, M, N, K), M, N);
}

int mfq_int8_matmul(const int8_t* x, int64_t x_stride, const float* x_scales, const int8_t* w, int64_t w_stride, const float* w_scales,
                    const void* bias, int64_t M, int64_t N, int64_t K, void* y, int dtype, void* workspace, size_t workspace_bytes,
                    void* stream) {
  if (!known(dtype)) return MFQ_EDTYPE;
  if (int rc = check_int8(M, N, K)) return rc;
  if (!x || !x_scales || !w || !w_scales || !y) return MFQ_ENULL;
  if (x_stride < 0 || w_stride < 0 || x_stride >= (1 << 20) || w_stride >= (1 << 20)) return MFQ_ESHAPE;
  if (!mfq::aligned16(x) || !mfq::aligned16(w) || !mfq::aligned16(y) || x_stride % 16 || w_stride % 16) return MFQ_EALIGN;
  const mfq::Int8Plan p = mfq::int8_plan(dtype, M, N, K);
  const size_t need = mfq::int8_workspace_bytes(p, M, N);
  if (need && !workspace) return MFQ_ENULL;
  if (need > workspace_bytes) return MFQ_ESCRATCH;
  if (need && !mfq::aligned16(workspace)) return MFQ_EALIGN;
  const mfq::Int8Call c = {x, w, x_scales, w_scales, bias, y, M, N, K, N, x_stride, w_stride};
  return mfq::launch_int8_matmul(dtype, c, p, workspace, (hipStream_t)stream);
}

}  // extern "C"
