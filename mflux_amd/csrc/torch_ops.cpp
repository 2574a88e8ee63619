// torch.ops.mfq.*: the PyTorch-ROCm face of libmfq.  Each op checks its tensors,
// allocates the outputs from torch's caching allocator on the inputs' device,
// and calls the C ABI of include/mfq.h on torch's current HIP stream: no device
// synchronisation, no state of its own.  (PyTorch-ROCm presents its HIP devices
// under the "cuda" device type, hence the ...MasqueradingAsCUDA guard and the
// CUDA dispatch key.)  Only the HIP dispatch key is
// registered, so a CPU tensor is refused by the dispatcher (there is no CPU
// implementation to fall back to).  mflux_amd.core calls these ops; the error
// texts a user sees for bad arguments are produced there, in MLX's wording.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <memory>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/mfq.h"

namespace {

using at::Tensor;

int dtype_code(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return MFQ_F32;
    case at::kHalf: return MFQ_F16;
    case at::kBFloat16: return MFQ_BF16;
    default: TORCH_CHECK(false, "mfq: ", what, " must be float32, float16 or bfloat16, got ", t);
  }
}

void check_status(const char* fn, int rc) {
  TORCH_CHECK(rc == MFQ_OK, fn, " failed: ", mfq_strerror(rc), " (status ", rc, ")");
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check_packed(const Tensor& wq, const Tensor& scales, const Tensor& biases) {
  TORCH_CHECK(wq.scalar_type() == at::kUInt32, "mfq: the packed weight must be uint32, got ", wq.scalar_type());
  TORCH_CHECK(wq.dim() == 2 && scales.dim() == 2 && biases.dim() == 2, "mfq: packed weight, scales and biases are 2-D");
  TORCH_CHECK(scales.scalar_type() == biases.scalar_type() && scales.sizes() == biases.sizes(),
              "mfq: scales and biases must agree in dtype and shape");
  TORCH_CHECK(wq.is_contiguous() && scales.is_contiguous() && biases.is_contiguous(), "mfq: operands must be contiguous");
  TORCH_CHECK(scales.device() == wq.device() && biases.device() == wq.device(), "mfq: operands on different devices");
}

std::tuple<Tensor, Tensor, Tensor> quantize_affine(const Tensor& w, int64_t group_size, int64_t bits) {
  TORCH_CHECK(w.dim() == 2 && w.is_contiguous(), "mfq::quantize_affine: w must be a contiguous matrix");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(w.device());
  const int64_t rows = w.size(0), K = w.size(1);
  TORCH_CHECK(group_size > 0 && K % group_size == 0 && (K * bits) % 32 == 0, "mfq::quantize_affine: bad K");
  Tensor wq = at::empty({rows, K * bits / 32}, w.options().dtype(at::kUInt32));
  Tensor scales = at::empty({rows, K / group_size}, w.options());
  Tensor biases = at::empty_like(scales);
  if (rows == 0) return {wq, scales, biases};
  check_status("mfq_quantize_affine",
               mfq_quantize_affine(w.data_ptr(), dtype_code(w.scalar_type(), "w"), rows, K, (int)group_size, (int)bits,
                                   static_cast<uint32_t*>(wq.data_ptr()), scales.data_ptr(), biases.data_ptr(),
                                   stream_of(w)));
  return {wq, scales, biases};
}

Tensor dequantize_affine(const Tensor& wq, const Tensor& scales, const Tensor& biases, int64_t group_size, int64_t bits,
                         at::ScalarType out_dtype) {
  check_packed(wq, scales, biases);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(wq.device());
  const int64_t rows = wq.size(0), K = wq.size(1) * 32 / bits;
  Tensor out = at::empty({rows, K}, scales.options().dtype(out_dtype));
  if (rows == 0) return out;
  check_status("mfq_dequantize_affine",
               mfq_dequantize_affine(static_cast<const uint32_t*>(wq.data_ptr()), scales.data_ptr(), biases.data_ptr(),
                                     dtype_code(scales.scalar_type(), "scales"), rows, K, (int)group_size, (int)bits,
                                     out.data_ptr(), dtype_code(out_dtype, "the output"), stream_of(wq)));
  return out;
}

Tensor dequantize_rows(const Tensor& wq, const Tensor& scales, const Tensor& biases, const Tensor& indices,
                       int64_t group_size, int64_t bits, at::ScalarType out_dtype) {
  check_packed(wq, scales, biases);
  TORCH_CHECK(indices.scalar_type() == at::kLong && indices.dim() == 1 && indices.is_contiguous() &&
                  indices.device() == wq.device(),
              "mfq::dequantize_rows: indices must be a contiguous int64 vector on the table's device");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(wq.device());
  const int64_t K = wq.size(1) * 32 / bits;
  Tensor out = at::empty({indices.size(0), K}, scales.options().dtype(out_dtype));
  if (indices.size(0) == 0) return out;
  check_status("mfq_dequantize_rows",
               mfq_dequantize_rows(static_cast<const uint32_t*>(wq.data_ptr()), scales.data_ptr(), biases.data_ptr(),
                                   dtype_code(scales.scalar_type(), "scales"), indices.data_ptr<int64_t>(),
                                   indices.size(0), wq.size(0), K, (int)group_size, (int)bits, out.data_ptr(),
                                   dtype_code(out_dtype, "the output"), stream_of(wq)));
  return out;
}

struct Matmul {
  int64_t M, K, N;
  int sb;
  const void* bias;
};

// common checks of the products; x is [M, K] in the scales' dtype
Matmul check_matmul(const char* fn, const Tensor& x, const Tensor& wq, const Tensor& scales, const Tensor& biases,
                    const c10::optional<Tensor>& bias, int64_t bits) {
  check_packed(wq, scales, biases);
  TORCH_CHECK(x.dim() == 2 && x.is_contiguous() && x.device() == wq.device(), fn, ": x must be a contiguous matrix on ",
              wq.device());
  TORCH_CHECK(x.scalar_type() == scales.scalar_type(), fn, ": x and scales must share a 16-bit dtype");
  Matmul m{x.size(0), wq.size(1) * 32 / bits, wq.size(0), dtype_code(scales.scalar_type(), "scales"), nullptr};
  TORCH_CHECK(x.size(1) == m.K, fn, ": x has ", x.size(1), " columns, the weight ", m.K);
  if (bias.has_value()) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == m.N && bias->scalar_type() == scales.scalar_type() &&
                    bias->is_contiguous() && bias->device() == wq.device(),
                fn, ": bias must be a contiguous [N] vector of the scales' dtype");
    m.bias = bias->data_ptr();
  }
  return m;
}

// y = x @ dequantize(wq)^T (+ t @ bs^T) (+ bias); the float32 planes of a K
// split come from torch's allocator on the current stream, so their reuse is
// ordered after this call.  `ok` is false (and y undefined) when the library
// has no kernel for the combination (MFQ_EUNSUPPORTED).
std::tuple<Tensor, bool> qmm_t(const Tensor& x, const Tensor& wq, const Tensor& scales, const Tensor& biases,
             const c10::optional<Tensor>& bias, int64_t group_size, int64_t bits, at::ScalarType out_dtype,
             const c10::optional<Tensor>& lr_t, const c10::optional<Tensor>& lr_bs) {
  const Matmul m = check_matmul("mfq::qmm_t", x, wq, scales, biases, bias, bits);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor y = at::empty({m.M, m.N}, x.options().dtype(out_dtype));
  if (m.M == 0) return {y, true};
  const void *t = nullptr, *bs = nullptr;
  int64_t rank = 0;
  if (lr_t.has_value() || lr_bs.has_value()) {
    TORCH_CHECK(lr_t.has_value() && lr_bs.has_value(), "mfq::qmm_t: the low-rank update needs both t and bs");
    rank = lr_bs->size(1);
    TORCH_CHECK(lr_t->dim() == 2 && lr_bs->dim() == 2 && lr_t->size(0) == m.M && lr_t->size(1) == rank &&
                    lr_bs->size(0) == m.N && lr_t->scalar_type() == x.scalar_type() &&
                    lr_bs->scalar_type() == x.scalar_type() && lr_t->is_contiguous() && lr_bs->is_contiguous(),
                "mfq::qmm_t: the low-rank update is t [M, R], bs [N, R], contiguous, in x's dtype");
    t = lr_t->data_ptr();
    bs = lr_bs->data_ptr();
  }
  size_t ws_bytes = 0;
  if (rank && out_dtype == at::kFloat)  // (an update with a float32 result: the kernels that dequantise in the GEMM)
    ws_bytes = mfq_qmm_t_workspace_bytes(m.M, m.K, m.N, (int)group_size, (int)bits);
  else
    mfq_qmm_t_plan(m.M, m.K, m.N, (int)group_size, (int)bits, 0, nullptr, nullptr, nullptr, &ws_bytes);
  Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, x.options().dtype(at::kByte));
  const int rc = mfq_qmm_t_low_rank(x.data_ptr(), m.sb, m.M, m.K, static_cast<const uint32_t*>(wq.data_ptr()),
                                    scales.data_ptr(), biases.data_ptr(), m.sb, m.bias, m.N, (int)group_size, (int)bits,
                                    t, bs, rank, y.data_ptr(), dtype_code(out_dtype, "the output"),
                                    ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, stream_of(x));
  if (rc == MFQ_EUNSUPPORTED) return {y, false};
  check_status("mfq_qmm_t_low_rank", rc);
  return {y, true};
}

// qmm_t with an epilogue of include/mfq.h's mfq_qmm_t_epilogue (1: gelu_approx from column act_from on,
// 2: residual + gate * y, 3: SwiGLU of gate / up rows stacked in blocks of 32, y is [M, N/2]); `ok` is false
// (and y undefined) when no kernel fuses it for the shape
std::tuple<Tensor, bool> qmm_t_epilogue(const Tensor& x, const Tensor& wq, const Tensor& scales, const Tensor& biases,
                                        const c10::optional<Tensor>& bias, int64_t group_size, int64_t bits,
                                        int64_t epilogue, const c10::optional<Tensor>& gate,
                                        const c10::optional<Tensor>& residual, int64_t act_from) {
  const Matmul m = check_matmul("mfq::qmm_t_epilogue", x, wq, scales, biases, bias, bits);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const void *gate_p = nullptr, *res_p = nullptr;
  if (epilogue == MFQ_EPILOGUE_GATE_RESIDUAL) {
    TORCH_CHECK(gate.has_value() && residual.has_value(), "mfq::qmm_t_epilogue: gate and residual are required");
    TORCH_CHECK(gate->dim() == 1 && gate->size(0) == m.N && gate->scalar_type() == x.scalar_type() &&
                    gate->is_contiguous() && gate->device() == x.device(),
                "mfq::qmm_t_epilogue: gate must be a contiguous [N] vector of x's dtype");
    TORCH_CHECK(residual->dim() == 2 && residual->size(0) == m.M && residual->size(1) == m.N &&
                    residual->scalar_type() == x.scalar_type() && residual->is_contiguous() &&
                    residual->device() == x.device(),
                "mfq::qmm_t_epilogue: residual must be a contiguous [M, N] matrix of x's dtype");
    gate_p = gate->data_ptr();
    res_p = residual->data_ptr();
  }
  const int64_t n_out = epilogue == MFQ_EPILOGUE_SWIGLU ? m.N / 2 : m.N;
  Tensor y = at::empty({m.M, n_out}, x.options());
  if (m.M == 0) return {y, true};
  size_t ws_bytes = 0;
  mfq_qmm_t_plan(m.M, m.K, m.N, (int)group_size, (int)bits, (int)epilogue, nullptr, nullptr, nullptr, &ws_bytes);
  Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, x.options().dtype(at::kByte));
  const int rc = mfq_qmm_t_epilogue(x.data_ptr(), m.sb, m.M, m.K, static_cast<const uint32_t*>(wq.data_ptr()),
                                    scales.data_ptr(), biases.data_ptr(), m.sb, m.bias, m.N, (int)group_size,
                                    (int)bits, (int)epilogue, gate_p, res_p, act_from, y.data_ptr(), m.sb,
                                    ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, stream_of(x));
  if (rc == MFQ_EUNSUPPORTED) return {y, false};
  check_status("mfq_qmm_t_epilogue", rc);
  return {y, true};
}

// y[M, K] = x[M, N] @ dequantize(wq[N, K]) (+ t @ bs^T); `ok` is false when N is not a multiple of 8
std::tuple<Tensor, bool> qmm_n(const Tensor& x, const Tensor& wq, const Tensor& scales, const Tensor& biases,
                               int64_t group_size, int64_t bits, at::ScalarType out_dtype,
                               const c10::optional<Tensor>& lr_t, const c10::optional<Tensor>& lr_bs) {
  check_packed(wq, scales, biases);
  TORCH_CHECK(x.dim() == 2 && x.is_contiguous() && x.device() == wq.device() && x.size(1) == wq.size(0) &&
                  x.scalar_type() == scales.scalar_type(),
              "mfq::qmm_n: x must be a contiguous [M, N] matrix of the scales' dtype on the weight's device");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t M = x.size(0), N = wq.size(0), K = wq.size(1) * 32 / bits;
  Tensor y = at::empty({M, K}, x.options().dtype(out_dtype));
  if (M == 0) return {y, true};
  const int sb = dtype_code(scales.scalar_type(), "scales");
  const void *t = nullptr, *bs = nullptr;
  int64_t rank = 0;
  if (lr_t.has_value() || lr_bs.has_value()) {
    TORCH_CHECK(lr_t.has_value() && lr_bs.has_value(), "mfq::qmm_n: the low-rank update needs both t and bs");
    TORCH_CHECK(lr_t->dim() == 2 && lr_bs->dim() == 2 && lr_t->size(0) == M && lr_bs->size(0) == K &&
                    lr_t->size(1) == lr_bs->size(1) && lr_t->scalar_type() == x.scalar_type() &&
                    lr_bs->scalar_type() == x.scalar_type() && lr_t->is_contiguous() && lr_bs->is_contiguous() &&
                    lr_t->device() == x.device() && lr_bs->device() == x.device(),
                "mfq::qmm_n: the low-rank update is t [M, R], bs [K, R], contiguous, in x's dtype");
    rank = lr_bs->size(1);
    t = lr_t->data_ptr();
    bs = lr_bs->data_ptr();
  }
  // the transposed 16-bit copy of the two-kernel path (and the planes of its K cut), where that is used
  const size_t ws_bytes = mfq_qmm_n_workspace_bytes(M, N, K, (int)group_size, (int)bits);
  Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, x.options().dtype(at::kByte));
  const int rc = mfq_qmm_n_low_rank(x.data_ptr(), sb, M, N, static_cast<const uint32_t*>(wq.data_ptr()),
                                    scales.data_ptr(), biases.data_ptr(), sb, K, (int)group_size, (int)bits, t, bs, rank,
                                    y.data_ptr(), dtype_code(out_dtype, "the output"),
                                    ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, stream_of(x));
  if (rc == MFQ_EUNSUPPORTED) return {y, false};
  check_status("mfq_qmm_n", rc);
  return {y, true};
}

// one to four rows of silu(x) against the weights in one kernel; `ok` is false
// (and y undefined) when no fused kernel takes the shape
std::tuple<Tensor, bool> qmv_silu(const Tensor& x, const Tensor& wq, const Tensor& scales, const Tensor& biases,
                                  const c10::optional<Tensor>& bias, int64_t group_size, int64_t bits) {
  const Matmul m = check_matmul("mfq::qmv_silu", x, wq, scales, biases, bias, bits);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor y = at::empty({m.M, m.N}, x.options());
  const int rc = mfq_qmv_silu(x.data_ptr(), m.sb, m.M, m.K, static_cast<const uint32_t*>(wq.data_ptr()),
                              scales.data_ptr(), biases.data_ptr(), m.sb, m.bias, m.N, (int)group_size, (int)bits,
                              y.data_ptr(), m.sb, stream_of(x));
  if (rc == MFQ_EUNSUPPORTED) return {y, false};
  check_status("mfq_qmv_silu", rc);
  return {y, true};
}

// LayerNorm(x, eps) * (1 + scale) + shift over the rows of x [M, K]; scale and shift [B, K] with M % B == 0 (or
// neither); `ok` is false when the rows are too long for the kernel
std::tuple<Tensor, bool> layer_norm_modulate(const Tensor& x, const c10::optional<Tensor>& scale,
                                             const c10::optional<Tensor>& shift, double eps) {
  TORCH_CHECK(x.dim() == 2 && x.is_contiguous(), "mfq::layer_norm_modulate: x must be a contiguous matrix");
  TORCH_CHECK(scale.has_value() == shift.has_value(), "mfq::layer_norm_modulate: scale and shift come together");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t M = x.size(0), K = x.size(1);
  int64_t rows_per_vector = M;
  const void *sc = nullptr, *sh = nullptr;
  if (scale.has_value()) {
    TORCH_CHECK(scale->dim() == 2 && scale->size(1) == K && scale->sizes() == shift->sizes() && scale->size(0) > 0 &&
                    M % scale->size(0) == 0 && scale->scalar_type() == x.scalar_type() &&
                    shift->scalar_type() == x.scalar_type() && scale->is_contiguous() && shift->is_contiguous() &&
                    scale->device() == x.device() && shift->device() == x.device(),
                "mfq::layer_norm_modulate: scale and shift must be contiguous [B, K] matrices of x's dtype, M % B == 0");
    rows_per_vector = M / scale->size(0);
    sc = scale->data_ptr();
    sh = shift->data_ptr();
  }
  Tensor y = at::empty_like(x);
  if (M == 0) return {y, true};
  const int rc = mfq_layer_norm_modulate(x.data_ptr(), dtype_code(x.scalar_type(), "x"), M, K, sc, sh, rows_per_vector,
                                         (float)eps, y.data_ptr(), stream_of(x));
  if (rc == MFQ_EUNSUPPORTED) return {y, false};
  check_status("mfq_layer_norm_modulate", rc);
  return {y, true};
}

// t = x @ A, A in the fragment order of mfq_low_rank_down ([R/16, K/32, 4, 16, 8])
Tensor low_rank_down(const Tensor& x, const Tensor& af) {
  TORCH_CHECK(x.dim() == 2 && af.dim() == 5 && x.is_contiguous() && af.is_contiguous() && af.size(2) == 4 &&
                  af.size(3) == 16 && af.size(4) == 8 && x.size(1) == 32 * af.size(1) &&
                  x.scalar_type() == af.scalar_type(),
              "mfq::low_rank_down: x [M, K], af [R/16, K/32, 4, 16, 8], contiguous, of one 16-bit type");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t R = 16 * af.size(0);
  Tensor t = at::empty({x.size(0), R}, x.options());
  check_status("mfq_low_rank_down", mfq_low_rank_down(x.data_ptr(), af.data_ptr(), dtype_code(x.scalar_type(), "x"),
                                                      x.size(0), x.size(1), R, t.data_ptr(), stream_of(x)));
  return t;
}

// ---- a trainable adapter's products (include/mfq.h, mfq_low_rank_pack and what follows it)
int64_t training_rank(int64_t rank) { return rank <= 16 ? 16 : 32; }

void check_factor(const char* fn, const Tensor& t, int64_t rows, int64_t columns, const Tensor& like) {
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == columns && t.is_contiguous() &&
                  t.scalar_type() == like.scalar_type() && t.device() == like.device(),
              fn, ": expected a contiguous [", rows, ", ", columns, "] matrix of ", like.scalar_type(), " on ", like.device());
}

void check_fragments(const char* fn, const Tensor& t, int64_t steps, const Tensor& like) {
  TORCH_CHECK(t.dim() == 5 && t.size(1) == steps && t.size(2) == 4 && t.size(3) == 16 && t.size(4) == 8 && t.is_contiguous() &&
                  t.scalar_type() == like.scalar_type() && t.device() == like.device(),
              fn, ": expected fragments [R/16, ", steps, ", 4, 16, 8] of ", like.scalar_type(), " on ", like.device());
}

// lora_A [K, rank], lora_B [rank, N] -> their fragments, scale lora_B^T [N, R] and lora_A [K, R]: new tensors all, also at the
// ranks where lora_A needs no padding, so that backward sees the factors that forward saw, whatever is written to them between
std::tuple<Tensor, Tensor, Tensor, Tensor> low_rank_pack(const Tensor& a, const Tensor& b, double scale) {
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2, "mfq::low_rank_pack: lora_A [K, rank], lora_B [rank, N]");
  const int64_t K = a.size(0), rank = a.size(1), N = b.size(1), R = training_rank(rank);
  check_factor("mfq::low_rank_pack", a, K, rank, a);
  check_factor("mfq::low_rank_pack", b, rank, N, a);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  Tensor af = at::empty({R / 16, K / 32, 4, 16, 8}, a.options()), bf = at::empty({R / 16, N / 32, 4, 16, 8}, a.options());
  Tensor bs = at::empty({N, R}, a.options()), ap = at::empty({K, R}, a.options());
  check_status("mfq_low_rank_pack",
               mfq_low_rank_pack(a.data_ptr(), b.data_ptr(), dtype_code(a.scalar_type(), "lora_A"), K, N, rank, R, (float)scale,
                                 af.data_ptr(), bf.data_ptr(), bs.data_ptr(), ap.data_ptr(), stream_of(a)));
  return {af, bf, bs, ap};
}

// t [M, R] = x @ lora_A and its fragments
std::tuple<Tensor, Tensor> low_rank_forward(const Tensor& x, const Tensor& af, int64_t rank) {
  TORCH_CHECK(x.dim() == 2, "mfq::low_rank_forward: x [M, K]");
  const int64_t M = x.size(0), K = x.size(1);
  check_factor("mfq::low_rank_forward", x, M, K, x);
  check_fragments("mfq::low_rank_forward", af, K / 32, x);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t R = 16 * af.size(0);
  Tensor t = at::empty({M, R}, x.options()), tf = at::empty({R / 16, (M + 31) / 32, 4, 16, 8}, x.options());
  check_status("mfq_low_rank_forward", mfq_low_rank_forward(x.data_ptr(), af.data_ptr(), dtype_code(x.scalar_type(), "x"), M, K,
                                                            rank, R, t.data_ptr(), tf.data_ptr(), stream_of(x)));
  return {t, tf};
}

// (gt [M, R], its fragments, the gradient of lora_B [rank, N]); what is not wanted comes back empty
std::tuple<Tensor, Tensor, Tensor> low_rank_gradient(const Tensor& g, const Tensor& bf, const Tensor& tf, int64_t rank, double scale,
                                                     bool want_gt, bool want_db) {
  TORCH_CHECK(g.dim() == 2, "mfq::low_rank_gradient: g [M, N]");
  const int64_t M = g.size(0), N = g.size(1);
  check_factor("mfq::low_rank_gradient", g, M, N, g);
  check_fragments("mfq::low_rank_gradient", bf, N / 32, g);
  check_fragments("mfq::low_rank_gradient", tf, (M + 31) / 32, g);
  TORCH_CHECK(tf.size(0) == bf.size(0), "mfq::low_rank_gradient: fragments of different ranks");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(g.device());
  const int64_t R = 16 * bf.size(0);
  Tensor gt, gtf, db;
  if (want_gt) {
    gt = at::empty({M, R}, g.options());
    gtf = at::empty({R / 16, (M + 31) / 32, 4, 16, 8}, g.options());
  } else {
    gt = gtf = at::empty({0}, g.options());
  }
  db = at::empty({want_db ? rank : 0, N}, g.options());
  if (!want_gt && !want_db) return {gt, gtf, db};
  check_status("mfq_low_rank_gradient",
               mfq_low_rank_gradient(g.data_ptr(), bf.data_ptr(), tf.data_ptr(), dtype_code(g.scalar_type(), "g"), M, N, rank, R,
                                     (float)scale, want_gt ? gt.data_ptr() : nullptr, want_gt ? gtf.data_ptr() : nullptr,
                                     want_db ? db.data_ptr() : nullptr, stream_of(g)));
  return {gt, gtf, db};
}

// x^T @ t [K, rank], t in fragments
Tensor low_rank_up(const Tensor& x, const Tensor& tf, int64_t rank) {
  TORCH_CHECK(x.dim() == 2, "mfq::low_rank_up: x [M, K]");
  const int64_t M = x.size(0), K = x.size(1);
  check_factor("mfq::low_rank_up", x, M, K, x);
  check_fragments("mfq::low_rank_up", tf, (M + 31) / 32, x);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor out = at::empty({K, rank}, x.options());
  check_status("mfq_low_rank_up", mfq_low_rank_up(x.data_ptr(), tf.data_ptr(), dtype_code(x.scalar_type(), "x"), M, K, rank,
                                                  16 * tf.size(0), out.data_ptr(), stream_of(x)));
  return out;
}

// y += t @ bs^T in place
void low_rank_add_(Tensor& y, const Tensor& t, const Tensor& bs) {
  TORCH_CHECK(y.dim() == 2 && t.dim() == 2 && bs.dim() == 2 && y.is_contiguous() && t.is_contiguous() &&
                  bs.is_contiguous() && t.size(0) == y.size(0) && bs.size(0) == y.size(1) && t.size(1) == bs.size(1) &&
                  t.scalar_type() == bs.scalar_type(),
              "mfq::low_rank_add_: y [M, N], t [M, R], bs [N, R], contiguous");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(y.device());
  check_status("mfq_low_rank_add",
               mfq_low_rank_add(t.data_ptr(), bs.data_ptr(), dtype_code(t.scalar_type(), "t"), y.size(0), y.size(1),
                                t.size(1), y.data_ptr(), dtype_code(y.scalar_type(), "y"), stream_of(y)));
}

// ---- the heads of an attention block (include/mfq.h, mfq_rotary and mfq_attention)
Tensor device_int32(const char* fn, const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt, fn, ": ", name, " must be int32 on ", like.device());
  return t.contiguous();
}

// The angles that a position adds, pair by pair, of `dim` channels; scaling: 0 none, 1 linear, 2 ntk, 3 yarn (mflux_amd.heads.rotary_tables)
void rotary_frequencies(int64_t dim, double base, int64_t scaling, double factor, double length, double fast, double slow,
                        std::vector<double>& out) {
  const double d = (double)dim;
  if (scaling == 2) base *= std::pow(factor, d / (d - 2));
  auto pair_of = [&](double turns) { return d * std::log(length / (turns * 2 * M_PI)) / (2 * std::log(base)); };  // that turns so often over length
  double low = 0, high = 0;
  if (scaling == 3) {
    low = std::max(std::floor(pair_of(fast)), 0.0);
    high = std::min(std::ceil(pair_of(slow)), d - 1);
  }
  for (int64_t i = 0; i < dim / 2; ++i) {
    double f = std::pow(base, -2.0 * (double)i / d);
    if (scaling == 1) f /= factor;
    if (scaling == 3) {
      const double stretched = std::min(std::max(((double)i - low) / std::max(high - low, 0.001), 0.0), 1.0);
      f = f / factor * stretched + f * (1.0 - stretched);
    }
    out.push_back(f);
  }
}

std::tuple<Tensor, Tensor> rotary_tables(const Tensor& positions, at::IntArrayRef dims, double base, int64_t scaling, double factor, double length,
                                         double fast, double slow, double table_factor) {
  TORCH_CHECK(positions.dim() == 2 && positions.scalar_type() == at::kInt && positions.size(1) == (int64_t)dims.size() && !dims.empty(),
              "mfq::rotary_tables: positions must be an int32 matrix with a column for each dimension");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(positions.device());
  std::vector<double> frequencies;
  uint8_t axis[MFQ_ROTARY_MAX_PAIRS];
  for (size_t a = 0; a < dims.size(); ++a) {
    TORCH_CHECK(dims[a] > 0 && dims[a] % 2 == 0 && (int64_t)frequencies.size() + dims[a] / 2 <= MFQ_ROTARY_MAX_PAIRS,
                "mfq::rotary_tables: dimensions must be even, of at most 512 channels in all");
    for (int64_t i = 0; i < dims[a] / 2; ++i) axis[frequencies.size() + i] = (uint8_t)a;
    rotary_frequencies(dims[a], base, scaling, factor, length, fast, slow, frequencies);
  }
  const Tensor p = positions.contiguous();
  const int64_t n = p.size(0), pairs = (int64_t)frequencies.size();
  Tensor cos = at::empty({n, pairs}, p.options().dtype(at::kFloat)), sin = at::empty_like(cos);
  if (n == 0) return {cos, sin};
  check_status("mfq_rotary_tables", mfq_rotary_tables(p.data_ptr<int32_t>(), n, (int)p.size(1), (int)pairs, frequencies.data(), axis,
                                                      (float)table_factor, cos.data_ptr<float>(), sin.data_ptr<float>(), stream_of(p)));
  return {cos, sin};
}

// x [B, S, H, D]; what has no dense last axis is copied
Tensor dense_rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

void set_strides(int64_t (&to)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

struct RotaryOperands {
  mfq_rotary_args a = {};
  std::vector<Tensor> keep;  // what the pointers point into

  RotaryOperands(const char* fn, const Tensor& q, const c10::optional<Tensor>& k, const Tensor& cos, const Tensor& sin,
                 const c10::optional<Tensor>& positions, const c10::optional<Tensor>& q_weight, const c10::optional<Tensor>& k_weight,
                 int64_t layout, double eps) {
    TORCH_CHECK(q.dim() == 4 && cos.dim() == 2 && cos.sizes() == sin.sizes(), fn, ": q [B, S, H, D], cos and sin [P, R / 2]");
    TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.device() == q.device() && sin.device() == q.device(),
                fn, ": cos and sin must be float32 on ", q.device());
    a.dtype = dtype_code(q.scalar_type(), "q");
    a.layout = (int32_t)layout;
    a.dim = (int32_t)q.size(3);
    a.rotated = (int32_t)cos.size(1) * 2;
    a.batch = q.size(0);
    a.tokens = q.size(1);
    a.table_rows = cos.size(0);
    a.eps = (float)eps;
    keep.push_back(cos.contiguous());
    a.cos = keep.back().data_ptr<float>();
    keep.push_back(sin.contiguous());
    a.sin = keep.back().data_ptr<float>();
    if (positions.has_value()) {
      TORCH_CHECK(positions->dim() == 2 && positions->size(1) == a.tokens && (positions->size(0) == a.batch || positions->size(0) == 1), fn,
                  ": positions [B, S] or [1, S]");
      keep.push_back(device_int32(fn, "positions", *positions, q));
      a.positions = keep.back().data_ptr<int32_t>();
      a.position_batch = positions->size(0) > 1 ? a.tokens : 0;
    } else {
      TORCH_CHECK(cos.size(0) >= a.tokens, fn, ": the tables are shorter than the tokens");
    }
    tensor(fn, a.q, q, q_weight, q);
    if (k.has_value()) tensor(fn, a.k, *k, k_weight, q);
  }
  void tensor(const char* fn, mfq_rotary_tensor& to, const Tensor& t, const c10::optional<Tensor>& weight, const Tensor& q) {
    TORCH_CHECK(t.dim() == 4 && t.scalar_type() == q.scalar_type() && t.device() == q.device() && t.size(0) == q.size(0) &&
                    t.size(1) == q.size(1) && t.size(3) == q.size(3) && t.size(2) > 0,
                fn, ": q and k must agree in type, device and all axes but the heads");
    keep.push_back(dense_rows(t));
    to.x = keep.back().data_ptr();
    set_strides(to.x_stride, keep.back());
    to.heads = t.size(2);
    if (weight.has_value()) {
      TORCH_CHECK(weight->dim() == 1 && weight->size(0) == q.size(3) && weight->scalar_type() == q.scalar_type() && weight->device() == q.device(),
                  fn, ": a weight must be a [D] vector of q's type");
      keep.push_back(weight->contiguous());
      to.weight = keep.back().data_ptr();
    }
  }
  void gradient(const char* fn, mfq_rotary_tensor& to, const Tensor& dy, const Tensor& x) {
    TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(), fn,
                ": a gradient must be as its tensor");
    keep.push_back(dense_rows(dy));
    to.dy = keep.back().data_ptr();
    set_strides(to.dy_stride, keep.back());
  }
};

std::tuple<Tensor, Tensor> rotary(const Tensor& q, const c10::optional<Tensor>& k, const Tensor& cos, const Tensor& sin,
                                  const c10::optional<Tensor>& positions, const c10::optional<Tensor>& q_weight,
                                  const c10::optional<Tensor>& k_weight, int64_t layout, double eps) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  RotaryOperands o("mfq::rotary", q, k, cos, sin, positions, q_weight, k_weight, layout, eps);
  Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.has_value() ? k->sizes() : at::IntArrayRef({0}), q.options());
  if (q.numel() == 0) return {yq, yk};
  o.a.q.out = yq.data_ptr();
  if (k.has_value()) o.a.k.out = yk.data_ptr();
  check_status("mfq_rotary", mfq_rotary(&o.a, stream_of(q)));
  return {yq, yk};
}

// (dq, dk, the weights' gradients); what there is not comes back empty
std::tuple<Tensor, Tensor, Tensor, Tensor> rotary_backward(const Tensor& dyq, const c10::optional<Tensor>& dyk, const Tensor& q,
                                                           const c10::optional<Tensor>& k, const Tensor& cos, const Tensor& sin,
                                                           const c10::optional<Tensor>& positions, const c10::optional<Tensor>& q_weight,
                                                           const c10::optional<Tensor>& k_weight, int64_t layout, double eps, bool want_x,
                                                           bool want_q_weight, bool want_k_weight) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  TORCH_CHECK(k.has_value() == dyk.has_value(), "mfq::rotary_backward: a gradient for each tensor");
  TORCH_CHECK((!want_q_weight || q_weight.has_value()) && (!want_k_weight || k_weight.has_value()), "mfq::rotary_backward: no such weight");
  RotaryOperands o("mfq::rotary_backward", q, k, cos, sin, positions, q_weight, k_weight, layout, eps);
  o.gradient("mfq::rotary_backward", o.a.q, dyq, q);
  if (k.has_value()) o.gradient("mfq::rotary_backward", o.a.k, *dyk, *k);
  const Tensor none = at::empty({0}, q.options());
  Tensor dq = want_x ? at::empty(q.sizes(), q.options()) : none, dk = want_x && k.has_value() ? at::empty(k->sizes(), q.options()) : none;
  Tensor dwq = want_q_weight ? at::empty({q.size(3)}, q.options()) : none, dwk = want_k_weight ? at::empty({q.size(3)}, q.options()) : none;
  if (q.numel() == 0) return {dq, dk, dwq.zero_(), dwk.zero_()};
  if (want_x) {
    o.a.q.out = dq.data_ptr();
    if (k.has_value()) o.a.k.out = dk.data_ptr();
  }
  if (want_q_weight) o.a.q.dweight = dwq.data_ptr();
  if (want_k_weight) o.a.k.dweight = dwk.data_ptr();
  const size_t bytes = mfq_rotary_workspace_bytes(&o.a);
  Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check_status("mfq_rotary_backward", mfq_rotary_backward(&o.a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
  return {dq, dk, dwq, dwk};
}

// A tensor of mfq_attention: rows of whole 16 bytes at whole 16 bytes; anything else is copied
void attention_tensor(std::vector<Tensor>& keep, mfq_attention_tensor& to, const Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) >= 0));
  const int64_t token = t.dim() - 3;
  ok = ok && (t.size(token) <= 1 || t.stride(token) < (1 << 24));
  keep.push_back(ok ? t : t.clone(at::MemoryFormat::Contiguous));
  const Tensor& k = keep.back();
  to.p = k.data_ptr();
  for (int i = 0; i < 3; ++i) {
    const int64_t axis = token - 1 + i;
    to.stride[i] = axis >= 0 && k.size(axis) > 1 ? k.stride(axis) : 0;
  }
}

struct AttentionOperands {
  mfq_attention_args a = {};
  std::vector<Tensor> keep;

  AttentionOperands(const char* fn, const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& q_offsets,
                    const c10::optional<Tensor>& k_offsets, const c10::optional<Tensor>& q_lengths, const c10::optional<Tensor>& k_lengths,
                    bool causal, double scale) {
    const bool packed = q_offsets.has_value();
    const int64_t d = packed ? 3 : 4;
    TORCH_CHECK(k_offsets.has_value() == packed && q.dim() == d && k.dim() == d && v.sizes() == k.sizes(), fn,
                ": q [B, S, H, D] and k, v [B, S, Hkv, D], or packed without the batch and with both offsets");
    TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() && k.device() == q.device() && v.device() == q.device() &&
                    q.size(-1) == k.size(-1) && (packed || q.size(0) == k.size(0)),
                fn, ": q, k and v must agree in type, device, head size and batch");
    a.dtype = dtype_code(q.scalar_type(), "q");
    a.causal = causal;
    a.dim = (int32_t)q.size(-1);
    a.scale = (float)scale;
    a.heads = q.size(-2);
    a.kv_heads = k.size(-2);
    a.q_tokens = q.size(-3);
    a.k_tokens = k.size(-3);
    keep.reserve(16);
    if (packed) {
      TORCH_CHECK(q_offsets->dim() == 1 && q_offsets->size(0) >= 2 && k_offsets->sizes() == q_offsets->sizes(), fn,
                  ": offsets of one more value than there are sequences");
      a.batch = q_offsets->size(0) - 1;
      a.q_offsets = ints(fn, "q_offsets", q_offsets, q);
      a.k_offsets = ints(fn, "k_offsets", k_offsets, q);
    } else {
      a.batch = q.size(0);
      for (const auto* l : {&q_lengths, &k_lengths})
        TORCH_CHECK(!l->has_value() || ((*l)->dim() == 1 && (*l)->size(0) == a.batch), fn, ": lengths of one value an entry");
      a.q_lengths = ints(fn, "q_lengths", q_lengths, q);
      a.k_lengths = ints(fn, "k_lengths", k_lengths, q);
    }
    attention_tensor(keep, a.q, q);
    attention_tensor(keep, a.k, k);
    attention_tensor(keep, a.v, v);
  }
  const int32_t* ints(const char* fn, const char* name, const c10::optional<Tensor>& t, const Tensor& q) {
    if (!t.has_value()) return nullptr;
    keep.push_back(device_int32(fn, name, *t, q));
    return keep.back().data_ptr<int32_t>();
  }
  int64_t rows() const { return (a.q_offsets ? 1 : a.batch) * a.q_tokens; }
};

// y, and for a backward pass (rest and lse not nullptr) what y's rounding left and the rows' log-sum-exps
Tensor attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& q_offsets,
                         const c10::optional<Tensor>& k_offsets, const c10::optional<Tensor>& q_lengths, const c10::optional<Tensor>& k_lengths,
                         bool causal, double scale, Tensor* rest, Tensor* lse) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  AttentionOperands o("mfq::attention", q, k, v, q_offsets, k_offsets, q_lengths, k_lengths, causal, scale);
  Tensor y = at::empty(q.sizes(), q.options());
  if (rest) {
    *rest = at::empty(q.sizes(), q.options());
    *lse = at::empty({o.a.heads, o.rows()}, q.options().dtype(at::kFloat));
  }
  if (q.numel() == 0) return y;
  if (k.numel() == 0) {
    if (rest) {
      rest->zero_();
      lse->fill_(std::numeric_limits<float>::infinity());
    }
    return y.zero_();
  }
  o.a.out = y.data_ptr();
  if (rest) {
    o.a.rest = rest->data_ptr();
    o.a.lse = lse->data_ptr<float>();
  }
  const size_t bytes = mfq_attention_workspace_bytes(&o.a);
  Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check_status("mfq_attention", mfq_attention(&o.a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
  return y;
}

std::tuple<Tensor, Tensor, Tensor> attention(const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& q_offsets,
                                             const c10::optional<Tensor>& k_offsets, const c10::optional<Tensor>& q_lengths,
                                             const c10::optional<Tensor>& k_lengths, bool causal, double scale) {
  Tensor rest, lse;
  Tensor y = attention_forward(q, k, v, q_offsets, k_offsets, q_lengths, k_lengths, causal, scale, &rest, &lse);
  return {y, rest, lse};
}

std::tuple<Tensor, Tensor, Tensor> attention_backward(const Tensor& dy, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& y,
                                                      const Tensor& rest, const Tensor& lse, const c10::optional<Tensor>& q_offsets,
                                                      const c10::optional<Tensor>& k_offsets, const c10::optional<Tensor>& q_lengths,
                                                      const c10::optional<Tensor>& k_lengths, bool causal, double scale, bool want_dq,
                                                      bool want_dkv) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  AttentionOperands o("mfq::attention_backward", q, k, v, q_offsets, k_offsets, q_lengths, k_lengths, causal, scale);
  TORCH_CHECK(dy.sizes() == q.sizes() && y.sizes() == q.sizes() && dy.scalar_type() == q.scalar_type() && y.scalar_type() == q.scalar_type() &&
                  dy.device() == q.device() && y.device() == q.device(),
              "mfq::attention_backward: dy and y must be as q");
  const Tensor none = at::empty({0}, q.options());
  Tensor dq = want_dq ? at::empty(q.sizes(), q.options()) : none;
  Tensor dk = want_dkv ? at::empty(k.sizes(), q.options()) : none, dv = want_dkv ? at::empty(k.sizes(), q.options()) : none;
  if (q.numel() == 0 || k.numel() == 0 || (!want_dq && !want_dkv)) return {dq.zero_(), dk.zero_(), dv.zero_()};
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.numel() == o.a.heads * o.rows() && lse.device() == q.device(),
              "mfq::attention_backward: lse [H, rows] of the forward pass");
  TORCH_CHECK(rest.sizes() == q.sizes() && rest.scalar_type() == q.scalar_type() && rest.is_contiguous() && rest.device() == q.device(),
              "mfq::attention_backward: the rest of y's rounding as the forward pass gave it");
  o.a.rest = rest.data_ptr();
  attention_tensor(o.keep, o.a.y, y);
  attention_tensor(o.keep, o.a.dy, dy);
  Tensor delta = at::empty_like(lse);
  o.a.lse = lse.data_ptr<float>();
  o.a.delta = delta.data_ptr<float>();
  if (want_dq) o.a.dq = dq.data_ptr();
  if (want_dkv) {
    o.a.dk = dk.data_ptr();
    o.a.dv = dv.data_ptr();
  }
  const size_t bytes = mfq_attention_backward_workspace_bytes(&o.a);
  Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check_status("mfq_attention_backward", mfq_attention_backward(&o.a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
  return {dq, dk, dv};
}

// ---- the two with their gradients: what mflux_amd.heads calls
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients of a backward pass that is itself recorded: a second derivative asks for what is not there, with an error
variable_list once(const char* fn, variable_list gradients) {
  if (!at::GradMode::is_enabled()) return gradients;
  variable_list some;
  for (const auto& g : gradients)
    if (g.defined()) some.push_back(g.detach().set_requires_grad(true));
  variable_list marked = (*std::make_shared<torch::autograd::DelayedError>(std::string(fn) + ": trying to differentiate twice a function that has "
                                                                           "no second derivative", (int)some.size()))(std::move(some));
  size_t n = 0;
  for (auto& g : gradients)
    if (g.defined()) g = marked[n++];
  return gradients;
}

c10::optional<Tensor> if_defined(const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; }
Tensor or_none(const c10::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
bool wanted(const c10::optional<Tensor>& t) { return t.has_value() && t->requires_grad(); }

// A forward-mode derivative is not there either, and below autograd a tangent would be dropped without a word
void check_forward_mode(const char* fn, std::initializer_list<const c10::optional<Tensor>*> operands) {
  for (const auto* t : operands)
    TORCH_CHECK(!t->has_value() || !(*t)->_fw_grad(0).defined(), fn, ": trying to differentiate in forward mode a function that has no "
                "forward-mode derivative");
}

// A backward pass that is captured into a graph hands a leaf's gradient to the node that an earlier, still living graph of the leaf made for
// it on the stream of its time.  Where that is the default stream the engine makes the capture wait for it, which HIP forbids, in a
// thread that cannot hand the error on: the process ends.  Such a call is refused while there is nothing to lose.
void check_capture(const char* fn, std::initializer_list<const c10::optional<Tensor>*> leaves, const Tensor& like) {
  const auto stream = c10::hip::getCurrentHIPStream(like.get_device());
  if (!stream.stream()) return;  // the default stream is never captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  for (const auto* t : leaves) {
    if (!wanted(*t) || !(*t)->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(**t);
    const auto of = node ? node->stream() : c10::nullopt;
    TORCH_CHECK(!of.has_value() || of->id() != 0, fn, ": a graph is being captured while an earlier result computed from the same leaf on the default "
                "stream still lives; its gradient would make the capture wait for that stream.  Delete that result first.");
  }
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const c10::optional<Tensor>& k, const Tensor& cos, const Tensor& sin,
                               const c10::optional<Tensor>& positions, const c10::optional<Tensor>& q_weight,
                               const c10::optional<Tensor>& k_weight, int64_t layout, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [yq, yk] = rotary(q, k, cos, sin, positions, q_weight, k_weight, layout, eps);
    // without a norm the turn back needs no input: it is neither kept nor held to its values
    ctx->save_for_backward({q_weight.has_value() ? q : Tensor(), k_weight.has_value() ? or_none(k) : Tensor(), cos, sin, or_none(positions),
                            or_none(q_weight), or_none(k_weight)});
    ctx->saved_data["layout"] = layout;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["wanted"] = (int64_t)(wanted(q) | wanted(k) << 1 | wanted(q_weight) << 2 | wanted(k_weight) << 3);
    if (!k.has_value()) return {yq};
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& q = saved[0].defined() ? saved[0] : dy[0];  // (for its shape alone)
    c10::optional<Tensor> k, dyk;
    if (dy.size() > 1) {
      dyk = dy[1];
      k = saved[1].defined() ? saved[1] : dy[1];
    }
    const int64_t want = ctx->saved_data["wanted"].toInt();
    variable_list out(9);
    std::tuple<Tensor, Tensor, Tensor, Tensor> g;
    {
      at::AutoGradMode off(false);
      at::AutoDispatchBelowADInplaceOrView guard;
      g = rotary_backward(dy[0], dyk, q, k, saved[2], saved[3], if_defined(saved[4]), if_defined(saved[5]),
                          if_defined(saved[6]), ctx->saved_data["layout"].toInt(), ctx->saved_data["eps"].toDouble(), want & 3, want & 4, want & 8);
    }
    if (want & 1) out[0] = std::get<0>(g);
    if (want & 2) out[1] = std::get<1>(g);
    if (want & 4) out[5] = std::get<2>(g);
    if (want & 8) out[6] = std::get<3>(g);
    return once("mfq::rotary", std::move(out));
  }
};

std::tuple<Tensor, Tensor> rotary_call(const Tensor& q, const c10::optional<Tensor>& k, const Tensor& cos, const Tensor& sin,
                                       const c10::optional<Tensor>& positions, const c10::optional<Tensor>& q_weight,
                                       const c10::optional<Tensor>& k_weight, int64_t layout, double eps) {
  const c10::optional<Tensor> first(q), c(cos), s(sin);
  check_forward_mode("mfq::rotary", {&first, &k, &c, &s, &q_weight, &k_weight});
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(q_weight) || wanted(k_weight))) {
    check_capture("mfq::rotary", {&first, &k, &q_weight, &k_weight}, q);
    auto out = RotaryFunction::apply(q, k, cos, sin, positions, q_weight, k_weight, layout, eps);
    return {out[0], out.size() > 1 ? out[1] : at::empty({0}, q.options())};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return rotary(q, k, cos, sin, positions, q_weight, k_weight, layout, eps);
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& q_offsets,
                        const c10::optional<Tensor>& k_offsets, const c10::optional<Tensor>& q_lengths, const c10::optional<Tensor>& k_lengths,
                        bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, rest, lse] = attention(q, k, v, q_offsets, k_offsets, q_lengths, k_lengths, causal, scale);
    ctx->save_for_backward({q, k, v, y, rest, lse, or_none(q_offsets), or_none(k_offsets), or_none(q_lengths), or_none(k_lengths)});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["wanted"] = (int64_t)(wanted(q) | wanted(k) << 1 | wanted(v) << 2);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    const int64_t want = ctx->saved_data["wanted"].toInt();
    variable_list out(9);
    std::tuple<Tensor, Tensor, Tensor> g;
    {
      at::AutoGradMode off(false);
      at::AutoDispatchBelowADInplaceOrView guard;
      g = attention_backward(dy[0], saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], if_defined(saved[6]), if_defined(saved[7]),
                             if_defined(saved[8]), if_defined(saved[9]), ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
                             want & 1, want & 6);
    }
    if (want & 1) out[0] = std::get<0>(g);
    if (want & 2) out[1] = std::get<1>(g);
    if (want & 4) out[2] = std::get<2>(g);
    return once("mfq::attention", std::move(out));
  }
};

Tensor attention_call(const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& q_offsets,
                      const c10::optional<Tensor>& k_offsets, const c10::optional<Tensor>& q_lengths, const c10::optional<Tensor>& k_lengths,
                      bool causal, double scale) {
  const c10::optional<Tensor> a(q), b(k), c(v);
  check_forward_mode("mfq::attention", {&a, &b, &c});
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v))) {
    check_capture("mfq::attention", {&a, &b, &c}, q);
    return AttentionFunction::apply(q, k, v, q_offsets, k_offsets, q_lengths, k_lengths, causal, scale);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return attention_forward(q, k, v, q_offsets, k_offsets, q_lengths, k_lengths, causal, scale, nullptr, nullptr);
}

}  // namespace

TORCH_LIBRARY(mfq, m) {
  m.def("quantize_affine(Tensor w, int group_size, int bits) -> (Tensor, Tensor, Tensor)");
  m.def("dequantize_affine(Tensor wq, Tensor scales, Tensor biases, int group_size, int bits, ScalarType out_dtype) -> Tensor");
  m.def("dequantize_rows(Tensor wq, Tensor scales, Tensor biases, Tensor indices, int group_size, int bits, ScalarType out_dtype) -> Tensor");
  m.def("qmm_t(Tensor x, Tensor wq, Tensor scales, Tensor biases, Tensor? bias, int group_size, int bits, ScalarType out_dtype, Tensor? lr_t, Tensor? lr_bs) -> (Tensor, bool)");
  m.def("qmm_t_epilogue(Tensor x, Tensor wq, Tensor scales, Tensor biases, Tensor? bias, int group_size, int bits, int epilogue, Tensor? gate, Tensor? residual, int act_from) -> (Tensor, bool)");
  m.def("qmm_n(Tensor x, Tensor wq, Tensor scales, Tensor biases, int group_size, int bits, ScalarType out_dtype, Tensor? lr_t=None, Tensor? lr_bs=None) -> (Tensor, bool)");
  m.def("qmv_silu(Tensor x, Tensor wq, Tensor scales, Tensor biases, Tensor? bias, int group_size, int bits) -> (Tensor, bool)");
  m.def("layer_norm_modulate(Tensor x, Tensor? scale, Tensor? shift, float eps) -> (Tensor, bool)");
  m.def("low_rank_add_(Tensor(a!) y, Tensor t, Tensor bs) -> ()");
  m.def("low_rank_down(Tensor x, Tensor af) -> Tensor");
  m.def("low_rank_pack(Tensor lora_a, Tensor lora_b, float scale) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("low_rank_forward(Tensor x, Tensor af, int rank) -> (Tensor, Tensor)");
  m.def("low_rank_gradient(Tensor g, Tensor bf, Tensor tf, int rank, float scale, bool want_gt, bool want_db) -> (Tensor, Tensor, Tensor)");
  m.def("low_rank_up(Tensor x, Tensor tf, int rank) -> Tensor");
  m.def("rotary_tables(Tensor positions, int[] dims, float base, int scaling, float factor, float length, float fast, float slow, float table_factor) -> (Tensor, Tensor)");
  m.def("rotary(Tensor q, Tensor? k, Tensor cos, Tensor sin, Tensor? positions, Tensor? q_weight, Tensor? k_weight, int layout, float eps) -> (Tensor, Tensor)");
  m.def("rotary_backward(Tensor dyq, Tensor? dyk, Tensor q, Tensor? k, Tensor cos, Tensor sin, Tensor? positions, Tensor? q_weight, Tensor? k_weight, int layout, float eps, bool want_x, bool want_q_weight, bool want_k_weight) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? q_offsets, Tensor? k_offsets, Tensor? q_lengths, Tensor? k_lengths, bool causal, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("rotary_call(Tensor q, Tensor? k, Tensor cos, Tensor sin, Tensor? positions, Tensor? q_weight, Tensor? k_weight, int layout, float eps) -> (Tensor, Tensor)");
  m.def("attention_call(Tensor q, Tensor k, Tensor v, Tensor? q_offsets, Tensor? k_offsets, Tensor? q_lengths, Tensor? k_lengths, bool causal, float scale) -> Tensor");
  m.def("attention_backward(Tensor dy, Tensor q, Tensor k, Tensor v, Tensor y, Tensor rest, Tensor lse, Tensor? q_offsets, Tensor? k_offsets, Tensor? q_lengths, Tensor? k_lengths, bool causal, float scale, bool want_dq, bool want_dkv) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mfq, CUDA, m) {  // the HIP backend answers to torch's CUDA dispatch key
  m.impl("quantize_affine", quantize_affine);
  m.impl("dequantize_affine", dequantize_affine);
  m.impl("dequantize_rows", dequantize_rows);
  m.impl("qmm_t", qmm_t);
  m.impl("qmm_t_epilogue", qmm_t_epilogue);
  m.impl("qmm_n", qmm_n);
  m.impl("qmv_silu", qmv_silu);
  m.impl("layer_norm_modulate", layer_norm_modulate);
  m.impl("low_rank_add_", low_rank_add_);
  m.impl("low_rank_down", low_rank_down);
  m.impl("low_rank_pack", low_rank_pack);
  m.impl("low_rank_forward", low_rank_forward);
  m.impl("low_rank_gradient", low_rank_gradient);
  m.impl("low_rank_up", low_rank_up);
  m.impl("rotary_tables", rotary_tables);
  m.impl("rotary", rotary);
  m.impl("rotary_backward", rotary_backward);
  m.impl("attention", attention);
  m.impl("attention_backward", attention_backward);
  m.impl("rotary_call", rotary_call);
  m.impl("attention_call", attention_call);
}

TORCH_LIBRARY_IMPL(mfq, AutogradCUDA, m) {  // the ops with gradients; the others are called from these and from Python functions
  m.impl("rotary_call", rotary_call);
  m.impl("attention_call", attention_call);
}
