// Rotary positions, with the RMS norm of the heads in front of them, for q and k in one launch:
//   n = x / sqrt(mean(x^2) + eps) * w   (where a weight is given)
//   y = n with its first R channels turned, pair (a, b) -> (a cos - b sin, b cos + a sin)
// (AttentionUtils.process_qkv and apply_rope,
// src/mflux/models/flux/model/flux_transformer/common/attention_utils.py), the tables of the angles, and the
// gradients:  dn = the turned back dy,  dw = sum dn x r,  dx = r (w dn - x r mean(w dn x r)),  r = 1 / sqrt(mean(x^2) + eps).
// Everything between a load and its store is float32 and rounded once; sums over rows are float32 and in a fixed order.
//
// Bound by HBM: every element is read and written once.  A lane holds kVec pairs of a row, as many lanes as that takes a row, and
// rows (token, head) are dealt to the wavefronts.  4608 tokens, 24 + 24 heads of 128 with norms, bfloat16: 28 us, 4.1 TB/s (a large copy:
// 4.9); backward of 4110 tokens, 16 + 4 heads, float16: 23 us, and 4 for the weights' sums.
#include "common.h"

#include <algorithm>

namespace mfq {
namespace {

constexpr int kThreads = 256;

// N consecutive elements as float32; N * size is 4 to 32 bytes or one element
template <typename T, int N>
__device__ inline void load_vec(const typename T::storage* p, float (&v)[N]) {
  if constexpr (sizeof(typename T::storage) == 4) {
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] = a[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = p[i];
    }
  } else if constexpr (N >= 4) {
    typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
    const words a = *reinterpret_cast<const words*>(p);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      v[2 * i] = lo_f32<T>(a[i]);
      v[2 * i + 1] = hi_f32<T>(a[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = T::to_f32(p[i]);
  }
}

template <typename T, int N>
__device__ inline void store_vec(typename T::storage* p, const float (&v)[N]) {
  if constexpr (sizeof(typename T::storage) == 4) {
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4*>(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = v[i];
    }
  } else if constexpr (N >= 4) {
    typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
    words a;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) a[i] = T::pack2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<words*>(p) = a;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = T::from_f32(v[i]);
  }
}

// One of q and k.  In the backward pass `x` is the forward's input (only needed with a weight) and `dy`, `out` the gradients.
struct RotaryTensor {
  const void* x;
  const void* dy;
  const void* weight;
  void* out;
  float* dw;                        // partial sums, [workgroups][dim]
  int64_t x_batch, x_token, x_head;     // strides in elements
  int64_t dy_batch, dy_token, dy_head;
  uint32_t heads;
  uint32_t rows;                    // tokens * heads
};

struct RotaryCall {
  RotaryTensor t[2];
  const float *cos, *sin;      // [table_rows, rotated / 2]
  const int32_t* positions;    // token -> row of the tables, or nullptr: the token's place
  int64_t position_batch;      // 0: the same positions for every entry
  uint32_t per_batch;          // tokens of an entry
  int table_rows, dim, rotated, half_layout;
  int lanes;                   // of a row: a power of two
  float eps;
};

// kVec pairs to a unit, kUnits units to a lane
template <typename T, int kVec, int kUnits, bool kBackward>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryCall c) {
  using E = typename T::storage;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int in_row = lane & (c.lanes - 1), row_of_wave = lane / c.lanes, per_pass = kWave / c.lanes;
  const int units = c.dim / (2 * kVec), turned = c.rotated / (2 * kVec), half = c.rotated / 2;
  // a unit's pairs: elements at[u] + i and at[u] + half + i, or, where they lie side by side, at[u] + 2 i and + 1
  int at[kUnits];
  bool inside[kUnits], turns[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = in_row + u * c.lanes;
    inside[u] = unit < units;
    turns[u] = unit < turned;
    at[u] = c.half_layout && turns[u] ? unit * kVec : unit * 2 * kVec;
  }
  auto load_unit = [&](const E* row, int u, float (&a)[kVec], float (&b)[kVec]) __attribute__((always_inline)) {
    if (c.half_layout && turns[u]) {
      load_vec<T, kVec>(row + at[u], a);
      load_vec<T, kVec>(row + at[u] + half, b);
    } else {
      float w[2 * kVec];
      load_vec<T, kVec>(row + at[u], *reinterpret_cast<float(*)[kVec]>(w));
      load_vec<T, kVec>(row + at[u] + kVec, *reinterpret_cast<float(*)[kVec]>(w + kVec));
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        a[i] = w[2 * i];
        b[i] = w[2 * i + 1];
      }
    }
  };
  auto store_unit = [&](E* row, int u, const float (&a)[kVec], const float (&b)[kVec]) __attribute__((always_inline)) {
    if (c.half_layout && turns[u]) {
      store_vec<T, kVec>(row + at[u], a);
      store_vec<T, kVec>(row + at[u] + half, b);
    } else {
      float w[2 * kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        w[2 * i] = a[i];
        w[2 * i + 1] = b[i];
      }
      store_vec<T, kVec>(row + at[u], *reinterpret_cast<const float(*)[kVec]>(w));
      store_vec<T, kVec>(row + at[u] + kVec, *reinterpret_cast<const float(*)[kVec]>(w + kVec));
    }
  };

  const int64_t waves = (int64_t)gridDim.x * (kThreads / kWave), id = (int64_t)blockIdx.x * (kThreads / kWave) + wave;
  // one of the two tensors: passes of `per_pass` rows (token, head), dealt to the wavefronts in turn from `start` on (as neighbours to
  // one wavefront, with a token's angles loaded once for them, 4110 tokens x 20 heads take 32 us in the backward pass, like this 25)
  auto walk = [&](const RotaryTensor& t, int64_t start) __attribute__((always_inline)) {
    const E* weight = static_cast<const E*>(t.weight);
    float wa[kUnits][kVec], wb[kUnits][kVec], dw[kUnits][2 * kVec];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (weight && inside[u]) load_unit(weight, u, wa[u], wb[u]);
#pragma unroll
      for (int i = 0; i < 2 * kVec; ++i) dw[u][i] = 0.f;
    }
    for (int64_t pass = start; pass * per_pass < t.rows; pass += waves) {
      const uint32_t any = (uint32_t)(pass * per_pass) + row_of_wave;
      const bool live = any < t.rows;
      const uint32_t row = live ? any : t.rows - 1;
      const uint32_t token = row / t.heads, head = row - token * t.heads, batch = token / c.per_batch, place = token - batch * c.per_batch;
      int64_t angle = place;
      if (c.positions) angle = c.positions[batch * c.position_batch + place];
      angle = min(max(angle, (int64_t)0), (int64_t)c.table_rows - 1) * half;
      const E* x = static_cast<const E*>(t.x) + (batch * t.x_batch + place * t.x_token + head * t.x_head);
      const E* dy = static_cast<const E*>(t.dy) + (batch * t.dy_batch + place * t.dy_token + head * t.dy_head);
      float a[kUnits][kVec], b[kUnits][kVec];  // the turned row, in the backward pass the turned back gradient
      float xa[kUnits][kVec], xb[kUnits][kVec], cs[kUnits][kVec], sn[kUnits][kVec];
      // everything the row needs is requested before the first sum over its lanes
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (!inside[u]) continue;
        if constexpr (kBackward) load_unit(dy, u, a[u], b[u]);
        if (!kBackward || weight) load_unit(x, u, xa[u], xb[u]);
        if (turns[u]) {
          load_vec<F32, kVec>(c.cos + angle + (in_row + u * c.lanes) * kVec, cs[u]);
          load_vec<F32, kVec>(c.sin + angle + (in_row + u * c.lanes) * kVec, sn[u]);
        }
      }
      float squares = 0.f, dot = 0.f;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (!inside[u]) continue;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          if (!turns[u]) {
            cs[u][i] = 1.f;
            sn[u][i] = 0.f;
          }
          if constexpr (kBackward) {
            const float g = a[u][i], h = b[u][i];
            a[u][i] = __builtin_fmaf(g, cs[u][i], h * sn[u][i]);
            b[u][i] = __builtin_fmaf(h, cs[u][i], -(g * sn[u][i]));
          }
          if (weight) {
            squares = __builtin_fmaf(xa[u][i], xa[u][i], __builtin_fmaf(xb[u][i], xb[u][i], squares));
            if constexpr (kBackward) dot = __builtin_fmaf(a[u][i] * wa[u][i], xa[u][i], __builtin_fmaf(b[u][i] * wb[u][i], xb[u][i], dot));
          }
        }
      }
      float r = 1.f, mean = 0.f;
      if (weight) {
        for (int d = 1; d < c.lanes; d *= 2) {
          squares += __shfl_xor(squares, d);
          if constexpr (kBackward) dot += __shfl_xor(dot, d);
        }
        r = 1.0f / __builtin_sqrtf(squares / (float)c.dim + c.eps);
        mean = r * dot / (float)c.dim;
      }
      if (!live) continue;
      E* out = static_cast<E*>(t.out);
      if (out) out += (int64_t)row * c.dim;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (!inside[u]) continue;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          if constexpr (!kBackward) {
            if (weight) {
              xa[u][i] = xa[u][i] * r * wa[u][i];
              xb[u][i] = xb[u][i] * r * wb[u][i];
            }
            a[u][i] = __builtin_fmaf(xa[u][i], cs[u][i], -(xb[u][i] * sn[u][i]));
            b[u][i] = __builtin_fmaf(xb[u][i], cs[u][i], xa[u][i] * sn[u][i]);
          } else if (weight) {
            const float m = xa[u][i] * r, n = xb[u][i] * r;  // the normalised row
            dw[u][2 * i] = __builtin_fmaf(a[u][i], m, dw[u][2 * i]);
            dw[u][2 * i + 1] = __builtin_fmaf(b[u][i], n, dw[u][2 * i + 1]);
            a[u][i] = r * __builtin_fmaf(-mean, m, a[u][i] * wa[u][i]);
            b[u][i] = r * __builtin_fmaf(-mean, n, b[u][i] * wb[u][i]);
          }
        }
        if (out) store_unit(out, u, a[u], b[u]);
      }
    }
    if constexpr (kBackward) {
      if (t.dw) {  // the workgroup's sums for the weight's gradient: a slot in LDS for every row that its wavefronts hold at a time
        __shared__ float sums[kThreads * kUnits * 2 * kVec];
        float* mine = sums + (wave * per_pass + row_of_wave) * c.dim;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          if (!inside[u]) continue;
          const bool apart = c.half_layout && turns[u];
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            mine[apart ? at[u] + i : at[u] + 2 * i] = dw[u][2 * i];
            mine[apart ? at[u] + half + i : at[u] + 2 * i + 1] = dw[u][2 * i + 1];
          }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < c.dim; e += kThreads) {
          float v = 0.f;
          for (int k = 0; k < kThreads / kWave * per_pass; ++k) v += sums[k * c.dim + e];
          t.dw[(int64_t)blockIdx.x * c.dim + e] = v;
        }
        __syncthreads();
      }
    }
  };
  walk(c.t[0], id);
  if (c.t[1].rows) walk(c.t[1], (id + waves - (c.t[0].rows + per_pass - 1) / per_pass % waves) % waves);  // from where the first one ended
}

// dw = sum of the workgroups' partial sums: a workgroup to 16 columns, 64 threads to a column
template <typename T>
__global__ __launch_bounds__(1024) void rotary_weight_kernel(const float* parts0, const float* parts1, int n, int dim, void* dw0, void* dw1) {
  const float* parts = blockIdx.y ? parts1 : parts0;
  auto* dw = static_cast<typename T::storage*>(blockIdx.y ? dw1 : dw0);
  if (!dw) return;
  const int e = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
  float v = 0.f;
  if (e < dim) {
#pragma unroll 8
    for (int i = part; i < n; i += 64) v += parts[(int64_t)i * dim + e];
  }
  __shared__ float sums[64][17];
  sums[part][threadIdx.x & 15] = v;
  __syncthreads();
  if (part || e >= dim) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) v += sums[i][threadIdx.x & 15];
  dw[e] = T::from_f32(v);
}

struct Shape {
  int vec, lanes;
  int64_t groups;
};

bool shape_of(const mfq_rotary_args& a, bool wide, bool backward, Shape& s) {
  const int dim = a.dim, rotated = a.rotated;
  s.vec = wide && dim % 16 == 0 && rotated % 16 == 0 ? 8 : wide && dim % 8 == 0 && rotated % 8 == 0 ? 4 : 1;
  const int units = s.vec == 1 ? 4 : 1;  // of a lane
  s.lanes = 1;
  while (s.lanes * units * 2 * s.vec < dim) s.lanes *= 2;
  if (s.lanes > kWave) return false;
  const int64_t tokens = a.batch * a.tokens, per_pass = kWave / s.lanes;
  const int64_t passes = (tokens * a.q.heads + per_pass - 1) / per_pass + (tokens * a.k.heads + per_pass - 1) / per_pass;
  // as many passes to every wavefront, of as many workgroups as the compute units hold at a time (three or four)
  const int64_t most = (backward ? 3 : 4) * (int64_t)compute_units(), groups = (passes + kThreads / kWave - 1) / (kThreads / kWave);
  const int64_t each = (groups + most - 1) / most;
  s.groups = (groups + each - 1) / each;
  return true;
}

template <typename T, bool kBackward>
int launch(const Shape& s, const RotaryCall& c, hipStream_t stream) {
  const dim3 grid((unsigned)s.groups), block(kThreads);
  if (s.vec == 8) hipLaunchKernelGGL((rotary_kernel<T, 8, 1, kBackward>), grid, block, 0, stream, c);
  else if (s.vec == 4) hipLaunchKernelGGL((rotary_kernel<T, 4, 1, kBackward>), grid, block, 0, stream, c);
  else hipLaunchKernelGGL((rotary_kernel<T, 1, 4, kBackward>), grid, block, 0, stream, c);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

// the angles' frequencies travel in the launch: no copy to the device, nothing a captured graph could find changed
struct Frequencies {
  double f[MFQ_ROTARY_MAX_PAIRS];
  uint8_t axis[MFQ_ROTARY_MAX_PAIRS];
};

// Sine and cosine of an angle of up to 2^33 (a position times a frequency of up to 4) in float64, times a factor and rounded once: less
// the nearest multiple of pi / 2 (whose second half makes up for the first's rounding, the products being exact in an fma), then the
// series in up to |r| = pi / 4, cut where the next term is below 2^-33.  The multiple is rounded by adding 1.5 * 2^52, which leaves it in the sum's low bits.
__device__ inline void sine_cosine(double angle, double factor, float& s, float& c) {
  const double shifted = __builtin_fma(angle, 0.63661977236758134308, 6755399441055744.0), quarter = shifted - 6755399441055744.0;
  const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, shifted);
  const double r = __builtin_fma(-quarter, 6.123233995736765886e-17, __builtin_fma(-quarter, 1.57079632679489661923, angle)), x = r * r;
  double sn = __builtin_fma(x, -1.0 / 39916800, 1.0 / 362880), cs = __builtin_fma(x, 1.0 / 479001600, -1.0 / 3628800);
  sn = __builtin_fma(x, sn, -1.0 / 5040);
  cs = __builtin_fma(x, cs, 1.0 / 40320);
  sn = __builtin_fma(x, sn, 1.0 / 120);
  cs = __builtin_fma(x, cs, -1.0 / 720);
  sn = __builtin_fma(x, sn, -1.0 / 6);
  cs = __builtin_fma(x, cs, 1.0 / 24);
  cs = __builtin_fma(x, cs, -0.5);
  sn = __builtin_fma(r * x, sn, r);
  cs = __builtin_fma(x, cs, 1.0);
  if (factor != 1.0) {
    sn *= factor;
    cs *= factor;
  }
  const float a = (float)sn, b = (float)cs;
  s = __uint_as_float(__float_as_uint(n & 1 ? b : a) ^ (n & 2) << 30);
  c = __uint_as_float(__float_as_uint(n & 1 ? a : b) ^ ((n + 1) & 2) << 30);
}

// A thread to kVec angles of every so many rows, so that it reads its frequencies once.  position * frequency is a float64 product and
// its sine and cosine are taken in float64: at position 10^5 a float32 angle is off by 4 10^-3.  Bound by the stores.
template <int kVec>
__global__ __launch_bounds__(256) void rotary_tables_kernel(const int32_t* positions, int64_t n, int axes, int pairs, Frequencies f, float factor,
                                                            float* cos, float* sin) {
  const int per_row = pairs / kVec, rows = 256 / per_row;
  const int first = threadIdx.x / per_row, pair = (threadIdx.x - first * per_row) * kVec;
  if (first >= rows) return;
  double frequency[kVec];
  int axis[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) {
    frequency[v] = f.f[pair + v];
    axis[v] = f.axis[pair + v];
  }
  for (int64_t row = (int64_t)blockIdx.x * rows + first; row < n; row += (int64_t)gridDim.x * rows) {
    float c[kVec], s[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) sine_cosine((double)positions[row * axes + axis[v]] * frequency[v], (double)factor, s[v], c[v]);
    store_vec<F32, kVec>(cos + row * pairs + pair, c);
    store_vec<F32, kVec>(sin + row * pairs + pair, s);
  }
}

}  // namespace

int launch_rotary_tables(const int32_t* positions, int64_t n, int axes, int pairs, const double* frequencies, const uint8_t* axis, float factor,
                         float* cos, float* sin, hipStream_t stream) {
  Frequencies f = {};
  for (int i = 0; i < pairs; ++i) {
    f.f[i] = frequencies[i];
    f.axis[i] = axis[i];
  }
  const bool wide = pairs % 4 == 0 && aligned16(cos) && aligned16(sin);
  const int64_t rows = 256 / (wide ? pairs / 4 : pairs);
  const dim3 grid((unsigned)std::min<int64_t>((n + rows - 1) / rows, 8 * (int64_t)compute_units()));
  if (wide) hipLaunchKernelGGL(rotary_tables_kernel<4>, grid, dim3(256), 0, stream, positions, n, axes, pairs, f, factor, cos, sin);
  else hipLaunchKernelGGL(rotary_tables_kernel<1>, grid, dim3(256), 0, stream, positions, n, axes, pairs, f, factor, cos, sin);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

size_t rotary_workspace_bytes(const mfq_rotary_args& a) {
  return ((a.q.dweight ? 1 : 0) + (a.k.dweight ? 1 : 0)) * (size_t)(3 * compute_units()) * a.dim * 4;
}

int launch_rotary(const mfq_rotary_args& a, bool wide, bool backward, float* workspace, hipStream_t stream) {
  Shape s;
  if (!shape_of(a, wide, backward, s)) return MFQ_EUNSUPPORTED;
  RotaryCall c = {};
  const mfq_rotary_tensor* in[2] = {&a.q, &a.k};
  for (int i = 0; i < 2; ++i) {
    const mfq_rotary_tensor& t = *in[i];
    c.t[i] = {t.x, t.dy, t.weight, t.out, nullptr, t.x_stride[0], t.x_stride[1], t.x_stride[2], t.dy_stride[0], t.dy_stride[1], t.dy_stride[2],
              (uint32_t)t.heads, (uint32_t)(a.batch * a.tokens * t.heads)};
    if (backward && t.dweight) {
      c.t[i].dw = workspace;
      workspace += (int64_t)(3 * compute_units()) * a.dim;  // a row of a workgroup
    }
  }
  c.cos = a.cos;
  c.sin = a.sin;
  c.positions = a.positions;
  c.position_batch = a.position_batch;
  c.per_batch = (uint32_t)a.tokens;
  c.table_rows = (int)a.table_rows;
  c.dim = a.dim;
  c.rotated = a.rotated;
  c.half_layout = a.layout == MFQ_ROTARY_HALF;
  c.lanes = s.lanes;
  c.eps = a.eps;
  int rc;
  if (a.dtype == MFQ_BF16) rc = backward ? launch<BF16, true>(s, c, stream) : launch<BF16, false>(s, c, stream);
  else if (a.dtype == MFQ_F16) rc = backward ? launch<F16, true>(s, c, stream) : launch<F16, false>(s, c, stream);
  else rc = backward ? launch<F32, true>(s, c, stream) : launch<F32, false>(s, c, stream);
  if (rc != MFQ_OK || !backward || (!a.q.dweight && !a.k.dweight)) return rc;
  const dim3 grid((unsigned)((a.dim + 15) / 16), 2);
#define MFQ_WEIGHTS(T) \
  hipLaunchKernelGGL(rotary_weight_kernel<T>, grid, dim3(1024), 0, stream, c.t[0].dw, c.t[1].dw, (int)s.groups, a.dim, a.q.dweight, a.k.dweight)
  if (a.dtype == MFQ_BF16) MFQ_WEIGHTS(BF16);
  else if (a.dtype == MFQ_F16) MFQ_WEIGHTS(F16);
  else MFQ_WEIGHTS(F32);
#undef MFQ_WEIGHTS
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

}  // namespace mfq
