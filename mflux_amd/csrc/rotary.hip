// Rotary positions, with the RMS norm of the heads in front of them, for q and k in one launch:
//   n = x / sqrt(mean(x^2) + eps) * w   (where a weight is given)
//   y = n with its first R channels turned, pair (a, b) -> (a cos - b sin, b cos + a sin)
// (AttentionUtils.process_qkv and apply_rope,
// src/mflux/models/flux/model/flux_transformer/common/attention_utils.py), the tables of the angles, and the
// gradients:  dn = the turned back dy,  dw = sum dn x r,  dx = r (w dn - x r mean(w dn x r)),  r = 1 / sqrt(mean(x^2) + eps).
// Everything between a load and its store is float32 and rounded once; sums over rows are float32 and in a fixed order.
//
// Bound by HBM: every element is read and written once.  A lane holds kVec pairs of a row, as many lanes as that takes a row, and a
// wavefront a token's rows: its cosines and sines are loaded once for all heads it walks.
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

// One of q and k.  In the backward pass `x` is the forward's input (only needed with a weight) and `y`, `out` the gradients.
struct RotaryTensor {
  const void* x;
  const void* dy;
  const void* weight;
  void* out;
  float* dw;                        // partial sums, [workgroups][dim]
  int64_t x_batch, x_token, x_head;     // strides in elements
  int64_t dy_batch, dy_token, dy_head;
  int heads;
};

struct RotaryCall {
  RotaryTensor t[2];
  const float *cos, *sin;      // [table_rows, rotated / 2]
  const int32_t* positions;    // token -> row of the tables, or nullptr: the token's place
  int64_t position_batch;      // 0: the same positions for every entry
  int64_t tokens;              // of all entries
  int per_batch;               // of an entry
  int table_rows, dim, rotated, half_layout;
  int lanes;                   // of a row: a power of two
  int passes;                  // of a wavefront over the heads
  int chunks;                  // of heads: passes * (64 / lanes) heads each
  float eps;
};

// kVec pairs to a unit, kUnits units to a lane
template <typename T, int kVec, int kUnits, bool kBackward>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryCall c) {
  using E = typename T::storage;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int in_row = lane & (c.lanes - 1), row_of_wave = lane / c.lanes, rows_per_pass = kWave / c.lanes;
  const int units = c.dim / (2 * kVec), turned = c.rotated / (2 * kVec), half = c.rotated / 2;
  // a unit's pairs: elements at[u] + i and at[u] + step + i (or, pairs side by side, at[u] + 2 i and + 1)
  int at[kUnits];
  bool inside[kUnits], turns[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = in_row + u * c.lanes;
    inside[u] = unit < units;
    turns[u] = unit < turned;
    at[u] = c.half_layout && turns[u] ? unit * kVec : unit * 2 * kVec;
  }
  const int heads = c.t[0].heads + c.t[1].heads;
  float dw[2][kUnits][2 * kVec];
  if constexpr (kBackward) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int i = 0; i < 2 * kVec; ++i) dw[w][u][i] = 0.f;
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

  const int64_t items = c.tokens * c.chunks;
  for (int64_t item = (int64_t)blockIdx.x * (kThreads / kWave) + wave; item < items; item += (int64_t)gridDim.x * (kThreads / kWave)) {
    const int64_t token = item / c.chunks;
    const int chunk = (int)(item - token * c.chunks);
    const int64_t batch = token / c.per_batch, place = token - batch * c.per_batch;
    int64_t row = place;
    if (c.positions) row = c.positions[batch * c.position_batch + place];
    row = min(max(row, (int64_t)0), (int64_t)c.table_rows - 1);
    float cs[kUnits][kVec], sn[kUnits][kVec];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (turns[u]) {
        load_vec<F32, kVec>(c.cos + row * half + (in_row + u * c.lanes) * kVec, cs[u]);
        load_vec<F32, kVec>(c.sin + row * half + (in_row + u * c.lanes) * kVec, sn[u]);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          cs[u][i] = 1.f;
          sn[u][i] = 0.f;
        }
      }
      if constexpr (kBackward) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) sn[u][i] = -sn[u][i];
      }
    }
    for (int pass = 0; pass < c.passes; ++pass) {
      const int any_head = (chunk * c.passes + pass) * rows_per_pass + row_of_wave;
      const bool live = any_head < heads;
      const int which = live && any_head >= c.t[0].heads;
      const RotaryTensor& t = c.t[which];
      const int head = live ? any_head - which * c.t[0].heads : 0;
      const E* x = static_cast<const E*>(t.x) + (batch * t.x_batch + place * t.x_token + head * t.x_head);
      const E* w = static_cast<const E*>(t.weight);
      E* out = static_cast<E*>(t.out) + (token * t.heads + head) * c.dim;
      float a[kUnits][kVec], b[kUnits][kVec];  // the row (forward) or its turned back gradient
      float xa[kUnits][kVec], xb[kUnits][kVec];
      float squares = 0.f;
      if (live && (!kBackward || w)) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if (inside[u]) {
            load_unit(x, u, xa[u], xb[u]);
#pragma unroll
            for (int i = 0; i < kVec; ++i) squares = __builtin_fmaf(xa[u][i], xa[u][i], __builtin_fmaf(xb[u][i], xb[u][i], squares));
          }
      }
      // lanes of a row always come here together; rows of both tensors may share a wavefront
      for (int d = 1; d < c.lanes; d *= 2) squares += __shfl_xor(squares, d);
      const float r = w ? 1.0f / __builtin_sqrtf(squares / (float)c.dim + c.eps) : 1.0f;
      if constexpr (!kBackward) {
        if (!live) continue;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if (inside[u]) {
            if (w) {
              float wa[kVec], wb[kVec];
              load_unit(w, u, wa, wb);
#pragma unroll
              for (int i = 0; i < kVec; ++i) {
                xa[u][i] = xa[u][i] * r * wa[i];
                xb[u][i] = xb[u][i] * r * wb[i];
              }
            }
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
              a[u][i] = __builtin_fmaf(xa[u][i], cs[u][i], -(xb[u][i] * sn[u][i]));
              b[u][i] = __builtin_fmaf(xb[u][i], cs[u][i], xa[u][i] * sn[u][i]);
            }
            store_unit(out, u, a[u], b[u]);
          }
      } else {
        const E* dy = static_cast<const E*>(t.dy) + (batch * t.dy_batch + place * t.dy_token + head * t.dy_head);
        float dot = 0.f;
        if (live) {
#pragma unroll
          for (int u = 0; u < kUnits; ++u)
            if (inside[u]) {
              float ga[kVec], gb[kVec];
              load_unit(dy, u, ga, gb);
#pragma unroll
              for (int i = 0; i < kVec; ++i) {
                a[u][i] = __builtin_fmaf(ga[i], cs[u][i], -(gb[i] * sn[u][i]));
                b[u][i] = __builtin_fmaf(gb[i], cs[u][i], ga[i] * sn[u][i]);
              }
              if (w) {
                float wa[kVec], wb[kVec];
                load_unit(w, u, wa, wb);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                  xa[u][i] *= r;  // the normalised row
                  xb[u][i] *= r;
                  if (which) {
                    dw[1][u][2 * i] = __builtin_fmaf(a[u][i], xa[u][i], dw[1][u][2 * i]);
                    dw[1][u][2 * i + 1] = __builtin_fmaf(b[u][i], xb[u][i], dw[1][u][2 * i + 1]);
                  } else {
                    dw[0][u][2 * i] = __builtin_fmaf(a[u][i], xa[u][i], dw[0][u][2 * i]);
                    dw[0][u][2 * i + 1] = __builtin_fmaf(b[u][i], xb[u][i], dw[0][u][2 * i + 1]);
                  }
                  a[u][i] *= wa[i];
                  b[u][i] *= wb[i];
                  dot = __builtin_fmaf(a[u][i], xa[u][i], __builtin_fmaf(b[u][i], xb[u][i], dot));
                }
              }
            }
        }
        for (int d = 1; d < c.lanes; d *= 2) dot += __shfl_xor(dot, d);
        if (!live || !out) continue;
        const float mean = dot / (float)c.dim;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if (inside[u]) {
            if (w) {
#pragma unroll
              for (int i = 0; i < kVec; ++i) {
                a[u][i] = r * __builtin_fmaf(-mean, xa[u][i], a[u][i]);
                b[u][i] = r * __builtin_fmaf(-mean, xb[u][i], b[u][i]);
              }
            }
            store_unit(out, u, a[u], b[u]);
          }
      }
    }
  }
  if constexpr (kBackward) {
    // the workgroup's sums for the weights' gradients: rows of a wavefront by shuffles, wavefronts through LDS
    __shared__ float sums[kThreads / kWave][kUnits * kWave * 2 * kVec];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (!c.t[which].dw) continue;
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int i = 0; i < 2 * kVec; ++i) {
          float v = dw[which][u][i];
          for (int d = c.lanes; d < kWave; d *= 2) v += __shfl_xor(v, d);
          if (row_of_wave == 0) {
            const int pair = i >> 1;
            const int e = c.half_layout && turns[u] ? at[u] + (i & 1) * half + pair : at[u] + 2 * pair + (i & 1);
            if (inside[u]) sums[wave][e] = v;
          }
        }
      __syncthreads();
      for (int e = threadIdx.x; e < c.dim; e += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kThreads / kWave; ++k) v += sums[k][e];
        c.t[which].dw[(int64_t)blockIdx.x * c.dim + e] = v;
      }
      __syncthreads();
    }
  }
}

// dw = sum of the workgroups' partial sums: a workgroup to 16 columns, 16 threads to a column
template <typename T>
__global__ __launch_bounds__(256) void rotary_weight_kernel(const float* parts0, const float* parts1, int n, int dim, void* dw0, void* dw1) {
  const float* parts = blockIdx.y ? parts1 : parts0;
  auto* dw = static_cast<typename T::storage*>(blockIdx.y ? dw1 : dw0);
  if (!dw) return;
  const int e = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
  float v = 0.f;
  if (e < dim)
    for (int i = part; i < n; i += 16) v += parts[(int64_t)i * dim + e];
  __shared__ float sums[16][17];
  sums[part][threadIdx.x & 15] = v;
  __syncthreads();
  if (part || e >= dim) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v += sums[i][threadIdx.x & 15];
  dw[e] = T::from_f32(v);
}

constexpr int kBackwardGroups = 512;

struct Shape {
  int vec, units, lanes, passes, chunks;
  int64_t groups;
};

bool shape_of(const mfq_rotary_args& a, bool wide, bool backward, Shape& s) {
  const int dim = a.dim, rotated = a.rotated;
  s.vec = wide && dim % 16 == 0 && rotated % 16 == 0 ? 8 : wide && dim % 8 == 0 && rotated % 8 == 0 ? 4 : 1;
  const int units = dim / (2 * s.vec);
  s.units = s.vec == 1 ? 4 : 1;
  s.lanes = 1;
  while (s.lanes * s.units < units) s.lanes *= 2;
  if (s.lanes > kWave) return false;
  const int64_t tokens = a.batch * a.tokens;
  const int heads = (int)(a.q.heads + a.k.heads), all = (heads + kWave / s.lanes - 1) / (kWave / s.lanes);
  // few tokens: the heads of one over several wavefronts, until there are two for every SIMD
  s.passes = (int)std::max<int64_t>(1, std::min<int64_t>(all, tokens * all / (8 * (int64_t)compute_units())));
  s.chunks = (all + s.passes - 1) / s.passes;
  s.groups = (tokens * s.chunks + kThreads / kWave - 1) / (kThreads / kWave);
  if (backward) s.groups = std::min<int64_t>(s.groups, kBackwardGroups);
  else s.groups = std::min<int64_t>(s.groups, 1 << 20);
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

// A thread to an angle.  position * frequency is a float64 product and its sine and cosine are taken in float64: at position 10^5 a
// float32 angle is off by 4 10^-3.
__global__ __launch_bounds__(256) void rotary_tables_kernel(const int32_t* positions, int64_t n, int axes, int pairs, Frequencies f, float factor,
                                                            float* cos, float* sin) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * pairs) return;
  const int64_t row = i / pairs;
  const int pair = (int)(i - row * pairs);
  const double angle = (double)positions[row * axes + f.axis[pair]] * f.f[pair];
  double s, c;
  ::sincos(angle, &s, &c);
  cos[i] = (float)(c * (double)factor);
  sin[i] = (float)(s * (double)factor);
}

}  // namespace

int launch_rotary_tables(const int32_t* positions, int64_t n, int axes, int pairs, const double* frequencies, const uint8_t* axis, float factor,
                         float* cos, float* sin, hipStream_t stream) {
  Frequencies f = {};
  for (int i = 0; i < pairs; ++i) {
    f.f[i] = frequencies[i];
    f.axis[i] = axis[i];
  }
  hipLaunchKernelGGL(rotary_tables_kernel, dim3((unsigned)((n * pairs + 255) / 256)), dim3(256), 0, stream, positions, n, axes, pairs, f, factor,
                     cos, sin);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

size_t rotary_workspace_bytes(const mfq_rotary_args& a) {
  return ((a.q.dweight ? 1 : 0) + (a.k.dweight ? 1 : 0)) * (size_t)kBackwardGroups * a.dim * 4;
}

int launch_rotary(const mfq_rotary_args& a, bool wide, bool backward, float* workspace, hipStream_t stream) {
  Shape s;
  if (!shape_of(a, wide, backward, s)) return MFQ_EUNSUPPORTED;
  RotaryCall c = {};
  const mfq_rotary_tensor* in[2] = {&a.q, &a.k};
  for (int i = 0; i < 2; ++i) {
    const mfq_rotary_tensor& t = *in[i];
    c.t[i] = {t.x, t.dy, t.weight, t.out, nullptr, t.x_stride[0], t.x_stride[1], t.x_stride[2], t.dy_stride[0], t.dy_stride[1], t.dy_stride[2],
              (int)t.heads};
    if (backward && t.dweight) {
      c.t[i].dw = workspace;
      workspace += (int64_t)kBackwardGroups * a.dim;
    }
  }
  c.cos = a.cos;
  c.sin = a.sin;
  c.positions = a.positions;
  c.position_batch = a.position_batch;
  c.tokens = a.batch * a.tokens;
  c.per_batch = (int)a.tokens;
  c.table_rows = (int)a.table_rows;
  c.dim = a.dim;
  c.rotated = a.rotated;
  c.half_layout = a.layout == MFQ_ROTARY_HALF;
  c.lanes = s.lanes;
  c.passes = s.passes;
  c.chunks = s.chunks;
  c.eps = a.eps;
  int rc;
  if (a.dtype == MFQ_BF16) rc = backward ? launch<BF16, true>(s, c, stream) : launch<BF16, false>(s, c, stream);
  else if (a.dtype == MFQ_F16) rc = backward ? launch<F16, true>(s, c, stream) : launch<F16, false>(s, c, stream);
  else rc = backward ? launch<F32, true>(s, c, stream) : launch<F32, false>(s, c, stream);
  if (rc != MFQ_OK || !backward || (!a.q.dweight && !a.k.dweight)) return rc;
  const dim3 grid((unsigned)((a.dim + 15) / 16), 2);
#define MFQ_WEIGHTS(T) \
  hipLaunchKernelGGL(rotary_weight_kernel<T>, grid, dim3(256), 0, stream, c.t[0].dw, c.t[1].dw, (int)s.groups, a.dim, a.q.dweight, a.k.dweight)
  if (a.dtype == MFQ_BF16) MFQ_WEIGHTS(BF16);
  else if (a.dtype == MFQ_F16) MFQ_WEIGHTS(F16);
  else MFQ_WEIGHTS(F32);
#undef MFQ_WEIGHTS
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

}  // namespace mfq
