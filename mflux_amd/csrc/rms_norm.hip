// RMS norm of rows with the residual's addition in front of it, its gradients, and rows in 8-bit integers with a scale each:
//   s = round(x + residual)                       (or x), what the next block's residual stream goes on with
//   y = round(s r w),  r = 1 / sqrt(mean(s^2) + eps)
//   codes = rint(127 p / max|p|), scale = r max|p| / 127,  p = s w   (without a norm p = x and r = 1)
//   dx = r (w dy - s r^2 mean(w dy s)) + ds,  dw = sum over the rows of dy s r
// All of it is bound by memory: a row is read once, into registers, and written once.  A row takes one wavefront or one
// workgroup of four, whichever has it in at most eight 16-byte pieces a lane; the weight stays in registers from row to row.
// A code does not depend on r, so it is decided by the products p alone, and exactly: where the float32 quotient is within
// 2^-13 of a border between two codes (its own error is below 2^-14), the sign of 254 |p| - (2 l + 1) max|p| in float64
// decides, where both products are exact for the 16-bit types.
// Sums are float32 (eight to some hundred terms a lane, then a tree), in an order that the row's length alone fixes.
#include <type_traits>

#include "rows.h"

namespace mfq {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxChunks = 8;

template <int kCtrl, typename V>
__device__ inline V dpp(V v) {
  return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, false));
}
template <typename V>
__device__ inline V lane_of(V v, int lane) {
  return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ inline float join(float a, float b) { return a + b; }
__device__ inline uint32_t join(uint32_t a, uint32_t b) { return max(a, b); }
__device__ inline uint64_t join(uint64_t a, uint64_t b) { return max(a, b); }
// the sum (of a float) or the largest (of an unsigned) over the 64 lanes, in every lane
template <typename V>
__device__ inline V over_wave(V v) {
  if constexpr (sizeof(V) == 8) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) v = join(v, (V)__shfl_xor((unsigned long long)v, d));
    return v;
  } else {
    v = join(v, dpp<0xB1>(v));   // quad_perm [1,0,3,2]
    v = join(v, dpp<0x4E>(v));   // quad_perm [2,3,0,1]
    v = join(v, dpp<0x141>(v));  // row_half_mirror
    v = join(v, dpp<0x140>(v));  // row_mirror: of the lane's row of 16
    return join(join(lane_of(v, 0), lane_of(v, 16)), join(lane_of(v, 32), lane_of(v, 48)));
  }
}
// the same over a row's lanes: a wavefront, or the workgroup's four, which meet in LDS (two sets of slots in turn, so that
// one barrier is enough)
template <int kLanes, typename A, typename B>
__device__ inline void over_row(A& a, B& b, int turn) {
  a = over_wave(a);
  b = over_wave(b);
  if constexpr (kLanes > kWave) {
    __shared__ A sa[2][kWaves];
    __shared__ B sb[2][kWaves];
    const int wave = threadIdx.x / kWave, set = turn & 1;
    if ((threadIdx.x & (kWave - 1)) == 0) {
      sa[set][wave] = a;
      sb[set][wave] = b;
    }
    __syncthreads();
    a = join(join(sa[set][0], sa[set][1]), join(sa[set][2], sa[set][3]));
    b = join(join(sb[set][0], sb[set][1]), join(sb[set][2], sb[set][3]));
  }
}

template <typename T>
constexpr int kVecOf = 16 / (int)sizeof(typename T::storage);

template <typename T>
__device__ inline void unpack(u32x4 raw, float (&v)[kVecOf<T>]) {
  if constexpr (sizeof(typename T::storage) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = lo_f32<T>(raw[i]);
      v[2 * i + 1] = hi_f32<T>(raw[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(raw[i]);
  }
}
template <typename T>
__device__ inline u32x4 pack(const float (&v)[kVecOf<T>]) {
  u32x4 raw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(typename T::storage) == 2) raw[i] = T::pack2(v[2 * i], v[2 * i + 1]);
    else raw[i] = __float_as_uint(v[i]);
  }
  return raw;
}
template <typename T>
__device__ inline u32x4 add(u32x4 a, u32x4 b) {
  float x[kVecOf<T>], y[kVecOf<T>];
  unpack<T>(a, x);
  unpack<T>(b, y);
#pragma unroll
  for (int i = 0; i < kVecOf<T>; ++i) x[i] += y[i];
  return pack<T>(x);
}

// ---- codes.  The product p of a value and its weight: exact in float32 for the 16-bit types, in float64 for float32.
template <typename T>
using Product = std::conditional_t<sizeof(typename T::storage) == 2, float, double>;
template <typename T>
using Bits = std::conditional_t<sizeof(typename T::storage) == 2, uint32_t, uint64_t>;

// |p| as an unsigned: its order is that of the magnitudes, with infinity above all numbers and NaN above that
template <typename T>
__device__ inline Bits<T> magnitude(Product<T> p) {
  return __builtin_bit_cast(Bits<T>, p) & (~(Bits<T>)0 >> 1);
}

// What the codes of a row are made with
template <typename T>
struct Coder {
  Product<T> top;
  float inverse;
  bool finite, some, tiny;
  __device__ inline Coder(Bits<T> largest) {
    top = __builtin_bit_cast(Product<T>, largest);
    finite = top < (Product<T>)__builtin_inff();
    some = finite && largest;
    tiny = top < (Product<T>)0x1p-100f;  // its inverse may be no float32
    inverse = 127.0f / (float)top;
  }
  // the scale of p's row, p being what it is times `factor`
  __device__ inline float scale(float factor) const { return finite ? (float)top * factor / 127.0f : __builtin_nanf(""); }
  __device__ inline int code(Product<T> p) const {
    if (!some) return 0;
    const Product<T> m = __builtin_bit_cast(Product<T>, magnitude<T>(p));
    const float t = tiny ? (float)((double)m * (127.0 / (double)top)) : (float)m * inverse;
    const float low = __builtin_floorf(t), rest = t - low;
    bool up = rest > 0.5f;
    if (__builtin_fabsf(rest - 0.5f) < 0x1p-13f) {
      const double d = __builtin_fma(254.0, (double)m, -((2.0 * (double)low + 1.0) * (double)top));
      up = d > 0.0 || (d == 0.0 && ((int)low & 1));
    }
    const int c = min((int)low + (up ? 1 : 0), 127);
    return p < 0 ? -c : c;
  }
};

template <typename T>
__device__ inline Product<T> product(float s, float w) {
  return (Product<T>)s * (Product<T>)w;
}

__device__ inline uint32_t pack_codes(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// kLanes lanes to a row, each kChunks of its 16-byte pieces
template <typename T, int kLanes, int kChunks, bool kCodes>
__global__ __launch_bounds__(kThreads) void rows_kernel(RowsCall c) {
  using E = typename T::storage;
  constexpr int V = kVecOf<T>, kRows = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, units = (int)(c.columns / V);
  u32x4 w[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u)
    if (c.weight && lane + u * kLanes < units) w[u] = static_cast<const u32x4*>(c.weight)[lane + u * kLanes];
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes; row < c.rows; row += (int64_t)gridDim.x * kRows, ++turn) {
    const u32x4* x = reinterpret_cast<const u32x4*>(static_cast<const E*>(c.x) + row * c.x_stride);
    const u32x4* residual = reinterpret_cast<const u32x4*>(static_cast<const E*>(c.residual) + row * c.residual_stride);
    u32x4 s[kChunks], r[kChunks];
#pragma unroll
    for (int u = 0; u < kChunks; ++u)
      if (lane + u * kLanes < units) s[u] = x[lane + u * kLanes];
    if (c.residual) {
#pragma unroll
      for (int u = 0; u < kChunks; ++u)
        if (lane + u * kLanes < units) r[u] = residual[lane + u * kLanes];
    }
    float squares = 0.f;
    Bits<T> largest = 0;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      if (c.residual) {
        s[u] = add<T>(s[u], r[u]);
        reinterpret_cast<u32x4*>(static_cast<E*>(c.sum) + row * c.columns)[lane + u * kLanes] = s[u];
      }
      float v[V], g[V];
      unpack<T>(s[u], v);
      if (kCodes && c.weight) unpack<T>(w[u], g);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        squares = __builtin_fmaf(v[i], v[i], squares);
        if constexpr (kCodes) largest = join(largest, magnitude<T>(c.weight ? product<T>(v[i], g[i]) : (Product<T>)v[i]));
      }
    }
    over_row<kLanes>(squares, largest, turn);
    const float rstd = c.norm ? 1.0f / __builtin_sqrtf(squares / (float)c.columns + c.eps) : 1.0f;
    const Coder<T> coder(largest);
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      float v[V], g[V];
      unpack<T>(s[u], v);
      if (c.weight) unpack<T>(w[u], g);
      if constexpr (kCodes) {
        uint32_t packed[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          int k[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) k[e] = coder.code(c.weight ? product<T>(v[4 * i + e], g[4 * i + e]) : (Product<T>)v[4 * i + e]);
          packed[i] = pack_codes(k[0], k[1], k[2], k[3]);
        }
        int8_t* to = c.codes + row * c.code_stride + (int64_t)(lane + u * kLanes) * V;
        if constexpr (V == 8) *reinterpret_cast<u32x2*>(to) = u32x2{packed[0], packed[1]};
        else *reinterpret_cast<uint32_t*>(to) = packed[0];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[i] *= rstd;
          if (c.weight) v[i] *= g[i];
        }
        reinterpret_cast<u32x4*>(static_cast<E*>(c.y) + row * c.columns)[lane + u * kLanes] = pack<T>(v);
      }
    }
    if (kCodes && lane == 0) c.scales[row] = coder.scale(rstd);
  }
}

// Rows of any length, alignment and stride: a workgroup to a row, element by element, which is read again (from a cache,
// where it fits one) for the results.
template <typename T, bool kCodes>
__global__ __launch_bounds__(kThreads) void rows_any_kernel(RowsCall c) {
  using E = typename T::storage;
  const E* weight = static_cast<const E*>(c.weight);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < c.rows; row += gridDim.x, ++turn) {
    const E* x = static_cast<const E*>(c.x) + row * c.x_stride;
    const E* residual = static_cast<const E*>(c.residual) + row * c.residual_stride;
    auto value = [&](int64_t k) __attribute__((always_inline)) {
      return c.residual ? T::to_f32(T::from_f32(T::to_f32(x[k]) + T::to_f32(residual[k]))) : T::to_f32(x[k]);
    };
    float squares = 0.f;
    Bits<T> largest = 0;
    for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
      const float s = value(k);
      if (c.residual) static_cast<E*>(c.sum)[row * c.columns + k] = T::from_f32(s);
      squares = __builtin_fmaf(s, s, squares);
      if constexpr (kCodes) largest = join(largest, magnitude<T>(weight ? product<T>(s, T::to_f32(weight[k])) : (Product<T>)s));
    }
    over_row<kThreads>(squares, largest, turn);
    const float rstd = c.norm ? 1.0f / __builtin_sqrtf(squares / (float)c.columns + c.eps) : 1.0f;
    const Coder<T> coder(largest);
    for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
      float s = value(k);
      if constexpr (kCodes) {
        c.codes[row * c.code_stride + k] = (int8_t)coder.code(weight ? product<T>(s, T::to_f32(weight[k])) : (Product<T>)s);
      } else {
        s *= rstd;
        if (weight) s *= T::to_f32(weight[k]);
        static_cast<E*>(c.y)[row * c.columns + k] = T::from_f32(s);
      }
    }
    if (kCodes && threadIdx.x == 0) c.scales[row] = coder.scale(rstd);
  }
}

// ---- gradients
template <typename T, int kLanes, int kChunks, bool kWeight>
__global__ __launch_bounds__(kThreads) void rows_backward_kernel(RowsCall c) {
  using E = typename T::storage;
  constexpr int V = kVecOf<T>, kRows = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, units = (int)(c.columns / V);
  u32x4 w[kChunks];
  float dw[kWeight ? kChunks : 1][V];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    if (c.weight && lane + u * kLanes < units) w[u] = static_cast<const u32x4*>(c.weight)[lane + u * kLanes];
    if constexpr (kWeight) {
#pragma unroll
      for (int i = 0; i < V; ++i) dw[u][i] = 0.f;
    }
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes; row < c.rows; row += (int64_t)gridDim.x * kRows, ++turn) {
    const u32x4* x = reinterpret_cast<const u32x4*>(static_cast<const E*>(c.x) + row * c.x_stride);
    const u32x4* dy = reinterpret_cast<const u32x4*>(static_cast<const E*>(c.dy) + row * c.dy_stride);
    const u32x4* dsum = reinterpret_cast<const u32x4*>(static_cast<const E*>(c.dsum) + row * c.dsum_stride);
    u32x4 s[kChunks], g[kChunks], d[kChunks];
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      s[u] = x[lane + u * kLanes];
      g[u] = dy[lane + u * kLanes];
      if (c.dsum && c.dx) d[u] = dsum[lane + u * kLanes];
    }
    float squares = 0.f, dot = 0.f;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      float v[V], a[V], b[V];
      unpack<T>(s[u], v);
      unpack<T>(g[u], a);
      if (c.weight) unpack<T>(w[u], b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        squares = __builtin_fmaf(v[i], v[i], squares);
        dot = __builtin_fmaf(c.weight ? a[i] * b[i] : a[i], v[i], dot);
      }
    }
    over_row<kLanes>(squares, dot, turn);
    const float rstd = 1.0f / __builtin_sqrtf(squares / (float)c.columns + c.eps), mean = rstd * dot / (float)c.columns;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      float v[V], a[V], b[V];
      unpack<T>(s[u], v);
      unpack<T>(g[u], a);
      if (c.weight) unpack<T>(w[u], b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float n = v[i] * rstd;
        if constexpr (kWeight) dw[u][i] = __builtin_fmaf(a[i], n, dw[u][i]);
        a[i] = rstd * __builtin_fmaf(-mean, n, c.weight ? a[i] * b[i] : a[i]);
      }
      if (!c.dx) continue;
      if (c.dsum) {
        unpack<T>(d[u], b);
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] += b[i];
      }
      reinterpret_cast<u32x4*>(static_cast<E*>(c.dx) + row * c.columns)[lane + u * kLanes] = pack<T>(a);
    }
  }
  if constexpr (kWeight) {  // the workgroup's sums: one row of the partial sums
    float* parts = c.parts + (int64_t)blockIdx.x * c.columns;
    if constexpr (kRows == 1) {
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        if (lane + u * kLanes >= units) continue;
#pragma unroll
        for (int i = 0; i < V; i += 4)
          *reinterpret_cast<f32x4*>(parts + (int64_t)(lane + u * kLanes) * V + i) = f32x4{dw[u][i], dw[u][i + 1], dw[u][i + 2], dw[u][i + 3]};
      }
    } else {
      __shared__ float sums[kRows][kLanes * kChunks * V];
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        if (lane + u * kLanes >= units) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) sums[threadIdx.x / kLanes][(lane + u * kLanes) * V + i] = dw[u][i];
      }
      __syncthreads();
      for (int k = threadIdx.x; k < (int)c.columns; k += kThreads) {
        float v = sums[0][k];
#pragma unroll
        for (int i = 1; i < kRows; ++i) v += sums[i][k];
        parts[k] = v;
      }
    }
  }
}

// of any length, alignment and stride; a workgroup adds its rows' shares of the weight's gradient up in its own row of `parts`
template <typename T>
__global__ __launch_bounds__(kThreads) void rows_backward_any_kernel(RowsCall c) {
  using E = typename T::storage;
  const E* weight = static_cast<const E*>(c.weight);
  float* parts = c.parts ? c.parts + (int64_t)blockIdx.x * c.columns : nullptr;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < c.rows; row += gridDim.x, ++turn) {
    const E* x = static_cast<const E*>(c.x) + row * c.x_stride;
    const E* dy = static_cast<const E*>(c.dy) + row * c.dy_stride;
    const E* dsum = static_cast<const E*>(c.dsum) + row * c.dsum_stride;
    float squares = 0.f, dot = 0.f;
    for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
      const float s = T::to_f32(x[k]), a = T::to_f32(dy[k]);
      squares = __builtin_fmaf(s, s, squares);
      dot = __builtin_fmaf(weight ? a * T::to_f32(weight[k]) : a, s, dot);
    }
    over_row<kThreads>(squares, dot, turn);
    const float rstd = 1.0f / __builtin_sqrtf(squares / (float)c.columns + c.eps), mean = rstd * dot / (float)c.columns;
    for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
      const float n = T::to_f32(x[k]) * rstd, a = T::to_f32(dy[k]);
      if (parts) parts[k] = turn ? __builtin_fmaf(a, n, parts[k]) : a * n;
      if (!c.dx) continue;
      float d = rstd * __builtin_fmaf(-mean, n, weight ? a * T::to_f32(weight[k]) : a);
      if (c.dsum) d += T::to_f32(dsum[k]);
      static_cast<E*>(c.dx)[row * c.columns + k] = T::from_f32(d);
    }
  }
}

// dw = sum of the workgroups' partial sums: a workgroup to 16 columns, 64 threads to a column
template <typename T>
__global__ __launch_bounds__(1024) void rows_weight_kernel(const float* parts, int n, int64_t columns, void* dw) {
  const int64_t column = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const int part = threadIdx.x >> 4;
  float v = 0.f;
  if (column < columns) {
#pragma unroll 8
    for (int i = part; i < n; i += 64) v += parts[i * columns + column];
  }
  __shared__ float sums[64][17];
  sums[part][threadIdx.x & 15] = v;
  __syncthreads();
  if (part || column >= columns) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) v += sums[i][threadIdx.x & 15];
  static_cast<typename T::storage*>(dw)[column] = T::from_f32(v);
}

// ---- codes times their row's scale
template <typename T, bool kWide>
__global__ __launch_bounds__(kThreads) void rows_values_kernel(const int8_t* codes, int64_t stride, const float* scales, int64_t rows,
                                                               int64_t columns, void* out) {
  using E = typename T::storage;
  constexpr int kEach = kWide ? 16 : 1;
  const int64_t per_row = columns / kEach, n = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / per_row, k = (i - row * per_row) * kEach;
    const float scale = scales[row];
    E* to = static_cast<E*>(out) + row * columns + k;
    if constexpr (kWide) {
      const u32x4 raw = *reinterpret_cast<const u32x4*>(codes + row * stride + k);
      constexpr int V = kVecOf<T>;
#pragma unroll
      for (int p = 0; p < 16 / V; ++p) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)(int8_t)(raw[(p * V + e) / 4] >> (8 * (e & 3))) * scale;
        reinterpret_cast<u32x4*>(to)[p] = pack<T>(v);
      }
    } else {
      *to = T::from_f32((float)codes[row * stride + k] * scale);
    }
  }
}

// lanes of a row and 16-byte pieces of a lane; false: the row does not fit the registers
bool form_of(int64_t units, int& lanes, int& chunks) {
  lanes = units <= 4 * kWave ? kWave : kThreads;
  const int64_t each = (units + lanes - 1) / lanes;
  chunks = 1;
  while (chunks < each) chunks *= 2;
  return chunks <= kMaxChunks;
}

constexpr int kBackwardGroups = 2;  // workgroups of a backward pass to a compute unit: rows of partial sums

int64_t groups_of(int64_t rows, int per_group, int64_t most) {
  const int64_t groups = (rows + per_group - 1) / per_group, each = (groups + most - 1) / most;
  return (groups + each - 1) / each;
}

template <typename T, int kLanes, int kChunks>
void launch_form(const RowsCall& c, bool backward, int64_t groups, hipStream_t stream) {
  const dim3 grid((unsigned)groups), block(kThreads);
  if (backward) {
    if (c.parts) hipLaunchKernelGGL((rows_backward_kernel<T, kLanes, kChunks, true>), grid, block, 0, stream, c);
    else hipLaunchKernelGGL((rows_backward_kernel<T, kLanes, kChunks, false>), grid, block, 0, stream, c);
  } else if (c.codes) {
    hipLaunchKernelGGL((rows_kernel<T, kLanes, kChunks, true>), grid, block, 0, stream, c);
  } else {
    hipLaunchKernelGGL((rows_kernel<T, kLanes, kChunks, false>), grid, block, 0, stream, c);
  }
}

template <typename T>
int launch(const RowsCall& c, bool wide, bool backward, hipStream_t stream) {
  int lanes, chunks;
  const bool fits = wide && form_of(c.columns / kVecOf<T>, lanes, chunks);
  int64_t groups;
  if (!fits) {
    groups = groups_of(c.rows, 1, (backward ? kBackwardGroups : 8) * (int64_t)compute_units());
    const dim3 grid((unsigned)groups), block(kThreads);
    if (backward) hipLaunchKernelGGL((rows_backward_any_kernel<T>), grid, block, 0, stream, c);
    else if (c.codes) hipLaunchKernelGGL((rows_any_kernel<T, true>), grid, block, 0, stream, c);
    else hipLaunchKernelGGL((rows_any_kernel<T, false>), grid, block, 0, stream, c);
  } else {
    groups = groups_of(c.rows, kThreads / lanes, (backward ? kBackwardGroups : 8) * (int64_t)compute_units());
    if (lanes == kWave) {
      if (chunks == 1) launch_form<T, kWave, 1>(c, backward, groups, stream);
      else if (chunks == 2) launch_form<T, kWave, 2>(c, backward, groups, stream);
      else launch_form<T, kWave, 4>(c, backward, groups, stream);
    } else {
      if (chunks <= 2) launch_form<T, kThreads, 2>(c, backward, groups, stream);
      else if (chunks == 4) launch_form<T, kThreads, 4>(c, backward, groups, stream);
      else launch_form<T, kThreads, 8>(c, backward, groups, stream);
    }
  }
  if (hipGetLastError() != hipSuccess) return MFQ_ELAUNCH;
  if (!backward || !c.parts) return MFQ_OK;
  hipLaunchKernelGGL(rows_weight_kernel<T>, dim3((unsigned)((c.columns + 15) / 16)), dim3(1024), 0, stream, c.parts, (int)groups, c.columns,
                     c.dweight);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

}  // namespace

size_t rows_workspace_bytes(int64_t rows, int64_t columns) {
  const int64_t most = kBackwardGroups * (int64_t)compute_units();
  return (size_t)(rows < most ? rows : most) * (size_t)columns * 4;
}

int launch_rows(int dtype, const RowsCall& c, bool wide, bool backward, hipStream_t stream) {
  if (dtype == MFQ_BF16) return launch<BF16>(c, wide, backward, stream);
  if (dtype == MFQ_F16) return launch<F16>(c, wide, backward, stream);
  return launch<F32>(c, wide, backward, stream);
}

int launch_rows_values(const int8_t* codes, int64_t stride, const float* scales, int64_t rows, int64_t columns, int dtype, void* out,
                       hipStream_t stream) {
  const bool wide = columns % 16 == 0 && stride % 16 == 0 && aligned16(codes) && aligned16(out);
  const int64_t n = rows * (wide ? columns / 16 : columns), most = 16 * (int64_t)compute_units();
  const dim3 grid((unsigned)((n + kThreads - 1) / kThreads < most ? (n + kThreads - 1) / kThreads : most)), block(kThreads);
#define MFQ_VALUES(T)                                                                                                            \
  if (wide) hipLaunchKernelGGL((rows_values_kernel<T, true>), grid, block, 0, stream, codes, stride, scales, rows, columns, out); \
  else hipLaunchKernelGGL((rows_values_kernel<T, false>), grid, block, 0, stream, codes, stride, scales, rows, columns, out)
  if (dtype == MFQ_BF16) {
    MFQ_VALUES(BF16);
  } else if (dtype == MFQ_F16) {
    MFQ_VALUES(F16);
  } else {
    MFQ_VALUES(F32);
  }
#undef MFQ_VALUES
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

}  // namespace mfq
