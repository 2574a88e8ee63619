// RMS norm of rows with the residual's addition in front of it, its gradients, and rows in 8-bit integers with a scale each:
//   s = round(x + residual)                       (or x), what the next block's residual stream goes on with
//   y = round(s r w),  r = 1 / sqrt(mean(s^2) + eps)
//   codes = rint(127 p / max|p|), scale = r max|p| / 127,  p = s w   (without a norm p = x and r = 1)
//   dx = r (w dy - s r^2 mean(w dy s)) + ds,  dw = sum over the rows of dy s r
// All of it is bound by memory: a row is read once, into registers, and written once.  A row takes a wavefront or a workgroup of 2 to
// 16, by its length; the weight stays in registers from row to row.
// A code does not depend on r, so it is decided by the products p alone, and exactly: where the float32 quotient is next to a
// border between two codes it is taken again in float64, which tells 16-bit types' products apart.
// A row's sums are float32 where registers hold it (up to 32 terms a lane, then a tree), and float64, or 32 terms at a time in float32 and
// these in float64, where they do not: in an order that its length and alignment alone fix.
#include <type_traits>

#include "rows.h"

namespace mfq {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;  // of the kernels that are not a row's lanes wide

template <int kCtrl, typename V>
__device__ inline V dpp(V v) {
  if constexpr (sizeof(V) == 8) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(V, u32x2{dpp<kCtrl>(w[0]), dpp<kCtrl>(w[1])});
  } else {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, false));
  }
}
template <typename V>
__device__ inline V lane_of(V v, int lane) {
  if constexpr (sizeof(V) == 8) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(V, u32x2{lane_of(w[0], lane), lane_of(w[1], lane)});
  } else {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  }
}
__device__ inline float join(float a, float b) { return a + b; }
__device__ inline double join(double a, double b) { return a + b; }
__device__ inline uint32_t join(uint32_t a, uint32_t b) { return max(a, b); }
__device__ inline uint64_t join(uint64_t a, uint64_t b) { return max(a, b); }
// the sum (of floating point numbers) or the largest (of an unsigned) over the 64 lanes, in every lane
template <typename V>
__device__ inline V over_wave(V v) {
  if constexpr (std::is_same_v<V, uint64_t>) {  // by shuffles, which leave the lanes' own work its place: 20000 x 77 10.6 us, without them 11.1
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) v = join(v, (V)__shfl_xor((unsigned long long)v, d));
    return v;
  }
  v = join(v, dpp<0xB1>(v));   // quad_perm [1,0,3,2]
  v = join(v, dpp<0x4E>(v));   // quad_perm [2,3,0,1]
  v = join(v, dpp<0x141>(v));  // row_half_mirror
  v = join(v, dpp<0x140>(v));  // row_mirror: of the lane's row of 16
  return join(join(lane_of(v, 0), lane_of(v, 16)), join(lane_of(v, 32), lane_of(v, 48)));
}
// the same over a row's lanes: a wavefront, or a workgroup's, which meet in LDS (two sets of slots in turn, so that one barrier is
// enough: `turn` counts the calls)
template <int kLanes, typename A, typename B>
__device__ inline void over_row(A& a, B& b, int turn) {
  a = over_wave(a);
  b = over_wave(b);
  if constexpr (kLanes > kWave) {
    constexpr int kWaves = kLanes / kWave;
    __shared__ A sa[2][kWaves];
    __shared__ B sb[2][kWaves];
    const int wave = threadIdx.x / kWave, set = turn & 1;
    if ((threadIdx.x & (kWave - 1)) == 0) {
      sa[set][wave] = a;
      sb[set][wave] = b;
    }
    __syncthreads();
    a = sa[set][0];
    b = sb[set][0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
      a = join(a, sa[set][i]);
      b = join(b, sb[set][i]);
    }
  }
}

template <typename T>
constexpr int kVecOf = 16 / (int)sizeof(typename T::storage);

// A unit of a row: 16 bytes, or one element where rows are not whole and aligned 16 bytes
template <typename T, int V>
using Unit = std::conditional_t<V == 1, typename T::storage, u32x4>;

template <typename T, int V>
__device__ inline void unpack(const Unit<T, V>& raw, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = T::to_f32(raw);
  } else if constexpr (sizeof(typename T::storage) == 2) {
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
template <typename T, int V>
__device__ inline Unit<T, V> pack(const float (&v)[V]) {
  if constexpr (V == 1) {
    return T::from_f32(v[0]);
  } else {
    u32x4 raw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(typename T::storage) == 2) raw[i] = T::pack2(v[2 * i], v[2 * i + 1]);
      else raw[i] = __float_as_uint(v[i]);
    }
    return raw;
  }
}
template <typename T, int V>
__device__ inline Unit<T, V> add(const Unit<T, V>& a, const Unit<T, V>& b) {
  float x[V], y[V];
  unpack<T, V>(a, x);
  unpack<T, V>(b, y);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] += y[i];
  return pack<T, V>(x);
}

// ---- rows whose sum of squares float32 does not hold: it overflows for values above some 10^17, and squares below its normal numbers count
// for values below 10^-19 with as small an eps.  The values of such a row are multiplied by a power of two, in the registers that hold
// them, and its sums are taken again.  A branch for all of the row's lanes, and nothing else in the way of other rows: 4352 x 3840
// bfloat16 22.0 -> 22.1 us, its gradients 25.6 -> 26.1 (in float64, from memory or behind the other rows: up to 1.5 times as much, by the
// registers that it takes from them).
template <typename T>
constexpr bool kFarValues = !std::is_same_v<T, F16>;  // float16 has no such values
// of a sum that all of the row's lanes have, and its mean with eps
__device__ inline bool far_row(float squares, float size) {
  return __builtin_amdgcn_readfirstlane((int)!(squares <= 0x1.fffffep127f && size >= 0x1p-120f));
}
// the power of two: 2^15 values below 2^128, or values down to 2^-149, whose squares float32 then adds up
__device__ inline float lift_of(float squares) { return squares <= 0x1.fffffep127f ? 0x1p100f : 0x1p-73f; }
template <typename T, int V>
__device__ inline Unit<T, V> lifted(const Unit<T, V>& raw, float lift) {
  float v[V];
  unpack<T, V>(raw, v);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] *= lift;
  return pack<T, V>(v);
}

// ---- codes.  The product p of a value and its weight: exact in float32 for the 16-bit types, in float64 for float32.
template <typename T, bool kWeighted>
using Product = std::conditional_t<kWeighted && sizeof(typename T::storage) == 4, double, float>;
template <typename P>
using Bits = std::conditional_t<sizeof(P) == 8, uint64_t, uint32_t>;

// |p| as an unsigned: its order is that of the magnitudes, with infinity above all numbers and NaN above that
template <typename P>
__device__ inline Bits<P> magnitude(P p) {
  return __builtin_bit_cast(Bits<P>, p) & (~(Bits<P>)0 >> 1);
}

// What the codes of a row are made with
template <typename P>
struct Coder {
  P top;
  float inverse;
  bool finite, some, far;
  __device__ inline Coder(Bits<P> largest) {
    top = __builtin_bit_cast(P, largest);
    finite = top < (P)__builtin_inff();
    some = finite && largest;
    far = top < (P)0x1p-100f || top > (P)0x1p120f;  // its inverse may be no normal float32
    inverse = 127.0f / (float)top;
  }
  // the scale of p's row, p being what it is times `factor`
  __device__ inline float scale(float factor) const { return finite ? (float)(top * (P)factor / (P)127) : __builtin_nanf(""); }
  __device__ inline float scale(double factor) const { return finite ? (float)((double)top * factor / 127.0) : __builtin_nanf(""); }
  // The codes of N products, in the low bytes, the first lowest.  Adding 1.5 2^23 rounds a quotient to a whole number, ties to even,
  // and leaves it in the sum's low bits; what the sum lost is how far the quotient is from it.  p * inverse is off by at most
  // 127 * 4 * 2^-24 < 2^-14 (the inverse, the product, and for float32 the rounding of p and max|p|).
  template <int N>
  __device__ inline uint32_t codes(const P (&p)[N]) const {
    if (!some) return 0;
    float sum[N], off = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = (float)p[i];
      sum[i] = __builtin_fmaf(v, inverse, 12582912.0f);
      off = __builtin_fmaxf(off, __builtin_fabsf(__builtin_fmaf(v, inverse, 12582912.0f - sum[i])));
    }
    if (far || off > 0.5f - 0x1p-14f) {  // one of them is next to a border
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] = 12582912.0f + (float)__builtin_rint(127.0 * (double)p[i] / (double)top);
    }
    if constexpr (N == 1) return __float_as_uint(sum[0]);
    const uint32_t low = __builtin_amdgcn_perm(__float_as_uint(sum[1 % N]), __float_as_uint(sum[0]), 0x0c0c0400u);
    return low | __builtin_amdgcn_perm(__float_as_uint(sum[3 % N]), __float_as_uint(sum[2 % N]), 0x04000c0cu);
  }
};

enum Result { kNormalised, kCodes, kNormalisedCodes, kWeightedCodes };  // kCodes: of the values as they are, without a norm

// kLanes lanes to a row, each kChunks of its units of V elements; up to 256 threads, workgroups of several rows.  4352 x 3840
// bfloat16 with a residual 22.4 us (6.0 TB/s, part of it from the last cache), with codes 22.4; 10240 x 3840 into codes without a norm 28;
// a few rows 4, a launch and one trip to memory each way.  Element by element (rows of no whole 16 bytes) 4096 x 4099 takes 43.
template <typename T, int V, int kLanes, int kChunks, int kResult>
__global__ __launch_bounds__(kLanes > kWave ? kLanes : kThreads) void rows_kernel(RowsCall c) {
  using E = typename T::storage;
  using U = Unit<T, V>;
  constexpr bool kCoded = kResult != kNormalised, kNorm = kResult != kCodes;
  using P = Product<T, kResult == kWeightedCodes>;
  constexpr int kRows = kLanes > kWave ? 1 : kThreads / kWave;
  const int lane = threadIdx.x % kLanes, units = (int)(c.columns / V);
  const bool weighted = kCoded ? kResult == kWeightedCodes : c.weight != nullptr;
  U w[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u)
    if (weighted && lane + u * kLanes < units) w[u] = static_cast<const U*>(c.weight)[lane + u * kLanes];
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes; row < c.rows; row += (int64_t)gridDim.x * kRows) {
    const U* x = reinterpret_cast<const U*>(static_cast<const E*>(c.x) + row * c.x_stride);
    const U* residual = reinterpret_cast<const U*>(static_cast<const E*>(c.residual) + row * c.residual_stride);
    U s[kChunks], r[kChunks];
#pragma unroll
    for (int u = 0; u < kChunks; ++u)
      if (lane + u * kLanes < units) s[u] = x[lane + u * kLanes];
    if (c.residual) {
#pragma unroll
      for (int u = 0; u < kChunks; ++u)
        if (lane + u * kLanes < units) r[u] = residual[lane + u * kLanes];
    }
    auto products = [&](int u, P (&p)[V]) __attribute__((always_inline)) {
      float v[V], g[V];
      unpack<T, V>(s[u], v);
      if constexpr (kResult == kWeightedCodes) unpack<T, V>(w[u], g);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (kResult == kWeightedCodes) p[i] = (P)v[i] * (P)g[i];
        else p[i] = v[i];
      }
    };
    float squares = 0.f;
    Bits<P> largest = 0;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      if (c.residual) {
        s[u] = add<T, V>(s[u], r[u]);
        reinterpret_cast<U*>(static_cast<E*>(c.sum) + row * c.columns)[lane + u * kLanes] = s[u];
      }
      float v[V];
      unpack<T, V>(s[u], v);
#pragma unroll
      for (int i = 0; kNorm && i < V; ++i) squares = __builtin_fmaf(v[i], v[i], squares);
      if constexpr (kCoded) {
        P p[V];
        products(u, p);
#pragma unroll
        for (int i = 0; i < V; ++i) largest = join(largest, magnitude(p[i]));
      }
    }
    over_row<kLanes>(squares, largest, turn++);
    const float size = squares / (float)c.columns + c.eps;
    float rstd = kNorm ? 1.0f / __builtin_sqrtf(size) : 1.0f;
    const Coder<P> coder(largest);
    float scale = kCoded ? coder.scale(rstd) : 0.f;
    if (kFarValues<T> && kNorm && far_row(squares, size)) {
      const float lift = lift_of(squares);
      squares = 0.f;
      Bits<P> none = 0;
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        if (lane + u * kLanes >= units) continue;
        const U t = lifted<T, V>(s[u], lift);
        float v[V];
        unpack<T, V>(t, v);
#pragma unroll
        for (int i = 0; i < V; ++i) squares = __builtin_fmaf(v[i], v[i], squares);
        if constexpr (!kCoded) s[u] = t;
      }
      over_row<kLanes>(squares, none, turn++);
      rstd = 1.0f / __builtin_sqrtf(squares / (float)c.columns + c.eps * lift * lift);
      if constexpr (kCoded) scale = coder.scale((double)rstd * (double)lift);
    }
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      if constexpr (kCoded) {
        P p[V];
        products(u, p);
        int8_t* to = c.codes + row * c.code_stride + (int64_t)(lane + u * kLanes) * V;
        if constexpr (V == 1) {
          *to = (int8_t)coder.codes(p);
        } else {
          uint32_t packed[V / 4];
#pragma unroll
          for (int i = 0; i < V / 4; ++i) {
            const P four[4] = {p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]};
            packed[i] = coder.codes(four);
          }
          if constexpr (V == 8) *reinterpret_cast<u32x2*>(to) = u32x2{packed[0], packed[1]};
          else *reinterpret_cast<uint32_t*>(to) = packed[0];
        }
      } else {
        float v[V], g[V];
        unpack<T, V>(s[u], v);
        if (weighted) unpack<T, V>(w[u], g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[i] *= rstd;
          if (weighted) v[i] *= g[i];
        }
        reinterpret_cast<U*>(static_cast<E*>(c.y) + row * c.columns)[lane + u * kLanes] = pack<T, V>(v);
      }
    }
    if (kCoded && lane == 0) c.scales[row] = scale;
  }
}

// Rows that no registers hold: a workgroup to a row, element by element, which is read again (from a cache, where it fits one) for
// the results.  A thread's sum has up to 2^20 terms and is float64 (equal values of a row of 2^22 would drift 10^-4 away in float32).
template <typename T, int kResult>
__global__ __launch_bounds__(kThreads) void rows_any_kernel(RowsCall c) {
  using E = typename T::storage;
  constexpr bool kCoded = kResult != kNormalised, kNorm = kResult != kCodes;
  using P = Product<T, kResult == kWeightedCodes>;
  const E* weight = static_cast<const E*>(c.weight);
  const double share = 1.0 / (double)c.columns;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < c.rows; row += gridDim.x, ++turn) {
    const E* x = static_cast<const E*>(c.x) + row * c.x_stride;
    const E* residual = static_cast<const E*>(c.residual) + row * c.residual_stride;
    auto value = [&](int64_t k) __attribute__((always_inline)) {
      return c.residual ? T::to_f32(T::from_f32(T::to_f32(x[k]) + T::to_f32(residual[k]))) : T::to_f32(x[k]);
    };
    auto product = [&](float s, int64_t k) __attribute__((always_inline)) {
      if constexpr (kResult == kWeightedCodes) return (P)s * (P)T::to_f32(weight[k]);
      else return (P)s;
    };
    double squares = 0.;
    Bits<P> largest = 0;
    for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
      const float s = value(k);
      if (c.residual) static_cast<E*>(c.sum)[row * c.columns + k] = T::from_f32(s);
      if (kNorm) squares = __builtin_fma((double)s, (double)s, squares);
      if constexpr (kCoded) largest = join(largest, magnitude(product(s, k)));
    }
    over_row<kThreads>(squares, largest, turn);
    const double root = kNorm ? 1.0 / __builtin_sqrt(squares * share + (double)c.eps) : 1.0;
    // the root as two factors where float32 may not hold it, in the order whose first product stays inside
    const float lift = !kFarValues<T> ? 1.f : root < 0x1p-60 ? 0x1p-84f : root > 0x1p60 ? 0x1p100f : 1.f, rstd = (float)(root / (double)lift);
    const float first = lift > 1.f ? lift : rstd, second = lift > 1.f ? rstd : lift;
    const Coder<P> coder(largest);
    for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
      float s = value(k);
      if constexpr (kCoded) {
        const P p[1] = {product(s, k)};
        c.codes[row * c.code_stride + k] = (int8_t)coder.codes(p);
      } else {
        s = s * first * second;
        if (weight) s *= T::to_f32(weight[k]);
        static_cast<E*>(c.y)[row * c.columns + k] = T::from_f32(s);
      }
    }
    if (kCoded && threadIdx.x == 0) c.scales[row] = kNorm ? coder.scale(root) : coder.scale(1.f);
  }
}

// ---- gradients.  A row's two sums are taken again from what was normalised (one more read instead of one more array), so a pass
// reads three arrays and writes one: 4099 x 4096 bfloat16 26.1 us (5.1 TB/s), and 4 for the partial sums' own kernel.  Element by
// element 4096 x 4099 takes 136.
template <typename T, int V, int kLanes, int kChunks, bool kWeight>
__global__ __launch_bounds__(kLanes > kWave ? kLanes : kThreads) void rows_backward_kernel(RowsCall c) {
  using E = typename T::storage;
  using U = Unit<T, V>;
  constexpr int kRows = kLanes > kWave ? 1 : kThreads / kWave;
  const int lane = threadIdx.x % kLanes, units = (int)(c.columns / V);
  U w[kChunks];
  float dw[kWeight ? kChunks : 1][V];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    if (c.weight && lane + u * kLanes < units) w[u] = static_cast<const U*>(c.weight)[lane + u * kLanes];
    if constexpr (kWeight) {
#pragma unroll
      for (int i = 0; i < V; ++i) dw[u][i] = 0.f;
    }
  }
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes; row < c.rows; row += (int64_t)gridDim.x * kRows) {
    const U* x = reinterpret_cast<const U*>(static_cast<const E*>(c.x) + row * c.x_stride);
    const U* dy = reinterpret_cast<const U*>(static_cast<const E*>(c.dy) + row * c.dy_stride);
    const U* dsum = reinterpret_cast<const U*>(static_cast<const E*>(c.dsum) + row * c.dsum_stride);
    U s[kChunks], g[kChunks], d[kChunks];
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
      unpack<T, V>(s[u], v);
      unpack<T, V>(g[u], a);
      if (c.weight) unpack<T, V>(w[u], b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        squares = __builtin_fmaf(v[i], v[i], squares);
        dot = __builtin_fmaf(c.weight ? a[i] * b[i] : a[i], v[i], dot);
      }
    }
    over_row<kLanes>(squares, dot, turn++);
    const float size = squares / (float)c.columns + c.eps;
    float rstd = 1.0f / __builtin_sqrtf(size), slope = rstd;  // r of what is in registers, and r
    if (kFarValues<T> && far_row(squares, size)) {
      const float lift = lift_of(squares);
      squares = dot = 0.f;
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        if (lane + u * kLanes >= units) continue;
        s[u] = lifted<T, V>(s[u], lift);
        float v[V], a[V], b[V];
        unpack<T, V>(s[u], v);
        unpack<T, V>(g[u], a);
        if (c.weight) unpack<T, V>(w[u], b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          squares = __builtin_fmaf(v[i], v[i], squares);
          dot = __builtin_fmaf(c.weight ? a[i] * b[i] : a[i], v[i], dot);
        }
      }
      over_row<kLanes>(squares, dot, turn++);
      rstd = 1.0f / __builtin_sqrtf(squares / (float)c.columns + c.eps * lift * lift);
      slope = rstd * lift;
    }
    const float mean = rstd * dot / (float)c.columns;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
      float v[V], a[V], b[V];
      unpack<T, V>(s[u], v);
      unpack<T, V>(g[u], a);
      if (c.weight) unpack<T, V>(w[u], b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float n = v[i] * rstd;
        if constexpr (kWeight) dw[u][i] = __builtin_fmaf(a[i], n, dw[u][i]);
        a[i] = slope * __builtin_fmaf(-mean, n, c.weight ? a[i] * b[i] : a[i]);
      }
      if (!c.dx) continue;
      if (c.dsum) {
        unpack<T, V>(d[u], b);
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] += b[i];
      }
      reinterpret_cast<U*>(static_cast<E*>(c.dx) + row * c.columns)[lane + u * kLanes] = pack<T, V>(a);
    }
  }
  if constexpr (kWeight) {  // the workgroup's sums: one row of the partial sums
    float* parts = c.parts + (int64_t)blockIdx.x * c.columns;
    __shared__ float sums[kRows > 1 ? kRows : 1][kRows > 1 ? kLanes * kChunks * V : 1];
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (lane + u * kLanes >= units) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (kRows > 1) sums[threadIdx.x / kLanes][(lane + u * kLanes) * V + i] = dw[u][i];
        else parts[(int64_t)(lane + u * kLanes) * V + i] = dw[u][i];
      }
    }
    if constexpr (kRows > 1) {
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

constexpr int kAtATime = 32;  // terms of a thread's sums in float32, before they go on in float64 (all of them there: 1.2 times as long in float32)

// rows that no registers hold; a workgroup adds its rows' shares of the weight's gradient up in its own row of `parts`
template <typename T>
__global__ __launch_bounds__(kThreads) void rows_backward_any_kernel(RowsCall c) {
  using E = typename T::storage;
  const E* weight = static_cast<const E*>(c.weight);
  float* parts = c.parts ? c.parts + (int64_t)blockIdx.x * c.columns : nullptr;
  const double share = 1.0 / (double)c.columns;
  int turn = 0;
  bool added = false;
  for (int64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
    const E* x = static_cast<const E*>(c.x) + row * c.x_stride;
    const E* dy = static_cast<const E*>(c.dy) + row * c.dy_stride;
    const E* dsum = static_cast<const E*>(c.dsum) + row * c.dsum_stride;
    double squares = 0., dot = 0.;
    for (int64_t from = threadIdx.x; from < c.columns; from += kAtATime * kThreads) {
      const int64_t to = min(from + kAtATime * kThreads, c.columns);
      float some = 0.f, some_dot = 0.f;
      for (int64_t k = from; k < to; k += kThreads) {
        const float s = T::to_f32(x[k]), a = T::to_f32(dy[k]);
        some = __builtin_fmaf(s, s, some);
        some_dot = __builtin_fmaf(weight ? a * T::to_f32(weight[k]) : a, s, some_dot);
      }
      squares += (double)some;
      dot += (double)some_dot;
    }
    over_row<kThreads>(squares, dot, turn++);
    double size = squares * share + (double)c.eps;
    float lift = 1.f;
    if (kFarValues<T> && far_row((float)squares, (float)size)) {
      lift = lift_of((float)squares);
      squares = dot = 0.;
#pragma unroll 1
      for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
        const double s = T::to_f32(x[k]) * lift, a = T::to_f32(dy[k]);
        squares = __builtin_fma(s, s, squares);
        dot = __builtin_fma(weight ? a * (double)T::to_f32(weight[k]) : a, s, dot);
      }
      over_row<kThreads>(squares, dot, turn++);
      size = squares * share + (double)c.eps * (double)lift * (double)lift;
    }
    const double root = 1.0 / __builtin_sqrt(size);
    const float rstd = (float)root, mean = (float)(root * dot * share), slope = rstd * lift;
    for (int64_t k = threadIdx.x; k < c.columns; k += kThreads) {
      const float n = T::to_f32(x[k]) * lift * rstd, a = T::to_f32(dy[k]);
      if (parts) parts[k] = added ? __builtin_fmaf(a, n, parts[k]) : a * n;
      if (!c.dx) continue;
      float d = slope * __builtin_fmaf(-mean, n, weight ? a * T::to_f32(weight[k]) : a);
      if (c.dsum) d += T::to_f32(dsum[k]);
      static_cast<E*>(c.dx)[row * c.columns + k] = T::from_f32(d);
    }
    added = true;
  }
}

// dw = sum of the workgroups' partial sums, in float64: rounded once, whatever their number.  A workgroup to 16 columns, 64 threads to a
// column, and on to other columns where there are more than a launch has (fewer than 2^32 threads: rows of up to 2^28 values would ask
// for 2^34).
template <typename T>
__global__ __launch_bounds__(1024) void rows_weight_kernel(const float* parts, int n, int64_t columns, void* dw) {
  constexpr int kWaves = 1024 / kWave;
  const int own = threadIdx.x & 15, part = threadIdx.x >> 4, wave = threadIdx.x / kWave;
  __shared__ double sums[kWaves][16];
  for (int64_t first = (int64_t)blockIdx.x * 16; first < columns; first += (int64_t)gridDim.x * 16) {
    const int64_t column = first + own;
    double v = 0.;
    if (column < columns) {
#pragma unroll 8
      for (int i = part; i < n; i += 64) v += (double)parts[i * columns + column];
    }
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    if ((threadIdx.x & (kWave - 1)) < 16) sums[wave][own] = v;
    __syncthreads();
    if (part == 0 && column < columns) {
#pragma unroll
      for (int i = 1; i < kWaves; ++i) v += sums[i][own];
      static_cast<typename T::storage*>(dw)[column] = T::from_f32((float)v);
    }
    __syncthreads();
  }
}

// ---- codes times their row's scale: 4352 x 3840 to bfloat16 10.8 us (4.6 TB/s)
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
        reinterpret_cast<u32x4*>(to)[p] = pack<T, V>(v);
      }
    } else {
      *to = T::from_f32((float)codes[row * stride + k] * scale);
    }
  }
}

// Workgroups of a backward pass, each of them a row of partial sums: two to a compute unit, and more of them where a lane would add up more
// than 128 rows in float32 (equal terms drift: 2048 of them some 300 roundings away, 128 of them 8 to 19)
constexpr int kBackwardGroups = 2, kBackwardRows = 128;
int64_t most_backward_groups(int64_t rows, int per_group) {
  const int64_t few = kBackwardGroups * (int64_t)compute_units(), each = kBackwardRows * per_group, many = (rows + each - 1) / each;
  return many < few ? few : many < (1 << 22) ? many : 1 << 22;  // (of up to 512 threads: fewer than 2^32)
}

// as many rows to every workgroup
int64_t groups_of(int64_t rows, int per_group, int64_t most) {
  const int64_t groups = (rows + per_group - 1) / per_group, each = (groups + most - 1) / most;
  return (groups + each - 1) / each;
}

template <typename T, int V, int kLanes, int kChunks>
int64_t forward_form(const RowsCall& c, hipStream_t stream) {
  constexpr int kBlock = kLanes > kWave ? kLanes : kThreads;
  const int64_t groups = groups_of(c.rows, kBlock / kLanes, 2048 / kBlock * (int64_t)compute_units());
  const dim3 grid((unsigned)groups), block(kBlock);
  if (!c.codes) hipLaunchKernelGGL((rows_kernel<T, V, kLanes, kChunks, kNormalised>), grid, block, 0, stream, c);
  else if (!c.norm) hipLaunchKernelGGL((rows_kernel<T, V, kLanes, kChunks, kCodes>), grid, block, 0, stream, c);
  else if (c.weight) hipLaunchKernelGGL((rows_kernel<T, V, kLanes, kChunks, kWeightedCodes>), grid, block, 0, stream, c);
  else hipLaunchKernelGGL((rows_kernel<T, V, kLanes, kChunks, kNormalisedCodes>), grid, block, 0, stream, c);
  return groups;
}

template <typename T, int V, int kLanes, int kChunks>
int64_t backward_form(const RowsCall& c, hipStream_t stream) {
  constexpr int kBlock = kLanes > kWave ? kLanes : kThreads;
  constexpr int kRows = kBlock / kLanes;
  const int64_t groups = groups_of(c.rows, kRows, most_backward_groups(c.rows, kRows));
  const dim3 grid((unsigned)groups), block(kBlock);
  if (c.parts) hipLaunchKernelGGL((rows_backward_kernel<T, V, kLanes, kChunks, true>), grid, block, 0, stream, c);
  else hipLaunchKernelGGL((rows_backward_kernel<T, V, kLanes, kChunks, false>), grid, block, 0, stream, c);
  return groups;
}

// The form of a row: as many lanes as hold it in two units each, which leaves registers for many rows on their way to a compute unit
// (4352 x 3840 bfloat16: 256 lanes of two 25 us and 24 with codes, 128 lanes of four 34 and 34); a backward pass, whose workgroups each
// cost a row of partial sums, in fewer workgroups with more of a row to a lane.
template <typename T>
int64_t launch_forward(const RowsCall& c, bool wide, hipStream_t stream) {
  constexpr int V = kVecOf<T>;
  const int64_t units = wide ? c.columns / V : c.columns;
  if (wide) {
    if (units <= 64) return forward_form<T, V, 64, 1>(c, stream);
    if (units <= 128) return forward_form<T, V, 64, 2>(c, stream);
    if (units <= 256) return forward_form<T, V, 128, 2>(c, stream);
    if (units <= 512) return forward_form<T, V, 256, 2>(c, stream);
    if (units <= 1024) return forward_form<T, V, 512, 2>(c, stream);
    if (units <= 2048) return forward_form<T, V, 1024, 2>(c, stream);
    if (units <= 4096) return forward_form<T, V, 1024, 4>(c, stream);
  } else {
    if (units <= 512) return forward_form<T, 1, 64, 8>(c, stream);
    if (units <= 1024) return forward_form<T, 1, 256, 4>(c, stream);
    if (units <= 4096) return forward_form<T, 1, 256, 16>(c, stream);
  }
  const int64_t groups = groups_of(c.rows, 1, 8 * (int64_t)compute_units());
  const dim3 grid((unsigned)groups), block(kThreads);
  if (!c.codes) hipLaunchKernelGGL((rows_any_kernel<T, kNormalised>), grid, block, 0, stream, c);
  else if (!c.norm) hipLaunchKernelGGL((rows_any_kernel<T, kCodes>), grid, block, 0, stream, c);
  else if (c.weight) hipLaunchKernelGGL((rows_any_kernel<T, kWeightedCodes>), grid, block, 0, stream, c);
  else hipLaunchKernelGGL((rows_any_kernel<T, kNormalisedCodes>), grid, block, 0, stream, c);
  return groups;
}

template <typename T>
int64_t launch_backward(const RowsCall& c, bool wide, hipStream_t stream) {
  constexpr int V = kVecOf<T>;
  const int64_t units = wide ? c.columns / V : c.columns;
  if (wide) {
    if (units <= 64) return backward_form<T, V, 64, 1>(c, stream);
    if (units <= 128) return backward_form<T, V, 64, 2>(c, stream);
    if (units <= 256) return backward_form<T, V, 64, 4>(c, stream);
    if (units <= 512) return backward_form<T, V, 256, 2>(c, stream);
    if (units <= 1024) return backward_form<T, V, 256, 4>(c, stream);
    if (units <= 2048) return backward_form<T, V, 512, 4>(c, stream);
  } else {
    if (units <= 512) return backward_form<T, 1, 64, 8>(c, stream);
    if (units <= 1024) return backward_form<T, 1, 256, 4>(c, stream);
    if (units <= 4096) return backward_form<T, 1, 256, 16>(c, stream);
  }
  const int64_t groups = groups_of(c.rows, 1, most_backward_groups(c.rows, 1));
  hipLaunchKernelGGL((rows_backward_any_kernel<T>), dim3((unsigned)groups), dim3(kThreads), 0, stream, c);
  return groups;
}

template <typename T>
int launch(const RowsCall& c, bool wide, bool backward, hipStream_t stream) {
  const int64_t groups = backward ? launch_backward<T>(c, wide, stream) : launch_forward<T>(c, wide, stream);
  if (hipGetLastError() != hipSuccess) return MFQ_ELAUNCH;
  if (!backward || !c.parts) return MFQ_OK;
  const int64_t sixteens = (c.columns + 15) / 16, most = 8 * (int64_t)compute_units();
  hipLaunchKernelGGL(rows_weight_kernel<T>, dim3((unsigned)(sixteens < most ? sixteens : most)), dim3(1024), 0, stream, c.parts, (int)groups,
                     c.columns, c.dweight);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

}  // namespace

size_t rows_workspace_bytes(int64_t rows, int64_t columns) {
  const int64_t most = most_backward_groups(rows, 1);  // as many as any form of a row has
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
