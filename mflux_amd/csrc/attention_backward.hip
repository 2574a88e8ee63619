// The gradients of attention (attention.hip):
//   P = softmax(scale q k^T + mask), dP = dy v^T, dS = P (dP - sum(dy y)), dv = P^T dy, dq = scale dS k, dk = scale dS^T q
// with P made again from the forward pass's log-sum-exp of each row.  Two launches: one walks the keys of a tile of queries (dq, and
// the rows' sums of dy y, which the other needs), one the queries of a tile of keys (dk and dv, over all heads that share them).
// That makes the scores twice, 14 instead of 10 operations a pair and element of a head, and no sum is made by atomics, so the
// gradients are the same bits every time.  All sums are float32; P and dS are rounded to the inputs' type for the second products,
// as P is in the forward pass.  sum(dy y) is taken from y and what its rounding left: with the roundings of bfloat16 put into a
// 64-bit calculation (1024 causal tokens, D = 128) dq is off by 2.6 10^-3 of its norm from the rounded y, by 2.4 from this one.
//
// 4608 tokens, 24 heads of 128, bfloat16: dq 374 to 391 us, 1.00 to 1.05 PFLOP/s of its 6 operations a pair and element; dk and dv 572 to
// 593 us, 0.88 to 0.91 of their 8 (float16: 425 and 636 us); causal 0.91 to 0.93 and 0.88 to 0.91.  4099 causal tokens in three sequences, 24 / 8 heads: 124 and 186 us, and 19 to join the parts; there the
// counters show the matrix units busy in 28 and 30 % of the cycles.
#include "attention.h"

#include <algorithm>
#include <type_traits>

namespace mfq {
namespace {

constexpr int pitch_of(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// a step over what every row sees, over what some see, and the same where a row is not finite (attention.h, tile_not_finite)
enum { kWhole, kEdge, kRowByRow };
template <int kMode>
using Mode = std::integral_constant<int, kMode>;

// float16 has neither the range nor the small numbers for the scores' gradients of any loss (a few keys and a large dy: above 65504, many
// keys and a small one: below 2^-24, with results that float16 holds), so they are rounded as multiples of a power of two that each
// lane's column of sums has for itself: taken from the first gradients that are not zero, and again, with the sums, from larger ones.
// bfloat16 has float32's range and needs none.
template <typename T, int kBlocks>
struct ColumnUnit {
  float unit = 0.f;  // what values are multiplied with, 0: none yet

  __device__ __attribute__((always_inline)) inline void apply(f32x16& ds, f32x16 (&sums)[kBlocks]) {
    if constexpr (T::code == MFQ_F16) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, __builtin_fabsf(ds[i]));
      most = max_halves(most);
      const bool low = most * unit > 16384.f || (unit == 0.f && most > 0.f);
      if (__any(low && most < 3e38f)) {
        // 2^4 over the power of two that `most` lies above
        const int exponent = min(max(131 + 127 - (int)(__float_as_uint(most) >> 23), 1), 254);
        const float next = low && most < 3e38f ? __uint_as_float((uint32_t)exponent << 23) : unit;
        const float factor = unit == 0.f ? 1.f : next / unit;
        unit = next;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) sums[b][i] *= factor;
      }
      const float by = unit == 0.f ? 1.f : unit;
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] *= by;
    }
  }
  __device__ __attribute__((always_inline)) inline void remove(f32x16 (&sums)[kBlocks]) {
    if constexpr (T::code == MFQ_F16) {
      const float by = unit == 0.f ? 1.f : 1.f / unit;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[b][i] *= by;
      unit = 0.f;
    }
  }
};
// and probabilities as multiples of 2^-13, for those that many queries give to a key that none of them looks at in earnest (attention.h, kLift;
// what is left to float16's 2^16 is for scores of millions, whose float32 log-sum-exp is itself off by more than 1)
template <typename T>
constexpr float kProbabilityShift = T::code == MFQ_F16 ? 13.f : 0.f;

constexpr int kKeys = 64;  // of a step of the first kernel

// kHalves == 2: a workgroup has 64 queries, and two wavefronts the same 32, each one half of every tile's keys, joined in LDS at the end
template <typename T, int kDim, bool kPadded, int kHalves>
__global__ __launch_bounds__(256, kDim <= 128 ? 2 : 1) void attention_dq_kernel(AttentionCall c, int tiles) {
  constexpr int kQueries = 128 / kHalves;
  constexpr int kPitch = pitch_of(kDim), kSteps = kDim / 16, kBlocks = kDim / 32;
  constexpr int kTileBytes = kKeys * kPitch * 2;
  using vec8 = typename T::vec8;
  using Row = QueryState<T, kDim, kPitch>;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // K, V, K, V
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = uniform(thread / kWave);
  int head, index;
  head_and_tile(blockIdx.x, c.heads, tiles, c.causal || c.q_offsets, head, index);
  const Run run = find_run<kQueries>(c, index, false, c.causal);
  if (!run.valid) return;
  const int kv_head = head / (c.heads / c.kv_heads);
  const int half = wave / (4 / kHalves);
  const int row = run.tile * kQueries + wave % (4 / kHalves) * 32 + (lane & 31);
  const int limit = visible_keys(run, row, c.causal);
  const int keys = uniform(run.tile * kQueries < run.nq ? visible_keys(run, min(run.tile * kQueries + kQueries, run.nq) - 1, c.causal) : 0);
  const int least = wave_min(row < run.nq ? limit : INT32_MAX), most = wave_max(limit);
  const int64_t rows = (int64_t)(c.q_offsets ? 1 : c.batch) * c.q_tokens;
  const int64_t at = (int64_t)run.batch * c.q_tokens + run.q0 + row;

  f32x16 dq[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) dq[b] = zero16();
  ColumnUnit<T, kBlocks> unit;
  float delta = 0.f;
  if (keys > 0) {
    const int64_t inside = run.q0 + min(row, run.nq - 1);
    vec8 q[kSteps], dy[kSteps];
    Row::load_row(q, c.q.p + run.batch * c.q.batch + inside * c.q.token + head * c.q.head, c.dim, lane);
    Row::load_row(dy, c.dy.p + run.batch * c.dy.batch + inside * c.dy.token + head * c.dy.head, c.dim, lane);
    {
      vec8 y[kSteps], rest[kSteps];
      Row::load_row(rest, c.rest ? c.rest + (((int64_t)run.batch * c.q_tokens + inside) * c.heads + head) * c.dim : nullptr, c.rest ? c.dim : 0, lane);
      Row::load_row(y, c.y.p + run.batch * c.y.batch + inside * c.y.token + head * c.y.head, c.dim, lane);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const u32x4a a = __builtin_bit_cast(u32x4a, dy[s]), b = __builtin_bit_cast(u32x4a, y[s]), r = __builtin_bit_cast(u32x4a, rest[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          delta = __builtin_fmaf(lo_f32<T>(a[i]), lo_f32<T>(b[i]) + lo_f32<T>(r[i]), delta);
          delta = __builtin_fmaf(hi_f32<T>(a[i]), hi_f32<T>(b[i]) + hi_f32<T>(r[i]), delta);
        }
      }
      delta = sum_halves(delta);
    }
    const float lse = c.lse[head * rows + (int64_t)run.batch * c.q_tokens + inside];
    const uint16_t* k = uniform(c.k.p + run.batch * c.k.batch + (int64_t)run.k0 * c.k.token + kv_head * c.k.head);
    const uint16_t* v = uniform(c.v.p + run.batch * c.v.batch + (int64_t)run.k0 * c.v.token + kv_head * c.v.head);
    TileLoader<kPitch, kKeys, 256, kPadded> load_k;
    TileLoader<kPitch, kKeys, 256> load_v;
    load_k.init(thread, c.k.token, c.dim);
    load_v.init(thread, c.v.token, c.dim);
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;
    const float scale = c.scale * kLog2e;

    // 32 keys
    auto step = [&](const char* k32, const char* v32, int left, auto mode) __attribute__((always_inline)) {
      constexpr bool kMasked = decltype(mode)::value != kWhole, kOneByOne = decltype(mode)::value == kRowByRow;
      bool not_finite = false;
      {
        f32x16 s = zero16(), dp = zero16();
        // operands are read a step ahead of the matrix instructions that take them
        vec8 a[2][2] = {{tile_rows<T, kPitch>(k32, 0, lane), tile_rows<T, kPitch>(v32, 0, lane)}};
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
          if (e + 1 < kSteps) {
            a[(e + 1) & 1][0] = tile_rows<T, kPitch>(k32, e + 1, lane);
            a[(e + 1) & 1][1] = tile_rows<T, kPitch>(v32, e + 1, lane);
          }
          s = mfma32(a[e & 1][0], q[e], s);
          dp = mfma32(a[e & 1][1], dy[e], dp);
          __builtin_amdgcn_sched_barrier(0);
        }
        vec8 w[2][kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) w[0][b] = tile_columns<T, kPitch>(k32, b, lane);
        // a row of K that is not finite shows in every score of it (attention.h, tile_not_finite)
        if constexpr (kMasked && !kOneByOne) not_finite = __any(times_zero(s, 0.f) != 0.f);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale, -lse));
          s[i] = p * (dp[i] - delta);
          if constexpr (kMasked) s[i] = result_row(i, lane) < left ? s[i] : 0.f;
        }
        unit.apply(s, dq);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const vec8 ds = result_operand<T>(s, n);
          if constexpr (kOneByOne) {
            add_columns_one_by_one<T, kPitch, kBlocks>(dq, k32 + n * 16 * kPitch * 2, ds, lane, [&](int r) { return 16 * n + r < left; });
          } else {
            if (n == 0) {
#pragma unroll
              for (int b = 0; b < kBlocks; ++b) w[1][b] = tile_columns<T, kPitch>(k32 + 16 * kPitch * 2, b, lane);
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) dq[b] = mfma32(w[n][b], ds, dq[b]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      return not_finite;
    };
    if constexpr (kPadded) {
      clear_padding<kPitch, kDim>(lds, kKeys, c.dim, thread, 256);
      clear_padding<kPitch, kDim>(lds + 2 * kTileBytes, kKeys, c.dim, thread, 256);
    }
    load_k.load(k, lds_at, keys, thread);
    load_v.load(v, lds_at + kTileBytes, keys, thread);
    auto advance = [&](int first, int buffer) __attribute__((always_inline)) {
      arrive_and_sync();
      const int next = first + kKeys;
      if (next < keys) {
        const uint32_t to = lds_at + (buffer ^ 1) * 2 * kTileBytes;
        load_k.load(k + (int64_t)next * c.k.token, to, keys - next, thread);
        load_v.load(v + (int64_t)next * c.v.token, to + kTileBytes, keys - next, thread);
      }
    };
    // as in the forward pass: whole tiles first
    const int whole = uniform(c.causal ? visible_keys(run, run.tile * kQueries, 1) : run.nk);
    int first = 0, buffer = 0;
    constexpr int kHalf = 32 * kPitch * 2;
    auto whole_tile = [&](const char* k64) __attribute__((always_inline)) {
      if constexpr (kHalves == 2) {
        step(k64 + half * kHalf, k64 + kTileBytes + half * kHalf, 32, Mode<kWhole>());
      } else {
        step(k64, k64 + kTileBytes, 32, Mode<kWhole>());
        step(k64 + kHalf, k64 + kTileBytes + kHalf, 32, Mode<kWhole>());
      }
    };
    for (; first + 2 * kKeys <= whole; first += 2 * kKeys) {
      advance(first, 0);
      whole_tile(lds);
      advance(first + kKeys, 1);
      whole_tile(lds + 2 * kTileBytes);
    }
    // at the largest heads what follows has offsets and rows of its own, as in the forward pass
    auto separate = [&]() __attribute__((always_inline)) {
      if constexpr (kDim > 192) {
        int own = thread;
        asm volatile("" : "+v"(own));
        load_k.init(own, c.k.token, c.dim);
        load_v.init(own, c.v.token, c.dim);
        int64_t at = inside;
        asm volatile("" : "+v"(at));
        Row::load_row(q, c.q.p + run.batch * c.q.batch + at * c.q.token + head * c.q.head, c.dim, own & (kWave - 1));
        Row::load_row(dy, c.dy.p + run.batch * c.dy.batch + at * c.dy.token + head * c.dy.head, c.dim, own & (kWave - 1));
      }
    };
    separate();
    bool not_finite = false;
#pragma unroll 1
    for (; first < keys; first += kKeys, buffer ^= 1) {
      advance(first, buffer);
#pragma unroll 1
      for (int at = first + (kHalves == 2 ? 32 * half : 0); at < min(first + kKeys, most); at += 32 * kHalves) {
        const char* k32 = lds + buffer * 2 * kTileBytes + (at - first) * kPitch * 2;
        if (at + 32 <= least) step(k32, k32 + kTileBytes, 32, Mode<kWhole>());
        else not_finite |= step(k32, k32 + kTileBytes, limit - at, Mode<kEdge>());
      }
    }
    if (any_wave<4>(not_finite, lds)) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) dq[b] = zero16();
      unit = {};
      separate();
      load_k.load(k, lds_at, keys, thread);
      load_v.load(v, lds_at + kTileBytes, keys, thread);
#pragma unroll 1
      for (first = 0, buffer = 0; first < keys; first += kKeys, buffer ^= 1) {
        advance(first, buffer);
#pragma unroll 1
        for (int at = first + (kHalves == 2 ? 32 * half : 0); at < min(first + kKeys, most); at += 32 * kHalves) {
          const char* k32 = lds + buffer * 2 * kTileBytes + (at - first) * kPitch * 2;
          step(k32, k32 + kTileBytes, limit - at, Mode<kRowByRow>());
        }
      }
    }
  }
  unit.remove(dq);
  if constexpr (kHalves == 2) {
    constexpr int kFloats = kDim + 4;
    float* slot = reinterpret_cast<float*>(lds) + (wave % 2 * 32 + (lane & 31)) * kFloats;
    __syncthreads();  // (nothing is in flight, and what has been requested has been read)
    if (half) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<f32x4*>(slot + 32 * b + result_row(i, lane)) = f32x4{dq[b][i], dq[b][i + 1], dq[b][i + 2], dq[b][i + 3]};
    }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 o = *reinterpret_cast<const f32x4*>(slot + 32 * b + result_row(i, lane));
#pragma unroll
        for (int j = 0; j < 4; ++j) dq[b][i + j] += o[j];
      }
  }
  if (row >= run.rows) return;
  if (lane < 32) c.delta[head * rows + at] = delta;
  if (c.dq) store_row<T, kBlocks>(c.dq + (at * c.heads + head) * c.dim, nullptr, dq, limit > 0, c.scale, c.dim, lane);
}

// The second kernel.  A workgroup has 128 keys of one head, 32 a wavefront, and walks the queries: a stage in LDS is q and dy of
// some rows with their log-sum-exps and sums.  Up to 128 elements a head there are eight wavefronts, two to the same keys, each with one
// half of a stage's 64 rows, so that two share a SIMD (one computes exponentials while the other multiplies) with 256 registers each:
// the sums (2 x 64) stay in them, the rows of K and V are read from LDS again for each product.  The halves are joined in LDS at the
// end.  Above 128 elements four wavefronts have 512 registers each, and K stays in them.
constexpr int kKeyRows = 128;
template <int kDim>
struct KeyShape {
  static constexpr int kPitch = pitch_of(kDim), kWaves = kDim <= 128 ? 8 : 4, kHalves = kWaves / 4, kRows = 32 * kHalves;
  static constexpr bool kHoldK = kDim > 128;
  static constexpr int kKeyTile = kKeyRows * kPitch * 2;      // bytes
  static constexpr int kV = kKeyTile * (kHoldK ? 1 : 2);      // V, and K where it is not held
  static constexpr int kTile = kRows * kPitch * 2;            // q or dy of a stage
  static constexpr int kStage = 2 * kTile + 512;              // and 64 log-sum-exps, 64 sums
  static constexpr int kFloats = kDim + 4;                    // a row of sums on its way to the other half
  static constexpr int kLds = kV + 2 * kStage;
  static_assert(kHalves == 1 || kKeyRows * kFloats * 4 <= kLds, "the halves are joined in place");
};

// 32 or 64 floats from a row on into LDS, those past `rows` repeating the last one
__device__ inline void load_floats(const float* base, uint32_t lds, int rows, int count, int lane) {
  const uint32_t o = 4u * (uint32_t)min(min(lane, count - 1), rows - 1);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(o), "s"(uniform(base)), "s"(uniform((int)lds)) : "memory", "m0");
}

// parts: of the query heads that share a key head, each with sums of its own (part_k, part_v: float32 planes [parts][rows][kv_heads][dim])
template <typename T, int kDim>
__global__ __launch_bounds__(64 * KeyShape<kDim>::kWaves, KeyShape<kDim>::kWaves / 4) void attention_dkv_kernel(AttentionCall c, int tiles, int parts,
                                                                                                               float* part_k, float* part_v) {
  using S = KeyShape<kDim>;
  constexpr int kPitch = S::kPitch, kSteps = kDim / 16, kBlocks = kDim / 32, kRows = S::kRows;
  using vec8 = typename T::vec8;
  using Row = QueryState<T, kDim, kPitch>;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // V, and two stages
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = uniform(thread / kWave);
  const int keys_of = wave & 3, half = wave >> 2;
  int which, index;
  head_and_tile(blockIdx.x, c.kv_heads * parts, tiles, c.causal || c.q_offsets, which, index);
  const int kv_head = which / parts, part = which - kv_head * parts;
  const Run run = find_run<kKeyRows>(c, index, true, false);  // causal: the first keys have the most queries
  if (!run.valid) return;
  const int group = c.heads / c.kv_heads;
  const int head0 = kv_head * group + part * group / parts, heads = (part + 1) * group / parts - part * group / parts;
  const int key0 = run.tile * kKeyRows;
  const int row = key0 + keys_of * 32 + (lane & 31);  // the lane's key
  const int shift = run.nk - run.nq;                  // causal: query i sees the keys up to i + shift
  // the queries that see a key are [from(key), nq)
  auto from = [&](int key) { return key >= run.nk ? run.nq : c.causal ? min(max(key - shift, 0), run.nq) : 0; };
  const int mine = from(row);
  const int first_query = uniform(from(key0)), last_from = uniform(from(min(key0 + kKeyRows, run.nk) - 1));
  // tiles of queries: [t0, t3) that any of the keys is seen by, [t1, t2) whole and seeing all the keys
  const int t0 = first_query / kRows, t3 = first_query < run.nq ? (run.nq + kRows - 1) / kRows : t0;
  const int t1 = min((last_from + kRows - 1) / kRows, t3), t2 = max(run.nq / kRows, t1);
  const int whole = t3 > t0 ? min(t2, t3) - t1 : 0, edge = t3 - t0 - whole;

  f32x16 dk[kBlocks], dv[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) dk[b] = dv[b] = zero16();
  ColumnUnit<T, kBlocks> unit;
  constexpr float kShift = kProbabilityShift<T>;
  if (t3 > t0 && heads > 0) {
    const int64_t inside = run.k0 + min(row, run.nk - 1);
    vec8 k[S::kHoldK ? kSteps : 1];
    if constexpr (S::kHoldK) Row::load_row(k, c.k.p + run.batch * c.k.batch + inside * c.k.token + kv_head * c.k.head, c.dim, lane);
    const uint16_t* v0 = uniform(c.v.p + run.batch * c.v.batch + (int64_t)(run.k0 + key0) * c.v.token + kv_head * c.v.head);
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;
    {
      TileLoader<kPitch, kKeyRows, 64 * S::kWaves> load_v;
      load_v.init(thread, c.v.token, c.dim);
      load_v.load(v0, lds_at, run.nk - key0, thread);
      if constexpr (!S::kHoldK) {
        load_v.init(thread, c.k.token, c.dim);
        load_v.load(uniform(c.k.p + run.batch * c.k.batch + (int64_t)(run.k0 + key0) * c.k.token + kv_head * c.k.head), lds_at + S::kKeyTile,
                    run.nk - key0, thread);
      }
    }
    TileLoader<kPitch, kRows, 64 * S::kWaves> load_q, load_dy;
    load_q.init(thread, c.q.token, c.dim);
    load_dy.init(thread, c.dy.token, c.dim);
    const uint16_t* q0 = uniform(c.q.p + run.batch * c.q.batch + (int64_t)run.q0 * c.q.token + (int64_t)head0 * c.q.head);
    const uint16_t* dy0 = uniform(c.dy.p + run.batch * c.dy.batch + (int64_t)run.q0 * c.dy.token + (int64_t)head0 * c.dy.head);
    const int64_t rows = (int64_t)(c.q_offsets ? 1 : c.batch) * c.q_tokens;
    const float* lse0 = uniform(c.lse + head0 * rows + (int64_t)run.batch * c.q_tokens + run.q0);
    const float* delta0 = uniform(c.delta + head0 * rows + (int64_t)run.batch * c.q_tokens + run.q0);
    const float scale = c.scale * kLog2e;
    const char* v32 = lds + keys_of * 32 * kPitch * 2;
    const char* k32 = v32 + S::kKeyTile;

    // item i: a head and a tile of its queries; all heads' whole tiles first, then those at an edge
    const int items = heads * (whole + edge);
    auto first_of = [&](int i, int& head) __attribute__((always_inline)) {
      if (i < heads * whole) {
        head = i / whole;
        return (t1 + i - head * whole) * kRows;
      }
      i -= heads * whole;
      head = i / edge;
      const int e = t0 + i - head * edge;
      return (e < t1 ? e : e + whole) * kRows;
    };
    auto request = [&](int i, int stage) __attribute__((always_inline)) {
      int head;
      const int first = first_of(i, head);
      const uint32_t to = lds_at + S::kV + stage * S::kStage;
      load_q.load(q0 + head * c.q.head + (int64_t)first * c.q.token, to, run.nq - first, thread);
      load_dy.load(dy0 + head * c.dy.head + (int64_t)first * c.dy.token, to + S::kTile, run.nq - first, thread);
      if (wave == 0) load_floats(lse0 + head * rows + first, to + 2 * S::kTile, run.nq - first, kRows, lane);
      if (wave == 1) load_floats(delta0 + head * rows + first, to + 2 * S::kTile + 256, run.nq - first, kRows, lane);
    };
    // masked: the queries [start, left) of the wavefront's 32 are there and see the lane's key
    auto step = [&](const char* stage, int start, int left, auto mode) __attribute__((always_inline)) {
      constexpr bool kMasked = decltype(mode)::value != kWhole, kOneByOne = decltype(mode)::value == kRowByRow;
      const char* q32 = stage + half * 32 * kPitch * 2;
      const char* dy32 = q32 + S::kTile;
      const float* lse = reinterpret_cast<const float*>(stage + 2 * S::kTile) + half * 32;
      const float* delta = lse + 64;
      bool not_finite = false;
      f32x16 s = zero16(), dp = zero16();
      vec8 a[2][4];
      auto operands = [&](int e) __attribute__((always_inline)) {
        a[e & 1][0] = tile_rows<T, kPitch>(q32, e, lane);
        a[e & 1][1] = tile_rows<T, kPitch>(dy32, e, lane);
        a[e & 1][2] = tile_rows<T, kPitch>(v32, e, lane);
        if constexpr (S::kHoldK) a[e & 1][3] = k[e];
        else a[e & 1][3] = tile_rows<T, kPitch>(k32, e, lane);
      };
      operands(0);
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        if (e + 1 < kSteps) operands(e + 1);
        s = mfma32(a[e & 1][0], a[e & 1][3], s);
        dp = mfma32(a[e & 1][1], a[e & 1][2], dp);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (kMasked && !kOneByOne) not_finite = __any(times_zero(s, times_zero(dp, 0.f)) != 0.f);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int r = result_row(i, lane);
        const f32x4 l = *reinterpret_cast<const f32x4*>(lse + r), d = *reinterpret_cast<const f32x4*>(delta + r);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + j], scale, kShift - l[j])), ds = p * (dp[i + j] - d[j]);
          const bool see = !kMasked || ((r + j >= start) & (r + j < left));
          s[i + j] = see ? p : 0.f;
          dp[i + j] = see ? ds : 0.f;
        }
      }
      unit.apply(dp, dk);
      if constexpr (kOneByOne) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          auto visible = [&](int r) { return 16 * n + r >= start && 16 * n + r < left; };
          add_columns_one_by_one<T, kPitch, kBlocks>(dv, dy32 + n * 16 * kPitch * 2, result_operand<T>(s, n), lane, visible);
          add_columns_one_by_one<T, kPitch, kBlocks>(dk, q32 + n * 16 * kPitch * 2, result_operand<T>(dp, n), lane, visible);
        }
      } else {
        // four products of 16 rows each: dv, dk, dv, dk
        vec8 w[2][kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) w[0][b] = tile_columns<T, kPitch>(dy32, b, lane);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          if (n < 3) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
              w[(n + 1) & 1][b] = tile_columns<T, kPitch>((n & 1 ? dy32 : q32) + ((n + 1) >> 1) * 16 * kPitch * 2, b, lane);
          }
          const vec8 x = result_operand<T>(n & 1 ? dp : s, n >> 1);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            if (n & 1) dk[b] = mfma32(w[n & 1][b], x, dk[b]);
            else dv[b] = mfma32(w[n & 1][b], x, dv[b]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      return not_finite;
    };
    request(0, 0);
    if (c.dim < kDim) {
      // both operands of the first products come out of LDS, where the pieces past the head's end repeat its last: one side has to be zero
      arrive_and_sync();
      clear_padding<kPitch, kDim>(lds, S::kV / (kPitch * 2), c.dim, thread, 64 * S::kWaves);  // K's tile lies 128 rows behind V's
    }
    int i = 0;
    for (; i + 2 <= heads * whole; i += 2) {
      arrive_and_sync();
      request(i + 1, 1);
      step(lds + S::kV, 0, 32, Mode<kWhole>());
      arrive_and_sync();
      if (i + 2 < items) request(i + 2, 0);
      step(lds + S::kV + S::kStage, 0, 32, Mode<kWhole>());
    }
    int stage = 0;
    auto edges = [&](auto mode) __attribute__((always_inline)) {
      bool not_finite = false;
#pragma unroll 1
      for (; i < items; ++i, stage ^= 1) {
        arrive_and_sync();
        if (i + 1 < items) request(i + 1, stage ^ 1);
        int head;
        const int first = first_of(i, head) + 32 * half;
        not_finite |= step(lds + S::kV + stage * S::kStage, mine - first, run.nq - first, mode);
      }
      return not_finite;
    };
    auto separate = [&]() __attribute__((always_inline)) {  // as in the dq kernel
      if constexpr (kDim > 192) {
        int own = thread;
        asm volatile("" : "+v"(own));
        load_q.init(own, c.q.token, c.dim);
        load_dy.init(own, c.dy.token, c.dim);
        if constexpr (S::kHoldK) {
          int64_t at = inside;
          asm volatile("" : "+v"(at));
          Row::load_row(k, c.k.p + run.batch * c.k.batch + at * c.k.token + kv_head * c.k.head, c.dim, own & (kWave - 1));
        }
      }
    };
    separate();
    const bool not_finite = edges(Mode<kEdge>());
    if (edge > 0 && any_wave<S::kWaves>(not_finite, lds + S::kV)) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) dk[b] = dv[b] = zero16();
      unit = {};
      i = stage = 0;
      separate();
      request(0, 0);
      edges(Mode<kRowByRow>());
    }
  }
  unit.remove(dk);
  const float k_factor = c.scale * __builtin_amdgcn_exp2f(-kShift), v_factor = __builtin_amdgcn_exp2f(-kShift);
  if constexpr (S::kHalves == 2) {
    // the second half's sums to the first, one array after the other
    float* slot = reinterpret_cast<float*>(lds) + (keys_of * 32 + (lane & 31)) * S::kFloats;
    auto join = [&](f32x16(&acc)[kBlocks]) __attribute__((always_inline)) {
      __syncthreads();
      if (half) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<f32x4*>(slot + 32 * b + result_row(i, lane)) = f32x4{acc[b][i], acc[b][i + 1], acc[b][i + 2], acc[b][i + 3]};
      }
      __syncthreads();
      if (!half) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4 o = *reinterpret_cast<const f32x4*>(slot + 32 * b + result_row(i, lane));
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[b][i + j] += o[j];
          }
      }
    };
    join(dk);
    join(dv);
    if (half) return;
  }
  if (row >= run.rows) return;
  const int64_t at = ((int64_t)run.batch * c.k_tokens + run.k0 + row) * c.kv_heads + kv_head;
  const bool seen = mine < run.nq;
  if (parts == 1) {
    if (c.dk) store_row<T, kBlocks>(c.dk + at * c.dim, nullptr, dk, seen, k_factor, c.dim, lane);
    if (c.dv) store_row<T, kBlocks>(c.dv + at * c.dim, nullptr, dv, seen, v_factor, c.dim, lane);
    return;
  }
  const int64_t plane = (int64_t)(c.q_offsets ? 1 : c.batch) * c.k_tokens * c.kv_heads * c.dim;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * b + result_row(i, lane);
      if (d >= c.dim) continue;
      f32x4 x, y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = seen ? dk[b][i + j] * k_factor : 0.f;
        y[j] = seen ? dv[b][i + j] * v_factor : 0.f;
      }
      *reinterpret_cast<f32x4*>(part_k + part * plane + at * c.dim + d) = x;
      *reinterpret_cast<f32x4*>(part_v + part * plane + at * c.dim + d) = y;
    }
}

// dk and dv = the parts' sums, rounded: a thread to eight elements
template <typename T>
__global__ __launch_bounds__(256) void attention_dkv_join_kernel(const float* part_k, const float* part_v, int parts, int64_t n, uint16_t* dk,
                                                                 uint16_t* dv) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  uint16_t* to = blockIdx.y ? dv : dk;
  if (i >= n || !to) return;
  const float* from = blockIdx.y ? part_v : part_k;
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
  for (int p = 0; p < parts; ++p) {
    a += *reinterpret_cast<const f32x4*>(from + p * n + i);
    b += *reinterpret_cast<const f32x4*>(from + p * n + i + 4);
  }
  const u32x2 x = pack4<T>(a), y = pack4<T>(b);
  *reinterpret_cast<u32x4a*>(to + i) = u32x4a{x[0], x[1], y[0], y[1]};
}

int64_t key_tiles(const AttentionCall& c) {
  return c.q_offsets ? c.k_tokens / kKeyRows + c.batch + 2 : (int64_t)((c.k_tokens + kKeyRows - 1) / kKeyRows) * c.batch;
}
int64_t key_values(const AttentionCall& c) { return (int64_t)(c.q_offsets ? 1 : c.batch) * c.k_tokens * c.kv_heads * c.dim; }

template <typename T, int kDim, bool kPadded, int kHalves>
int launch_dq(const AttentionCall& c, hipStream_t stream) {
  constexpr int kQueries = 128 / kHalves, kBytes = 4 * kKeys * pitch_of(kDim) * 2;
  const int64_t tiles = c.q_offsets ? (int64_t)c.q_tokens / kQueries + c.batch + 2 : (int64_t)((c.q_tokens + kQueries - 1) / kQueries) * c.batch;
  if (!launches(tiles * c.heads, 256)) return MFQ_ESHAPE;
  static PerDeviceInt configured;
  if (!raise_lds_limit(configured, reinterpret_cast<const void*>(&attention_dq_kernel<T, kDim, kPadded, kHalves>), kBytes)) return MFQ_ELAUNCH;
  hipLaunchKernelGGL((attention_dq_kernel<T, kDim, kPadded, kHalves>), dim3((unsigned)(tiles * c.heads)), dim3(256), kBytes, stream, c, (int)tiles);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T, int kDim>
int launch(const AttentionCall& c, int parts, float* workspace, hipStream_t stream) {
  using S = KeyShape<kDim>;
  const int64_t tiles = key_tiles(c), n = key_values(c);
  if ((c.dk || c.dv) && !launches(tiles * c.kv_heads * parts, 64 * S::kWaves)) return MFQ_ESHAPE;
  // 64 queries to a workgroup where 128 leave compute units idle, or (causal) the longest of them working alone: causal heads of 128,
  // 2048 tokens x 8 heads (128 such workgroups) 49 against 60 us, 4096 x 16 (512) 131 and 156, 4608 x 24 (864) 242 and 220; not causal,
  // 1500 x 24 (288) 90 and 71, 2048 x 24 (384) 93 and 89.
  const int64_t groups = (c.q_offsets ? c.q_tokens / 128 + c.batch : (int64_t)((c.q_tokens + 127) / 128) * c.batch) * c.heads;
  const bool halves = 2 * groups <= (c.causal ? 4 : 1) * (int64_t)compute_units();
  int rc;
  if constexpr (kDim <= 128)
    rc = c.dim < kDim ? (halves ? launch_dq<T, kDim, true, 2>(c, stream) : launch_dq<T, kDim, true, 1>(c, stream))
                      : (halves ? launch_dq<T, kDim, false, 2>(c, stream) : launch_dq<T, kDim, false, 1>(c, stream));
  else
    rc = c.dim < kDim ? launch_dq<T, kDim, true, 1>(c, stream) : launch_dq<T, kDim, false, 1>(c, stream);
  if (rc != MFQ_OK) return rc;
  if (!c.dk && !c.dv) return MFQ_OK;
  static PerDeviceInt configured;
  if (!raise_lds_limit(configured, reinterpret_cast<const void*>(&attention_dkv_kernel<T, kDim>), S::kLds)) return MFQ_ELAUNCH;
  float* part_v = parts > 1 ? workspace + parts * n : nullptr;
  hipLaunchKernelGGL((attention_dkv_kernel<T, kDim>), dim3((unsigned)(tiles * c.kv_heads * parts)), dim3(64 * S::kWaves), S::kLds, stream, c,
                     (int)tiles, parts, workspace, part_v);
  if (hipGetLastError() != hipSuccess) return MFQ_ELAUNCH;
  if (parts == 1) return MFQ_OK;
  hipLaunchKernelGGL(attention_dkv_join_kernel<T>, dim3((unsigned)((n / 8 + 255) / 256), 2), dim3(256), 0, stream, workspace, part_v, parts, n,
                     c.dk, c.dv);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T>
int launch_dim(const AttentionCall& c, int parts, float* workspace, hipStream_t stream) {
  if (c.dim <= 64) return launch<T, 64>(c, parts, workspace, stream);
  if (c.dim <= 96) return launch<T, 96>(c, parts, workspace, stream);
  if (c.dim <= 128) return launch<T, 128>(c, parts, workspace, stream);
  if (c.dim <= 192) return launch<T, 192>(c, parts, workspace, stream);
  return launch<T, 256>(c, parts, workspace, stream);
}

}  // namespace

int attention_backward_parts(const AttentionCall& c) {
  if (!c.dk && !c.dv) return 1;
  // three workgroups for every compute unit: causal ones differ in length by any factor
  const int64_t groups = key_tiles(c) * c.kv_heads, want = 3 * (int64_t)compute_units();
  return (int)std::min<int64_t>(c.heads / c.kv_heads, std::max<int64_t>(1, (want + groups - 1) / groups));
}

size_t attention_backward_bytes(const AttentionCall& c, int parts) { return parts > 1 ? (size_t)(2 * parts * key_values(c)) * 4 : 0; }

int launch_attention_backward(int dtype, const AttentionCall& c, int parts, void* workspace, hipStream_t stream) {
  return dtype == MFQ_BF16 ? launch_dim<BF16>(c, parts, (float*)workspace, stream) : launch_dim<F16>(c, parts, (float*)workspace, stream);
}

}  // namespace mfq
