// The gradients of attention (attention.hip):
//   P = softmax(scale q k^T + mask), dP = dy v^T, dS = P (dP - sum(dy y)), dv = P^T dy, dq = scale dS k, dk = scale dS^T q
// with P made again from the forward pass's log-sum-exp of each row.  Two launches: one walks the keys of a tile of queries (dq, and
// the rows' sums of dy y, which the other needs), one the queries of a tile of keys (dk and dv, over all heads that share them).
// That makes the scores twice, 14 instead of 10 operations a pair and element of a head, and no sum is made by atomics, so the
// gradients are the same bits every time.  All sums are float32; P and dS are rounded to the inputs' type for the second products,
// as P is in the forward pass.
#include "attention.h"

#include <type_traits>

namespace mfq {
namespace {

constexpr int pitch_of(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

constexpr int kQueries = 128;  // of a workgroup of the first kernel
constexpr int kKeys = 64;      // of its step

template <typename T, int kDim>
__global__ __launch_bounds__(256, kDim <= 96 ? 2 : 1) void attention_dq_kernel(AttentionCall c, int tiles) {
  constexpr int kPitch = pitch_of(kDim), kSteps = kDim / 16, kBlocks = kDim / 32;
  constexpr int kTileBytes = kKeys * kPitch * 2;
  using vec8 = typename T::vec8;
  using Row = QueryState<T, kDim, kPitch>;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // K, V, K, V
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = uniform(thread / kWave);
  int head, index;
  head_and_tile(blockIdx.x, c.heads, tiles, head, index);
  const Run run = find_run<kQueries>(c, index, false, c.causal);
  if (!run.valid) return;
  const int kv_head = head / (c.heads / c.kv_heads);
  const int row = run.tile * kQueries + wave * 32 + (lane & 31);
  const int limit = visible_keys(run, row, c.causal);
  const int keys = uniform(run.tile * kQueries < run.nq ? visible_keys(run, min(run.tile * kQueries + kQueries, run.nq) - 1, c.causal) : 0);
  const int least = wave_min(limit), most = wave_max(limit);
  const int64_t rows = (int64_t)(c.q_offsets ? 1 : c.batch) * c.q_tokens;
  const int64_t at = (int64_t)run.batch * c.q_tokens + run.q0 + row;

  f32x16 dq[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) dq[b] = zero16();
  float delta = 0.f;
  if (keys > 0) {
    const int64_t inside = run.q0 + min(row, run.nq - 1);
    vec8 q[kSteps], dy[kSteps];
    Row::load_row(q, c.q.p + run.batch * c.q.batch + inside * c.q.token + head * c.q.head, c.dim, lane);
    Row::load_row(dy, c.dy.p + run.batch * c.dy.batch + inside * c.dy.token + head * c.dy.head, c.dim, lane);
    {
      vec8 y[kSteps];
      Row::load_row(y, c.y.p + run.batch * c.y.batch + inside * c.y.token + head * c.y.head, c.dim, lane);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const u32x4a a = __builtin_bit_cast(u32x4a, dy[s]), b = __builtin_bit_cast(u32x4a, y[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          delta = __builtin_fmaf(lo_f32<T>(a[i]), lo_f32<T>(b[i]), delta);
          delta = __builtin_fmaf(hi_f32<T>(a[i]), hi_f32<T>(b[i]), delta);
        }
      }
      delta = sum_halves(delta);
    }
    const float lse = c.lse[head * rows + (int64_t)run.batch * c.q_tokens + inside];
    const uint16_t* k = uniform(c.k.p + run.batch * c.k.batch + (int64_t)run.k0 * c.k.token + kv_head * c.k.head);
    const uint16_t* v = uniform(c.v.p + run.batch * c.v.batch + (int64_t)run.k0 * c.v.token + kv_head * c.v.head);
    TileLoader<kPitch, kKeys, 256> load_k, load_v;
    load_k.init(thread, c.k.token, c.dim);
    load_v.init(thread, c.v.token, c.dim);
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;
    const float scale = c.scale * kLog2e;

    auto step = [&](const char* k_tile, const char* v_tile, int left, auto masked) __attribute__((always_inline)) {
      constexpr bool kMasked = decltype(masked)::value;
      bool one_by_one = false;
      if constexpr (kMasked) one_by_one = tile_not_finite<T, kPitch, kSteps, kKeys / 32>(k_tile, lane);
#pragma unroll
      for (int t = 0; t < kKeys / 32; ++t) {
        const char* k32 = k_tile + t * 32 * kPitch * 2;
        const char* v32 = v_tile + t * 32 * kPitch * 2;
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int e = 0; e < kSteps; ++e) s = mfma32(tile_rows<T, kPitch>(k32, e, lane), q[e], s);
#pragma unroll
        for (int e = 0; e < kSteps; ++e) dp = mfma32(tile_rows<T, kPitch>(v32, e, lane), dy[e], dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale, -lse));
          s[i] = p * (dp[i] - delta);
          if (kMasked && 32 * t + result_row(i, lane) >= left) s[i] = 0.f;
        }
#pragma unroll
        for (int slab = 0; slab < 2; ++slab) {
          const vec8 ds = result_operand<T>(s, slab);
          const char* k16 = k32 + slab * 16 * kPitch * 2;
          if (kMasked && __builtin_expect(one_by_one, 0))
            add_columns_one_by_one<T, kPitch, kBlocks>(dq, k16, ds, lane, [&](int r) { return 32 * t + 16 * slab + r < left; });
          else
            add_columns<T, kPitch, kBlocks>(dq, k16, ds, lane);
        }
      }
    };
    load_k.load(k, lds_at, keys, thread);
    load_v.load(v, lds_at + kTileBytes, keys, thread);
    for (int first = 0, buffer = 0; first < keys; first += kKeys, buffer ^= 1) {
      arrive_and_sync();
      const int next = first + kKeys;
      if (next < keys) {
        const uint32_t to = lds_at + (buffer ^ 1) * 2 * kTileBytes;
        load_k.load(k + (int64_t)next * c.k.token, to, keys - next, thread);
        load_v.load(v + (int64_t)next * c.v.token, to + kTileBytes, keys - next, thread);
      }
      const char* k_tile = lds + buffer * 2 * kTileBytes;
      if (next <= least) step(k_tile, k_tile + kTileBytes, kKeys, std::false_type());
      else if (first < most) step(k_tile, k_tile + kTileBytes, limit - first, std::true_type());
    }
  }
  if (row >= run.rows) return;
  if (c.delta && lane < 32) c.delta[head * rows + at] = delta;
  if (c.dq) store_row<T, kBlocks>(c.dq + (at * c.heads + head) * c.dim, dq, limit > 0 ? c.scale : 0.f, c.dim, lane);
}

constexpr int kKeyRows = 128;  // of a workgroup of the second kernel
constexpr int query_step(int dim) { return dim <= 128 ? 64 : 32; }

// 64 (32) floats from a row on into LDS, those past `rows` repeating the last one
__device__ inline void load_floats(const float* base, uint32_t lds, int rows, int count, int lane) {
  const uint32_t o = 4u * (uint32_t)min(min(lane, count - 1), rows - 1);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(o), "s"(uniform(base)), "s"(uniform((int)lds)) : "memory", "m0");
}

template <typename T, int kDim>
__global__ __launch_bounds__(256, 1) void attention_dkv_kernel(AttentionCall c, int tiles) {
  constexpr int kPitch = pitch_of(kDim), kSteps = kDim / 16, kBlocks = kDim / 32, kRows = query_step(kDim);
  constexpr int kTileBytes = kRows * kPitch * 2, kStage = 2 * kTileBytes + 512;  // q, dy, 64 log-sum-exps, 64 sums
  using vec8 = typename T::vec8;
  using Row = QueryState<T, kDim, kPitch>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = uniform(thread / kWave);
  int kv_head, index;
  head_and_tile(blockIdx.x, c.kv_heads, tiles, kv_head, index);
  const Run run = find_run<kKeyRows>(c, index, true, false);  // causal: the first keys have the most queries
  if (!run.valid) return;
  const int group = c.heads / c.kv_heads;
  const int row = run.tile * kKeyRows + wave * 32 + (lane & 31);  // the lane's key
  const int shift = run.nk - run.nq;  // causal: query i sees the keys up to i + shift
  // the queries that see the lane's key are [from, nq)
  const int from = row >= run.nk ? run.nq : c.causal ? min(max(row - shift, 0), run.nq) : 0;
  const int first_query = uniform(run.tile * kKeyRows >= run.nk ? run.nq : c.causal ? min(max(run.tile * kKeyRows - shift, 0), run.nq) : 0);
  const int wave_first = wave_min(from), wave_last = wave_max(from);
  const int begin = first_query / kRows * kRows;
  const int per_head = first_query < run.nq ? (run.nq - begin + kRows - 1) / kRows : 0;

  f32x16 dk[kBlocks], dv[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) dk[b] = dv[b] = zero16();
  if (per_head > 0) {
    const int64_t inside = run.k0 + min(row, run.nk - 1);
    vec8 k[kSteps], v[kSteps];
    Row::load_row(k, c.k.p + run.batch * c.k.batch + inside * c.k.token + kv_head * c.k.head, c.dim, lane);
    Row::load_row(v, c.v.p + run.batch * c.v.batch + inside * c.v.token + kv_head * c.v.head, c.dim, lane);
    TileLoader<kPitch, kRows, 256> load_q, load_dy;
    load_q.init(thread, c.q.token, c.dim);
    load_dy.init(thread, c.dy.token, c.dim);
    const uint16_t* q0 = uniform(c.q.p + run.batch * c.q.batch + (int64_t)run.q0 * c.q.token + (int64_t)kv_head * group * c.q.head);
    const uint16_t* dy0 = uniform(c.dy.p + run.batch * c.dy.batch + (int64_t)run.q0 * c.dy.token + (int64_t)kv_head * group * c.dy.head);
    const int64_t rows = (int64_t)(c.q_offsets ? 1 : c.batch) * c.q_tokens;
    const float* lse0 = uniform(c.lse + kv_head * group * rows + (int64_t)run.batch * c.q_tokens + run.q0);
    const float* delta0 = uniform(c.delta + kv_head * group * rows + (int64_t)run.batch * c.q_tokens + run.q0);
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;
    const float scale = c.scale * kLog2e;

    auto request = [&](int head, int first, int stage) __attribute__((always_inline)) {
      const uint32_t to = lds_at + stage * kStage;
      load_q.load(q0 + head * c.q.head + (int64_t)first * c.q.token, to, run.nq - first, thread);
      load_dy.load(dy0 + head * c.dy.head + (int64_t)first * c.dy.token, to + kTileBytes, run.nq - first, thread);
      if (wave == 0) load_floats(lse0 + head * rows + first, to + 2 * kTileBytes, run.nq - first, kRows, lane);
      if (wave == 1) load_floats(delta0 + head * rows + first, to + 2 * kTileBytes + 256, run.nq - first, kRows, lane);
    };
    // masked: left = the queries of the tile that there are, start = the first of them that sees the lane's key
    auto step = [&](const char* q_tile, int start, int left, auto masked) __attribute__((always_inline)) {
      constexpr bool kMasked = decltype(masked)::value;
      const char* dy_tile = q_tile + kTileBytes;
      const float* lse = reinterpret_cast<const float*>(q_tile + 2 * kTileBytes);
      const float* delta = lse + 64;
      bool one_by_one = false;
      if constexpr (kMasked)
        one_by_one = tile_not_finite<T, kPitch, kSteps, kRows / 32>(q_tile, lane) ||
                     tile_not_finite<T, kPitch, kSteps, kRows / 32>(dy_tile, lane);
#pragma unroll
      for (int t = 0; t < kRows / 32; ++t) {
        const char* q32 = q_tile + t * 32 * kPitch * 2;
        const char* dy32 = dy_tile + t * 32 * kPitch * 2;
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int e = 0; e < kSteps; ++e) s = mfma32(tile_rows<T, kPitch>(q32, e, lane), k[e], s);
#pragma unroll
        for (int e = 0; e < kSteps; ++e) dp = mfma32(tile_rows<T, kPitch>(dy32, e, lane), v[e], dp);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int r = 32 * t + result_row(i, lane);
          const f32x4 l = *reinterpret_cast<const f32x4*>(lse + r), d = *reinterpret_cast<const f32x4*>(delta + r);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + j], scale, -l[j]));
            float ds = p * (dp[i + j] - d[j]);
            if (kMasked && (r + j < start || r + j >= left)) p = ds = 0.f;
            s[i + j] = p;
            dp[i + j] = ds;
          }
        }
#pragma unroll
        for (int slab = 0; slab < 2; ++slab) {
          const vec8 p = result_operand<T>(s, slab), ds = result_operand<T>(dp, slab);
          const char* q16 = q32 + slab * 16 * kPitch * 2;
          const char* dy16 = dy32 + slab * 16 * kPitch * 2;
          if (kMasked && __builtin_expect(one_by_one, 0)) {
            auto visible = [&](int r) { return 32 * t + 16 * slab + r >= start && 32 * t + 16 * slab + r < left; };
            add_columns_one_by_one<T, kPitch, kBlocks>(dv, dy16, p, lane, visible);
            add_columns_one_by_one<T, kPitch, kBlocks>(dk, q16, ds, lane, visible);
          } else {
            add_columns<T, kPitch, kBlocks>(dv, dy16, p, lane);
            add_columns<T, kPitch, kBlocks>(dk, q16, ds, lane);
          }
        }
      }
    };
    request(0, begin, 0);
    int head = 0, first = begin;
    for (int i = 0, stage = 0; i < per_head * group; ++i, stage ^= 1) {
      arrive_and_sync();
      int next = first + kRows, next_head = head;
      if (next >= run.nq) {
        next = begin;
        ++next_head;
      }
      if (i + 1 < per_head * group) request(next_head, next, stage ^ 1);
      const char* q_tile = lds + stage * kStage;
      if (first >= wave_last && first + kRows <= run.nq) step(q_tile, 0, kRows, std::false_type());
      else if (first + kRows > wave_first) step(q_tile, from - first, run.nq - first, std::true_type());
      head = next_head;
      first = next;
    }
  }
  if (row >= run.rows) return;
  const int64_t at = ((int64_t)run.batch * c.k_tokens + run.k0 + row) * c.kv_heads + kv_head;
  const bool seen = from < run.nq;
  if (c.dk) store_row<T, kBlocks>(c.dk + at * c.dim, dk, seen ? c.scale : 0.f, c.dim, lane);
  if (c.dv) store_row<T, kBlocks>(c.dv + at * c.dim, dv, seen ? 1.f : 0.f, c.dim, lane);
}

template <typename T, int kDim>
int launch(const AttentionCall& c, hipStream_t stream) {
  const int64_t more = c.q_offsets ? c.batch + 2 : 0;  // as in the forward pass
  {
    constexpr int kBytes = 4 * kKeys * pitch_of(kDim) * 2;
    static PerDeviceInt configured;
    if (!raise_lds_limit(configured, reinterpret_cast<const void*>(&attention_dq_kernel<T, kDim>), kBytes)) return MFQ_ELAUNCH;
    const int64_t tiles = more ? c.q_tokens / kQueries + more : (int64_t)((c.q_tokens + kQueries - 1) / kQueries) * c.batch;
    if (tiles * c.heads > INT32_MAX) return MFQ_ESHAPE;
    hipLaunchKernelGGL((attention_dq_kernel<T, kDim>), dim3((unsigned)(tiles * c.heads)), dim3(256), kBytes, stream, c, (int)tiles);
    if (hipGetLastError() != hipSuccess) return MFQ_ELAUNCH;
  }
  if (!c.dk && !c.dv) return MFQ_OK;
  constexpr int kBytes = 2 * (2 * query_step(kDim) * pitch_of(kDim) * 2 + 512);
  static PerDeviceInt configured;
  if (!raise_lds_limit(configured, reinterpret_cast<const void*>(&attention_dkv_kernel<T, kDim>), kBytes)) return MFQ_ELAUNCH;
  const int64_t tiles = more ? c.k_tokens / kKeyRows + more : (int64_t)((c.k_tokens + kKeyRows - 1) / kKeyRows) * c.batch;
  if (tiles * c.kv_heads > INT32_MAX) return MFQ_ESHAPE;
  hipLaunchKernelGGL((attention_dkv_kernel<T, kDim>), dim3((unsigned)(tiles * c.kv_heads)), dim3(256), kBytes, stream, c, (int)tiles);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T>
int launch_dim(const AttentionCall& c, hipStream_t stream) {
  if (c.dim <= 64) return launch<T, 64>(c, stream);
  if (c.dim <= 96) return launch<T, 96>(c, stream);
  if (c.dim <= 128) return launch<T, 128>(c, stream);
  if (c.dim <= 192) return launch<T, 192>(c, stream);
  return launch<T, 256>(c, stream);
}

}  // namespace

int launch_attention_backward(int dtype, const AttentionCall& c, hipStream_t stream) {
  return dtype == MFQ_BF16 ? launch_dim<BF16>(c, stream) : launch_dim<F16>(c, stream);
}

}  // namespace mfq
