// Attention of few queries against many keys (single tokens over a cache): y = softmax(scale q k^T + mask) v with the key axis
// split over workgroups and joined behind them.
//
// Bound by the bytes of K and V, which are read once: the query heads that share a key head are the columns of one product (32
// rows = tokens x heads of a group to a workgroup), and every wavefront streams key tiles of its own through a ring in LDS
// that no other wavefront waits for.  The wavefronts of a workgroup are joined in LDS, the workgroups of a sequence by a second
// launch over their float32 partial results (none if the axis is not split).
//
// One token of 32 sequences of up to 8192 keys, 32 / 8 heads of 128: 124 us, 602 MB, 4.9 TB/s (as a large copy), 5 us of them the join;
// 205 MB of keys and values of one sequence: 47 us, 4.4 TB/s, 6 of them the join.  Prompts too small for tiles of 128 queries come
// here as well (attention_splits).
#include "attention.h"

#include <algorithm>
#include <type_traits>

namespace mfq {
namespace {

constexpr int kRows = 32;  // of a workgroup: (token, head of the group) pairs
constexpr int kStep = 32;  // keys of a step of a wavefront

constexpr int pitch_of(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
constexpr int waves_of(int dim) { return dim <= 128 ? 4 : 2; }

template <typename T, int kDim>
struct SplitShape {
  static constexpr int kPitch = pitch_of(kDim), kWaves = waves_of(kDim);
  static constexpr int kTile = kStep * kPitch * 2;            // bytes
  static constexpr int kRing = 2 * kTile > kRows * (kDim + 4) * 4 ? 2 * kTile : kRows * (kDim + 4) * 4;  // of a wavefront: K, V
  static constexpr int kPart = kRows * (kDim + 4) * 4;        // a wavefront's result on its way to the others
  static constexpr int kStats = kWaves * kRing;               // where its statistics lie
  static constexpr int kLds = kStats + kWaves * kRows * 8;
  static_assert(kPart <= kRing, "a wavefront's result fits its ring");
};

template <typename T, int kDim, bool kPadded>
__global__ __launch_bounds__(64 * waves_of(kDim), kDim <= 128 ? 2 : 1) void attention_split_kernel(AttentionCall c, int splits, int least_chunk, float* part_o,
                                                                                 float2* part_stats) {
  using S = SplitShape<T, kDim>;
  constexpr int kPitch = S::kPitch, kWaves = S::kWaves;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = uniform(thread / kWave);
  // neighbours: the heads of the same tokens, which lie side by side in memory
  const int kv_head = blockIdx.x % c.kv_heads, item = blockIdx.x / c.kv_heads;
  const int split = item % splits, group = c.heads / c.kv_heads;
  const Run run = find_run<kRows>(c, item / splits, false, false, group);
  if (!run.valid) return;

  const int row = run.tile * kRows + (lane & 31), token = row / group, head = kv_head * group + row % group;
  const int limit = visible_keys(run, token, c.causal);
  const int most = wave_max(limit), least = wave_min(token < run.nq ? limit : INT32_MAX);
  const int chunk = max(((run.nk + splits - 1) / splits + kStep - 1) / kStep * kStep, least_chunk);
  const int begin = split * chunk, end = min(min(begin + chunk, run.nk), most);

  QueryState<T, kDim, kPitch> state;
  state.init();
  if (begin < end) {
    const int64_t q_at = run.batch * c.q.batch + (int64_t)(run.q0 + min(token, run.nq - 1)) * c.q.token + head * c.q.head;
    state.load_row(state.q, c.q.p + q_at, c.dim, lane);
    const uint16_t* k = uniform(c.k.p + run.batch * c.k.batch + (int64_t)run.k0 * c.k.token + kv_head * c.k.head);
    const uint16_t* v = uniform(c.v.p + run.batch * c.v.batch + (int64_t)run.k0 * c.v.token + kv_head * c.v.head);
    TileLoader<kPitch, kStep, 64, kPadded> load_k;
    TileLoader<kPitch, kStep, 64> load_v;
    load_k.init(lane, c.k.token, c.dim);
    load_v.init(lane, c.v.token, c.dim);
    const uint32_t ring_at = (uint32_t)(uintptr_t)lds + wave * S::kRing;
    const float scale = c.scale * kLog2e;
    // A tile of K and one of V in LDS: the next K is requested when the scores are made, the next V behind the second product, so one
    // of them is always in flight (and eight wavefronts share a compute unit).  A wavefront's requests arrive in order: with the later
    // tile's still out, the earlier one is there.
    constexpr int kRequests = TileLoader<kPitch, kStep, 64>::kLoads;
    const char* k_tile = lds + wave * S::kRing;
    const char* v_tile = k_tile + S::kTile;
    auto request_k = [&](int first) __attribute__((always_inline)) {
      load_k.load(k + (int64_t)first * c.k.token, ring_at, run.nk - first, lane);
    };
    auto request_v = [&](int first) __attribute__((always_inline)) {
      load_v.load(v + (int64_t)first * c.v.token, ring_at + S::kTile, run.nk - first, lane);
    };
    int first = begin + wave * kStep;
    auto start = [&]() __attribute__((always_inline)) {
      if (first < end) {
        request_k(first);
        request_v(first);
      }
    };
    enum { kWhole, kEdge, kRowByRow };
    // the tile at `first`, whose mode is one value
    auto tile = [&](auto mode) __attribute__((always_inline)) {
      constexpr int kMode = decltype(mode)::value;
      bool not_finite = false;
      const int next = first + kWaves * kStep;
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kRequests) : "memory");
      auto between = [&]() __attribute__((always_inline)) {
        if (next < end) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read
          request_k(next);
          asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kRequests) : "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
      };
      if constexpr (kMode == kWhole) state.template step<1, false>(k_tile, v_tile, kStep, scale, lane, between);
      else not_finite = state.template step<1, true, kMode == kRowByRow>(k_tile, v_tile, limit - first, scale, lane, between);
      if (next < end) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and V
        request_v(next);
      }
      first = next;
      return not_finite;
    };
    // at the largest heads what follows the whole tiles has offsets and queries of its own (attention.hip has the reason)
    auto separate = [&]() __attribute__((always_inline)) {
      if constexpr (kDim > 192) {
        int own = lane;
        asm volatile("" : "+v"(own));
        load_k.init(own, c.k.token, c.dim);
        load_v.init(own, c.v.token, c.dim);
        int64_t at = q_at;
        asm volatile("" : "+v"(at));
        state.load_row(state.q, c.q.p + at, c.dim, own);
      }
    };
    if constexpr (kPadded) clear_padding<kPitch, kDim>(lds + wave * S::kRing, kStep, c.dim, lane, kWave);
    start();
#pragma unroll 1
    while (first < end && first + kStep <= least) tile(std::integral_constant<int, kWhole>());
    separate();
    bool not_finite = false;
#pragma unroll 1
    while (first < end) not_finite |= tile(std::integral_constant<int, kEdge>());
    if (not_finite) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      state.init();
      separate();
      first = begin + wave * kStep;
      start();
#pragma unroll 1
      while (first < end) tile(std::integral_constant<int, kRowByRow>());
    }
  }

  // join the wavefronts: their accumulators and statistics through LDS, rows of kDim + 4 floats
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  constexpr int kFloats = kDim + 4;
  float* mine = reinterpret_cast<float*>(lds + wave * S::kRing) + (lane & 31) * kFloats;
#pragma unroll
  for (int b = 0; b < kDim / 32; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<f32x4*>(mine + 32 * b + result_row(i, lane)) = f32x4{state.o[b][i], state.o[b][i + 1], state.o[b][i + 2], state.o[b][i + 3]};
  float2* stats = reinterpret_cast<float2*>(lds + S::kStats);
  const float sum = sum_halves(state.sum);
  if (lane < 32) stats[wave * kRows + lane] = make_float2(state.top, sum);
  __syncthreads();
  const float c2 = c.scale * kLog2e;
  const int64_t rows = (int64_t)(c.q_offsets ? 1 : c.batch) * c.q_tokens;
  // a thread: four elements of a row at a time
  for (int i = thread; i < kRows * (kDim / 4); i += kWaves * kWave) {
    const int r = i / (kDim / 4), d = i % (kDim / 4) * 4;
    const int p = run.tile * kRows + r, tok = p / group;
    if (tok >= run.rows || d >= c.dim) continue;
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w * kRows + r].x);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 st = stats[w * kRows + r];
      // a part without keys has the factor 0; where the reference is an infinity the scores' own NaN stay
      const float f = st.x == top ? 1.f : __builtin_amdgcn_exp2f((st.x - top) * c2);
      total += st.y * f;
      const f32x4 a = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * S::kRing) + r * kFloats + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += a[e] * f;
    }
    const int64_t at = ((int64_t)run.batch * c.q_tokens + run.q0 + tok) * c.heads + kv_head * group + p % group;
    if (splits == 1) {
      const bool seen = visible_keys(run, tok, c.causal) > 0;
      const float f = 1.0f / total;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = seen ? o[e] * f : 0.f;
      const u32x2 packed = pack4<T>(o);
      *reinterpret_cast<u32x2*>(c.out + at * c.dim + d) = packed;
      if (c.rest) *reinterpret_cast<u32x2*>(c.rest + at * c.dim + d) = pack4_rest<T>(o, packed);
      if (c.lse && d == 0)
        c.lse[(at % c.heads) * rows + at / c.heads] = seen ? state.log_sum(top, total, c2) : __builtin_inff();
    } else {
      const int64_t slot = (int64_t)split * rows * c.heads + at;
      if (begin < run.nk) *reinterpret_cast<f32x4*>(part_o + slot * c.dim + d) = o;
      // a range in which the row sees no key has the sum -1: one in which its scores are all -infinity has the sum 0
      if (d == 0) part_stats[slot] = make_float2(top, visible_keys(run, tok, c.causal) > begin ? total : -1.f);
    }
  }
}

// y = the partial results of a row joined: a workgroup to a row, a quarter wavefront (half of one above 64 elements, a whole one
// above 128) to every split of its own, four elements a lane
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(AttentionCall c, int64_t rows, int splits, const float* part_o, const float2* part_stats) {
  __shared__ float tops[4], sums[4];
  __shared__ __attribute__((aligned(16))) float parts[16][256];
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = thread / kWave;
  const int64_t at = blockIdx.x, step = rows * c.heads;
  const float c2 = c.scale * kLog2e;
  float top = -__builtin_inff();
  for (int s = thread; s < splits; s += 256) top = fmaxf(top, part_stats[s * step + at].x);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const int lanes = c.dim <= 64 ? 16 : c.dim <= 128 ? 32 : 64, groups = 256 / lanes;
  const int mine = thread / lanes, d = thread % lanes * 4;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float total = 0.f;
#pragma unroll 4
  for (int s = mine; s < splits; s += groups) {
    const float2 st = part_stats[s * step + at];
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    const bool seen = !(st.y < 0.f);  // (a sum that is NaN is a row's own)
    if (d < c.dim && seen) a = *reinterpret_cast<const f32x4*>(part_o + (s * step + at) * c.dim + d);
    // where the reference is an infinity the scores' own NaN stay
    const float f = st.x == top ? 1.f : __builtin_amdgcn_exp2f((st.x - top) * c2);
    total += seen ? st.y * f : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += a[e] * f;
  }
  if (thread % lanes != 0) total = 0.f;  // one lane of a group counts
#pragma unroll
  for (int n = 1; n < kWave; n *= 2) total += __shfl_xor(total, n);
  if (lane == 0) sums[wave] = total;
  *reinterpret_cast<f32x4*>(&parts[mine][d]) = o;
  __syncthreads();
  if (mine) return;
  total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  const bool empty = part_stats[at].y < 0.f;  // a row that sees any key sees the first one
  const float f = 1.0f / total;
  if (d < c.dim) {
    for (int g = 1; g < groups; ++g) o += *reinterpret_cast<const f32x4*>(&parts[g][d]);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = empty ? 0.f : o[e] * f;
    const u32x2 packed = pack4<T>(o);
    *reinterpret_cast<u32x2*>(c.out + at * c.dim + d) = packed;
    if (c.rest) *reinterpret_cast<u32x2*>(c.rest + at * c.dim + d) = pack4_rest<T>(o, packed);
  }
  if (c.lse && thread == 0) c.lse[(at % c.heads) * rows + at / c.heads] = empty ? __builtin_inff() : top * c2 + (__builtin_amdgcn_logf(total) - kLift<T>);
}

// keys of a call's longest sequence as the host knows it, over the splits
int least_chunk(const AttentionCall& c, int splits) {
  const int64_t keys = c.q_offsets ? (c.k_tokens + c.batch - 1) / c.batch : c.k_tokens;
  return (int)(((keys + splits - 1) / splits + kStep - 1) / kStep * kStep);
}

int64_t rows_of(const AttentionCall& c) { return (int64_t)(c.q_offsets ? 1 : c.batch) * c.q_tokens; }
int64_t tiles_of(const AttentionCall& c) {
  const int64_t group = c.heads / c.kv_heads;
  return c.q_offsets ? c.q_tokens * group / kRows + c.batch + 2 : (c.q_tokens * group + kRows - 1) / kRows * c.batch;
}

template <typename T, int kDim, bool kPadded>
int launch(const AttentionCall& c, int splits, float* workspace, hipStream_t stream) {
  using S = SplitShape<T, kDim>;
  const int64_t tiles = tiles_of(c), rows = rows_of(c), grid = tiles * c.kv_heads * splits;
  if (!launches(grid, 64 * S::kWaves)) return MFQ_ESHAPE;
  static PerDeviceInt configured;
  if (!raise_lds_limit(configured, reinterpret_cast<const void*>(&attention_split_kernel<T, kDim, kPadded>), S::kLds)) return MFQ_ELAUNCH;
  float* part_o = workspace;
  float2* part_stats = splits > 1 ? reinterpret_cast<float2*>(workspace + splits * rows * c.heads * c.dim) : nullptr;
  hipLaunchKernelGGL((attention_split_kernel<T, kDim, kPadded>), dim3((unsigned)grid), dim3(64 * S::kWaves), S::kLds, stream, c, splits,
                     least_chunk(c, splits), part_o, part_stats);
  if (hipGetLastError() != hipSuccess) return MFQ_ELAUNCH;
  if (splits == 1) return MFQ_OK;
  hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)(rows * c.heads)), dim3(256), 0, stream, c, rows, splits, part_o, part_stats);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T, int kDim>
int launch_padded(const AttentionCall& c, int splits, float* workspace, hipStream_t stream) {
  return c.dim < kDim ? launch<T, kDim, true>(c, splits, workspace, stream) : launch<T, kDim, false>(c, splits, workspace, stream);
}

template <typename T>
int launch_dim(const AttentionCall& c, int splits, float* workspace, hipStream_t stream) {
  if (c.dim <= 64) return launch_padded<T, 64>(c, splits, workspace, stream);
  if (c.dim <= 96) return launch_padded<T, 96>(c, splits, workspace, stream);
  if (c.dim <= 128) return launch_padded<T, 128>(c, splits, workspace, stream);
  if (c.dim <= 192) return launch_padded<T, 192>(c, splits, workspace, stream);
  return launch_padded<T, 256>(c, splits, workspace, stream);
}

}  // namespace

int attention_splits(const AttentionCall& c) {
  const int64_t group = c.heads / c.kv_heads, units = compute_units();
  // mean queries and keys of a sequence
  const int64_t queries = c.q_offsets ? (c.q_tokens + c.batch - 1) / c.batch : c.q_tokens;
  const int64_t keys = c.q_offsets ? (c.k_tokens + c.batch - 1) / c.batch : c.k_tokens;
  const int64_t items = std::max<int64_t>(tiles_of(c) - (c.q_offsets ? 2 : 0), 1) * c.kv_heads;
  if (queries * group <= kRows) {
    // Single tokens: eight workgroups for every compute unit, so that sequences of different lengths fill it evenly (32 of them, 1024 to
    // 8192 keys, 8 key heads: 129, 137, 126, 125 us with one, four, eight, sixteen ranges), each with 256 keys at least; and at most 64
    // ranges, which the join reads behind each other (one sequence of 100003 keys, 4 key heads, from a cache: 39, 43, 50 us with 64, 128, 256).
    // The keys of a range are counted by the tensor's length where a sequence's own is shorter.
    const int64_t want = (8 * units + items - 1) / items;
    return (int)std::min({std::max<int64_t>(keys / 256, 1), want, (int64_t)64});
  }
  // A prompt whose tiles of 128 queries leave compute units idle: 32 rows to a workgroup, the keys dealt to its wavefronts, is as much
  // work on four times the units (heads of 128, causal: 1024 tokens x 8 heads 15.1 us here, 25.3 there; 2048 x 8, 128 such tiles, 28.2
  // and 42.4; 1024 x 24, 192, 25.0 and 26.8).  The limit is one for all calls and lies between theirs: at 256 tiles (2048 x 16, causal) heads of
  // 64 take 25.7 and 32.0, of 128 42.0 and 43.6, of 256 114 and 99; without a mask 2048 x 8 heads of 128 take 31.0 and 40.6, 1024 x 24 29.2 and 25.1.
  const int64_t tiles = (c.q_offsets ? c.q_tokens / 128 + c.batch : (int64_t)((c.q_tokens + 127) / 128) * c.batch) * c.heads;
  if (4 * tiles > 3 * units) return 0;
  // and the keys in ranges where even those are few (128 queries x 8 heads against 32768 keys: 301, 86, 50, 43, 79 us with 1, 4, 8, 16
  // and 32; 128 against 4096: 37, 18, 15, 16, 23), but not where the join has as many rows again (1024 x 8: 14.3 us with 1, 24 with 2)
  if (2 * items > units) return 1;
  return (int)std::max<int64_t>(std::min({keys / 512, 2 * units / items, (int64_t)64}), 1);
}

size_t attention_split_bytes(const AttentionCall& c, int splits) {
  return splits > 1 ? (size_t)(splits * rows_of(c) * c.heads) * (c.dim + 2) * 4 : 0;
}

int launch_attention_split(int dtype, const AttentionCall& c, int splits, void* workspace, hipStream_t stream) {
  return dtype == MFQ_BF16 ? launch_dim<BF16>(c, splits, (float*)workspace, stream) : launch_dim<F16>(c, splits, (float*)workspace, stream);
}

}  // namespace mfq
