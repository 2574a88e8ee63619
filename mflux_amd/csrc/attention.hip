// Attention over whole prompts and images: y = softmax(scale q k^T + mask) v for
// batched or packed sequences, grouped heads, causal or not
// (mx.fast.scaled_dot_product_attention in the reference,
// src/mflux/models/flux/model/flux_transformer/common/attention_utils.py:49).
//
// One pass over the keys with the softmax's running maximum and sum in float32; the scores never leave the registers.
// A workgroup of four wavefronts has 128 queries of one head, 32 a wavefront, and walks the keys 64 at a time: K and V
// tiles go straight from memory into LDS (two of each, the next in flight while the current one is multiplied) and are
// read by all four wavefronts.  Two workgroups share a compute unit.  See attention.h for the orientation of the products.
//
// 4608 tokens, 24 heads of 128, bfloat16, calls behind each other: 274 to 284 us on three cards, 0.92 to 0.95 PFLOP/s (a large library product: 1.39); 16384
// causal tokens, 28 / 4 heads: 1.84 to 1.92 ms, 1.00 to 1.04.  The counters show the matrix units busy in 41 % of the cycles, six vector instructions
// to a matrix instruction and no bank conflicts; power has a part as well, on zeros the first of these calls takes 227 us.  256 queries to a
// workgroup, three stages of tiles, 128 keys a step and wavefront priorities were tried and were no faster.
#include "attention.h"

namespace mfq {
namespace {

constexpr int kKeys = 64;  // of a step

constexpr int pitch_of(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// kPadded: the head is smaller than kDim
template <typename T, int kDim, bool kPadded>
__global__ __launch_bounds__(256, kDim <= 128 ? 2 : 1) void attention_kernel(AttentionCall c, int tiles) {
  constexpr int kQueries = 128;  // of a workgroup
  constexpr int kPitch = pitch_of(kDim);
  constexpr int kTileBytes = kKeys * kPitch * 2;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // K, V, K, V
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = uniform(thread / kWave);
  int head, index;
  head_and_tile(blockIdx.x, c.heads, tiles, c.causal || c.q_offsets, head, index);
  const Run run = find_run<kQueries>(c, index, false, c.causal);
  if (!run.valid) return;
  const int kv_head = head / (c.heads / c.kv_heads);

  const int row = run.tile * kQueries + wave * 32 + (lane & 31);  // of the run: the lane's query
  const int limit = visible_keys(run, row, c.causal);
  // keys that any query of the workgroup sees: the last one's, as limits grow along the rows
  const int keys = uniform(run.tile * kQueries < run.nq ? visible_keys(run, min(run.tile * kQueries + kQueries, run.nq) - 1, c.causal) : 0);
  const int least = wave_min(row < run.nq ? limit : INT32_MAX), most = wave_max(limit);

  QueryState<T, kDim, kPitch> state;
  state.init();
  if (keys > 0) {
    const int64_t q_at = run.batch * c.q.batch + (int64_t)(run.q0 + min(row, run.nq - 1)) * c.q.token + head * c.q.head;
    state.load_row(state.q, c.q.p + q_at, c.dim, lane);
    const uint16_t* k = uniform(c.k.p + run.batch * c.k.batch + (int64_t)run.k0 * c.k.token + kv_head * c.k.head);
    const uint16_t* v = uniform(c.v.p + run.batch * c.v.batch + (int64_t)run.k0 * c.v.token + kv_head * c.v.head);
    TileLoader<kPitch, kKeys, 256, kPadded> load_k;
    TileLoader<kPitch, kKeys, 256> load_v;
    load_k.init(thread, c.k.token, c.dim);
    load_v.init(thread, c.v.token, c.dim);
    const uint32_t lds_at = (uint32_t)(uintptr_t)lds;
    const float scale = c.scale * kLog2e;
    auto request_k = [&](int first) __attribute__((always_inline)) {
      load_k.load(k + (int64_t)first * c.k.token, lds_at + (first / kKeys & 1) * 2 * kTileBytes, keys - first, thread);
    };
    auto request_v = [&](int first) __attribute__((always_inline)) {
      load_v.load(v + (int64_t)first * c.v.token, lds_at + (first / kKeys & 1) * 2 * kTileBytes + kTileBytes, keys - first, thread);
    };
    if constexpr (kPadded) {
      clear_padding<kPitch, kDim>(lds, kKeys, c.dim, thread, 256);
      clear_padding<kPitch, kDim>(lds + 2 * kTileBytes, kKeys, c.dim, thread, 256);
    }
    request_k(0);
    request_v(0);
    // Tiles that every query of the workgroup sees all of (those that are there: the others' rows are not stored) come first, by pairs, so
    // that their places in LDS are constants, in blocks of 32 keys whose two halves overlap with the neighbours'.  At the first block of a
    // tile its K has arrived (its V may be on the way), everyone is done with the K of the tile before, and the next one's is
    // requested into its place; at the second block the same goes for V.
    constexpr int kRequests = TileLoader<kPitch, kKeys, 256>::kLoads, kHalf = 32 * kPitch * 2;
    const int whole = uniform(c.causal ? visible_keys(run, run.tile * kQueries, 1) : run.nk) / (2 * kKeys) * (2 * kKeys);
    int first = 0, buffer = 0;
    if (whole > 0) {
      f32x16 s0, s1;
      auto arrive_k = [&](int at) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(kRequests) : "memory");
        if (at + kKeys < keys) request_k(at + kKeys);
      };
      auto arrive_v = [&](int at) __attribute__((always_inline)) {
        if (at + kKeys < keys) {
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(kRequests) : "memory");
          request_v(at + kKeys);
        } else {
          arrive_and_sync();
        }
      };
      constexpr int k0 = 0, v0 = kTileBytes, k1 = 2 * kTileBytes, v1 = 3 * kTileBytes;
      typename QueryState<T, kDim, kPitch>::Addresses places;
      places.init(lds, lane);
      auto three_blocks = [&](int at) __attribute__((always_inline)) {
        arrive_v(at);
        state.template overlapped<true>(s0, s1, places, k0 + kHalf, v0, scale);
        arrive_k(at + kKeys);
        state.template overlapped<true>(s1, s0, places, k1, v0 + kHalf, scale);
        arrive_v(at + kKeys);
        state.template overlapped<true>(s0, s1, places, k1 + kHalf, v1, scale);
      };
      arrive_k(0);
      state.scores(s0, places, k0);
      state.follow(state.maximum(s0), scale);
      three_blocks(0);
      for (first = 2 * kKeys; first < whole; first += 2 * kKeys) {
        arrive_k(first);
        state.template overlapped<true>(s1, s0, places, k0, v1 + kHalf, scale);
        three_blocks(first);
      }
      state.template overlapped<false>(s1, s0, places, 0, v1 + kHalf, scale);
    }
    // At the large heads what follows has offsets and queries of its own: with those of the loop above kept for it, the compiler spilled
    // them there as well, and as memory answers in order, each reload waited for the tiles requested before it
    // (4608 tokens x 24 heads of 192: 1615 us against 520; of 256: 2465 against 703).
    auto separate = [&]() __attribute__((always_inline)) {
      if constexpr (kDim > 128) {
        int own = thread;
        asm volatile("" : "+v"(own));
        load_k.init(own, c.k.token, c.dim);
        load_v.init(own, c.v.token, c.dim);
        int64_t at = q_at;
        asm volatile("" : "+v"(at));
        state.load_row(state.q, c.q.p + at, c.dim, own & (kWave - 1));
      }
    };
    // the tile of `buffer` has arrived and the next one is requested
    auto advance = [&](int at) __attribute__((always_inline)) {
      arrive_and_sync();
      if (at + kKeys < keys) {
        request_k(at + kKeys);
        request_v(at + kKeys);
      }
    };
    // the others in blocks of 32 keys, so that of a wavefront's own edge only what lies across it is masked
    bool not_finite = false;
    separate();
#pragma unroll 1
    for (; first < keys; first += kKeys, buffer ^= 1) {
      advance(first);
#pragma unroll 1
      for (int at = first; at < min(first + kKeys, most); at += 32) {
        const char* k32 = lds + buffer * 2 * kTileBytes + (at - first) * kPitch * 2;
        if (at + 32 <= least) state.template step<1, false>(k32, k32 + kTileBytes, 32, scale, lane);
        else not_finite |= state.template step<1, true>(k32, k32 + kTileBytes, limit - at, scale, lane);
      }
    }
    if (whole < keys && any_wave<4>(not_finite, lds)) {
      state.init();
      separate();
      request_k(0);
      request_v(0);
#pragma unroll 1
      for (first = 0, buffer = 0; first < keys; first += kKeys, buffer ^= 1) {
        advance(first);
#pragma unroll 1
        for (int at = first; at < min(first + kKeys, most); at += 32) {
          const char* k32 = lds + buffer * 2 * kTileBytes + (at - first) * kPitch * 2;
          state.template step<1, true, true>(k32, k32 + kTileBytes, limit - at, scale, lane);
        }
      }
    }
  }
  if (row >= run.rows) return;
  const float sum = sum_halves(state.sum);
  const int64_t at = (int64_t)run.batch * c.q_tokens + run.q0 + row;  // of the densely packed result
  const bool seen = limit > 0;
  const int64_t to = (at * c.heads + head) * c.dim;
  store_row<T, kDim / 32>(c.out + to, c.rest ? c.rest + to : nullptr, state.o, seen, 1.0f / sum, c.dim, lane);
  if (c.lse && lane < 32) {
    const int64_t rows = (int64_t)(c.q_offsets ? 1 : c.batch) * c.q_tokens;
    c.lse[head * rows + at] = seen ? state.log_sum(state.top, sum, c.scale * kLog2e) : __builtin_inff();
  }
}

template <typename T, int kDim, bool kPadded>
int launch(const AttentionCall& c, hipStream_t stream) {
  constexpr int kQueries = 128;  // of a workgroup
  constexpr int kBytes = 4 * kKeys * pitch_of(kDim) * 2;
  // packed: a tile that is not full for every sequence at most, and for the rows in front of and behind them
  const int64_t tiles = c.q_offsets ? (int64_t)c.q_tokens / kQueries + c.batch + 2 : (int64_t)((c.q_tokens + kQueries - 1) / kQueries) * c.batch;
  if (!launches(tiles * c.heads, 256)) return MFQ_ESHAPE;
  static PerDeviceInt configured;
  if (!raise_lds_limit(configured, reinterpret_cast<const void*>(&attention_kernel<T, kDim, kPadded>), kBytes)) return MFQ_ELAUNCH;
  hipLaunchKernelGGL((attention_kernel<T, kDim, kPadded>), dim3((unsigned)(tiles * c.heads)), dim3(256), kBytes, stream, c, (int)tiles);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T, int kDim>
int launch_padded(const AttentionCall& c, hipStream_t stream) {
  return c.dim < kDim ? launch<T, kDim, true>(c, stream) : launch<T, kDim, false>(c, stream);
}

template <typename T>
int launch_dim(const AttentionCall& c, hipStream_t stream) {
  if (c.dim <= 64) return launch_padded<T, 64>(c, stream);
  if (c.dim <= 96) return launch_padded<T, 96>(c, stream);
  if (c.dim <= 128) return launch_padded<T, 128>(c, stream);
  if (c.dim <= 192) return launch_padded<T, 192>(c, stream);
  return launch_padded<T, 256>(c, stream);
}

}  // namespace

int launch_attention(int dtype, const AttentionCall& c, hipStream_t stream) {
  return dtype == MFQ_BF16 ? launch_dim<BF16>(c, stream) : launch_dim<F16>(c, stream);
}

}  // namespace mfq
