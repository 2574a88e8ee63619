// What the attention kernels (attention.hip, attention_split.hip,
// attention_backward.hip) share: which rows a workgroup has, tiles in LDS, and
// the products of tiles.
//
// One orientation throughout, on 32x32x16 matrix instructions.  A tile of scores
// is computed transposed, S^T = K Q^T (rows: keys, columns: queries), so a lane
// holds 16 keys' scores of ONE query: the softmax's maximum and sum are taken
// within a lane and over one exchange between the two halves of the wavefront,
// and its statistics are one register each.  The instruction's result is at once
// the next product's right operand, O^T = V^T P^T: lane (column, half h) holds keys
// {4h .. 4h+3} and {8+4h .. 8+4h+3} of each 16, and the left operand is read with
// the same order of keys (the transposing LDS read hands out four consecutive
// rows of a column at a time), so probabilities never move between lanes.
#pragma once

#include "common.h"

namespace mfq {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;

// ---- the call, as the kernels take it -------------------------------------------------------------------
struct AttentionTensor {
  const uint16_t* p = nullptr;
  int64_t batch = 0;         // elements from a batch entry to the next
  int64_t token = 0, head = 0;  // from a token, a head to the next
};

struct AttentionCall {
  AttentionTensor q, k, v, y, dy;  // y: the result, or in the backward pass the forward's
  uint16_t* rest = nullptr;  // y before its rounding minus y, densely packed: forward writes it where not nullptr, backward reads it
  uint16_t *out = nullptr, *dq = nullptr, *dk = nullptr, *dv = nullptr;  // densely packed, [(batch,) tokens, heads, dim]
  float* lse = nullptr;    // [heads][rows]: log2 of the sum of exp2 of the scaled scores, +inf for a row that sees nothing
  float* delta = nullptr;  // [heads][rows]: sum of dy * y
  const int32_t *q_offsets = nullptr, *k_offsets = nullptr;  // packed: batch + 1 each
  const int32_t *q_lengths = nullptr, *k_lengths = nullptr;  // batched: optional, batch each
  int batch = 0, heads = 0, kv_heads = 0, dim = 0;
  int q_tokens = 0, k_tokens = 0;  // batched: of an entry; packed: of all
  int causal = 0;
  float scale = 0.f;
};

// A run of rows that a workgroup walks: queries [q0, q0 + nq) and keys [k0, k0 + nk) of one sequence, in rows of its tensor
// (batched: of the entry).  Rows of the run that belong to no sequence have nq (nk) less than `rows`: they are written as zeros.
struct Run {
  int batch;       // entry of a batched call, 0 in a packed one
  int q0, nq, k0, nk;
  int rows;        // rows to write from q0 (k0 where a kernel goes by keys) on
  int tile;        // the workgroup's tile of `rows`
  bool valid;
};

__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <typename P>
__device__ inline const P* uniform(const P* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t low = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), high = __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return reinterpret_cast<const P*>((uintptr_t)((uint64_t)high << 32 | low));
}

// inclusive sum over the lanes
__device__ inline int wave_scan(int v) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Tile `index` of kTile rows among all sequences' tiles.  Packed calls: offsets are read clamped to the tensor (whatever they
// hold, no row outside it is touched), the rows in front of the first and behind the last sequence count as sequences without
// keys, and the sequences' tiles are counted by the lanes, one to a sequence, so the host needs no sequence's length: up to 62
// of them by decreasing number of keys, so that the longest workgroups start first, more in their own order.  `by_key`: tiles
// of key rows instead of query rows; `per`: rows that a token counts for.  `reverse`: the last tile first (causal: the longest
// first).
template <int kTile>
__device__ inline Run find_run(const AttentionCall& c, int index, bool by_key, bool reverse, int per = 1) {
  Run r;
  const int tokens = by_key ? c.k_tokens : c.q_tokens;
  if (!c.q_offsets) {
    const int tiles = (tokens * per + kTile - 1) / kTile;
    r.valid = index < tiles * c.batch;
    // tiles of the same place of all entries behind each other, so that a causal call starts all its long ones first
    const int place = index / c.batch;
    r.batch = index - place * c.batch;
    r.tile = reverse ? tiles - 1 - place : place;
    r.q0 = r.k0 = 0;
    const int b = r.valid ? r.batch : 0;
    r.nq = c.q_lengths ? min(max(c.q_lengths[b], 0), c.q_tokens) : c.q_tokens;
    r.nk = c.k_lengths ? min(max(c.k_lengths[b], 0), c.k_tokens) : c.k_tokens;
    r.rows = tokens;
    r.nq = uniform(r.nq);
    r.nk = uniform(r.nk);
    return r;
  }
  const int lane = threadIdx.x & (kWave - 1);
  const int n = c.batch + 2;
  const int32_t* offsets = by_key ? c.k_offsets : c.q_offsets;
  // the rows of sequence s - 1 (0 and n - 1: the rows in front of and behind all sequences)
  auto bounds = [&](const int32_t* o, int limit, int s, int& first, int& count) {
    const int a = s == 0 ? 0 : min(max(o[min(s, n - 1) - 1], 0), limit);
    const int b = s >= n - 1 ? limit : min(max(o[s], 0), limit);
    first = a;
    count = max(b - a, 0);
  };
  auto tiles_of = [&](int s) {
    int first, count = 0;
    if (s < n) bounds(offsets, tokens, s, first, count);
    return (count * per + kTile - 1) / kTile;
  };
  r.valid = false;
  r.batch = r.q0 = r.nq = r.k0 = r.nk = r.rows = r.tile = 0;
  if (n <= kWave) {
    int q0 = 0, nq = 0, k0 = 0, nk = 0;
    if (lane < n) {
      bounds(c.q_offsets, c.q_tokens, lane, q0, nq);
      bounds(c.k_offsets, c.k_tokens, lane, k0, nk);
    }
    const int rows = by_key ? nk : nq, tiles = (rows * per + kTile - 1) / kTile;
    if (lane == 0 || lane >= n - 1) nq = nk = 0;
    int before = 0;
    for (int i = 0; i < n; ++i) {
      const int keys = __builtin_amdgcn_readlane(nk, i), count = __builtin_amdgcn_readlane(tiles, i);
      before += keys > nk || (keys == nk && i < lane) ? count : 0;
    }
    const uint64_t here = __ballot(lane < n && index >= before && index < before + tiles);
    if (!here) return r;
    const int l = __builtin_ctzll(here);
    r.valid = true;
    r.tile = index - __builtin_amdgcn_readlane(before, l);
    if (reverse) r.tile = __builtin_amdgcn_readlane(tiles, l) - 1 - r.tile;
    r.q0 = __builtin_amdgcn_readlane(q0, l);
    r.nq = __builtin_amdgcn_readlane(nq, l);
    r.k0 = __builtin_amdgcn_readlane(k0, l);
    r.nk = __builtin_amdgcn_readlane(nk, l);
    r.rows = __builtin_amdgcn_readlane(rows, l);
    return r;
  }
  int total = 0;
  if (reverse) {
    for (int s = 0; s < n; s += kWave) total += __shfl(wave_scan(tiles_of(s + lane)), kWave - 1);
    index = total - 1 - index;
  }
  if (index < 0) return r;
  int before = 0;
  for (int s = 0; s < n; s += kWave) {
    const int tiles = tiles_of(s + lane), sum = before + wave_scan(tiles);
    const uint64_t here = __ballot(sum > index);
    if (here) {
      const int l = __builtin_ctzll(here), seq = s + l;
      r.valid = true;
      r.tile = uniform(index - __shfl(sum - tiles, l));
      bounds(c.q_offsets, c.q_tokens, seq, r.q0, r.nq);
      bounds(c.k_offsets, c.k_tokens, seq, r.k0, r.nk);
      r.rows = by_key ? r.nk : r.nq;
      if (seq == 0 || seq == n - 1) r.nq = r.nk = 0;
      r.q0 = uniform(r.q0);
      r.nq = uniform(r.nq);
      r.k0 = uniform(r.k0);
      r.nk = uniform(r.nk);
      r.rows = uniform(r.rows);
      return r;
    }
    before = uniform(__shfl(sum, kWave - 1));
  }
  return r;
}

// The (head, tile) of workgroup `id` of heads x tiles.  Workgroups are dealt round-robin to the 8 XCDs, each with an L2 of its
// own: an XCD takes whole heads, neighbours (which share their keys and values in a grouped call), one behind the other, so that all its
// workgroups in flight read the same head's keys; the heads past a multiple of 8 are spread tile by tile.  `uneven`: tiles of different
// lengths, the longest first: then an XCD takes its heads' tiles in turn, or the last head's longest would start last.
__device__ inline void head_and_tile(int id, int heads, int tiles, bool uneven, int& head, int& tile) {
  const int per_xcd = heads / 8, whole = per_xcd * 8 * tiles;
  if (id < whole) {
    const int x = id & 7, j = id >> 3;
    head = x * per_xcd + (uneven ? j % per_xcd : j / tiles);
    tile = uneven ? j / per_xcd : j % tiles;
  } else {
    const int rest = heads - per_xcd * 8, j = id - whole;
    head = per_xcd * 8 + j % rest;
    tile = j / rest;
  }
}

// ---- tiles in LDS -----------------------------------------------------------------------------------------
// A tile is rows of kPitch elements (a power of two, the head's 16-byte pieces padded up to it), the pieces of a row permuted by
// an exclusive or with the row's bits: pieces of the same number of 16 rows lie in different banks (a matrix operand's rows), and so
// do 64 bytes of each of four consecutive rows (what 32 lanes of the transposing read take).
template <int kPitch>
__device__ inline int swizzle(int row) {
  if constexpr (kPitch == 64) return (row >> 1 & 1) << 2 | (row >> 2 & 1) << 1 | (row >> 3 & 1);  // (two rows to a turn of the banks)
  return (row & 3) << 2 | (row >> 2 & 1) << 1 | (row >> 3 & 1);
}

// Loads a tile of kRows rows straight into LDS with kThreads threads, 16 bytes a lane and instruction; rows past `rows` repeat the
// last one and pieces past the head's end its last piece, so that nothing outside the tensor is read (their scores are masked,
// and the other operand is zero there).  kSkip: pieces past the head's end are left alone, for a tile in which they have been cleared: an
// infinity that the head ends with would come to a NaN in the product with zero.  Every instruction loads whole rows, so none is
// without lanes, and a count of requests in flight holds.
template <int kPitch, int kRows, int kThreads, bool kSkip = false>
struct TileLoader {
  static constexpr int kPieces = kPitch / 8;  // of a row
  static constexpr int kLoads = kRows * kPieces / kThreads;
  static constexpr uint32_t kNone = ~0u;  // no offset: 127 rows of less than 2^25 bytes and a head lie below
  static_assert(kRows * kPieces % kThreads == 0 && kWave % kPieces == 0, "whole instructions of whole rows");
  uint32_t row_bytes;
  uint32_t offset[kLoads];

  __device__ inline void init(int thread, int64_t token_stride, int dim) {
    row_bytes = (uint32_t)token_stride * 2u;
    const int wave = thread / kWave, lane = thread & (kWave - 1);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = (wave * kLoads + i) * kWave + lane, row = piece / kPieces, slot = piece % kPieces;
      const int place = slot ^ swizzle<kPitch>(row);
      offset[i] = (uint32_t)row * row_bytes + 16u * (uint32_t)min(place, dim / 8 - 1);
      if (kSkip && place >= dim / 8) offset[i] = kNone;
    }
  }
  // `base`: the tile's first row in memory; `lds`: the tile's address in LDS; `rows`: those that are there, at least one
  __device__ inline void load(const uint16_t* base, uint32_t lds, int rows, int thread) const {
    const int wave = uniform(thread / kWave), lane = thread & (kWave - 1);
    const uint32_t to = lds + (uint32_t)(wave * kLoads * kWave * 16);
    base = uniform(base);  // (the compiler loses track of what is one value for the wavefront)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t o = offset[i];
      if (rows < kRows) {
        const int row = ((wave * kLoads + i) * kWave + lane) / kPieces;
        if (row >= rows) o -= (uint32_t)(row - rows + 1) * row_bytes;
      }
      if (kSkip && offset[i] == kNone) continue;
      // one wait state behind the write of m0, which the compiler does not see to inside a statement of assembly
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(o), "s"(base), "s"(uniform((int)(to + (uint32_t)i * kWave * 16u)))
                   : "memory", "m0");
    }
  }
};

// The pieces past the head's end of `rows` rows of a tile, up to the size it is padded to, become zero; by `threads` threads
template <int kPitch, int kDim>
__device__ inline void clear_padding(char* tile, int rows, int dim, int thread, int threads) {
  const int from = dim / 8, pieces = kDim / 8 - from;
  for (int n = thread; n < rows * pieces; n += threads) {
    const int r = n / pieces, piece = from + n % pieces;
    *reinterpret_cast<u32x4a*>(tile + r * kPitch * 2 + 16 * (piece ^ swizzle<kPitch>(r))) = u32x4a{0u, 0u, 0u, 0u};
  }
}

// Whether any of the workgroup's kWaves wavefronts says so; `at`: LDS that nobody reads any more.  Nothing is in flight afterwards.
template <int kWaves>
__device__ inline bool any_wave(bool mine, char* at) {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  int* flags = reinterpret_cast<int*>(at);
  if ((threadIdx.x & (kWave - 1)) == 0) flags[threadIdx.x / kWave] = mine;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) any |= flags[w];
  __syncthreads();
  return uniform(any);
}

// this wavefront's requests have arrived, and everyone's reads so far are done
__device__ inline void arrive_and_sync() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// rows 0 .. 31 of a tile as a left operand: lane (row l % 32, half l / 32) holds elements 16 step + 8 half ..
template <typename T, int kPitch>
__device__ inline typename T::vec8 tile_rows(const char* tile, int step, int lane) {
  const int row = lane & 31, piece = 2 * step + (lane >> 5);
  return *reinterpret_cast<const typename T::vec8*>(tile + row * (kPitch * 2) + 16 * (piece ^ swizzle<kPitch>(row)));
}

// columns 32 block .. +31 of 16 rows of a tile as a left operand (the tile transposed): lane (column l % 32, half h) holds rows
// {4h .. 4h+3} and {8+4h .. 8+4h+3}, the order in which a score tile's result holds them
template <typename T, int kPitch>
__device__ inline typename T::vec8 tile_columns(const char* tile, int block, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int i = lane & 15, row = 4 * (lane >> 5) + (i >> 2), piece = 4 * block + 2 * (lane >> 4 & 1) + (i >> 1 & 1);
  const char* a = tile + row * (kPitch * 2) + 16 * (piece ^ swizzle<kPitch>(row)) + 8 * (i & 1);
  const char* b = tile + (row + 8) * (kPitch * 2) + 16 * (piece ^ swizzle<kPitch>(row + 8)) + 8 * (i & 1);
  const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a);
  const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)b);
  return __builtin_bit_cast(typename T::vec8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The same by addresses in LDS that a lane computes once: operand e of tile_rows lies at rows[e], the two halves of block b of
// tile_columns at columns[0][b] and [1][b], from the tile's first row on, so that a tile, a block of rows and a half of it are constants
// in the instruction.  (Left to itself the compiler makes them again for every read, 90 vector instructions a step of 64 keys.)
typedef __attribute__((address_space(3))) const char* LdsAddress;
template <int kPitch, int kSteps, int kBlocks>
struct OperandAddresses {
  uint32_t rows[kSteps], columns[2][kBlocks];

  __device__ inline void init(const char* lds, int lane) {
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    const int row = lane & 31, i = lane & 15, first = 4 * (lane >> 5) + (i >> 2), piece = 2 * (lane >> 4 & 1) + (i >> 1 & 1);
    const uint32_t r = row * (kPitch * 2) + 16 * ((lane >> 5) ^ swizzle<kPitch>(row));
    const uint32_t c = first * (kPitch * 2) + 16 * (piece ^ swizzle<kPitch>(first)) + 8 * (i & 1);
#pragma unroll
    for (int e = 0; e < kSteps; ++e) {
      rows[e] = base + (r ^ (32 * e));
      asm volatile("" : "+v"(rows[e]));
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      columns[0][b] = base + (c ^ (64 * b));
      columns[1][b] = base + (c ^ (64 * b) ^ 16) + 8 * kPitch * 2;  // eight rows on: the swizzle's low bit turns
      asm volatile("" : "+v"(columns[0][b]), "+v"(columns[1][b]));
    }
  }
  template <typename T>
  __device__ inline typename T::vec8 row_operand(int e, int offset) const {
    typedef __attribute__((address_space(3))) const typename T::vec8 operand;
    return *(operand*)(LdsAddress)(uintptr_t)(rows[e] + offset);
  }
  template <typename T>
  __device__ inline typename T::vec8 column_operand(int b, int offset) const {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(columns[0][b] + offset));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(columns[1][b] + offset));
    return __builtin_bit_cast(typename T::vec8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

__device__ inline f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// the row of a 32-row result that register i of a lane holds
__device__ inline int result_row(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

// registers 8 slab .. +7 of a result as a right operand's 16 rows, rounded to the 16-bit type
template <typename T>
__device__ inline typename T::vec8 result_operand(const f32x16& s, int slab) {
  u32x4a w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = T::pack2(s[8 * slab + 2 * i], s[8 * slab + 2 * i + 1]);
  return __builtin_bit_cast(typename T::vec8, w);
}

// The values of the lane's column in the wavefront's two halves (lanes l and l ^ 32)
struct Halves {
  float low, high;
};
__device__ inline Halves halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return {__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
__device__ inline float sum_halves(float v) {
  const Halves h = halves(v);
  return h.low + h.high;
}
__device__ inline float max_halves(float v) {
  const Halves h = halves(v);
  return fmaxf(h.low, h.high);
}

// sum + the operand's eight values: what the second product weighs with is what the sum divides by, rounded alike
template <typename T>
__device__ inline float add_sum(typename T::vec8 p, float sum) {
  const u32x4a w = __builtin_bit_cast(u32x4a, p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T::code == MFQ_BF16) {
      typedef __bf16 pair __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, (uint32_t)w[i]), __builtin_bit_cast(pair, 0x3f803f80u), sum, false);
    } else {
      typedef __fp16 pair __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, (uint32_t)w[i]), __builtin_bit_cast(pair, 0x3c003c00u), sum, false);
    }
  }
  return sum;
}

// Whether a tile of kTiles x 32 rows holds an infinity or a NaN: in a product with zeros every finite element gives zero.  Asked of
// tiles at a mask's edge alone: a masked row's probability is zero, but zero times such an element is NaN, which the product would
// hand to columns that never see the row.  A workgroup (in the split form a wavefront) that met such a tile begins again and adds every
// row by itself: code of its own, so that it costs the other calls no register.
template <typename T, int kPitch, int kSteps, int kTiles>
__device__ inline bool tile_not_finite(const char* tile, int lane) {
  using vec8 = typename T::vec8;
  const vec8 none = __builtin_bit_cast(vec8, u32x4a{0u, 0u, 0u, 0u});
  f32x16 probe = zero16();
#pragma unroll 1
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int e = 0; e < kSteps; ++e) probe = mfma32(tile_rows<T, kPitch>(tile + t * 32 * kPitch * 2, e, lane), none, probe);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += probe[i];
  return __any(sum != 0.f);
}

// The product of a 32 x 32 tile of results with zeros: 0, or NaN if any of them is not finite
__device__ inline float times_zero(const f32x16& s, float sum) {
#pragma unroll
  for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(s[i], 0.f, sum);
  return sum;
}

// acc += tile^T p for 16 rows of a tile, row by row, each added only where it is visible.  visible(row): of the lane's column.
template <typename T, int kPitch, int kBlocks, typename Visible>
__device__ inline void add_columns_one_by_one(f32x16 (&acc)[kBlocks], const char* tile16, typename T::vec8 p, int lane, Visible visible) {
  using vec8 = typename T::vec8;
  typedef short s16x8 __attribute__((ext_vector_type(8)));
#pragma unroll 1
  for (int row = 0; row < 16; ++row) {
    s16x8 keep;
#pragma unroll
    for (int s = 0; s < 8; ++s) keep[s] = row == 8 * (s >> 2) + 4 * (lane >> 5) + (s & 3) ? (short)-1 : (short)0;
    const vec8 one = __builtin_bit_cast(vec8, (s16x8)(__builtin_bit_cast(s16x8, p) & keep));
    const bool see = visible(row);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const s16x8 v = __builtin_bit_cast(s16x8, tile_columns<T, kPitch>(tile16, b, lane)) & keep;
      const f32x16 part = mfma32(__builtin_bit_cast(vec8, v), one, zero16());
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[b][i] += see ? part[i] : 0.f;
    }
  }
}

// The exponentials' reference follows a row's maximum only where that has grown by more than a factor of 2^kLag: up to there float32
// sums and 16-bit probabilities hold them as well as values up to 1, and the accumulators need no pass.  bfloat16 has the range for any
// lag.  float16 ends at 2^16 and loses bits below 2^-14 and everything below 2^-25, so its probabilities are multiples of 2^-kLift, and so is
// the sum that they are divided by: at most 2^-35 of the largest is lost.  (Without it 8192 keys of weight e^-18 each beside a strong one
// vanished together.)  A lag of 4 takes the time that one of 8 takes on scores of a standard deviation of 1 (4608 tokens x 24 heads of 128: 286
// us), and 294 instead of 288 us at 3; a lag of 1 and three more powers cost 10 and 18 us.
template <typename T>
constexpr float kLag = T::code == MFQ_F16 ? 4.f : 8.f;
template <typename T>
constexpr float kLift = T::code == MFQ_F16 ? 10.f : 0.f;

// ---- a lane's query as the softmax goes over its keys -----------------------------------------------------------
// kDim: the head's size padded to a multiple of 32.  O^T accumulates in kDim / 32 results.
template <typename T, int kDim, int kPitch>
struct QueryState {
  static constexpr int kBlocks = kDim / 32, kSteps = kDim / 16;
  using vec8 = typename T::vec8;
  vec8 q[kSteps];  // the query as a right operand: elements 16 step + 8 half ..
  f32x16 o[kBlocks];
  float top;   // the reference the exponentials are taken against, unscaled
  float sum;   // of this half's exponentials

  __device__ inline void init() {
    top = -__builtin_inff();
    sum = 0.f;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) o[b] = zero16();
  }
  // p: the query's row; pieces past the head's end are zero
  __device__ inline static void load_row(vec8 (&to)[kSteps], const uint16_t* p, int dim, int lane) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      u32x4a w = {0u, 0u, 0u, 0u};
      if (d < dim) w = *reinterpret_cast<const u32x4a*>(p + d);
      to[s] = __builtin_bit_cast(vec8, w);
    }
  }

  // One step over kTiles x 32 keys, tiles of K and V in LDS.  `limit`: keys of the tile that the lane's query sees (may be
  // negative or beyond the tile); kMasked: whether any lane's ends inside it (code of its own: a branch around these parts has the
  // compiler copy every accumulator twice a step).  c: scale * log2(e).  between(): run when K's tile has been read, before V's is.
  // A masked step answers whether V's tile holds an infinity or a NaN: then its result is not to be used, and kOneByOne gives it.
  struct Nothing {
    __device__ inline void operator()() const {}
  };
  template <int kTiles, bool kMasked, bool kOneByOne = false, typename Between = Nothing>
  __device__ __attribute__((always_inline)) inline bool step(const char* k_tile, const char* v_tile, int limit, float c, int lane,
                                                             Between between = Between()) {
    f32x16 s[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) s[t] = zero16();
    // operands are read two steps ahead of the matrix instructions that take them
    vec8 a[3][kTiles];
    auto rows = [&](int e) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) a[e % 3][t] = tile_rows<T, kPitch>(k_tile + t * 32 * kPitch * 2, e, lane);
    };
    rows(0);
    rows(1);
#pragma unroll
    for (int e = 0; e < kSteps; ++e) {
      if (e + 2 < kSteps) rows(e + 2);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) s[t] = mfma32(a[e % 3][t], q[e], s[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
    between();
    vec8 w[2][kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) w[0][b] = tile_columns<T, kPitch>(v_tile, b, lane);
    bool not_finite = false;
    if constexpr (kMasked) {
      if constexpr (!kOneByOne) not_finite = tile_not_finite<T, kPitch, kSteps, kTiles>(v_tile, lane);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = 32 * t + result_row(i, lane) < limit ? s[t][i] : -__builtin_inff();
    }
    float most = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, s[t][i]);
    most = max_halves(most);
    if (__any((most - top) * c > kLag<T>)) {
      const float next = fmaxf(top, most);
      const float factor = next == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((top - next) * c);
      top = next;
      sum *= factor;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= factor;
    }
    const float shift = reference(c);
#pragma unroll
    for (int n = 0; n < 2 * kTiles; ++n) {
      const vec8 p = probabilities(s[n / 2], n & 1, c, shift);
      if constexpr (kOneByOne) {
        add_columns_one_by_one<T, kPitch, kBlocks>(o, v_tile + n * 16 * kPitch * 2, p, lane, [&](int row) { return 16 * n + row < limit; });
      } else {
        if (n + 1 < 2 * kTiles) {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) w[(n + 1) & 1][b] = tile_columns<T, kPitch>(v_tile + (n + 1) * 16 * kPitch * 2, b, lane);
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) o[b] = mfma32(w[n & 1][b], p, o[b]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    return not_finite;
  }
  // what the scaled scores are taken against
  __device__ __attribute__((always_inline)) inline float reference(float c) const { return top == -__builtin_inff() ? 0.f : top * c - kLift<T>; }
  // the row's log2 of the sum of exp2 of the scaled scores; `total`: of both halves and all parts
  __device__ static inline float log_sum(float top, float total, float c) { return top * c + (__builtin_amdgcn_logf(total) - kLift<T>); }
  // exponentials of half a score tile as the second product's operand, added to the sum
  __device__ __attribute__((always_inline)) inline vec8 probabilities(f32x16& s, int slab, float c, float shift) {
#pragma unroll
    for (int i = 8 * slab; i < 8 * slab + 8; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -shift));
    const vec8 p = result_operand<T>(s, slab);
    sum = add_sum<T>(p, sum);
    return p;
  }
  // ---- the same over 32 keys in two halves that overlap: while the matrix pipeline makes the next block's scores, the vector pipeline
  // takes this one's exponentials, and while it multiplies with V, the maximum over the next block's.
  using Addresses = OperandAddresses<kPitch, kSteps, kBlocks>;
  // scores of a block alone (the first one), k32: its place in LDS
  __device__ __attribute__((always_inline)) inline void scores(f32x16& s, const Addresses& at, int k32) {
    s = zero16();
#pragma unroll
    for (int e = 0; e < kSteps; ++e) s = mfma32(at.template row_operand<T>(e, k32), q[e], s);
  }
  // the reference follows the block's maximum (see step)
  __device__ __attribute__((always_inline)) inline void follow(float most, float c) {
    most = max_halves(most);
    if (__any((most - top) * c > kLag<T>)) {
      const float next = fmaxf(top, most);
      const float factor = next == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((top - next) * c);
      top = next;
      sum *= factor;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= factor;
    }
  }
  __device__ __attribute__((always_inline)) static inline float maximum(const f32x16& s) {
    float most = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
    return most;
  }
  // s: the block's scores; kNext: next = the scores of the block at k32
  template <bool kNext>
  __device__ __attribute__((always_inline)) inline void overlapped(f32x16& s, f32x16& next, const Addresses& at, int k32, int v32, float c) {
    const float shift = reference(c);
    vec8 p[2], w[2][kBlocks], a[3];
    if constexpr (kNext) {
      next = zero16();
      a[0] = at.template row_operand<T>(0, k32);
      a[1] = at.template row_operand<T>(1, k32);
    }
#pragma unroll
    for (int e = 0; e < kSteps; ++e) {
      if constexpr (kNext) {
        if (e + 2 < kSteps) a[(e + 2) % 3] = at.template row_operand<T>(e + 2, k32);
        next = mfma32(a[e % 3], q[e], next);
      }
      // V's first operands, when the reads of K end
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        if (b * 2 / kBlocks + kSteps - 2 == e) w[0][b] = at.template column_operand<T>(b, v32);
#pragma unroll
      for (int i = 16 * e / kSteps; i < 16 * (e + 1) / kSteps; ++i) {
        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -shift));
        if ((i & 7) == 7) {
          p[i >> 3] = result_operand<T>(s, i >> 3);
          sum = add_sum<T>(p[i >> 3], sum);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    float most[4] = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        if (n == 0) w[1][b] = at.template column_operand<T>(b, v32 + 16 * kPitch * 2);
        o[b] = mfma32(w[n][b], p[n], o[b]);
        if constexpr (kNext) {
          const int g = n * kBlocks + b;
#pragma unroll
          for (int i = 16 * g / (2 * kBlocks); i < 16 * (g + 1) / (2 * kBlocks); ++i) most[i & 3] = fmaxf(most[i & 3], next[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (kNext) follow(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), c);
  }
};

// the last key (+ 1) that query i of a sequence sees
__device__ inline int visible_keys(const Run& r, int i, int causal) {
  if (i >= r.nq) return 0;
  return causal ? min(max(i + 1 + r.nk - r.nq, 0), r.nk) : r.nk;
}

__device__ inline int wave_min(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v = min(v, __shfl_xor(v, d));
  return uniform(v);
}
__device__ inline int wave_max(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v = max(v, __shfl_xor(v, d));
  return uniform(v);
}

// four values as 16-bit elements, and what their rounding left of them
template <typename T>
__device__ inline u32x2 pack4(f32x4 v) { return u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])}; }
template <typename T>
__device__ inline u32x2 pack4_rest(f32x4 v, u32x2 p) {
  return u32x2{T::pack2(v[0] - lo_f32<T>(p[0]), v[1] - hi_f32<T>(p[0])), T::pack2(v[2] - lo_f32<T>(p[1]), v[3] - hi_f32<T>(p[1]))};
}

// A column of results (kDim / 32 of them) as a row of the output, zeros where it is not `seen`; `rest`: of the rounding, or nullptr.
// Four consecutive elements a store.
template <typename T, int kBlocks>
__device__ inline void store_row(uint16_t* row, uint16_t* rest, const f32x16 (&o)[kBlocks], bool seen, float factor, int dim, int lane) {
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * b + result_row(i, lane);
      if (d >= dim) continue;
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = seen ? o[b][i + j] * factor : 0.f;
      const u32x2 p = pack4<T>(v);
      *reinterpret_cast<u32x2*>(row + d) = p;
      if (rest) *reinterpret_cast<u32x2*>(rest + d) = pack4_rest<T>(v, p);
    }
}

// whether a launch may have so many workgroups: fewer than 2^32 threads in all
inline bool launches(int64_t groups, int threads) { return groups <= UINT32_MAX / threads; }

int launch_attention(int dtype, const AttentionCall& c, hipStream_t stream);
// few queries against many keys: into how many ranges the key axis is cut, 0 where launch_attention is the faster
int attention_splits(const AttentionCall& c);
size_t attention_split_bytes(const AttentionCall& c, int splits);  // of workspace, 16-byte aligned
int launch_attention_split(int dtype, const AttentionCall& c, int splits, void* workspace, hipStream_t stream);
// into how many parts the query heads that share a key head are cut, each with float32 sums of its own
int attention_backward_parts(const AttentionCall& c);
size_t attention_backward_bytes(const AttentionCall& c, int parts);  // of workspace, 16-byte aligned
int launch_attention_backward(int dtype, const AttentionCall& c, int parts, void* workspace, hipStream_t stream);

}  // namespace mfq
