// The product of two matrices of 8-bit integers with a scale for each row of either:
//   y[m][n] = x_scales[m] w_scales[n] sum_k x[m][k] w[n][k] (+ bias[n])
// The sum is exact (32-bit integers: |x w| <= 2^14 and K < 2^17), so its order is free: K may be cut between wavefronts and
// workgroups, and the lanes' k within a matrix instruction may be any as long as both operands agree.  What follows is float32,
// rounded once to y's type.
#include <type_traits>

#include "rows.h"

namespace mfq {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int BK = 128;  // k of a step: a cache line of a row
constexpr int kMaxLds = 160 * 1024;

struct I32 {  // a range's sums as they are, for the kernel that joins them
  using storage = int32_t;
};

__device__ inline float value_of(int sum, float xs, float ws, float add) { return (float)sum * xs * ws + add; }

// ---- tiles -------------------------------------------------------------------------------------------------------------
// A workgroup of four wavefronts computes kM x kN outputs, a wavefront kWM x kWN of them on v_mfma_i32_16x16x64_i8 with w as
// the first operand (a lane's registers are four neighbouring columns of y, of one row).
//   - x and w go from memory straight into LDS, a step's 128 bytes of a row at a time, into a ring of units (a step of x, then
//     a step of w, in turn), the 16-byte column of a row XORed with swz_mask(row);
//   - the fragments of half a step (64 k) are read while the half before them is multiplied, across the end of a step too: the
//     one barrier of a step lies in front of its second half, where the fragments of that half are in registers (the step's two
//     units are free) and the next step's units have arrived;
//   - workgroups stay and walk tiles; the ring runs on over a tile's end, and results go from the registers to memory.
// Large products are bound by power: matrix instructions alone, on operands that stay in registers (codes of a normal
// distribution), reach 4.0 PFLOP/s where the second operand stays from one instruction to the next, 3.4 where the first one
// does, 3.0 where both change (32x32x32: 3.4; zeros, bound by issue: 4.2, 32x32x32 4.9).  8192^3 takes 395 us (2.78 PFLOP/s),
// 16384 x 4096 x 12288 580, 4352 x 20480 x 3840 298 (2.30; 19200 columns of it in five whole rounds, the others on 128 x 192).
// Below some 2000 rows it is the way into LDS, about 50 bytes a ns and compute unit whatever the tile: 512 x 3840 x 3840 16.7 us,
// 333 x 11520 x 3840 25 (a quarter of the matrix units' time), 24 x 3840 x 10240 9 and 3 for its join.
template <int kM_, int kN_, int kWM_, int kWN_, int kUnits_>
struct Tile {
  static constexpr int kM = kM_, kN = kN_, kWM = kWM_, kWN = kWN_, kUnits = kUnits_;
  static constexpr int kAcross = kM / kWM, kWaves = kAcross * (kN / kWN), kThreads = kWaves * kWave;
  static constexpr int kI = kWM / 16, kJ = kWN / 16;
  static constexpr int kXLoads = kM / 8 / kWaves, kWLoads = kN / 8 / kWaves;  // of a wavefront for a unit, a KiB each
  static constexpr int kUnitBytes = (kM > kN ? kM : kN) * BK;
  static constexpr int kLds = kUnits * kUnitBytes;
  static constexpr int loads(int unit) { return unit % 2 ? kWLoads : kXLoads; }
  // loads of the units from `from` to the last one requested, before the next request (of units kUnits, kUnits + 1)
  static constexpr int behind(int from) {
    int n = 0;
    for (int u = from; u < kUnits; ++u) n += loads(u);
    return n;
  }
  static_assert(kM % (8 * kWaves) == 0 && kN % (8 * kWaves) == 0 && kLds <= kMaxLds && kUnits >= 4 && behind(2) < 64, "");
};

// The 16-byte column of a 128-byte row of LDS is XORed with this, so that the rows of a fragment that are read together (columns
// 2 (lane / 16) + half) spread over the banks: see qmm_frag.hip
__device__ inline int swz_mask(int row) {
  const int i = (row >> 1) & 7;
  return (i & 4) | ((i & 1) << 1) | ((i >> 2) ^ ((i >> 1) & 1));
}

// An item's part of the product: a tile and a range of K
struct Item {
  int64_t m0, n0;
  int split, first, steps;
};

template <typename S>
__device__ inline Item item_of(int item, int tiles_m, int tiles_n, int splits, int all_steps) {
  const int n_tiles = tiles_m * tiles_n, split = item / n_tiles;
  int tile = item - split * n_tiles;
  // an XCD (every eighth workgroup) walks a contiguous run of the tiles, in bands of four tile rows
  const int per_xcd = n_tiles / 8;
  if (tile < per_xcd * 8) tile = (tile & 7) * per_xcd + (tile >> 3);
  constexpr int kBand = 4;
  const int band = tile / (kBand * tiles_n), band_rows = min(tiles_m - band * kBand, kBand), in_band = tile - band * kBand * tiles_n;
  Item it;
  it.m0 = (int64_t)__builtin_amdgcn_readfirstlane(band * kBand + in_band % band_rows) * S::kM;
  it.n0 = (int64_t)__builtin_amdgcn_readfirstlane(in_band / band_rows) * S::kN;
  it.split = __builtin_amdgcn_readfirstlane(split);
  it.first = __builtin_amdgcn_readfirstlane(all_steps * split / splits);  // of at most 1024 steps and 64 ranges
  it.steps = __builtin_amdgcn_readfirstlane(all_steps * (split + 1) / splits) - it.first;
  return it;
}

template <typename S, typename T>
__global__ __launch_bounds__(S::kThreads) void int8_tile_kernel(Int8Call c, int tiles_m, int tiles_n, int splits, void* out) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kI = S::kI, kJ = S::kJ;
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int r = lane & 15, q4 = lane >> 4;
  const int items = tiles_m * tiles_n * splits, all_steps = ((int)c.K + BK - 1) / BK;
  auto item_at = [&](int item) __attribute__((always_inline)) { return item_of<S>(item, tiles_m, tiles_n, splits, all_steps); };

  // ---- requests: eight rows x 128 bytes an instruction, a unit's rows dealt to the wavefronts in turn.  x and w have a
  // place of their own in the sequence of (item, step).  Behind the last item they stay where they are.
  const int own_row = wave * 8 + (lane >> 3);
  const uint32_t column = 16 * ((lane & 7) ^ swz_mask(own_row));  // of a row, that goes to the lane's place
  const uint32_t tail = (uint32_t)((c.K - 1) & (BK - 1)) + 1;        // bytes of a row in the last step of all
  const uint32_t last_column = min(column, tail - 16);                // the bytes past the end of K repeat others; x's are cleared below
  const uint32_t lds_addr = (uint32_t)(uintptr_t)lds + (uint32_t)(wave * 8 * BK);
  struct Place {
    int item, at, left;  // step of K, steps left of the item
    const int8_t* p;
  };
  Place px, pw;
  uint32_t x_row[S::kXLoads], w_row[S::kWLoads];
  auto begin = [&](auto is_x, Place& to, uint32_t* rows, int item) __attribute__((always_inline)) {
    const Item it = item_at(item);
    const int64_t from = is_x ? it.m0 : it.n0, stride = is_x ? c.x_stride : c.w_stride;
    const int last = (int)min((is_x ? c.M : c.N) - from, (int64_t)(is_x ? S::kM : S::kN)) - 1;
#pragma unroll
    for (int l = 0; l < (is_x ? S::kXLoads : S::kWLoads); ++l) rows[l] = (uint32_t)min(own_row + 8 * S::kWaves * l, last) * (uint32_t)stride;
    to.item = item;
    to.at = it.first;
    to.left = it.steps;
    to.p = (is_x ? c.x : c.w) + from * stride + (int64_t)it.first * BK;
  };
  auto advance = [&](auto is_x, Place& to, uint32_t* rows) __attribute__((always_inline)) {
    if (--to.left) {
      to.p += BK;
      ++to.at;
    } else if (to.item + (int)gridDim.x < items) {
      begin(is_x, to, rows, to.item + (int)gridDim.x);
    } else {
      to.left = 1;
    }
  };
  constexpr std::true_type kX{};
  constexpr std::false_type kW{};
  auto request = [&](auto is_x, int l, int slot) __attribute__((always_inline)) {
    const Place& from = is_x ? px : pw;
    const uint32_t off = (is_x ? x_row : w_row)[l] + (from.at == all_steps - 1 ? last_column : column);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr + (uint32_t)(slot * S::kUnitBytes));
    asm volatile("s_add_i32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 ::"v"(off), "s"(from.p), "s"(to), "i"(l * S::kWaves * 1024) : "memory", "m0", "scc");
  };
  // the slots of the ring, a step's x and w: (slot, slot + 1)
  auto next_slot = [](int slot, int by) __attribute__((always_inline)) { return slot + by >= S::kUnits ? slot + by - S::kUnits : slot + by; };
  // x past the end of K, once it has arrived
  auto clear_tail = [&](int slot) __attribute__((always_inline)) {
    if (column >= tail) {
#pragma unroll
      for (int l = 0; l < S::kXLoads; ++l)
        *reinterpret_cast<u32x4*>(lds + slot * S::kUnitBytes + (wave + l * S::kWaves) * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  // ---- fragments.  Lane (r, q4) has 16 bytes of row r, those of column 2 q4 + half of a step.
  const int wm = wave % S::kAcross * S::kWM, wn = wave / S::kAcross * S::kWN;
  i32x4 xf[2][kI], wf[2][kJ];
  const int x_at = (wm + r) * BK, w_at = (wn + r) * BK, swz = swz_mask(r);
  // fragment f of a half, in the order of their use: the first of x, those of w, the others of x
  auto read = [&](int set, int slot, int half, int f) __attribute__((always_inline)) {
    const int at = ((2 * q4 + half) ^ swz) << 4;
    if (f >= 1 && f <= kJ) wf[set][f - 1] = *reinterpret_cast<const i32x4*>(lds + next_slot(slot, 1) * S::kUnitBytes + at + w_at + (f - 1) * 16 * BK);
    else xf[set][f ? f - kJ : 0] = *reinterpret_cast<const i32x4*>(lds + slot * S::kUnitBytes + at + x_at + (f ? f - kJ : 0) * 16 * BK);
  };
  i32x4 acc[kI][kJ];
  // Multiplies half a step's fragments (`fresh`: the first of an item); in between, reads those of (slot, next) into the other set
  // and requests a unit.  Reads and requests are dealt out over the first three quarters of the instructions.
  constexpr int kOneX = 1, kOneW = 2;
  auto half_step = [&](auto fresh_c, auto set_c, auto unit_c, int slot, int next, int to) __attribute__((always_inline)) {
    constexpr int set = decltype(set_c)::value, unit = decltype(unit_c)::value;
    constexpr int kInstr = kI * kJ, kSpan = kInstr >= 16 ? kInstr * 3 / 4 : kInstr, kReads = kI + kJ;
    constexpr int kRequests = unit == kOneX ? S::kXLoads : S::kWLoads;
#pragma unroll
    for (int n = 0; n < kInstr; ++n) {
      const int i = n / kJ, j = n % kJ;
      acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[set][j], xf[set][i], decltype(fresh_c)::value ? i32x4{0, 0, 0, 0} : acc[i][j], 0, 0, 0);
      if (n < kSpan) {
#pragma unroll
        for (int f = kReads * n / kSpan; f < kReads * (n + 1) / kSpan; ++f) read(set ^ 1, slot, next, f);
#pragma unroll
        for (int l = kRequests * n / kSpan; l < kRequests * (n + 1) / kSpan; ++l) {
          if constexpr (unit == kOneX) request(kX, l, to);
          else request(kW, l, to);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (unit == kOneX) advance(kX, px, x_row);
    else advance(kW, pw, w_row);
  };
#define MFQ_C(v) std::integral_constant<int, v>{}

  // ---- results.  Element e of acc[i][j] is row wm + 16 i + r, column wn + 16 j + 4 q4 + e.  16-bit types: two neighbouring
  // blocks of 16 columns exchange quads, so that a lane has eight columns of one of them.
  using E = typename T::storage;
  constexpr bool kRaw = std::is_same_v<T, I32>;
  auto store = [&](const Item& it) __attribute__((always_inline)) {
    constexpr int kEach = 16 / (int)sizeof(E);
    const int64_t stride = kRaw ? c.N : c.y_stride;
    const bool whole = c.N % kEach == 0 && stride % kEach == 0;
    const int64_t n0 = it.n0 + wn, m0 = it.m0 + wm + r;
    char* y = static_cast<char*>(out) + ((kRaw ? (int64_t)it.split * c.M : 0) + m0) * stride * (int64_t)sizeof(E);
    float xs[kI];
#pragma unroll
    for (int i = 0; i < kI; ++i) xs[i] = kRaw ? 0.f : c.x_scales[min(m0 + 16 * i, c.M - 1)];
    constexpr int kPair = sizeof(E) == 2 ? 2 : 1;  // blocks of columns at a time
#pragma unroll
    for (int j = 0; j < kJ; j += kPair) {
      if (n0 + 16 * j >= c.N) continue;
      float ws[kPair][4], add[kPair][4];
      if constexpr (!kRaw) {
#pragma unroll
        for (int p = 0; p < kPair; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t n = min(n0 + 16 * (j + p) + 4 * q4 + e, c.N - 1);
            ws[p][e] = c.w_scales[n];
            add[p][e] = 0.f;
            if (c.bias) add[p][e] = T::to_f32(static_cast<const E*>(c.bias)[n]);
          }
      }
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        E* row = reinterpret_cast<E*>(y + (int64_t)(16 * i) * stride * (int64_t)sizeof(E));
        const bool inside = m0 + 16 * i < c.M;
#pragma unroll
        for (int p = 0; p < kPair; ++p) asm volatile("" : "+a"(acc[i][j + p]));  // (or all of acc is moved to vector registers at the loop's end)
        if constexpr (sizeof(E) == 2) {
          uint32_t a[2], b[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            a[k] = T::pack2(value_of(acc[i][j][2 * k], xs[i], ws[0][2 * k], add[0][2 * k]),
                            value_of(acc[i][j][2 * k + 1], xs[i], ws[0][2 * k + 1], add[0][2 * k + 1]));
            b[k] = T::pack2(value_of(acc[i][j + 1][2 * k], xs[i], ws[1][2 * k], add[1][2 * k]),
                            value_of(acc[i][j + 1][2 * k + 1], xs[i], ws[1][2 * k + 1], add[1][2 * k + 1]));
            // a of odd q4 and b of even q4 change places: lane q4 has the quads q4 & ~1 and q4 | 1 of block j + q4 % 2
            const auto s = __builtin_amdgcn_permlane16_swap(a[k], b[k], false, false);
            a[k] = s[0];
            b[k] = s[1];
          }
          const int64_t n = n0 + 16 * (j + (q4 & 1)) + 8 * (q4 >> 1);
          if (!inside) continue;
          if (whole) {
            if (n < c.N) *reinterpret_cast<u32x4*>(row + n) = u32x4{a[0], a[1], b[0], b[1]};
          } else {
            const uint64_t low = a[0] | (uint64_t)a[1] << 32, high = b[0] | (uint64_t)b[1] << 32;
#pragma unroll 1
            for (int k = 0; k < 8 && n + k < c.N; ++k) row[n + k] = (E)((k < 4 ? low : high) >> (16 * (k & 3)));
          }
        } else {
          E q[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (kRaw) q[k] = acc[i][j][k];
            else q[k] = value_of(acc[i][j][k], xs[i], ws[0][k], add[0][k]);
          }
          const int64_t n = n0 + 16 * j + 4 * q4;
          if (!inside) continue;
          typedef E quad __attribute__((ext_vector_type(4)));
          if (whole) {
            if (n < c.N) *reinterpret_cast<quad*>(row + n) = quad{q[0], q[1], q[2], q[3]};
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n + k < c.N) row[n + k] = q[k];
          }
        }
      }
    }
  };

  // ---- the walk
  int item = blockIdx.x;
  Item it = item_at(item);
  begin(kX, px, x_row, item);
  begin(kW, pw, w_row, item);
#pragma unroll
  for (int u = 0; u < S::kUnits - 1; ++u) {
    if (u % 2 == 0) {
#pragma unroll
      for (int l = 0; l < S::kXLoads; ++l) request(kX, l, u);
      advance(kX, px, x_row);
    } else {
#pragma unroll
      for (int l = 0; l < S::kWLoads; ++l) request(kW, l, u);
      advance(kW, pw, w_row);
    }
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::behind(2) - S::loads(S::kUnits - 1)) : "memory");
  if (tail < BK && it.first == all_steps - 1) clear_tail(0);
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int f = 0; f < kI + kJ; ++f) read(0, 0, 0, f);
  // The units requested in a step: the one that takes the place of its x, in its second half, and the one that takes that of its
  // w, in the next step's first
  constexpr int kFirst = S::kUnits % 2 ? kOneW : kOneX, kSecond = S::kUnits % 2 ? kOneX : kOneW;
  int slot = 0, pending = S::kUnits - 1;
  auto step = [&](auto fresh, int next_at) __attribute__((always_inline)) {  // next_at: step of K of the one after
    half_step(fresh, MFQ_C(0), MFQ_C(kSecond), slot, 1, pending);
    // everything read is in registers, the next step's units have arrived: for all wavefronts, behind the barrier.  (Behind the
    // last step of all the ring goes round as well: what is requested and read there is not used.)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(S::behind(4)) : "memory");
    const int after = next_slot(slot, 2);
    if (tail < BK && next_at == all_steps - 1) clear_tail(after);
    asm volatile("s_barrier" ::: "memory");
    half_step(std::false_type{}, MFQ_C(1), MFQ_C(kFirst), after, 0, slot);
    pending = next_slot(slot, 1);
    slot = after;
  };
  for (;;) {
    const int next_first = item + (int)gridDim.x < items ? item_at(item + (int)gridDim.x).first : 0;
    step(std::true_type{}, it.steps > 1 ? it.first + 1 : next_first);
    for (int q = 1; q < it.steps; ++q) step(std::false_type{}, q + 1 < it.steps ? it.first + q + 1 : next_first);
    store(it);
    item += (int)gridDim.x;
    if (item >= items) break;
    it = item_at(item);
  }
#undef MFQ_C
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // requests on their way into LDS
}

// ---- few rows of x --------------------------------------------------------------------------------------------------------
// Bound by the bytes of w, which go from memory straight into registers, kRing KiB of a wavefront ahead.  On v_mfma_i32_16x16x64_i8
// lane (j, q) = (lane % 16, lane / 16) supplies 16 bytes of row j of either operand.  One load instruction of w takes eight rows x
// 128 bytes, whole cache lines: operand row j is row j / 2, bytes 64 (j % 2) + 16 q.  x enters as eight rows x 128 bytes as
// well, operand row j being row j % 8, bytes 64 (j / 8) + 16 q.  Of the 16 x 16 results those belong together whose halves are the
// same (row 8 h + token, column 2 row + h); the others are dropped.
// A workgroup walks a run of blocks of eight rows of w, its wavefronts have a range of K each; a lane keeps its share of x in
// LDS (nothing is exchanged before the end), and the wavefronts' sums meet there behind the last block.
// Up to 32 rows of x go through a workgroup, and up to four workgroups share a run of w.
// 1 x 10240 x 3840: 8.5 us with w in the last cache, 10 without (3.9 TB/s); 1 x 3840 x 10240 11.9; 1 x 2048 x 1024 3.6.
constexpr int kFewMaxWaves = 16;

// LDS of a workgroup: x, and a block's sums
__host__ __device__ inline int few_image(int tokens8, int steps, int waves) { return tokens8 * 1024 * steps * waves; }
__host__ __device__ inline int few_sums(int tokens8, int waves) { return tokens8 * 512 * waves; }

template <int kX, int kRing, typename T>
__global__ __launch_bounds__(kFewMaxWaves* kWave) void int8_few_kernel(Int8Call c, int waves, int steps, int per_group, int groups) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  using E = typename T::storage;
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int j = lane & 15, q = lane >> 4;
  // the workgroups of a run of w are eight apart, on one XCD: all but the first find w in a cache
  const int eight = (int)blockIdx.x >> 3, run = eight / groups * 8 + ((int)blockIdx.x & 7), token0 = eight % groups * 8 * kX;
  const int64_t all_blocks = (c.N + 7) / 8, first_block = (int64_t)run * per_group;
  const int blocks = (int)max(min(all_blocks - first_block, (int64_t)per_group), (int64_t)0);
  const int all_steps = ((int)c.K + BK - 1) / BK, tail = (int)((c.K - 1) & (BK - 1)) + 1;
  const int first = min(wave * steps, all_steps), mine = min(first + steps, all_steps) - first;  // the wavefront's steps

  // ---- w: position p of the wavefront is step p % mine of block p / mine; positions behind the last repeat it
  const int column = 64 * (j & 1) + 16 * q, last_column = min(column, tail - 16);
  int ahead_block = 0, ahead_step = 0;
  i32x4 w[kRing];
  auto load = [&](int u) __attribute__((always_inline)) {
    const int64_t row0 = (first_block + ahead_block) * 8;
    const int row = (int)min((int64_t)(j >> 1), c.N - 1 - row0), at = first + ahead_step;
    const int8_t* p = c.w + row0 * c.w_stride + (int64_t)at * BK;
    w[u] = *reinterpret_cast<const i32x4*>(p + (row * (uint32_t)c.w_stride + (uint32_t)(at == all_steps - 1 ? last_column : column)));
    if (ahead_step + 1 < mine) {
      ++ahead_step;
    } else if (ahead_block + 1 < blocks) {
      ++ahead_block;
      ahead_step = 0;
    }
  };
  char* x = lds + wave * few_image(kX, steps, 1) + lane * 16;
  int* sums = reinterpret_cast<int*>(lds + few_image(kX, steps, waves)) + wave * (few_sums(kX, 1) / 4);
  const int block_ints = few_sums(kX, waves) / 4;
  if (mine > 0 && blocks > 0) {
    // x is requested before w, some steps at a time
    const int x_column = 64 * (j >> 3) + 16 * q;
    constexpr int kAtOnce = kX > 2 ? 2 : 4;
    i32x4 v[kAtOnce][kX];
    auto load_x = [&](int from) __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s) {
        const int at = first + min(from + s, mine - 1), most = at == all_steps - 1 ? tail - 16 : BK - 16;
#pragma unroll
        for (int a = 0; a < kX; ++a) {
          v[s][a] = *reinterpret_cast<const i32x4*>(c.x + min((int64_t)(token0 + 8 * a + (j & 7)), c.M - 1) * c.x_stride + (int64_t)at * BK + min(x_column, most));
          if (x_column > most) v[s][a] = i32x4{0, 0, 0, 0};
        }
      }
    };
    auto keep_x = [&](int from) __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s)
        if (from + s < mine) {
#pragma unroll
          for (int a = 0; a < kX; ++a) *reinterpret_cast<i32x4*>(x + ((from + s) * kX + a) * 1024) = v[s][a];
        }
    };
    load_x(0);
#pragma unroll
    for (int u = 0; u < kRing; ++u) load(u);
    keep_x(0);
    for (int s = kAtOnce; s < mine; s += kAtOnce) {
      load_x(s);
      keep_x(s);
    }
    i32x4 acc[kX];
#pragma unroll
    for (int a = 0; a < kX; ++a) acc[a] = i32x4{0, 0, 0, 0};
    int step = 0;
    auto multiply = [&](int u) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < kX; ++a)
        acc[a] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4*>(x + (step * kX + a) * 1024), w[u], acc[a], 0, 0, 0);
      if (++step < mine) return;
      // the end of a block.  Register e of a lane: operand row 4 q + e (half q / 2, token 4 (q % 2) + e), column j (row j / 2 of w, half j % 2)
      if ((j & 1) == (q >> 1)) {
#pragma unroll
        for (int a = 0; a < kX; ++a) *reinterpret_cast<i32x4*>(sums + a * 128 + (j & 1) * 64 + (j >> 1) * 8 + 4 * (q & 1)) = acc[a];
      }
#pragma unroll
      for (int a = 0; a < kX; ++a) acc[a] = i32x4{0, 0, 0, 0};
      sums += block_ints;
      step = 0;
    };
    int left = blocks * mine;
    for (; left > kRing; left -= kRing) {
#pragma unroll
      for (int u = 0; u < kRing; ++u) {
        multiply(u);
        load(u);
      }
    }
#pragma unroll
    for (int u = 0; u < kRing; ++u)
      if (u < left) multiply(u);
  } else {
    for (int b = 0; b < blocks; ++b)
      for (int k = lane; k < kX * 128; k += kWave) sums[b * block_ints + k] = 0;
  }
  __syncthreads();
  const int* all = reinterpret_cast<const int*>(lds + few_image(kX, steps, waves));
  for (int o = t; o < blocks * kX * 64; o += waves * kWave) {
    const int row = o & 7, token = token0 + (o >> 3) % (8 * kX), block = o / (64 * kX), in_group = token - token0;
    const int64_t n = (first_block + block) * 8 + row;
    if (token >= c.M || n >= c.N) continue;
    const int* s = all + block * block_ints + (in_group >> 3) * 128 + row * 8 + (in_group & 7);
    int sum = 0;
    for (int k = 0; k < waves; ++k) sum += s[k * kX * 128] + s[k * kX * 128 + 64];
    const float v = value_of(sum, c.x_scales[token], c.w_scales[n], c.bias ? T::to_f32(static_cast<const E*>(c.bias)[n]) : 0.f);
    static_cast<E*>(c.y)[token * c.y_stride + n] = T::from_f32(v);
  }
}

// ---- the ranges of a cut K joined: four outputs to a thread where rows are whole fours.  Bound by the launch and its first bytes
// (24 x 3840 of eight ranges 3 us, 3 MB).
template <typename T, bool kWide>
__global__ __launch_bounds__(256) void int8_join_kernel(Int8Call c, const int* planes, int splits) {
  using E = typename T::storage;
  constexpr int kEach = kWide ? 4 : 1;
  const int64_t outputs = c.M * c.N, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * kEach;
  if (i >= outputs) return;
  int sum[kEach] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    if constexpr (kWide) {
      const i32x4 v = *reinterpret_cast<const i32x4*>(planes + s * outputs + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    } else {
      sum[0] += planes[s * outputs + i];
    }
  }
  const int64_t m = i / c.N, n = i - m * c.N;
  float v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    v[e] = value_of(sum[e], c.x_scales[m], c.w_scales[n + e], c.bias ? T::to_f32(static_cast<const E*>(c.bias)[n + e]) : 0.f);
  E* y = static_cast<E*>(c.y) + i;
  if constexpr (!kWide) *y = T::from_f32(v[0]);
  else if constexpr (sizeof(E) == 2) *reinterpret_cast<u32x2*>(y) = u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
  else *reinterpret_cast<f32x4*>(y) = f32x4{v[0], v[1], v[2], v[3]};
}

// The tiles.  The small ones, whose steps are bound by latency, keep more steps on their way.
using Tile32x64 = Tile<32, 64, 16, 32, 20>;
using Tile64x64 = Tile<64, 64, 32, 32, 20>;
using Tile64x128 = Tile<64, 128, 32, 64, 10>;
using Tile128x128 = Tile<128, 128, 64, 64, 10>;
using Tile128x128Two = Tile<128, 128, 64, 64, 5>;  // two workgroups to a compute unit
using Tile128x192 = Tile<128, 192, 64, 96, 6>;
using Tile256x256 = Tile<256, 256, 128, 128, 5>;

template <typename S, typename T>
int launch_tiles(const Int8Call& c, int splits, void* out, hipStream_t stream) {
  static PerDeviceInt limit;
  const void* kernel = reinterpret_cast<const void*>(&int8_tile_kernel<S, T>);
  if (!raise_lds_limit(limit, kernel, S::kLds)) return MFQ_ELAUNCH;
  const int64_t tiles_m = (c.M + S::kM - 1) / S::kM, tiles_n = (c.N + S::kN - 1) / S::kN;
  const int64_t items = tiles_m * tiles_n * splits, places = (int64_t)compute_units() * (kMaxLds / S::kLds);
  if (items + places > INT32_MAX) return MFQ_ESHAPE;
  hipLaunchKernelGGL((int8_tile_kernel<S, T>), dim3((unsigned)(items < places ? items : places)), dim3(S::kThreads), S::kLds, stream, c,
                     (int)tiles_m, (int)tiles_n, splits, out);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T>
int launch_tiles_of(const Int8Call& c, const Int8Tiles& t, int splits, void* out, hipStream_t stream) {
  switch (t.rows * 1000 + t.columns) {
    case 32064: return launch_tiles<Tile32x64, T>(c, splits, out, stream);
    case 64064: return launch_tiles<Tile64x64, T>(c, splits, out, stream);
    case 64128: return launch_tiles<Tile64x128, T>(c, splits, out, stream);
    case 128128: return t.places == 2 ? launch_tiles<Tile128x128Two, T>(c, splits, out, stream) : launch_tiles<Tile128x128, T>(c, splits, out, stream);
    case 128192: return launch_tiles<Tile128x192, T>(c, splits, out, stream);
    default:
      if constexpr (sizeof(typename T::storage) == 2) return launch_tiles<Tile256x256, T>(c, splits, out, stream);
      else return MFQ_EUNSUPPORTED;  // the plan has none
  }
}

// Wavefronts of a workgroup and steps of a wavefront: the fewest steps left over, of 8 to 16 wavefronts
void few_shape(int64_t K, int& waves, int& steps) {
  const int all = (int)((K + BK - 1) / BK);
  waves = all < 8 ? all : 8;
  steps = (all + 7) / 8;
  for (int w = 9; w <= kFewMaxWaves; ++w) {
    const int each = (all + w - 1) / w;
    if (each * w < steps * waves) waves = w, steps = each;
  }
}
struct Few {
  int waves, steps, per_group, groups, rounds;
  int64_t grid;
};
// A product of groups of 8 tokens8 rows of x; false: x does not fit
bool few_of(int64_t M, int64_t N, int64_t K, int tokens8, Few& f) {
  few_shape(K, f.waves, f.steps);
  // One workgroup to a compute unit (two or three, each with fewer blocks, take 15 us where one takes 12: 10240 x 3840), in as many
  // equal rounds as the room for sums asks for
  const int64_t most = (kMaxLds - few_image(tokens8, f.steps, f.waves)) / few_sums(tokens8, f.waves), places = compute_units();
  if (most < 2) return false;
  const int64_t blocks = (N + 7) / 8, groups = (M + 8 * tokens8 - 1) / (8 * tokens8);
  const int64_t rounds = (blocks * groups + places * most - 1) / (places * most);
  const int64_t per_group = (blocks * groups + places * rounds - 1) / (places * rounds), runs = (blocks + per_group - 1) / per_group;
  f.per_group = (int)per_group;
  f.groups = (int)groups;
  f.rounds = (int)rounds;
  f.grid = (runs + 7) / 8 * 8 * groups;
  return true;
}

template <int kX, int kRing, typename T>
int launch_few_of(const Int8Call& c, const Few& f, hipStream_t stream) {
  static PerDeviceInt limit;
  if (!raise_lds_limit(limit, reinterpret_cast<const void*>(&int8_few_kernel<kX, kRing, T>), kMaxLds)) return MFQ_ELAUNCH;
  const int lds = few_image(kX, f.steps, f.waves) + f.per_group * few_sums(kX, f.waves);
  hipLaunchKernelGGL((int8_few_kernel<kX, kRing, T>), dim3((unsigned)f.grid), dim3(f.waves * kWave), lds, stream, c, f.waves, f.steps, f.per_group,
                     f.groups);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <int kX, typename T>
int launch_few(const Int8Call& c, hipStream_t stream) {
  Few f;
  if (!few_of(c.M, c.N, c.K, kX, f)) return MFQ_EUNSUPPORTED;  // the plan has none
  const int64_t positions = (int64_t)f.per_group * f.steps;  // requests of a wavefront: those behind the last are in vain
  if (positions <= 2) return launch_few_of<kX, 2, T>(c, f, stream);
  return positions <= 5 ? launch_few_of<kX, 4, T>(c, f, stream) : launch_few_of<kX, 8, T>(c, f, stream);
}

template <typename T>
int launch(const Int8Call& c, const Int8Plan& p, void* workspace, hipStream_t stream) {
  if (p.kernel == MFQ_INT8_FEW) {
    switch (p.tiles.rows) {
      case 8: return launch_few<1, T>(c, stream);
      case 16: return launch_few<2, T>(c, stream);
      case 24: return launch_few<3, T>(c, stream);
      default: return launch_few<4, T>(c, stream);
    }
  }
  if (p.first) {  // two products side by side, of columns that fill whole rounds of workgroups and of the others
    using E = typename T::storage;
    Int8Call part = c;
    part.N = p.first;
    if (int rc = launch_tiles_of<T>(part, p.tiles, 1, part.y, stream)) return rc;
    part.N = c.N - p.first;
    part.w += p.first * c.w_stride;
    part.w_scales += p.first;
    if (part.bias) part.bias = static_cast<const E*>(c.bias) + p.first;
    part.y = static_cast<E*>(c.y) + p.first;
    return launch_tiles_of<T>(part, p.rest, 1, part.y, stream);
  }
  if (p.splits == 1) return launch_tiles_of<T>(c, p.tiles, 1, c.y, stream);
  if (int rc = launch_tiles_of<I32>(c, p.tiles, p.splits, workspace, stream)) return rc;
  const bool wide = c.N % 4 == 0;
  const int64_t threads = c.M * c.N / (wide ? 4 : 1);
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (wide) hipLaunchKernelGGL((int8_join_kernel<T, true>), grid, dim3(256), 0, stream, c, static_cast<const int*>(workspace), p.splits);
  else hipLaunchKernelGGL((int8_join_kernel<T, false>), grid, dim3(256), 0, stream, c, static_cast<const int*>(workspace), p.splits);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

}  // namespace

// What a product is estimated to take, in us, and the tile of the least: launch and first bytes 3, a round of workgroups as many steps
// as its range of K has at the tile's time each, a cut K 4 for the second launch and its planes at 3 TB/s written and read.  Times of a
// step measured with all compute units busy (30 and 80 steps, 120 to 1360 tiles): they follow the tile's bytes through LDS and a
// latency, not its matrix instructions, but for the largest.
struct Choice {
  Int8Tiles tiles;
  float step;
};
constexpr Choice kChoices[] = {{{32, 64, 1}, 0.30f},   {{64, 64, 1}, 0.40f},   {{64, 128, 1}, 0.47f},  {{128, 128, 1}, 0.66f},
                               {{128, 128, 2}, 1.12f}, {{128, 192, 1}, 0.84f}, {{256, 256, 1}, 1.58f}};

float least_time(int dtype, int64_t M, int64_t N, int64_t steps, bool cut_k, Int8Tiles& tiles, int& splits) {
  float least = 1e30f;
  for (const Choice& o : kChoices) {
    if (o.tiles.rows == 256 && dtype == MFQ_F32) continue;
    const int64_t n = ((M + o.tiles.rows - 1) / o.tiles.rows) * ((N + o.tiles.columns - 1) / o.tiles.columns);
    const int64_t places = (int64_t)compute_units() * o.tiles.places;
    int64_t most = o.tiles.rows == 256 || !cut_k ? 1 : places / n;
    if (most > steps / 4) most = steps / 4;
    if (most > 16) most = 16;
    for (int cut = 0; cut < 2; ++cut) {
      const int64_t s = cut ? most : 1;
      if (cut && s < 2) break;
      float t = 3.f + (float)((n * s + places - 1) / places) * (float)((steps + s - 1) / s) * o.step;
      if (s > 1) t += 4.f + (float)(s * M * N) * 4.f / 3e6f;
      if (t < least) {
        least = t;
        tiles = o.tiles;
        splits = (int)s;
      }
    }
  }
  return least;
}

Int8Plan int8_plan(int dtype, int64_t M, int64_t N, int64_t K) {
  Int8Plan p = {MFQ_INT8_TILES, 1, {}, 0, {}};
  const int64_t steps = (K + BK - 1) / BK;
  const int groups = (int)((M + 31) / 32), tokens8 = M <= 128 ? (int)((M + 8 * groups - 1) / (8 * groups)) : 0;
  Few f;
  const bool few = tokens8 && few_of(M, N, K, tokens8, f);
  if (few && M <= 16) {
    p.kernel = MFQ_INT8_FEW;
    p.tiles = {8 * tokens8, 8, 1};
    return p;
  }
  const float whole = least_time(dtype, M, N, steps, true, p.tiles, p.splits);
  // Few rows: always up to 16, where w's bytes bound it.  Above, by an estimate: a workgroup's x (KiB of LDS, once a round) and its
  // blocks of w at 33 bytes a ns, and 0.7 us a block.  24 x 2048 x 1024 6.2 -> 4.2 us, 24 x 3840 x 3840 10.0 -> 8.1, 128 x 512 x 2048
  // 7.5 -> 5.3 (four groups), but 24 x 10240 x 3840 would take 20 instead of 15.
  if (few) {
    const float kib = (float)(few_image(tokens8, f.steps, f.waves) + 8 * f.per_group * K) / 1024.f;
    if (1.8f + (float)f.rounds * (0.03f * kib + 0.7f * (float)f.per_group) < whole) {
      p.kernel = MFQ_INT8_FEW;
      p.splits = 1;
      p.tiles = {8 * tokens8, 8, 1};
      return p;
    }
  }
  if (p.tiles.rows != 256) return p;
  // The largest tiles' last round may leave most compute units idle: whole rounds of them, and smaller tiles for the columns behind
  // (one launch -> two: 2000 x 10240 x 3840 96 -> 81 us, 5000 x 3840 x 10240 212 -> 175, 4352 x 12288 x 4096 201 -> 193,
  // 4352 x 20480 x 3840, five rounds and a third, 305 -> 302, and 2 % slower at most, 3000 x 20480 x 3840)
  const int64_t units = compute_units(), down = (M + 255) / 256, across = (N + 255) / 256, columns = down * across / units * units / down;
  if (columns == 0 || columns >= across) return p;
  int one;
  Int8Tiles rest;
  const float behind = least_time(dtype, M, N - 256 * columns, steps, false, rest, one);
  if (3.f + (float)((down * columns + units - 1) / units) * (float)steps * 1.58f + behind < whole) {
    p.first = 256 * columns;
    p.rest = rest;
  }
  return p;
}

size_t int8_workspace_bytes(const Int8Plan& p, int64_t M, int64_t N) { return p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0; }

int launch_int8_matmul(int dtype, const Int8Call& c, const Int8Plan& p, void* workspace, hipStream_t stream) {
  if (dtype == MFQ_BF16) return launch<BF16>(c, p, workspace, stream);
  if (dtype == MFQ_F16) return launch<F16>(c, p, workspace, stream);
  return launch<F32>(c, p, workspace, stream);
}

}  // namespace mfq
