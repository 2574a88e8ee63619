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
// does, 3.0 where both change (32x32x32: 3.4; zeros, bound by issue: 4.2, 32x32x32 4.9).
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
    const bool whole = c.N % kEach == 0;
    const int64_t n0 = it.n0 + wn, m0 = it.m0 + wm + r;
    char* y = static_cast<char*>(out) + ((kRaw ? (int64_t)it.split * c.M : 0) + m0) * c.N * (int64_t)sizeof(E);
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
        E* row = reinterpret_cast<E*>(y + (int64_t)(16 * i) * c.N * (int64_t)sizeof(E));
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
// Up to 16 rows of x: bound by the bytes of w, which go from memory straight into registers.  On v_mfma_i32_16x16x64_i8 lane
// (j, q) = (lane % 16, lane / 16) supplies 16 bytes of row j of either operand.  One load instruction of w takes eight rows x
// 128 bytes, whole cache lines: operand row j is row j / 2, bytes 64 (j % 2) + 16 q.  x enters as eight rows x 128 bytes as
// well, operand row j being row j % 8, bytes 64 (j / 8) + 16 q.  Of the 16 x 16 results those belong together whose halves are the
// same (row 8 h + token, column 2 row + h); the others are dropped.  The wavefronts of a workgroup take a range of K each of
// the same 16 rows of w, and their sums meet in LDS.
template <int kTokens, int kWaves, typename T>
__global__ __launch_bounds__(kWaves* kWave) void int8_few_kernel(Int8Call c) {
  using E = typename T::storage;
  constexpr int kX = kTokens / 8, kW = 2, kAhead = 4;
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int j = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int all_steps = (int)((c.K + BK - 1) / BK), tail = (int)((c.K - 1) & (BK - 1)) + 1;
  const int first = (int)((int64_t)all_steps * wave / kWaves), end = (int)((int64_t)all_steps * (wave + 1) / kWaves);
  const int w_column = 64 * (j & 1) + 16 * q, x_column = 64 * (j >> 3) + 16 * q;
  const int8_t *wp[kW], *xp[kX];
#pragma unroll
  for (int b = 0; b < kW; ++b) wp[b] = c.w + min(n0 + 8 * b + (j >> 1), c.N - 1) * c.w_stride;
#pragma unroll
  for (int b = 0; b < kX; ++b) xp[b] = c.x + min((int64_t)(8 * b + (j & 7)), c.M - 1) * c.x_stride;
  i32x4 w[kAhead][kW], x[kAhead][kX], acc[kW][kX];
#pragma unroll
  for (int b = 0; b < kW; ++b)
#pragma unroll
    for (int a = 0; a < kX; ++a) acc[b][a] = i32x4{0, 0, 0, 0};
  // steps past the wavefront's end repeat its last one and are never multiplied; bytes past the end of K repeat others, x's are 0
  auto load = [&](int s, int slot) __attribute__((always_inline)) {
    const int at = max(min(s, end - 1), 0), most = at == all_steps - 1 ? tail - 16 : BK - 16;
    const bool past = x_column > most;
#pragma unroll
    for (int b = 0; b < kW; ++b) w[slot][b] = *reinterpret_cast<const i32x4*>(wp[b] + (int64_t)at * BK + min(w_column, most));
#pragma unroll
    for (int a = 0; a < kX; ++a) {
      x[slot][a] = *reinterpret_cast<const i32x4*>(xp[a] + (int64_t)at * BK + min(x_column, most));
      if (past) x[slot][a] = i32x4{0, 0, 0, 0};
    }
  };
#pragma unroll
  for (int s = 0; s < kAhead; ++s) load(first + s, s);
  for (int s = first; s < end; s += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s + u < end) {
#pragma unroll
        for (int b = 0; b < kW; ++b)
#pragma unroll
          for (int a = 0; a < kX; ++a) acc[b][a] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[u][a], w[u][b], acc[b][a], 0, 0, 0);
      }
      load(s + u + kAhead, u);
    }
  }
  // register e of a lane: operand row 4 q + e (half q / 2, token 4 (q % 2) + e), column j (row j / 2 of w, half j % 2)
  __shared__ int sums[2 * kWaves][kTokens][kW * 8];
  if ((j & 1) == (q >> 1)) {
#pragma unroll
    for (int b = 0; b < kW; ++b)
#pragma unroll
      for (int a = 0; a < kX; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[2 * wave + (j & 1)][8 * a + 4 * (q & 1) + e][8 * b + (j >> 1)] = acc[b][a][e];
  }
  __syncthreads();
  for (int o = t; o < kTokens * kW * 8; o += kWaves * kWave) {
    const int token = o / (kW * 8), row = o % (kW * 8);
    const int64_t n = n0 + row;
    if (token >= c.M || n >= c.N) continue;
    int sum = 0;
#pragma unroll
    for (int k = 0; k < 2 * kWaves; ++k) sum += sums[k][token][row];
    const float v = value_of(sum, c.x_scales[token], c.w_scales[n], c.bias ? T::to_f32(static_cast<const E*>(c.bias)[n]) : 0.f);
    static_cast<E*>(c.y)[token * c.N + n] = T::from_f32(v);
  }
}

// ---- the ranges of a cut K joined: four outputs to a thread where rows are whole fours
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

using Tile32 = Tile<32, 128, 32, 32, 5>;
using Tile64 = Tile<64, 64, 32, 32, 10>;
using Tile128 = Tile<128, 128, 64, 64, 5>;
using Tile256 = Tile<256, 256, 128, 128, 5>;

template <typename S, typename T>
int launch_tiles(const Int8Call& c, int splits, void* out, hipStream_t stream) {
  static PerDeviceInt limit;
  const void* kernel = reinterpret_cast<const void*>(&int8_tile_kernel<S, T>);
  if (!raise_lds_limit(limit, kernel, S::kLds)) return MFQ_ELAUNCH;
  const int64_t tiles_m = (c.M + S::kM - 1) / S::kM, tiles_n = (c.N + S::kN - 1) / S::kN;
  const int64_t items = tiles_m * tiles_n * splits, places = (int64_t)compute_units() * (kMaxLds / S::kLds);
  hipLaunchKernelGGL((int8_tile_kernel<S, T>), dim3((unsigned)(items < places ? items : places)), dim3(S::kThreads), S::kLds, stream, c,
                     (int)tiles_m, (int)tiles_n, splits, out);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T>
int launch_tiles_of(const Int8Call& c, const Int8Plan& p, void* out, hipStream_t stream) {
  if (p.rows == 32) return launch_tiles<Tile32, T>(c, p.splits, out, stream);
  if (p.rows == 64) return launch_tiles<Tile64, T>(c, p.splits, out, stream);
  if (p.rows == 128) return launch_tiles<Tile128, T>(c, p.splits, out, stream);
  if constexpr (sizeof(typename T::storage) == 2) {
    if (p.rows == 256) return launch_tiles<Tile256, T>(c, p.splits, out, stream);
  }
  return MFQ_EUNSUPPORTED;
}

template <typename T>
int launch(const Int8Call& c, const Int8Plan& p, void* workspace, hipStream_t stream) {
  if (p.kernel == MFQ_INT8_FEW) {
    const dim3 grid((unsigned)((c.N + 15) / 16));
    if (c.M <= 8) hipLaunchKernelGGL((int8_few_kernel<8, 8, T>), grid, dim3(8 * kWave), 0, stream, c);
    else hipLaunchKernelGGL((int8_few_kernel<16, 8, T>), grid, dim3(8 * kWave), 0, stream, c);
    return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
  }
  if (p.splits == 1) return launch_tiles_of<T>(c, p, c.y, stream);
  if (int rc = launch_tiles_of<I32>(c, p, workspace, stream)) return rc;
  const bool wide = c.N % 4 == 0;
  const int64_t threads = c.M * c.N / (wide ? 4 : 1);
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (wide) hipLaunchKernelGGL((int8_join_kernel<T, true>), grid, dim3(256), 0, stream, c, static_cast<const int*>(workspace), p.splits);
  else hipLaunchKernelGGL((int8_join_kernel<T, false>), grid, dim3(256), 0, stream, c, static_cast<const int*>(workspace), p.splits);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

}  // namespace

Int8Plan int8_plan(int dtype, int64_t M, int64_t N, int64_t K) {
  if (M <= 16) return {MFQ_INT8_FEW, 1, (int)M, 16};
  const int64_t units = compute_units(), steps = (K + BK - 1) / BK;
  Int8Plan p = {MFQ_INT8_TILES, 1, 256, 256};
  if (M <= 32) p.rows = 32, p.columns = 128;
  else if (M <= 64) p.rows = p.columns = 64;
  else if (dtype == MFQ_F32 || ((M + 255) / 256) * ((N + 255) / 256) < units * 3 / 4) p.rows = p.columns = 128;
  const int64_t tiles = ((M + p.rows - 1) / p.rows) * ((N + p.columns - 1) / p.columns);
  const int64_t places = p.rows == 256 ? units : 2 * units;
  if (tiles * 2 <= places) {
    int64_t s = places / tiles, most = steps / 4;
    if (s > most) s = most;
    if (s > 16) s = 16;
    if (s >= 2) p.splits = (int)s;
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
