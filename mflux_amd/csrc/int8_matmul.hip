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
// A workgroup of four wavefronts computes kM x kN outputs, a wavefront kWM x kWN of them on v_mfma_i32_32x32x32_i8 with w as
// the first operand (a lane's registers are four neighbouring columns of y each, of one row).
//   - x and w go from memory straight into LDS, 128 bytes of a row at a time: kStages steps of both, the 16-byte column of a row
//     XORed with (row / 2) % 8, so that the 32 rows of a fragment spread over the banks;
//   - the fragments of a quarter step (32 k) are read while the one before them is multiplied, across the end of a step too:
//     the one barrier of a step lies in front of its last quarter, where the fragments of that quarter are in registers (the
//     step's LDS is free for the step kStages later) and the next step's LDS has arrived.
template <int kM_, int kN_, int kWM_, int kWN_, int kStages_>
struct Tile {
  static constexpr int kM = kM_, kN = kN_, kWM = kWM_, kWN = kWN_, kStages = kStages_;
  static constexpr int kAcross = kM / kWM, kWaves = kAcross * (kN / kWN), kThreads = kWaves * kWave;
  static constexpr int kI = kWM / 32, kJ = kWN / 32;
  static constexpr int kStageBytes = (kM + kN) * BK;
  static constexpr int kLoads = (kM + kN) / 8 / kWaves;  // of a wavefront, a KiB each
  static constexpr int kOutStride = kWN * 4 + 16;        // a staged row of results, of 32-bit types
  static constexpr int kOutBytes = kWaves * (32 * kOutStride + 2 * kWN * 4);  // and w's scales and the bias of a wavefront's columns
  static constexpr int kLds = kStages * kStageBytes > kOutBytes ? kStages * kStageBytes : kOutBytes;
  static constexpr int kXLoads = kM / 8 / kWaves;
  static_assert(kM % (8 * kWaves) == 0 && kN % (8 * kWaves) == 0 && kLds <= kMaxLds, "");
};

template <typename S, typename T>
__global__ __launch_bounds__(S::kThreads) void int8_tile_kernel(Int8Call c, int tiles_m, int tiles_n, int splits, void* out) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kI = S::kI, kJ = S::kJ, kLoads = S::kLoads;
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int r = lane & 31, h = lane >> 5;

  // Work item = (range of K, tile); an XCD walks a contiguous run of the tiles, in bands of four tile rows
  const int n_tiles = tiles_m * tiles_n;
  const int split = __builtin_amdgcn_readfirstlane((int)blockIdx.x / n_tiles);
  int tile = (int)blockIdx.x - split * n_tiles;
  const int per_xcd = n_tiles / 8;
  if (tile < per_xcd * 8) tile = (tile & 7) * per_xcd + (tile >> 3);
  constexpr int kBand = 4;
  const int band = tile / (kBand * tiles_n), band_rows = min(tiles_m - band * kBand, kBand), in_band = tile - band * kBand * tiles_n;
  const int64_t m0 = (int64_t)__builtin_amdgcn_readfirstlane(band * kBand + in_band % band_rows) * S::kM;
  const int64_t n0 = (int64_t)__builtin_amdgcn_readfirstlane(in_band / band_rows) * S::kN;

  const int all_steps = ((int)c.K + BK - 1) / BK;  // at most 1024, of at most 1024 ranges
  const int first = __builtin_amdgcn_readfirstlane(all_steps * split / splits);
  const int steps = __builtin_amdgcn_readfirstlane(all_steps * (split + 1) / splits) - first;

  // ---- what the wavefront loads: eight rows x 128 bytes an instruction, the tile's rows of x dealt to the wavefronts in
  // turn, then those of w
  const int own_row = wave * 8 + (lane >> 3);
  const int last_x = (int)min(c.M - m0, (int64_t)S::kM) - 1, last_w = (int)min(c.N - n0, (int64_t)S::kN) - 1;
  uint32_t row_at[kLoads];
#pragma unroll
  for (int l = 0; l < kLoads; ++l)
    row_at[l] = l < S::kXLoads ? (uint32_t)min(own_row + 8 * S::kWaves * l, last_x) * (uint32_t)c.x_stride
                               : (uint32_t)min(own_row + 8 * S::kWaves * (l - S::kXLoads), last_w) * (uint32_t)c.w_stride;
  const int8_t *x0 = c.x + m0 * c.x_stride, *w0 = c.w + n0 * c.w_stride;
  const uint32_t column = 16 * ((lane & 7) ^ ((own_row >> 1) & 7));  // of a row, that goes to the lane's place
  const uint32_t lds_addr = (uint32_t)(uintptr_t)lds + (uint32_t)(wave * 8 * BK);
  const uint32_t tail = (uint32_t)((c.K - 1) & (BK - 1)) + 1;  // bytes of a row in the last step of all
  // Step q of the item into its stage.  The bytes of the last step past the end of K repeat others; x's are cleared below.
  auto load = [&](int q, int stage) __attribute__((always_inline)) {
    const int at = first + q;
    const uint32_t col = min(column, at == all_steps - 1 ? tail - 16 : (uint32_t)BK - 16);
    const uint32_t to = lds_addr + (uint32_t)(stage * S::kStageBytes);
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      asm volatile("s_add_i32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                   ::"v"(row_at[l] + col), "s"((l < S::kXLoads ? x0 : w0) + (int64_t)at * BK), "s"(to), "i"(l * S::kWaves * 1024)
                   : "memory", "m0", "scc");
  };
  // x past the end of K, once it has arrived
  auto clear_tail = [&](int stage) __attribute__((always_inline)) {
    if (column < tail) return;
#pragma unroll
    for (int l = 0; l < S::kXLoads; ++l)
      *reinterpret_cast<u32x4*>(lds + stage * S::kStageBytes + (wave + l * S::kWaves) * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
  };

  // ---- fragments
  const int wm = wave % S::kAcross * S::kWM, wn = wave / S::kAcross * S::kWN;
  i32x4 xf[2][kI], wf[2][kJ];
  const int swz = (r >> 1) & 7;
  auto read = [&](int set, int stage, int quarter) __attribute__((always_inline)) {
    const char* p = lds + stage * S::kStageBytes + r * BK + (((2 * quarter + h) ^ swz) << 4);
#pragma unroll
    for (int j = 0; j < kJ; ++j) wf[set][j] = *reinterpret_cast<const i32x4*>(p + (S::kM + wn + 32 * j) * BK);
#pragma unroll
    for (int i = 0; i < kI; ++i) xf[set][i] = *reinterpret_cast<const i32x4*>(p + (wm + 32 * i) * BK);
  };
  i32x16 acc[kI][kJ];
#pragma unroll
  for (int i = 0; i < kI; ++i)
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int i = 0; i < kI; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[set][j], xf[set][i], acc[i][j], 0, 0, 0);
  };
  // own loads of the next step have arrived (and everything the wavefront has read from LDS is in registers), for all wavefronts
  auto arrive = [&](int q) __attribute__((always_inline)) {  // q: the step that must be there
    if (S::kStages > 2 && q + S::kStages - 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S::kStages - 2) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if (tail < BK && first + q == all_steps - 1) {
      clear_tail(q % S::kStages);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    asm volatile("s_barrier" ::: "memory");
  };

  if (steps > 0) {
#pragma unroll
    for (int q = 0; q < S::kStages; ++q)
      if (q < steps) load(q, q);
    if (S::kStages > 1 && steps >= S::kStages) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S::kStages - 1) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (tail < BK && first == all_steps - 1) {
      clear_tail(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    asm volatile("s_barrier" ::: "memory");
    read(0, 0, 0);
    int stage = 0;
    for (int q = 0; q < steps; ++q) {
      const int after = stage + 1 == S::kStages ? 0 : stage + 1;
      read(1, stage, 1);
      multiply(0);
      read(0, stage, 2);
      multiply(1);
      read(1, stage, 3);
      multiply(0);
      if (q + 1 < steps) {
        arrive(q + 1);
        if (q + S::kStages < steps) load(q + S::kStages, stage);
        read(0, after, 0);
      }
      multiply(1);
      stage = after;
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // LDS is free for the results

  // ---- results: strips of 32 rows through a private region of LDS, so that whole row segments are written
  // register e of acc[i][j] is row wm + 32 i + r, column wn + 32 j + 8 (e / 4) + 4 h + e % 4
  using E = typename T::storage;
  constexpr bool kRaw = std::is_same_v<T, I32>;
  constexpr int kEach = 16 / (int)sizeof(E);               // values of a 16-byte piece
  constexpr int kStride = S::kWN * (int)sizeof(E) + 16;
  constexpr int kPieces = S::kWN / kEach, kRowsAtOnce = kWave / kPieces;
  char* strip = lds + wave * 32 * S::kOutStride;
  E* y = static_cast<E*>(out) + (kRaw ? (int64_t)split * c.M * c.N : 0);
  const E* bias = static_cast<const E*>(c.bias);
  const bool whole = c.N % kEach == 0;
  float* w_scales = reinterpret_cast<float*>(lds + S::kWaves * 32 * S::kOutStride) + wave * 2 * S::kWN;
  if constexpr (!kRaw) {
#pragma unroll
    for (int k = lane; k < S::kWN; k += kWave) {
      const int64_t n = min(n0 + wn + k, c.N - 1);
      w_scales[k] = c.w_scales[n];
      w_scales[S::kWN + k] = bias ? T::to_f32(bias[n]) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < kI; ++i) {
    const int64_t m = m0 + wm + 32 * i + r;
    float xs = 0.f;
    if constexpr (!kRaw) xs = c.x_scales[min(m, c.M - 1)];
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int col = 32 * j + 8 * b + 4 * h;
        if constexpr (kRaw) {
          *reinterpret_cast<i32x4*>(strip + r * kStride + col * 4) =
              i32x4{acc[i][j][4 * b], acc[i][j][4 * b + 1], acc[i][j][4 * b + 2], acc[i][j][4 * b + 3]};
        } else {
          const f32x4 ws = *reinterpret_cast<const f32x4*>(w_scales + col), add = *reinterpret_cast<const f32x4*>(w_scales + S::kWN + col);
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = value_of(acc[i][j][4 * b + e], xs, ws[e], add[e]);
          if constexpr (sizeof(E) == 2) *reinterpret_cast<u32x2*>(strip + r * kStride + col * 2) = u32x2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
          else *reinterpret_cast<f32x4*>(strip + r * kStride + col * 4) = f32x4{v[0], v[1], v[2], v[3]};
        }
      }
    }
    const int piece = lane % kPieces;
    const int64_t n = n0 + wn + piece * kEach;
#pragma unroll
    for (int k = 0; k < 32 / kRowsAtOnce; ++k) {
      const int row = k * kRowsAtOnce + lane / kPieces;
      const u32x4 v = *reinterpret_cast<const u32x4*>(strip + row * kStride + piece * 16);
      const int64_t at = m0 + wm + 32 * i + row;
      if (at >= c.M) continue;
      if (whole) {
        if (n < c.N) *reinterpret_cast<u32x4*>(y + at * c.N + n) = v;
      } else {
        const E* e = reinterpret_cast<const E*>(&v);
#pragma unroll
        for (int k2 = 0; k2 < kEach; ++k2)
          if (n + k2 < c.N) y[at * c.N + n + k2] = e[k2];
      }
    }
  }
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

using Tile32 = Tile<32, 128, 32, 32, 4>;
using Tile64 = Tile<64, 64, 32, 32, 4>;
using Tile128 = Tile<128, 128, 64, 64, 2>;
using Tile256 = Tile<256, 256, 128, 128, 2>;

template <typename S, typename T>
int launch_tiles(const Int8Call& c, int splits, void* out, hipStream_t stream) {
  static PerDeviceInt limit;
  const void* kernel = reinterpret_cast<const void*>(&int8_tile_kernel<S, T>);
  if (!raise_lds_limit(limit, kernel, S::kLds)) return MFQ_ELAUNCH;
  const int64_t tiles_m = (c.M + S::kM - 1) / S::kM, tiles_n = (c.N + S::kN - 1) / S::kN;
  hipLaunchKernelGGL((int8_tile_kernel<S, T>), dim3((unsigned)(tiles_m * tiles_n * splits)), dim3(S::kThreads), S::kLds, stream, c, (int)tiles_m,
                     (int)tiles_n, splits, out);
  return hipGetLastError() == hipSuccess ? MFQ_OK : MFQ_ELAUNCH;
}

template <typename T>
int launch_tiles_of(const Int8Call& c, const Int8Plan& p, void* out, hipStream_t stream) {
  if (p.rows == 32) return launch_tiles<Tile32, T>(c, p.splits, out, stream);
  if (p.rows == 64) return launch_tiles<Tile64, T>(c, p.splits, out, stream);
  if (p.rows == 128) return launch_tiles<Tile128, T>(c, p.splits, out, stream);
  return launch_tiles<Tile256, T>(c, p.splits, out, stream);
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

Int8Plan int8_plan(int64_t M, int64_t N, int64_t K) {
  if (M <= 16) return {MFQ_INT8_FEW, 1, (int)M, 16};
  const int64_t units = compute_units(), steps = (K + BK - 1) / BK;
  Int8Plan p = {MFQ_INT8_TILES, 1, 256, 256};
  if (M <= 32) p.rows = 32, p.columns = 128;
  else if (M <= 64) p.rows = p.columns = 64;
  else if (((M + 255) / 256) * ((N + 255) / 256) < units * 3 / 4) p.rows = p.columns = 128;
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
