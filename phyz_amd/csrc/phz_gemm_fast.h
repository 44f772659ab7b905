// phz_gemm_fast.h — the matrix product for aligned operands:
//
//   C[i][j] = sum_k A(i, k) B(j, k)
//
// Operands are one plane of 16-bit elements, f32 (through the f32 matrix
// instructions: exact products at a sixteenth of the rate), or a sum of planes:
//   two    A = hi + lo, f32 data cut in f16: lo hi + hi lo + hi hi (lo lo, at
//          most 2^-22 of a product, is left out as the cut's own 2^-23 are), for
//          data of a known range;
//   three  A = h + m + l, f32 data cut in bf16 without loss (cut3): six of the
//          nine products, as in phz_gemm.h, for any data.
// A may have two planes where B has one: lo b + hi b, f32 data (cut2) with bf16.
// Rows are 16-byte aligned and, along k (or along rows, for
// operands dense along rows), whole 16 bytes long or padded with zeros to them.
#pragma once
#include <algorithm>

#include "phz_gemm.h"

namespace phzop {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

struct half_t { uint16_t bits; };
__device__ __forceinline__ float to_f32(half_t v) { return (float)__builtin_bit_cast(_Float16, v.bits); }
template <> __device__ __forceinline__ half_t from_f32<half_t>(float v) {
  return half_t{__builtin_bit_cast(uint16_t, (_Float16)v)};
}

// Products of two fragments of 16 bytes a lane: kStep of k.
template <class T> struct Mfma;
template <> struct Mfma<float> {
  static constexpr int kStep = 8;  // as multiply() in phz_gemm.h
  static __device__ __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};
template <> struct Mfma<bf16> {
  static constexpr int kStep = 16;
  static __device__ __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mfma<half_t> {
  static constexpr int kStep = 16;
  static __device__ __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

struct FastArgs {
  const char *a, *b, *zeros;
  int64_t a_row, b_row, a_batch, b_batch;  // bytes
  uint32_t a_plane, b_plane;               // bytes from a plane to the next
  int32_t m, n, k;
  int32_t a_rows, b_rows;   // rows that exist (dense along rows: whole 16 bytes)
  int32_t k_split, splits;  // contraction per split, a multiple of 64
  int32_t tiles_m, tiles_n;
};

// 16 bytes a lane from global memory to LDS at `lds` + 16 lane, without passing
// registers. Written as asm so that the compiler does not wait for it at the
// next LDS read: the loop below waits for a stage's loads itself. There is no
// output register; the wait state is the one that a write of m0 needs.
__device__ __forceinline__ void dma16(uint32_t lds, const char* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma16(uint32_t lds, const char* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory", "m0");
}

// One operand's tile of ROWS rows by BK: how it lies in LDS, how NW waves
// bring it there, and how a lane reads a fragment (eight k of one row).
//
// Dense along k: rows of 2 BK bytes. The 16-byte chunks of row r stand in the
// order c ^ f(r), with f such that the reads of 16 consecutive rows fall into
// all 64 banks. Dense along rows: BK rows (one a k) of 2 ROWS bytes, read
// through the transposing LDS read, which hands each lane of 16 a column of a
// 4 x 16 block; 64-byte groups of the row of k stand in the order g ^ (k % 4),
// so the four rows of a block fall into all banks (with rows of 128 bytes, two
// of them a bank row, g ^ (k / 2 % 2)). Measured (counters): no
// bank conflicts in either.
// With two planes the tile holds SK = 32 of k twice: hi's, then lo's. With
// three it is three tiles of 32 of k.
template <class T, bool ALONG_K, int ROWS, int SLOTS, int NW, int PL>
struct FastTile {
  static constexpr int ES = sizeof(T), EL = 16 / ES;  // bytes of an element, elements of 16 bytes
  static constexpr int kParts = PL == 3 ? 3 : 1, BK = SLOTS / kParts, SK = SLOTS / PL;
  static constexpr int kPart = ROWS * BK * ES, kBytes = kParts * kPart;
  static constexpr int kPerWave = kBytes / 1024 / NW;  // 1 KB loads of each wave
  static constexpr int kChunks = (ALONG_K ? BK : ROWS) / EL, kRows = 64 / kChunks;  // 16-byte chunks of a row, rows of a load
  static_assert(kPerWave * NW * 1024 == kBytes, "whole loads for every wave");
  uint32_t off[kPerWave];
  int32_t kk[kPerWave];  // first k of the lane's 16 bytes within the tile

  // What the row r's (k's) chunks are permuted by.
  static __device__ __forceinline__ int order(int r) {
    if (ALONG_K) return BK * ES == 64 ? (r >> 2) & 3 : (r >> 1) & 7;
    if (ES == 4) return 0;  // read an element a lane: no two share a bank
    return (ROWS == 64 ? (r >> 1) & 1 : r & 3) << 2;
  }

  __device__ __forceinline__ void init(int wave, int lane, int row0, int rows, int64_t row_bytes, uint32_t plane) {
#pragma unroll
    for (int i = 0; i < kPerWave; i++) {
      const int at = wave * kPerWave + i, part = at / (kPart / 1024);
      const int r = at % (kPart / 1024) * kRows + lane / kChunks;
      if (ALONG_K) {
        const int c = (lane % kChunks) ^ order(r);
        // Rows past the end repeat the last one: their sums are not stored.
        kk[i] = c * EL % SK;
        off[i] = (uint32_t)((min(row0 + r, rows - 1) - row0) * row_bytes) + kk[i] * ES + (part + c * EL / SK) * plane;
      } else {
        const int c = (lane % kChunks) ^ order(r);
        kk[i] = r % SK;
        off[i] = (uint32_t)(kk[i] * row_bytes) + (min(row0 + c * EL, rows - EL) - row0) * ES + (part + r / SK) * plane;
      }
    }
  }
  // `left`: k of this tile that exist.
  __device__ __forceinline__ void load(uint32_t lds, const char* base, const char* zeros, int wave, int left) const {
    if (left >= SK) {
#pragma unroll
      for (int i = 0; i < kPerWave; i++) dma16(lds + (wave * kPerWave + i) * 1024, base, off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kPerWave; i++)
        dma16(lds + (wave * kPerWave + i) * 1024, kk[i] < left ? base + off[i] : zeros);
    }
  }
  // The fragment of rows row + lane % 32, plane h: EL of k from kk + EL (lane / 32).
  static __device__ __forceinline__ s16x8 read(const char* l, int lane, int row, int h, int kk) {
    const int k = kParts == 1 ? h * SK + kk : kk;
    if (kParts > 1) l += h * kPart;
    if constexpr (ALONG_K) {
      const int r = row + (lane & 31), c = (k / EL + (lane >> 5)) ^ order(r);
      return *(const s16x8*)(l + r * (BK * ES) + c * 16);
    }
    if constexpr (ES == 4) {
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = *(const float*)(l + ((k + (lane >> 5) * 4 + j) * ROWS + row + (lane & 31)) * 4);
      return __builtin_bit_cast(s16x8, v);
    }
    const int p = lane & 15;
    const int at = (k + (lane >> 5) * 8 + (p >> 2)) * (ROWS * 2) +
                   ((row * 2 + ((lane >> 4) & 1) * 32 + (p & 3) * 8) ^ (order(p >> 2) << 4));
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(l + at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(l + at + 4 * ROWS * 2));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// A tile BM x BN, BK slots of contraction a stage (SK = BK / planes of k), NS stages of LDS, MW x NW waves, and
// NG such groups of waves: each takes every NG-th stage of the contraction, and
// their sums are added in order at the end. One group where the tiles fill the
// chip; several where they do not, so that a compute unit has other waves to
// run while one waits.
template <int BM_, int BN_, int BK_, int NS_, int MW_, int NW_, int NG_ = 1>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, NS = NS_, MW = MW_, NW = NW_, NG = NG_;
  static constexpr int kThreads = MW_ * NW_ * NG_ * 64;
};

// Bound by the matrix cores and the reads of LDS that feed them, which take
// about as long on 64 x 64 of a wave and two thirds on 128 x 64: 8192 x 8192 x
// 8192 bf16 903 us, 1217 TFLOP/s; 32768 x 1024 -> 4096 with GELU and residual
// 381 to 404 us (720 to 680 TFLOP/s) by card in a steady train of launches, 420
// after an idle moment and up to 480 in the first ten, where every 16 stages a
// tile's way out has the compute unit to itself.
// PL, PB: planes of A and of B.
template <class T, int PL, int PB, bool AK, bool BKD, class Shape, bool RAGGED, class Epi>
__global__ __launch_bounds__(Shape::kThreads, 2) void gemm_fast(FastArgs p, Epi epi) {
  constexpr int BM = Shape::BM, BN = Shape::BN, BK = Shape::BK, NS = Shape::NS, NG = Shape::NG;
  constexpr int NWAVE = Shape::MW * Shape::NW;
  constexpr int WM = BM / Shape::MW, WN = BN / Shape::NW, TM = WM / 32, TN = WN / 32, SK = BK / PL;
  using TA = FastTile<T, AK, BM, BK, NWAVE, PL>;
  using TB = FastTile<T, BKD, BN, SK * PB, NWAVE, PB>;
  constexpr int kOne = TA::kBytes + TB::kBytes, kStage = NG * kOne, kLoads = TA::kPerWave + TB::kPerWave;
  constexpr int kOutRow = WN + 4;  // floats of one staged output row
  constexpr int kOut = NG * NWAVE * 32 * kOutRow * 4;
  constexpr int kLds = NS * kStage > kOut ? NS * kStage : kOut;
  static_assert(kLds <= 160 * 1024, "the compute unit's LDS");
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  const int lane = threadIdx.x & 63;
  const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = NG == 1 ? 0 : all / NWAVE, wave = NG == 1 ? all : all % NWAVE;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + group * kOne;

  // Consecutive workgroups go to the eight dies in turn: each die takes a run of
  // tiles, and a run goes through groups of eight rows of tiles column by
  // column, so that what its tiles read meets in its L2.
  const int tiles = p.tiles_m * p.tiles_n;
  const int die = blockIdx.x & 7, per = tiles >> 3, rest = tiles & 7;
  const int tile = die * per + min(die, rest) + (blockIdx.x >> 3);
  const int band = tile / (8 * p.tiles_n), rows = min(8, p.tiles_m - band * 8), in = tile - band * 8 * p.tiles_n;
  const int m0 = (band * 8 + in % rows) * BM, n0 = in / rows * BN;
  const int q = blockIdx.y, split = blockIdx.z;
  const int k0 = split * p.k_split, k1 = min(p.k, k0 + p.k_split);

  TA ta;
  TB tb;
  ta.init(wave, lane, m0, p.a_rows, p.a_row, p.a_plane);
  tb.init(wave, lane, n0, p.b_rows, p.b_row, p.b_plane);
  constexpr int ES = sizeof(T);
  const int64_t a_step = AK ? ES : p.a_row, b_step = BKD ? ES : p.b_row;
  const char* ga = p.a + q * p.a_batch + (AK ? m0 * p.a_row : (int64_t)m0 * ES);
  const char* gb = p.b + q * p.b_batch + (BKD ? n0 * p.b_row : (int64_t)n0 * ES);

  // The groups take the stages in turn.
  const int total = (k1 - k0 + SK - 1) / SK, steps = (total + NG - 1) / NG;
  int k = k0 + group * SK;  // the next stage to load
  auto load = [&](uint32_t to) {
    if (NG > 1 && k >= k1) return;
    ta.load(to, ga + k * a_step, p.zeros, wave, k1 - k);
    tb.load(to + TA::kBytes, gb + k * b_step, p.zeros, wave, k1 - k);
    k += NG * SK;
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;

  const int wm = wave / Shape::NW * WM, wn = wave % Shape::NW * WN;
#pragma unroll
  for (int t = 0; t < NS - 1; t++)
    if (t < steps) load(base + t * kStage);
  int now = 0;
  // Waits for stage t: this wave's loads of it have landed (those of later
  // stages may be in flight; a group's last ones may be fewer, then all of them
  // are waited for) and its reads of the last one are done; past the barrier
  // that holds for every wave, and the last stage may be overwritten.
  auto arrive = [&](int t) {
    if (t + NS - 1 + (NG > 1) <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  auto compute = [&] {
    const char* l = lds + group * kOne + now;
    now = now == (NS - 1) * kStage ? 0 : now + kStage;
#pragma unroll
    for (int kk = 0; kk < SK; kk += Mfma<T>::kStep) {
      s16x8 fa[PL][TM], fb[PB][TN];
#pragma unroll
      for (int h = 0; h < PL; h++) {
#pragma unroll
        for (int i = 0; i < TM; i++) fa[h][i] = TA::read(l, lane, wm + i * 32, h, kk);
        if (h < PB) {
#pragma unroll
          for (int j = 0; j < TN; j++) fb[h][j] = TB::read(l + TA::kBytes, lane, wn + j * 32, h, kk);
        }
      }
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) {
          if constexpr (PL == 3) {
            acc[i][j] = Mfma<T>::run(fa[2][i], fb[0][j], acc[i][j]);
            acc[i][j] = Mfma<T>::run(fa[0][i], fb[2][j], acc[i][j]);
            acc[i][j] = Mfma<T>::run(fa[1][i], fb[1][j], acc[i][j]);
          }
          if constexpr (PL >= 2) {
            acc[i][j] = Mfma<T>::run(fa[1][i], fb[0][j], acc[i][j]);
            if constexpr (PB >= 2) acc[i][j] = Mfma<T>::run(fa[0][i], fb[1][j], acc[i][j]);
          }
          acc[i][j] = Mfma<T>::run(fa[0][i], fb[0][j], acc[i][j]);
        }
    }
  };
  for (int t = 0; t + 1 < steps; t++) {
    arrive(t);
    if (t + NS - 1 < steps) load(base + (now == 0 ? (NS - 1) * kStage : now - kStage));
    compute();
  }

  // What the epilogue reads is under way during the last stage: each lane's
  // eight columns of the first 32 rows of its wave's part.
  constexpr int kLanes = WN / 8, kRows = 64 / kLanes;  // lanes along a row, rows at once
  constexpr int kShare = 32 / NG;  // rows that a group puts out; where they are fewer than kRows, lanes idle
  constexpr int kPuts = kShare < kRows ? 1 : kShare / kRows;
  const int col = n0 + wn + (lane % kLanes) * 8;
  const int left = RAGGED ? min(8, p.n - col) : 8;
  const bool mine = kShare >= kRows || lane / kLanes < kShare;
  auto row_of = [&](int i, int r) { return m0 + wm + i * 32 + group * kShare + r * kRows + lane / kLanes; };
  typename Epi::Held held[2][kPuts];
  auto fetch = [&](int i) {
#pragma unroll
    for (int r = 0; r < kPuts; r++)
      if (mine && row_of(i, r) < p.m && col < p.n) epi.fetch(q, row_of(i, r), col, left, held[i & 1][r]);
  };
  typename Epi::Columns columns;
  arrive(steps - 1);
  if (col < p.n) epi.columns(col, left, columns);
  fetch(0);
  if (NG == 1 || (steps - 1) * NG + group < total) compute();  // a group may have no last stage

  // Out through LDS, 32 rows of a wave's part at a time, so that each lane
  // holds eight neighbouring columns: wide loads and stores, whole lines. The
  // groups' sums meet here, and each group puts out its share of the rows.
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  float* out = (float*)lds + wave * 32 * kOutRow;
  constexpr int kGroup = NWAVE * 32 * kOutRow;  // floats between groups
#pragma unroll
  for (int i = 0; i < TM; i++) {
    if (i + 1 < TM) fetch(i + 1);
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        out[group * kGroup + ((r >> 2) * 8 + (lane >> 5) * 4 + (r & 3)) * kOutRow + j * 32 + (lane & 31)] = acc[i][j][r];
    if (NG > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < kPuts; r++) {
      const int row = row_of(i, r);
      if (!mine || row >= p.m || col >= p.n) continue;
      float v[8];
      const float* s = out + (group * kShare + r * kRows + lane / kLanes) * kOutRow + (lane % kLanes) * 8;
      *(f32x4*)v = *(const f32x4*)s;
      *(f32x4*)(v + 4) = *(const f32x4*)(s + 4);
#pragma unroll
      for (int g = 1; g < NG; g++)
#pragma unroll
        for (int c = 0; c < 8; c++) v[c] += s[g * kGroup + c];
      if (!RAGGED || left == 8) epi.put8(q, split, row, col, 8, v, held[i & 1][r], columns);
      else epi.put8(q, split, row, col, left, v, held[i & 1][r], columns);
    }
    if (NG > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
  }
}

// ── which tile, and over how many splits of the contraction ─────────────────

template <class T, int PL> struct Tiles {
  typedef Tile<256, 256, 64, 2, 2, 4> Big;
  typedef Tile<128, 128, 64, 2, 2, 2, 2> Mid;
  typedef Tile<64, 64, 64, 4, 2, 2, 2> Deep;   // one a compute unit
  typedef Tile<64, 64, 64, 2, 2, 2, 2> Small;  // two
  typedef Tile<128, 128, 64, 2, 2, 2> Two;     // two
};
template <> struct Tiles<bf16, 3> {
  typedef Tile<256, 128, 96, 2, 4, 2> Big;
  typedef Tile<128, 128, 96, 3, 2, 2> Mid;
  typedef Tile<64, 64, 96, 3, 2, 2, 2> Deep;
  typedef Tile<64, 64, 96, 3, 2, 2> Small;
};
template <> struct Tiles<float, 1> {
  typedef Tile<64, 64, 32, 2, 2, 2, 2> Deep;
  typedef Tile<64, 64, 32, 2, 2, 2> Small;  // four
};

// plan_fast's names for f32 operands as they are, and for two planes by one.
enum { PLANES_F32 = 0, PLANES_2BY1 = 21 };

struct FastPlan {
  int tile;  // 0 big, 1 mid, 2 deep, 3 small, 4 two
  int32_t splits, k_split;
  uint64_t part_bytes;  // workspace for the splits' sums
};

// The least of an estimate: rounds of workgroups over the chip, times the
// stages of a workgroup's contraction at the tile's measured time, and for a
// split contraction the sums' way through memory. One MI355X, bf16, us:
//
//                         256x256  128x128  128x128g2  64x64g2  64x64g2  library
//                         one a CU two      one        one      two
//   8192 x 8192 x 8192    903      1023     .          .        .        860
//   4096 x 4096 x 1024    36.7     38.3     .          .        .        29.8
//   8192 x 1000 x 1000    .        24.2     28.1       51.4     40.7     .
//   2048 x 2048 x 2048    51.6     24.6     21.9       36.6     28.6     21.9
//   1024 x 4096 x 1024    28.1     13.4     12.9       21.7     16.6     14.0
//   1024 x 1024 x 4096    91.2     40.8     33.8       17.8     23.0     19.3
//   1024 x 1024 x 1024    27.1     11.6     11.1       6.4      6.4      8.3
//   512 x 512 x 2048      47.4     .        19.2       10.9     10.8     7.4
//   4096 x 256 x 256      11.0     .        6.1        4.4      4.3      6.1
//
// Large tiles read LDS and L2 least for each product and win where there are
// enough of them; below, what counts is that every compute unit has one. f32
// products are bound by their instructions and take small tiles throughout
// (4096 x 2048 x 2048: 64x64 four a CU 265, 128x128 273; 1024 x 1024 x 1024:
// 64x64g2 21, 128x128 66). Two planes by one, linear layers' dx with their dz (21
// us of it), 256x256 / 128x128g2 / 128x128: 8191 x 1000 -> 1001 77 / 77 / 68, 4096
// x 2048 -> 2048 107 / 98 / 83, 16384 x 1024 -> 1024 95 / 116 / 103.
inline FastPlan plan_fast(const phz_ops* o, int64_t m, int64_t n, int64_t k, int64_t batch, int planes, bool may_split) {
  // Time of a stage of 64 (of 32 for two and three planes, and for f32) with
  // one workgroup a compute unit, and with all that fit.
  struct Kind { int bm, bn, per_cu; double alone, full; };
  const Kind one[5] = {{256, 256, 1, 1.7, 1.7}, {128, 128, 1, 0.6, 0.6}, {64, 64, 1, 0.24, 0.24}, {64, 64, 2, 0.32, 0.42},
                       {128, 128, 2, 0.68, 1.3}};
  const Kind two_by_one[5] = {{256, 256, 1, 1.6, 1.6}, {128, 128, 1, 0.62, 0.62}, {64, 64, 1, 0.24, 0.24}, {64, 64, 2, 0.32, 0.44},
                              {128, 128, 2, 0.8, 1.05}};
  const Kind three[4] = {{256, 128, 1, 2.8, 2.8}, {128, 128, 1, 1.5, 1.5}, {64, 64, 1, 0.45, 0.45}, {64, 64, 2, 0.6, 0.8}};
  const Kind f32[4] = {{}, {}, {64, 64, 1, 0.57, 0.57}, {64, 64, 4, 0.6, 2.0}};
  const Kind* kinds = planes == 3 ? three : planes == PLANES_F32 ? f32 : planes == PLANES_2BY1 ? two_by_one : one;
  const int64_t sk = planes == 1 ? 64 : 32, stages = std::max<int64_t>(1, ceil_div(k, sk));
  FastPlan best{};
  double least = 1e30;
  for (int t = planes == PLANES_F32 ? 2 : 0; t < (kinds == three || kinds == f32 ? 4 : 5); t++) {
    const Kind& kind = kinds[t];
    const int64_t tiles = ceil_div(m, kind.bm) * ceil_div(n, kind.bn) * batch;
    for (int64_t splits = 1; splits <= (may_split ? 64 : 1); splits *= 2) {
      if (splits > 1 && stages < 8 * splits) break;
      const int64_t rounds = ceil_div(tiles * splits, (int64_t)o->cus * kind.per_cu);
      const int64_t beside = std::min<int64_t>(kind.per_cu, ceil_div(tiles * splits, o->cus));
      const double stage =
          kind.per_cu == 1 ? kind.full : kind.alone + (kind.full - kind.alone) * (beside - 1) / (kind.per_cu - 1);
      double us = rounds * (3.0 + ceil_div(stages, splits) * stage);
      if (splits > 1) us += 3.0 + 0.1 * splits + (2.0 * splits + 1) * m * n * batch * 4 / 8e6;  // sums stay in the caches
      if (us < least) {
        least = us;
        best.tile = t;
        best.splits = (int32_t)splits;
      }
    }
  }
  const int64_t per = ceil_div(ceil_div(k, best.splits), 64) * 64;
  best.k_split = (int32_t)std::max<int64_t>(64, per);
  best.splits = (int32_t)std::max<int64_t>(1, ceil_div(k, best.k_split));
  best.part_bytes = best.splits > 1 ? (uint64_t)best.splits * batch * m * ((n + 7) / 8 * 8) * 4 : 0;
  return best;
}

// Sums of one split, joined by join_kernel, in rows of whole eights.
struct PartOut : NothingAhead {
  static constexpr bool kRagged = false;
  float* part;
  int64_t row, batch, split;
  PartOut(float* p, int64_t r, int64_t b, int64_t s) : part(p), row(r), batch(b), split(s) {}
  __device__ __forceinline__ void put8(int q, int s, int i, int j, int, const float* sums, const Held&, const Columns&) const {
    float* at = part + s * split + q * batch + i * row + j;
    *(f32x4*)at = *(const f32x4*)sums;
    *(f32x4*)(at + 4) = *(const f32x4*)(sums + 4);
  }
  __device__ __forceinline__ void put1(int q, int s, int i, int j, float sum) const {
    part[s * split + q * batch + i * row + j] = sum;
  }
};

// What a join's first blocks may do beside it, to save a launch.
struct NothingBeside {
  static constexpr unsigned blocks = 0;
  __device__ __forceinline__ void run(unsigned) const {}
};

// The splits' sums to the epilogue, added in a fixed order: four threads for
// eight elements, each every fourth split.
template <class Epi, class Beside>
__global__ __launch_bounds__(256) void join_kernel(PartOut p, int splits, int32_t m, int32_t n, Epi epi, Beside beside) {
  if (blockIdx.x < beside.blocks) return beside.run(blockIdx.x);
  __shared__ float s[3][64][9];
  const uint32_t per = (n + 7) / 8;
  const int q = blockIdx.y, unit = threadIdx.x & 63, lane = threadIdx.x >> 6;
  const int64_t stride = (int64_t)(gridDim.x - beside.blocks) * 64;
  for (int64_t t0 = (int64_t)(blockIdx.x - beside.blocks) * 64; t0 < (int64_t)m * per; t0 += stride) {
    const int64_t t = t0 + unit;
    const bool live = t < (int64_t)m * per;
    const int i = live ? (int)(t / per) : 0, j = live ? (int)(t - (int64_t)i * per) * 8 : 0;
    const float* at = p.part + q * p.batch + i * p.row + j;
    typename Epi::Held held;
    typename Epi::Columns columns;
    if (live && lane == 0) epi.fetch(q, i, j, min(8, n - j), held), epi.columns(j, min(8, n - j), columns);
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = 0.0f;
#pragma unroll 4
    for (int k = lane; k < splits; k += 4) {
      const f32x4 lo = *(const f32x4*)(at + k * p.split), hi = *(const f32x4*)(at + k * p.split + 4);
#pragma unroll
      for (int c = 0; c < 4; c++) v[c] += lo[c], v[4 + c] += hi[c];
    }
    if (lane) {
#pragma unroll
      for (int c = 0; c < 8; c++) s[lane - 1][unit][c] = v[c];
    }
    __syncthreads();
    if (lane == 0 && live) {
#pragma unroll
      for (int l = 0; l < 3; l++)
#pragma unroll
        for (int c = 0; c < 8; c++) v[c] += s[l][unit][c];
      if (j + 8 <= n) epi.put8(q, 0, i, j, 8, v, held, columns);
      else epi.put8(q, 0, i, j, n - j, v, held, columns);
    }
    __syncthreads();
  }
}

template <class Epi, class Beside>
void launch_join(hipStream_t stream, const PartOut& sums, int batch, int splits, int32_t m, int32_t n, const Epi& epi,
                 const Beside& beside) {
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div((int64_t)m * ((n + 7) / 8), 64), 8192);
  hipLaunchKernelGGL((join_kernel<Epi, Beside>), dim3(beside.blocks + blocks, (unsigned)batch), dim3(256), 0, stream, sums,
                     splits, m, n, epi, beside);
}

// `part`: plan.part_bytes of workspace. `beside` goes with the join: to plans
// with splits, and one matrix, only.
template <class T, int PL, bool AK, bool BKD, int PB = PL, class Epi, class Beside = NothingBeside>
void launch_gemm_fast(const phz_ops* o, hipStream_t stream, FastArgs p, int batch, const FastPlan& plan, float* part,
                      const Epi& epi, const Beside& beside = {}) {
  p.zeros = (const char*)o->zeros;
  p.splits = plan.splits;
  p.k_split = plan.k_split;
  const PartOut sums{part, (p.n + 7) / 8 * 8, (int64_t)p.m * ((p.n + 7) / 8 * 8),
                     (int64_t)batch * p.m * ((p.n + 7) / 8 * 8)};
  auto go = [&](auto shape) {
    using S = decltype(shape);
    p.tiles_m = (int32_t)ceil_div(p.m, S::BM);
    p.tiles_n = (int32_t)ceil_div(p.n, S::BN);
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)batch, (unsigned)p.splits);
    const dim3 block(S::kThreads);
    if (p.splits > 1) {
      hipLaunchKernelGGL((gemm_fast<T, PL, PB, AK, BKD, S, false, PartOut>), grid, block, 0, stream, p, sums);
      return;
    }
    if constexpr (Epi::kRagged) {
      if (p.n % 8) {
        hipLaunchKernelGGL((gemm_fast<T, PL, PB, AK, BKD, S, true, Epi>), grid, block, 0, stream, p, epi);
        return;
      }
    }
    hipLaunchKernelGGL((gemm_fast<T, PL, PB, AK, BKD, S, false, Epi>), grid, block, 0, stream, p, epi);
  };
  if constexpr (sizeof(T) == 2) {
    if (plan.tile == 0) go(typename Tiles<T, PL>::Big{});
    if (plan.tile == 1) go(typename Tiles<T, PL>::Mid{});
  }
  if constexpr (sizeof(T) == 2 && PL < 3) {
    if (plan.tile == 4) go(typename Tiles<T, PL>::Two{});
  }
  if (plan.tile == 2) go(typename Tiles<T, PL>::Deep{});
  if (plan.tile == 3) go(typename Tiles<T, PL>::Small{});
  if (p.splits > 1) launch_join(stream, sums, batch, p.splits, p.m, p.n, epi, beside);
}

// gemm_any's contraction in splits where its tiles are few: a stage of tile_k
// takes about 1.1 us alone, a join 4, so splits keep at least four stages, and
// there are at most two workgroups a compute unit.
struct AnyPlan {
  int32_t splits, k_split;
  uint64_t part_bytes;
};
template <class E>
AnyPlan plan_any(const phz_ops* o, int64_t m, int64_t n, int64_t k) {
  const int64_t bk = Any<E>::tile_k, stages = ceil_div(k, bk), tiles = ceil_div(m, 64) * ceil_div(n, 64);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(ceil_div(2 * o->cus, tiles), stages / 4));
  AnyPlan p{};
  p.k_split = (int32_t)(std::max<int64_t>(1, ceil_div(stages, want)) * bk);
  p.splits = (int32_t)std::max<int64_t>(1, ceil_div(k, p.k_split));
  p.part_bytes = p.splits > 1 ? (uint64_t)p.splits * m * ((n + 7) / 8 * 8) * 4 : 0;
  return p;
}
template <class E, bool AK, bool BKD, int PA = 1, class Epi, class Beside = NothingBeside>
void launch_any(const phz_ops* o, hipStream_t stream, Operand a, Operand b, int64_t m, int64_t n, int64_t k,
                const AnyPlan& plan, float* part, const Epi& epi, const Beside& beside = {}) {
  const GemmShape s{(int32_t)m, (int32_t)n, (int32_t)k, plan.k_split, plan.splits};
  if (plan.splits == 1) return launch_gemm_any<E, AK, BKD, PA>(o, stream, a, b, s, 1, epi);
  const int64_t row = (n + 7) / 8 * 8;
  const PartOut sums{part, row, m * row, m * row};
  launch_gemm_any<E, AK, BKD, PA>(o, stream, a, b, s, 1, sums);
  launch_join(stream, sums, 1, plan.splits, s.m, s.n, epi, beside);
}

}  // namespace phzop
