// phz_gemm_fast.h — the matrix product for large aligned operands of 16 bits:
//
//   C[i][j] = sum_k A(i, k) B(j, k)
//
// Operands are one plane of 16-bit elements, or two: A = hi + lo, f32 data cut
// in f16, whose product is taken as lo hi + hi lo + hi hi (lo lo is below what
// f32 sums hold). Rows are 16-byte aligned and, along k (or along rows, for
// operands dense along rows), a multiple of eight elements long or padded with
// zeros to one.
#pragma once
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

template <class T> struct Mfma;
template <> struct Mfma<bf16> {
  static __device__ __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mfma<half_t> {
  static __device__ __forceinline__ f32x16 run(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

struct FastArgs {
  const char *a, *b, *zeros;
  int64_t a_row, b_row, a_batch, b_batch;  // bytes
  uint32_t a_plane, b_plane;               // bytes from hi to lo
  int32_t m, n, k;
  int32_t a_rows, b_rows;   // rows that exist (dense along rows: a multiple of eight)
  int32_t k_split, splits;  // contraction per split, a multiple of 64
  int32_t tiles_m, tiles_n;
};

// 16 bytes a lane from global memory to LDS at `lds` + 16 lane, without passing
// registers. Written as asm so that the compiler does not wait for it at the
// next LDS read: the loop below waits for a stage's loads itself. There is no
// output register; the wait state is the one that a write of m0 needs.
__device__ __forceinline__ void dma16(uint32_t lds, const char* base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base)
               : "memory");
}
__device__ __forceinline__ void dma16(uint32_t lds, const char* at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(at) : "memory");
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
// With two planes the tile holds SK = BK / 2 of k twice: hi's, then lo's.
template <bool ALONG_K, int ROWS, int BK, int NW, int PL>
struct FastTile {
  static constexpr int SK = BK / PL;
  static constexpr int kBytes = ROWS * BK * 2;
  static constexpr int kPerWave = kBytes / 1024 / NW;  // 1 KB loads of each wave
  static constexpr int kChunks = ALONG_K ? BK / 8 : ROWS / 8, kRows = 64 / kChunks;  // 16-byte chunks of a row, rows of a load
  static_assert(kPerWave * NW * 1024 == kBytes, "whole loads for every wave");
  uint32_t off[kPerWave];
  int32_t kk[kPerWave];  // first k of the lane's 16 bytes within the tile

  // What the row r's (k's) chunks are permuted by.
  static __device__ __forceinline__ int order(int r) {
    if (ALONG_K) return BK == 32 ? (r >> 2) & 3 : (r >> 1) & 7;
    return (ROWS == 64 ? (r >> 1) & 1 : r & 3) << 2;
  }

  __device__ __forceinline__ void init(int wave, int lane, int row0, int rows, int64_t row_bytes, uint32_t plane) {
#pragma unroll
    for (int i = 0; i < kPerWave; i++) {
      const int r = (wave * kPerWave + i) * kRows + lane / kChunks;
      if (ALONG_K) {
        const int c = (lane % kChunks) ^ order(r);
        // Rows past the end repeat the last one: their sums are not stored.
        kk[i] = c * 8 % SK;
        off[i] = (uint32_t)((min(row0 + r, rows - 1) - row0) * row_bytes) + kk[i] * 2 + (c * 8 / SK) * plane;
      } else {
        const int c = (lane % kChunks) ^ order(r);
        kk[i] = r % SK;
        off[i] = (uint32_t)(kk[i] * row_bytes) + (min(row0 + c * 8, rows - 8) - row0) * 2 + (r / SK) * plane;
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
  // The fragment of rows row + lane % 32, the tile's k from k + 8 (lane / 32).
  static __device__ __forceinline__ s16x8 read(const char* l, int lane, int row, int k) {
    if constexpr (ALONG_K) {
      const int r = row + (lane & 31), c = ((k >> 3) + (lane >> 5)) ^ order(r);
      return *(const s16x8*)(l + r * (BK * 2) + c * 16);
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

// A tile BM x BN, contraction BK a stage, NS stages of LDS, MW x NW waves, and
// NG such groups of waves: each takes every NG-th stage of the contraction, and
// their sums are added in order at the end. One group where the tiles fill the
// chip; several where they do not, so that a compute unit has other waves to
// run while one waits.
template <int BM_, int BN_, int BK_, int NS_, int MW_, int NW_, int NG_ = 1>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, NS = NS_, MW = MW_, NW = NW_, NG = NG_;
  static constexpr int kThreads = MW_ * NW_ * NG_ * 64;
};

template <class T, int PL, bool AK, bool BKD, class Shape, class Epi>
__global__ __launch_bounds__(Shape::kThreads, 2) void gemm_fast(FastArgs p, Epi epi) {
  constexpr int BM = Shape::BM, BN = Shape::BN, BK = Shape::BK, NS = Shape::NS, NG = Shape::NG;
  constexpr int NWAVE = Shape::MW * Shape::NW;
  constexpr int WM = BM / Shape::MW, WN = BN / Shape::NW, TM = WM / 32, TN = WN / 32, SK = BK / PL;
  using TA = FastTile<AK, BM, BK, NWAVE, PL>;
  using TB = FastTile<BKD, BN, BK, NWAVE, PL>;
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
  const int64_t a_step = AK ? 2 : p.a_row, b_step = BKD ? 2 : p.b_row;
  const char* ga = p.a + q * p.a_batch + (AK ? m0 * p.a_row : (int64_t)m0 * 2);
  const char* gb = p.b + q * p.b_batch + (BKD ? n0 * p.b_row : (int64_t)n0 * 2);

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
  for (int t = 0; t < steps; t++) {
    // This wave's loads of this stage have landed (those of later stages may be
    // in flight; a group's last ones may be fewer, then all of them are waited
    // for) and its reads of the last one are done; past the barrier that holds
    // for every wave, and the last stage may be overwritten.
    if (t + NS - 1 + (NG > 1) <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + NS - 1 < steps) load(base + (now == 0 ? (NS - 1) * kStage : now - kStage));
    if (NG > 1 && t * NG + group >= total) continue;  // no stage is left for this group
    const char* l = lds + group * kOne + now;
    now = now == (NS - 1) * kStage ? 0 : now + kStage;
#pragma unroll
    for (int kk = 0; kk < SK; kk += 16) {
      s16x8 fa[PL][TM], fb[PL][TN];
#pragma unroll
      for (int h = 0; h < PL; h++) {
#pragma unroll
        for (int i = 0; i < TM; i++) fa[h][i] = TA::read(l, lane, wm + i * 32, h * SK + kk);
#pragma unroll
        for (int j = 0; j < TN; j++) fb[h][j] = TB::read(l + TA::kBytes, lane, wn + j * 32, h * SK + kk);
      }
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) {
          if constexpr (PL == 2) {
            acc[i][j] = Mfma<T>::run(fa[1][i], fb[0][j], acc[i][j]);
            acc[i][j] = Mfma<T>::run(fa[0][i], fb[1][j], acc[i][j]);
          }
          acc[i][j] = Mfma<T>::run(fa[0][i], fb[0][j], acc[i][j]);
        }
    }
  }

  // Out through LDS, 32 rows of a wave's part at a time, so that each lane
  // holds eight neighbouring columns: wide loads and stores, whole lines. The
  // groups' sums meet here, and each group puts out its share of the rows.
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  float* out = (float*)lds + wave * 32 * kOutRow;
  constexpr int kGroup = NWAVE * 32 * kOutRow;       // floats between groups
  constexpr int kLanes = WN / 8, kRows = 64 / kLanes;  // lanes along a row, rows at once
  constexpr int kShare = 32 / NG;  // rows that a group puts out; where they are fewer than kRows, lanes idle
  const int col = n0 + wn + (lane % kLanes) * 8;
#pragma unroll
  for (int i = 0; i < TM; i++) {
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        out[group * kGroup + ((r >> 2) * 8 + (lane >> 5) * 4 + (r & 3)) * kOutRow + j * 32 + (lane & 31)] = acc[i][j][r];
    if (NG > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r0 = 0; r0 < kShare; r0 += kRows) {
      if (kShare < kRows && lane / kLanes >= kShare) break;
      const int r = group * kShare + r0 + lane / kLanes, row = m0 + wm + i * 32 + r;
      float v[8];
      const float* s = out + r * kOutRow + (lane % kLanes) * 8;
      *(f32x4*)v = *(const f32x4*)s;
      *(f32x4*)(v + 4) = *(const f32x4*)(s + 4);
#pragma unroll
      for (int g = 1; g < NG; g++)
#pragma unroll
        for (int c = 0; c < 8; c++) v[c] += s[g * kGroup + c];
      if (row < p.m) {
        if (col + 8 <= p.n) epi.template put<8>(q, split, row, col, v);
        else
          for (int c = 0; c < 8 && col + c < p.n; c++) epi.template put<1>(q, split, row, col + c, v + c);
      }
    }
    if (NG > 1) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
  }
}

// The four tiles and when each is taken, for `tiles` of its size over all
// batches and splits (one MI355X, bf16, us; torch's library beside them):
//
//                         256x256  128x128  128x128g2  64x64g2  64x64g2  library
//                         8 waves  2 a CU   1 a CU     1 a CU   2 a CU
//   8192 x 8192 x 8192    903      1023     .          .        .        860
//   4096 x 4096 x 1024    36.7     38.3     .          .        .        29.8
//   2048 x 2048 x 2048    51.6     26.9     23.9       42.9     30.3     21.9
//   1024 x 4096 x 1024    28.1     15.0     14.2       25.4     18.4     14.0
//   1500 x 1000 x 3000    78.1     40.8     36.8       31.3     26.6     26.6
//   1024 x 1024 x 4096    91.2     44.1     36.5       21.1     26.3     19.3
//   512 x 512 x 2048      47.4     21.9     19.2       10.9     10.8     7.4
//   4096 x 256 x 256      11.0     6.2      6.1        4.4      4.3      6.1
//
// Large tiles read LDS and L2 least for each product and win where there are
// enough of them; below, what counts is that every compute unit has one.
typedef Tile<256, 256, 64, 2, 2, 4> TileBig;
typedef Tile<128, 128, 64, 2, 2, 2, 2> TileMid;
typedef Tile<64, 64, 64, 4, 2, 2, 2> TileDeep;
typedef Tile<64, 64, 64, 2, 2, 2, 2> TileSmall;

template <class T, int PL, bool AK, bool BKD, class Epi>
void launch_gemm_fast(const phz_ops* o, hipStream_t stream, FastArgs p, int batch, const Epi& epi) {
  p.zeros = (const char*)o->zeros;
  const int64_t z = (int64_t)batch * p.splits;
  auto tiles = [&](int bm, int bn) { return ceil_div(p.m, bm) * ceil_div(p.n, bn) * z; };
  auto go = [&](auto shape) {
    using S = decltype(shape);
    p.tiles_m = (int32_t)ceil_div(p.m, S::BM);
    p.tiles_n = (int32_t)ceil_div(p.n, S::BN);
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)batch, (unsigned)p.splits);
    hipLaunchKernelGGL((gemm_fast<T, PL, AK, BKD, S, Epi>), grid, dim3(S::kThreads), 0, stream, p, epi);
  };
  if (tiles(256, 256) >= o->cus) go(TileBig{});
  else if (tiles(128, 128) >= o->cus * 3 / 4) go(TileMid{});
  else if (tiles(64, 64) <= o->cus) go(TileDeep{});
  else go(TileSmall{});
}

}  // namespace phzop
