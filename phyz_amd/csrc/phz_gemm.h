// phz_gemm.h — the matrix product under the linear layer and Newton-Schulz:
//
//   C[i][j] = sum_k A(i, k) B(j, k)
//
// on the matrix cores, each operand dense along k or along its rows, at any
// size, stride and alignment.
//
// bf16 operands take the bf16 matrix instructions, f32 operands the f32 ones,
// whose products are exact: the path for small sizes, any layout and any value.
// Sums are f32. (Large f32 products are faster cut in bf16 pieces, see cut3 and
// phz_gemm_fast.h: the f32 instructions have a sixteenth of the bf16 rate.)
#pragma once
#include "phz_ops.h"

namespace phzop {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Element (i, k) of an operand, batch q: data + q batch + i row + k, or, dense
// along rows, data + q batch + k row + i.
struct Operand {
  const void* data;
  int64_t row, batch;
  int64_t plane;  // of A, where it is the sum of two planes
};

struct GemmShape {
  int32_t m, n, k;
  int32_t k_split;  // contraction per split, a multiple of the k tile
  int32_t splits;
};

// Contraction per tile, and elements between a tile's rows in LDS: four or
// eight more than it, so that the 16-byte reads of 16 consecutive rows fall
// into all 64 banks.
template <class E> struct Any;
template <> struct Any<bf16> { static constexpr int tile_k = 64, ld = 72; };
template <> struct Any<float> { static constexpr int tile_k = 32, ld = 36; };

// x = h + m + l in bf16 pieces, each the nearest to what the ones before leave
// (h cut off where the nearest is infinite). For |x| in [2^e, 2^(e+1)) what h
// leaves is at most 2^(e-8) and a multiple of 2^(e-23), what m leaves at most
// 2^(e-17): seven bits, so the cut is exact (from 2^-110 on; a smaller x loses
// what is below bf16's least, 2^-133). Of the nine products of two numbers'
// pieces the six largest are taken (hh, hm, mh, mm, hl, lh); what is left out,
// ml + lm + ll, is at most 2^-24 (1 + 2^-9) of |a||b|, of either sign: no more
// than one rounding to f32. Six products of the bf16 rate are 2.7 times the rate
// of the f32 matrix instructions.
//
// The three pieces of x. One that is not finite is (+-1, 0, x): the last piece
// meets only the other operand's first one, which is 0 where the operand is, so
// every product is what f32 makes of it: infinity times a number that infinity,
// times 0 NaN, times infinity (h l and l h) theirs.
__device__ __forceinline__ void cut3(float x, uint16_t& h, uint16_t& m, uint16_t& l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  if ((b & 0x7f800000u) == 0x7f800000u) {
    h = (uint16_t)((b >> 16 & 0x8000u) | 0x3f80u), m = 0;
    l = (uint16_t)(b & 0x007fffffu ? 0x7fc0u : b >> 16);
    return;
  }
  bf16 p = from_f32<bf16>(x);
  if ((p.bits & 0x7f80u) == 0x7f80u) p.bits = (uint16_t)(b >> 16);
  const float r = x - to_f32(p);
  const bf16 q = from_f32<bf16>(r);
  h = p.bits, m = q.bits, l = from_f32<bf16>(r - to_f32(q)).bits;
}

// v = hi + lo to 2^-16 of itself, of one sign: hi v's first eight bits, lo the
// nearest to the rest. lo is never 0 beside a number hi (2^-30 of it instead, or
// 1 beside infinity), so that infinity times v is infinity in both products.
__device__ __forceinline__ void cut2(float v, bf16& hi, bf16& lo) {
  hi.bits = (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16);
  const float h = to_f32(hi);
  if (v != v) hi.bits = 0x7fc0u;
  const float rest = fabsf(h) < __builtin_inff() ? v - h : copysignf(1.0f, h);
  lo = from_f32<bf16>(rest != 0.0f ? rest : h * 0x1p-30f);
}

// Moves one operand's tile of ROWS rows by tile_k through registers into LDS,
// laid out [row][k]. A chunk is eight k of one row (dense along k), or of R
// rows (dense along rows: then a wave's loads are contiguous along rows, and
// the transpose is done in registers).
template <class E, bool ALONG_K, int ROWS>
struct Stage {
  static constexpr int BK = Any<E>::tile_k, LD = Any<E>::ld, KC = BK / 8;
  static constexpr int R = ALONG_K ? 1 : (int)(4 / sizeof(E));
  static constexpr int kChunks = ROWS / R * KC, N = kChunks / 256;
  static_assert(kChunks % 256 == 0, "whole chunks for every thread");
  E v[N][R][8];

  __device__ __forceinline__ static void place(int c, int& row, int& k) {
    if (ALONG_K) row = c / KC, k = c % KC * 8;
    else row = c % (ROWS / R) * R, k = c / (ROWS / R) * 8;
  }
  __device__ __forceinline__ void load(const E* base, int64_t ld, int row0, int rows, int k0, int k_end) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      int row, k;
      place(threadIdx.x + i * 256, row, k);
      row += row0;
      k += k0;
      if (ALONG_K) {
        if (row < rows && k + 8 <= k_end) {
          const Pack<E, 8> p = *(const Pack<E, 8>*)(base + row * ld + k);
#pragma unroll
          for (int j = 0; j < 8; j++) v[i][0][j] = p.v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) v[i][0][j] = row < rows && k + j < k_end ? base[row * ld + k + j] : E{};
        }
      } else if (row + R <= rows && k + 8 <= k_end) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const Pack<E, R> p = *(const Pack<E, R>*)(base + (int64_t)(k + j) * ld + row);
#pragma unroll
          for (int r = 0; r < R; r++) v[i][r][j] = p.v[r];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
          for (int r = 0; r < R; r++)
            v[i][r][j] = row + r < rows && k + j < k_end ? base[(int64_t)(k + j) * ld + row + r] : E{};
      }
    }
  }
  __device__ __forceinline__ void store(E* lds) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      int row, k;
      place(threadIdx.x + i * 256, row, k);
#pragma unroll
      for (int r = 0; r < R; r++) {
        E* to = lds + (row + r) * LD + k;
        if constexpr (sizeof(E) == 2) {
          u32x4 q;
#pragma unroll
          for (int j = 0; j < 4; j++) q[j] = (uint32_t)v[i][r][2 * j].bits | (uint32_t)v[i][r][2 * j + 1].bits << 16;
          *(u32x4*)to = q;
        } else {
#pragma unroll
          for (int j = 0; j < 8; j += 4) *(f32x4*)(to + j) = f32x4{v[i][r][j], v[i][r][j + 1], v[i][r][j + 2], v[i][r][j + 3]};
        }
      }
    }
  }
};

// What a lane takes of 32 rows in one 16-byte read, and the products of it:
// bf16, 16 of k in one instruction; f32, eight of k in four, where an
// instruction pairs the k of lanes below 32 with that four further on. Both
// operands pair alike, so the sum is the same.
__device__ __forceinline__ f32x16 multiply(const bf16* a, const bf16* b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)a, *(const bf16x8*)b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply(const float* a, const float* b, f32x16 c) {
  const f32x4 x = *(const f32x4*)a, y = *(const f32x4*)b;
#pragma unroll
  for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
  return c;
}

// Eight elements, or the first `left` of them.
template <class E>
__device__ __forceinline__ void load_some(Pack<E, 8>& to, const E* p, int left) {
  if (left >= 8) {
    to = *(const Pack<E, 8>*)p;
  } else {
#pragma unroll
    for (int c = 0; c < 8; c++) to.v[c] = c < left ? p[c] : E{};
  }
}
template <class E>
__device__ __forceinline__ void store_some(E* p, const Pack<E, 8>& from, int left) {
  if (left >= 8) {
    *(Pack<E, 8>*)p = from;
  } else {
#pragma unroll
    for (int c = 0; c < 8; c++)
      if (c < left) p[c] = from.v[c];
  }
}

// Any size and layout: a workgroup of four waves per BM x BN tile, registers
// holding the next k tile while the matrix cores work on the one in LDS. Bound
// by the latency of a stage (about 1.1 us with a workgroup or two a compute
// unit): for small calls and odd rows. 4096 x 55 -> 256 f32 6.4 us.
//
// An epilogue has
//   Columns, columns(j, left, c)                what it reads for eight columns, once
//   Held, fetch(q, i, j, left, held)            what it reads for eight elements, ahead
//   put8(q, split, i, j, left, sums, held, c)   eight neighbouring sums of row i
//   kRagged                                     whether rows may end inside eight
// of which, at a ragged end, only the first `left` exist; else that is the
// constant 8. RAGGED is a kernel of its own: its single accesses, all on their
// way together, take registers that whole rows would miss (32768 x 1024 -> 4096
// bf16 388 us, 412 with both in one), and one at a time, after each other, cost
// a load's latency each (54038 x 252 -> 135: 73 us, so 49).
//
// PA: planes of A, both in a stage.
template <class E, bool AK, bool BKD, int PA, int BM, int BN, bool RAGGED, class Epi>
__global__ __launch_bounds__(256) void gemm_any(Operand a, Operand b, GemmShape s, Epi epi) {
  constexpr int BK = Any<E>::tile_k, LD = Any<E>::ld, PER = 16 / sizeof(E);
  constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 32, TN = WN / 32;
  using SA = Stage<E, AK, BM>;
  using SB = Stage<E, BKD, BN>;
  constexpr int kOutRow = WN + 4;  // floats of one staged output row
  static_assert(4 * 32 * kOutRow * 4 <= (BM + BN) * LD * (int)sizeof(E), "output rows fit the tiles");
  __shared__ __attribute__((aligned(16))) E la[(PA * BM + BN) * LD];
  E* lb = la + PA * BM * LD;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  const int q = blockIdx.z / s.splits, split = blockIdx.z - q * s.splits;
  const int k0 = split * s.k_split, k_end = min(s.k, k0 + s.k_split);
  const E* pa = (const E*)a.data + q * a.batch;
  const E* pb = (const E*)b.data + q * b.batch;
  const int wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
  const int fr = lane & 31, fk = (lane >> 5) * PER;

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
  SA sa[PA];
  SB sb;
  auto load = [&](int k) {
#pragma unroll
    for (int h = 0; h < PA; h++) sa[h].load(h ? pa + a.plane : pa, a.row, m0, s.m, k, k_end);
    sb.load(pb, b.row, n0, s.n, k, k_end);
  };
  load(k0);
  for (int k = k0; k < k_end; k += BK) {
    __syncthreads();
#pragma unroll
    for (int h = 0; h < PA; h++) sa[h].store(la + h * BM * LD);
    sb.store(lb);
    __syncthreads();
    if (k + BK < k_end) load(k + BK);
#pragma unroll
    for (int kk = 0; kk < BK; kk += 2 * PER)
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
          for (int h = PA - 1; h >= 0; h--)
            acc[i][j] = multiply(la + (h * BM + wm + i * 32 + fr) * LD + kk + fk, lb + (wn + j * 32 + fr) * LD + kk + fk, acc[i][j]);
  }

  // Out through LDS, 32 rows of a wave's part at a time, so that each lane
  // holds eight neighbouring columns. Accumulator layout: register r of a lane
  // is row (r / 4) 8 + (lane / 32) 4 + r % 4, column lane % 32 of its block.
  __syncthreads();
  float* out = (float*)la + wave * 32 * kOutRow;
  constexpr int kLanes = WN / 8, kRows = 64 / kLanes, kPuts = 32 / kRows;
  const int col = n0 + wn + (lane % kLanes) * 8;
  typename Epi::Columns columns;
  const int left = RAGGED ? min(8, s.n - col) : 8;
  if (col < s.n) epi.columns(col, left, columns);
#pragma unroll
  for (int i = 0; i < TM; i++) {
    typename Epi::Held held[kPuts];
#pragma unroll
    for (int r = 0; r < kPuts; r++) {
      const int row = m0 + wm + i * 32 + r * kRows + lane / kLanes;
      if (row < s.m && col < s.n) epi.fetch(q, row, col, left, held[r]);
    }
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        out[((r >> 2) * 8 + (lane >> 5) * 4 + (r & 3)) * kOutRow + j * 32 + fr] = acc[i][j][r];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < kPuts; r++) {
      const int row = m0 + wm + i * 32 + r * kRows + lane / kLanes;
      float v[8];
      const float* p = out + (r * kRows + lane / kLanes) * kOutRow + (lane % kLanes) * 8;
      *(f32x4*)v = *(const f32x4*)p;
      *(f32x4*)(v + 4) = *(const f32x4*)(p + 4);
      if (row >= s.m || col >= s.n) continue;
      if (!RAGGED || left == 8) epi.put8(q, split, row, col, 8, v, held[r], columns);
      else epi.put8(q, split, row, col, left, v, held[r], columns);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// For epilogues that read nothing for columns, or nothing ahead.
struct NoColumns {
  struct Columns {};
  __device__ __forceinline__ void columns(int, int, Columns&) const {}
};
struct NothingAhead : NoColumns {
  struct Held {};
  __device__ __forceinline__ void fetch(int, int, int, int, Held&) const {}
};

// Launches gemm_any with the tile that fills the chip: 128 x 128 where those
// are two for every compute unit and not mostly beyond the edge, 64 x 64 below.
template <class E, bool AK, bool BKD, int PA = 1, class Epi>
void launch_gemm_any(const phz_ops* o, hipStream_t stream, Operand a, Operand b, GemmShape s, int batch, Epi epi) {
  const int64_t z = (int64_t)batch * s.splits;
  const bool large = s.m > 64 && s.n > 64 && ceil_div(s.m, 128) * ceil_div(s.n, 128) * z >= 2ll * o->cus;
  const int tile = large ? 128 : 64;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(ceil_div(s.n, tile), ceil_div(s.m, tile), z), dim3(256), 0, stream, a, b, s, epi);
  };
  if constexpr (Epi::kRagged) {
    if (s.n % 8) {
      large ? go(gemm_any<E, AK, BKD, PA, 128, 128, true, Epi>) : go(gemm_any<E, AK, BKD, PA, 64, 64, true, Epi>);
      return;
    }
  }
  large ? go(gemm_any<E, AK, BKD, PA, 128, 128, false, Epi>) : go(gemm_any<E, AK, BKD, PA, 64, 64, false, Epi>);
}

}  // namespace phzop
