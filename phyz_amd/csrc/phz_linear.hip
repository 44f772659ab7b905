// phz_linear.hip — the linear layer with its epilogue, y = act(x W^T + b) + r,
// and its gradients dx = dz W, dw = dz^T x, db = sum of dz over rows, for
// dz = dy act'(pre).
#include "phz_gemm_fast.h"

#include <algorithm>
#include <type_traits>

using namespace phzop;

namespace {

// ── activations ─────────────────────────────────────────────────────────────

// tanh(p) = 1 - 2 / (1 + exp(2 p)), and where that cancels (|p| < 0.3) its
// series to p^9, whose next term is 1382/155925 p^10 < 6e-8 of it. The device
// library's took 60 us more over 134 million elements.
__device__ __forceinline__ float tanh_of(float p) {
  const float s = p * p;
  const float small = p * fmaf(s, fmaf(s, fmaf(s, fmaf(s, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  const float large = fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __expf(2.0f * p)), 1.0f);
  return fabsf(p) < 0.3f ? small : large;
}

// sigmoid(p), with signed_gate's relative error: (1.25 |p| + 8) 2^-24 where p is
// far below 0, 8 2^-24 above.
__device__ __forceinline__ float gate_of(float p) { return __builtin_amdgcn_rcpf(1.0f + __expf(-p)); }

constexpr float kGeluA = 0.79788456080286536f, kGeluB = 0.044715f;  // sqrt(2 / pi)

// The activation in place; the choice is outside the loop.
template <int N>
__device__ __forceinline__ void act_of(int act, float* p) {
  switch (act) {
    case PHZ_ACT_TANH:
#pragma unroll
      for (int c = 0; c < N; c++) p[c] = tanh_of(p[c]);
      break;
    case PHZ_ACT_RELU:
#pragma unroll
      for (int c = 0; c < N; c++) p[c] = p[c] < 0.0f ? 0.0f : p[c];  // NaN stays
      break;
    case PHZ_ACT_SILU:
      // p sigmoid(p); -inf has the limit 0, not the product's NaN.
#pragma unroll
      for (int c = 0; c < N; c++) p[c] = p[c] == -__builtin_inff() ? 0.0f : p[c] * gate_of(p[c]);
      break;
    case PHZ_ACT_GELU:
      // 0.5 (1 + tanh(u)) = sigmoid(2 u)
#pragma unroll
      for (int c = 0; c < N; c++)
        p[c] = p[c] == -__builtin_inff() ? 0.0f
                                         : p[c] * gate_of(p[c] * fmaf(2.0f * kGeluA * kGeluB * p[c], p[c], 2.0f * kGeluA));
      break;
    default: break;
  }
}

__device__ __forceinline__ float act_grad(int act, float p) {
  switch (act) {
    case PHZ_ACT_TANH: {
      // 1 - tanh^2 = 4 t / (1 + t)^2 with t = exp(-2|p|), without cancellation.
      const float t = __expf(-2.0f * fabsf(p)), r = __builtin_amdgcn_rcpf(1.0f + t);
      return 4.0f * t * r * r;
    }
    case PHZ_ACT_RELU: return p > 0.0f ? 1.0f : p <= 0.0f ? 0.0f : p;
    case PHZ_ACT_SILU: {
      const float q = fabsf(signed_gate(p)), g = gate_of(p);
      const float d = fabsf(p) == __builtin_inff() ? 0.0f : p * (q * (1.0f - q));
      return g + d;
    }
    case PHZ_ACT_GELU: {
      const float u = 2.0f * kGeluA * p * fmaf(kGeluB * p, p, 1.0f);
      const float q = fabsf(signed_gate(u)), g = gate_of(u);
      const float du = 2.0f * kGeluA * fmaf(3.0f * kGeluB * p, p, 1.0f);
      const float c = q * (1.0f - q);
      return g + (c == 0.0f ? 0.0f : p * c * du);
    }
    default: return 1.0f;
  }
}

// ── epilogues ───────────────────────────────────────────────────────────────

template <class E>
struct LinearOut {
  const E *bias, *residual;
  E *pre, *y;
  int64_t residual_row, pre_row, y_row, bias_step;
  int act;
  static constexpr bool kRagged = true;
  struct Columns {
    Pack<E, 8> bias;
  };
  struct Held {
    Pack<E, 8> residual;
  };
  __device__ __forceinline__ void columns(int j, int left, Columns& c) const {
    if (!bias) return;
    if (bias_step == 1) {
      load_some(c.bias, bias + j, left);
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) c.bias.v[k] = k < left ? bias[(j + k) * bias_step] : E{};
    }
  }
  __device__ __forceinline__ void fetch(int, int i, int j, int left, Held& h) const {
    if (residual) load_some(h.residual, residual + i * residual_row + j, left);
  }
  __device__ __forceinline__ void put8(int, int, int i, int j, int left, const float* sums, const Held& h,
                                       const Columns& col) const {
    float p[8];
    Pack<E, 8> out;
#pragma unroll
    for (int c = 0; c < 8; c++) p[c] = bias ? sums[c] + to_f32(col.bias.v[c]) : sums[c];
    if (pre) {
#pragma unroll
      for (int c = 0; c < 8; c++) out.v[c] = from_f32<E>(p[c]);
      store_some(pre + i * pre_row + j, out, left);
    }
    act_of<8>(act, p);
#pragma unroll
    for (int c = 0; c < 8; c++) out.v[c] = from_f32<E>(residual ? p[c] + to_f32(h.residual.v[c]) : p[c]);
    store_some(y + i * y_row + j, out, left);
  }
  __device__ __forceinline__ void put1(int, int, int i, int j, float p) const {
    if (bias) p += to_f32(bias[j * bias_step]);
    if (pre) pre[i * pre_row + j] = from_f32<E>(p);
    act_of<1>(act, &p);
    if (residual) p += to_f32(residual[i * residual_row + j]);
    y[i * y_row + j] = from_f32<E>(p);
  }
};

template <class E>
struct PlainOut : NothingAhead {
  static constexpr bool kRagged = true;
  E* y;
  int64_t row;
  PlainOut(E* p, int64_t r) : y(p), row(r) {}
  __device__ __forceinline__ void put8(int, int, int i, int j, int left, const float* sums, const Held&, const Columns&) const {
    Pack<E, 8> out;
#pragma unroll
    for (int c = 0; c < 8; c++) out.v[c] = from_f32<E>(sums[c]);
    store_some(y + i * row + j, out, left);
  }
};

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

// ── few rows ────────────────────────────────────────────────────────────────
//
// Up to 64 rows (a policy acting, a serving batch): the weights are read once
// and everything else is small, so the floor is their way from memory. A
// workgroup takes 16 TN outputs, its eight waves every eighth run of 128 bytes
// of each weight row, straight into the matrix cores' fragments: lane l holds
// the 16 bytes of row l % 16 at l / 16, and so does it of the inputs' row l %
// 16; which k an instruction pairs is the same on both sides and does not
// matter to the sum. The waves' sums meet in LDS in order. f32 takes the f32
// matrix instructions: exact products, and still below the weights' time.
// 16 x 2048 -> 8192 bf16: 8.8 us, 3.8 TB/s (a large copy: 7.2 us). From 33 rows
// on the inputs' way from L2 counts too: 64 x 2048 -> 4096 bf16 13.2 us against
// 10.7 by tiles, but 64 x 1852 -> 3995 13.3 against 21.8, f32 512 -> 2048 7.3
// against 11.0, and equal elsewhere.

template <class E> struct Small;
template <> struct Small<bf16> {
  static constexpr int kPer = 8;
  static __device__ __forceinline__ f32x4 run(const Pack<bf16, 8>& a, const Pack<bf16, 8>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Small<float> {
  static constexpr int kPer = 4;
  static __device__ __forceinline__ f32x4 run(const Pack<float, 4>& a, const Pack<float, 4>& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
  }
};

constexpr int kSmallRows = 64, kSmallWaves = 8;

template <class E, int TM, int TN, class Epi>
__global__ __launch_bounds__(kSmallWaves * 64) void few_rows(const E* x, int64_t x_row, const E* w, int64_t w_row,
                                                             int32_t m, int32_t n, int32_t k, int32_t k_split, Epi epi) {
  constexpr int PER = Small<E>::kPer, U = 2;  // U loads of 64 bytes a row make a line
  typedef Pack<E, PER> Frag;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, at = (lane >> 4) * PER;
  const int n0 = blockIdx.x * 16 * TN;
  const E* wp[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) wp[j] = w + min(n0 + j * 16 + r, n - 1) * w_row + at;
  const E* xp[TM];
#pragma unroll
  for (int i = 0; i < TM; i++) xp[i] = x + min(i * 16 + r, m - 1) * x_row + at;
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int kRun = 4 * PER * U;
  const int split = blockIdx.y;
  int k0 = split * k_split + wave * kRun;
  k = min(k, (split + 1) * k_split);
#pragma unroll 2
  for (; k0 + kRun <= k; k0 += kSmallWaves * kRun) {
    Frag fw[U][TN], fx[U][TM];
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
      for (int j = 0; j < TN; j++) fw[u][j] = *(const Frag*)(wp[j] + k0 + u * 4 * PER);
#pragma unroll
      for (int i = 0; i < TM; i++) fx[u][i] = *(const Frag*)(xp[i] + k0 + u * 4 * PER);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = Small<E>::run(fw[u][j], fx[u][i], acc[i][j]);
  }
  if (k0 < k) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      Frag fw[TN], fx[TM];
      const int left = k - (k0 + u * 4 * PER + at);  // of this lane's elements
#pragma unroll
      for (int c = 0; c < PER; c++) {
#pragma unroll
        for (int j = 0; j < TN; j++) fw[j].v[c] = c < left ? wp[j][k0 + u * 4 * PER + c] : E{};
#pragma unroll
        for (int i = 0; i < TM; i++) fx[i].v[c] = c < left ? xp[i][k0 + u * 4 * PER + c] : E{};
      }
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = Small<E>::run(fw[j], fx[i], acc[i][j]);
    }
  }
  // Rows past m repeat the last one; their sums are not stored.
  // [wave][input row][output], outputs one apart: row (lane / 16) 4 + r of the
  // accumulator is an output, column lane % 16 an input row.
  constexpr int kRow = 16 * TN + 1;
  __shared__ float sums[kSmallWaves][16 * TM][kRow];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) sums[wave][i * 16 + r][j * 16 + (lane >> 4) * 4 + c] = acc[i][j][c];
  __syncthreads();
  for (int t = threadIdx.x; t < 16 * TM * 16 * TN; t += kSmallWaves * 64) {
    const int i = t / (16 * TN), j = t % (16 * TN);
    float v = sums[0][i][j];
#pragma unroll
    for (int g = 1; g < kSmallWaves; g++) v += sums[g][i][j];
    if (i < m && n0 + j < n) epi.put1(0, split, i, n0 + j, v);
  }
}

// 32 outputs a workgroup where that still is one for every compute unit, and
// the contraction in splits where 16 leave units idle and their time (of runs
// of k, by rows and type, measured) pays for the join: 32 x 4096 -> 1024 15.2 us
// in one, 10.5 in four.
struct FewPlan {
  bool wide;
  int32_t splits, k_split;
  uint64_t part_bytes;
};
template <class E>
FewPlan plan_few(const phz_ops* o, int64_t m, int64_t n, int64_t k) {
  constexpr int64_t kAll = kSmallWaves * 8 * Small<E>::kPer;  // a run of every wave
  const double us = k * (sizeof(E) == 2 ? 1.5 + 0.045 * m : 2.0 + 0.105 * m) / 1000;
  FewPlan p{ceil_div(n, 32) >= o->cus, 1, 0, 0};
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>(o->cus / ceil_div(n, 16), k / (2 * kAll)));
  if (us * (1 - 1.0 / splits) < 5) splits = 1;
  p.k_split = (int32_t)(std::max<int64_t>(1, ceil_div(ceil_div(k, splits), kAll)) * kAll);
  p.splits = (int32_t)std::max<int64_t>(1, ceil_div(k, p.k_split));
  p.part_bytes = p.splits > 1 ? (uint64_t)p.splits * m * pad8(n) * 4 : 0;
  return p;
}

template <class E, class Epi>
void launch_few_rows(hipStream_t stream, const phz_tensor* x, const phz_tensor* w, const FewPlan& p, Epi epi) {
  const int32_t m = (int32_t)x->size[0], k = (int32_t)x->size[1], n = (int32_t)w->size[0];
  auto go = [&](auto kernel, int per) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(n, per), (unsigned)p.splits), dim3(kSmallWaves * 64), 0, stream,
                       (const E*)x->data, x->stride[0], (const E*)w->data, w->stride[0], m, n, k, p.k_split, epi);
  };
  if (m <= 16) p.wide ? go(few_rows<E, 1, 2, Epi>, 32) : go(few_rows<E, 1, 1, Epi>, 16);
  else if (m <= 32) p.wide ? go(few_rows<E, 2, 2, Epi>, 32) : go(few_rows<E, 2, 1, Epi>, 16);
  else p.wide ? go(few_rows<E, 4, 2, Epi>, 32) : go(few_rows<E, 4, 1, Epi>, 16);
}

// Eight f32 as two planes of bf16, the second `plane` elements on.
__device__ __forceinline__ void put_two(bf16* to, int64_t plane, const float* v) {
  Pack<bf16, 8> hi, lo;
#pragma unroll
  for (int c = 0; c < 8; c++) cut2(v[c], hi.v[c], lo.v[c]);
  *(Pack<bf16, 8>*)to = hi;
  *(Pack<bf16, 8>*)(to + plane) = lo;
}

// Eight f32 as three planes of bf16.
__device__ __forceinline__ void put_cut(bf16* to, int64_t plane, const float* v) {
  Pack<bf16, 8> h, m, l;
#pragma unroll
  for (int c = 0; c < 8; c++) cut3(v[c], h.v[c].bits, m.v[c].bits, l.v[c].bits);
  *(Pack<bf16, 8>*)to = h;
  *(Pack<bf16, 8>*)(to + plane) = m;
  *(Pack<bf16, 8>*)(to + 2 * plane) = l;
}

// dz = dy act'(pre) (where there is an activation, or the copy is wanted) in
// rows of `dz_row` with zeros past n, or cut into three planes of such rows, and
// the sums of dz over each block's rows, which ColumnSums adds up in order. For
// bf16 operands with an activation dz is two planes of bf16 (cut2), the second
// `plane` on in the same row: rounded to one, it would be a second rounding of
// the gradients, as large as their own (1 x 33 -> 13: 0.0033 off 64 bits,
// relative, for 0.0020). A thread takes eight columns; `across` (a power of two, at most 32) of them lie
// along a row, the others take rows in turn. Bound by memory: 40793 x 1760 bf16
// 77 us for 431 MB (5.6 TB/s), 16384 x 256 f32 10.7 us for 50 MB, of which some
// 4 us are the launch's ramp and the sums.
template <class E>
__global__ __launch_bounds__(256) void dz_rows(int act, const E* dy, int64_t dy_row, const E* pre, int64_t pre_row,
                                               E* dz, bf16* cut, int64_t plane, int64_t dz_row, float* sums, E* db,
                                               int64_t db_step, int32_t m, int32_t n, int32_t rows, int32_t across) {
  const int lanes = 256 / across, at = threadIdx.x & (across - 1), lane = threadIdx.x / across;
  const int j = (blockIdx.x * across + at) * 8;
  const int64_t i0 = (int64_t)blockIdx.y * rows, i1 = min((int64_t)m, i0 + rows);
  float total[8];
#pragma unroll
  for (int c = 0; c < 8; c++) total[c] = 0.0f;
  if (j + 8 <= n) {
#pragma unroll 4
    for (int64_t i = i0 + lane; i < i1; i += lanes) {
      const Pack<E, 8> d = *(const Pack<E, 8>*)(dy + i * dy_row + j);
      Pack<E, 8> p, out;
      float all[8];
      if (act != PHZ_ACT_NONE) p = *(const Pack<E, 8>*)(pre + i * pre_row + j);
#pragma unroll
      for (int c = 0; c < 8; c++) {
        float v = to_f32(d.v[c]);
        if (act != PHZ_ACT_NONE) v *= act_grad(act, to_f32(p.v[c]));
        total[c] += v;
        out.v[c] = from_f32<E>(v);
        all[c] = v;
      }
      if constexpr (sizeof(E) == 2) {
        if (dz && plane) put_two(dz + i * dz_row + j, plane, all);
        else if (dz) *(Pack<E, 8>*)(dz + i * dz_row + j) = out;
      } else {
        if (dz) *(Pack<E, 8>*)(dz + i * dz_row + j) = out;
        if (cut) put_cut(cut + i * dz_row + j, plane, all);
      }
    }
  } else if (j < n) {
    for (int64_t i = i0 + lane; i < i1; i += lanes) {
      float all[8];
#pragma unroll
      for (int c = 0; c < 8; c++) {
        float v = 0.0f;
        if (j + c < n) {
          v = to_f32(dy[i * dy_row + j + c]);
          if (act != PHZ_ACT_NONE) v *= act_grad(act, to_f32(pre[i * pre_row + j + c]));
          total[c] += v;
        }
        all[c] = v;
        if (dz && !(sizeof(E) == 2 && plane)) dz[i * dz_row + j + c] = from_f32<E>(v);  // rows are whole eights
      }
      if constexpr (sizeof(E) == 2) {
        if (dz && plane) put_two(dz + i * dz_row + j, plane, all);
      } else {
        if (cut) put_cut(cut + i * dz_row + j, plane, all);
      }
    }
  }
  if (!sums && !db) return;
  __shared__ float s[256][9];  // [lane][eight of columns][column], one apart
  __shared__ float part[256];
#pragma unroll
  for (int c = 0; c < 8; c++) s[threadIdx.x][c] = total[c];
  __syncthreads();
  // A thread adds eight lanes of a column, and the first ones those sums.
  const int wide = across * 8, at_col = threadIdx.x & (wide - 1), first = threadIdx.x / wide * 8;
  float v = 0.0f;
#pragma unroll
  for (int l = 0; l < 8; l++) v += s[(first + l) * across + at_col / 8][at_col % 8];
  part[threadIdx.x] = v;
  __syncthreads();
  const int col = blockIdx.x * wide + at_col;
  if (first == 0 && col < n) {
    for (int l = wide; l < 256; l += wide) v += part[l + at_col];
    if (sums) sums[(int64_t)blockIdx.y * n + col] = v;
    else db[col * db_step] = from_f32<E>(v);
  }
}

// db from the blocks' sums of dz: eight columns a workgroup, 32 threads a
// column, each every 32nd block's sum. Latency only (3 to 4 us by itself), so it
// goes beside the join of dw's splits where there is one.
template <class E>
struct ColumnSums {
  const float* sums;
  E* db;
  int64_t step;
  int32_t parts, n;
  unsigned blocks;  // workgroups, 0 where there is no db
  __device__ __forceinline__ void run(unsigned block) const {
    __shared__ float s[4][8];
    const int c = threadIdx.x & 7, j = block * 8 + c;
    float v = 0.0f;
    if (j < n) {
#pragma unroll 8
      for (int i = threadIdx.x >> 3; i < parts; i += 32) v += sums[(int64_t)i * n + j];
    }
#pragma unroll
    for (int k = 8; k < 64; k *= 2) v += __shfl_xor(v, k);
    if ((threadIdx.x & 63) < 8) s[threadIdx.x >> 6][c] = v;
    __syncthreads();
    if (threadIdx.x < 8 && j < n) db[j * step] = from_f32<E>((s[0][c] + s[1][c]) + (s[2][c] + s[3][c]));
  }
};
template <class E>
__global__ __launch_bounds__(256) void column_sums(ColumnSums<E> c) {
  c.run(blockIdx.x);
}

// Rows of n elements into rows of `to_row`, zeros between: as they are, or f32
// cut into three planes. Bound by memory: 54038 x 252 bf16 12 us, 4.5 TB/s.
template <class E>
__global__ __launch_bounds__(256) void pack_rows(const E* from, int64_t from_row, E* to, bf16* cut, int64_t to_row,
                                                 int64_t plane, int32_t m, int32_t n) {
  const int64_t per = to_row / 8;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < m * per; t += (int64_t)gridDim.x * 256) {
    const int64_t i = t / per, j = (t - i * per) * 8;
    const E* p = from + i * from_row + j;
    Pack<E, 8> v{};
    if (j + 8 <= n) v = *(const Pack<E, 8>*)p;
    else
      for (int c = 0; c < 8 && j + c < n; c++) v.v[c] = p[c];
    if (to) *(Pack<E, 8>*)(to + i * to_row + j) = v;
    if constexpr (sizeof(E) == 4)
      if (cut) put_cut(cut + i * to_row + j, plane, v.v);
  }
}

template <class E>
__global__ void fill_zero(E* y, int64_t row, int32_t n, int64_t total) {
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < total; t += (int64_t)gridDim.x * blockDim.x)
    y[t / n * row + t % n] = E{};
}

// ── hosts ───────────────────────────────────────────────────────────────────

bool check_act(phz_ops* o, int act) {
  if (act >= PHZ_ACT_NONE && act <= PHZ_ACT_GELU) return true;
  o->err = "unknown activation";
  return false;
}

bool check_type(phz_ops* o, const char* name, const phz_tensor* t) {
  if (!t) return o->err = fmt("%s is missing", name), false;
  if (t->dtype == PHZ_F32 || t->dtype == PHZ_BF16) return true;
  o->err = fmt("%s is %s, expected f32 or bf16", name, dtype_name(t->dtype));
  return false;
}

bool check_limits(phz_ops* o, int64_t m, int64_t n, int64_t k) {
  // Tile counts along rows and columns fit the grid's 65535 and 2^31.
  if (m > 65535ll * 64 || n > 65535ll * 64 || k > 65535ll * 64)
    return o->err = "rows, n_in and n_out have to be at most 4194240", false;
  return true;
}

// Workspace of one call, handed out in pieces of whole 256 bytes: first counted,
// then taken.
struct Carve {
  char* base = nullptr;
  uint64_t used = 0;
  template <class T> T* take(uint64_t bytes) {
    T* p = (T*)(base ? base + used : nullptr);
    used += (bytes + 255) & ~255ull;
    return p;
  }
};

// How a product's operands go to gemm_fast: as they are, copied into whole
// eights where they do not lie well (rows of whole 16 bytes, and a tile's rows
// within 32-bit offsets); or, f32, cut in three planes.
enum Way { AS_IS, CUT, ANY };  // ANY: gemm_any

// By sizes alone, so a view's strides do not change the result's bits. `whole`:
// the sizes along dense axes are whole 16 bytes, so that usually nothing needs
// a copy; from `copy_from` multiply-adds on the copies pay all the same. f32
// goes to bf16 pieces from 2^33 multiply-adds on, where their rate pays for the
// cuts (us, f32 instructions / pieces: 2048 x 1024 -> 1024 45 / 53, 4096 x 1024
// -> 1024 77 / 70, 8192 x 1024 -> 1024 139 / 107, 16384 x 1024 -> 1024 265 / 198;
// not at every size: 4100 x 2056 -> 1032 174 / 200).
template <class E>
Way way_of(int64_t m, int64_t n, int64_t k, bool whole) {
  constexpr int64_t copy_from = 1ll << 30;
  const int64_t work = m * n * k;
  if (sizeof(E) == 4 && work >= 1ll << 33 && m * pad8(k) < 1ll << 29 && m * pad8(n) < 1ll << 29 && n * pad8(k) < 1ll << 29)
    return CUT;  // planes keep their distance within the 32 bits of a tile's offsets
  return whole || work >= copy_from ? AS_IS : ANY;
}

template <class E>
struct Lain {
  const E* from;
  int64_t from_row, rows, cols;
  Way way;
  bool well, two = false;  // two: a copy of two planes, a row of one beside the other's
  char* copy = nullptr;
  Lain(const phz_tensor* t, Way w)
      : from((const E*)t->data), from_row(t->stride[0]), rows(t->size[0]), cols(t->size[1]), way(w) {
    constexpr int64_t el = 16 / sizeof(E);
    well = way == ANY || (way == AS_IS && (uintptr_t)from % 16 == 0 && from_row % el == 0 && cols % el == 0 &&
                          from_row <= 1 << 22);
  }
  int64_t plane() const {  // elements
    return way == CUT ? (rows * pad8(cols) + 127) / 128 * 128 : two ? pad8(cols) : 0;
  }
  uint64_t bytes() const { return way == CUT ? 3 * plane() * 2 : rows * row() * sizeof(E); }
  const void* data() const { return well ? (const void*)from : copy; }
  int64_t row() const { return well ? from_row : pad8(cols) * (two ? 2 : 1); }
  int64_t whole_cols() const { return well ? cols : pad8(cols); }
  void lay(hipStream_t stream) const {
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(rows * (pad8(cols) / 8), 256), 8192);
    if (!well)
      hipLaunchKernelGGL(pack_rows<E>, dim3(blocks), dim3(256), 0, stream, from, from_row, (E*)(way == CUT ? nullptr : copy),
                         (bf16*)(way == CUT ? copy : nullptr), pad8(cols), plane(), (int32_t)rows, (int32_t)cols);
  }
};

template <class E>
FastPlan plan(const phz_ops* o, Way way, int64_t m, int64_t n, int64_t k, bool two = false) {
  return plan_fast(o, m, n, k, 1, way == CUT ? 3 : sizeof(E) == 4 ? (int)PLANES_F32 : two ? (int)PLANES_2BY1 : 1, true);
}

// The product of two operands, C of m x n, contraction k; AK, BK: dense along
// it.
template <class E, bool AK, bool BK, class Epi, class Beside = NothingBeside>
void product(const phz_ops* o, hipStream_t stream, const Lain<E>& a, const Lain<E>& b, int64_t m, int64_t n, int64_t k,
             const FastPlan& plan, float* part, const Epi& epi, const Beside& beside = {}) {
  const int64_t e = a.way == CUT ? 2 : sizeof(E);
  FastArgs f{};
  f.a = (const char*)a.data(), f.b = (const char*)b.data(), f.a_row = a.row() * e, f.b_row = b.row() * e;
  f.a_plane = (uint32_t)(a.plane() * 2), f.b_plane = (uint32_t)(b.plane() * 2);
  f.m = (int32_t)m, f.n = (int32_t)n, f.k = (int32_t)k;
  f.a_rows = (int32_t)(AK ? a.rows : a.whole_cols()), f.b_rows = (int32_t)(BK ? b.rows : b.whole_cols());
  if constexpr (sizeof(E) == 4) {
    if (a.way == CUT) return launch_gemm_fast<bf16, 3, AK, BK>(o, stream, f, 1, plan, part, epi, beside);
  } else if constexpr (!BK) {  // A is dz
    if (a.two) return launch_gemm_fast<bf16, 2, AK, BK, 1>(o, stream, f, 1, plan, part, epi, beside);
  }
  launch_gemm_fast<E, 1, AK, BK>(o, stream, f, 1, plan, part, epi, beside);
}

template <class E>
int linear(phz_ops* o, hipStream_t stream, int act, const phz_tensor* x, const phz_tensor* w, const phz_tensor* bias,
           const phz_tensor* residual, const phz_tensor* pre, const phz_tensor* y) {
  const int64_t m = x->size[0], k = x->size[1], n = w->size[0];
  LinearOut<E> out{};
  if (bias) out.bias = (const E*)bias->data, out.bias_step = bias->stride[0];
  if (residual) out.residual = (const E*)residual->data, out.residual_row = residual->stride[0];
  if (pre) out.pre = (E*)pre->data, out.pre_row = pre->stride[0];
  out.y = (E*)y->data, out.y_row = y->stride[0];
  out.act = act;
  if (m <= kSmallRows) {
    const FewPlan how = plan_few<E>(o, m, n, k);
    if (how.splits == 1) {
      launch_few_rows<E>(stream, x, w, how, out);
    } else {
      float* part = (float*)o->workspace(stream, how.part_bytes);
      if (!part) return 1;
      const PartOut sums{part, pad8(n), m * pad8(n), m * pad8(n)};
      launch_few_rows<E>(stream, x, w, how, sums);
      launch_join(stream, sums, 1, how.splits, (int32_t)m, (int32_t)n, out, NothingBeside{});
    }
    return launched(o, "linear") ? 0 : 1;
  }
  const Way way = k == 0 ? ANY : way_of<E>(m, n, k, k % (16 / sizeof(E)) == 0);
  if (way != ANY) {
    Lain<E> a(x, way), b(w, way);
    const FastPlan how = plan<E>(o, way, m, n, pad8(k));
    Carve c;
    float* part = nullptr;
    for (int pass = 0; pass < 2; pass++) {
      c.used = 0;
      if (!a.well) a.copy = c.take<char>(a.bytes());
      if (!b.well) b.copy = c.take<char>(b.bytes());
      part = c.take<float>(how.part_bytes);
      if (pass == 0 && c.used && !(c.base = o->workspace(stream, c.used))) return 1;
    }
    a.lay(stream);
    b.lay(stream);
    product<E, true, true>(o, stream, a, b, m, n, k, how, part, out);
  } else {
    const AnyPlan how = plan_any<E>(o, m, n, k);
    float* part = how.part_bytes ? (float*)o->workspace(stream, how.part_bytes) : nullptr;
    if (how.part_bytes && !part) return 1;
    launch_any<E, true, true>(o, stream, Operand{x->data, x->stride[0], 0}, Operand{w->data, w->stride[0], 0}, m, n, k, how,
                              part, out);
  }
  return launched(o, "linear") ? 0 : 1;
}

template <class E>
int linear_backward(phz_ops* o, hipStream_t stream, int act, const phz_tensor* dy, const phz_tensor* x,
                    const phz_tensor* w, const phz_tensor* pre, const phz_tensor* dx, const phz_tensor* dw,
                    const phz_tensor* db) {
  const int64_t m = x->size[0], k = x->size[1], n = w->size[0];
  const bool need_dx = dx && m > 0 && k > 0, need_dw = dw && k > 0 && m > 0;
  constexpr int64_t el = 16 / sizeof(E);
  const Way way = way_of<E>(m, n, k, k % el == 0 && n % el == 0);
  const bool fast = way != ANY;
  Lain<E> d(dy, way), xo(x, way), wo(w, way);
  if (act != PHZ_ACT_NONE) d.well = false;  // dz is made here
  d.two = sizeof(E) == 2 && act != PHZ_ACT_NONE;
  FastPlan dx_plan{}, dw_plan{};
  if (fast && need_dx) dx_plan = plan<E>(o, way, m, k, pad8(n), d.two);
  if (fast && need_dw) dw_plan = plan<E>(o, way, n, k, m, d.two);
  AnyPlan dx_any{1, 1, 0}, dw_any{1, 1, 0};
  if (!fast && need_dx) dx_any = plan_any<E>(o, m, k, n);
  if (!fast && need_dw) dw_any = plan_any<E>(o, n, k, m);
  const bool lay_d = (need_dx || need_dw) && (fast ? !d.well : act != PHZ_ACT_NONE);
  // Blocks of rows whose sums of dz are added up in the end: four workgroups a
  // compute unit in all, 64 to 512 blocks of at least 16 rows. Up to 128 rows
  // are one block, of 64 rows at a time, which leaves db itself (a launch less:
  // 25.3 -> 22.1 us for 2 x 57 -> 914; 323 x 558 -> 20 would take 34 for 25).
  const bool one = m <= 128;
  int across = one ? 4 : 32;
  while (across > 1 && across * 4 >= n) across /= 2;
  const int64_t wanted = std::min<int64_t>(512, std::max<int64_t>(64, 4 * o->cus / ceil_div(n, across * 8)));
  const int64_t rows = one ? 128 : std::max<int64_t>(16, ceil_div(ceil_div(m, wanted), 8) * 8), blocks = ceil_div(m, rows);

  Carve c;
  float *sums = nullptr, *part = nullptr;
  for (int pass = 0; pass < 2; pass++) {
    c.used = 0;
    if (lay_d) d.copy = c.take<char>(d.bytes());
    if (db && !one) sums = c.take<float>(blocks * n * 4);
    if (fast && need_dw && !xo.well) xo.copy = c.take<char>(xo.bytes());
    if (fast && need_dx && !wo.well) wo.copy = c.take<char>(wo.bytes());
    part = c.take<float>(std::max({dx_plan.part_bytes, dw_plan.part_bytes, dx_any.part_bytes, dw_any.part_bytes}));
    if (pass == 0 && c.used && !(c.base = o->workspace(stream, c.used))) return 1;
  }
  if (m > 0 && (lay_d || db)) {
    hipLaunchKernelGGL(dz_rows<E>, dim3((unsigned)ceil_div(n, across * 8), (unsigned)blocks), dim3(256), 0, stream, act,
                       (const E*)dy->data, dy->stride[0], pre ? (const E*)pre->data : nullptr, pre ? pre->stride[0] : 0,
                       (E*)(way == CUT ? nullptr : d.copy), (bf16*)(way == CUT ? d.copy : nullptr), d.plane(),
                       pad8(n) * (d.two ? 2 : 1), sums, db ? (E*)db->data : nullptr, db ? db->stride[0] : 0, (int32_t)m, (int32_t)n, (int32_t)rows, across);
  }
  // db goes with the join of dw's splits where there is one.
  const ColumnSums<E> bias{sums, db ? (E*)db->data : nullptr, db ? db->stride[0] : 0, (int32_t)blocks, (int32_t)n,
                           db && (!one || m == 0) ? (unsigned)ceil_div(n, 8) : 0u};
  const bool joined = need_dw && (fast ? dw_plan.splits : dw_any.splits) > 1;
  if (bias.blocks && !joined) hipLaunchKernelGGL(column_sums<E>, dim3(bias.blocks), dim3(256), 0, stream, bias);
  if (fast) {
    if (need_dx) {
      wo.lay(stream);
      product<E, true, false>(o, stream, d, wo, m, k, n, dx_plan, part, PlainOut<E>{(E*)dx->data, dx->stride[0]});
    }
    if (need_dw) {
      xo.lay(stream);
      product<E, false, false>(o, stream, d, xo, n, k, m, dw_plan, part, PlainOut<E>{(E*)dw->data, dw->stride[0]}, bias);
    }
  } else {
    const Operand dop{d.copy ? d.copy : dy->data, d.copy ? pad8(n) * (d.two ? 2 : 1) : dy->stride[0], 0, d.plane()},
        xa{x->data, x->stride[0], 0}, wa{w->data, w->stride[0], 0};
    auto both = [&](auto planes) {
      constexpr int PA = decltype(planes)::value;
      if (need_dx)
        launch_any<E, true, false, PA>(o, stream, dop, wa, m, k, n, dx_any, part, PlainOut<E>{(E*)dx->data, dx->stride[0]});
      if (need_dw)
        launch_any<E, false, false, PA>(o, stream, dop, xa, n, k, m, dw_any, part, PlainOut<E>{(E*)dw->data, dw->stride[0]},
                                        bias);
    };
    if constexpr (sizeof(E) == 2) {
      d.two ? both(std::integral_constant<int, 2>{}) : both(std::integral_constant<int, 1>{});
    } else {
      both(std::integral_constant<int, 1>{});
    }
  }
  if (dw && k > 0 && m == 0)
    hipLaunchKernelGGL(fill_zero<E>, dim3(256), dim3(256), 0, stream, (E*)dw->data, dw->stride[0], (int32_t)k, n * k);
  return launched(o, "linear backward") ? 0 : 1;
}

bool same_view(const phz_tensor* a, const phz_tensor* b) {
  return a->data == b->data && (a->size[0] <= 1 || a->stride[0] == b->stride[0]);
}

}  // namespace

extern "C" {

int phz_linear(phz_ops* o, void* stream, int act, const phz_tensor* x, const phz_tensor* w, const phz_tensor* bias,
               const phz_tensor* residual, const phz_tensor* pre, const phz_tensor* y) {
  return guarded(o, [&] {
    if (!check_act(o, act) || !check_type(o, "x", x)) return 1;
    const int d = x->dtype;
    if (!check(o, "x", x, Want{2, {-1, -1, 0}, d, true, false})) return 1;
    const int64_t m = x->size[0], k = x->size[1];
    if (!check(o, "w", w, Want{2, {-1, k, 0}, d, true, false})) return 1;
    const int64_t n = w->size[0];
    if ((bias && !check(o, "bias", bias, Want{1, {n, 0, 0}, d, false, false})) ||
        (residual && !check(o, "residual", residual, Want{2, {m, n, 0}, d, true, false})) ||
        (pre && !check(o, "pre", pre, Want{2, {m, n, 0}, d, true, true})) ||
        !check(o, "y", y, Want{2, {m, n, 0}, d, true, true}) || !check_limits(o, m, n, k))
      return 1;
    const bool in_place = residual && !empty(y) && same_view(y, residual);
    for (const phz_tensor* t : {y, pre}) {
      const char* name = t == y ? "y" : "pre";
      if (!apart(o, name, t, "x", x) || !apart(o, name, t, "w", w) || !apart(o, name, t, "bias", bias)) return 1;
      if (!(t == y && in_place) && !apart(o, name, t, "residual", residual)) return 1;
    }
    if (!apart(o, "y", y, "pre", pre)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (m == 0 || n == 0) return 0;
    DeviceGuard g(o);
    if (!g.ok) return 1;
    return d == PHZ_F32 ? linear<float>(o, (hipStream_t)stream, act, x, w, bias, residual, pre, y)
                        : linear<bf16>(o, (hipStream_t)stream, act, x, w, bias, residual, pre, y);
  });
}

int phz_linear_backward(phz_ops* o, void* stream, int act, const phz_tensor* dy, const phz_tensor* x,
                        const phz_tensor* w, const phz_tensor* pre, const phz_tensor* dx, const phz_tensor* dw,
                        const phz_tensor* db) {
  return guarded(o, [&] {
    if (!check_act(o, act) || !check_type(o, "x", x)) return 1;
    const int d = x->dtype;
    if (!check(o, "x", x, Want{2, {-1, -1, 0}, d, true, false})) return 1;
    const int64_t m = x->size[0], k = x->size[1];
    if (!check(o, "w", w, Want{2, {-1, k, 0}, d, true, false})) return 1;
    const int64_t n = w->size[0];
    if (act != PHZ_ACT_NONE && !pre) return o->fail("pre is missing: the activation's gradient needs it");
    if (!check(o, "dy", dy, Want{2, {m, n, 0}, d, true, false}) ||
        (pre && !check(o, "pre", pre, Want{2, {m, n, 0}, d, true, false})) ||
        (dx && !check(o, "dx", dx, Want{2, {m, k, 0}, d, true, true})) ||
        (dw && !check(o, "dw", dw, Want{2, {n, k, 0}, d, true, true})) ||
        (db && !check(o, "db", db, Want{1, {n, 0, 0}, d, false, true})) || !check_limits(o, m, n, k))
      return 1;
    const struct { const char* name; const phz_tensor* t; } outs[] = {{"dx", dx}, {"dw", dw}, {"db", db}},
        ins[] = {{"dy", dy}, {"x", x}, {"w", w}, {"pre", pre}};
    for (auto& u : outs)
      for (auto& v : ins)
        if (!apart(o, u.name, u.t, v.name, v.t)) return 1;
    if (!apart(o, "dx", dx, "dw", dw) || !apart(o, "dx", dx, "db", db) || !apart(o, "dw", dw, "db", db)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    DeviceGuard g(o);
    if (!g.ok) return 1;
    if (n == 0) {
      if (dx && m > 0 && k > 0) {
        if (d == PHZ_F32)
          hipLaunchKernelGGL(fill_zero<float>, dim3(256), dim3(256), 0, (hipStream_t)stream, (float*)dx->data,
                             dx->stride[0], (int32_t)k, m * k);
        else
          hipLaunchKernelGGL(fill_zero<bf16>, dim3(256), dim3(256), 0, (hipStream_t)stream, (bf16*)dx->data,
                             dx->stride[0], (int32_t)k, m * k);
      }
      return launched(o, "linear backward") ? 0 : 1;
    }
    return d == PHZ_F32 ? linear_backward<float>(o, (hipStream_t)stream, act, dy, x, w, pre, dx, dw, db)
                        : linear_backward<bf16>(o, (hipStream_t)stream, act, dy, x, w, pre, dx, dw, db);
  });
}

}  // extern "C"
