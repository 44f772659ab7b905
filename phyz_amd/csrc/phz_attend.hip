// phz_attend.hip — linear attention with a decay for each head, over rollouts
// and one step at a time, with its gradients.
//
//   S_t = a_t S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t,  a_t = exp(g_t), or 0
//                                                           where an episode begins
//   E_t = scale q_t do_t^T + a_{t+1} E_{t+1}
//   dq_t = scale S_t do_t,  dk_t = E_t v_t,  dv_t = E_t^T k_t,
//   dg_t = a_t <E_t, S_{t-1}>,  ds0 = a_0 E_0
//
// Steps are taken in chunks of C (64 in bf16, 32 in f32), in which the recurrence
// is four matrix products. With L[t][s] = a_{s+1} .. a_t for s <= t (0 where an
// episode begins between), e_t = L from the chunk's start, r_s = L to its end and
// f over all of it,
//   A = scale (Q K^T) o L,   O = A V + scale e o (Q S),   S <- f S + K^T (r o V)
// A workgroup takes one head of one world through its chunks (or a segment of
// them, where heads are few), the state in its waves' registers: the data is read
// once. L comes from running sums of g in f64, as differences of long ones are
// taken.
#include "phz_ops.h"

#include <algorithm>
#include <type_traits>

using namespace phzop;

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_of_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxSize = 128;       // of a head's keys and values
constexpr float kForgets = -104.0f; // exp of less is 0 in f32: an episode begins

// One of q, k, v, o and their gradients: [steps][worlds][heads of its own * size].
struct Rows {
  void* p;
  int64_t t, b;  // strides
  int32_t per;   // heads of g that one of its heads serves
};
// States [worlds][heads][size_k * size_v], or null.
struct States {
  float* p;
  int64_t b, h;
};

struct AttendArgs {
  Rows q, k, v, o, dq, dk, dv;  // o: the output, or its gradient
  const float* g;
  float* dg;
  const uint8_t* reset;
  States s0, s1, ds, ds0;  // first and last state, their gradients
  int64_t g_t, g_b, g_h, dg_t, dg_b, dg_h, r_t, r_b;
  int32_t steps, worlds, heads, nk, nv;
  float scale;
  const uint32_t* flags;  // heads to take, or null: all
};

template <class E>
__device__ __forceinline__ const E* row_of(const Rows& r, int b, int h, int size) {
  return (const E*)r.p + b * r.b + (int64_t)(h / r.per) * size;
}

// The lane, as a value that the compiler finds anew: the addresses that follow from
// it are then not all kept in registers through a loop over steps or chunks.
__device__ __forceinline__ int fresh_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// ── one step after another ──────────────────────────────────────────────────
//
// A wave holds 16 columns of one head's state: lane (c, g) = (lane % 16, lane /
// 16) has its column's rows 16 i + 4 g + r. A sweep is
//   s <- a s + key val^T,  out = s^T read
// over the steps in either direction; the four gradients' and the forward pass's
// are all of this form.
struct Sweep {
  const void *read, *key, *val;
  int64_t read_t, key_t, val_t;
  int32_t rows, cols;   // key's (and read's) size, and val's
  float key_scale, out_scale;
  const float* first;   // the state that it starts from, or null
  int64_t f_row, f_col; // strides of its elements
  bool back;
};

// What is left of the state that comes into a step: exp(g) of it, or 0 where an
// episode begins. Below f32's normal numbers exp(g) is a product of two, since the
// state may be large enough to need its digits.
struct Keep {
  float by, rest;
  bool forget;
  __device__ __forceinline__ Keep(float x, bool reset) : forget(reset || x < kForgets) {
    const bool small = x < -87.0f;
    by = expf(small ? 0.5f * x : x);
    rest = small ? by : 1.0f;
  }
  __device__ __forceinline__ float of(float s) const { return forget ? 0.0f : s * by * rest; }
};
__device__ __forceinline__ Keep keep_of(const AttendArgs& a, int b, int h, int64_t t) {
  if (t >= a.steps) return Keep(0.0f, false);
  return Keep(a.g[b * a.g_b + h * a.g_h + t * a.g_t], a.reset && a.reset[b * a.r_b + t * a.r_t]);
}
__device__ __forceinline__ void first_state(const Sweep& w, int col0, float (&s)[8][4]) {
  const int lane = fresh_lane(), col = col0 + (lane & 15), g = lane >> 4;
#pragma unroll
  for (int i = 0; i < 8; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int d = 16 * i + 4 * g + r;
      s[i][r] = w.first && col < w.cols && d < w.rows ? w.first[d * w.f_row + col * w.f_col] : 0.0f;
    }
}
// Step t, and the column's sum over the lane's rows of read. (Rows that do not exist
// are left alone: a value that is not finite times their 0 is not 0.)
template <class E>
__device__ __forceinline__ float take_step(const AttendArgs& a, const Sweep& w, int b, int h, int64_t t, int col0, float (&s)[8][4]) {
  const int lane = fresh_lane(), col = col0 + (lane & 15), g = lane >> 4;
  // Backwards the state of step t + 1 comes in by that step's gate.
  const Keep keep = keep_of(a, b, h, w.back ? t + 1 : t);
  const E* key = (const E*)w.key + t * w.key_t;
  const E* read = (const E*)w.read + t * w.read_t;
  const float val = col < w.cols ? to_f32(((const E*)w.val)[t * w.val_t + col]) * w.key_scale : 0.0f;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if (16 * i >= w.rows) break;
    const int d = 16 * i + 4 * g;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t at = (uint32_t)min(d + r, w.rows - 1);
      const bool there = d + r < w.rows;
      const float x = fmaf(to_f32(key[at]), val, keep.of(s[i][r]));
      s[i][r] = there ? x : s[i][r];
      sum = there ? fmaf(to_f32(read[at]), x, sum) : sum;
    }
  }
  return sum;
}
template <class E, class Before, class Out>
__device__ __forceinline__ void sweep(const AttendArgs& a, const Sweep& w, int b, int h, int col0, float (&s)[8][4], Before&& before,
                                      Out&& out) {
  const int col = col0 + (threadIdx.x & 15);
  first_state(w, col0, s);
#pragma unroll 1
  for (int n = 0; n < a.steps; n++) {
    const int64_t t = w.back ? a.steps - 1 - n : n;
    before(t);
    float sum = take_step<E>(a, w, b, h, t, col0, s);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    out(t, col, col < w.cols, sum * w.out_scale);
  }
}

template <class E>
__device__ __forceinline__ void put(const Rows& r, int64_t t, int b, int h, int size, int col, float v, bool wide) {
  // Heads that share one of theirs leave f32 sums of their own, joined later.
  if (wide) ((float*)r.p)[t * r.t + b * r.b + (int64_t)h * size + col] = v;
  else ((E*)r.p)[t * r.t + b * r.b + (int64_t)h * size + col] = from_f32<E>(v);
}

// The elements of the state that a lane holds, rows and columns within the head.
template <class F>
__device__ __forceinline__ void each_element(int rows, int col, bool live, float (&s)[8][4], F&& f) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < 8; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int d = 16 * i + 4 * g + r;
      if (live && d < rows) f(d, s[i][r]);
    }
}

// A head whose steps are taken one after the other: what the chunks' products
// cannot do is right here, infinities and NaN that a reset cuts off from the
// steps behind it. A workgroup looks through its heads' flags, a thread a head at a
// time (one wave's look at each in turn took 17 us for 16384 heads, this 6).
struct Flagged {
  const AttendArgs& a;
  int32_t marks;
  uint64_t* mask;  // of 8, in LDS
  int64_t all;
  // Calls f(head) for each of the workgroup's heads that is marked, or for all.
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    for (int64_t bh0 = blockIdx.x; bh0 < all; bh0 += 512 * (int64_t)gridDim.x) {
      const int64_t mine = bh0 + threadIdx.x * (int64_t)gridDim.x;
      uint32_t any = 0;
      if (mine < all) {
        any = !a.flags;
        #pragma unroll 16
        for (int m = 0; m < marks; m++) any |= a.flags[m * all + mine];
      }
      const uint64_t marked = __ballot(any != 0);
      if (!__syncthreads_or(any)) continue;
      if ((threadIdx.x & 63) == 0) mask[threadIdx.x >> 6] = marked;
      __syncthreads();
      for (int i = 0; i < 512; i++)
        if (mask[i >> 6] >> (i & 63) & 1) f(bh0 + i * (int64_t)gridDim.x);
      __syncthreads();
    }
  }
};
template <class E>
__global__ __launch_bounds__(512) void attend_sequential(AttendArgs a, int32_t marks) {
  const int wave = threadIdx.x >> 6, c = threadIdx.x & 15, col0 = 16 * wave;
  const int64_t all = (int64_t)a.worlds * a.heads;
  __shared__ uint64_t mask[8];
  Flagged{a, marks, mask, all}.each([&](int64_t bh) {
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    if (col0 >= a.nv) return;
    Sweep w{row_of<E>(a.q, b, h, a.nk), row_of<E>(a.k, b, h, a.nk), row_of<E>(a.v, b, h, a.nv), a.q.t, a.k.t, a.v.t, a.nk, a.nv,
            1.0f, a.scale, a.s0.p ? a.s0.p + b * a.s0.b + h * a.s0.h : nullptr, a.nv, 1, false};
    float s[8][4];
    sweep<E>(a, w, b, h, col0, s, [](int64_t) {}, [&](int64_t t, int col, bool live, float v) {
      if (live && (threadIdx.x & 63) < 16) put<E>(a.o, t, b, h, a.nv, col, v, false);
    });
    if (a.s1.p) {
      float* last = a.s1.p + b * a.s1.b + h * a.s1.h;
      const int col = col0 + c;
      each_element(a.nk, col, col < a.nv, s, [&](int d, float v) { last[(int64_t)d * a.nv + col] = v; });
    }
  });
}

// Its gradients. `wide`: which of dq, dk, dv are sums of each head's own (1, 2, 4).
// dg = exp(g_t) <E_t, S_{t-1}> by that formula: what is not finite reaches the steps
// that the formula says, and no others, and no sum is taken over steps. E goes back
// from the last step; the states that it meets, as many steps' at a time as LDS holds,
// are found again from the one before their `chunk` steps, which the first pass leaves
// in `kept`, one a chunk from chunk `from` on (blocks: 16 rows each of a padded state):
// the passes over the products are done with that memory. A head of 4000 steps of 64 and
// 64 f32 takes 61 ms, 0.1 where all is finite.
struct Kept {
  float* p;
  int64_t step;  // elements to the next chunk's
  int32_t size, blocks, from, chunk;
};
template <class E>
__global__ __launch_bounds__(512) void attend_sequential_backward(AttendArgs a, int32_t marks, int32_t wide, Kept kept) {
  // 16 blocks of 16 rows of states, beside one in registers.
  __shared__ float met[16 * 4][512];
  const int most = 16 / kept.blocks + 1;
  __shared__ float part[8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, col0 = 16 * wave;
  const int64_t all = (int64_t)a.worlds * a.heads;
  // The sum of one value of each lane over the workgroup, in every thread.
  auto total = [&](float v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
    if (lane == 0) part[wave] = v;
    __syncthreads();
    float sum = 0.0f;
    for (int i = 0; i < 8; i++) sum += part[i];
    __syncthreads();
    return sum;
  };
  __shared__ uint64_t mask[8];
  Flagged{a, marks, mask, all}.each([&](int64_t bh) {
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    const E *q = row_of<E>(a.q, b, h, a.nk), *k = row_of<E>(a.k, b, h, a.nk), *v = row_of<E>(a.v, b, h, a.nv),
            *d_o = row_of<E>(a.o, b, h, a.nv);
    const float* s0 = a.s0.p ? a.s0.p + b * a.s0.b + h * a.s0.h : nullptr;
    const float* ds = a.ds.p ? a.ds.p + b * a.ds.b + h * a.ds.h : nullptr;
    // The states' transposes: dq reads S, dk and dg E, by their columns d.
    const Sweep of_s{d_o, v, k, a.o.t, a.v.t, a.k.t, a.nv, a.nk, 1.0f, a.scale, s0, 1, a.nv, false};
    const Sweep of_e{v, d_o, q, a.v.t, a.o.t, a.q.t, a.nv, a.nk, a.scale, 1.0f, ds, 1, a.nv, true};
    auto slot = [&](int64_t t) {
      return kept.p + (t / kept.chunk - kept.from) * kept.step + bh * kept.size + wave * kept.blocks * 256 + lane;
    };
    const bool holds = a.dg && col0 < a.nk;
    float s[8][4];
    sweep<E>(a, of_s, b, h, col0, s,
             [&](int64_t t) {
               if (!holds || t == 0 || t % kept.chunk) return;
               float* p = slot(t);
#pragma unroll
               for (int i = 0; i < 8; i++)
                 if (i < kept.blocks)
#pragma unroll
                   for (int r = 0; r < 4; r++) p[(i * 4 + r) * 64] = s[i][r];
             },
             [&](int64_t t, int col, bool live, float x) {
               if (live && lane < 16) put<E>(a.dq, t, b, h, a.nk, col, x, wide & 1);
             });
    sweep<E>(a, of_e, b, h, col0, s, [](int64_t) {}, [&](int64_t t, int col, bool live, float x) {
      if (live && lane < 16) put<E>(a.dk, t, b, h, a.nk, col, x, wide & 2);
    });
    sweep<E>(a, Sweep{k, q, d_o, a.k.t, a.q.t, a.o.t, a.nk, a.nv, a.scale, 1.0f, ds, a.nv, 1, true}, b, h, col0, s, [](int64_t) {},
             [&](int64_t t, int col, bool live, float x) {
               if (live && lane < 16) put<E>(a.dv, t, b, h, a.nv, col, x, wide & 4);
             });
    if (a.ds0.p) {
      float* out = a.ds0.p + b * a.ds0.b + h * a.ds0.h;
      const Keep keep = keep_of(a, b, h, 0);
      const int col = col0 + c;
      each_element(a.nk, col, col < a.nv, s, [&](int d, float x) { out[(int64_t)d * a.nv + col] = keep.of(x); });
    }
    if (!a.dg) return;
    float* dg = a.dg + b * a.dg_b + h * a.dg_h;
    float e[8][4];
    first_state(of_e, col0, e);
    for (int64_t t1 = a.steps; t1 > 0;) {
      // Steps from t1 - n to t1 - 1, of the chunk that begins at t0.
      const int64_t t0 = (t1 - 1) / kept.chunk * kept.chunk;
      const int n = (int)min((int64_t)most, t1 - t0);
      if (t0 == 0) {
        first_state(of_s, col0, s);
      } else if (holds) {
        const float* p = slot(t0);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) s[i][r] = i < kept.blocks ? p[(i * 4 + r) * 64] : 0.0f;
      }
#pragma unroll 1
      for (int64_t t = t0; t < t1 - 1; t++) {
        const int m = (int)(t - (t1 - n));
        if (m >= 0) {
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (i < kept.blocks)
#pragma unroll
              for (int r = 0; r < 4; r++) met[(m * kept.blocks + i) * 4 + r][threadIdx.x] = s[i][r];
        }
        (void)take_step<E>(a, of_s, b, h, t, col0, s);
      }
#pragma unroll 1
      for (int m = n - 1; m >= 0; m--) {
        const int64_t t = t1 - n + m;
        (void)take_step<E>(a, of_e, b, h, t, col0, e);
        // The gate before the sum, which may pass f32's range without it.
        const Keep keep = keep_of(a, b, h, t);
        float mine = 0.0f;
        if (col0 + c < a.nk) {
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (i < kept.blocks)
#pragma unroll
              for (int r = 0; r < 4; r++)
                mine = fmaf(keep.of(e[i][r]), m + 1 < n ? met[(m * kept.blocks + i) * 4 + r][threadIdx.x] : s[i][r], mine);
        }
        const float sum = total(mine);
        if (threadIdx.x == 0) dg[t * a.dg_t] = keep.forget ? 0.0f : sum;
      }
      t1 -= n;
    }
  });
}

// ── chunks: products of tiles of 16 ─────────────────────────────────────────
//
// A fragment is, of a lane (c, g) = (lane % 16, lane / 16), four neighbouring
// elements 4 g .. 4 g + 3 of a block of 16 along the contraction, of row (or
// column) c. The matrix instructions' result has that form too, its rows along the
// contraction: a state that one product leaves in registers is the next one's
// operand as it is.
// kSide: chains of products side by side (f32's take as long to issue as to end).
template <class E> struct Kind;
template <> struct Kind<float> {
  typedef f32x4 Frag;
  static constexpr int C = 32, kPieces = 1, kSide = 1;
};
// bf16: operands that are f32 (scores, states, what is added to a state) go in
// three pieces, each the rounding of what the ones before leave, which hold what f32
// does. (Two leave 2^-17 of each: bf16 results were then 8e-5 to 1.1e-4 of their norm
// from the rounding of 64 bits', now at most 4e-5, for 2 to 9% of the time.)
template <> struct Kind<bf16> {
  typedef s16x4 Frag;
  static constexpr int C = 64, kPieces = 3, kSide = 2;
};

// c + A B over N blocks of 16.
template <int N>
__device__ __forceinline__ f32x4 mma(const f32x4* a, const f32x4* b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][r], b[i][r], c, 0, 0, 0);
  return c;
}
template <int N>
__device__ __forceinline__ f32x4 mma(const s16x4* a, const s16x4* b, f32x4 c) {
  static_assert(N % 2 == 0, "an instruction takes two blocks");
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const s16x8 x = __builtin_shufflevector(a[i], a[i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    const s16x8 y = __builtin_shufflevector(b[i], b[i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  }
  return c;
}

// U of them side by side, chains that do not wait for each other: c[u] + A B with
// the operands' fragments sa and sb apart.
template <int N, int U>
__device__ __forceinline__ void mma_side(const f32x4* a, int sa, const f32x4* b, int sb, f32x4* c) {
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int u = 0; u < U; u++) c[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u * sa + i][r], b[u * sb + i][r], c[u], 0, 0, 0);
}
template <int N, int U>
__device__ __forceinline__ void mma_side(const s16x4* a, int sa, const s16x4* b, int sb, f32x4* c) {
#pragma unroll
  for (int i = 0; i < N; i += 2)
#pragma unroll
    for (int u = 0; u < U; u++) c[u] = mma<2>(a + u * sa + i, b + u * sb + i, c[u]);
}

// The two bf16 of a word.
__device__ __forceinline__ float low_half(uint32_t x) { return __builtin_bit_cast(float, x << 16); }
__device__ __forceinline__ float high_half(uint32_t x) { return __builtin_bit_cast(float, x & 0xffff0000u); }

// v in NP pieces, each `stride` fragments from the last.
template <int NP>
__device__ __forceinline__ void cut(f32x4 v, f32x4* out, int) {
  static_assert(NP == 1, "f32 is whole");
  out[0] = v;
}
template <int NP>
__device__ __forceinline__ void cut(f32x4 v, s16x4* out, int stride) {
#pragma unroll
  for (int p = 0; p < NP; p++) {
    u32x2 x;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const f32x2 pair{v[2 * i], v[2 * i + 1]};
      x[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2));
      if (p + 1 < NP) v[2 * i] -= low_half(x[i]), v[2 * i + 1] -= high_half(x[i]);
    }
    out[p * stride] = __builtin_bit_cast(s16x4, x);
  }
}
__device__ __forceinline__ f32x4 widen(f32x4 v) { return v; }
__device__ __forceinline__ f32x4 widen(s16x4 v) {
  const u32x2 x = __builtin_bit_cast(u32x2, v);
  return f32x4{low_half(x[0]), high_half(x[0]), low_half(x[1]), high_half(x[1])};
}
// What decays leave of a state, times `by`: 0, whatever x is, where an episode begins
// between; else x times the square of their root, which f32 holds down to 2^-252 of
// it (an infinity stays one, or becomes a NaN, which sends the head to the steps one
// after the other).
__device__ __forceinline__ f32x4 left_of(f32x4 x, float root, float by) {
  const float f = root * by;
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = root < 0.0f ? 0.0f : x[i] * root * f;
  return x;
}

// A tile of ROWS x D in LDS, rows 16 bytes apart from whole banks: fragments along
// a row and down a column fall into all banks.
template <class E, int D>
struct Tile {
  typedef typename Kind<E>::Frag Frag;
  static constexpr int kRow = D * sizeof(E) + 16;
  static __device__ __forceinline__ Frag along(const char* l, int row, int block, int lane) {
    return *(const Frag*)(l + (row + (lane & 15)) * kRow + (16 * block + (lane >> 4) * 4) * (int)sizeof(E));
  }
  // Rows 16 block + 4 g .. + 3 of column col + c.
  static __device__ __forceinline__ Frag down(const char* l, int block, int col, int lane) {
    const int c = lane & 15, g = lane >> 4;
    if constexpr (sizeof(E) == 4) {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; r++) v[r] = *(const float*)(l + (16 * block + 4 * g + r) * kRow + (col + c) * 4);
      return v;
    } else {
      // The transposing read hands each lane of 16 a column of a 4 x 16 block.
      typedef __attribute__((address_space(3))) s16x4 lds4;
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(l + (16 * block + 4 * g + (c >> 2)) * kRow + col * 2 + (c & 3) * 8));
    }
  }
};

// A chunk's scores in LDS: the tiles on and below the diagonal alone, so that three
// pieces are smaller than two whole squares. Block b's b + 1 tiles stand beside those
// of the block as far from the other end: rows of one length, 16 bytes apart from
// whole banks.
template <class E>
struct Scores {
  typedef typename Kind<E>::Frag Frag;
  static constexpr int NB = Kind<E>::C / 16, kTileRow = 16 * sizeof(E), kRow = kTileRow * (NB + 1) + 16, kSize = NB / 2 * 16 * kRow;
  static __device__ __forceinline__ constexpr int at(int a, int b) {
    return b >= NB / 2 ? (NB - 1 - b) * 16 * kRow + kTileRow * a : b * 16 * kRow + kTileRow * (NB - b + a);
  }
  // Row c of block b, columns 16 a + 4 g .. + 3, for a <= b.
  static __device__ __forceinline__ int place(int a, int b, int lane) {
    return at(a, b) + (lane & 15) * kRow + (lane >> 4) * 4 * (int)sizeof(E);
  }
  // Fragments of the tile of rows b and columns a: along its rows, and down its
  // columns; nothing above the diagonal.
  static __device__ __forceinline__ Frag along(const char* l, int b, int a, int lane) {
    return a <= b ? *(const Frag*)(l + place(a, b, lane)) : Frag{};
  }
  static __device__ __forceinline__ Frag down(const char* l, int b, int a, int lane) {
    if (a > b) return Frag{};
    const int c = lane & 15, g = lane >> 4;
    if constexpr (sizeof(E) == 4) {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; r++) v[r] = *(const float*)(l + at(a, b) + (4 * g + r) * kRow + 4 * c);
      return v;
    } else {
      typedef __attribute__((address_space(3))) s16x4 lds4;
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(l + at(a, b) + (4 * g + (c >> 2)) * kRow + (c & 3) * 8));
    }
  }
};

// A chunk's rows of one tensor on their way from memory to LDS through registers,
// NT threads, each a column of 16 bytes. Rows behind the last step are that step's
// again: what they come to is not stored, and adds nothing to the state (their
// weights are 0). Columns that do not exist are 0; a column that ends within the
// 16 bytes goes to LDS an element at a time, when the others leave registers.
// What follows from these is found where it is used, and not kept in registers
// through the loop over chunks (which it would fill).
__device__ __forceinline__ void again(int& x, int& y) { asm volatile("" : "+v"(x), "+v"(y)); }

template <class E, int D, int NT>
struct Load {
  static constexpr int C = Kind<E>::C, EL = 16 / sizeof(E), kPer = D / EL, kStep = NT / kPer;
  static constexpr int N = (C + kStep - 1) / kStep;
  Pack<E, EL> x[N];
  __device__ __forceinline__ void fetch(const E* base, int64_t stride, int left, int d) {
    int col = threadIdx.x % kPer * EL, row0 = threadIdx.x / kPer;
    again(col, row0);
    // (Also says that what the registers held before is not needed any more.)
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = Pack<E, EL>{};
    if (col + EL > d || left <= 0) return;
    const E* p = base + col;
    if (left == C) {
      p += (uint32_t)row0 * (uint64_t)stride;
#pragma unroll
      for (int i = 0; i < N; i++, p += kStep * stride)
        if (C % kStep == 0 || row0 + i * kStep < C) {
          // f32 past the caches (404 us against 421 for 64 steps of 16384 heads); lines
          // of bf16 are shared by heads.
          if constexpr (sizeof(E) == 4) x[i] = __builtin_bit_cast(std::remove_reference_t<decltype(x[i])>, __builtin_nontemporal_load((const f32x4_of_4*)p));
          else x[i] = *(const Pack<E, EL>*)p;
        }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = *(const Pack<E, EL>*)(p + min(row0 + i * kStep, left - 1) * stride);
    }
  }
  // The same base, stride and d as fetch had.
  __device__ __forceinline__ void stash(char* l, const E* base, int64_t stride, int left, int d) const {
    int col = threadIdx.x % kPer * EL, row0 = threadIdx.x / kPer;
    again(col, row0);
    l += row0 * Tile<E, D>::kRow + col * (int)sizeof(E);
    if (col + EL <= d || col >= d) {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (C % kStep == 0 || row0 + i * kStep < C)
          *(f32x4*)(l + i * kStep * Tile<E, D>::kRow) = __builtin_bit_cast(f32x4, x[i]);
      return;
    }
    const int n = d - col;
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (C % kStep != 0 && row0 + i * kStep >= C) continue;
      const E* p = base + min(row0 + i * kStep, left - 1) * stride + col;
      Pack<E, EL> y;
#pragma unroll
      for (int e = 0; e < EL; e++) y.v[e] = e < n ? p[e] : E{};
      *(f32x4*)(l + i * kStep * Tile<E, D>::kRow) = __builtin_bit_cast(f32x4, y);
    }
  }
};

// What the gates of a chunk come to.
template <int C>
struct Decays {
  double sum[C];            // of log2 of the gates up to t
  float e[C], r[C];         // from the start to t, from t to the end; 0 behind or before a reset
  float e_root[C], r_root[C];  // their roots, negative there
  float u[C], w[C];         // from the end of the tile of 16 before to t, from t to the end of its tile
  int32_t since[C];         // the last step up to t at which an episode begins, or 0; C behind the last step
  float f_root;             // of that over all of it, negative where a reset is in it
  double all;               // log2 of it without resets
  uint64_t resets;
};
// As it was read: a comparison would wait for the loads.
struct Gate {
  float x;
  uint32_t reset;
  bool live;
};
// A lane a step; by one wave.
__device__ __forceinline__ Gate fetch_gate(const float* g, int64_t g_t, const uint8_t* reset, int64_t r_t, int left) {
  const int lane = threadIdx.x & 63;
  Gate v{0.0f, 0, lane < left};
  if (lane < left) {
    v.x = g[lane * g_t];
    if (reset) v.reset = reset[lane * r_t];
  }
  return v;
}
// x moved between lanes by a DPP control; 0 where there is no such lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double x) {
  const u32x2 v = __builtin_bit_cast(u32x2, x);
  const u32x2 y{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)v[0], CTRL, ROWS, 0xf, false),
                (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v[1], CTRL, ROWS, 0xf, false)};
  return __builtin_bit_cast(double, y);
}
__device__ __forceinline__ double of_lane(double x, int lane) {
  const u32x2 v = __builtin_bit_cast(u32x2, x);
  const u32x2 y{(uint32_t)__builtin_amdgcn_readlane((int)v[0], lane), (uint32_t)__builtin_amdgcn_readlane((int)v[1], lane)};
  return __builtin_bit_cast(double, y);
}
template <int C>
__device__ __forceinline__ void find_decays(Gate v, Decays<C>* d) {
  const int lane = threadIdx.x & 63;
  const bool reset = v.reset != 0 || v.x < kForgets;
  // A reset's own gate does not count: what is left of before is nothing.
  double x = reset ? 0.0 : (double)v.x * 1.4426950408889634074;
  x += moved<0x111, 0xf>(x);  // row_shr by 1, 2, 4, 8: sums within rows of 16 lanes
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  const double mine = x, row = moved<0x15f, 0xf>(x);  // the row's last lane's
  x += moved<0x142, 0xa>(x);  // lane 15 to the row behind it, in rows 1 and 3
  x += moved<0x143, 0xc>(x);  // lane 31 to rows 2 and 3
  const uint64_t resets = __ballot(reset);
  const double all = of_lane(x, C - 1);
  if (lane >= C) return;
  const uint64_t upto = resets & (2ull << lane) - 1ull;
  const int at = resets ? 63 - __builtin_clzll(resets) : 0;
  d->sum[lane] = x;
  const bool from_start = v.live && !upto, to_end = v.live && lane >= at;
  const float e_root = __builtin_amdgcn_exp2f(0.5f * (float)x), r_root = __builtin_amdgcn_exp2f(0.5f * (float)(all - x));
  d->e[lane] = from_start ? e_root * e_root : 0.0f;
  d->r[lane] = to_end ? r_root * r_root : 0.0f;
  d->e_root[lane] = from_start ? e_root : -1.0f;
  d->r_root[lane] = to_end ? r_root : -1.0f;
  d->u[lane] = __builtin_amdgcn_exp2f((float)mine);
  d->w[lane] = __builtin_amdgcn_exp2f((float)(row - mine));
  d->since[lane] = !v.live ? C : upto ? 63 - __builtin_clzll(upto) : 0;
  if (lane == 0) {
    d->f_root = resets ? -1.0f : __builtin_amdgcn_exp2f(0.5f * (float)all);
    d->all = all;
    d->resets = resets;
  }
}
// L[t][s] for the lane's t = 16 b + c and s = 16 a + 4 g .. + 3: between tiles the
// product of the way from s to its tile's end, from there to t's tile, and on to t.
template <int C>
__device__ __forceinline__ f32x4 decay_between(const Decays<C>& d, int a, int b, int lane) {
  const int t = 16 * b + (lane & 15), s = 16 * a + (lane >> 4) * 4, since = d.since[t];
  f32x4 x;
  if (a == b) {
    const double at = d.sum[t];
#pragma unroll
    for (int r = 0; r < 4; r++)
      x[r] = s + r <= t && s + r >= since ? __builtin_amdgcn_exp2f((float)(at - d.sum[s + r])) : 0.0f;
  } else {
    float way = d.u[t];
    if (b > a + 1) way *= __builtin_amdgcn_exp2f((float)(d.sum[16 * b - 1] - d.sum[16 * a + 15]));
    const f32x4 w = *(const f32x4*)&d.w[s];
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] = s + r >= since ? way * w[r] : 0.0f;
  }
  return x;
}
// Tile n of the C / 16 (C / 16 + 1) / 2 with a <= b.
__device__ __forceinline__ void tile_of(int n, int* a, int* b) {
  *b = n >= 6 ? 3 : n >= 3 ? 2 : n >= 1 ? 1 : 0;
  *a = n - *b * (*b + 1) / 2;
}

// Segments: `chunks` chunks each, one a workgroup. The states between them stand in
// `states` [count - 1][heads of all worlds][rows * columns, padded] as the waves
// hold them, a lane's four rows of a column together.
struct Segments {
  int32_t chunks, count;
  float* states;
  float* decay;           // [count - 1][heads]: root of that over a segment, negative where a reset is in it
  uint32_t* flags;        // [count][heads]: results that are not finite
  uint32_t* state_flags;  // [count - 1][heads]: states that are not
};

// A workgroup's head and segment. Neighbouring heads share lines of memory: 16 of
// them go to one XCD. (More, and the XCDs are far apart in each row: 64 steps of 8192
// heads' gradients 593 us with an eighth of all a XCD, 568 so; one, and lines are
// read twice: 777 steps of 222 heads 220 us against 218, 1023 of 305 forward 110
// against 108; 64 steps of 16384 in bf16 lose 2% so.)
__device__ __forceinline__ void place_of(const AttendArgs& a, int64_t* bh, int* segment, int* b, int* h) {
  const uint32_t n = gridDim.x, i = blockIdx.x, heads = (uint32_t)(a.worlds * a.heads);
  const uint32_t id = i < n / 128 * 128 ? i / 128 * 128 + i % 8 * 16 + i % 128 / 8 : i;
  const uint32_t s = id / heads, at = id - s * heads;
  *segment = (int)s;
  *bh = at;
  *b = (int)(at / (uint32_t)a.heads);
  *h = (int)(at % (uint32_t)a.heads);
}

__device__ __forceinline__ bool not_finite(float sum_of_zeros) { return sum_of_zeros != 0.0f || sum_of_zeros != sum_of_zeros; }
__device__ __forceinline__ float zeros_of(f32x4 x, float z) {
#pragma unroll
  for (int i = 0; i < 4; i++) z = fmaf(x[i], 0.0f, z);
  return z;
}

// NB blocks, from `block` on, of 16 columns of a state in the caller's layout, as
// rows of keys or of values (TURNED): a lane's four neighbouring rows are nv elements
// apart, or one.
template <bool TURNED, int NB>
__device__ __forceinline__ void read_state(const float* p, int nk, int nv, int col0, int block, f32x4 (&s)[NB]) {
  const int lane = fresh_lane(), col = col0 + (lane & 15), row0 = (lane >> 4) * 4 + 16 * block;
  const int rows = TURNED ? nv : nk, cols = TURNED ? nk : nv;
#pragma unroll
  for (int i = 0; i < NB; i++) s[i] = f32x4{};
  if (!p || col >= cols) return;
  p += TURNED ? row0 + col * nv : row0 * nv + col;
  if (TURNED) {
#pragma unroll
    for (int i = 0; i < NB; i++) {
      if (row0 + 16 * i + 4 <= rows) {
        s[i] = __builtin_bit_cast(f32x4, *(const Pack<float, 4>*)(p + 16 * i));
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (row0 + 16 * i + r < rows) s[i][r] = p[16 * i + r];
      }
    }
  } else {
    // One pointer that moves on: 4 NB of them would fill the registers.
#pragma unroll
    for (int i = 0; i < NB; i++, p += 16 * nv) {
      const float* at = p;
#pragma unroll
      for (int r = 0; r < 4; r++, at += nv)
        if (row0 + 16 * i + r < rows) s[i][r] = *at;
    }
  }
}
template <int NB>
__device__ __forceinline__ void write_state(float* p, int nk, int nv, int col0, const f32x4 (&s)[NB]) {
  const int lane = fresh_lane(), col = col0 + (lane & 15), row0 = (lane >> 4) * 4;
  if (col >= nv) return;
  p += row0 * nv + col;
#pragma unroll
  for (int i = 0; i < NB; i++, p += 16 * nv) {
    float* at = p;
#pragma unroll
    for (int r = 0; r < 4; r++, at += nv)
      if (row0 + 16 * i + r < nk) *at = s[i][r];
  }
}

// Four neighbouring elements of an output's row, of which it has `left` more.
// LAST: f32 that is not read again here goes past the caches (404 us against 425 for
// 64 steps of 16384 heads); the half lines of bf16 have to meet there.
template <bool LAST, class E>
__device__ __forceinline__ void put4(E* p, int left, f32x4 v) {
  if (LAST && sizeof(E) == 4 && left >= 4) {
    __builtin_nontemporal_store(v, (f32x4_of_4*)p);
  } else if (left >= 4) {
    Pack<E, 4> y;
#pragma unroll
    for (int i = 0; i < 4; i++) y.v[i] = from_f32<E>(v[i]);
    *(Pack<E, 4>*)p = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < left) p[i] = from_f32<E>(v[i]);
  }
}
// A wave's 16 columns, from col0 on, of a chunk's rows of one head: a lane's four of
// row 16 i + c. `wide`: f32 sums of each head's own. Whole tiles need no questions.
template <class E, int C>
struct Put {
  char* p;
  int64_t step;  // bytes to 16 rows further
  int rows, cols;
  bool whole, wide;
  __device__ __forceinline__ Put(const Rows& r, int64_t t0, int left, int b, int h, int size, int col0, int lane, bool wide_) : wide(wide_) {
    const uint32_t c = lane & 15, g = lane >> 4;
    const int e = wide ? 4 : (int)sizeof(E);
    p = (char*)r.p + (t0 * r.t + b * r.b + (int64_t)h * size + col0) * e + (c * (uint64_t)r.t + 4 * g) * e;
    step = 16 * r.t * e;
    rows = left - (int)c, cols = size - col0 - 4 * (int)g;
    whole = left == C && col0 + 16 <= size;
  }
  __device__ __forceinline__ void operator()(int i, f32x4 v) const {
    char* at = p + i * step;
    if (!whole && 16 * i >= rows) return;
    const int left = whole ? 4 : cols;
    if (wide) put4<false>((float*)at, left, v);
    else put4<true>((E*)at, left, v);
  }
};

// s <- f s + rows^T (weight o cols) of one chunk, f by its root: the wave's 16 columns, SIDE blocks
// of rows at a time (one where registers are short).
template <class E, int DR, int DC, int SIDE = Kind<E>::kSide>
__device__ __forceinline__ void advance_state(const char* rows, const char* cols, const float* weight, float scale, float f_root, int col0,
                                              f32x4 (&s)[DR / 16]) {
  typedef Kind<E> K;
  typedef typename K::Frag Frag;
  // (Few registers: two blocks of steps at a time as well, 308 us against 342 for 256
  // steps of 2048 heads of 64 backwards in bf16, 553 against 610 for 4096 of 64 of 128.)
  constexpr int NB = K::C / 16, U = SIDE, NJ = SIDE == 1 ? 2 : NB;
  const int lane = fresh_lane(), g = lane >> 4;
#pragma unroll
  for (int j0 = 0; j0 < NB; j0 += NJ) {
    Frag v[K::kPieces][NJ];
#pragma unroll
    for (int i = 0; i < NJ; i++) {
      f32x4 x = widen(Tile<E, DC>::down(cols, j0 + i, col0, lane));
      const f32x4 w = *(const f32x4*)(weight + 16 * (j0 + i) + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; r++) x[r] *= w[r] * scale;
      cut<K::kPieces>(x, &v[0][i], NJ);
    }
#pragma unroll
    for (int i = 0; i < DR / 16; i += U) {
      Frag k[U][NJ];
      f32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
#pragma unroll
        for (int j = 0; j < NJ; j++) k[u][j] = Tile<E, DR>::down(rows, j0 + j, 16 * (i + u), lane);
        x[u] = j0 ? s[i + u] : left_of(s[i + u], f_root, 1.0f);
      }
#pragma unroll
      for (int p = K::kPieces - 1; p >= 0; p--) mma_side<NJ, U>(k[0], NJ, v[p], 0, x);
#pragma unroll
      for (int u = 0; u < U; u++) s[i + u] = x[u];
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// The forward pass. Wave w has columns 16 w .. 16 w + 15 of the state and of o.
// Scores are found a tile of 16 x 16 at a time by all waves, and meet in LDS, where
// q and k were: half the LDS again would be two workgroups a compute unit less.
// Long rollouts of many heads are bound by memory (64 steps of 16384 heads of 64 f32:
// 377 us, 4.3 TB/s); in bf16, and where heads are few, by the chain of a chunk's
// phases: 32768 steps of 8 heads of 128 take 107 us here, two workgroups a compute
// unit, of which the matrix units are busy 24% and the vector units issue 47%.
template <class E, int DK, int DV>
__global__ __launch_bounds__(DV * 4, DV == 128 ? 4 : DK > DV ? 2 : 3) void attend_chunks(AttendArgs a, Segments seg) {
  typedef Kind<E> K;
  typedef typename K::Frag Frag;
  constexpr int C = K::C, NT = DV * 4, NW = NT / 64, NB = C / 16, NK = DK / 16;
  constexpr int two = sizeof(E) == 2 ? 2 : 1, U = K::kSide;  // blocks of an instruction, chains
  constexpr int kTiles = NB * (NB + 1) / 2, kMine = (kTiles + NW - 1) / NW, NH = 2;
  // The next chunk's loads go out before this one's products where registers allow
  // it (1024 steps of 512 heads of 64 bf16: 112 us against 133), in f32 behind them,
  // which is bound by memory anyway (64 of 16384: 404 against 426).
  constexpr bool kEarly = sizeof(E) == 2 && DK <= 64;
  constexpr int kTile = C * Tile<E, DK>::kRow, kScore = Scores<E>::kSize;
  __shared__ __align__(16) char shared[2 * kTile > K::kPieces * kScore ? 2 * kTile : K::kPieces * kScore];
  __shared__ __align__(16) char v_tile[C * Tile<E, DV>::kRow];
  __shared__ __align__(16) Decays<C> decays;
  __shared__ uint32_t bad;
  char *q_tile = shared, *k_tile = shared + kTile;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col0 = 16 * wave;
  const bool live = col0 < a.nv;  // else the wave helps with loads and scores alone
  const int64_t heads = (int64_t)a.worlds * a.heads;
  int64_t bh;
  int segment, b, h;
  place_of(a, &bh, &segment, &b, &h);
  const int64_t first = (int64_t)segment * seg.chunks * C;
  const int64_t end = min((int64_t)a.steps, first + (int64_t)seg.chunks * C);
  const E *q = row_of<E>(a.q, b, h, a.nk), *k = row_of<E>(a.k, b, h, a.nk), *v = row_of<E>(a.v, b, h, a.nv);
  const float* gate = a.g + b * a.g_b + h * a.g_h;
  const uint8_t* reset = a.reset ? a.reset + b * a.r_b : nullptr;

  Load<E, DK, NT> lq, lk;
  Load<E, DV, NT> lv;
  Gate lg{};
  auto fetch = [&](int64_t t) {
    const int left = (int)max((int64_t)0, min((int64_t)C, end - t));
    if (wave == 0) lg = fetch_gate(gate + t * a.g_t, a.g_t, reset ? reset + t * a.r_t : nullptr, a.r_t, left);
    lq.fetch(q + t * a.q.t, a.q.t, left, a.nk);
    lk.fetch(k + t * a.k.t, a.k.t, left, a.nk);
    lv.fetch(v + t * a.v.t, a.v.t, left, a.nv);
  };
  fetch(first);
  f32x4 s[NK];
  if (segment == 0) {
    read_state<false>(a.s0.p ? a.s0.p + b * a.s0.b + h * a.s0.h : nullptr, a.nk, a.nv, col0, 0, s);
  } else {
    const f32x4* p = (const f32x4*)(seg.states + ((segment - 1) * heads + bh) * (DK * DV)) + wave * NK * 64 + fresh_lane();
#pragma unroll
    for (int i = 0; i < NK; i++) s[i] = p[i * 64];
  }
  if (threadIdx.x == 0) bad = 0;
  float zeros = 0.0f;
  for (int64_t t0 = first; t0 < end; t0 += C) {
    __syncthreads();  // the last chunk's tiles are read
    const int left = (int)min((int64_t)C, end - t0);
    lq.stash(q_tile, q + t0 * a.q.t, a.q.t, left, a.nk);
    lk.stash(k_tile, k + t0 * a.k.t, a.k.t, left, a.nk);
    lv.stash(v_tile, v + t0 * a.v.t, a.v.t, left, a.nv);
    if (wave == 0) find_decays(lg, &decays);
    __syncthreads();
    if (kEarly) fetch(t0 + C);
    Frag mine[kMine][K::kPieces];
#pragma unroll
    for (int m = 0; m < kMine; m++) {
      const int lane = fresh_lane();
      const int n = wave + m * NW;
      if (n >= kTiles) break;
      int ta, tb;
      tile_of(n, &ta, &tb);
      Frag x[NK], y[NK];
#pragma unroll
      for (int i = 0; i < NK; i++) {
        x[i] = Tile<E, DK>::along(k_tile, 16 * ta, i, lane);
        y[i] = Tile<E, DK>::along(q_tile, 16 * tb, i, lane);
      }
      f32x4 p = mma<NK>(x, y, f32x4{});
      const f32x4 l = decay_between(decays, ta, tb, lane);
#pragma unroll
      for (int r = 0; r < 4; r++) p[r] = l[r] != 0.0f ? p[r] * l[r] * a.scale : 0.0f;
      cut<K::kPieces>(p, mine[m], 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    // What the state from before the chunk answers: o^T = S^T Q^T.
    // Some of the state's rows at a time: all its pieces would fill the registers.
    f32x4 acc[NB] = {};
    const int at = fresh_lane();
    if (live) {
#pragma unroll
      for (int half = 0; half < NK; half += NH) {
        Frag sp[K::kPieces][NH];
#pragma unroll
        for (int i = 0; i < NH; i++) cut<K::kPieces>(s[half + i], &sp[0][i], NH);
#pragma unroll
        for (int i = 0; i < NB; i += U) {
          Frag y[U][NH];
#pragma unroll
          for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < NH; j++) y[u][j] = Tile<E, DK>::along(q_tile, 16 * (i + u), half + j, at);
#pragma unroll
          for (int p = K::kPieces - 1; p >= 0; p--) mma_side<NH, U>(sp[p], 0, y[0], NH, &acc[i]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int i = 0; i < NB; i++) acc[i] = left_of(acc[i], decays.e_root[16 * i + (at & 15)], a.scale);
      advance_state<E, DK, DV>(k_tile, v_tile, decays.r, 1.0f, decays.f_root, col0, s);
    }
    __syncthreads();  // q and k are read
    if (!kEarly) fetch(t0 + C);  // nothing where that is the end
    const int lane = fresh_lane();
#pragma unroll
    for (int m = 0; m < kMine; m++) {
      const int n = wave + m * NW;
      if (n >= kTiles) break;
      int ta, tb;
      tile_of(n, &ta, &tb);
      char* at = shared + Scores<E>::place(ta, tb, lane);
#pragma unroll
      for (int i = 0; i < K::kPieces; i++) *(Frag*)(at + i * kScore) = mine[m][i];
    }
    Frag vf[NB];
    if (live) {
#pragma unroll
      for (int i = 0; i < NB; i++) vf[i] = Tile<E, DV>::down(v_tile, i, col0, lane);
    }
    __syncthreads();  // the scores are there
    if (live) {
      const Put<E, C> put(a.o, t0, left, b, h, a.nv, col0, lane, false);
#pragma unroll
      for (int i = 0; i < NB; i += two) {
        // In bf16 two tiles of rows take the same pairs of blocks.
#pragma unroll
        for (int p = K::kPieces - 1; p >= 0; p--) {
          Frag y[two][NB];
#pragma unroll
          for (int u = 0; u < two; u++)
#pragma unroll
            for (int j = 0; j < i + two; j++) y[u][j] = Scores<E>::along(shared + p * kScore, i + u, j, lane);
#pragma unroll
          for (int j = 0; j < i + two; j += two) mma_side<two, two>(&vf[j], 0, &y[0][j], NB, &acc[i]);
        }
#pragma unroll
        for (int u = 0; u < two; u++) {
          zeros = zeros_of(acc[i + u], zeros);
          put(i + u, acc[i + u]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (end == a.steps && a.s1.p) write_state(a.s1.p + b * a.s1.b + h * a.s1.h, a.nk, a.nv, col0, s);
#pragma unroll
  for (int i = 0; i < NK; i++) zeros = zeros_of(s[i], zeros);
  if (not_finite(zeros)) bad = 1;
  __syncthreads();
  if (threadIdx.x == 0) seg.flags[segment * heads + bh] = bad;
}

// A state's rows and columns: what key and val are to it, and where an element of
// it stands in the caller's.
struct Roles {
  Rows rows, cols;
  int32_t nr, nc;
  int64_t row_stride, col_stride;
  States first;
};

// States alone, of one segment a workgroup:
//   ADDS   what a segment but the last adds to the state, from 0, and how much it
//          leaves of it
//   BACK   the same of the gradient's, E, from the end, of a segment but the first
//   EACH   the state before each chunk but the first, which stands elsewhere
enum { ADDS, BACK, EACH };
template <class E, int DR, int DC, int MODE>
__global__ __launch_bounds__(DC * 4, DR > 2 * DC ? 2 : 4) void segment_states(AttendArgs a, Roles x, Segments seg, f32x4* each) {
  typedef Kind<E> K;
  constexpr int C = K::C, NT = DC * 4, NR = DR / 16;
  __shared__ __align__(16) char r_tile[C * Tile<E, DR>::kRow], c_tile[C * Tile<E, DC>::kRow];
  __shared__ __align__(16) Decays<C> decays;
  __shared__ uint32_t bad;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col0 = 16 * wave;
  const int64_t heads = (int64_t)a.worlds * a.heads;
  int64_t bh;
  int slot, b, h;
  place_of(a, &bh, &slot, &b, &h);
  const int segment = MODE == BACK ? slot + 1 : slot;
  const int64_t first = (int64_t)segment * seg.chunks * C, end = min((int64_t)a.steps, first + (int64_t)seg.chunks * C);
  const E *rp = row_of<E>(x.rows, b, h, x.nr), *cp = row_of<E>(x.cols, b, h, x.nc);
  const float* gate = a.g + b * a.g_b + h * a.g_h;
  const uint8_t* reset = a.reset ? a.reset + b * a.r_b : nullptr;
  f32x4 s[NR];
  if (MODE == EACH && segment == 0) {
    read_state<true>(x.first.p ? x.first.p + b * x.first.b + h * x.first.h : nullptr, x.nc, x.nr, col0, 0, s);
  } else {
    const f32x4* p = (const f32x4*)(seg.states + ((segment - 1) * heads + bh) * (DR * DC)) + wave * NR * 64 + lane;
#pragma unroll
    for (int i = 0; i < NR; i++) s[i] = MODE == EACH ? p[i * 64] : f32x4{};
  }
  if (threadIdx.x == 0) bad = 0;
  Load<E, DR, NT> lr;
  Load<E, DC, NT> lc;
  Gate lg{};
  auto fetch = [&](int64_t t) {
    const int left = (int)max((int64_t)0, min((int64_t)C, end - t));
    lr.fetch(rp + t * x.rows.t, x.rows.t, left, x.nr);
    lc.fetch(cp + t * x.cols.t, x.cols.t, left, x.nc);
    if (wave == 0) lg = fetch_gate(gate + t * a.g_t, a.g_t, reset ? reset + t * a.r_t : nullptr, a.r_t, left);
  };
  const int64_t chunks = (end - first + C - 1) / C;
  auto start = [&](int64_t n) { return first + (MODE == BACK ? chunks - 1 - n : n) * C; };
  fetch(start(0));
  double all = 0.0;
  bool forgets = false;
  for (int64_t n = 0; n < chunks; n++) {
    if (MODE == EACH && n > 0) {
      f32x4* p = each + ((start(n) / C * heads + bh) * (DC / 16) + wave) * NR * 64 + lane;
#pragma unroll
      for (int i = 0; i < NR; i++) p[i * 64] = s[i];
    }
    if (MODE == EACH && n + 1 == chunks) break;
    __syncthreads();
    const int64_t t0 = start(n);
    const int left = (int)min((int64_t)C, end - t0);
    lr.stash(r_tile, rp + t0 * x.rows.t, x.rows.t, left, x.nr);
    lc.stash(c_tile, cp + t0 * x.cols.t, x.cols.t, left, x.nc);
    if (wave == 0) find_decays(lg, &decays);
    __syncthreads();
    if (n + 1 < chunks) fetch(start(n + 1));
    if (col0 < x.nc)
      advance_state<E, DR, DC>(r_tile, c_tile, MODE == BACK ? decays.e : decays.r, MODE == BACK ? a.scale : 1.0f, decays.f_root, col0, s);
    all += decays.all;
    forgets = forgets || decays.resets;
  }
  if (MODE == EACH) return;
  f32x4* p = (f32x4*)(seg.states + (slot * heads + bh) * (DR * DC)) + wave * NR * 64 + lane;
  float zeros = 0.0f;
#pragma unroll
  for (int i = 0; i < NR; i++) {
    p[i * 64] = s[i];
    zeros = zeros_of(s[i], zeros);
  }
  __syncthreads();
  if (not_finite(zeros)) bad = 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    seg.decay[slot * heads + bh] = forgets ? -1.0f : (float)exp2(0.5 * all);
    seg.state_flags[slot * heads + bh] = bad;
  }
}

// The state before each segment but the first (the gradient behind each but the
// last), from what each adds: in place. 63 segments of 8 heads of 128: 12 us for 66 MB
// both ways (22 with one load after the other).
template <int DR, int DC>
__global__ __launch_bounds__(256) void join_segments(AttendArgs a, Roles x, Segments seg, bool back) {
  const int64_t heads = (int64_t)a.worlds * a.heads, bh = blockIdx.x / (DR * DC / 256);
  const int i = blockIdx.x % (DR * DC / 256) * 256 + threadIdx.x;
  const int r = i & 3, lane = i >> 2 & 63, tile = i >> 8, row = tile % (DR / 16) * 16 + (lane >> 4) * 4 + r;
  const int col = tile / (DR / 16) * 16 + (lane & 15), b = (int)(bh / a.heads), h = (int)(bh % a.heads);
  float s = x.first.p && row < x.nr && col < x.nc
                ? x.first.p[b * x.first.b + h * x.first.h + row * x.row_stride + col * x.col_stride]
                : 0.0f;
  const int slots = seg.count - 1;
  const int64_t step = (back ? -1 : 1) * heads * (DR * DC), from = back ? slots - 1 : 0;
  float* p = seg.states + (from * heads + bh) * (DR * DC) + i;
  const float* f = seg.decay + from * heads + bh;
  const int64_t f_step = back ? -heads : heads;
  // Sixteen at a time: their loads wait together.
  constexpr int N = 16;
  for (int n = 0; n < slots; n += N) {
    float add[N], keep[N];
#pragma unroll
    for (int j = 0; j < N; j++)
      if (n + j < slots) add[j] = p[j * step], keep[j] = f[j * f_step];
#pragma unroll
    for (int j = 0; j < N; j++)
      if (n + j < slots) {
        s = keep[j] < 0.0f ? add[j] : fmaf(keep[j] * s, keep[j], add[j]);
        p[j * step] = s;
      }
    p += N * step;
    f += N * f_step;
  }
}

// Sums over lanes, in each of them, that stay in registers: over a row of 16, and of
// the four rows' values of a lane.
template <int N>
__device__ __forceinline__ float rotated(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float sum_of_row(float x) {
  x += rotated<8>(x);
  x += rotated<4>(x);
  x += rotated<2>(x);
  return x + rotated<1>(x);
}
__device__ __forceinline__ float sum_of_rows(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto y = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t v = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, (uint32_t)y[0]) + __builtin_bit_cast(float, (uint32_t)y[1]));
  const auto z = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_bit_cast(float, (uint32_t)z[0]) + __builtin_bit_cast(float, (uint32_t)z[1]);
}

// Sums over the lanes up to each.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float sums_up_to(float x) {
  x += moved<0x111, 0xf>(x);
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);
  return x + moved<0x143, 0xc>(x);
}

__device__ __forceinline__ float dot4(f32x4 x, f32x4 y) {
  return fmaf(x[0], y[0], fmaf(x[1], y[1], fmaf(x[2], y[2], x[3] * y[3])));
}

// The gradients, chunks from the last to the first. Beside the forward pass's
// products, with S the state before the chunk, E the loss's gradient for the one
// behind it, and W = dO V^T, dA = scale W o L:
//   dQ = dA K + scale e o (dO S^T),  dK = dA^T Q + r o (V E^T),  dV = A^T dO + r o (K E),
//   E <- f E + scale (e o Q)^T dO.
// E is held twice: as rows of values by the first NK waves, 16 columns of keys each,
// which find dK, and as rows of keys by the NV others, which find dV. dQ's tiles are
// dealt out to all. (One wave for a column of each takes twice the registers: when the
// roles were dealt, 458 us against 254 at 256 steps of 2048 heads of 64 in bf16, the
// same in f32.)
// A gate's gradient sums over all ways across it: from the state before to the
// gradient behind, X = f <S, E>; from steps u >= t to the state before,
// q_u . (the state's part of dq_u); from steps s < t to the gradient behind,
// k_s . (its part of dk_s); and between steps of the chunk, M = A o W over u >= t >
// s, R_{t+1} = R_t + sum_u M[u][t] - sum_s M[t][s].
// No sum is taken over more than a chunk, so nothing large cancels.
// 64 steps of 8192 heads of 64 f32: 490 us at 3.0 TB/s, of whose time the matrix
// units are busy 37% and the vector units a third; 777 steps of 222 heads of 48 and
// 80 in bf16: 159 us, one workgroup of twelve waves a compute unit, phases again.
template <int DK, int DV>
constexpr int kGradientThreads = (DK + DV) * 4;

template <class E, int DK, int DV>
__global__ __launch_bounds__((kGradientThreads<DK, DV>), 4) void attend_gradients(AttendArgs a, Segments seg, const float* forth,
                                                                                  const f32x4* each, int32_t wide) {
  typedef Kind<E> K;
  typedef typename K::Frag Frag;
  constexpr int C = K::C, NT = kGradientThreads<DK, DV>, NW = NT / 64, NB = C / 16, NK = DK / 16, NV = DV / 16;
  constexpr int two = sizeof(E) == 2 ? 2 : 1;  // blocks of an instruction
  // dQ's tiles: each in kParts parts of kPer blocks of steps, by a wave of the first
  // and some of the second kind.
  constexpr int kParts = 1 + NV / NK < NB ? 1 + NV / NK : NB, kPer = (NB + kParts - 1) / kParts;
  __shared__ __align__(16) char q_tile[C * Tile<E, DK>::kRow], k_tile[C * Tile<E, DK>::kRow];
  __shared__ __align__(16) char v_tile[C * Tile<E, DV>::kRow], o_tile[C * Tile<E, DV>::kRow];
  __shared__ __align__(16) char score[K::kPieces][Scores<E>::kSize], dscore[K::kPieces][Scores<E>::kSize];
  __shared__ __align__(16) Decays<C> decays;
  __shared__ __align__(16) float row_sum[NB][C], col_sum[NB][C], q_dot[NK][C], k_dot[NK][C], x_dot[NK];
  __shared__ uint32_t bad;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool keys = wave < NK;  // else values
  const int col0 = 16 * (keys ? wave : wave - NK);
  const int tile = wave % NK, part = wave / NK;  // of dQ
  const bool asks = part < kParts && part * kPer < NB && 16 * tile < a.nk;
  const bool live = col0 < (keys ? a.nk : a.nv);  // else the wave helps with loads and scores alone
  const int64_t heads = (int64_t)a.worlds * a.heads;
  int64_t bh;
  int segment, b, h;
  place_of(a, &bh, &segment, &b, &h);
  const int64_t first = (int64_t)segment * seg.chunks * C;
  const int64_t end = min((int64_t)a.steps, first + (int64_t)seg.chunks * C);
  const E *q = row_of<E>(a.q, b, h, a.nk), *k = row_of<E>(a.k, b, h, a.nk), *v = row_of<E>(a.v, b, h, a.nv),
          *d_o = row_of<E>(a.o, b, h, a.nv);
  const float* gate = a.g + b * a.g_b + h * a.g_h;
  const uint8_t* reset = a.reset ? a.reset + b * a.r_b : nullptr;
  float* dg = a.dg ? a.dg + b * a.dg_b + h * a.dg_h : nullptr;

  constexpr int NE = NK > NV ? NK : NV;
  f32x4 e[NE] = {};  // rows of values (NV blocks), or of keys (NK)
  {
    const int lane = fresh_lane(), c = lane & 15, g = lane >> 4;
    if (segment + 1 == seg.count) {
      const float* ds = a.ds.p ? a.ds.p + b * a.ds.b + h * a.ds.h : nullptr;
      if (keys) read_state<true>(ds, a.nk, a.nv, col0, 0, *(f32x4(*)[NV])e);
      else read_state<false>(ds, a.nk, a.nv, col0, 0, *(f32x4(*)[NK])e);
    } else {
      const float* p = seg.states + (segment * heads + bh) * (DK * DV);
      if (keys) {
        // Element (row d, column j) stands at tile j / 16 * NK + d / 16, lane d % 16 / 4 * 16 + j % 16, row d % 4.
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) e[i][r] = p[(((i * NK + wave) * 64) + (c >> 2) * 16 + 4 * g + r) * 4 + (c & 3)];
      } else {
#pragma unroll
        for (int i = 0; i < NK; i++) e[i] = ((const f32x4*)p)[((wave - NK) * NK + i) * 64 + lane];
      }
    }
  }
  // (Tiles of columns that do not exist leave theirs so.)
  for (int i = threadIdx.x; i < NK * C; i += NT) (&q_dot[0][0])[i] = (&k_dot[0][0])[i] = 0.0f;
  if (threadIdx.x < NK) x_dot[threadIdx.x] = 0.0f;
  if (threadIdx.x == 0) bad = 0;
  Load<E, DK, NT> lq, lk;
  Load<E, DV, NT> lv, lo;
  Gate lg{};
  auto fetch = [&](int64_t t) {
    const int left = (int)max((int64_t)0, min((int64_t)C, end - t));
    lq.fetch(q + t * a.q.t, a.q.t, left, a.nk);
    lk.fetch(k + t * a.k.t, a.k.t, left, a.nk);
    lv.fetch(v + t * a.v.t, a.v.t, left, a.nv);
    lo.fetch(d_o + t * a.o.t, a.o.t, left, a.nv);
    if (wave == 0) lg = fetch_gate(gate + t * a.g_t, a.g_t, reset ? reset + t * a.r_t : nullptr, a.r_t, left);
  };
  float zeros = 0.0f;
  // The gates' gradients of the chunk at t0, by the last wave, a lane a step.
  auto gates = [&](int64_t t0, float f_root, uint64_t resets) {
    const int lane = fresh_lane(), t = lane, tile = t / 16;
    float x = 0.0f, qd = 0.0f, kd = 0.0f, m = 0.0f;
    for (int w = 0; w < NK; w++) x += x_dot[w];
    if (t < C) {
      // (q's from the last step on.)
      for (int w = 0; w < NK; w++) qd += q_dot[w][C - 1 - t], kd += k_dot[w][t];
      for (int i = tile; i < NB; i++) m += col_sum[i][t];
      for (int i = 0; i <= tile; i++) m -= row_sum[i][t];
    }
    // Of the steps before: not with t's own taken off again, which a gate that closes
    // leaves far larger than the others.
    const float up = __shfl_up(sums_up_to(kd + m), 1), before = lane ? up : 0.0f;
    const float sum = (f_root < 0.0f ? 0.0f : x * f_root * f_root) + __shfl(sums_up_to(qd), (C - 1 - t) & 63) + before;
    const int64_t step = t0 + t;
    if (t < C && step < end) {
      const float out = resets >> t & 1 ? 0.0f : sum;
      zeros = fmaf(out, 0.0f, zeros);
      dg[step * a.dg_t] = out;
    }
  };
  // acc + the intra-chunk product: A's fragments `x` (a block of steps each) with
  // the scores' of tile i, along their rows or down their columns.
  auto add = [&](const Frag* x, const char (&scores)[K::kPieces][Scores<E>::kSize], int i, bool along, f32x4 acc, int lane) {
#pragma unroll
    for (int p = K::kPieces - 1; p >= 0; p--)
#pragma unroll
      for (int j = 0; j < NB; j += two) {
        if (along ? j > i : j + two <= i) continue;
        Frag y[two];
#pragma unroll
        for (int m = 0; m < two; m++)
          y[m] = along ? Scores<E>::along(scores[p], i, j + m, lane) : Scores<E>::down(scores[p], j + m, i, lane);
        acc = mma<two>(x + j, y, acc);
      }
    zeros = zeros_of(acc, zeros);
    return acc;
  };
  const int64_t chunks = (end - first + C - 1) / C;
  fetch(first + (chunks - 1) * C);
  float f_before = 0.0f;
  uint64_t resets_before = 0;
  for (int64_t n = chunks - 1; n >= 0; n--) {
    const int64_t t0 = first + n * C;
    __syncthreads();  // the chunk before is done with its tiles, and its sums are there
    if (dg && n + 1 < chunks && wave == NW - 1) gates(t0 + C, f_before, resets_before);
    const int left = (int)min((int64_t)C, end - t0);
    lq.stash(q_tile, q + t0 * a.q.t, a.q.t, left, a.nk);
    lk.stash(k_tile, k + t0 * a.k.t, a.k.t, left, a.nk);
    lv.stash(v_tile, v + t0 * a.v.t, a.v.t, left, a.nv);
    lo.stash(o_tile, d_o + t0 * a.o.t, a.o.t, left, a.nv);
    if (wave == 0) find_decays(lg, &decays);
    __syncthreads();
    // Blocks of the state before the chunk: rows of values, the tile's columns of keys.
    constexpr int NS = NV < 4 ? NV : 4;
    auto state_before = [&](int block, f32x4 (&s)[NS]) {
      if (n == 0 && segment == 0) {
        read_state<true>(a.s0.p ? a.s0.p + b * a.s0.b + h * a.s0.h : nullptr, a.nk, a.nv, 16 * tile, block, s);
      } else {
        const f32x4* p = n == 0 ? (const f32x4*)forth + ((segment - 1) * heads + bh) * (NK * NV * 64) : each + (t0 / C * heads + bh) * (NK * NV * 64);
        p += (tile * NV + block) * 64 + fresh_lane();
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] = p[i * 64];
      }
    };
    f32x4 s[NS];
    if (asks) state_before(0, s);
    for (int m = wave; m < NB * (NB + 1) / 2; m += NW) {
      const int lane = fresh_lane(), c = lane & 15, g = lane >> 4;
      int ta, tb;
      tile_of(m, &ta, &tb);
      // c + the tile's products, four blocks at a time.
      auto score_of = [&](auto tag, const char* left, const char* right) {
        constexpr int D = decltype(tag)::value, N = D / 16 < 4 ? D / 16 : 4;
        f32x4 p{};
#pragma unroll
        for (int i = 0; i < D / 16; i += N) {
          Frag x[N], y[N];
#pragma unroll
          for (int j = 0; j < N; j++) {
            x[j] = Tile<E, D>::along(left, 16 * ta, i + j, lane);
            y[j] = Tile<E, D>::along(right, 16 * tb, i + j, lane);
          }
          p = mma<N>(x, y, p);
        }
        return p;
      };
      f32x4 p = score_of(std::integral_constant<int, DK>(), k_tile, q_tile);
      f32x4 w = score_of(std::integral_constant<int, DV>(), v_tile, o_tile);
      const f32x4 l = decay_between(decays, ta, tb, lane);
      f32x4 ways;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const bool there = l[r] != 0.0f;
        p[r] = there ? p[r] * l[r] * a.scale : 0.0f;
        ways[r] = there && (ta != tb || 4 * g + r != c) ? p[r] * w[r] : 0.0f;
        w[r] = there ? w[r] * l[r] * a.scale : 0.0f;
        sum += ways[r];
      }
      const int at = Scores<E>::place(ta, tb, lane);
      Frag z[K::kPieces];
      cut<K::kPieces>(p, z, 1);
#pragma unroll
      for (int i = 0; i < K::kPieces; i++) *(Frag*)(score[i] + at) = z[i];
      cut<K::kPieces>(w, z, 1);
#pragma unroll
      for (int i = 0; i < K::kPieces; i++) *(Frag*)(dscore[i] + at) = z[i];
      if (dg) {
        sum = sum_of_rows(sum);
        if (g == 0) row_sum[ta][16 * tb + c] = sum;
#pragma unroll
        for (int r = 0; r < 4; r++) ways[r] = sum_of_row(ways[r]);
        if (c == 0) *(f32x4*)&col_sum[tb][16 * ta + 4 * g] = ways;
      }
    }
    __syncthreads();
    f_before = decays.f_root;
    resets_before = decays.resets;
    // acc[i] += (state's columns)^T (rows of `with`, of steps' blocks from i0 on) over
    // up to four blocks of the contraction, from `block` on.
    auto far = [&](auto rows, const f32x4* state, const char* with, int block, int i0, auto& acc, int lane) {
      constexpr int NP = K::kPieces, D = decltype(rows)::value, NF = D / 16 < 4 ? D / 16 : 4;
      constexpr int M = sizeof acc / sizeof acc[0], N = 2;
      // Two blocks' pieces at a time: four fill the registers (684 us against 606 for
      // 4096 steps of 64 heads of 128 and 128 in bf16).
#pragma unroll
      for (int k = 0; k < NF; k += N) {
        Frag big[NP][N];
#pragma unroll
        for (int i = 0; i < N; i++) cut<NP>(state[k + i], &big[0][i], N);
#pragma unroll
        for (int i = 0; i < M; i++) {
          Frag y[N];
#pragma unroll
          for (int j = 0; j < N; j++) y[j] = Tile<E, D>::along(with, 16 * (i0 + i), block + k + j, lane);
#pragma unroll
          for (int p = NP - 1; p >= 0; p--) acc[i] = mma<N>(big[p], y, acc[i]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    constexpr std::integral_constant<int, DK> dk{};
    constexpr std::integral_constant<int, DV> dv{};
    // A dot product with a row of q or k, over the tile's 16 columns.
    auto dot = [&](f32x4 x, const char* rows, int i, int column, float* to, int lane) {
      const float d = sum_of_rows(dot4(x, widen(Tile<E, DK>::along(rows, 16 * i, column, lane))));
      if (lane < 16) to[16 * i + lane] = d;
    };
    if (asks) {
      const int lane = fresh_lane(), c = lane & 15;
      f32x4 acc[kPer] = {};
      float d = 0.0f;
#pragma unroll
      for (int block = 0; block < NV; block += NS) {
        if (block) state_before(block, s);
        if (dg && keys) {
#pragma unroll
          for (int i = 0; i < NS; i++) d += dot4(s[i], e[block + i]);
        }
        far(dv, s, o_tile, block, part * kPer, acc, lane);
      }
      if (dg && keys) {
        d = sum_of_rows(sum_of_row(d));
        if (lane == 0) x_dot[wave] = d;
      }
      Frag x[NB];
#pragma unroll
      for (int i = 0; i < NB; i++) x[i] = Tile<E, DK>::down(k_tile, i, 16 * tile, lane);
      const Put<E, C> put(a.dq, t0, left, b, h, a.nk, 16 * tile, lane, wide & 1);
#pragma unroll
      for (int m = 0; m < kParts; m++)
        if (m == part) {
#pragma unroll
          for (int n = 0; n < kPer; n++) {
            const int i = m * kPer + n;
            if (i >= NB) break;
            f32x4 y = left_of(acc[n], decays.e_root[16 * i + c], a.scale);
            if (dg) dot(y, q_tile, i, tile, q_dot[tile], lane);
            y = add(x, dscore, i, true, y, lane);
            put(i, y);
          }
        }
    }
    if (n > 0) fetch(t0 - C);
    if (!live) {
    } else if (keys) {
      const int lane = fresh_lane(), c = lane & 15;
      f32x4 acc[NB] = {};
#pragma unroll
      for (int block = 0; block < NV; block += NS) far(dv, e + block, v_tile, block, 0, acc, lane);
      Frag x[NB];
#pragma unroll
      for (int i = 0; i < NB; i++) x[i] = Tile<E, DK>::down(q_tile, i, col0, lane);
      const Put<E, C> put(a.dk, t0, left, b, h, a.nk, col0, lane, wide & 2);
#pragma unroll
      for (int i = 0; i < NB; i++) {
        f32x4 y = left_of(acc[i], decays.r_root[16 * i + c], 1.0f);
        if (dg) dot(y, k_tile, i, wave, k_dot[wave], lane);
        y = add(x, dscore, i, false, y, lane);
        put(i, y);
      }
      advance_state<E, DV, DK, 1>(o_tile, q_tile, decays.e, a.scale, decays.f_root, col0, *(f32x4(*)[NV])e);
    } else {
      const int lane = fresh_lane(), c = lane & 15;
      f32x4 acc[NB] = {};
#pragma unroll
      for (int block = 0; block < NK; block += 4) far(dk, e + block, k_tile, block, 0, acc, lane);
      Frag x[NB];
#pragma unroll
      for (int i = 0; i < NB; i++) x[i] = Tile<E, DV>::down(o_tile, i, col0, lane);
      const Put<E, C> put(a.dv, t0, left, b, h, a.nv, col0, lane, wide & 4);
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const f32x4 y = add(x, score, i, false, left_of(acc[i], decays.r_root[16 * i + c], 1.0f), lane);
        put(i, y);
      }
      advance_state<E, DK, DV, 1>(q_tile, o_tile, decays.e, a.scale, decays.f_root, col0, *(f32x4(*)[NK])e);
    }
  }
  __syncthreads();
  if (dg && wave == NW - 1) gates(first, f_before, resets_before);
  if (!keys) {
    if (segment == 0 && a.ds0.p)
      write_state(a.ds0.p + b * a.ds0.b + h * a.ds0.h, a.nk, a.nv, col0, *(f32x4(*)[NK])e);
#pragma unroll
    for (int i = 0; i < NK; i++) zeros = zeros_of(e[i], zeros);
  }
  if (not_finite(zeros)) bad = 1;
  __syncthreads();
  if (threadIdx.x == 0) seg.flags[segment * heads + bh] = bad;
}

// ── a single step ───────────────────────────────────────────────────────────
//
// A workgroup takes `width` columns of one head's state: a thread four
// neighbouring columns of every RP-th row, read, replaced and read by q; the
// rows' sums meet in LDS. One pass over the states: 1024 worlds x 4 heads of 64 in 23
// us, 6.0 TB/s (a part of them from the memory-side cache); 8 x 8 heads of 128 in 8 us,
// which is two trips to memory and the launch.
constexpr int kStepThreads = 256;

template <class E>
__global__ __launch_bounds__(kStepThreads) void attend_step(AttendArgs a, int32_t parts, int32_t width) {
  __shared__ float sum[kStepThreads * 4];
  const int64_t at = blockIdx.x;
  const int part = (int)(at % parts);
  const int64_t bh = at / parts;
  const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
  const int j0 = part * width, cols = min(width, a.nv - j0);
  const int groups = (cols + 3) / 4, rows = kStepThreads / groups;
  const int jj = threadIdx.x % groups, rr = threadIdx.x / groups;
  const Keep keep(a.g[b * a.g_b + h * a.g_h], a.reset && a.reset[b * a.r_b]);
  float* s = a.s1.p + b * a.s1.b + h * a.s1.h + j0;
  const E *q = row_of<E>(a.q, b, h, a.nk), *k = row_of<E>(a.k, b, h, a.nk), *v = row_of<E>(a.v, b, h, a.nv) + j0;
  float acc[4] = {};
  const int j = 4 * jj, n = min(4, cols - j);
  if (rr < rows) {
    float val[4];
#pragma unroll
    for (int i = 0; i < 4; i++) val[i] = i < n ? to_f32(v[j + i]) : 0.0f;
    if (n == 4) {
      // Four rows at a time: their loads wait together.
      constexpr int R = 4;
      for (int d0 = rr; d0 < a.nk; d0 += R * rows) {
        Pack<float, 4> w[R];
        E kd[R], qd[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
          const int d = d0 + r * rows;
          if (d < a.nk) w[r] = *(const Pack<float, 4>*)(s + d * a.nv + j), kd[r] = k[d], qd[r] = q[d];
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
          const int d = d0 + r * rows;
          if (d >= a.nk) break;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            w[r].v[i] = fmaf(to_f32(kd[r]), val[i], keep.of(w[r].v[i]));
            acc[i] = fmaf(to_f32(qd[r]), w[r].v[i], acc[i]);
          }
          *(Pack<float, 4>*)(s + d * a.nv + j) = w[r];
        }
      }
    } else {
      for (int d = rr; d < a.nk; d += rows) {
        const float kd = to_f32(k[d]), qd = to_f32(q[d]);
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (i < n) {
            float& w = s[(int64_t)d * a.nv + j + i];
            w = fmaf(kd, val[i], keep.of(w));
            acc[i] = fmaf(qd, w, acc[i]);
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) sum[threadIdx.x * 4 + i] = acc[i];
  __syncthreads();
  const int used = min(rows, a.nk);
  for (int i = threadIdx.x; i < cols; i += kStepThreads) {
    float o = 0.0f;
    for (int r = 0; r < used; r++) o += sum[r * groups * 4 + i];
    ((E*)a.o.p)[b * a.o.b + (int64_t)h * a.nv + j0 + i] = from_f32<E>(o * a.scale);
  }
}

// ── the rest ────────────────────────────────────────────────────────────────

// States copied, or zeros, where there are no steps.
__global__ void copy_states(States from, States to, int32_t heads, int32_t n) {
  const int b = blockIdx.x / heads, h = blockIdx.x % heads;
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    to.p[b * to.b + h * to.h + i] = from.p ? from.p[b * from.b + h * from.h + i] : 0.0f;
}

// The sums of heads that share one: from [steps][worlds][heads * size] f32, dense, VEC
// neighbouring elements a lane. (One at a time, with 64-bit divisions: 37 us for the
// sums of 28749 rows of 6 heads of 48 and of 80, against 20.)
template <class E, int VEC>
__global__ void join_heads(const float* from, Rows to, int64_t rows, int32_t worlds, int32_t heads, int32_t size) {
  const int32_t own = heads / to.per, width = own * size;
  const int64_t n = rows * (width / VEC);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    int64_t row, t;
    if (n <= 0xffffffffll) row = (uint32_t)i / (uint32_t)(width / VEC), t = (uint32_t)row / (uint32_t)worlds;
    else row = i / (width / VEC), t = row / worlds;
    const int32_t x = (int32_t)(i - row * (width / VEC)) * VEC, h = x / size, d = x - h * size;
    const float* f = from + (row * heads + (int64_t)h * to.per) * size + d;
    Pack<float, VEC> s{};
    for (int p = 0; p < to.per; p++) {
      const Pack<float, VEC> y = *(const Pack<float, VEC>*)(f + (int64_t)p * size);
#pragma unroll
      for (int j = 0; j < VEC; j++) s.v[j] += y.v[j];
    }
    Pack<E, VEC> out;
#pragma unroll
    for (int j = 0; j < VEC; j++) out.v[j] = from_f32<E>(s.v[j]);
    *(Pack<E, VEC>*)((E*)to.p + t * to.t + (row - t * worlds) * to.b + x) = out;
  }
}

// ── arguments ───────────────────────────────────────────────────────────────

struct Named {
  const char* name;
  const phz_tensor* t;
};

// Sizes from cfg, q, k, v and g; false, with the error set, where they do not fit.
// ndim 3: with the axis of steps.
bool take(phz_ops* o, const phz_attention_cfg* cfg, const phz_tensor* q, const phz_tensor* k, const phz_tensor* v,
          const phz_tensor* g, const phz_tensor* reset, int ndim, AttendArgs* a) {
  if (!cfg) return o->err = "configuration is missing", false;
  if (cfg->size_k < 1 || cfg->size_k > kMaxSize || cfg->size_v < 1 || cfg->size_v > kMaxSize)
    return o->err = fmt("size_k and size_v have to be 1 to %d, not %d and %d", kMaxSize, cfg->size_k, cfg->size_v), false;
  if (!(cfg->scale >= -3e38 && cfg->scale <= 3e38)) return o->err = "scale has to be finite", false;
  if (!q) return o->err = "q is missing", false;
  if (q->dtype != PHZ_F32 && q->dtype != PHZ_BF16)
    return o->err = fmt("q is %s, expected f32 or bf16", dtype_name(q->dtype)), false;
  const int last = ndim - 1;
  Want any{ndim, {-1, -1, -1}, q->dtype, true, false};
  if (!check(o, "q", q, any)) return false;
  const int64_t T = ndim == 3 ? q->size[0] : 1, B = q->size[last - 1];
  Want rows = any;
  rows.size[0] = ndim == 3 ? T : B;
  if (ndim == 3) rows.size[1] = B;
  if (!check(o, "k", k, rows) || !check(o, "v", v, rows)) return false;
  rows.dtype = PHZ_F32;
  rows.dense = false;
  if (!check(o, "g", g, rows)) return false;
  const int64_t H = g->size[last];
  if (T > 0x3fff0000ll || B > 0x3fff0000ll || H > 0xffffll || H < 1)
    return o->err = "steps and worlds have to be below 2^30, heads 1 to 65535", false;
  if (B * H > 0x3fff0000ll) return o->err = "too many heads of all worlds", false;
  const struct { const char* name; const phz_tensor* t; int size; Rows* to; } each[] = {
      {"q", q, cfg->size_k, &a->q}, {"k", k, cfg->size_k, &a->k}, {"v", v, cfg->size_v, &a->v}};
  for (auto& x : each) {
    const int64_t n = x.t->size[last];
    if (n < 1 || n % x.size || H % (n / x.size))
      return o->err = fmt("%s has %lld elements along axis %d: heads of %d, as many as g's %lld or a divisor of them", x.name,
                          (long long)n, last, x.size, (long long)H),
             false;
    *x.to = Rows{x.t->data, ndim == 3 ? x.t->stride[0] : 0, x.t->stride[last - 1], (int32_t)(H / (n / x.size))};
  }
  Want mask{ndim - 1, {ndim == 3 ? T : B, B, 0}, PHZ_U8, false, false};
  if (reset && !check(o, "reset", reset, mask)) return false;
  a->g = (const float*)g->data;
  a->g_t = ndim == 3 ? g->stride[0] : 0, a->g_b = g->stride[last - 1], a->g_h = g->stride[last];
  if (reset) {
    a->reset = (const uint8_t*)reset->data;
    a->r_t = ndim == 3 ? reset->stride[0] : 0, a->r_b = reset->stride[ndim - 2];
  }
  a->steps = (int32_t)T, a->worlds = (int32_t)B, a->heads = (int32_t)H;
  a->nk = cfg->size_k, a->nv = cfg->size_v;
  a->scale = (float)cfg->scale;
  return true;
}

// One of the tensors of whole states.
bool take_states(phz_ops* o, const char* name, const phz_tensor* t, bool output, const AttendArgs& a, States* to) {
  if (!t) return true;
  const Want want{3, {a.worlds, a.heads, (int64_t)a.nk * a.nv}, PHZ_F32, true, output};
  if (!check(o, name, t, want)) return false;
  *to = States{(float*)t->data, t->stride[0], t->stride[1]};
  return true;
}

// Outputs that share elements with inputs or with each other.
bool all_apart(phz_ops* o, std::initializer_list<Named> outs, std::initializer_list<Named> ins) {
  for (auto u = outs.begin(); u != outs.end(); u++) {
    for (auto& v : ins)
      if (!apart(o, u->name, u->t, v.name, v.t)) return false;
    for (auto v = u + 1; v != outs.end(); v++)
      if (!apart(o, u->name, u->t, v->name, v->t)) return false;
  }
  return true;
}

// A launch has fewer than 2^32 threads, a workgroup up to 1024 of them: calls of more
// heads of all worlds take some worlds at a time, one after the other in the stream.
constexpr int64_t kMostHeads = (1 << 22) - 1;
template <class F>
int by_worlds(const AttendArgs& a, int64_t elem, F&& f) {
  const int64_t most = kMostHeads / a.heads;
  for (int64_t b = 0; b < a.worlds; b += most) {
    AttendArgs x = a;
    x.worlds = (int32_t)std::min(most, a.worlds - b);
    for (Rows* r : {&x.q, &x.k, &x.v, &x.o, &x.dq, &x.dk, &x.dv})
      if (r->p) r->p = (char*)r->p + b * r->b * elem;
    for (States* s : {&x.s0, &x.s1, &x.ds, &x.ds0})
      if (s->p) s->p += b * s->b;
    if (x.g) x.g += b * x.g_b;
    if (x.dg) x.dg += b * x.dg_b;
    if (x.reset) x.reset += b * x.r_b;
    if (f(x)) return 1;
  }
  return 0;
}

// ── how the steps are spread ────────────────────────────────────────────────

int padded(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }

// Few heads take their steps in segments, as many as the chip holds workgroups at a
// time (`resident` a compute unit); each has four chunks at least, since the segments'
// states are found in a pass of its own. Heads that fill more than half of it do not:
// 1023 steps of 305 heads in one 108 us, in two 138.
Segments segments_of(const phz_ops* o, const AttendArgs& a, int chunk, int resident) {
  const int64_t heads = (int64_t)a.worlds * a.heads, chunks = ceil_div(a.steps, chunk);
  Segments s{};
  const int64_t want = std::max<int64_t>(1, std::min((int64_t)resident * o->cus / heads, chunks / 4));
  s.chunks = (int32_t)ceil_div(chunks, want);
  s.count = (int32_t)ceil_div(chunks, s.chunks);
  return s;
}

// Workgroups of a kernel that a compute unit holds.
template <class Kernel>
int resident_of(Kernel kernel, int threads) {
  int n = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, (const void*)kernel, threads, 0) != hipSuccess) {
    (void)hipGetLastError();
    return 1;
  }
  return std::max(n, 1);
}

// Calls f with the padded sizes as constants.
template <class F>
void with_size(int n, F&& f) {
  if (n <= 32) f(std::integral_constant<int, 32>());
  else if (n <= 64) f(std::integral_constant<int, 64>());
  else f(std::integral_constant<int, 128>());
}

// A call's pieces of workspace, each at a multiple of 256 bytes.
struct Pieces {
  int64_t size = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = size;
    size += ceil_div(bytes, 256) * 256;
    return at;
  }
};

template <class E>
int forward(phz_ops* o, hipStream_t stream, const AttendArgs& a) {
  const int64_t heads = (int64_t)a.worlds * a.heads, state = (int64_t)padded(a.nk) * padded(a.nv) * 4;
  int resident = 1;
  with_size(a.nk, [&](auto dk) {
    with_size(a.nv, [&](auto dv) {
      static const int n = resident_of(attend_chunks<E, dk(), dv()>, dv() * 4);
      resident = n;
    });
  });
  Segments seg = segments_of(o, a, Kind<E>::C, resident);
  const int slots = seg.count - 1;
  Pieces p;
  const int64_t flags = p.take((seg.count + slots) * heads * 4), decay = p.take(slots * heads * 4), states = p.take(slots * heads * state);
  char* work = o->workspace(stream, p.size);
  if (!work) return 1;
  seg.flags = (uint32_t*)(work + flags);
  seg.state_flags = seg.flags + seg.count * heads;
  seg.decay = (float*)(work + decay);
  seg.states = (float*)(work + states);
  with_size(a.nk, [&](auto dk) {
    with_size(a.nv, [&](auto dv) {
      constexpr int DK = dk(), DV = dv();
      if (slots) {
        const Roles x{a.k, a.v, a.nk, a.nv, a.nv, 1, a.s0};
        hipLaunchKernelGGL((segment_states<E, DK, DV, ADDS>), dim3((unsigned)(heads * slots)), dim3(DV * 4), 0, stream, a, x, seg,
                           nullptr);
        hipLaunchKernelGGL((join_segments<DK, DV>), dim3((unsigned)(heads * (DK * DV / 256))), dim3(256), 0, stream, a, x, seg, false);
      }
      hipLaunchKernelGGL((attend_chunks<E, DK, DV>), dim3((unsigned)(heads * seg.count)), dim3(DV * 4), 0, stream, a, seg);
    });
  });
  if (!launched(o, "linear attention")) return 1;
  AttendArgs again = a;
  again.flags = seg.flags;
  hipLaunchKernelGGL(attend_sequential<E>, dim3((unsigned)std::min<int64_t>(heads, 2 * o->cus)), dim3(512), 0, stream, again,
                     seg.count + slots);
  return launched(o, "linear attention") ? 0 : 1;
}

// dq, dk and dv of shared heads go through f32 sums of each head's own.
template <class E>
int backward(phz_ops* o, hipStream_t stream, AttendArgs a) {
  const Rows outs[3] = {a.dq, a.dk, a.dv};
  const int64_t T = a.steps, heads = (int64_t)a.worlds * a.heads, state = (int64_t)padded(a.nk) * padded(a.nv) * 4;
  const int sizes[3] = {a.nk, a.nk, a.nv};
  int resident = 1;
  with_size(a.nk, [&](auto dk) {
    with_size(a.nv, [&](auto dv) {
      static const int n = resident_of(attend_gradients<E, dk(), dv()>, kGradientThreads<dk(), dv()>);
      resident = n;
    });
  });
  Segments seg = segments_of(o, a, Kind<E>::C, resident);
  const int64_t chunks = ceil_div(T, Kind<E>::C), slots = seg.count - 1;
  Pieces p;
  int64_t own[3];
  for (int i = 0; i < 3; i++) own[i] = outs[i].per > 1 ? p.take(T * heads * sizes[i] * 4) : -1;
  const int64_t flags = p.take((seg.count + 2 * slots) * heads * 4), decay = p.take(slots * heads * 4);
  const int64_t forth = p.take(slots * heads * state), back = p.take(slots * heads * state);
  const int64_t each = p.take(seg.chunks > 1 ? chunks * heads * state : 0);
  char* work = o->workspace(stream, p.size);
  if (!work) return 1;
  int wide = 0;
  Rows* to[3] = {&a.dq, &a.dk, &a.dv};
  for (int i = 0; i < 3; i++) {
    *to[i] = outs[i];
    if (own[i] >= 0) {
      wide |= 1 << i;
      *to[i] = Rows{work + own[i], heads * sizes[i], (int64_t)a.heads * sizes[i], 1};
    }
  }
  seg.flags = (uint32_t*)(work + flags);
  seg.decay = (float*)(work + decay);
  with_size(a.nk, [&](auto dk) {
    with_size(a.nv, [&](auto dv) {
      constexpr int DK = dk(), DV = dv();
      const unsigned join = (unsigned)(heads * (DK * DV / 256)), most = (unsigned)(heads * seg.count);
      // States have rows of values here, as dq reads them.
      const Roles s{a.v, a.k, a.nv, a.nk, 1, a.nv, a.s0}, e{a.q, a.o, a.nk, a.nv, a.nv, 1, a.ds};
      if (slots) {
        seg.states = (float*)(work + forth);
        seg.state_flags = seg.flags + seg.count * heads;
        hipLaunchKernelGGL((segment_states<E, DV, DK, ADDS>), dim3((unsigned)(heads * slots)), dim3(DK * 4), 0, stream, a, s, seg,
                           nullptr);
        hipLaunchKernelGGL((join_segments<DV, DK>), dim3(join), dim3(256), 0, stream, a, s, seg, false);
      }
      if (seg.chunks > 1) {
        seg.states = (float*)(work + forth);
        hipLaunchKernelGGL((segment_states<E, DV, DK, EACH>), dim3(most), dim3(DK * 4), 0, stream, a, s, seg, (f32x4*)(work + each));
      }
      if (slots) {
        seg.states = (float*)(work + back);
        seg.state_flags = seg.flags + (seg.count + slots) * heads;
        hipLaunchKernelGGL((segment_states<E, DK, DV, BACK>), dim3((unsigned)(heads * slots)), dim3(DV * 4), 0, stream, a, e, seg,
                           nullptr);
        hipLaunchKernelGGL((join_segments<DK, DV>), dim3(join), dim3(256), 0, stream, a, e, seg, true);
      }
      hipLaunchKernelGGL((attend_gradients<E, DK, DV>), dim3(most), dim3(kGradientThreads<DK, DV>), 0, stream, a, seg,
                         (const float*)(work + forth), (const f32x4*)(work + each), wide);
    });
  });
  if (!launched(o, "linear attention backward")) return 1;
  AttendArgs again = a;
  again.flags = seg.flags;
  // (A compute unit holds one workgroup of it.)
  const Kept kept{(float*)(work + (seg.chunks > 1 ? each : forth)), heads * (state / 4), (int32_t)(state / 4), padded(a.nv) / 16,
                  seg.chunks > 1 ? 0 : 1, Kind<E>::C};
  hipLaunchKernelGGL(attend_sequential_backward<E>, dim3((unsigned)std::min<int64_t>(heads, o->cus)), dim3(512), 0, stream, again,
                     (int32_t)(seg.count + 2 * slots), wide, kept);
  for (int i = 0; i < 3; i++) {
    if (own[i] < 0) continue;
    const bool four = sizes[i] % 4 == 0;
    const unsigned n = (unsigned)std::min<int64_t>(ceil_div(T * heads / outs[i].per * sizes[i], four ? 1024 : 256), 16 * o->cus);
    hipLaunchKernelGGL((four ? join_heads<E, 4> : join_heads<E, 1>), dim3(n), dim3(256), 0, stream, (const float*)to[i]->p, outs[i],
                       T * a.worlds, a.worlds, a.heads, sizes[i]);
  }
  return launched(o, "linear attention backward") ? 0 : 1;
}

}  // namespace

extern "C" {

int phz_linear_attention(phz_ops* o, void* stream_, const phz_attention_cfg* cfg, const phz_tensor* q, const phz_tensor* k,
                         const phz_tensor* v, const phz_tensor* g, const phz_tensor* s0, const phz_tensor* reset,
                         const phz_tensor* out, const phz_tensor* s_last) {
  return guarded(o, [&] {
    AttendArgs a{};
    if (!take(o, cfg, q, k, v, g, reset, 3, &a)) return 1;
    const Want like{3, {a.steps, a.worlds, (int64_t)a.heads * a.nv}, q->dtype, true, true};
    if (!check(o, "o", out, like) || !take_states(o, "s0", s0, false, a, &a.s0) ||
        !take_states(o, "s_last", s_last, true, a, &a.s1) ||
        !all_apart(o, {{"o", out}, {"s_last", s_last}},
                   {{"q", q}, {"k", k}, {"v", v}, {"g", g}, {"s0", s0}, {"reset", reset}}))
      return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (a.worlds == 0) return 0;
    a.o = Rows{out->data, out->stride[0], out->stride[1], 1};
    auto stream = (hipStream_t)stream_;
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    return by_worlds(a, elem_bytes(q->dtype), [&](const AttendArgs& x) {
      if (x.steps == 0) {
        if (x.s1.p)
          hipLaunchKernelGGL(copy_states, dim3(x.worlds * x.heads), dim3(256), 0, stream, x.s0, x.s1, x.heads, x.nk * x.nv);
        return launched(o, "linear attention") ? 0 : 1;
      }
      return q->dtype == PHZ_F32 ? forward<float>(o, stream, x) : forward<bf16>(o, stream, x);
    });
  });
}

int phz_linear_attention_backward(phz_ops* o, void* stream_, const phz_attention_cfg* cfg, const phz_tensor* d_o,
                                  const phz_tensor* ds, const phz_tensor* q, const phz_tensor* k, const phz_tensor* v,
                                  const phz_tensor* g, const phz_tensor* s0, const phz_tensor* reset, const phz_tensor* dq,
                                  const phz_tensor* dk, const phz_tensor* dv, const phz_tensor* dg, const phz_tensor* ds0) {
  return guarded(o, [&] {
    AttendArgs a{};
    if (!take(o, cfg, q, k, v, g, reset, 3, &a)) return 1;
    const int64_t T = a.steps, B = a.worlds, H = a.heads;
    const Want grad{3, {T, B, H * a.nv}, q->dtype, true, false};
    const Want gates{3, {T, B, H}, PHZ_F32, false, true};
    if (!check(o, "do", d_o, grad)) return 1;
    for (const auto& x : {std::pair<Named, const phz_tensor*>{{"dq", dq}, q}, {{"dk", dk}, k}, {{"dv", dv}, v}})
      if (!check(o, x.first.name, x.first.t, Want{3, {T, B, x.second->size[2]}, q->dtype, true, true})) return 1;
    if ((dg && !check(o, "dg", dg, gates)) || !take_states(o, "s0", s0, false, a, &a.s0) ||
        !take_states(o, "ds", ds, false, a, &a.ds) || !take_states(o, "ds0", ds0, true, a, &a.ds0) ||
        !all_apart(o, {{"dq", dq}, {"dk", dk}, {"dv", dv}, {"dg", dg}, {"ds0", ds0}},
                   {{"do", d_o}, {"ds", ds}, {"q", q}, {"k", k}, {"v", v}, {"g", g}, {"s0", s0}, {"reset", reset}}))
      return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (B == 0) return 0;
    auto stream = (hipStream_t)stream_;
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    a.o = Rows{d_o->data, d_o->stride[0], d_o->stride[1], 1};
    if (dg) a.dg = (float*)dg->data, a.dg_t = dg->stride[0], a.dg_b = dg->stride[1], a.dg_h = dg->stride[2];
    a.dq = Rows{dq->data, dq->stride[0], dq->stride[1], a.q.per};
    a.dk = Rows{dk->data, dk->stride[0], dk->stride[1], a.k.per};
    a.dv = Rows{dv->data, dv->stride[0], dv->stride[1], a.v.per};
    return by_worlds(a, elem_bytes(q->dtype), [&](const AttendArgs& x) {
      if (x.steps == 0) {
        if (x.ds0.p)
          hipLaunchKernelGGL(copy_states, dim3(x.worlds * x.heads), dim3(256), 0, stream, x.ds, x.ds0, x.heads, x.nk * x.nv);
        return launched(o, "linear attention backward") ? 0 : 1;
      }
      return q->dtype == PHZ_F32 ? backward<float>(o, stream, x) : backward<bf16>(o, stream, x);
    });
  });
}

int phz_linear_attention_step(phz_ops* o, void* stream_, const phz_attention_cfg* cfg, const phz_tensor* q,
                              const phz_tensor* k, const phz_tensor* v, const phz_tensor* g, const phz_tensor* reset,
                              const phz_tensor* s, const phz_tensor* out) {
  return guarded(o, [&] {
    AttendArgs a{};
    if (!take(o, cfg, q, k, v, g, reset, 2, &a)) return 1;
    const Want like{2, {a.worlds, (int64_t)a.heads * a.nv, 0}, q->dtype, true, true};
    if (!s) return o->fail("s is missing");
    if (!check(o, "o", out, like) || !take_states(o, "s", s, true, a, &a.s1) ||
        !all_apart(o, {{"s", s}, {"o", out}}, {{"q", q}, {"k", k}, {"v", v}, {"g", g}, {"reset", reset}}))
      return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (a.worlds == 0) return 0;
    a.o = Rows{out->data, 0, out->stride[0], 1};
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    return by_worlds(a, elem_bytes(q->dtype), [&](const AttendArgs& x) {
      const int64_t all = (int64_t)x.worlds * x.heads;
      // Few heads: several workgroups to one, of 16 columns at least.
      int width = (x.nv + 3) / 4 * 4;
      while (all * ceil_div(x.nv, width) < 2 * o->cus && width % 32 == 0) width /= 2;
      const int parts = (int)ceil_div(x.nv, width);
      hipLaunchKernelGGL((q->dtype == PHZ_F32 ? attend_step<float> : attend_step<bf16>), dim3((unsigned)(all * parts)),
                         dim3(kStepThreads), 0, (hipStream_t)stream_, x, parts, width);
      return launched(o, "linear attention step") ? 0 : 1;
    });
  });
}

}  // extern "C"
