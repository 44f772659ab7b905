// phz_scan.hip — the gated linear recurrence over rollouts, forward and
// backward, and its single step.
//
//   forward   h_t = c_t h_{t-1} + u_t                       t = 0 .. T-1
//   backward  e_t = dh_t + k_{t+1},  k_t = c_t e_t           t = T-1 .. 0
//             dx_t = (1 - c_t) e_t,  dz_t = e_t (h_{t-1} - x_t) c_t (1 - c_t)
//             (decay: dx_t = e_t, dz_t = e_t h_{t-1}),  dh0 = k_0
//
// with c = sigmoid(z), u = (1 - c) x or c = z, u = x, and h_{t-1} := 0 where an
// episode begins. Both directions are one affine recurrence per channel,
// s <- c s + v, over the steps in processing order; a span of steps composes to
// s <- A s + H with A the product of its c. The layout of the work follows:
//
//   lane    VEC neighbouring channels of one world; the state in f32 registers
//   wave    64 lanes, U steps loaded ahead of the ones being computed
//   group   NW waves (4 or 16) take NW consecutive runs of U steps of the same channels
//           (a slab): each wave composes its run from registers, the runs'
//           (A, H) meet in LDS, and each wave then runs its steps from the
//           state that the earlier ones leave. The data is read once.
//   chunk   where the channels do not fill the chip, the steps are split in S
//           chunks over the grid: one pass composes each chunk, the second
//           starts each chunk from its predecessors' (A, H), folded in order.
//           That pass visits the chunks in the opposite order, so what the
//           first one read last is still in the memory-side cache.
//
// Every composition has a fixed order, so results do not depend on timing.
#include "phz_ops.h"

#include <algorithm>

using namespace phzop;

namespace {

constexpr int kWaveLanes = 64;

// How waves share a sequence's steps.
enum Spread {
  ALONE = 1,   // a wave takes all of them
  CHUNKS = 4,  // a group of four shares a slab, and takes one of several chunks
  SLABS = 16   // a group of sixteen shares a slab, and takes all of them
};

struct ScanArgs {
  const void *z, *x, *h, *dh;   // h and dh: backward only
  void *o1, *o2;                // h | dz, dx
  const float* start;           // h0 | dh_last, or null
  const float* h0;              // backward: the state before the first step, or null
  float* end;                   // h_last | dh0, or null
  const uint8_t* reset;
  int64_t z_t, z_b, x_t, x_b, h_t, h_b, dh_t, dh_b, o1_t, o1_b, o2_t, o2_b, r_t, r_b, start_b, h0_b, end_b;
  int64_t lanes;                // worlds * groups
  int32_t steps, width, groups; // groups: lanes that cover one world's width
  int32_t chunk, chunks;        // steps per chunk
  float* agg;                   // [chunks][chunk_words][lanes][VEC]: each chunk's A, H (decay: m, H, e of A = m 2^e)
};
constexpr int chunk_words(int form) { return form == PHZ_GATE_DECAY ? 3 : 2; }

// A span in which an episode begins keeps nothing of the state before it, be
// that infinite or NaN: its A is this NaN, and stands for "forget", which a
// product that underflows to 0 does not. (A gate that is NaN makes H NaN, so
// no other NaN in A matters.) A state of 0 passes a span as 0.
constexpr uint32_t kForget = 0x7fc5a5a5u;
__device__ __forceinline__ bool forgets(float a) { return __builtin_bit_cast(uint32_t, a) == kForget; }
__device__ __forceinline__ float compose(float a, float s, float h) {
  return forgets(a) || s == 0.0f ? h : fmaf(a, s, h);
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

// A where f32 does not hold it: m 2^e, with 1 <= |m| < 2, or 0. In the decay form
// a product of gates may leave f32's range, and come back, where product times
// state does not (130 gates of 2 on a state of 0.001, then 130 of 1/2). Sigmoid
// gates are at most 1: a product below f32's range never grows again, and what it
// loses is below 2^-126 of the state.
struct Wide {
  float m = 1.0f;
  int32_t e = 0;
  // A run of these between settles: each at most halves m.
  __device__ __forceinline__ void times(float c) {
    m *= __builtin_amdgcn_frexp_mantf(c);
    e += __builtin_amdgcn_frexp_expf(c);
  }
  __device__ __forceinline__ void settle() {
    e = min(max(e + __builtin_amdgcn_frexp_expf(m) - 1, -(1 << 30)), 1 << 30);
    m = 2.0f * __builtin_amdgcn_frexp_mantf(m);
  }
  __device__ __forceinline__ float compose(float s, float h) const {
    return forgets(m) ? h : fmaf(m, __builtin_amdgcn_ldexpf(s, e), h);
  }
};
// A run's A is plain f32 where all its gates are within 2^-15 and 2^15, so that
// the products of its up to eight are in range; else it is this mark, and the
// Wide product stands beside it.
constexpr uint32_t kApart = 0x7fc5a5a6u;
constexpr uint32_t kNarrowLeast = 0x38000000u, kNarrowMost = 0x47000000u;  // 2^-15 and 2^15

// One step's affine map and outputs. `s` is h (forward) or k (backward).
template <int FORM>
struct Step;

template <>
struct Step<PHZ_GATE_SIGMOID> {
  // The gate as its smaller side c with z's sign (signed_gate):
  // h' = h + c (x - h) where the gate keeps, x + c (h - x) where it writes, so
  // a gate at rest leaves the state exactly as it is. Differences are taken of
  // halves, which stay in f32's range where x - h does not; the bits are the same.
  static __device__ __forceinline__ float gate(float z) { return signed_gate(z); }
  static __device__ __forceinline__ float keep(float q) { return __float_as_int(q) < 0 ? fabsf(q) : 1.0f - fabsf(q); }
  static __device__ __forceinline__ float write(float q) { return __float_as_int(q) < 0 ? 1.0f - fabsf(q) : fabsf(q); }
  static __device__ __forceinline__ float next(float h, float q, float x) {
    const bool w = __float_as_int(q) < 0;
    const float base = w ? x : h, other = w ? h : x;
    return fmaf(2.0f * fabsf(q), fmaf(-0.5f, base, 0.5f * other), base);
  }
  static __device__ __forceinline__ float dz(float e, float hp, float x, float q) {
    const float c = fabsf(q);
    return e * fmaf(-0.5f, x, 0.5f * hp) * (2.0f * c * (1.0f - c));
  }
};

template <>
struct Step<PHZ_GATE_DECAY> {
  static __device__ __forceinline__ float gate(float z) { return z; }
  static __device__ __forceinline__ float keep(float q) { return q; }
  static __device__ __forceinline__ float write(float) { return 1.0f; }
  static __device__ __forceinline__ float next(float h, float q, float x) { return fmaf(q, h, x); }
  static __device__ __forceinline__ float dz(float e, float hp, float, float) { return e * hp; }
};

template <class E, int VEC>
__device__ __forceinline__ Pack<E, VEC> load(const void* base, int64_t at) {
  return *(const Pack<E, VEC>*)((const E*)base + at);
}
template <class E, int VEC>
__device__ __forceinline__ void store(void* base, int64_t at, const float* v) {
  Pack<E, VEC> p;
#pragma unroll
  for (int i = 0; i < VEC; i++) p.v[i] = from_f32<E>(v[i]);
  *(Pack<E, VEC>*)((E*)base + at) = p;
}

// A run of U steps as loaded. Backward: a = dh and hp = h_{t-1}; the decay
// form's gradients do not need x.
template <class E, int VEC, int U, bool BACK, bool NEED_X>
struct Run {
  Pack<E, VEC> z[U], x[NEED_X ? U : 1], a[BACK ? U : 1], hp[BACK ? U : 1];
  // Whether episodes begin, as loaded: step u in reset[u], or, where a wave's
  // lanes are of one world, step u in lane u's reset[0].
  uint32_t reset[U];
};

template <class E, int FORM, bool BACK, int VEC, int NW, int U, bool AGG>
__global__ __launch_bounds__(NW * kWaveLanes) void gated_scan_kernel(ScanArgs p) {
  static_assert(NW > 1 || !AGG, "chunks are of several waves");
  using S = Step<FORM>;
  constexpr bool kWide = FORM == PHZ_GATE_DECAY;
  constexpr int kWords = kWide ? 4 : 2;  // of a run in LDS: A, H, and m and e of an A apart
  constexpr int kChunkWords = chunk_words(FORM);
  // What a chunk's map needs: forward z, x; backward z and dh only.
  constexpr bool kNeedX = BACK ? (FORM == PHZ_GATE_SIGMOID && !AGG) : true;
  constexpr bool kNeedH = BACK && !AGG;
  using R = Run<E, VEC, U, BACK, kNeedX>;
  // Double-buffered, so one barrier a slab is enough.
  __shared__ float lds[NW > 1 ? 2 * NW * kWords * VEC * kWaveLanes : 1];

  const int lane = threadIdx.x & 63;
  const int wave = NW > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int64_t id = (int64_t)blockIdx.x * kWaveLanes + lane;
  const bool live = id < p.lanes;
  const int64_t idc = live ? id : p.lanes - 1;  // idle lanes follow the last one, and store nothing
  const int64_t b = idc / p.groups;
  // The last group of a world starts early where VEC does not divide the
  // width: its first channels are computed twice, to the same bits.
  const int d = min((int)(idc - b * p.groups) * VEC, p.width - VEC);
  const int chunk = p.chunks == 1 ? 0 : AGG ? (int)blockIdx.y : p.chunks - 1 - (int)blockIdx.y;
  const int first = chunk * p.chunk, last = min(p.steps, first + p.chunk);

  const E* z = (const E*)p.z + b * p.z_b + d;
  const E* x = kNeedX ? (const E*)p.x + b * p.x_b + d : nullptr;
  const E* dh = BACK ? (const E*)p.dh + b * p.dh_b + d : nullptr;
  const E* h = kNeedH ? (const E*)p.h + b * p.h_b + d : nullptr;
  const uint8_t* rs = p.reset ? p.reset + b * p.r_b : nullptr;

  auto step_of = [&](int i) { return (int64_t)(BACK ? p.steps - 1 - i : i); };
  float s[VEC];
  float prod[VEC];
  Wide wide[VEC];       // the same, where gates may be above 1
  bool forgot = false;  // the chunk so far (AGG)
#pragma unroll
  for (int v = 0; v < VEC; v++) s[v] = 0.0f, prod[v] = 1.0f;

  // The steps [from, to) themselves, one after the other. A span's H grows from
  // 0 and may leave f32's range, or a gate be infinite, where the state that
  // goes through the span stays finite: where A and H make a state that is not
  // finite of one that is, the steps decide. Once a state is not finite it stays
  // so until the next episode, so this is taken about once an episode at most.
  auto walk = [&](float st, int v, int from, int to) {
#pragma unroll 1
    for (int i = from; i < to; i++) {
      const int64_t t = step_of(i);
      const float q = S::gate(to_f32(z[t * p.z_t + v])), a = to_f32(BACK ? dh[t * p.dh_t + v] : x[t * p.x_t + v]);
      const bool rst = rs && rs[t * p.r_t];
      if (BACK) st = rst ? 0.0f : S::keep(q) * (a + st);
      else st = S::next(rst ? 0.0f : st, q, a);
    }
    return st;
  };
  // Channel v's state after the steps [from, to), whose map is (a, h). (An
  // infinite state stays so whatever finite inputs add, be the sum of those
  // alone the other infinity.)
  auto pass = [&](const Wide& a, float h, int v, int from, int to) {
    const float r = a.compose(s[v], fabsf(s[v]) == __builtin_inff() && fabsf(h) == __builtin_inff() && !forgets(a.m) ? 0.0f : h);
    s[v] = !forgets(a.m) && finite(s[v]) && !finite(r) ? walk(s[v], v, from, to) : r;
  };

  if (!AGG) {
    if (p.start) {
#pragma unroll
      for (int v = 0; v < VEC; v++) s[v] = p.start[b * p.start_b + d + v];
    }
    // The state that the earlier chunks leave.
    constexpr int kAhead = 32 / VEC;  // chunks whose (A, H) are loaded together
    constexpr bool kWideChunks = kWide && NW == CHUNKS;
    const int64_t word = p.lanes * VEC;
    bool odd = false;
    for (int j0 = 0; j0 < chunk; j0 += kAhead) {
      Pack<float, VEC> A[kAhead], X[kWideChunks ? kAhead : 1], H[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const float* a = p.agg + ((int64_t)min(j0 + j, chunk - 1) * kChunkWords * p.lanes + idc) * VEC;
        A[j] = load<float, VEC>(a, 0), H[j] = load<float, VEC>(a, word);
        if constexpr (kWideChunks) X[j] = load<float, VEC>(a, 2 * word);
      }
#pragma unroll
      for (int j = 0; j < kAhead; j++)
        if (j0 + j < chunk) {
#pragma unroll
          for (int v = 0; v < VEC; v++) {
            if constexpr (kWideChunks) {
              s[v] = Wide{A[j].v[v], __builtin_bit_cast(int32_t, X[j].v[v])}.compose(s[v], H[j].v[v]);
              odd = odd || !finite(s[v]);
            } else {
              s[v] = compose(A[j].v[v], s[v], H[j].v[v]);
            }
          }
        }
    }
    if constexpr (kWideChunks) {
      if (odd) {
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          s[v] = p.start ? p.start[b * p.start_b + d + v] : 0.0f;
#pragma unroll 1
          for (int j = 0; j < chunk; j++) {
            const float* a = p.agg + ((int64_t)j * kChunkWords * p.lanes + idc) * VEC + v;
            pass(Wide{a[0], __builtin_bit_cast(int32_t, a[2 * word])}, a[word], v, j * p.chunk, (j + 1) * p.chunk);
          }
        }
      }
    }
  }

  const bool one_world = __all(b == (int64_t)__builtin_amdgcn_readfirstlane((int)b));
  auto fetch = [&](R& r, int base) {
    if (rs && one_world) r.reset[0] = lane < U && base + lane < last ? rs[step_of(base + lane) * p.r_t] : 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = base + u;
      if (i < last) {
        const int64_t t = step_of(i);
        r.z[u] = load<E, VEC>(z, t * p.z_t);
        if (kNeedX) r.x[u] = load<E, VEC>(x, t * p.x_t);
        if (BACK) r.a[u] = load<E, VEC>(dh, t * p.dh_t);
        if (kNeedH && t > 0) r.hp[u] = load<E, VEC>(h, (t - 1) * p.h_t);
        if (rs && !one_world) r.reset[u] = rs[t * p.r_t];
      }
    }
  };

  const int stride = NW * U;
  R cur, nxt;
  int base = first + wave * U;
  fetch(cur, base);
  int buf = 0;
  for (int slab = first; slab < last; slab += stride, base += stride) {
    if (slab + stride < last) fetch(nxt, base + stride);
    uint32_t reset = 0;  // bit u: an episode begins at step u of the run
    if (rs && one_world) {
      reset = (uint32_t)__ballot(cur.reset[0] != 0);
    } else if (rs) {
#pragma unroll
      for (int u = 0; u < U; u++) reset |= (base + u < last && cur.reset[u] ? 1u : 0u) << u;
    }
    float q[U][VEC];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int v = 0; v < VEC; v++) q[u][v] = S::gate(to_f32(cur.z[u].v[v]));

    // One step of the affine recurrence: forward to h_t, backward to k_t.
    auto advance = [&](float st, int u, int v, bool rst) {
      if (BACK) return rst ? 0.0f : S::keep(q[u][v]) * (to_f32(cur.a[u].v[v]) + st);
      return S::next(rst ? 0.0f : st, q[u][v], to_f32(cur.x[kNeedX ? u : 0].v[v]));
    };

    if constexpr (NW > 1) {
      // Compose this wave's run.
      float A[VEC], H[VEC];
      bool forget = false;
      uint32_t reach = 0;  // of the gates' magnitudes above the least that is narrow
#pragma unroll
      for (int v = 0; v < VEC; v++) A[v] = 1.0f, H[v] = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
        if (base + u < last) {
          const bool rst = (reset >> u) & 1u;
#pragma unroll
          for (int v = 0; v < VEC; v++) {
            H[v] = advance(H[v], u, v, rst);
            A[v] *= S::keep(q[u][v]);
            if (kWide) reach = max(reach, 2 * __builtin_bit_cast(uint32_t, q[u][v]) - 2 * kNarrowLeast);
          }
          forget = forget || rst;
        }
      constexpr int kWord = kWaveLanes * VEC;
      float* mine = lds + buf * (NW * kWords * kWord);
      auto word_of = [&](int w, int i, int v) -> float& { return mine[(w * kWords + i) * kWord + lane * VEC + v]; };
      if (kWide && !forget && reach > 2 * (kNarrowMost - kNarrowLeast)) {
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          Wide a;
#pragma unroll
          for (int u = 0; u < U; u++)
            if (base + u < last) a.times(q[u][v]);
          a.settle();
          word_of(wave, 2, v) = a.m, word_of(wave, 3, v) = __builtin_bit_cast(float, a.e);
          A[v] = __builtin_bit_cast(float, kApart);
        }
      }
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        word_of(wave, 0, v) = forget ? __builtin_bit_cast(float, kForget) : A[v];
        word_of(wave, 1, v) = H[v];
      }
      __syncthreads();
      // Fold every run of the slab in order; keep the state before this
      // wave's own.
      float before[VEC], slab_s[VEC];
      float odd = 0.0f;  // NaN where some state is not finite
#pragma unroll
      for (int v = 0; v < VEC; v++) before[v] = slab_s[v] = s[v];
#pragma unroll
      for (int w = 0; w < NW; w++) {
        if (w == wave) {
#pragma unroll
          for (int v = 0; v < VEC; v++) before[v] = s[v];
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
          const float a = word_of(w, 0, v);
          s[v] = compose(a, s[v], word_of(w, 1, v));
          if (kWide) odd = fmaf(0.0f, s[v], odd);
          if (AGG) {
            forgot = forgot || forgets(a);
            prod[v] *= a;
          }
        }
      }
      if constexpr (kWide) {
        auto run_of = [&](int w, int v) {
          const float a = word_of(w, 0, v);
          Wide r{a, 0};
          if (__builtin_bit_cast(uint32_t, a) == kApart)
            r.m = word_of(w, 2, v), r.e = __builtin_bit_cast(int32_t, word_of(w, 3, v));
          return r;
        };
        // An A apart, or a state that is not finite: each run with care.
        if (odd != odd) {
#pragma unroll
          for (int v = 0; v < VEC; v++) {
            s[v] = slab_s[v];
#pragma unroll 1
            for (int w = 0; w < NW; w++) {
              if (w == wave) before[v] = s[v];
              pass(run_of(w, v), word_of(w, 1, v), v, min(slab + w * U, last), min(slab + (w + 1) * U, last));
            }
          }
        }
        if (AGG && wave == 0) {  // who stores it
#pragma unroll
          for (int w = 0; w < NW; w++)
#pragma unroll
            for (int v = 0; v < VEC; v++) {
              const Wide r = run_of(w, v);
              wide[v].times(r.m);
              wide[v].e += r.e;
            }
#pragma unroll
          for (int v = 0; v < VEC; v++) wide[v].settle();
        }
      }
      if (!AGG) {
        // The outputs, from the state before the run; s stays the slab's end.
#pragma unroll
        for (int u = 0; u < U; u++)
          if (base + u < last) {
            const int64_t t = step_of(base + u);
            const bool rst = (reset >> u) & 1u;
            if (BACK) {
              float dz[VEC], dx[VEC];
#pragma unroll
              for (int v = 0; v < VEC; v++) {
                const float e = to_f32(cur.a[u].v[v]) + before[v];
                float hp = 0.0f;
                if (!rst) {
                  if (t > 0) hp = to_f32(cur.hp[kNeedH ? u : 0].v[v]);
                  else if (p.h0) hp = p.h0[b * p.h0_b + d + v];
                }
                dz[v] = S::dz(e, hp, kNeedX ? to_f32(cur.x[kNeedX ? u : 0].v[v]) : 0.0f, q[u][v]);
                dx[v] = S::write(q[u][v]) * e;
                before[v] = rst ? 0.0f : S::keep(q[u][v]) * e;
              }
              if (live) {
                store<E, VEC>(p.o1, b * p.o1_b + d + t * p.o1_t, dz);
                store<E, VEC>(p.o2, b * p.o2_b + d + t * p.o2_t, dx);
              }
            } else {
#pragma unroll
              for (int v = 0; v < VEC; v++) before[v] = advance(before[v], u, v, rst);
              if (live) store<E, VEC>(p.o1, b * p.o1_b + d + t * p.o1_t, before);
            }
          }
      }
      buf ^= 1;
    } else {
#pragma unroll
      for (int u = 0; u < U; u++)
        if (base + u < last) {
          const int64_t t = step_of(base + u);
          const bool rst = (reset >> u) & 1u;
          if (BACK) {
            float dz[VEC], dx[VEC];
#pragma unroll
            for (int v = 0; v < VEC; v++) {
              const float e = to_f32(cur.a[u].v[v]) + s[v];
              float hp = 0.0f;
              if (!rst) {
                if (t > 0) hp = to_f32(cur.hp[kNeedH ? u : 0].v[v]);
                else if (p.h0) hp = p.h0[b * p.h0_b + d + v];
              }
              dz[v] = S::dz(e, hp, kNeedX ? to_f32(cur.x[kNeedX ? u : 0].v[v]) : 0.0f, q[u][v]);
              dx[v] = S::write(q[u][v]) * e;
              s[v] = rst ? 0.0f : S::keep(q[u][v]) * e;
            }
            if (live) {
              store<E, VEC>(p.o1, b * p.o1_b + d + t * p.o1_t, dz);
              store<E, VEC>(p.o2, b * p.o2_b + d + t * p.o2_t, dx);
            }
          } else {
#pragma unroll
            for (int v = 0; v < VEC; v++) s[v] = advance(s[v], u, v, rst);
            if (live) store<E, VEC>(p.o1, b * p.o1_b + d + t * p.o1_t, s);
          }
        }
    }
    cur = nxt;
  }

  if (AGG) {
    if (live && wave == 0) {
      const int64_t word = p.lanes * VEC;
      float* a = p.agg + ((int64_t)chunk * kChunkWords * p.lanes + id) * VEC;
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        a[v] = forgot ? __builtin_bit_cast(float, kForget) : kWide ? wide[v].m : prod[v], a[word + v] = s[v];
        if (kWide) a[2 * word + v] = __builtin_bit_cast(float, wide[v].e);
      }
    }
  } else if (p.end && chunk == p.chunks - 1 && live && wave == 0) {
#pragma unroll
    for (int v = 0; v < VEC; v++) p.end[b * p.end_b + d + v] = s[v];
  }
}

// The steps that each wave loads ahead of the ones it computes: more hide more
// of memory's latency, and leave registers for fewer waves.
template <class E>
constexpr int run_steps(bool back, int spread) {
  return spread == ALONE ? (back ? 2 : 4) : back && sizeof(E) == 4 ? 4 : 8;
}

template <class E, int FORM, bool BACK, int VEC, int NW>
void launch_as(const ScanArgs& p, hipStream_t stream) {
  constexpr int U = run_steps<E>(BACK, NW);
  const unsigned groups = (unsigned)ceil_div(p.lanes, kWaveLanes);
  if constexpr (NW == CHUNKS) {
    if (p.chunks > 1)  // nobody starts from the last chunk
      hipLaunchKernelGGL((gated_scan_kernel<E, FORM, BACK, VEC, NW, U, true>), dim3(groups, p.chunks - 1), dim3(NW * 64), 0,
                         stream, p);
  }
  hipLaunchKernelGGL((gated_scan_kernel<E, FORM, BACK, VEC, NW, U, false>), dim3(groups, p.chunks), dim3(NW * 64), 0, stream,
                     p);
}

template <class E, int FORM, bool BACK>
void launch(const ScanArgs& p, int vec, int spread, hipStream_t stream) {
  if (spread == SLABS) vec == 2 ? launch_as<E, FORM, BACK, 2, SLABS>(p, stream) : launch_as<E, FORM, BACK, 1, SLABS>(p, stream);
  else if (spread == CHUNKS)
    vec == 4 ? launch_as<E, FORM, BACK, 4, CHUNKS>(p, stream) : launch_as<E, FORM, BACK, 1, CHUNKS>(p, stream);
  else vec == 4 ? launch_as<E, FORM, BACK, 4, ALONE>(p, stream) : launch_as<E, FORM, BACK, 1, ALONE>(p, stream);
}

template <class E>
void launch_any(const ScanArgs& p, int form, bool back, int vec, int spread, hipStream_t stream) {
  auto go = [&](auto f, auto bk) { launch<E, decltype(f)::value, decltype(bk)::value>(p, vec, spread, stream); };
  using Sg = std::integral_constant<int, PHZ_GATE_SIGMOID>;
  using Dc = std::integral_constant<int, PHZ_GATE_DECAY>;
  if (form == PHZ_GATE_SIGMOID) back ? go(Sg{}, std::true_type{}) : go(Sg{}, std::false_type{});
  else back ? go(Dc{}, std::true_type{}) : go(Dc{}, std::false_type{});
}

// What is left where there are no steps: the last state is the first one.
__global__ void copy_rows(const float* src, int64_t src_b, float* dst, int64_t dst_b, int64_t rows, int32_t width) {
  const int64_t n = rows * width;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / width, c = i - r * width;
    dst[r * dst_b + c] = src ? src[r * src_b + c] : 0.0f;
  }
}

// One step for every channel, the state replaced in place: 16 bytes a channel
// in f32. Bound by a launch's latency below about a million channels (1024 x
// 256: 2.7 us, 0.9 of them at a copy's rate), by memory above.
template <class E, int FORM, int VEC>
__global__ __launch_bounds__(256) void gated_step_kernel(const void* z, int64_t z_b, const void* x, int64_t x_b,
                                                         const uint8_t* reset, int64_t r_b, float* h, int64_t h_b,
                                                         int64_t lanes, int32_t groups, int32_t width) {
  using S = Step<FORM>;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < lanes; id += (int64_t)gridDim.x * 256) {
    const int64_t b = id / groups;
    const int d = (int)(id - b * groups) * VEC;
    const bool rst = reset && reset[b * r_b];
    float* hs = h + b * h_b + d;
    if (d + VEC <= width) {
      const auto zv = load<E, VEC>(z, b * z_b + d), xv = load<E, VEC>(x, b * x_b + d);
      auto hv = load<float, VEC>(hs, 0);
#pragma unroll
      for (int v = 0; v < VEC; v++)
        hv.v[v] = S::next(rst ? 0.0f : hv.v[v], S::gate(to_f32(zv.v[v])), to_f32(xv.v[v]));
      *(Pack<float, VEC>*)hs = hv;
    } else {
      for (int v = 0; d + v < width; v++)
        hs[v] = S::next(rst ? 0.0f : hs[v], S::gate(to_f32(((const E*)z)[b * z_b + d + v])),
                        to_f32(((const E*)x)[b * x_b + d + v]));
    }
  }
}

// Which spread. Waves alone where the channels, four a lane, give four waves a
// compute unit; groups of sixteen, two channels a lane, where those are one for
// every second compute unit, so that the data is read once; below, chunks of at
// least two slabs up to 16 waves a compute unit in all, at most 64 chunks (each
// start folds its predecessors), of lanes of four channels, or of one where
// even so the waves would be few.
// One MI355X, us:                            alone  sixteen  chunks  bytes at a copy's rate
//   64 x 4096 x 256 f32, forward             159    214      164     173
//   512 x 64 x 512 f32, forward              155    39       63      43
//   512 x 64 x 512 f32, backward             393    87       100     86
//   1023 x 61 x 515 bf16 decay, backward     662    96       119     69
//   4000 x 100 x 128 f32, backward           .      448      372     264
//   32768 x 1 x 2048 bf16, forward           .      1261     167     86
//   4096 x 1 x 512 f32, forward              .      162      15.8    5.4
// (sigmoid where not said otherwise; decay takes less, though the exponents of its
// products are 1 to 7% of its sixteen and 2 to 15% of its chunks.)
// What chunks cost above their bytes is the second reading.
struct Plan {
  int vec, spread, chunk, chunks;
  int64_t groups, lanes;
};

Plan plan(const phz_ops* o, int dtype, int64_t steps, int64_t worlds, int64_t width, bool back) {
  Plan p{};
  auto lay = [&](int vec, Spread spread) {
    p.spread = spread;
    p.vec = width >= vec ? vec : 1;
    p.groups = ceil_div(width, p.vec);
    p.lanes = worlds * p.groups;
    p.chunk = (int)steps;
    p.chunks = 1;
    return ceil_div(p.lanes, kWaveLanes);
  };
  if (lay(4, ALONE) >= 4 * o->cus || steps <= 16) return p;
  if (lay(2, SLABS) >= o->cus / 2) return p;
  for (int vec : {4, 1}) {
    const int64_t want = 16ll * o->cus, waves = lay(vec, CHUNKS) * CHUNKS;
    const int64_t slab = CHUNKS * (dtype == PHZ_F32 ? run_steps<float>(back, CHUNKS) : run_steps<bf16>(back, CHUNKS));
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({ceil_div(want, waves), steps / (2 * slab), 64}));
    p.chunk = (int)(ceil_div(ceil_div(steps, chunks), slab) * slab);
    p.chunks = (int)ceil_div(steps, p.chunk);
    if (waves * p.chunks >= want / 2) break;
  }
  return p;
}

bool check_form(phz_ops* o, int form) {
  if (form == PHZ_GATE_SIGMOID || form == PHZ_GATE_DECAY) return true;
  o->err = "unknown gate form";
  return false;
}

bool check_type(phz_ops* o, const char* name, const phz_tensor* t) {
  if (!t) return o->err = fmt("%s is missing", name), false;
  if (t->dtype == PHZ_F32 || t->dtype == PHZ_BF16) return true;
  o->err = fmt("%s is %s, expected f32 or bf16", name, dtype_name(t->dtype));
  return false;
}

bool check_limits(phz_ops* o, int64_t steps, int64_t worlds, int64_t width) {
  if (steps > 0x7fff0000ll || width > 0x7fff0000ll || worlds > 0x7fff0000ll)
    return o->err = "steps, worlds and width have to be below 2^31", false;
  // Lanes (of four channels) are counted in the launch's 32 bits.
  if (worlds * (width < 4 ? width : ceil_div(width, 4)) > 0xffff0000ll) return o->err = "too many channels", false;
  return true;
}

int scan(phz_ops* o, hipStream_t stream, int form, bool back, ScanArgs a, int dtype, int64_t steps, int64_t worlds,
         int64_t width) {
  if (worlds == 0 || width == 0) return 0;
  DeviceGuard g(o);
  if (!g.ok) return 1;
  if (steps == 0) {
    if (a.end) {
      const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(worlds * width, 256), 4096);
      hipLaunchKernelGGL(copy_rows, dim3(blocks), dim3(256), 0, stream, a.start, a.start_b, a.end, a.end_b, worlds,
                         (int32_t)width);
    }
    return launched(o, "gated scan") ? 0 : 1;
  }
  const Plan p = plan(o, dtype, steps, worlds, width, back);
  a.steps = (int32_t)steps;
  a.width = (int32_t)width;
  a.groups = (int32_t)p.groups;
  a.lanes = p.lanes;
  a.chunk = p.chunk;
  a.chunks = p.chunks;
  if (p.chunks > 1) {
    a.agg = (float*)o->workspace(stream, (uint64_t)p.chunks * chunk_words(form) * p.lanes * p.vec * sizeof(float));
    if (!a.agg) return 1;
  }
  if (dtype == PHZ_F32) launch_any<float>(a, form, back, p.vec, p.spread, stream);
  else launch_any<bf16>(a, form, back, p.vec, p.spread, stream);
  return launched(o, "gated scan") ? 0 : 1;
}

}  // namespace

extern "C" {

int phz_gated_scan(phz_ops* o, void* stream, int form, const phz_tensor* z, const phz_tensor* x, const phz_tensor* h0,
                   const phz_tensor* reset, const phz_tensor* h, const phz_tensor* h_last) {
  return guarded(o, [&] {
    if (!check_form(o, form) || !check_type(o, "z", z)) return 1;
    const Want in{3, {-1, -1, -1}, z->dtype, true, false};
    if (!check(o, "z", z, in)) return 1;
    const int64_t T = z->size[0], B = z->size[1], D = z->size[2];
    const Want like{3, {T, B, D}, z->dtype, true, false}, out{3, {T, B, D}, z->dtype, true, true};
    const Want row{2, {B, D, 0}, PHZ_F32, true, false}, row_out{2, {B, D, 0}, PHZ_F32, true, true};
    const Want mask{2, {T, B, 0}, PHZ_U8, false, false};
    if (!check(o, "x", x, like) || !check(o, "h", h, out) || (h0 && !check(o, "h0", h0, row)) ||
        (reset && !check(o, "reset", reset, mask)) || (h_last && !check(o, "h_last", h_last, row_out)) ||
        !check_limits(o, T, B, D))
      return 1;
    for (const phz_tensor* t : {h, h_last}) {
      const char* name = t == h ? "h" : "h_last";
      if (!apart(o, name, t, "z", z) || !apart(o, name, t, "x", x) || !apart(o, name, t, "h0", h0) ||
          !apart(o, name, t, "reset", reset))
        return 1;
    }
    if (!apart(o, "h", h, "h_last", h_last)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    ScanArgs a{};
    a.z = z->data, a.z_t = z->stride[0], a.z_b = z->stride[1];
    a.x = x->data, a.x_t = x->stride[0], a.x_b = x->stride[1];
    a.o1 = h->data, a.o1_t = h->stride[0], a.o1_b = h->stride[1];
    if (h0) a.start = (const float*)h0->data, a.start_b = h0->stride[0];
    if (h_last) a.end = (float*)h_last->data, a.end_b = h_last->stride[0];
    if (reset) a.reset = (const uint8_t*)reset->data, a.r_t = reset->stride[0], a.r_b = reset->stride[1];
    return scan(o, (hipStream_t)stream, form, false, a, z->dtype, T, B, D);
  });
}

int phz_gated_scan_backward(phz_ops* o, void* stream, int form, const phz_tensor* dh, const phz_tensor* dh_last,
                            const phz_tensor* z, const phz_tensor* x, const phz_tensor* h, const phz_tensor* h0,
                            const phz_tensor* reset, const phz_tensor* dz, const phz_tensor* dx, const phz_tensor* dh0) {
  return guarded(o, [&] {
    if (!check_form(o, form) || !check_type(o, "z", z)) return 1;
    const Want in{3, {-1, -1, -1}, z->dtype, true, false};
    if (!check(o, "z", z, in)) return 1;
    const int64_t T = z->size[0], B = z->size[1], D = z->size[2];
    const Want like{3, {T, B, D}, z->dtype, true, false}, out{3, {T, B, D}, z->dtype, true, true};
    const Want row{2, {B, D, 0}, PHZ_F32, true, false}, row_out{2, {B, D, 0}, PHZ_F32, true, true};
    const Want mask{2, {T, B, 0}, PHZ_U8, false, false};
    if (!check(o, "x", x, like) || !check(o, "h", h, like) || !check(o, "dh", dh, like) || !check(o, "dz", dz, out) ||
        !check(o, "dx", dx, out) || (h0 && !check(o, "h0", h0, row)) || (dh_last && !check(o, "dh_last", dh_last, row)) ||
        (reset && !check(o, "reset", reset, mask)) || (dh0 && !check(o, "dh0", dh0, row_out)) ||
        !check_limits(o, T, B, D))
      return 1;
    const struct { const char* name; const phz_tensor* t; } outs[] = {{"dz", dz}, {"dx", dx}, {"dh0", dh0}},
        ins[] = {{"dh", dh}, {"dh_last", dh_last}, {"z", z}, {"x", x}, {"h", h}, {"h0", h0}, {"reset", reset}};
    for (auto& u : outs)
      for (auto& v : ins)
        if (!apart(o, u.name, u.t, v.name, v.t)) return 1;
    if (!apart(o, "dz", dz, "dx", dx) || !apart(o, "dz", dz, "dh0", dh0) || !apart(o, "dx", dx, "dh0", dh0)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    ScanArgs a{};
    a.z = z->data, a.z_t = z->stride[0], a.z_b = z->stride[1];
    a.x = x->data, a.x_t = x->stride[0], a.x_b = x->stride[1];
    a.h = h->data, a.h_t = h->stride[0], a.h_b = h->stride[1];
    a.dh = dh->data, a.dh_t = dh->stride[0], a.dh_b = dh->stride[1];
    a.o1 = dz->data, a.o1_t = dz->stride[0], a.o1_b = dz->stride[1];
    a.o2 = dx->data, a.o2_t = dx->stride[0], a.o2_b = dx->stride[1];
    if (dh_last) a.start = (const float*)dh_last->data, a.start_b = dh_last->stride[0];
    if (h0) a.h0 = (const float*)h0->data, a.h0_b = h0->stride[0];
    if (dh0) a.end = (float*)dh0->data, a.end_b = dh0->stride[0];
    if (reset) a.reset = (const uint8_t*)reset->data, a.r_t = reset->stride[0], a.r_b = reset->stride[1];
    return scan(o, (hipStream_t)stream, form, true, a, z->dtype, T, B, D);
  });
}

int phz_gated_step(phz_ops* o, void* stream, int form, const phz_tensor* z, const phz_tensor* x,
                   const phz_tensor* reset, const phz_tensor* h) {
  return guarded(o, [&] {
    if (!check_form(o, form) || !check_type(o, "z", z)) return 1;
    if (!check(o, "z", z, Want{2, {-1, -1, 0}, z->dtype, true, false})) return 1;
    const int64_t B = z->size[0], D = z->size[1];
    if (!check(o, "x", x, Want{2, {B, D, 0}, z->dtype, true, false}) ||
        (reset && !check(o, "reset", reset, Want{1, {B, 0, 0}, PHZ_U8, false, false})) ||
        !check(o, "h", h, Want{2, {B, D, 0}, PHZ_F32, true, true}) || !check_limits(o, 1, B, D) ||
        !apart(o, "h", h, "z", z) || !apart(o, "h", h, "x", x) || !apart(o, "h", h, "reset", reset))
      return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (B == 0 || D == 0) return 0;
    DeviceGuard g(o);
    if (!g.ok) return 1;
    constexpr int VEC = 4;
    const int64_t groups = ceil_div(D, VEC), lanes = B * groups;
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(lanes, 256), 1 << 20);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, z->data, z->stride[0], x->data,
                         x->stride[0], reset ? (const uint8_t*)reset->data : nullptr, reset ? reset->stride[0] : 0,
                         (float*)h->data, h->stride[0], lanes, (int32_t)groups, (int32_t)D);
    };
    if (z->dtype == PHZ_F32)
      form == PHZ_GATE_SIGMOID ? go(gated_step_kernel<float, PHZ_GATE_SIGMOID, VEC>)
                               : go(gated_step_kernel<float, PHZ_GATE_DECAY, VEC>);
    else
      form == PHZ_GATE_SIGMOID ? go(gated_step_kernel<bf16, PHZ_GATE_SIGMOID, VEC>)
                               : go(gated_step_kernel<bf16, PHZ_GATE_DECAY, VEC>);
    return launched(o, "gated step") ? 0 : 1;
  });
}

}  // extern "C"
