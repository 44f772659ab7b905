// phz_adamw.hip — AdamW over many tensors at once, its moments in 32 bits or in
// 8 with an exponent for each 256 elements.
//
//   m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2
//   w <- (1 - lr wd) w - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by memory: 28 bytes an element in f32, 14 with bf16 gradients and 8-bit
// moments. The tensors of a launch travel in its arguments (a captured graph then
// holds them itself), up to kTensors; a workgroup finds its tensor among them.
#include "phz_ops.h"

#include <math.h>

#include <algorithm>
#include <vector>

using namespace phzop;

namespace {

constexpr int kBlock = 256;     // elements that share an exponent
constexpr int kTensors = 56;    // of a launch: its arguments stay below 4 KB
// Threads of a workgroup, and its elements: many where the tensors fill the chip so
// too, else few, so that they spread (the 8 tensors of a policy, 0.28 M elements: 8.0
// us at 4096, 4.7 at 1024).
constexpr int kThreads = 256, kSpan = 4096, kSmallSpan = 1024;
constexpr int kTopM = 14, kTopV = 30;        // code exponents of a block's largest element
constexpr uint32_t kInf = 0x7f800000u;

struct One {
  void *w, *m, *v;
  const void* g;
  uint8_t* e;
  int64_t n;
  uint32_t first;  // workgroup
  uint32_t key;    // the tensor's place in the list
};
struct AdamWArgs {
  const float* fix;  // lr / (1 - b1^t), 1 / (1 - b2^t), and the step's random bits, from `advance`
  float b1, b2, c1, c2, keep, eps;
  int32_t count, span;
  One t[kTensors];
};
static_assert(sizeof(AdamWArgs) <= 4096, "kernel arguments");

// 32 bits to 32 bits, each of the result's depending on all of them.
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0xb504f335u;
  x = (x ^ (x >> 15)) * 0xb7e15163u;
  return x ^ (x >> 16);
}

// t = ++*step, and what follows from it for every element. A launch of its own,
// since the update's workgroups all read it.
__global__ void advance(int64_t* step, double lr, double b1, double b2, uint32_t seed, float* out) {
  const int64_t t = ++*step;
  out[0] = (float)fmax(-3e38, fmin(3e38, lr / (1.0 - pow(b1, (double)t))));
  out[1] = (float)(1.0 / (1.0 - pow(b2, (double)t)));
  ((uint32_t*)out)[2] = mix((uint32_t)t ^ 0x9e3779b9u) + seed;
}

// A code's value below block exponent e, and the code of a value. Every step is
// exact, so the codes do not depend on how they are computed.
template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t code, int e) {
  constexpr int top = SIGNED ? kTopM : kTopV;
  if (code == (SIGNED ? 0x80u : 0xffu)) return __builtin_nanf("");
  // Below the leading one, the code above without that one.
  const uint32_t size = SIGNED ? code & 0x7f : code, least = (uint32_t)(e - top + 1) << 23;
  const bool small = size < 8;
  const uint32_t bits = (size << 20) + (least - (small ? 0 : 1u << 23));
  const float value = __builtin_bit_cast(float, bits) - (small ? __builtin_bit_cast(float, least) : 0.0f);
  return SIGNED && code > 0x80 ? -value : value;
}
// (Both ways of a code are taken and one is chosen: 8 elements a lane on different
// ways cost more.)
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(float x, int e, uint32_t dither) {
  constexpr int top = SIGNED ? kTopM : kTopV;
  const uint32_t bits = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  const uint32_t base = (uint32_t)(e - top) << 3;
  // Below, whole multiples of the least step, to 20 further bits.
  const float fine = __builtin_amdgcn_ldexpf(__builtin_bit_cast(float, bits), 149 + top - e);
  const uint32_t least = (uint32_t)fine + dither, normal = bits + dither;
  uint32_t code = bits >= (base + 8) << 20 ? (normal >> 20) - base : least >> 20;
  if (!SIGNED) code = max(code, min(bits, 1u));
  if (SIGNED) code |= x < 0.0f && code ? 0x80 : 0;
  return bits >= kInf ? (SIGNED ? 0x80 : 0xff) : code;
}

// sqrt(x) to the instruction's unit in the last place, also for x below its range.
__device__ __forceinline__ float root(float x) {
  const bool small = x < 0x1p-96f;
  return __builtin_amdgcn_sqrtf(small ? x * 0x1p64f : x) * (small ? 0x1p-32f : 1.0f);
}

// x a + y b and x^2 with every product and sum rounded: codes follow from them, and
// are the same in any implementation that does so.
__device__ __forceinline__ float blend(float x, float a, float y, float b) {
#pragma clang fp contract(off)
  const float p = x * a, q = y * b;
  return p + q;
}
__device__ __forceinline__ float square(float x) {
#pragma clang fp contract(off)
  return x * x;
}

// The largest biased exponent of a wave's finite values, at least 40.
__device__ __forceinline__ int block_exponent(uint32_t most) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, m));
  return max((int)(most >> 23), 40);
}
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return b < kInf ? b : 0;
}

template <class E>
__device__ __forceinline__ void fetch(const E* p, int n, float* x) {
  if (n == 4) {
    const Pack<E, 4> v = *(const Pack<E, 4>*)p;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = to_f32(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = i < n ? to_f32(p[i]) : 0.0f;
  }
}
template <class E>
__device__ __forceinline__ void stash(E* p, int n, const float* x) {
  if (n == 4) {
    Pack<E, 4> v;
#pragma unroll
    for (int i = 0; i < 4; i++) v.v[i] = from_f32<E>(x[i]);
    *(Pack<E, 4>*)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) p[i] = from_f32<E>(x[i]);
  }
}

// Four codes as one word; those that do not exist are 0.
__device__ __forceinline__ uint32_t fetch_codes(const uint8_t* p, int n) {
  if (n == 4) return __builtin_bit_cast(uint32_t, *(const Pack<uint8_t, 4>*)p);
  uint32_t x = 0;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (i < n) x |= (uint32_t)p[i] << 8 * i;
  return x;
}
__device__ __forceinline__ void stash_codes(uint8_t* p, int n, uint32_t x) {
  if (n == 4) {
    *(Pack<uint8_t, 4>*)p = __builtin_bit_cast(Pack<uint8_t, 4>, x);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) p[i] = (uint8_t)(x >> 8 * i);
  }
}

// A wave takes 256 elements at a time, a lane four of them. In 8 bits that is a
// block, whose exponent the wave's lanes find together. There the codes' arithmetic
// takes about as long as the memory: 67 M elements with bf16 gradients in 198 us
// (4.7 TB/s), 335 with codes fetched, branched on and stored a byte at a time.
template <class W, class G, bool EIGHT>
__global__ __launch_bounds__(kThreads) void adamw_kernel(AdamWArgs a) {
  int at = 0;
  for (int i = 1; i < a.count; i++) at = blockIdx.x >= a.t[i].first ? i : at;
  const One& t = a.t[at];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float fix1 = a.fix[0], fix2 = a.fix[1];
  const uint32_t key = EIGHT ? mix(mix(((const uint32_t*)a.fix)[2]) + t.key * 0x243f6a89u) : 0;
  const int64_t start = (int64_t)(blockIdx.x - t.first) * a.span;
  const int64_t blocks = ceil_div(t.n, kBlock);
  for (int u = 0; u < a.span / (kThreads * 4); u++) {
    const int64_t block = start / kBlock + u * (kThreads / 64) + wave;
    if (block >= blocks) return;
    const int64_t i0 = block * kBlock + lane * 4;
    const int n = (int)min((int64_t)4, max((int64_t)0, t.n - i0));
    float w[4], g[4], m[4], v[4];
    fetch((const W*)t.w + i0, n, w);
    fetch((const G*)t.g + i0, n, g);
    if constexpr (EIGHT) {
      const int em = t.e[block], ev = t.e[blocks + block];
      const uint32_t cm = fetch_codes((const uint8_t*)t.m + i0, n), cv = fetch_codes((const uint8_t*)t.v + i0, n);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        m[i] = decode<true>(cm >> 8 * i & 0xff, em);
        v[i] = decode<false>(cv >> 8 * i & 0xff, ev);
      }
    } else {
      fetch((const float*)t.m + i0, n, m);
      fetch((const float*)t.v + i0, n, v);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      m[i] = blend(m[i], a.b1, g[i], a.c1);
      v[i] = blend(v[i], a.b2, square(g[i]), a.c2);
      // Nine roundings of the step at most, two of them in its quotient.
      w[i] = w[i] * a.keep - m[i] * fix1 * __builtin_amdgcn_rcpf(root(v[i] * fix2) + a.eps);
    }
    stash((W*)t.w + i0, n, w);
    if constexpr (EIGHT) {
      uint32_t mm = 0, mv = 0;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < n) mm = max(mm, finite_bits(m[i])), mv = max(mv, finite_bits(v[i]));
      const int em = block_exponent(mm), ev = block_exponent(mv);
      if (lane == 0) t.e[block] = (uint8_t)em, t.e[blocks + block] = (uint8_t)ev;
      uint32_t cm = 0, cv = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t h = mix((uint32_t)(i0 + i) * 0x9e3779b9u ^ key);
        cm |= encode<true>(m[i], em, (h & 0xffff) * 16 + 8) << 8 * i;
        cv |= encode<false>(v[i], ev, (h >> 16) * 16 + 8) << 8 * i;
      }
      stash_codes((uint8_t*)t.m + i0, n, cm);
      stash_codes((uint8_t*)t.v + i0, n, cv);
    } else {
      stash((float*)t.m + i0, n, m);
      stash((float*)t.v + i0, n, v);
    }
  }
}

// The values of codes. One's m and v are the codes, g and w the values' places. A
// thread takes eight neighbours, which one block has: 66 us for 67 M elements, against
// 270 an element at a time.
__global__ __launch_bounds__(kThreads) void values_kernel(AdamWArgs a) {
  int at = 0;
  for (int i = 1; i < a.count; i++) at = blockIdx.x >= a.t[i].first ? i : at;
  const One& t = a.t[at];
  const int64_t blocks = ceil_div(t.n, kBlock), start = (int64_t)(blockIdx.x - t.first) * a.span;
#pragma unroll 2
  for (int u = threadIdx.x * 8; u < a.span; u += kThreads * 8) {
    const int64_t i = start + u;
    if (i >= t.n) return;
    const int em = t.e[i / kBlock], ev = t.e[blocks + i / kBlock];
    const uint8_t *m = (const uint8_t*)t.m + i, *v = (const uint8_t*)t.v + i;
    bf16 *to_m = (bf16*)t.w + i, *to_v = (bf16*)t.g + i;
    if (i + 8 <= t.n) {
      const Pack<uint8_t, 8> cm = *(const Pack<uint8_t, 8>*)m, cv = *(const Pack<uint8_t, 8>*)v;
      Pack<bf16, 8> x, y;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x.v[j] = from_f32<bf16>(decode<true>(cm.v[j], em));
        y.v[j] = from_f32<bf16>(decode<false>(cv.v[j], ev));
      }
      *(Pack<bf16, 8>*)to_m = x;
      *(Pack<bf16, 8>*)to_v = y;
    } else {
      for (int j = 0; j < t.n - i; j++) {
        to_m[j] = from_f32<bf16>(decode<true>(m[j], em));
        to_v[j] = from_f32<bf16>(decode<false>(v[j], ev));
      }
    }
  }
}

// One list's tensors: vectors of the sizes of w's (or of m's). What is as it has to
// be is seen at once: a name for the complaint costs more than the kernels do.
bool vectors(phz_ops* o, const char* name, int64_t i, const phz_tensor* t, int64_t n, int dtype, bool output) {
  if (t->ndim == 1 && t->dtype == dtype && t->size[0] >= 0 && t->size[0] <= 1ll << 40 && (n < 0 || t->size[0] == n) &&
      (t->size[0] <= 1 || t->stride[0] == 1) && (!t->size[0] || (t->data && t->stride[0] >= 0 && t->stride[0] <= 1ll << 48)) &&
      (uintptr_t)t->data % (uintptr_t)elem_bytes(dtype) == 0)
    return true;
  const std::string full = fmt("%s[%lld]", name, (long long)i);
  return check(o, full.c_str(), t, Want{1, {n, 0, 0}, dtype, true, output});
}

// Outputs that share memory with anything else: spans sorted by address. A list's
// tensors mostly stand in order, so lists are merged.
struct Span {
  uintptr_t lo, hi;
  const char* name;
  int64_t i;
  bool output;
};
struct Spans {
  std::vector<Span> all;
  size_t begin = 0;  // of the present list
  static bool before(const Span& a, const Span& b) { return a.lo < b.lo; }
  void add(const char* name, int64_t i, const phz_tensor* t, bool output) {
    if (empty(t)) return;
    const uintptr_t lo = (uintptr_t)t->data;
    all.push_back({lo, lo + (uintptr_t)(t->size[0] * elem_bytes(t->dtype)), name, i, output});
  }
  void add(const char* name, const phz_tensor* t, int64_t n, bool output) {
    for (int64_t i = 0; i < n; i++) add(name, i, t + i, output);
    end_list();
  }
  void end_list() {
    if (!std::is_sorted(all.begin() + begin, all.end(), before)) std::sort(all.begin() + begin, all.end(), before);
    std::inplace_merge(all.begin(), all.begin() + begin, all.end(), before);
    begin = all.size();
  }
  bool apart(phz_ops* o) const {
    // The span that reaches furthest so far, of outputs and of all.
    const Span *far = nullptr, *far_out = nullptr;
    for (auto& s : all) {
      const Span* hit = s.output ? far : far_out;
      if (hit && hit->hi > s.lo) {
        const Span &a = s.output ? s : *hit, &b = s.output ? *hit : s;
        o->err = fmt("%s[%lld] overlaps %s[%lld]", a.name, (long long)a.i, b.name, (long long)b.i);
        return false;
      }
      if (!far || s.hi > far->hi) far = &s;
      if (s.output && (!far_out || s.hi > far_out->hi)) far_out = &s;
    }
    return true;
  }
};

// Launches over the entries, kTensors and fewer than 2^32 threads at a time.
constexpr uint64_t kMostGroups = (1ull << 32) / kThreads - 1;
template <class F>
void in_launches(const phz_ops* o, const std::vector<One>& all, AdamWArgs a, F&& launch) {
  int64_t wide = 0;
  for (auto& t : all) wide += ceil_div(t.n, kSpan);
  a.span = wide < 4 * o->cus ? kSmallSpan : kSpan;
  size_t i = 0;
  while (i < all.size()) {
    a.count = 0;
    uint64_t groups = 0;
    while (i < all.size() && a.count < kTensors) {
      const uint64_t more = (uint64_t)ceil_div(all[i].n, a.span);
      if (a.count && groups + more > kMostGroups) break;
      a.t[a.count] = all[i++];
      a.t[a.count++].first = (uint32_t)groups;
      groups += more;
    }
    launch(a, (unsigned)groups);
  }
}

constexpr int64_t kMostElements = (int64_t)kMostGroups * kSpan;  // of a tensor: its workgroups fit a launch

bool check_exponents(phz_ops* o, int64_t i, const phz_tensor* e, int64_t n) {
  return vectors(o, "exponents", i, e, 2 * ceil_div(n, kBlock), PHZ_U8, true);
}

}  // namespace

extern "C" {

int phz_adamw_step(phz_ops* o, void* stream_, const phz_adamw_cfg* cfg, int64_t n, const phz_tensor* w, const phz_tensor* g,
                   const phz_tensor* m, const phz_tensor* v, const phz_tensor* exponents, const phz_tensor* step) {
  return guarded(o, [&] {
    if (!cfg) return o->fail("configuration is missing");
    if (!(fabs(cfg->lr) <= 1e30 && fabs(cfg->weight_decay) <= 1e30)) return o->fail("lr and weight_decay have to be finite");
    if (!(cfg->beta1 >= 0 && cfg->beta1 < 1 && cfg->beta2 >= 0 && cfg->beta2 < 1)) return o->fail("betas have to be in [0, 1)");
    if (!(cfg->eps >= 0 && cfg->eps <= 1e30)) return o->fail("eps has to be finite and not negative");
    if (n < 0 || n > 1 << 24) return o->fail("too many tensors");
    if (n && (!w || !g || !m || !v)) return o->fail("a list of tensors is missing");
    if (!check(o, "step", step, Want{1, {1, 0, 0}, PHZ_I64, true, true})) return 1;
    const bool eight = n && m[0].dtype == PHZ_U8;
    if (n && eight != (exponents != nullptr))
      return o->fail(eight ? "exponents are missing: m is u8" : "exponents are given, but m is not u8");
    std::vector<One> each[4];
    for (int64_t i = 0; i < n; i++) {
      for (const auto& x : {std::make_pair("w", w + i), std::make_pair("g", g + i)})
        if (x.second->dtype != PHZ_F32 && x.second->dtype != PHZ_BF16)
          return o->fail(fmt("%s[%lld] is %s, expected f32 or bf16", x.first, (long long)i, dtype_name(x.second->dtype)));
      if (!vectors(o, "w", i, w + i, -1, w[i].dtype, true)) return 1;
      const int64_t size = w[i].size[0];
      if (size > kMostElements) return o->fail(fmt("w[%lld] is too large", (long long)i));
      const int dt = eight ? PHZ_U8 : PHZ_F32;
      if (!vectors(o, "g", i, g + i, size, g[i].dtype, false) || !vectors(o, "m", i, m + i, size, dt, true) ||
          !vectors(o, "v", i, v + i, size, dt, true) || (eight && !check_exponents(o, i, exponents + i, size)))
        return 1;
      if (size)
        each[(w[i].dtype == PHZ_BF16) * 2 + (g[i].dtype == PHZ_BF16)].push_back(
            One{w[i].data, m[i].data, v[i].data, g[i].data, eight ? (uint8_t*)exponents[i].data : nullptr, size, 0, (uint32_t)i});
    }
    Spans spans;
    spans.all.reserve((size_t)n * 5 + 1);
    spans.add("w", w, n, true);
    spans.add("g", g, n, false);
    spans.add("m", m, n, true);
    spans.add("v", v, n, true);
    if (eight) spans.add("exponents", exponents, n, true);
    spans.add("step", step, 1, true);
    if (!spans.apart(o)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    auto stream = (hipStream_t)stream_;
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    auto* fix = (float*)o->workspace(stream, 64);
    if (!fix) return 1;
    AdamWArgs a{};
    a.fix = fix;
    a.b1 = (float)cfg->beta1, a.b2 = (float)cfg->beta2;
    a.c1 = (float)(1.0 - cfg->beta1), a.c2 = (float)(1.0 - cfg->beta2);
    // (An eps that is not 0 keeps 0 / (0 + eps) at 0, also where f32 has no such number.)
    a.keep = (float)(1.0 - cfg->lr * cfg->weight_decay), a.eps = cfg->eps > 0 ? (float)fmax(cfg->eps, 0x1p-126) : 0.0f;
    hipLaunchKernelGGL(advance, dim3(1), dim3(1), 0, stream, (int64_t*)step->data, cfg->lr, cfg->beta1, cfg->beta2, cfg->seed, fix);
    for (int k = 0; k < 4; k++) {
      auto go = [&](auto kernel) {
        in_launches(o, each[k], a, [&](const AdamWArgs& x, unsigned groups) {
          hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), 0, stream, x);
        });
      };
      if (eight)
        k == 0   ? go(adamw_kernel<float, float, true>)
        : k == 1 ? go(adamw_kernel<float, bf16, true>)
        : k == 2 ? go(adamw_kernel<bf16, float, true>)
                 : go(adamw_kernel<bf16, bf16, true>);
      else
        k == 0   ? go(adamw_kernel<float, float, false>)
        : k == 1 ? go(adamw_kernel<float, bf16, false>)
        : k == 2 ? go(adamw_kernel<bf16, float, false>)
                 : go(adamw_kernel<bf16, bf16, false>);
    }
    return launched(o, "AdamW") ? 0 : 1;
  });
}

int phz_adamw_values(phz_ops* o, void* stream, int64_t n, const phz_tensor* m, const phz_tensor* v, const phz_tensor* exponents,
                     const phz_tensor* m_values, const phz_tensor* v_values) {
  return guarded(o, [&] {
    if (n < 0 || n > 1 << 24) return o->fail("too many tensors");
    if (n && (!m || !v || !exponents || !m_values || !v_values)) return o->fail("a list of tensors is missing");
    std::vector<One> all;
    for (int64_t i = 0; i < n; i++) {
      if (!vectors(o, "m", i, m + i, -1, PHZ_U8, false)) return 1;
      const int64_t size = m[i].size[0];
      if (size > kMostElements) return o->fail(fmt("m[%lld] is too large", (long long)i));
      if (!vectors(o, "v", i, v + i, size, PHZ_U8, false) || !check_exponents(o, i, exponents + i, size) ||
          !vectors(o, "m_values", i, m_values + i, size, PHZ_BF16, true) ||
          !vectors(o, "v_values", i, v_values + i, size, PHZ_BF16, true))
        return 1;
      if (size) all.push_back(One{m_values[i].data, m[i].data, v[i].data, v_values[i].data, (uint8_t*)exponents[i].data, size, 0, 0});
    }
    Spans spans;
    spans.all.reserve((size_t)n * 5);
    spans.add("m", m, n, false);
    spans.add("v", v, n, false);
    spans.add("exponents", exponents, n, false);
    spans.add("m_values", m_values, n, true);
    spans.add("v_values", v_values, n, true);
    if (!spans.apart(o)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    in_launches(o, all, AdamWArgs{}, [&](const AdamWArgs& x, unsigned groups) {
      hipLaunchKernelGGL(values_kernel, dim3(groups), dim3(kThreads), 0, (hipStream_t)stream, x);
    });
    return launched(o, "AdamW values") ? 0 : 1;
  });
}

}  // extern "C"
