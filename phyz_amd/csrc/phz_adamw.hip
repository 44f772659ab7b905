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
constexpr int kThreads = 256, kSpan = 4096;  // threads and elements of a workgroup
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
  const float* fix;  // 1 - b1^t, 1 - b2^t, and the step's random bits, from `advance`
  float b1, b2, c1, c2, lr, keep, eps;
  int32_t count;
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
__global__ void advance(int64_t* step, double b1, double b2, uint32_t seed, float* out) {
  const int64_t t = ++*step;
  out[0] = (float)(1.0 - pow(b1, (double)t));
  out[1] = (float)(1.0 - pow(b2, (double)t));
  ((uint32_t*)out)[2] = mix((uint32_t)t ^ 0x9e3779b9u) + seed;
}

// The power of two with biased exponent e (1 to 254).
__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, e << 23); }

// A code's value below block exponent e, and the code of a value. Every step is
// exact, so the codes do not depend on how they are computed.
template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t code, int e) {
  constexpr int top = SIGNED ? kTopM : kTopV;
  if (code == (SIGNED ? 0x80u : 0xffu)) return __builtin_nanf("");
  const uint32_t size = SIGNED ? code & 0x7f : code, exp = size >> 3;
  const float digits = (float)(exp ? 8 + (size & 7) : size);
  const float value = digits * power(e - top - 3 + (int)max(exp, 1u));
  return SIGNED && code > 0x80 ? -value : value;
}
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(float x, int e, uint32_t dither) {
  constexpr int top = SIGNED ? kTopM : kTopV;
  const uint32_t bits = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  if (bits >= kInf) return SIGNED ? 0x80 : 0xff;
  const int exp = (int)(bits >> 23) - e + top;
  uint32_t code;
  if (exp >= 1) {
    code = ((bits + dither) >> 20) - ((uint32_t)(e - top) << 3);
  } else {
    // Whole multiples of the least step, to 20 further bits.
    const uint32_t fixed = (uint32_t)__builtin_amdgcn_ldexpf(__builtin_bit_cast(float, bits), 129 + top - e + 20);
    code = (fixed + dither) >> 20;
  }
  if (SIGNED) return x < 0.0f && code ? code + 0x80 : code;
  return bits ? max(code, 1u) : 0;
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

// A wave takes 256 elements at a time, a lane four of them. In 8 bits that is a
// block, whose exponent the wave's lanes find together.
template <class W, class G, bool EIGHT>
__global__ __launch_bounds__(kThreads) void adamw_kernel(AdamWArgs a) {
  int at = 0;
  for (int i = 1; i < a.count; i++) at = blockIdx.x >= a.t[i].first ? i : at;
  const One& t = a.t[at];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float fix1 = a.fix[0], fix2 = a.fix[1];
  const uint32_t key = EIGHT ? mix(mix(((const uint32_t*)a.fix)[2]) + t.key * 0x243f6a89u) : 0;
  const int64_t start = (int64_t)(blockIdx.x - t.first) * kSpan;
  const int64_t blocks = ceil_div(t.n, kBlock);
#pragma unroll 2
  for (int u = 0; u < kSpan / kThreads / 4; u++) {
    const int64_t block = start / kBlock + u * (kThreads / 64) + wave;
    if (block >= blocks) return;
    const int64_t i0 = block * kBlock + lane * 4;
    const int n = (int)min((int64_t)4, max((int64_t)0, t.n - i0));
    float w[4], g[4], m[4], v[4];
    fetch((const W*)t.w + i0, n, w);
    fetch((const G*)t.g + i0, n, g);
    if constexpr (EIGHT) {
      const int em = t.e[block], ev = t.e[blocks + block];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        m[i] = i < n ? decode<true>(((const uint8_t*)t.m)[i0 + i], em) : 0.0f;
        v[i] = i < n ? decode<false>(((const uint8_t*)t.v)[i0 + i], ev) : 0.0f;
      }
    } else {
      fetch((const float*)t.m + i0, n, m);
      fetch((const float*)t.v + i0, n, v);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      m[i] = blend(m[i], a.b1, g[i], a.c1);
      v[i] = blend(v[i], a.b2, square(g[i]), a.c2);
      w[i] = w[i] * a.keep - (m[i] / fix1) * a.lr / (sqrtf(v[i] / fix2) + a.eps);
    }
    stash((W*)t.w + i0, n, w);
    if constexpr (EIGHT) {
      uint32_t mm = 0, mv = 0;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < n) mm = max(mm, finite_bits(m[i])), mv = max(mv, finite_bits(v[i]));
      const int em = block_exponent(mm), ev = block_exponent(mv);
      if (lane == 0) t.e[block] = (uint8_t)em, t.e[blocks + block] = (uint8_t)ev;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (i >= n) break;
        const uint32_t h = mix((uint32_t)(i0 + i) * 0x9e3779b9u ^ key);
        ((uint8_t*)t.m)[i0 + i] = (uint8_t)encode<true>(m[i], em, (h & 0xffff) * 16 + 8);
        ((uint8_t*)t.v)[i0 + i] = (uint8_t)encode<false>(v[i], ev, (h >> 16) * 16 + 8);
      }
    } else {
      stash((float*)t.m + i0, n, m);
      stash((float*)t.v + i0, n, v);
    }
  }
}

// The values of codes. One's m and v are the codes, g and w the values' places.
__global__ __launch_bounds__(kThreads) void values_kernel(AdamWArgs a) {
  int at = 0;
  for (int i = 1; i < a.count; i++) at = blockIdx.x >= a.t[i].first ? i : at;
  const One& t = a.t[at];
  const int64_t blocks = ceil_div(t.n, kBlock), start = (int64_t)(blockIdx.x - t.first) * kSpan;
  for (int u = 0; u < kSpan / kThreads; u++) {
    const int64_t i = start + u * kThreads + threadIdx.x;
    if (i >= t.n) return;
    ((bf16*)t.w)[i] = from_f32<bf16>(decode<true>(((const uint8_t*)t.m)[i], t.e[i / kBlock]));
    ((bf16*)t.g)[i] = from_f32<bf16>(decode<false>(((const uint8_t*)t.v)[i], t.e[blocks + i / kBlock]));
  }
}

// One list's tensors: vectors of the sizes of w's (or of m's).
bool vectors(phz_ops* o, const char* name, int64_t i, const phz_tensor* t, int64_t n, int dtype, bool output) {
  const std::string full = fmt("%s[%lld]", name, (long long)i);
  return check(o, full.c_str(), t, Want{1, {n, 0, 0}, dtype, true, output});
}

// Outputs that share memory with anything else: spans sorted by address.
struct Span {
  uintptr_t lo, hi;
  const char* name;
  int64_t i;
  bool output;
};
void add_span(std::vector<Span>& spans, const char* name, int64_t i, const phz_tensor* t, bool output) {
  if (empty(t)) return;
  const uintptr_t lo = (uintptr_t)t->data;
  spans.push_back({lo, lo + (uintptr_t)(t->size[0] * elem_bytes(t->dtype)), name, i, output});
}
bool spans_apart(phz_ops* o, std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  // The span that reaches furthest so far, of outputs and of all.
  const Span *far = nullptr, *far_out = nullptr;
  for (auto& s : spans) {
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

// Launches over the entries, kTensors and 2^31 workgroups at a time.
template <class F>
void in_launches(const std::vector<One>& all, AdamWArgs a, F&& launch) {
  size_t i = 0;
  while (i < all.size()) {
    a.count = 0;
    uint64_t groups = 0;
    while (i < all.size() && a.count < kTensors) {
      const uint64_t more = (uint64_t)ceil_div(all[i].n, kSpan);
      if (a.count && groups + more > 0x7fffffffull) break;
      a.t[a.count] = all[i++];
      a.t[a.count++].first = (uint32_t)groups;
      groups += more;
    }
    launch(a, (unsigned)groups);
  }
}

constexpr int64_t kMostElements = 1ll << 40;  // of a tensor: its workgroups fit a launch

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
    std::vector<Span> spans;
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
      add_span(spans, "w", i, w + i, true);
      add_span(spans, "g", i, g + i, false);
      add_span(spans, "m", i, m + i, true);
      add_span(spans, "v", i, v + i, true);
      if (eight) add_span(spans, "exponents", i, exponents + i, true);
      if (size)
        each[(w[i].dtype == PHZ_BF16) * 2 + (g[i].dtype == PHZ_BF16)].push_back(
            One{w[i].data, m[i].data, v[i].data, g[i].data, eight ? (uint8_t*)exponents[i].data : nullptr, size, 0, (uint32_t)i});
    }
    add_span(spans, "step", 0, step, true);
    if (!spans_apart(o, spans)) return 1;
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
    a.lr = (float)cfg->lr, a.keep = (float)(1.0 - cfg->lr * cfg->weight_decay), a.eps = (float)cfg->eps;
    hipLaunchKernelGGL(advance, dim3(1), dim3(1), 0, stream, (int64_t*)step->data, cfg->beta1, cfg->beta2, cfg->seed, fix);
    for (int k = 0; k < 4; k++) {
      auto go = [&](auto kernel) {
        in_launches(each[k], a, [&](const AdamWArgs& x, unsigned groups) {
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
    std::vector<Span> spans;
    std::vector<One> all;
    for (int64_t i = 0; i < n; i++) {
      if (!vectors(o, "m", i, m + i, -1, PHZ_U8, false)) return 1;
      const int64_t size = m[i].size[0];
      if (size > kMostElements) return o->fail(fmt("m[%lld] is too large", (long long)i));
      if (!vectors(o, "v", i, v + i, size, PHZ_U8, false) || !check_exponents(o, i, exponents + i, size) ||
          !vectors(o, "m_values", i, m_values + i, size, PHZ_BF16, true) ||
          !vectors(o, "v_values", i, v_values + i, size, PHZ_BF16, true))
        return 1;
      add_span(spans, "m", i, m + i, false);
      add_span(spans, "v", i, v + i, false);
      add_span(spans, "exponents", i, exponents + i, false);
      add_span(spans, "m_values", i, m_values + i, true);
      add_span(spans, "v_values", i, v_values + i, true);
      if (size) all.push_back(One{m_values[i].data, m[i].data, v[i].data, v_values[i].data, (uint8_t*)exponents[i].data, size, 0, 0});
    }
    if (!spans_apart(o, spans)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    in_launches(all, AdamWArgs{}, [&](const AdamWArgs& x, unsigned groups) {
      hipLaunchKernelGGL(values_kernel, dim3(groups), dim3(kThreads), 0, (hipStream_t)stream, x);
    });
    return launched(o, "AdamW values") ? 0 : 1;
  });
}

}  // extern "C"
