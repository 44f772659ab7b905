// phz_rotary.hip — rotary positions: pairs of elements of each head turned by an
// angle that is the position times the pair's frequency.
//
// A turn is taken in three steps: position * freq / 2 pi in f64, less its nearest
// whole number (at freq 1 a position of 2^40 still leaves some 15 bits of a turn),
// the rest in f32, and sine and cosine by their series on a quarter turn. A
// lane takes one pair of a row, or four neighbours where rows are many, and turns
// them in every head, so the angles are found once a row. Bound by memory: 262144 rows
// of 8 heads of 64 bf16 in 104 us, 5.2 TB/s (133 with one pair a lane and 64-bit
// divisions); a step of 1024 worlds is a launch (4 us).
#include "phz_ops.h"

#include <algorithm>

using namespace phzop;

namespace {

constexpr double kTurn = 0.15915494309189533577;  // 1 / 2 pi

// (cos, sin) of 2 pi u for |u| <= 1/2. On |r| <= pi/4 the series to r^8 and r^9
// leave at most the terms after them, (pi/4)^10 / 10! = 2^-25.3 and (pi/4)^11 / 11! =
// 2^-29.1; with the roundings on the way cos is within 1.3 and sin 1.6 of 2^-24, and u's own,
// up to 2^-26 of a turn, is 2^-23.3 of an angle.
__device__ __forceinline__ void turn(float u, float* c, float* s) {
  const float quarter = rintf(4.0f * u);
  const float r = 6.2831853071795865f * fmaf(-0.25f, quarter, u), x = r * r;
  const float sn = r * fmaf(x, fmaf(x, fmaf(x, fmaf(x, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), 1.0f);
  const float cs = fmaf(x, fmaf(x, fmaf(x, fmaf(x, 2.4801587e-5f, -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.0f);
  const int k = (int)quarter & 3;
  const float a = k & 1 ? sn : cs, b = k & 1 ? cs : sn;
  *c = k == 1 || k == 2 ? -a : a;
  *s = k >= 2 ? -b : b;
}

struct RotaryArgs {
  const void* x;
  void* y;
  const void* pos;
  const double* freq;
  int64_t x_t, x_b, y_t, y_b, p_t, p_b, f_s;
  int64_t rows;
  int32_t worlds, heads, size, pairs;
  float scale, sign;
};

// A lane VEC neighbouring pairs of a row, or VEC elements behind the pairs.
template <class E, class P, int VEC>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, int32_t pairs_layout) {
  const int32_t each = (a.size - a.pairs) / VEC;
  const int64_t n = a.rows * each;
  const bool half = pairs_layout == PHZ_PAIRS_HALF;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    int64_t row, t;
    int32_t p, b;
    if (n <= 0xffffffffll) {
      const uint32_t r = (uint32_t)i / (uint32_t)each, s = r / (uint32_t)a.worlds;
      row = r, t = s, p = (int32_t)((uint32_t)i - r * each), b = (int32_t)(r - s * a.worlds);
    } else {
      row = i / each, t = row / a.worlds, p = (int32_t)(i - row * each), b = (int32_t)(row - t * a.worlds);
    }
    p *= VEC;
    const E* x = (const E*)a.x + t * a.x_t + b * a.x_b;
    E* y = (E*)a.y + t * a.y_t + b * a.y_b;
    if (p >= a.pairs) {
      x += p + a.pairs, y += p + a.pairs;
      for (int h = 0; h < a.heads; h++, x += a.size, y += a.size) *(Pack<E, VEC>*)y = *(const Pack<E, VEC>*)x;
      continue;
    }
    const double position = (double)((const P*)a.pos)[t * a.p_t + b * a.p_b];
    float c[VEC], s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      const double turns = position * (a.freq[(p + j) * a.f_s] * kTurn);
      turn((float)(turns - rint(turns)), &c[j], &s[j]);
      c[j] *= a.scale, s[j] *= a.scale * a.sign;
    }
    auto turned = [&](int j, E& v0, E& v1) {
      const float x0 = to_f32(v0), x1 = to_f32(v1);
      v0 = from_f32<E>(fmaf(x0, c[j], -x1 * s[j]));
      v1 = from_f32<E>(fmaf(x0, s[j], x1 * c[j]));
    };
    if (half) {
      x += p, y += p;
      for (int h = 0; h < a.heads; h++, x += a.size, y += a.size) {
        Pack<E, VEC> v0 = *(const Pack<E, VEC>*)x, v1 = *(const Pack<E, VEC>*)(x + a.pairs);
#pragma unroll
        for (int j = 0; j < VEC; j++) turned(j, v0.v[j], v1.v[j]);
        *(Pack<E, VEC>*)y = v0;
        *(Pack<E, VEC>*)(y + a.pairs) = v1;
      }
    } else {
      x += 2 * p, y += 2 * p;
      for (int h = 0; h < a.heads; h++, x += a.size, y += a.size) {
        Pack<E, 2 * VEC> v = *(const Pack<E, 2 * VEC>*)x;
#pragma unroll
        for (int j = 0; j < VEC; j++) turned(j, v.v[2 * j], v.v[2 * j + 1]);
        *(Pack<E, 2 * VEC>*)y = v;
      }
    }
  }
}

}  // namespace

extern "C" int phz_rotary(phz_ops* o, void* stream, const phz_rotary_cfg* cfg, const phz_tensor* x, const phz_tensor* positions,
                          const phz_tensor* freq, const phz_tensor* y) {
  return guarded(o, [&] {
    if (!cfg) return o->fail("configuration is missing");
    if (cfg->pairs != PHZ_PAIRS_HALF && cfg->pairs != PHZ_PAIRS_INTERLEAVED) return o->fail("unknown layout of pairs");
    if (!(cfg->scale >= -3e38 && cfg->scale <= 3e38)) return o->fail("scale has to be finite");
    if (!x) return o->fail("x is missing");
    if (x->dtype != PHZ_F32 && x->dtype != PHZ_BF16)
      return o->fail(fmt("x is %s, expected f32 or bf16", dtype_name(x->dtype)));
    if (!check(o, "x", x, Want{3, {-1, -1, -1}, x->dtype, true, false})) return 1;
    const int64_t T = x->size[0], B = x->size[1], W = x->size[2];
    if (!positions) return o->fail("positions is missing");
    if (positions->dtype != PHZ_I32 && positions->dtype != PHZ_I64)
      return o->fail(fmt("positions is %s, expected i32 or i64", dtype_name(positions->dtype)));
    if (!check(o, "positions", positions, Want{2, {T, B, 0}, positions->dtype, false, false}) ||
        !check(o, "freq", freq, Want{1, {-1, 0, 0}, PHZ_F64, false, false}) ||
        !check(o, "y", y, Want{3, {T, B, W}, x->dtype, true, true}))
      return 1;
    if (cfg->heads < 1 || W % cfg->heads) return o->fail(fmt("x has %lld elements along axis 2, not %d heads", (long long)W, cfg->heads));
    const int64_t size = W / cfg->heads;
    if (2 * freq->size[0] > size)
      return o->fail(fmt("freq has %lld pairs, more than fit heads of %lld", (long long)freq->size[0], (long long)size));
    if (T > 0x3fff0000ll || B > 0x3fff0000ll || W > 0x3fff0000ll) return o->fail("steps, worlds and width have to be below 2^30");
    const bool same = x->data == y->data && x->stride[0] == y->stride[0] && x->stride[1] == y->stride[1];
    if ((!same && !apart(o, "y", y, "x", x)) || !apart(o, "y", y, "positions", positions) || !apart(o, "y", y, "freq", freq)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (T == 0 || B == 0 || W == 0) return 0;
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    RotaryArgs a{x->data, y->data, positions->data, (const double*)freq->data, x->stride[0], x->stride[1], y->stride[0],
                 y->stride[1], positions->stride[0], positions->stride[1], freq->stride[0], T * B, (int32_t)B, cfg->heads,
                 (int32_t)size, (int32_t)freq->size[0], (float)cfg->scale, cfg->inverse ? -1.0f : 1.0f};
    // Four pairs a lane where that still fills the chip.
    const int64_t n = a.rows * (a.size - a.pairs);
    const bool four = a.pairs % 4 == 0 && a.size % 4 == 0 && n >= 4 * 512 * (int64_t)o->cus;
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(four ? n / 4 : n, 256), 1 << 20);
    auto go = [&](auto one, auto many) {
      hipLaunchKernelGGL(four ? many : one, dim3(blocks), dim3(256), 0, (hipStream_t)stream, a, cfg->pairs);
    };
    const bool wide = positions->dtype == PHZ_I64;
    if (x->dtype == PHZ_F32)
      wide ? go(rotary_kernel<float, int64_t, 1>, rotary_kernel<float, int64_t, 4>)
           : go(rotary_kernel<float, int32_t, 1>, rotary_kernel<float, int32_t, 4>);
    else
      wide ? go(rotary_kernel<bf16, int64_t, 1>, rotary_kernel<bf16, int64_t, 4>)
           : go(rotary_kernel<bf16, int32_t, 1>, rotary_kernel<bf16, int32_t, 4>);
    return launched(o, "rotary") ? 0 : 1;
  });
}
