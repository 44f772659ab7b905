// phz_muon.hip — orthogonalised updates: Newton-Schulz steps on a gradient's
// matrix (or a batch of them) and Muon's update of the weights.
//
//   X = g / (|g|_F + eps);   X <- a X + (b A + c A^2) X,  A = X X^T
//
// on whichever side is shorter: for tall matrices A = X^T X and
// X <- a X + X (b A + c A^2), so nothing is transposed.
#include "phz_gemm.h"

#include <math.h>

#include <algorithm>

using namespace phzop;

namespace {

constexpr int kNormBlocks = 64;  // partial sums of squares per matrix

struct View {
  void* data;
  int64_t batch, row;
};

// The matrix to orthogonalise into X (f32, dense) and partial sums of its
// squares, in f64: gradients whose squares leave f32's range have a norm too.
// With a momentum, m <- mu m + g comes first and the matrix is g + mu m or m.
template <class E>
__global__ __launch_bounds__(256) void gather_kernel(View g, View m, float mu, int nesterov, float* x, double* part,
                                                     int32_t rows, int32_t cols) {
  const int q = blockIdx.y;
  const int64_t n = (int64_t)rows * cols;
  double sum = 0.0;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)kNormBlocks * 256) {
    const int64_t i = t / cols, j = t - i * cols;
    float v = to_f32(((const E*)g.data)[q * g.batch + i * g.row + j]);
    if (m.data) {
      float* mp = (float*)m.data + q * m.batch + i * m.row + j;
      const float mn = fmaf(mu, *mp, v);
      *mp = mn;
      v = nesterov ? fmaf(mu, mn, v) : mn;
    }
    x[q * n + t] = v;
    sum += (double)v * v;
  }
  __shared__ double s[256];
  s[threadIdx.x] = sum;
  __syncthreads();
  for (int k = 128; k; k >>= 1) {
    if (threadIdx.x < k) s[threadIdx.x] += s[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) part[q * kNormBlocks + blockIdx.x] = s[0];
}

__global__ __launch_bounds__(256) void scale_kernel(float* x, const double* part, double eps, int64_t n) {
  const int q = blockIdx.y;
  double sum = 0.0;
  for (int i = 0; i < kNormBlocks; i++) sum += part[q * kNormBlocks + i];
  const double inv = 1.0 / (sqrt(sum) + eps);
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256)
    x[q * n + t] = (float)(x[q * n + t] * inv);
}

// C = alpha * product + beta * D
struct Axpby {
  float *y;
  const float* d;
  float alpha, beta;
  int64_t row, batch;
  __device__ __forceinline__ void operator()(int q, int, int i, int j, float p) const {
    const int64_t at = q * batch + i * row + j;
    y[at] = fmaf(alpha, p, d ? beta * d[at] : 0.0f);
  }
};

// The last step's X' as o, or into the weights: w <- keep w - step X'.
template <class E>
struct LastOut {
  const float* x;
  float a;
  int64_t row, batch;
  E* o;
  int64_t o_row, o_batch;
  float keep, step;
  int update;
  __device__ __forceinline__ void operator()(int q, int, int i, int j, float p) const {
    const float v = fmaf(a, x[q * batch + i * row + j], p);
    E* at = o + q * o_batch + i * o_row + j;
    *at = from_f32<E>(update ? fmaf(-step, v, keep * to_f32(*at)) : v);
  }
};

template <class E>
__global__ __launch_bounds__(256) void finish_kernel(LastOut<E> out, int32_t rows, int32_t cols) {
  const int64_t n = (int64_t)rows * cols;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256)
    out(blockIdx.y, 0, (int)(t / cols), (int)(t % cols), 0.0f);
}

template <class G, class O>
int newton_schulz(phz_ops* o, hipStream_t stream, const phz_muon_cfg& cfg, int64_t batch, int32_t rows, int32_t cols,
                  View g, View m, LastOut<O> last) {
  const int64_t n = (int64_t)rows * cols, s = std::min(rows, cols);
  const uint64_t part_bytes = ((uint64_t)batch * kNormBlocks * 8 + 255) & ~255ull;
  const uint64_t bytes = part_bytes + (uint64_t)batch * (2 * n + 2 * s * s) * 4;
  char* ws = o->workspace(stream, bytes);
  if (!ws) return 1;
  double* part = (double*)ws;
  float* x = (float*)(ws + part_bytes);
  float *y = x + batch * n, *a = y + batch * n, *p = a + batch * s * s;
  hipLaunchKernelGGL(gather_kernel<G>, dim3(kNormBlocks, (unsigned)batch), dim3(256), 0, stream, g, m,
                     (float)cfg.momentum, cfg.nesterov, x, part, rows, cols);
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n, 256), 4096);
  hipLaunchKernelGGL(scale_kernel, dim3(blocks, (unsigned)batch), dim3(256), 0, stream, x, part, cfg.eps, n);
  const bool wide = rows <= cols;
  const int32_t si = (int32_t)s, l = std::max(rows, cols);
  last.row = cols, last.batch = n;
  if (cfg.steps == 0) {
    last.x = x, last.a = 1.0f;
    hipLaunchKernelGGL(finish_kernel<O>, dim3(blocks, (unsigned)batch), dim3(256), 0, stream, last, rows, cols);
  }
  for (int k = 0; k < cfg.steps; k++) {
    const Operand xo{x, cols, n}, ao{a, s, s * s}, po{p, s, s * s};
    const Axpby gram{a, nullptr, 1.0f, 0.0f, s, s * s};
    const GemmShape gs{si, si, l, l, 1}, ss{si, si, si, si, 1};
    if (wide) launch_gemm_any<float, true, true>(o, stream, xo, xo, gs, (int)batch, gram);
    else launch_gemm_any<float, false, false>(o, stream, xo, xo, gs, (int)batch, gram);
    launch_gemm_any<float, true, true>(o, stream, ao, ao, ss, (int)batch,
                                       Axpby{p, a, (float)cfg.c, (float)cfg.b, s, s * s});
    const GemmShape xs{rows, cols, si, si, 1};
    if (k + 1 < cfg.steps) {
      const Axpby next{y, x, 1.0f, (float)cfg.a, cols, n};
      if (wide) launch_gemm_any<float, true, false>(o, stream, po, xo, xs, (int)batch, next);
      else launch_gemm_any<float, true, true>(o, stream, xo, po, xs, (int)batch, next);
    } else {
      last.x = x, last.a = (float)cfg.a;
      if (wide) launch_gemm_any<float, true, false>(o, stream, po, xo, xs, (int)batch, last);
      else launch_gemm_any<float, true, true>(o, stream, xo, po, xs, (int)batch, last);
    }
    std::swap(x, y);
  }
  return launched(o, "orthogonalize") ? 0 : 1;
}

bool check_cfg(phz_ops* o, const phz_muon_cfg* c, bool step) {
  if (!c) return o->err = "configuration is missing", false;
  if (c->steps < 0 || c->steps > 64) return o->err = fmt("steps is %d, expected 0 to 64", c->steps), false;
  if (!isfinite(c->a) || !isfinite(c->b) || !isfinite(c->c)) return o->err = "coefficients have to be finite", false;
  if (!(c->eps >= 0) || !isfinite(c->eps)) return o->err = "eps has to be finite and not negative", false;
  if (step && (!isfinite(c->lr) || !isfinite(c->momentum) || !isfinite(c->weight_decay)))
    return o->err = "lr, momentum and weight_decay have to be finite", false;
  return true;
}

// Batch, rows and cols of a matrix or a batch of them.
struct Sizes {
  int64_t batch, rows, cols;
};
bool sizes(phz_ops* o, const char* name, const phz_tensor* t, Sizes* s) {
  if (!t) return o->err = fmt("%s is missing", name), false;
  if (t->dtype != PHZ_F32 && t->dtype != PHZ_BF16)
    return o->err = fmt("%s is %s, expected f32 or bf16", name, dtype_name(t->dtype)), false;
  if (t->ndim != 2 && t->ndim != 3)
    return o->err = fmt("%s has %d dimensions, expected a matrix or a batch of them", name, t->ndim), false;
  const int k = t->ndim - 2;
  *s = Sizes{k ? t->size[0] : 1, t->size[k], t->size[k + 1]};
  if (s->rows > 32768 || s->cols > 1 << 20 || s->cols * s->rows > 1ll << 30 || std::min(s->rows, s->cols) > 32768)
    return o->err = fmt("%s is %lld x %lld: at most 32768 rows and 2^30 elements a matrix", name, (long long)s->rows,
                        (long long)s->cols),
           false;
  if (s->batch > 65535) return o->err = "at most 65535 matrices a call", false;
  return true;
}
View view(const phz_tensor* t) {
  const int k = t->ndim - 2;
  return View{t->data, k ? t->stride[0] : 0, t->stride[k]};
}

}  // namespace

extern "C" {

int phz_orthogonalize(phz_ops* o, void* stream, const phz_muon_cfg* cfg, const phz_tensor* g, const phz_tensor* out) {
  return guarded(o, [&] {
    Sizes s;
    if (!check_cfg(o, cfg, false) || !sizes(o, "g", g, &s)) return 1;
    Want in{g->ndim, {g->size[0], g->size[1], g->ndim == 3 ? g->size[2] : 0}, g->dtype, true, false};
    if (!check(o, "g", g, in)) return 1;
    in.output = true;
    if (!check(o, "o", out, in) || !apart(o, "o", out, "g", g)) return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (empty(g)) return 0;
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    const View ov = view(out);
    phz_muon_cfg c = *cfg;
    if (g->dtype == PHZ_F32) {
      LastOut<float> last{};
      last.o = (float*)ov.data, last.o_row = ov.row, last.o_batch = ov.batch;
      return newton_schulz<float, float>(o, (hipStream_t)stream, c, s.batch, (int32_t)s.rows, (int32_t)s.cols, view(g),
                                         View{}, last);
    }
    LastOut<bf16> last{};
    last.o = (bf16*)ov.data, last.o_row = ov.row, last.o_batch = ov.batch;
    return newton_schulz<bf16, bf16>(o, (hipStream_t)stream, c, s.batch, (int32_t)s.rows, (int32_t)s.cols, view(g),
                                     View{}, last);
  });
}

int phz_muon_step(phz_ops* o, void* stream, const phz_muon_cfg* cfg, const phz_tensor* w, const phz_tensor* g,
                  const phz_tensor* m) {
  return guarded(o, [&] {
    Sizes s;
    if (!check_cfg(o, cfg, true) || !sizes(o, "g", g, &s)) return 1;
    Want in{g->ndim, {g->size[0], g->size[1], g->ndim == 3 ? g->size[2] : 0}, g->dtype, true, false};
    if (!check(o, "g", g, in)) return 1;
    in.output = true;
    in.dtype = PHZ_F32;
    if (!check(o, "w", w, in) || !check(o, "m", m, in) || !apart(o, "w", w, "g", g) || !apart(o, "m", m, "g", g) ||
        !apart(o, "w", w, "m", m))
      return 1;
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    if (empty(g)) return 0;
    DeviceGuard guard(o);
    if (!guard.ok) return 1;
    const View wv = view(w);
    LastOut<float> last{};
    last.o = (float*)wv.data, last.o_row = wv.row, last.o_batch = wv.batch;
    last.update = 1;
    last.keep = (float)(1.0 - cfg->lr * cfg->weight_decay);
    last.step = (float)(cfg->lr * sqrt(std::max(1.0, (double)s.rows / (double)s.cols)));
    return g->dtype == PHZ_F32
               ? newton_schulz<float, float>(o, (hipStream_t)stream, *cfg, s.batch, (int32_t)s.rows, (int32_t)s.cols,
                                             view(g), view(m), last)
               : newton_schulz<bf16, float>(o, (hipStream_t)stream, *cfg, s.batch, (int32_t)s.rows, (int32_t)s.cols,
                                            view(g), view(m), last);
  });
}

}  // extern "C"
