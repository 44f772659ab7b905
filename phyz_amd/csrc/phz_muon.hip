// phz_muon.hip — orthogonalised updates: Newton-Schulz steps on a gradient's
// matrix (or a batch of them) and Muon's update of the weights.
//
//   X = g / (|g|_F + eps);   X <- a X + (b A + c A^2) X,  A = X X^T
//
// on whichever side is shorter: for tall matrices A = X^T X and
// X <- a X + X (b A + c A^2), so nothing is transposed.
#include "phz_gemm_fast.h"

#include <math.h>

#include <algorithm>

using namespace phzop;

namespace {

struct View {
  void* data;
  int64_t batch, row;
};

// Blocks that share a matrix's sum of squares; each leaves one partial.
int norm_blocks(int64_t elements) { return (int)std::max<int64_t>(1, std::min<int64_t>(512, elements / 4096)); }

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s[4];
#pragma unroll
  for (int k = 32; k; k >>= 1) v += __shfl_xor(v, k);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Eight neighbouring elements of a row (fewer at its end: zeros).
template <class E>
__device__ __forceinline__ void load8(const View& t, int q, int64_t i, int j, int cols, float* v) {
  const E* p = (const E*)t.data + q * t.batch + i * t.row + j;
  if (j + 8 <= cols) {
    const Pack<E, 8> w = *(const Pack<E, 8>*)p;
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = to_f32(w.v[c]);
  } else {
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = j + c < cols ? to_f32(p[c]) : 0.0f;
  }
}

// The matrix: g, or with a momentum m (already updated) what Muon
// orthogonalises.
template <class E>
struct Source {
  View g, m;
  float mu;
  int nesterov;
  __device__ __forceinline__ void at(int q, int64_t i, int j, int cols, float* v) const {
    if (!m.data) return load8<E>(g, q, i, j, cols, v);
    load8<float>(m, q, i, j, cols, v);
    if (nesterov) {
      float d[8];
      load8<E>(g, q, i, j, cols, d);
#pragma unroll
      for (int c = 0; c < 8; c++) v[c] = fmaf(mu, v[c], d[c]);
    }
  }
};

// m <- mu m + g where there is a momentum, for eight elements; the sum of the
// squares of what is orthogonalised, in f64: gradients whose squares leave
// f32's range have a norm too.
template <class E>
__device__ __forceinline__ double update8(const Source<E>& s, int q, int64_t i, int j, int cols) {
  float v[8];
  if (s.m.data) {
    float d[8];
    load8<float>(s.m, q, i, j, cols, v);
    load8<E>(s.g, q, i, j, cols, d);
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = fmaf(s.mu, v[c], d[c]);
    float* mp = (float*)s.m.data + q * s.m.batch + i * s.m.row + j;
    if (j + 8 <= cols) {
      Pack<float, 8> w;
#pragma unroll
      for (int c = 0; c < 8; c++) w.v[c] = v[c];
      *(Pack<float, 8>*)mp = w;
    } else {
      for (int c = 0; j + c < cols; c++) mp[c] = v[c];
    }
    if (s.nesterov) {
#pragma unroll
      for (int c = 0; c < 8; c++) v[c] = fmaf(s.mu, v[c], d[c]);
    }
  } else {
    load8<E>(s.g, q, i, j, cols, v);
  }
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < 8; c++) sum = fma((double)v[c], (double)v[c], sum);
  return sum;
}

// A launch's latency at a policy's sizes (2 x 256 x 256 f32 3.5 us), memory above
// (1024 x 4096 bf16 5.0 us for 8.4 MB).
template <class E>
__global__ __launch_bounds__(256) void norm_kernel(Source<E> s, double* part, int32_t rows, int32_t cols) {
  const int q = blockIdx.y;
  const uint32_t per = (cols + 7) / 8, n = (uint32_t)rows * per;  // eights
  double sum = 0.0;
  for (uint32_t t = blockIdx.x * 256 + threadIdx.x; t < n; t += gridDim.x * 256) {
    const uint32_t i = t / per;
    sum += update8(s, q, i, (t - i * per) * 8, cols);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) part[(int64_t)q * gridDim.x + blockIdx.x] = sum;
}

// X as planes of f16: the value times `scale` as hi + lo (or hi alone), rows of
// `ld` (a multiple of eight), zeros past the matrix's columns.
struct Planes {
  half_t* data;
  int64_t plane, row, batch;  // elements
};

template <int P>
__device__ __forceinline__ void put_planes(const Planes& p, int64_t at, const float* v) {
  Pack<half_t, 8> hi, lo;
#pragma unroll
  for (int c = 0; c < 8; c++) {
    hi.v[c] = from_f32<half_t>(v[c]);
    if (P == 2) lo.v[c] = from_f32<half_t>(v[c] - to_f32(hi.v[c]));
  }
  *(Pack<half_t, 8>*)(p.data + at) = hi;
  if (P == 2) *(Pack<half_t, 8>*)(p.data + p.plane + at) = lo;
}
template <int P>
struct PlaneEight {
  Pack<half_t, 8> hi, lo;
  __device__ __forceinline__ void get(const Planes& p, int64_t at) {
    hi = *(const Pack<half_t, 8>*)(p.data + at);
    if (P == 2) lo = *(const Pack<half_t, 8>*)(p.data + p.plane + at);
  }
  __device__ __forceinline__ float value(int c) const { return P == 2 ? to_f32(hi.v[c]) + to_f32(lo.v[c]) : to_f32(hi.v[c]); }
};

__device__ __forceinline__ double inverse_norm(const double* part, int parts, int q, double eps) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) sum += part[(int64_t)q * parts + i];
  return 1.0 / (sqrt(block_sum(sum)) + eps);
}

// X = the matrix over its norm, as two planes, or in f32 where xf is given. Each
// workgroup adds the norm's parts itself, its first elements being on their way
// meanwhile: 2 x 256 x 256 f32 3.5 us, 1024 x 4096 bf16 10.6 us for 25 MB.
template <class E>
__global__ __launch_bounds__(256) void scale_kernel(Source<E> s, const double* part, int parts, double eps, float scale,
                                                    Planes x, float* xf, int32_t rows, int32_t cols) {
  const int q = blockIdx.y;
  const uint32_t per = (cols + 7) / 8, n = (uint32_t)rows * per;
  uint32_t t = blockIdx.x * 256 + threadIdx.x, i = t / per;
  int j = (t - i * per) * 8;
  float v[8];
  if (t < n) s.at(q, i, j, cols, v);  // on its way during the norm's sum
  const double inv = inverse_norm(part, parts, q, eps) * scale;
  while (t < n) {
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = (float)(v[c] * inv);
    if (xf) {
#pragma unroll
      for (int c = 0; c < 8; c++)
        if (j + c < cols) xf[((int64_t)q * rows + i) * cols + j + c] = v[c];
    } else {
      put_planes<2>(x, q * x.batch + i * x.row + j, v);
    }
    t += gridDim.x * 256;
    i = t / per, j = (t - i * per) * 8;
    if (t < n) s.at(q, i, j, cols, v);
  }
}

// y = alpha sum + beta d, as PY planes; d has PD.
template <int PY, int PD>
struct PlanesOut : NoColumns {
  static constexpr bool kRagged = false;  // rows of planes are whole eights
  Planes y, d;
  float alpha, beta;
  int32_t cols;  // columns that exist: zeros beyond
  PlanesOut(Planes y_, Planes d_, float al, float be, int32_t c) : y(y_), d(d_), alpha(al), beta(be), cols(c) {}
  typedef PlaneEight<PD> Held;
  __device__ __forceinline__ void fetch(int q, int i, int j, int, Held& h) const {
    if (d.data) h.get(d, q * d.batch + i * d.row + j);
  }
  __device__ __forceinline__ void put8(int q, int, int i, int j, int, const float* sums, const Held& h, const Columns&) const {
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; c++)
      v[c] = j + c < cols ? (d.data ? fmaf(alpha, sums[c], beta * h.value(c)) : alpha * sums[c]) : 0.0f;
    put_planes<PY>(y, q * y.batch + i * y.row + j, v);
  }
};

// The last X' as o, or into the weights: w <- keep w - step X'.
template <class O>
struct Result {
  O* o;
  int64_t row, batch;
  float keep, step;
  int update;
  __device__ __forceinline__ void put(int q, int64_t i, int64_t j, float v) const {
    O* at = o + q * batch + i * row + j;
    *at = from_f32<O>(update ? fmaf(-step, v, keep * to_f32(*at)) : v);
  }
  __device__ __forceinline__ void put8(int q, int64_t i, int64_t j, const float* v, const Pack<O, 8>& before) const {
    Pack<O, 8> w;
#pragma unroll
    for (int c = 0; c < 8; c++) w.v[c] = from_f32<O>(update ? fmaf(-step, v[c], keep * to_f32(before.v[c])) : v[c]);
    *(Pack<O, 8>*)(o + q * batch + i * row + j) = w;
  }
};

// alpha sum + beta X into the result.
template <class O>
struct LastOut : NoColumns {
  static constexpr bool kRagged = false;  // rows of planes are whole eights
  Planes x;
  float alpha, beta;
  int32_t cols;
  Result<O> out;
  LastOut(Planes x_, float al, float be, int32_t c, const Result<O>& o) : x(x_), alpha(al), beta(be), cols(c), out(o) {}
  struct Held {
    PlaneEight<2> x;
    Pack<O, 8> before;
  };
  __device__ __forceinline__ void fetch(int q, int i, int j, int, Held& h) const {
    h.x.get(x, q * x.batch + i * x.row + j);
    if (out.update && j + 8 <= cols) h.before = *(const Pack<O, 8>*)(out.o + q * out.batch + i * out.row + j);
  }
  __device__ __forceinline__ void put8(int q, int, int i, int j, int, const float* sums, const Held& h, const Columns&) const {
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = fmaf(alpha, sums[c], beta * h.x.value(c));
    if (j + 8 <= cols) out.put8(q, i, j, v, h.before);
    else
      for (int c = 0; c < 8 && j + c < cols; c++) out.put(q, i, j + c, v[c]);
  }
};

// C = alpha product + beta D in f32 (any coefficients; see newton_schulz_any).
struct Axpby : NothingAhead {
  static constexpr bool kRagged = true;
  float *y;
  const float* d;
  float alpha, beta;
  int64_t row, batch;
  Axpby(float* y_, const float* d_, float al, float be, int64_t r, int64_t b)
      : y(y_), d(d_), alpha(al), beta(be), row(r), batch(b) {}
  __device__ __forceinline__ void put8(int q, int s, int i, int j, int left, const float* p, const Held&, const Columns&) const {
    for (int c = 0; c < 8 && c < left; c++) put1(q, s, i, j + c, p[c]);
  }
  __device__ __forceinline__ void put1(int q, int, int i, int j, float p) const {
    const int64_t at = q * batch + i * row + j;
    y[at] = fmaf(alpha, p, d ? beta * d[at] : 0.0f);
  }
};

template <class O>
struct LastAny : NothingAhead {
  static constexpr bool kRagged = true;
  const float* x;
  float a;
  int64_t row, batch;
  Result<O> out;
  LastAny(const float* x_, float a_, int64_t r, int64_t b, const Result<O>& o) : x(x_), a(a_), row(r), batch(b), out(o) {}
  __device__ __forceinline__ void put8(int q, int s, int i, int j, int left, const float* p, const Held&, const Columns&) const {
    for (int c = 0; c < 8 && c < left; c++) put1(q, s, i, j + c, p[c]);
  }
  __device__ __forceinline__ void put1(int q, int, int i, int j, float p) const {
    out.put(q, i, j, fmaf(a, x[q * batch + i * row + j], p));
  }
};

template <class O>
__global__ __launch_bounds__(256) void finish_kernel(LastAny<O> out, int32_t rows, int32_t cols) {
  const int64_t n = (int64_t)rows * cols;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256)
    out.put1(blockIdx.y, 0, (int)(t / cols), (int)(t % cols), 0.0f);
}

// The largest |p(s)| for s in [0, top], p odd: p(s) = a s + b s^3 + c s^5, at
// the ends or where p' = 0, a quadratic in s^2.
double quintic_top(double a, double b, double c, double top) {
  auto p = [&](double s) { return fabs(s * (a + s * s * (b + s * s * c))); };
  double best = p(top);
  auto at = [&](double t) {
    if (t > 0 && t < top * top) best = std::max(best, p(sqrt(t)));
  };
  if (c == 0.0) {
    if (b != 0.0) at(-a / (3 * b));
  } else if (9 * b * b >= 20 * a * c) {
    const double d = sqrt(9 * b * b - 20 * a * c);
    at((-3 * b + d) / (10 * c));
    at((-3 * b - d) / (10 * c));
  }
  return best;
}

// What the iterates' singular values stay below, and so every element: of X,
// of A, and of b A + c A^2.
struct Bounds {
  double x, a, p;
};
Bounds bounds(const phz_muon_cfg& g) {
  Bounds m{1.0, 1.0, 0.0};
  double top = 1.0;
  for (int k = 0; k < g.steps; k++) {
    const double t = top * top;
    m.a = std::max(m.a, t);
    m.p = std::max(m.p, fabs(t * (g.b + g.c * t)));
    if (g.c != 0.0 && -g.b / (2 * g.c) > 0 && -g.b / (2 * g.c) < t) m.p = std::max(m.p, g.b * g.b / fabs(4 * g.c));
    top = quintic_top(g.a, g.b, g.c, top) * 1.001;
    if (!(top < 1e30)) {  // or NaN
      m.x = INFINITY;
      break;
    }
    m.x = std::max(m.x, top);
  }
  return m;
}

// The power of two that puts values up to `bound` within half of f16's range.
double f16_scale(double bound) { return exp2(floor(log2(32768.0 / bound))); }

// Any coefficients: products of f32 operands at any size (phz_gemm.h).
template <class G, class O>
int newton_schulz_any(phz_ops* o, hipStream_t stream, const phz_muon_cfg& cfg, int64_t batch, int32_t rows,
                      int32_t cols, const Source<G>& src, const Result<O>& out) {
  const int64_t n = (int64_t)rows * cols, s = std::min(rows, cols);
  const int parts = norm_blocks(n);
  const uint64_t part_bytes = ((uint64_t)batch * parts * 8 + 255) & ~255ull;
  char* ws = o->workspace(stream, part_bytes + (uint64_t)batch * (2 * n + 2 * s * s) * 4);
  if (!ws) return 1;
  double* part = (double*)ws;
  float* x = (float*)(ws + part_bytes);
  float *y = x + batch * n, *a = y + batch * n, *p = a + batch * s * s;
  hipLaunchKernelGGL(norm_kernel<G>, dim3(parts, (unsigned)batch), dim3(256), 0, stream, src, part, rows, cols);
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n, 2048), 2048);
  hipLaunchKernelGGL(scale_kernel<G>, dim3(blocks, (unsigned)batch), dim3(256), 0, stream, src, part, parts, cfg.eps,
                     1.0f, Planes{}, x, rows, cols);
  const bool wide = rows <= cols;
  const int32_t si = (int32_t)s, l = std::max(rows, cols);
  if (cfg.steps == 0)
    hipLaunchKernelGGL(finish_kernel<O>, dim3(blocks, (unsigned)batch), dim3(256), 0, stream,
                       LastAny<O>{x, 1.0f, cols, n, out}, rows, cols);
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
      const LastAny<O> last{x, (float)cfg.a, cols, n, out};
      if (wide) launch_gemm_any<float, true, false>(o, stream, po, xo, xs, (int)batch, last);
      else launch_gemm_any<float, true, true>(o, stream, xo, po, xs, (int)batch, last);
    }
    std::swap(x, y);
  }
  return launched(o, "orthogonalize") ? 0 : 1;
}

FastArgs product(const Planes& a, const Planes& b, int32_t m, int32_t n, int32_t k, int32_t a_rows, int32_t b_rows) {
  FastArgs f{};
  f.a = (const char*)a.data, f.b = (const char*)b.data;
  f.a_row = a.row * 2, f.b_row = b.row * 2, f.a_batch = a.batch * 2, f.b_batch = b.batch * 2;
  f.a_plane = (uint32_t)(a.plane * 2), f.b_plane = (uint32_t)(b.plane * 2);
  f.m = m, f.n = n, f.k = k, f.a_rows = a_rows, f.b_rows = b_rows;
  return f;
}

// The iterates as f16 planes. X starts at norm 1 and its singular values stay
// below a bound that the coefficients give, so a power of two puts every
// element in f16's range: no element leaves it, and what falls below its
// smallest is 2^-39 of what the bound allows.
//
// P = 2, for f32 gradients: every operand is hi + lo, 22 bits. P = 1, for bf16
// ones: products take hi alone, 11 bits to the gradient's 8, but X is carried
// as hi + lo through a X. Its rounding to 11 bits would be noise in every
// direction, which the steps raise along with the small singular values (3.3e-3
// of the result at 1024 x 4096 with a few directions ten times the rest,
// against 1.7e-3 for rounding the result alone); that of A and of the products
// only moves the directions that are large.
//
// Bound, product by product, by one round of tiles: its start from the memory-
// side cache (the last product's tiles were written by other dies), its stages,
// its way out. 2 x 256 x 256 f32 94 us in 17 launches of 3.5 to 6; 1024 x 4096
// bf16 213, 15 products of 7 to 19; 1501 x 1001 f32 287, of 16 to 25.
template <class G, class O, int P>
int newton_schulz(phz_ops* o, hipStream_t stream, const phz_muon_cfg& cfg, const Bounds& top, int64_t batch,
                  int32_t rows, int32_t cols, const Source<G>& src, const Result<O>& out) {
  const bool wide = rows <= cols;
  const int32_t s = std::min(rows, cols), l = std::max(rows, cols), s8 = (s + 7) & ~7, c8 = (cols + 7) & ~7;
  const int parts = norm_blocks((int64_t)rows * cols);
  const uint64_t part_bytes = ((uint64_t)batch * parts * 8 + 255) & ~255ull;
  // A matrix's planes lie together, each from a multiple of 256 bytes.
  const int64_t xn = ((int64_t)rows * c8 + 127) & ~127ll, an = ((int64_t)s * s8 + 127) & ~127ll;
  // The Gram product is long and has few tiles: it may be split.
  const FastPlan gplan = plan_fast(o, s, s8, wide ? c8 : l, batch, P, true), pplan = plan_fast(o, s, s8, s8, batch, P, true),
                 xplan = plan_fast(o, rows, c8, s, batch, P, false);
  const uint64_t split_bytes = (std::max(gplan.part_bytes, pplan.part_bytes) + 255) & ~255ull;
  char* ws = o->workspace(stream, part_bytes + split_bytes + (uint64_t)batch * (4 * xn + 2 * P * an) * 2);
  if (!ws) return 1;
  double* part = (double*)ws;
  float* sums = (float*)(ws + part_bytes);
  half_t* h = (half_t*)(ws + part_bytes + split_bytes);
  Planes x{h, xn, c8, 2 * xn}, y{h + 2 * batch * xn, xn, c8, 2 * xn};
  const Planes a{h + 4 * batch * xn, an, s8, P * an}, p{h + (4 * xn + P * an) * batch, an, s8, P * an};
  const double sx = f16_scale(top.x), sa = f16_scale(top.a), sp = f16_scale(top.p > 0 ? top.p : 1.0);
  hipLaunchKernelGGL(norm_kernel<G>, dim3(parts, (unsigned)batch), dim3(256), 0, stream, src, part, rows, cols);
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div((int64_t)rows * c8, 2048), 1024);
  hipLaunchKernelGGL(scale_kernel<G>, dim3(blocks, (unsigned)batch), dim3(256), 0, stream, src, part, parts, cfg.eps,
                     (float)sx, x, nullptr, rows, cols);
  for (int k = 0; k < cfg.steps; k++) {
    const PlanesOut<P, P> gram{a, Planes{}, (float)(sa / (sx * sx)), 0.0f, s};
    if (wide) launch_gemm_fast<half_t, P, true, true>(o, stream, product(x, x, s, s8, c8, s, s), (int)batch, gplan, sums,
                                                           gram);
    else launch_gemm_fast<half_t, P, false, false>(o, stream, product(x, x, s, s8, l, s8, s8), (int)batch, gplan, sums,
                                                     gram);
    const PlanesOut<P, P> poly{p, a, (float)(cfg.c * sp / (sa * sa)), (float)(cfg.b * sp / sa), s};
    launch_gemm_fast<half_t, P, true, true>(o, stream, product(a, a, s, s8, s8, s, s), (int)batch, pplan, sums, poly);
    const FastArgs f = wide ? product(p, x, rows, c8, s, s, c8) : product(x, p, rows, c8, s8, rows, s);
    if (k + 1 < cfg.steps) {
      const PlanesOut<2, 2> next{y, x, (float)(1.0 / sp), (float)cfg.a, cols};
      if (wide) launch_gemm_fast<half_t, P, true, false>(o, stream, f, (int)batch, xplan, nullptr, next);
      else launch_gemm_fast<half_t, P, true, true>(o, stream, f, (int)batch, xplan, nullptr, next);
    } else {
      const LastOut<O> last{x, (float)(1.0 / (sp * sx)), (float)(cfg.a / sx), cols, out};
      if (wide) launch_gemm_fast<half_t, P, true, false>(o, stream, f, (int)batch, xplan, nullptr, last);
      else launch_gemm_fast<half_t, P, true, true>(o, stream, f, (int)batch, xplan, nullptr, last);
    }
    std::swap(x, y);
  }
  return launched(o, "orthogonalize") ? 0 : 1;
}

// ── a matrix that fits a compute unit ───────────────────────────────────────
//
// Up to about 128 x 160 or 64 x 500, one workgroup does all of it: the
// seventeen launches of the path above would each take a few microseconds for
// next to no work. X lies in LDS as hi + lo, shorter side along rows (tall
// matrices transposed on the way in and out), A and then b A + c A^2 beside it.
// Each product's 32 x 32 blocks are shared among sixteen waves, which hold their
// sums until everybody has read what they replace. Sums come out with four
// neighbouring rows in a lane: A and the polynomial are symmetric and X' is
// taken as X^T P, so those are four neighbours along a row of LDS, too.
// Rows of LDS are eight elements longer than whole 32, which puts 16 rows'
// reads on all banks. Bound by the latency of its barriers and LDS reads: 34 x 33
// f32 60 -> 20 us against those launches, 8 x 103 x 47 f32 72 -> 27, 128 x 128
// bf16 65 -> 35.
constexpr int kOneWaves = 16, kOneBlocks = 3, kOneLds = 156 * 1024, kOneLittle = 40 * 1024;

struct OneShape {
  int32_t s, l;    // shorter and longer side, in whole 32
  int32_t xr, ar;  // elements between rows of X and of A
  int64_t bytes;
};
OneShape one_shape(int64_t rows, int64_t cols, int planes) {
  OneShape o{};
  o.s = (int32_t)((std::min(rows, cols) + 31) / 32 * 32), o.l = (int32_t)((std::max(rows, cols) + 31) / 32 * 32);
  o.xr = o.l + 8, o.ar = o.s + 8;
  o.bytes = (int64_t)o.s * o.xr * 4 + (int64_t)o.s * o.ar * 2 * planes;
  return o;
}

struct Four {
  half_t v[4];
};

template <class G, class O, int P, int LDS>
__global__ __launch_bounds__(kOneWaves * 64) void one_kernel(Source<G> src, phz_muon_cfg cfg, OneShape sh, float sx, float sa,
                                                             float sp, Result<O> out, int32_t rows, int32_t cols) {
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  __shared__ double norm;
  half_t* xh = (half_t*)lds;
  half_t* xl = xh + sh.s * sh.xr;
  half_t* ah = xl + sh.s * sh.xr;
  half_t* al = ah + sh.s * sh.ar;  // P = 2
  const int q = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool wide = rows <= cols;
  constexpr int T = kOneWaves * 64;

  // The matrix's norm (and the momentum's update), then X over it; a thread
  // meets the same elements in both passes.
  for (int t = threadIdx.x; t < sh.s * sh.xr / 4; t += T) ((uint64_t*)lds)[t] = 0, ((uint64_t*)xl)[t] = 0;
  const uint32_t per = (cols + 7) / 8, n = (uint32_t)rows * per;  // eights
  double sum = 0.0;
  for (uint32_t t = threadIdx.x; t < n; t += T) {
    const uint32_t i = t / per;
    sum += update8(src, q, i, (t - i * per) * 8, cols);
  }
  __shared__ double part[kOneWaves];
#pragma unroll
  for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < kOneWaves; w++) all += part[w];
    norm = sx / (sqrt(all) + cfg.eps);
  }
  __syncthreads();
  const double inv = norm;
  for (uint32_t t = threadIdx.x; t < n; t += T) {
    const uint32_t i = t / per;
    const int j = (t - i * per) * 8;
    float v[8];
    src.at(q, i, j, cols, v);
#pragma unroll
    for (int c = 0; c < 8; c++) {
      if (j + c >= cols) break;
      const float x = (float)(v[c] * inv);
      const int at = wide ? i * sh.xr + j + c : (j + c) * sh.xr + i;
      xh[at] = from_f32<half_t>(x);
      xl[at] = from_f32<half_t>(x - to_f32(xh[at]));
    }
  }
  __syncthreads();

  const int fr = lane & 31, fk = (lane >> 5) * 8;  // fragments: row lane % 32, eight k from here
  auto along = [&](const half_t* p, int pitch, int row, int k) { return *(const s16x8*)(p + (row + fr) * pitch + k + fk); };
  // Eight k (rows of X) of column col + lane % 32.
  auto across = [&](const half_t* p, int col, int k) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const half_t* at = p + (k + fk + ((lane & 15) >> 2)) * sh.xr + col + (lane & 16) + (lane & 3) * 4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + 4 * sh.xr));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto times = [&](s16x8 ahi, s16x8 alo, s16x8 bhi, s16x8 blo, f32x16 c) {
    if (P == 2) {
      c = Mfma<half_t>::run(alo, bhi, c);
      c = Mfma<half_t>::run(ahi, blo, c);
    }
    return Mfma<half_t>::run(ahi, bhi, c);
  };
  auto put4 = [&](half_t* hi, half_t* lo, int at, const float* v) {
    Four h, l;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      h.v[c] = from_f32<half_t>(v[c]);
      if (lo) l.v[c] = from_f32<half_t>(v[c] - to_f32(h.v[c]));
    }
    *(Four*)(hi + at) = h;
    if (lo) *(Four*)(lo + at) = l;
  };
  // Where a block's group of four sums lies: column `col` + lane % 32 of the
  // product, its row `row` + 8 g + 4 (lane / 32).
  auto place = [&](int pitch, int row, int col, int g) { return (col + fr) * pitch + row + g * 8 + (lane >> 5) * 4; };
  const int sb = sh.s / 32, lb = sh.l / 32, ablocks = sb * sb, xblocks = sb * lb;  // at most 16, 48
  const int ai = wave / sb * 32, aj = wave % sb * 32;
  const float to_a = sa / (sx * sx), to_c = (float)cfg.c * (sp / (sa * sa)), to_b = (float)cfg.b * (sp / sa);
  for (int step = 0; step < cfg.steps; step++) {
    // A = X X^T: nothing is replaced that others read.
    f32x16 c;
    if (wave < ablocks) {
#pragma unroll
      for (int r = 0; r < 16; r++) c[r] = 0.0f;
#pragma unroll 2
      for (int k = 0; k < sh.l; k += 16)
        c = times(along(xh, sh.xr, ai, k), P == 2 ? along(xl, sh.xr, ai, k) : s16x8{}, along(xh, sh.xr, aj, k),
                  P == 2 ? along(xl, sh.xr, aj, k) : s16x8{}, c);
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = c[g * 4 + r] * to_a;
        put4(ah, P == 2 ? al : nullptr, place(sh.ar, ai, aj, g), v);
      }
    }
    __syncthreads();
    // b A + c A^2, in A's place once everybody has read A.
    if (wave < ablocks) {
#pragma unroll
      for (int r = 0; r < 16; r++) c[r] = 0.0f;
#pragma unroll 2
      for (int k = 0; k < sh.s; k += 16)
        c = times(along(ah, sh.ar, ai, k), P == 2 ? along(al, sh.ar, ai, k) : s16x8{}, along(ah, sh.ar, aj, k),
                  P == 2 ? along(al, sh.ar, aj, k) : s16x8{}, c);
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const Four h = *(const Four*)(ah + place(sh.ar, ai, aj, g));
        Four l{};
        if (P == 2) l = *(const Four*)(al + place(sh.ar, ai, aj, g));
#pragma unroll
        for (int r = 0; r < 4; r++)
          c[g * 4 + r] = fmaf(to_c, c[g * 4 + r], to_b * (P == 2 ? to_f32(h.v[r]) + to_f32(l.v[r]) : to_f32(h.v[r])));
      }
    }
    __syncthreads();
    if (wave < ablocks) {
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = c[g * 4 + r];
        put4(ah, P == 2 ? al : nullptr, place(sh.ar, ai, aj, g), v);
      }
    }
    __syncthreads();
    // X' = a X + (X^T P)^T, block columns of X by block rows of P.
    f32x16 d[kOneBlocks];
#pragma unroll
    for (int u = 0; u < kOneBlocks; u++) {
      const int t = wave + u * kOneWaves;
      if (t < xblocks) {
        const int col = t / sb * 32, row = t % sb * 32;
#pragma unroll
        for (int r = 0; r < 16; r++) d[u][r] = 0.0f;
#pragma unroll 2
        for (int k = 0; k < sh.s; k += 16)
          d[u] = times(across(xh, col, k), P == 2 ? across(xl, col, k) : s16x8{}, along(ah, sh.ar, row, k),
                       P == 2 ? along(al, sh.ar, row, k) : s16x8{}, d[u]);
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const int at = place(sh.xr, col, row, g);
          const Four h = *(const Four*)(xh + at), l = *(const Four*)(xl + at);
#pragma unroll
          for (int r = 0; r < 4; r++)
            d[u][g * 4 + r] = fmaf((float)cfg.a, to_f32(h.v[r]) + to_f32(l.v[r]), d[u][g * 4 + r] * (1.0f / sp));
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOneBlocks; u++) {
      const int t = wave + u * kOneWaves;
      if (t < xblocks) {
        const int col = t / sb * 32, row = t % sb * 32;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; r++) v[r] = d[u][g * 4 + r];
          put4(xh, xl, place(sh.xr, col, row, g), v);
        }
      }
    }
    __syncthreads();
  }
  for (uint32_t t = threadIdx.x; t < n; t += T) {
    const uint32_t i = t / per;
    const int j = (t - i * per) * 8;
    const bool whole = j + 8 <= cols;
    Pack<O, 8> before{};
    if (out.update && whole) before = *(const Pack<O, 8>*)(out.o + q * out.batch + i * out.row + j);
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; c++) {
      const int at = min(j + c, cols - 1) * (wide ? 1 : sh.xr) + i * (wide ? sh.xr : 1);
      v[c] = (to_f32(xh[at]) + to_f32(xl[at])) * (1.0f / sx);
    }
    if (whole) out.put8(q, i, j, v, before);
    else
      for (int c = 0; j + c < cols; c++) out.put(q, i, j + c, v[c]);
  }
}

template <class G, class O>
int orthogonal(phz_ops* o, hipStream_t stream, const phz_muon_cfg& cfg, int64_t batch, int64_t rows, int64_t cols,
               View g, View m, const Result<O>& out) {
  const Source<G> src{g, m, (float)cfg.momentum, cfg.nesterov};
  const Bounds top = bounds(cfg);
  // Coefficients that let the iterates grow past f16 (or no step at all).
  if (cfg.steps == 0 || !(top.x <= 64) || !(top.a <= 4096) || !(top.p <= 4096))
    return newton_schulz_any<G, O>(o, stream, cfg, batch, (int32_t)rows, (int32_t)cols, src, out);
  constexpr int P = sizeof(O) == 2 ? 1 : 2;
  const OneShape shape = one_shape(rows, cols, P);
  if (shape.s <= 128 && shape.bytes <= kOneLds && shape.s / 32 * (shape.l / 32) <= kOneBlocks * kOneWaves) {
    const float sx = (float)f16_scale(top.x), sa = (float)f16_scale(top.a), sp = (float)f16_scale(top.p > 0 ? top.p : 1.0);
    if (shape.bytes <= kOneLittle)
      hipLaunchKernelGGL((one_kernel<G, O, P, kOneLittle>), dim3((unsigned)batch), dim3(kOneWaves * 64), 0, stream, src, cfg,
                         shape, sx, sa, sp, out, (int32_t)rows, (int32_t)cols);
    else
      hipLaunchKernelGGL((one_kernel<G, O, P, kOneLds>), dim3((unsigned)batch), dim3(kOneWaves * 64), 0, stream, src, cfg,
                         shape, sx, sa, sp, out, (int32_t)rows, (int32_t)cols);
    return launched(o, "orthogonalize") ? 0 : 1;
  }
  return newton_schulz<G, O, P>(o, stream, cfg, top, batch, (int32_t)rows, (int32_t)cols, src, out);
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
  if (s->rows > 32768 || s->cols > 1 << 20 || s->cols * s->rows > 1ll << 30)
    return o->err = fmt("%s is %lld x %lld: at most 32768 rows, 2^20 columns and 2^30 elements a matrix", name,
                        (long long)s->rows, (long long)s->cols),
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
    if (g->dtype == PHZ_F32)
      return orthogonal<float, float>(o, (hipStream_t)stream, *cfg, s.batch, s.rows, s.cols, view(g), View{},
                                      Result<float>{(float*)ov.data, ov.row, ov.batch, 0.0f, 0.0f, 0});
    return orthogonal<bf16, bf16>(o, (hipStream_t)stream, *cfg, s.batch, s.rows, s.cols, view(g), View{},
                                  Result<bf16>{(bf16*)ov.data, ov.row, ov.batch, 0.0f, 0.0f, 0});
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
    const double shape = sqrt(std::max(1.0, (double)s.rows / (double)s.cols));
    const Result<float> out{(float*)wv.data, wv.row, wv.batch, (float)(1.0 - cfg->lr * cfg->weight_decay),
                            (float)(cfg->lr * shape), 1};
    return g->dtype == PHZ_F32
               ? orthogonal<float, float>(o, (hipStream_t)stream, *cfg, s.batch, s.rows, s.cols, view(g), view(m), out)
               : orthogonal<bf16, float>(o, (hipStream_t)stream, *cfg, s.batch, s.rows, s.cols, view(g), view(m), out);
  });
}

}  // extern "C"
