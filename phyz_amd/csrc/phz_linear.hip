// phz_linear.hip — the linear layer with its epilogue, y = act(x W^T + b) + r,
// and its gradients dx = dz W, dw = dz^T x, db = sum of dz over rows, for
// dz = dy act'(pre).
#include "phz_gemm.h"

#include <algorithm>

using namespace phzop;

namespace {

// ── activations ─────────────────────────────────────────────────────────────

// tanh as ocml's (2 ulp): its 1 - t cancels near 0 in any form made of one
// exponential, and f32 callers see that.
__device__ __forceinline__ float gate_of(float p) {  // sigmoid(p)
  const float q = signed_gate(p);
  return __float_as_int(q) < 0 ? fabsf(q) : 1.0f - fabsf(q);
}

constexpr float kGeluA = 0.79788456080286536f, kGeluB = 0.044715f;  // sqrt(2 / pi)

__device__ __forceinline__ float act_of(int act, float p) {
  switch (act) {
    case PHZ_ACT_TANH: return tanhf(p);
    case PHZ_ACT_RELU: return p < 0.0f ? 0.0f : p;  // NaN stays
    // p sigmoid(p); -inf has the limit 0, not the product's NaN.
    case PHZ_ACT_SILU: return p == -__builtin_inff() ? 0.0f : p * gate_of(p);
    // 0.5 (1 + tanh(u)) = sigmoid(2 u)
    case PHZ_ACT_GELU:
      return p == -__builtin_inff() ? 0.0f : p * gate_of(2.0f * kGeluA * p * fmaf(kGeluB * p, p, 1.0f));
    default: return p;
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
  template <int N>
  __device__ __forceinline__ void put(int, int, int i, int j, const float* sums) const {
    float p[N];
    Pack<E, N> r, out;
    if (residual) r = *(const Pack<E, N>*)(residual + i * residual_row + j);
#pragma unroll
    for (int c = 0; c < N; c++) p[c] = bias ? sums[c] + to_f32(bias[(j + c) * bias_step]) : sums[c];
    if (pre) {
#pragma unroll
      for (int c = 0; c < N; c++) out.v[c] = from_f32<E>(p[c]);
      *(Pack<E, N>*)(pre + i * pre_row + j) = out;
    }
#pragma unroll
    for (int c = 0; c < N; c++) {
      p[c] = act_of(act, p[c]);
      out.v[c] = from_f32<E>(residual ? p[c] + to_f32(r.v[c]) : p[c]);
    }
    *(Pack<E, N>*)(y + i * y_row + j) = out;
  }
};

template <class E>
struct PlainOut {
  E* y;
  int64_t row;
  template <int N>
  __device__ __forceinline__ void put(int, int, int i, int j, const float* sums) const {
    Pack<E, N> out;
#pragma unroll
    for (int c = 0; c < N; c++) out.v[c] = from_f32<E>(sums[c]);
    *(Pack<E, N>*)(y + i * row + j) = out;
  }
};

// Sums of one split of the contraction, joined by join_splits.
struct SplitOut {
  float* part;
  int64_t row, split;
  template <int N>
  __device__ __forceinline__ void put(int, int s, int i, int j, const float* sums) const {
    Pack<float, N> out;
#pragma unroll
    for (int c = 0; c < N; c++) out.v[c] = sums[c];
    *(Pack<float, N>*)(part + s * split + i * row + j) = out;
  }
};

// y[i][j] = the splits' sums, added in order.
template <class E>
__global__ __launch_bounds__(256) void join_splits(const float* part, int splits, int64_t split, E* y, int64_t row,
                                                   int32_t n, int64_t total) {
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    float v = part[t];
    for (int s = 1; s < splits; s++) v += part[s * split + t];
    const int64_t i = t / n;
    y[i * row + (t - i * n)] = from_f32<E>(v);
  }
}

constexpr int kDzRows = 64;

// dz = dy act'(pre) (where there is an activation) and the sums of dz over
// each block of kDzRows rows, which column_sums adds up in order.
template <class E>
__global__ __launch_bounds__(256) void dz_rows(int act, const E* dy, int64_t dy_row, const E* pre, int64_t pre_row,
                                               E* dz, int64_t dz_row, float* sums, int32_t m, int32_t n) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  const int i0 = blockIdx.y * kDzRows, i1 = min(m, i0 + kDzRows);
  float total = 0.0f;
#pragma unroll 8
  for (int i = i0; i < i1; i++) {
    float d = to_f32(dy[i * dy_row + j]);
    if (act != PHZ_ACT_NONE) d *= act_grad(act, to_f32(pre[i * pre_row + j]));
    total += d;
    if (dz) dz[i * dz_row + j] = from_f32<E>(d);
  }
  if (sums) sums[(int64_t)blockIdx.y * n + j] = total;
}

template <class E>
__global__ __launch_bounds__(256) void column_sums(const float* sums, int32_t blocks, int32_t n, E* db, int64_t step) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  float v = 0.0f;
  for (int i = 0; i < blocks; i++) v += sums[(int64_t)i * n + j];
  db[j * step] = from_f32<E>(v);
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

template <class E>
int linear(phz_ops* o, hipStream_t stream, int act, const phz_tensor* x, const phz_tensor* w, const phz_tensor* bias,
           const phz_tensor* residual, const phz_tensor* pre, const phz_tensor* y) {
  const int32_t m = (int32_t)x->size[0], k = (int32_t)x->size[1], n = (int32_t)w->size[0];
  LinearOut<E> out{};
  if (bias) out.bias = (const E*)bias->data, out.bias_step = bias->stride[0];
  if (residual) out.residual = (const E*)residual->data, out.residual_row = residual->stride[0];
  if (pre) out.pre = (E*)pre->data, out.pre_row = pre->stride[0];
  out.y = (E*)y->data, out.y_row = y->stride[0];
  out.act = act;
  const Operand a{x->data, x->stride[0], 0}, b{w->data, w->stride[0], 0};
  launch_gemm_any<E, true, true>(o, stream, a, b, GemmShape{m, n, k, std::max(k, 1), 1}, 1, out);
  return launched(o, "linear") ? 0 : 1;
}

template <class E>
int linear_backward(phz_ops* o, hipStream_t stream, int act, const phz_tensor* dy, const phz_tensor* x,
                    const phz_tensor* w, const phz_tensor* pre, const phz_tensor* dx, const phz_tensor* dw,
                    const phz_tensor* db) {
  const int32_t m = (int32_t)x->size[0], k = (int32_t)x->size[1], n = (int32_t)w->size[0];
  const bool products = (dx || dw) && m > 0;
  // The contraction of dw runs over rows: split where its few tiles would not
  // fill the chip.
  const int64_t tiles = ceil_div(n, 64) * ceil_div(k, 64);
  const int bk = Cut<E>::tile_k;
  int64_t splits = dw ? std::min<int64_t>(ceil_div(2 * o->cus, tiles), ceil_div(m, 4 * bk)) : 1;
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, 256));
  const int32_t k_split = (int32_t)std::max<int64_t>(bk, ceil_div(ceil_div(m, splits), bk) * bk);
  splits = std::max<int64_t>(1, ceil_div(m, k_split));
  const int64_t dz_row = (n + 7) / 8 * 8, blocks = ceil_div(m, kDzRows);
  const uint64_t dz_bytes = act != PHZ_ACT_NONE && products ? ((uint64_t)m * dz_row * sizeof(E) + 255) & ~255ull : 0;
  const uint64_t sum_bytes = db ? ((uint64_t)blocks * n * 4 + 255) & ~255ull : 0;
  const uint64_t part_bytes = dw && splits > 1 ? (uint64_t)splits * n * k * 4 : 0;
  char* ws = nullptr;
  if (dz_bytes + sum_bytes + part_bytes && !(ws = o->workspace(stream, dz_bytes + sum_bytes + part_bytes))) return 1;
  E* dz = dz_bytes ? (E*)ws : nullptr;
  float* sums = sum_bytes ? (float*)(ws + dz_bytes) : nullptr;
  float* part = (float*)(ws + dz_bytes + sum_bytes);
  if (dz || db) {
    if (blocks)
      hipLaunchKernelGGL(dz_rows<E>, dim3((unsigned)ceil_div(n, 256), (unsigned)blocks), dim3(256), 0, stream, act,
                         (const E*)dy->data, dy->stride[0], pre ? (const E*)pre->data : nullptr,
                         pre ? pre->stride[0] : 0, dz, dz_row, sums, m, n);
    if (db)
      hipLaunchKernelGGL(column_sums<E>, dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, stream, sums, (int32_t)blocks, n,
                         (E*)db->data, db->stride[0]);
  }
  const Operand d{dz ? dz : dy->data, dz ? dz_row : dy->stride[0], 0};
  if (dx && m > 0 && k > 0)
    launch_gemm_any<E, true, false>(o, stream, d, Operand{w->data, w->stride[0], 0}, GemmShape{m, k, n, std::max(n, 1), 1},
                                    1, PlainOut<E>{(E*)dx->data, dx->stride[0]});
  if (dw && n > 0 && k > 0) {
    const Operand xo{x->data, x->stride[0], 0};
    if (m == 0) {
      hipLaunchKernelGGL(fill_zero<E>, dim3(256), dim3(256), 0, stream, (E*)dw->data, dw->stride[0], k, (int64_t)n * k);
    } else if (splits == 1) {
      launch_gemm_any<E, false, false>(o, stream, d, xo, GemmShape{n, k, m, k_split, 1}, 1,
                                       PlainOut<E>{(E*)dw->data, dw->stride[0]});
    } else {
      launch_gemm_any<E, false, false>(o, stream, d, xo, GemmShape{n, k, m, k_split, (int32_t)splits}, 1,
                                       SplitOut{part, k, (int64_t)n * k});
      const int64_t total = (int64_t)n * k;
      hipLaunchKernelGGL(join_splits<E>, dim3((unsigned)std::min<int64_t>(ceil_div(total, 256), 8192)), dim3(256), 0,
                         stream, part, (int)splits, total, (E*)dw->data, dw->stride[0], k, total);
    }
  }
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
