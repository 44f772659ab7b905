// phz_ops.h — what the operators of sequence policies share: the handle, its
// workspaces, the checks of tensor arguments, and element conversions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <exception>
#include <string>
#include <vector>

#include "../../include/phyz_amd.h"

struct phz_ops {
  int device = -1;
  int cus = 256;
  std::string err;
  // Zeros that out-of-range lanes of direct-to-LDS loads read.
  const void* zeros = nullptr;
  // One for a stream's own calls, and for each capture on it that needed one.
  struct Block { void* stream; void* data; uint64_t bytes; bool graph; unsigned long long capture; };
  std::vector<Block> blocks;

  int fail(const std::string& m) {
    err = m;
    return 1;
  }
  bool hip_ok(hipError_t e, const char* what) {
    if (e == hipSuccess) return true;
    err = std::string(what) + ": " + hipGetErrorString(e);
    return false;
  }
  // The stream's workspace, at least `bytes` long (256-byte aligned), or NULL
  // with the error set.
  char* workspace(hipStream_t stream, uint64_t bytes);
};

namespace phzop {

inline std::string fmt(const char* f, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, f);
  vsnprintf(buf, sizeof buf, f, ap);
  va_end(ap);
  return buf;
}

// The calling thread's current device is the handle's while a call runs.
struct DeviceGuard {
  int before = -1;
  bool ok = true;
  explicit DeviceGuard(phz_ops* o) {
    int now = -1;
    ok = o->hip_ok(hipGetDevice(&now), "hipGetDevice");
    if (ok && now != o->device) {
      ok = o->hip_ok(hipSetDevice(o->device), "hipSetDevice");
      before = now;
    }
  }
  ~DeviceGuard() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// Runs a call's body; nothing thrown inside leaves the C interface.
template <class F>
int guarded(phz_ops* o, F&& body) {
  if (!o) return 1;
  try {
    o->err.clear();
    return body();
  } catch (const std::exception& e) {
    try {
      o->err = e.what();
    } catch (...) {
    }
    return 1;
  } catch (...) {
    return 1;
  }
}

inline const char* dtype_name(int d) {
  return d == PHZ_F32    ? "f32"
         : d == PHZ_BF16 ? "bf16"
         : d == PHZ_U8   ? "u8"
         : d == PHZ_F64  ? "f64"
         : d == PHZ_I32  ? "i32"
         : d == PHZ_I64  ? "i64"
                         : "unknown";
}
inline int64_t elem_bytes(int d) {
  return d == PHZ_F64 || d == PHZ_I64 ? 8 : d == PHZ_F32 || d == PHZ_I32 ? 4 : d == PHZ_BF16 ? 2 : 1;
}

// Shape, type and layout of one argument. `size`: what each axis has to be,
// -1 for any. The last axis has to be dense where `dense` is set; strides may
// not be negative, and an output's axes of more than one element not broadcast.
struct Want {
  int ndim;
  int64_t size[3];
  int dtype;
  bool dense;
  bool output;
};
bool check(phz_ops* o, const char* name, const phz_tensor* t, const Want& want);
// False, with the error set, where output `a` shares an element with `b`.
bool apart(phz_ops* o, const char* an, const phz_tensor* a, const char* bn, const phz_tensor* b);
inline bool empty(const phz_tensor* t) {
  for (int i = 0; i < t->ndim; i++)
    if (t->size[i] == 0) return true;
  return false;
}
inline bool launched(phz_ops* o, const char* what) { return o->hip_ok(hipGetLastError(), what); }
__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ── device side ─────────────────────────────────────────────────────────────

struct bf16 { uint16_t bits; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __builtin_bit_cast(float, (uint32_t)v.bits << 16); }
// To nearest, ties to even; NaN stays NaN (one v_cvt on gfx950).
template <class E> __device__ __forceinline__ E from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) {
  return bf16{__builtin_bit_cast(uint16_t, (__bf16)v)};
}

// N elements whose address is aligned to one element only: gfx950 loads and
// stores global memory at any alignment, so odd strides keep wide accesses.
template <class E, int N>
struct __attribute__((packed, aligned(sizeof(E)))) Pack {
  E v[N];
};

// sigmoid(z) as (the smaller of it and its complement), with z's sign: both
// gates then have a relative error of at most (1.25 |z| + 8) 2^-24, which
// 1 - sigmoid(z) has not where the gate saturates. The part that grows is the
// exponential's argument, |z| log2(e) rounded to f32 (and the constant's own
// rounding); that is up to 16 units of f32's last place at |z| = 20, where the gate is
// 2e-9, and taking the argument in two parts would cost two instructions more.
__device__ __forceinline__ float signed_gate(float z) {
  const float t = __expf(-fabsf(z));
  return copysignf(t * __builtin_amdgcn_rcpf(1.0f + t), z);
}

}  // namespace phzop
