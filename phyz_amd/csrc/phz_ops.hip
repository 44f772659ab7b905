// phz_ops.hip — the handle of the sequence operators: create and destroy, the
// per-stream workspaces, and the checks that every operator makes of its
// tensors before it launches anything.
#include "phz_ops.h"

#include <string.h>

#include <algorithm>
#include <map>
#include <mutex>

using namespace phzop;

namespace {

thread_local std::string g_ops_create_error;

// 256 zero bytes on a device, which captured graphs read too: one for all handles,
// never freed.
const void* zeros_of(phz_ops* o) {
  static std::mutex lock;
  static std::map<int, void*> made;
  std::lock_guard<std::mutex> hold(lock);
  void*& z = made[o->device];
  if (!z) {
    void* p = nullptr;
    if (!o->hip_ok(hipMalloc(&p, 256), "zeros")) return nullptr;
    if (!o->hip_ok(hipMemset(p, 0, 256), "zeros") || !o->hip_ok(hipDeviceSynchronize(), "create")) {
      (void)hipFree(p);
      return nullptr;
    }
    z = p;
  }
  return z;
}

}  // namespace

// A stream's own calls and each capture on it work in blocks of their own, since
// a graph may be replayed on any stream, beside another one's replay and beside
// the stream's own calls. A capture takes the block that the stream's calls have
// grown (they get another when they next need one), or, where an earlier capture
// has taken that, allocates its like.
char* phz_ops::workspace(hipStream_t stream, uint64_t bytes) {
  bytes = std::max<uint64_t>((bytes + 255) & ~255ull, 256);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long capture = 0;
  if (!hip_ok(hipStreamIsCapturing(stream, &status), "hipStreamIsCapturing")) return nullptr;
  const bool capturing = status != hipStreamCaptureStatusNone;
  if (capturing && !hip_ok(hipStreamGetCaptureInfo(stream, &status, &capture), "hipStreamGetCaptureInfo")) return nullptr;
  Block *own = nullptr, *eager = nullptr;
  uint64_t known = 0;  // the most that the stream's calls or captures have had
  for (auto& x : blocks)
    if (x.stream == (void*)stream) {
      known = std::max(known, x.bytes);
      if (!x.graph) eager = &x;
      if (x.graph == capturing && x.capture == capture && (!own || own->bytes < x.bytes)) own = &x;
    }
  if (own && own->bytes >= bytes) return (char*)own->data;
  if (capturing) {
    if (eager && eager->bytes >= bytes) {
      eager->graph = true;
      eager->capture = capture;
      return (char*)eager->data;
    }
    if (known < bytes) {
      err = fmt("the stream is being captured and its workspace would have to grow to %llu bytes: run the call once "
                "before, or phz_ops_reserve",
                (unsigned long long)bytes);
      return nullptr;
    }
    // An allocation is no part of the capture; this mode lets it pass.
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    if (!hip_ok(hipThreadExchangeStreamCaptureMode(&mode), "hipThreadExchangeStreamCaptureMode")) return nullptr;
    void* p = nullptr;
    const bool ok = hip_ok(hipMalloc(&p, known), "workspace");
    (void)hipThreadExchangeStreamCaptureMode(&mode);
    if (!ok) {
      (void)hipGetLastError();
      return nullptr;
    }
    blocks.push_back(Block{(void*)stream, p, known, true, capture});
    return (char*)p;
  }
  // Half as much again as asked, so that growing sizes do not allocate on
  // every call.
  uint64_t want = std::max(bytes + bytes / 2, known);
  void* p = nullptr;
  if (hipMalloc(&p, want) != hipSuccess) {
    (void)hipGetLastError();
    want = bytes;
    if (!hip_ok(hipMalloc(&p, want), "workspace")) {
      (void)hipGetLastError();
      return nullptr;
    }
  }
  if (own) {
    (void)hipFree(own->data);  // waits for the device, so work in flight has ended
    own->data = p;
    own->bytes = want;
  } else {
    blocks.push_back(Block{(void*)stream, p, want, false, 0});
  }
  return (char*)p;
}

namespace phzop {

bool check(phz_ops* o, const char* name, const phz_tensor* t, const Want& want) {
  if (!t) return o->err = fmt("%s is missing", name), false;
  if (t->ndim != want.ndim) return o->err = fmt("%s has %d dimensions, expected %d", name, t->ndim, want.ndim), false;
  if (t->dtype != want.dtype)
    return o->err = fmt("%s is %s, expected %s", name, dtype_name(t->dtype), dtype_name(want.dtype)), false;
  for (int i = 0; i < want.ndim; i++) {
    if (t->size[i] < 0) return o->err = fmt("%s has a negative size", name), false;
    if (want.size[i] >= 0 && t->size[i] != want.size[i])
      return o->err = fmt("%s has %lld elements along axis %d, expected %lld", name, (long long)t->size[i], i,
                          (long long)want.size[i]),
             false;
  }
  if (empty(t)) return true;
  if (!t->data) return o->err = fmt("%s has no data", name), false;
  int64_t extent = 1;
  for (int i = 0; i < want.ndim; i++) {
    if (t->stride[i] < 0 || t->stride[i] > (1ll << 48) || t->size[i] > (1ll << 40))
      return o->err = fmt("%s has a negative or absurd stride or size along axis %d", name, i), false;
    if (want.output && t->size[i] > 1 && t->stride[i] == 0)
      return o->err = fmt("%s is broadcast along axis %d: an output's elements have to be its own", name, i), false;
    if (t->size[i] > 1 && __builtin_add_overflow(extent, (t->size[i] - 1) * (__int128)t->stride[i] > (1ll << 56)
                                                             ? (1ll << 62)
                                                             : (t->size[i] - 1) * t->stride[i],
                                                 &extent))
      return o->err = fmt("%s is too large", name), false;
  }
  if (extent > (1ll << 56)) return o->err = fmt("%s is too large", name), false;
  if (want.output) {
    // Axes from the smallest stride up: each has to step over all of those below.
    int axis[3], n = 0;
    for (int i = 0; i < want.ndim; i++)
      if (t->size[i] > 1) axis[n++] = i;
    std::sort(axis, axis + n, [&](int a, int b) { return t->stride[a] < t->stride[b]; });
    int64_t below = 1;
    for (int k = 0; k < n; k++) {
      if (t->stride[axis[k]] < below) return o->err = fmt("%s overlaps itself along axis %d", name, axis[k]), false;
      below += (t->size[axis[k]] - 1) * t->stride[axis[k]];
    }
  }
  if (want.dense && t->size[want.ndim - 1] > 1 && t->stride[want.ndim - 1] != 1)
    return o->err = fmt("%s: the last axis has to be dense (stride %lld)", name, (long long)t->stride[want.ndim - 1]),
           false;
  if ((uintptr_t)t->data % (uintptr_t)elem_bytes(t->dtype))
    return o->err = fmt("%s is not aligned to its elements", name), false;
  return true;
}

namespace {

void span(const phz_tensor* t, uintptr_t* lo, uintptr_t* hi) {
  int64_t n = 1;
  for (int i = 0; i < t->ndim; i++) n += (t->size[i] - 1) * t->stride[i];
  *lo = (uintptr_t)t->data;
  *hi = *lo + (uintptr_t)(n * elem_bytes(t->dtype));
}

}  // namespace

bool apart(phz_ops* o, const char* an, const phz_tensor* a, const char* bn, const phz_tensor* b) {
  if (!a || !b || empty(a) || empty(b)) return true;
  uintptr_t al, ah, bl, bh;
  span(a, &al, &ah);
  span(b, &bl, &bh);
  if (ah <= bl || bh <= al) return true;
  // Interleaved views (halves of a buffer's rows, a record's first step beside its
  // others): modulo a stride of either, axes whose strides are its multiples
  // vanish, and the rest of each view is within one stretch of residues. Where
  // those do not meet, no element does.
  const int64_t ea = elem_bytes(a->dtype), eb = elem_bytes(b->dtype);
  auto stretch = [](const phz_tensor* t, int64_t e, int64_t mod) {
    int64_t n = e;
    for (int i = 0; i < t->ndim; i++)
      if (t->size[i] > 1 && t->stride[i] * e % mod) n += (t->size[i] - 1) * t->stride[i] * e;
    return n;
  };
  for (int k = 0; k < a->ndim + b->ndim; k++) {
    const phz_tensor* t = k < a->ndim ? a : b;
    const int i = k < a->ndim ? k : k - a->ndim;
    const int64_t mod = t->size[i] > 1 ? t->stride[i] * (t == a ? ea : eb) : 0;
    if (mod <= 0) continue;
    const int64_t off = (((int64_t)(bl - al) % mod) + mod) % mod;
    if (off >= stretch(a, ea, mod) && mod - off >= stretch(b, eb, mod)) return true;
  }
  o->err = fmt("%s overlaps %s", an, bn);
  return false;
}

}  // namespace phzop

extern "C" {

int phz_ops_create(int device_ordinal, phz_ops** out) {
  try {
    g_ops_create_error.clear();
    if (!out) return g_ops_create_error = "null output pointer", 1;
    *out = nullptr;
    if (device_ordinal == -1) {
      *out = new phz_ops();
      return 0;
    }
    int count = 0;
    if (hipGetDeviceCount(&count) != hipSuccess || count == 0) return g_ops_create_error = "no HIP device available", 1;
    if (device_ordinal < 0 || device_ordinal >= count)
      return g_ops_create_error = fmt("device ordinal %d out of range (%d devices)", device_ordinal, count), 1;
    auto* o = new phz_ops();
    o->device = device_ordinal;
    DeviceGuard g(o);
    int cus = 0;
    bool ok = g.ok && o->hip_ok(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device_ordinal),
                                "compute units");
    ok = ok && (o->zeros = zeros_of(o));
    if (!ok) {
      g_ops_create_error = o->err;
      delete o;
      return 1;
    }
    o->cus = cus;
    *out = o;
    return 0;
  } catch (const std::exception& e) {
    g_ops_create_error = e.what();
    return 1;
  }
}

void phz_ops_destroy(phz_ops* o) {
  if (!o) return;
  if (o->device >= 0) {
    DeviceGuard g(o);
    for (auto& b : o->blocks) (void)hipFree(b.data);
  }
  delete o;
}

const char* phz_ops_last_error(const phz_ops* o) { return o ? o->err.c_str() : g_ops_create_error.c_str(); }

int phz_ops_reserve(phz_ops* o, void* stream, uint64_t bytes) {
  return guarded(o, [&] {
    if (o->device < 0) return o->fail("host-only handle (device -1)");
    DeviceGuard g(o);
    return g.ok && o->workspace((hipStream_t)stream, bytes) ? 0 : 1;
  });
}

uint64_t phz_ops_workspace_bytes(const phz_ops* o) {
  uint64_t n = 0;
  if (o) {
    for (auto& b : o->blocks) n += b.bytes;
  }
  return n;
}

uint64_t phz_ops_graph_bytes(const phz_ops* o) {
  uint64_t n = 0;
  if (o)
    for (auto& b : o->blocks) n += b.graph ? b.bytes : 0;
  return n;
}

}  // extern "C"
