// qserve_host.h - what the serving operators' entry points (qserve.h) share: refusals,
// the device of a call, and launches on the caller's stream.
#ifndef QSERVE_HOST_H
#define QSERVE_HOST_H

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <cstdio>

#include "qserve.h"

namespace qs {

inline int refuse(const char *fn, const char *why) {
  fprintf(stderr, "Error: %s: %s\n", fn, why);
  return 1;
}

inline bool misaligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

// The device that holds `p` is the current one while this lives.  `why` is set when `p`
// is no device memory or the stream belongs to another device.
class OnDevice {
 public:
  OnDevice(const void *p, hipStream_t stream) {
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess || (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged)) {
      (void)hipGetLastError();
      why = "no GPU, or an argument that is not device memory";
      return;
    }
    int cur = 0, sdev = a.device;
    if (stream && hipStreamGetDevice(stream, &sdev) != hipSuccess) {
      (void)hipGetLastError();
      why = "not a stream";
      return;
    }
    if (sdev != a.device) { why = "the stream is on another device than the buffers"; return; }
    if (hipGetDevice(&cur) == hipSuccess && cur != a.device) {
      if (hipSetDevice(a.device) != hipSuccess) { (void)hipGetLastError(); why = "hipSetDevice failed"; return; }
      back_ = cur;
    }
  }
  ~OnDevice() {
    if (back_ >= 0) (void)hipSetDevice(back_);
  }
  OnDevice(const OnDevice &) = delete;
  OnDevice &operator=(const OnDevice &) = delete;
  const char *why = nullptr;

 private:
  int back_ = -1;
};

// Why a cache view cannot be served, or NULL.
inline const char *bad_cache(const QPagedKV *c) {
  if (!c || !c->k || !c->v) return "null cache";
  if (c->type < QLLAMA_KV_F32 || c->type > QLLAMA_KV_I8) return "unknown cache type";
  if (c->n_pages < 1 || c->page_size < 1 || (int64_t)c->n_pages * c->page_size > INT_MAX) return "bad number or size of pages";
  if (c->n_kv < 1 || c->n_kv > 65535) return "bad number of KV heads";
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8) return "head_dim must be a multiple of 8, at most 256";
  if (c->slot_stride < c->head_dim || c->head_stride < c->head_dim || c->page_stride < c->head_dim ||
      (c->slot_stride | c->head_stride | c->page_stride) % 8 || c->slot_stride > (1 << 24))
    return "strides must be multiples of 8, at least head_dim (slots: at most 2^24)";
  if (misaligned(c->k, 16) || misaligned(c->v, 16)) return "k and v must be 16-byte aligned";
  if (c->type == QLLAMA_KV_I8) {
    if (!c->k_scale || !c->v_scale || misaligned(c->k_scale, 4) || misaligned(c->v_scale, 4)) return "an int8 cache needs scales";
    if (c->scale_slot_stride < 1 || c->scale_head_stride < 1 || c->scale_page_stride < 1 || c->scale_slot_stride > (1 << 24))
      return "bad strides of the scales";
  }
  return nullptr;
}

template <typename P>
struct Same { using type = P; };         // a kernel's parameters follow from the kernel alone
template <typename... P>
inline hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t shmem, hipStream_t stream, typename Same<P>::type... args) {
  void *at[] = {&args...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, at, shmem, stream);
  if (e != hipSuccess) (void)hipGetLastError();      // told by the call's own return
  return e;
}

}  // namespace qs

// Launch on the caller's stream; on an error the enclosing entry point refuses.  The
// launch's own result counts: the thread's last error may be that of an earlier call of
// the caller's, and is left for the caller to find.
#define QS_LAUNCH(fn, kernel, grid, block, shmem, stream, ...)                       \
  do {                                                                               \
    const hipError_t qs_e_ = qs::launch(kernel, grid, block, shmem, stream, __VA_ARGS__); \
    if (qs_e_ != hipSuccess) return qs::refuse(fn, hipGetErrorString(qs_e_));        \
  } while (0)

#endif
