// operators.h -- what the device operators (scan.cu, rotate.cu, losses.cu) share:
// storage types and the frame of a C entry point.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <exception>

#include "../../include/topos_b200.h"
#include "kernels.h"
#include "launch.h"

namespace tb {

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }

// Two f32 operations in one instruction (sm_100's packed f32x2 forms, each rounded as its scalar).
__device__ __forceinline__ unsigned long long packed(float2 v) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 unpacked(unsigned long long r) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)));
  return unpacked(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)));
  return unpacked(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)), "l"(packed(c)));
  return unpacked(r);
}
__device__ __forceinline__ float2 both(float v) { return {v, v}; }

// Two bf16 values of one word, the lower first, and back.
__device__ __forceinline__ float2 unpack_bf16(unsigned r) {
  return {__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u)};
}
__device__ __forceinline__ unsigned pack_bf16(float2 v) {
  unsigned r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
  return r;
}

// The frame of an operator's entry point: the request is checked first, then the library's
// state, then the work is enqueued on the caller's stream.
class OperatorCall {
 public:
  OperatorCall(const char* name, void* stream) : name_(name), stream_((cudaStream_t)stream) {}
  cudaStream_t stream() const { return stream_; }

  int invalid(const char* why) const {
    char text[256];
    snprintf(text, sizeof text, "%s: %s", name_, why);
    set_last_error(text);
    return TB_INVALID;
  }

  // TB_OK when work may be enqueued.
  int ready() {
    static std::atomic<bool> device_seen{false};
    if (!device_seen.load(std::memory_order_relaxed)) {
      int count = 0;
      if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
        cudaGetLastError();
        return fail(TB_PLATFORM_UNSUPPORTED, "no CUDA device");
      }
      device_seen.store(true, std::memory_order_relaxed);
    }
    if (poisoned()) return fail(TB_POISONED, "the backend is poisoned");
    cudaGetLastError();  // a launch error left by earlier, unrelated work is not this call's
    return TB_OK;
  }

  // The launches' outcome.
  int finish(cudaError_t e) const {
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e == cudaSuccess) return TB_OK;
    // refused before anything ran, and the device is well
    if (e == cudaErrorInvalidResourceHandle)
      return invalid("the stream is not one of the current device");
    if (e >= cudaErrorStreamCaptureUnsupported && e <= cudaErrorStreamCaptureWrongThread)
      return invalid("not taken by the capture of a stream");  // that is lost, or would be
    if (e == cudaErrorInvalidConfiguration) return invalid("more work than one launch takes");
    char text[256];
    snprintf(text, sizeof text, "%s: %s", name_, cudaGetErrorString(e));
    poison_library(text);
    return TB_RUNTIME;
  }

 private:
  int fail(int code, const char* why) const {
    char text[256];
    snprintf(text, sizeof text, "%s: %s", name_, why);
    set_last_error(text);
    return code;
  }
  const char* name_;
  cudaStream_t stream_;
};

// Runs an entry point's body; no C++ exception leaves the library.
template <typename F>
inline int guarded(F body) noexcept {
  try {
    return body();
  } catch (const std::exception&) {
    return TB_RUNTIME;
  } catch (...) {
    return TB_RUNTIME;
  }
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device; `allowed` remembers the
// devices where it already may.  48 KB may always be used, 16 KB of it static.
inline cudaError_t allow_shared(const void* kernel, size_t bytes, std::atomic<uint64_t>& allowed) {
  if (bytes <= 32 * 1024) return cudaSuccess;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device)) return e;
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (device < 64 && (allowed.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && device < 64) allowed.fetch_or(bit, std::memory_order_release);
  return e;
}

inline bool aligned_to(const void* p, int64_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
// Extents a request may have: each, and their product, far below what 64-bit sizes hold.
inline bool extents_fit(std::initializer_list<int64_t> extents) {
  double product = 1;
  for (int64_t e : extents) {
    if (e < 0 || e > (int64_t(1) << 40)) return false;
    product *= e > 0 ? (double)e : 1.0;
  }
  return product < (double)(int64_t(1) << 44);
}

// Whether rows of `inner` elements, counted along each axis and set `strides` apart, keep clear of
// one another: along the axes by rising stride, each step passes all that the ones before reach.
template <int N>
inline bool rows_apart(int64_t inner, const int64_t (&counts)[N], const int64_t (&strides)[N]) {
  int64_t count[N], stride[N];
  int axes = 0;
  for (int i = 0; i < N; ++i) {
    if (counts[i] == 0) return true;
    if (counts[i] == 1) continue;
    int at = axes++;
    for (; at > 0 && stride[at - 1] > strides[i]; --at) {
      stride[at] = stride[at - 1];
      count[at] = count[at - 1];
    }
    stride[at] = strides[i];
    count[at] = counts[i];
  }
  double reach = (double)inner;  // sizes may pass 64 bits in a malformed request
  for (int i = 0; i < axes; ++i) {
    if ((double)stride[i] < reach) return false;
    reach += (double)stride[i] * (double)(count[i] - 1);
  }
  return true;
}

}  // namespace tb
