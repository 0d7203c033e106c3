// tg_attn.h — what the attention operators on device tensors share
// (tg_attn_prompt.cu, tg_attn_shared.cu, tg_kv_evict.cu): element types,
// argument checks of their C entries, conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "tg_runtime.h"

namespace tg {

enum { ATTN_BF16 = 0, ATTN_FP16 = 1 };
constexpr int ATTN_MAX_HD = 128;   // head_dim limit of the operators, a multiple of 8
constexpr float LOG2E = 1.4426950408889634f;

// The softmax weights that meet the values are 2^(c s - m + OFF), m a running
// reference that a score exceeds by LIFT at most, in 16 bits.  bf16 has fp32's
// range.  fp16 ends at 2^16 and loses bits below 2^-14, so its weights use the
// range up to 2^15: those above 2^-24 of the reference's keep all 11 bits, and
// smaller ones are off by 2^-35 of it at most (2^-25 without OFF: thousands
// of keys of 2^-24.5, all of an output beside keys without a value, counted 1.4
// times).  Sums have the same factor, which cancels.  The smaller LIFT, the more
// often an accumulator is scaled: 8 x 1,024 tokens 103 us with OFF 10 and LIFT 5,
// 107 with 11 and 4, 101 with 0 and 8; 8,192 tokens 446, 468, 438.
template <typename T>
struct AttnRange {
  static constexpr float OFF = 0.f, LIFT = 8.f;
};
template <>
struct AttnRange<__half> {
  static constexpr float OFF = 10.f, LIFT = 5.f;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

// The checks of one C entry: the first failure records an error (code 3, bad
// arguments; 2, no device) under the entry's name and sticks.
struct ArgCheck {
  const char* what;
  int dev = -1;
  int rc = 0;
  bool known;   // pointers are known to be null or device memory of the current device
  explicit ArgCheck(const char* w, bool k = false) : what(w), known(k) {}
  // A condition on the arguments; the text says what is wanted.
  bool need(bool ok, const char* text) {
    if (!ok && !rc) {
      set_host_error(3, "%s: %s", what, text);
      rc = 3;
    }
    return rc == 0;
  }
  bool device() {
    if (rc) return false;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
      set_host_error(2, "%s: no usable CUDA device (%s)", what, cudaGetErrorString(e));
      rc = 2;
    }
    return rc == 0;
  }
  // Device memory of the current device, aligned to `align` bytes.
  bool ptr(const void* p, unsigned align, const char* name) {
    if (rc) return false;
    cudaPointerAttributes a{};
    const bool ok = p && (known || (cudaPointerGetAttributes(&a, p) == cudaSuccess &&
                                    (a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged) && a.device == dev));
    if (!ok) {
      cudaGetLastError();
      set_host_error(3, "%s: %s must be device memory on the current device %d", what, name, dev);
      rc = 3;
    } else if ((uintptr_t)p % align) {
      set_host_error(3, "%s: %s must be %u-byte aligned", what, name, align);
      rc = 3;
    }
    return rc == 0;
  }
  // The stride, in elements, of a 16-bit tensor's dimension of n values: a
  // positive multiple of 8 (16 bytes).  One that no index uses may be anything.
  long long stride(int64_t s, long long n) {
    if (n <= 1) return 8;
    need(s > 0 && s % 8 == 0 && s < (1ll << 38), "strides must be positive multiples of 8 elements");
    return s;
  }
  // The result of the launches.
  int done(cudaError_t e) {
    if (!rc && e != cudaSuccess) {
      rc = 100 + (int)e;
      set_host_error(rc, "%s: launch failed: %s", what, cudaGetErrorString(e));
    }
    return rc;
  }
};

}  // namespace tg
