// Shared by the model kernels (attention, token log probabilities, residual
// norm): element types, 8-element vectors at any element alignment, wave
// reductions, and the guard that every C entry runs under.

#pragma once

#include <hip/hip_runtime.h>

#include "model_api.h"

namespace sofa_model {

using fp16 = _Float16;

constexpr int kWave = 64;

// Vectors of 8 elements that are aligned like one element: rows of odd length
// start anywhere, and gfx950 loads and stores 16 bytes from any address.
template <typename T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  typename Vec8<T>::type v = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float) v[j];
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  typename Vec8<T>::type v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T) x[j];
  *reinterpret_cast<typename Vec8<T>::type*>(p) = v;
}

// `n` of 8 elements are there (n may be <= 0); the others read as `fill`
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8], int n,
                                      float fill = 0.f) {
  if (n >= 8) {
    load8(p, x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? (float) p[j] : fill;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], int n) {
  if (n >= 8) {
    store8(p, x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T) x[j];
  }
}

// small vectors (weights, gates), whose type is known at run time only
__device__ __forceinline__ void load8_any(const void* p, int type, int64_t at,
                                          float (&x)[8], int n) {
  if (type == kFloat32)
    load8(static_cast<const float*>(p) + at, x, n);
  else if (type == kBFloat16)
    load8(static_cast<const bf16*>(p) + at, x, n);
  else
    load8(static_cast<const fp16*>(p) + at, x, n);
}

__device__ __forceinline__ void store_any(void* p, int type, int64_t at,
                                          float x) {
  if (type == kFloat32)
    static_cast<float*>(p)[at] = x;
  else if (type == kBFloat16)
    static_cast<bf16*>(p)[at] = (bf16) x;
  else
    static_cast<fp16*>(p)[at] = (fp16) x;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// exp and log in base 2 as single instructions (1 ulp); subnormal results of
// exp2 are flushed, which is 2^-126 next to a largest term of 1
__device__ __forceinline__ float exp2_fast(float x) {
  return __builtin_amdgcn_exp2f(x);
}
__device__ __forceinline__ float log2_fast(float x) {
  return __builtin_amdgcn_logf(x);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Makes `device` current for the launches of one C entry and puts the
// caller's device back.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    status_ = hipGetDevice(&before_);
    if (status_ == hipSuccess && before_ != device) {
      status_ = hipSetDevice(device);
      changed_ = status_ == hipSuccess;
    }
  }
  ~DeviceGuard() {
    if (changed_) (void) hipSetDevice(before_);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  int status() const { return (int) status_; }

 private:
  hipError_t status_;
  int before_ = 0;
  bool changed_ = false;
};

}  // namespace sofa_model
