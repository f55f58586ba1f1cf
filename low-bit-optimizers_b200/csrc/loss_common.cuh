// Device helpers shared by the training-loss kernels (distill.cu, balance.cu): loads of 16 bytes as fp32 values for
// the three element types, stores with one rounding to nearest even, the hardware exponential, index loads.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace lpmm_b200 {

template <typename T>
struct Elem;  // VE elements are 16 bytes
template <>
struct Elem<float> {
  static constexpr int VE = 4;
  static __device__ __forceinline__ float widen(float v) { return v; }
  static __device__ __forceinline__ float narrow(float v) { return v; }
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int VE = 8;
  static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void two(uint32_t w, float* x) {  // a bf16 is the upper half of its fp32 value
    x[0] = __uint_as_float(w << 16), x[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t join(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    two(r.x, x), two(r.y, x + 2), two(r.z, x + 4), two(r.w, x + 6);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(join(x[0], x[1]), join(x[2], x[3]), join(x[4], x[5]), join(x[6], x[7]));
  }
};
template <>
struct Elem<__half> {
  static constexpr int VE = 8;
  static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void two(uint32_t w, float* x) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x[0] = f.x, x[1] = f.y;
  }
  static __device__ __forceinline__ uint32_t join(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    two(r.x, x), two(r.y, x + 2), two(r.z, x + 4), two(r.w, x + 6);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(join(x[0], x[1]), join(x[2], x[3]), join(x[4], x[5]), join(x[6], x[7]));
  }
};

// 2^x by the hardware instruction (about 2^-22 relative; results below 2^-126 are 0, which no sum of terms of which
// one is 1, and no gradient, can tell from the denormal value)
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float load_any(const void* p, long long i, int dtype) {
  if (dtype == LPMM_B200_DTYPE_FP32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == LPMM_B200_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ long long load_index(const void* p, long long i, int bits) {
  return bits == 64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fc00000); }

}  // namespace lpmm_b200
