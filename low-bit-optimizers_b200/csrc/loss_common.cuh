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
  static __device__ __forceinline__ uint32_t raw(const float* p) { return *reinterpret_cast<const uint32_t*>(p); }
  static __device__ __forceinline__ float of_raw(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ float type_of(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  template <int N>
  static __device__ __forceinline__ float maximum(const uint4* u) {  // NaN is passed over, here and below
    float m = __uint_as_float(u[0].x);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      m = fmaxf(m, fmaxf(__uint_as_float(u[j].x), __uint_as_float(u[j].y)));
      m = fmaxf(m, fmaxf(__uint_as_float(u[j].z), __uint_as_float(u[j].w)));
    }
    return m;
  }
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
  static __device__ __forceinline__ uint32_t raw(const __nv_bfloat16* p) { return *reinterpret_cast<const unsigned short*>(p); }
  static __device__ __forceinline__ float of_raw(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ __nv_bfloat16 type_of(uint32_t w) { return __ushort_as_bfloat16((unsigned short)w); }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  template <int N>
  static __device__ __forceinline__ float maximum(const uint4* u) {
    __nv_bfloat162 m = as2(u[0].x);
#pragma unroll
    for (int j = 0; j < N; ++j)
      m = __hmax2(m, __hmax2(__hmax2(as2(u[j].x), as2(u[j].y)), __hmax2(as2(u[j].z), as2(u[j].w))));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ __nv_bfloat162 as2(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
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
  static __device__ __forceinline__ uint32_t raw(const __half* p) { return *reinterpret_cast<const unsigned short*>(p); }
  static __device__ __forceinline__ float of_raw(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)w)); }
  static __device__ __forceinline__ __half type_of(uint32_t w) { return __ushort_as_half((unsigned short)w); }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  template <int N>
  static __device__ __forceinline__ float maximum(const uint4* u) {
    __half2 m = as2(u[0].x);
#pragma unroll
    for (int j = 0; j < N; ++j)
      m = __hmax2(m, __hmax2(__hmax2(as2(u[j].x), as2(u[j].y)), __hmax2(as2(u[j].z), as2(u[j].w))));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ __half2 as2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
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

// first element of a row; rows and inner < 2^31, so the division is one of 32 bits
__device__ __forceinline__ long long row_at(long long row, long long inner, long long outer_stride, long long inner_stride) {
  if (inner == 1) return row * outer_stride;
  const unsigned o = (unsigned)row / (unsigned)inner;
  return o * outer_stride + ((unsigned)row - o * (unsigned)inner) * inner_stride;
}
// ---------------------------------------------------------------------------------------------
// barriers in shared memory and bulk copies into it
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* b, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(unsigned long long* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(b)) : "memory");
}
__device__ __forceinline__ void mbar_expect(unsigned long long* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(b)), "r"(bytes) : "memory");
}
// A wait is a matter of microseconds.  One try sleeps for up to WAIT_NS, the limit is some seconds of tries.
constexpr uint32_t WAIT_NS = 20000;
constexpr int WAIT_LIMIT = 1 << 18;
__device__ __forceinline__ bool mbar_test(unsigned long long* b, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_at(b)), "r"(parity), "r"(WAIT_NS)
      : "memory");
  return done;
}
__device__ __forceinline__ bool mbar_test_cluster(unsigned long long* b, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_at(b)), "r"(parity), "r"(WAIT_NS)
      : "memory");
  return done;
}
// Waits for the phase; gives up (false) when the limit is reached or another thread of the CTA has given up (*failed).  The
// caller goes on in either case (its data are then worthless, its accesses in range) but starts no more copies, waits for those
// under way, and the kernel ends as it should.
__device__ __forceinline__ bool mbar_wait(unsigned long long* b, uint32_t parity, int* failed) {
  if (mbar_test(b, parity)) return true;
  for (int i = 0; i < WAIT_LIMIT; ++i) {
    if (mbar_test(b, parity)) return true;
    if (*(volatile int*)failed) return false;
  }
  *(volatile int*)failed = 1;
  return false;
}
// the same for data that other CTAs of the cluster send
__device__ __forceinline__ void mbar_wait_cluster(unsigned long long* b, uint32_t parity, int* failed) {
  for (int i = 0; i < WAIT_LIMIT; ++i) {
    if (mbar_test_cluster(b, parity) || *(volatile int*)failed) return;
  }
  *(volatile int*)failed = 1;
}
// 8 bytes to the address `to`, counted by the barrier `b`, of CTA `rank` of the cluster
__device__ __forceinline__ void send_async(void* to, float2 v, unsigned long long* b, int rank) {
  asm volatile(
      "{\n .reg .b32 t, r;\n mapa.shared::cluster.u32 t, %0, %4;\n mapa.shared::cluster.u32 r, %3, %4;\n"
      " st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [t], {%1, %2}, [r];\n}" ::"r"(smem_at(to)),
      "f"(v.x), "f"(v.y), "r"(smem_at(b)), "r"(rank)
      : "memory");
}
__device__ __forceinline__ void mbar_wait_landed(unsigned long long* b, uint32_t parity) {
  for (int i = 0; i < WAIT_LIMIT; ++i)
    if (mbar_test(b, parity)) return;
}
// between a thread's own accesses to shared memory and a bulk copy over it that follows a barrier
__device__ __forceinline__ void bulk_load_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(void* to, const void* from, uint32_t bytes, unsigned long long* b) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_at(to)),
               "l"(from), "r"(bytes), "r"(smem_at(b))
               : "memory");
}

// A kernel launched with launch_after(): waits until the kernel before it has finished and its results can be read.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// lets a kernel launched with launch_after() start (it still waits for this one's end in pdl_wait)
__device__ __forceinline__ void pdl_start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fc00000); }

}  // namespace lpmm_b200
