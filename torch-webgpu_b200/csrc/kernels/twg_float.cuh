// Element access for the kernels that read and write float32, float16 or bfloat16 and compute in
// float32: 16-byte vectors of any of the three, and single elements.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "twg_launch.cuh"

namespace twg {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// The one rounding of a result: to nearest, ties to even.
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Elements of T in one 16-byte vector.
template <class T> constexpr int kVecOf = 16 / (int)sizeof(T);

// A vector of `BYTES` bytes, and its accesses (as in twg_pointwise.cuh: no line in L1, evicted first).
template <int BYTES> struct VecBytes;
template <> struct VecBytes<16> { using type = uint4; };
template <> struct VecBytes<8> { using type = uint2; };
template <> struct VecBytes<4> { using type = u32; };
__device__ __forceinline__ void ld_vec(uint4& v, const void* p) { v = ld_v4(p); }
__device__ __forceinline__ void ld_vec(uint2& v, const void* p) {
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
}
__device__ __forceinline__ void ld_vec(u32& v, const void* p) { v = ld_b32(p); }
__device__ __forceinline__ void st_vec(void* p, const uint4& v) { st_v4(p, v); }
__device__ __forceinline__ void st_vec(void* p, const uint2& v) {
  asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void st_vec(void* p, const u32& v) { st_b32(p, v); }

// The words of a vector.
__device__ __forceinline__ void words(const uint4& r, u32 (&w)[4]) { w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w; }
__device__ __forceinline__ void words(const uint2& r, u32 (&w)[2]) { w[0] = r.x; w[1] = r.y; }
__device__ __forceinline__ void words(const u32& r, u32 (&w)[1]) { w[0] = r; }
__device__ __forceinline__ void from_words(uint4& r, const u32 (&w)[4]) { r = make_uint4(w[0], w[1], w[2], w[3]); }
__device__ __forceinline__ void from_words(uint2& r, const u32 (&w)[2]) { r = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void from_words(u32& r, const u32 (&w)[1]) { r = w[0]; }

template <class VEC, int N>
__device__ __forceinline__ void unpack(const VEC& r, float (&f)[N], const float*) {
  u32 w[N];
  words(r, w);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = as_f(w[i]);
}
template <class VEC, int N>
__device__ __forceinline__ void unpack(const VEC& r, float (&f)[N], const __half*) {
  u32 w[N / 2];
  words(r, w);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    __half2 h;
    *reinterpret_cast<u32*>(&h) = w[i];
    const float2 v = __half22float2(h);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <class VEC, int N>
__device__ __forceinline__ void unpack(const VEC& r, float (&f)[N], const __nv_bfloat16*) {
  u32 w[N / 2];
  words(r, w);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    f[2 * i] = as_f(w[i] << 16);
    f[2 * i + 1] = as_f(w[i] & 0xffff0000u);
  }
}
template <int N>
__device__ __forceinline__ auto pack(const float (&f)[N], const float*) {
  typename VecBytes<4 * N>::type r;
  u32 w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = as_u(f[i]);
  from_words(r, w);
  return r;
}
template <int N>
__device__ __forceinline__ auto pack(const float (&f)[N], const __half*) {
  typename VecBytes<2 * N>::type r;
  u32 w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const u32*>(&h);
  }
  from_words(r, w);
  return r;
}
template <int N>
__device__ __forceinline__ auto pack(const float (&f)[N], const __nv_bfloat16*) {
  typename VecBytes<2 * N>::type r;
  u32 w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const u32*>(&h);
  }
  from_words(r, w);
  return r;
}

// A vector of global memory to shared memory, on its way until a wait: copy_async_wait<N> returns when
// at most the calling thread's N latest commits are still under way.
__device__ __forceinline__ void copy_async(uint4* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((u32)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
template <class VEC>
__device__ __forceinline__ void copy_async(VEC* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((u32)__cvta_generic_to_shared(to)), "l"(from), "n"(sizeof(VEC)) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two float32 values in one register pair, and arithmetic on both in one instruction.
struct Two {
  u64 v;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ void get(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
};
__device__ __forceinline__ Two add(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Host side: bytes of a floating element type this family of kernels takes, 0 for any other.
inline int float_size(int dtype) {
  return dtype == TWG_DTYPE_F32 ? 4 : (dtype == TWG_DTYPE_F16 || dtype == TWG_DTYPE_BF16) ? 2 : 0;
}

// Call `fn` with a null pointer of the element type behind `dtype` (one of the three).
template <class Fn>
int dispatch_float(int dtype, Fn&& fn) {
  if (dtype == TWG_DTYPE_F32) return fn(static_cast<float*>(nullptr));
  if (dtype == TWG_DTYPE_F16) return fn(static_cast<__half*>(nullptr));
  return fn(static_cast<__nv_bfloat16*>(nullptr));
}

}  // namespace twg
