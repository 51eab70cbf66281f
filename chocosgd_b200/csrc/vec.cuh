// Runs of 1 - 8 consecutive elements of fp32 / bf16 / fp16 tensors, read and written with one access and
// held as fp32 in between (each value is rounded once, when it is stored).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

// element types of the C entry points
#define DT_F32 0
#define DT_BF16 1
#define DT_F16 2

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { typedef uint4 type; };
template <> struct RawVec<8> { typedef uint2 type; };
template <> struct RawVec<4> { typedef uint32_t type; };
template <> struct RawVec<2> { typedef uint16_t type; };

// hides a value's origin from the compiler, which else keeps conversions of it alive instead of doing them again
__device__ __forceinline__ void opaque(uint4& v) { asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)); }
__device__ __forceinline__ void opaque(uint2& v) { asm volatile("" : "+r"(v.x), "+r"(v.y)); }
__device__ __forceinline__ void opaque(uint32_t& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void opaque(uint16_t& v) { asm volatile("" : "+h"(v)); }

// V elements of T as they lie in memory
template <typename T, int V> struct Vec {
  typedef typename RawVec<sizeof(T) * V>::type Raw;
  union { Raw raw; T e[V]; };
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void clear() { raw = Raw(); }
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// one element of a tensor whose type is only known at run time
__device__ __forceinline__ float load_any(const void* p, int dt, long long i) {
  if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (dt == DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dt, long long i, float v) {
  if (dt == DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == DT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// ---- pairs of fp32 numbers: one instruction works on both ------------------------------------------------------------
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float2 f2_get(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float f2_sum(F2 a) {
  const float2 p = f2_get(a);
  return p.x + p.y;
}
// elements 2 i and 2 i + 1 of a vector
__device__ __forceinline__ F2 pair_of(const Vec<float, 4>& v, int i) { return f2(v.e[2 * i], v.e[2 * i + 1]); }
__device__ __forceinline__ F2 pair_of(const Vec<__nv_bfloat16, 8>& v, int i) {
  const uint32_t w = i == 0 ? v.raw.x : (i == 1 ? v.raw.y : (i == 2 ? v.raw.z : v.raw.w));
  return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ F2 pair_of(const Vec<__half, 8>& v, int i) {
  const uint32_t w = i == 0 ? v.raw.x : (i == 1 ? v.raw.y : (i == 2 ? v.raw.z : v.raw.w));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2(f.x, f.y);
}
// a vector of pairs, each rounded once (no address of a register is taken: it would end in local memory)
__device__ __forceinline__ uint32_t pack_bf16x2(F2 a) {
  const float2 f = f2_get(a);
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_f16x2(F2 a) {
  const float2 f = f2_get(a);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_pairs(float* p, const F2 (&a)[2]) {
  const float2 x = f2_get(a[0]), y = f2_get(a[1]);
  *reinterpret_cast<float4*>(p) = make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ void store_pairs(__nv_bfloat16* p, const F2 (&a)[4]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(a[0]), pack_bf16x2(a[1]), pack_bf16x2(a[2]), pack_bf16x2(a[3]));
}
__device__ __forceinline__ void store_pairs(__half* p, const F2 (&a)[4]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_f16x2(a[0]), pack_f16x2(a[1]), pack_f16x2(a[2]), pack_f16x2(a[3]));
}

static inline int dt_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }
