// kv_common.cuh — pieces shared by the kernels of libdsa_kv.so (C ABI:
// include/dsa_kv.h): index arithmetic, 16-bit and 8-bit element formats.
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "dsa_kv.h"

namespace kv {

constexpr float kMinScale = 1.0e-12f;

// Division of n < 2^31 by d >= 1 with a precomputed multiplier (the round-up
// method of Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994).
struct FastDiv {
  uint32_t d, mul, shift;
  __host__ void init(uint32_t v) {
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < v) ++l;
    d = v;
    mul = (uint32_t)(((1ull << 32) * ((1ull << l) - v)) / v + 1);
    shift = l;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
  __device__ __forceinline__ void divmod(uint32_t n, uint32_t* q, uint32_t* r) const {
    *q = div(n);
    *r = n - *q * d;
  }
};

// A dense [B, Q, H, D] tensor of 2-byte elements; strides in bytes.
struct Dense {
  uint8_t* ptr;
  int64_t sb, sq, sh;
  __device__ __forceinline__ uint8_t* row(uint32_t b, uint32_t q, uint32_t h) const {
    return ptr + b * sb + q * sq + h * sh;
  }
};

// One side (keys or values) of the cache; strides in bytes (codes) and floats (scales).
struct CacheSide {
  uint8_t* codes;
  float* scale;
  int64_t sp, sh, st;
  int64_t ssp, ssh, sst;
};

// No load of these kernels is of the read-only kind (ld.global.nc): a grid that
// was launched early is already running while the one before it writes what
// it will read.
__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int bytes) {
  return bytes == 8 ? (int64_t)reinterpret_cast<const long long*>(p)[i]
                    : (int64_t)reinterpret_cast<const int*>(p)[i];
}

// Programmatic dependent launch: the grid may start while the previous kernel
// of the stream drains; it waits for it before its first global access, and
// lets the next launch begin its own set-up.
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}

// ------------------------------------------------------------- fp32 pairs
// Two fp32 values in one register pair: one instruction for both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// ------------------------------------------------------------ 16-bit formats
template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80u;
  __device__ __forceinline__ static float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Half16<__half> {
  static constexpr uint32_t kInf = 0x7c00u;
  __device__ __forceinline__ static float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float f[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Half16<T>::unpack(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float f[8]) {
  return make_uint4(Half16<T>::pack(f[0], f[1]), Half16<T>::pack(f[2], f[3]), Half16<T>::pack(f[4], f[5]),
                    Half16<T>::pack(f[6], f[7]));
}

// ------------------------------------------------------------- 8-bit formats
// Four e4m3 codes of four values, lowest byte first (nearest even, saturating at 448).
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
// Two e4m3 codes as two fp16 values (exact: e4m3 is a subset of fp16).
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
__device__ __forceinline__ uint32_t to_s8(float v) { return (uint32_t)__float2int_rn(v) & 0xffu; }
__device__ __forceinline__ uint32_t to_s8x4(float a, float b, float c, float d) {
  return to_s8(a) | (to_s8(b) << 8) | (to_s8(c) << 16) | (to_s8(d) << 24);
}
// Four codes as two pairs of fp32 values.
template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, f32x2& lo, f32x2& hi) {
  if (E4M3) {
    const uint32_t a = e4m3x2_to_half2((uint16_t)w), b = e4m3x2_to_half2((uint16_t)(w >> 16));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    lo = pair(x.x, x.y);
    hi = pair(y.x, y.y);
  } else {
    const int v = (int)w;
    lo = pair((float)(int8_t)v, (float)(int8_t)(v >> 8));
    hi = pair((float)(int8_t)(v >> 16), (float)(v >> 24));
  }
}

}  // namespace kv
