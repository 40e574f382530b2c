// Element types of the memory-bound training kernels: 16 bytes of bf16, fp16 or fp32 to and from fp32 registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200train {

// Two fp32 values in one 64-bit register pair: sm_100 adds, multiplies and multiply-adds both in one instruction.
using F2 = unsigned long long;
__device__ __forceinline__ F2 make2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split2(F2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Elem<T>: N elements fill 16 bytes; unpack / pack convert a whole 16-byte word, load1 / store1 a single element.
template <typename T>
struct Elem;

template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack2(uint32_t w, float* f) {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};

template <>
struct Elem<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack2(uint32_t w, float* f) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    f[0] = v.x;
    f[1] = v.y;
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }
};

template <>
struct Elem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float load1(const float* p) { return *p; }
  static __device__ __forceinline__ void store1(float* p, float v) { *p = v; }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  if constexpr (Elem<T>::N == 8) {
    Elem<T>::unpack2(v.x, f);
    Elem<T>::unpack2(v.y, f + 2);
    Elem<T>::unpack2(v.z, f + 4);
    Elem<T>::unpack2(v.w, f + 6);
  } else {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float* f) {
  if constexpr (Elem<T>::N == 8) {
    return make_uint4(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]), Elem<T>::pack2(f[4], f[5]), Elem<T>::pack2(f[6], f[7]));
  } else {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
}

// The same with the elements in pairs: N / 2 of them fill 16 bytes.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, F2* f) {
  float e[Elem<T>::N];
  unpack<T>(v, e);
#pragma unroll
  for (int i = 0; i < Elem<T>::N / 2; ++i) f[i] = make2(e[2 * i], e[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const F2* f) {
  float e[Elem<T>::N];
#pragma unroll
  for (int i = 0; i < Elem<T>::N / 2; ++i) {
    const float2 p = split2(f[i]);
    e[2 * i] = p.x;
    e[2 * i + 1] = p.y;
  }
  return pack<T>(e);
}

}  // namespace b200train
