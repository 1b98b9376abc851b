// Two neighbouring elements at a time: the instructions that work on pairs of floats, and pairs of elements
// of a row in memory.
#pragma once

#include "m3_common.cuh"

namespace m3 {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two floats in one register pair, for the instructions that work on both
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float a, float b) {
  f2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void unpack2(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}

// 1 / (1 + e^-x), from the hardware's 2^x and reciprocal (relative error a few 1e-7)
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ f2 sigmoid2(f2 x) {
  float a, b;
  unpack2(mul2(x, pack2(-kLog2e, -kLog2e)), a, b);
  unpack2(add2(pack2(ex2(a), ex2(b)), pack2(1.f, 1.f)), a, b);
  return pack2(rcp(a), rcp(b));
}
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  unpack2(sigmoid2(pack2(x.x, x.y)), x.x, x.y);
  return x;
}

// A sum in two floats, hi + lo, with what each addition of hi rounds away kept in lo: 48 bits or so, without
// conversions to 64-bit floats and their few units.
struct Two {
  float hi, lo;
  __device__ __forceinline__ void add(float x) {
    const float s = __fadd_rn(hi, x), part = __fsub_rn(s, hi);
    lo = __fadd_rn(lo, __fadd_rn(__fsub_rn(hi, __fsub_rn(s, part)), __fsub_rn(x, part)));
    hi = s;
  }
  __device__ __forceinline__ void add(const Two& o) {
    add(o.hi);
    lo = __fadd_rn(lo, o.lo);
  }
  __device__ __forceinline__ Two shuffled(int mask) const {
    return Two{__shfl_xor_sync(0xffffffffu, hi, mask), __shfl_xor_sync(0xffffffffu, lo, mask)};
  }
  __device__ __forceinline__ float value() const { return __fadd_rn(hi, lo); }
};

// Two neighbouring elements of a row as they lie in memory, converted when they are used, so that loads can
// stay in flight. W32: the row is fp32 whatever T is.
template <typename T> struct Raw2 { uint32_t v; };
template <> struct Raw2<float> { float2 v; };
__device__ __forceinline__ float2 value2(Raw2<float> r) { return r.v; }
__device__ __forceinline__ float2 value2(Raw2<__nv_bfloat16> r) {
  return make_float2(__uint_as_float(r.v << 16), __uint_as_float(r.v & 0xffff0000u));
}
__device__ __forceinline__ float2 value2(Raw2<__half> r) { return __half22float2(*reinterpret_cast<__half2*>(&r.v)); }
// vec: both at once (the address is on a boundary of the pair); else one by one, the second at `second`
template <typename T>
__device__ __forceinline__ Raw2<T> load2(const T* p, bool vec, int second) {
  Raw2<T> r;
  if constexpr (sizeof(T) == 4) {
    if (vec) r.v = *reinterpret_cast<const float2*>(p);
    else r.v = make_float2(p[0], p[second]);
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    if (vec) r.v = *reinterpret_cast<const uint32_t*>(p);
    else r.v = (uint32_t)h[0] | (uint32_t)h[second] << 16;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store2(T* p, bool vec, bool both, float a, float b) {
  if (vec) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(a, b);
    else {
      T v[2] = {from_f32<T>(a), from_f32<T>(b)};
      *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(v);
    }
  } else {
    st(p, a);
    if (both) st(p + 1, b);
  }
}
}  // namespace m3
