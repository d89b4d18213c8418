// rtg_vec.h — 16-byte accesses at element alignment and the float / bf16 conversions around them (the bandwidth kernels of
// rtg_layernorm.hip and rtg_gradnorm.hip).
#pragma once
#include "rtg_common.h"

struct rtg_bf16 { unsigned short u; };

// sixteen bytes of global memory at any 2- or 4-byte address: the memory pipeline splits an access that straddles a line by
// itself, so a tensor that starts in the middle of a flat buffer, or a row of odd length, needs no scalar form of a kernel
typedef unsigned u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float rtg_up(float v) { return v; }
__device__ __forceinline__ float rtg_up(rtg_bf16 v) { return __uint_as_float((unsigned)v.u << 16); }
__device__ __forceinline__ void rtg_down(float v, float& out) { out = v; }
// (bf16: round to nearest even, the one rounding of a result)
__device__ __forceinline__ void rtg_down(float v, rtg_bf16& out) { out.u = __builtin_bit_cast(unsigned short, (__bf16)v); }

// the value is computed here, not later (volatile statements keep their order)
__device__ __forceinline__ void rtg_pin(float& v) { asm volatile("" : "+v"(v)); }

// N elements of T as they lie in memory.  hold(): the compiler forgets what it has computed from the vector, so a kernel that
// reads its tile several times converts it again (a shift an element) instead of keeping every element's float in a register;
// behind rtg_pin of what was summed from it (else the sums move behind hold() and the vector is kept twice).
template <class T> struct RtgVec;
template <> struct RtgVec<float> {
  static constexpr int N = 4;
  u32x4 r;
  __device__ __forceinline__ void load(const float* p) { r = *reinterpret_cast<const u32x4_a4*>(p); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<u32x4_a4*>(p) = r; }
  __device__ __forceinline__ float get(int e) const { return __uint_as_float(r[e]); }
  __device__ __forceinline__ void set(const float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(v[e]);
  }
  __device__ __forceinline__ void zero() { r = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void hold() {}
};
template <> struct RtgVec<rtg_bf16> {
  static constexpr int N = 8;
  u32x4 r;
  __device__ __forceinline__ void load(const rtg_bf16* p) { r = *reinterpret_cast<const u32x4_a2*>(p); }
  __device__ __forceinline__ void store(rtg_bf16* p) const { *reinterpret_cast<u32x4_a2*>(p) = r; }
  __device__ __forceinline__ float get(int e) const {
    return __uint_as_float(e & 1 ? r[e >> 1] & 0xffff0000u : r[e >> 1] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned lo = __builtin_bit_cast(unsigned short, (__bf16)v[2 * e]);
      const unsigned hi = __builtin_bit_cast(unsigned short, (__bf16)v[2 * e + 1]);
      r[e] = lo | (hi << 16);
    }
  }
  __device__ __forceinline__ void zero() { r = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void hold() { asm volatile("" : "+v"(r)); }
};
