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
  using T = float;
  static constexpr int N = 4;
  u32x4 r;
  __device__ __forceinline__ void load(const float* p) { r = *reinterpret_cast<const u32x4_a4*>(p); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<u32x4_a4*>(p) = r; }
  // ... that nobody reads again soon: the line is the first to leave the caches
  __device__ __forceinline__ void load_once(const float* p) { r = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a4*>(p)); }
  __device__ __forceinline__ void store_once(float* p) const {
    const u32x4_a4 v = r;
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_a4*>(p));
  }
  __device__ __forceinline__ float get(int e) const { return __uint_as_float(r[e]); }
  __device__ __forceinline__ void set(const float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(v[e]);
  }
  __device__ __forceinline__ void zero() { r = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void hold() {}
};
template <> struct RtgVec<rtg_bf16> {
  using T = rtg_bf16;
  static constexpr int N = 8;
  u32x4 r;
  __device__ __forceinline__ void load(const rtg_bf16* p) { r = *reinterpret_cast<const u32x4_a2*>(p); }
  __device__ __forceinline__ void store(rtg_bf16* p) const { *reinterpret_cast<u32x4_a2*>(p) = r; }
  __device__ __forceinline__ void load_once(const rtg_bf16* p) { r = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2*>(p)); }
  __device__ __forceinline__ void store_once(rtg_bf16* p) const {
    const u32x4_a2 v = r;
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_a2*>(p));
  }
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

template <bool ONCE, class V, class T>
__device__ __forceinline__ void rtg_load(V& v, const T* p) {
  if constexpr (ONCE) v.load_once(p);
  else v.load(p);
}
template <bool ONCE, class V, class T>
__device__ __forceinline__ void rtg_store(const V& v, T* p) {
  if constexpr (ONCE) v.store_once(p);
  else v.store(p);
}

// a single element in the place of a vector: axes shorter than one
template <class E> struct RtgOne {
  using T = E;
  static constexpr int N = 1;
  E r;
  __device__ __forceinline__ void load(const E* p) { r = *p; }
  __device__ __forceinline__ void load_once(const E* p) { r = *p; }
  __device__ __forceinline__ void store(E* p) const { *p = r; }
  __device__ __forceinline__ float get(int) const { return rtg_up(r); }
  __device__ __forceinline__ void set(const float (&v)[1]) { rtg_down(v[0], r); }
  __device__ __forceinline__ void zero() { r = E{}; }
  __device__ __forceinline__ void hold() {}
};

// v + (v of another lane), by vector instructions alone (a shuffle goes through LDS: six of them are ~400 cycles of a short
// row's time).  CTRL: a DPP pattern inside 16 lanes
template <int CTRL>
__device__ __forceinline__ float rtg_add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int RTG_DPP_XOR1 = 0xB1, RTG_DPP_XOR2 = 0x4E, RTG_DPP_HALF_MIRROR = 0x141, RTG_DPP_MIRROR = 0x140,
              RTG_DPP_QUAD_MIRROR = 0x1B, RTG_DPP_ROR8 = 0x128;
// ... of the lane 16 / 32 away (the two halves of a swap of v with itself: the even and the odd rows / the lower and upper half)
__device__ __forceinline__ float rtg_add_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float rtg_add_32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// the sum over groups of L adjacent lanes (8 .. 64), in every lane
template <int L>
__device__ __forceinline__ float rtg_group_sum(float v) {
  v = rtg_add_dpp<RTG_DPP_XOR1>(v);
  v = rtg_add_dpp<RTG_DPP_XOR2>(v);
  v = rtg_add_dpp<RTG_DPP_HALF_MIRROR>(v);              // (quads are of one value: a mirror is a swap of the two)
  if constexpr (L >= 16) v = rtg_add_dpp<RTG_DPP_MIRROR>(v);
  if constexpr (L >= 32) v = rtg_add_16(v);
  if constexpr (L >= 64) v = rtg_add_32(v);
  return v;
}
// v of the lane L away (lane ^ L)
template <int L>
__device__ __forceinline__ float rtg_swap(float v) {
  static_assert(L == 2 || L == 4 || L == 8, "inside a row of 16 lanes");
  const int i = __float_as_int(v);
  if constexpr (L == 2) return __int_as_float(__builtin_amdgcn_update_dpp(0, i, RTG_DPP_XOR2, 0xf, 0xf, true));
  if constexpr (L == 8) return __int_as_float(__builtin_amdgcn_update_dpp(0, i, RTG_DPP_ROR8, 0xf, 0xf, true));
  // a mirror of every eight lanes (lane ^ 7), then of every four (lane ^ 3)
  const int m = __builtin_amdgcn_update_dpp(0, i, RTG_DPP_HALF_MIRROR, 0xf, 0xf, true);
  return __int_as_float(__builtin_amdgcn_update_dpp(0, m, RTG_DPP_QUAD_MIRROR, 0xf, 0xf, true));
}
__device__ __forceinline__ bool rtg_upper(int l) { return (threadIdx.x & l) != 0; }

// Sums over the lanes that agree in lane % LP, of V values at once: at each level a lane hands half of its values to its partner
// and adds the partner's to the half it keeps (a swap instruction and an addition for two sums), so that V sums over 64 / LP
// lanes cost V - 1 exchanges, not V times their logarithm, and what follows from a sum is computed once, not in every lane.
// rtg_scatter_sum leaves max(1, V LP / 64) sums in a lane (v[0 ..]); rtg_gather gives every lane all V of what it made of them.
template <int L>
__device__ __forceinline__ float rtg_sum_two(float a, float b) {          // lower lanes: the sum of a, upper lanes: of b
  if constexpr (L == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else if constexpr (L == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    const bool up = rtg_upper(L);
    return (up ? b : a) + rtg_swap<L>(up ? a : b);
  }
}
template <int L>
__device__ __forceinline__ float rtg_sum_one(float v) {
  if constexpr (L >= 16) return rtg_sum_two<L>(v, v);
  else return v + rtg_swap<L>(v);
}
template <int L>
__device__ __forceinline__ void rtg_spread(float& lower, float& upper) {   // `lower` of the lower and of the upper lanes
  const unsigned u = __float_as_uint(lower);
  if constexpr (L == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    lower = __uint_as_float(r[0]);
    upper = __uint_as_float(r[1]);
  } else if constexpr (L == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    lower = __uint_as_float(r[0]);
    upper = __uint_as_float(r[1]);
  } else {
    const float mine = lower, other = rtg_swap<L>(lower);
    const bool up = rtg_upper(L);
    lower = up ? other : mine;
    upper = up ? mine : other;
  }
}
template <int LP, int V, int L = 32>
__device__ __forceinline__ void rtg_scatter_sum(float* v) {
  if constexpr (L >= LP) {
    if constexpr (V > 1) {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) v[k] = rtg_sum_two<L>(v[k], v[k + V / 2]);
      rtg_scatter_sum<LP, V / 2, L / 2>(v);
    } else {
      v[0] = rtg_sum_one<L>(v[0]);
      rtg_scatter_sum<LP, 1, L / 2>(v);
    }
  }
}
template <int LP, int V, int L = 32>
__device__ __forceinline__ void rtg_gather(float* v) {
  if constexpr (L >= LP && V > 1) {
    rtg_gather<LP, V / 2, L / 2>(v);
#pragma unroll
    for (int k = V / 2 - 1; k >= 0; --k) rtg_spread<L>(v[k], v[k + V / 2]);
  }
}
constexpr int rtg_scattered(int lp, int v) { return v * lp > 64 ? v * lp / 64 : 1; }
