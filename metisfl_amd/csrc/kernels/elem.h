// Element types of the any-type operators: 16-byte packs of fp32 / bf16 / fp16
// that may start at any element (rows of odd width or stride), as floats.
#pragma once
#include "kernels/common.h"

namespace mfl {

struct BF16 {
  uint16_t u;
};
typedef _Float16 F16;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(BF16 v) { return bf2f(v.u); }
__device__ __forceinline__ float to_f(F16 v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ BF16 from_f<BF16>(float v) {
  return BF16{f2bf(v)};
}
template <>
__device__ __forceinline__ F16 from_f<F16>(float v) {
  return (F16)v;
}

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
};

// N elements from p, aligned to the element alone: gfx950's global loads and
// stores take 16 bytes at any such address.
template <typename T, int N>
struct Pack {
  T e[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& v) {
  __builtin_memcpy(p, &v, sizeof(v));
}

// The same past the caches' write-back (16 bytes), for results larger than the
// caches: a stream of stores then does not fetch or evict lines.
template <typename T, int N>
__device__ __forceinline__ void stream_pack(T* p, const Pack<T, N>& v) {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  static_assert(sizeof(v) == 16, "16 bytes");
  Words w;
  __builtin_memcpy(&w, &v, sizeof(w));
  __builtin_nontemporal_store(w, reinterpret_cast<Words*>(p));
}

// Reductions over a wave's rows of 16 lanes by DPP rotations (every lane gets
// the result; a rotation costs a VALU instruction where a shuffle goes through
// LDS), and over all 64 lanes by four lane reads more.  The lanes of a row (of
// the wave) must all be active.
template <int N>
__device__ __forceinline__ float row_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ float sum16(float v) {
  v += row_ror<8>(v);
  v += row_ror<4>(v);
  v += row_ror<2>(v);
  return v + row_ror<1>(v);
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, row_ror<8>(v));
  v = fmaxf(v, row_ror<4>(v));
  v = fmaxf(v, row_ror<2>(v));
  return fmaxf(v, row_ror<1>(v));
}
__device__ __forceinline__ float max4(float v) {  // of a quad
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, false)));  // 1 0 3 2
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, false)));  // 2 3 0 1
}
// Sum over aligned groups of L (16 or 64) lanes.
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
  static_assert(L == 16 || L == 64, "a row of 16 lanes or a wave");
  v = sum16(v);
  if constexpr (L == 64) v = (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
  return v;
}
__device__ __forceinline__ float max64(float v) {
  v = max16(v);
  return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}

}  // namespace mfl
