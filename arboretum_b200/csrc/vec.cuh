// Short vectors of fp32 / bf16 / fp16 elements in registers, loaded and stored in one access of
// up to 16 bytes; arithmetic on them is always in fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace arb {

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<4> { using type = unsigned; };
template <> struct RawVec<2> { using type = unsigned short; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
// rounding to the nearest, ties to even
__device__ __forceinline__ void from_f32(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half &o) { o = __float2half_rn(v); }

// VEC elements of T at `p`, which is aligned to min(16, VEC * sizeof(T)) bytes
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[VEC]) {
  constexpr int kBytes = VEC * int(sizeof(T)) < 16 ? VEC * int(sizeof(T)) : 16;
  constexpr int kEach = kBytes / int(sizeof(T));
  using Raw = typename RawVec<kBytes>::type;
#pragma unroll
  for (int j = 0; j < VEC / kEach; ++j) {
    const Raw r = reinterpret_cast<const Raw *>(p)[j];
    T e[kEach];
    memcpy(e, &r, kBytes);
#pragma unroll
    for (int k = 0; k < kEach; ++k) v[j * kEach + k] = to_f32(e[k]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[VEC]) {
  constexpr int kBytes = VEC * int(sizeof(T)) < 16 ? VEC * int(sizeof(T)) : 16;
  constexpr int kEach = kBytes / int(sizeof(T));
  using Raw = typename RawVec<kBytes>::type;
#pragma unroll
  for (int j = 0; j < VEC / kEach; ++j) {
    T e[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) from_f32(v[j * kEach + k], e[k]);
    Raw r;
    memcpy(&r, e, kBytes);
    reinterpret_cast<Raw *>(p)[j] = r;
  }
}

}  // namespace arb
