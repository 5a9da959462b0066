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

// VEC neighbouring elements of T as they lie in memory: loaded now, turned into fp32 when used (half
// the registers of fp32 while the load is in flight).  The address is aligned to
// min(16, VEC * sizeof(T)) bytes.
template <typename T, int VEC>
struct Vec {
  static constexpr int kBytes = VEC * int(sizeof(T)) < 16 ? VEC * int(sizeof(T)) : 16;
  static constexpr int kEach = kBytes / int(sizeof(T));
  static constexpr int kParts = VEC / kEach;
  using Raw = typename RawVec<kBytes>::type;
  Raw raw[kParts];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int j = 0; j < kParts; ++j) raw[j] = reinterpret_cast<const Raw *>(p)[j];
  }
  __device__ __forceinline__ void clear() { memset(raw, 0, sizeof raw); }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      T e[kEach];
      memcpy(e, &raw[j], kBytes);
#pragma unroll
      for (int k = 0; k < kEach; ++k) v[j * kEach + k] = to_f32(e[k]);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      T e[kEach];
#pragma unroll
      for (int k = 0; k < kEach; ++k) from_f32(v[j * kEach + k], e[k]);
      memcpy(&raw[j], e, kBytes);
    }
  }
  __device__ __forceinline__ void add_to(float (&v)[VEC]) const {
    float x[VEC];
    get(x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] += x[k];
  }
  __device__ __forceinline__ void store(T *p) const {
#pragma unroll
    for (int j = 0; j < kParts; ++j) reinterpret_cast<Raw *>(p)[j] = raw[j];
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[VEC]) {
  Vec<T, VEC> x;
  x.load(p);
  x.get(v);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[VEC]) {
  Vec<T, VEC> x;
  x.set(v);
  x.store(p);
}

}  // namespace arb
