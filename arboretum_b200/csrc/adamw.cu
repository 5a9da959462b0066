// AdamW step over many tensors in one launch, moments in fp32 or in 8 bits:
//
//   g' = grad * grad_scale          m = beta1 m + (1 - beta1) g'       v = beta2 v + (1 - beta2) g'^2
//   p  = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// all in fp32; p is rounded to its type at the end (or kept in fp32 beside a rounded copy).
//
// Moments in 8 bits: 128 elements of a tensor share a power of two, and an element is that times an
// e4m3 number; the second moment is kept as its square root, which halves the range of exponents it
// needs.  A moment moves by (1 - beta) of its distance a step, often less than half an e4m3 step,
// so rounding to the nearest would freeze it: the rounding is dithered by a hash of (element, step,
// seed), an element goes up with the probability of its remainder.  A root above zero never becomes
// zero (it is divided by).  A block that holds an infinity or a NaN reads back as NaN.
#include <algorithm>
#include <cmath>

#include "operators.h"
#include "vec.cuh"

namespace arb {

namespace {

constexpr int kMaxGrads = 2048;  // gradient pointers of one launch (kernel parameters: 16 KB)
struct GradPointers {
  const void *at[kMaxGrads];
};

// the same mixing as the dither of the boosting gradients, here for 32 bits of it
__device__ __forceinline__ unsigned hash_bits(unsigned long long index, unsigned step, unsigned seed) {
  unsigned x = unsigned(index) ^ (unsigned(index >> 32) * 0x9E3779B1u) ^ (step * 0x85EBCA6Bu) ^ (seed * 0xC2B2AE35u);
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  x ^= x >> 16;
  return x;
}

// e4m3 magnitude: shifted to the top of the mantissa it is a float whose exponent is 2^120 short
__device__ __forceinline__ float decode(unsigned code, float scale) {
  const float v = __uint_as_float((code & 127u) << 20) * 0x1p120f * scale;
  return code & 128u ? -v : v;
}
__device__ __forceinline__ unsigned encode(float x, float inv_scale, unsigned random16) {
  const unsigned bits = __float_as_uint(fabsf(x) * inv_scale * 0x1p-120f);
  return min((bits + (random16 << 4) + 8u) >> 20, 126u);
}
// exponent field of the scale of a block whose largest magnitude has these bits: the largest code
// stands for 448 = 1.75 * 2^8.  255: the block holds a value that is not finite
__device__ __forceinline__ unsigned scale_field(unsigned top_bits) {
  const unsigned e = (top_bits + 0x1FFFFFu) >> 23;
  return e >= 255u ? 255u : max(int(e) - 8, 1);
}
__device__ __forceinline__ float scale_of(unsigned field) {
  return __uint_as_float(field == 255u ? 0x7FC00000u : field << 23);
}
__device__ __forceinline__ float inv_scale_of(unsigned field) {
  return __uint_as_float(field == 255u ? 0u : (254u - field) << 23);
}

struct Scalars {
  float beta1, one_beta1, beta2, one_beta2, inv_root_bc2, step_size, keep, eps, grad_scale;
  unsigned step;
};

__device__ __forceinline__ Scalars scalars_of(const AdamWLaunch &a) {
  Scalars c;
  const double b1t = a.state->beta1_t * a.beta1, b2t = a.state->beta2_t * a.beta2;
  const double lr = a.lr_device ? double(*a.lr_device) : a.lr;
  c.beta1 = float(a.beta1), c.one_beta1 = float(1.0 - a.beta1);
  c.beta2 = float(a.beta2), c.one_beta2 = float(1.0 - a.beta2);
  c.inv_root_bc2 = float(1.0 / sqrt(1.0 - b2t));
  c.step_size = float(lr / (1.0 - b1t));
  c.keep = float(1.0 - lr * a.decay);
  c.eps = a.eps;
  c.grad_scale = a.grad_scale ? *a.grad_scale : 1.0f;
  c.step = unsigned(a.state->step + 1);
  return c;
}

// Eight neighbouring elements of a tensor of type T.  `vec`: the tensor starts on a 16-byte
// boundary; the last elements of a tensor, and tensors that start elsewhere, go one by one.
constexpr int kEach = 8;
template <typename T>
__device__ __forceinline__ void load_each(const T *p, long long i, int left, bool vec, float (&v)[kEach]) {
  if (vec && left >= kEach) {
    load_vec<T, kEach>(p + i, v);
  } else {
#pragma unroll
    for (int j = 0; j < kEach; ++j) v[j] = j < left ? to_f32(p[i + j]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_each(T *p, long long i, int left, bool vec, const float (&v)[kEach]) {
  if (vec && left >= kEach) {
    store_vec<T, kEach>(p + i, v);
  } else {
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (j < left) from_f32(v[j], p[i + j]);
  }
}
__device__ __forceinline__ void load_typed(const void *p, int type, long long i, int left, bool vec, float (&v)[kEach]) {
  if (type == kF32) load_each(static_cast<const float *>(p), i, left, vec, v);
  else if (type == kBF16) load_each(static_cast<const __nv_bfloat16 *>(p), i, left, vec, v);
  else load_each(static_cast<const __half *>(p), i, left, vec, v);
}
__device__ __forceinline__ void store_typed(void *p, int type, long long i, int left, bool vec, const float (&v)[kEach]) {
  if (type == kF32) store_each(static_cast<float *>(p), i, left, vec, v);
  else if (type == kBF16) store_each(static_cast<__nv_bfloat16 *>(p), i, left, vec, v);
  else store_each(static_cast<__half *>(p), i, left, vec, v);
}

constexpr int kThreads = 256;
constexpr int kLanes = kMomentBlock / kEach;  // lanes that hold an 8-bit block: half a warp

// A thread takes eight neighbouring elements: 16 bytes of a half-precision tensor, two accesses of 16
// of a float one, 8 bytes of codes; half a warp holds a block, so its largest magnitude is found with
// shuffles.  All loads of an element are issued before the first is used: 128 bytes a thread in flight.
template <int BITS>
__global__ void __launch_bounds__(kThreads) adamw_kernel(AdamWLaunch a, const __grid_constant__ GradPointers grads,
                                                         int first_tensor, int first_chunk, int n_chunks, bool last) {
  __shared__ Scalars shared_scalars;
  if (threadIdx.x == 0) shared_scalars = scalars_of(a);
  __syncthreads();
  const Scalars c = shared_scalars;
  for (int k = blockIdx.x; k < n_chunks; k += gridDim.x) {
    const AdamWChunk ch = a.chunks[first_chunk + k];
    const AdamWTensor t = a.tensors[ch.tensor];
    const void *grad = grads.at[ch.tensor - first_tensor];
    if (grad == nullptr) continue;
    const int grad_type = a.grad_f32 ? kF32 : t.type;
    const bool grad_vec = reinterpret_cast<unsigned long long>(grad) % 16 == 0, vec = t.vec != 0;
    const long long i1 = min(t.n, (ch.index + 1ll) * kAdamWChunk);
    for (long long i0 = (long long)ch.index * kAdamWChunk; i0 < i1; i0 += kThreads * kEach) {
      const long long i = i0 + threadIdx.x * kEach, at = t.slot + i;
      const int left = int(min((long long)kEach, i1 - i));  // <= 0: nothing here, the lane only takes part in the shuffles
      if (BITS == 32 && left <= 0) continue;
      float p[kEach], g[kEach], m[kEach], v[kEach];
      load_typed(grad, grad_type, i, left, grad_vec, g);
      if (a.master) load_each(a.master, at, left, true, p);
      else load_typed(t.param, t.type, i, left, vec, p);
      if (BITS == 32) {
        load_each(static_cast<float *>(a.moment1), at, left, true, m);
        load_each(static_cast<float *>(a.moment2), at, left, true, v);
      } else if (left > 0) {  // slots are whole blocks: the codes behind a tensor's end are there
        const uint2 cm = *reinterpret_cast<const uint2 *>(static_cast<unsigned char *>(a.moment1) + at);
        const uint2 cr = *reinterpret_cast<const uint2 *>(static_cast<unsigned char *>(a.moment2) + at);
        const float s1 = a.scale1[at / kMomentBlock], s2 = a.scale2[at / kMomentBlock];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          m[j] = decode((j < 4 ? cm.x : cm.y) >> (j % 4 * 8) & 255u, s1);
          const float r = decode((j < 4 ? cr.x : cr.y) >> (j % 4 * 8) & 255u, s2);
          v[j] = r * r;
        }
      }
      unsigned top_m = 0, top_r = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const float gj = g[j] * c.grad_scale;
        m[j] = m[j] * c.beta1 + gj * c.one_beta1;
        v[j] = v[j] * c.beta2 + (gj * gj) * c.one_beta2;
        const float root = sqrtf(v[j]);
        p[j] = p[j] * c.keep - (m[j] / (root * c.inv_root_bc2 + c.eps)) * c.step_size;
        if (BITS == 8) {
          v[j] = root;
          if (j < left) {
            top_m = max(top_m, __float_as_uint(m[j]) & 0x7FFFFFFFu);
            top_r = max(top_r, __float_as_uint(root) & 0x7FFFFFFFu);
          }
        }
      }
      store_typed(t.param, t.type, i, left, vec, p);
      if (a.master) store_each(a.master, at, left, true, p);
      if (BITS == 32) {
        store_each(static_cast<float *>(a.moment1), at, left, true, m);
        store_each(static_cast<float *>(a.moment2), at, left, true, v);
      } else {
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) {
          top_m = max(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
          top_r = max(top_r, __shfl_xor_sync(0xffffffffu, top_r, o));
        }
        if (left > 0) {
          const unsigned fm = scale_field(top_m), fr = scale_field(top_r);
          const float im = inv_scale_of(fm), ir = inv_scale_of(fr);
          uint2 cm = make_uint2(0u, 0u), cr = make_uint2(0u, 0u);
#pragma unroll
          for (int j = 0; j < kEach; ++j) {
            if (j < left) {
              const unsigned h = hash_bits((unsigned long long)(at + j), c.step, a.seed);
              const unsigned em = encode(m[j], im, h & 0xffffu) | (m[j] < 0.0f ? 128u : 0u);
              unsigned er = encode(v[j], ir, h >> 16);
              if (v[j] > 0.0f) er = max(er, 1u);
              (j < 4 ? cm.x : cm.y) |= em << (j % 4 * 8);
              (j < 4 ? cr.x : cr.y) |= er << (j % 4 * 8);
            }
          }
          *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(a.moment1) + at) = cm;
          *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(a.moment2) + at) = cr;
          if (threadIdx.x % kLanes == 0) {
            a.scale1[at / kMomentBlock] = scale_of(fm);
            a.scale2[at / kMomentBlock] = scale_of(fr);
          }
        }
      }
    }
  }
  // the last CTA of the step's last launch moves the step count on: every CTA has read it by then
  __syncthreads();
  if (last && threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(&a.state->done, 1u) == gridDim.x - 1) {
      a.state->beta1_t *= a.beta1;
      a.state->beta2_t *= a.beta2;
      a.state->step += 1;
      a.state->done = 0;
    }
  }
}

}  // namespace

void launch_adamw(const AdamWLaunch &a, const void *const *grads, const std::vector<int> &first_chunk,
                  int n_tensors, cudaStream_t s) {
  GradPointers g;
  for (int t0 = 0;; t0 += kMaxGrads) {
    const int t1 = std::min(n_tensors, t0 + kMaxGrads);
    const bool last = t1 == n_tensors;
    std::copy(grads + t0, grads + t1, g.at);
    const int chunks = first_chunk[t1] - first_chunk[t0];
    if (chunks > 0 || last) {  // a step without elements still counts
      const int grid = std::max(1, std::min(chunks, device_sm_count() * 8));
      if (a.bits == 8) adamw_kernel<8><<<grid, kThreads, 0, s>>>(a, g, t0, first_chunk[t0], chunks, last);
      else adamw_kernel<32><<<grid, kThreads, 0, s>>>(a, g, t0, first_chunk[t0], chunks, last);
      ARB_CUDA(cudaGetLastError());
      count_launch();
    }
    if (last) break;
  }
}

}  // namespace arb
