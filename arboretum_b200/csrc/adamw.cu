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

__device__ __forceinline__ float load_as(const void *p, int type, long long i) {
  if (type == kF32) return static_cast<const float *>(p)[i];
  if (type == kBF16) return to_f32(static_cast<const __nv_bfloat16 *>(p)[i]);
  return to_f32(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_as(void *p, int type, long long i, float v) {
  if (type == kF32) static_cast<float *>(p)[i] = v;
  else if (type == kBF16) from_f32(v, static_cast<__nv_bfloat16 *>(p)[i]);
  else from_f32(v, static_cast<__half *>(p)[i]);
}

constexpr int kThreads = 128;  // a CTA step covers one 8-bit block

template <int BITS>
__global__ void __launch_bounds__(kThreads) adamw_kernel(AdamWLaunch a, const __grid_constant__ GradPointers grads,
                                                         int first_tensor, int first_chunk, int n_chunks, bool last) {
  __shared__ unsigned warp_m[4], warp_r[4];
  const Scalars c = scalars_of(a);
  for (int k = blockIdx.x; k < n_chunks; k += gridDim.x) {
    const AdamWChunk ch = a.chunks[first_chunk + k];
    const AdamWTensor t = a.tensors[ch.tensor];
    const void *grad = grads.at[ch.tensor - first_tensor];
    if (grad == nullptr) continue;
    const int grad_type = a.grad_f32 ? kF32 : t.type;
    const long long i1 = min(t.n, (ch.index + 1ll) * kAdamWChunk);
    for (long long i0 = (long long)ch.index * kAdamWChunk; i0 < i1; i0 += kThreads) {
      const long long i = i0 + threadIdx.x, at = t.slot + i;
      const bool in = i < i1;
      float m = 0.0f, v = 0.0f, root = 0.0f;
      if (in) {
        const float g = load_as(grad, grad_type, i) * c.grad_scale;
        float p = a.master ? a.master[at] : load_as(t.param, t.type, i);
        if (BITS == 8) {
          m = decode(static_cast<unsigned char *>(a.moment1)[at], a.scale1[at / kMomentBlock]);
          const float r = decode(static_cast<unsigned char *>(a.moment2)[at], a.scale2[at / kMomentBlock]);
          v = r * r;
        } else {
          m = static_cast<float *>(a.moment1)[at];
          v = static_cast<float *>(a.moment2)[at];
        }
        m = m * c.beta1 + g * c.one_beta1;
        v = v * c.beta2 + (g * g) * c.one_beta2;
        root = sqrtf(v);
        p = p * c.keep - (m / (root * c.inv_root_bc2 + c.eps)) * c.step_size;
        store_as(t.param, t.type, i, p);
        if (a.master) a.master[at] = p;
        if (BITS == 32) {
          static_cast<float *>(a.moment1)[at] = m;
          static_cast<float *>(a.moment2)[at] = v;
        }
      }
      if (BITS == 8) {
        const unsigned mm = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(m)));
        const unsigned mr = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(root)));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) warp_m[threadIdx.x >> 5] = mm, warp_r[threadIdx.x >> 5] = mr;
        __syncthreads();
        const unsigned fm = scale_field(max(max(warp_m[0], warp_m[1]), max(warp_m[2], warp_m[3])));
        const unsigned fr = scale_field(max(max(warp_r[0], warp_r[1]), max(warp_r[2], warp_r[3])));
        if (in) {
          const unsigned h = hash_bits((unsigned long long)at, c.step, a.seed);
          const unsigned cm = encode(m, inv_scale_of(fm), h & 0xffffu) | (m < 0.0f ? 128u : 0u);
          unsigned cr = encode(root, inv_scale_of(fr), h >> 16);
          if (root > 0.0f) cr = max(cr, 1u);
          static_cast<unsigned char *>(a.moment1)[at] = (unsigned char)cm;
          static_cast<unsigned char *>(a.moment2)[at] = (unsigned char)cr;
        }
        if (threadIdx.x == 0) {
          a.scale1[at / kMomentBlock] = scale_of(fm);
          a.scale2[at / kMomentBlock] = scale_of(fr);
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
      const int grid = std::max(1, std::min(chunks, device_sm_count() * 16));
      if (a.bits == 8) adamw_kernel<8><<<grid, kThreads, 0, s>>>(a, g, t0, first_chunk[t0], chunks, last);
      else adamw_kernel<32><<<grid, kThreads, 0, s>>>(a, g, t0, first_chunk[t0], chunks, last);
      ARB_CUDA(cudaGetLastError());
      count_launch();
    }
    if (last) break;
  }
}

}  // namespace arb
