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
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "operators.h"
#include "vec.cuh"

namespace arb {

namespace {

constexpr int kMaxGrads = 2048;  // gradient pointers of one launch (kernel parameters: 16 KB)
struct GradPointers {
  const void *at[kMaxGrads];
};

// 32 bits for an element: the mixing of the boosting gradients' dither.  `key` holds what the eight
// elements of a thread share: the upper half of the index, the step and the seed.
__device__ __forceinline__ unsigned hash_key(unsigned long long index, unsigned step, unsigned seed) {
  return unsigned(index) ^ (unsigned(index >> 32) * 0x9E3779B1u) ^ (step * 0x85EBCA6Bu) ^ (seed * 0xC2B2AE35u);
}
__device__ __forceinline__ unsigned hash_bits(unsigned x) {
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  x ^= x >> 16;
  return x;
}

// two e4m3 codes as floats
__device__ __forceinline__ float2 decode2(unsigned codes) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3)));
}
// Magnitude of the code for x = value / scale * 2^-120 >= 0: there e4m3's exponents are float's
// smallest, so a code is the top of the bits, and the dither is added to the 20 bits that go.
// `random` holds 16 bits, shifted up by four.
__device__ __forceinline__ unsigned encode(float x, unsigned random) {
  return min((__float_as_uint(x) + ((random & 0xFFFF0u) | 8u)) >> 20, 126u);
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
  const double lr = a.lr_device ? double(*a.lr_device) : a.lr;
  c.beta1 = float(a.beta1), c.one_beta1 = float(1.0 - a.beta1);
  c.beta2 = float(a.beta2), c.one_beta2 = float(1.0 - a.beta2);
  c.inv_root_bc2 = a.state->inv_root_bc2;
  c.step_size = float(lr * a.state->inv_bc1);
  c.keep = float(1.0 - lr * a.decay);
  c.eps = a.eps;
  c.grad_scale = a.grad_scale ? *a.grad_scale : 1.0f;
  c.step = unsigned(a.state->step + 1);
  return c;
}

// Root of v >= 0, rounded to the nearest like sqrtf: one Newton step on the hardware's reciprocal root
// with the residual in a fused multiply-add (Markstein's correction), a third of sqrtf's instructions.
// Exhaustively equal to sqrtf for zero and all of [2^-100, 2^126]; the others take sqrtf.
__device__ __forceinline__ float root_of(float v) {
  float q;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(fmaxf(v, 0x1p-100f)));  // v == 0: finite, the product is zero
  const float s = __fmul_rn(v, q);
  return __fmaf_rn(__fmaf_rn(-s, s, v), __fmul_rn(0.5f, q), s);
}
__device__ __forceinline__ bool root_is_plain(unsigned largest, unsigned smallest_less_one) {
  return largest <= 0x7E800000u && smallest_less_one >= 0x0D800000u - 1u;  // 2^126, 2^-100; zero less one is large
}
// larger magnitude; a NaN stays
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// quotient off by two units in the last place at most: a millionth of the step it scales
__device__ __forceinline__ float quotient(float a, float b) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b));
  return a * r;
}

constexpr int kThreads = 256;
constexpr int kEach = 8;                      // neighbouring elements of a thread
constexpr int kTileElems = kThreads * kEach;  // elements of a CTA at a time
constexpr int kLanes = kMomentBlock / kEach;  // lanes that hold an 8-bit block: half a warp

// eight elements as they lie in memory; `whole`: all are there and the address is 16-byte aligned
template <typename T>
__device__ __forceinline__ void load_each(Vec<T, kEach> &v, const T *p, int left, bool whole) {
  if (whole) {
    v.load(p);
  } else {
    float x[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) x[j] = j < left ? to_f32(p[j]) : 0.0f;
    v.set(x);
  }
}
template <typename T>
__device__ __forceinline__ void store_each(T *p, const float (&x)[kEach], int left, bool whole) {
  if (whole) {
    store_vec<T, kEach>(p, x);
  } else {
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (j < left) from_f32(x[j], p[j]);
  }
}

// A thread's share of a tile.  All loads of a tile are issued before the first value is used.
template <int BITS, typename P, typename G, bool MASTER>
struct Tile {
  using W = typename std::conditional<MASTER, float, P>::type;
  Vec<W, kEach> w;
  Vec<G, kEach> g;
  Vec<float, kEach> m32, v32;
  uint2 cm, cr;
  float s1, s2;

  __device__ __forceinline__ void load(const AdamWLaunch &a, const P *param, const G *grad, long long at, int left, bool vec,
                                       bool grad_vec) {
    const bool full = left >= kEach;
    load_each(g, grad, left, full && grad_vec);
    if constexpr (MASTER) load_each(w, a.master + at, left, full);
    else load_each(w, param, left, full && vec);
    if constexpr (BITS == 32) {
      load_each(m32, static_cast<const float *>(a.moment1) + at, left, full);
      load_each(v32, static_cast<const float *>(a.moment2) + at, left, full);
    } else {
      cm = cr = make_uint2(0u, 0u);
      s1 = s2 = 0.0f;
      if (left > 0) {  // slots are whole blocks: the codes behind a tensor's end are there, zeros
        cm = *reinterpret_cast<const uint2 *>(static_cast<const unsigned char *>(a.moment1) + at);
        cr = *reinterpret_cast<const uint2 *>(static_cast<const unsigned char *>(a.moment2) + at);
        s1 = a.scale1[at / kMomentBlock];
        s2 = a.scale2[at / kMomentBlock];
      }
    }
  }

  // (elements past a tensor's end have no weight and no gradient, and moments of zero: they stay so)
  __device__ __forceinline__ void step(const AdamWLaunch &a, const Scalars &c, P *param, long long at, int left, bool vec) const {
    float p[kEach], gr[kEach], m[kEach], v[kEach];
    g.get(gr);
    w.get(p);
    if constexpr (BITS == 32) {
      m32.get(m);
      v32.get(v);
    } else {
#pragma unroll
      for (int j = 0; j < kEach; j += 2) {
        const float2 mj = decode2((j < 4 ? cm.x : cm.y) >> (j % 4 * 8) & 0xFFFFu);
        const float2 rj = decode2((j < 4 ? cr.x : cr.y) >> (j % 4 * 8) & 0xFFFFu);
        m[j] = mj.x * s1, m[j + 1] = mj.y * s1;
        const float r0 = rj.x * s2, r1 = rj.y * s2;
        v[j] = r0 * r0, v[j + 1] = r1 * r1;
      }
    }
    unsigned largest = 0, smallest = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const float gj = gr[j] * c.grad_scale;
      m[j] = m[j] * c.beta1 + gj * c.one_beta1;
      v[j] = v[j] * c.beta2 + (gj * gj) * c.one_beta2;
      largest = max(largest, __float_as_uint(v[j]));
      smallest = min(smallest, __float_as_uint(v[j]) - 1u);
    }
    float root[kEach];
    if (root_is_plain(largest, smallest)) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) root[j] = root_of(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kEach; ++j) root[j] = sqrtf(v[j]);
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      p[j] = p[j] * c.keep - quotient(m[j], root[j] * c.inv_root_bc2 + c.eps) * c.step_size;
    const bool full = left >= kEach;
    store_each(param, p, left, full && vec);
    if constexpr (MASTER) store_each(a.master + at, p, left, full);
    if constexpr (BITS == 32) {
      store_each(static_cast<float *>(a.moment1) + at, m, left, full);
      store_each(static_cast<float *>(a.moment2) + at, v, left, full);
    } else {
      float top_m = 0.0f, top_r = 0.0f;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        top_m = larger(top_m, fabsf(m[j]));
        top_r = larger(top_r, root[j]);
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        top_m = larger(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
        top_r = larger(top_r, __shfl_xor_sync(0xffffffffu, top_r, o));
      }
      if (left <= 0) return;
      const unsigned fm = scale_field(__float_as_uint(top_m) & 0x7FFFFFFFu), fr = scale_field(__float_as_uint(top_r) & 0x7FFFFFFFu);
      const unsigned key = hash_key((unsigned long long)at, c.step, a.seed);  // at is a multiple of eight
      unsigned em[kEach], er[kEach];
      // the scale's inverse and e4m3's shift of 2^-120 are one factor unless it would fall below float's
      // smallest normal number: moments beyond 448 * 64
      if (fm <= 133u && fr <= 133u) {
        const float im = __uint_as_float((134u - fm) << 23), ir = __uint_as_float((134u - fr) << 23);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          const unsigned h = hash_bits(key ^ unsigned(j));
          em[j] = encode(fabsf(m[j]) * im, h << 4);
          er[j] = encode(root[j] * ir, h >> 12);
        }
      } else {
        const float im = inv_scale_of(fm), ir = inv_scale_of(fr);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          const unsigned h = hash_bits(key ^ unsigned(j));
          em[j] = encode(fabsf(m[j]) * im * 0x1p-120f, h << 4);
          er[j] = encode(root[j] * ir * 0x1p-120f, h >> 12);
        }
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        em[j] |= m[j] < 0.0f ? 128u : 0u;
        er[j] = max(er[j], min(__float_as_uint(root[j]), 1u));  // above zero stays above zero
      }
      const auto pack = [](const unsigned *e) { return e[0] | e[1] << 8 | e[2] << 16 | e[3] << 24; };
      *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(a.moment1) + at) = make_uint2(pack(em), pack(em + 4));
      *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(a.moment2) + at) = make_uint2(pack(er), pack(er + 4));
      if (threadIdx.x % kLanes == 0) {
        a.scale1[at / kMomentBlock] = scale_of(fm);
        a.scale2[at / kMomentBlock] = scale_of(fr);
      }
    }
  }
};

template <int BITS, typename P, typename G, bool MASTER>
__device__ __forceinline__ void step_chunk(const AdamWLaunch &a, const Scalars &c, const AdamWTensor &t, const void *grad_at,
                                           long long first) {
  const bool vec = t.vec != 0, grad_vec = reinterpret_cast<unsigned long long>(grad_at) % 16 == 0;
  P *param = static_cast<P *>(t.param) + first;
  const G *grad = static_cast<const G *>(grad_at) + first;
  const long long slot = t.slot + first;
  const int n = int(min(t.n - first, (long long)kAdamWChunk));
  // a thread behind the end (n - i <= 0) loads and stores nothing, but takes part in the shuffles
  int i = threadIdx.x * kEach;
  Tile<BITS, P, G, MASTER> tile;
  if constexpr (BITS == 8) tile.load(a, param + i, grad + i, slot + i, n - i, vec, grad_vec);
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kTileElems, i += kTileElems) {
    if constexpr (BITS == 8) {  // few bytes and much arithmetic: the next tile is on its way meanwhile
      const Tile<BITS, P, G, MASTER> now = tile;
      const int next = i + kTileElems;
      tile.load(a, param + next, grad + next, slot + next, n - next, vec, grad_vec);
      now.step(a, c, param + i, slot + i, n - i, vec);
    } else {
      tile.load(a, param + i, grad + i, slot + i, n - i, vec, grad_vec);
      tile.step(a, c, param + i, slot + i, n - i, vec);
    }
  }
}

template <int BITS, bool MASTER>
__global__ void __launch_bounds__(kThreads, BITS == 8 ? 3 : 4) adamw_kernel(AdamWLaunch a, const __grid_constant__ GradPointers grads,
                                                            int first_tensor, int first_chunk, int n_chunks, bool last) {
  __shared__ Scalars shared_scalars;
  if (threadIdx.x == 0) shared_scalars = scalars_of(a);
  const AdamWChunk ch = int(blockIdx.x) < n_chunks ? a.chunks[first_chunk + blockIdx.x] : AdamWChunk{-1, 0};
  __syncthreads();
  const Scalars c = shared_scalars;
  const void *grad = ch.tensor < 0 ? nullptr : grads.at[ch.tensor - first_tensor];
  if (grad != nullptr) {
    const AdamWTensor t = a.tensors[ch.tensor];
    const long long first = (long long)ch.index * kAdamWChunk;
    if (t.type == kF32) step_chunk<BITS, float, float, MASTER>(a, c, t, grad, first);
    else if (t.type == kBF16 && a.grad_f32) step_chunk<BITS, __nv_bfloat16, float, MASTER>(a, c, t, grad, first);
    else if (t.type == kBF16) step_chunk<BITS, __nv_bfloat16, __nv_bfloat16, MASTER>(a, c, t, grad, first);
    else if (a.grad_f32) step_chunk<BITS, __half, float, MASTER>(a, c, t, grad, first);
    else step_chunk<BITS, __half, __half, MASTER>(a, c, t, grad, first);
  }
  // the last CTA of the step's last launch moves the step count on: every CTA has read it by then
  if (last && threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(&a.state->done, 1u) == gridDim.x - 1) {
      AdamWState st = *a.state;
      st.advance(a.beta1, a.beta2);
      st.done = 0;
      *a.state = st;
    }
  }
}

}  // namespace

namespace {
// a chunk a CTA: the chunks of a step are uneven (tensors end inside them), so the device hands them out
template <int BITS, bool MASTER>
void launch_with(const AdamWLaunch &a, const GradPointers &g, int first_tensor, int first_chunk, int chunks, bool last,
                 cudaStream_t s) {
  adamw_kernel<BITS, MASTER><<<std::max(1, chunks), kThreads, 0, s>>>(a, g, first_tensor, first_chunk, chunks, last);
  ARB_CUDA(cudaGetLastError());
  count_launch();
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
      const auto launch = a.bits == 8 ? (a.master ? launch_with<8, true> : launch_with<8, false>)
                                      : (a.master ? launch_with<32, true> : launch_with<32, false>);
      launch(a, g, t0, first_chunk[t0], chunks, last, s);
    }
    if (last) break;
  }
}

}  // namespace arb
