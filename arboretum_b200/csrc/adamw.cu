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
#include "root.cuh"
#include "vec.cuh"

namespace arb {

namespace {

// Gradient addresses of one launch, kernel parameters: 16 KB of them at most, 512 bytes for few tensors.
constexpr int kMaxGrads = 2048, kFewGrads = 64, kSomeGrads = 512;
template <int N>
struct GradPointers {
  const void *at[N];
};

// 32 bits for an element, by the mixing of the boosting gradients' dither:
//   x = index ^ step, seed, upper half of index;  x ^= x >> 16;  x *= A;  x ^= x >> 15;  x *= B;  x ^= x >> 16
// The first fold is the same for the eight elements of a thread, whose indices differ in three bits; the
// last one leaves the upper half as it is.
__device__ __forceinline__ unsigned hash_key(unsigned long long index, unsigned step, unsigned seed) {
  const unsigned x = unsigned(index) ^ (unsigned(index >> 32) * 0x9E3779B1u) ^ (step * 0x85EBCA6Bu) ^ (seed * 0xC2B2AE35u);
  return x ^ (x >> 16);
}
__device__ __forceinline__ unsigned hash_before_last(unsigned x) {  // x: key ^ element
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  return x * 0x846CA68Bu;
}

// two e4m3 codes as floats
__device__ __forceinline__ float2 decode2(unsigned codes) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3)));
}
// x = |value| / scale * 2^-120: there e4m3's exponents are float's smallest, so a code is the seven bits
// from 20 on, and the dither is added to the 20 bits that go.  `random` holds 16 bits, shifted up by four.
constexpr unsigned kCodeOne = 1u << 20, kCodeMost = (126u << 20) | 0xFFFFFu;
__device__ __forceinline__ unsigned dithered(float x, unsigned random) { return min(__float_as_uint(x) + random + 8u, kCodeMost); }
// the upper bytes of four words
__device__ __forceinline__ unsigned upper_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
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
  float beta1, one_beta1, beta2, one_beta2, inv_root_bc2, step_size, keep, eps, grad_scale, one;
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
  c.one = a.state->one;
  c.step = unsigned(a.state->step + 1);
  return c;
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

template <int BITS>
constexpr int kThreads = BITS == 8 ? 128 : 256;
constexpr int kEach = 8;                      // neighbouring elements of a thread
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
  static constexpr int kPairs = kEach / 2;
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
    float gr[kEach], pr[kEach];
    float2 m[kPairs], v[kPairs];
    g.get(gr);
    w.get(pr);
    if constexpr (BITS == 32) {
      float x[kEach];
      m32.get(x);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) m[j] = make_float2(x[2 * j], x[2 * j + 1]);
      v32.get(x);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[j] = make_float2(x[2 * j], x[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        m[j] = mul2(decode2((j < 2 ? cm.x : cm.y) >> (j % 2 * 16) & 0xFFFFu), both(s1));
        const float2 r = mul2(decode2((j < 2 ? cr.x : cr.y) >> (j % 2 * 16) & 0xFFFFu), both(s2));
        v[j] = mul2(r, r);
      }
    }
    unsigned largest = 0, smallest = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 gj = mul2(make_float2(gr[2 * j], gr[2 * j + 1]), both(c.grad_scale));
      m[j] = add2(mul2(m[j], both(c.beta1)), mul2(gj, both(c.one_beta1)), c.one);
      v[j] = add2(mul2(v[j], both(c.beta2)), mul2(mul2(gj, gj), both(c.one_beta2)), c.one);
      largest = max(max(largest, __float_as_uint(v[j].x)), __float_as_uint(v[j].y));
      smallest = min(min(smallest, __float_as_uint(v[j].x)), __float_as_uint(v[j].y));
    }
    const bool plain = root_is_plain(largest, smallest);
    float im = 0.0f, ir = 0.0f;
    bool one = true;
    if constexpr (BITS == 8) {
      float top_m = 0.0f;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) top_m = larger(larger(top_m, fabsf(m[j].x)), fabsf(m[j].y));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        top_m = larger(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));  // v >= 0: its bits are in its order
      }
      const float top_r = sqrtf(__uint_as_float(largest));  // the largest root is the root of the largest
      const unsigned fm = scale_field(__float_as_uint(top_m) & 0x7FFFFFFFu), fr = scale_field(__float_as_uint(top_r) & 0x7FFFFFFFu);
      if (threadIdx.x % kLanes == 0 && left > 0) {
        a.scale1[at / kMomentBlock] = scale_of(fm);
        a.scale2[at / kMomentBlock] = scale_of(fr);
      }
      // The scale's inverse and e4m3's shift of 2^-120 are one factor unless it would fall below float's
      // smallest normal number (moments beyond 448 * 64): then the second factor follows.
      one = fm <= 133u && fr <= 133u;
      im = one ? __uint_as_float((134u - fm) << 23) : inv_scale_of(fm);
      ir = one ? __uint_as_float((134u - fr) << 23) : inv_scale_of(fr);
    }
    if (left <= 0) return;
    // zeros and very small or large second moments take a path of their own: it is the same step
    if (plain) finish<true>(a, c, param, at, left, vec, pr, m, v, im, ir, one);
    else finish<false>(a, c, param, at, left, vec, pr, m, v, im, ir, one);
  }

  // from the moments on; PLAIN: all second moments are in [2^-100, 2^126]
  template <bool PLAIN>
  __device__ __forceinline__ void finish(const AdamWLaunch &a, const Scalars &c, P *param, long long at, int left, bool vec,
                                         float (&pr)[kEach], const float2 (&m)[kPairs], const float2 (&v)[kPairs],
                                         float im, float ir, bool one) const {
    float2 p[kPairs], root[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) root[j] = PLAIN ? root_of(v[j]) : make_float2(sqrtf(v[j].x), sqrtf(v[j].y));
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 below = add2(mul2(root[j], both(c.inv_root_bc2)), both(c.eps), c.one);
      const float2 part = mul2(make_float2(quotient(m[j].x, below.x), quotient(m[j].y, below.y)), both(-c.step_size));
      p[j] = add2(mul2(make_float2(pr[2 * j], pr[2 * j + 1]), both(c.keep)), part, c.one);
    }
    const auto flat = [](const float2 (&x)[kPairs], float (&y)[kEach]) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) y[2 * j] = x[j].x, y[2 * j + 1] = x[j].y;
    };
    const bool full = left >= kEach;
    flat(p, pr);
    store_each(param, pr, left, full && vec);
    if constexpr (MASTER) store_each(a.master + at, pr, left, full);
    if constexpr (BITS == 32) {
      float x[kEach];
      flat(m, x);
      store_each(static_cast<float *>(a.moment1) + at, x, left, full);
      flat(v, x);
      store_each(static_cast<float *>(a.moment2) + at, x, left, full);
    } else {
      unsigned em[kEach], er[kEach];
      const unsigned key = hash_key((unsigned long long)at, c.step, a.seed);  // at is a multiple of eight
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const float2 mj = m[j / 2], rj = root[j / 2];
        const float mx = j % 2 ? mj.y : mj.x, rx = j % 2 ? rj.y : rj.x;
        float ym = fabsf(mx) * im, yr = rx * ir;
        if (!one) ym *= 0x1p-120f, yr *= 0x1p-120f;
        const unsigned h = hash_before_last(key ^ unsigned(j)), upper = h >> 12;
        // the code in the upper byte, below the sign; a root above zero stays above zero
        em[j] = dithered(ym, ((h << 4) ^ upper) & 0xFFFF0u) << 4 | (__float_as_uint(mx) & 0x80000000u);
        er[j] = max(dithered(yr, upper & 0xFFFF0u), PLAIN ? kCodeOne : min(__float_as_uint(rx), kCodeOne)) << 4;
      }
      *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(a.moment1) + at) =
          make_uint2(upper_bytes(em[0], em[1], em[2], em[3]), upper_bytes(em[4], em[5], em[6], em[7]));
      *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(a.moment2) + at) =
          make_uint2(upper_bytes(er[0], er[1], er[2], er[3]), upper_bytes(er[4], er[5], er[6], er[7]));
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
  const int n = int(min(t.n - first, (long long)a.chunk));
  // a thread behind the end (n - i <= 0) loads and stores nothing, but takes part in the shuffles
  constexpr int kTileElems = kThreads<BITS> * kEach;  // elements of a CTA at a time
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kTileElems) {
    const int i = i0 + threadIdx.x * kEach;
    Tile<BITS, P, G, MASTER> tile;
    tile.load(a, param + i, grad + i, slot + i, n - i, vec, grad_vec);
    tile.step(a, c, param + i, slot + i, n - i, vec);
  }
}

// Many small CTAs: with moments in 8 bits the step issues 69 instructions an element, three quarters of the
// time, and waits for a tile's loads the rest; it wants as many warps as 40 registers allow: one bf16
// tensor of 128 M elements takes 309 us with 12 CTAs of 128 threads an SM, 354 with 5 of 256.  Moments in
// 32 bits are bound by memory: 64 M elements with a copy take 279 us.
template <int BITS, bool MASTER, int N>
__global__ void __launch_bounds__(kThreads<BITS>, BITS == 8 ? 12 : 4) adamw_kernel(AdamWLaunch a, const __grid_constant__ GradPointers<N> grads,
                                                            int first_tensor, int first_chunk, int n_chunks, bool last) {
  __shared__ Scalars shared_scalars;
  if (threadIdx.x == 0) shared_scalars = scalars_of(a);
  const AdamWChunk ch = int(blockIdx.x) < n_chunks ? a.chunks[first_chunk + blockIdx.x] : AdamWChunk{-1, 0};
  __syncthreads();
  const Scalars c = shared_scalars;
  const void *grad = ch.tensor < 0 ? nullptr : grads.at[ch.tensor - first_tensor];
  if (grad != nullptr) {
    const AdamWTensor t = a.tensors[ch.tensor];
    const long long first = (long long)ch.index * a.chunk;
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
template <int BITS, bool MASTER, int N>
void launch_with(const AdamWLaunch &a, const void *const *grads, int n, int first_tensor, int first_chunk, int chunks, bool last,
                 cudaStream_t s) {
  GradPointers<N> g;
  std::copy(grads, grads + n, g.at);
  adamw_kernel<BITS, MASTER, N><<<std::max(1, chunks), kThreads<BITS>, 0, s>>>(a, g, first_tensor, first_chunk, chunks, last);
  ARB_CUDA(cudaGetLastError());
  count_launch();
}
template <int N, typename... Args>
void launch_variant(const AdamWLaunch &a, Args... args) {
  if (a.bits == 8 && a.master) launch_with<8, true, N>(a, args...);
  else if (a.bits == 8) launch_with<8, false, N>(a, args...);
  else if (a.master) launch_with<32, true, N>(a, args...);
  else launch_with<32, false, N>(a, args...);
}
}  // namespace

void launch_adamw(const AdamWLaunch &a, const void *const *grads, const std::vector<int> &first_chunk,
                  int n_tensors, cudaStream_t s) {
  for (int t0 = 0;; t0 += kMaxGrads) {
    const int t1 = std::min(n_tensors, t0 + kMaxGrads), n = t1 - t0;
    const bool last = t1 == n_tensors;
    const int chunks = first_chunk[t1] - first_chunk[t0];
    if (chunks > 0 || last) {  // a step without elements still counts
      if (n <= kFewGrads) launch_variant<kFewGrads>(a, grads + t0, n, t0, first_chunk[t0], chunks, last, s);
      else if (n <= kSomeGrads) launch_variant<kSomeGrads>(a, grads + t0, n, t0, first_chunk[t0], chunks, last, s);
      else launch_variant<kMaxGrads>(a, grads + t0, n, t0, first_chunk[t0], chunks, last, s);
    }
    if (last) break;
  }
}

}  // namespace arb
