// Lookup of table rows by token with scaling, its gradient by sorted tokens, and the sort itself.
//
//   out[b, :] = round(scale * sum_t table[tok[b, t], :])
//   dtable[v, :] = round(scale * sum_{(b, t): tok[b, t] = v} grad[b, :])
//
// Sums are held in fp32 and rounded once to the output's type.  No floating-point atomics: the
// gradient of a row is summed by its owner over the sorted tokens, in an order that only the tokens
// decide, so two calls on the same tokens give the same bits.
#include <algorithm>

#include "operators.h"
#include "vec.cuh"

namespace arb {

namespace {

template <typename I>
__device__ __forceinline__ long long token_at(const TokenView &t, long long b, long long k) {
  return (long long)(static_cast<const I *>(t.at)[b * t.bag_stride + k * t.token_stride]);
}

template <typename T, typename O, typename I>
__global__ void lookup_kernel(LookupLaunch a) {
  const long long total = a.tokens.bags * a.dim;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long b = i / a.dim, d = i - b * a.dim;
    float sum = 0.0f;
    for (long long k = 0; k < a.tokens.per_bag; ++k) {
      const long long tok = token_at<I>(a.tokens, b, k);
      if (tok >= 0 && tok < a.rows) sum += to_f32(static_cast<const T *>(a.table)[tok * a.row_stride + d]);
    }
    from_f32(sum * a.scale, static_cast<O *>(a.out)[b * a.out_stride + d]);
  }
}

// ---- the sort --------------------------------------------------------------------------------
// Least-significant-digit radix sort of (token, bag): every pass counts the digits of each tile,
// turns the counts into positions (digit by digit, tile by tile) and moves the pairs, keeping the
// order of equal digits.  An empty slot sorts as token `rows`, behind everything.
constexpr int kDigitBits = 8, kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 256, kSortItems = 16, kTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32;

struct SortPass {
  TokenView tokens;        // first pass: where keys come from
  long long rows;
  const unsigned *key_in, *bag_in;  // later passes
  unsigned *key_out, *bag_out;
  unsigned *counts;        // [digit][tile]
  unsigned *totals;        // [digit]
  long long n;
  int tiles, shift;
  bool first, by_slot;     // by_slot: pairs are numbered slot after slot (neighbouring bags lie side by side)
};

template <typename I>
__device__ __forceinline__ void sort_pair(const SortPass &p, long long i, unsigned &key, unsigned &bag) {
  if (!p.first) {
    key = p.key_in[i];
    bag = p.bag_in[i];
    return;
  }
  const long long b = p.by_slot ? i % p.tokens.bags : i / p.tokens.per_bag;
  const long long k = p.by_slot ? i / p.tokens.bags : i - b * p.tokens.per_bag;
  const long long tok = token_at<I>(p.tokens, b, k);
  key = tok >= 0 && tok < p.rows ? unsigned(tok) : unsigned(p.rows);
  bag = unsigned(b);
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortPass p) {
  __shared__ unsigned cnt[kDigits];
  for (int i = threadIdx.x; i < kDigits; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
  const long long t0 = blockIdx.x * (long long)kTile;
  for (int j = 0; j < kSortItems; ++j) {
    const long long i = t0 + j * kSortThreads + threadIdx.x;
    if (i < p.n) {
      unsigned key, bag;
      sort_pair<I>(p, i, key, bag);
      atomicAdd(&cnt[(key >> p.shift) & (kDigits - 1)], 1u);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kDigits; i += kSortThreads) p.counts[size_t(i) * p.tiles + blockIdx.x] = cnt[i];
}

// exclusive sum over a CTA's 256 threads
__device__ __forceinline__ unsigned block_exclusive(unsigned v, unsigned *total) {
  __shared__ unsigned warp_sum[8];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  unsigned x = v;
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sum[w] = x;
  __syncthreads();
  unsigned before = 0, all = 0;
  for (int i = 0; i < 8; ++i) {
    if (i < w) before += warp_sum[i];
    all += warp_sum[i];
  }
  __syncthreads();
  *total = all;
  return before + x - v;
}

// one CTA a digit: its counts become exclusive sums over the tiles
__global__ void __launch_bounds__(256) sort_scan_kernel(SortPass p) {
  unsigned *row = p.counts + size_t(blockIdx.x) * p.tiles;
  unsigned run = 0;
  for (int t = 0; t < p.tiles; t += 256) {
    const int i = t + int(threadIdx.x);
    const unsigned v = i < p.tiles ? row[i] : 0u;
    unsigned all;
    const unsigned before = block_exclusive(v, &all);
    if (i < p.tiles) row[i] = run + before;
    run += all;
  }
  if (threadIdx.x == 0) p.totals[blockIdx.x] = run;
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(SortPass p) {
  __shared__ unsigned warp_cnt[kSortWarps][kDigits];
  __shared__ unsigned base[kDigits];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&warp_cnt[0][0])[i] = 0;
  {
    unsigned all;
    const unsigned before = block_exclusive(p.totals[threadIdx.x], &all);
    base[threadIdx.x] = before + p.counts[size_t(threadIdx.x) * p.tiles + blockIdx.x];
  }
  __syncthreads();
  // a warp owns kSortItems * 32 neighbouring pairs; equal digits keep their order
  const long long w0 = blockIdx.x * (long long)kTile + w * (kSortItems * 32);
  unsigned key[kSortItems], bag[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const long long i = w0 + j * 32 + lane;
    const bool in = i < p.n;
    key[j] = bag[j] = rank[j] = 0;
    if (in) sort_pair<I>(p, i, key[j], bag[j]);
    const unsigned digit = in ? (key[j] >> p.shift) & (kDigits - 1) : kDigits;
    const unsigned same = __match_any_sync(0xffffffffu, digit);
    const unsigned below = __popc(same & ((1u << lane) - 1u));
    if (in) rank[j] = warp_cnt[w][digit] + below;
    __syncwarp();
    if (in && below == 0) warp_cnt[w][digit] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  {
    unsigned run = 0;
    for (int i = 0; i < kSortWarps; ++i) {
      const unsigned c = warp_cnt[i][threadIdx.x];
      warp_cnt[i][threadIdx.x] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const long long i = w0 + j * 32 + lane;
    if (i < p.n) {
      const unsigned digit = (key[j] >> p.shift) & (kDigits - 1);
      const unsigned to = base[digit] + warp_cnt[w][digit] + rank[j];
      p.key_out[to] = key[j];
      p.bag_out[to] = bag[j];
    }
  }
}

// begin[v] = first position of a token >= v: position p fills the rows behind its predecessor's
// token up to its own; a warp fills the gaps of its 32 positions together
__global__ void order_begin_kernel(const unsigned *__restrict__ key, long long n, long long rows,
                                   unsigned *__restrict__ begin) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * blockDim.x / 32;
  for (long long w = (blockIdx.x * (long long)blockDim.x + threadIdx.x) / 32; w * 32 <= n; w += warps) {
    const long long p = w * 32 + lane;
    long long lo = 0, hi = -1;  // rows this position fills
    if (p <= n) {
      lo = p == 0 ? 0 : (long long)key[p - 1] + 1;
      hi = p == n ? rows : (long long)key[p];
    }
    unsigned todo = __ballot_sync(0xffffffffu, lo <= hi);
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      const long long l = __shfl_sync(0xffffffffu, lo, src), h = __shfl_sync(0xffffffffu, hi, src);
      for (long long v = l + lane; v <= h; v += 32) begin[v] = unsigned(w * 32 + src);
    }
  }
}

// ---- the gradient ----------------------------------------------------------------------------
template <typename T, typename O>
__global__ void lookup_grad_kernel(LookupGradLaunch a, const unsigned *__restrict__ bag,
                                   const unsigned *__restrict__ begin, long long rows) {
  const long long total = rows * a.dim;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long v = i / a.dim, d = i - v * a.dim;
    const unsigned p0 = begin[v], p1 = begin[v + 1];
    O *o = static_cast<O *>(a.out) + v * a.out_stride + d;
    if (a.accumulate && p0 == p1) continue;
    float sum = 0.0f;
    for (unsigned p = p0; p < p1; ++p)
      sum += to_f32(static_cast<const T *>(a.grad)[(long long)bag[p] * a.grad_stride + d]);
    sum *= a.scale;
    if (a.accumulate) sum += to_f32(*o);
    from_f32(sum, *o);
  }
}

inline int grid_of(long long n, int threads, int per_sm) {
  return int(std::max<long long>(1, std::min<long long>((n + threads - 1) / threads, (long long)device_sm_count() * per_sm)));
}

int key_bits(int64_t rows) {  // keys are 0 .. rows
  int b = 1;
  while ((uint64_t(rows) >> b) != 0) ++b;
  return b;
}

// scratch of the sort: two buffers of pairs, the digit counts
struct SortScratch {
  unsigned *key[2], *bag[2], *counts, *totals;
  size_t bytes;
  SortScratch(void *mem, int64_t n, int64_t rows) {
    (void)rows;
    const size_t pair = (size_t(n) * 4 + 255) / 256 * 256;
    const size_t tiles = size_t((n + kTile - 1) / kTile);
    char *p = static_cast<char *>(mem);
    size_t at = 0;
    auto take = [&](size_t b) {
      char *q = p + at;
      at += (b + 255) / 256 * 256;
      return reinterpret_cast<unsigned *>(q);
    };
    key[0] = take(pair), key[1] = take(pair), bag[0] = take(pair), bag[1] = take(pair);
    counts = take(tiles * kDigits * 4);
    totals = take(kDigits * 4);
    bytes = at;
  }
};

}  // namespace

#define ARB_BY_TYPE(type, out_type, CALL)                                            \
  do {                                                                               \
    if ((type) == kF32 && (out_type) == kF32) { CALL(float, float); }                \
    else if ((type) == kBF16 && (out_type) == kBF16) { CALL(__nv_bfloat16, __nv_bfloat16); } \
    else if ((type) == kBF16 && (out_type) == kF32) { CALL(__nv_bfloat16, float); }  \
    else if ((type) == kF16 && (out_type) == kF16) { CALL(__half, __half); }         \
    else if ((type) == kF16 && (out_type) == kF32) { CALL(__half, float); }          \
    else throw std::runtime_error("the output has the input's type or fp32");        \
  } while (0)

void launch_lookup(const LookupLaunch &a, cudaStream_t s) {
  if (a.tokens.bags == 0 || a.dim == 0) return;
  const int threads = 256, grid = grid_of(a.tokens.bags * a.dim, threads, 16);
#define ARB_CALL(T, O)                                                                      \
  if (a.tokens.bytes == 4) lookup_kernel<T, O, int32_t><<<grid, threads, 0, s>>>(a);        \
  else lookup_kernel<T, O, int64_t><<<grid, threads, 0, s>>>(a)
  ARB_BY_TYPE(a.type, a.out_type, ARB_CALL);
#undef ARB_CALL
  ARB_CUDA(cudaGetLastError());
  count_launch();
}

size_t TokenOrder::bytes(int64_t count, int64_t rows) {
  return (size_t(count) * 4 + 255) / 256 * 256 + (size_t(rows + 1) * 4 + 255) / 256 * 256;
}
TokenOrder::TokenOrder(void *mem, int64_t count_, int64_t rows_) : count(count_), rows(rows_) {
  bag = static_cast<unsigned *>(mem);
  begin = reinterpret_cast<unsigned *>(static_cast<char *>(mem) + (size_t(count) * 4 + 255) / 256 * 256);
}

size_t token_order_scratch(int64_t count, int64_t rows) { return SortScratch(nullptr, count, rows).bytes; }

void launch_token_order(const TokenView &t, const TokenOrder &o, void *scratch, cudaStream_t s) {
  const int64_t n = t.count();
  const SortScratch sc(scratch, n, o.rows);
  const int passes = (key_bits(o.rows) + kDigitBits - 1) / kDigitBits;
  SortPass p;
  p.tokens = t;
  p.rows = o.rows;
  p.n = n;
  p.tiles = int((n + kTile - 1) / kTile);
  p.counts = sc.counts;
  p.totals = sc.totals;
  p.by_slot = t.bag_stride < t.token_stride;
  for (int i = 0; i < passes && n > 0; ++i) {
    p.first = i == 0;
    p.shift = i * kDigitBits;
    p.key_in = sc.key[(i + 1) & 1];
    p.bag_in = sc.bag[(i + 1) & 1];
    p.key_out = sc.key[i & 1];
    p.bag_out = i == passes - 1 ? o.bag : sc.bag[i & 1];
    if (t.bytes == 4) sort_count_kernel<int32_t><<<p.tiles, kSortThreads, 0, s>>>(p);
    else sort_count_kernel<int64_t><<<p.tiles, kSortThreads, 0, s>>>(p);
    sort_scan_kernel<<<kDigits, 256, 0, s>>>(p);
    if (t.bytes == 4) sort_move_kernel<int32_t><<<p.tiles, kSortThreads, 0, s>>>(p);
    else sort_move_kernel<int64_t><<<p.tiles, kSortThreads, 0, s>>>(p);
    ARB_CUDA(cudaGetLastError());
    count_launch(3);
  }
  order_begin_kernel<<<grid_of(n + 1, 256, 8), 256, 0, s>>>(sc.key[(passes - 1) & 1], n, o.rows, o.begin);
  ARB_CUDA(cudaGetLastError());
  count_launch();
}

size_t lookup_grad_scratch(int64_t, int64_t, int64_t) { return 0; }

void launch_lookup_grad(const LookupGradLaunch &a, const TokenOrder &o, void *, cudaStream_t s) {
  if (o.rows == 0 || a.dim == 0) return;
  const int threads = 256, grid = grid_of(o.rows * a.dim, threads, 16);
#define ARB_CALL(T, O) lookup_grad_kernel<T, O><<<grid, threads, 0, s>>>(a, o.bag, o.begin, o.rows)
  ARB_BY_TYPE(a.type, a.out_type, ARB_CALL);
#undef ARB_CALL
  ARB_CUDA(cudaGetLastError());
  count_launch();
}

}  // namespace arb
