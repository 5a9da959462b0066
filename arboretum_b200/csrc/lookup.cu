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
// row of a token, or -1 for an empty slot
__device__ __forceinline__ long long row_at(const TokenView &t, long long rows, long long b, long long k) {
  const long long tok = t.bytes == 4 ? token_at<int32_t>(t, b, k) : token_at<int64_t>(t, b, k);
  return tok >= 0 && tok < rows ? tok : -1;
}

// How the threads of a CTA share the work: a group of tx lanes across the columns and ly lanes
// along the tokens of a bag makes a unit's sums (tx and ly powers of two).
struct LaneShape {
  int tx_bits, ly_bits;
};

// A unit is a bag and a run of tx * U vectors of VEC columns.  Memory bound: the rows are read once
// and the result written once; a thread issues the loads of U column vectors and of K tokens before
// it adds the first, so that enough bytes are in flight.  With few bags the tokens of a bag are
// split over ly lanes, which join their sums through shared memory in a fixed order.
constexpr int kLookupThreads = 256;
template <typename T, typename O, int VEC, int U, int K>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(LookupLaunch a, LaneShape sh, int vecs, int chunks) {
  __shared__ float part[K > 1 ? kLookupThreads * U * VEC : 1];  // one token a bag: nothing to join
  const int tx = 1 << sh.tx_bits, ly = 1 << sh.ly_bits;
  const int lane = threadIdx.x & (tx - 1), slice = (threadIdx.x >> sh.tx_bits) & (ly - 1);
  const int group = threadIdx.x >> (sh.tx_bits + sh.ly_bits), groups = kLookupThreads >> (sh.tx_bits + sh.ly_bits);
  const T *table = static_cast<const T *>(a.table);
  const long long b = blockIdx.x * (long long)groups + group;
  for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
    const int c0 = chunk * (tx * U) + lane;
    float sum[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[u][j] = 0.0f;
    if (b < a.tokens.bags) {
      for (long long k0 = slice; k0 < a.tokens.per_bag; k0 += ly * K) {
        long long row[K];
#pragma unroll
        for (int k = 0; k < K; ++k) row[k] = k0 + k * ly < a.tokens.per_bag ? row_at(a.tokens, a.rows, b, k0 + k * ly) : -1;
        float v[K][U][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (row[k] >= 0 && c0 + u * tx < vecs) {
              load_vec<T, VEC>(table + row[k] * a.row_stride + (long long)(c0 + u * tx) * VEC, v[k][u]);
            } else {
#pragma unroll
              for (int j = 0; j < VEC; ++j) v[k][u][j] = 0.0f;
            }
          }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum[u][j] += v[k][u][j];
      }
    }
    if (K > 1 && ly > 1) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[(u * VEC + j) * kLookupThreads + threadIdx.x] = sum[u][j];
      for (int half = ly >> 1; half > 0; half >>= 1) {
        __syncthreads();
        if (slice < half) {
#pragma unroll
          for (int i = 0; i < U * VEC; ++i)
            part[i * kLookupThreads + threadIdx.x] += part[i * kLookupThreads + threadIdx.x + half * tx];
        }
      }
      if (slice != 0) continue;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[u][j] = part[(u * VEC + j) * kLookupThreads + threadIdx.x];
    }
    if (b < a.tokens.bags) {
      O *out = static_cast<O *>(a.out) + b * a.out_stride;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + u * tx < vecs) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) sum[u][j] *= a.scale;
          store_vec<O, VEC>(out + (long long)(c0 + u * tx) * VEC, sum[u]);
        }
      }
    }
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

// ---- rows named by many bags -----------------------------------------------------------------
// A row named by more than `piece` bags is cut into pieces of that many, so that the sum of a
// frequent token is shared by many warps.  Which slot a row's pieces get depends on the order of
// arrival here; no value does: a row's pieces are joined in their own order.
__device__ __forceinline__ void add_frequent(const TokenOrder &o, unsigned row, unsigned len) {
  const unsigned pieces = (len + o.piece - 1) / o.piece;
  const unsigned long long at = atomicAdd(o.counts, (1ull << 32) | pieces);
  o.frequent[at >> 32] = make_uint2(row, unsigned(at));  // ascending in the first piece's number
}

__global__ void order_plan_kernel(TokenOrder o) {
  for (long long v = blockIdx.x * (long long)blockDim.x + threadIdx.x; v < o.rows; v += (long long)gridDim.x * blockDim.x) {
    const unsigned len = o.begin[v + 1] - o.begin[v];
    if (len > o.piece) add_frequent(o, unsigned(v), len);
  }
}

// ---- the gradient ----------------------------------------------------------------------------
struct GradLanes {
  int tx_bits;      // lanes across the columns
  int ly_row_bits;  // lanes along the bags of a row
  int ly_item_bits; // ... of a piece of a frequent row
};

constexpr int kGradThreads = 256;

// sum over positions p0 + slice, p0 + slice + ly, .. below p1 of the gradient rows they name
template <typename T, int VEC, int U>
__device__ __forceinline__ void sum_bags(const LookupGradLaunch &a, const unsigned *__restrict__ bag, unsigned p0, unsigned p1,
                                         int slice, int ly, int tx, int c0, int vecs, float (&sum)[U][VEC]) {
  constexpr int K = U * VEC >= 16 ? 2 : 4;  // bags whose loads are in flight together
  const T *grad = static_cast<const T *>(a.grad);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[u][j] = 0.0f;
  for (unsigned p = p0 + slice; p < p1; p += ly * K) {
    long long row[K];
#pragma unroll
    for (int k = 0; k < K; ++k) row[k] = p + k * ly < p1 ? (long long)bag[p + k * ly] * a.grad_stride : -1;
    float v[K][U][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row[k] >= 0 && c0 + u * tx < vecs) {
          load_vec<T, VEC>(grad + row[k] + (long long)(c0 + u * tx) * VEC, v[k][u]);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[k][u][j] = 0.0f;
        }
      }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[u][j] += v[k][u][j];
  }
  for (int o = tx; o < tx * ly; o <<= 1)  // the slices of a group are neighbouring lanes of a warp
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[u][j] += __shfl_xor_sync(0xffffffffu, sum[u][j], o);
}

template <typename O, int VEC, int U>
__device__ __forceinline__ void write_row(const LookupGradLaunch &a, long long row, int c0, int tx, int vecs,
                                          float (&sum)[U][VEC]) {
  O *out = static_cast<O *>(a.out) + row * a.out_stride;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (c0 + u * tx < vecs) {
      O *at = out + (long long)(c0 + u * tx) * VEC;
      if (a.accumulate) {
        float old[VEC];
        load_vec<O, VEC>(at, old);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[u][j] = sum[u][j] * a.scale + old[j];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[u][j] *= a.scale;
      }
      store_vec<O, VEC>(at, sum[u]);
    }
  }
}

// CTAs below item_blocks sum the pieces of frequent rows into `partial` [piece][dim]; the others
// take the rows of the table in order: zeros where no bag names a row, else its sum.  (The sums
// behind the loops are uniform over a warp: lanes without a row of their own go through them empty.)
template <typename T, typename O, int VEC, int U>
__global__ void __launch_bounds__(kGradThreads) lookup_grad_kernel(LookupGradLaunch a, TokenOrder o, GradLanes sh, int vecs,
                                                                   int chunks, unsigned item_blocks, float *partial) {
  const int tx = 1 << sh.tx_bits, lane = threadIdx.x & (tx - 1);
  if (blockIdx.x < item_blocks) {
    const int ly = 1 << sh.ly_item_bits, slice = (threadIdx.x >> sh.tx_bits) & (ly - 1);
    const int bits = sh.tx_bits + sh.ly_item_bits;
    const unsigned group = threadIdx.x >> bits, groups = kGradThreads >> bits;
    const unsigned long long counts = *o.counts;
    const unsigned items = unsigned(counts), n_frequent = unsigned(counts >> 32);
    for (unsigned i0 = blockIdx.x * groups; i0 < items; i0 += item_blocks * groups) {
      const unsigned i = i0 + group;
      unsigned p0 = 0, p1 = 0;
      if (i < items) {  // the last frequent row whose pieces start at or below i
        unsigned lo = 0, hi = n_frequent;
        while (hi - lo > 1) {
          const unsigned mid = (lo + hi) / 2;
          if (o.frequent[mid].y <= i) lo = mid;
          else hi = mid;
        }
        const uint2 f = o.frequent[lo];
        const unsigned end = o.begin[f.x + 1];
        p0 = o.begin[f.x] + (i - f.y) * o.piece;
        p1 = end - p0 > o.piece ? p0 + o.piece : end;
      }
      for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
        const int c0 = chunk * (tx * U) + lane;
        float sum[U][VEC];
        sum_bags<T, VEC, U>(a, o.bag, p0, p1, slice, ly, tx, c0, vecs, sum);
        if (slice == 0 && i < items) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + u * tx < vecs) {
#pragma unroll
              for (int j = 0; j < VEC; ++j) partial[(size_t(i) * vecs + (c0 + u * tx)) * VEC + j] = sum[u][j];
            }
        }
      }
    }
    return;
  }
  const int ly = 1 << sh.ly_row_bits, slice = (threadIdx.x >> sh.tx_bits) & (ly - 1);
  const int bits = sh.tx_bits + sh.ly_row_bits;
  const long long row = (blockIdx.x - item_blocks) * (long long)(kGradThreads >> bits) + (threadIdx.x >> bits);
  unsigned p0 = 0, p1 = 0;
  if (row < o.rows) p0 = o.begin[row], p1 = o.begin[row + 1];
  const bool mine = row < o.rows && p1 - p0 <= o.piece && !(a.accumulate && p0 == p1);
  if (!mine) p1 = p0;
  for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
    const int c0 = chunk * (tx * U) + lane;
    float sum[U][VEC];
    sum_bags<T, VEC, U>(a, o.bag, p0, p1, slice, ly, tx, c0, vecs, sum);
    if (mine && slice == 0) write_row<O, VEC, U>(a, row, c0, tx, vecs, sum);
  }
}

// the pieces of a frequent row, joined in their order
template <typename O, int VEC>
__global__ void __launch_bounds__(kGradThreads) lookup_grad_join_kernel(LookupGradLaunch a, TokenOrder o, int vecs,
                                                                        const float *__restrict__ partial) {
  const unsigned n_frequent = unsigned(*o.counts >> 32);
  for (unsigned h = blockIdx.x; h < n_frequent; h += gridDim.x) {
    const uint2 f = o.frequent[h];
    const unsigned pieces = (o.begin[f.x + 1] - o.begin[f.x] + o.piece - 1) / o.piece;
    for (int c = blockIdx.y * kGradThreads + threadIdx.x; c < vecs; c += gridDim.y * kGradThreads) {
      float sum[1][VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[0][j] = 0.0f;
#pragma unroll 4
      for (unsigned k = 0; k < pieces; ++k) {
        const float *at = partial + (size_t(f.y + k) * vecs + c) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[0][j] += at[j];
      }
      write_row<O, VEC, 1>(a, f.x, c, 0, vecs, sum);
    }
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

namespace {

int log2_floor(int64_t v) {
  int b = 0;
  while ((v >> (b + 1)) > 0) ++b;
  return b;
}

// Elements a thread may move in one access: the widest of 16 bytes, 4 bytes and one element that
// the columns, the distances of the rows and both starts allow.
int vec_of(int type, int64_t dim, const void *p, int64_t stride, const void *q, int out_type, int64_t out_stride) {
  const int widths[2] = {int(16 / elem_size(type)), int(4 / elem_size(type))};
  for (int v : widths) {
    const auto fits = [&](const void *at, int t, int64_t st) {
      const size_t bytes = std::min<size_t>(16, v * elem_size(t));
      return reinterpret_cast<uintptr_t>(at) % bytes == 0 && size_t(st) * elem_size(t) % bytes == 0;
    };
    if (v > 1 && dim % v == 0 && fits(p, type, stride) && fits(q, out_type, out_stride)) return v;
  }
  return 1;
}

template <typename T, typename O, int VEC>
void lookup_with(const LookupLaunch &a, cudaStream_t s) {
  const int64_t vecs = a.dim / VEC;
  ARB_CHECK(vecs <= (int64_t(1) << 30), "rows of more than 2^30 vectors");
  const bool pooled = a.tokens.per_bag > 1;
  const int u = !pooled && vecs >= 256 ? 4 : 1;
  LaneShape sh;
  // lanes across the columns: enough for the row, at most a CTA
  sh.tx_bits = std::min(7, log2_floor(std::max<int64_t>(1, (vecs + u - 1) / u * 2 - 1)));
  // lanes along the tokens: where a bag's tokens lie side by side a narrow group reads them as one
  // line, and where the bags alone do not fill the device they share the loop
  const int64_t threads_wanted = int64_t(device_sm_count()) * 1024;
  int64_t have = a.tokens.bags * ((vecs + u - 1) / u);
  const bool side_by_side = std::abs(a.tokens.token_stride) < std::abs(a.tokens.bag_stride);
  sh.ly_bits = 0;
  while (pooled && sh.tx_bits + sh.ly_bits < 8 && (int64_t(4) << sh.ly_bits) < a.tokens.per_bag &&
         ((have << sh.ly_bits) < threads_wanted || (side_by_side && sh.tx_bits + sh.ly_bits < 3)))
    ++sh.ly_bits;
  const int groups = kLookupThreads >> (sh.tx_bits + sh.ly_bits);
  const int chunks = int((vecs + (int64_t(u) << sh.tx_bits) - 1) / (int64_t(u) << sh.tx_bits));
  const dim3 grid(unsigned((a.tokens.bags + groups - 1) / groups), unsigned(std::min(chunks, 65535)));
  if (pooled) lookup_kernel<T, O, VEC, 1, 4><<<grid, kLookupThreads, 0, s>>>(a, sh, int(vecs), chunks);
  else if (u == 4) lookup_kernel<T, O, VEC, 4, 1><<<grid, kLookupThreads, 0, s>>>(a, sh, int(vecs), chunks);
  else lookup_kernel<T, O, VEC, 1, 1><<<grid, kLookupThreads, 0, s>>>(a, sh, int(vecs), chunks);
}

}  // namespace

void launch_lookup(const LookupLaunch &a, cudaStream_t s) {
  if (a.tokens.bags == 0 || a.dim == 0) return;
  const int vec = vec_of(a.type, a.dim, a.table, a.row_stride, a.out, a.out_type, a.out_stride);
#define ARB_CALL(T, O)                                              \
  if (vec * sizeof(T) == 16) lookup_with<T, O, 16 / sizeof(T)>(a, s); \
  else if (vec > 1) lookup_with<T, O, 4 / sizeof(T)>(a, s);         \
  else lookup_with<T, O, 1>(a, s)
  ARB_BY_TYPE(a.type, a.out_type, ARB_CALL);
#undef ARB_CALL
  ARB_CUDA(cudaGetLastError());
  count_launch();
}

namespace {
size_t pad256(size_t b) { return (b + 255) / 256 * 256; }
// Bags of a piece: few tokens want short pieces, so that a frequent row is shared widely; a large
// batch has pieces enough, and longer ones cost fewer partial sums.
unsigned piece_of(int64_t count) {
  unsigned p = 32;
  while (p < 4096 && int64_t(p) * 8192 < count) p *= 2;
  return p;
}
// a frequent row has more than `piece` bags, so its pieces are fewer than two for every `piece` bags
int64_t most_pieces(int64_t count) { return count / piece_of(count) * 2 + 1; }
}  // namespace

size_t TokenOrder::bytes(int64_t count, int64_t rows) {
  return 256 + pad256(size_t(count) * 4) + pad256(size_t(rows + 1) * 4) + pad256(size_t(count / piece_of(count) + 1) * 8);
}
TokenOrder::TokenOrder(void *mem, int64_t count_, int64_t rows_) : count(count_), rows(rows_), piece(piece_of(count_)) {
  char *p = static_cast<char *>(mem);
  counts = reinterpret_cast<unsigned long long *>(p);
  bag = reinterpret_cast<unsigned *>(p + 256);
  begin = reinterpret_cast<unsigned *>(p + 256 + pad256(size_t(count) * 4));
  frequent = reinterpret_cast<uint2 *>(p + 256 + pad256(size_t(count) * 4) + pad256(size_t(rows + 1) * 4));
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
  ARB_CUDA(cudaMemsetAsync(o.counts, 0, sizeof *o.counts, s));
  order_plan_kernel<<<grid_of(o.rows, 256, 8), 256, 0, s>>>(o);
  ARB_CUDA(cudaGetLastError());
  count_launch(2);
}

size_t lookup_grad_scratch(int64_t count, int64_t rows, int64_t dim) {
  (void)rows;
  return count > piece_of(count) ? pad256(size_t(most_pieces(count)) * size_t(dim) * sizeof(float)) : 0;
}

namespace {

template <typename T, typename O, int VEC, int U>
void lookup_grad_with(const LookupGradLaunch &a, const TokenOrder &o, float *partial, cudaStream_t s) {
  const int vecs = int(a.dim / VEC);
  GradLanes sh;
  sh.tx_bits = std::min(5, log2_floor(std::max(1, (vecs + U - 1) / U * 2 - 1)));
  sh.ly_item_bits = 5 - sh.tx_bits;
  // a row is named by count / rows bags: that many lanes share it
  sh.ly_row_bits = 0;
  while (sh.tx_bits + sh.ly_row_bits < 5 && (o.rows << sh.ly_row_bits) < o.count) ++sh.ly_row_bits;
  const int chunks = (vecs + (U << sh.tx_bits) - 1) / (U << sh.tx_bits);
  const int64_t groups = kGradThreads >> (sh.tx_bits + sh.ly_row_bits);
  const int64_t item_groups = kGradThreads >> (sh.tx_bits + sh.ly_item_bits);
  unsigned item_blocks = 0;
  if (o.count > o.piece)
    item_blocks = unsigned(std::min<int64_t>((most_pieces(o.count) + item_groups - 1) / item_groups, device_sm_count() * 16));
  const dim3 grid(unsigned((o.rows + groups - 1) / groups) + item_blocks, unsigned(std::min(chunks, 65535)));
  lookup_grad_kernel<T, O, VEC, U><<<grid, kGradThreads, 0, s>>>(a, o, sh, vecs, chunks, item_blocks, partial);
  if (item_blocks) {
    const dim3 join(unsigned(std::min<int64_t>(o.count / o.piece, device_sm_count() * 8)),
                    unsigned(std::min<int64_t>((vecs + kGradThreads - 1) / kGradThreads, 65535)));
    lookup_grad_join_kernel<O, VEC><<<join, kGradThreads, 0, s>>>(a, o, vecs, partial);
    count_launch();
  }
}

template <typename T, typename O, int VEC>
void lookup_grad_vec(const LookupGradLaunch &a, const TokenOrder &o, float *partial, cudaStream_t s) {
  ARB_CHECK(a.dim / VEC <= (int64_t(1) << 30), "rows of more than 2^30 vectors");
  // a wide row gives every lane several vectors: more bytes in flight for one look at the row's bags
  if (VEC > 1 && a.dim / VEC >= 128) lookup_grad_with<T, O, VEC, VEC == 1 ? 1 : 4>(a, o, partial, s);
  else lookup_grad_with<T, O, VEC, 1>(a, o, partial, s);
}

}  // namespace

void launch_lookup_grad(const LookupGradLaunch &a, const TokenOrder &o, void *scratch, cudaStream_t s) {
  if (o.rows == 0 || a.dim == 0) return;
  const int vec = vec_of(a.type, a.dim, a.grad, a.grad_stride, a.out, a.out_type, a.out_stride);
  float *partial = static_cast<float *>(scratch);
#define ARB_CALL(T, O)                                                             \
  if (vec * sizeof(T) == 16) lookup_grad_vec<T, O, 16 / sizeof(T)>(a, o, partial, s); \
  else if (vec > 1) lookup_grad_vec<T, O, 4 / sizeof(T)>(a, o, partial, s);         \
  else lookup_grad_vec<T, O, 1>(a, o, partial, s)
  ARB_BY_TYPE(a.type, a.out_type, ARB_CALL);
#undef ARB_CALL
  ARB_CUDA(cudaGetLastError());
  count_launch();
}

}  // namespace arb
