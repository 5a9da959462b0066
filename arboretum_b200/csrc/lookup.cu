// Lookup of table rows by token with scaling, its gradient by sorted tokens, and the sort itself.
//
//   out[b, :] = round(scale * sum_t table[tok[b, t], :])
//   dtable[v, :] = round(scale * sum_{(b, t): tok[b, t] = v} grad[b, :])
//
// Sums are held in fp32 and rounded once to the output's type.  No floating-point atomics: the
// gradient of a row is summed by its owner over the sorted tokens, in an order that only the tokens
// decide, so two calls on the same tokens give the same bits.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

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

constexpr int kLookupThreads = 256;

// Rows a lane adds up in fp32 before the sum is set aside and begun anew: a bag of a million tokens would
// drift by thousands of half steps in one chain.
constexpr int kChain = 1024;

// A thread's vector of the sum over the tokens begin + slice, begin + slice + ly, .. below `end` of bag b,
// K rows in flight.
// TOGETHER: the lanes of a group (at least eight) fetch a token each and hand them around, so that a
// bag's tokens cost one access and empty slots cost nothing.
template <typename T, int VEC, int K, bool TOGETHER>
__device__ __forceinline__ void sum_tokens(const LookupLaunch &a, long long b, long long begin, long long end, int slice, int ly, int tx,
                                           int c, int vecs, float (&sum)[VEC]) {
  const T *table = static_cast<const T *>(a.table) + (long long)c * VEC;
  const long long mine = b < a.tokens.bags ? end : begin;
  if (TOGETHER) {
    const int width = min(tx, 32), lane = threadIdx.x & 31, group0 = lane & ~(width - 1);
    // every lane of the warp makes as many rounds as a whole bag needs: the shuffles want them all
    for (long long k0 = begin; k0 < end; k0 += (long long)ly * width) {
      const long long k = k0 + slice + (long long)(lane - group0) * ly;
      const long long row = k < mine ? row_at(a.tokens, a.rows, b, k) : -1;
      const int index = int(row);  // rows fit 31 bits
      unsigned todo = (__ballot_sync(0xffffffffu, row >= 0) >> group0) & (width == 32 ? 0xffffffffu : (1u << width) - 1u);
      while (__any_sync(0xffffffffu, todo != 0)) {
        Vec<T, VEC> v[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
          const int src = todo ? __ffs(todo) - 1 : 0;
          const int r = __shfl_sync(0xffffffffu, index, group0 + src);
          v[i].clear();
          if (todo && c < vecs) v[i].load(table + (long long)r * a.row_stride);
          todo &= todo - 1;
        }
#pragma unroll
        for (int i = 0; i < K; ++i) v[i].add_to(sum);
      }
    }
  } else {
    for (long long k0 = begin + slice; k0 < mine; k0 += (long long)ly * K) {
      long long row[K];
#pragma unroll
      for (int i = 0; i < K; ++i) row[i] = k0 + i * ly < mine ? row_at(a.tokens, a.rows, b, k0 + i * ly) : -1;
      Vec<T, VEC> v[K];
#pragma unroll
      for (int i = 0; i < K; ++i) {
        v[i].clear();
        if (row[i] >= 0 && c < vecs) v[i].load(table + row[i] * a.row_stride);
      }
#pragma unroll
      for (int i = 0; i < K; ++i) v[i].add_to(sum);
    }
  }
}

// Bags of several tokens.  A unit is a bag and a run of tx vectors of VEC columns.  Memory bound: the
// rows are read once and the result written once; a thread has the loads of K rows in flight before it
// adds the first.  With few bags the tokens of a bag are split over ly groups of lanes, which join
// their sums through shared memory in a fixed order.  20011 bags of up to 12 rows of 100 fp16 columns, a
// table that the second-level cache holds: 14.3 us (six CTAs an SM; 16.6 with the five that fit without a
// limit on registers).  Issue is busy half of that time and warps wait for a turn more than for a load:
// all eight slots of a round are executed, whatever is left of a bag.
// LONG: bags of more than kChain rows a lane, whose sums are set aside; apart from the others, which would
// pay for it with registers (a million bags of 128 rows of one column: 294 us, 329 in one kernel).
template <typename T, typename O, int VEC, bool TOGETHER, bool LONG>
__global__ void __launch_bounds__(kLookupThreads, 6) lookup_kernel(LookupLaunch a, LaneShape sh, int vecs, int chunks) {
  __shared__ float part[kLookupThreads * VEC];
  const int tx = 1 << sh.tx_bits, ly = 1 << sh.ly_bits;
  const int lane = threadIdx.x & (tx - 1), slice = (threadIdx.x >> sh.tx_bits) & (ly - 1);
  const int group = threadIdx.x >> (sh.tx_bits + sh.ly_bits), groups = kLookupThreads >> (sh.tx_bits + sh.ly_bits);
  const long long b = blockIdx.x * (long long)groups + group;
  for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
    const int c = chunk * tx + lane;
    float sum[VEC];
    if constexpr (!LONG) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
      sum_tokens<T, VEC, 8, TOGETHER>(a, b, 0, a.tokens.per_bag, slice, ly, tx, c, vecs, sum);
    } else {
      __syncthreads();  // others may still read what they join of the columns before
      for (long long k = 0; k < a.tokens.per_bag; k += (long long)kChain * ly) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
        sum_tokens<T, VEC, 8, TOGETHER>(a, b, k, min(k + (long long)kChain * ly, (long long)a.tokens.per_bag), slice, ly, tx, c, vecs, sum);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float &total = part[j * kLookupThreads + threadIdx.x];
          if (k != 0) sum[j] += total;
          total = sum[j];
        }
      }
    }
    if (ly > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VEC; ++j) part[j * kLookupThreads + threadIdx.x] = sum[j];
      for (int half = ly >> 1; half > 0; half >>= 1) {
        __syncthreads();
        if (slice < half) {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            part[j * kLookupThreads + threadIdx.x] += part[j * kLookupThreads + threadIdx.x + half * tx];
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] = part[j * kLookupThreads + threadIdx.x];
    }
    if (b < a.tokens.bags && slice == 0 && c < vecs) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] *= a.scale;
      store_vec<O, VEC>(static_cast<O *>(a.out) + b * a.out_stride + (long long)c * VEC, sum);
    }
  }
}

// One token a bag: a row is copied, scaled, from the table to the output.  A group of tx lanes takes a
// run of tx * U vectors of one row.  Memory bound: 16384 rows of 4096 bf16 in 44 us, 5.9 TB/s (with the
// bags' loop and its sums around the same accesses 53).
template <typename T, typename O, int VEC, int U>
__global__ void __launch_bounds__(kLookupThreads) lookup_rows_kernel(LookupLaunch a, int tx_bits, int vecs, int chunks) {
  const int tx = 1 << tx_bits, lane = threadIdx.x & (tx - 1);
  const long long b = blockIdx.x * (long long)(kLookupThreads >> tx_bits) + (threadIdx.x >> tx_bits);
  if (b >= a.tokens.bags) return;
  const long long row = row_at(a.tokens, a.rows, b, 0);
  const T *from = static_cast<const T *>(a.table) + row * a.row_stride;
  O *out = static_cast<O *>(a.out) + b * a.out_stride;
  for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
    const int c0 = chunk * (tx * U) + lane;
    Vec<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].clear();
      if (row >= 0 && c0 + u * tx < vecs) v[u].load(from + (long long)(c0 + u * tx) * VEC);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VEC];
      v[u].get(x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] *= a.scale;
      if (c0 + u * tx < vecs) store_vec<O, VEC>(out + (long long)(c0 + u * tx) * VEC, x);
    }
  }
}

// The same for 16-bit rows that begin on any two bytes (an odd number of columns): four-byte accesses all
// the same.  A row's elements are taken as they share aligned words where they lie; where the output's
// words pair them differently, a word's halves come from two neighbouring lanes.  10608 rows of 4545
// bf16: 51 us, 66 with an access an element (32 at 4546, 23 at 4544); bound by issued instructions.
template <typename T>
__device__ __forceinline__ unsigned load_pair(const T *row, long long e, long long dim) {  // elements e, e + 1; row + e on four bytes
  if (e >= 0 && e + 1 < dim) return *reinterpret_cast<const unsigned *>(row + e);
  unsigned lo = 0, hi = 0;
  if (e >= 0 && e < dim) lo = *reinterpret_cast<const unsigned short *>(row + e);
  if (e + 1 >= 0 && e + 1 < dim) hi = *reinterpret_cast<const unsigned short *>(row + e + 1);
  return hi << 16 | lo;
}
template <typename T, int U>
__global__ void __launch_bounds__(kLookupThreads) lookup_odd_rows_kernel(LookupLaunch a, int chunks) {
  const int lane = threadIdx.x & 31;
  const long long b = blockIdx.x * (long long)(kLookupThreads / 32) + threadIdx.x / 32;  // a warp a row
  if (b >= a.tokens.bags) return;
  const long long token = row_at(a.tokens, a.rows, b, 0);
  const T *from = static_cast<const T *>(a.table) + max(token, 0ll) * a.row_stride;
  T *out = static_cast<T *>(a.out) + b * a.out_stride;
  const long long dim = token < 0 ? 0 : a.dim;  // an empty slot loads nothing
  const int s = int(reinterpret_cast<uintptr_t>(from) / 2 & 1), d = int(reinterpret_cast<uintptr_t>(out) / 2 & 1);
  for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
    // output word w holds elements 2 w - d and the next; its first one is in the row's word w + (s && !d),
    // the halves swapped where s and d differ
    const long long w0 = (long long)chunk * (32 * U) + lane;
    unsigned word[U], next = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) word[u] = load_pair(from, 2 * (w0 + u * 32) - s - (d && !s ? 2 : 0), dim);
    if (s != d && lane == 31) next = load_pair(from, 2 * (w0 + (U - 1) * 32 + 1) - s - (d && !s ? 2 : 0), dim);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unsigned pair = word[u];
      if (s != d) {  // the same for the whole warp
        const unsigned from_next = __shfl_down_sync(0xffffffffu, word[u], 1);
        const unsigned from_first = u + 1 < U ? __shfl_sync(0xffffffffu, word[u + 1 < U ? u + 1 : u], 0) : next;
        pair = __byte_perm(word[u], lane == 31 ? from_first : from_next, 0x5432);  // upper half, then the next one's lower
      }
      T e[2];
      memcpy(e, &pair, 4);
      from_f32(to_f32(e[0]) * a.scale, e[0]);
      from_f32(to_f32(e[1]) * a.scale, e[1]);
      memcpy(&pair, e, 4);
      const long long at = 2 * (w0 + u * 32) - d;
      if (at >= 0 && at + 1 < a.dim) {
        *reinterpret_cast<unsigned *>(out + at) = pair;
      } else {
        if (at >= 0 && at < a.dim) out[at] = e[0];
        if (at + 1 >= 0 && at + 1 < a.dim) out[at + 1] = e[1];
      }
    }
  }
}

// Bags of many tokens over a narrow table that fits into shared memory (the leaf values of a forest):
// every CTA holds the whole table and a thread the sums of two neighbouring bags, whose tokens lie
// side by side in memory, tree after tree.  The tokens are all that is read from device memory; the
// table's values come from shared memory, where 32 random words cost a few cycles and a gather
// through the first-level cache one for every line it touches.  A million bags of 128 int32 tokens over
// 32768 values: 96 us, 5.4 TB/s (350 through the cache).
constexpr int kTableThreads = 1024;
// tokens of two bags, K slots
template <typename I, int K>
struct TokenPairs {
  struct alignas(2 * sizeof(I)) Both { I v[2]; };
  Both tok[K];
  __device__ __forceinline__ void load(const I *p, long long step, long long other, bool paired) {
    if (paired) {  // one access for both bags
#pragma unroll
      for (int k = 0; k < K; ++k) tok[k] = *reinterpret_cast<const Both *>(p + k * step);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) tok[k].v[0] = p[k * step], tok[k].v[1] = p[k * step + other];
    }
  }
  template <int DIM>
  __device__ __forceinline__ void add(const float *values, unsigned rows, float (&sum)[2][DIM]) const {
    using U = typename std::make_unsigned<I>::type;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const unsigned r = U(tok[k].v[e]) < U(rows) ? unsigned(tok[k].v[e]) : rows;
#pragma unroll
        for (int d = 0; d < DIM; ++d) sum[e][d] += values[r * DIM + d];
      }
  }
};

template <typename T, typename O, typename I, int DIM>
__global__ void __launch_bounds__(kTableThreads) lookup_table_kernel(LookupLaunch a, bool paired) {
  extern __shared__ float values[];  // [rows][DIM], and a row of zeros for empty slots
  const unsigned rows = unsigned(a.rows);
  for (unsigned i = threadIdx.x; i < (rows + 1) * DIM; i += blockDim.x) {
    const unsigned r = i / DIM, d = i - r * DIM;
    values[i] = r < rows ? to_f32(static_cast<const T *>(a.table)[(long long)r * a.row_stride + d]) : 0.0f;
  }
  __syncthreads();
  constexpr int K = 32 / int(sizeof(I));  // slots whose tokens are under way while as many others are summed
  const int per_bag = int(a.tokens.per_bag), full = per_bag / K * K;
  const long long step = a.tokens.token_stride;
  for (long long b = (blockIdx.x * (long long)blockDim.x + threadIdx.x) * 2; b < a.tokens.bags;
       b += (long long)gridDim.x * blockDim.x * 2) {
    const bool two = b + 1 < a.tokens.bags;
    const long long other = two ? a.tokens.bag_stride : 0;  // a last bag alone is summed twice
    const bool both = paired && two;
    const I *p = static_cast<const I *>(a.tokens.at) + b * a.tokens.bag_stride;
    float sum[2][DIM];
#pragma unroll
    for (int d = 0; d < DIM; ++d) sum[0][d] = sum[1][d] = 0.0f;
    if (full) {
      TokenPairs<I, K> now;
      now.load(p, step, other, both);
#pragma unroll 2
      for (int k = K; k < full; k += K) {
        p += K * step;
        TokenPairs<I, K> next;
        next.load(p, step, other, both);
        now.add(values, rows, sum);
        now = next;
      }
      now.add(values, rows, sum);
      p += K * step;
    }
    for (int k = full; k < per_bag; ++k, p += step) {
      TokenPairs<I, 1> last;
      last.load(p, step, other, both);
      last.add(values, rows, sum);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (e == 0 || two) {
        O *out = static_cast<O *>(a.out) + (b + e) * a.out_stride;
#pragma unroll
        for (int d = 0; d < DIM; ++d) from_f32(sum[e][d] * a.scale, out[d]);
      }
  }
}

// ---- the sort --------------------------------------------------------------------------------
// Least-significant-digit radix sort of (token, bag): every pass counts the digits of each tile,
// turns the counts into positions (digit by digit, tile by tile) and moves the pairs, keeping the
// order of equal digits.  An empty slot sorts as token `rows`, behind everything.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortThreads = kDigits, kSortWarps = kSortThreads / 32;  // a thread takes a digit
// pairs of a thread: few of them give every SM a tile of a small batch, many long runs of a large one
constexpr int kFewItems = 4, kManyItems = 16;
constexpr int64_t kManyTokens = int64_t(1) << 20;

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
  bool blocked;            // keys are (run of bags, token)
  unsigned *clear_counts;  // first pass of an order that is not blocked: what its items count in and mark is cleared
  unsigned char *clear_named;
};

__device__ __forceinline__ void sort_pair(const SortPass &p, long long i, unsigned &key, unsigned &bag) {
  if (!p.first) {
    key = p.key_in[i];
    bag = p.bag_in[i];
    return;
  }
  const unsigned at = unsigned(i), by = unsigned(p.by_slot ? p.tokens.bags : p.tokens.per_bag);  // both below 2^31
  const unsigned hi = by == 1 ? at : at / by, lo = at - hi * by;
  const long long b = p.by_slot ? lo : hi, k = p.by_slot ? hi : lo;
  const long long row = row_at(p.tokens, p.rows, b, k);
  key = row >= 0 ? unsigned(row) : unsigned(p.rows);
  bag = unsigned(b);
  if (p.blocked) key += bag / kBlockBags * unsigned(p.rows + 1);
}

// lanes of the warp with the same digit: a ballot a bit (the match instruction takes its time with many
// different values)
__device__ __forceinline__ unsigned lanes_with(unsigned digit, int bits) {
  unsigned same = 0xffffffffu;
  for (int i = 0; i < bits; ++i) {
    const unsigned set = __ballot_sync(0xffffffffu, digit >> i & 1u);
    same &= digit >> i & 1u ? set : ~set;
  }
  return same;
}

template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortPass p) {
  __shared__ unsigned cnt[kDigits];
  overlap_release();
  overlap_wait();
  cnt[threadIdx.x] = 0;
  if (p.clear_named != nullptr) {
    if (blockIdx.x == 0 && threadIdx.x < 2) p.clear_counts[threadIdx.x] = 0;
    const long long step = (long long)gridDim.x * kSortThreads;
    for (long long i = blockIdx.x * (long long)kSortThreads + threadIdx.x; i < (p.rows + 15) / 16; i += step)
      reinterpret_cast<uint4 *>(p.clear_named)[i] = make_uint4(0u, 0u, 0u, 0u);  // padded to 256 bytes
  }
  __syncthreads();
  const long long t0 = blockIdx.x * (long long)(kSortThreads * ITEMS);
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const long long i = t0 + j * kSortThreads + threadIdx.x;
    if (i < p.n) {
      unsigned key, bag;
      sort_pair(p, i, key, bag);
      atomicAdd(&cnt[(key >> p.shift) & (kDigits - 1)], 1u);
    }
  }
  __syncthreads();
  p.counts[size_t(threadIdx.x) * p.tiles + blockIdx.x] = cnt[threadIdx.x];
}

// exclusive sum over the threads of a CTA
__device__ __forceinline__ unsigned block_exclusive(unsigned v, unsigned *total) {
  __shared__ unsigned warp_sum[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  unsigned x = v;
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sum[w] = x;
  __syncthreads();
  unsigned before = 0, all = 0;
  for (int i = 0; i < warps; ++i) {
    if (i < w) before += warp_sum[i];
    all += warp_sum[i];
  }
  __syncthreads();
  *total = all;
  return before + x - v;
}

// one CTA a digit: its counts become exclusive sums over the tiles
__global__ void __launch_bounds__(256) sort_scan_kernel(SortPass p) {
  overlap_release();
  overlap_wait();
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

// Pairs are put in order inside the tile first, so that what goes to one digit's place in memory leaves
// as a run.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_move_kernel(SortPass p) {
  extern __shared__ uint2 staged[];  // [kSortThreads * ITEMS]
  __shared__ unsigned short warp_cnt[kSortWarps][kDigits];
  __shared__ unsigned base[kDigits];          // where the tile's pairs of a digit go
  __shared__ unsigned short first[kDigits];   // and where they begin in the tile
  overlap_release();
  overlap_wait();
  constexpr int kTile = kSortThreads * ITEMS;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  for (int i = 0; i < kSortWarps; ++i) warp_cnt[i][tid] = 0;
  {
    unsigned all;
    const unsigned before = block_exclusive(p.totals[tid], &all);
    base[tid] = before + p.counts[size_t(tid) * p.tiles + blockIdx.x];
  }
  __syncthreads();
  // a warp owns ITEMS * 32 neighbouring pairs; equal digits keep their order
  const long long t0 = blockIdx.x * (long long)kTile, w0 = t0 + w * (ITEMS * 32);
  unsigned key[ITEMS], bag[ITEMS];
  unsigned short rank[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const long long i = w0 + j * 32 + lane;
    key[j] = 0xffffffffu, bag[j] = 0;
    if (i < p.n) sort_pair(p, i, key[j], bag[j]);
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const bool in = w0 + j * 32 + lane < p.n;
    const unsigned digit = (key[j] >> p.shift) & (kDigits - 1);
    const unsigned same = lanes_with(digit, kDigitBits) & __ballot_sync(0xffffffffu, in);
    const unsigned below = __popc(same & ((1u << lane) - 1u));
    rank[j] = (unsigned short)(warp_cnt[w][digit] + below);
    __syncwarp();
    if (in && below == 0) warp_cnt[w][digit] += (unsigned short)__popc(same);
    __syncwarp();
  }
  __syncthreads();
  {
    unsigned run = 0, all;
#pragma unroll
    for (int i = 0; i < kSortWarps; ++i) {
      const unsigned c = warp_cnt[i][tid];
      warp_cnt[i][tid] = (unsigned short)run;
      run += c;
    }
    first[tid] = (unsigned short)block_exclusive(run, &all);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    if (w0 + j * 32 + lane < p.n) {
      const unsigned digit = (key[j] >> p.shift) & (kDigits - 1);
      staged[first[digit] + warp_cnt[w][digit] + rank[j]] = make_uint2(key[j], bag[j]);
    }
  }
  __syncthreads();
  const int n = int(min((long long)kTile, p.n - t0));
  for (int i = tid; i < n; i += kSortThreads) {
    const uint2 v = staged[i];
    const unsigned digit = (v.x >> p.shift) & (kDigits - 1);
    const unsigned to = base[digit] + (i - first[digit]);
    p.key_out[to] = v.x;
    p.bag_out[to] = v.y;
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

// ---- vectors of a blocked order ----------------------------------------------------------------
// A segment (run, row) takes as many vectors of eight bags as it needs, the empty slots behind a run's
// last row none.  Sums over tiles of segments, their exclusive sums, then every segment's first vector.
constexpr int kVecTile = 2048;
__device__ __forceinline__ unsigned vectors_of(const unsigned *__restrict__ begin, long long k, const TokenOrder &o) {
  return k < o.segments() && k % (o.rows + 1) != o.rows ? (begin[k + 1] - begin[k] + 7) / 8 : 0u;
}
__global__ void __launch_bounds__(256) vec_count_kernel(const unsigned *__restrict__ begin, TokenOrder o, unsigned *__restrict__ tile) {
  unsigned sum = 0;
  for (int j = 0; j < kVecTile / 256; ++j) sum += vectors_of(begin, blockIdx.x * (long long)kVecTile + j * 256 + threadIdx.x, o);
  unsigned all;
  block_exclusive(sum, &all);
  if (threadIdx.x == 0) tile[blockIdx.x] = all;
}
__global__ void __launch_bounds__(256) vec_tiles_kernel(unsigned *tile, int tiles) {
  unsigned run = 0;
  for (int t = 0; t < tiles; t += 256) {
    const int i = t + int(threadIdx.x);
    const unsigned v = i < tiles ? tile[i] : 0u;
    unsigned all;
    const unsigned before = block_exclusive(v, &all);
    if (i < tiles) tile[i] = run + before;
    run += all;
  }
}
__global__ void __launch_bounds__(256) vec_begin_kernel(const unsigned *__restrict__ begin, TokenOrder o, const unsigned *__restrict__ tile) {
  unsigned run = tile[blockIdx.x];
  for (int j = 0; j < kVecTile / 256; ++j) {
    const long long k = blockIdx.x * (long long)kVecTile + j * 256 + threadIdx.x;
    const unsigned n = vectors_of(begin, k, o);
    unsigned all;
    const unsigned first = run + block_exclusive(n, &all);
    run += all;
    if (k > o.segments()) continue;
    o.vec_begin[k] = first;
    if (n)  // the end of the last vector
      for (unsigned p = begin[k + 1] - begin[k]; p < n * 8; ++p) o.local[size_t(first) * 8 + p] = kNoBag;
  }
}
__global__ void vec_move_kernel(const unsigned *__restrict__ key, const unsigned *__restrict__ bag, const unsigned *__restrict__ begin,
                                TokenOrder o) {
  const unsigned rows1 = unsigned(o.rows + 1);
  for (long long p = blockIdx.x * (long long)blockDim.x + threadIdx.x; p < o.count; p += (long long)gridDim.x * blockDim.x) {
    const unsigned k = key[p], run = k / rows1;
    if (k - run * rows1 == unsigned(o.rows)) continue;
    o.local[size_t(o.vec_begin[k]) * 8 + (unsigned(p) - begin[k])] = (unsigned short)((bag[p] - run * kBlockBags) * 4);
  }
}

// ---- items of work -----------------------------------------------------------------------------
// The bags of a row, in pieces: a frequent token's sum is shared by many warps.  The order of the list
// depends on the order of arrival here; no value does: where a row is cut follows from the sorted
// positions alone, and its pieces are joined in their own order.
// Called by whole warps; `at(i)` is the token at sorted position i, row[] that of the positions
// q0 + 32 j + lane. One atomic addition a warp, whatever the number of positions.
template <int ITEMS, typename At>
__device__ __forceinline__ void add_items(const TokenOrder &o, long long q0, const unsigned (&row)[ITEMS], const At &at) {
  const unsigned n = unsigned(o.count), piece = o.piece;
  const int lane = threadIdx.x & 31;
  // p a multiple inside the row: is another one before or behind it in the row?
  const auto cut_at = [&](unsigned p, unsigned r) {
    return (p >= piece && at(p - piece) == r) || (p + piece < n && at(p + piece) == r);
  };
  bool first[ITEMS], item[ITEMS];
  unsigned items = 0;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const long long ql = q0 + 32 * j + lane;
    const unsigned q = unsigned(ql);
    const bool valid = ql < (long long)n && (long long)row[j] < o.rows;
    first[j] = valid && (q == 0 || at(q - 1) != row[j]);
    item[j] = first[j] || (valid && (q & (piece - 1)) == 0 && cut_at(q, row[j]));
    items += __popc(__ballot_sync(0xffffffffu, item[j]));
  }
  if (items == 0) return;
  unsigned slot = 0;
  if (lane == 0) slot = atomicAdd(&o.counts[0], items);
  slot = __shfl_sync(0xffffffffu, slot, 0);
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const unsigned same = __ballot_sync(0xffffffffu, item[j]);
    const unsigned mine = slot + __popc(same & ((1u << lane) - 1u));
    slot += __popc(same);
    if (!item[j]) continue;
    const unsigned q = unsigned(q0 + 32 * j + lane), r = row[j];
    // first position behind q, below `most`, of another row
    const auto end_of = [&](unsigned most) {
      unsigned lo = q, hi = most;  // at(lo) is the row's, hi is not or is the end
      while (hi - lo > 1) {
        const unsigned mid = lo + (hi - lo) / 2;
        if (at(mid) == r) lo = mid;
        else hi = mid;
      }
      return hi;
    };
    const unsigned next = (q / piece + 1) * piece;  // the next multiple; within the row it cuts if it is one of two
    unsigned end;
    bool whole = first[j];
    if (next < n && at(next) == r && cut_at(next, r)) {
      end = next;
      if (first[j]) o.frequent[atomicAdd(&o.counts[1], 1u)] = make_uint4(q, end_of(n), r, 0u);
      whole = false;
    } else if (q + 1 >= n || at(q + 1) != r) {  // most rows have one bag
      end = q + 1;
    } else {
      end = end_of(n - q > 2 * piece ? q + 2 * piece : n);
    }
    o.item[mine] = make_uint4(q, end, r, whole ? 1u : 0u);
    if (first[j]) o.named[r] = 1;
  }
}

__global__ void order_items_kernel(TokenOrder o, const unsigned *key) {
  overlap_release();
  overlap_wait();
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long q0 = blockIdx.x * (long long)blockDim.x + (threadIdx.x & ~31u); q0 < o.count; q0 += step) {
    const long long q = q0 + (threadIdx.x & 31);
    const unsigned row[1] = {q < o.count ? key[q] : 0xffffffffu};
    add_items<1>(o, q0, row, [&](unsigned i) { return key[i]; });
  }
}

// A few tokens: one CTA, and a token's place is the number of tokens before it, counted.  (The digits'
// passes of the cluster take 10 us whatever the number of tokens.)
constexpr int kFewTokens = 512;
constexpr int64_t kFewRows = 1 << 18;  // marks that the sort clears itself
__global__ void __launch_bounds__(kFewTokens) order_few_kernel(SortPass p, TokenOrder o, bool clear) {
  __shared__ __align__(16) unsigned key[kFewTokens];
  __shared__ unsigned sorted[kFewTokens];
  const int tid = threadIdx.x, n = int(p.n);
  if (tid < 2) o.counts[tid] = 0;
  if (clear)
    for (long long i = tid; i < (p.rows + 15) / 16; i += blockDim.x)
      reinterpret_cast<uint4 *>(o.named)[i] = make_uint4(0u, 0u, 0u, 0u);  // padded to 256 bytes
  unsigned mine = 0xffffffffu, bag = 0;
  if (tid < n) sort_pair(p, tid, mine, bag);
  key[tid] = mine;
  sorted[tid] = 0xffffffffu;
  __syncthreads();
  unsigned place = 0;
  for (int i = 0; i < n; i += 4) {
    const uint4 k = *reinterpret_cast<const uint4 *>(key + i);  // behind the last token: above all tokens
    place += k.x < mine || (k.x == mine && i < tid);
    place += k.y < mine || (k.y == mine && i + 1 < tid);
    place += k.z < mine || (k.z == mine && i + 2 < tid);
    place += k.w < mine || (k.w == mine && i + 3 < tid);
  }
  if (tid < n) {
    sorted[place] = mine;
    o.bag[place] = bag;
  }
  __syncthreads();
  const unsigned row[1] = {sorted[tid]};
  add_items<1>(o, tid & ~31, row, [&](unsigned i) { return sorted[i]; });
}

// Where the sum of the piece that begins at position q goes.  Of the pieces that begin within one run of
// `piece` positions at most two belong to cut rows: one that begins with the run, and the first one of a
// row that ends beyond it.
__device__ __forceinline__ size_t slot_of(unsigned q, unsigned piece) {
  return size_t(q / piece) * 2 + ((q & (piece - 1)) != 0 ? 1 : 0);
}

// ---- the gradient ----------------------------------------------------------------------------
struct GradLanes {
  int tx_bits, ly_bits;  // of a sum: lanes across the columns, lanes along the bags
  int zero_bits;         // lanes across the columns of an untouched row
  int chunks;            // runs of tx * U vectors in a row
};

constexpr int kGradThreads = 256;

// The vectors of one gradient row that a lane takes.  ODD: 16-bit rows that begin on any two bytes, in
// pairs of columns (VEC = 2) read by aligned words; where a row's words pair the columns differently, a
// pair's halves come from two neighbouring lanes.  A warp has one row then.
template <typename T, int VEC, int U, bool ODD>
struct RowPart {
  Vec<T, VEC> v[U];
  unsigned next;  // ODD: lane 31's word behind its last one
  bool shifted;   // ODD: the row's words begin with odd columns; the same for the whole warp
  __device__ __forceinline__ void load(const LookupGradLaunch &a, bool in, unsigned bag, int c0, int tx, int vecs) {
    const T *row = static_cast<const T *>(a.grad) + (long long)bag * a.grad_stride;
    if constexpr (ODD) {
      shifted = reinterpret_cast<uintptr_t>(row) / 2 & 1;
      const long long dim = in ? a.dim : 0;
      const int s = shifted ? 1 : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) v[u].raw[0] = load_pair(row, 2ll * (c0 + u * 32) - s, dim);
      next = s && (threadIdx.x & 31) == 31 ? load_pair(row, 2ll * (c0 + (U - 1) * 32 + 1) - s, dim) : 0u;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u].clear();
        if (in && c0 + u * tx < vecs) v[u].load(row + (long long)(c0 + u * tx) * VEC);
      }
    }
  }
  // whole warps: the halves change lanes
  __device__ __forceinline__ void add_to(float (&sum)[U][VEC]) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec<T, VEC> x = v[u];
      if constexpr (ODD) {
        if (shifted) {
          const unsigned from_next = __shfl_down_sync(0xffffffffu, v[u].raw[0], 1);
          const unsigned from_first = u + 1 < U ? __shfl_sync(0xffffffffu, v[u + 1 < U ? u + 1 : u].raw[0], 0) : next;
          x.raw[0] = __byte_perm(v[u].raw[0], (threadIdx.x & 31) == 31 ? from_first : from_next, 0x5432);
        }
      }
      x.add_to(sum[u]);
    }
  }
};

// Sum over the sorted positions p .. end of the gradient rows they name, for a group of tx * ly lanes:
// the group's lanes fetch as many bags at once and hand them around; slice s takes every ly-th position.
// `id` is the bag of this lane's position of the first tx * ly, `head` the row of its slice's first
// position, both already fetched.  For whole warps.
template <typename T, int VEC, int U, bool ODD>
__device__ __forceinline__ void sum_bags(const LookupGradLaunch &a, const unsigned *__restrict__ bag, unsigned p, unsigned end,
                                         unsigned id, const RowPart<T, VEC, U, ODD> &head, int slice, int ly, int tx, int c0, int vecs,
                                         float (&sum)[U][VEC]) {
  constexpr int K = U > 1 ? 3 : 8;  // bags whose loads are in flight together
  const int width = tx * ly, group0 = threadIdx.x & 31 & ~(width - 1), place = threadIdx.x & (width - 1);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[u][j] = 0.0f;
  head.add_to(sum);
  for (int k_first = ly;; k_first = 0) {
    const int n = int(min(end - p, unsigned(width)));
    for (int k0 = k_first; __any_sync(0xffffffffu, k0 < n); k0 += ly * K) {
      RowPart<T, VEC, U, ODD> row[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int at = k0 + k * ly + slice;
        const unsigned b = __shfl_sync(0xffffffffu, id, group0 + (at & (width - 1)));
        row[k].load(a, at < n, b, c0, tx, vecs);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) row[k].add_to(sum);
    }
    const bool more = end - p > unsigned(width);
    if (!__any_sync(0xffffffffu, more)) break;
    p = more ? p + width : end;
    id = p + place < end ? bag[p + place] : 0u;
  }
  for (int o = tx; o < tx * ly; o <<= 1)  // the slices of a group are neighbouring lanes of a warp
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[u][j] += __shfl_xor_sync(0xffffffffu, sum[u][j], o);
}

template <typename O, int VEC, int U, bool ODD = false>
__device__ __forceinline__ void write_row(const LookupGradLaunch &a, long long row, int c0, int tx, int vecs,
                                          float (&sum)[U][VEC]) {
  if constexpr (ODD) {  // pairs of columns, written one by one: the output's rows begin anywhere
    O *at = static_cast<O *>(a.out) + row * a.out_stride;
    float old[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const long long c = (long long)(c0 + u * tx) * VEC + j;
        old[u][j] = a.accumulate && c < a.dim ? to_f32(at[c]) : 0.0f;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const long long c = (long long)(c0 + u * tx) * VEC + j;
        if (c < a.dim) from_f32(a.accumulate ? sum[u][j] * a.scale + old[u][j] : sum[u][j] * a.scale, at[c]);
      }
    return;
  }
  O *out = static_cast<O *>(a.out) + row * a.out_stride + (long long)c0 * VEC;
  Vec<O, VEC> old[U];  // all on their way before the first is needed
  if (a.accumulate) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * tx < vecs) old[u].load(out + (long long)(u * tx) * VEC);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (c0 + u * tx >= vecs) continue;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[u][j] *= a.scale;
    if (a.accumulate) old[u].add_to(sum[u]);
    store_vec<O, VEC>(out + (long long)(u * tx) * VEC, sum[u]);
  }
}

// Zeros for one row by tx lanes: 16-byte stores wherever the row begins, single ones before and behind.
template <typename O>
__device__ __forceinline__ void zero_row(O *row, long long dim, int lane, int tx) {
  const long long head = min((long long)((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(O)), dim);
  const long long vecs = (dim - head) / (16 / int(sizeof(O))), tail = head + vecs * (16 / int(sizeof(O)));
  O zero;
  from_f32(0.0f, zero);
  for (long long c = lane; c < head; c += tx) row[c] = zero;
  for (long long c = lane; c < vecs; c += tx) reinterpret_cast<uint4 *>(row + head)[c] = make_uint4(0u, 0u, 0u, 0u);
  for (long long c = tail + lane; c < dim; c += tx) row[c] = zero;
}

// CTAs below item_blocks sum the items' bags: a whole row is written at once, a piece of a frequent one
// goes to `partial`.  The other CTAs write the zeros of the rows that no bag names, kZeroRows rows a
// group of lanes: the marks of all of them are read at once, and the stores wait for nothing else.
constexpr int kZeroRows = 8;
template <typename T, typename O, int VEC, int U, bool ODD>
__global__ void __launch_bounds__(kGradThreads) lookup_grad_kernel(LookupGradLaunch a, TokenOrder o, GradLanes sh, int vecs,
                                                                   unsigned item_blocks, float *partial) {
  overlap_release();
  overlap_wait();
  if (blockIdx.x < item_blocks) {
    const int tx = 1 << sh.tx_bits, lane = threadIdx.x & (tx - 1);
    const int ly = 1 << sh.ly_bits, slice = (threadIdx.x >> sh.tx_bits) & (ly - 1);
    const int bits = sh.tx_bits + sh.ly_bits;
    const int chunks = sh.chunks;
    // Neighbouring groups take the chunks of one item.  Most items are one bag, so the accesses of an item
    // are a chain (item, bag, row) of a few hundred bytes each: they are spread over the items before it.
    // While an item is summed, the first rows of the next one, the bags of the one after that and the place
    // of a third are being fetched.
    const unsigned items = o.counts[0];
    // a group's units are `groups` apart; item and chunk of the next one follow by addition
    const unsigned groups = item_blocks * (kGradThreads >> bits), next_item = groups / chunks, next_chunk = groups % chunks;
    struct Unit {
      unsigned item;
      int chunk;
    };
    const auto after = [&](Unit u) {
      u.item += next_item, u.chunk += int(next_chunk);
      if (u.chunk >= chunks) u.chunk -= chunks, ++u.item;
      return u;
    };
    const auto item_of = [&](const Unit &u) { return u.item < items ? o.item[u.item] : make_uint4(0, 0, 0, 0); };
    const int place = threadIdx.x & (tx * ly - 1), group0 = threadIdx.x & 31 & ~(tx * ly - 1);
    const auto bag_of = [&](const uint4 &it) { return it.x + place < it.y ? o.bag[it.x + place] : 0u; };
    const auto head_of = [&](const uint4 &it, unsigned id, int c0) {
      RowPart<T, VEC, U, ODD> head;
      head.load(a, it.x + slice < it.y, __shfl_sync(0xffffffffu, id, group0 + slice), c0, tx, vecs);
      return head;
    };
    const unsigned begin = blockIdx.x * (kGradThreads >> bits) + (threadIdx.x >> bits);
    Unit u = {begin / chunks, int(begin % chunks)}, u1 = after(u), u2 = after(u1);
    uint4 it = item_of(u), it1 = item_of(u1), it2 = item_of(u2);
    unsigned id = bag_of(it), id1 = bag_of(it1);
    RowPart<T, VEC, U, ODD> head = head_of(it, id, u.chunk * (tx * U) + lane);
    while (__any_sync(0xffffffffu, u.item < items)) {
      const Unit u3 = after(u2);
      const uint4 it3 = item_of(u3);
      const unsigned id2 = bag_of(it2);
      const RowPart<T, VEC, U, ODD> head1 = head_of(it1, id1, u1.chunk * (tx * U) + lane);
      const int c0 = u.chunk * (tx * U) + lane;
      float sum[U][VEC];
      sum_bags<T, VEC, U, ODD>(a, o.bag, it.x, it.y, id, head, slice, ly, tx, c0, vecs, sum);
      if (u.item < items && slice == 0) {
        if (it.w) {
          write_row<O, VEC, U, ODD>(a, it.z, c0, tx, vecs, sum);
        } else {
          float *to = partial + slot_of(it.x, o.piece) * size_t(a.dim);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + u * tx < vecs) {
#pragma unroll
              for (int j = 0; j < VEC; ++j)
                if (!ODD || (long long)(c0 + u * tx) * VEC + j < a.dim) to[(long long)(c0 + u * tx) * VEC + j] = sum[u][j];
            }
        }
      }
      u = u1, u1 = u2, u2 = u3, it = it1, it1 = it2, it2 = it3, id = id1, id1 = id2, head = head1;
    }
    return;
  }
  const int tx = 1 << sh.zero_bits, groups = kGradThreads >> sh.zero_bits;
  const long long row0 = (blockIdx.x - item_blocks) * (long long)(groups * kZeroRows) + (threadIdx.x >> sh.zero_bits);
  unsigned char named[kZeroRows];
#pragma unroll
  for (int r = 0; r < kZeroRows; ++r) named[r] = row0 + r * groups < o.rows ? o.named[row0 + r * groups] : 1;
  const int lane = threadIdx.x & (tx - 1);
#pragma unroll
  for (int r = 0; r < kZeroRows; ++r) {
    if (named[r]) continue;
    O *out = static_cast<O *>(a.out) + (row0 + r * groups) * a.out_stride;
    if constexpr (!ODD && VEC * sizeof(O) >= 16) {  // every row begins on 16 bytes
      constexpr int kWords = VEC * int(sizeof(O)) / 16;
      for (int c = lane; c < vecs * kWords; c += tx) reinterpret_cast<uint4 *>(out)[c] = make_uint4(0u, 0u, 0u, 0u);
    } else {
      zero_row(out, a.dim, lane, tx);
    }
  }
}

// The pieces of a frequent row, joined in their order: eight groups of 32 lanes take every eighth piece
// of a run of columns, and the groups' sums are added one after another.
template <typename O, int VEC, int U>
__global__ void __launch_bounds__(kGradThreads) lookup_grad_join_kernel(LookupGradLaunch a, TokenOrder o, int vecs, int chunks,
                                                                        const float *__restrict__ partial) {
  __shared__ float part[kGradThreads * VEC * U];
  constexpr int kSlices = kGradThreads / 32, K = 4;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  overlap_release();
  overlap_wait();
  const unsigned frequent = o.counts[1];
  for (unsigned h = blockIdx.x; h < frequent; h += gridDim.x) {
    const uint4 f = o.frequent[h];
    const unsigned second = (f.x / o.piece + 1) * o.piece;  // pieces: the first, then one at every multiple
    const unsigned pieces = 1 + (f.y - second + o.piece - 1) / o.piece;
    for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
      const int c0 = chunk * (32 * U) + lane;
      float sum[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[u][j] = 0.0f;
      for (unsigned k0 = slice; k0 < pieces; k0 += kSlices * K) {
        float v[K][U][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const unsigned n = k0 + k * kSlices;
          const unsigned q = n == 0 ? f.x : second + (n - 1) * o.piece;
          const float *at = partial + slot_of(q, o.piece) * size_t(a.dim) + (long long)c0 * VEC;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[k][u][j] = n < pieces && c0 + u * 32 < vecs ? at[u * 32 * VEC + j] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum[u][j] += v[k][u][j];
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[(u * VEC + j) * kGradThreads + threadIdx.x] = sum[u][j];
      __syncthreads();
      if (slice == 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            for (int g = 1; g < kSlices; ++g) sum[u][j] += part[(u * VEC + j) * kGradThreads + g * 32 + lane];
        write_row<O, VEC, U>(a, f.z, c0, 32, vecs, sum);
      }
    }
  }
}

// ---- the gradient over a blocked order -------------------------------------------------------
// Narrow rows: a CTA brings the gradients of one run of bags into shared memory and sums the rows of
// its share of the table over them: 2 bytes a token are read from device memory, the gradient's
// values from shared memory, where 32 random words take three to four cycles.  (Gathered through the
// second-level cache, 4 bytes of a 32-byte sector each, the same sums of 128 M leaf tokens took 478 us,
// that cache's bandwidth; a few lanes a row instead of a stream, 162 us.)
//
// A warp walks the vectors of up to 32 rows as one stream, 32 vectors at a time: a lane sums its vector's eight
// values, a segmented sum over the lanes adds up the vectors of a row, and what is left of a row at the
// end of the 32 is carried on.  Every address is known in advance, so the next vectors are on their way.
// Three CTAs an SM hold 60 warps: 110 us for 128 M tokens, against 137 with 48 of them.
constexpr int kNarrowThreads = 640;
template <typename T, int DIM>
__global__ void __launch_bounds__(kNarrowThreads, DIM == 1 ? 3 : 1) narrow_grad_kernel(LookupGradLaunch a, TokenOrder o, float *__restrict__ partial) {
  extern __shared__ float grads[];  // [kBlockBags][DIM], and zeros for kNoBag
  overlap_release();
  overlap_wait();
  const long long bag0 = (long long)blockIdx.y * kBlockBags;
  const int n = int(min((long long)kBlockBags, o.bags - bag0));
  for (int i = threadIdx.x; i < n * DIM; i += kNarrowThreads) {
    const int r = i / DIM, d = i - r * DIM;
    grads[i] = to_f32(static_cast<const T *>(a.grad)[(bag0 + r) * a.grad_stride + d]);
  }
  if (threadIdx.x < DIM) grads[kBlockBags * DIM + threadIdx.x] = 0.0f;
  __syncthreads();
  const unsigned *begin = o.vec_begin + size_t(blockIdx.y) * (o.rows + 1);
  float *out = partial + size_t(blockIdx.y) * o.rows * DIM;
  const int lane = threadIdx.x & 31;
  const unsigned below = (2u << lane) - 1u;  // this lane and those before it
  const long long v_end = min((long long)o.rows, (blockIdx.x + 1ll) * a.rows_per_cta);
  const int span = a.rows_per_warp;  // at most 32
  for (long long v0 = blockIdx.x * (long long)a.rows_per_cta + threadIdx.x / 32 * span; v0 < v_end; v0 += kNarrowThreads / 32 * span) {
    // lane l looks after row v0 + l: its vectors are first .. last
    const bool mine = lane < span && v0 + lane < v_end;
    const long long v = min(v0 + min(lane, span - 1), (long long)v_end - 1);
    const unsigned first = begin[v], last = mine ? begin[v + 1] : first;
    const unsigned w_end = __shfl_sync(0xffffffffu, begin[v + 1], 31);
    unsigned w0 = __shfl_sync(0xffffffffu, first, 0);
    const uint4 *stream = reinterpret_cast<const uint4 *>(o.local) + lane;
    const uint4 none = make_uint4(kNoBag * 0x10001u, kNoBag * 0x10001u, kNoBag * 0x10001u, kNoBag * 0x10001u);
    float total[DIM], carry[DIM];
#pragma unroll
    for (int d = 0; d < DIM; ++d) total[d] = carry[d] = 0.0f;
    uint4 ids = w0 + lane < w_end ? stream[w0] : none;
    for (; w0 < w_end; w0 += 32) {
      const uint4 next = w0 + 32 + lane < w_end ? stream[w0 + 32] : none;
      const unsigned word[4] = {ids.x, ids.y, ids.z, ids.w};
      float sum[DIM];
#pragma unroll
      for (int d = 0; d < DIM; ++d) sum[d] = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned offset = (j % 2 ? word[j / 2] >> 16 : word[j / 2] & 0xFFFFu) * DIM;
#pragma unroll
        for (int d = 0; d < DIM; ++d) sum[d] += *reinterpret_cast<const float *>(reinterpret_cast<const char *>(grads) + offset + 4 * d);
      }
      // lanes whose vector is the first of its row
      const unsigned starts = __reduce_or_sync(0xffffffffu, first != last && first - w0 < 32u ? 1u << (first - w0) : 0u);
      const unsigned before = starts & below;
      const int from = before ? 31 - __clz(before) : 0;  // first lane of this lane's row
#pragma unroll
      for (int d = 0; d < DIM; ++d) {
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const float x = __shfl_up_sync(0xffffffffu, sum[d], s);
          if (lane - s >= from) sum[d] += x;
        }
        if (!before) sum[d] += carry[d];  // the row began in an earlier 32
        carry[d] = __shfl_sync(0xffffffffu, sum[d], 31);
        const float x = __shfl_sync(0xffffffffu, sum[d], int(last - 1 - w0) & 31);
        if (first != last && last - 1 - w0 < 32u) total[d] = x;
      }
      ids = next;
    }
    if (mine)
#pragma unroll
      for (int d = 0; d < DIM; ++d) out[(v0 + lane) * DIM + d] = total[d];
  }
}

// Wider rows over a blocked order: a group of tx lanes takes a row's columns over a share of the runs
// (blockIdx.z of `splits`), from device memory.  A share of a row that every bag names is one group's sum
// over a hundred thousand bags and more, so it is held in 64 bits: left to right in fp32 a sum of 100003
// equal values was off by 8200 half steps.  Bound by that chain where rows are few: 65536 bags of 4 over
// 2 x 8 fp32 columns keep 5 CTAs busy.
template <typename T, int VEC>
__global__ void __launch_bounds__(kGradThreads, 4) blocked_grad_kernel(LookupGradLaunch a, TokenOrder o, int tx_bits, int vecs,
                                                                    int chunks, int splits, float *__restrict__ partial) {
  overlap_release();
  overlap_wait();
  const int tx = 1 << tx_bits, lane = threadIdx.x & (tx - 1);
  const long long v = blockIdx.x * (long long)(kGradThreads >> tx_bits) + (threadIdx.x >> tx_bits);
  if (v >= o.rows) return;
  const int k0 = int((long long)o.blocks * blockIdx.z / splits), k1 = int((long long)o.blocks * (blockIdx.z + 1) / splits);
  for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
    const int c = chunk * tx + lane;
    if (c >= vecs) continue;
    const T *grad = static_cast<const T *>(a.grad) + (long long)c * VEC;
    double total[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) total[j] = 0.0;
    for (int k = k0; k < k1; ++k) {
      const unsigned *begin = o.vec_begin + size_t(k) * (o.rows + 1) + v;
      const long long bag0 = (long long)k * kBlockBags;
      const unsigned end = begin[1];
      for (unsigned w = begin[0]; w < end; ++w) {
        const uint4 ids = reinterpret_cast<const uint4 *>(o.local)[w];
        const unsigned word[4] = {ids.x, ids.y, ids.z, ids.w};
        Vec<T, VEC> x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned id = i % 2 ? word[i / 2] >> 16 : word[i / 2] & 0xFFFFu;
          x[i].clear();
          if (id != kNoBag) x[i].load(grad + (bag0 + id / 4) * a.grad_stride);
        }
        float sum[VEC];  // of eight bags: seven additions
        x[0].get(sum);
#pragma unroll
        for (int i = 1; i < 8; ++i) x[i].add_to(sum);
#pragma unroll
        for (int j = 0; j < VEC; ++j) total[j] += double(sum[j]);
      }
    }
    // one rounding a share; the shares are joined in 64 bits again
    float *out = partial + ((size_t(blockIdx.z) * o.rows + v) * vecs + c) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = float(total[j]);
  }
}

// the shares' sums, in 64 bits (there may be 65535 of them): eight groups of lanes take every eighth
// share, and their sums are added in order
template <typename O>
__global__ void __launch_bounds__(kGradThreads) blocked_join_kernel(LookupGradLaunch a, long long rows, int splits,
                                                                    const float *__restrict__ partial) {
  __shared__ double part[kGradThreads];
  constexpr int kSlices = kGradThreads / 32;
  overlap_release();
  overlap_wait();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long long n = rows * a.dim;
  for (long long i0 = blockIdx.x * 32ll; i0 < n; i0 += gridDim.x * 32ll) {
    const long long i = i0 + lane;
    double total = 0.0;
    if (i < n)
#pragma unroll 8
      for (int k = slice; k < splits; k += kSlices) total += double(partial[size_t(k) * n + i]);
    __syncthreads();
    part[threadIdx.x] = total;
    __syncthreads();
    if (slice != 0 || i >= n) continue;
#pragma unroll
    for (int g = 1; g < kSlices; ++g) total += part[g * 32 + lane];
    const float sum = float(total) * a.scale;
    O *at = static_cast<O *>(a.out) + i / a.dim * a.out_stride + i % a.dim;
    if (!a.accumulate) from_f32(sum, *at);
    else if (sum != 0.0f) from_f32(to_f32(*at) + sum, *at);  // a row without bags keeps its bits
  }
}

// ---- the sort of a batch in one launch -------------------------------------------------------
// Up to 32768 tokens are sorted by one cluster of at most eight CTAs: the pairs stay in shared
// memory, a pass exchanges digit counts and moves the pairs through distributed shared memory, and
// the rows' first positions and the items come out of the same launch.  Bound by latency: barriers and
// dependent accesses.  (The general sort takes three launches a pass and leaves the device to a few
// tiles at these sizes: 16384 tokens over 131072 rows took 109 us in it, 18 here.)
namespace cg = cooperative_groups;
constexpr int kClusterThreads = 512, kClusterWarps = kClusterThreads / 32;
constexpr int kMostClusterBits = 9, kMostClusterDigits = 1 << kMostClusterBits;
static_assert(kMostClusterDigits == kClusterThreads, "a thread takes a digit");
constexpr int kMostClusterItems = 8;

struct ClusterSortMemory {
  unsigned short warp_cnt[kClusterWarps][kMostClusterDigits];
  unsigned cta_cnt[kMostClusterDigits];
  unsigned base[kMostClusterDigits];
  unsigned warp_sum[kClusterWarps];
};

template <int ITEMS>
__global__ void __launch_bounds__(kClusterThreads) order_cluster_kernel(SortPass p, TokenOrder o, int digit_bits, int passes, bool clear) {
  extern __shared__ __align__(16) unsigned char raw[];
  uint2 *pair = reinterpret_cast<uint2 *>(raw);
  ClusterSortMemory &m = *reinterpret_cast<ClusterSortMemory *>(raw + sizeof(uint2) * kClusterThreads * ITEMS);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = int(cluster.block_rank()), ctas = int(cluster.num_blocks());
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  constexpr int kSpan = kClusterThreads * ITEMS;  // pairs of a CTA
  const int digits = 1 << digit_bits;
  const int at0 = w * (ITEMS * 32) + lane;  // this thread's pairs: at0, at0 + 32, ..
  unsigned key[ITEMS], bag[ITEMS], rank_in[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const long long i = (long long)rank * kSpan + at0 + j * 32;
    key[j] = 0xffffffffu;  // behind everything, empty slots included: it comes after them and digits are stable
    bag[j] = 0;
    if (i < p.n) sort_pair(p, i, key[j], bag[j]);
  }
  if (rank == 0 && tid < 2) o.counts[tid] = 0;
  if (clear)
    for (long long i = (long long)rank * kClusterThreads + tid; i < (p.rows + 15) / 16; i += ctas * kClusterThreads)
      reinterpret_cast<uint4 *>(o.named)[i] = make_uint4(0u, 0u, 0u, 0u);  // padded to 256 bytes
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    for (int i = tid; i < kClusterWarps * kMostClusterDigits / 2; i += kClusterThreads)
      reinterpret_cast<unsigned *>(&m.warp_cnt[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const unsigned digit = (key[j] >> shift) & (digits - 1);
      const unsigned same = lanes_with(digit, digit_bits);
      const unsigned below = __popc(same & ((1u << lane) - 1u));
      rank_in[j] = m.warp_cnt[w][digit] + below;
      __syncwarp();
      if (below == 0) m.warp_cnt[w][digit] += (unsigned short)__popc(same);
      __syncwarp();
    }
    __syncthreads();
    if (tid < digits) {
      unsigned c[kClusterWarps], run = 0;
#pragma unroll
      for (int i = 0; i < kClusterWarps; ++i) c[i] = m.warp_cnt[i][tid];
#pragma unroll
      for (int i = 0; i < kClusterWarps; ++i) {
        m.warp_cnt[i][tid] = (unsigned short)run;  // below kSpan
        run += c[i];
      }
      m.cta_cnt[tid] = run;
    }
    cluster.sync();  // the counts are there, and every CTA holds its pairs in registers
    unsigned before = 0, total = 0;
    if (tid < digits) {
      unsigned c[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) c[r] = r < ctas ? cluster.map_shared_rank(m.cta_cnt, r)[tid] : 0u;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r < rank) before += c[r];
        total += c[r];
      }
    }
    // exclusive sum of the digits' totals
    unsigned x = total;
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) m.warp_sum[w] = x;
    __syncthreads();
    unsigned ahead = 0;
#pragma unroll
    for (int i = 0; i < kClusterWarps; ++i) ahead += i < w ? m.warp_sum[i] : 0u;
    m.base[tid] = ahead + x - total + before;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const unsigned digit = (key[j] >> shift) & (digits - 1);
      const unsigned to = m.base[digit] + m.warp_cnt[w][digit] + rank_in[j];
      cluster.map_shared_rank(pair, int(to / kSpan))[to % kSpan] = make_uint2(key[j], bag[j]);
    }
    cluster.sync();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const uint2 v = pair[at0 + j * 32];
      key[j] = v.x;
      bag[j] = v.y;
    }
  }
  const long long q0 = (long long)rank * kSpan + w * (ITEMS * 32);
  if (q0 < p.n) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (q0 + j * 32 + lane < p.n) o.bag[q0 + j * 32 + lane] = bag[j];
    add_items<ITEMS>(o, q0, key, [&](unsigned i) {
      return int(i / kSpan) == rank ? pair[i % kSpan].x : cluster.map_shared_rank(pair, int(i / kSpan))[i % kSpan].x;
    });
  }
  cluster.sync();  // no CTA's memory goes while another may look at it
}

inline int grid_of(long long n, int threads, int per_sm) {
  return int(std::max<long long>(1, std::min<long long>((n + threads - 1) / threads, (long long)device_sm_count() * per_sm)));
}

int key_bits(int64_t rows) {  // keys are 0 .. rows
  int b = 1;
  while ((uint64_t(rows) >> b) != 0) ++b;
  return b;
}

int64_t tiles_of(int64_t n) {
  const int64_t tile = kSortThreads * (n < kManyTokens ? kFewItems : kManyItems);
  return (n + tile - 1) / tile;
}
template <int ITEMS>
void sort_pass(const SortPass &p, cudaStream_t s) {
  constexpr int smem = kSortThreads * ITEMS * int(sizeof(uint2));
  static bool ready[kMaxDevices] = {};
  const int dev = current_device();
  if (!ready[dev]) {
    ARB_CUDA(cudaFuncSetAttribute(sort_move_kernel<ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    ready[dev] = true;
  }
  launch_overlapped(sort_count_kernel<ITEMS>, dim3(p.tiles), dim3(kSortThreads), 0, s, p);
  launch_overlapped(sort_scan_kernel, dim3(kDigits), dim3(256), 0, s, p);
  launch_overlapped(sort_move_kernel<ITEMS>, dim3(p.tiles), dim3(kSortThreads), smem, s, p);
  count_launch(3);
}

// scratch of the sort: two buffers of pairs, the digit counts
struct SortScratch {
  unsigned *key[2], *bag[2], *counts, *totals;
  size_t bytes;
  SortScratch(void *mem, int64_t n) {
    const size_t pair = (size_t(n) * 4 + 255) / 256 * 256;
    const size_t tiles = size_t(tiles_of(n));
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

// Elements a thread may move in one access: the widest of 16, 8 and 4 bytes and one element that
// the columns, the distances of the rows and both starts allow.
int vec_of(int type, int64_t dim, const void *p, int64_t stride, const void *q, int out_type, int64_t out_stride) {
  const int widths[3] = {int(16 / elem_size(type)), int(8 / elem_size(type)), int(4 / elem_size(type))};
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
  const bool pooled = a.tokens.per_bag != 1;
  // one token a bag: 64 bytes of a wide row a lane, in vectors as wide as its alignment allows
  constexpr int kWide = std::min(8, 64 / (VEC * int(sizeof(T))));
  const int u = !pooled && vecs >= 32 * kWide ? kWide : 1;
  LaneShape sh;
  // lanes across the columns: enough for the row, at most half a CTA
  sh.tx_bits = std::min(7, log2_floor(std::max<int64_t>(1, (vecs + u - 1) / u * 2 - 1)));
  // lanes along the tokens: where a bag's tokens lie side by side a narrow group reads them as one
  // line, and where the bags alone do not fill the device they share the loop
  const int64_t threads_wanted = int64_t(device_sm_count()) * 1024;
  const int64_t have = a.tokens.bags * vecs;
  const bool side_by_side = std::abs(a.tokens.token_stride) < std::abs(a.tokens.bag_stride);
  sh.ly_bits = 0;
  while (pooled && sh.tx_bits + sh.ly_bits < 8 && (int64_t(4) << sh.ly_bits) < a.tokens.per_bag &&
         ((have << sh.ly_bits) < threads_wanted || (side_by_side && sh.tx_bits + sh.ly_bits < 3)))
    ++sh.ly_bits;
  if constexpr (VEC == 1 && sizeof(T) == 2 && std::is_same<T, O>::value) {
    if (u > 1) {  // a wide row
      constexpr int kWords = 8;
      const int runs = int((a.dim / 2 + 1 + 32 * kWords - 1) / (32 * kWords));
      const dim3 grid(unsigned((a.tokens.bags + kLookupThreads / 32 - 1) / (kLookupThreads / 32)), unsigned(std::min(runs, 65535)));
      lookup_odd_rows_kernel<T, kWords><<<grid, kLookupThreads, 0, s>>>(a, runs);
      return;
    }
  }
  const int groups = kLookupThreads >> (sh.tx_bits + sh.ly_bits);
  const int chunks = int((vecs + (int64_t(u) << sh.tx_bits) - 1) / (int64_t(u) << sh.tx_bits));
  const dim3 grid(unsigned((a.tokens.bags + groups - 1) / groups), unsigned(std::min(chunks, 65535)));
  const bool together = sh.tx_bits >= 3, long_bags = a.tokens.per_bag > int64_t(kChain) << sh.ly_bits;
  if (long_bags && together) lookup_kernel<T, O, VEC, true, true><<<grid, kLookupThreads, 0, s>>>(a, sh, int(vecs), chunks);
  else if (long_bags) lookup_kernel<T, O, VEC, false, true><<<grid, kLookupThreads, 0, s>>>(a, sh, int(vecs), chunks);
  else if (pooled && together) lookup_kernel<T, O, VEC, true, false><<<grid, kLookupThreads, 0, s>>>(a, sh, int(vecs), chunks);
  else if (pooled) lookup_kernel<T, O, VEC, false, false><<<grid, kLookupThreads, 0, s>>>(a, sh, int(vecs), chunks);
  else if (u > 1) lookup_rows_kernel<T, O, VEC, kWide><<<grid, kLookupThreads, 0, s>>>(a, sh.tx_bits, int(vecs), chunks);
  else lookup_rows_kernel<T, O, VEC, 1><<<grid, kLookupThreads, 0, s>>>(a, sh.tx_bits, int(vecs), chunks);
}

constexpr size_t kMostTableBytes = 200 << 10;  // of shared memory, one CTA an SM
// Tokens of a bag that one thread adds up in fp32.  Setting sums aside like lookup_kernel costs the usual
// bags 5 % here (122 us instead of 115 for a million of 128 tokens), and a table of more trees that fits
// has no more than a dozen leaves a tree.
constexpr int64_t kMostTableTokens = 4 * kChain;

template <typename T, typename O, typename I, int DIM>
void lookup_table_with(const LookupLaunch &a, cudaStream_t s) {
  static bool ready[kMaxDevices] = {};
  const int dev = current_device();
  if (!ready[dev]) {
    ARB_CUDA(cudaFuncSetAttribute(lookup_table_kernel<T, O, I, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  int(kMostTableBytes)));
    ready[dev] = true;
  }
  const size_t smem = size_t(a.rows + 1) * DIM * sizeof(float);
  const bool paired = a.tokens.bag_stride == 1 && a.tokens.token_stride % 2 == 0 &&
                      reinterpret_cast<uintptr_t>(a.tokens.at) % (2 * sizeof(I)) == 0;
  // as many rounds as 1024 threads an SM need, and then no more threads than fill them evenly
  const int64_t pairs = (a.tokens.bags + 1) / 2, sms = device_sm_count();
  const int64_t rounds = (pairs + sms * kTableThreads - 1) / (sms * kTableThreads);
  const int threads = int(std::max<int64_t>(256, ((pairs + sms * rounds - 1) / (sms * rounds) + 31) / 32 * 32));
  lookup_table_kernel<T, O, I, DIM><<<int(sms), threads, smem, s>>>(a, paired);
}

template <typename T, typename O>
bool lookup_table(const LookupLaunch &a, cudaStream_t s) {
  // Instances are there for one to three columns (a leaf's values for a few classes); wider rows go through
  // the cache.  Only where the bags of one slot lie next to one another, the table fits, the lookups are many times
  // the words every SM has to copy first, and a thread's chain of additions is not too long.
  const TokenView &t = a.tokens;
  if (a.dim > 3 || t.per_bag < 2 || t.per_bag > kMostTableTokens || std::abs(t.bag_stride) >= std::abs(t.token_stride) ||
      size_t(a.rows + 1) * size_t(a.dim) * sizeof(float) > kMostTableBytes ||
      t.count() < 4 * a.rows * device_sm_count())
    return false;
#define ARB_DIM(D)                                                     \
  if (a.dim == D) {                                                    \
    if (t.bytes == 4) lookup_table_with<T, O, int32_t, D>(a, s);       \
    else lookup_table_with<T, O, int64_t, D>(a, s);                    \
  }
  ARB_DIM(1) ARB_DIM(2) ARB_DIM(3)
#undef ARB_DIM
  return true;
}

}  // namespace

void launch_lookup(const LookupLaunch &a, cudaStream_t s) {
  if (a.tokens.bags == 0 || a.dim == 0) return;
  const int vec = vec_of(a.type, a.dim, a.table, a.row_stride, a.out, a.out_type, a.out_stride);
#define ARB_CALL(T, O)                                                      \
  if (lookup_table<T, O>(a, s)) {}                                          \
  else if (vec * sizeof(T) == 16) lookup_with<T, O, 16 / sizeof(T)>(a, s);  \
  else if (vec * sizeof(T) == 8) lookup_with<T, O, 8 / sizeof(T)>(a, s);    \
  else if (vec > 1) lookup_with<T, O, 4 / sizeof(T)>(a, s);                 \
  else lookup_with<T, O, 1>(a, s)
  ARB_BY_TYPE(a.type, a.out_type, ARB_CALL);
#undef ARB_CALL
  ARB_CUDA(cudaGetLastError());
  count_launch();
}

namespace {
size_t pad256(size_t b) { return (b + 255) / 256 * 256; }
// Bags of a piece: few tokens want short pieces, so that a frequent row is shared widely (2340 tokens of
// which some come 300 times: 40 us with 16, 57 with 32), but not so short that ordinary rows are cut
// (20275 slots over 367 rows of 1392 columns: 57 with 16, 39 with 32); a large batch has pieces enough,
// and longer ones cost fewer partial sums.
unsigned piece_of(int64_t count, int64_t rows) {
  unsigned p = count / 8 < rows ? 16 : 32;
  while (p < 4096 && int64_t(p) * 8192 < count) p *= 2;
  return p;
}
}  // namespace

namespace {
constexpr int64_t kMostClusterTokens = int64_t(8) * kClusterThreads * kMostClusterItems;
// An order is kept by runs of bags where a row has 32 bags a run or more, on average: then a run's
// sums are worth more than the look at where its bags begin.  Chosen for rows of up to three columns,
// whose gradients of a run fit shared memory; an order does not know the columns, so wider rows over few
// rows take it too, at the price named at blocked_grad_kernel.
int blocks_of(int64_t bags, int64_t per_bag, int64_t rows) {
  const int64_t blocks = (bags + kBlockBags - 1) / kBlockBags;
  const bool many = per_bag > 1 && bags * per_bag > kMostClusterTokens && bags * per_bag >= 32 * rows * blocks;
  return many && blocks < 65536 && blocks * (rows + 1) < (int64_t(1) << 31) ? int(blocks) : 1;
}
}  // namespace

TokenOrder::TokenOrder(void *mem, int64_t bags_, int64_t per_bag, int64_t rows_)
    : bags(bags_), count(bags_ * per_bag), rows(rows_), blocks(blocks_of(bags_, per_bag, rows_)), piece(piece_of(count, rows_)) {
  size_t at = 0;
  auto take = [&](size_t b) {
    char *q = static_cast<char *>(mem) + at;
    at += pad256(b);
    return static_cast<void *>(q);
  };
  counts = static_cast<unsigned *>(take(256));
  bag = nullptr, local = nullptr, vec_begin = nullptr, frequent = item = nullptr, named = nullptr;
  if (blocks > 1) {
    vec_begin = static_cast<unsigned *>(take(size_t(segments() + 1) * 4));
    local = static_cast<unsigned short *>(take(size_t(most_vectors()) * 16));
  } else {
    named = static_cast<unsigned char *>(take(size_t(rows)));
    bag = static_cast<unsigned *>(take(size_t(count) * 4));
    item = static_cast<uint4 *>(take(size_t(most_items()) * 16));
    frequent = static_cast<uint4 *>(take(size_t(count / piece + 1) * 16));
  }
  bytes = at;
}

namespace {
int vec_tiles(const TokenOrder &o) { return int((o.segments() + 1 + kVecTile - 1) / kVecTile); }
}  // namespace

size_t token_order_scratch(const TokenOrder &o) {
  if (o.count <= kMostClusterTokens) return 0;
  const size_t vectors = o.blocks > 1 ? pad256(size_t(o.segments() + 1) * 4) + pad256(size_t(vec_tiles(o)) * 4) : 0;
  return SortScratch(nullptr, o.count).bytes + vectors;
}

namespace {
template <int ITEMS>
void launch_cluster_order(const SortPass &p, const TokenOrder &o, bool clear, cudaStream_t s) {
  constexpr size_t smem = sizeof(uint2) * kClusterThreads * ITEMS + sizeof(ClusterSortMemory);
  static bool ready[kMaxDevices] = {};  // setting it twice does no harm
  const int dev = current_device();
  if (!ready[dev]) {
    ARB_CUDA(cudaFuncSetAttribute(order_cluster_kernel<ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    ready[dev] = true;
  }
  int ctas = 1;
  while (int64_t(ctas) * kClusterThreads * ITEMS < p.n) ctas *= 2;
  const int bits = key_bits(o.rows), passes = (bits + kMostClusterBits - 1) / kMostClusterBits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ctas);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ARB_CUDA(cudaLaunchKernelEx(&cfg, order_cluster_kernel<ITEMS>, p, o, (bits + passes - 1) / passes, passes, clear));
  count_launch();
}
}  // namespace

void launch_token_order(const TokenView &t, const TokenOrder &o, void *scratch, cudaStream_t s) {
  const int64_t n = t.count();
  SortPass p = {};
  p.tokens = t;
  p.rows = o.rows;
  p.n = n;
  p.first = true;
  p.by_slot = std::abs(t.bag_stride) < std::abs(t.token_stride);
  if (n > 0 && n <= kMostClusterTokens) {
    const bool clear = o.rows <= kFewRows;  // else the marks are cleared by the whole device
    if (!clear) ARB_CUDA(cudaMemsetAsync(o.named, 0, size_t(o.rows), s));
    if (n <= kFewTokens) {
      order_few_kernel<<<1, kFewTokens, 0, s>>>(p, o, clear);
      ARB_CUDA(cudaGetLastError());
      count_launch();
    } else if (n <= int64_t(8) * kClusterThreads * 4) {
      launch_cluster_order<4>(p, o, clear, s);
    } else {
      launch_cluster_order<kMostClusterItems>(p, o, clear, s);
    }
    return;
  }
  const int64_t keys = o.blocks * (o.rows + 1) - 1;  // the largest key
  const unsigned *sorted = nullptr, *sorted_bag = nullptr;
  if (n > 0) {
    const SortScratch sc(scratch, n);
    const int passes = (key_bits(keys) + kDigitBits - 1) / kDigitBits;
    p.tiles = int(tiles_of(n));
    p.counts = sc.counts;
    p.totals = sc.totals;
    p.blocked = o.blocks > 1;
    // The first pass clears what the items count in and mark: two launches fewer, and the items' kernel
    // follows the sort without a gap (38933 bags of 181 rows with their gradient: 42 us, 35 so). With
    // more than 16 rows a token its blocks would have more to clear than to sort: a fill by the whole device.
    const bool clear = o.blocks == 1 && o.rows <= 16 * n;
    if (o.blocks == 1 && !clear) {
      ARB_CUDA(cudaMemsetAsync(o.counts, 0, 2 * sizeof *o.counts, s));
      ARB_CUDA(cudaMemsetAsync(o.named, 0, size_t(o.rows), s));
    }
    for (int i = 0; i < passes; ++i) {
      const bool last = i == passes - 1;
      p.first = i == 0;
      p.clear_counts = i == 0 && clear ? o.counts : nullptr;
      p.clear_named = i == 0 && clear ? o.named : nullptr;
      p.shift = i * kDigitBits;
      p.key_in = sc.key[(i + 1) & 1];
      p.bag_in = sc.bag[(i + 1) & 1];
      p.key_out = sc.key[i & 1];
      p.bag_out = last && o.blocks == 1 ? o.bag : sc.bag[i & 1];
      if (n < kManyTokens) sort_pass<kFewItems>(p, s);
      else sort_pass<kManyItems>(p, s);
    }
    sorted = sc.key[(passes - 1) & 1];
    sorted_bag = sc.bag[(passes - 1) & 1];
  }
  if (o.blocks > 1) {
    const SortScratch sc(scratch, n);
    unsigned *begin = reinterpret_cast<unsigned *>(static_cast<char *>(scratch) + sc.bytes);
    unsigned *tile = begin + pad256(size_t(o.segments() + 1) * 4) / 4;
    order_begin_kernel<<<grid_of(n + 1, 256, 8), 256, 0, s>>>(sorted, n, o.segments(), begin);
    vec_count_kernel<<<vec_tiles(o), 256, 0, s>>>(begin, o, tile);
    vec_tiles_kernel<<<1, 256, 0, s>>>(tile, vec_tiles(o));
    vec_begin_kernel<<<vec_tiles(o), 256, 0, s>>>(begin, o, tile);
    vec_move_kernel<<<grid_of(n, 256, 8), 256, 0, s>>>(sorted, sorted_bag, begin, o);
    count_launch(5);
  } else {
    if (n > 0) {
      launch_overlapped(order_items_kernel, dim3(grid_of(n, 256, 8)), dim3(256), 0, s, o, sorted);
      count_launch();
    } else {  // no sort has cleared them
      ARB_CUDA(cudaMemsetAsync(o.counts, 0, 2 * sizeof *o.counts, s));
      if (o.rows > 0) ARB_CUDA(cudaMemsetAsync(o.named, 0, size_t(o.rows), s));
    }
  }
  ARB_CUDA(cudaGetLastError());
}

namespace {

// shares a row's runs are divided into: one run a share where they fit shared memory, else as many
// shares as it takes to fill the device, but no more than there are runs
int splits_of(const TokenOrder &o, int64_t dim) {
  if (dim <= 3) return o.blocks;
  const int64_t lanes = std::max<int64_t>(1, o.rows * ((dim + 7) / 8));
  const int64_t want = (int64_t(device_sm_count()) * 2048 + lanes - 1) / lanes;
  return int(std::max<int64_t>(1, std::min<int64_t>(o.blocks, want)));
}

template <typename T, int DIM>
void narrow_grad_with(LookupGradLaunch a, const TokenOrder &o, float *partial, cudaStream_t s) {
  static bool ready[kMaxDevices] = {};
  const int dev = current_device();
  constexpr int smem = (kBlockBags + 1) * DIM * int(sizeof(float));
  if (!ready[dev]) {
    ARB_CUDA(cudaFuncSetAttribute(narrow_grad_kernel<T, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    ready[dev] = true;
  }
  // shares of the table a run: a few CTAs for every place on the device, so that the last ones fill it;
  // with few rows the warps take fewer of them at a time
  const int64_t places = device_sm_count() * (DIM == 1 ? 3 : 1);
  const int64_t shares = std::max<int64_t>(1, (4 * places + o.blocks - 1) / o.blocks);
  constexpr int kWarps = kNarrowThreads / 32;
  a.rows_per_warp = 32;
  while (a.rows_per_warp > 2 && o.blocks * ((o.rows + kWarps * a.rows_per_warp - 1) / (kWarps * a.rows_per_warp)) < 2 * places)
    a.rows_per_warp /= 2;
  const int64_t step = kWarps * a.rows_per_warp;  // rows a CTA takes at a time
  a.rows_per_cta = int(std::max<int64_t>(step, ((o.rows + shares - 1) / shares + step - 1) / step * step));
  const dim3 grid(unsigned((o.rows + a.rows_per_cta - 1) / a.rows_per_cta), unsigned(o.blocks));
  launch_overlapped(narrow_grad_kernel<T, DIM>, grid, dim3(kNarrowThreads), smem, s, a, o, partial);
}

template <typename T, int VEC>
void blocked_grad_with(const LookupGradLaunch &a, const TokenOrder &o, int splits, float *partial, cudaStream_t s) {
  const int vecs = int(a.dim / VEC);
  const int tx_bits = std::min(5, log2_floor(std::max(1, vecs * 2 - 1)));
  const int chunks = (vecs + (1 << tx_bits) - 1) >> tx_bits;
  const int64_t groups = kGradThreads >> tx_bits;
  const dim3 grid(unsigned((o.rows + groups - 1) / groups), unsigned(std::min(chunks, 65535)), unsigned(splits));
  launch_overlapped(blocked_grad_kernel<T, VEC>, grid, dim3(kGradThreads), 0, s, a, o, tx_bits, vecs, chunks, splits, partial);
}

template <typename T, typename O>
void blocked_grad(const LookupGradLaunch &a, const TokenOrder &o, int vec, float *partial, cudaStream_t s) {
  const int splits = splits_of(o, a.dim);
  ARB_CHECK(a.dim / vec <= (int64_t(1) << 30), "rows of more than 2^30 vectors");
  if (a.dim == 1) narrow_grad_with<T, 1>(a, o, partial, s);
  else if (a.dim == 2) narrow_grad_with<T, 2>(a, o, partial, s);
  else if (a.dim == 3) narrow_grad_with<T, 3>(a, o, partial, s);
  else if (vec >= 4) blocked_grad_with<T, 4>(a, o, splits, partial, s);
  else if (vec * sizeof(T) >= 4) blocked_grad_with<T, 4 / sizeof(T)>(a, o, splits, partial, s);
  else blocked_grad_with<T, 1>(a, o, splits, partial, s);
  launch_overlapped(blocked_join_kernel<O>, dim3(grid_of(o.rows * a.dim, 32, 32)), dim3(kGradThreads), 0, s, a,
                    (long long)o.rows, splits, static_cast<const float *>(partial));
  count_launch();
}

}  // namespace

size_t lookup_grad_scratch(const TokenOrder &o, int64_t dim) {
  if (o.blocks > 1) return pad256(size_t(splits_of(o, dim)) * size_t(o.rows) * size_t(dim) * sizeof(float));
  return o.count > o.piece ? pad256((size_t(o.count / o.piece) + 1) * 2 * size_t(dim) * sizeof(float)) : 0;
}

namespace {

// CTAs of the sums' kernel that the device holds at once
template <typename T, typename O, int VEC, int U, bool ODD>
int64_t resident_sums() {
  static int ctas[kMaxDevices] = {};
  const int dev = current_device();
  if (!ctas[dev]) {
    int n = 0;
    ARB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, lookup_grad_kernel<T, O, VEC, U, ODD>, kGradThreads, 0));
    ctas[dev] = std::max(1, n);
  }
  return int64_t(ctas[dev]) * device_sm_count();
}

template <typename T, typename O, int VEC, int U, bool ODD = false>
void lookup_grad_with(const LookupGradLaunch &a, const TokenOrder &o, float *partial, cudaStream_t s) {
  const int vecs = int((a.dim + VEC - 1) / VEC);
  GradLanes sh;
  sh.tx_bits = std::min(5, log2_floor(std::max(1, (vecs + U - 1) / U * 2 - 1)));
  // a row has count / rows bags, a piece no more than `piece`: that many lanes share them
  const int64_t length = std::min<int64_t>(o.piece, o.count / std::max<int64_t>(1, std::min(o.count, o.rows)));
  sh.ly_bits = 0;
  while (sh.tx_bits + sh.ly_bits < 5 && (int64_t(1) << sh.ly_bits) < length) ++sh.ly_bits;
  const int64_t zero_words = (a.dim * int64_t(sizeof(O)) + 15) / 16;
  sh.zero_bits = int(std::min(8, log2_floor(std::max<int64_t>(1, zero_words * 2 - 1))));
  sh.chunks = (vecs + (U << sh.tx_bits) - 1) / (U << sh.tx_bits);
  const int64_t groups = kGradThreads >> (sh.tx_bits + sh.ly_bits);
  const int64_t item_blocks = std::min<int64_t>((o.most_items() * sh.chunks + groups - 1) / groups, resident_sums<T, O, VEC, U, ODD>());
  const int64_t zero_groups = kGradThreads >> sh.zero_bits;
  const int64_t zero_blocks = a.accumulate ? 0 : (o.rows + zero_groups * kZeroRows - 1) / (zero_groups * kZeroRows);
  if (item_blocks + zero_blocks == 0) return;
  launch_overlapped(lookup_grad_kernel<T, O, VEC, U, ODD>, dim3(unsigned(item_blocks + zero_blocks)), dim3(kGradThreads), 0, s,
                    a, o, sh, vecs, unsigned(item_blocks), partial);
  if (o.count > o.piece) {
    constexpr int kWidth = ODD ? 1 : VEC, kJoin = kWidth < 4 ? 4 / kWidth : 1;
    const int join_vecs = int(a.dim / kWidth), join_chunks = (join_vecs + 32 * kJoin - 1) / (32 * kJoin);
    const dim3 join(unsigned(std::min<int64_t>(o.count / o.piece, device_sm_count() * 2)), unsigned(std::min(join_chunks, 65535)));
    launch_overlapped(lookup_grad_join_kernel<O, kWidth, kJoin>, join, dim3(kGradThreads), 0, s, a, o, join_vecs,
                      join_chunks, static_cast<const float *>(partial));
    count_launch();
  }
}

template <typename T, typename O, int VEC>
void lookup_grad_vec(const LookupGradLaunch &a, const TokenOrder &o, float *partial, cudaStream_t s) {
  ARB_CHECK(a.dim / VEC <= (int64_t(1) << 30), "rows of more than 2^30 vectors");
  // A wide row gives every lane up to four vectors and 32 bytes of it: more in flight for one look at the
  // row's bags.  With three bags in flight (sums alone, us): 16384 x 4096 bf16 198, 2340 x 5301 fp32 40;
  // two vectors and two bags 208 and -, four and eight 308 and -, eight vectors of one element 59 for the
  // latter: past 128 registers the SM holds too few warps.
  constexpr int kWide = std::min(4, 32 / (VEC * int(sizeof(T))));
  if constexpr (VEC == 1 && sizeof(T) == 2) {
    if (a.dim >= 256) {  // 16-bit rows that begin anywhere: words of two columns
      lookup_grad_with<T, O, 2, 4, true>(a, o, partial, s);
      return;
    }
  }
  if (a.dim / VEC >= 32 * kWide) lookup_grad_with<T, O, VEC, kWide>(a, o, partial, s);
  else lookup_grad_with<T, O, VEC, 1>(a, o, partial, s);
}

}  // namespace

void launch_lookup_grad(const LookupGradLaunch &a, const TokenOrder &o, void *scratch, cudaStream_t s) {
  if (o.rows == 0 || a.dim == 0) return;
  const int vec = vec_of(a.type, a.dim, a.grad, a.grad_stride, a.out, a.out_type, a.out_stride);
  float *partial = static_cast<float *>(scratch);
#define ARB_CALL(T, O)                                                             \
  if (o.blocks > 1) blocked_grad<T, O>(a, o, vec, partial, s);                      \
  else if (vec * sizeof(T) == 16) lookup_grad_vec<T, O, 16 / sizeof(T)>(a, o, partial, s); \
  else if (vec * sizeof(T) == 8) lookup_grad_vec<T, O, 8 / sizeof(T)>(a, o, partial, s); \
  else if (vec > 1) lookup_grad_vec<T, O, 4 / sizeof(T)>(a, o, partial, s);         \
  else lookup_grad_vec<T, O, 1>(a, o, partial, s)
  ARB_BY_TYPE(a.type, a.out_type, ARB_CALL);
#undef ARB_CALL
  ARB_CUDA(cudaGetLastError());
  count_launch();
}

}  // namespace arb
