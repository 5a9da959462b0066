// Operators on tables of learned rows (leaf values, embeddings): lookup, its gradient by sorted
// tokens, and the AdamW step over many tensors.  All launchers enqueue on the given stream, never
// synchronise and never allocate: outputs and scratch memory come from the caller, so that a call
// can be captured into a CUDA graph.
#pragma once
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <vector>

#include "common.cuh"

namespace arb {

enum ElemType { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline size_t elem_size(int t) { return t == kF32 ? 4 : 2; }

// Tokens of `bags` bags of `per_bag` each: token t of bag b is at[b * bag_stride + t * token_stride]
// (strides in elements, int32 or int64).  A token outside [0, rows) is an empty slot.
struct TokenView {
  const void *at;
  int bytes;  // 4 or 8
  int64_t bags, per_bag, bag_stride, token_stride;
  int64_t count() const { return bags * per_bag; }
};

struct LookupLaunch {
  const void *table;
  int type;
  int64_t rows, dim, row_stride;
  TokenView tokens;
  float scale;
  void *out;
  int out_type;
  int64_t out_stride;
};
void launch_lookup(const LookupLaunch &a, cudaStream_t s);

// The tokens' order, in memory of the caller: for every row v of the table, the bags that name it,
// in a fixed order that only the tokens decide.
//
// blocks == 1: the bags sorted by token, and the sorted positions cut into items of work.
// blocks > 1: many bags of several tokens over few rows (the leaves of a forest).  The order is kept
// apart for every run of kBlockBags bags, whose gradients fit into shared memory.  Bags are numbered
// from the run's first one, times four (the byte of a float), in 16 bits; within a run the bags of row v
// are vectors of eight, vec_begin[k * (rows + 1) + v] .. vec_begin[k * (rows + 1) + v + 1], the last one
// filled up with kNoBag: no vector holds bags of two rows, and all are 16-byte aligned.
constexpr int kBlockBags = 16383;
constexpr unsigned short kNoBag = kBlockBags * 4;
struct TokenOrder {
  int64_t bags, count, rows;
  int blocks;
  unsigned short *local;  // blocks > 1: eight a vector
  unsigned *vec_begin;    // blocks > 1: segments() + 1
  __host__ __device__ int64_t segments() const { return blocks * (rows + 1); }
  int64_t most_vectors() const { return count / 8 + blocks * rows + 1; }
  unsigned *bag;          // blocks == 1, and the rest: count
  // The bags of a row are cut at multiples of `piece` (a power of two) where two of these lie inside
  // them, so an item has fewer than 2 * piece bags.
  unsigned piece;
  uint4 *item;           // first position, end, row, 1 if these are all the row's bags
  uint4 *frequent;       // the same of a whole row that is cut
  unsigned char *named;  // per row: a bag names it
  unsigned *counts;      // items, cut rows
  int64_t most_items() const { return count / piece + (count < rows ? count : rows) + 1; }
  size_t bytes;
  TokenOrder(void *mem, int64_t bags, int64_t per_bag, int64_t rows);
};
size_t token_order_scratch(const TokenOrder &o);
void launch_token_order(const TokenView &t, const TokenOrder &o, void *scratch, cudaStream_t s);

struct LookupGradLaunch {
  const void *grad;  // [bags][dim], rows grad_stride apart (0: the same row for every bag)
  int type;
  int64_t dim, grad_stride;
  float scale;
  void *out;  // [rows][dim]
  int out_type;
  int64_t out_stride;
  bool accumulate;
  int rows_per_cta = 0, rows_per_warp = 0;  // set by the launcher
};
size_t lookup_grad_scratch(const TokenOrder &o, int64_t dim);
void launch_lookup_grad(const LookupGradLaunch &a, const TokenOrder &o, void *scratch, cudaStream_t s);

// ---- AdamW ---------------------------------------------------------------------------------
constexpr int kMomentBlock = 128;  // elements of an 8-bit block; tensors' slots are padded to it
// Elements a CTA takes: with few of them short chunks give every SM some and keep a CTA's chain of tiles
// short, with many the start of a CTA counts.  One tensor of bf16, no copy; moments in 8 bits (us for
// chunks of 2048 / 4096 / 8192):
// 1 M elements 8.5 / 10.5 / 14.5, 12 M 36 / 35 / 37, 24 M 71 / 68 / 70, 128 M 341 / 314 / 308; moments in
// 32 bits: 1 M 8.4 / 8.4 / 10.4, 4 M 20 / 17 / 17, 128 M 541 / 496 / 474.
constexpr int kLeastAdamWChunk = 2048;
inline int adamw_chunk(int64_t elements, int bits) {
  const int64_t few = int64_t(bits == 8 ? 8 : 2) << 20, many = int64_t(bits == 8 ? 48 : 4) << 20;
  return elements < few ? kLeastAdamWChunk : elements < many ? 4096 : 8192;
}

struct AdamWTensor {  // device table, one record a tensor
  void *param;
  long long n;
  long long slot;  // first element in the flat moment buffers, a multiple of kMomentBlock
  int type;
  int vec;         // the parameter is 16-byte aligned
};
struct AdamWChunk {
  int tensor;
  int index;  // elements index * chunk ..
};
struct AdamWState {  // device: the step count and what follows from it, advanced by the kernel
  double beta1_t, beta2_t;  // powers of the betas for the coming step
  double inv_bc1;           // 1 / (1 - beta1_t)
  float inv_root_bc2;       // 1 / sqrt(1 - beta2_t)
  unsigned done;            // CTAs of the running step that have finished
  long long step;           // steps taken
  float one;                // 1
  __host__ __device__ void derive() {
    inv_bc1 = 1.0 / (1.0 - beta1_t);
    inv_root_bc2 = float(1.0 / sqrt(1.0 - beta2_t));
  }
  __host__ __device__ void advance(double beta1, double beta2) {
    beta1_t *= beta1;
    beta2_t *= beta2;
    step += 1;
    derive();
  }
};
struct AdamWLaunch {
  const AdamWTensor *tensors;
  const AdamWChunk *chunks;
  AdamWState *state;
  void *moment1, *moment2;  // float, or e4m3 codes when bits == 8
  float *scale1, *scale2;   // one a block, bits == 8
  float *master;            // single-precision copy of the parameters in the slots' layout, or nullptr
  int bits;
  int chunk;                // elements of a chunk
  double beta1, beta2;
  float eps;
  double decay, lr;
  const float *lr_device;    // takes lr's place when not nullptr
  const float *grad_scale;   // device factor on every gradient, or nullptr
  unsigned seed;
  bool grad_f32;             // all gradients are fp32; else each has its parameter's type
};
// grads[i] belongs to tensor first_tensor + i (nullptr: that tensor is left as it is)
void launch_adamw(const AdamWLaunch &a, const void *const *grads, const std::vector<int> &first_chunk,
                  int n_tensors, cudaStream_t s);

}  // namespace arb
