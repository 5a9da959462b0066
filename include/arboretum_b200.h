/* C ABI of libarboretum.so (B200 build).
 *
 * The first fourteen functions are the reference's python-wrapper ABI
 * (python-wrapper/arboretum_wrapper.h:4-39), re-exported one to one so that the
 * reference's python-package/arboretum/core.py loads this library unchanged.
 * Every function returns NULL on success, else a NUL-terminated message owned by
 * the library (valid until the next failing call on the same thread).  Handles
 * are opaque; a NULL handle passed to a free function is ignored.  Unlike the
 * reference no call ever exits the process or lets a C++ exception escape.
 *
 * The functions below the "additive" line do not exist in the reference.
 */
#ifndef ARBORETUM_B200_H
#define ARBORETUM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void *VoidPointer;

/* arboretum_wrapper.h:6-9 / arboretum_wrapper.cu:16-39.  `data` is row-major
 * [nrow][ncol] fp32, `categories` row-major [nrow][ccol] or NULL; both are
 * copied.  `missing` is accepted and ignored, like in the reference. */
const char *ACreateFromDenseMatrix(const float *data, const unsigned int *categories, int nrow,
                                   int ncol, int ccol, float missing, VoidPointer *out);
/* arboretum_wrapper.h:11 / .cu:41-55 */
const char *ASetY(VoidPointer data, const float *y);
/* arboretum_wrapper.h:13 / .cu:57-71 */
const char *ASetLabel(VoidPointer data, const unsigned char *labels);
/* arboretum_wrapper.h:15 / .cu:73-86 */
const char *ASetWeights(VoidPointer data, const float *weights);
/* arboretum_wrapper.h:17-18 / .cu:88-99: nested JSON configuration */
const char *AInitGarden(const char *configuration, VoidPointer *garden);
/* arboretum_wrapper.h:20-21 / .cu:101-111: one boosting round (labels_count trees).
 * The first call quantises `data` and binds the garden to it. */
const char *AGrowTree(VoidPointer garden, VoidPointer data, const float *grad);
/* arboretum_wrapper.h:23 / .cu:180-191 */
const char *AAppendLastTree(VoidPointer garden, VoidPointer data);
/* arboretum_wrapper.h:25-26 / .cu:153-178: *out = new float[rows * labels] */
const char *AGetY(VoidPointer garden, VoidPointer data, const float **out);
/* arboretum_wrapper.h:28-29 / .cu:113-139: n_rounds == -1 means all trees */
const char *APredict(VoidPointer garden, VoidPointer data, const float **out, const int n_rounds);
/* arboretum_wrapper.h:31 / .cu:141-145: *model = heap C string (argument order as there) */
const char *ADumpModel(const char **model, VoidPointer garden);
/* arboretum_wrapper.h:33 / .cu:147-151 */
const char *ALoadModel(const char *model, VoidPointer garden);
/* arboretum_wrapper.h:35-39 / .cu:193-205 */
const char *AFreeDMatrix(VoidPointer ptr);
const char *AFreeGarden(VoidPointer ptr);
const char *ADeleteArray(float *in);

/* ------------------------------- additive ---------------------------------- */

/* Rows that are already binned (uint8 ids < hist_size, row-major [nrow][ncol]);
 * the reference ingests fp32 only (arboretum_wrapper.h:6-9).  `bins` may point to host or
 * to device memory (rows generated or decoded on the GPU); so may ASetY's `y` for a matrix
 * that lives in device memory. */
const char *ACreateFromBinnedMatrix(const uint8_t *bins, int64_t nrow, int ncol, int hist_size,
                                    VoidPointer *out);
/* Thresholds computed elsewhere (e.g. on the whole data set before sharding rows
 * over GPUs): thr is [ncol][hist_size], size[f] = bins in use.  Must precede the
 * first AGrowTree. */
const char *ASetThresholds(VoidPointer data, const float *thr, const int *size, int hist_size);
/* Quantise now (what the first AGrowTree would do) and read the result back:
 * thr [ncol][hist_size], size [ncol], bins [nrow][ncol] uint16; any may be NULL. */
const char *AQuantize(VoidPointer data, int hist_size, int missing_bin, float *thr, int *size,
                      uint16_t *bins);
/* Training-time predictions of the bound DMatrix, internal scale, [labels][rows]. */
const char *AGetTrainY(VoidPointer garden, float *out);
/* Split records of level `level` of the last grown tree: arrays of 1 << level
 * entries (node_begin: one more).  Sums are in gradient units. */
const char *AGetLevelStats(VoidPointer garden, int level, unsigned *node_begin, float *gain,
                           int *fid, int *bin, double *left_g, double *left_h, double *tot_g,
                           double *tot_h, unsigned *left_count);
/* The same for tree `tree_in_round` (0 .. labels_count - 1, -1 = the last) of the last round:
 * multi:softmax grows one tree per class in every round. */
const char *AGetLevelStatsOf(VoidPointer garden, int tree_in_round, int level, unsigned *node_begin,
                             float *gain, int *fid, int *bin, double *left_g, double *left_h,
                             double *tot_g, double *tot_h, unsigned *left_count);
/* The fixed-point steps of the last round: every gradient (hessian) entered the histograms
 * as an integer multiple of *g_step (*h_step), off from its float value by less than one
 * step. */
const char *AGetGradientStep(VoidPointer garden, double *g_step, double *h_step);
/* CUDA-event timing of the kernel classes: switch on, then read a JSON summary. */
const char *ASetProfile(VoidPointer garden, int on);
const char *AGetTimings(VoidPointer garden, const char **json);
/* One histogram launch over host buffers (kernel-level parity and measurement):
 * bins row-major [nrow][ncol] of `bin_bytes`-byte ids, grad [nrow] (pair == 0) or
 * [nrow][2]; rowid (NULL = identity) grouped by node with node_begin[n_nodes + 1];
 * out_g / out_h [n_nodes][ncol][hist_size + 1] doubles.  When `reps` > 0 the
 * launch is repeated and its mean device time is stored in *ms. */
const char *ABuildHistogram(const void *bins, int bin_bytes, int64_t nrow, int ncol, int hist_size,
                            const float *grad, int pair, const unsigned *rowid,
                            const unsigned *node_begin, int n_nodes, int quant_bits, double *out_g,
                            double *out_h, int reps, float *ms);
/* The same launch with the subtraction trick (hist_grad_sum.cu:6-33,288-290 of the reference):
 * nodes 2p and 2p + 1 are the children of parent p, whose sums parent_g / parent_h
 * [n_nodes / 2][ncol][hist_size + 1] are given (multiples of the fixed-point step, e.g.
 * integers); only the smaller child of every pair is scanned (ties: the left one), the other
 * is parent - scanned. */
const char *ABuildHistogramFromParents(const void *bins, int bin_bytes, int64_t nrow, int ncol, int hist_size,
                                       const float *grad, int pair, const unsigned *rowid,
                                       const unsigned *node_begin, int n_nodes, int quant_bits,
                                       const double *parent_g, const double *parent_h, double *out_g,
                                       double *out_h);
/* Multi-GPU: rows are sharded over one process per GPU; every level's histogram
 * is summed over the ranks with ncclAllReduce, and the first AGrowTree finds the
 * thresholds of the whole data set with the other ranks (unless ASetThresholds gave
 * them), so bins and trees equal those of the unsharded matrix.  `id` is the 128-byte
 * ncclUniqueId made by rank 0 (ANcclUniqueId) and sent to the others by the host.
 * The first communicator of a process is kept until the process exits; a later Garden
 * of the same rank and world size attaches it when AInitNccl is given id128 == NULL
 * (no bootstrap, no host traffic).  Gardens that share a communicator must not train at
 * the same time. */
const char *ANcclUniqueId(char *id128);
const char *AInitNccl(VoidPointer garden, int rank, int world, const char *id128);

/* No counterpart in the reference.  The waits of the exchange between row shards over peer
 * memory are bounded: a peer that never answers makes a kernel give up after a time limit,
 * record where, and return (the host then reports an error after the tree; the context stays
 * usable).  This call exercises exactly that wait on a word that nothing sets, on the
 * current device: *timed_out becomes 1, *waited_ms about limit_ms (at most 2000). */
const char *APeerWaitProbe(double limit_ms, int *timed_out, double *waited_ms);

/* No counterpart in the reference.  Threshold search of ONE feature for callers that
 * must not allocate device memory (a process whose GPU memory is owned by one
 * arena, a fixed-budget service, a latency-critical section): `sorted_device` holds
 * the column's n values in ascending fp32 radix order in device memory,
 * `thr_device` receives hist_size thresholds (device memory), `stream` is a
 * cudaStream_t (NULL = default stream).  The call only launches kernels; its
 * scratch is a 128 KB array inside the library image, which every GPU that loads
 * the library holds until the process exits.  n may not exceed 67,108,864 (2^26):
 * larger columns return an error and should go through AQuantize.  The first call on
 * a device looks the array's address up (cudaGetSymbolAddress) and may make the
 * runtime load the library's kernels, which takes device memory once: make one
 * warm-up call before a section that must not allocate.  All calls on a device share the array, so two
 * calls that overlap on the GPU (different streams, different threads) race; calls
 * on one stream are safe.  Nothing of an earlier call's scratch contents is read. */
const char *AThresholdsNoAlloc(const float *sorted_device, long long n, int hist_size,
                               float *thr_device, void *stream);

/* Additive (no counterpart in the reference): the library takes its device memory from the
 * current device's stream-ordered pool and keeps what it frees, so that the next matrix or
 * model does not pay for cudaMalloc again; this call hands the unused part back to the
 * driver (for a process that shares the GPU with other allocators), together with the few
 * small pinned host blocks it keeps for the same reason. */
const char *AReleaseCachedMemory(void);

/* Additive (no counterpart in the reference): measures, on the current device, how many
 * (gradient, hessian) pair updates per second the histogram kernels' two shared-memory
 * reductions sustain when nothing else is done (no loads, staging or stores) -- the
 * ceiling of their inner loop.  `steps` x 8 updates per thread of a full grid; a few
 * thousand steps run for a millisecond. */
const char *ASharedAtomicPeak(int steps, double *pair_updates_per_s);

/* ---- operators on tables of learned rows (no counterpart in the reference) ------------------
 * A forest of T trees with L leaves is a table of T * L rows, a row of the data set a bag of T
 * tokens (ALeafTokens) and its prediction the sum of the rows they name.  The operators take
 * tables of any width: lookup, its gradient, and the AdamW step on what is learned.
 *
 * All pointers below are device memory of `device` (an ordinal) unless said otherwise, `stream`
 * is a cudaStream_t of that device (NULL = its default stream).  AEmbedding, ATokenOrder,
 * AEmbeddingGrad and AAdamWStep only enqueue: no synchronisation, no allocation, so they can be
 * captured into a CUDA graph; the other calls may allocate and wait.  Outputs and scratch memory
 * belong to the caller and must live until the work is done.  Two calls that may overlap need
 * scratch of their own.  Strides are in elements.
 * Element types: 0 = fp32, 1 = bf16, 2 = fp16; an output has the input's type or fp32.
 * Tokens are int32 (token_bytes 4) or int64 (8): token t of bag b is
 * tokens[b * bag_stride + t * token_stride].  A token outside [0, rows) is an empty slot: it adds
 * nothing and gets no gradient.  bags * per_bag and rows must be below 2^31 - 1.  scale is finite. */

/* Trees of the model (labels_count a boosting round). */
const char *ATreeCount(VoidPointer garden, int *count);
/* Ordinal of the device the model works on: `device` of its configuration, else the one that was
 * current when it first needed one (this call, at the latest). */
const char *AModelDevice(VoidPointer garden, int *device);
/* The leaf that every row of `data` reaches in each of the first n_rounds trees (-1: all; a count of
 * trees, like APredict's): out[tree][row] = tree * 2^(depth - 1) + leaf, host memory or memory of the
 * model's device. */
const char *ALeafTokens(VoidPointer garden, VoidPointer data, int n_rounds, int *out);
/* `steps` AdamW steps on the leaf values of all trees together, on the gradient of the mean loss over
 * `data` (its targets; the garden's objective, with labels_count 1 unless it is multi:softmax): lookup,
 * gradient by sorted tokens and AdamW step as below, one tensor a tree.  The trees' tests stay.
 * Training can go on afterwards; predictions that AAppendLastTree has accumulated follow the new values
 * in the next AGetY or AAppendLastTree (an error when another model has added to the same matrix). */
const char *ARefineLeaves(VoidPointer garden, VoidPointer data, int steps, double lr, double beta1, double beta2, double eps,
                          double weight_decay, int state_bits);

/* out[b][:] = scale * sum over t of table[token(b, t)][:], summed in fp32, rounded once */
const char *AEmbedding(const void *table, int type, int64_t rows, int64_t dim, int64_t row_stride,
                       const void *tokens, int token_bytes, int64_t bags, int64_t per_bag,
                       int64_t bag_stride, int64_t token_stride, double scale, void *out, int out_type,
                       int64_t out_stride, int device, void *stream);
/* Bytes that ATokenOrder needs: the order itself (kept as long as it is used) and scratch (free
 * after the call; may be 0).  Both 256-byte aligned. */
const char *ATokenOrderBytes(int64_t bags, int64_t per_bag, int64_t rows, int64_t *order_bytes, int64_t *scratch_bytes);
/* Sorts the bags by the tokens that name them, for AEmbeddingGrad: stable, so equal tokens give
 * equal orders. */
const char *ATokenOrder(const void *tokens, int token_bytes, int64_t bags, int64_t per_bag, int64_t bag_stride,
                        int64_t token_stride, int64_t rows, void *order, void *scratch, int device, void *stream);
const char *AEmbeddingGradBytes(int64_t bags, int64_t per_bag, int64_t rows, int64_t dim, int device,
                                int64_t *scratch_bytes);
/* out[v][:] = scale * sum of grad[b][:] over all (b, t) whose token is v (accumulate: added to out,
 * rows no token names stay untouched; else they become zero).  `order` of the same bags, tokens a
 * bag and rows.  Summed in fp32 or more in a fixed order: the same inputs give the same bits on the same
 * device.  grad_stride 0: one row for all bags. */
const char *AEmbeddingGrad(const void *grad, int type, int64_t bags, int64_t dim, int64_t grad_stride,
                           const void *order, int64_t per_bag, int64_t rows, double scale, void *out, int out_type,
                           int64_t out_stride, int accumulate, void *scratch, int device, void *stream);

/* AdamW over many tensors in one launch.  Element i of tensor k has its moments at element
 * slot[k] + i of the flat moment buffers; slots start at multiples of 128 in the order of the
 * tensors: slot[0] = 0, slot[k + 1] = slot[k] + (size[k] rounded up to 128).  `length` is the end
 * of the last slot.
 *   state_bits 32: moment1, moment2 = fp32 first and second moment.
 *   state_bits 8:  moment1, moment2 = e4m3 codes, scale1, scale2 = one fp32 power of two for every
 *                  128 elements; moment2 holds the SQUARE ROOT of the second moment.  Rounded with
 *                  a dither keyed by (element, step, seed).
 * master: fp32 copy of the parameters in the slots' layout, or NULL; with it a step updates the
 * copy and stores it rounded to each parameter's type. */
typedef struct {
  void *param;   /* contiguous */
  int64_t size;  /* elements, may be 0 */
  int type;      /* element type */
} AAdamWParam;
typedef struct {
  double beta1, beta2;  /* in [0, 1) */
  double eps;           /* 0, or at least 2^-126 */
  double weight_decay;
  int state_bits;
  unsigned seed;
  void *moment1, *moment2;
  float *scale1, *scale2;
  float *master;
} AAdamWConfig;
/* params is host memory.  *length: elements of the moment buffers; *workspace_bytes: what the
 * optimizer keeps beside them in device memory of the caller. */
const char *AAdamWBytes(const AAdamWParam *params, int count, int64_t *length, int64_t *workspace_bytes);
/* params and config are host memory and copied; the buffers they name and the workspace must
 * outlive the handle.  Waits for the upload of the workspace.  The moments are taken as they are. */
const char *AAdamWCreate(const AAdamWParam *params, int count, const AAdamWConfig *config, void *workspace,
                         int device, VoidPointer *out);
/* The step count, which lives in device memory (a captured step counts every replay): set, or
 * read back after waiting for `stream`. */
const char *AAdamWSetStep(VoidPointer optimizer, int64_t step, void *stream);
const char *AAdamWGetStep(VoidPointer optimizer, int64_t *step, void *stream);
/* One step.  grads: host array of `count` device pointers, contiguous gradients (NULL: that tensor
 * and its moments stay as they are); all fp32 (grads_fp32 != 0) or each of its parameter's type.
 * lr_device (fp32, NULL: lr) and grad_scale (fp32 factor on all gradients, NULL: 1) are read by the
 * kernel.  Steps of one optimizer must be ordered on the device. */
const char *AAdamWStep(VoidPointer optimizer, const void *const *grads, int count, int grads_fp32, double lr,
                       const float *lr_device, const float *grad_scale, void *stream);
const char *AFreeAdamW(VoidPointer optimizer);

#ifdef __cplusplus
}
#endif
#endif /* ARBORETUM_B200_H */
