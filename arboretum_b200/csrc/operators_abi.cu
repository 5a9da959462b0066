// extern "C" boundary of the operators in operators.h: arguments are checked here, on the host,
// before anything is enqueued.
#include <cmath>
#include <memory>

#include "../../include/arboretum_b200.h"
#include "abi.h"
#include "operators.h"

using namespace arb;

namespace {

constexpr int64_t kMostTokens = (int64_t(1) << 31) - 2, kMostRows = (int64_t(1) << 31) - 2;
constexpr int64_t kMostElements = int64_t(1) << 46;  // of one tensor: keeps byte offsets inside 63 bits

// Makes `device` current for the call and puts the caller's device back.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    ARB_CUDA(cudaGetDevice(&before_));
    if (device == before_) return;
    if (const cudaError_t e = cudaSetDevice(device)) {
      cudaGetLastError();  // the launches after a later, good call look at it
      throw std::runtime_error(std::string("CUDA error ") + cudaGetErrorString(e) + " for device " + std::to_string(device));
    }
    changed_ = true;
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(before_);
  }
  DeviceScope(const DeviceScope &) = delete;
  DeviceScope &operator=(const DeviceScope &) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

void check_type(int type) { ARB_CHECK(type == kF32 || type == kBF16 || type == kF16, "unknown element type"); }
void check_aligned(const void *p, size_t bytes, const char *what) {
  if (reinterpret_cast<uintptr_t>(p) % bytes != 0) throw std::runtime_error(std::string(what) + " is not aligned to its type");
}
void check_matrix(const void *p, int type, int64_t rows, int64_t dim, int64_t stride, const char *what) {
  check_type(type);
  if (rows == 0 || dim == 0) return;
  if (p == nullptr) throw std::runtime_error(std::string(what) + " is NULL");
  check_aligned(p, elem_size(type), what);
  if (stride < 0 || (stride != 0 && rows > kMostElements / stride))
    throw std::runtime_error(std::string(what) + ": stride out of range");
}

void check_counts(int64_t bags, int64_t per_bag, int64_t rows) {
  ARB_CHECK(bags >= 0 && per_bag >= 0, "negative token count");
  ARB_CHECK(bags <= kMostTokens && per_bag <= kMostTokens && (per_bag == 0 || bags <= kMostTokens / per_bag),
            "more than 2^31 - 2 tokens in one call");
  ARB_CHECK(rows >= 0 && rows <= kMostRows, "a table has at most 2^31 - 2 rows");
}

TokenView check_tokens(const void *tokens, int bytes, int64_t bags, int64_t per_bag, int64_t bag_stride,
                       int64_t token_stride, int64_t rows) {
  ARB_CHECK(bytes == 4 || bytes == 8, "tokens are int32 or int64");
  check_counts(bags, per_bag, rows);
  for (int64_t stride : {bag_stride, token_stride})  // (the least int64 has no absolute value)
    ARB_CHECK(stride >= -kMostElements && stride <= kMostElements, "token stride out of range");
  if (bags * per_bag > 0) {
    ARB_CHECK(tokens != nullptr, "tokens is NULL");
    check_aligned(tokens, size_t(bytes), "tokens");
  }
  return TokenView{tokens, bytes, bags, per_bag, bag_stride, token_stride};
}

void check_out(int type, int out_type) {
  check_type(out_type);
  ARB_CHECK(out_type == type || out_type == kF32, "the output has the input's type or fp32");
}

// a sum of nothing is zero, and stays so
void check_scale(double scale) { ARB_CHECK(std::isfinite(float(scale)), "scale is not finite in fp32"); }

struct AdamW {
  int device = 0;
  AdamWLaunch launch;
  std::vector<int> first_chunk;  // per tensor, one more at the end
  std::vector<int> type;
  int count = 0;
};

int64_t padded(int64_t n) { return (n + kMomentBlock - 1) / kMomentBlock * kMomentBlock; }

// where the parts of an optimizer's workspace lie
struct AdamWLayout {
  int64_t length = 0, chunks = 0;  // chunks: room for the shortest
  size_t tensors_at, chunks_at, bytes;
  AdamWLayout(const AAdamWParam *params, int count) {
    ARB_CHECK(count >= 0 && (count == 0 || params != nullptr), "params is NULL");
    for (int i = 0; i < count; ++i) {
      ARB_CHECK(params[i].size >= 0 && params[i].size <= kMostElements, "tensor size out of range");
      length += padded(params[i].size);
      ARB_CHECK(length <= kMostElements, "too many elements for one optimizer");
    }
    for (int i = 0; i < count; ++i) chunks += (params[i].size + kLeastAdamWChunk - 1) / kLeastAdamWChunk;
    ARB_CHECK(chunks <= (int64_t(1) << 30), "too many elements for one optimizer");
    tensors_at = 256;  // the state comes first
    chunks_at = tensors_at + (size_t(count) * sizeof(AdamWTensor) + 255) / 256 * 256;
    bytes = chunks_at + (size_t(chunks) * sizeof(AdamWChunk) + 255) / 256 * 256;
  }
};

void put_step(AdamW *o, int64_t step, cudaStream_t s) {
  AdamWState st;
  st.beta1_t = std::pow(o->launch.beta1, double(step) + 1);
  st.beta2_t = std::pow(o->launch.beta2, double(step) + 1);
  st.step = step;
  st.done = 0;
  st.one = 1.0f;
  st.derive();
  ARB_CUDA(cudaMemcpyAsync(o->launch.state, &st, sizeof st, cudaMemcpyHostToDevice, s));
  ARB_CUDA(cudaStreamSynchronize(s));
}

}  // namespace

extern "C" {

const char *AEmbedding(const void *table, int type, int64_t rows, int64_t dim, int64_t row_stride,
                       const void *tokens, int token_bytes, int64_t bags, int64_t per_bag,
                       int64_t bag_stride, int64_t token_stride, double scale, void *out, int out_type,
                       int64_t out_stride, int device, void *stream) {
  ARB_TRY
  LookupLaunch a;
  a.tokens = check_tokens(tokens, token_bytes, bags, per_bag, bag_stride, token_stride, rows);
  ARB_CHECK(dim >= 0 && dim <= kMostElements, "row width out of range");
  check_matrix(table, type, rows, dim, row_stride, "table");
  check_out(type, out_type);
  check_matrix(out, out_type, bags, dim, out_stride, "out");
  ARB_CHECK(bags < 2 || out_stride >= dim, "rows of out overlap");
  check_scale(scale);
  a.table = table, a.type = type, a.rows = rows, a.dim = dim, a.row_stride = row_stride;
  a.scale = float(scale);
  a.out = out, a.out_type = out_type, a.out_stride = out_stride;
  if (bags == 0 || dim == 0) return nullptr;
  DeviceScope scope(device);
  launch_lookup(a, static_cast<cudaStream_t>(stream));
  ARB_CATCH
}

const char *ATokenOrderBytes(int64_t bags, int64_t per_bag, int64_t rows, int64_t *order_bytes, int64_t *scratch_bytes) {
  ARB_TRY
  ARB_CHECK(order_bytes && scratch_bytes, "NULL argument");
  check_counts(bags, per_bag, rows);
  const TokenOrder o(nullptr, bags, per_bag, rows);
  *order_bytes = int64_t(o.bytes);
  *scratch_bytes = int64_t(token_order_scratch(o));
  ARB_CATCH
}

const char *ATokenOrder(const void *tokens, int token_bytes, int64_t bags, int64_t per_bag, int64_t bag_stride,
                        int64_t token_stride, int64_t rows, void *order, void *scratch, int device, void *stream) {
  ARB_TRY
  const TokenView t = check_tokens(tokens, token_bytes, bags, per_bag, bag_stride, token_stride, rows);
  const TokenOrder o(order, bags, per_bag, rows);
  ARB_CHECK(order && (scratch || token_order_scratch(o) == 0), "NULL argument");
  check_aligned(order, 256, "order");
  check_aligned(scratch, 256, "scratch");
  DeviceScope scope(device);
  launch_token_order(t, o, scratch, static_cast<cudaStream_t>(stream));
  ARB_CATCH
}

const char *AEmbeddingGradBytes(int64_t bags, int64_t per_bag, int64_t rows, int64_t dim, int device, int64_t *scratch_bytes) {
  ARB_TRY
  ARB_CHECK(scratch_bytes, "NULL argument");
  check_counts(bags, per_bag, rows);
  ARB_CHECK(dim >= 0 && dim <= kMostElements, "row width out of range");
  const TokenOrder o(nullptr, bags, per_bag, rows);
  if (o.blocks > 1) {  // goes by the device's size
    DeviceScope scope(device);
    *scratch_bytes = int64_t(lookup_grad_scratch(o, dim));
  } else {
    *scratch_bytes = int64_t(lookup_grad_scratch(o, dim));
  }
  ARB_CATCH
}

const char *AEmbeddingGrad(const void *grad, int type, int64_t bags, int64_t dim, int64_t grad_stride,
                           const void *order, int64_t per_bag, int64_t rows, double scale, void *out, int out_type,
                           int64_t out_stride, int accumulate, void *scratch, int device, void *stream) {
  ARB_TRY
  check_counts(bags, per_bag, rows);
  ARB_CHECK(dim >= 0 && dim <= kMostElements, "row width out of range");
  check_matrix(grad, type, bags, dim, grad_stride, "grad");
  check_out(type, out_type);
  check_matrix(out, out_type, rows, dim, out_stride, "out");
  ARB_CHECK(rows < 2 || out_stride >= dim, "rows of out overlap");
  check_scale(scale);
  ARB_CHECK(order != nullptr, "order is NULL");
  check_aligned(order, 256, "order");
  check_aligned(scratch, 256, "scratch");
  if (rows == 0 || dim == 0) return nullptr;
  const TokenOrder o(const_cast<void *>(order), bags, per_bag, rows);
  DeviceScope scope(device);
  ARB_CHECK(scratch != nullptr || lookup_grad_scratch(o, dim) == 0, "scratch is NULL");
  LookupGradLaunch a;
  a.grad = grad, a.type = type, a.dim = dim, a.grad_stride = grad_stride;
  a.scale = float(scale);
  a.out = out, a.out_type = out_type, a.out_stride = out_stride;
  a.accumulate = accumulate != 0;
  launch_lookup_grad(a, o, scratch, static_cast<cudaStream_t>(stream));
  ARB_CATCH
}

const char *AAdamWBytes(const AAdamWParam *params, int count, int64_t *length, int64_t *workspace_bytes) {
  ARB_TRY
  ARB_CHECK(length && workspace_bytes, "NULL argument");
  const AdamWLayout l(params, count);
  *length = l.length;
  *workspace_bytes = int64_t(l.bytes);
  ARB_CATCH
}

const char *AAdamWCreate(const AAdamWParam *params, int count, const AAdamWConfig *config, void *workspace,
                         int device, VoidPointer *out) {
  ARB_TRY
  ARB_CHECK(config && workspace && out, "NULL argument");
  const AAdamWConfig &c = *config;
  ARB_CHECK(c.state_bits == 8 || c.state_bits == 32, "state_bits must be 8 or 32");
  ARB_CHECK(c.beta1 >= 0 && c.beta1 < 1 && c.beta2 >= 0 && c.beta2 < 1, "betas must be in [0, 1)");
  ARB_CHECK(c.eps >= 0 && std::isfinite(c.eps) && c.weight_decay >= 0 && std::isfinite(c.weight_decay),
            "eps and weight_decay must be finite and not negative");
  // the kernel's reciprocal takes a divisor below float's smallest normal number for zero: a second
  // moment of zero would give 0 / 0
  ARB_CHECK(c.eps == 0 || float(c.eps) >= 0x1p-126f, "eps must be 0 or at least 2^-126");
  const AdamWLayout l(params, count);
  check_aligned(workspace, 256, "workspace");
  if (l.length > 0) {
    ARB_CHECK(c.moment1 && c.moment2, "the moment buffers are NULL");
    ARB_CHECK(c.state_bits == 32 || (c.scale1 && c.scale2), "the scale buffers are NULL");
    for (const void *p : {static_cast<const void *>(c.moment1), static_cast<const void *>(c.moment2),
                          static_cast<const void *>(c.scale1), static_cast<const void *>(c.scale2),
                          static_cast<const void *>(c.master)})
      check_aligned(p, 16, "an optimizer buffer");
  }
  std::unique_ptr<AdamW> o(new AdamW());
  std::vector<AdamWTensor> tensors(static_cast<size_t>(count));
  std::vector<AdamWChunk> chunks;
  chunks.reserve(size_t(l.chunks));
  const int chunk = adamw_chunk(l.length, c.state_bits);
  int64_t slot = 0;
  for (int i = 0; i < count; ++i) {
    check_type(params[i].type);
    ARB_CHECK(params[i].param != nullptr || params[i].size == 0, "a parameter is NULL");
    check_aligned(params[i].param, elem_size(params[i].type), "a parameter");
    tensors[i] = AdamWTensor{params[i].param, params[i].size, slot, params[i].type,
                             reinterpret_cast<uintptr_t>(params[i].param) % 16 == 0 ? 1 : 0};
    o->first_chunk.push_back(int(chunks.size()));
    o->type.push_back(params[i].type);
    for (int64_t k = 0; k * chunk < params[i].size; ++k) chunks.push_back(AdamWChunk{i, int(k)});
    slot += padded(params[i].size);
  }
  o->first_chunk.push_back(int(chunks.size()));
  o->count = count;
  o->device = device;
  char *w = static_cast<char *>(workspace);
  AdamWLaunch &a = o->launch;
  a.state = reinterpret_cast<AdamWState *>(w);
  a.tensors = reinterpret_cast<AdamWTensor *>(w + l.tensors_at);
  a.chunks = reinterpret_cast<AdamWChunk *>(w + l.chunks_at);
  a.moment1 = c.moment1, a.moment2 = c.moment2, a.scale1 = c.scale1, a.scale2 = c.scale2, a.master = c.master;
  a.bits = c.state_bits;
  a.chunk = chunk;
  a.beta1 = c.beta1, a.beta2 = c.beta2, a.eps = float(c.eps), a.decay = c.weight_decay;
  a.seed = c.seed;
  DeviceScope scope(device);
  if (count > 0)
    ARB_CUDA(cudaMemcpy(w + l.tensors_at, tensors.data(), tensors.size() * sizeof(AdamWTensor), cudaMemcpyHostToDevice));
  if (!chunks.empty())
    ARB_CUDA(cudaMemcpy(w + l.chunks_at, chunks.data(), chunks.size() * sizeof(AdamWChunk), cudaMemcpyHostToDevice));
  put_step(o.get(), 0, nullptr);
  *out = o.release();
  ARB_CATCH
}

const char *AAdamWSetStep(VoidPointer optimizer, int64_t step, void *stream) {
  ARB_TRY
  ARB_CHECK(optimizer, "NULL argument");
  ARB_CHECK(step >= 0, "negative step count");
  AdamW *o = static_cast<AdamW *>(optimizer);
  DeviceScope scope(o->device);
  put_step(o, step, static_cast<cudaStream_t>(stream));
  ARB_CATCH
}

const char *AAdamWGetStep(VoidPointer optimizer, int64_t *step, void *stream) {
  ARB_TRY
  ARB_CHECK(optimizer && step, "NULL argument");
  AdamW *o = static_cast<AdamW *>(optimizer);
  DeviceScope scope(o->device);
  AdamWState st;
  ARB_CUDA(cudaMemcpyAsync(&st, o->launch.state, sizeof st, cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream)));
  ARB_CUDA(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)));
  *step = st.step;
  ARB_CATCH
}

const char *AAdamWStep(VoidPointer optimizer, const void *const *grads, int count, int grads_fp32, double lr,
                       const float *lr_device, const float *grad_scale, void *stream) {
  ARB_TRY
  ARB_CHECK(optimizer, "NULL argument");
  const AdamW *o = static_cast<const AdamW *>(optimizer);
  ARB_CHECK(count == o->count && (count == 0 || grads != nullptr), "one gradient (or NULL) for every parameter");
  ARB_CHECK(lr_device != nullptr || std::isfinite(lr), "lr is not finite");
  for (int i = 0; i < count; ++i) check_aligned(grads[i], grads_fp32 ? 4 : elem_size(o->type[i]), "a gradient");
  check_aligned(lr_device, 4, "lr_device");
  check_aligned(grad_scale, 4, "grad_scale");
  AdamWLaunch a = o->launch;
  a.lr = lr;
  a.lr_device = lr_device;
  a.grad_scale = grad_scale;
  a.grad_f32 = grads_fp32 != 0;
  DeviceScope scope(o->device);
  launch_adamw(a, grads, o->first_chunk, count, static_cast<cudaStream_t>(stream));
  ARB_CATCH
}

const char *AFreeAdamW(VoidPointer optimizer) {
  ARB_TRY
  delete static_cast<AdamW *>(optimizer);
  ARB_CATCH
}

}  // extern "C"
