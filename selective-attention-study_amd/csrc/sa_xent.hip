// The C ABI of the vocabulary loss (include/sa.h): argument checks and dispatch; the kernels are in sa_xent_bf16.hip,
// sa_xent_f16.hip and sa_xent_f32.hip.

#include <math.h>

#include "sa_xent.h"

namespace {

bool xent_sizes_ok(int64_t tokens, int64_t vocab, int64_t width) {
  return tokens >= 1 && tokens < ((int64_t)1 << 28) && vocab >= 1 && vocab < ((int64_t)1 << 28) && width >= 1 && width <= ((int64_t)1 << 16) &&
         cdiv(tokens, 128) * cdiv(vocab, 128) < ((int64_t)1 << 23);   // (a launch holds fewer than 2^32 threads)
}
bool xent_types_ok(int x_dtype, int w_dtype, int dtype) { return lm_elem_size(x_dtype) && lm_elem_size(w_dtype) && lm_elem_size(dtype); }
bool on_elements(const void* p, int dtype) { return (uintptr_t)p % lm_elem_size(dtype) == 0; }
bool on_16(const void* p) { return (uintptr_t)p % 16 == 0; }
bool xent_ld_ok(int64_t ld) { return ld >= 0 && ld < ((int64_t)1 << 40); }

int64_t xent_space(const XentCall& c, int dtype, bool backward) {
  return dtype == SA_DTYPE_BF16 ? xent_bytes_bf16(c, backward) : dtype == SA_DTYPE_F16 ? xent_bytes_f16(c, backward) : xent_bytes_f32(c, backward);
}
int xent_run(const XentCall& c, int dtype, bool backward) {
  return dtype == SA_DTYPE_BF16 ? xent_bf16(c, backward) : dtype == SA_DTYPE_F16 ? xent_f16(c, backward) : xent_f32(c, backward);
}

}  // namespace

extern "C" {

int64_t sa_linear_xent_workspace_bytes(const void* x, int64_t x_ld, const void* weight, int64_t weight_ld, int64_t tokens,
                                       int64_t vocab, int64_t width, int reduction, int train, int x_dtype, int weight_dtype, int dtype) {
  if (!xent_sizes_ok(tokens, vocab, width) || !xent_types_ok(x_dtype, weight_dtype, dtype)) return -1;
  float lse = 0.f;
  XentCall c{};
  c.x = x, c.x_ld = x_ld, c.w = weight, c.w_ld = weight_ld, c.tokens = tokens, c.vocab = vocab, c.width = width;
  c.reduction = reduction, c.x_t = x_dtype, c.w_t = weight_dtype, c.lse = train ? &lse : nullptr, c.cus = device_cus();
  return xent_space(c, dtype, false);
}

int sa_linear_xent(const void* x, int64_t x_ld, const void* weight, int64_t weight_ld, const int64_t* targets, float* loss, float* lse,
                   int32_t* rows, void* workspace, int64_t workspace_bytes, int64_t tokens, int64_t vocab, int64_t width,
                   int64_t ignore, int reduction, int x_dtype, int weight_dtype, int dtype, void* stream) {
  if (!xent_types_ok(x_dtype, weight_dtype, dtype)) return SA_ERR_DTYPE;
  if (!xent_sizes_ok(tokens, vocab, width) || !xent_ld_ok(x_ld) || !xent_ld_ok(weight_ld) || reduction < SA_REDUCE_NONE ||
      reduction > SA_REDUCE_SUM)
    return SA_ERR_ARGUMENT;
  if (!x || !weight || !targets || !loss || !rows || !on_elements(x, x_dtype) || !on_elements(weight, weight_dtype) ||
      (uintptr_t)targets % 8 || (uintptr_t)loss % 4 || (uintptr_t)lse % 4 || (uintptr_t)rows % 4)
    return SA_ERR_ARGUMENT;
  XentCall c{};
  c.x = x, c.x_ld = x_ld, c.w = weight, c.w_ld = weight_ld, c.targets = targets, c.loss = loss, c.lse = lse, c.rows = rows;
  c.ws = workspace, c.tokens = tokens, c.vocab = vocab, c.width = width, c.ignore = ignore, c.reduction = reduction;
  c.x_t = x_dtype, c.w_t = weight_dtype, c.cus = device_cus(), c.st = static_cast<hipStream_t>(stream);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < xent_space(c, dtype, false)) return SA_ERR_WORKSPACE;
  return xent_run(c, dtype, false);
}

int64_t sa_linear_xent_backward_workspace_bytes(const void* weight, int64_t weight_ld, int64_t tokens, int64_t vocab, int64_t width,
                                                int need_dx, int need_dweight, int weight_dtype, int dtype) {
  if (!xent_sizes_ok(tokens, vocab, width) || !xent_types_ok(dtype, weight_dtype, dtype)) return -1;
  char some = 0;
  XentCall c{};
  c.w = weight, c.w_ld = weight_ld, c.tokens = tokens, c.vocab = vocab, c.width = width, c.w_t = weight_dtype, c.x_t = dtype;
  c.dx = need_dx ? &some : nullptr, c.dw = need_dweight ? &some : nullptr, c.lse = (float*)&c, c.cus = device_cus();
  return xent_space(c, dtype, true);
}

int sa_linear_xent_backward(const void* x, int64_t x_ld, const void* weight, int64_t weight_ld, const int64_t* targets,
                            const float* lse, const int32_t* rows, const float* dloss, void* dx, void* dweight, void* workspace,
                            int64_t workspace_bytes, int64_t tokens, int64_t vocab, int64_t width, int reduction, int x_dtype,
                            int weight_dtype, int dtype, void* stream) {
  if (!xent_types_ok(x_dtype, weight_dtype, dtype)) return SA_ERR_DTYPE;
  if (!xent_sizes_ok(tokens, vocab, width) || !xent_ld_ok(x_ld) || !xent_ld_ok(weight_ld) || reduction < SA_REDUCE_NONE ||
      reduction > SA_REDUCE_SUM)
    return SA_ERR_ARGUMENT;
  if (!x || !weight || !targets || !lse || !rows || !dloss || !on_elements(x, x_dtype) || !on_elements(weight, weight_dtype) ||
      (uintptr_t)targets % 8 || (uintptr_t)lse % 4 || (uintptr_t)rows % 4 || (uintptr_t)dloss % 4 || !on_16(dx) || !on_16(dweight))
    return SA_ERR_ARGUMENT;
  if (!dx && !dweight) return SA_OK;
  XentCall c{};
  c.x = x, c.x_ld = x_ld, c.w = weight, c.w_ld = weight_ld, c.targets = targets, c.lse = const_cast<float*>(lse);
  c.rows = const_cast<int32_t*>(rows), c.dloss = dloss, c.dx = dx, c.dw = dweight;
  c.ws = workspace, c.tokens = tokens, c.vocab = vocab, c.width = width, c.reduction = reduction;
  c.x_t = x_dtype, c.w_t = weight_dtype, c.cus = device_cus(), c.st = static_cast<hipStream_t>(stream);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < xent_space(c, dtype, true)) return SA_ERR_WORKSPACE;
  return xent_run(c, dtype, true);
}

}  // extern "C"
