// C-ABI entry points of the operators that train and serve adapters on a packed model
// (include/cdclq.h): validation, workspace plans and the k_ckpt.hip / k_loss.hip launches. They
// enqueue on the caller's stream and return; nothing here allocates device memory or waits.
#include <hip/hip_runtime.h>

#include <string>

#include "cdclq.h"
#include "ctx.h"
#include "kernels.h"

namespace {

using namespace cdclq;

// The context's GPU for the length of a call; the caller's current device comes back afterwards.
struct OnDevice {
  int before = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

int check_half(cdclq_ctx* ctx, int dtype) {
  if (dtype != CDCLQ_DTYPE_F16 && dtype != CDCLQ_DTYPE_BF16)
    return fail(ctx, CDCLQ_INVALID_ARG, "unsupported dtype " + std::to_string(dtype) + " (need F16 or BF16)");
  return CDCLQ_OK;
}

// Sizes whose tiles and tables are counted in 32 bits.
constexpr size_t kMaxTokens = (size_t)1 << 24, kMaxWidth = (size_t)1 << 20, kMaxVocab = (size_t)1 << 28;

int check_size(cdclq_ctx* ctx, const char* what, size_t got, size_t most) {
  if (got > most)
    return fail(ctx, CDCLQ_INVALID_ARG,
                std::string(what) + " " + std::to_string(got) + " exceeds this build's limit of " + std::to_string(most));
  return CDCLQ_OK;
}

int check_rows(cdclq_ctx* ctx, const char* what, size_t ld, size_t cols) {
  if (ld < cols)
    return fail(ctx, CDCLQ_INVALID_ARG, std::string("row stride ") + std::to_string(ld) + " of " + what +
                                            " is below its " + std::to_string(cols) + " columns");
  return CDCLQ_OK;
}

int check_work(cdclq_ctx* ctx, const void* work, size_t got, size_t need) {
  if (need && (!work || got < need))
    return fail(ctx, CDCLQ_INVALID_ARG,
                "workspace holds " + std::to_string(work ? got : 0) + " bytes, the call needs " + std::to_string(need));
  if ((uintptr_t)work % 256) return fail(ctx, CDCLQ_INVALID_ARG, "workspace is not aligned to 256 bytes");
  return CDCLQ_OK;
}

bool loss_pads_w(const void* w, size_t ldw, size_t d) { return d % 8 || ldw % 8 || (uintptr_t)w % 16; }

int check_loss(cdclq_ctx* ctx, const void* x, size_t ldx, const void* w, size_t ldw, size_t t, size_t d, size_t v,
               int dtype, const int64_t* targets) {
  CK(check_half(ctx, dtype));
  if (d == 0 || v == 0) return fail(ctx, CDCLQ_INVALID_ARG, "hidden width and vocabulary must be > 0");
  CK(check_size(ctx, "token count", t, kMaxTokens));
  CK(check_size(ctx, "hidden width", d, kMaxWidth));
  CK(check_size(ctx, "vocabulary", v, kMaxVocab));
  CK(check_rows(ctx, "x", ldx, d));
  CK(check_rows(ctx, "w", ldw, d));
  if (!w || (t && (!x || !targets))) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  return CDCLQ_OK;
}

}  // namespace

extern "C" {

int cdclq_checkpoint_save_device(cdclq_ctx* ctx, const void* x, size_t ldx, size_t t, size_t n, int dtype,
                                 int8_t* codes, float* scales, void* stream) {
  if (!ctx) return CDCLQ_INVALID_ARG;
  ctx->err.clear();
  CK(check_half(ctx, dtype));
  CK(check_size(ctx, "width", n, (size_t)1 << 30));
  CK(check_rows(ctx, "x", ldx, n));
  if (t == 0 || n == 0) return CDCLQ_OK;
  if (!x || !codes || !scales) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  OnDevice on(ctx->device);
  HIPCK(on.err);
  HIPCK(ckpt_save((hipStream_t)stream, dtype, static_cast<const uint16_t*>(x), (long)ldx, (long)t, (long)n, codes, scales));
  return CDCLQ_OK;
}

int cdclq_checkpoint_restore_device(cdclq_ctx* ctx, const int8_t* codes, const float* scales, size_t t, size_t n,
                                    int dtype, void* out, size_t ldo, void* stream) {
  if (!ctx) return CDCLQ_INVALID_ARG;
  ctx->err.clear();
  CK(check_half(ctx, dtype));
  CK(check_size(ctx, "width", n, (size_t)1 << 30));
  CK(check_rows(ctx, "out", ldo, n));
  if (t == 0 || n == 0) return CDCLQ_OK;
  if (!codes || !scales || !out) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  OnDevice on(ctx->device);
  HIPCK(on.err);
  HIPCK(ckpt_restore((hipStream_t)stream, dtype, codes, scales, (long)t, (long)n, static_cast<uint16_t*>(out), (long)ldo));
  return CDCLQ_OK;
}

size_t cdclq_vocab_work_bytes(size_t t, size_t d, size_t v, const void* w, size_t ldw, int grad) {
  if (d == 0 || v == 0 || t > kMaxTokens || d > kMaxWidth || v > kMaxVocab) return 0;
  return loss_plan((long)t, (long)d, (long)v, loss_pads_w(w, ldw, d), grad != 0).bytes;
}

int cdclq_vocab_loss_device(cdclq_ctx* ctx, const void* x, size_t ldx, const void* w, size_t ldw, size_t t, size_t d,
                            size_t v, int dtype, const int64_t* targets, int64_t ignore_index, float* loss, float* lse,
                            void* work, size_t work_bytes, void* stream) {
  if (!ctx) return CDCLQ_INVALID_ARG;
  ctx->err.clear();
  CK(check_loss(ctx, x, ldx, w, ldw, t, d, v, dtype, targets));
  if (t == 0) return CDCLQ_OK;
  if (!loss || !lse) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  const LossPlan p = loss_plan((long)t, (long)d, (long)v, loss_pads_w(w, ldw, d), false);
  CK(check_work(ctx, work, work_bytes, p.bytes));
  LossArgs a = {};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = (long)ldx;
  a.w = static_cast<const uint16_t*>(w);
  a.ldw = (long)ldw;
  a.t = (long)t, a.d = (long)d, a.v = (long)v;
  a.targets = targets;
  a.ignore = ignore_index;
  a.loss = loss;
  a.lse_out = lse;
  a.work = work;
  OnDevice on(ctx->device);
  HIPCK(on.err);
  HIPCK(loss_forward((hipStream_t)stream, dtype, a, p));
  return CDCLQ_OK;
}

int cdclq_vocab_loss_backward_device(cdclq_ctx* ctx, const void* x, size_t ldx, const void* w, size_t ldw, size_t t,
                                     size_t d, size_t v, int dtype, const int64_t* targets, int64_t ignore_index,
                                     const float* lse, const float* dloss, void* dx, size_t lddx, void* dw, size_t lddw,
                                     void* work, size_t work_bytes, void* stream) {
  if (!ctx) return CDCLQ_INVALID_ARG;
  ctx->err.clear();
  CK(check_loss(ctx, x, ldx, w, ldw, t, d, v, dtype, targets));
  CK(check_rows(ctx, "dx", lddx, d));
  if (dw) CK(check_rows(ctx, "dw", lddw, d));
  if (t == 0 && !dw) return CDCLQ_OK;
  if (t && (!lse || !dloss || !dx)) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  const LossPlan p = loss_plan((long)t, (long)d, (long)v, loss_pads_w(w, ldw, d), true);
  CK(check_work(ctx, work, work_bytes, p.bytes));
  LossArgs a = {};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = (long)ldx;
  a.w = static_cast<const uint16_t*>(w);
  a.ldw = (long)ldw;
  a.t = (long)t, a.d = (long)d, a.v = (long)v;
  a.targets = targets;
  a.ignore = ignore_index;
  a.lse_in = lse;
  a.dloss = dloss;
  a.dx = static_cast<uint16_t*>(dx);
  a.lddx = (long)lddx;
  a.dw = static_cast<uint16_t*>(dw);
  a.lddw = (long)lddw;
  a.work = work;
  OnDevice on(ctx->device);
  HIPCK(on.err);
  HIPCK(loss_backward((hipStream_t)stream, dtype, a, p));
  return CDCLQ_OK;
}

}  // extern "C"
