// C-ABI entry points of the operators that train and serve adapters on a packed model
// (include/cdclq.h): validation, workspace plans and the k_ckpt.hip / k_loss.hip / k_packed.hip /
// k_adapt.hip launches. They enqueue on the caller's stream and return; only the opening and closing of
// a packed layer allocates device memory and waits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <new>
#include <string>
#include <vector>

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

// Sizes whose tiles and tables are counted in 32 bits (and items in a grid's second dimension).
constexpr size_t kMaxTokens = (size_t)1 << 22, kMaxWidth = (size_t)1 << 20, kMaxVocab = (size_t)1 << 24;

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

// A packed layer in the layout of packed.h: one allocation on its GPU.
struct cdclq_packed {
  int device = 0;
  size_t bytes = 0;
  void* blob = nullptr;
  cdclq::PackedView view = {};
};

namespace {

// Tokens up to which the packed codes are decoded in the product's registers, 64 at a time (the most whose sums
// a wavefront holds for two row tiles); for more the weights are expanded to 16 bits first. 4096 -> 14336 in 4
// bits: 128 tokens 58 us against 79 expanded, 192 84 and 90, 256 96 and 91; 4096 -> 4096 in 8: 192 50 and 51,
// 256 65 and 52; 2048 -> 2048 in 4: 192 18 and 30.
constexpr size_t kFewTokens = 192;

int open_packed(cdclq_ctx* ctx, size_t m, size_t n, size_t group, const uint8_t* gbits, size_t ngroups,
                const uint8_t* qweight, size_t qweight_bytes, const uint16_t* scales, const uint8_t* qzeros,
                const int32_t* perm, cdclq_packed* p) {
  size_t rb = 0;
  if (m == 0 || n == 0) return fail(ctx, CDCLQ_INVALID_ARG, "a packed layer needs rows and columns");
  if (cdclq_row_bytes(n, group, gbits, ngroups, &rb) != CDCLQ_OK)
    return fail(ctx, CDCLQ_INVALID_ARG, "invalid packed layout (d_in " + std::to_string(n) + ", group " +
                                            std::to_string(group) + ", " + std::to_string(ngroups) + " groups)");
  CK(check_size(ctx, "d_out", m, (size_t)1 << 24));
  if (!qweight || !scales || !qzeros || !perm) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  if (qweight_bytes < m * rb)
    return fail(ctx, CDCLQ_INVALID_ARG, "qweight holds " + std::to_string(qweight_bytes) + " bytes, the layer needs " +
                                            std::to_string(m * rb));
  std::vector<int32_t> order(n);
  HIPCK(hipMemcpy(order.data(), perm, n * 4, hipMemcpyDeviceToHost));
  std::vector<uint8_t> seen(n, 0);
  for (int32_t c : order) {
    if (c < 0 || (size_t)c >= n || seen[c])
      return fail(ctx, CDCLQ_INVALID_ARG, "perm is not a permutation of 0..d_in (" + std::to_string(n) + ")");
    seen[c] = 1;
  }
  const size_t g = std::min(group, n), ng = (n + g - 1) / g;
  std::vector<int32_t> slotpos;
  std::vector<uint32_t> grp, coff(n);
  std::vector<uint8_t> cwid(n);
  for (size_t i = 0; i < ng; ++i) {
    const size_t c0 = i * g, c1 = std::min(n, c0 + g);
    for (size_t c = c0; c < c1; ++c) slotpos.push_back((int32_t)c);
    slotpos.resize((slotpos.size() + 31) / 32 * 32, -1);
    grp.resize(slotpos.size() / 32, (uint32_t)i);
  }
  slotpos.resize((slotpos.size() + 127) / 128 * 128, -1);
  grp.resize(slotpos.size() / 32, (uint32_t)(ng - 1));
  CK(check_size(ctx, "slot count", slotpos.size(), (size_t)1 << 22));
  uint32_t bit = 0;
  for (size_t c = 0; c < n; ++c) {
    coff[c] = bit;
    cwid[c] = gbits[c / group];
    bit += cwid[c];
  }
  const size_t nkb = slotpos.size() / 128;
  std::vector<uint32_t> kinfo(nkb);
  std::vector<int32_t> col(slotpos.size());
  std::vector<int32_t> slot(n);
  for (size_t i = 0; i < col.size(); ++i) {
    col[i] = slotpos[i] < 0 ? -1 : order[slotpos[i]];
    if (col[i] >= 0) slot[col[i]] = (int32_t)i;
  }
  uint32_t at = 0;
  int bits = -1;
  for (size_t k = 0; k < nkb; ++k) {
    uint32_t w = 0, ends = 8;
    for (size_t s = 0; s < 4; ++s) {
      w = std::max<uint32_t>(w, gbits[grp[4 * k + s]]);
      if (s < 3 && grp[4 * k + s] != grp[4 * k + s + 1]) ends |= 1u << s;
    }
    kinfo[k] = at << 8 | ends << 4 | w;
    at += w;
    bits = bits < 0 || bits == (int)w ? (int)w : 0;
  }
  PackedView& v = p->view;
  v.m = (int)m, v.n = (int)n, v.tiles = (int)((m + 15) / 16), v.ng = (int)ng, v.nkb = (int)nkb, v.bits = bits;
  v.tile_bytes = 256l * at;
  // one blob: codes, scales, then the tables
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t codes = up((size_t)v.tiles * v.tile_bytes), scl = up((size_t)v.tiles * ng * 64);
  const size_t tab[] = {up(4 * nkb), up(4 * grp.size()), up(4 * col.size()), up(4 * n)};
  const size_t tables = tab[0] + tab[1] + tab[2] + tab[3];
  const size_t build[] = {up(4 * slotpos.size()), up(4 * n), up(n)};
  p->bytes = codes + scl + tables;
  hipError_t e = hipMalloc(&p->blob, p->bytes);
  if (e != hipSuccess) {
    p->blob = nullptr;
    (void)hipGetLastError();
    return fail(ctx, CDCLQ_OOM, "device allocation of " + std::to_string(p->bytes) + " bytes failed (" +
                                    hipGetErrorString(e) + ")");
  }
  char* base = static_cast<char*>(p->blob);
  char* t = base + codes + scl;
  v.codes = reinterpret_cast<uint8_t*>(base);
  v.scl = reinterpret_cast<uint32_t*>(base + codes);
  v.kinfo = reinterpret_cast<uint32_t*>(t);
  v.grp = reinterpret_cast<uint32_t*>(t + tab[0]);
  v.col = reinterpret_cast<int*>(t + tab[0] + tab[1]);
  v.slot = reinterpret_cast<int*>(t + tab[0] + tab[1] + tab[2]);
  std::vector<char> host(tables + build[0] + build[1] + build[2], 0);
  std::memcpy(host.data(), kinfo.data(), 4 * nkb);
  std::memcpy(host.data() + tab[0], grp.data(), 4 * grp.size());
  std::memcpy(host.data() + tab[0] + tab[1], col.data(), 4 * col.size());
  std::memcpy(host.data() + tab[0] + tab[1] + tab[2], slot.data(), 4 * n);
  char* h = host.data() + tables;
  std::memcpy(h, slotpos.data(), 4 * slotpos.size());
  std::memcpy(h + build[0], coff.data(), 4 * n);
  std::memcpy(h + build[0] + build[1], cwid.data(), n);
  CK(ensure(ctx, ctx->pk_tab[2], build[0] + build[1] + build[2]));
  char* d = P<char>(ctx->pk_tab[2]);
  HIPCK(hipMemcpy(t, host.data(), tables, hipMemcpyHostToDevice));
  HIPCK(hipMemcpy(d, h, build[0] + build[1] + build[2], hipMemcpyHostToDevice));
  HIPCK(packed_layout(ctx->st, v, (int)ngroups, qweight, (long)rb, scales, qzeros, reinterpret_cast<int*>(d),
                      reinterpret_cast<uint32_t*>(d + build[0]), reinterpret_cast<uint8_t*>(d + build[0] + build[1]),
                      reinterpret_cast<uint8_t*>(base), reinterpret_cast<uint32_t*>(base + codes)));
  HIPCK(hipStreamSynchronize(ctx->st));
  return CDCLQ_OK;
}

int check_adapters(cdclq_ctx* ctx, const cdclq_packed* p, size_t t, int dtype, size_t adapters, size_t rank,
                   const void* a, const void* b, const float* scaling, const int32_t* request) {
  if (!p) return fail(ctx, CDCLQ_INVALID_ARG, "null packed layer");
  if (p->device != ctx->device)
    return fail(ctx, CDCLQ_INVALID_ARG, "the packed layer is on GPU " + std::to_string(p->device) + ", the context on " +
                                            std::to_string(ctx->device));
  CK(check_half(ctx, dtype));
  CK(check_size(ctx, "token count", t, kMaxTokens));
  CK(check_size(ctx, "adapter count", adapters, 32768));
  CK(check_size(ctx, "rank", rank, 128));
  if ((adapters == 0) != (rank == 0)) return fail(ctx, CDCLQ_INVALID_ARG, "adapters without a rank, or a rank without adapters");
  if (rank && (!a || !b || !scaling || (t && !request))) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  return CDCLQ_OK;
}

AdapterArgs adapter_args(const void* x, size_t ldx, size_t t, const void* a, const void* b, const float* scaling,
                         size_t adapters, size_t rank, const int32_t* request) {
  AdapterArgs r = {};
  r.t = (long)t;
  r.x = static_cast<const uint16_t*>(x);
  r.ldx = (long)ldx;
  r.a = static_cast<const uint16_t*>(a);
  r.b = static_cast<const uint16_t*>(b);
  r.scaling = scaling;
  r.adapters = (int)adapters;
  r.rank = (int)rank;
  r.request = request;
  return r;
}

size_t linear_bytes(const PackedView& v, const AdapterArgs& r) {
  return (size_t)r.t <= kFewTokens ? few_work_bytes(v, r.t, r.rank) : wide_work_bytes(v, r);
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

int cdclq_packed_open_device(cdclq_ctx* ctx, size_t d_out, size_t d_in, size_t group, const uint8_t* gbits,
                             size_t ngroups, const uint8_t* qweight, size_t qweight_bytes, const uint16_t* scales_f16,
                             const uint8_t* qzeros, const int32_t* perm_i32, cdclq_packed** out) {
  if (!ctx) return CDCLQ_INVALID_ARG;
  ctx->err.clear();
  if (!out) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  *out = nullptr;
  OnDevice on(ctx->device);
  HIPCK(on.err);
  cdclq_packed* p = new (std::nothrow) cdclq_packed();
  if (!p) return fail(ctx, CDCLQ_OOM, "host allocation failed");
  p->device = ctx->device;
  int rc;
  try {
    rc = open_packed(ctx, d_out, d_in, group, gbits, ngroups, qweight, qweight_bytes, scales_f16, qzeros, perm_i32, p);
  } catch (const std::bad_alloc&) {
    rc = fail(ctx, CDCLQ_OOM, "host allocation failed");
  }
  if (rc != CDCLQ_OK) {
    cdclq_packed_close(p);
    return rc;
  }
  *out = p;
  return CDCLQ_OK;
}

void cdclq_packed_close(cdclq_packed* p) {
  if (!p) return;
  {
    OnDevice on(p->device);
    if (p->blob) (void)hipFree(p->blob);  // waits for the GPU's work
  }
  delete p;
}

size_t cdclq_packed_bytes(const cdclq_packed* p) { return p ? p->bytes : 0; }

size_t cdclq_adapter_work_bytes(const cdclq_packed* packed, const void* x, size_t ldx, size_t t, const void* a,
                                const void* b, size_t adapters, size_t rank, int grad) {
  if (!packed || t > kMaxTokens || adapters > 32768 || rank > 128) return 0;
  const AdapterArgs r = adapter_args(x, ldx, t, a, b, nullptr, adapters, rank, nullptr);
  return grad ? grad_work_bytes(packed->view, r) : linear_bytes(packed->view, r);
}

int cdclq_adapter_linear_device(cdclq_ctx* ctx, const cdclq_packed* packed, const void* x, size_t ldx, size_t t,
                                int dtype, const void* a, const void* b, const float* scaling, size_t adapters,
                                size_t rank, const int32_t* request, void* y, size_t ldy, float* low, void* work,
                                size_t work_bytes, void* stream) {
  if (!ctx) return CDCLQ_INVALID_ARG;
  ctx->err.clear();
  CK(check_adapters(ctx, packed, t, dtype, adapters, rank, a, b, scaling, request));
  const PackedView& v = packed->view;
  CK(check_rows(ctx, "x", ldx, v.n));
  CK(check_rows(ctx, "y", ldy, v.m));
  if (t == 0) return CDCLQ_OK;
  if (!x || !y) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  AdapterArgs r = adapter_args(x, ldx, t, a, b, scaling, adapters, rank, request);
  r.y = static_cast<uint16_t*>(y);
  r.ldy = (long)ldy;
  r.low = low;
  CK(check_work(ctx, work, work_bytes, linear_bytes(v, r)));
  OnDevice on(ctx->device);
  HIPCK(on.err);
  if (t <= kFewTokens) HIPCK(adapter_few((hipStream_t)stream, dtype, v, r, work));
  else HIPCK(adapter_wide((hipStream_t)stream, dtype, v, r, work));
  return CDCLQ_OK;
}

int cdclq_adapter_backward_device(cdclq_ctx* ctx, const cdclq_packed* packed, const void* dy, size_t lddy, size_t t,
                                  int dtype, const int8_t* codes, const float* scales, const float* low, const void* a,
                                  const void* b, const float* scaling, size_t adapters, size_t rank,
                                  const int32_t* request, void* dx, size_t lddx, void* da, void* db, void* work,
                                  size_t work_bytes, void* stream) {
  if (!ctx) return CDCLQ_INVALID_ARG;
  ctx->err.clear();
  CK(check_adapters(ctx, packed, t, dtype, adapters, rank, a, b, scaling, request));
  const PackedView& v = packed->view;
  CK(check_rows(ctx, "dy", lddy, v.m));
  CK(check_rows(ctx, "dx", lddx, v.n));
  if (t && (!dy || !dx)) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  if (rank && (!da || !db || (t && (!codes || !scales || !low)))) return fail(ctx, CDCLQ_INVALID_ARG, "null buffer argument");
  if (t == 0 && rank == 0) return CDCLQ_OK;
  AdapterArgs r = adapter_args(dy, lddy, t, a, b, scaling, adapters, rank, request);
  r.y = static_cast<uint16_t*>(dx);
  r.ldy = (long)lddx;
  r.low = const_cast<float*>(low);
  r.codes = codes;
  r.scales = scales;
  r.da = static_cast<uint16_t*>(da);
  r.db = static_cast<uint16_t*>(db);
  CK(check_work(ctx, work, work_bytes, grad_work_bytes(v, r)));
  OnDevice on(ctx->device);
  HIPCK(on.err);
  HIPCK(adapter_grad((hipStream_t)stream, dtype, v, r, work));
  return CDCLQ_OK;
}

}  // extern "C"
