// torch.ops.tdc.* of the row operators (rows_*.hip).  Unlike the iteration's ops, which write
// into buffers of the engine, these return new tensors: a request is one call from Python,
// and under graph capture the allocations belong to the graph's own pool.  The gradients are
// C++ nodes: the autograd engine's worker thread runs them without the interpreter (measured
// with rms_norm of 4 x 64 rows, forward and torch.autograd.grad: 59 us against 83 us with
// nodes in Python).
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <cmath>
#include <limits>

#include "kernels.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using c10::SymInt;
using DevGuard = at::hip::HIPGuardMasqueradingAsCUDA;

hipStream_t cur_stream() { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

constexpr int64_t MAX_WIDTH = 16384;
constexpr int64_t MAX_SLOTS = std::numeric_limits<int32_t>::max() - 1;
constexpr int64_t MAX_COLUMNS = 1 << 24;  // of grouped rows: passes over a row are grid blocks

int code_of(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return TDC_F32;
    case at::kHalf: return TDC_F16;
    case at::kBFloat16: return TDC_BF16;
    default: TORCH_CHECK_VALUE(false, what, " must be fp32, fp16 or bf16, got ", t);
  }
  return -1;
}

void check(int err, const char* what) {
  TORCH_CHECK(err == 0, "tdc: ", what, " failed: ", hipGetErrorString((hipError_t)err), " (code ",
              err, ")");
}

// A new tensor on `like`'s device, without the dispatcher's rounds (0.4 us each).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType t, const Tensor& like) {
  return at::detail::empty_cuda(sizes, t, like.device(), std::nullopt);
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

// Arguments that a caller gets wrong raise ValueError, as the checks of the CPU path do.  The
// checks are those of the shape functions too, where sizes may be symbols.
void check_rows(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.dim() == 2, name, " must be rows [N, D], got ", x.sym_sizes());
  TORCH_CHECK_VALUE(x.sym_size(1) >= 1, name, " has no columns");
  TORCH_CHECK_VALUE(x.sym_stride(1) == 1 || x.sym_size(1) == 1, name,
                    " must have contiguous columns, got strides ", x.sym_strides());
}

void check_like(const Tensor& t, const Tensor& x, const char* name) {
  check_rows(t, name);
  TORCH_CHECK_VALUE(t.device() == x.device() && t.scalar_type() == x.scalar_type() &&
                        t.sym_sizes() == x.sym_sizes(),
                    name, " must have the shape, type and device of the rows");
}

// Weights of shape `sizes`: null, fp32 (w32) or the rows' type.
void check_weights(const OptTensor& w, const Tensor& x, c10::SymIntArrayRef sizes, const char* name) {
  if (!has(w)) return;
  TORCH_CHECK_VALUE(w->sym_sizes() == sizes && w->is_contiguous(), name, " must be contiguous ",
                    sizes, ", got ", w->sym_sizes());
  TORCH_CHECK_VALUE(w->device() == x.device(), name, " is on ", w->device(), ", the rows on ",
                    x.device());
  TORCH_CHECK_VALUE(w->scalar_type() == at::kFloat || w->scalar_type() == x.scalar_type(), name,
                    " must be fp32 or of the rows' type, got ", w->scalar_type());
}
const void* weights_of(const OptTensor& w, bool& w32) {
  w32 = !has(w) || w->scalar_type() == at::kFloat;
  return has(w) ? w->data_ptr() : nullptr;
}

void check_index(const Tensor& t, const Tensor& x, const SymInt& n, const char* name) {
  TORCH_CHECK_VALUE(t.device() == x.device(), "the plan is on ", t.device(), ", the rows on ",
                    x.device());
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.is_contiguous() && t.sym_numel() == n, "tdc: ", name,
                    " must be int32 [", n, "]");
}

int num_cus(const Tensor& t) {
  int v = 0;
  if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, t.device().index()) !=
          hipSuccess || v <= 0)
    v = 256;
  return v;
}

// ------------------------------------------------------------------ norm
int check_norm(const Tensor& x, const OptTensor& w, const OptTensor& r, double eps, int64_t fp8_width) {
  check_rows(x, "x");
  const SymInt d = x.sym_size(1);
  const int code = code_of(x.scalar_type(), "x");
  TORCH_CHECK_VALUE(d <= MAX_WIDTH && fp8_width <= MAX_WIDTH, "rms_norm takes up to ", MAX_WIDTH,
                    " columns, got ", d);
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps must be finite and not negative, got ", eps);
  TORCH_CHECK(fp8_width == 0 || (fp8_width % 32 == 0 && d <= fp8_width), "tdc.rms_norm: fp8 width");
  if (has(r)) check_like(*r, x, "residual");
  check_weights(w, x, {d}, "weight");
  return code;
}

std::vector<Tensor> norm_impl(const Tensor& x, const OptTensor& w, const OptTensor& r, double eps,
                              bool want_rstd, int64_t fp8_width) {
  const int code = check_norm(x, w, r, eps, fp8_width);
  const int64_t n = x.size(0), d = x.size(1);
  bool w32;
  const void* wp = weights_of(w, w32);
  const DevGuard guard(x.device());
  std::vector<Tensor> res;
  Tensor q, s, y;
  if (fp8_width) {
    q = fresh({n, fp8_width}, at::kFloat8_e4m3fn, x);
    s = fresh({n, fp8_width / 32}, at::kByte, x);
    res = {q, s};
  } else {
    y = fresh({n, d}, x.scalar_type(), x);
    res = {y};
  }
  Tensor h, rstd;
  if (has(r)) {
    h = fresh({n, d}, x.scalar_type(), x);
    res.push_back(h);
  }
  if (want_rstd) {
    rstd = fresh({n}, at::kFloat, x);
    res.push_back(rstd);
  }
  check(tdc_rms_norm(code, x.data_ptr(), x.stride(0), has(r) ? r->data_ptr() : nullptr,
                     has(r) ? r->stride(0) : 0, wp, w32, n, (int)d, eps,
                     y.defined() ? y.data_ptr() : nullptr, q.defined() ? q.data_ptr() : nullptr,
                     s.defined() ? s.data_ptr() : nullptr, (int)fp8_width,
                     h.defined() ? h.data_ptr() : nullptr,
                     rstd.defined() ? rstd.data_ptr<float>() : nullptr, cur_stream()),
        "rms_norm");
  return res;
}

std::vector<Tensor> rms_norm(const Tensor& x, const OptTensor& w, const OptTensor& r, double eps) {
  return norm_impl(x, w, r, eps, false, 0);
}
// with what the gradient needs: y[, h], rstd
std::vector<Tensor> rms_norm_train(const Tensor& x, const OptTensor& w, const OptTensor& r,
                                   double eps) {
  return norm_impl(x, w, r, eps, true, 0);
}
std::vector<Tensor> rms_norm_fp8(const Tensor& x, const OptTensor& w, const OptTensor& r, double eps,
                                 int64_t width) {
  TORCH_CHECK(width > 0, "tdc.rms_norm_fp8: width");
  return norm_impl(x, w, r, eps, false, width);
}

std::vector<Tensor> rms_norm_bwd(const Tensor& h, const OptTensor& w, const Tensor& rstd,
                                 const Tensor& dy, const OptTensor& dh, bool want_dx,
                                 bool want_dw) {
  check_rows(h, "h");
  check_like(dy, h, "dy");
  if (has(dh)) check_like(*dh, h, "dh");
  const int64_t n = h.size(0), d = h.size(1);
  const int code = code_of(h.scalar_type(), "h");
  check_weights(w, h, {SymInt(d)}, "weight");
  TORCH_CHECK(d >= 1 && d <= MAX_WIDTH, "tdc.rms_norm_bwd: width");
  TORCH_CHECK(rstd.device() == h.device() && rstd.scalar_type() == at::kFloat &&
                  rstd.is_contiguous() && rstd.numel() == n, "tdc.rms_norm_bwd: rstd fp32 [N]");
  TORCH_CHECK(!want_dw || has(w), "tdc.rms_norm_bwd: dw needs the weights");
  TORCH_CHECK(want_dx || (want_dw && !has(dh)), "tdc.rms_norm_bwd: nothing to compute, or dh without dx");
  bool w32;
  const void* wp = weights_of(w, w32);
  const DevGuard guard(h.device());
  std::vector<Tensor> res;
  Tensor dx, part, dw;
  if (want_dx) {
    dx = fresh({n, d}, h.scalar_type(), h);
    res.push_back(dx);
  }
  const int parts = tdc_rms_norm_bwd_parts(n, num_cus(h));
  if (want_dw) {
    dw = fresh({d}, w->scalar_type(), *w);
    part = fresh({parts, d}, at::kFloat, h);
    res.push_back(dw);
  }
  check(tdc_rms_norm_bwd(code, h.data_ptr(), h.stride(0), rstd.data_ptr<float>(), wp, w32,
                         dy.data_ptr(), dy.stride(0), has(dh) ? dh->data_ptr() : nullptr,
                         has(dh) ? dh->stride(0) : 0, n, (int)d,
                         dx.defined() ? dx.data_ptr() : nullptr,
                         part.defined() ? part.data_ptr<float>() : nullptr, parts,
                         dw.defined() ? dw.data_ptr() : nullptr, cur_stream()),
        "rms_norm_bwd");
  return res;
}

Tensor dequant_fp8(const Tensor& q, const Tensor& s, int64_t d, at::ScalarType dtype) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kFloat8_e4m3fn && q.dim() == 2 &&
                  q.is_contiguous() && q.size(1) % 32 == 0 && d >= 1 && d <= q.size(1) &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "tdc.dequant_fp8: q float8_e4m3fn [N, 32 m], 16-byte aligned");
  TORCH_CHECK(s.device() == q.device() && s.scalar_type() == at::kByte && s.is_contiguous() &&
                  s.numel() == q.size(0) * (q.size(1) / 32), "tdc.dequant_fp8: s uint8 [N, m]");
  const int code = code_of(dtype, "dtype");
  const DevGuard guard(q.device());
  Tensor out = fresh({q.size(0), d}, dtype, q);
  check(tdc_dequant_fp8(code, q.data_ptr(), s.data_ptr(), q.size(0), (int)d, (int)q.size(1),
                        out.data_ptr(), cur_stream()),
        "dequant_fp8");
  return out;
}

// ------------------------------------------------------------------ gate
void check_mask(const OptTensor& mask, const Tensor& scores) {
  if (!has(mask)) return;
  TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool, "mask must be a bool tensor");
  TORCH_CHECK_VALUE(mask->device() == scores.device(), "mask is on ", mask->device(),
                    ", the scores on ", scores.device());
  TORCH_CHECK_VALUE(mask->sym_sizes() == scores.sym_sizes(), "mask must be [N, K], got ",
                    mask->sym_sizes());
}

struct MaskArg {
  const uint8_t* p = nullptr;
  int64_t rs = 0, cs = 0;
};

MaskArg mask_of(const OptTensor& mask) {
  MaskArg m;
  if (!has(mask)) return m;
  m.p = static_cast<const uint8_t*>(mask->data_ptr());
  m.rs = mask->stride(0);
  m.cs = mask->stride(1);
  return m;
}

int check_gate(const Tensor& scores, const OptTensor& mask, int64_t k) {
  check_rows(scores, "scores");
  const SymInt n = scores.sym_size(0), K = scores.sym_size(1);
  const int code = code_of(scores.scalar_type(), "scores");
  TORCH_CHECK_VALUE(k >= 1 && k <= 16 && K >= k, "k must be 1 to ", K.min(16), ", got ", k);
  TORCH_CHECK_VALUE(K <= (1 << 30) && n <= MAX_SLOTS, "too many scores: ", scores.sym_sizes());
  check_mask(mask, scores);
  return code;
}

std::vector<Tensor> gate_impl(const Tensor& scores, const OptTensor& mask, int64_t k, bool normalize,
                              bool train) {
  const int code = check_gate(scores, mask, k);
  const int64_t n = scores.size(0), K = scores.size(1);
  const MaskArg m = mask_of(mask);
  const DevGuard guard(scores.device());
  Tensor w = fresh({n, k}, at::kFloat, scores);
  Tensor labels = fresh({n, k}, at::kInt, scores);
  std::vector<Tensor> res = {w, labels};
  Tensor chosen, stat;
  if (train) {
    chosen = fresh({n, k, 2}, at::kInt, scores);
    res.push_back(chosen);
    if (!normalize) {
      stat = fresh({n, 2}, at::kFloat, scores);
      res.push_back(stat);
    }
  }
  check(tdc_topk_gate(code, scores.data_ptr(), scores.stride(0), m.p, m.rs, m.cs, n, (int)K, (int)k,
                      normalize, w.data_ptr<float>(), labels.data_ptr<int32_t>(),
                      chosen.defined() ? chosen.data_ptr() : nullptr,
                      stat.defined() ? stat.data_ptr<float>() : nullptr, cur_stream()),
        "topk_gate");
  return res;
}

std::tuple<Tensor, Tensor> topk_gate(const Tensor& scores, const OptTensor& mask, int64_t k,
                                     bool normalize) {
  const std::vector<Tensor> out = gate_impl(scores, mask, k, normalize, false);
  return {out[0], out[1]};
}
// with what the gradient needs: w, labels, both again as pairs int32 [N, k, 2][, stat]
std::vector<Tensor> topk_gate_train(const Tensor& scores, const OptTensor& mask, int64_t k,
                                    bool normalize) {
  return gate_impl(scores, mask, k, normalize, true);
}

// scores, mask, stat: given without `normalize` only.
Tensor topk_gate_bwd(const OptTensor& scores, const OptTensor& mask, const Tensor& chosen,
                     const OptTensor& stat, const Tensor& dw, int64_t K, at::ScalarType dtype) {
  TORCH_CHECK(chosen.is_cuda() && chosen.dim() == 3 && chosen.size(2) == 2 &&
                  chosen.scalar_type() == at::kInt && chosen.is_contiguous(),
              "tdc.topk_gate_bwd: chosen int32 [N, k, 2]");
  const int64_t n = chosen.size(0), k = chosen.size(1);
  TORCH_CHECK(dw.device() == chosen.device() && dw.scalar_type() == at::kFloat && dw.is_contiguous() &&
                  dw.numel() == n * k, "tdc.topk_gate_bwd: dw fp32 [N, k]");
  const int code = code_of(dtype, "scores");
  const bool normalize = !has(scores);
  MaskArg m;
  if (!normalize) {
    check_rows(*scores, "scores");
    TORCH_CHECK(scores->device() == chosen.device() && scores->scalar_type() == dtype &&
                    scores->size(0) == n && scores->size(1) == K, "tdc.topk_gate_bwd: scores");
    TORCH_CHECK(has(stat) && stat->device() == chosen.device() &&
                    stat->scalar_type() == at::kFloat && stat->is_contiguous() && stat->numel() == 2 * n, "tdc.topk_gate_bwd: stat");
    check_mask(mask, *scores);
    m = mask_of(mask);
  }
  const DevGuard guard(chosen.device());
  Tensor ds = fresh({n, K}, dtype, chosen);
  check(tdc_topk_gate_bwd(code, normalize ? nullptr : scores->data_ptr(),
                          normalize ? 0 : scores->stride(0), m.p, m.rs, m.cs, chosen.data_ptr(),
                          normalize ? nullptr : stat->data_ptr<float>(),
                          dw.data_ptr<float>(), n, (int)K, (int)k, normalize, ds.data_ptr(),
                          cur_stream()),
        "topk_gate_bwd");
  return ds;
}

// ------------------------------------------------------------------ groups
void check_plan(const Tensor& given, int64_t K) {
  TORCH_CHECK_VALUE((given.dim() == 1 || given.dim() == 2) &&
                        (given.scalar_type() == at::kInt || given.scalar_type() == at::kLong),
                    "labels must be int32 or int64 [N] or [N, k], got ", given.scalar_type(), " ",
                    given.sym_sizes());
  TORCH_CHECK_VALUE(given.dim() == 1 || given.sym_size(1) >= 1, "labels have no columns");
  TORCH_CHECK_VALUE(K >= 1 && K < (1 << 22), "n_clusters must be 1 to ", (1 << 22) - 1, ", got ", K);
  TORCH_CHECK_VALUE(given.sym_numel() <= MAX_SLOTS, "at most ", MAX_SLOTS, " labels, got ",
                    given.sym_numel());
}

std::vector<Tensor> group_plan(const Tensor& given, int64_t K) {
  check_plan(given, K);
  const int64_t m = given.numel();
  const Tensor labels = given.contiguous();
  const DevGuard guard(labels.device());
  Tensor offsets = fresh({K + 1}, at::kInt, labels);
  Tensor order = fresh({m}, at::kInt, labels);
  Tensor pos = fresh(labels.sizes(), at::kInt, labels);
  const int64_t words = tdc_group_plan_work(m, (int)K);
  Tensor work;
  if (words) work = fresh({words}, at::kInt, labels);
  check(tdc_group_plan(labels.scalar_type() == at::kLong, labels.data_ptr(), m, (int)K,
                       words ? work.data_ptr<int32_t>() : nullptr, order.data_ptr<int32_t>(),
                       pos.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), cur_stream()),
        "group_plan");
  return {offsets, order, pos};
}

// pos int32 [N, k] or [N]: the slots of each row.
SymInt slots_of(const Tensor& offsets, const Tensor& pos, const Tensor& like) {
  TORCH_CHECK((pos.dim() == 1 || pos.dim() == 2) && offsets.dim() == 1 && offsets.sym_numel() >= 2,
              "tdc: pos [N] or [N, k], offsets [K + 1]");
  check_index(offsets, like, offsets.sym_numel(), "offsets");
  check_index(pos, like, pos.sym_numel(), "pos");
  TORCH_CHECK(pos.sym_numel() <= MAX_SLOTS, "tdc: too many slots");
  return pos.dim() == 1 ? SymInt(1) : pos.sym_size(1);
}
int64_t slots(const Tensor& pos) { return pos.dim() == 1 ? 1 : pos.size(1); }

int check_group(const Tensor& x, const Tensor& offsets, const Tensor& pos) {
  check_rows(x, "x");
  slots_of(offsets, pos, x);
  const int code = code_of(x.scalar_type(), "x");
  TORCH_CHECK_VALUE(pos.sym_size(0) == x.sym_size(0), "the plan is of ", pos.sym_size(0),
                    " rows, x has ", x.sym_size(0));
  TORCH_CHECK_VALUE(x.sym_size(1) <= MAX_COLUMNS, "at most ", MAX_COLUMNS, " columns, got ",
                    x.sym_size(1));
  return code;
}

Tensor group_rows(const Tensor& x, const Tensor& offsets, const Tensor& pos) {
  const int code = check_group(x, offsets, pos);
  const int64_t n = x.size(0), d = x.size(1), k = slots(pos);
  const DevGuard guard(x.device());
  Tensor out = fresh({n * k, d}, x.scalar_type(), x);
  check(tdc_group_rows(code, x.data_ptr(), x.stride(0), n, (int)k, (int)d,
                       offsets.data_ptr<int32_t>(), (int)offsets.numel() - 1,
                       pos.data_ptr<int32_t>(), out.data_ptr(), cur_stream()),
        "group_rows");
  return out;
}

int check_combine(const Tensor& y, const Tensor& offsets, const Tensor& pos, const OptTensor& w) {
  check_rows(y, "y");
  const SymInt places = slots_of(offsets, pos, y) * pos.sym_size(0);
  const int code = code_of(y.scalar_type(), "y");
  TORCH_CHECK_VALUE(y.sym_size(0) == places, "the plan is of ", places, " places, y has ",
                    y.sym_size(0), " rows");
  TORCH_CHECK_VALUE(y.sym_size(1) <= MAX_COLUMNS, "at most ", MAX_COLUMNS, " columns, got ",
                    y.sym_size(1));
  check_weights(w, y, pos.sym_sizes(), "weights");
  return code;
}

Tensor combine_rows(const Tensor& y, const Tensor& offsets, const Tensor& pos, const OptTensor& w) {
  const int code = check_combine(y, offsets, pos, w);
  const int64_t n = pos.size(0), d = y.size(1), k = slots(pos);
  bool w32;
  const void* wp = weights_of(w, w32);
  const DevGuard guard(y.device());
  Tensor out = fresh({n, d}, y.scalar_type(), y);
  check(tdc_combine_rows(code, y.data_ptr(), y.stride(0), n, (int)k, (int)d,
                         offsets.data_ptr<int32_t>(), (int)offsets.numel() - 1,
                         pos.data_ptr<int32_t>(), wp, w32, out.data_ptr(), cur_stream()),
        "combine_rows");
  return out;
}

// y: given where the weights' gradient is wanted.
std::vector<Tensor> combine_rows_bwd(const Tensor& dout, const OptTensor& y, const Tensor& offsets,
                                     const Tensor& pos, const OptTensor& w, bool want_dy) {
  check_rows(dout, "dout");
  slots_of(offsets, pos, dout);
  const int64_t n = dout.size(0), d = dout.size(1), k = slots(pos);
  const int code = code_of(dout.scalar_type(), "dout");
  TORCH_CHECK(pos.size(0) == n && d >= 1 && d <= MAX_SLOTS,
              "tdc.combine_rows_bwd: rows do not fit the plan");
  check_weights(w, dout, pos.sym_sizes(), "weights");
  bool w32;
  const void* wp = weights_of(w, w32);
  const bool want_dw = has(y);
  if (want_dw) {
    check_rows(*y, "y");
    TORCH_CHECK(wp != nullptr || n * k == 0, "tdc.combine_rows_bwd: dw needs the weights");
    TORCH_CHECK(has(w) && y->device() == dout.device() && y->scalar_type() == dout.scalar_type() &&
                    y->size(0) == n * k && y->size(1) == d, "tdc.combine_rows_bwd: y");
  }
  const DevGuard guard(dout.device());
  Tensor dy, dw;
  std::vector<Tensor> res;
  if (want_dy) {
    dy = fresh({n * k, d}, dout.scalar_type(), dout);
    res.push_back(dy);
  }
  if (want_dw) {
    dw = fresh(w->sizes(), w->scalar_type(), *w);
    res.push_back(dw);
  }
  check(tdc_combine_rows_bwd(code, dout.data_ptr(), dout.stride(0),
                             want_dw ? y->data_ptr() : nullptr, want_dw ? y->stride(0) : 0, n,
                             (int)k, (int)d, offsets.data_ptr<int32_t>(), (int)offsets.numel() - 1,
                             pos.data_ptr<int32_t>(), wp, w32, want_dy ? dy.data_ptr() : nullptr,
                             want_dw ? dw.data_ptr() : nullptr, cur_stream()),
        "combine_rows_bwd");
  return res;
}

// ------------------------------------------------------------------ shapes
// The results of each operator as tensors without data: what tracing and compilation run in
// the kernels' place.
Tensor shaped(c10::SymIntArrayRef sizes, at::ScalarType t, const Tensor& like) {
  return at::empty_symint(sizes, at::TensorOptions().dtype(t).device(like.device()));
}

std::vector<Tensor> norm_shapes(const Tensor& x, const OptTensor& w, const OptTensor& r, double eps,
                                bool want_rstd, int64_t fp8_width) {
  check_norm(x, w, r, eps, fp8_width);
  const SymInt n = x.sym_size(0), d = x.sym_size(1);
  std::vector<Tensor> res;
  if (fp8_width) {
    res = {shaped({n, fp8_width}, at::kFloat8_e4m3fn, x), shaped({n, fp8_width / 32}, at::kByte, x)};
  } else {
    res = {shaped({n, d}, x.scalar_type(), x)};
  }
  if (has(r)) res.push_back(shaped({n, d}, x.scalar_type(), x));
  if (want_rstd) res.push_back(shaped({n}, at::kFloat, x));
  return res;
}
std::vector<Tensor> rms_norm_shapes(const Tensor& x, const OptTensor& w, const OptTensor& r,
                                    double eps) {
  return norm_shapes(x, w, r, eps, false, 0);
}
std::vector<Tensor> rms_norm_train_shapes(const Tensor& x, const OptTensor& w, const OptTensor& r,
                                          double eps) {
  return norm_shapes(x, w, r, eps, true, 0);
}
std::vector<Tensor> rms_norm_fp8_shapes(const Tensor& x, const OptTensor& w, const OptTensor& r,
                                        double eps, int64_t width) {
  return norm_shapes(x, w, r, eps, false, width);
}
std::vector<Tensor> rms_norm_bwd_shapes(const Tensor& h, const OptTensor& w, const Tensor&,
                                        const Tensor&, const OptTensor&, bool want_dx,
                                        bool want_dw) {
  std::vector<Tensor> res;
  if (want_dx) res.push_back(shaped(h.sym_sizes(), h.scalar_type(), h));
  if (want_dw) res.push_back(shaped(w->sym_sizes(), w->scalar_type(), *w));
  return res;
}
Tensor dequant_fp8_shapes(const Tensor& q, const Tensor&, SymInt d, at::ScalarType dtype) {
  return shaped({q.sym_size(0), std::move(d)}, dtype, q);
}

std::tuple<Tensor, Tensor> topk_gate_shapes(const Tensor& scores, const OptTensor& mask, int64_t k,
                                            bool) {
  check_gate(scores, mask, k);
  const SymInt n = scores.sym_size(0);
  return {shaped({n, k}, at::kFloat, scores), shaped({n, k}, at::kInt, scores)};
}
std::vector<Tensor> topk_gate_train_shapes(const Tensor& scores, const OptTensor& mask, int64_t k,
                                           bool normalize) {
  const auto [w, labels] = topk_gate_shapes(scores, mask, k, normalize);
  const SymInt n = scores.sym_size(0);
  const Tensor chosen = shaped({n, k, 2}, at::kInt, scores);
  if (normalize) return {w, labels, chosen};
  return {w, labels, chosen, shaped({n, 2}, at::kFloat, scores)};
}
Tensor topk_gate_bwd_shapes(const OptTensor&, const OptTensor&, const Tensor& chosen,
                            const OptTensor&, const Tensor&, SymInt K, at::ScalarType dtype) {
  return shaped({chosen.sym_size(0), std::move(K)}, dtype, chosen);
}

std::vector<Tensor> group_plan_shapes(const Tensor& labels, int64_t K) {
  check_plan(labels, K);
  return {shaped({K + 1}, at::kInt, labels), shaped({labels.sym_numel()}, at::kInt, labels),
          shaped(labels.sym_sizes(), at::kInt, labels)};
}
Tensor group_rows_shapes(const Tensor& x, const Tensor& offsets, const Tensor& pos) {
  check_group(x, offsets, pos);
  return shaped({pos.sym_numel(), x.sym_size(1)}, x.scalar_type(), x);
}
Tensor combine_rows_shapes(const Tensor& y, const Tensor& offsets, const Tensor& pos,
                           const OptTensor& w) {
  check_combine(y, offsets, pos, w);
  return shaped({pos.sym_size(0), y.sym_size(1)}, y.scalar_type(), y);
}
std::vector<Tensor> combine_rows_bwd_shapes(const Tensor& dout, const OptTensor& y, const Tensor&,
                                            const Tensor& pos, const OptTensor& w, bool want_dy) {
  std::vector<Tensor> res;
  if (want_dy) res.push_back(shaped({pos.sym_numel(), dout.sym_size(1)}, dout.scalar_type(), dout));
  if (has(y)) res.push_back(shaped(w->sym_sizes(), w->scalar_type(), *w));
  return res;
}

// ------------------------------------------------------------------ autograd
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// The operator tdc::NAME below autograd, with the signature of its kernel.  Not the kernel
// itself: what stands between the two (dispatch modes, tracing) sees the call as it sees
// PyTorch's own (0.1 us of a call).
#define TDC_BELOW_AUTOGRAD(NAME, ...)                                                     \
  [&] {                                                                                   \
    static const auto op =                                                                \
        c10::Dispatcher::singleton().findSchemaOrThrow("tdc::" #NAME, "").typed<decltype(NAME##_shapes)>(); \
    const at::AutoDispatchBelowADInplaceOrView below;                                     \
    return op.call(__VA_ARGS__);                                                          \
  }()

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return has(t) && t->requires_grad(); }

// An incoming gradient in a layout that the kernels take (broadcast ones are laid out).
Tensor laid_out(const Tensor& g) {
  if (!g.defined() || g.sym_size(1) <= 1 || g.sym_stride(1) == 1) return g;
  return g.contiguous();
}

// The gradients are not differentiable: asked for a graph, they give one that leads back to
// what they were computed `from` and raises when it is used.
variable_list once(variable_list grads, const variable_list& in, const variable_list& saved) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list have;
  for (const Tensor& g : grads)
    if (g.defined()) have.push_back(g);
  for (const variable_list* from : {&in, &saved})
    for (const Tensor& t : *from)
      if (wants_grad(t)) have.push_back(t);
  auto fn = std::make_shared<torch::autograd::DelayedError>(
      "tdc: the gradients of the row operators are not differentiable", (int64_t)have.size());
  have = (*fn)(std::move(have));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = have[i++];
  return grads;
}

// A gradient that is being captured may not go on to a node of the default stream, such as
// the accumulator that a leaf keeps while an eager graph of it lives: the engine would have
// that stream wait for the captured one, which ends the process.  Raises before it does.
void check_capture() {
  const at::hip::HIPStreamMasqueradingAsCUDA now = at::hip::getCurrentHIPStreamMasqueradingAsCUDA();
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(now.stream(), &status) != hipSuccess ||
      status == hipStreamCaptureStatusNone)
    return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const c10::Stream none =
      at::hip::getDefaultHIPStreamMasqueradingAsCUDA(now.device_index()).unwrap();
  for (const auto& edge : node->next_edges()) {
    if (!edge.is_valid()) continue;
    const auto stream = edge.function->stream();
    TORCH_CHECK(!stream || stream->device_index() != none.device_index() || *stream != none,
                "tdc: this gradient is being captured, but its input belongs to an autograd graph "
                "made outside of the capture: capture the forward pass too, and drop other graphs "
                "of the same leaves (or detach them) first");
  }
}

// Stand-ins for the inputs of the node that runs, for `once`: the gate's gradient is made from
// copies that no longer lead back to its scores.
variable_list inputs_of_node() {
  variable_list res;
  const auto node = torch::autograd::get_current_node();
  if (!node || !at::GradMode::is_enabled()) return res;
  for (const auto& edge : node->next_edges()) {
    if (!edge.is_valid()) continue;
    res.push_back(at::empty({0}, at::kFloat));
    torch::autograd::impl::set_gradient_edge(res.back(), edge);
  }
  return res;
}

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

struct RmsNorm : public Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w,
                               const OptTensor& r, double eps) {
    std::vector<Tensor> out = TDC_BELOW_AUTOGRAD(rms_norm_train, x, w, r, eps);
    Tensor rstd = out.back();
    out.pop_back();
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({has(r) ? out[1] : x, has(w) ? *w : Tensor(), rstd});
    ctx->saved_data["residual"] = has(r);
    // without a gradient of the rows, their sum has none either
    const bool rows = wants_grad(x) || wants_grad(r);
    if (has(r) && !rows) ctx->mark_non_differentiable({out[1]});
    ctx->saved_data["dx"] = rows;
    ctx->saved_data["dw"] = wants_grad(w);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    const auto saved = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    const bool want_dx = ctx->saved_data["dx"].toBool();
    const bool want_dw = ctx->saved_data["dw"].toBool();
    const Tensor dh = grads.size() > 1 ? laid_out(grads[1]) : Tensor();
    variable_list res(4);
    if (!grads[0].defined()) {  // only the sum was used
      res[0] = dh;
    } else {
      const std::vector<Tensor> g =
          TDC_BELOW_AUTOGRAD(rms_norm_bwd, saved[0], opt(saved[1]), saved[2], laid_out(grads[0]),
                             opt(dh), want_dx, want_dw);
      if (want_dx) res[0] = g[0];
      if (want_dw) res[1] = g.back();
    }
    if (residual) res[2] = res[0];
    return once(res, grads, saved);
  }
};

struct TopkGate : public Function<TopkGate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& scores, const OptTensor& mask,
                               int64_t k, bool normalize) {
    std::vector<Tensor> out = TDC_BELOW_AUTOGRAD(topk_gate_train, scores, mask, k, normalize);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[1]});
    // not the outputs, which the caller may edit; the weights over the chosen say all about
    // their gradient, those over every cluster need the scores again
    if (normalize)
      ctx->save_for_backward({out[2]});
    else
      ctx->save_for_backward({out[2], scores, out[3], has(mask) ? *mask : Tensor()});
    ctx->saved_data["clusters"] = scores.sym_size(1);
    ctx->saved_data["dtype"] = (int64_t)scores.scalar_type();
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    variable_list res(4);
    if (!grads[0].defined()) return res;
    const auto saved = ctx->get_saved_variables();
    const bool normalize = saved.size() == 1;
    const OptTensor none;
    res[0] = TDC_BELOW_AUTOGRAD(topk_gate_bwd, normalize ? none : opt(saved[1]),
                                normalize ? none : opt(saved[3]), saved[0],
                                normalize ? none : opt(saved[2]), grads[0].contiguous(),
                                ctx->saved_data["clusters"].toSymInt(),
                                (at::ScalarType)ctx->saved_data["dtype"].toInt());
    return once(res, grads, inputs_of_node());
  }
};

struct GroupRows : public Function<GroupRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& offsets,
                        const Tensor& pos) {
    ctx->save_for_backward({offsets, pos});
    return TDC_BELOW_AUTOGRAD(group_rows, x, offsets, pos);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    const auto saved = ctx->get_saved_variables();
    variable_list res(3);
    res[0] = TDC_BELOW_AUTOGRAD(combine_rows, laid_out(grads[0]), saved[0], saved[1], OptTensor());
    return once(res, grads, saved);
  }
};

struct CombineRows : public Function<CombineRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& offsets,
                        const Tensor& pos, const OptTensor& w) {
    ctx->save_for_backward({offsets, pos, has(w) ? *w : Tensor(), wants_grad(w) ? y : Tensor()});
    ctx->saved_data["dy"] = wants_grad(y);
    return TDC_BELOW_AUTOGRAD(combine_rows, y, offsets, pos, w);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    const auto saved = ctx->get_saved_variables();
    const bool want_dy = ctx->saved_data["dy"].toBool();
    const std::vector<Tensor> g =
        TDC_BELOW_AUTOGRAD(combine_rows_bwd, laid_out(grads[0]), opt(saved[3]), saved[0], saved[1],
                           opt(saved[2]), want_dy);
    variable_list res(4);
    if (want_dy) res[0] = g[0];
    if (saved[3].defined()) res[3] = g.back();
    return once(res, grads, saved);
  }
};

bool no_graph() { return !at::GradMode::is_enabled(); }

// There are no forward-mode formulas: an input with a tangent is refused, whether or not it
// asks for a gradient, since the result would go on without one.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), "tdc: ", what,
                              " has no forward-mode gradient");
}
void no_tangent(const OptTensor& t, const char* what) {
  if (t.has_value()) no_tangent(*t, what);
}

std::vector<Tensor> rms_norm_ad(const Tensor& x, const OptTensor& w, const OptTensor& r, double eps) {
  no_tangent(x, "rms_norm");
  no_tangent(w, "rms_norm");
  no_tangent(r, "rms_norm");
  if (no_graph() || !(wants_grad(x) || wants_grad(w) || wants_grad(r)))
    return TDC_BELOW_AUTOGRAD(rms_norm, x, w, r, eps);
  return RmsNorm::apply(x, w, r, eps);
}

std::vector<Tensor> rms_norm_fp8_ad(const Tensor& x, const OptTensor& w, const OptTensor& r,
                                    double eps, int64_t width) {
  no_tangent(x, "rms_norm_fp8");
  no_tangent(w, "rms_norm_fp8");
  no_tangent(r, "rms_norm_fp8");
  return TDC_BELOW_AUTOGRAD(rms_norm_fp8, x, w, r, eps, width);
}

std::tuple<Tensor, Tensor> topk_gate_ad(const Tensor& scores, const OptTensor& mask, int64_t k,
                                        bool normalize) {
  no_tangent(scores, "topk_gate");
  if (no_graph() || !wants_grad(scores))
    return TDC_BELOW_AUTOGRAD(topk_gate, scores, mask, k, normalize);
  const variable_list out = TopkGate::apply(scores, mask, k, normalize);
  return {out[0], out[1]};
}

Tensor group_rows_ad(const Tensor& x, const Tensor& offsets, const Tensor& pos) {
  no_tangent(x, "group_rows");
  if (no_graph() || !wants_grad(x)) return TDC_BELOW_AUTOGRAD(group_rows, x, offsets, pos);
  return GroupRows::apply(x, offsets, pos);
}

Tensor combine_rows_ad(const Tensor& y, const Tensor& offsets, const Tensor& pos, const OptTensor& w) {
  no_tangent(y, "combine_rows");
  no_tangent(w, "combine_rows");
  if (no_graph() || !(wants_grad(y) || wants_grad(w)))
    return TDC_BELOW_AUTOGRAD(combine_rows, y, offsets, pos, w);
  return CombineRows::apply(y, offsets, pos, w);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(tdc, m) {
  m.def("rms_norm(Tensor x, Tensor? w, Tensor? r, float eps) -> Tensor[]");
  m.def("rms_norm_fp8(Tensor x, Tensor? w, Tensor? r, float eps, int width) -> Tensor[]");
  m.def("dequant_fp8(Tensor q, Tensor s, SymInt d, ScalarType dtype) -> Tensor");
  m.def("topk_gate(Tensor scores, Tensor? mask, int k, bool normalize) -> (Tensor, Tensor)");
  m.def("group_plan(Tensor labels, int K) -> Tensor[]");
  m.def("group_rows(Tensor x, Tensor offsets, Tensor pos) -> Tensor");
  m.def("combine_rows(Tensor y, Tensor offsets, Tensor pos, Tensor? w) -> Tensor");
  // the two halves of the autograd nodes
  m.def("rms_norm_train(Tensor x, Tensor? w, Tensor? r, float eps) -> Tensor[]");
  m.def("rms_norm_bwd(Tensor h, Tensor? w, Tensor rstd, Tensor dy, Tensor? dh, "
        "bool want_dx, bool want_dw) -> Tensor[]");
  m.def("topk_gate_train(Tensor scores, Tensor? mask, int k, bool normalize) -> Tensor[]");
  m.def("topk_gate_bwd(Tensor? scores, Tensor? mask, Tensor chosen, Tensor? stat, Tensor dw, "
        "SymInt K, ScalarType dtype) -> Tensor");
  m.def("combine_rows_bwd(Tensor dout, Tensor? y, Tensor offsets, Tensor pos, Tensor? w, "
        "bool want_dy) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(tdc, CUDA, m) {
  m.impl("rms_norm", &rms_norm);
  m.impl("rms_norm_fp8", &rms_norm_fp8);
  m.impl("dequant_fp8", &dequant_fp8);
  m.impl("topk_gate", &topk_gate);
  m.impl("group_plan", &group_plan);
  m.impl("group_rows", &group_rows);
  m.impl("combine_rows", &combine_rows);
  m.impl("rms_norm_train", &rms_norm_train);
  m.impl("rms_norm_bwd", &rms_norm_bwd);
  m.impl("topk_gate_train", &topk_gate_train);
  m.impl("topk_gate_bwd", &topk_gate_bwd);
  m.impl("combine_rows_bwd", &combine_rows_bwd);
}

TORCH_LIBRARY_IMPL(tdc, Meta, m) {
  m.impl("rms_norm", &rms_norm_shapes);
  m.impl("rms_norm_fp8", &rms_norm_fp8_shapes);
  m.impl("dequant_fp8", &dequant_fp8_shapes);
  m.impl("topk_gate", &topk_gate_shapes);
  m.impl("group_plan", &group_plan_shapes);
  m.impl("group_rows", &group_rows_shapes);
  m.impl("combine_rows", &combine_rows_shapes);
  m.impl("rms_norm_train", &rms_norm_train_shapes);
  m.impl("rms_norm_bwd", &rms_norm_bwd_shapes);
  m.impl("topk_gate_train", &topk_gate_train_shapes);
  m.impl("topk_gate_bwd", &topk_gate_bwd_shapes);
  m.impl("combine_rows_bwd", &combine_rows_bwd_shapes);
}

TORCH_LIBRARY_IMPL(tdc, AutogradCUDA, m) {
  m.impl("rms_norm", &rms_norm_ad);
  m.impl("rms_norm_fp8", &rms_norm_fp8_ad);
  m.impl("topk_gate", &topk_gate_ad);
  m.impl("group_rows", &group_rows_ad);
  m.impl("combine_rows", &combine_rows_ad);
}
