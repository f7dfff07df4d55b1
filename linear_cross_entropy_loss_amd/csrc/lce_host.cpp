// Host path of the Python operator (ops.py) for ordinary calls: from the tensors to one call of the C ABI (include/lce.h) and its
// results, without the interpreter in between.
//
// A step of a small problem is bound by the host: N=256, H=256, V=4096 in bf16 has 43 us of kernels and took 81 us of host time in
// Python, 51 here -- 160 and 106 where the threads of a backward, which wait for each other, sleep long enough for the processor's
// deeper idle states.
//
// What is no such call -- a tensor subclass, strides in no order of rows, a problem that the library refuses -- is not handled
// here: the functions return None before anything has been allocated or launched, and ops.py goes on as for any call, errors
// included.  Device calls go to the current device and the stream that is handed over; allocations come from torch's caching
// allocator, as the current stream's.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/Allocator.h>
#include <c10/core/InferenceMode.h>

#include <vector>

#include "../../include/lce.h"

namespace {

// The C ABI's functions, by the addresses that the loader of the library gives (bind).
struct Abi {
  decltype(&lce_strerror) strerror;
  decltype(&lce_last_hip_error) last_hip_error;
  decltype(&lce_check_problem) check_problem;
  decltype(&lce_workspace_bytes) workspace_bytes;
  decltype(&lce_forward) forward;
  decltype(&lce_backward) backward;
  decltype(&lce_forward_backward_workspace_bytes) forward_backward_workspace_bytes;
  decltype(&lce_forward_backward_plan) forward_backward_plan;
  decltype(&lce_forward_backward) forward_backward;
  decltype(&lce_stand_in) stand_in;
  decltype(&lce_unit_gradient) unit_gradient;
  decltype(&lce_pad_rows) pad_rows;
  decltype(&lce_transpose_rows) transpose_rows;
  decltype(&lce_soft_targets) soft_targets;
  decltype(&lce_distill_workspace_bytes) distill_workspace_bytes;
  decltype(&lce_distill) distill;
  decltype(&lce_top_logits) top_logits;
  decltype(&lce_sample) sample;
  decltype(&lce_token_labels) token_labels;
  decltype(&lce_token_logits_workspace_bytes) token_logits_workspace_bytes;
  decltype(&lce_token_logits) token_logits;
  decltype(&lce_token_logits_backward) token_logits_backward;
  decltype(&lce_quantize_rows) quantize_rows;
  decltype(&lce_quantize_columns) quantize_columns;
  decltype(&lce_int8_logits_workspace_bytes) int8_logits_workspace_bytes;
  decltype(&lce_int8_logits) int8_logits;
  decltype(&lce_clip_workspace_bytes) clip_workspace_bytes;
  decltype(&lce_clip) clip;
} abi;

template <class F> void bind_one(const py::dict& d, const char* name, F& f) { f = reinterpret_cast<F>(d[name].cast<uintptr_t>()); }
void bind(const py::dict& d) {
  bind_one(d, "lce_strerror", abi.strerror);
  bind_one(d, "lce_last_hip_error", abi.last_hip_error);
  bind_one(d, "lce_check_problem", abi.check_problem);
  bind_one(d, "lce_workspace_bytes", abi.workspace_bytes);
  bind_one(d, "lce_forward", abi.forward);
  bind_one(d, "lce_backward", abi.backward);
  bind_one(d, "lce_forward_backward_workspace_bytes", abi.forward_backward_workspace_bytes);
  bind_one(d, "lce_forward_backward_plan", abi.forward_backward_plan);
  bind_one(d, "lce_forward_backward", abi.forward_backward);
  bind_one(d, "lce_stand_in", abi.stand_in);
  bind_one(d, "lce_unit_gradient", abi.unit_gradient);
  bind_one(d, "lce_pad_rows", abi.pad_rows);
  bind_one(d, "lce_transpose_rows", abi.transpose_rows);
  bind_one(d, "lce_soft_targets", abi.soft_targets);
  bind_one(d, "lce_distill_workspace_bytes", abi.distill_workspace_bytes);
  bind_one(d, "lce_distill", abi.distill);
  bind_one(d, "lce_top_logits", abi.top_logits);
  bind_one(d, "lce_sample", abi.sample);
  bind_one(d, "lce_token_labels", abi.token_labels);
  bind_one(d, "lce_token_logits_workspace_bytes", abi.token_logits_workspace_bytes);
  bind_one(d, "lce_token_logits", abi.token_logits);
  bind_one(d, "lce_token_logits_backward", abi.token_logits_backward);
  bind_one(d, "lce_quantize_rows", abi.quantize_rows);
  bind_one(d, "lce_quantize_columns", abi.quantize_columns);
  bind_one(d, "lce_int8_logits_workspace_bytes", abi.int8_logits_workspace_bytes);
  bind_one(d, "lce_int8_logits", abi.int8_logits);
  bind_one(d, "lce_clip_workspace_bytes", abi.clip_workspace_bytes);
  bind_one(d, "lce_clip", abi.clip);
}

int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? LCE_BF16 : t == at::kHalf ? LCE_F16 : t == at::kFloat ? LCE_F32 : -1;
}
int64_t row_multiple(at::ScalarType t) { return t == at::kFloat ? 4 : 8; }

// A dense tensor on a GPU that is nothing but that.
bool plain(const at::Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.is_neg() &&
         !t.is_conj();
}
bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Memory that is given back when the call's launches have been issued (the allocator hands it out again in stream order).
struct Workspace {
  c10::DataPtr data;
  explicit Workspace(size_t n) : data(n > 0 ? c10::GetAllocator(c10::DeviceType::CUDA)->allocate(n) : c10::DataPtr()) {}
};

py::object tensor_or_none(const at::Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

// Row strides of matrices that are laid out here (ops.py, _padded_cols and _dx_cols).
int64_t padded_cols(int64_t cols, at::ScalarType t) {
  int64_t m = row_multiple(t);
  if (cols % m == 0) return cols;
  if (2 * cols >= 8 * m) m *= 8;
  return (cols + m - 1) / m * m;
}
int64_t dx_cols(int64_t H, at::ScalarType t) { return H % 4 == 0 ? H : padded_cols(H, t); }

// How the kernels come to a matrix: as it is, or from a copy whose rows start on 16-byte boundaries.
enum Copy { kInPlace, kByRows, kTransposed };
struct Call {
  lce_problem p;
  Copy x, w;
};

// x: rows of H, contiguous or (`strided`) with a row stride.  At: (H, V), as the operator takes it.  False: no ordinary call.
bool describe(const at::Tensor& x, const at::Tensor& At, bool strided, Call& c) {
  memset(&c, 0, sizeof(c));
  if (!plain(x) || !plain(At) || x.dim() < 1 || At.dim() != 2 || x.device() != At.device()) return false;
  const at::ScalarType xt = x.scalar_type(), wt = At.scalar_type();
  const int xd = dtype_code(xt), wd = dtype_code(wt);
  if (xd < 0 || (wd != xd && wd != LCE_F32)) return false;
  const int64_t H = x.size(-1), V = At.size(1), m = row_multiple(wt);
  if (H <= 0 || V <= 0 || At.size(0) != H || x.numel() <= 0) return false;
  lce_problem& p = c.p;
  if (strided) {
    if (x.dim() != 2 || x.stride(1) != 1 || x.stride(0) % row_multiple(xt) != 0 || x.stride(0) < H || !aligned(x)) return false;
    p.ldx = x.stride(0);
  } else {
    if (!x.is_contiguous()) return false;
    c.x = H % row_multiple(xt) == 0 && aligned(x) ? kInPlace : kByRows;
    p.ldx = c.x == kInPlace ? H : padded_cols(H, xt);
  }
  p.N = x.numel() / H;
  p.H = H;
  p.V = V;
  p.lddx = dx_cols(H, xt);
  p.x_dtype = p.dx_dtype = xd;
  p.w_dtype = p.dw_dtype = wd;
  p.w_layout = LCE_W_HV;
  if (At.stride(1) == 1 && At.stride(0) % m == 0 && At.stride(0) >= V) {
    if (!aligned(At)) return false;
    p.ldw = At.stride(0);
  } else if (xd != LCE_F32 && H % 8 == 0 && V > 1 && At.stride(0) == 1 && At.stride(1) % m == 0 && At.stride(1) >= H) {
    if (!aligned(At)) return false;
    p.w_layout = LCE_W_VH;
    p.ldw = At.stride(1);
  } else {
    if (At.stride(1) == 1 && At.stride(0) >= V) c.w = kByRows;
    else if (At.stride(0) == 1 && At.stride(1) >= H) c.w = kTransposed;
    else return false;
    p.ldw = padded_cols(V, wt);
  }
  p.lddw = padded_cols(p.w_layout == LCE_W_VH ? H : V, wt);
  return true;
}

at::Tensor rows_of(int64_t rows, int64_t cols, int64_t ld, const at::TensorOptions& o) {
  at::Tensor t = at::empty({rows, ld}, o);
  return ld == cols ? t : t.narrow(1, 0, cols);
}
int copy_rows(Copy how, const at::Tensor& from, int64_t rows, int64_t cols, const at::Tensor& to, int64_t ld, void* stream) {
  const int d = dtype_code(to.scalar_type());
  return how == kByRows ? abi.pad_rows(from.data_ptr(), d, rows, cols, from.dim() == 2 ? from.stride(0) : cols, to.data_ptr(), ld, stream)
                        : abi.transpose_rows(from.data_ptr(), d, rows, cols, from.stride(1), to.data_ptr(), ld, stream);
}

// The loss, and with `route` (1: where the library says so, 2: wherever it fits) and a gradient wanted, that too if one evaluation of
// the logits gives both: (out5, lse, n_valid, x, y, w, layout, dx, dw, pre), as ops.py's _one_pass_impl and _forward_impl return
// them, then whether the gradients are there; (status, name) where the C ABI refused; None: not handled.  `copy_w`: a weight that
// cannot be read in place may be copied here (ops.py says so to the user once).
py::object forward(const at::Tensor& x_in, const at::Tensor& y, const at::Tensor& At, int64_t ignore_index, double z_reg, double scale,
                   int64_t n_chunk, bool monitoring, int pack, int route, bool exact, bool need_dx, bool need_dw, bool copy_w, uintptr_t stream) {
  Call c;
  lce_problem& p = c.p;
  if (!describe(x_in, At, false, c) || (c.w != kInPlace && !copy_w) || !plain(y) || y.scalar_type() != at::kLong || y.device() != x_in.device() || !y.is_contiguous() ||
      y.numel() != p.N)
    return py::none();
  p.ignore_index = ignore_index;
  p.logit_scale = (float)scale;
  p.z_reg = (float)z_reg;
  p.n_chunk = n_chunk;
  p.monitoring = monitoring ? 1 : 0;
  p.pack_rows = pack;
  const bool grads = route > 0 && (need_dx || need_dw);
  if (grads)
    p.route = (route == 2 ? LCE_ROUTE_ONE_PASS : LCE_ROUTE_AUTO) | (exact ? LCE_ROUTE_EXACT_SUMS : 0) |
              (p.x_dtype == LCE_F32 ? LCE_ROUTE_KEEP_LOGITS : 0);
  if (abi.check_problem(&p) != LCE_OK) return py::none();
  int64_t chunks = 0;
  if (grads && abi.forward_backward_plan(&p, &chunks, nullptr) != LCE_OK) return py::none();
  size_t bytes = 0;
  if ((chunks > 0 ? abi.forward_backward_workspace_bytes(&p, &bytes) : abi.workspace_bytes(&p, &bytes, nullptr)) != LCE_OK)
    return py::none();

  at::NoGradGuard no_grad;
  const auto o = x_in.options();
  const at::Tensor y1 = y.dim() == 1 ? y : y.view({p.N});
  const at::Tensor x = c.x != kInPlace ? rows_of(p.N, p.H, p.ldx, o) : x_in.dim() == 2 ? x_in : x_in.view({p.N, p.H});
  const at::Tensor w = c.w != kInPlace ? rows_of(p.H, p.V, p.ldw, At.options()) : p.w_layout == LCE_W_VH ? At.t() : At;
  at::Tensor dx, dw, pre;
  if (chunks > 0 && need_dx) dx = rows_of(p.N, p.H, p.lddx, o);
  if (chunks > 0 && need_dw) dw = rows_of(w.size(0), w.size(1), p.lddw, At.options());
  const auto f32 = o.dtype(at::kFloat);
  const at::Tensor lse = at::empty({p.N}, f32), out5 = at::empty({5}, f32), n_valid = at::empty({1}, y.options());
  if (chunks > 0 && p.x_dtype == LCE_F16) pre = at::empty({1}, f32);
  Workspace ws(bytes);
  void* const s = reinterpret_cast<void*>(stream);
  int rc = LCE_OK;
  const char* what = chunks > 0 ? "lce_forward_backward" : "lce_forward";
  {
    py::gil_scoped_release release;
    if (c.x != kInPlace) rc = copy_rows(c.x, x_in, p.N, p.H, x, p.ldx, s);
    if (rc == LCE_OK && c.w != kInPlace) rc = copy_rows(c.w, At, p.H, p.V, w, p.ldw, s);
    if (rc != LCE_OK) {
      what = "lce_pad_rows";
    } else if (chunks > 0) {
      const float* g = nullptr;
      if (pre.defined()) {
        rc = abi.stand_in((const int64_t*)y1.data_ptr(), p.N, ignore_index, (float*)pre.data_ptr(), s);
        g = (const float*)pre.data_ptr();
      } else {
        rc = abi.unit_gradient(&g);
      }
      if (rc == LCE_OK)
        rc = abi.forward_backward(&p, x.data_ptr(), w.data_ptr(), (const int64_t*)y1.data_ptr(), g, (float*)lse.data_ptr(),
                                  (float*)out5.data_ptr(), (int64_t*)n_valid.data_ptr(), ptr(dx), ptr(dw), ws.data.get(), bytes, s);
    } else {
      rc = abi.forward(&p, x.data_ptr(), w.data_ptr(), (const int64_t*)y1.data_ptr(), (float*)lse.data_ptr(), (float*)out5.data_ptr(),
                       (int64_t*)n_valid.data_ptr(), ws.data.get(), bytes, s);
    }
  }
  if (rc != LCE_OK) return py::make_tuple(rc, what);
  return py::make_tuple(out5, lse, n_valid, x, y1, w, p.w_layout, tensor_or_none(dx), tensor_or_none(dw), tensor_or_none(pre),
                        chunks > 0);
}

// The gradients by recomputing the logits, of what forward saved: (dx, dw), dense, dw as it is stored.  None: not handled.
py::object backward(const at::Tensor& x, const at::Tensor& y1, const at::Tensor& w, const at::Tensor& lse, const at::Tensor& n_valid,
                    const at::Tensor& g, int64_t ignore_index, double z_reg, double scale, int64_t n_chunk, bool need_dx, bool need_dw,
                    int pack, int layout, uintptr_t stream) {
  Call c;
  lce_problem& p = c.p;
  if (!(need_dx || need_dw) || w.dim() != 2) return py::none();
  if (!describe(x, layout == LCE_W_VH ? w.t() : w, true, c) || c.w != kInPlace || p.w_layout != layout) return py::none();
  for (const at::Tensor& t : {y1, lse, n_valid, g})
    if (!plain(t) || t.device() != x.device() || !t.is_contiguous()) return py::none();
  if (y1.scalar_type() != at::kLong || y1.numel() != p.N || lse.scalar_type() != at::kFloat || lse.numel() != p.N ||
      n_valid.scalar_type() != at::kLong || g.scalar_type() != at::kFloat || g.numel() != 1)
    return py::none();
  p.ignore_index = ignore_index;
  p.logit_scale = (float)scale;
  p.z_reg = (float)z_reg;
  p.n_chunk = n_chunk;
  p.pack_rows = pack;
  size_t bytes = 0;
  if (abi.check_problem(&p) != LCE_OK || abi.workspace_bytes(&p, nullptr, &bytes) != LCE_OK) return py::none();

  at::NoGradGuard no_grad;
  at::Tensor dx, dw;
  if (need_dx) dx = rows_of(p.N, p.H, p.lddx, x.options());
  if (need_dw) dw = rows_of(w.size(0), w.size(1), p.lddw, w.options());
  Workspace ws(bytes);
  int rc;
  {
    py::gil_scoped_release release;
    rc = abi.backward(&p, x.data_ptr(), w.data_ptr(), (const int64_t*)y1.data_ptr(), (const float*)lse.data_ptr(),
                      (const int64_t*)n_valid.data_ptr(), (const float*)g.data_ptr(), ptr(dx), ptr(dw), ws.data.get(), bytes,
                      reinterpret_cast<void*>(stream));
  }
  if (rc != LCE_OK) return py::make_tuple(rc, "lce_backward", py::none());
  if (need_dx) dx = dx.contiguous();
  if (need_dw) dw = dw.contiguous();
  return py::make_tuple(tensor_or_none(dx), tensor_or_none(dw));
}

// Distillation (distillation.py): (loss, dx, dw, pre, x, w, w_layout, columns, q, y), as LinearDistillationImplementation keeps them;
// (status, name) where the C ABI refused; None: not handled.  index, logits: (..., K), contiguous.  scale: of the student's logits, the
// temperature in it.
py::object distill(const at::Tensor& x_in, const at::Tensor& At, const at::Tensor& index, const at::Tensor& logits, double temperature,
                   double scale, int64_t n_chunk, int pack, int route, bool exact, bool need_dx, bool need_dw, bool copy_w, uintptr_t stream) {
  Call c;
  lce_problem& p = c.p;
  if (!describe(x_in, At, false, c) || (c.w != kInPlace && !copy_w)) return py::none();
  for (const at::Tensor& t : {index, logits})
    if (!plain(t) || t.device() != x_in.device() || !t.is_contiguous() || t.dim() < 1) return py::none();
  const int64_t K = index.size(-1);
  const int ld = dtype_code(logits.scalar_type());
  if (index.scalar_type() != at::kLong || ld < 0 || K < 1 || index.numel() != p.N * K || logits.numel() != p.N * K) return py::none();
  p.ignore_index = -1;
  p.logit_scale = (float)scale;
  p.n_chunk = n_chunk;
  p.pack_rows = pack;
  p.route = (route == 2 ? LCE_ROUTE_ONE_PASS : route == 0 ? LCE_ROUTE_TWO_PASS : LCE_ROUTE_AUTO) | (exact ? LCE_ROUTE_EXACT_SUMS : 0) |
            (p.x_dtype == LCE_F32 ? LCE_ROUTE_KEEP_LOGITS : 0);
  const bool grads = need_dx || need_dw;
  size_t bytes = 0;
  if (abi.distill_workspace_bytes(&p, K, grads, &bytes) != LCE_OK) return py::none();

  at::NoGradGuard no_grad;
  const auto o = x_in.options();
  const at::Tensor x = c.x != kInPlace ? rows_of(p.N, p.H, p.ldx, o) : x_in.dim() == 2 ? x_in : x_in.view({p.N, p.H});
  const at::Tensor w = c.w != kInPlace ? rows_of(p.H, p.V, p.ldw, At.options()) : p.w_layout == LCE_W_VH ? At.t() : At;
  at::Tensor dx, dw, pre;
  if (need_dx) dx = rows_of(p.N, p.H, p.lddx, o);
  if (need_dw) dw = rows_of(w.size(0), w.size(1), p.lddw, At.options());
  const auto f32 = o.dtype(at::kFloat);
  const at::Tensor columns = at::empty({p.N, K}, o.dtype(at::kInt)), q = at::empty({p.N, K}, f32), y = at::empty({p.N}, o.dtype(at::kLong));
  const at::Tensor loss = at::empty({}, f32);
  if (grads && p.x_dtype == LCE_F16) pre = at::empty({1}, f32);
  const size_t lse_bytes = ((size_t)p.N * 4 + 255) & ~(size_t)255;
  Workspace ws(bytes), kept(lse_bytes + 256);  // (lse and the number of rows)
  float* const lse = (float*)kept.data.get();
  int64_t* const n_valid = (int64_t*)((char*)kept.data.get() + lse_bytes);
  void* const s = reinterpret_cast<void*>(stream);
  int rc = LCE_OK;
  const char* what = "lce_distill";
  {
    py::gil_scoped_release release;
    if (c.x != kInPlace) rc = copy_rows(c.x, x_in, p.N, p.H, x, p.ldx, s);
    if (rc == LCE_OK && c.w != kInPlace) rc = copy_rows(c.w, At, p.H, p.V, w, p.ldw, s);
    if (rc != LCE_OK) what = "lce_pad_rows";
    else if ((rc = abi.soft_targets(p.N, K, p.V, (const int64_t*)index.data_ptr(), K, logits.data_ptr(), ld, K, (float)temperature,
                                    (int32_t*)columns.data_ptr(), (float*)q.data_ptr(), (int64_t*)y.data_ptr(), s)) != LCE_OK)
      what = "lce_soft_targets";
    const float* g = nullptr;
    if (rc == LCE_OK && pre.defined()) {
      rc = abi.stand_in((const int64_t*)y.data_ptr(), p.N, -1, (float*)pre.data_ptr(), s);
      g = (const float*)pre.data_ptr();
    } else if (rc == LCE_OK) {
      rc = abi.unit_gradient(&g);
    }
    if (rc == LCE_OK)
      rc = abi.distill(&p, K, (const int32_t*)columns.data_ptr(), (const float*)q.data_ptr(), (const int64_t*)y.data_ptr(), x.data_ptr(),
                       w.data_ptr(), g, lse, (float*)loss.data_ptr(), n_valid, ptr(dx), ptr(dw), ws.data.get(), bytes, s);
  }
  if (rc != LCE_OK) return py::make_tuple(rc, what);
  return py::make_tuple(loss, tensor_or_none(dx), tensor_or_none(dw), tensor_or_none(pre), x, w, p.w_layout, columns, q, y);
}

// Rows of logits (selection.py), read in place: the last dimension dense, the others one stride apart.  A selection from one short row is
// 7 us of the device and was 14 us of Python (20 with settings by row); 6 and 5 here.
struct Rows {
  int64_t rows = 0, cols = 0, ld = 0;
  int dtype = -1;
};
bool describe_rows(const at::Tensor& logits, Rows& r) {
  if (!plain(logits) || logits.dim() < 1 || logits.size(-1) < 1 || logits.numel() == 0) return false;
  r.dtype = dtype_code(logits.scalar_type());
  r.cols = logits.size(-1);
  r.rows = logits.numel() / r.cols;
  r.ld = r.cols;
  if (!logits.is_contiguous()) {
    if (logits.dim() != 2 || (logits.stride(1) != 1 && r.cols > 1)) return false;
    r.ld = logits.stride(0);
  }
  return r.dtype >= 0;
}

// (values, index, lse) of top_logits; (status, name) where the C ABI refused; None: not handled.
py::object top_logits(const at::Tensor& logits, int64_t k, uintptr_t stream) {
  Rows r;
  if (!describe_rows(logits, r)) return py::none();
  at::NoGradGuard no_grad;
  auto shape = logits.sizes().vec();
  shape.back() = k;
  const auto o = logits.options().requires_grad(false);
  const at::Tensor values = at::empty(shape, o), index = at::empty(shape, o.dtype(at::kLong));
  shape.pop_back();
  const at::Tensor lse = at::empty(shape, o.dtype(at::kFloat));
  int rc;
  {
    py::gil_scoped_release release;
    rc = abi.top_logits(logits.data_ptr(), r.dtype, r.rows, r.cols, r.ld, k, values.data_ptr(), (int64_t*)index.data_ptr(),
                        (float*)lse.data_ptr(), reinterpret_cast<void*>(stream));
  }
  if (rc != LCE_OK) return py::make_tuple(rc, "top_logits");
  return py::make_tuple(values, index, lse);
}

// A setting of sample_logits: a number, or a tensor with one for each row.  False: neither of these as the C ABI takes it.
template <class T> bool setting(const py::handle& value, const at::Tensor& logits, const at::Tensor& u, at::ScalarType type, T* number, const T** rows) {
  if (THPVariable_Check(value.ptr())) {
    const at::Tensor& t = THPVariable_Unpack(value.ptr());
    if (!plain(t) || t.scalar_type() != type || t.device() != logits.device() || t.sizes() != u.sizes() || !t.is_contiguous()) return false;
    *rows = (const T*)t.data_ptr();
    return true;
  }
  if (PyLong_Check(value.ptr())) {
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(value.ptr(), &overflow);
    *number = (T)v;
    return overflow == 0;
  }
  if constexpr (std::is_same_v<T, float>) {
    if (!PyFloat_Check(value.ptr())) return false;
    *number = (float)PyFloat_AS_DOUBLE(value.ptr());
    return true;
  }
  return false;
}

// The tokens of sample_logits; None: not handled, or refused by the C ABI.
py::object sample_logits(const at::Tensor& logits, const at::Tensor& u, const py::object& temperature, const py::object& top_k,
                         const py::object& top_p, const py::object& min_p, uintptr_t stream) {
  Rows r;
  if (!describe_rows(logits, r)) return py::none();
  if (!plain(u) || u.scalar_type() != at::kFloat || u.device() != logits.device() || !u.is_contiguous() ||
      u.sizes() != logits.sizes().slice(0, logits.dim() - 1))
    return py::none();
  lce_sampling s = {1.f, 1.f, 0.f, 0, nullptr, nullptr, nullptr, nullptr};
  if (!setting(temperature, logits, u, at::kFloat, &s.temperature, &s.temperature_rows) ||
      !setting(top_p, logits, u, at::kFloat, &s.top_p, &s.top_p_rows) || !setting(min_p, logits, u, at::kFloat, &s.min_p, &s.min_p_rows) ||
      !setting(top_k, logits, u, at::kLong, &s.top_k, &s.top_k_rows))
    return py::none();
  at::NoGradGuard no_grad;
  const at::Tensor token = at::empty(u.sizes(), u.options().dtype(at::kLong).requires_grad(false));
  int rc;
  {
    py::gil_scoped_release release;
    rc = abi.sample(logits.data_ptr(), r.dtype, r.rows, r.cols, r.ld, (const float*)u.data_ptr(), &s, (int64_t*)token.data_ptr(),
                    reinterpret_cast<void*>(stream));
  }
  if (rc != LCE_OK) return py::none();
  return py::cast(token);
}

// Logits of given tokens (token_logits.py).  A call as the C ABI takes it, the settings that its backward needs too, and its results.
struct TokenCall {
  Call c;
  bool piece;
  int64_t ignore_index, vocab_start, vocab_size;  // of the tokens; the problem's are of the labels
  size_t bytes;
  void* stream;
  int rc = LCE_OK;
  at::Tensor logits, lse, x, w, labels;
  at::Tensor scales;  // of float32 tensors, for the backward
};

// False: no ordinary call.
bool describe_tokens(const at::Tensor& x_in, const at::Tensor& At, const at::Tensor& tokens, int64_t ignore_index, double scale, int64_t n_chunk,
                     int64_t vocab_start, int64_t vocab_size, int pack, bool copy_w, uintptr_t stream, TokenCall& t) {
  lce_problem& p = t.c.p;
  if (!describe(x_in, At, false, t.c) || (t.c.w != kInPlace && !copy_w) || !plain(tokens) || tokens.scalar_type() != at::kLong ||
      tokens.device() != x_in.device() || !tokens.is_contiguous() || tokens.sizes() != x_in.sizes().slice(0, x_in.dim() - 1))
    return false;
  t.piece = vocab_size != p.V;
  t.ignore_index = ignore_index;
  t.vocab_start = vocab_start;
  t.vocab_size = vocab_size;
  t.stream = reinterpret_cast<void*>(stream);
  p.ignore_index = t.piece ? -1 : ignore_index;
  p.logit_scale = (float)scale;
  p.n_chunk = n_chunk;
  p.pack_rows = pack;
  return abi.token_logits_workspace_bytes(&p, &t.bytes, nullptr) == LCE_OK;
}

// (the interpreter's lock is not needed)
void run_tokens(const at::Tensor& x_in, const at::Tensor& At, const at::Tensor& tokens, TokenCall& t) {
  const Call& c = t.c;
  const lce_problem& p = c.p;
  at::NoGradGuard no_grad;
  const auto o = x_in.options().requires_grad(false);
  t.x = c.x != kInPlace ? rows_of(p.N, p.H, p.ldx, o) : x_in.dim() == 2 ? x_in : x_in.view({p.N, p.H});
  t.w = c.w != kInPlace ? rows_of(p.H, p.V, p.ldw, At.options().requires_grad(false)) : p.w_layout == LCE_W_VH ? At.t() : At;
  const at::Tensor given = tokens.dim() == 1 ? tokens : tokens.view({p.N});
  t.labels = t.piece ? at::empty({p.N}, tokens.options()) : given;
  t.logits = at::empty(tokens.sizes(), o.dtype(at::kFloat));
  t.lse = at::empty(tokens.sizes(), o.dtype(at::kFloat));
  if (p.x_dtype == LCE_F32) t.scales = at::empty({LCE_PAIR_SCALES}, o);
  Workspace ws(t.bytes);
  if (c.x != kInPlace) t.rc = copy_rows(c.x, x_in, p.N, p.H, t.x, p.ldx, t.stream);
  if (t.rc == LCE_OK && c.w != kInPlace) t.rc = copy_rows(c.w, At, p.H, p.V, t.w, p.ldw, t.stream);
  if (t.rc == LCE_OK && t.piece)
    t.rc = abi.token_labels((const int64_t*)given.data_ptr(), p.N, t.ignore_index, t.vocab_start, p.V, t.vocab_size, (int64_t*)t.labels.data_ptr(),
                            t.stream);
  if (t.rc == LCE_OK)
    t.rc = abi.token_logits(&p, t.x.data_ptr(), t.w.data_ptr(), (const int64_t*)t.labels.data_ptr(), t.piece ? p.V : t.ignore_index,
                            (float*)t.logits.data_ptr(), (float*)t.lse.data_ptr(), (float*)ptr(t.scales), ws.data.get(), t.bytes, t.stream);
}

// (logits, lse, x, w, w_layout, labels, ignore_index), as _forward of token_logits.py returns them; (status, name) where the C ABI refused; None:
// not handled.
py::object token_logits(const at::Tensor& x_in, const at::Tensor& At, const at::Tensor& tokens, int64_t ignore_index, double scale, int64_t n_chunk,
                        int64_t vocab_start, int64_t vocab_size, int pack, bool copy_w, uintptr_t stream) {
  TokenCall t;
  if (!describe_tokens(x_in, At, tokens, ignore_index, scale, n_chunk, vocab_start, vocab_size, pack, copy_w, stream, t)) return py::none();
  {
    py::gil_scoped_release release;
    run_tokens(x_in, At, tokens, t);
  }
  if (t.rc != LCE_OK) return py::make_tuple(t.rc, "linear_token_logits");
  return py::make_tuple(t.logits, t.lse, t.x, t.w, t.c.p.w_layout, t.labels, t.c.p.ignore_index);
}

// The gradients, dense, dw as it is stored.  False: not handled, nothing is launched.
bool run_tokens_backward(const at::Tensor& x, const at::Tensor& w, int layout, const at::Tensor& labels, const at::Tensor& logits,
                         const at::Tensor& lse, const at::Tensor& g_logits, const at::Tensor& g_lse, int64_t ignore_index, double scale,
                         const at::Tensor& scales, int64_t n_chunk, int pack, bool need_dx, bool need_dw, void* stream, at::Tensor& dx,
                         at::Tensor& dw, int& rc) {
  Call c;
  lce_problem& p = c.p;
  if (!(need_dx || need_dw) || w.dim() != 2) return false;
  if (!describe(x, layout == LCE_W_VH ? w.t() : w, true, c) || c.w != kInPlace || p.w_layout != layout) return false;
  for (const at::Tensor& t : {logits, lse, g_logits, g_lse})
    if (!plain(t) || t.device() != x.device() || !t.is_contiguous() || t.scalar_type() != at::kFloat || t.numel() != p.N) return false;
  if (!plain(labels) || labels.scalar_type() != at::kLong || labels.device() != x.device() || !labels.is_contiguous() || labels.numel() != p.N)
    return false;
  p.ignore_index = ignore_index;
  p.logit_scale = (float)scale;
  p.n_chunk = n_chunk;
  p.pack_rows = pack;
  size_t bytes = 0;
  if (abi.token_logits_workspace_bytes(&p, nullptr, &bytes) != LCE_OK) return false;

  at::NoGradGuard no_grad;
  if (need_dx) dx = rows_of(p.N, p.H, p.lddx, x.options().requires_grad(false));
  if (need_dw) dw = rows_of(w.size(0), w.size(1), p.lddw, w.options().requires_grad(false));
  Workspace ws(bytes);
  rc = abi.token_logits_backward(&p, x.data_ptr(), w.data_ptr(), (const int64_t*)labels.data_ptr(), (const float*)logits.data_ptr(),
                                 (const float*)lse.data_ptr(), (const float*)g_logits.data_ptr(), (const float*)g_lse.data_ptr(), (const float*)ptr(scales),
                                 ptr(dx), ptr(dw),
                                 ws.data.get(), bytes, stream);
  if (rc != LCE_OK) return true;
  if (need_dx) dx = dx.contiguous();
  if (need_dw) dw = dw.contiguous();
  return true;
}

// (dx, dw); (status, name, None) where the C ABI refused; None: not handled.
py::object token_logits_backward(const at::Tensor& x, const at::Tensor& w, int layout, const at::Tensor& labels, const at::Tensor& logits,
                                 const at::Tensor& lse, const at::Tensor& g_logits, const at::Tensor& g_lse, int64_t ignore_index, double scale,
                                 int64_t n_chunk, int pack, bool need_dx, bool need_dw, uintptr_t stream) {
  at::Tensor dx, dw;
  int rc = LCE_OK;
  bool handled;
  {
    py::gil_scoped_release release;
    handled = run_tokens_backward(x, w, layout, labels, logits, lse, g_logits, g_lse, ignore_index, scale, at::Tensor(), n_chunk, pack, need_dx, need_dw,
                                  reinterpret_cast<void*>(stream), dx, dw, rc);
  }
  if (!handled) return py::none();
  if (rc != LCE_OK) return py::make_tuple(rc, "linear_token_logits", py::none());
  return py::make_tuple(tensor_or_none(dx), tensor_or_none(dw));
}

// The operator with its place in the autograd graph, whose backward does not wait for the interpreter: a forward and backward of 64 rows of
// 256 x 4096, 41 us on the GPU, in 80 us, by TokenLogitsImplementation (token_logits.py) 107.
struct TokenLogits : public torch::autograd::Function<TokenLogits> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x_in, const at::Tensor& At,
                                                const at::Tensor& tokens, TokenCall* t) {
    run_tokens(x_in, At, tokens, *t);
    TORCH_CHECK(t->rc == LCE_OK, "linear_token_logits");  // (differentiable_token_logits has the status)
    ctx->save_for_backward({t->x, t->w, t->labels, t->logits, t->lse, t->scales});
    const lce_problem& p = t->c.p;
    ctx->saved_data["layout"] = (int64_t)p.w_layout;
    ctx->saved_data["ignore_index"] = p.ignore_index;
    ctx->saved_data["scale"] = (double)p.logit_scale;
    ctx->saved_data["n_chunk"] = p.n_chunk;
    ctx->saved_data["pack"] = (int64_t)p.pack_rows;
    ctx->saved_data["shape"] = x_in.sizes().vec();
    ctx->saved_data["stream"] = (int64_t)reinterpret_cast<uintptr_t>(t->stream);  // (the engine runs the backward on the forward's)
    return {t->logits, t->lse};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const auto saved = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    const int layout = (int)d["layout"].toInt();
    // (hooks on saved tensors may bring them back with other strides)
    const auto rows = [](const at::Tensor& t) {
      if (t.stride(1) == 1 && t.stride(0) % row_multiple(t.scalar_type()) == 0 && t.stride(0) >= t.size(1) && aligned(t)) return t;
      at::NoGradGuard no_grad;
      at::Tensor copy = rows_of(t.size(0), t.size(1), padded_cols(t.size(1), t.scalar_type()), t.options().requires_grad(false));
      return copy.copy_(t);
    };
    const at::Tensor g_logits = g[0].contiguous(), g_lse = g[1].contiguous();
    at::Tensor dx, dw;
    int rc = LCE_OK;
    const bool handled = run_tokens_backward(rows(saved[0]), rows(saved[1]), layout, saved[2].contiguous(), saved[3].contiguous(), saved[4].contiguous(), g_logits, g_lse,
                                             d["ignore_index"].toInt(), d["scale"].toDouble(), saved[5], d["n_chunk"].toInt(), (int)d["pack"].toInt(),
                                             ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                             reinterpret_cast<void*>((uintptr_t)d["stream"].toInt()), dx, dw, rc);
    TORCH_CHECK(handled, "linear_token_logits: upstream gradients or saved tensors that are no dense tensors of the forward's device and sizes");
    TORCH_CHECK(rc == LCE_OK, "linear_token_logits: ", abi.strerror(rc), rc == LCE_EHIP ? ": " : "", rc == LCE_EHIP ? abi.last_hip_error() : "");
    if (dx.defined()) dx = dx.view(d["shape"].toIntVector());
    if (dw.defined() && layout == LCE_W_VH) dw = dw.t();
    torch::autograd::variable_list out = {dx, dw};
    if (at::GradMode::is_enabled()) {  // (create_graph: a second derivative is an error, not zero)
      for (at::Tensor& t : out)
        if (t.defined()) t.requires_grad_(true);
      out = (*std::make_shared<torch::autograd::DelayedError>("linear_token_logits is differentiable once", (int64_t)out.size()))(std::move(out));
    }
    return {out[0], out[1], at::Tensor(), at::Tensor()};
  }
};

// linear_token_logits: (logits, lse); (status, name, None) where the C ABI refused; None: not handled.
py::object differentiable_token_logits(const at::Tensor& x_in, const at::Tensor& At, const at::Tensor& tokens, int64_t ignore_index, double scale,
                                       int64_t n_chunk, int64_t vocab_start, int64_t vocab_size, int pack, bool copy_w, uintptr_t stream) {
  TokenCall t;
  if (!describe_tokens(x_in, At, tokens, ignore_index, scale, n_chunk, vocab_start, vocab_size, pack, copy_w, stream, t)) return py::none();
  torch::autograd::variable_list out;
  {
    py::gil_scoped_release release;
    try {
      out = TokenLogits::apply(x_in, At, tokens, &t);
    } catch (const c10::Error&) {
      if (t.rc == LCE_OK) throw;
    }
  }
  if (t.rc != LCE_OK) return py::make_tuple(t.rc, "linear_token_logits", py::none());
  return py::make_tuple(out[0], out[1]);
}

// What quantize_rows and, of the columns of a matrix, quantize_weight (quantization.py) return, the values with rows of `ldq` bytes; (status,
// name, None) where the C ABI refused; None: not handled.
py::object quantize(const at::Tensor& t, bool columns, int64_t ldq, uintptr_t stream) {
  Rows r;
  if (!describe_rows(t, r) || r.rows < 1 || (columns && t.dim() != 2)) return py::none();
  const int64_t depth = columns ? r.rows : r.cols, others = columns ? r.cols : r.rows;
  at::NoGradGuard no_grad;
  const auto o = t.options().requires_grad(false);
  auto shape = t.sizes().vec();
  if (columns) std::swap(shape[0], shape[1]);
  std::vector<int64_t> strides(shape.size());
  strides.back() = 1;
  int64_t n = ldq;
  for (int i = (int)shape.size() - 2; i >= 0; --i) {
    strides[i] = n;
    n *= shape[i];
  }
  // (whole rows of memory, of which the values are the first `depth` of each)
  const at::Tensor values = at::empty({others, ldq}, o.dtype(at::kChar)).as_strided(shape, strides);
  shape.pop_back();
  const at::Tensor scales = at::empty(shape, o.dtype(at::kFloat));
  int rc;
  {
    py::gil_scoped_release release;
    rc = columns ? abi.quantize_columns(t.data_ptr(), r.dtype, depth, others, r.ld, (int8_t*)values.data_ptr(), ldq, (float*)scales.data_ptr(),
                                        reinterpret_cast<void*>(stream))
                 : abi.quantize_rows(t.data_ptr(), r.dtype, others, depth, r.ld, (int8_t*)values.data_ptr(), ldq, (float*)scales.data_ptr(),
                                     reinterpret_cast<void*>(stream));
  }
  if (rc != LCE_OK) return py::make_tuple(rc, columns ? "quantize_weight" : "quantize_rows", py::none());
  return py::make_tuple(values, scales);
}

// quantized_logits (quantization.py); (status, name) where the C ABI refused; None: not handled.
py::object quantized_logits(const at::Tensor& x, const at::Tensor& values, const at::Tensor& scales, double scale, py::object dtype, uintptr_t stream) {
  Rows r;
  if (!describe_rows(x, r) || !plain(values) || !plain(scales) || values.scalar_type() != at::kChar || scales.scalar_type() != at::kFloat ||
      values.device() != x.device() || scales.device() != x.device() || values.dim() != 2 || values.size(0) < 1 || values.size(1) != r.cols ||
      values.stride(1) != 1 || values.stride(0) < r.cols || values.stride(0) > 2 * LCE_INT8_DEPTH || values.stride(0) % 16 != 0 ||
      !aligned(values) || scales.dim() != 1 || scales.size(0) != values.size(0) || !scales.is_contiguous())
    return py::none();
  const at::ScalarType type = dtype.is_none() ? x.scalar_type() : reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
  const int code = dtype_code(type);
  const int64_t V = values.size(0);
  size_t bytes = 0;
  if (code < 0 || abi.int8_logits_workspace_bytes(r.rows, r.cols, V, &bytes) != LCE_OK) return py::none();
  at::NoGradGuard no_grad;
  auto shape = x.sizes().vec();
  shape.back() = V;
  const at::Tensor out = at::empty(shape, x.options().dtype(type).requires_grad(false));
  Workspace ws(bytes);
  int rc;
  {
    py::gil_scoped_release release;
    rc = abi.int8_logits(x.data_ptr(), r.dtype, r.rows, r.cols, V, r.ld, (const int8_t*)values.data_ptr(), values.stride(0),
                         (const float*)scales.data_ptr(), (float)scale, out.data_ptr(), code, V, ws.data.get(), bytes,
                         reinterpret_cast<void*>(stream));
  }
  if (rc != LCE_OK) return py::make_tuple(rc, "quantized_logits");
  return py::cast(out);
}

// The norm that clip_gradients (clipping.py) returns; (status, name) where the C ABI refused; None: not handled.  grads, out: lists of the
// same length; divisor_rows: None or a tensor with the divisor.
py::object clip(const py::list& grads, const py::list& out, double max_norm, double divisor, const py::object& divisor_tensor, uintptr_t stream) {
  const size_t n = grads.size();
  if (n == 0 || out.size() != n) return py::none();
  std::vector<lce_tensor> t(n);
  at::TensorOptions options;
  c10::Device device(c10::kCPU);
  for (size_t i = 0; i < n; ++i) {
    const py::handle gh = grads[i], oh = out[i];
    if (!THPVariable_Check(gh.ptr()) || !THPVariable_Check(oh.ptr())) return py::none();
    const at::Tensor &g = THPVariable_Unpack(gh.ptr()), &o = THPVariable_Unpack(oh.ptr());
    if (!plain(g) || !plain(o) || g.sizes() != o.sizes() || g.strides() != o.strides() || !g.is_non_overlapping_and_dense()) return py::none();
    if (o.is_inference() && !c10::InferenceMode::is_enabled()) return py::none();
    if (i == 0) {
      device = g.device();
      options = g.options();
    }
    const int gd = dtype_code(g.scalar_type()), od = dtype_code(o.scalar_type());
    if (g.device() != device || o.device() != device || gd < 0 || (od != gd && od != LCE_F32)) return py::none();
    t[i] = {g.data_ptr(), o.data_ptr(), g.numel(), gd, od};
  }
  const float* by = nullptr;
  if (!divisor_tensor.is_none()) {
    const at::Tensor& d = THPVariable_Unpack(divisor_tensor.ptr());
    if (!plain(d) || d.scalar_type() != at::kFloat || d.numel() != 1 || d.device() != device) return py::none();
    by = (const float*)d.data_ptr();
  }
  size_t bytes = 0;
  if (abi.clip_workspace_bytes(t.data(), (int64_t)n, &bytes) != LCE_OK) return py::none();
  at::NoGradGuard no_grad;
  const at::Tensor norm = at::empty({}, options.dtype(at::kFloat).requires_grad(false));
  Workspace ws(bytes);
  int rc;
  {
    py::gil_scoped_release release;
    rc = abi.clip(t.data(), (int64_t)n, (float)max_norm, (float)divisor, by, (float*)norm.data_ptr(), ws.data.get(), bytes,
                  reinterpret_cast<void*>(stream));
  }
  if (rc != LCE_OK) return py::make_tuple(rc, "clip_gradients");
  for (size_t i = 0; i < n; ++i) THPVariable_Unpack(py::handle(out[i]).ptr()).unsafeGetTensorImpl()->bump_version();
  return py::cast(norm);
}

}  // namespace

PYBIND11_MODULE(_lce_host, m) {
  m.def("bind", &bind);
  m.def("forward", &forward);
  m.def("backward", &backward);
  m.def("distill", &distill);
  m.def("top_logits", &top_logits);
  m.def("sample_logits", &sample_logits);
  m.def("token_logits", &token_logits);
  m.def("differentiable_token_logits", &differentiable_token_logits);
  m.def("token_logits_backward", &token_logits_backward);
  m.def("quantize", &quantize);
  m.def("quantized_logits", &quantized_logits);
  m.def("clip", &clip);
}
