// Host side of the feed-forward operators (hot_amd/ffn.py): argument checks, result and workspace tensors, autograd nodes, and the
// launches through the C entries of libhotk.so.  In C++ because a call is a few microseconds of GPU work at the small end: with
// the same steps in Python (ctypes arguments, a Python autograd function) a norm of one token took 22 us a call and one with
// its gradients 160, against 4.7 and 55 here, of which torch's own engine takes 31.
//
// The entries' addresses come from Python's loaded library (bind), so both bindings run the same build of it; with timing on
// (_lib.timing_begin) every launch is reported to the same hook as Python's own.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/python.h>

#include <atomic>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/hotk.h"

namespace py = pybind11;
using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Refused : std::runtime_error {      // becomes hot_amd._lib.HotkError
  using std::runtime_error::runtime_error;
};
PyObject* error_type = nullptr;

template <class... A>
[[noreturn]] void refuse(const A&... parts) {
  throw Refused(c10::str(parts...));
}

// ---- the library -------------------------------------------------------------------------------------------------------
struct Entries {
  decltype(&hotk_strerror) strerror;
  decltype(&hotk_rmsnorm_supported) rmsnorm_supported;
  decltype(&hotk_rmsnorm_fwd) rmsnorm_fwd;
  decltype(&hotk_rmsnorm_quant) rmsnorm_quant;
  decltype(&hotk_quantize_rows) quantize_rows;
  decltype(&hotk_rmsnorm_partials) rmsnorm_partials;
  decltype(&hotk_rmsnorm_bwd) rmsnorm_bwd;
  decltype(&hotk_sum_partials) sum_partials;
  decltype(&hotk_linear_workspace_bytes) linear_workspace_bytes;
  decltype(&hotk_linear_act) linear_act;
  decltype(&hotk_linear_dz_partials) linear_dz_partials;
  decltype(&hotk_linear_dz) linear_dz;
  decltype(&hotk_pad_rows) pad_rows;
} L{};

template <class F>
void bind_one(F& f, const py::dict& d, const char* name) {
  f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}

void bind(const py::dict& d, py::object error) {
  bind_one(L.strerror, d, "hotk_strerror");
  bind_one(L.rmsnorm_supported, d, "hotk_rmsnorm_supported");
  bind_one(L.rmsnorm_fwd, d, "hotk_rmsnorm_fwd");
  bind_one(L.rmsnorm_quant, d, "hotk_rmsnorm_quant");
  bind_one(L.quantize_rows, d, "hotk_quantize_rows");
  bind_one(L.rmsnorm_partials, d, "hotk_rmsnorm_partials");
  bind_one(L.rmsnorm_bwd, d, "hotk_rmsnorm_bwd");
  bind_one(L.sum_partials, d, "hotk_sum_partials");
  bind_one(L.linear_workspace_bytes, d, "hotk_linear_workspace_bytes");
  bind_one(L.linear_act, d, "hotk_linear_act");
  bind_one(L.linear_dz_partials, d, "hotk_linear_dz_partials");
  bind_one(L.linear_dz, d, "hotk_linear_dz");
  bind_one(L.pad_rows, d, "hotk_pad_rows");
  error_type = error.release().ptr();      // kept for the process
}

void check(int rc, const char* what) {
  if (rc != HOTK_OK) refuse(what, " failed: ", L.strerror(rc), " (", rc, ")");
}

// the timing hook: called with (name, bytes, True) before and (name, bytes, False) after a launch while it is set
std::atomic<bool> timing{false};
PyObject* timing_hook = nullptr;           // touched under the GIL only

void set_timing(py::object hook) {
  Py_XDECREF(timing_hook);
  timing_hook = hook.is_none() ? nullptr : hook.release().ptr();
  timing = timing_hook != nullptr;
}

template <class F>
void launch(const char* name, int64_t bytes, F&& f) {
  int rc;
  if (timing.load(std::memory_order_relaxed)) {
    py::gil_scoped_acquire gil;
    py::object hook = timing_hook ? py::reinterpret_borrow<py::object>(timing_hook) : py::none();
    if (!hook.is_none()) hook(name, bytes, true);
    rc = f();
    if (!hook.is_none()) hook(name, bytes, false);
  } else {
    rc = f();
  }
  check(rc, name);
}

// ---- arguments ---------------------------------------------------------------------------------------------------------
int type_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HOTK_F32;
    case at::kBFloat16: return HOTK_BF16;
    case at::kHalf: return HOTK_F16;
    case at::kFloat8_e4m3fn: return HOTK_E4M3;
    default: return -1;
  }
}

// derivatives are of first order and in reverse: a tensor that carries a forward derivative would lose it here
void check_tangent(const Tensor& t, const char* what) {
  if (t._fw_grad(/*level=*/0).defined())
    refuse(what, " carries a forward-mode derivative: there are gradients in reverse mode only");
}

// a tensor with memory of its own: one that stands for others (under torch.func's transforms, a class with __torch_dispatch__
// such as a distributed or a fake tensor) has none, and an optional operand without memory would count as one not given
void check_plain(const Tensor& t, const char* what) {
  using c10::DispatchKey;
  if (t.key_set().has_any(c10::DispatchKeySet({DispatchKey::Python, DispatchKey::Batched, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                                  DispatchKey::Functionalize})))
    refuse(what, ": a plain tensor is expected, not one that stands for others (torch.func, vmap, __torch_dispatch__)");
  check_tangent(t, what);
}

// the values are what the memory holds
void check_memory(const Tensor& t, const char* what) {
  if (t.layout() != at::kStrided) refuse(what, ": a strided tensor is expected");
  if (t.is_neg() || t._is_zerotensor()) refuse(what, " is a view that negates (or stands for zeros without memory): call resolve_neg() or clone() first");
}

void check_input(const Tensor& x, const char* what, bool eight = false) {
  if (!x.defined()) refuse(what, ": a tensor is expected");
  check_plain(x, what);
  if (!x.is_cuda())
    refuse("hot_amd kernels run on a HIP device only; ", what, " is on ", x.device(), ". There is no CPU path: move it to the GPU.");
  const int ty = type_of(x.scalar_type());
  if (eight ? ty != HOTK_E4M3 : (ty < 0 || ty == HOTK_E4M3))
    refuse(what, ": ", eight ? "float8_e4m3fn" : "fp32, bf16 or fp16", " expected, got ", x.scalar_type());
  check_memory(x, what);
  if (x.dim() < 1 || x.size(-1) == 0) refuse(what, ": [..., width] with width >= 1 expected, got shape ", x.sizes());
}

// an operand that goes with `ref`: on its device, of this type and shape
void check_with(const Tensor& ref, const Tensor& t, const char* what, at::IntArrayRef shape, at::ScalarType type) {
  if (!t.defined()) refuse(what, ": a tensor is expected");
  check_plain(t, what);
  if (t.device() != ref.device()) refuse(what, " is on ", t.device(), ", the input on ", ref.device());
  if (t.scalar_type() != type) refuse(what, ": ", type, " expected, got ", t.scalar_type());
  check_memory(t, what);
  if (t.sizes() != shape) refuse(what, ": shape ", shape, " expected, got ", t.sizes());
}

// what the forward pass kept as memory of `n` elements in a row, as the backward pass finds it: a saved-tensor hook may have put another
// tensor in its place, so its values are taken in any layout, and anything but n values of this type beside `ref` is refused
Tensor kept_values(const Tensor& ref, const Tensor& t, const char* what, int64_t n, at::ScalarType type) {
  if (!t.defined()) refuse(what, " kept for the backward pass did not come back");
  check_with(ref, t, what, t.sizes(), type);
  if (t.numel() != n) refuse(what, " kept for the backward pass came back with ", t.numel(), " elements instead of ", n);
  return t.contiguous();
}

// [..., C] as rows in place: the tensor, elements from row to row, rows; a copy where the rows lie at no single stride
struct Rows {
  Tensor t;
  int64_t ld = 0, n = 0;
  bool zeros = false;                      // made here with zeros from a row's end to the next
  const void* p() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};

Rows rows(const Tensor& given) {
  // (a gradient may be such a view; inputs were checked)
  const Tensor x = given.is_neg() || given._is_zerotensor() ? given.clone() : given;
  const int64_t C = x.size(-1), n = x.numel() / C;
  if (n == 0) return {x, C, 0};
  if (x.stride(-1) == 1 || C == 1) {
    int64_t ld = -1, span = 1;             // span: rows that the dimensions to the right hold
    bool ok = true;
    for (int64_t k = x.dim() - 2; k >= 0 && ok; --k) {
      if (x.size(k) != 1) {
        if (ld < 0) ld = x.stride(k);      // the innermost dimension of more than one
        ok = x.stride(k) == ld * span;
      }
      span *= x.size(k);
    }
    if (ld < 0) ld = C;
    if (ok && ld >= C) return {x, ld, n};
  }
  return {x.contiguous(), C, n};
}
Rows rows(const optional<Tensor>& x) { return x ? rows(*x) : Rows{}; }

void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream(); }
Tensor like(const Tensor& x, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, x.options().dtype(type)); }
Tensor like(const Tensor& x) { return like(x, x.sizes(), x.scalar_type()); }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const optional<Tensor>& t) { return t && wants_grad(*t); }
template <class... T>
void refuse_grad(const char* what, const T&... t) {
  if (at::GradMode::is_enabled() && (wants_grad(t) || ...))
    refuse(what, " has no gradient: call it under torch.no_grad() or on detached tensors");
}
void first_order(const char* what, const variable_list& gradients) {
  if (at::GradMode::is_enabled()) refuse(what, " has gradients of first order only (create_graph=True asks for more)");
  for (const Tensor& g : gradients)
    if (g.defined()) check_plain(g, "a gradient");
}

// ---- norm --------------------------------------------------------------------------------------------------------------
void check_norm(const Tensor& x, const Tensor& w, const optional<Tensor>& r, const optional<Tensor>& kind, int64_t keep, double eps) {
  check_input(x, "x");
  const int64_t D = x.size(-1);
  check_with(x, w, "weight", {D}, x.scalar_type());
  if (r) check_with(x, *r, "residual", x.sizes(), x.scalar_type());
  if (L.rmsnorm_supported(D, type_of(x.scalar_type())) != 1) refuse("rows of up to 32768 elements are normalised, got ", D);
  if (keep < 0 || keep > 0xffffffffll) refuse("keep: a bit set over kinds expected, got ", keep);
  if (!(eps >= 0.)) refuse("eps: a number >= 0 expected, got ", eps);
  if (kind && kind->defined()) check_plain(*kind, "kind");
  if (kind && (!kind->defined() || kind->scalar_type() != at::kByte || kind->numel() != x.numel() / D || kind->device() != x.device()))
    refuse("kind: uint8, one per row (", x.numel() / D, "), on ", x.device(), " expected");
}
Tensor kind_of(const optional<Tensor>& kind) { return kind ? kind->contiguous() : Tensor(); }
const uint8_t* kind_ptr(const Tensor& k) { return k.defined() ? k.const_data_ptr<uint8_t>() : nullptr; }

// y (and h), and what the backward pass needs
struct Normed {
  Tensor y, h, rstd, w, kind;
};
Normed norm_forward(const Tensor& x, const Tensor& weight, const optional<Tensor>& r, const optional<Tensor>& kind, int64_t keep,
                    double eps, bool grad) {
  const c10::DeviceGuard guard(x.device());
  const int64_t D = x.size(-1);
  const Rows xs = rows(x), rs = rows(r);
  Normed o;
  o.w = weight.contiguous();
  o.kind = kind_of(kind);
  o.y = like(x);
  if (r) o.h = like(x);
  if (grad) o.rstd = like(x, {xs.n}, at::kFloat);
  if (xs.n)
    launch("hotk_rmsnorm_fwd", (r ? 4 : 2) * x.numel() * x.element_size(), [&] {
      return L.rmsnorm_fwd(xs.p(), xs.ld, rs.p(), rs.ld, o.w.const_data_ptr(), kind_ptr(o.kind), (unsigned)keep, (float)eps, o.y.data_ptr(),
                           out(o.h), (float*)out(o.rstd), xs.n, D, type_of(x.scalar_type()), stream_of(x));
    });
  return o;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& r,
                               const optional<Tensor>& kind, int64_t keep, double eps) {
    ctx->set_materialize_grads(false);
    Normed o = norm_forward(x, weight, r, kind, keep, eps, true);
    ctx->save_for_backward({r ? o.h : x, o.rstd, o.w, o.kind});
    ctx->saved_data["keep"] = keep;
    ctx->saved_data["wants"] = (int64_t)(wants_grad(x) | wants_grad(weight) << 1 | wants_grad(r) << 2 | (r ? 1 : 0) << 3 | (kind ? 1 : 0) << 4);
    if (r) return {o.y, o.h};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("rms_norm", g);
    const auto saved = ctx->get_saved_variables();
    const int64_t wants = ctx->saved_data["wants"].toInt(), keep = ctx->saved_data["keep"].toInt();
    const bool has_r = wants & 8;
    Tensor dy = g[0], dh = has_r ? g[1] : Tensor(), dx, dw;
    if (dy.defined() || dh.defined()) {
      const Tensor& ref = dy.defined() ? dy : dh;      // of the rows' device, type and shape
      const c10::DeviceGuard guard(ref.device());
      const auto type = ref.scalar_type();
      const int ty = type_of(type);
      const int64_t D = ref.size(-1), n = ref.numel() / D;
      const Tensor& h = saved[0];
      check_with(ref, h, "the stream", ref.sizes(), type);
      const Tensor rstd = kept_values(ref, saved[1], "a norm's statistics", n, at::kFloat), w = kept_values(ref, saved[2], "weight", D, type);
      const Tensor kind = wants & 16 ? kept_values(ref, saved[3], "kind", n, at::kByte) : Tensor();
      if (!dy.defined()) dy = at::zeros_like(h);
      const Rows hs = rows(h), gs = rows(dy), ss = dh.defined() ? rows(dh) : Rows{};
      void* st = stream_of(h);
      int64_t parts = 0;
      if (wants & 2) {
        check(L.rmsnorm_partials(hs.n, D, ty, &parts), "hotk_rmsnorm_partials");
        dw = like(h, {D}, type);
      }
      dx = like(h);
      const Tensor part = parts ? like(h, {parts, D}, at::kFloat) : Tensor();
      launch("hotk_rmsnorm_bwd", (dh.defined() ? 4 : 3) * h.numel() * h.element_size(), [&] {
        return L.rmsnorm_bwd(gs.p(), gs.ld, ss.p(), ss.ld, hs.p(), hs.ld, rstd.const_data_ptr<float>(), w.const_data_ptr(), kind_ptr(kind),
                             (unsigned)keep, dx.data_ptr(), (float*)out(part), parts ? nullptr : out(dw), hs.n, D, ty, st);
      });
      if (parts) launch("hotk_sum_partials", 4 * parts * D, [&] { return L.sum_partials(part.const_data_ptr<float>(), parts, D, dw.data_ptr(), ty, st); });
    }
    return {wants & 1 ? dx : Tensor(), dw, wants & 4 ? dx : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

py::object rms_norm(const Tensor& x, const Tensor& weight, const optional<Tensor>& r, double eps, const optional<Tensor>& kind, int64_t keep) {
  check_norm(x, weight, r, kind, keep, eps);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(r))) {
    const variable_list o = RmsNorm::apply(x, weight, r, kind, keep, eps);
    return r ? py::object(py::make_tuple(o[0], o[1])) : py::cast(o[0]);
  }
  const Normed o = norm_forward(x, weight, r, kind, keep, eps, false);
  return r ? py::object(py::make_tuple(o.y, o.h)) : py::cast(o.y);
}

py::tuple rms_norm_quantized(const Tensor& x, const Tensor& weight, const optional<Tensor>& r, double eps, const optional<Tensor>& kind,
                             int64_t keep) {
  check_norm(x, weight, r, kind, keep, eps);
  refuse_grad("rms_norm_quantized", x, weight, r);
  const c10::DeviceGuard guard(x.device());
  const int64_t D = x.size(-1);
  const Rows xs = rows(x), rs = rows(r);
  const Tensor w = weight.contiguous(), k = kind_of(kind), q = like(x, x.sizes(), at::kFloat8_e4m3fn);
  const Tensor scale = like(x, x.sizes().slice(0, x.dim() - 1), at::kFloat), h = r ? like(x) : Tensor();
  if (xs.n)
    launch("hotk_rmsnorm_quant", x.numel() * (1 + (r ? 3 : 1) * x.element_size()), [&] {
      return L.rmsnorm_quant(xs.p(), xs.ld, rs.p(), rs.ld, w.const_data_ptr(), kind_ptr(k), (unsigned)keep, (float)eps, (uint8_t*)q.data_ptr(),
                             scale.data_ptr<float>(), out(h), xs.n, D, type_of(x.scalar_type()), stream_of(x));
    });
  return r ? py::make_tuple(q, scale, h) : py::make_tuple(q, scale);
}

py::tuple quantize_rows(const Tensor& x) {
  check_input(x, "x");
  refuse_grad("quantize_rows", x);
  const int64_t D = x.size(-1);
  const int ty = type_of(x.scalar_type());
  if (L.rmsnorm_supported(D, ty) != 1) refuse("rows of up to 32768 elements are quantized, got ", D);
  const c10::DeviceGuard guard(x.device());
  const Rows xs = rows(x);
  const Tensor q = like(x, x.sizes(), at::kFloat8_e4m3fn), scale = like(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  if (xs.n)
    launch("hotk_quantize_rows", x.numel() * (1 + x.element_size()), [&] {
      return L.quantize_rows(xs.p(), xs.ld, (uint8_t*)q.data_ptr(), scale.data_ptr<float>(), xs.n, D, ty, stream_of(x));
    });
  return py::make_tuple(q, scale);
}

// ---- product -----------------------------------------------------------------------------------------------------------
int64_t up(int64_t n, int64_t size) {      // n elements of `size` bytes in whole 16-byte pieces
  const int64_t m = 16 / size;
  return (n + m - 1) / m * m;
}
bool whole(const Rows& x, int64_t C) {     // rows as the tiles read them: whole, aligned 16-byte pieces, zeros behind the row
  const int64_t e = x.t.element_size();
  return (C * e % 16 == 0 || x.zeros) && x.ld * e % 16 == 0 && (uintptr_t)x.p() % 16 == 0;
}
Rows padded(const Rows& in, int64_t C) {   // itself where it is whole, else a copy with zeros behind each row
  if (in.n == 0 || whole(in, C)) return in;
  const int64_t e = in.t.element_size(), ld = up(C, e);
  const Tensor o = like(in.t, {in.n, ld}, in.t.scalar_type());
  launch("hotk_pad_rows", 2 * in.n * C * e, [&] { return L.pad_rows(in.p(), in.ld * e, o.data_ptr(), ld * e, in.n, C * e, stream_of(in.t)); });
  return {o, ld, in.n, true};
}

// operands of a product: its tiles reach rows by 32-bit offsets, at strides of up to 8 MiB; short rows further apart are copied
constexpr int64_t MAX_ROW_BYTES = 1 << 23;
Rows operand(const Tensor& t) {
  const Rows r = rows(t);
  const int64_t e = t.element_size(), C = t.size(-1);
  if (r.ld * e <= MAX_ROW_BYTES || C * e > MAX_ROW_BYTES) return r;
  return {r.t.clone(at::MemoryFormat::Contiguous), C, r.n};
}

struct Extras {
  Tensor bias, save, x_scale, w_scale;
  Rows res;
  const void* x_lo = nullptr;
  int act = HOTK_ACT_NONE, flags = 0;
};
// epilogue(x w^T) [M, N] as a new tensor of this shape (no view: the caller may go on in place), copies of operands
// that it had to make in `made`
Tensor product(const Rows& x, const Rows& w, int64_t M, int64_t N, int64_t K, at::IntArrayRef shape, at::ScalarType type, const Extras& e,
               Rows* made = nullptr) {
  const Tensor y = like(x.t, shape, type);
  if (M == 0) return y;
  const int ty = type_of(x.t.scalar_type());
  hotk_linear_args a{};
  a.M = M; a.N = N; a.K = K;
  a.x = x.p(); a.ld_x = x.ld;
  a.w = w.p(); a.ld_w = w.ld;
  a.bias = out(e.bias);
  a.res = e.res.p(); a.ld_res = e.res.ld;
  a.y = y.data_ptr(); a.ld_y = N;
  a.save = out(e.save);
  a.x_scale = (const float*)out(e.x_scale); a.w_scale = (const float*)out(e.w_scale);
  a.type = ty; a.out_type = type_of(type); a.act = e.act; a.flags = e.flags; a.x_lo = e.x_lo;
  if (x.zeros && (w.zeros || (a.flags & HOTK_LINEAR_W_DOWN))) a.flags |= HOTK_LINEAR_PADDED;
  size_t need = 0;
  int rc = L.linear_workspace_bytes(&a, &need);
  Rows copies[2];
  if (rc == HOTK_EUNSUPPORTED && !(a.flags & HOTK_LINEAR_X_DOWN)) {      // not in whole pieces: copies that are
    copies[0] = padded(x, K);
    copies[1] = padded(w, a.flags & HOTK_LINEAR_W_DOWN ? N : K);
    a.x = copies[0].p(); a.ld_x = copies[0].ld;
    a.w = copies[1].p(); a.ld_w = copies[1].ld;
    a.flags |= HOTK_LINEAR_PADDED;       // (a row that needed no copy ends with a piece)
    rc = L.linear_workspace_bytes(&a, &need);
    if (made) {
      made[0] = copies[0];
      made[1] = copies[1];
    }
  }
  check(rc, "hotk_linear_act");
  const Tensor ws = need ? like(x.t, {(int64_t)need}, at::kByte) : Tensor();
  launch("hotk_linear_act", (M + N) * K * x.t.element_size() + M * N * y.element_size() * (1 + e.res.t.defined()),
         [&] { return L.linear_act(&a, out(ws), need, stream_of(x.t)); });
  return y;
}

int act_code(const std::string& act) {
  static const char* const names[] = {"none", "relu", "leakyrelu", "gelu", "tanh", "silu"};
  for (int i = 0; i < 6; ++i)
    if (act == names[i]) return i;
  refuse("act: one of none, relu, leakyrelu, gelu, tanh, silu expected, got ", act);
}

std::vector<int64_t> result_shape(const Tensor& x, int64_t N) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = N;
  return s;
}

void check_linear(const Tensor& x, const Tensor& w, const optional<Tensor>& b, const optional<Tensor>& r, at::ScalarType type) {
  if (!w.defined() || w.dim() != 2 || w.size(0) == 0) refuse("weight: [N, K] with N >= 1 expected");
  const int64_t N = w.size(0), K = w.size(1);
  if (x.size(-1) != K) refuse("x has rows of ", x.size(-1), ", weight of ", K);
  check_with(x, w, "weight", {N, K}, x.scalar_type());
  if (b) check_with(x, *b, "bias", {N}, type);
  if (r) check_with(x, *r, "residual", result_shape(x, N), type);
}

// what the backward pass reads: the slopes, and the operands as rows (copies where the product made some)
struct Kept {
  Tensor save;
  Rows x, w;
};
Tensor linear_forward(const Tensor& x, const Tensor& weight, const optional<Tensor>& b, const optional<Tensor>& r, int act, bool grad,
                      Kept* kept) {
  const c10::DeviceGuard guard(x.device());
  const int64_t K = x.size(-1), N = weight.size(0);
  const Rows xs = operand(x), ws = operand(weight);
  Extras e;
  e.act = act;
  if (b) e.bias = b->contiguous();
  e.res = rows(r);
  if (grad && act) kept->save = e.save = like(x, {xs.n, N}, x.scalar_type() == at::kFloat ? at::kFloat : at::kShort);
  Rows made[2] = {xs, ws};
  const Tensor y = product(xs, ws, xs.n, N, K, result_shape(x, N), x.scalar_type(), e, made);
  if (kept) {
    kept->x = made[0];
    kept->w = made[1];
  }
  return y;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& b, const optional<Tensor>& r,
                        int64_t act, int64_t dz_parts) {
    ctx->set_materialize_grads(false);
    Kept kept;
    const bool inner = wants_grad(x) || wants_grad(weight) || wants_grad(b);
    if ((wants_grad(x) || wants_grad(weight)) && up(weight.size(0), x.element_size()) * x.element_size() > MAX_ROW_BYTES)
      refuse("gradients of rows of up to 8 MiB: the result's rows have ", weight.size(0), " elements");      // (now, not in the backward pass)
    const Tensor y = linear_forward(x, weight, b, r, (int)act, inner, &kept);
    // what a gradient needs: x for the weight's, the weight for x's; the input itself where it was read in place (so that a later
    // change of it is noticed), else the copy
    const bool own_x = !kept.x.t.is_same(x) && kept.x.n, own_w = !kept.w.t.is_same(weight);
    ctx->save_for_backward({!wants_grad(weight) ? Tensor() : own_x ? kept.x.t : x, !wants_grad(x) ? Tensor() : own_w ? kept.w.t : weight, kept.save});
    ctx->saved_data["act"] = act;
    ctx->saved_data["dz_parts"] = dz_parts;
    ctx->saved_data["shape"] = std::vector<int64_t>(x.sizes().begin(), x.sizes().end());
    ctx->saved_data["ld"] = std::vector<int64_t>{own_x ? kept.x.ld : 0, own_w ? kept.w.ld : 0};
    ctx->saved_data["wants"] = (int64_t)(wants_grad(x) | wants_grad(weight) << 1 | wants_grad(b) << 2 | wants_grad(r) << 3);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("linear_act", g);
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = g[0];
    const int act = (int)ctx->saved_data["act"].toInt();
    const int64_t wants = ctx->saved_data["wants"].toInt();
    const auto shape = ctx->saved_data["shape"].toIntVector(), ld = ctx->saved_data["ld"].toIntVector();
    Tensor dx, dw, db;
    if (dy.defined() && (wants & 7)) {
      const c10::DeviceGuard guard(dy.device());
      const auto type = dy.scalar_type();
      const int64_t K = shape.back(), N = dy.size(-1), M = dy.numel() / N;
      // an operand: itself in any layout, or a copy of rows `ld` apart
      const auto kept = [&](int i, const char* what, at::IntArrayRef own, int64_t n) {
        if (ld[i]) return Rows{kept_values(dy, saved[i], what, n * ld[i], type), ld[i], n, true};
        check_with(dy, saved[i], what, own, type);
        return operand(saved[i]);
      };
      const Tensor save = act != HOTK_ACT_NONE ? kept_values(dy, saved[2], "slopes", M * N, type == at::kFloat ? at::kFloat : at::kShort) : Tensor();
      if (M == 0) {
        if (wants & 1) dx = at::zeros(shape, dy.options());
        if (wants & 2) dw = at::zeros({N, K}, dy.options());
        if (wants & 4) db = at::zeros({N}, dy.options());
      } else {
        const Rows gs = operand(dy);
        const int ty = type_of(type);
        // one pass over dy: dz where it is not dy itself, and its column sums
        Rows dz = gs;
        const bool itself = act == HOTK_ACT_NONE && whole(gs, N);
        // dz is rounded to the type for the products, which adds as much error as the result's own rounding; as two numbers of the
        // type it leaves the result's alone, for twice the matrix work.  The caller says which, or (0) its size: two up to 2^25
        // multiplications, where an eager call hides the second part behind its launches (1 to 5 us of the two products' 10 to 20,
        // beside 50 that the host takes; a replayed graph pays them in full), and at 2^28 it would be 7 of 14
        const int64_t parts = ctx->saved_data["dz_parts"].toInt();
        const bool two_parts = act != HOTK_ACT_NONE && type != at::kFloat && (parts ? parts == 2 : (double)M * N * K <= 33554432.);
        if ((wants & 3) && !itself) {
          const int64_t ld = up(N, dy.element_size());
          dz = {like(dy, {two_parts ? 2 * M : M, ld}, type), ld, M, true};
        }
        Tensor part;
        if (wants & 4) {
          int64_t n = 0;
          check(L.linear_dz_partials(M, &n), "hotk_linear_dz_partials");
          db = like(dy, {N}, type);
          if (n > 1) part = like(dy, {n, N}, at::kFloat);
        }
        const bool write = (wants & 3) && !itself;
        void* lo = write && two_parts ? (char*)dz.t.data_ptr() + M * dz.ld * dy.element_size() : nullptr;
        if (write || db.defined())
          launch("hotk_linear_dz", M * N * dy.element_size() * (1 + write + (act != HOTK_ACT_NONE)), [&] {
            return L.linear_dz(gs.p(), gs.ld, out(save), act, write ? dz.t.data_ptr() : nullptr, lo, dz.ld, (float*)out(part), part.defined() ? nullptr : out(db),
                               M, N, ty, stream_of(dy));
          });
        if (part.defined())
          launch("hotk_sum_partials", 4 * part.numel(), [&] {
            return L.sum_partials(part.const_data_ptr<float>(), part.size(0), N, db.data_ptr(), ty, stream_of(dy));
          });
        Extras e;
        e.x_lo = lo;
        if (wants & 1) {
          e.flags = HOTK_LINEAR_W_DOWN;
          dx = product(dz, padded(kept(1, "weight", {N, K}, N), K), M, K, N, shape, type, e);
        }
        if (wants & 2) {
          e.flags = HOTK_LINEAR_X_DOWN | HOTK_LINEAR_W_DOWN;
          dw = product(dz, padded(kept(0, "x", shape, M), K), N, K, M, {N, K}, type, e);
        }
      }
    }
    return {dx, dw, db, wants & 8 ? dy : Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear_act(const Tensor& x, const Tensor& weight, const optional<Tensor>& b, const std::string& act, const optional<Tensor>& r,
                  const optional<int64_t>& dz_parts) {
  check_input(x, "x");
  if (dz_parts && *dz_parts != 1 && *dz_parts != 2) refuse("dz_parts: 1, 2 or None expected, got ", *dz_parts);
  const int code = act_code(act);
  check_linear(x, weight, b, r, x.scalar_type());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(b) || wants_grad(r)))
    return LinearAct::apply(x, weight, b, r, (int64_t)code, dz_parts.value_or(0));
  return linear_forward(x, weight, b, r, code, false, nullptr);
}

Tensor linear_act_quantized(const Tensor& xq, const Tensor& x_scale, const Tensor& wq, const Tensor& w_scale, const optional<Tensor>& b,
                            const std::string& act, const optional<Tensor>& r, py::object out_dtype) {
  check_input(xq, "xq", true);
  if (!THPDtype_Check(out_dtype.ptr())) refuse("out_dtype: fp32, bf16 or fp16 expected");
  const auto type = reinterpret_cast<THPDtype*>(out_dtype.ptr())->scalar_type;
  if (type_of(type) < 0 || type_of(type) == HOTK_E4M3) refuse("out_dtype: fp32, bf16 or fp16 expected, got ", type);
  const int code = act_code(act);
  check_linear(xq, wq, b, r, type);
  check_with(xq, x_scale, "x_scale", xq.sizes().slice(0, xq.dim() - 1), at::kFloat);
  check_with(xq, w_scale, "w_scale", {wq.size(0)}, at::kFloat);
  refuse_grad("linear_act_quantized", b, r, x_scale, w_scale);
  const c10::DeviceGuard guard(xq.device());
  const int64_t K = xq.size(-1);
  Extras e;
  e.act = code;
  if (b) e.bias = b->contiguous();
  e.res = rows(r);
  e.x_scale = x_scale.contiguous();
  e.w_scale = w_scale.contiguous();
  return product(operand(xq), operand(wq), xq.numel() / K, wq.size(0), K, result_shape(xq, wq.size(0)), type, e);
}

}  // namespace

PYBIND11_MODULE(_ffn, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Refused& e) {
      PyErr_SetString(error_type ? error_type : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("set_timing", &set_timing);
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_quantized", &rms_norm_quantized);
  m.def("quantize_rows", &quantize_rows);
  m.def("linear_act", &linear_act);
  m.def("linear_act_quantized", &linear_act_quantized);
}
