// Native binding of the operators that are called token by token: the 8-bit
// linears and the expert routing.  Argument checks, allocation and the call into
// the C ABI in one step, and the routing's autograd nodes; a call costs a few
// microseconds of host time where the same in Python costs 12 to 20 (and a
// gradient step some 50 instead of 125), which is what a decoding step's small
// launches wait for.
//
// The C ABI's functions come in by address (`bind`), from the library that the
// Python side loaded, so that both bindings share one copy of it.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>

#include "g2ptq_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxK = 131071;  // |a b| <= 128 * 128: longer sums could leave 32 bits
constexpr int64_t kMaxExperts = 1024;

// ---------------------------------------------------------------------------
// the C ABI
// ---------------------------------------------------------------------------

#define G2Q_FUNCTIONS(X)                                                                     \
  X(g2q_quantize_tokens) X(g2q_int8_matmul) X(g2q_int8_matmul_workspace_bytes)               \
  X(g2q_int8_matmul_grouped) X(g2q_int8_linear) X(g2q_int8_linear_workspace_bytes)           \
  X(g2q_route) X(g2q_route_workspace_bytes) X(g2q_dispatch_rows) X(g2q_combine_rows)         \
  X(g2q_combine_rows_backward) X(g2q_status_string)

struct Api {
#define X(name) decltype(&::name) name = nullptr;
  G2Q_FUNCTIONS(X)
#undef X
} api;

// Never freed: they outlive the interpreter that would have to be asked.
py::object* g_error;        // (name, status) -> exception
py::object* g_status_word;  // device index -> address, 0 for none

void bind(const py::dict& addresses, py::object error, py::object status_word) {
#define X(name) \
  api.name = reinterpret_cast<decltype(api.name)>(addresses[#name].cast<uintptr_t>());
  G2Q_FUNCTIONS(X)
#undef X
  g_error = new py::object(std::move(error));
  g_status_word = new py::object(std::move(status_word));
}

void run(const char* name, int status) {
  if (status >= 0) return;
  // (a backward runs without the interpreter's lock: a plain error there)
  TORCH_CHECK(PyGILState_Check(), name, " failed: ", api.g2q_status_string(status), " (status ",
              status, ")");
  py::object e = (*g_error)(name, status);
  PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(e.ptr())), e.ptr());
  throw py::error_already_set();
}
#define G2Q_RUN(name, ...) run(#name, api.name(__VA_ARGS__))

// The device's status word for tensor-core timeouts.
int* status_word(int dev) {
  return reinterpret_cast<int*>((*g_status_word)(dev).cast<uintptr_t>());
}

// ---------------------------------------------------------------------------
// checks
// ---------------------------------------------------------------------------

// The CUDA device of the first tensor, which the others share; made current.
struct On {
  int dev;
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t, std::initializer_list<const Tensor*> rest)
      : dev(check(t, rest)), guard(dev), stream(c10::cuda::getCurrentCUDAStream(dev).stream()) {}

  static int check(const Tensor& t, std::initializer_list<const Tensor*> rest) {
    auto one = [](const Tensor& u) {
      TORCH_CHECK(u.is_cuda(), "g2ptq_b200 ops require CUDA tensors (no CPU fallback)");
    };
    one(t);
    for (const Tensor* u : rest) {
      if (!u || !u->defined()) continue;
      one(*u);
      TORCH_CHECK_VALUE(u->get_device() == t.get_device(),
                        "g2ptq_b200 ops require every tensor on the same device");
    }
    return t.get_device();
  }
};

int dtype_code(at::ScalarType t) {
  if (t == at::kBFloat16) return G2Q_DTYPE_BF16;
  if (t == at::kFloat) return G2Q_DTYPE_F32;
  TORCH_CHECK_TYPE(t == at::kHalf, "unsupported dtype ", t);
  return G2Q_DTYPE_F16;
}

struct Matrix {
  int64_t rows, cols, ld;
};

// 2-D with unit column stride and rows that do not overlap.
Matrix matrix(const char* name, const Tensor& t) {
  TORCH_CHECK_VALUE(t.dim() == 2, name, " must be 2-D, got shape ", t.sizes());
  const int64_t r = t.size(0), c = t.size(1);
  TORCH_CHECK_VALUE(c <= 1 || t.stride(1) == 1, name, " needs unit column stride");
  if (r <= 1) return {r, c, c > 1 ? c : 1};
  TORCH_CHECK_VALUE(t.stride(0) >= c, name, " has overlapping rows");
  return {r, c, t.stride(0)};
}

void vector(const char* name, const Tensor& t, int64_t n, at::ScalarType type) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.dim() == 1 && t.size(0) == n, name, " must be ",
                    type, " of shape (", n, ",), got ", t.scalar_type(), " of shape ", t.sizes());
  TORCH_CHECK_VALUE(n <= 1 || t.stride(0) == 1, name, " must be contiguous");
}

const Tensor* given(const optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }
const float* fdata(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }
const float* fdata(const optional<Tensor>& t) { return t.has_value() ? fdata(*t) : nullptr; }
const int8_t* bdata(const Tensor& t) { return static_cast<const int8_t*>(t.const_data_ptr()); }
const int32_t* idata(const Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

// Derivatives that an operator does not have are refused, not dropped without a
// word: a forward-mode tangent, and where nothing is recorded any gradient.
void no_tangent(const char* what, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), what,
                " has no forward-mode derivative");
}

void no_gradient(const char* what, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t || !t->defined() || !at::GradMode::is_enabled() || !t->requires_grad(), what,
                " records no gradient: detach its inputs or call it under torch.no_grad()");
  no_tangent(what, inputs);
}

struct Bytes {  // scratch of a call, from the caching allocator
  Tensor t;
  size_t n;
  Bytes(size_t n, const Tensor& like) : n(n) {
    if (n) t = at::empty({(int64_t)n}, like.options().dtype(at::kByte));
  }
  void* get() const { return n ? t.data_ptr() : nullptr; }
};

// ---------------------------------------------------------------------------
// 8-bit linears
// ---------------------------------------------------------------------------

struct Weight {
  int64_t N, ldb, E, gs;
};

void columns(int64_t K, int64_t have, int64_t N) {
  TORCH_CHECK_VALUE(have == K, "the tokens have ", K, " columns and the weight ", have);
  TORCH_CHECK_VALUE(K > 0 && K <= kMaxK && N > 0, "needs 1 to ", kMaxK,
                    " columns and at least one channel");
}

Weight weight(const Tensor& b, const Tensor& scale, int64_t K) {
  TORCH_CHECK_TYPE(b.scalar_type() == at::kChar, "the weight must be int8 codes, got ",
                   b.scalar_type());
  const Matrix m = matrix("the weight", b);
  columns(K, m.cols, m.rows);
  vector("its scale", scale, m.rows, at::kFloat);
  return {m.rows, m.ld, 0, 0};
}

Weight expert_weight(const Tensor& b, const Tensor& scale, const Tensor& offsets, int64_t K) {
  TORCH_CHECK_TYPE(b.scalar_type() == at::kChar, "the weight must be int8 codes, got ",
                   b.scalar_type());
  TORCH_CHECK_VALUE(b.dim() == 3, "the weight must be [experts, channels, columns], got shape ",
                    b.sizes());
  const int64_t E = b.size(0), N = b.size(1);
  columns(K, b.size(2), N);
  TORCH_CHECK_VALUE(E > 0 && E <= kMaxExperts, "needs 1 to ", kMaxExperts, " experts, got ", E);
  const int64_t ldb = N > 1 ? b.stride(1) : K;
  TORCH_CHECK_VALUE((K == 1 || b.stride(2) == 1) && ldb >= K && (E == 1 || b.stride(0) >= N * ldb),
                    "the weight needs unit column stride and experts and rows that do not overlap");
  TORCH_CHECK_VALUE(scale.scalar_type() == at::kFloat && scale.dim() == 2 && scale.size(0) == E &&
                        scale.size(1) == N && scale.is_contiguous(),
                    "its scale must be contiguous fp32 of shape (", E, ", ", N, ")");
  vector("offsets", offsets, E + 1, at::kInt);
  return {N, ldb, E, E > 1 ? b.stride(0) : N * ldb};
}

Matrix codes_of(const Tensor& a, const Tensor& scale) {
  TORCH_CHECK_TYPE(a.scalar_type() == at::kChar, "the tokens must be int8 codes, got ",
                   a.scalar_type());
  const Matrix m = matrix("the tokens", a);
  vector("their scale", scale, m.rows, at::kFloat);
  return m;
}

std::tuple<Tensor, Tensor> quantize_tokens(const Tensor& x) {
  On on(x, {});
  const Matrix m = matrix("x", x);
  TORCH_CHECK_VALUE(m.cols > 0, "quantize_tokens needs at least one column");
  const int dt = dtype_code(x.scalar_type());
  const int64_t ldq = (m.cols + 15) / 16 * 16;
  Tensor codes = at::empty({m.rows, ldq}, x.options().dtype(at::kChar)).narrow(1, 0, m.cols);
  Tensor scale = at::empty({m.rows}, x.options().dtype(at::kFloat));
  G2Q_RUN(g2q_quantize_tokens, static_cast<int8_t*>(codes.data_ptr()), ldq,
          static_cast<float*>(scale.data_ptr()), x.const_data_ptr(), dt, m.ld, m.rows, m.cols,
          on.stream);
  return {codes, scale};
}

Tensor int8_matmul(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale,
                   const optional<Tensor>& bias, const py::object& out_dtype) {
  no_gradient("int8_matmul", {&a_scale, &b_scale, given(bias)});
  On on(a, {&a_scale, &b, &b_scale, given(bias)});
  const Matrix m = codes_of(a, a_scale);
  const Weight w = weight(b, b_scale, m.cols);
  if (bias) vector("bias", *bias, w.N, at::kFloat);
  const at::ScalarType type = torch::python::detail::py_object_to_dtype(out_dtype);
  const int dt = dtype_code(type);
  Tensor out = at::empty({m.rows, w.N}, a.options().dtype(type));
  Bytes ws(api.g2q_int8_matmul_workspace_bytes(m.rows, w.N, m.cols), a);
  G2Q_RUN(g2q_int8_matmul, out.data_ptr(), dt, w.N, bdata(a), m.ld, fdata(a_scale), bdata(b), w.ldb,
          fdata(b_scale), fdata(bias), m.rows, w.N, m.cols, ws.get(), ws.n, status_word(on.dev),
          on.stream);
  return out;
}

Tensor int8_matmul_grouped(const Tensor& a, const Tensor& a_scale, const Tensor& b,
                           const Tensor& b_scale, const Tensor& offsets,
                           const py::object& out_dtype) {
  no_gradient("int8_matmul_grouped", {&a_scale, &b_scale});
  On on(a, {&a_scale, &b, &b_scale, &offsets});
  const Matrix m = codes_of(a, a_scale);
  const Weight w = expert_weight(b, b_scale, offsets, m.cols);
  const at::ScalarType type = torch::python::detail::py_object_to_dtype(out_dtype);
  const int dt = dtype_code(type);
  Tensor out = at::empty({m.rows, w.N}, a.options().dtype(type));
  G2Q_RUN(g2q_int8_matmul_grouped, out.data_ptr(), dt, w.N, bdata(a), m.ld, fdata(a_scale),
          bdata(b), w.ldb, w.gs, fdata(b_scale), idata(offsets), w.E, m.rows, w.N, m.cols,
          status_word(on.dev), on.stream);
  return out;
}

Tensor linear(const On& on, const Tensor& x, const Matrix& m, const Tensor& codes, const Weight& w,
              const Tensor& scale, const float* bias, const int32_t* offsets) {
  const int dt = dtype_code(x.scalar_type());
  Tensor out = at::empty({m.rows, w.N}, x.options());
  const int8_t* b = bdata(codes);
  // strides that are never stepped over do not count
  const int64_t ldb = w.N > 1 ? w.ldb : 0, gs = w.E > 1 ? w.gs : 0;
  const int aligned = ((reinterpret_cast<uintptr_t>(b) | (uintptr_t)ldb | (uintptr_t)gs) & 15) == 0;
  Bytes ws(api.g2q_int8_linear_workspace_bytes(m.rows, w.N, m.cols, w.E, aligned), x);
  G2Q_RUN(g2q_int8_linear, out.data_ptr(), dt, w.N, x.const_data_ptr(), dt, m.ld, b, w.ldb, w.gs,
          fdata(scale), bias, offsets, w.E, m.rows, w.N, m.cols, ws.get(), ws.n,
          status_word(on.dev), on.stream);
  return out;
}

Tensor int8_linear(const Tensor& x, const Tensor& codes, const Tensor& scale,
                   const optional<Tensor>& bias) {
  no_gradient("int8_linear", {&x, &scale, given(bias)});
  On on(x, {&codes, &scale, given(bias)});
  const Matrix m = matrix("x", x);
  const Weight w = weight(codes, scale, m.cols);
  if (bias) vector("bias", *bias, w.N, at::kFloat);
  return linear(on, x, m, codes, w, scale, fdata(bias), nullptr);
}

Tensor int8_linear_grouped(const Tensor& x, const Tensor& codes, const Tensor& scale,
                           const Tensor& offsets) {
  no_gradient("int8_linear_grouped", {&x, &scale});
  On on(x, {&codes, &scale, &offsets});
  const Matrix m = matrix("x", x);
  const Weight w = expert_weight(codes, scale, offsets, m.cols);
  return linear(on, x, m, codes, w, scale, nullptr, idata(offsets));
}

// ---------------------------------------------------------------------------
// expert routing
// ---------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> route(const Tensor& experts, int64_t num_experts) {
  On on(experts, {});
  TORCH_CHECK_VALUE(experts.dim() == 2 && experts.size(1) > 0,
                    "experts must be [tokens, slots], got shape ", experts.sizes());
  const bool wide = experts.scalar_type() == at::kLong;
  TORCH_CHECK_TYPE(wide || experts.scalar_type() == at::kInt, "experts must be int32 or int64, got ",
                   experts.scalar_type());
  TORCH_CHECK_VALUE(num_experts > 0 && num_experts <= kMaxExperts, "1 to ", kMaxExperts,
                    " experts, got ", num_experts);
  TORCH_CHECK_VALUE(experts.is_contiguous(), "experts must be contiguous");
  const int64_t n = experts.numel();
  const auto ints = experts.options().dtype(at::kInt);
  Tensor order = at::empty({n}, ints), position = at::empty(experts.sizes(), ints);
  Tensor offsets = at::empty({num_experts + 1}, ints);
  Bytes ws(api.g2q_route_workspace_bytes(n, num_experts), experts);
  G2Q_RUN(g2q_route, static_cast<int32_t*>(order.data_ptr()),
          static_cast<int32_t*>(position.data_ptr()), static_cast<int32_t*>(offsets.data_ptr()),
          experts.const_data_ptr(), (int)wide, n, num_experts, ws.get(), ws.n, on.stream);
  return {order, position, offsets};
}

struct Slots {
  int64_t T, k;
};

Slots slots(const Tensor& position) {
  TORCH_CHECK_VALUE(position.scalar_type() == at::kInt && position.dim() == 2 &&
                        position.size(1) > 0,
                    "position must be int32 [tokens, slots]");
  TORCH_CHECK_VALUE(position.is_contiguous(), "position must be contiguous");
  return {position.size(0), position.size(1)};
}

int weights_code(const Tensor& w, const Tensor& position) {
  if (!w.defined()) return 0;
  TORCH_CHECK_VALUE(w.sizes() == position.sizes(), "weights must have shape ", position.sizes());
  TORCH_CHECK_VALUE(w.is_contiguous(), "weights must be contiguous");
  return dtype_code(w.scalar_type());
}

const void* data_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

Tensor dispatch_rows(const Tensor& x, const Tensor& position) {
  On on(x, {&position});
  const Slots s = slots(position);
  const Matrix m = matrix("x", x);
  TORCH_CHECK_VALUE(m.rows == s.T && m.cols > 0, "x must have ", s.T,
                    " rows and at least one column");
  const int64_t eb = x.element_size();
  TORCH_CHECK_TYPE(eb == 1 || eb == 2 || eb == 4, "unsupported dtype ", x.scalar_type());
  Tensor out = at::empty({s.T * s.k, m.cols}, x.options());
  G2Q_RUN(g2q_dispatch_rows, out.data_ptr(), m.cols, x.const_data_ptr(), m.ld, (int)eb,
          idata(position), s.T, s.k, m.cols, on.stream);
  return out;
}

Tensor combine(const Tensor& y, const Tensor& position, const Tensor& w) {
  On on(y, {&position, &w});
  const Slots s = slots(position);
  const Matrix m = matrix("y", y);
  TORCH_CHECK_VALUE(m.rows == s.T * s.k && m.cols > 0, "y must have ", s.T * s.k,
                    " rows and at least one column");
  const int dt = dtype_code(y.scalar_type()), wdt = weights_code(w, position);
  Tensor out = at::empty({s.T, m.cols}, y.options());
  G2Q_RUN(g2q_combine_rows, out.data_ptr(), m.cols, y.const_data_ptr(), m.ld, dt, idata(position),
          data_or_null(w), wdt, s.T, s.k, m.cols, on.stream);
  return out;
}

Tensor combine_rows(const Tensor& y, const Tensor& position, const optional<Tensor>& weights) {
  return combine(y, position, weights.value_or(Tensor()));
}

std::tuple<Tensor, Tensor> combine_backward(const Tensor& grad, const Tensor& y_in,
                                            const Tensor& position, const Tensor& w, bool need_y,
                                            bool need_w) {
  const Tensor y = need_w ? y_in : Tensor();
  On on(grad, {&y, &position, &w});
  const Slots s = slots(position);
  const Matrix m = matrix("grad", grad);
  TORCH_CHECK_VALUE(m.rows == s.T && m.cols > 0, "grad must have ", s.T,
                    " rows and at least one column");
  TORCH_CHECK_VALUE(w.defined(), "combine_rows_backward needs the weights");
  const int dt = dtype_code(grad.scalar_type()), wdt = weights_code(w, position);
  int64_t ldy = m.cols;
  if (need_w) {
    TORCH_CHECK_VALUE(y.defined(), "the weights' gradient needs y");
    const Matrix ym = matrix("y", y);
    TORCH_CHECK_VALUE(ym.rows == s.T * s.k && ym.cols == m.cols &&
                          y.scalar_type() == grad.scalar_type(),
                      "y must be ", grad.scalar_type(), " of shape (", s.T * s.k, ", ", m.cols, ")");
    ldy = ym.ld;
  }
  Tensor gy, gw;
  if (need_y) gy = at::empty({s.T * s.k, m.cols}, grad.options());
  if (need_w) gw = at::empty(w.sizes(), w.options());
  G2Q_RUN(g2q_combine_rows_backward, need_y ? gy.data_ptr() : nullptr, m.cols,
          need_w ? gw.data_ptr() : nullptr, grad.const_data_ptr(), m.ld, data_or_null(y), ldy, dt,
          idata(position), w.const_data_ptr(), wdt, s.T, s.k, m.cols, on.stream);
  return {gy, gw};
}

std::tuple<optional<Tensor>, optional<Tensor>> combine_rows_backward(
    const Tensor& grad, const optional<Tensor>& y, const Tensor& position,
    const optional<Tensor>& weights, bool need_y, bool need_weights) {
  auto [gy, gw] = combine_backward(grad, y.value_or(Tensor()), position,
                                   weights.value_or(Tensor()), need_y, need_weights);
  auto opt = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; };
  return {opt(gy), opt(gw)};
}

// ---------------------------------------------------------------------------
// autograd
// ---------------------------------------------------------------------------

// With unit column stride and rows that do not overlap (a gradient that autograd
// broadcast can have stride zero).
Tensor plain_rows(const Tensor& t) {
  if (t.dim() != 2) return t;
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
    return t.contiguous();
  return t;
}

void once() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "the routing's gradients cannot be differentiated a second time");
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& position) {
    ctx->save_for_backward({position});
    return dispatch_rows(x, position);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    return {combine(plain_rows(grads[0]), ctx->get_saved_variables()[0], Tensor()), Tensor()};
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& position,
                        const Tensor& w) {
    ctx->save_for_backward({w.requires_grad() ? y : Tensor(), position, w});
    ctx->saved_data["y"] = y.requires_grad();
    return combine(y, position, w);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& y = saved[0];
    auto [gy, gw] = combine_backward(plain_rows(grads[0]), y, saved[1], saved[2],
                                     ctx->saved_data["y"].toBool(), y.defined());
    return {gy, Tensor(), gw};
  }
};

struct CombineOnes : torch::autograd::Function<CombineOnes> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& position) {
    ctx->save_for_backward({position});
    return combine(y, position, Tensor());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    return {dispatch_rows(plain_rows(grads[0]), ctx->get_saved_variables()[0]), Tensor()};
  }
};

Tensor dispatch_grad(const Tensor& x_in, const Tensor& position) {
  no_tangent("dispatch", {&x_in});
  const Tensor x = plain_rows(x_in);
  if (!(at::GradMode::is_enabled() && x.requires_grad())) return dispatch_rows(x, position);
  On::check(x, {&position});
  dtype_code(x.scalar_type());
  return Dispatch::apply(x, position);
}

Tensor combine_grad(const Tensor& y_in, const Tensor& position, const optional<Tensor>& weights) {
  no_tangent("combine", {&y_in, given(weights)});
  const Tensor y = plain_rows(y_in);
  const Tensor w = weights ? weights->contiguous() : Tensor();
  if (!(at::GradMode::is_enabled() && (y.requires_grad() || (w.defined() && w.requires_grad()))))
    return combine(y, position, w);
  On::check(y, {&position, &w});
  return w.defined() ? Combine::apply(y, position, w) : CombineOnes::apply(y, position);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  using torch::wrap_pybind_function;
  namespace py = pybind11;
  m.def("bind", &bind);
  m.def("quantize_tokens", wrap_pybind_function(&quantize_tokens));
  m.def("int8_matmul", wrap_pybind_function(&int8_matmul));
  m.def("int8_matmul_grouped", wrap_pybind_function(&int8_matmul_grouped));
  m.def("int8_linear", wrap_pybind_function(&int8_linear));
  m.def("int8_linear_grouped", wrap_pybind_function(&int8_linear_grouped));
  m.def("route", wrap_pybind_function(&route));
  m.def("dispatch_rows", wrap_pybind_function(&dispatch_rows));
  m.def("combine_rows", wrap_pybind_function(&combine_rows));
  m.def("combine_rows_backward", wrap_pybind_function(&combine_rows_backward));
  m.def("dispatch", wrap_pybind_function(&dispatch_grad));
  m.def("combine", wrap_pybind_function(&combine_grad));
}
