// Host side of the training operators: checks of arguments, allocation of results and workspaces from torch's caching
// allocator, and the calls of libcogaim.so's entry points.  The same in Python (ctypes) took 10 to 15 us a call, three to
// five times the smallest kernels; here it is 3.5 to 5 (linear forward 3.6, pack8 4.1, layer norm 4.9), most of it the launches.  The entry points' addresses
// come from the Python side (`bind`), which loads the library.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include "../../include/cogaim.h"

namespace {
namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using OptType = std::optional<at::ScalarType>;

constexpr int64_t GROUP = 32, MAX_NORM_WIDTH = 16384, MAX_LEADING_DIM = 1 << 21, MAX_ROWS = 0x7fffffff - 511, MAX_WIDTH = 1 << 30;
enum { ACT_NONE, ACT_RELU, ACT_GELU };

#define ENTRIES(X)                                                                                                        \
  X(cogaim_pack8) X(cogaim_unpack8) X(cogaim_activation_bwd) X(cogaim_layernorm_train_fwd) X(cogaim_layernorm_bwd)        \
  X(cogaim_layernorm_bwd_workspace_bytes) X(cogaim_linear_fwd) X(cogaim_linear_fwd_workspace_bytes)                       \
  X(cogaim_linear_bwd_input) X(cogaim_linear_bwd_input_workspace_bytes) X(cogaim_linear_bwd_weight)                       \
  X(cogaim_linear_bwd_weight_workspace_bytes) X(cogaim_scale_unit)       \
  X(cogaim_activation_bwd_from)
#define DECLARE(n) decltype(&::n) n##_;
ENTRIES(DECLARE)
PyObject* error_class = nullptr;

void bind(const py::dict& addresses, py::object error) {
#define LOOK_UP(n) n##_ = reinterpret_cast<decltype(&::n)>(py::cast<uintptr_t>(addresses[#n]));
  ENTRIES(LOOK_UP)
  error_class = error.release().ptr();
}
std::vector<std::string> entries() {
  std::vector<std::string> v;
#define NAME(n) v.push_back(#n);
  ENTRIES(NAME)
  return v;
}

void check(int rc, const char* name) {
  if (rc == 0) return;
  PyErr_Format(error_class, "%s failed with code %d", name, rc);
  throw py::error_already_set();
}

// ---- arguments ---------------------------------------------------------------------------------------------------
bool is_half(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool is_float(at::ScalarType t) { return is_half(t) || t == at::kFloat; }
int code(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : 2; }

void floats(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(is_float(t.scalar_type()), name, " must be bf16, fp16 or fp32, not ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name, " needs at least one column");
}
void halves(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(is_half(t.scalar_type()), name, " must be bf16 or fp16, not ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, name, " needs at least one column");
}
at::ScalarType out_type(OptType t, at::ScalarType otherwise) {
  const at::ScalarType o = t ? *t : otherwise;
  TORCH_CHECK_TYPE(is_float(o), "out_dtype must be bf16, fp16 or fp32, not ", o);
  return o;
}
int activation(const std::string& name) {
  if (name == "none") return ACT_NONE;
  if (name == "relu") return ACT_RELU;
  if (name == "gelu") return ACT_GELU;
  TORCH_CHECK_VALUE(false, "activation must be 'none', 'relu' or 'gelu', not '", name, "'");
}
void same_shape(const Tensor& t, const char* name, at::IntArrayRef shape, const at::Device& dev) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " has shape ", t.sizes(), ", ", shape, " is needed");
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", the rows are on ", dev);
}
OptTensor vec(const OptTensor& t, const char* name, int64_t n, const at::Device& dev) {
  if (!t) return t;
  TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == n, name, " must be a float32 vector of ", n);
  TORCH_CHECK_VALUE(t->device() == dev, name, " is on ", t->device(), ", the rows are on ", dev);
  return t->is_contiguous() ? t : OptTensor(t->contiguous());
}
Tensor needed_vec(const OptTensor& t, const char* name, int64_t n, const at::Device& dev) {
  TORCH_CHECK_VALUE(t.has_value(), name, " is needed");
  return *vec(t, name, n, dev);
}
Tensor stat(const OptTensor& t, const char* name, at::IntArrayRef lead, const at::Device& dev) {
  TORCH_CHECK_TYPE(t && t->scalar_type() == at::kFloat, name, " must be a float32 tensor");
  same_shape(*t, name, lead, dev);
  return t->contiguous();
}
struct Saved { Tensor codes, exponents; };
at::DimVector with_last(at::IntArrayRef lead, int64_t last) {
  at::DimVector v(lead.begin(), lead.end());
  v.push_back(last);
  return v;
}
Saved saved8(const Tensor& codes, const Tensor& exponents, const char* name, at::IntArrayRef shape, const at::Device& dev) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kChar && exponents.scalar_type() == at::kByte, name, ": codes must be int8 and exponents uint8");
  same_shape(codes, name, shape, dev);
  same_shape(exponents, name, with_last(shape.slice(0, shape.size() - 1), (shape.back() + GROUP - 1) / GROUP), dev);
  return Saved{codes.contiguous(), exponents.contiguous()};
}
// [rows, columns] of a tensor; a copy when its columns are not contiguous or its rows overlap
struct Rows { Tensor keep; void* p; int64_t ld; int n; };
Rows rows(const Tensor& t) {
  const int64_t D = t.size(-1);
  auto take = [&](const Tensor& u, int64_t n, int64_t ld) {
    TORCH_CHECK_VALUE(n <= MAX_ROWS, "more rows than the kernels count");
    return Rows{u, u.data_ptr(), ld, (int)n};
  };
  if (t.is_contiguous()) return take(t, t.numel() / D, D);
  const Tensor u = t.dim() == 2 ? t : t.reshape({t.numel() / D, D});
  const int64_t n = u.size(0), ld = n > 1 ? u.stride(0) : D;
  if (ld >= D && (D == 1 || u.stride(1) == 1)) return take(u, n, ld);
  const Tensor v = u.contiguous();
  return take(v, n, D);
}
int64_t leading(int64_t ld, const char* name) {
  TORCH_CHECK_VALUE(ld <= MAX_LEADING_DIM, "rows of ", name, " are ", ld, " elements apart: at most ", MAX_LEADING_DIM);
  return ld;
}
int narrow(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n <= MAX_WIDTH, name, " is wider than ", MAX_WIDTH);
  return (int)n;
}

// the tensors' device made current, and its current stream
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const at::Device& dev) : guard(checked(dev)), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream()) {}
  static const at::Device& checked(const at::Device& dev) {
    TORCH_CHECK(dev.is_cuda(), "the training operators run only on a ROCm device (no CPU path)");
    return dev;
  }
};
Tensor fresh(const Tensor& like, at::IntArrayRef shape, at::ScalarType t) { return at::empty(shape, like.options().dtype(t).requires_grad(false)); }
Saved fresh8(const Tensor& like, at::IntArrayRef lead, int64_t D) {
  return Saved{fresh(like, with_last(lead, D), at::kChar), fresh(like, with_last(lead, (D + GROUP - 1) / GROUP), at::kByte)};
}
template <class T = void> T* ptr(const OptTensor& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

// ---- 8-bit activations -------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> pack8(const Tensor& x) {
  floats(x, "x");
  const int64_t D = x.size(-1);
  narrow(D, "x");
  const On on(x.device());
  const Saved out = fresh8(x, x.sizes().slice(0, x.dim() - 1), D);
  const Rows v = rows(x);
  if (v.n)
    check(cogaim_pack8_(v.p, code(x.scalar_type()), v.ld, out.codes.data_ptr(), out.exponents.data_ptr(), v.n, (int)D, on.stream), "cogaim_pack8");
  return {out.codes, out.exponents};
}

Tensor unpack8(const Tensor& codes, const Tensor& exponents, at::ScalarType dtype) {
  const at::ScalarType t = out_type(dtype, dtype);
  TORCH_CHECK_VALUE(codes.dim() >= 1 && codes.size(-1) >= 1, "saved needs at least one column");
  const Saved s = saved8(codes, exponents, "saved", codes.sizes(), codes.device());
  const int D = narrow(codes.size(-1), "saved");
  const On on(codes.device());
  const Tensor out = fresh(codes, codes.sizes(), t);
  const int64_t M = codes.numel() / D;
  TORCH_CHECK_VALUE(M <= MAX_ROWS, "more rows than the kernels count");
  if (M)
    check(cogaim_unpack8_(s.codes.data_ptr(), s.exponents.data_ptr(), out.data_ptr(), code(t), D, (int)M, D, D, on.stream), "cogaim_unpack8");
  return out;
}

Tensor activation_backward(const Tensor& dy, const OptTensor& u, const OptTensor& codes, const OptTensor& exponents, const std::string& name, OptType dtype) {
  floats(dy, "dy");
  const int act = activation(name);
  TORCH_CHECK_VALUE(act != ACT_NONE, "activation must be 'relu' or 'gelu'");
  const at::ScalarType t = out_type(dtype, dy.scalar_type());
  if (u) {
    floats(*u, "saved");
    same_shape(*u, "saved", dy.sizes(), dy.device());
    const int D = narrow(dy.size(-1), "dy");
    const On on(dy.device());
    const Tensor out = fresh(dy, dy.sizes(), t);
    const Rows v = rows(dy), uv = rows(*u);
    if (v.n)
      check(cogaim_activation_bwd_from_(v.p, code(dy.scalar_type()), v.ld, uv.p, code(u->scalar_type()), uv.ld, out.data_ptr(), code(t), D, act, v.n, D,
                                        on.stream), "cogaim_activation_bwd_from");
    return out;
  }
  const Saved s = saved8(*codes, *exponents, "saved", dy.sizes(), dy.device());
  const int D = narrow(dy.size(-1), "dy");
  const On on(dy.device());
  const Tensor out = fresh(dy, dy.sizes(), t);
  const Rows v = rows(dy);
  if (v.n)
    check(cogaim_activation_bwd_(v.p, code(dy.scalar_type()), v.ld, s.codes.data_ptr(), s.exponents.data_ptr(), out.data_ptr(), code(t), D, act,
                                 v.n, D, on.stream), "cogaim_activation_bwd");
  return out;
}

// ---- layer norm --------------------------------------------------------------------------------------------------
int norm_width(const Tensor& x) {
  TORCH_CHECK_VALUE(x.size(-1) <= MAX_NORM_WIDTH, "layer norm of ", x.size(-1), " columns: at most ", MAX_NORM_WIDTH);
  return (int)x.size(-1);
}

std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor> layer_norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                                                            double eps, OptType dtype, bool checkpoint) {
  floats(x, "x");
  const int D = norm_width(x);
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative");
  const Tensor w = needed_vec(weight, "weight", D, x.device()), b = needed_vec(bias, "bias", D, x.device());
  const at::ScalarType t = out_type(dtype, x.scalar_type());
  const On on(x.device());
  const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
  const Tensor y = fresh(x, x.sizes(), t), mean = fresh(x, lead, at::kFloat), rstd = fresh(x, lead, at::kFloat);
  OptTensor codes, exponents;
  if (checkpoint) {
    const Saved s = fresh8(x, lead, D);
    codes = s.codes; exponents = s.exponents;
  }
  const Rows v = rows(x);
  if (v.n)
    check(cogaim_layernorm_train_fwd_(v.p, code(x.scalar_type()), v.ld, (const float*)w.data_ptr(), (const float*)b.data_ptr(), y.data_ptr(), code(t),
                                      D, (float*)mean.data_ptr(), (float*)rstd.data_ptr(), ptr(codes), ptr(exponents), v.n, D, (float)eps, on.stream),
          "cogaim_layernorm_train_fwd");
  return {y, mean, rstd, codes, exponents};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& dy, const OptTensor& x, const OptTensor& codes, const OptTensor& exponents,
                                                       const OptTensor& mean, const OptTensor& rstd, const OptTensor& weight, const OptTensor& add,
                                                       OptType dtype) {
  floats(dy, "dy");
  const int D = norm_width(dy);
  const at::Device dev = dy.device();
  const at::IntArrayRef lead = dy.sizes().slice(0, dy.dim() - 1);
  const Tensor w = needed_vec(weight, "weight", D, dev), r = stat(rstd, "rstd", lead, dev);
  OptTensor m, c, e;
  at::ScalarType t;
  if (x) {
    floats(*x, "saved");
    same_shape(*x, "saved", dy.sizes(), dev);
    m = stat(mean, "mean", lead, dev);
    t = out_type(dtype, x->scalar_type());
  } else {
    const Saved s = saved8(*codes, *exponents, "saved", dy.sizes(), dev);
    c = s.codes; e = s.exponents;
    t = out_type(dtype, dy.scalar_type());
  }
  if (add) {
    floats(*add, "add");
    same_shape(*add, "add", dy.sizes(), dev);
  }
  const On on(dev);
  const Tensor dx = fresh(dy, dy.sizes(), t);
  const Rows v = rows(dy);
  if (!v.n) return {dx, at::zeros({D}, w.options().requires_grad(false)), at::zeros({D}, w.options().requires_grad(false))};
  const Tensor dw = fresh(w, {D}, at::kFloat), db = fresh(w, {D}, at::kFloat);
  const long long bytes = cogaim_layernorm_bwd_workspace_bytes_(v.n, D);
  const Tensor ws = fresh(dy, {bytes}, at::kByte);
  const Rows xv = x ? rows(*x) : Rows{Tensor(), nullptr, 0, 0}, av = add ? rows(*add) : Rows{Tensor(), nullptr, 0, 0};
  check(cogaim_layernorm_bwd_(v.p, code(dy.scalar_type()), v.ld, xv.p, x ? code(x->scalar_type()) : 0, xv.ld, ptr(c), ptr(e), ptr<float>(m),
                              (const float*)r.data_ptr(), (const float*)w.data_ptr(), av.p, add ? code(add->scalar_type()) : 0, av.ld, dx.data_ptr(),
                              code(t), D, (float*)dw.data_ptr(), (float*)db.data_ptr(), v.n, D, ws.data_ptr(), bytes, on.stream),
        "cogaim_layernorm_bwd");
  return {dx, dw, db};
}

// scale times a power of two that brings small scales towards 1, and the 1-element tensor that undoes it
std::tuple<Tensor, Tensor> scale_unit(const Tensor& scale) {
  TORCH_CHECK_VALUE(scale.dim() == 1 && scale.size(0) >= 1, "scale must be a vector");
  const OptTensor s = vec(scale, "scale", narrow(scale.size(0), "scale"), scale.device());
  const On on(scale.device());
  const Tensor scaled = fresh(scale, scale.sizes(), at::kFloat), unit = fresh(scale, {1}, at::kFloat);
  check(cogaim_scale_unit_((const float*)s->data_ptr(), (float*)scaled.data_ptr(), (float*)unit.data_ptr(), (int)scale.size(0), on.stream), "cogaim_scale_unit");
  return {scaled, unit};
}

// ---- linear layers -----------------------------------------------------------------------------------------------
template <class Desc>
void run(const Desc& d, long long (*size)(const Desc*), int (*launch)(const Desc*, void*, long long, void*), const char* name, const Tensor& like, void* stream) {
  const long long bytes = size(&d);
  TORCH_CHECK_VALUE(bytes >= 0, name, ": arguments the kernels do not take");
  if (bytes == 0) return check(launch(&d, nullptr, 0, stream), name);
  const Tensor ws = fresh(like, {(int64_t)bytes}, at::kByte);
  check(launch(&d, ws.data_ptr(), bytes, stream), name);
}
void matrix(const Tensor& w) {
  halves(w, "weight");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 1, "weight must be a matrix");
}

std::tuple<Tensor, OptTensor, OptTensor, OptTensor> linear_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const std::string& name,
                                                                   const OptTensor& scale, const OptTensor& residual, OptType dtype, bool checkpoint,
                                                                   bool pre_activation) {
  halves(x, "x");
  matrix(weight);
  const int act = activation(name);
  const int N = narrow(weight.size(0), "weight"), K = narrow(weight.size(1), "weight");
  const at::Device dev = x.device();
  TORCH_CHECK_VALUE(x.size(-1) == K && weight.scalar_type() == x.scalar_type() && weight.device() == dev, "x ", x.sizes(), " ", x.scalar_type(), " on ",
                    dev, " does not go with weight ", weight.sizes(), " ", weight.scalar_type(), " on ", weight.device());
  TORCH_CHECK_VALUE(!scale || act == ACT_NONE, "scale goes with activation 'none'");
  TORCH_CHECK_VALUE(!checkpoint || !pre_activation, "checkpoint and pre_activation are two ways to keep one thing");
  const OptTensor b = vec(bias, "bias", N, dev), s = vec(scale, "scale", N, dev);
  const at::ScalarType t = out_type(dtype, x.scalar_type());
  const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
  const at::DimVector shape = with_last(lead, N);
  if (residual) {
    floats(*residual, "residual");
    same_shape(*residual, "residual", shape, dev);
  }
  const On on(dev);
  const Tensor y = fresh(x, shape, t);
  OptTensor codes, exponents, pre;
  if (checkpoint) {
    const Saved k = fresh8(x, lead, N);
    codes = k.codes; exponents = k.exponents;
  }
  if (pre_activation) pre = fresh(x, shape, x.scalar_type());
  const Rows xv = rows(x);
  if (xv.n) {
    const Rows wv = rows(weight), rv = residual ? rows(*residual) : Rows{Tensor(), nullptr, 0, 0};
    cogaim_linear_fwd_desc d{};
    d.x = xv.p; d.w = wv.p; d.bias = ptr<float>(b); d.scale = ptr<float>(s); d.residual = rv.p; d.y = y.data_ptr();
    d.codes = ptr(codes); d.exponents = ptr(exponents);
    d.ldx = leading(xv.ld, "x"); d.ldw = leading(wv.ld, "weight"); d.ldr = leading(rv.ld, "residual"); d.ldy = leading(N, "y");
    d.M = xv.n; d.N = N; d.K = K; d.dtype = code(x.scalar_type()); d.residual_dtype = residual ? code(residual->scalar_type()) : 0;
    d.y_dtype = code(t); d.activation = act; d.extended = 1; d.pre = ptr(pre);
    run(d, cogaim_linear_fwd_workspace_bytes_, cogaim_linear_fwd_, "cogaim_linear_fwd", x, on.stream);
  }
  return {y, codes, exponents, pre};
}

std::tuple<Tensor, OptTensor> linear_backward_input(const Tensor& dy, const Tensor& weight, const std::string& name, const OptTensor& codes,
                                                    const OptTensor& exponents, const OptTensor& scale, OptType dtype, bool want_activation) {
  halves(dy, "dy");
  matrix(weight);
  const int act = activation(name);
  const int N = narrow(weight.size(0), "weight"), K = narrow(weight.size(1), "weight");
  const at::Device dev = dy.device();
  TORCH_CHECK_VALUE(dy.size(-1) == N && weight.scalar_type() == dy.scalar_type() && weight.device() == dev, "dy ", dy.sizes(), " ", dy.scalar_type(),
                    " on ", dev, " does not go with weight ", weight.sizes(), " ", weight.scalar_type(), " on ", weight.device());
  TORCH_CHECK_VALUE((act != ACT_NONE) == codes.has_value(), "saved is the pre-activation of an activation: give both or neither");
  TORCH_CHECK_VALUE(!want_activation || act != ACT_NONE, "want_activation needs an activation");
  const OptTensor s = vec(scale, "scale", N, dev);
  const at::ScalarType t = out_type(dtype, dy.scalar_type());
  const at::DimVector shape = with_last(dy.sizes().slice(0, dy.dim() - 1), K);
  OptTensor c, e;
  if (codes) {
    const Saved k = saved8(*codes, *exponents, "saved", shape, dev);
    c = k.codes; e = k.exponents;
  }
  const On on(dev);
  const Tensor dx = fresh(dy, shape, t);
  OptTensor a;
  if (want_activation) a = fresh(dy, shape, dy.scalar_type());
  const Rows v = rows(dy);
  if (v.n) {
    const Rows wv = rows(weight);
    cogaim_linear_bwd_input_desc d{};
    d.dy = v.p; d.w = wv.p; d.scale = ptr<float>(s); d.codes = ptr(c); d.exponents = ptr(e); d.dx = dx.data_ptr(); d.a = ptr(a);
    d.lddy = leading(v.ld, "dy"); d.ldw = leading(wv.ld, "weight"); d.lddx = leading(K, "dx"); d.lda = K;
    d.M = v.n; d.N = N; d.K = K; d.dtype = code(dy.scalar_type()); d.dx_dtype = code(t); d.activation = act;
    run(d, cogaim_linear_bwd_input_workspace_bytes_, cogaim_linear_bwd_input_, "cogaim_linear_bwd_input", dy, on.stream);
  }
  return {dx, a};
}

std::tuple<Tensor, Tensor, OptTensor> linear_backward_weight(const Tensor& dy, const OptTensor& x, const OptTensor& codes, const OptTensor& exponents,
                                                             const OptTensor& weight, const OptTensor& bias, const OptTensor& scale,
                                                             const OptTensor& x_scale, const OptTensor& x_shift, at::ScalarType dtype) {
  halves(dy, "dy");
  const int N = narrow(dy.size(-1), "dy");
  const at::Device dev = dy.device();
  const at::IntArrayRef lead = dy.sizes().slice(0, dy.dim() - 1);
  OptTensor c, e;
  int K;
  if (x) {
    halves(*x, "x");
    K = narrow(x->size(-1), "x");
    same_shape(*x, "x", with_last(lead, K), dev);
    TORCH_CHECK_TYPE(x->scalar_type() == dy.scalar_type(), "x is ", x->scalar_type(), ", dy ", dy.scalar_type());
    TORCH_CHECK_VALUE(!x_scale && !x_shift, "x_scale and x_shift go with an 8-bit x");
  } else {
    TORCH_CHECK_VALUE(codes->dim() >= 1 && codes->size(-1) >= 1, "x needs at least one column");
    K = narrow(codes->size(-1), "x");
    const Saved k = saved8(*codes, *exponents, "x", with_last(lead, K), dev);
    c = k.codes; e = k.exponents;
  }
  const OptTensor xs = vec(x_scale, "x_scale", K, dev), xt = vec(x_shift, "x_shift", K, dev), s = vec(scale, "scale", N, dev);
  OptTensor b;
  if (s) {
    TORCH_CHECK_VALUE(weight.has_value(), "scale needs the forward's weight");
    matrix(*weight);
    same_shape(*weight, "weight", {N, K}, dev);
    TORCH_CHECK_TYPE(weight->scalar_type() == dy.scalar_type(), "weight is ", weight->scalar_type(), ", dy ", dy.scalar_type());
    b = vec(bias, "bias", N, dev);
  } else {
    TORCH_CHECK_VALUE(!weight && !bias, "weight and bias go with scale");
  }
  const at::ScalarType t = out_type(dtype, dtype);
  const On on(dev);
  const Rows v = rows(dy);
  const Tensor dw = fresh(dy, {N, K}, t), db = fresh(dy, {N}, at::kFloat);
  OptTensor ds;
  if (s) ds = fresh(dy, {N}, at::kFloat);
  if (!v.n) {
    dw.zero_(); db.zero_();
    if (ds) ds->zero_();
    return {dw, db, ds};
  }
  const Rows xv = x ? rows(*x) : Rows{Tensor(), nullptr, 0, 0}, wv = s ? rows(*weight) : Rows{Tensor(), nullptr, 0, 0};
  cogaim_linear_bwd_weight_desc d{};
  d.dy = v.p; d.x = xv.p; d.codes = ptr(c); d.exponents = ptr(e); d.x_scale = ptr<float>(xs); d.x_shift = ptr<float>(xt);
  d.w = wv.p; d.bias = ptr<float>(b); d.scale = ptr<float>(s); d.dw = dw.data_ptr(); d.db = (float*)db.data_ptr(); d.ds = ptr<float>(ds);
  d.lddy = leading(v.ld, "dy"); d.ldx = leading(xv.ld, "x"); d.ldw = leading(wv.ld, "weight"); d.lddw = leading(K, "dW");
  d.M = v.n; d.N = N; d.K = K; d.dtype = code(dy.scalar_type()); d.dw_dtype = code(t);
  run(d, cogaim_linear_bwd_weight_workspace_bytes_, cogaim_linear_bwd_weight_, "cogaim_linear_bwd_weight", dy, on.stream);
  return {dw, db, ds};
}
}  // namespace

PYBIND11_MODULE(_host, m) {
  m.def("bind", &bind);
  m.def("entries", &entries);
  m.def("pack8", &pack8);
  m.def("unpack8", &unpack8);
  m.def("activation_backward", &activation_backward);
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("scale_unit", &scale_unit);
  m.def("linear_forward", &linear_forward);
  m.def("linear_backward_input", &linear_backward_input);
  m.def("linear_backward_weight", &linear_backward_weight);
}
