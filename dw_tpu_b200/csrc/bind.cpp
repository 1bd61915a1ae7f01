// The calls of the operators around the expert layer from Python without
// ctypes: dense_matmul, route_grouped_topk and block_norm check torch tensors,
// allocate what is not given and call the C ABI on the current stream of the
// tensors' device. A decode step makes these calls for kernels of 2-10 us, where
// ~40 attribute lookups and a ctypes call cost more than the kernel: host time of
// post_norm with most arguments 24.6 us that way, 5.2 us here; pre_norm 17.4 and
// 4.3, dense_matmul 16.0 and 4.4.
//
// The C ABI stays the one implementation: its functions are looked up in
// libdw_moe.so (init), and what they refuse raises ValueError with their
// message, as for every other op.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <dlfcn.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <optional>
#include <string>

#include "../../include/dw_moe.h"

namespace {

using at::Tensor;
using Opt = std::optional<Tensor>;

decltype(&dwm_dense_matmul) g_dense;
decltype(&dwm_route_grouped_topk) g_route;
decltype(&dwm_block_norm) g_norm;
decltype(&dwm_last_error) g_error;

void check_rc(int rc, const char* what) {
  if (rc == DWM_OK) return;
  TORCH_CHECK_VALUE(rc != DWM_ERR_INVALID && rc != DWM_ERR_UNSUPPORTED, what, ": ", g_error());
  TORCH_CHECK(rc < 0, what, ": CUDA error ", rc, ": ", g_error());
  TORCH_CHECK(false, what, ": ", g_error());
}

// ---- arguments -------------------------------------------------------------
Tensor tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
Opt optional_tensor(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor(o, name);
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
int int32(PyObject* o, const char* name) {
  const long long v = integer(o);
  TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, name, "=", v, " is out of range");
  return (int)v;
}
float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return (float)v;
}
// An explicit cudaStream_t (an int), or None: the current stream of `dev`.
void* stream_of(PyObject* o, c10::Device dev) {
  if (o != Py_None) return reinterpret_cast<void*>(integer(o));
  return c10::cuda::getCurrentCUDAStream(dev.index()).stream();
}

// ---- tensors ---------------------------------------------------------------
void* data(const Opt& t) { return t ? t->data_ptr() : nullptr; }

void same_device(c10::Device dev, const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device().str(), ", not on ", dev.str());
}
c10::Device cuda_device(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "dw_tpu_b200 ops take CUDA tensors (no CPU path)");
  return t.device();
}
// Inputs that autograd would expect a gradient for, or that carry a forward-mode
// tangent, are refused: these ops are for inference and record none.
void no_grad(const Tensor& t) {
  TORCH_CHECK_VALUE(!(t._fw_grad(/*level=*/0).defined() &&
                      c10::AutogradState::get_tls_state().get_fw_grad_mode()),
                    "inference only: an input has a forward-mode tangent");
  TORCH_CHECK_VALUE(!(t.requires_grad() && c10::GradMode::is_enabled()),
                    "inference only: an input requires a gradient (call under torch.no_grad() or "
                    "detach it)");
}
void no_grad(const Opt& t) {
  if (t) no_grad(*t);
}

int dtype_of(const Tensor& t, const char* name) {
  const auto d = t.scalar_type();
  TORCH_CHECK_VALUE(d == at::kBFloat16 || d == at::kFloat, name, " dtype ", d, " not supported");
  return d == at::kFloat ? DWM_F32 : DWM_BF16;
}
at::ScalarType type_of(int code) { return code == DWM_F32 ? at::kFloat : at::kBFloat16; }

// A 2-D tensor with unit stride along its rows; returns its row stride.
int64_t rows(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 2, name, " must be 2-D, got ", t.sizes());
  TORCH_CHECK_VALUE(t.stride(1) == 1 || t.size(1) <= 1, name,
                    " must have unit stride along its rows");
  return t.stride(0);
}
int64_t rows(const Tensor& t, const char* name, int64_t m, int64_t n) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == m && t.size(1) == n, name, " must be [", m, ", ",
                    n, "], got ", t.sizes());
  return rows(t, name);
}
void vector(const Tensor& t, const char* name, int64_t n) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, name, " must be a vector of ", n, ", got ",
                    t.sizes());
  TORCH_CHECK_VALUE(n <= 1 || t.stride(0) == 1, name, " must be contiguous");
}
int size32(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v <= INT32_MAX, name, "=", v, " is too large");
  return (int)v;
}
// A new output, of the current stream's memory: a call on a stream of its own
// brings its outputs.
Tensor fresh(int64_t m, int64_t n, at::ScalarType dt, c10::Device dev, PyObject* stream) {
  TORCH_CHECK_VALUE(stream == Py_None, "a call with a stream of its own needs its outputs given");
  return at::detail::empty_cuda({m, n}, dt, dev, std::nullopt);  // (at::empty: 0.25 us more)
}
Tensor fresh(int64_t m, int64_t n, int code, c10::Device dev, PyObject* stream) {
  return fresh(m, n, type_of(code), dev, stream);
}

// ---- the calls -------------------------------------------------------------
// Positional arguments only; ops.py names them.

// (x, w, bias, act, act_limit, residual, residual_scale, out, out_dtype, stream)
PyObject* dense_matmul(PyObject*, PyObject* const* v, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n_args == 10, "dense_matmul takes 10 arguments");
  const Tensor x = tensor(v[0], "x"), w = tensor(v[1], "w");
  const Opt bias = optional_tensor(v[2], "bias"), res = optional_tensor(v[5], "residual");
  Opt out = optional_tensor(v[7], "out");
  const int act = int32(v[3], "act");
  no_grad(x);
  no_grad(w);
  no_grad(bias);
  no_grad(res);
  no_grad(out);
  const c10::Device dev = cuda_device(x);
  same_device(dev, w, "w");
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16,
                    "x and w must be bf16, got ", x.scalar_type(), " and ", w.scalar_type());
  const int64_t ldx = rows(x, "x"), ldw = rows(w, "w");
  const int m = size32(x.size(0), "m"), k = size32(x.size(1), "k"), n = size32(w.size(0), "n");
  TORCH_CHECK_VALUE(w.size(1) == k, "x has k=", k, ", w k=", w.size(1));
  const int n_out = act == DWM_ACT_SWIGLU || act == DWM_ACT_SWIGLU_CLAMP ? n / 2 : n;
  if (bias) {
    same_device(dev, *bias, "bias");
    vector(*bias, "bias", n);
  }
  int64_t ldr = 0;
  if (res) {
    same_device(dev, *res, "residual");
    ldr = rows(*res, "residual", m, n_out);
  }
  const c10::cuda::OptionalCUDAGuard guard(dev);
  if (out) {
    same_device(dev, *out, "out");
  } else {
    out = fresh(m, n_out, int32(v[8], "out_dtype"), dev, v[9]);
  }
  const int64_t ldo = rows(*out, "out", m, n_out);
  check_rc(g_dense(x.data_ptr(), ldx, w.data_ptr(), ldw, m, n, k, data(bias),
                   bias ? dtype_of(*bias, "bias") : DWM_F32, act, real(v[4]), data(res),
                   res ? dtype_of(*res, "residual") : DWM_F32, ldr, real(v[6]), data(out),
                   dtype_of(*out, "out"), ldo, stream_of(v[9], dev)),
           "dense_matmul");
  return THPVariable_Wrap(*out);
  END_HANDLE_TH_ERRORS
}

// (logits, top_k, num_groups, topk_groups, scoring, group_score, renormalize, routed_scale, bias,
//  num_valid, weights_dtype, ids, w32, w16, stream) -> (weights, ids)
// ids / w32 / w16 None: ids and weights of weights_dtype are allocated.
PyObject* route_grouped_topk(PyObject*, PyObject* const* v, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n_args == 15, "route_grouped_topk takes 15 arguments");
  const Tensor logits = tensor(v[0], "logits");
  const Opt bias = optional_tensor(v[8], "bias");
  Opt ids = optional_tensor(v[11], "ids_out"), w32 = optional_tensor(v[12], "w32_out"),
      w16 = optional_tensor(v[13], "w16_out");
  no_grad(logits);
  no_grad(bias);
  no_grad(w32);
  no_grad(w16);
  const c10::Device dev = cuda_device(logits);
  const int64_t ld = rows(logits, "logits");
  const int t = size32(logits.size(0), "t"), e = size32(logits.size(1), "e");
  const int top_k = int32(v[1], "top_k");
  const int dt = logits.scalar_type() == at::kDouble ? DWM_F64 : dtype_of(logits, "logits");
  if (bias) {
    same_device(dev, *bias, "bias");
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat, "bias must be f32");
    vector(*bias, "bias", e);
  }
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const bool own = !ids;
  if (own) {
    TORCH_CHECK_VALUE(top_k >= 1 && top_k <= 32, "top_k=", top_k, " must be in [1, 32]");
    const int type = int32(v[10], "dtype");
    ids = fresh(t, top_k, at::kInt, dev, v[14]);
    (type == DWM_F32 ? w32 : w16) = fresh(t, top_k, type, dev, v[14]);
  } else {
    auto given = [&](const Opt& o, at::ScalarType type, const char* name) {
      if (!o) return;
      same_device(dev, *o, name);
      TORCH_CHECK_VALUE(o->dim() == 2 && o->size(0) == t && o->size(1) == top_k &&
                            o->scalar_type() == type && o->is_contiguous(),
                        name, " must be a contiguous ", type, " [", t, ", ", top_k, "] tensor");
    };
    given(ids, at::kInt, "ids_out");
    given(w32, at::kFloat, "w32_out");
    given(w16, at::kBFloat16, "w16_out");
  }
  check_rc(g_route(logits.data_ptr(), dt, ld, t, e, top_k, int32(v[2], "num_groups"),
                   int32(v[3], "topk_groups"), int32(v[4], "scoring"), int32(v[5], "group_score"),
                   int32(v[6], "renormalize"), real(v[7]), static_cast<float*>(data(bias)),
                   int32(v[9], "num_valid_tokens"), static_cast<int32_t*>(data(ids)),
                   static_cast<float*>(data(w32)), data(w16), stream_of(v[14], dev)),
           "route_grouped_topk");
  if (!own) Py_RETURN_NONE;
  THPObjectPtr a(THPVariable_Wrap(w32 ? *w32 : *w16)), b(THPVariable_Wrap(*ids));
  if (!a || !b) return nullptr;
  return PyTuple_Pack(2, a.get(), b.get());
  END_HANDLE_TH_ERRORS
}

// (residual, y, norm_weight, norm_bias, gate, scale, residual_scale, weight, bias, eps, kind,
//  r_out, h_out, h_dtype, want_h, stream) -> (r_out, h_out)
// r_out (with y) and h_out (want_h) are allocated where they are None.
PyObject* block_norm(PyObject*, PyObject* const* v, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n_args == 16, "block_norm takes 16 arguments");
  const Tensor res = tensor(v[0], "residual");
  const Opt y = optional_tensor(v[1], "y"), gate = optional_tensor(v[4], "gate");
  const Opt vec[4] = {optional_tensor(v[2], "norm_weight"), optional_tensor(v[3], "norm_bias"),
                      optional_tensor(v[7], "weight"), optional_tensor(v[8], "bias")};
  Opt r_out = optional_tensor(v[11], "r_out"), h_out = optional_tensor(v[12], "h_out");
  const bool want_h = integer(v[14]) != 0;
  no_grad(res);
  no_grad(y);
  no_grad(gate);
  for (const Opt& x : vec) no_grad(x);
  no_grad(r_out);
  no_grad(h_out);
  const c10::Device dev = cuda_device(res);
  const int64_t ldres = rows(res, "residual");
  const int t = size32(res.size(0), "t"), h = size32(res.size(1), "h");
  const int res_dt = dtype_of(res, "residual");
  const char* names[4] = {"norm_weight", "norm_bias", "weight", "bias"};
  int w_dt = -1;
  for (int i = 0; i < 4; ++i) {
    if (!vec[i]) continue;
    same_device(dev, *vec[i], names[i]);
    vector(*vec[i], names[i], h);
    const int d = dtype_of(*vec[i], names[i]);
    TORCH_CHECK_VALUE(w_dt < 0 || w_dt == d,
                      "the norms' weights and biases must share one dtype");
    w_dt = d;
  }
  TORCH_CHECK_VALUE(!vec[1] || vec[0], "norm_bias needs norm_weight");
  TORCH_CHECK_VALUE(want_h ? vec[2].has_value() : !vec[3] && !vec[2] && !h_out,
                    "h_out, weight and bias belong together: h_out = norm(r) * weight + bias");
  TORCH_CHECK_VALUE(y || (!r_out && !gate && !vec[0]),
                    "r_out, gate and norm_weight go with y");
  int64_t ldy = 0, ldg = 0, ldr = 0, ldh = 0;
  int mode = DWM_GATE_NONE;
  if (y) {
    same_device(dev, *y, "y");
    ldy = rows(*y, "y", t, h);
  }
  if (gate) {
    same_device(dev, *gate, "gate");
    TORCH_CHECK_VALUE(gate->scalar_type() == y->scalar_type(), "gate must have y's dtype");
    if (gate->dim() == 1) {
      vector(*gate, "gate", h);
      mode = DWM_GATE_CHANNEL;
    } else {
      const bool one = gate->dim() == 2 && gate->size(1) == 1;
      ldg = rows(*gate, "gate", t, one ? 1 : h);
      mode = one ? DWM_GATE_TOKEN : DWM_GATE_FULL;
    }
  }
  const c10::cuda::OptionalCUDAGuard guard(dev);
  if (y) {
    if (r_out) {
      same_device(dev, *r_out, "r_out");
      TORCH_CHECK_VALUE(r_out->scalar_type() == res.scalar_type(),
                        "r_out must have residual's dtype");
    } else {
      r_out = fresh(t, h, res_dt, dev, v[15]);
    }
    ldr = rows(*r_out, "r_out", t, h);
  }
  int h_dt = DWM_BF16;
  if (want_h) {
    if (h_out) {
      same_device(dev, *h_out, "h_out");
    } else {
      h_out = fresh(t, h, int32(v[13], "h_dtype"), dev, v[15]);
    }
    ldh = rows(*h_out, "h_out", t, h);
    h_dt = dtype_of(*h_out, "h_out");
  }
  check_rc(g_norm(data(y), y ? dtype_of(*y, "y") : DWM_BF16, ldy, res.data_ptr(), res_dt, ldres, t,
                  h, int32(v[10], "kind"), real(v[9]), vec[0].has_value(), data(vec[0]),
                  data(vec[1]), data(gate), mode, ldg, real(v[5]), real(v[6]), data(vec[2]),
                  data(vec[3]), w_dt == DWM_F32 ? DWM_F32 : DWM_BF16, data(r_out), ldr,
                  data(h_out), h_dt, ldh, stream_of(v[15], dev)),
           "block_norm");
  auto wrap = [](const Opt& o) { return o ? THPVariable_Wrap(*o) : Py_NewRef(Py_None); };
  THPObjectPtr a(wrap(r_out)), b(wrap(h_out));
  if (!a || !b) return nullptr;
  return PyTuple_Pack(2, a.get(), b.get());
  END_HANDLE_TH_ERRORS
}

// init(path): takes the C ABI from the library at `path`.
PyObject* init(PyObject*, PyObject* path) {
  HANDLE_TH_ERRORS
  const char* p = PyUnicode_AsUTF8(path);
  if (!p) return nullptr;
  void* lib = dlopen(p, RTLD_NOW | RTLD_LOCAL);
  if (!lib) {
    PyErr_Format(PyExc_ImportError, "%s", dlerror());
    return nullptr;
  }
  g_dense = reinterpret_cast<decltype(g_dense)>(dlsym(lib, "dwm_dense_matmul"));
  g_route = reinterpret_cast<decltype(g_route)>(dlsym(lib, "dwm_route_grouped_topk"));
  g_norm = reinterpret_cast<decltype(g_norm)>(dlsym(lib, "dwm_block_norm"));
  g_error = reinterpret_cast<decltype(g_error)>(dlsym(lib, "dwm_last_error"));
  if (!g_dense || !g_route || !g_norm || !g_error) {
    PyErr_Format(PyExc_ImportError, "%s lacks an entry point: build it anew", p);
    return nullptr;
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"init", init, METH_O, "init(path of libdw_moe.so)"},
    {"dense_matmul", reinterpret_cast<PyCFunction>(dense_matmul), METH_FASTCALL, nullptr},
    {"route_grouped_topk", reinterpret_cast<PyCFunction>(route_grouped_topk), METH_FASTCALL,
     nullptr},
    {"block_norm", reinterpret_cast<PyCFunction>(block_norm), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, kMethods};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit__bind() {
  PyObject* m = PyModule_Create(&kModule);
  // The torch whose internals it is compiled against.
  if (m && PyModule_AddStringConstant(m, "torch_version", DWM_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
