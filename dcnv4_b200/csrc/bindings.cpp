// Fast route of the LayerNorm training passes from Python into the C ABI: one C call that checks the tensors, allocates
// the results and launches, for what an ordinary call looks like (CUDA tensors on the current device, contiguous, types and
// sizes that fit, at least one row).  Anything else returns None, and the Python route -- which raises what is wrong with
// the arguments, changes the device or handles empty tensors -- takes the call.
//
// A LayerNorm of a small feature map runs in 2 us; checked, allocated and passed through ctypes argument by argument, a
// forward and a backward call took 13 and 19 us of host time; this way they take 6 and 9.
//
// The library itself stays free of framework types: its functions are handed over as addresses (`init`).
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

namespace {

using FwdFn = int (*)(const void*, const void*, const void*, const void*, const void*, const float*, void*, void*, float*,
                      float*, int, int, int, int, long long, int, long long, float, int, void*);
using BwdFn = int (*)(const void*, const void*, const void*, const float*, const float*, const void*, const void*,
                      const void*, const float*, void*, void*, void*, void*, void*, void*, size_t, int, int, int, int,
                      long long, int, long long, int, void*);
using SeamBwdFn = int (*)(const void*, const void*, const void*, const void*, const float*, const float*, const void*,
                          const float*, void*, void*, void*, void*, void*, size_t, int, int, long long, int, long long, void*);
using WorkspaceFn = size_t (*)(int, long long, int);

FwdFn g_fwd = nullptr;
BwdFn g_bwd = nullptr;
WorkspaceFn g_workspace = nullptr;
SeamBwdFn g_seam_bwd = nullptr;

constexpr int kPlain = 0, kPost = 1, kPre = 2;
constexpr int64_t kMaxChannels = 8192, kMaxRows = (int64_t)1 << 30;

// Type code of the C ABI, or -1.
inline int code_of(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1;
}
inline at::ScalarType type_of(int code) { return code == 0 ? at::kFloat : code == 1 ? at::kHalf : at::kBFloat16; }

// A tensor argument, or nullptr for None; `ok` turns false for anything else, and for tensor subclasses.
inline const at::Tensor* tensor(PyObject* o, bool& ok) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_CheckExact(o)) { ok = false; return nullptr; }
  return &THPVariable_Unpack(o);
}
inline bool plain(const at::Tensor& t, at::Device dev, at::ScalarType type) {
  return t.device() == dev && t.scalar_type() == type && t.is_contiguous() && !t.unsafeGetTensorImpl()->is_python_dispatch();
}
inline void* data(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// The interpreter goes on while results are allocated and kernels launched (a kernel's first launch loads it).
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// What both passes check; fills rows, channels and rows per sample.
bool accept(const at::Tensor& x, at::ScalarType x_type, at::ScalarType out_type, const at::Tensor& w, const at::Tensor& b,
            const at::Tensor* gamma, const at::Tensor* s, int64_t& rows, int64_t& C, int64_t& per) {
  const at::Device dev = x.device();
  const at::ScalarType p = w.scalar_type();
  if (!x.is_cuda() || dev.index() != c10::cuda::current_device() || x.dim() < 1 || x.numel() == 0 ||
      !plain(x, dev, x.scalar_type()) || code_of(x.scalar_type()) < 0 || code_of(x_type) < 0)
    return false;
  C = x.size(-1);
  rows = x.numel() / C;
  per = rows;
  if (C > kMaxChannels || rows > kMaxRows || (out_type != x_type && out_type != at::kFloat) ||
      (p != x_type && p != at::kFloat) || !plain(w, dev, p) || w.numel() != C || !plain(b, dev, p) || b.numel() != C)
    return false;
  if (gamma && (!plain(*gamma, dev, p) || gamma->numel() != C)) return false;
  if (s) {
    const int64_t n = s->numel();
    if (!plain(*s, dev, at::kFloat) || n == 0 || x.dim() < 2 || x.size(0) % n != 0) return false;
    per = rows / n;
  }
  return true;
}

// init(forward, backward, workspace bytes, backward of the seam from branch and residual): addresses of the library's functions.
PyObject* py_init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) { PyErr_SetString(PyExc_TypeError, "init takes four addresses"); return nullptr; }
  g_fwd = reinterpret_cast<FwdFn>(PyLong_AsVoidPtr(a[0]));
  g_bwd = reinterpret_cast<BwdFn>(PyLong_AsVoidPtr(a[1]));
  g_workspace = reinterpret_cast<WorkspaceFn>(PyLong_AsVoidPtr(a[2]));
  g_seam_bwd = reinterpret_cast<SeamBwdFn>(PyLong_AsVoidPtr(a[3]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// ln_forward(mode, x, residual, weight, bias, eps, layer_scale, sample_scale, activation, out type code)
// -> (y, mean, rstd), with the sum in front for the pre-norm seam; an error code; or None.
PyObject* py_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !g_fwd) Py_RETURN_NONE;
  bool ok = true;
  const int mode = (int)PyLong_AsLong(a[0]), act = (int)PyLong_AsLong(a[8]), out_code = (int)PyLong_AsLong(a[9]);
  const double eps = PyFloat_AsDouble(a[5]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *x = tensor(a[1], ok), *res = tensor(a[2], ok), *w = tensor(a[3], ok), *b = tensor(a[4], ok);
  const at::Tensor *gamma = tensor(a[6], ok), *s = tensor(a[7], ok);
  if (!ok || !x || !w || !b || (mode != kPlain) != (res != nullptr) || out_code < 0 || out_code > 2) Py_RETURN_NONE;
  const at::ScalarType out = type_of(out_code);
  int64_t rows, C, per;
  if (!accept(*x, x->scalar_type(), out, *w, *b, gamma, s, rows, C, per)) Py_RETURN_NONE;
  if (res && (!plain(*res, x->device(), out) || res->sizes() != x->sizes())) Py_RETURN_NONE;
  at::Tensor y, h, mean, rstd;
  int rc;
  {
    Unlocked unlocked;
    const auto opts = x->options().requires_grad(false);
    y = at::empty(x->sizes(), opts.dtype(out));
    mean = at::empty({rows}, opts.dtype(at::kFloat));
    rstd = at::empty({rows}, opts.dtype(at::kFloat));
    if (mode == kPre) h = at::empty(x->sizes(), opts.dtype(out));
    rc = g_fwd(x->data_ptr(), data(res), w->data_ptr(), b->data_ptr(), data(gamma), static_cast<const float*>(data(s)),
               y.data_ptr(), mode == kPre ? h.data_ptr() : nullptr, mean.data_ptr<float>(), rstd.data_ptr<float>(), mode,
               code_of(x->scalar_type()), out_code, code_of(w->scalar_type()), rows, (int)C, per, (float)eps, act,
               c10::cuda::getCurrentCUDAStream(x->device().index()).stream());
  }
  if (rc) return PyLong_FromLong(rc);
  const int extra = mode == kPre;
  PyObject* tuple = PyTuple_New(3 + extra);
  if (!tuple) return nullptr;
  if (extra) PyTuple_SET_ITEM(tuple, 0, THPVariable_Wrap(std::move(h)));
  PyTuple_SET_ITEM(tuple, extra, THPVariable_Wrap(std::move(y)));
  PyTuple_SET_ITEM(tuple, extra + 1, THPVariable_Wrap(std::move(mean)));
  PyTuple_SET_ITEM(tuple, extra + 2, THPVariable_Wrap(std::move(rstd)));
  return tuple;
  END_HANDLE_TH_ERRORS
}

// ln_backward(mode, grad_y, grad_h, x or h, residual, mean, rstd, weight, bias, layer_scale, sample_scale, activation, type
// code of the branch input) -> (grad_x, grad_branch, grad_weight, grad_bias, grad_layer_scale), an error code, or None.
// With a residual (pre-norm seam in 16 bits) x is the branch.  grad_branch is grad_x itself where the two are equal;
// grad_layer_scale is None without a layer scale.
PyObject* py_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13 || !g_bwd) Py_RETURN_NONE;
  bool ok = true;
  const int mode = (int)PyLong_AsLong(a[0]), act = (int)PyLong_AsLong(a[11]), code = (int)PyLong_AsLong(a[12]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *gy = tensor(a[1], ok), *gh = tensor(a[2], ok), *x = tensor(a[3], ok), *res = tensor(a[4], ok);
  const at::Tensor *mean = tensor(a[5], ok), *rstd = tensor(a[6], ok), *w = tensor(a[7], ok), *b = tensor(a[8], ok);
  const at::Tensor *gamma = tensor(a[9], ok), *s = tensor(a[10], ok);
  if (!ok || !gy || !x || !mean || !rstd || !w || !b || code < 0 || code > 2) Py_RETURN_NONE;
  const bool pre = mode == kPre;
  const at::ScalarType branch_type = type_of(code), out = gy->scalar_type();
  int64_t rows, C, per;
  if (!accept(*x, branch_type, out, *w, *b, gamma, s, rows, C, per)) Py_RETURN_NONE;
  const at::Device dev = x->device();
  if (res && (!pre || branch_type != out || out == at::kFloat || !plain(*res, dev, out) || res->sizes() != x->sizes()))
    Py_RETURN_NONE;
  if (x->scalar_type() != (pre ? out : branch_type) || !plain(*gy, dev, out) || gy->sizes() != x->sizes() ||
      (gh && (!plain(*gh, dev, out) || gh->sizes() != x->sizes())) || !plain(*mean, dev, at::kFloat) ||
      mean->numel() != rows || !plain(*rstd, dev, at::kFloat) || rstd->numel() != rows)
    Py_RETURN_NONE;
  at::Tensor gx, branch, gw, gb, gs;
  int rc;
  {
    Unlocked unlocked;
    const auto opts = x->options().requires_grad(false);
    const auto param = opts.dtype(w->scalar_type());
    gx = at::empty(x->sizes(), opts);
    if (pre && (s || branch_type != out)) branch = at::empty(x->sizes(), opts.dtype(branch_type));
    gw = at::empty(w->sizes(), param);
    gb = at::empty(b->sizes(), param);
    if (gamma) gs = at::empty(gamma->sizes(), param);
    const size_t bytes = g_workspace(code, rows, (int)C);
    at::Tensor ws = at::empty({(int64_t)bytes}, opts.dtype(at::kByte));
    void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    void* branch_ptr = branch.defined() ? branch.data_ptr() : nullptr;
    if (res)
      rc = g_seam_bwd(gy->data_ptr(), data(gh), x->data_ptr(), res->data_ptr(), mean->data_ptr<float>(), rstd->data_ptr<float>(),
                      w->data_ptr(), static_cast<const float*>(data(s)), gx.data_ptr(), branch_ptr, gw.data_ptr(),
                      gb.data_ptr(), ws.data_ptr(), bytes, code, code_of(w->scalar_type()), rows, (int)C, per, stream);
    else
      rc = g_bwd(gy->data_ptr(), pre ? data(gh) : nullptr, x->data_ptr(), mean->data_ptr<float>(), rstd->data_ptr<float>(),
                 w->data_ptr(), b->data_ptr(), data(gamma), static_cast<const float*>(data(s)), gx.data_ptr(), branch_ptr,
                 gw.data_ptr(), gb.data_ptr(), gs.defined() ? gs.data_ptr() : nullptr, ws.data_ptr(), bytes, mode, code,
                 code_of(out), code_of(w->scalar_type()), rows, (int)C, per, act, stream);
  }
  if (rc) return PyLong_FromLong(rc);
  PyObject* tuple = PyTuple_New(5);
  if (!tuple) return nullptr;
  PyObject* first = THPVariable_Wrap(std::move(gx));
  PyTuple_SET_ITEM(tuple, 0, first);
  if (branch.defined()) {
    PyTuple_SET_ITEM(tuple, 1, THPVariable_Wrap(std::move(branch)));
  } else {
    Py_INCREF(first);
    PyTuple_SET_ITEM(tuple, 1, first);
  }
  PyTuple_SET_ITEM(tuple, 2, THPVariable_Wrap(std::move(gw)));
  PyTuple_SET_ITEM(tuple, 3, THPVariable_Wrap(std::move(gb)));
  if (gs.defined()) {
    PyTuple_SET_ITEM(tuple, 4, THPVariable_Wrap(std::move(gs)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(tuple, 4, Py_None);
  }
  return tuple;
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"init", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_init)), METH_FASTCALL, nullptr},
    {"ln_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_forward)), METH_FASTCALL, nullptr},
    {"ln_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_backward)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "dcnv4_b200_bindings", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_dcnv4_b200_bindings(void) { return PyModule_Create(&kModule); }
