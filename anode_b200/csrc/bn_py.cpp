// Python side of the hot entry points: argument checks, tensor -> pointer, current stream and the C call in one
// native step.  A layer call through ctypes spent 12 - 20 us in the interpreter (one Python-level check per tensor,
// a stream object, twenty boxed arguments), several times the duration of the kernel on small layers; the same work
// here takes well under a microsecond.  The functions of the C ABI come in as addresses (bind), so this module is
// linked against nothing but Python and torch, and a library chosen at run time is honoured.
//
// Arguments mirror anode_b200/ops.py, which keeps the public signatures, defaults and error types.
// torch reports some conditions by C++ exceptions (no driver, a tensor without storage inside a function transform, a
// sparse one): every function turns them into Python errors (GUARDED), and nothing is asked of torch or CUDA once
// an argument was refused.
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <stdint.h>

#include <exception>

// Exceptions become Python errors by torch's own translation, which runs only when there is one: HANDLE_TH_ERRORS around
// every call would set up a buffer for C++ warnings each time.
namespace {
PyObject *translated(std::exception_ptr e)
{
  HANDLE_TH_ERRORS
  std::rethrow_exception(e);
  END_HANDLE_TH_ERRORS
}
}  // namespace
#define GUARDED try {
#define END_GUARDED } catch (...) { return translated(std::current_exception()); }

namespace {

struct KernelConfig { uint32_t block_sz, max_block_ct; };

// addresses of the C ABI, in the order of kNames
enum { F_FWD, F_FWD_ACT, F_FWD_ADD, F_BWD, F_BWD_ACT, F_BWD_ADD, F_INFER, F_NORMALIZE, F_ADJOINT,
       F_RMS_FWD, F_RMS_BWD, F_RMS_BWD_BYTES, F_RMS_QUANT, F_ROTARY_FWD, F_ROTARY_BWD, F_ROTARY_BWD_BYTES, F_COUNT };
const char *const kNames[F_COUNT] = {
    "anode_gpu_batch_norm_relu_fused_fwd_3d1_packed_f32", "anode_gpu_batch_norm_act_fused_fwd_3d1_packed_f32",
    "anode_gpu_batch_norm_add_act_fused_fwd_3d1_packed_f32", "anode_gpu_batch_norm_relu_fused_bwd_3d1_packed_f32",
    "anode_gpu_batch_norm_act_fused_bwd_3d1_packed_f32", "anode_gpu_batch_norm_add_act_fused_bwd_3d1_packed_f32",
    "anode_gpu_batch_norm_act_infer_3d1_packed_f32", "anode_gpu_batch_normalize_3d1_packed_f32",
    "anode_gpu_batch_normalize_adjoint_3d1_packed_f32", "anode_gpu_rms_norm_add_fwd", "anode_gpu_rms_norm_add_bwd",
    "anode_gpu_rms_norm_add_bwd_workspace_bytes", "anode_gpu_rms_norm_add_quant_fwd", "anode_gpu_rotary_positions_fwd",
    "anode_gpu_rotary_positions_bwd", "anode_gpu_rotary_positions_bwd_workspace_bytes"};
void *g_fn[F_COUNT] = {};

typedef const float *In;
typedef float *Out;
typedef int (*FwdFn)(uint32_t, uint32_t, uint32_t, float, float, int, In, In, In, Out, Out, Out, Out, Out, void *, size_t, const KernelConfig *, void *);
typedef int (*FwdActFn)(uint32_t, uint32_t, uint32_t, float, float, float, In, In, In, Out, Out, Out, Out, Out, void *, size_t, const KernelConfig *, void *);
typedef int (*FwdAddFn)(uint32_t, uint32_t, uint32_t, float, float, float, In, In, In, In, Out, Out, Out, Out, Out, void *, size_t, const KernelConfig *, void *);
typedef int (*BwdFn)(uint32_t, uint32_t, uint32_t, int, int, In, In, In, In, In, In, Out, Out, Out, void *, size_t, const KernelConfig *, void *);
typedef int (*BwdActFn)(uint32_t, uint32_t, uint32_t, float, int, In, In, In, In, In, In, Out, Out, Out, void *, size_t, const KernelConfig *, void *);
typedef int (*BwdAddFn)(uint32_t, uint32_t, uint32_t, float, int, In, In, In, In, In, In, In, Out, Out, Out, Out, void *, size_t, const KernelConfig *, void *);
typedef int (*InferFn)(uint32_t, uint32_t, uint32_t, float, In, In, In, In, In, Out, const KernelConfig *, void *);
typedef int (*NormalizeFn)(uint32_t, uint32_t, uint32_t, float, float, In, Out, Out, Out, Out, Out, const KernelConfig *, void *);
typedef int (*AdjointFn)(uint32_t, uint32_t, uint32_t, In, In, In, In, Out, Out, Out, const KernelConfig *, void *);

// The interpreter's lock is given back while this lives (exceptions included).
struct Unlocked {
  PyThreadState *state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// One call's arguments: the first failure sets the Python error and every later access does nothing.
struct Args {
  PyObject *const *v;
  bool ok = true;

  const at::Tensor *tensor(int i, bool null_ok)
  {
    if (!ok || (v[i] == Py_None && null_ok)) return nullptr;
    if (!THPVariable_Check(v[i])) {
      PyErr_SetString(PyExc_ValueError, "expected a contiguous float32 CUDA tensor");
      ok = false;
      return nullptr;
    }
    return &THPVariable_Unpack(v[i]);
  }
  // device pointer of a packed f32 array (the reference only implements packed arrays too, src/ops_gpu.rs:3777-3779)
  Out ptr(int i, bool null_ok = true)
  {
    const at::Tensor *t = tensor(i, null_ok);
    if (!t) return nullptr;
    if (!(t->is_cuda() && t->scalar_type() == at::kFloat && t->is_contiguous())) {
      PyErr_SetString(PyExc_ValueError, "expected a contiguous float32 CUDA tensor");
      ok = false;
      return nullptr;
    }
    return static_cast<float *>(t->data_ptr());
  }
  float f(int i)
  {
    if (!ok) return 0.f;
    const double d = PyFloat_AsDouble(v[i]);
    if (d == -1.0 && PyErr_Occurred()) ok = false;
    return (float)d;
  }
  int truth(int i)
  {
    if (!ok) return 0;
    const int r = PyObject_IsTrue(v[i]);
    if (r < 0) ok = false;
    return r > 0;
  }
  size_t size(int i)
  {
    if (!ok) return 0;
    const size_t r = PyLong_AsSize_t(v[i]);
    if (r == (size_t)-1 && PyErr_Occurred()) ok = false;
    return r;
  }
  void *raw(int i)
  {
    const at::Tensor *t = tensor(i, true);
    return t ? t->data_ptr() : nullptr;
  }
  // a torch stream, or None for the current one
  void *stream(int i)
  {
    if (!ok) return nullptr;
    if (v[i] == Py_None) return c10::cuda::getCurrentCUDAStream().stream();
    PyObject *h = PyObject_GetAttrString(v[i], "cuda_stream");
    if (!h) { ok = false; return nullptr; }
    void *p = PyLong_AsVoidPtr(h);
    Py_DECREF(h);
    if (PyErr_Occurred()) ok = false;
    return p;
  }
  // [N, C, *spatial] -> (dim0, dim1, dim2) as the apply closures compute them (src/ops_gpu.rs:3764-3766, :4911-4913);
  // `axes` (None: not checked) must be the positions of the spatial dimensions (src/ops_gpu.rs:3736)
  void dims(int axes, int i, uint32_t d[3])
  {
    const at::Tensor *t = tensor(i, false);
    if (!t) return;
    const int64_t nd = t->dim();
    if (axes >= 0 && v[axes] != Py_None) {
      // any iterable whose items equal 0, 1, ...; the usual list of integers without making another one
      bool usual = PyList_CheckExact(v[axes]) && PyList_GET_SIZE(v[axes]) == (nd > 2 ? nd - 2 : 0);
      for (Py_ssize_t k = 0; usual && k + 2 < nd; ++k) {
        PyObject *e = PyList_GET_ITEM(v[axes], k);
        usual = PyLong_CheckExact(e) && PyLong_AsLong(e) == (long)k;
        if (PyErr_Occurred()) PyErr_Clear();      // (an integer beyond a long)
      }
      PyObject *got = usual ? nullptr : PySequence_List(v[axes]), *want = got ? PyList_New(0) : nullptr;
      int same = usual ? 2 : want ? 1 : -1;
      for (int64_t k = 0; same == 1 && k + 2 < nd; ++k) {
        PyObject *e = PyLong_FromLongLong(k);
        if (!e || PyList_Append(want, e)) same = -1;
        Py_XDECREF(e);
      }
      if (same == 1) same = PyObject_RichCompareBool(got, want, Py_EQ);
      if (same == 0) PyErr_Format(PyExc_ValueError, "axes must be %R for a %d-D batch array", want, (int)(nd - 2));
      Py_XDECREF(got); Py_XDECREF(want);
      if (same <= 0) { ok = false; return; }
    }
    if (nd < 2) { PyErr_SetString(PyExc_IndexError, "expected an array [N, C, *spatial]"); ok = false; return; }
    uint64_t d0 = 1;
    for (int64_t k = 2; k < nd; ++k) d0 *= (uint64_t)t->size(k);
    d[0] = (uint32_t)d0; d[1] = (uint32_t)t->size(1); d[2] = (uint32_t)t->size(0);
  }
};

bool want_args(Py_ssize_t n, Py_ssize_t want)
{
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}
bool bound(int which)
{
  if (g_fn[which]) return true;
  PyErr_SetString(PyExc_ImportError, "the CUDA library is not loaded");
  return false;
}
const KernelConfig kDefaultCfg = {1024, 148 * 32};     // ops.py's default launch hint (the kernels choose their own shapes)

// fwd(axes, epsilon, avg_rate, x, residual, y, mean, var, avg_mean, avg_var, gamma, beta, relu, neg_slope | None, ws, ws_bytes, stream)
PyObject *py_fwd(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 17)) return nullptr;
  Args a{v};
  uint32_t d[3] = {0, 0, 0};
  a.dims(0, 3, d);
  const float eps = a.f(1), rate = a.f(2);
  const bool add = v[4] != Py_None, act = add || v[13] != Py_None;
  const float slope = act ? a.f(13) : 0.f;      // (the residual epilogue always has one: None is refused)
  In x = a.ptr(3), res = a.ptr(4), gamma = a.ptr(10), beta = a.ptr(11);
  Out y = a.ptr(5), mean = a.ptr(6), var = a.ptr(7), rm = a.ptr(8), rv = a.ptr(9);
  const int relu = a.truth(12);
  void *ws = a.raw(14);
  const size_t bytes = a.size(15);
  void *s = a.stream(16);
  if (!a.ok) return nullptr;
  const int which = add ? F_FWD_ADD : act ? F_FWD_ACT : F_FWD;
  if (!bound(which)) return nullptr;
  int rc;
  {
    Unlocked unlocked;
    if (add) rc = ((FwdAddFn)g_fn[which])(d[0], d[1], d[2], eps, rate, slope, x, res, gamma, beta, y, mean, var, rm, rv, ws, bytes, &kDefaultCfg, s);
    else if (act) rc = ((FwdActFn)g_fn[which])(d[0], d[1], d[2], eps, rate, slope, x, gamma, beta, y, mean, var, rm, rv, ws, bytes, &kDefaultCfg, s);
    else rc = ((FwdFn)g_fn[which])(d[0], d[1], d[2], eps, rate, relu, x, gamma, beta, y, mean, var, rm, rv, ws, bytes, &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// bwd(axes, dy, x, y | None, mean, var, dx, dresidual, gamma, beta, dgamma, dbeta, relu, neg_slope | None, accumulate, ws, ws_bytes, stream)
PyObject *py_bwd(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 18)) return nullptr;
  Args a{v};
  uint32_t d[3] = {0, 0, 0};
  a.dims(0, 2, d);
  const bool add = v[3] != Py_None, act = add || v[13] != Py_None;
  const float slope = act ? a.f(13) : 0.f;      // (the residual epilogue always has one: None is refused)
  In dy = a.ptr(1), x = a.ptr(2), y = a.ptr(3), mean = a.ptr(4), var = a.ptr(5), gamma = a.ptr(8), beta = a.ptr(9);
  Out dx = a.ptr(6), dres = a.ptr(7), dg = a.ptr(10), db = a.ptr(11);
  const int relu = a.truth(12), acc = a.truth(14);
  void *ws = a.raw(15);
  const size_t bytes = a.size(16);
  void *s = a.stream(17);
  if (!a.ok) return nullptr;
  const int which = add ? F_BWD_ADD : act ? F_BWD_ACT : F_BWD;
  if (!bound(which)) return nullptr;
  int rc;
  {
    Unlocked unlocked;
    if (add) rc = ((BwdAddFn)g_fn[which])(d[0], d[1], d[2], slope, acc, dy, x, y, mean, var, gamma, beta, dx, dres, dg, db, ws, bytes, &kDefaultCfg, s);
    else if (act) rc = ((BwdActFn)g_fn[which])(d[0], d[1], d[2], slope, acc, dy, x, mean, var, gamma, beta, dx, dg, db, ws, bytes, &kDefaultCfg, s);
    else rc = ((BwdFn)g_fn[which])(d[0], d[1], d[2], relu, acc, dy, x, mean, var, gamma, beta, dx, dg, db, ws, bytes, &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// infer(axes, x, mean, var, y, gamma, beta, neg_slope, stream)
PyObject *py_infer(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 9)) return nullptr;
  Args a{v};
  uint32_t d[3] = {0, 0, 0};
  a.dims(0, 1, d);
  const float slope = a.f(7);
  In x = a.ptr(1), mean = a.ptr(2), var = a.ptr(3), gamma = a.ptr(5), beta = a.ptr(6);
  Out y = a.ptr(4);
  void *s = a.stream(8);
  if (!a.ok || !bound(F_INFER)) return nullptr;
  int rc;
  {
    Unlocked unlocked;
    rc = ((InferFn)g_fn[F_INFER])(d[0], d[1], d[2], slope, x, mean, var, gamma, beta, y, &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// The outputs of the front end's composition are made here: three tensors through the interpreter took longer than the call.
at::Tensor like(const at::Tensor &x) { return at::empty_like(x); }
at::Tensor per_channel(const at::Tensor &x) { return at::empty({x.size(1)}, x.options()); }
Out data(const at::Tensor &t) { return static_cast<float *>(t.data_ptr()); }
// (status, a, b, c)
PyObject *answer(int rc, const at::Tensor &a, const at::Tensor &b, const at::Tensor &c)
{
  PyObject *t = PyTuple_New(4), *items[4] = {PyLong_FromLong(rc), THPVariable_Wrap(a), THPVariable_Wrap(b), THPVariable_Wrap(c)};
  bool ok = t != nullptr;
  for (int i = 0; i < 4; ++i) {
    ok = ok && items[i];
    if (t) PyTuple_SET_ITEM(t, i, items[i]); else Py_XDECREF(items[i]);
  }
  if (ok) return t;
  Py_XDECREF(t);
  return nullptr;
}

// normalize(axes, epsilon, avg_rate, x, avg_mean, avg_var, stream) -> status, y, mean, var
PyObject *py_normalize(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 7)) return nullptr;
  Args a{v};
  uint32_t d[3] = {0, 0, 0};
  a.dims(0, 3, d);
  const float eps = a.f(1), rate = a.f(2);
  In x = a.ptr(3, false);
  Out rm = a.ptr(4, false), rv = a.ptr(5, false);
  void *s = a.stream(6);
  if (!a.ok || !bound(F_NORMALIZE)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(v[3]);
  const at::Tensor mean = per_channel(t), var = per_channel(t), y = like(t);
  int rc;
  {
    Unlocked unlocked;
    rc = ((NormalizeFn)g_fn[F_NORMALIZE])(d[0], d[1], d[2], eps, rate, x, data(y), data(mean), data(var), rm, rv, &kDefaultCfg, s);
  }
  return answer(rc, y, mean, var);
  END_GUARDED
}

// adjoint(axes, dy, x, mean, var, stream) -> status, dx, dmean, dvar
PyObject *py_adjoint(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 6)) return nullptr;
  Args a{v};
  uint32_t d[3] = {0, 0, 0};
  a.dims(0, 2, d);
  In dy = a.ptr(1, false), x = a.ptr(2, false), mean = a.ptr(3, false), var = a.ptr(4, false);
  void *s = a.stream(5);
  if (!a.ok || !bound(F_ADJOINT)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(v[2]);
  const at::Tensor dvar = per_channel(t), dmean = per_channel(t), dx = like(t);
  int rc;
  {
    Unlocked unlocked;
    rc = ((AdjointFn)g_fn[F_ADJOINT])(d[0], d[1], d[2], dy, x, mean, var, data(dx), data(dmean), data(dvar), &kDefaultCfg, s);
  }
  return answer(rc, dx, dmean, dvar);
  END_GUARDED
}

// The tensors of one of the reference's own entry points: `lo` to `hi` of them, all required (these entry points have no
// status, and their kernels read and write what they are given).
struct Pointers {
  void *p[5] = {};
  Py_ssize_t k = 0;

  bool take(PyObject *tuple, Py_ssize_t lo, Py_ssize_t hi)
  {
    if (!PyTuple_Check(tuple)) { PyErr_SetString(PyExc_TypeError, "tensors: a tuple"); return false; }
    k = PyTuple_GET_SIZE(tuple);
    if (k < lo || k > hi) { PyErr_Format(PyExc_TypeError, "%zd to %zd tensors", lo, hi); return false; }
    PyObject *items[5];
    for (Py_ssize_t i = 0; i < k; ++i) items[i] = PyTuple_GET_ITEM(tuple, i);
    Args t{items};
    for (Py_ssize_t i = 0; i < k; ++i) {
      p[i] = t.ptr((int)i, false);
      if (t.ok && !p[i] && THPVariable_Unpack(items[i]).numel() != 0) {
        PyErr_SetString(PyExc_RuntimeError, "a tensor has no storage");
        t.ok = false;
      }
    }
    return t.ok;
  }
};
typedef void *P;
typedef const KernelConfig *K;

// The form of the C call is the function's, never read off the arguments' values.
// flat(address, tensors, stream): element count (of the first tensor) and 2 or 3 arrays
PyObject *py_flat(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 3)) return nullptr;
  void *fn = PyLong_AsVoidPtr(v[0]);
  if (PyErr_Occurred()) return nullptr;
  Args a{v};
  Pointers q;
  if (!q.take(v[1], 2, 3)) return nullptr;
  const uint32_t len = (uint32_t)THPVariable_Unpack(PyTuple_GET_ITEM(v[1], 0)).numel();
  void *s = a.stream(2);
  if (!a.ok) return nullptr;
  const KernelConfig *cfg = &kDefaultCfg;
  {
    Unlocked unlocked;
    if (q.k == 2) ((void (*)(uint32_t, P, P, K, P))fn)(len, q.p[0], q.p[1], cfg, s);
    else ((void (*)(uint32_t, P, P, P, K, P))fn)(len, q.p[0], q.p[1], q.p[2], cfg, s);
  }
  Py_RETURN_NONE;
  END_GUARDED
}

// packed(address, axes, like, tensors, stream): the dimensions of `like` and 2 to 5 arrays
PyObject *py_packed(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 5)) return nullptr;
  void *fn = PyLong_AsVoidPtr(v[0]);
  if (PyErr_Occurred()) return nullptr;
  Args a{v};
  uint32_t d[3] = {0, 0, 0};
  a.dims(1, 2, d);
  Pointers q;
  if (!a.ok || !q.take(v[3], 2, 5)) return nullptr;
  void *s = a.stream(4);
  if (!a.ok) return nullptr;
  const KernelConfig *cfg = &kDefaultCfg;
  {
    Unlocked unlocked;
    if (q.k == 2) ((void (*)(uint32_t, uint32_t, uint32_t, P, P, K, P))fn)(d[0], d[1], d[2], q.p[0], q.p[1], cfg, s);
    else if (q.k == 3) ((void (*)(uint32_t, uint32_t, uint32_t, P, P, P, K, P))fn)(d[0], d[1], d[2], q.p[0], q.p[1], q.p[2], cfg, s);
    else if (q.k == 4) ((void (*)(uint32_t, uint32_t, uint32_t, P, P, P, P, K, P))fn)(d[0], d[1], d[2], q.p[0], q.p[1], q.p[2], q.p[3], cfg, s);
    else ((void (*)(uint32_t, uint32_t, uint32_t, P, P, P, P, P, K, P))fn)(d[0], d[1], d[2], q.p[0], q.p[1], q.p[2], q.p[3], q.p[4], cfg, s);
  }
  Py_RETURN_NONE;
  END_GUARDED
}

// packed_eps(address, axes, like, tensors, epsilon, stream): the dimensions of `like`, epsilon and 3 arrays
PyObject *py_packed_eps(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 6)) return nullptr;
  void *fn = PyLong_AsVoidPtr(v[0]);
  if (PyErr_Occurred()) return nullptr;
  Args a{v};
  uint32_t d[3] = {0, 0, 0};
  a.dims(1, 2, d);
  const float eps = a.f(4);
  Pointers q;
  if (!a.ok || !q.take(v[3], 3, 3)) return nullptr;
  void *s = a.stream(5);
  if (!a.ok) return nullptr;
  {
    Unlocked unlocked;
    ((void (*)(uint32_t, uint32_t, uint32_t, float, P, P, P, K, P))fn)(d[0], d[1], d[2], eps, q.p[0], q.p[1], q.p[2], &kDefaultCfg, s);
  }
  Py_RETURN_NONE;
  END_GUARDED
}

// ---- row-wise operators: any of three element types, rows and heads at strides, everything on one device -----------------------

struct AnodeHeads { void *data; uint64_t batch_stride, seq_stride, head_stride; uint32_t heads; };
typedef const void *CV;
typedef uint64_t U8;
typedef int (*RmsFwdFn)(int, U8, uint32_t, float, CV, U8, CV, U8, CV, int, P, U8, P, U8, float *, K, P);
typedef int (*RmsBwdFn)(int, U8, uint32_t, CV, U8, CV, U8, const float *, CV, int, CV, U8, P, U8, P, P, size_t, K, P);
typedef size_t (*RmsBytesFn)(U8, uint32_t);
typedef int (*RmsQuantFn)(int, U8, uint32_t, float, uint32_t, CV, U8, CV, U8, CV, int, P, U8, float *, U8, U8, P, U8, K, P);
typedef const AnodeHeads *H;
typedef int (*RotaryFwdFn)(int, uint32_t, uint32_t, uint32_t, uint32_t, int, float, const double *, CV, int, U8, U8, int, float, CV, CV, int, H, H, H, H, K, P);
typedef int (*RotaryBwdFn)(int, uint32_t, uint32_t, uint32_t, uint32_t, int, float, const double *, CV, int, U8, U8, int, float, CV, CV, int, H, H, H, H, H, H,
                           P, P, P, size_t, K, P);
typedef size_t (*RotaryBytesFn)(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t);

int type_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1; }

// The arguments of a row-wise operator: the first failure sets the Python error and every later access does nothing.
struct RowArgs {
  PyObject *const *v;
  const char *const *name;
  bool ok = true;
  int device = -1;                       // of the first tensor
  int missing = -1;                      // a tensor without storage

  bool fail(int i, const char *what)
  {
    if (ok) PyErr_Format(PyExc_ValueError, "%s: %s", name[i], what);
    ok = false;
    return false;
  }
  const at::Tensor *tensor(int i, bool null_ok)
  {
    if (!ok || (v[i] == Py_None && null_ok)) return nullptr;
    if (!THPVariable_Check(v[i])) { fail(i, "expected a CUDA tensor"); return nullptr; }
    const at::Tensor *t = &THPVariable_Unpack(v[i]);
    if (!t->is_cuda() || t->layout() != at::kStrided) { fail(i, "expected a CUDA tensor"); return nullptr; }
    if (device < 0) device = t->get_device();
    if (t->get_device() != device) { fail(i, "on another device than the first tensor"); return nullptr; }
    return t;
  }
  bool given(int i) const { return v[i] != Py_None; }
  // one of the three element types, as a code
  int type(int i, const at::Tensor &t)
  {
    const int c = type_code(t.scalar_type());
    if (c < 0) fail(i, "expected float32, float16 or bfloat16");
    return c;
  }
  void *data(int i, const at::Tensor &t)
  {
    void *p = t.data_ptr();
    if (!p && t.numel() && missing < 0) missing = i;      // (refused once the arguments' sizes and types are known to be right)
    return p;
  }
  // the leading `lead` dimensions as rows at one distance
  bool collapse(int i, const at::Tensor &t, int64_t lead, U8 &rows, U8 &stride)
  {
    rows = 1; stride = 0;
    bool first = true;
    for (int64_t d = 0; d < lead; ++d)
      if (t.size(d) == 0) { rows = 0; return true; }
    for (int64_t d = lead - 1; d >= 0; --d) {
      const int64_t n = t.size(d);
      if (n == 1) continue;
      if (first) { stride = (U8)t.stride(d); first = false; }
      else if ((U8)t.stride(d) != stride * rows) return fail(i, "its rows do not lie at one distance");
      rows *= (U8)n;
    }
    if (first && lead) stride = (U8)t.size(t.dim() - 1);
    return true;
  }
  // [*, cols] of packed rows; of `like`'s sizes where that is given, and of its type unless `any_type`
  void *rows(int i, const at::Tensor *like, U8 &stride, bool null_ok = false, at::ScalarType as = at::ScalarType::Undefined)
  {
    stride = 0;
    const at::Tensor *t = tensor(i, null_ok);
    if (!t) return nullptr;
    if (t->dim() < 1) { fail(i, "expected an array [*, cols]"); return nullptr; }
    if (like && t->sizes() != like->sizes()) { fail(i, "has other sizes than the first tensor"); return nullptr; }
    const at::ScalarType want = as != at::ScalarType::Undefined ? as : like ? like->scalar_type() : t->scalar_type();
    if (t->scalar_type() != want) { fail(i, "has another type than this operator takes beside the first tensor's"); return nullptr; }
    if (t->size(t->dim() - 1) > 1 && t->stride(t->dim() - 1) != 1) { fail(i, "its last dimension is not packed"); return nullptr; }
    U8 n;
    if (!collapse(i, *t, t->dim() - 1, n, stride)) return nullptr;
    return data(i, *t);
  }
  // a packed vector of n weights of any of the three types
  void *weights(int i, int64_t n, int &code, bool null_ok = true)
  {
    const at::Tensor *t = tensor(i, null_ok);
    if (!t) return nullptr;
    const int c = type(i, *t);
    if (c < 0) return nullptr;
    if (t->numel() != n || !t->is_contiguous()) { fail(i, "expected a packed vector, one weight per column"); return nullptr; }
    if (code >= 0 && code != c) { fail(i, "has another type than the other weights"); return nullptr; }
    code = c;
    return data(i, *t);
  }
  // a packed array of n elements of one type
  void *packed(int i, at::ScalarType as, int64_t n, const char *what, bool null_ok)
  {
    const at::Tensor *t = tensor(i, null_ok);
    if (!t) return nullptr;
    if (t->scalar_type() != as || t->numel() != n || !t->is_contiguous()) { fail(i, what); return nullptr; }
    return data(i, *t);
  }
  double f(int i)
  {
    if (!ok) return 0.;
    const double d = PyFloat_AsDouble(v[i]);
    if (d == -1.0 && PyErr_Occurred()) ok = false;
    return d;
  }
  int truth(int i)
  {
    if (!ok) return 0;
    const int r = PyObject_IsTrue(v[i]);
    if (r < 0) ok = false;
    return r > 0;
  }
  // a torch stream of the tensors' device, or None for that device's current one
  void *stream(int i)
  {
    if (ok && missing >= 0) fail(missing, "has no storage");
    if (!ok) return nullptr;
    if (v[i] == Py_None) return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    PyObject *h = PyObject_GetAttrString(v[i], "cuda_stream"), *d = h ? PyObject_GetAttrString(v[i], "device_index") : nullptr;
    void *p = h ? PyLong_AsVoidPtr(h) : nullptr;
    const long at = d ? PyLong_AsLong(d) : -1;
    Py_XDECREF(h); Py_XDECREF(d);
    if (PyErr_Occurred()) { ok = false; return nullptr; }
    if (at != device) fail(i, "belongs to another device than the tensors");
    return p;
  }
  // the call's workspace: the caller's, or one of `bytes` that belongs to the call's stream
  void *workspace(int i, int stream_at, void *s, size_t &bytes, at::Tensor &own)
  {
    if (!ok || bytes == 0) return nullptr;
    if (v[i] != Py_None) {
      const at::Tensor *t = tensor(i, false);
      if (!t) return nullptr;
      if (!t->is_contiguous()) { fail(i, "expected a packed array"); return nullptr; }
      bytes = t->nbytes();
      return data(i, *t);
    }
    const auto options = at::TensorOptions().dtype(at::kByte).device(at::kCUDA, (c10::DeviceIndex)device);
    if (v[stream_at] == Py_None) own = at::empty({(int64_t)bytes}, options);
    else {
      const c10::cuda::CUDAStreamGuard guard(c10::cuda::getStreamFromExternal((cudaStream_t)s, (c10::DeviceIndex)device));
      own = at::empty({(int64_t)bytes}, options);
    }
    return own.data_ptr();
  }
};
bool cols_of(RowArgs &a, int i, const at::Tensor &t, U8 &rows, uint32_t &cols)
{
  U8 stride;
  const int64_t c = t.size(t.dim() - 1);
  if (c > 0x7fffffffll) return a.fail(i, "too many columns");
  cols = (uint32_t)c;
  return a.collapse(i, t, t.dim() - 1, rows, stride);
}

// rms_fwd(epsilon, x, y, gamma, residual, total, inv_rms, stream)
PyObject *py_rms_fwd(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 8)) return nullptr;
  static const char *const names[] = {"epsilon", "x", "y", "gamma", "residual", "total", "inv_rms", "stream"};
  RowArgs a{v, names};
  U8 rows = 0, sx, sy, sr, st;
  uint32_t cols = 0;
  const double eps = a.f(0);
  CV x = a.rows(1, nullptr, sx);
  if (!a.ok) return nullptr;
  const at::Tensor &like = THPVariable_Unpack(v[1]);
  const int type = a.type(1, like);
  int gt = -1;
  if (!a.ok || !cols_of(a, 1, like, rows, cols)) return nullptr;
  P y = a.rows(2, &like, sy);
  CV g = a.weights(3, cols, gt), r = a.rows(4, &like, sr, true);
  P t = a.rows(5, &like, st, true);
  if (a.ok && a.given(5) && !a.given(4)) a.fail(5, "is the sum with a residual: without one it would be a copy of x");
  float *inv = (float *)a.packed(6, at::kFloat, (int64_t)rows, "expected a packed float32 array, one value per row", true);
  void *s = a.stream(7);
  if (!a.ok || !bound(F_RMS_FWD)) return nullptr;
  const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)a.device));
  int rc;
  {
    Unlocked unlocked;
    rc = ((RmsFwdFn)g_fn[F_RMS_FWD])(type, rows, cols, (float)eps, x, sx, r, sr, g, gt, y, sy, t, st, inv, &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// rms_bwd(dy, total, inv_rms, dx, gamma, dtotal, dgamma, accumulate, workspace, stream)
PyObject *py_rms_bwd(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 10)) return nullptr;
  static const char *const names[] = {"dy", "total", "inv_rms", "dx", "gamma", "dtotal", "dgamma", "cap", "workspace", "stream"};
  RowArgs a{v, names};
  U8 rows = 0, sy, st, sx, sd;
  uint32_t cols = 0;
  CV dy = a.rows(0, nullptr, sy);
  if (!a.ok) return nullptr;
  const at::Tensor &like = THPVariable_Unpack(v[0]);
  const int type = a.type(0, like);
  int gt = -1;
  if (!a.ok || !cols_of(a, 0, like, rows, cols)) return nullptr;
  CV t = a.rows(1, &like, st);
  const float *inv = (const float *)a.packed(2, at::kFloat, (int64_t)rows, "expected a packed float32 array, one value per row", false);
  P dx = a.rows(3, &like, sx);
  CV g = a.weights(4, cols, gt), dt = a.rows(5, &like, sd, true);
  P dg = a.weights(6, cols, gt);
  if (a.truth(7)) {
    if (a.ok && a.given(5)) a.fail(7, "Accumulate adds into dx, which takes the place of dtotal: give one of them");
    dt = dx; sd = sx;
  }
  void *s = a.stream(9);
  if (!a.ok || !bound(F_RMS_BWD) || !bound(F_RMS_BWD_BYTES)) return nullptr;
  const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)a.device));
  size_t bytes = dg ? ((RmsBytesFn)g_fn[F_RMS_BWD_BYTES])(rows, cols) : 0;
  at::Tensor own;
  void *ws = a.workspace(8, 9, s, bytes, own);
  if (!a.ok) return nullptr;
  int rc;
  {
    Unlocked unlocked;
    rc = ((RmsBwdFn)g_fn[F_RMS_BWD])(type, rows, cols, dy, sy, t, st, inv, g, gt, dt, sd, dx, sx, dg, ws, bytes, &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// rms_quant(epsilon, x, q, scale, gamma, residual, total, stream)
PyObject *py_rms_quant(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 8)) return nullptr;
  static const char *const names[] = {"epsilon", "x", "q", "scale", "gamma", "residual", "total", "stream"};
  RowArgs a{v, names};
  U8 rows = 0, sx, sq, sr, st, scale_rows = 0, scale_row = 0, scale_group = 0;
  uint32_t cols = 0, block = 0;
  const double eps = a.f(0);
  CV x = a.rows(1, nullptr, sx);
  if (!a.ok) return nullptr;
  const at::Tensor &like = THPVariable_Unpack(v[1]);
  const int type = a.type(1, like);
  int gt = -1;
  if (!a.ok || !cols_of(a, 1, like, rows, cols)) return nullptr;
  P q = a.rows(2, &like, sq, false, at::kFloat8_e4m3fn);
  const at::Tensor *scale = a.tensor(3, false);
  if (!a.ok) return nullptr;
  // [*] of x's rows, or [*, groups]
  const int64_t lead = like.dim() - 1;
  bool fits = scale->scalar_type() == at::kFloat && (scale->dim() == lead || scale->dim() == lead + 1);
  for (int64_t d = 0; fits && d < lead; ++d) fits = scale->size(d) == like.size(d);
  if (fits && scale->dim() == lead + 1) {
    block = 128;
    fits = scale->size(lead) == ((int64_t)cols + 127) / 128;
    scale_group = (U8)scale->stride(lead);
  }
  if (!fits) { a.fail(3, "expected float32, one per row or one per 128 columns of a row"); return nullptr; }
  if (!a.collapse(3, *scale, lead, scale_rows, scale_row)) return nullptr;
  void *sc = a.data(3, *scale);
  CV g = a.weights(4, cols, gt), r = a.rows(5, &like, sr, true);
  P t = a.rows(6, &like, st, true);
  if (a.ok && a.given(6) && !a.given(5)) a.fail(6, "is the sum with a residual: without one it would be a copy of x");
  void *s = a.stream(7);
  if (!a.ok || !bound(F_RMS_QUANT)) return nullptr;
  const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)a.device));
  int rc;
  {
    Unlocked unlocked;
    rc = ((RmsQuantFn)g_fn[F_RMS_QUANT])(type, rows, cols, (float)eps, block, x, sx, r, sr, g, gt, q, sq, (float *)sc, scale_row, scale_group, t, st,
                                         &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// What both directions of the rotary positions begin with: [tokens, heads, dim] or [batch, seq, heads, dim] arrays.
struct RotaryHeads {
  RowArgs &a;
  int type = -1;
  int64_t batch = 0, seq = 0, dim = 0;

  // array i into h; of the first one's batch, seq, dim and type, and of `heads` heads where that is not negative
  bool take(int i, AnodeHeads &h, int64_t heads, bool null_ok)
  {
    const at::Tensor *t = a.tensor(i, null_ok);
    if (!t) return false;
    const int64_t nd = t->dim();
    if (nd != 3 && nd != 4) return a.fail(i, "expected [tokens, heads, dim] or [batch, seq, heads, dim]");
    const int64_t b = nd == 4 ? t->size(0) : 1, s = t->size(nd - 3), n = t->size(nd - 2), d = t->size(nd - 1);
    const int c = a.type(i, *t);
    if (c < 0) return false;
    if (type < 0) { type = c; batch = b; seq = s; dim = d; dims = nd; }
    if (c != type) return a.fail(i, "has another type than the first array");
    if (nd != dims || b != batch || s != seq || d != dim) return a.fail(i, "has other sizes than the first array");
    if (heads >= 0 && n != heads) return a.fail(i, "has another number of heads than its input");
    if (batch > 0xffffffffll || seq > 0xffffffffll || n > 0xffffffffll || dim > 0xffffffffll) return a.fail(i, "too large");
    if (d > 1 && t->stride(nd - 1) != 1) return a.fail(i, "its last dimension is not packed");
    h = AnodeHeads{a.data(i, *t), nd == 4 ? (U8)t->stride(0) : 0, (U8)t->stride(nd - 3), (U8)t->stride(nd - 2), (uint32_t)n};
    return a.ok;
  }
  int64_t dims = 0;
  // [tokens], [batch, seq] or [seq] of 32- or 64-bit integers
  CV positions(int i, int &bytes, U8 &batch_stride, U8 &seq_stride)
  {
    const at::Tensor *t = a.tensor(i, false);
    if (!t) return nullptr;
    const bool each = dims == 4 && t->dim() == 2;
    if ((t->scalar_type() != at::kLong && t->scalar_type() != at::kInt) || !(t->dim() == 1 || each) || t->size(t->dim() - 1) != seq || (each && t->size(0) != batch)) {
      a.fail(i, "expected int32 or int64, one position per token");
      return nullptr;
    }
    bytes = t->scalar_type() == at::kLong ? 8 : 4;
    batch_stride = each ? (U8)t->stride(0) : 0;
    seq_stride = (U8)t->stride(t->dim() - 1);
    return a.data(i, *t);
  }
  const double *freq(int i, uint32_t &rot)
  {
    const at::Tensor *t = a.tensor(i, false);
    if (!t) return nullptr;
    if (t->scalar_type() != at::kDouble || t->dim() != 1 || !t->is_contiguous() || t->numel() > 0x3fffffff) {
      a.fail(i, "expected a packed float64 vector, one frequency per pair");
      return nullptr;
    }
    rot = 2 * (uint32_t)t->numel();
    return (const double *)a.data(i, *t);
  }
};

// rotary_fwd(positions, freq, q, k, q_out, k_out, interleaved, amplitude, epsilon | None, gamma_q, gamma_k, stream)
PyObject *py_rotary_fwd(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 12)) return nullptr;
  static const char *const names[] = {"positions", "freq", "q", "k", "q_out", "k_out", "interleaved", "amplitude", "epsilon", "gamma_q", "gamma_k", "stream"};
  RowArgs a{v, names};
  RotaryHeads r{a};
  AnodeHeads q, k, qo, ko;
  if (!r.take(2, q, -1, false)) return nullptr;
  const bool two = r.take(3, k, -1, true);
  if (!a.ok || !r.take(4, qo, q.heads, false)) return nullptr;
  if (two != (v[5] != Py_None)) { a.fail(5, "k and k_out are given together"); return nullptr; }
  if (two && !r.take(5, ko, k.heads, false)) return nullptr;
  int bytes = 0, gt = -1;
  U8 pb = 0, ps = 0;
  uint32_t rot = 0;
  CV positions = r.positions(0, bytes, pb, ps);
  const double *freq = r.freq(1, rot);
  const int interleaved = a.truth(6);
  const double amplitude = a.f(7);
  const bool norm = v[8] != Py_None;
  const double eps = norm ? a.f(8) : 0.0;
  CV gq = a.weights(9, r.dim, gt), gk = a.weights(10, r.dim, gt);
  if (a.ok && !norm && (a.given(9) || a.given(10))) a.fail(a.given(9) ? 9 : 10, "is the norm's weight, and epsilon=None means no norm");
  void *s = a.stream(11);
  if (!a.ok || !bound(F_ROTARY_FWD)) return nullptr;
  const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)a.device));
  int rc;
  {
    Unlocked unlocked;
    rc = ((RotaryFwdFn)g_fn[F_ROTARY_FWD])(r.type, (uint32_t)r.batch, (uint32_t)r.seq, (uint32_t)r.dim, rot, interleaved, (float)amplitude, freq, positions,
                                           bytes, pb, ps, norm, (float)eps, gq, gk, gt, &q, two ? &k : nullptr, &qo, two ? &ko : nullptr, &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// rotary_bwd(positions, freq, dq_out, dk_out, dq, dk, interleaved, amplitude, epsilon | None, q, k, gamma_q, gamma_k, dgamma_q, dgamma_k, workspace, stream)
PyObject *py_rotary_bwd(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 17)) return nullptr;
  static const char *const names[] = {"positions", "freq", "dq_out", "dk_out", "dq", "dk", "interleaved", "amplitude", "epsilon", "q", "k", "gamma_q", "gamma_k",
                                      "dgamma_q", "dgamma_k", "workspace", "stream"};
  RowArgs a{v, names};
  RotaryHeads r{a};
  AnodeHeads dqo, dko, dq, dk, q, k;
  if (!r.take(2, dqo, -1, false)) return nullptr;
  const bool two = r.take(3, dko, -1, true);
  if (!a.ok || !r.take(4, dq, dqo.heads, false)) return nullptr;
  if (two != (v[5] != Py_None)) { a.fail(5, "dk_out and dk are given together"); return nullptr; }
  if (two && !r.take(5, dk, dko.heads, false)) return nullptr;
  int bytes = 0, gt = -1;
  U8 pb = 0, ps = 0;
  uint32_t rot = 0;
  CV positions = r.positions(0, bytes, pb, ps);
  const double *freq = r.freq(1, rot);
  const int interleaved = a.truth(6);
  const double amplitude = a.f(7);
  const bool norm = v[8] != Py_None;
  const double eps = norm ? a.f(8) : 0.0;
  if (!a.ok) return nullptr;
  if (norm) {
    if (!r.take(9, q, dqo.heads, false) || (two && !r.take(10, k, dko.heads, false))) return nullptr;
  }
  CV gq = a.weights(11, r.dim, gt), gk = a.weights(12, r.dim, gt);
  P dgq = a.weights(13, r.dim, gt), dgk = a.weights(14, r.dim, gt);
  for (int i = 11; i < 15; ++i)
    if (a.ok && !norm && a.given(i)) a.fail(i, "belongs to the norm's weight, and epsilon=None means no norm");
  if (a.ok && !two && a.given(14)) a.fail(14, "there are no keys");
  void *s = a.stream(16);
  if (!a.ok || !bound(F_ROTARY_BWD) || !bound(F_ROTARY_BWD_BYTES)) return nullptr;
  const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)a.device));
  size_t need = dgq || dgk ? ((RotaryBytesFn)g_fn[F_ROTARY_BWD_BYTES])((uint32_t)r.batch, (uint32_t)r.seq, dqo.heads, two ? dko.heads : 0, (uint32_t)r.dim) : 0;
  at::Tensor own;
  void *ws = a.workspace(15, 16, s, need, own);
  if (!a.ok) return nullptr;
  int rc;
  {
    Unlocked unlocked;
    rc = ((RotaryBwdFn)g_fn[F_ROTARY_BWD])(r.type, (uint32_t)r.batch, (uint32_t)r.seq, (uint32_t)r.dim, rot, interleaved, (float)amplitude, freq, positions,
                                           bytes, pb, ps, norm, (float)eps, gq, gk, gt, &dqo, two ? &dko : nullptr, norm ? &q : nullptr,
                                           norm && two ? &k : nullptr, &dq, two ? &dk : nullptr, dgq, dgk, ws, need, &kDefaultCfg, s);
  }
  return PyLong_FromLong(rc);
  END_GUARDED
}

// bind({name: address}): the C ABI's functions
PyObject *py_bind(PyObject *, PyObject *const *v, Py_ssize_t n)
{
  GUARDED
  if (!want_args(n, 1)) return nullptr;
  for (int i = 0; i < F_COUNT; ++i) {
    PyObject *e = PyDict_GetItemString(v[0], kNames[i]);
    if (!e) { PyErr_Format(PyExc_KeyError, "%s", kNames[i]); return nullptr; }
    g_fn[i] = PyLong_AsVoidPtr(e);
    if (PyErr_Occurred()) return nullptr;
  }
  Py_RETURN_NONE;
  END_GUARDED
}

PyMethodDef kMethods[] = {
    {"bind", (PyCFunction)(void *)py_bind, METH_FASTCALL, nullptr},
    {"fwd", (PyCFunction)(void *)py_fwd, METH_FASTCALL, nullptr},
    {"bwd", (PyCFunction)(void *)py_bwd, METH_FASTCALL, nullptr},
    {"infer", (PyCFunction)(void *)py_infer, METH_FASTCALL, nullptr},
    {"normalize", (PyCFunction)(void *)py_normalize, METH_FASTCALL, nullptr},
    {"adjoint", (PyCFunction)(void *)py_adjoint, METH_FASTCALL, nullptr},
    {"flat", (PyCFunction)(void *)py_flat, METH_FASTCALL, nullptr},
    {"packed", (PyCFunction)(void *)py_packed, METH_FASTCALL, nullptr},
    {"packed_eps", (PyCFunction)(void *)py_packed_eps, METH_FASTCALL, nullptr},
    {"rms_fwd", (PyCFunction)(void *)py_rms_fwd, METH_FASTCALL, nullptr},
    {"rms_bwd", (PyCFunction)(void *)py_rms_bwd, METH_FASTCALL, nullptr},
    {"rms_quant", (PyCFunction)(void *)py_rms_quant, METH_FASTCALL, nullptr},
    {"rotary_fwd", (PyCFunction)(void *)py_rotary_fwd, METH_FASTCALL, nullptr},
    {"rotary_bwd", (PyCFunction)(void *)py_rotary_bwd, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", "Fast paths of anode_b200.ops into the C ABI.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void)
{
  PyObject *m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "built_for", ANODE_BUILT_FOR) < 0) { Py_DECREF(m); return nullptr; }
  return m;
}
