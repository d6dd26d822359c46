// The Python launchers' way to the C-ABI (include/iris_amd.h): a CPython module that checks the operands, fills the
// argument struct and launches on torch's current stream without going through Python for any of it.
//
// A launch of a few rows is 7 us of GPU work.  Checked and filled in Python (nine tensors, some sixty attribute
// reads, a ctypes struct, a device context) it cost 15 us of host time a launch, and a stream of such launches ran at the
// host's pace; here it costs what the runtime's launch call does.
//
// Every function takes the ordinary, well-formed call and nothing else.  Anything it is not sure of (a tensor of
// another type, a subclass, a wrong extent, another current device) it declines before anything is launched, and
// the Python code behind it runs the full checks, which raise what they always did.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <utility>

#include "../../../include/iris_amd.h"

namespace {

constexpr int DECLINED = -1;

// Read off the file by iris_amd/build.py and iris_amd/_native.py before it is loaded.
__attribute__((used)) const char built_for[] = "iris_amd._launch built for " IRIS_BUILT_FOR;

// A plain strided tensor of the device, or (for None) nothing.  False: not for this module.
struct Operand {
  const at::Tensor* t = nullptr;
  explicit operator bool() const { return t != nullptr; }
  void* ptr() const { return t ? t->data_ptr() : nullptr; }
};

bool plain(const at::Tensor& t) {
  using c10::DispatchKey;
  static const c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::Conjugate,
                                            DispatchKey::Negative, DispatchKey::ZeroTensor, DispatchKey::FuncTorchBatched,
                                            DispatchKey::FuncTorchGradWrapper});
  return t.defined() && t.layout() == c10::kStrided && t.has_storage() && !t.key_set().has_any(wrapped);
}

// Whether this thread is being traced, or inside a transform or a dispatch mode (torch.func, functionalization,
// make_fx, ...): autograd's apply records a function there, or refuses it, and a launch of our own would pass it by.
bool watched() {
  using c10::DispatchKey;
  static const c10::DispatchKeySet modes({DispatchKey::FuncTorchDynamicLayerFrontMode, DispatchKey::FuncTorchDynamicLayerBackMode,
                                          DispatchKey::FuncTorchVmapMode, DispatchKey::FuncTorchBatched,
                                          DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize, DispatchKey::Python,
                                          DispatchKey::PythonTLSSnapshot, DispatchKey::PythonDispatcher, DispatchKey::PreDispatch,
                                          DispatchKey::Tracer});
  return torch::jit::tracer::isTracing() || c10::impl::tls_local_dispatch_key_set().included_.has_any(modes);
}

// Whether autograd has business with a tensor among the arguments: a gradient, or a tangent (forward mode).
bool differentiated(PyObject* const* x, Py_ssize_t n) {
  for (Py_ssize_t i = 0; i < n; ++i) {
    // (what most arguments are: the check for a tensor asks its metaclass about each of these)
    if (x[i] == Py_None || PyLong_Check(x[i]) || PyUnicode_Check(x[i]) || !THPVariable_Check(x[i])) continue;
    const at::Tensor& t = THPVariable_Unpack(x[i]);
    if (!plain(t) || (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(/*level=*/0).defined()) return true;
  }
  return false;
}

bool operand(PyObject* o, int device, Operand* out) {
  if (o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!plain(t) || !t.is_cuda() || t.get_device() != device) return false;
  out->t = &t;
  return true;
}

// Python ints (bools too) only: anything else is left to the Python code's conversions.
bool integer(PyObject* o, int64_t lo, int64_t hi, int64_t* out) {
  if (!PyLong_Check(o)) return false;
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  if (overflow || v < lo || v > hi) return false;
  *out = v;
  return true;
}
bool int32(PyObject* o, int32_t* out) {
  int64_t v;
  if (!integer(o, INT32_MIN, INT32_MAX, &v)) return false;
  *out = (int32_t)v;
  return true;
}
bool ticks(PyObject* o, uint64_t* out) {
  int64_t v;
  if (!integer(o, 0, INT64_MAX, &v)) return false;
  *out = (uint64_t)v;
  return true;
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return IRIS_DTYPE_F32;
    case at::kHalf: return IRIS_DTYPE_F16;
    case at::kBFloat16: return IRIS_DTYPE_BF16;
    default: return -1;
  }
}

bool matrix_of(const Operand& t, int64_t rows, int64_t cols) {
  return t && t.t->dim() == 2 && t.t->size(0) >= rows && t.t->size(1) >= cols;
}

bool contiguous(const Operand& t, at::ScalarType type, int64_t numel) {
  return t.t->scalar_type() == type && t.t->numel() >= numel && t.t->is_contiguous();
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool flags_ok(const Operand& flags, int64_t tiles) { return !flags || contiguous(flags, at::kInt, tiles); }

bool bases_ok(const Operand& bases, int64_t ranks) {
  if (!bases) return ranks <= 1;
  const auto type = bases.t->scalar_type();
  return (type == at::kUInt64 || type == at::kLong) && bases.t->numel() >= ranks;
}

// The device a launch's tensors must share: the first one's, which must be the current one too.
int launch_device(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return -1;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!plain(t) || !t.is_cuda()) return -1;
  int current = -1;
  if (hipGetDevice(&current) != hipSuccess || current != t.get_device()) return -1;
  return current;
}

void* current_stream(int device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

template <class Launch>
int unlocked(Launch launch) {
  int err;
  Py_BEGIN_ALLOW_THREADS;
  err = launch();
  Py_END_ALLOW_THREADS;
  return err;
}

struct GemmOperands {
  Operand a, b, c, c_global, flags, bases, ts_begin, ts_end, status, partials, locks;
};

// The tensors' share of iris_gemm_args, checked as ops.gemm_launch documents it; `g` holds the numbers already.
bool fill_gemm(const GemmOperands& t, iris_gemm_args* g) {
  if (!t.a || !t.b || t.a.t->dim() != 2 || t.b.t->dim() != 2) return false;
  const int64_t M = t.a.t->size(0), K = t.a.t->size(1), N = t.b.t->size(1);
  if (t.b.t->size(0) != K || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return false;
  const int dt = dtype_code(*t.a.t);
  if (dt < 0 || t.b.t->scalar_type() != t.a.t->scalar_type()) return false;
  if (g->block_m <= 0 || g->block_n <= 0 || g->group_size_m <= 0 || g->num_sms <= 0 || g->world_size <= 0) return false;
  const int64_t tiles = cdiv(M, g->block_m) * cdiv(N, g->block_n);
  switch (g->epilogue) {
    case IRIS_EPI_ALL_SCATTER:
      if (!matrix_of(t.c_global, M, N * g->world_size)) return false;
      break;
    case IRIS_EPI_ATOMIC_ADD:
      if (!matrix_of(t.c_global, M, N)) return false;
      break;
    case IRIS_EPI_ONE_SHOT:
      if (!matrix_of(t.c, M, N) || !matrix_of(t.c_global, M, N)) return false;
      break;
    default: return false;
  }
  if (!flags_ok(t.flags, tiles) || !bases_ok(t.bases, g->world_size)) return false;
  if (t.ts_begin && !contiguous(t.ts_begin, at::kLong, tiles)) return false;
  if (t.ts_end && !contiguous(t.ts_end, at::kLong, tiles)) return false;
  if (t.status && !((t.status.t->scalar_type() == at::kInt || t.status.t->scalar_type() == at::kUInt32) && t.status.t->numel() >= 1))
    return false;
  g->a = t.a.ptr();
  g->b = t.b.ptr();
  g->c = t.c.ptr();
  g->c_global = t.c_global.ptr();
  g->tile_completed = static_cast<int32_t*>(t.flags.ptr());
  g->heap_bases = static_cast<const uint64_t*>(t.bases.ptr());
  g->mm_begin_timestamp = static_cast<int64_t*>(t.ts_begin.ptr());
  g->mm_end_timestamp = static_cast<int64_t*>(t.ts_end.ptr());
  g->status = static_cast<uint32_t*>(t.status.ptr());
  g->M = (int32_t)M;
  g->N = (int32_t)N;
  g->K = (int32_t)K;
  g->stride_am = t.a.t->stride(0);
  g->stride_ak = t.a.t->stride(1);
  g->stride_bk = t.b.t->stride(0);
  g->stride_bn = t.b.t->stride(1);
  g->ab_dtype = dt;
  if (t.c) {
    if (t.c.t->dim() != 2 || (g->c_dtype = dtype_code(*t.c.t)) < 0) return false;
    g->stride_cm = t.c.t->stride(0);
    g->stride_cn = t.c.t->stride(1);
  }
  if (t.c_global) {
    if ((g->c_global_dtype = dtype_code(*t.c_global.t)) < 0) return false;
    g->stride_cm_global = t.c_global.t->stride(0);
    g->stride_cn_global = t.c_global.t->stride(1);
  }
  if (t.locks) {
    if (!contiguous(t.locks, at::kInt, g->num_sms)) return false;
    g->locks = static_cast<int32_t*>(t.locks.ptr());
  }
  if (t.partials) {
    if (!t.locks || t.partials.t->scalar_type() != at::kFloat || t.partials.t->dim() != 2 || !t.partials.t->is_contiguous() ||
        t.partials.t->size(0) < g->num_sms)
      return false;
    g->partials = static_cast<float*>(t.partials.ptr());
    g->partials_slot_elems = t.partials.t->size(1);
  } else if (g->split_k > 1 || g->split_k == IRIS_GEMM_SPLIT_STREAM_K) {
    return false;
  }
  return true;
}

// gemm(a, b, c, c_global, tile_completed, heap_bases, mm_begin_timestamp, mm_end_timestamp, status, partials, locks,
//      rank, world_size, num_sms, BLK_M, BLK_N, BLK_K, gsize_m, epilogue, phase, notify, num_xcds, scope, variant,
//      spin_timeout_ticks, split_k, split_handover, flag_sem, touch_ahead)
// -> hipError_t of the launch, or -1: declined, nothing launched.
PyObject* gemm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 29) {
    PyErr_SetString(PyExc_TypeError, "gemm takes 29 arguments");
    return nullptr;
  }
  const int device = launch_device(v[0]);
  GemmOperands t;
  iris_gemm_args g{};
  int32_t notify = PyObject_IsTrue(v[20]);
  const bool ok =
      device >= 0 && operand(v[0], device, &t.a) && operand(v[1], device, &t.b) && operand(v[2], device, &t.c) &&
      operand(v[3], device, &t.c_global) && operand(v[4], device, &t.flags) && operand(v[5], device, &t.bases) &&
      operand(v[6], device, &t.ts_begin) && operand(v[7], device, &t.ts_end) && operand(v[8], device, &t.status) &&
      operand(v[9], device, &t.partials) && operand(v[10], device, &t.locks) && int32(v[11], &g.cur_rank) &&
      int32(v[12], &g.world_size) && int32(v[13], &g.num_sms) && int32(v[14], &g.block_m) && int32(v[15], &g.block_n) &&
      int32(v[16], &g.block_k) && int32(v[17], &g.group_size_m) && int32(v[18], &g.epilogue) && int32(v[19], &g.phase) &&
      notify >= 0 && int32(v[21], &g.num_xcds) && int32(v[22], &g.scope) && int32(v[23], &g.variant) &&
      ticks(v[24], &g.spin_timeout_ticks) && int32(v[25], &g.split_k) && int32(v[26], &g.split_handover) &&
      int32(v[27], &g.flag_sem) && int32(v[28], &g.touch_ahead);
  g.notify = notify;
  PyErr_Clear();
  if (!ok || !fill_gemm(t, &g)) return PyLong_FromLong(DECLINED);
  void* stream = current_stream(device);
  return PyLong_FromLong(unlocked([&] { return iris_gemm_launch(&g, stream); }));
}

// The wrappers' P / locks buffers (benchmark.py:136-142) where they have the reference's shapes, else neither.
void workspace(PyObject* P, PyObject* locks, int device, iris_gemm_args* g, GemmOperands* t) {
  Operand p, l;
  if (!operand(P, device, &p) || !operand(locks, device, &l) || !p || !l) return;
  if (p.t->scalar_type() != at::kFloat || p.t->dim() != 2 || !p.t->is_contiguous() || p.t->size(0) < g->num_sms ||
      p.t->size(1) < (int64_t)g->block_m * g->block_n || !contiguous(l, at::kInt, g->num_sms))
    return;
  t->partials = p;
  t->locks = l;
}

// Class attributes of a `matmul` class that steer its launch.
PyObject *s_debug, *s_notify, *s_phase, *s_scope, *s_variant, *s_status, *s_ticks, *s_split_k;

struct Attr {
  PyObject* o;
  Attr(PyObject* cls, PyObject* name) : o(PyObject_GetAttr(cls, name)) {}
  ~Attr() { Py_XDECREF(o); }
  Attr(const Attr&) = delete;
  bool truth(int32_t* out) const { return o && (*out = PyObject_IsTrue(o)) >= 0; }
};

// matmul_apply(cls, epilogue, args): the positional `matmul.apply(*args)` of a wrapper class, when it is not in debug
// mode, no operand wants a gradient or carries a tangent, and nothing traces or transforms the call.  -> what autograd's
// apply returns (a view of `c`, or None); NotImplemented: declined, nothing launched, the caller takes the long way; or the
// hipError_t of a launch that failed (its first kernel may have run, so it is not tried again).
PyObject* matmul_apply(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 3 || !PyTuple_Check(v[2])) {
    PyErr_SetString(PyExc_TypeError, "matmul_apply(cls, epilogue, args)");
    return nullptr;
  }
  PyObject* const cls = v[0];
  PyObject* const* x = &PyTuple_GET_ITEM(v[2], 0);
  const Py_ssize_t nx = PyTuple_GET_SIZE(v[2]);
  auto decline = [] {
    PyErr_Clear();
    Py_RETURN_NOTIMPLEMENTED;
  };
  // a, b, c, c_global, bias, P, locks, tile_completed, rank, world_size, grid, BLK_M, BLK_N, BLK_K, gsize_m, two_tiles,
  // num_stages, num_warps, waves_per_eu, mfmaInstrSize, kpack, heap_bases_ptr, cu_count, COLLECT_TIMESTAMPS, begin, end
  if (nx < 22 || nx > 26) return decline();
  const int device = launch_device(x[0]);
  if (device < 0) return decline();
  const Attr debug(cls, s_debug), notify(cls, s_notify), phase(cls, s_phase), scope(cls, s_scope), variant(cls, s_variant),
      status(cls, s_status), spin(cls, s_ticks), split_k(cls, s_split_k);
  GemmOperands t;
  iris_gemm_args g{};
  int32_t debug_on, cu_count = 304, collect = 0;
  if (!debug.truth(&debug_on) || debug_on || !notify.truth(&g.notify) || !phase.o || !int32(phase.o, &g.phase) || !scope.o ||
      !int32(scope.o, &g.scope) || !variant.o || !int32(variant.o, &g.variant) || !status.o ||
      !operand(status.o, device, &t.status) || !spin.o || !ticks(spin.o, &g.spin_timeout_ticks) || !split_k.o ||
      !int32(split_k.o, &g.split_k))
    return decline();
  if (!operand(x[0], device, &t.a) || !operand(x[1], device, &t.b) || !operand(x[2], device, &t.c) ||
      !operand(x[3], device, &t.c_global) || !operand(x[7], device, &t.flags) || !int32(x[8], &g.cur_rank) ||
      !int32(x[9], &g.world_size) || !int32(x[10], &g.num_sms) || !int32(x[11], &g.block_m) || !int32(x[12], &g.block_n) ||
      !int32(x[13], &g.block_k) || !int32(x[14], &g.group_size_m) || !operand(x[21], device, &t.bases) || !int32(v[1], &g.epilogue))
    return decline();
  if (nx > 22 && !int32(x[22], &cu_count)) return decline();
  if (nx > 23 && (collect = PyObject_IsTrue(x[23])) < 0) return decline();
  if (collect && ((nx > 24 && !operand(x[24], device, &t.ts_begin)) || (nx > 25 && !operand(x[25], device, &t.ts_end))))
    return decline();
  if (watched() || differentiated(x, nx)) return decline();
  // (ops.default_num_xcds)
  g.num_xcds = (cu_count == 304 || cu_count == 256) && g.num_sms % 8 == 0 ? 8 : 1;
  if (g.num_sms > 0 && g.block_m > 0 && g.block_n > 0) workspace(x[5], x[6], device, &g, &t);
  if (!fill_gemm(t, &g)) return decline();
  void* stream = current_stream(device);
  const int err = unlocked([&] { return iris_gemm_launch(&g, stream); });
  if (err != hipSuccess) return PyLong_FromLong(err);
  if (!t.c) Py_RETURN_NONE;
  try {
    at::NoGradGuard guard;
    return THPVariable_Wrap(t.c.t->view_as(*t.c.t));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// one_shot_reduce(c, c_global, tile_completed, heap_bases, status, rank, world_size, BLK_M, BLK_N, gsize_m, num_sms,
//                 num_xcds, scope, wait_flags, variant, spin_timeout_ticks, flag_sem)
PyObject* one_shot_reduce(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 17) {
    PyErr_SetString(PyExc_TypeError, "one_shot_reduce takes 17 arguments");
    return nullptr;
  }
  const int device = launch_device(v[0]);
  Operand c, c_global, flags, bases, status;
  iris_reduce_args r{};
  r.wait_flags = PyObject_IsTrue(v[13]);
  const bool ok = device >= 0 && operand(v[0], device, &c) && operand(v[1], device, &c_global) && operand(v[2], device, &flags) &&
                  operand(v[3], device, &bases) && operand(v[4], device, &status) && int32(v[5], &r.cur_rank) &&
                  int32(v[6], &r.world_size) && int32(v[7], &r.block_m) && int32(v[8], &r.block_n) &&
                  int32(v[9], &r.group_size_m) && int32(v[10], &r.num_sms) && int32(v[11], &r.num_xcds) &&
                  int32(v[12], &r.scope) && r.wait_flags >= 0 && int32(v[14], &r.variant) &&
                  ticks(v[15], &r.spin_timeout_ticks) && int32(v[16], &r.flag_sem);
  PyErr_Clear();
  if (!ok || c.t->dim() != 2 || !matrix_of(c_global, c.t->size(0), c.t->size(1)) || c.t->size(0) > INT32_MAX ||
      c.t->size(1) > INT32_MAX || r.block_m <= 0 || r.block_n <= 0 || r.group_size_m <= 0 || r.num_sms < 0)
    return PyLong_FromLong(DECLINED);
  const int64_t tiles = cdiv(c.t->size(0), r.block_m) * cdiv(c.t->size(1), r.block_n);
  r.c_dtype = dtype_code(*c.t);
  r.c_global_dtype = dtype_code(*c_global.t);
  if (r.c_dtype < 0 || r.c_global_dtype < 0 || (r.wait_flags && r.world_size > 1 && !flags) || !flags_ok(flags, tiles) ||
      !bases_ok(bases, r.world_size))
    return PyLong_FromLong(DECLINED);
  r.c = c.ptr();
  r.c_global = c_global.ptr();
  r.tile_completed = static_cast<int32_t*>(flags.ptr());
  r.heap_bases = static_cast<const uint64_t*>(bases.ptr());
  r.status = static_cast<uint32_t*>(status.ptr());
  r.M = (int32_t)c.t->size(0);
  r.N = (int32_t)c.t->size(1);
  r.stride_cm = c.t->stride(0);
  r.stride_cn = c.t->stride(1);
  r.stride_cm_global = c_global.t->stride(0);
  r.stride_cn_global = c_global.t->stride(1);
  void* stream = current_stream(device);
  return PyLong_FromLong(unlocked([&] { return iris_one_shot_reduce_launch(&r, stream); }));
}

// memset_i32(tensor, value)
PyObject* memset_i32(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "memset_i32(tensor, value)");
    return nullptr;
  }
  const int device = launch_device(v[0]);
  Operand t;
  int32_t value;
  if (device < 0 || !operand(v[0], device, &t) || t.t->scalar_type() != at::kInt || !t.t->is_contiguous() || !int32(v[1], &value))
    return PyLong_FromLong(DECLINED);
  int32_t* p = static_cast<int32_t*>(t.ptr());
  const int64_t count = t.t->numel();
  void* stream = current_stream(device);
  return PyLong_FromLong(unlocked([&] { return iris_memset_i32_launch(p, value, count, stream); }));
}

// ---- the attention block (iris_amd/attention.py documents what is checked) ----

constexpr int MAX_REQUESTS = 8192, MAX_HEAD_DIM = 512, MAX_ATTENTION_HEAD_DIM = 256;

bool real(PyObject* o, double* out) {
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  *out = PyFloat_AsDouble(o);
  return !PyErr_Occurred();
}
bool truth(PyObject* o, int32_t* out) { return (*out = PyObject_IsTrue(o)) >= 0; }

// Autograd's business with an operand: a tangent (forward mode), or a gradient.
bool tangent(const Operand& t) { return t && t.t->_fw_grad(/*level=*/0).defined(); }
bool differentiates(const Operand& t) { return t && ((at::GradMode::is_enabled() && t.t->requires_grad()) || tangent(t)); }

// A tensor [tokens, heads, head size] of `type` whose head elements are contiguous; sizes below 0 are free.
bool heads_of(const Operand& t, at::ScalarType type, int64_t tokens, int64_t heads, int64_t dim) {
  return t && t.t->dim() == 3 && t.t->scalar_type() == type && (tokens < 0 || t.t->size(0) == tokens) && (heads < 0 || t.t->size(1) == heads) &&
         (dim < 0 || t.t->size(2) == dim) && (t.t->size(2) <= 1 || t.t->stride(2) == 1) && t.t->size(0) <= INT32_MAX && t.t->size(1) <= INT32_MAX;
}

// Something that a kernel writes: elements of its own, and no gradient.
bool output(const Operand& t) {
  if (!t || differentiates(t)) return false;
  const int64_t n = t.t->dim();
  int64_t reach = 0, floor = -1;  // axes in the order of their strides
  for (int64_t taken = 0; taken < n; ++taken) {
    int64_t best = -1;
    for (int64_t i = 0; i < n; ++i) {
      const int64_t key = t.t->stride(i) * 8 + i;
      if (key > floor && (best < 0 || key < t.t->stride(best) * 8 + best)) best = i;
    }
    if (best < 0) return false;
    floor = t.t->stride(best) * 8 + best;
    if (t.t->size(best) <= 1) continue;
    if (t.t->stride(best) <= reach) return false;
    reach += t.t->stride(best) * (t.t->size(best) - 1);
  }
  return true;
}

// A tensor's elements lie in [lo, hi).
struct Span {
  const char *lo = nullptr, *hi = nullptr;
  bool meets(const Span& other) const { return lo < other.hi && other.lo < hi; }
};
Span span_of(const at::Tensor& t) {
  const auto sizes = t.sizes(), strides = t.strides();
  Span s;
  int64_t reach = 1;
  for (size_t d = 0; d < sizes.size(); ++d) {
    if (!sizes[d]) return s;
    reach += (sizes[d] - 1) * strides[d];
  }
  s.lo = (const char*)t.data_ptr();
  s.hi = s.lo + reach * (int64_t)t.element_size();
  return s;
}
// ... as runs of `run` bytes at every combination of its axes' steps, the longest step first.
struct Lattice {
  static constexpr int MOST_AXES = 8;
  int64_t step[MOST_AXES], count[MOST_AXES], run;
  int axes = 0;
};
Lattice lattice_of(const at::Tensor& t) {
  Lattice l;
  l.run = (int64_t)t.element_size();
  for (int64_t d = 0; d < t.dim(); ++d) {
    const int64_t n = t.size(d), step = t.stride(d) * (int64_t)t.element_size();
    if (n <= 1 || step == 0) continue;
    int i = l.axes++;
    for (; i > 0 && l.step[i - 1] < step; --i) l.step[i] = l.step[i - 1], l.count[i] = l.count[i - 1];
    l.step[i] = step, l.count[i] = n;
  }
  while (l.axes && l.step[l.axes - 1] == l.run) l.run *= l.count[--l.axes];
  return l;
}
// Whether the axes from i and j on of two lattices, the second `by` bytes further on, have a byte in common.  A step of the longest axis
// is looked at only where what is left of both can meet, which for tensors whose axes lie inside each other are two or three.
// `budget` ends the rest: what cannot be told apart counts as common.
bool meet(const Lattice& a, int i, const Lattice& b, int j, int64_t by, int* budget) {
  if (--*budget < 0) return true;
  int64_t reach_a = a.run, reach_b = b.run;
  for (int k = i; k < a.axes; ++k) reach_a += (a.count[k] - 1) * a.step[k];
  for (int k = j; k < b.axes; ++k) reach_b += (b.count[k] - 1) * b.step[k];
  if (by >= reach_a || -by >= reach_b) return false;
  if (i == a.axes && j == b.axes) return true;
  const int64_t step = std::max(i < a.axes ? a.step[i] : 0, j < b.axes ? b.step[j] : 0);
  const bool in_a = i < a.axes && a.step[i] == step, in_b = j < b.axes && b.step[j] == step;
  const int64_t most = in_a ? a.count[i] - 1 : 0, least = in_b ? 1 - b.count[j] : 0;  // of a's index less b's
  if (in_a) reach_a -= most * step;
  if (in_b) reach_b += least * step;
  // -reach_b < by - k step < reach_a
  const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t first = std::max(least, floor_div(by - reach_a, step) + 1), last = std::min(most, floor_div(by + reach_b - 1, step));
  for (int64_t k = first; k <= last; ++k)
    if (meet(a, i + in_a, b, j + in_b, by - k * step, budget)) return true;
  return false;
}
bool common(const at::Tensor& a, const at::Tensor& b) {
  if (a.dim() > Lattice::MOST_AXES || b.dim() > Lattice::MOST_AXES) return true;
  int budget = 4096;
  return meet(lattice_of(a), 0, lattice_of(b), 0, (const char*)b.data_ptr() - (const char*)a.data_ptr(), &budget);
}
bool same_view(const at::Tensor& a, const at::Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}
// Operands t[outs] lie apart from each other and, but for those in `late` (which are written when all inputs have been read), from
// t[ins].  An output may be one of its own inputs, element by element: (output, input) pairs in `in_place`.
bool apart(const Operand* t, std::initializer_list<int> outs, std::initializer_list<int> ins, std::initializer_list<std::pair<int, int>> in_place,
           std::initializer_list<int> late = {}) {
  Span span[16];
  for (const auto& list : {outs, ins})
    for (const int i : list)
      if (t[i]) span[i] = span_of(*t[i].t);
  for (auto o = outs.begin(); o != outs.end(); ++o) {
    for (auto p = outs.begin(); p != o; ++p)
      if (span[*o].meets(span[*p]) && common(*t[*o].t, *t[*p].t)) return false;
    if (std::find(late.begin(), late.end(), *o) != late.end()) continue;
    for (const int i : ins) {
      if (!span[*o].meets(span[i])) continue;
      if (std::find(in_place.begin(), in_place.end(), std::make_pair(*o, i)) != in_place.end() && same_view(*t[*o].t, *t[i].t)) continue;
      if (common(*t[*o].t, *t[i].t)) return false;
    }
  }
  return true;
}

// overlap(a, b) -> whether two tensors (of any device) have memory in common, or may have.
PyObject* overlap(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 2 || !THPVariable_Check(x[0]) || !THPVariable_Check(x[1])) {
    PyErr_SetString(PyExc_TypeError, "overlap takes two tensors");
    return nullptr;
  }
  const at::Tensor &a = THPVariable_Unpack(x[0]), &b = THPVariable_Unpack(x[1]);
  if (!plain(a) || !plain(b)) Py_RETURN_TRUE;
  return PyBool_FromLong(a.device() == b.device() && span_of(a).meets(span_of(b)) && common(a, b));
}

bool vector_of(const Operand& t, at::ScalarType type, int64_t numel) {
  return t && t.t->dim() == 1 && t.t->scalar_type() == type && t.t->numel() == numel && t.t->is_contiguous();
}
bool status_ok(const Operand& t) {
  return !t || ((t.t->scalar_type() == at::kInt || t.t->scalar_type() == at::kUInt32) && t.t->numel() >= 1);
}
bool rows_contiguous(const Operand& t) { return t && t.t->dim() == 2 && (t.t->size(1) <= 1 || t.t->stride(1) == 1); }

// build_block_tables(cached, new_tokens, block_table, pool, pool_state, lengths, pool_state_out, query_starts, positions, slots,
//                    status, page_size)
PyObject* block_tables(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 12) {
    PyErr_SetString(PyExc_TypeError, "block_tables takes 12 arguments");
    return nullptr;
  }
  const int device = launch_device(v[0]);
  Operand t[11];
  iris_block_tables_args a{};
  bool ok = device >= 0 && int32(v[11], &a.page_size) && a.page_size > 0;
  for (int i = 0; ok && i < 11; ++i) ok = operand(v[i], device, &t[i]);
  PyErr_Clear();
  enum { CACHED, NEW, TABLE, POOL, STATE, LENGTHS, STATE_OUT, STARTS, POSITIONS, SLOTS, STATUS };
  if (!ok || !t[CACHED] || !t[POOL] || !t[POSITIONS]) return PyLong_FromLong(DECLINED);
  const int64_t requests = t[CACHED].t->numel(), pool = t[POOL].t->numel(), tokens = t[POSITIONS].t->numel();
  if (requests > MAX_REQUESTS || pool < 1 || pool > INT32_MAX || tokens > INT32_MAX || !vector_of(t[CACHED], at::kInt, requests) ||
      !vector_of(t[NEW], at::kInt, requests) || !vector_of(t[LENGTHS], at::kInt, requests) || !vector_of(t[STARTS], at::kInt, requests + 1) ||
      !vector_of(t[POOL], at::kInt, pool) || !vector_of(t[STATE], at::kLong, 2) || !vector_of(t[STATE_OUT], at::kLong, 2) ||
      !vector_of(t[POSITIONS], at::kInt, tokens) || !vector_of(t[SLOTS], at::kLong, tokens) || !status_ok(t[STATUS]) || !rows_contiguous(t[TABLE]) ||
      t[TABLE].t->scalar_type() != at::kInt || t[TABLE].t->size(0) != requests || t[TABLE].t->size(1) > INT32_MAX ||
      (requests > 1 && !output(t[TABLE])))
    return PyLong_FromLong(DECLINED);
  // no operand lies in another
  for (int i = 0; i < STATUS; ++i) {
    const auto span = [&](int k, const char** lo, const char** hi) {
      int64_t reach = 1;
      for (int64_t d = 0; d < t[k].t->dim(); ++d) reach += t[k].t->stride(d) * (t[k].t->size(d) - 1);
      *lo = (const char*)t[k].ptr();
      *hi = *lo + (t[k].t->numel() ? reach * (int64_t)t[k].t->element_size() : 0);
    };
    const char *lo, *hi, *lo2, *hi2;
    span(i, &lo, &hi);
    for (int k = 0; k < i; ++k) {
      span(k, &lo2, &hi2);
      if (lo < hi2 && lo2 < hi) return PyLong_FromLong(DECLINED);
    }
  }
  a.cached = (const int32_t*)t[CACHED].ptr();
  a.new_tokens = (const int32_t*)t[NEW].ptr();
  a.block_table = (int32_t*)t[TABLE].ptr();
  a.pool = (int32_t*)t[POOL].ptr();
  a.pool_state = (const int64_t*)t[STATE].ptr();
  a.pool_state_out = (int64_t*)t[STATE_OUT].ptr();
  a.lengths = (int32_t*)t[LENGTHS].ptr();
  a.query_starts = (int32_t*)t[STARTS].ptr();
  a.positions = (int32_t*)t[POSITIONS].ptr();
  a.slots = (int64_t*)t[SLOTS].ptr();
  a.status = (uint32_t*)t[STATUS].ptr();
  a.requests = (int32_t)requests;
  a.table_width = (int32_t)t[TABLE].t->size(1);
  a.stride_table = std::max<int64_t>(t[TABLE].t->stride(0), a.table_width);
  a.pool_size = (int32_t)pool;
  a.max_tokens = (int32_t)tokens;
  void* stream = current_stream(device);
  return PyLong_FromLong(unlocked([&] { return iris_block_tables_launch(&a, stream); }));
}

// What the norms and the rotation take beside the heads.
template <class Args>
bool rope_operands(const Operand& positions, const Operand& cos, const Operand& sin, const Operand& qw, const Operand& kw, at::ScalarType type,
                   int64_t tokens, int64_t dim, Args* a) {
  if (dim % 2 || dim <= 0 || dim > MAX_HEAD_DIM || (bool)cos != (bool)sin) return false;
  if (cos) {
    if (!positions || cos.t->scalar_type() != at::kFloat || sin.t->scalar_type() != at::kFloat || !rows_contiguous(cos) || !rows_contiguous(sin) ||
        cos.t->sizes() != sin.t->sizes() || cos.t->size(0) < 1 || cos.t->size(0) > INT32_MAX || 2 * cos.t->size(1) > dim)
      return false;
    const bool wide = positions.t->scalar_type() == at::kLong;
    if (!vector_of(positions, wide ? at::kLong : at::kInt, tokens)) return false;
    a->cos = (const float*)cos.ptr();
    a->sin = (const float*)sin.ptr();
    a->positions = positions.ptr();
    a->stride_cos = cos.t->stride(0);
    a->stride_sin = sin.t->stride(0);
    a->rotary_dim = (int32_t)(2 * cos.t->size(1));
    a->max_positions = (int32_t)cos.t->size(0);
    a->positions_64 = wide;
  }
  for (const Operand* w : {&qw, &kw})
    if (*w && (!vector_of(*w, w->t->scalar_type(), dim) || (w->t->scalar_type() != type && w->t->scalar_type() != at::kFloat))) return false;
  if (qw && kw && qw.t->scalar_type() != kw.t->scalar_type()) return false;
  a->q_weight = qw.ptr();
  a->k_weight = kw.ptr();
  a->weight_fp32 = (qw && qw.t->scalar_type() == at::kFloat) || (kw && kw.t->scalar_type() == at::kFloat);
  a->tokens = (int32_t)tokens;
  a->head_dim = (int32_t)dim;
  return true;
}

struct CacheStrides {
  int64_t page, row, head;
};
bool cache_of(const Operand& t, at::ScalarType type, int64_t heads, int64_t dim, CacheStrides* s) {
  if (!t || t.t->dim() != 4 || t.t->scalar_type() != type || t.t->size(1) < 1 || t.t->size(2) != heads || t.t->size(3) != dim ||
      (dim > 1 && t.t->stride(3) != 1) || t.t->size(0) > INT32_MAX || t.t->size(1) > INT32_MAX)
    return false;
  int64_t* const out[3] = {&s->page, &s->row, &s->head};
  for (int i = 0; i < 3; ++i) *out[i] = t.t->size(i) > 1 ? t.t->stride(i) : 0;  // (the stride of an axis of one is never taken)
  return true;
}

void strides_of(const Operand& t, int64_t* token, int64_t* head) {
  *token = t.t->size(0) > 1 ? t.t->stride(0) : 0;
  *head = t.t->size(1) > 1 ? t.t->stride(1) : 0;
}

// qk_norm_rope(q, k, positions, cos, sin, q_out, k_out, q_weight, k_weight, v, k_cache, v_cache, slots, status, eps, interleaved)
PyObject* qk_norm_rope(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 16) {
    PyErr_SetString(PyExc_TypeError, "qk_norm_rope takes 16 arguments");
    return nullptr;
  }
  const int device = launch_device(x[0]);
  Operand t[14];
  iris_qk_norm_rope_args a{};
  double eps = 0;
  bool ok = device >= 0 && real(x[14], &eps) && truth(x[15], &a.interleaved);
  for (int i = 0; ok && i < 14; ++i) ok = operand(x[i], device, &t[i]);
  PyErr_Clear();
  enum { Q, K, POSITIONS, COS, SIN, Q_OUT, K_OUT, QW, KW, V, K_CACHE, V_CACHE, SLOTS, STATUS };
  if (!ok || !t[Q] || t[Q].t->dim() != 3 || dtype_code(*t[Q].t) < 0) return PyLong_FromLong(DECLINED);
  const auto type = t[Q].t->scalar_type();
  const int64_t tokens = t[Q].t->size(0), hq = t[Q].t->size(1), dim = t[Q].t->size(2);
  if (!heads_of(t[Q], type, -1, -1, -1) || !heads_of(t[K], type, tokens, -1, dim) || !heads_of(t[Q_OUT], type, tokens, hq, dim) || !output(t[Q_OUT]))
    return PyLong_FromLong(DECLINED);
  const int64_t hk = t[K].t->size(1);
  for (const int i : {Q, K, V, COS, SIN, QW, KW})
    if (differentiates(t[i])) return PyLong_FromLong(DECLINED);
  if (!rope_operands(t[POSITIONS], t[COS], t[SIN], t[QW], t[KW], type, tokens, dim, &a) || !status_ok(t[STATUS])) return PyLong_FromLong(DECLINED);
  if (t[K_OUT] ? !heads_of(t[K_OUT], type, tokens, hk, dim) || !output(t[K_OUT]) : !t[SLOTS] && hk) return PyLong_FromLong(DECLINED);
  if (t[SLOTS]) {
    CacheStrides k, w;
    if (!heads_of(t[V], type, tokens, hk, dim) || !vector_of(t[SLOTS], at::kLong, tokens) || !cache_of(t[K_CACHE], type, hk, dim, &k) ||
        !cache_of(t[V_CACHE], type, hk, dim, &w) || t[K_CACHE].t->sizes() != t[V_CACHE].t->sizes() || !output(t[K_CACHE]) || !output(t[V_CACHE]))
      return PyLong_FromLong(DECLINED);
    a.page_size = (int32_t)t[K_CACHE].t->size(1);
    a.num_slots = t[K_CACHE].t->size(0) * t[K_CACHE].t->size(1);
    if (a.num_slots > INT32_MAX) return PyLong_FromLong(DECLINED);
    a.stride_kc_page = k.page, a.stride_kc_row = k.row, a.stride_kc_head = k.head;
    a.stride_vc_page = w.page, a.stride_vc_row = w.row, a.stride_vc_head = w.head;
    strides_of(t[V], &a.stride_vt, &a.stride_vh);
  } else if (t[V] || t[K_CACHE] || t[V_CACHE]) {
    return PyLong_FromLong(DECLINED);
  }
  if (!apart(t, {Q_OUT, K_OUT, K_CACHE, V_CACHE}, {Q, K, V, POSITIONS, COS, SIN, QW, KW, SLOTS}, {{Q_OUT, Q}, {K_OUT, K}}))
    return PyLong_FromLong(DECLINED);
  a.q = t[Q].ptr();
  a.k = t[K].ptr();
  a.v = t[V].ptr();
  a.q_out = t[Q_OUT].ptr();
  a.k_out = t[K_OUT].ptr();
  a.k_cache = t[K_CACHE].ptr();
  a.v_cache = t[V_CACHE].ptr();
  a.slots = (const int64_t*)t[SLOTS].ptr();
  a.status = (uint32_t*)t[STATUS].ptr();
  strides_of(t[Q], &a.stride_qt, &a.stride_qh);
  strides_of(t[K], &a.stride_kt, &a.stride_kh);
  strides_of(t[Q_OUT], &a.stride_qot, &a.stride_qoh);
  if (t[K_OUT]) strides_of(t[K_OUT], &a.stride_kot, &a.stride_koh);
  a.q_heads = (int32_t)hq;
  a.k_heads = (int32_t)hk;
  a.dtype = dtype_code(*t[Q].t);
  a.eps = (float)eps;
  void* stream = current_stream(device);
  return PyLong_FromLong(unlocked([&] { return iris_qk_norm_rope_launch(&a, stream); }));
}

// qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, dq, dk, q_weight, k_weight, dq_weight, dk_weight, workspace,
//                       status, eps, interleaved)
PyObject* qk_norm_rope_backward(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 17) {
    PyErr_SetString(PyExc_TypeError, "qk_norm_rope_backward takes 17 arguments");
    return nullptr;
  }
  const int device = launch_device(x[2]);
  Operand t[15];
  iris_qk_norm_rope_backward_args a{};
  double eps = 0;
  bool ok = device >= 0 && real(x[15], &eps) && truth(x[16], &a.interleaved);
  for (int i = 0; ok && i < 15; ++i) ok = operand(x[i], device, &t[i]);
  PyErr_Clear();
  enum { DQ_OUT, DK_OUT, Q, K, POSITIONS, COS, SIN, DQ, DK, QW, KW, DQW, DKW, WORKSPACE, STATUS };
  if (!ok || !t[Q] || t[Q].t->dim() != 3 || dtype_code(*t[Q].t) < 0) return PyLong_FromLong(DECLINED);
  const auto type = t[Q].t->scalar_type();
  const int64_t tokens = t[Q].t->size(0), hq = t[Q].t->size(1), dim = t[Q].t->size(2);
  if (!heads_of(t[Q], type, -1, -1, -1) || !heads_of(t[K], type, tokens, -1, dim)) return PyLong_FromLong(DECLINED);
  const int64_t hk = t[K].t->size(1);
  if (!heads_of(t[DQ_OUT], type, tokens, hq, dim) || !heads_of(t[DQ], type, tokens, hq, dim) || !heads_of(t[DK_OUT], type, tokens, hk, dim) ||
      !heads_of(t[DK], type, tokens, hk, dim) || !output(t[DQ]) || !output(t[DK]) || !status_ok(t[STATUS]) ||
      !rope_operands(t[POSITIONS], t[COS], t[SIN], t[QW], t[KW], type, tokens, dim, &a))
    return PyLong_FromLong(DECLINED);
  for (const int i : {DQ_OUT, DK_OUT, Q, K, COS, SIN, QW, KW})
    if (tangent(t[i])) return PyLong_FromLong(DECLINED);
  if (t[DQW] || t[DKW]) {
    if ((t[DQW] && (!t[QW] || !vector_of(t[DQW], at::kFloat, dim) || !output(t[DQW]))) ||
        (t[DKW] && (!t[KW] || !vector_of(t[DKW], at::kFloat, dim) || !output(t[DKW]))) || !t[WORKSPACE] ||
        !contiguous(t[WORKSPACE], at::kFloat, 2 * dim))
      return PyLong_FromLong(DECLINED);
    a.workspace = (float*)t[WORKSPACE].ptr();
    a.workspace_elems = t[WORKSPACE].t->numel();
  }
  // (the weights' gradients are written by a launch of their own)
  if (!apart(t, {DQ, DK, WORKSPACE, DQW, DKW}, {DQ_OUT, DK_OUT, Q, K, POSITIONS, COS, SIN, QW, KW}, {{DQ, DQ_OUT}, {DQ, Q}, {DK, DK_OUT}, {DK, K}},
             {DQW, DKW}))
    return PyLong_FromLong(DECLINED);
  a.dq_out = t[DQ_OUT].ptr();
  a.dk_out = t[DK_OUT].ptr();
  a.q = t[Q].ptr();
  a.k = t[K].ptr();
  a.dq = t[DQ].ptr();
  a.dk = t[DK].ptr();
  a.dq_weight = (float*)t[DQW].ptr();
  a.dk_weight = (float*)t[DKW].ptr();
  a.status = (uint32_t*)t[STATUS].ptr();
  strides_of(t[DQ_OUT], &a.stride_dqot, &a.stride_dqoh);
  strides_of(t[DK_OUT], &a.stride_dkot, &a.stride_dkoh);
  strides_of(t[Q], &a.stride_qt, &a.stride_qh);
  strides_of(t[K], &a.stride_kt, &a.stride_kh);
  strides_of(t[DQ], &a.stride_dqt, &a.stride_dqh);
  strides_of(t[DK], &a.stride_dkt, &a.stride_dkh);
  a.q_heads = (int32_t)hq;
  a.k_heads = (int32_t)hk;
  a.dtype = dtype_code(*t[Q].t);
  a.eps = (float)eps;
  void* stream = current_stream(device);
  return PyLong_FromLong(unlocked([&] { return iris_qk_norm_rope_backward_launch(&a, stream); }));
}

// attention(q, k_cache, v_cache, block_table, lengths, query_starts, out, lse, workspace, status, scale, window, sinks)
PyObject* attention(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 13) {
    PyErr_SetString(PyExc_TypeError, "attention takes 13 arguments");
    return nullptr;
  }
  const int device = launch_device(x[0]);
  Operand t[10];
  iris_attention_args a{};
  double scale = 0;
  bool ok = device >= 0 && (x[10] == Py_None || real(x[10], &scale)) && int32(x[11], &a.window) && int32(x[12], &a.sinks);
  for (int i = 0; ok && i < 10; ++i) ok = operand(x[i], device, &t[i]);
  PyErr_Clear();
  enum { Q, K_CACHE, V_CACHE, TABLE, LENGTHS, STARTS, OUT, LSE, WORKSPACE, STATUS };
  if (!ok || !t[Q] || t[Q].t->dim() != 3 || dtype_code(*t[Q].t) < 0 || !t[K_CACHE] || t[K_CACHE].t->dim() != 4 || !rows_contiguous(t[TABLE]))
    return PyLong_FromLong(DECLINED);
  const auto type = t[Q].t->scalar_type();
  const int64_t tokens = t[Q].t->size(0), hq = t[Q].t->size(1), dim = t[Q].t->size(2), hk = t[K_CACHE].t->size(2);
  const int64_t requests = t[TABLE].t->size(0), width = t[TABLE].t->size(1), pages = t[K_CACHE].t->size(0), page_size = t[K_CACHE].t->size(1);
  const int64_t vec = 16 / (int64_t)t[Q].t->element_size();
  CacheStrides k, v;
  // (calls with nothing to do, and those whose sizes are refused, are the Python code's)
  if (!tokens || !hq || !hk || !requests || !width || !pages || hq % hk || dim % vec || dim <= 0 || dim > MAX_ATTENTION_HEAD_DIM ||
      width > INT32_MAX || requests > INT32_MAX || width * page_size > INT32_MAX)
    return PyLong_FromLong(DECLINED);
  if (!heads_of(t[Q], type, -1, -1, -1) || !heads_of(t[OUT], type, tokens, hq, dim) || !cache_of(t[K_CACHE], type, hk, dim, &k) ||
      !cache_of(t[V_CACHE], type, hk, dim, &v) || t[K_CACHE].t->sizes() != t[V_CACHE].t->sizes() || t[TABLE].t->scalar_type() != at::kInt ||
      !vector_of(t[LENGTHS], at::kInt, requests) || (t[STARTS] ? !vector_of(t[STARTS], at::kInt, requests + 1) : requests != tokens) ||
      !output(t[OUT]) || !status_ok(t[STATUS]))
    return PyLong_FromLong(DECLINED);
  for (const int i : {Q, K_CACHE, V_CACHE})
    if (differentiates(t[i])) return PyLong_FromLong(DECLINED);
  if (t[LSE]) {
    if (t[LSE].t->scalar_type() != at::kFloat || !rows_contiguous(t[LSE]) || t[LSE].t->size(0) != tokens || t[LSE].t->size(1) != hq || !output(t[LSE]))
      return PyLong_FromLong(DECLINED);
    a.lse = (float*)t[LSE].ptr();
    a.stride_lse = t[LSE].t->stride(0);
  }
  if (t[WORKSPACE]) {
    if (!contiguous(t[WORKSPACE], at::kFloat, 0)) return PyLong_FromLong(DECLINED);
    a.workspace = (float*)t[WORKSPACE].ptr();
    a.workspace_elems = t[WORKSPACE].t->numel();
  }
  if (!apart(t, {OUT, LSE, WORKSPACE}, {Q, K_CACHE, V_CACHE, TABLE, LENGTHS, STARTS}, {{OUT, Q}})) return PyLong_FromLong(DECLINED);
  a.q = t[Q].ptr();
  a.k_cache = t[K_CACHE].ptr();
  a.v_cache = t[V_CACHE].ptr();
  a.block_table = (const int32_t*)t[TABLE].ptr();
  a.lengths = (const int32_t*)t[LENGTHS].ptr();
  a.query_starts = (const int32_t*)t[STARTS].ptr();
  a.out = t[OUT].ptr();
  a.status = (uint32_t*)t[STATUS].ptr();
  strides_of(t[Q], &a.stride_qt, &a.stride_qh);
  strides_of(t[OUT], &a.stride_ot, &a.stride_oh);
  a.stride_kc_page = k.page, a.stride_kc_row = k.row, a.stride_kc_head = k.head;
  a.stride_vc_page = v.page, a.stride_vc_row = v.row, a.stride_vc_head = v.head;
  a.stride_table = requests > 1 ? std::max(t[TABLE].t->stride(0), width) : width;
  if (requests > 1 && t[TABLE].t->stride(0) < width) return PyLong_FromLong(DECLINED);
  a.requests = (int32_t)requests;
  a.tokens = (int32_t)tokens;
  a.q_heads = (int32_t)hq;
  a.k_heads = (int32_t)hk;
  a.head_dim = (int32_t)dim;
  a.page_size = (int32_t)page_size;
  a.table_width = (int32_t)width;
  a.num_pages = (int32_t)pages;
  a.dtype = dtype_code(*t[Q].t);
  a.scale = (float)(x[10] == Py_None ? 1.0 / std::sqrt((double)dim) : scale);
  void* stream = current_stream(device);
  return PyLong_FromLong(unlocked([&] { return iris_attention_launch(&a, stream); }));
}

PyMethodDef methods[] = {
    {"gemm", (PyCFunction)(void (*)(void))gemm, METH_FASTCALL, "launch a shard GEMM; -1: declined"},
    {"matmul_apply", (PyCFunction)(void (*)(void))matmul_apply, METH_FASTCALL, "matmul.apply; NotImplemented: declined, int: failed"},
    {"one_shot_reduce", (PyCFunction)(void (*)(void))one_shot_reduce, METH_FASTCALL, "launch the reduce; -1: declined"},
    {"memset_i32", (PyCFunction)(void (*)(void))memset_i32, METH_FASTCALL, "int32 fill; -1: declined"},
    {"block_tables", (PyCFunction)(void (*)(void))block_tables, METH_FASTCALL, "launch the block tables; -1: declined"},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, "launch norms and rotation; -1: declined"},
    {"qk_norm_rope_backward", (PyCFunction)(void (*)(void))qk_norm_rope_backward, METH_FASTCALL, "launch their gradient; -1: declined"},
    {"overlap", (PyCFunction)(void (*)(void))overlap, METH_FASTCALL, "whether two tensors have memory in common"},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, "launch attention over a paged cache; -1: declined"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", "launches through the C-ABI on torch's current stream", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__launch(void) {
  s_debug = PyUnicode_InternFromString("_debug");
  s_notify = PyUnicode_InternFromString("notify");
  s_phase = PyUnicode_InternFromString("phase");
  s_scope = PyUnicode_InternFromString("scope");
  s_variant = PyUnicode_InternFromString("variant");
  s_status = PyUnicode_InternFromString("status");
  s_ticks = PyUnicode_InternFromString("spin_timeout_ticks");
  s_split_k = PyUnicode_InternFromString("split_k");
  return PyModule_Create(&module);
}
