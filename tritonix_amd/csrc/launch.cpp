// Repeated calls of the Python entry points, from a kept argument struct to the launch, without the interpreter.
//
// A call of a size met before has nothing to decide: allocate the result, fill three pointers into a tnx_gemm_args, launch.  In
// Python that took 5.5 us around a launch of 3.5 (the tuple of sizes, strides and types that finds the struct, torch.empty,
// ctypes), which is what a small product waits for: its kernel takes 4 to 5.  Here it takes 1.2: 1024 x 768 x 512 through
// tritonix.matmul 8.97 -> 5.84 us, a small gated product 7.7 -> 4.9, conv2d 8.6 -> 5.5 and, in two launches, 12.4 -> 9.0.
//
// The entry points are looked up in the library that tritonix_amd/_C.py has loaded (their addresses are handed to bind()), the
// structs are the header's.  Every function answers None where the ordinary path has to take the call: a size not kept, a hook,
// a replaced config, a tensor on another than the current device, a subclass of torch.Tensor (but Parameter), an allocation that
// failed, a conv2d status other than TNX_OK.  That path then raises what is to be raised.  A product's status is raised here: its
// launch may have left counters set in the workspace, which is not to be launched over again.  All state is guarded by the
// interpreter lock, which no entry of the tables is read without.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/headeronly/version.h>

#include <cstring>
#include <mutex>
#include <unordered_map>

#include "../../include/tritonix_hip.h"

namespace {

int (*fn_gemm)(const tnx_gemm_args*) = nullptr;
int (*fn_gemm_f32)(const tnx_gemm_args*, void*, size_t) = nullptr;
int (*fn_conv)(const tnx_conv2d_args*) = nullptr;
PyObject* fn_workspace = nullptr;       // (device index, stream, bytes, atomic) -> tensor
PyObject* fn_failed = nullptr;          // (device index, stream, status, argument struct): raises

// What a launch depends on but its pointers.  Compared and hashed as bytes: zero-filled before it is written.
struct Key {
  int64_t tag;
  int64_t sizes[8], strides[8];
  int64_t options[6];
  int32_t type_a, type_b, type_c, device, aligned, count_c;
  bool operator==(const Key& o) const { return std::memcmp(this, &o, sizeof(Key)) == 0; }
};
struct Hash {
  size_t operator()(const Key& k) const {
    const unsigned char* p = (const unsigned char*)&k;
    uint64_t h = 0x9e3779b97f4a7c15ull;
    for (size_t i = 0; i < sizeof(Key); i += 8) {
      uint64_t w;
      std::memcpy(&w, p + i, 8);
      h = (h ^ w) * 0xff51afd7ed558ccdull;
      h ^= h >> 32;
    }
    return (size_t)h;
  }
};
static_assert(sizeof(Key) % 8 == 0, "hashed word by word");

struct Object {                          // a Python reference that goes with its plan
  PyObject* p = nullptr;
  Object() = default;
  explicit Object(PyObject* o) : p(o) { Py_XINCREF(p); }
  Object(Object&& o) noexcept : p(o.p) { o.p = nullptr; }
  Object& operator=(Object&& o) noexcept { std::swap(p, o.p); return *this; }
  ~Object() { Py_XDECREF(p); }
};

Object taken(PyObject* o) {              // a new reference
  Object t;
  t.p = o;
  return t;
}

struct Product {
  tnx_gemm_args args;
  int64_t rows, cols;
  at::ScalarType type;
  int64_t scratch, slices;
  bool atomic;
  Object memo_key, config;
};
struct Conv {
  tnx_conv2d_args args;
  int64_t shape[4], scratch;
};
// never destroyed: what they hold belongs to the interpreter, which is gone by the time destructors of statics run
std::unordered_map<Key, Product, Hash>& products = *new std::unordered_map<Key, Product, Hash>;
std::unordered_map<Key, Conv, Hash>& convs = *new std::unordered_map<Key, Conv, Hash>;

// an ordinary dense tensor on the GPU: nothing that intercepts the calls the Python path would make of it, no tangent of forward mode (which the Python
// path refuses where an operator has gradients)
bool plain(const at::Tensor& t, int64_t dim) {
  if (!t.defined() || !t.is_cuda() || t.dim() != dim || t.layout() != at::kStrided || t._fw_grad(0).defined()) return false;
  const c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  if (impl->is_python_dispatch()) return false;
  static const c10::DispatchKeySet other({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::Functionalize,
                                          c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                          c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::Batched,
                                          c10::DispatchKey::Negative});      // (the negative of its memory)
  return !impl->key_set().has_any(other);
}

bool operand_key(int64_t tag, const at::Tensor& a, const at::Tensor& b, Key* k) {
  std::memset(k, 0, sizeof *k);
  k->tag = tag;
  for (int i = 0; i < 2; ++i) {
    k->sizes[i] = a.size(i); k->sizes[2 + i] = b.size(i);
    k->strides[i] = a.stride(i); k->strides[2 + i] = b.stride(i);
  }
  k->type_a = (int32_t)a.scalar_type(); k->type_b = (int32_t)b.scalar_type();
  k->device = a.get_device();
  k->aligned = (((uintptr_t)a.data_ptr() | (uintptr_t)b.data_ptr()) & 15) == 0;
  return b.get_device() == k->device;
}

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, c10::DeviceIndex device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::DeviceType::CUDA, device)));
}

bool tensor_arg(PyObject* o) { return THPVariable_Check(o); }
// a torch.Tensor or Parameter itself: a subclass may answer the Python path's calls in its own way, and gives its type to a result
// that comes from one of its methods (new_empty)
bool own_tensor(PyObject* o) { return THPVariable_CheckExact(o); }

// The interpreter lock is given back while memory is allocated and the launch is queued: both may wait for the GPU (an allocation
// that frees cached blocks, a full queue), and what the GPU waits for may be a host function or a thread that needs the lock.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// None, whatever Exception is set (the ordinary path meets its cause again); an interrupt or an exit goes on its way
PyObject* none() {
  if (PyErr_Occurred() && !PyErr_ExceptionMatches(PyExc_Exception)) return nullptr;
  PyErr_Clear();
  Py_RETURN_NONE;
}

// bind(tnx_gemm, tnx_gemm_f32, tnx_conv2d_forward, workspace, failed): addresses of the entry points
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long g, f, c;
  PyObject *w, *e;
  if (!PyArg_ParseTuple(args, "KKKOO", &g, &f, &c, &w, &e)) return nullptr;
  fn_gemm = (decltype(fn_gemm))(uintptr_t)g;
  fn_gemm_f32 = (decltype(fn_gemm_f32))(uintptr_t)f;
  fn_conv = (decltype(fn_conv))(uintptr_t)c;
  Object workspace(w), failed(e);
  std::swap(fn_workspace, workspace.p);
  std::swap(fn_failed, failed.p);
  Py_RETURN_NONE;
}

// keep(tag, a, b, c, args, scratch, slices, atomic, memo key, config): the launch that gave c, from its argument struct's bytes
PyObject* keep(PyObject*, PyObject* args) {
  long long tag, scratch, slices;
  PyObject *a, *b, *c, *memo_key, *config;
  const char* bytes;
  Py_ssize_t len;
  int atomic;
  if (!PyArg_ParseTuple(args, "LOOOy#LLpOO", &tag, &a, &b, &c, &bytes, &len, &scratch, &slices, &atomic, &memo_key, &config)) return nullptr;
  if (len != (Py_ssize_t)sizeof(tnx_gemm_args) || !tensor_arg(a) || !tensor_arg(b) || !tensor_arg(c)) {
    PyErr_SetString(PyExc_ValueError, "keep: not an argument struct and its tensors");
    return nullptr;
  }
  try {
    const at::Tensor &ta = THPVariable_Unpack(a), &tb = THPVariable_Unpack(b), &tc = THPVariable_Unpack(c);
    Key k;
    if (!own_tensor(a) || !own_tensor(b) || !plain(ta, 2) || !plain(tb, 2) || !operand_key(tag, ta, tb, &k)) Py_RETURN_NONE;
    Product p;
    std::memcpy(&p.args, bytes, sizeof p.args);
    p.rows = tc.size(0); p.cols = tc.size(1);
    p.type = tc.scalar_type();
    p.scratch = scratch; p.slices = slices; p.atomic = atomic != 0;
    p.memo_key = Object(memo_key);
    p.config = Object(config);
    products[k] = std::move(p);
  } catch (...) {
    return none();
  }
  Py_RETURN_NONE;
}

// product(tag, a, b, memo, hooks) -> c, or None
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5 || !own_tensor(args[1]) || !own_tensor(args[2]) || !PyDict_Check(args[3]) || !PyList_Check(args[4]) ||
      PyList_GET_SIZE(args[4]) != 0)
    Py_RETURN_NONE;
  const long long tag = PyLong_AsLongLong(args[0]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor &a = THPVariable_Unpack(args[1]), &b = THPVariable_Unpack(args[2]);
    Key k;
    if (products.empty() || !plain(a, 2) || !plain(b, 2) || !operand_key(tag, a, b, &k)) Py_RETURN_NONE;
    const auto hit = products.find(k);
    if (hit == products.end()) Py_RETURN_NONE;
    // by value: the comparison and the workspace call below run Python, and the lock is given back, behind which the entry may be
    // forgotten
    const Product& kept = hit->second;
    const struct { int64_t rows, cols; at::ScalarType type; int64_t scratch, slices; bool atomic; } p = {
        kept.rows, kept.cols, kept.type, kept.scratch, kept.slices, kept.atomic};
    tnx_gemm_args g = kept.args;
    const Object memo_key(kept.memo_key.p), config(kept.config.p);
    PyObject* now = PyDict_GetItemWithError(args[3], memo_key.p);        // the config memo may hold another tile by now
    if (!now) return none();
    const Object held(now);
    if (PyObject_RichCompareBool(now, config.p, Py_EQ) != 1) return none();
    const c10::DeviceIndex device = (c10::DeviceIndex)k.device;
    if (c10::hip::current_device() != device) Py_RETURN_NONE;
    g.a = a.data_ptr(); g.b = b.data_ptr();
    g.stream = c10::hip::getCurrentHIPStream(device).stream();
    // held until the launch is queued: while the lock is given back another thread may have the buffer replaced by a larger one
    // or evicted, and a block that goes back to the stream's pool before then is handed out again -- to the result below, even
    Object workspace;
    if (p.slices > 0) {
      workspace = taken(PyObject_CallFunction(fn_workspace, "iKLi", (int)device, (unsigned long long)(uintptr_t)g.stream, (long long)p.slices, (int)p.atomic));
      if (!workspace.p || !tensor_arg(workspace.p)) return none();
      const at::Tensor& ws = THPVariable_Unpack(workspace.p);
      g.workspace = ws.data_ptr();
      g.workspace_bytes = (size_t)ws.nbytes();
    }
    at::Tensor c;
    int status;
    {
      const Unlocked unlocked;
      c = fresh({p.rows, p.cols}, p.type, device);
      g.c = c.data_ptr();
      if (g.in_dtype == TNX_F32) {
        at::Tensor scratch;
        if (p.scratch > 0) scratch = fresh({p.scratch}, at::kByte, device);
        status = fn_gemm_f32(&g, p.scratch > 0 ? scratch.data_ptr() : nullptr, (size_t)p.scratch);
      } else {
        status = fn_gemm(&g);
      }
    }
    if (status != TNX_OK) {
      taken(PyObject_CallFunction(fn_failed, "iKiy#", (int)device, (unsigned long long)(uintptr_t)g.stream, status, (const char*)&g, (Py_ssize_t)sizeof g));
      return PyErr_Occurred() ? nullptr : none();
    }
    return THPVariable_Wrap(c);
  } catch (...) {
    return none();
  }
}

bool pair_of(PyObject* t, int64_t* out) {
  if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != 2) return false;
  for (int i = 0; i < 2; ++i) {
    PyObject* v = PyTuple_GET_ITEM(t, i);
    if (!PyLong_CheckExact(v)) return false;
    out[i] = PyLong_AsLongLong(v);
  }
  return !PyErr_Occurred();
}

// (input, weight, bias or None, stride, padding, dilation) -> key; false: the ordinary path
bool conv_key(PyObject* const* args, Key* k) {
  if (!own_tensor(args[0]) || !own_tensor(args[1]) || !(args[2] == Py_None || own_tensor(args[2]))) return false;
  const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  if (!plain(x, 4) || !plain(w, 4) || !x.is_contiguous() || !w.is_contiguous()) return false;
  std::memset(k, 0, sizeof *k);
  for (int i = 0; i < 4; ++i) { k->sizes[i] = x.size(i); k->sizes[4 + i] = w.size(i); }
  for (int i = 0; i < 3; ++i)
    if (!pair_of(args[3 + i], k->options + 2 * i)) { PyErr_Clear(); return false; }
  k->type_a = (int32_t)x.scalar_type(); k->type_b = (int32_t)w.scalar_type();
  k->device = x.get_device();
  k->type_c = -1;
  if (w.get_device() != k->device) return false;
  if (args[2] != Py_None) {
    const at::Tensor& bias = THPVariable_Unpack(args[2]);
    if (!plain(bias, 1) || !bias.is_contiguous() || bias.get_device() != k->device) return false;
    k->type_c = (int32_t)bias.scalar_type();
    k->count_c = (int32_t)bias.numel();
  }
  return true;
}

// keep_conv(input, weight, bias, stride, padding, dilation, args, shape, scratch)
PyObject* keep_conv(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9 || !PyBytes_Check(args[6]) || PyBytes_GET_SIZE(args[6]) != (Py_ssize_t)sizeof(tnx_conv2d_args) || !PyTuple_Check(args[7]) ||
      PyTuple_GET_SIZE(args[7]) != 4) {
    PyErr_SetString(PyExc_ValueError, "keep_conv: not an argument struct, a shape and a size");
    return nullptr;
  }
  try {
    Key k;
    if (!conv_key(args, &k)) Py_RETURN_NONE;
    Conv p;
    std::memcpy(&p.args, PyBytes_AS_STRING(args[6]), sizeof p.args);
    for (int i = 0; i < 4; ++i) p.shape[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(args[7], i));
    p.scratch = PyLong_AsLongLong(args[8]);
    if (PyErr_Occurred()) return nullptr;
    convs[k] = p;
  } catch (...) {
    return none();
  }
  Py_RETURN_NONE;
}

// conv(input, weight, bias, stride, padding, dilation) -> output, or None
PyObject* conv(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6 || convs.empty()) Py_RETURN_NONE;
  try {
    Key k;
    if (!conv_key(args, &k)) Py_RETURN_NONE;
    const auto hit = convs.find(k);
    if (hit == convs.end()) Py_RETURN_NONE;
    const Conv p = hit->second;
    const c10::DeviceIndex device = (c10::DeviceIndex)k.device;
    if (c10::hip::current_device() != device) Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
    tnx_conv2d_args a = p.args;
    a.input = x.data_ptr(); a.weight = w.data_ptr();
    a.bias = args[2] == Py_None ? nullptr : THPVariable_Unpack(args[2]).data_ptr();
    a.stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor y;
    int status;
    {
      const Unlocked unlocked;
      y = fresh({p.shape[0], p.shape[1], p.shape[2], p.shape[3]}, (at::ScalarType)k.type_a, device);
      at::Tensor scratch;
      if (p.scratch > 0) {
        scratch = fresh({p.scratch}, at::kByte, device);
        a.workspace = scratch.data_ptr();
        a.workspace_bytes = (size_t)p.scratch;
      }
      a.output = y.data_ptr();
      status = fn_conv(&a);
    }
    if (status != TNX_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
  } catch (...) {
    return none();
  }
}

PyObject* forget(PyObject*, PyObject*) {
  products.clear();
  Py_RETURN_NONE;
}
PyObject* forget_convs(PyObject*, PyObject*) {
  convs.clear();
  Py_RETURN_NONE;
}

// the stream a launch on the device would go to, for tests
PyObject* stream_of(PyObject*, PyObject* arg) {
  const long index = PyLong_AsLong(arg);
  if (PyErr_Occurred()) return nullptr;
  return PyLong_FromUnsignedLongLong((unsigned long long)(uintptr_t)c10::hip::getCurrentHIPStream((c10::DeviceIndex)index).stream());
}

// ---------------------------------------------------------------------------------------------------------------------------
// Microscaled products and routing.  These calls have nothing to keep between them: the kernels' choice is the library's host arithmetic.
// What is saved is the interpreter's work around them, checks, torch.empty and the filling of structs: one token's routing 16.5 us -> 8.0, its
// product 10 -> 4.6, an ordinary product with its quantisation 16 -> 8.1.  As above, None hands the call to the ordinary path, which
// raises what is to be raised; a status other than TNX_OK does too (nothing is left behind by such a launch).
struct OpEntries {
  size_t (*code_bytes)(int64_t, int64_t);
  size_t (*scale_bytes)(int64_t, int64_t);
  int (*quantize)(const tnx_mx_args*);
  int (*quantize_both)(const tnx_mx_args*, void*, void*);
  int (*dequantize)(const tnx_mx_args*);
  int (*takes_rows)(int64_t, int64_t);
  int (*gemm)(const tnx_mx_gemm_args*);
  size_t (*gemm_workspace)(const tnx_mx_gemm_args*);
  size_t (*workspace_bytes)(int64_t, int32_t, int32_t);
  int (*route)(const tnx_moe_args*);
  int (*backward)(const tnx_moe_args*);
  int (*combine)(const void*, const int32_t*, const float*, void*, int64_t, int32_t, int64_t, int32_t, int32_t, void*);
} ops = {};
int64_t join_bytes = 0;

// bind_ops(addresses of the above, in their order, and the most bytes of a bfloat16 join's rows in 32 bits)
PyObject* bind_ops(PyObject*, PyObject* arg) {
  constexpr int N = sizeof(OpEntries) / sizeof(void*);
  if (!PyTuple_Check(arg) || PyTuple_GET_SIZE(arg) != N + 1) {
    PyErr_SetString(PyExc_ValueError, "bind_ops: not the entry points");
    return nullptr;
  }
  void* at[N];
  for (int i = 0; i < N; ++i) at[i] = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(arg, i));
  const long long most = PyLong_AsLongLong(PyTuple_GET_ITEM(arg, N));
  if (PyErr_Occurred()) return nullptr;
  join_bytes = most;
  static_assert(sizeof ops == sizeof at, "one pointer each");
  std::memcpy(&ops, at, sizeof ops);
  Py_RETURN_NONE;
}

// tnx_dtype of a float type that has kernels, or -1
int float_code(at::ScalarType t) {
  return t == at::kHalf ? TNX_F16 : t == at::kBFloat16 ? TNX_BF16 : t == at::kFloat ? TNX_F32 : -1;
}
at::ScalarType type_of(int code) { return code == TNX_F16 ? at::kHalf : code == TNX_BF16 ? at::kBFloat16 : at::kFloat; }

// integers from Python objects; false: not integers (and no error set)
template <int N> bool integers(PyObject* const* args, int64_t (&out)[N]) {
  for (int i = 0; i < N; ++i) {
    if (!PyLong_Check(args[i])) return false;
    out[i] = PyLong_AsLongLong(args[i]);
  }
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}

// a dense tensor of the current device; what it is for may be asked of it
bool here(PyObject* o, int64_t dim, const at::Tensor** t, c10::DeviceIndex* device) {
  if (!own_tensor(o)) return false;
  const at::Tensor& x = THPVariable_Unpack(o);
  if (!plain(x, dim)) return false;
  if (*device < 0) *device = (c10::DeviceIndex)x.get_device();
  *t = &x;
  return x.get_device() == *device && c10::hip::current_device() == *device;
}

// buffer of a quantised matrix of `rows` rows of k: codes, then scales
struct Quantised {
  at::Tensor buffer;
  int64_t code_bytes = 0;
  int status = TNX_OK;
};
Quantised room(int64_t rows, int64_t k, c10::DeviceIndex device) {
  Quantised q;
  q.code_bytes = (int64_t)ops.code_bytes(rows, k);
  q.buffer = fresh({q.code_bytes + (int64_t)ops.scale_bytes(rows, k)}, at::kByte, device);
  return q;
}
tnx_mx_args quantising(const at::Tensor& x, bool along_last, const Quantised& q, void* stream) {
  tnx_mx_args a = {};
  a.data = x.data_ptr();
  a.codes = q.buffer.data_ptr();
  a.scales = (uint8_t*)a.codes + q.code_bytes;
  a.batch = 1;
  a.rows = x.size(along_last ? 0 : 1); a.k = x.size(along_last ? 1 : 0);
  a.stride_row = x.stride(along_last ? 0 : 1); a.stride_k = x.stride(along_last ? 1 : 0);
  a.dtype = float_code(x.scalar_type());
  a.stream = stream;
  return a;
}
Quantised quantised(const at::Tensor& x, bool along_last, c10::DeviceIndex device, void* stream) {
  Quantised q = room(x.size(along_last ? 0 : 1), x.size(along_last ? 1 : 0), device);
  const tnx_mx_args a = quantising(x, along_last, q, stream);
  q.status = ops.quantize(&a);
  return q;
}
// along its last dimension, and along its first
struct QuantisedBoth {
  Quantised last, first;
};
QuantisedBoth quantised(const at::Tensor& x, bool last, bool first, c10::DeviceIndex device, void* stream) {
  if (!last || !first) return {last ? quantised(x, true, device, stream) : Quantised(), first ? quantised(x, false, device, stream) : Quantised()};
  QuantisedBoth b{room(x.size(0), x.size(1), device), room(x.size(1), x.size(0), device)};
  const tnx_mx_args a = quantising(x, true, b.last, stream);
  uint8_t* other = (uint8_t*)b.first.buffer.data_ptr();
  b.last.status = b.first.status = ops.quantize_both(&a, other, other + b.first.code_bytes);
  return b;
}

// the product, with the scratch that it is faster with
int multiply(tnx_mx_gemm_args* g, c10::DeviceIndex device) {
  const size_t bytes = ops.gemm_workspace(g);
  if (!bytes) return ops.gemm(g);
  const at::Tensor scratch = fresh({(int64_t)bytes}, at::kByte, device);
  g->workspace = scratch.data_ptr();
  g->workspace_bytes = bytes;
  return ops.gemm(g);
}

// mx_quantize(x, along its last dimension) -> (buffer, bytes of codes), or None
PyObject* mx_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) Py_RETURN_NONE;
  try {
    const at::Tensor* x;
    c10::DeviceIndex device = -1;
    if (!here(args[0], 2, &x, &device) || float_code(x->scalar_type()) < 0) Py_RETURN_NONE;
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    const bool along_last = PyObject_IsTrue(args[1]) == 1;
    Quantised q;
    {
      const Unlocked unlocked;
      q = quantised(*x, along_last, device, stream);
    }
    if (q.status != TNX_OK) Py_RETURN_NONE;
    const Object t = taken(THPVariable_Wrap(q.buffer)), bytes = taken(PyLong_FromLongLong(q.code_bytes));
    if (!t.p || !bytes.p) return nullptr;
    return PyTuple_Pack(2, t.p, bytes.p);
  } catch (...) {
    return none();
  }
}

// mx_dequantize(buffer, bytes of codes, rows, k, along its last dimension, tnx_dtype) -> the matrix, or None
PyObject* mx_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6) Py_RETURN_NONE;
  try {
    const at::Tensor* b;
    c10::DeviceIndex device = -1;
    int64_t v[5];
    if (!here(args[0], 1, &b, &device) || !integers(args + 1, v) || v[1] < 0 || v[2] < 0) Py_RETURN_NONE;
    tnx_mx_args a = {};
    a.codes = b->data_ptr();
    a.scales = (uint8_t*)a.codes + v[0];
    a.batch = 1; a.rows = v[1]; a.k = v[2];
    const bool along_last = v[3] != 0;
    a.stride_row = along_last ? v[2] : 1; a.stride_k = along_last ? 1 : v[1];
    a.dtype = (int32_t)v[4];
    a.stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor out;
    int status;
    {
      const Unlocked unlocked;
      out = fresh({along_last ? v[1] : v[2], along_last ? v[2] : v[1]}, type_of(a.dtype), device);
      a.data = out.data_ptr();
      status = ops.dequantize(&a);
    }
    if (status != TNX_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  } catch (...) {
    return none();
  }
}

// mx_product(a, buffer, bytes of codes, n, k, epilogue[, experts, top_k, offsets, order or None, rows or None, weights or None]) -> the product of
// the rows of a, quantised on the way in, or None.  With experts: of `order`'s pairs (gathered), or of a's rows as they lie, and
// with rows and weights the join of it
PyObject* mx_product(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6 && n != 12) Py_RETURN_NONE;
  try {
    const at::Tensor *a, *b, *offsets = nullptr, *order = nullptr, *rows = nullptr, *weights = nullptr;
    c10::DeviceIndex device = -1;
    int64_t v[4], ev[2] = {0, 1};
    if (!here(args[0], 2, &a, &device) || !here(args[1], 1, &b, &device) || !integers(args + 2, v)) Py_RETURN_NONE;
    const int code = float_code(a->scalar_type());
    const int64_t k = v[2], epilogue = v[3];
    if (code < 0 || a->size(1) != k || k <= 0 || (epilogue != TNX_EPI_NONE && v[1] % 2)) Py_RETURN_NONE;
    if (n == 12) {
      const int64_t most = a->size(0);
      if (!integers(args + 6, ev) || ev[0] <= 0 || ev[1] <= 0 || !here(args[8], 1, &offsets, &device) || offsets->numel() != ev[0] + 1 ||
          offsets->scalar_type() != at::kInt || !offsets->is_contiguous())
        Py_RETURN_NONE;
      if (args[9] != Py_None && (!here(args[9], 1, &order, &device) || order->numel() != most * ev[1] || order->scalar_type() != at::kInt || !order->is_contiguous()))
        Py_RETURN_NONE;
      if (args[10] != Py_None) {
        if (order || !here(args[10], 2, &rows, &device) || !here(args[11], 2, &weights, &device) || rows->numel() != most || rows->size(1) != ev[1] ||
            weights->sizes() != rows->sizes() || rows->scalar_type() != at::kInt || weights->scalar_type() != at::kFloat || !rows->is_contiguous() ||
            !weights->is_contiguous())
          Py_RETURN_NONE;
      }
    }
    tnx_mx_gemm_args g = {};
    g.b_codes = b->data_ptr();
    g.b_scales = (const uint8_t*)g.b_codes + v[0];
    g.a_rows = a->size(0);
    g.m = order ? order->numel() : g.a_rows;
    g.n = v[1]; g.k = k;
    g.stride_out = epilogue != TNX_EPI_NONE ? g.n / 2 : g.n;
    g.out_dtype = code; g.epilogue = (int32_t)epilogue;
    if (n == 12) {
      g.experts = (int32_t)ev[0]; g.top_k = (int32_t)ev[1];
      g.offsets = (const int32_t*)offsets->data_ptr();
      g.order = order ? (const int32_t*)order->data_ptr() : nullptr;
    }
    g.stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor out, joined;
    int status;
    {
      const Unlocked unlocked;
      Quantised q;
      if ((a->stride(1) == 1 || k == 1) && ops.takes_rows(g.a_rows, k)) {
        g.a_data = a->data_ptr(); g.a_dtype = code; g.stride_a = a->stride(0);
      } else {
        q = quantised(*a, true, device, g.stream);
        g.a_codes = q.buffer.data_ptr();
        g.a_scales = (const uint8_t*)g.a_codes + q.code_bytes;
      }
      // (the rows of a join: in 32 bits where moe.py has them so)
      if (rows && (code == TNX_F16 || g.m * g.n * 4 <= join_bytes)) g.out_dtype = TNX_F32;
      out = fresh({g.m, g.stride_out}, type_of(g.out_dtype), device);
      g.out = out.data_ptr();
      status = q.status != TNX_OK ? q.status : multiply(&g, device);
      if (status == TNX_OK && rows) {
        joined = fresh({rows->size(0), g.n}, a->scalar_type(), device);
        status = ops.combine(out.data_ptr(), (const int32_t*)rows->data_ptr(), (const float*)weights->data_ptr(), joined.data_ptr(), rows->size(0),
                             (int32_t)rows->size(1), g.n, g.out_dtype, code, g.stream);
      }
    }
    if (status != TNX_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(rows ? joined : out);
  } catch (...) {
    return none();
  }
}

// out[m, n] = a[m, k] b[k, n] of float tensors, both quantised along k
struct Multiplied {
  at::Tensor out;
  int status;
};
Multiplied multiplied(const Quantised& a, const Quantised& b, int64_t m, int64_t n, int64_t k, at::ScalarType type, c10::DeviceIndex device, void* stream) {
  Multiplied r{fresh({m, n}, type, device), a.status != TNX_OK ? a.status : b.status};
  if (r.status != TNX_OK) return r;
  tnx_mx_gemm_args g = {};
  g.a_codes = a.buffer.data_ptr(); g.a_scales = (const uint8_t*)g.a_codes + a.code_bytes;
  g.b_codes = b.buffer.data_ptr(); g.b_scales = (const uint8_t*)g.b_codes + b.code_bytes;
  g.out = r.out.data_ptr();
  g.m = g.a_rows = m; g.n = n; g.k = k; g.stride_out = n;
  g.out_dtype = float_code(type);
  g.stream = stream;
  r.status = multiply(&g, device);
  return r;
}

// What a backward pass returns, for a node of `inputs` inputs.  Where gradients of these gradients may be asked for, differentiating them is an error,
// not a silent zero.
torch::autograd::variable_list gradients(torch::autograd::variable_list out, size_t inputs, const char* message) {
  if (at::GradMode::is_enabled()) {
    for (at::Tensor& t : out)
      if (t.defined()) t.set_requires_grad(true);
    const int64_t count = (int64_t)out.size();
    out = (*std::make_shared<torch::autograd::DelayedError>(message, count))(std::move(out));
  }
  out.resize(inputs);
  return out;
}

// The training step of a linear layer as a node of the autograd graph: y = x w, dx = dy w^T, dw = x^T dy.  Each matrix is read once, for both of
// its quantisations; kept for the backward pass are the quantised x and w (17/32 of a byte an element) that its products take.
struct LinearStep : torch::autograd::Function<LinearStep> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, bool wants_dx, bool wants_dw) {
    const c10::DeviceIndex device = (c10::DeviceIndex)x.get_device();
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    const int64_t m = x.size(0), k = x.size(1), n = w.size(1);
    QuantisedBoth qx, qw;
    Multiplied y;
    {
      const Unlocked unlocked;
      qx = quantised(x, true, wants_dw, device, stream);
      qw = quantised(w, wants_dx, true, device, stream);
      y = multiplied(qx.last, qw.first, m, n, k, x.scalar_type(), device, stream);
    }
    if (y.status != TNX_OK || (wants_dw && qx.first.status != TNX_OK) || (wants_dx && qw.last.status != TNX_OK)) throw std::runtime_error("mx_linear");
    if (wants_dx || wants_dw) {
      ctx->save_for_backward({qx.first.buffer, qw.last.buffer});
      ctx->saved_data["m"] = m;
      ctx->saved_data["k"] = k;
      ctx->saved_data["n"] = n;
      ctx->saved_data["type"] = (int64_t)x.scalar_type();
    }
    return y.out;
  }
  // (on a thread of the engine's, with the streams and the device of the forward call)
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const at::Tensor& dy = grads[0];
    const auto saved = ctx->get_saved_variables();
    const int64_t m = ctx->saved_data["m"].toInt(), k = ctx->saved_data["k"].toInt(), n = ctx->saved_data["n"].toInt();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    TORCH_CHECK(plain(dy, 2) && dy.size(0) == m && dy.size(1) == n && dy.scalar_type() == type, "mx_linear: a gradient that is not an ordinary tensor of the result's size and type");
    const bool wants_dx = ctx->needs_input_grad(0) && saved[1].defined(), wants_dw = ctx->needs_input_grad(1) && saved[0].defined();
    const c10::DeviceIndex device = (c10::DeviceIndex)dy.get_device();
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    const QuantisedBoth qy = quantised(dy, wants_dx, wants_dw, device, stream);
    Multiplied dx{{}, TNX_OK}, dw{{}, TNX_OK};
    if (wants_dx) dx = multiplied(qy.last, {saved[1], (int64_t)ops.code_bytes(k, n), TNX_OK}, m, k, n, type, device, stream);
    if (wants_dw) dw = multiplied({saved[0], (int64_t)ops.code_bytes(k, m), TNX_OK}, qy.first, k, n, m, type, device, stream);
    TORCH_CHECK(dx.status == TNX_OK && dw.status == TNX_OK, "mx_linear: status ", dx.status != TNX_OK ? dx.status : dw.status, " in the backward pass");
    return gradients({dx.out, dw.out}, 4, "mx_linear has no second derivative");
  }
};

// mx_linear(x, w) -> x w with its place in the graph, or None
PyObject* mx_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) Py_RETURN_NONE;
  try {
    const at::Tensor *x, *w;
    c10::DeviceIndex device = -1;
    if (!here(args[0], 2, &x, &device) || !here(args[1], 2, &w, &device) || x->size(1) != w->size(0) || x->scalar_type() != w->scalar_type() ||
        float_code(x->scalar_type()) < 0 || x->numel() == 0 || w->numel() == 0)
      Py_RETURN_NONE;
    const bool graph = at::GradMode::is_enabled();
    return THPVariable_Wrap(LinearStep::apply(*x, *w, graph && x->requires_grad(), graph && w->requires_grad()));
  } catch (...) {
    return none();
  }
}

// weights, experts, offsets, order, rows of the routing that `a` describes
struct Routed {
  at::Tensor weights, experts, offsets, order, rows;
  int status;
};
Routed routed(tnx_moe_args a, c10::DeviceIndex device) {
  Routed r;
  r.weights = fresh({a.tokens, a.top_k}, at::kFloat, device);
  r.experts = fresh({a.tokens, a.top_k}, at::kInt, device);
  r.offsets = fresh({a.num_experts + 1}, at::kInt, device);
  r.order = fresh({a.tokens * a.top_k}, at::kInt, device);
  r.rows = fresh({a.tokens, a.top_k}, at::kInt, device);
  at::Tensor scratch;
  const size_t bytes = ops.workspace_bytes(a.tokens, a.top_k, a.num_experts);
  if (bytes) {
    scratch = fresh({(int64_t)bytes}, at::kByte, device);
    a.workspace = scratch.data_ptr();
    a.workspace_bytes = bytes;
  }
  a.weights = (float*)r.weights.data_ptr();
  a.experts = (int32_t*)r.experts.data_ptr();
  a.offsets = (int32_t*)r.offsets.data_ptr();
  a.order = (int32_t*)r.order.data_ptr();
  a.rows = (int32_t*)r.rows.data_ptr();
  r.status = ops.route(&a);
  return r;
}

// gradient of the logits; weights and experts [tokens, top_k] and grad of the same shape are contiguous
int route_gradient(const at::Tensor& logits, const at::Tensor& weights, const at::Tensor& experts, const at::Tensor& grad, int32_t scoring, int32_t renormalize,
                   float scale, c10::DeviceIndex device, void* stream, at::Tensor* out) {
  tnx_moe_args a = {};
  a.logits = logits.data_ptr();
  a.weights = (float*)weights.data_ptr();
  a.experts = (int32_t*)experts.data_ptr();
  a.grad = (const float*)grad.data_ptr();
  a.tokens = logits.size(0); a.stride_logits = logits.stride(0);
  a.num_experts = (int32_t)logits.size(1); a.top_k = (int32_t)weights.size(1); a.dtype = float_code(logits.scalar_type());
  a.scoring = scoring; a.renormalize = renormalize;
  a.num_groups = a.top_groups = a.group_top = 1;
  a.scale = scale;
  a.stream = stream;
  *out = fresh({a.tokens, a.num_experts}, logits.scalar_type(), device);
  a.grad_logits = out->data_ptr();
  return ops.backward(&a);
}

// The routing as a node of the autograd graph: the weights carry a gradient, the choice is held fixed
struct RouteStep : torch::autograd::Function<RouteStep> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const tnx_moe_args& a) {
    Routed r;
    {
      const Unlocked unlocked;
      r = routed(a, (c10::DeviceIndex)logits.get_device());
    }
    if (r.status != TNX_OK) throw std::runtime_error("moe_route");
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r.experts, r.offsets, r.order, r.rows});
    ctx->save_for_backward({logits, r.weights, r.experts});
    ctx->saved_data["scoring"] = (int64_t)a.scoring;
    ctx->saved_data["renormalize"] = (int64_t)a.renormalize;
    ctx->saved_data["scale"] = (double)a.scale;
    return {r.weights, r.experts, r.offsets, r.order, r.rows};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor()};
    const auto saved = ctx->get_saved_variables();
    TORCH_CHECK(plain(grads[0], 2) && grads[0].sizes() == saved[1].sizes(), "moe_route: a gradient that is not an ordinary tensor of the weights' size");
    const at::Tensor grad = grads[0].detach().to(at::kFloat).contiguous();
    const c10::DeviceIndex device = (c10::DeviceIndex)grad.get_device();
    at::Tensor out;
    const int status = route_gradient(saved[0], saved[1], saved[2], grad, (int32_t)ctx->saved_data["scoring"].toInt(), (int32_t)ctx->saved_data["renormalize"].toInt(),
                                      (float)ctx->saved_data["scale"].toDouble(), device, c10::hip::getCurrentHIPStream(device).stream(), &out);
    TORCH_CHECK(status == TNX_OK, "moe_route: status ", status, " in the backward pass");
    return gradients({out}, 2, "moe_route has no second derivative");
  }
};

// moe_route(logits, bias or None, top_k, scoring, num_groups, top_groups, group_top, renormalize, scale) -> (weights, experts, offsets, order,
// rows), the weights with their place in the graph, or None
PyObject* moe_route(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9 || !PyFloat_Check(args[8])) Py_RETURN_NONE;
  try {
    const at::Tensor *logits, *bias = nullptr;
    c10::DeviceIndex device = -1;
    int64_t v[6];
    if (!here(args[0], 2, &logits, &device) || !integers(args + 2, v)) Py_RETURN_NONE;
    if (args[1] != Py_None && (!here(args[1], 1, &bias, &device) || !bias->is_contiguous() || bias->scalar_type() != at::kFloat || bias->numel() != logits->size(1)))
      Py_RETURN_NONE;
    const int64_t tokens = logits->size(0), experts = logits->size(1), top_k = v[0];
    if (float_code(logits->scalar_type()) < 0 || experts < 1 || experts > TNX_MOE_MAX_EXPERTS || top_k < 1 || top_k > experts ||
        top_k > TNX_MOE_MAX_TOP_K || (logits->stride(1) != 1 && experts > 1))
      Py_RETURN_NONE;
    tnx_moe_args a = {};
    a.logits = logits->data_ptr();
    a.bias = bias ? (const float*)bias->data_ptr() : nullptr;
    a.tokens = tokens; a.stride_logits = logits->stride(0);
    a.num_experts = (int32_t)experts; a.top_k = (int32_t)top_k; a.dtype = float_code(logits->scalar_type());
    a.scoring = (int32_t)v[1]; a.num_groups = (int32_t)v[2]; a.top_groups = (int32_t)v[3]; a.group_top = (int32_t)v[4]; a.renormalize = (int32_t)v[5];
    a.scale = (float)PyFloat_AS_DOUBLE(args[8]);
    a.stream = c10::hip::getCurrentHIPStream(device).stream();
    Routed r;
    if (at::GradMode::is_enabled() && logits->requires_grad()) {
      const torch::autograd::variable_list out = RouteStep::apply(*logits, a);
      r = {out[0], out[1], out[2], out[3], out[4], TNX_OK};
    } else {
      const Unlocked unlocked;
      r = routed(a, device);
    }
    if (r.status != TNX_OK) Py_RETURN_NONE;
    const Object o[5] = {taken(THPVariable_Wrap(r.weights)), taken(THPVariable_Wrap(r.experts)), taken(THPVariable_Wrap(r.offsets)),
                         taken(THPVariable_Wrap(r.order)), taken(THPVariable_Wrap(r.rows))};
    for (const Object& x : o)
      if (!x.p) return nullptr;
    return PyTuple_Pack(5, o[0].p, o[1].p, o[2].p, o[3].p, o[4].p);
  } catch (...) {
    return none();
  }
}

// moe_backward(grad, logits, weights, experts, scoring, renormalize, scale) -> gradient of the logits, or None
PyObject* moe_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7 || !PyFloat_Check(args[6])) Py_RETURN_NONE;
  try {
    const at::Tensor *grad, *logits, *weights, *chosen;
    c10::DeviceIndex device = -1;
    int64_t v[2];
    if (!here(args[0], 2, &grad, &device) || !here(args[1], 2, &logits, &device) || !here(args[2], 2, &weights, &device) ||
        !here(args[3], 2, &chosen, &device) || !integers(args + 4, v))
      Py_RETURN_NONE;
    const int64_t tokens = logits->size(0), experts = logits->size(1);
    if (grad->sizes() != weights->sizes() || chosen->sizes() != weights->sizes() || weights->size(0) != tokens || grad->scalar_type() != at::kFloat ||
        weights->scalar_type() != at::kFloat || chosen->scalar_type() != at::kInt || !grad->is_contiguous() || !weights->is_contiguous() ||
        !chosen->is_contiguous() || (logits->stride(1) != 1 && experts > 1) || float_code(logits->scalar_type()) < 0)
      Py_RETURN_NONE;
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor out;
    int status;
    {
      const Unlocked unlocked;
      status = route_gradient(*logits, *weights, *chosen, *grad, (int32_t)v[0], (int32_t)v[1], (float)PyFloat_AS_DOUBLE(args[6]), device, stream, &out);
    }
    if (status != TNX_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  } catch (...) {
    return none();
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Linear layers, layer normalisation, grouped products: as above, with their nodes of the autograd graph.  A training step of a small
// layer (1025 x 770 x 514) is five launches of 5 to 12 us, 159 us a step through the interpreter and 79 us from here.  Matrices only: x of other dimensions is made one by
// ops/linear.py and ops/norm.py, which go on through the interpreter (1024 x 768 x 512 with gelu, a step: 71 us, of [8, 128, 512] 179; a token's call 7.0 and 14.6).
struct BlockEntries {
  size_t (*linear_workspace)(const tnx_linear_args*);
  size_t (*linear_scratch)(const tnx_linear_args*);
  int (*linear)(const tnx_linear_args*);
  size_t (*gradient_bytes)(const tnx_linear_gradient_args*);
  int (*gradient)(const tnx_linear_gradient_args*);
  int (*norm)(const tnx_norm_args*);
  size_t (*norm_workspace)(const tnx_norm_args*);
  int (*norm_backward)(const tnx_norm_args*);
  int (*grouped)(const tnx_grouped_args*);
  size_t (*grouped_workspace)(const tnx_grouped_args*);
} blocks = {};

// bind_blocks(addresses of the above, in their order)
PyObject* bind_blocks(PyObject*, PyObject* arg) {
  constexpr int N = sizeof(BlockEntries) / sizeof(void*);
  if (!PyTuple_Check(arg) || PyTuple_GET_SIZE(arg) != N) {
    PyErr_SetString(PyExc_ValueError, "bind_blocks: not the entry points");
    return nullptr;
  }
  void* at[N];
  for (int i = 0; i < N; ++i) at[i] = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(arg, i));
  if (PyErr_Occurred()) return nullptr;
  static_assert(sizeof blocks == sizeof at, "one pointer each");
  std::memcpy(&blocks, at, sizeof blocks);
  Py_RETURN_NONE;
}

// Scratch of products whose K is cut, its counters zero: a stream's own growing buffer (every launch leaves the counters zero).  Launches that
// are recorded into a HIP graph have one of the graph's memory (two graphs of one stream may be replayed on two), cleared by the first of a stream and
// capture: clearing it for each product of a graph took 3 us of 12.  Asked for without the interpreter lock, on any thread, with the
// stream the current one.
struct Counted {
  std::mutex lock;
  struct Entry {
    c10::DeviceIndex device;
    void* stream;
    unsigned long long capture;        // 0: none
    at::Tensor buffer;
    uint64_t used;
  };
  std::vector<Entry> entries;            // a program has few streams; the longest unused goes first
  uint64_t clock = 0;
  static at::Tensor made(int64_t bytes, c10::DeviceIndex device) {
    at::Tensor t = fresh({bytes}, at::kByte, device);
    t.narrow(0, 0, TNX_WS_COUNTER_BYTES).zero_();
    return t;
  }
  at::Tensor of(int64_t bytes, c10::DeviceIndex device, void* stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long capture = 0;
    if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &capture) != hipSuccess) {
      (void)hipGetLastError();
      return made(bytes, device);
    }
    if (status == hipStreamCaptureStatusNone) capture = 0;
    const std::lock_guard<std::mutex> held(lock);
    // (of an earlier capture: the graph keeps its memory, whose launches clear it with every replay)
    for (size_t i = 0; i < entries.size(); ++i)
      if (entries[i].device == device && entries[i].stream == stream && entries[i].capture && entries[i].capture != capture) entries.erase(entries.begin() + i--);
    for (Entry& e : entries)
      if (e.device == device && e.stream == stream && e.capture == capture) {
        if (e.buffer.numel() < bytes) e.buffer = made(bytes, device);
        e.used = ++clock;
        return e.buffer;
      }
    if (entries.size() >= 8) {
      size_t oldest = 0;
      for (size_t i = 1; i < entries.size(); ++i)
        if (entries[i].used < entries[oldest].used) oldest = i;
      entries.erase(entries.begin() + oldest);
    }
    entries.push_back({device, stream, capture, made(bytes < (1 << 20) ? 1 << 20 : bytes, device), ++clock});
    return entries.back().buffer;
  }
  void drop(c10::DeviceIndex device, void* stream) {
    const std::lock_guard<std::mutex> held(lock);
    for (size_t i = 0; i < entries.size(); ++i)
      if (entries[i].device == device && entries[i].stream == stream) entries.erase(entries.begin() + i--);
  }
};
Counted& counted_workspaces = *new Counted;      // never destroyed, as the tables above

// rows with neighbouring columns that do not overlap
bool row_major(const at::Tensor& t) { return (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) == 1 || t.stride(0) >= t.size(1)); }
bool column_major(const at::Tensor& t) { return t.stride(0) == 1 && t.stride(1) >= t.size(0); }

struct Made {
  at::Tensor y, z;
  int status = TNX_OK;
};
// y = act(x w + bias) + residual of operands as they lie, and z.  Called without the interpreter lock.
Made made_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor* bias, const at::Tensor* residual, int act, bool want_z, c10::DeviceIndex device,
                 void* stream) {
  tnx_linear_args a = {};
  a.x = x.data_ptr(); a.w = w.data_ptr();
  a.m = x.size(0); a.k = x.size(1); a.n = w.size(1);
  a.stride_xm = a.m == 1 ? a.k : x.stride(0); a.stride_xk = a.k == 1 ? 1 : x.stride(1);
  a.stride_wn = a.n == 1 ? 1 : w.stride(1);
  a.stride_wk = a.k == 1 && a.stride_wn == 1 ? a.n : w.stride(0);
  a.dtype = float_code(x.scalar_type());
  if (bias) { a.bias = bias->data_ptr(); a.bias_dtype = float_code(bias->scalar_type()); }
  if (residual) a.residual = residual->data_ptr();
  a.activation = act;
  a.stream = stream;
  Made r;
  r.y = fresh({a.m, a.n}, x.scalar_type(), device);
  if (want_z) r.z = fresh({a.m, a.n}, x.scalar_type(), device);
  a.y = r.y.data_ptr();
  a.z = want_z ? r.z.data_ptr() : nullptr;
  const size_t counted = blocks.linear_workspace(&a), bytes = blocks.linear_scratch(&a);
  at::Tensor ws, scratch;
  if (counted) {
    ws = counted_workspaces.of((int64_t)counted, device, stream);        // (held until the launch is queued)
    a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.nbytes();
  }
  if (bytes) {
    scratch = fresh({(int64_t)bytes}, at::kByte, device);
    a.scratch = scratch.data_ptr(); a.scratch_bytes = bytes;
  }
  r.status = blocks.linear(&a);
  if (r.status == TNX_E_HIP && counted) counted_workspaces.drop(device, stream);
  return r;
}

at::Tensor product_of(const at::Tensor& a, const at::Tensor& b, c10::DeviceIndex device, void* stream) {
  const at::Tensor x = row_major(a) || column_major(a) ? a : a.contiguous(), w = row_major(b) || column_major(b) ? b : b.contiguous();
  Made r = made_linear(x, w, nullptr, nullptr, TNX_ACT_NONE, false, device, stream);
  TORCH_CHECK(r.status == TNX_OK, "linear: status ", r.status, " in the backward pass");
  return r.y;
}

typedef std::optional<at::Tensor> MaybeTensor;

// What a node keeps of its forward call beside tensors: that it had a residual; that its weights are k-contiguous, transposes of row-major ones, and their gradient is to
// lie so too; the result's type and columns.
enum { HAS_RESIDUAL = 1, TRANSPOSED = 2 };
bool transposed(const at::Tensor& w) { return w.stride(-2) == 1 && w.stride(-1) != 1; }
int64_t what_of(const at::Tensor& y, int64_t flags) { return flags | (int64_t)y.scalar_type() << 8 | y.size(1) << 16; }
bool fits(const at::Tensor& dy, int64_t what) { return plain(dy, 2) && dy.size(1) == what >> 16 && (int64_t)dy.scalar_type() == (what >> 8 & 255); }

struct LinearLayer : torch::autograd::Function<LinearLayer> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const MaybeTensor& bias, const MaybeTensor& residual,
                            int64_t act) {
    const c10::DeviceIndex device = (c10::DeviceIndex)x.get_device();
    const bool derived = act != TNX_ACT_NONE && (x.requires_grad() || w.requires_grad() || (bias && bias->requires_grad()));
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    Made r;
    {
      const Unlocked unlocked;
      r = made_linear(x, w, bias ? &*bias : nullptr, residual ? &*residual : nullptr, (int)act, derived, device, stream);
    }
    if (r.status != TNX_OK) throw std::runtime_error("linear");
    ctx->set_materialize_grads(false);
    // (what no gradient that is asked for reads is not kept: it may change before the backward pass)
    ctx->save_for_backward({w.requires_grad() ? x : at::Tensor(), x.requires_grad() ? w : at::Tensor(), r.z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias ? (int64_t)bias->scalar_type() : (int64_t)-1;
    ctx->saved_data["what"] = what_of(r.y, (residual ? HAS_RESIDUAL : 0) | (transposed(w) ? TRANSPOSED : 0));
    return r.y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return torch::autograd::variable_list(5);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &z = saved[2];
    const int64_t what = ctx->saved_data["what"].toInt();
    const at::Tensor resolved = grads[0].resolve_neg(), given = resolved.detach();
    TORCH_CHECK(fits(resolved, what), "linear: a gradient that is not an ordinary tensor of the result's size and type");
    const int act = (int)ctx->saved_data["act"].toInt();
    const int64_t bias_type = ctx->saved_data["bias"].toInt();
    // (inputs that were not given are not counted)
    const bool wants_x = ctx->needs_input_grad(0), wants_w = ctx->needs_input_grad(1), wants_bias = bias_type >= 0 && ctx->needs_input_grad(2);
    const bool wants_residual = (what & HAS_RESIDUAL) && ctx->needs_input_grad(bias_type >= 0 ? 3 : 2);
    const c10::DeviceIndex device = (c10::DeviceIndex)given.get_device();
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor dx, dw, dbias;
    if (wants_x || wants_w || wants_bias) {
      const at::Tensor dy = given.contiguous();
      at::Tensor dz = dy;
      if (act != TNX_ACT_NONE || wants_bias) {
        tnx_linear_gradient_args a = {};
        a.dy = dy.data_ptr();
        a.m = dy.size(0); a.n = dy.size(1);
        a.dtype = float_code(dy.scalar_type());
        a.activation = act;
        if (act != TNX_ACT_NONE) {
          a.z = z.data_ptr();
          if (wants_x || wants_w) {
            dz = fresh({a.m, a.n}, dy.scalar_type(), device);
            a.dz = dz.data_ptr();
          }
        }
        if (wants_bias) {
          dbias = fresh({a.n}, (at::ScalarType)bias_type, device);
          a.dbias = dbias.data_ptr();
          a.bias_dtype = float_code((at::ScalarType)bias_type);
        }
        at::Tensor scratch;
        if (const size_t bytes = blocks.gradient_bytes(&a)) {
          scratch = fresh({(int64_t)bytes}, at::kByte, device);
          a.workspace = scratch.data_ptr(); a.workspace_bytes = bytes;
        }
        a.stream = stream;
        const int status = blocks.gradient(&a);
        TORCH_CHECK(status == TNX_OK, "linear: status ", status, " in the backward pass");
      }
      if (wants_x) dx = product_of(dz, w.t(), device, stream);
      // (a weight that is the transpose of a row-major one has its gradient so too)
      if (wants_w) dw = what & TRANSPOSED ? product_of(dz.t(), x, device, stream).t() : product_of(x.t(), dz, device, stream);
    }
    torch::autograd::variable_list out = gradients({dx, dw, dbias}, 5, "linear has no second derivative");
    // (the gradient itself, not another tensor of its memory: who takes it as his own looks whether others hold the tensor)
    if (wants_residual) out[3] = grads[0];
    return out;
  }
};

// linear(x, w, bias or None, residual or None, tnx_activation) -> y with its place in the graph, or None
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) Py_RETURN_NONE;
  try {
    const at::Tensor *x, *w, *bias = nullptr, *residual = nullptr;
    c10::DeviceIndex device = -1;
    int64_t v[1];
    if (!here(args[0], 2, &x, &device) || !here(args[1], 2, &w, &device) || !integers(args + 4, v)) Py_RETURN_NONE;
    const at::ScalarType type = x->scalar_type();
    if (x->size(1) != w->size(0) || type != w->scalar_type() || float_code(type) < 0 || x->numel() == 0 || w->size(0) < 16 || w->size(1) < 16 || !row_major(*x) ||
        !(row_major(*w) || column_major(*w)))
      Py_RETURN_NONE;
    if (args[2] != Py_None && (!here(args[2], 1, &bias, &device) || bias->size(0) != w->size(1) || !bias->is_contiguous() ||
                               (bias->scalar_type() != type && bias->scalar_type() != at::kFloat)))
      Py_RETURN_NONE;
    if (args[3] != Py_None && (!here(args[3], 2, &residual, &device) || residual->size(0) != x->size(0) || residual->size(1) != w->size(1) ||
                               !residual->is_contiguous() || residual->scalar_type() != type))
      Py_RETURN_NONE;
    if (at::GradMode::is_enabled() && (x->requires_grad() || w->requires_grad() || (bias && bias->requires_grad()) || (residual && residual->requires_grad())))
      return THPVariable_Wrap(LinearLayer::apply(*x, *w, bias ? MaybeTensor(*bias) : MaybeTensor(), residual ? MaybeTensor(*residual) : MaybeTensor(), v[0]));
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    Made r;
    {
      const Unlocked unlocked;
      r = made_linear(*x, *w, bias, residual, (int)v[0], false, device, stream);
    }
    if (r.status != TNX_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(r.y);
  } catch (...) {
    return none();
  }
}

tnx_norm_args norm_args(const at::Tensor& x, const at::Tensor* weight, const at::Tensor* bias, float eps, void* stream) {
  tnx_norm_args a = {};
  a.x = x.data_ptr();
  a.rows = x.size(0); a.n = x.size(1); a.stride_x = x.stride(0);
  a.dtype = float_code(x.scalar_type());
  a.eps = eps;
  if (weight) { a.weight = weight->data_ptr(); a.weight_dtype = float_code(weight->scalar_type()); }
  if (bias) { a.bias = bias->data_ptr(); a.bias_dtype = float_code(bias->scalar_type()); }
  a.stream = stream;
  return a;
}

struct NormLayer : torch::autograd::Function<NormLayer> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
    const c10::DeviceIndex device = (c10::DeviceIndex)x.get_device();
    tnx_norm_args a = norm_args(x, weight ? &*weight : nullptr, bias ? &*bias : nullptr, (float)eps, c10::hip::getCurrentHIPStream(device).stream());
    at::Tensor y, statistics;
    int status;
    {
      const Unlocked unlocked;
      y = fresh({a.rows, a.n}, x.scalar_type(), device);
      statistics = fresh({2, a.rows}, at::kFloat, device);
      a.y = y.data_ptr();
      a.mean = (float*)statistics.data_ptr();
      a.rstd = a.mean + a.rows;
      status = blocks.norm(&a);
    }
    if (status != TNX_OK) throw std::runtime_error("layer_norm");
    ctx->set_materialize_grads(false);
    // (x where dx or dweight is asked for, weight where dx is: what neither reads may change before the backward pass)
    const bool own = x.requires_grad();
    ctx->save_for_backward({own || (weight && weight->requires_grad()) ? x : at::Tensor(), own && weight ? *weight : at::Tensor(), statistics});
    ctx->saved_data["what"] = what_of(y, 0);
    ctx->saved_data["weight"] = weight ? (int64_t)weight->scalar_type() : (int64_t)-1;
    ctx->saved_data["bias"] = bias ? (int64_t)bias->scalar_type() : (int64_t)-1;
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return torch::autograd::variable_list(4);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &statistics = saved[2];
    const int64_t weight_type = ctx->saved_data["weight"].toInt(), bias_type = ctx->saved_data["bias"].toInt();
    const at::Tensor resolved = grads[0].resolve_neg(), given = resolved.detach();
    TORCH_CHECK(fits(resolved, ctx->saved_data["what"].toInt()) && given.size(0) == statistics.size(1),
                "layer_norm: a gradient that is not an ordinary tensor of the result's size and type");
    const at::Tensor dy = given.stride(1) == 1 || given.size(1) <= 1 ? given : given.contiguous();
    const c10::DeviceIndex device = (c10::DeviceIndex)dy.get_device();
    // (where only the bias asks, dx and dweight are not written and their sums not looked at: dy stands in for x)
    tnx_norm_args a = norm_args(x.defined() ? x : dy, weight.defined() ? &weight : nullptr, nullptr, 0.0f, c10::hip::getCurrentHIPStream(device).stream());
    a.mean = (float*)statistics.data_ptr();
    a.rstd = a.mean + a.rows;
    a.dy = dy.data_ptr();
    a.stride_dy = dy.stride(0);
    at::Tensor dx, dweight, dbias, scratch;
    if (ctx->needs_input_grad(0)) {
      dx = fresh({a.rows, a.n}, dy.scalar_type(), device);
      a.dx = dx.data_ptr();
    }
    if (weight_type >= 0 && ctx->needs_input_grad(1)) {
      dweight = fresh({a.n}, (at::ScalarType)weight_type, device);
      a.dweight = dweight.data_ptr();
      a.weight_dtype = float_code((at::ScalarType)weight_type);
    }
    if (bias_type >= 0 && ctx->needs_input_grad(weight_type >= 0 ? 2 : 1)) {       // (inputs that were not given are not counted)
      dbias = fresh({a.n}, (at::ScalarType)bias_type, device);
      a.dbias = dbias.data_ptr();
      a.bias_dtype = float_code((at::ScalarType)bias_type);
    }
    if (const size_t bytes = blocks.norm_workspace(&a)) {
      scratch = fresh({(int64_t)bytes}, at::kByte, device);
      a.workspace = scratch.data_ptr(); a.workspace_bytes = bytes;
    }
    const int status = blocks.norm_backward(&a);
    TORCH_CHECK(status == TNX_OK, "layer_norm: status ", status, " in the backward pass");
    return gradients({dx, dweight, dbias}, 4, "layer_norm has no second derivative");
  }
};

// layer_norm(x, weight or None, bias or None, eps) -> y with its place in the graph, or None
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || !PyFloat_Check(args[3])) Py_RETURN_NONE;
  try {
    const at::Tensor *x, *p[2] = {nullptr, nullptr};
    c10::DeviceIndex device = -1;
    const double eps = PyFloat_AS_DOUBLE(args[3]);
    if (!here(args[0], 2, &x, &device) || float_code(x->scalar_type()) < 0 || x->numel() == 0 || !(x->stride(1) == 1 || x->size(1) == 1) || !(eps >= 0.0))
      Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i) {
      if (args[1 + i] == Py_None) continue;
      if (!here(args[1 + i], 1, &p[i], &device) || p[i]->size(0) != x->size(1) || !p[i]->is_contiguous() ||
          (p[i]->scalar_type() != x->scalar_type() && p[i]->scalar_type() != at::kFloat))
        Py_RETURN_NONE;
    }
    if (at::GradMode::is_enabled() && (x->requires_grad() || (p[0] && p[0]->requires_grad()) || (p[1] && p[1]->requires_grad())))
      return THPVariable_Wrap(NormLayer::apply(*x, p[0] ? MaybeTensor(*p[0]) : MaybeTensor(), p[1] ? MaybeTensor(*p[1]) : MaybeTensor(), eps));
    tnx_norm_args a = norm_args(*x, p[0], p[1], (float)eps, c10::hip::getCurrentHIPStream(device).stream());
    at::Tensor y;
    int status;
    {
      const Unlocked unlocked;
      y = fresh({a.rows, a.n}, x->scalar_type(), device);
      a.y = y.data_ptr();
      status = blocks.norm(&a);
    }
    if (status != TNX_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
  } catch (...) {
    return none();
  }
}

// Operands of a grouped product as they lie: a with rows that do not overlap, matrices that are row-major or k-contiguous.
bool grouped_weights(const at::Tensor& w) {
  return (w.stride(2) == 1 && w.stride(1) >= w.size(2)) || (w.stride(1) == 1 && w.stride(2) >= w.size(1));
}
tnx_grouped_args grouped_args(int form, const at::Tensor& a, const at::Tensor& b, const at::Tensor& offsets, int64_t n, int64_t k, int64_t group, int64_t bk,
                              int64_t bn, void* stream) {
  tnx_grouped_args g = {};
  g.a = a.data_ptr(); g.b = b.data_ptr();
  g.offsets = (const int32_t*)offsets.data_ptr();
  g.rows = a.size(0); g.n = n; g.k = k;
  g.stride_ar = a.size(0) == 1 ? a.size(1) : a.stride(0); g.stride_ak = 1;
  g.stride_group = group; g.stride_bk = bk; g.stride_bn = bn;
  g.groups = (int32_t)(offsets.numel() - 1); g.dtype = float_code(a.scalar_type()); g.form = form;
  g.stream = stream;
  return g;
}
// the product, with the scratch that it is faster with
int grouped_launch(tnx_grouped_args* g, c10::DeviceIndex device) {
  at::Tensor scratch;
  if (const size_t bytes = blocks.grouped_workspace(g)) {
    scratch = fresh({(int64_t)bytes}, at::kByte, device);
    g->workspace = scratch.data_ptr(); g->workspace_bytes = bytes;
  }
  return blocks.grouped(g);
}
int rows_product(const at::Tensor& x, const at::Tensor& w, const at::Tensor& offsets, c10::DeviceIndex device, void* stream, at::Tensor* y) {
  tnx_grouped_args g = grouped_args(TNX_GROUPED_ROWS, x, w, offsets, w.size(2), x.size(1), w.stride(0), w.stride(1), w.stride(2), stream);
  *y = fresh({g.rows, g.n}, x.scalar_type(), device);
  g.c = y->data_ptr();
  return grouped_launch(&g, device);
}
int weight_gradient(const at::Tensor& x, const at::Tensor& dy, const at::Tensor& offsets, c10::DeviceIndex device, void* stream, at::Tensor* dw) {
  const int64_t k = x.size(1), n = dy.size(1);
  tnx_grouped_args g = grouped_args(TNX_GROUPED_WEIGHT_GRADIENT, x, dy, offsets, n, k, k * n, dy.size(0) == 1 ? n : dy.stride(0), 1, stream);
  *dw = fresh({(int64_t)g.groups, k, n}, x.scalar_type(), device);
  g.c = dw->data_ptr();
  return grouped_launch(&g, device);
}

struct GroupedProduct : torch::autograd::Function<GroupedProduct> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& offsets) {
    const c10::DeviceIndex device = (c10::DeviceIndex)x.get_device();
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor y;
    int status;
    {
      const Unlocked unlocked;
      status = rows_product(x, w, offsets, device, stream, &y);
    }
    if (status != TNX_OK) throw std::runtime_error("grouped_matmul");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({w.requires_grad() ? x : at::Tensor(), x.requires_grad() ? w : at::Tensor(), offsets});
    ctx->saved_data["what"] = what_of(y, transposed(w) ? TRANSPOSED : 0);
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return torch::autograd::variable_list(3);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &offsets = saved[2];
    const int64_t what = ctx->saved_data["what"].toInt();
    const at::Tensor resolved = grads[0].resolve_neg();
    at::Tensor dy = resolved.detach();
    TORCH_CHECK(fits(resolved, what), "grouped_matmul: a gradient that is not an ordinary tensor of the result's size and type");
    if (!row_major(dy)) dy = dy.contiguous();
    const c10::DeviceIndex device = (c10::DeviceIndex)dy.get_device();
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor dx, dw;
    int status = TNX_OK;
    if (ctx->needs_input_grad(0)) status = rows_product(dy, w.transpose(1, 2), offsets, device, stream, &dx);
    if (status == TNX_OK && ctx->needs_input_grad(1)) {
      // (as a linear layer's)
      const bool turned = what & TRANSPOSED;
      status = turned ? weight_gradient(dy, x, offsets, device, stream, &dw) : weight_gradient(x, dy, offsets, device, stream, &dw);
      if (turned) dw = dw.transpose(1, 2);
    }
    TORCH_CHECK(status == TNX_OK, "grouped_matmul: status ", status, " in the backward pass");
    return gradients({dx, dw}, 3, "grouped_matmul has no second derivative");
  }
};

// grouped_matmul(x, w, offsets) -> y with its place in the graph, or None
PyObject* grouped_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) Py_RETURN_NONE;
  try {
    const at::Tensor *x, *w, *offsets;
    c10::DeviceIndex device = -1;
    if (!here(args[0], 2, &x, &device) || !here(args[1], 3, &w, &device) || !here(args[2], 1, &offsets, &device)) Py_RETURN_NONE;
    // (rows shorter than a chunk may have to be padded)
    if (x->size(1) != w->size(1) || w->size(1) < 8 || w->size(2) < 8 || x->size(0) == 0 || w->size(0) < 1 || w->size(0) > TNX_GROUPED_MAX_GROUPS ||
        offsets->size(0) != w->size(0) + 1 || (offsets->scalar_type() != at::kInt && offsets->scalar_type() != at::kLong) || !offsets->is_contiguous() ||
        float_code(x->scalar_type()) < 0 || w->scalar_type() != x->scalar_type() || !row_major(*x) || !grouped_weights(*w))
      Py_RETURN_NONE;
    at::Tensor narrowed;
    if (offsets->scalar_type() == at::kLong) {            // (past 32 bits: the nearest inside)
      narrowed = at::clamp(*offsets, 0, x->size(0)).to(at::kInt);
      offsets = &narrowed;
    }
    if (at::GradMode::is_enabled() && (x->requires_grad() || w->requires_grad())) return THPVariable_Wrap(GroupedProduct::apply(*x, *w, *offsets));
    void* stream = c10::hip::getCurrentHIPStream(device).stream();
    at::Tensor y;
    int status;
    {
      const Unlocked unlocked;
      status = rows_product(*x, *w, *offsets, device, stream, &y);
    }
    if (status != TNX_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
  } catch (...) {
    return none();
  }
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"keep", keep, METH_VARARGS, nullptr},
    {"product", (PyCFunction)(void (*)(void))product, METH_FASTCALL, nullptr},
    {"keep_conv", (PyCFunction)(void (*)(void))keep_conv, METH_FASTCALL, nullptr},
    {"conv", (PyCFunction)(void (*)(void))conv, METH_FASTCALL, nullptr},
    {"forget", forget, METH_NOARGS, nullptr},
    {"forget_convs", forget_convs, METH_NOARGS, nullptr},
    {"stream_of", stream_of, METH_O, nullptr},
    {"bind_ops", bind_ops, METH_O, nullptr},
    {"mx_quantize", (PyCFunction)(void (*)(void))mx_quantize, METH_FASTCALL, nullptr},
    {"mx_dequantize", (PyCFunction)(void (*)(void))mx_dequantize, METH_FASTCALL, nullptr},
    {"mx_product", (PyCFunction)(void (*)(void))mx_product, METH_FASTCALL, nullptr},
    {"mx_linear", (PyCFunction)(void (*)(void))mx_linear, METH_FASTCALL, nullptr},
    {"moe_route", (PyCFunction)(void (*)(void))moe_route, METH_FASTCALL, nullptr},
    {"moe_backward", (PyCFunction)(void (*)(void))moe_backward, METH_FASTCALL, nullptr},
    {"bind_blocks", bind_blocks, METH_O, nullptr},
    {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr},
    {"layer_norm", (PyCFunction)(void (*)(void))layer_norm, METH_FASTCALL, nullptr},
    {"grouped_matmul", (PyCFunction)(void (*)(void))grouped_matmul, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__launch() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {      // whose classes it was compiled against
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
