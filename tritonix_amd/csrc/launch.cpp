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

// an ordinary dense tensor on the GPU: nothing that intercepts the calls the Python path would make of it
bool plain(const at::Tensor& t, int64_t dim) {
  if (!t.defined() || !t.is_cuda() || t.dim() != dim || t.layout() != at::kStrided) return false;
  const c10::TensorImpl* impl = t.unsafeGetTensorImpl();
  if (impl->is_python_dispatch()) return false;
  static const c10::DispatchKeySet other({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::Functionalize,
                                          c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                          c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::Batched});
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
