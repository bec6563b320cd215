// The operators' call path in native code: a CPython module over the C ABI for torch tensors.
//
// A call on one short sequence is a few microseconds of device time; argument checks, output allocation and the
// ctypes call in Python took 13 of the 15 us such a call cost.  The functions here do the same checks on the C++
// tensors, allocate the result (and scratch memory) from torch's caching allocator and call the C ABI: about 4 us,
// half of it the launch itself.
//
// Only the straight path lives here.  Whatever is out of the ordinary -- a wrong type or shape, a tensor on another
// device, an error code -- makes a function return None without having launched anything (or after a failed
// launch), and the caller in ops.py goes through its checks again and reports what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ditto_b200.h"

#include <algorithm>
#include <climits>
#include <cstring>
#include <initializer_list>
#include <string_view>
#include <type_traits>
#include <vector>

namespace {

using SoftmaxFn = int (*)(const void*, const void*, const void*, void*, int, int, int, int, int, int, int, float, int, void*,
                          size_t, int*, void*);
using MhaFn = int (*)(const void*, void*, int, int, int, int, int, float, int, int*, void*);
using GemmFn = int (*)(const void*, const void*, const void*, void*, int, int, int, int, int, int, int, int, void*, size_t,
                       int*, void*);
using FfnFn = int (*)(const void*, const void*, const void*, const void*, const void*, void*, int, int, int, int, int, int,
                      int, int, int, void*, size_t, int*, void*);
using BytesFn = size_t (*)(int, int, int, int, int, int, int);

SoftmaxFn g_softmax = nullptr;
MhaFn g_mha = nullptr;
GemmFn g_gemm = nullptr;
FfnFn g_ffn = nullptr;
BytesFn g_bytes = nullptr;
constexpr int kDevices = 64;
int* g_status[kDevices] = {};       // device status words, registered by ops.py

constexpr int kOpGemmReluGemm = 1, kOpLessScratch = 0x2000;

// What all tensors of a call have in common.
struct Common {
  int device = -1;
  at::ScalarType type = at::ScalarType::Undefined;
  int code = 0;
};

// The tensor behind `o` if it is a contiguous CUDA tensor that fits the call so far (the first one decides type and
// device: 16-bit floating point, on the current device).
const at::Tensor* take(PyObject* o, Common& c) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous()) return nullptr;
  const int dev = t.device().index();
  const at::ScalarType st = t.scalar_type();
  if (c.device < 0) {
    if (st == at::kHalf) c.code = 0;
    else if (st == at::kBFloat16) c.code = 1;
    else return nullptr;
    if (dev < 0 || dev >= kDevices || g_status[dev] == nullptr || dev != c10::cuda::current_device()) return nullptr;
    c.device = dev;
    c.type = st;
  } else if (dev != c.device || st != c.type) {
    return nullptr;
  }
  return &t;
}

bool fits(std::initializer_list<int64_t> v) {
  for (int64_t x : v)
    if (x < 0 || x > INT_MAX) return false;
  return true;
}

bool is_text(PyObject* o, const char* s) { return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, s) == 0; }

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)), std::nullopt);
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

bool shape_is(const at::Tensor& t, int64_t a, int64_t b, int64_t c) {
  return t.dim() == 3 && t.size(0) == a && t.size(1) == b && t.size(2) == c;
}

// A pair of two new references.
PyObject* pair_of(PyObject* first, PyObject* second) {
  PyObject* t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, first);
  PyTuple_SET_ITEM(t, 1, second);
  return t;
}

// Lets other Python threads run: around allocations and launches, which can block (a full launch queue, cudaMalloc, a queue that
// waits for a Python host callback).  Everything taken from Python objects -- addresses, shapes, texts -- is read before.
struct WithoutLock {
  PyThreadState* state = PyEval_SaveThread();
  WithoutLock() = default;
  WithoutLock(const WithoutLock&) = delete;
  WithoutLock& operator=(const WithoutLock&) = delete;
  ~WithoutLock() { PyEval_RestoreThread(state); }
};

// Runs `body` and returns what it returns; None for nullptr or an exception.
template <class F>
PyObject* guarded(F body) {
  try {
    PyObject* r = body();
    if (r != nullptr) return r;
  } catch (...) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

// The result: `given`, checked by the caller, or a new tensor.
class Result {
 public:
  Result(PyObject* given, const at::Tensor* t) : given_(given), address_(t ? t->data_ptr() : nullptr) {}
  // its address; allocates a new one (without the lock)
  void* address(const Common& c, at::IntArrayRef shape) {
    if (given_ != Py_None) return address_;
    fresh_ = make(shape, c.type, c.device);
    return fresh_.data_ptr();
  }
  PyObject* give() {
    if (given_ == Py_None) return THPVariable_Wrap(fresh_);
    Py_INCREF(given_);
    return given_;
  }

 private:
  PyObject* given_;
  void* address_;
  at::Tensor fresh_;
};

// Whether `given` can be the result; `t` is the tensor behind it (null for None).
bool result_ok(PyObject* given, Common& c, at::IntArrayRef shape, const at::Tensor** t) {
  *t = nullptr;
  if (given == Py_None) return true;
  *t = take(given, c);
  return *t != nullptr && (*t)->sizes() == shape;
}

// softmax(query, key, value, out, scale, key_layout, flags)
PyObject* py_softmax(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7 || g_softmax == nullptr) return nullptr;
    Common c;
    const at::Tensor *q = take(a[0], c), *k = q ? take(a[1], c) : nullptr, *v = k ? take(a[2], c) : nullptr;
    if (v == nullptr || q->dim() != 3 || k->dim() != 3 || v->dim() != 3) return nullptr;
    int layout;
    if (is_text(a[5], "LK")) layout = 1;
    else if (is_text(a[5], "KL")) layout = 0;
    else return nullptr;
    const int64_t b = q->size(0), M = q->size(1), K = q->size(2), L = v->size(1), N = v->size(2);
    if (!(layout ? shape_is(*k, b, L, K) : shape_is(*k, b, K, L)) || v->size(0) != b || !fits({b, M, N, K, L})) return nullptr;
    const double scale = PyFloat_AsDouble(a[4]);
    const long flags = PyLong_AsLong(a[6]);
    if (PyErr_Occurred() || flags < INT_MIN || flags > INT_MAX) return nullptr;
    const int64_t shape[3] = {b, M, N};
    const at::Tensor* given;
    if (!result_ok(a[3], c, shape, &given)) return nullptr;
    const void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr();
    Result out(a[3], given);
    int rc;
    {
      WithoutLock unlocked;
      rc = g_softmax(qp, kp, vp, out.address(c, shape), b, M, N, K, L, c.code, layout, static_cast<float>(scale),
                     static_cast<int>(flags), nullptr, 0, g_status[c.device], stream_of(c.device));
    }
    return rc ? nullptr : out.give();
  });
}

// mha(qkv, num_heads, out, scale, flags)
PyObject* py_mha(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 5 || g_mha == nullptr) return nullptr;
    Common c;
    const at::Tensor* x = take(a[0], c);
    if (x == nullptr || x->dim() != 3) return nullptr;
    const long heads = PyLong_AsLong(a[1]), flags = PyLong_AsLong(a[4]);
    const double scale = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred() || heads <= 0 || heads > INT_MAX || flags < INT_MIN || flags > INT_MAX) return nullptr;
    const int64_t b = x->size(0), M = x->size(1), k3 = x->size(2);
    if (k3 % (3 * heads) || !fits({b, M, k3})) return nullptr;
    const int64_t hidden = k3 / 3;
    const int64_t shape[3] = {b, M, hidden};
    const at::Tensor* given;
    if (!result_ok(a[2], c, shape, &given)) return nullptr;
    const void* xp = x->data_ptr();
    Result out(a[2], given);
    int rc;
    {
      WithoutLock unlocked;
      rc = g_mha(xp, out.address(c, shape), b, M, heads, hidden / heads, c.code, static_cast<float>(scale), static_cast<int>(flags),
                 g_status[c.device], stream_of(c.device));
    }
    return rc ? nullptr : out.give();
  });
}

// The operands of the MLP chain and the feed-forward block: x [M, K] or [batch, M, K], weights likewise.
struct Chain {
  const at::Tensor *x, *w1, *w2;
  const void *xp, *w1p, *w2p;     // their addresses
  int64_t b, M, N, K, L;
  int layout;                     // 1: weights [out, in]
  bool flat;                      // x is a matrix, and so is the result
};
bool chain_of(PyObject* px, PyObject* pw1, PyObject* pw2, PyObject* layout, Common& c, Chain& r) {
  r.x = take(px, c);
  r.w1 = r.x ? take(pw1, c) : nullptr;
  r.w2 = r.w1 ? take(pw2, c) : nullptr;
  if (r.w2 == nullptr) return false;
  if (is_text(layout, "OI")) r.layout = 1;
  else if (is_text(layout, "IO")) r.layout = 0;
  else return false;
  auto dims = [](const at::Tensor& t, int64_t (&d)[3]) {
    if (t.dim() != 2 && t.dim() != 3) return false;
    d[0] = t.dim() == 3 ? t.size(0) : 1;
    d[1] = t.size(t.dim() - 2);
    d[2] = t.size(t.dim() - 1);
    return true;
  };
  int64_t x[3], u[3], v[3];
  if (!dims(*r.x, x) || !dims(*r.w1, u) || !dims(*r.w2, v)) return false;
  r.flat = r.x->dim() == 2;
  r.b = x[0];
  r.M = x[1];
  r.K = x[2];
  r.L = r.layout ? u[1] : u[2];
  r.N = r.layout ? v[1] : v[2];
  r.xp = r.x->data_ptr();
  r.w1p = r.w1->data_ptr();
  r.w2p = r.w2->data_ptr();
  return u[0] == r.b && v[0] == r.b && (r.layout ? u[2] : u[1]) == r.K && (r.layout ? v[2] : v[1]) == r.L &&
         fits({r.b, r.M, r.N, r.K, r.L});
}
// As the operators' Python path takes it: a given result may be a matrix or have a batch dimension of its own.
bool chain_result_ok(PyObject* given, Common& c, const Chain& r, const at::Tensor** t) {
  *t = nullptr;
  if (given == Py_None) return true;
  *t = take(given, c);
  return *t != nullptr && (((*t)->dim() == 2 && r.b == 1 && (*t)->size(0) == r.M && (*t)->size(1) == r.N) || shape_is(**t, r.b, r.M, r.N));
}
// The shape of a new result.
struct ChainShape {
  int64_t d[3];
  bool flat;
  explicit ChainShape(const Chain& r) : d{r.b, r.M, r.N}, flat(r.flat) {}
  operator at::IntArrayRef() const { return flat ? at::IntArrayRef(d + 1, 2) : at::IntArrayRef(d, 3); }
};
// Whether the caching allocator can be expected to have `bytes` more in one piece: cached, or free on the device and within the process's share.
// Asked before a large request, because one that fails is dear: the allocator gives all its cached blocks back first, waiting for the device
// (16384 x 1024 -> 4096 -> 1024 with 100 MB left and no such question: 1073 us a call, 209 with it).
// An allocator that cannot tell is asked for the memory itself.
bool room_for(int device, size_t bytes) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return true;
  try {
    const auto index = static_cast<c10::DeviceIndex>(device);
    const auto s = c10::cuda::CUDACachingAllocator::getDeviceStats(index);
    const size_t reserved = static_cast<size_t>(s.reserved_bytes[0].current);
    // what the allocator can give back: cached segments of which no part is in use
    const size_t whole = reserved - static_cast<size_t>(s.allocated_bytes[0].current) - static_cast<size_t>(s.inactive_split_bytes[0].current);
    if (whole >= bytes) return true;
    size_t free = 0, total = 0, largest = 1;       // (a largest block of 0 would ask the device)
    if (cudaMemGetInfo(&free, &total) != cudaSuccess) {
      cudaGetLastError();
      return true;
    }
    const double share = c10::cuda::CUDACachingAllocator::getMemoryFraction(index) * static_cast<double>(total);
    const size_t allowed = share > static_cast<double>(reserved) ? static_cast<size_t>(share) - reserved : 0;
    if (whole + std::min(free, allowed) >= bytes) return true;
    c10::cuda::CUDACachingAllocator::cacheInfo(index, &largest);       // (walks all cached blocks)
    return largest >= bytes;
  } catch (const std::exception&) {
    return true;
  }
}
constexpr size_t kLargeScratch = 48u << 20;      // (what the question costs counts in small calls)

// Scratch memory of a call, in stream order from the caching allocator: its own for every stream, thread and captured graph.
// Where there is no memory left for the whole hidden layer of a large call, the ring of the next best form; none where there is
// none for that: the call then takes the form that needs none.
at::Tensor scratch_for(const Common& c, int64_t b, int64_t M, int64_t N, int64_t K, int64_t L, size_t* bytes) {
  for (const int op : {kOpGemmReluGemm, kOpGemmReluGemm | kOpLessScratch}) {
    *bytes = g_bytes(op, b, M, N, K, L, c.code);
    if (*bytes == 0) break;
    if (*bytes <= kLargeScratch || room_for(c.device, *bytes)) {
      try {
        return make({static_cast<int64_t>(*bytes)}, at::kByte, c.device);
      } catch (const c10::OutOfMemoryError&) {
      }
    }
    *bytes = 0;
  }
  return at::Tensor();
}

// gemm(x, w1, w2, out, activation, weight_layout, scratch)
PyObject* py_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7 || g_gemm == nullptr) return nullptr;
    int act;
    if (is_text(a[4], "relu")) act = 1;
    else if (is_text(a[4], "identity")) act = 0;
    else return nullptr;
    Common c;
    Chain r;
    if (!chain_of(a[0], a[1], a[2], a[5], c, r)) return nullptr;
    const at::Tensor* given;
    if (!chain_result_ok(a[3], c, r, &given)) return nullptr;
    const bool scratch = a[6] == Py_True;
    Result out(a[3], given);
    int rc;
    {
      WithoutLock unlocked;
      size_t bytes = 0;
      at::Tensor ws;
      void* y = out.address(c, ChainShape(r));
      if (scratch) ws = scratch_for(c, r.b, r.M, r.N, r.K, r.L, &bytes);
      rc = g_gemm(r.xp, r.w1p, r.w2p, y, r.b, r.M, r.N, r.K, r.L, c.code, r.layout, act, bytes ? ws.data_ptr() : nullptr, bytes,
                  g_status[c.device], stream_of(c.device));
    }
    return rc ? nullptr : out.give();
  });
}

int act_code(PyObject* o) { return is_text(o, "identity") ? 0 : is_text(o, "relu") ? 1 : is_text(o, "gelu") ? 2 : -1; }

// ffn(x, w1, b1, w2, b2, out, act1, act2, weight_layout)
PyObject* py_ffn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 9 || g_ffn == nullptr) return nullptr;
    const int act1 = act_code(a[6]), act2 = act_code(a[7]);
    if (act1 < 0 || act2 < 0) return nullptr;
    Common c;
    Chain r;
    if (!chain_of(a[0], a[1], a[3], a[8], c, r)) return nullptr;
    const void* bias[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
      PyObject* o = a[i == 0 ? 2 : 4];
      if (o == Py_None) continue;
      const at::Tensor* t = take(o, c);
      if (t == nullptr || t->numel() != r.b * (i == 0 ? r.L : r.N)) return nullptr;
      bias[i] = t->data_ptr();
    }
    const at::Tensor* given;
    if (!chain_result_ok(a[5], c, r, &given)) return nullptr;
    Result out(a[5], given);
    int rc;
    {
      WithoutLock unlocked;
      size_t bytes = 0;
      void* y = out.address(c, ChainShape(r));
      at::Tensor ws = scratch_for(c, r.b, r.M, r.N, r.K, r.L, &bytes);
      rc = g_ffn(r.xp, r.w1p, bias[0], r.w2p, bias[1], y, r.b, r.M, r.N, r.K, r.L, c.code, r.layout, act1, act2,
                 bytes ? ws.data_ptr() : nullptr, bytes, g_status[c.device], stream_of(c.device));
    }
    return rc ? nullptr : out.give();
  });
}

// ------------------------------------------------------------------ masked attention and the paged cache
// Entry points by their declared types, bound by name (bind_masked).
struct Masked {
  decltype(&ditto_b200_masked_workspace_bytes) bytes = nullptr;
  decltype(&ditto_b200_masked_attention) forward = nullptr;
  decltype(&ditto_b200_masked_attention_backward) backward = nullptr;
  decltype(&ditto_b200_paged_workspace_bytes) paged_bytes = nullptr;
  decltype(&ditto_b200_paged_attention) paged = nullptr;
  decltype(&ditto_b200_cache_append) append = nullptr;
  decltype(&ditto_b200_cache_workspace_bytes) cache_bytes = nullptr;
  decltype(&ditto_b200_cache_fork) fork = nullptr;
  decltype(&ditto_b200_cache_free) free = nullptr;
  decltype(&ditto_b200_cache_compact) compact = nullptr;
} g_masked;

// A 16-bit CUDA tensor of `dims` dimensions, not empty, its last one contiguous, the data and the other strides multiples of 16 bytes; the
// strides go to `strides` (dimensions of one entry: any valid one).
const at::Tensor* take_strided(PyObject* o, Common& c, int dims, long long* strides) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.dim() != dims || t.numel() == 0) return nullptr;
  const int dev = t.device().index();
  const at::ScalarType st = t.scalar_type();
  if (c.device < 0) {
    if (st == at::kHalf) c.code = 0;
    else if (st == at::kBFloat16) c.code = 1;
    else return nullptr;
    if (dev < 0 || dev >= kDevices || g_status[dev] == nullptr || dev != c10::cuda::current_device()) return nullptr;
    c.device = dev;
    c.type = st;
  } else if (dev != c.device || st != c.type) {
    return nullptr;
  }
  if (t.stride(dims - 1) != 1 && t.size(dims - 1) != 1) return nullptr;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return nullptr;
  for (int i = 0; i + 1 < dims; ++i) {
    if (t.size(i) > INT_MAX) return nullptr;
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8)) return nullptr;
    if (strides != nullptr) strides[i] = t.size(i) > 1 ? t.stride(i) : 8;
  }
  return &t;
}

// A contiguous CUDA tensor of another type on the call's device, of this many entries in its one dimension (below 0: any number).
const at::Tensor* take_vector(PyObject* o, int device, at::ScalarType type, int64_t n) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.device().index() != device || t.scalar_type() != type || t.dim() != 1 || !t.is_contiguous()) return nullptr;
  return n < 0 || t.size(0) == n ? &t : nullptr;
}
// ... or None: *out is its address or null.
template <class T>
bool optional_vector(PyObject* o, int device, at::ScalarType type, int64_t n, const T** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = take_vector(o, device, type, n);
  if (t == nullptr || t->requires_grad()) return false;
  *out = static_cast<const T*>(t->data_ptr());
  return true;
}
// A table of page ids with contiguous rows.
const at::Tensor* take_table(PyObject* o, int device) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.device().index() != device || t.scalar_type() != at::kInt || t.dim() != 2 || t.numel() == 0 || t.stride(1) != 1) return nullptr;
  if (t.size(0) > 1 && t.stride(0) < t.size(1)) return nullptr;
  return t.size(0) <= INT_MAX && t.size(1) <= INT_MAX ? &t : nullptr;
}
long long row_stride(const at::Tensor& t) { return std::max<int64_t>(t.stride(0), t.size(1)); }

bool number(PyObject* o, float* out) {
  const double v = PyFloat_AsDouble(o);
  *out = static_cast<float>(v);
  return !(v == -1.0 && PyErr_Occurred());
}
bool optional_cap(PyObject* o, float* out) {
  *out = 0.f;
  return o == Py_None || (number(o, out) && *out > 0.f);
}

at::Tensor workspace(size_t bytes, int device) {
  return bytes == 0 ? at::Tensor() : make({static_cast<int64_t>(bytes)}, at::kByte, device);
}

// The operands and rules from the arguments  q, k, v, out (may be None), scale, causal, prefix, documents, slopes, cap.
bool masked_args(PyObject* const* a, Common& c, ditto_b200_masked_args& r, const at::Tensor** query, const at::Tensor** key, const at::Tensor** out) {
  const at::Tensor* q = take_strided(a[0], c, 4, r.q_strides);
  const at::Tensor* k = q ? take_strided(a[1], c, 4, r.k_strides) : nullptr;
  const at::Tensor* v = k ? take_strided(a[2], c, 4, r.v_strides) : nullptr;
  if (v == nullptr || k->sizes() != v->sizes() || k->size(0) != q->size(0) || k->size(3) != q->size(3)) return false;
  *out = nullptr;
  if (a[3] != Py_None && ((*out = take_strided(a[3], c, 4, r.out_strides)) == nullptr || (*out)->sizes() != q->sizes())) return false;
  r.batch = q->size(0), r.M = q->size(1), r.heads = q->size(2), r.head_dim = q->size(3), r.L = k->size(1), r.kv_heads = k->size(2);
  r.dtype = c.code;
  if (r.kv_heads == 0 || r.heads % r.kv_heads) return false;
  if (!number(a[4], &r.scale) || !optional_cap(a[9], &r.cap)) return false;
  if (a[5] != Py_True && a[5] != Py_False) return false;
  r.causal = a[5] == Py_True;
  if (!optional_vector(a[6], c.device, at::kInt, r.batch, &r.prefix) || !optional_vector(a[8], c.device, at::kFloat, r.heads, &r.slopes)) return false;
  r.documents = nullptr;
  if (a[7] != Py_None) {
    const at::Tensor* d = take_table(a[7], c.device);
    if (d == nullptr || !d->is_contiguous() || d->size(0) != r.batch || d->size(1) != r.L) return false;
    r.documents = static_cast<const int*>(d->data_ptr());
  }
  r.q = q->data_ptr(), r.k = k->data_ptr(), r.v = v->data_ptr();
  r.out = *out ? (*out)->data_ptr() : nullptr;
  *query = q, *key = k;
  return true;
}
void compact_strides(const at::Tensor& t, long long* strides) {
  for (int i = 0; i < 3; ++i) strides[i] = t.size(i) > 1 ? t.stride(i) : 8;
}

// masked(query, key, value, out, scale, causal, prefix, documents, slopes, cap, return_lse)
PyObject* py_masked(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 11 || g_masked.forward == nullptr) return nullptr;
    Common c;
    ditto_b200_masked_args r = {};
    const at::Tensor *q, *k, *given;
    if (!masked_args(a, c, r, &q, &k, &given)) return nullptr;
    if (c10::GradMode::is_enabled() && (q->requires_grad() || k->requires_grad() || THPVariable_Unpack(a[2]).requires_grad())) return nullptr;
    const bool want_lse = a[10] == Py_True;
    at::Tensor out, lse;
    const std::vector<int64_t> shape = q->sizes().vec();
    int rc;
    {
      WithoutLock unlocked;
      if (given == nullptr) {
        out = make(shape, c.type, c.device);
        r.out = out.data_ptr();
        compact_strides(out, r.out_strides);
      }
      if (want_lse) {
        lse = make(at::IntArrayRef(shape.data(), 3), at::kFloat, c.device);
        r.lse = static_cast<float*>(lse.data_ptr());
      }
      const size_t bytes = r.documents != nullptr ? g_masked.bytes(&r, 0) : 0;
      at::Tensor ws = workspace(bytes, c.device);
      rc = g_masked.forward(&r, bytes ? ws.data_ptr() : nullptr, bytes, g_status[c.device], stream_of(c.device));
    }
    if (rc) return nullptr;
    PyObject* first = a[3];
    if (given == nullptr) first = THPVariable_Wrap(out);
    else Py_INCREF(first);
    if (!want_lse) return first;
    return pair_of(first, THPVariable_Wrap(lse));
  });
}

// masked_backward(grad_out, query, key, value, out, lse, scale, causal, prefix, documents, slopes, cap) -> (dq, dk, dv)
PyObject* py_masked_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 12 || g_masked.backward == nullptr || a[4] == Py_None) return nullptr;
    Common c;
    ditto_b200_masked_args r = {};
    const at::Tensor *q, *k, *out;
    PyObject* const args[10] = {a[1], a[2], a[3], a[4], a[6], a[7], a[8], a[9], a[10], a[11]};
    if (!masked_args(args, c, r, &q, &k, &out)) return nullptr;
    long long strides[3];
    const at::Tensor* g = take_strided(a[0], c, 4, strides);
    if (g == nullptr || g->sizes() != q->sizes() || !THPVariable_Check(a[5])) return nullptr;
    const at::Tensor& lse = THPVariable_Unpack(a[5]);
    if (!lse.is_cuda() || lse.device().index() != c.device || lse.scalar_type() != at::kFloat || !lse.is_contiguous() ||
        !shape_is(lse, r.batch, r.M, r.heads))
      return nullptr;
    r.lse = static_cast<float*>(lse.data_ptr());
    const void* gp = g->data_ptr();
    const std::vector<int64_t> rows = q->sizes().vec(), keys = k->sizes().vec();
    at::Tensor dq, dk, dv;
    int rc;
    {
      WithoutLock unlocked;
      dq = make(rows, c.type, c.device);
      dk = make(keys, c.type, c.device);
      dv = make(keys, c.type, c.device);
      const size_t bytes = g_masked.bytes(&r, 1);
      at::Tensor ws = workspace(bytes, c.device);
      rc = g_masked.backward(&r, gp, strides, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes,
                             g_status[c.device], stream_of(c.device));
    }
    if (rc) return nullptr;
    PyObject* t = PyTuple_New(3);
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(dq));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(dk));
    PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(dv));
    return t;
  });
}

// The cache of a call: key_pages, value_pages, block_table, lengths, query_starts (or None).
struct Cache {
  const at::Tensor *keys, *values, *table;
  const int *lengths, *starts;
  int batch;
};
bool cache_of(PyObject* const* a, Common& c, int64_t tokens, long long* key_strides, long long* value_strides, Cache& r) {
  r.keys = take_strided(a[0], c, 4, key_strides);
  r.values = r.keys ? take_strided(a[1], c, 4, value_strides) : nullptr;
  if (r.values == nullptr || r.keys->sizes() != r.values->sizes() || (r.table = take_table(a[2], c.device)) == nullptr) return false;
  r.batch = static_cast<int>(r.table->size(0));
  const at::Tensor* lengths = take_vector(a[3], c.device, at::kInt, r.batch);
  if (lengths == nullptr || !optional_vector(a[4], c.device, at::kInt, r.batch + 1, &r.starts)) return false;
  r.lengths = static_cast<const int*>(lengths->data_ptr());
  return r.starts != nullptr || tokens == r.batch;
}

// paged(query, key_pages, value_pages, block_table, lengths, query_starts, out, scale, prefix, slopes, cap)
PyObject* py_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 11 || g_masked.paged == nullptr) return nullptr;
    Common c;
    ditto_b200_paged_args r = {};
    Cache cache;
    const at::Tensor* q = take_strided(a[0], c, 3, r.q_strides);
    if (q == nullptr || !cache_of(a + 1, c, q->size(0), r.key_strides, r.value_strides, cache) || cache.keys->size(3) != q->size(2)) return nullptr;
    const at::Tensor* given = nullptr;
    if (a[6] != Py_None && ((given = take_strided(a[6], c, 3, r.out_strides)) == nullptr || given->sizes() != q->sizes())) return nullptr;
    r.tokens = q->size(0), r.heads = q->size(1), r.head_dim = q->size(2), r.batch = cache.batch;
    r.pages = cache.keys->size(0), r.page = cache.keys->size(1), r.kv_heads = cache.keys->size(2);
    r.table_cols = cache.table->size(1), r.table_stride = row_stride(*cache.table), r.dtype = c.code;
    if (!number(a[7], &r.scale) || !optional_cap(a[10], &r.cap) || !optional_vector(a[8], c.device, at::kInt, r.batch, &r.prefix) ||
        !optional_vector(a[9], c.device, at::kFloat, r.heads, &r.slopes))
      return nullptr;
    r.q = q->data_ptr(), r.key_pages = cache.keys->data_ptr(), r.value_pages = cache.values->data_ptr();
    r.table = static_cast<const int*>(cache.table->data_ptr()), r.lengths = cache.lengths, r.starts = cache.starts;
    r.out = given ? given->data_ptr() : nullptr;
    const int64_t shape[3] = {r.tokens, r.heads, r.head_dim};
    at::Tensor out;
    int rc;
    {
      WithoutLock unlocked;
      if (given == nullptr) {
        out = make(shape, c.type, c.device);
        if (r.starts != nullptr) out.zero_();          // (tokens of no sequence)
        r.out = out.data_ptr();
        for (int i = 0; i < 2; ++i) r.out_strides[i] = shape[i] > 1 ? out.stride(i) : 8;
      }
      const size_t bytes = g_masked.paged_bytes(&r);
      at::Tensor ws = workspace(bytes, c.device);
      rc = g_masked.paged(&r, bytes ? ws.data_ptr() : nullptr, bytes, g_status[c.device], stream_of(c.device));
    }
    if (rc) return nullptr;
    if (given == nullptr) return THPVariable_Wrap(out);
    Py_INCREF(a[6]);
    return a[6];
  });
}

// append(keys, values, key_pages, value_pages, block_table, lengths, query_starts) -> True
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7 || g_masked.append == nullptr) return nullptr;
    Common c;
    ditto_b200_append_args r = {};
    Cache cache;
    const at::Tensor *k = take_strided(a[0], c, 3, r.k_strides), *v = k ? take_strided(a[1], c, 3, r.v_strides) : nullptr;
    if (v == nullptr || k->sizes() != v->sizes() || !cache_of(a + 2, c, k->size(0), r.key_strides, r.value_strides, cache)) return nullptr;
    if (cache.keys->size(2) != k->size(1) || cache.keys->size(3) != k->size(2)) return nullptr;
    r.keys = k->data_ptr(), r.values = v->data_ptr(), r.key_pages = cache.keys->data_ptr(), r.value_pages = cache.values->data_ptr();
    r.table = static_cast<const int*>(cache.table->data_ptr()), r.lengths = cache.lengths, r.starts = cache.starts;
    r.table_stride = row_stride(*cache.table), r.table_cols = cache.table->size(1);
    r.tokens = k->size(0), r.batch = cache.batch, r.kv_heads = k->size(1), r.head_dim = k->size(2);
    r.pages = cache.keys->size(0), r.page = cache.keys->size(1);
    int rc;
    {
      WithoutLock unlocked;
      rc = g_masked.append(&r, g_status[c.device], stream_of(c.device));
    }
    if (rc) return nullptr;
    Py_RETURN_TRUE;
  });
}

// The tables of a cache; lengths may be null where the call does not need them.
bool tables_of(PyObject* table, PyObject* lengths, PyObject* references, int* device, ditto_b200_tables& r) {
  if (!THPVariable_Check(table)) return false;
  *device = THPVariable_Unpack(table).device().index();
  if (*device < 0 || *device >= kDevices || g_status[*device] == nullptr || *device != c10::cuda::current_device()) return false;
  const at::Tensor* t = take_table(table, *device);
  if (t == nullptr) return false;
  const at::Tensor* l = lengths ? take_vector(lengths, *device, at::kInt, t->size(0)) : nullptr;
  const at::Tensor* f = take_vector(references, *device, at::kInt, -1);
  if ((lengths && l == nullptr) || f == nullptr || f->size(0) == 0 || f->size(0) > INT_MAX) return false;
  r.table = static_cast<int*>(t->data_ptr()), r.lengths = l ? static_cast<int*>(l->data_ptr()) : nullptr;
  r.references = static_cast<int*>(f->data_ptr());
  r.stride = row_stride(*t), r.sequences = t->size(0), r.cols = t->size(1), r.page = 0, r.pages = f->size(0);
  return true;
}
// Pools [pages, ...] of one shape, type and stride, in a list or tuple.
bool pools_of(PyObject* o, int device, int64_t pages, std::vector<void*>& base, ditto_b200_pools& r) {
  if (!PyList_Check(o) && !PyTuple_Check(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  if (n == 0) return false;
  const at::Tensor* first = nullptr;
  base.resize(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* x = PySequence_Fast_GET_ITEM(o, i);
    if (!THPVariable_Check(x)) return false;
    const at::Tensor& t = THPVariable_Unpack(x);
    if (!t.is_cuda() || t.device().index() != device || t.dim() < 2) return false;
    if (first == nullptr) {
      first = &t;
      if (t.size(0) != pages || t.numel() == 0) return false;
      int64_t inner = 1;                               // a page is contiguous
      for (int64_t d = t.dim() - 1; d > 0; --d) {
        if (t.size(d) != 1 && t.stride(d) != inner) return false;
        inner *= t.size(d);
      }
      r.page_bytes = inner * t.element_size();
      r.stride_bytes = t.size(0) > 1 ? t.stride(0) * static_cast<int64_t>(t.element_size()) : r.page_bytes;
    } else if (t.sizes() != first->sizes() || t.strides() != first->strides() || t.scalar_type() != first->scalar_type()) {
      return false;
    }
    base[i] = t.data_ptr();
  }
  r.base = base.data(), r.count = static_cast<int>(n), r.pages = static_cast<int>(pages);
  return true;
}

// cache_free(block_table, lengths, references, sequences) -> True
PyObject* py_cache_free(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int device;
    ditto_b200_tables t;
    if (n != 4 || g_masked.free == nullptr || !tables_of(a[0], a[1], a[2], &device, t)) return nullptr;
    const at::Tensor* s = take_vector(a[3], device, at::kInt, -1);
    if (s == nullptr || s->size(0) == 0 || s->size(0) > INT_MAX) return nullptr;
    const int* sp = static_cast<const int*>(s->data_ptr());
    const int count = static_cast<int>(s->size(0));
    int rc;
    {
      WithoutLock unlocked;
      rc = g_masked.free(&t, sp, count, g_status[device], stream_of(device));
    }
    if (rc) return nullptr;
    Py_RETURN_TRUE;
  });
}

// cache_fork(pools, block_table, lengths, references, parents, children, page_size) -> True
PyObject* py_cache_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int device;
    ditto_b200_tables t;
    ditto_b200_pools pools;
    std::vector<void*> base;
    if (n != 7 || g_masked.fork == nullptr || !tables_of(a[1], a[2], a[3], &device, t) || !pools_of(a[0], device, t.pages, base, pools)) return nullptr;
    const at::Tensor *from = take_vector(a[4], device, at::kInt, -1), *to = from ? take_vector(a[5], device, at::kInt, from->size(0)) : nullptr;
    if (to == nullptr || to->size(0) == 0 || to->size(0) > t.sequences) return nullptr;
    const long page = PyLong_AsLong(a[6]);
    if (page <= 0 || page > INT_MAX) return nullptr;
    t.page = static_cast<int>(page);
    const int *fp = static_cast<const int*>(from->data_ptr()), *tp = static_cast<const int*>(to->data_ptr());
    const int count = static_cast<int>(to->size(0));
    int rc;
    {
      WithoutLock unlocked;
      const size_t bytes = g_masked.cache_bytes(&t, count);
      at::Tensor ws = workspace(bytes, device);
      rc = g_masked.fork(&pools, &t, fp, tp, count, ws.data_ptr(), bytes, g_status[device], stream_of(device));
    }
    if (rc) return nullptr;
    Py_RETURN_TRUE;
  });
}

// cache_compact(pools, block_table, references) -> (table, references)
PyObject* py_cache_compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int device;
    ditto_b200_tables t;
    ditto_b200_pools pools;
    std::vector<void*> base;
    if (n != 3 || g_masked.compact == nullptr || !tables_of(a[1], nullptr, a[2], &device, t) || !pools_of(a[0], device, t.pages, base, pools)) return nullptr;
    at::Tensor table, references;
    int rc;
    {
      WithoutLock unlocked;
      table = make({t.sequences, t.cols}, at::kInt, device);
      references = make({t.pages}, at::kInt, device);
      const size_t bytes = g_masked.cache_bytes(&t, 0);
      at::Tensor ws = workspace(bytes, device);
      rc = g_masked.compact(&pools, &t, static_cast<int*>(table.data_ptr()), t.cols, static_cast<int*>(references.data_ptr()), ws.data_ptr(), bytes,
                            g_status[device], stream_of(device));
    }
    if (rc) return nullptr;
    return pair_of(THPVariable_Wrap(table), THPVariable_Wrap(references));
  });
}

// bind_masked(name, address): a C entry point of the operators above
PyObject* py_bind_masked(PyObject*, PyObject* args) {
  const char* name;
  unsigned long long p;
  if (!PyArg_ParseTuple(args, "sK", &name, &p)) return nullptr;
  const std::string_view s(name);
  auto set = [&](const char* known, auto& fn) {
    if (s == known) fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p);
  };
  set("ditto_b200_masked_workspace_bytes", g_masked.bytes);
  set("ditto_b200_masked_attention", g_masked.forward);
  set("ditto_b200_masked_attention_backward", g_masked.backward);
  set("ditto_b200_paged_workspace_bytes", g_masked.paged_bytes);
  set("ditto_b200_paged_attention", g_masked.paged);
  set("ditto_b200_cache_append", g_masked.append);
  set("ditto_b200_cache_workspace_bytes", g_masked.cache_bytes);
  set("ditto_b200_cache_fork", g_masked.fork);
  set("ditto_b200_cache_free", g_masked.free);
  set("ditto_b200_cache_compact", g_masked.compact);
  Py_RETURN_NONE;
}

// A built module's compiled shape: plan(kind, batch, M, N, K, L, type code, heads, scale, act1, act2, bias1, bias2).
struct Plan {
  int kind;                       // 0 softmax, 1 GEMM chain, 2 packed attention, 3 feed-forward
  int64_t b, M, N, K, L;
  int code, heads, act1, act2, bias1, bias2;
  float scale;
};
constexpr const char* kPlanName = "ditto_b200.plan";
void free_plan(PyObject* cap) { delete static_cast<Plan*>(PyCapsule_GetPointer(cap, kPlanName)); }
PyObject* py_plan(PyObject*, PyObject* args) {
  Plan p;
  long long b, M, N, K, L;
  if (!PyArg_ParseTuple(args, "iLLLLLiifiiii", &p.kind, &b, &M, &N, &K, &L, &p.code, &p.heads, &p.scale, &p.act1, &p.act2, &p.bias1,
                        &p.bias2))
    return nullptr;
  p.b = b, p.M = M, p.N = N, p.K = K, p.L = L;
  return PyCapsule_New(new Plan(p), kPlanName, free_plan);
}

// call(plan, *tensors) -> True, or None where the checked path has to look at the arguments
PyObject* py_call(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n < 3 || !PyCapsule_IsValid(a[0], kPlanName)) return nullptr;
    const Plan& p = *static_cast<const Plan*>(PyCapsule_GetPointer(a[0], kPlanName));
    const at::Tensor* t[6];
    void* ptr[6];
    const int count = static_cast<int>(n - 1);
    if (count > 6) return nullptr;
    Common c;
    for (int i = 0; i < count; ++i) {
      if ((t[i] = take(a[i + 1], c)) == nullptr) return nullptr;
      ptr[i] = t[i]->data_ptr();
    }
    if (c.code != p.code) return nullptr;
    int* status = g_status[c.device];
    if (p.kind <= 1) {
      if (count != 4 || !shape_is(*t[0], p.b, p.M, p.K) || !shape_is(*t[1], p.b, p.K, p.L) || !shape_is(*t[2], p.b, p.L, p.N) ||
          !shape_is(*t[3], p.b, p.M, p.N))
        return nullptr;
    } else if (p.kind == 2) {
      if (count != 2 || !shape_is(*t[0], p.b, p.M, 3 * p.N) || !shape_is(*t[1], p.b, p.M, p.N)) return nullptr;
    } else {
      // x, w1 [L, K], (b1 [L]), w2 [N, L], (b2 [N]), out; x and out keep whatever leading dimensions the layer has
      if (count != 4 + p.bias1 + p.bias2) return nullptr;
      const int i2 = 2 + p.bias1;                      // w2
      auto matrix = [](const at::Tensor& m, int64_t r, int64_t k) { return m.dim() == 2 && m.size(0) == r && m.size(1) == k; };
      auto vector = [](const at::Tensor& v, int64_t k) { return v.dim() == 1 && v.size(0) == k; };
      if (t[0]->numel() != p.M * p.K || t[count - 1]->numel() != p.M * p.N || !matrix(*t[1], p.L, p.K) || !matrix(*t[i2], p.N, p.L) ||
          (p.bias1 && !vector(*t[2], p.L)) || (p.bias2 && !vector(*t[i2 + 1], p.N)))
        return nullptr;
    }
    int rc = -1;
    {
      WithoutLock unlocked;
      void* stream = stream_of(c.device);
      size_t bytes = 0;
      at::Tensor ws;
      if (p.kind == 0) {
        rc = g_softmax(ptr[0], ptr[1], ptr[2], ptr[3], p.b, p.M, p.N, p.K, p.L, p.code, 0, p.scale, 0, nullptr, 0, status, stream);
      } else if (p.kind == 1) {
        ws = scratch_for(c, p.b, p.M, p.N, p.K, p.L, &bytes);
        rc = g_gemm(ptr[0], ptr[1], ptr[2], ptr[3], p.b, p.M, p.N, p.K, p.L, p.code, 0, p.act1, bytes ? ws.data_ptr() : nullptr, bytes,
                    status, stream);
      } else if (p.kind == 2) {
        rc = g_mha(ptr[0], ptr[1], p.b, p.M, p.heads, p.N / p.heads, p.code, p.scale, 0, status, stream);
      } else {
        const int i2 = 2 + p.bias1;
        ws = scratch_for(c, 1, p.M, p.N, p.K, p.L, &bytes);
        rc = g_ffn(ptr[0], ptr[1], p.bias1 ? ptr[2] : nullptr, ptr[i2], p.bias2 ? ptr[i2 + 1] : nullptr, ptr[count - 1], 1, p.M, p.N, p.K,
                   p.L, p.code, 1, p.act1, p.act2, bytes ? ws.data_ptr() : nullptr, bytes, status, stream);
      }
    }
    if (rc != 0) return nullptr;
    Py_RETURN_TRUE;
  });
}

// bind(softmax, mha, gemm, ffn, bytes): addresses of the C entry points
PyObject* py_bind(PyObject*, PyObject* args) {
  unsigned long long s, m, g, f, b;
  if (!PyArg_ParseTuple(args, "KKKKK", &s, &m, &g, &f, &b)) return nullptr;
  g_softmax = reinterpret_cast<SoftmaxFn>(s);
  g_mha = reinterpret_cast<MhaFn>(m);
  g_gemm = reinterpret_cast<GemmFn>(g);
  g_ffn = reinterpret_cast<FfnFn>(f);
  g_bytes = reinterpret_cast<BytesFn>(b);
  Py_RETURN_NONE;
}
// status(device index, address of its status word)
PyObject* py_status(PyObject*, PyObject* args) {
  int dev;
  unsigned long long p;
  if (!PyArg_ParseTuple(args, "iK", &dev, &p)) return nullptr;
  if (dev >= 0 && dev < kDevices) g_status[dev] = reinterpret_cast<int*>(p);
  Py_RETURN_NONE;
}

#define DITTO_FAST(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fn)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {DITTO_FAST("softmax", py_softmax),
                          DITTO_FAST("mha", py_mha),
                          DITTO_FAST("gemm", py_gemm),
                          DITTO_FAST("ffn", py_ffn),
                          DITTO_FAST("call", py_call),
                          DITTO_FAST("masked", py_masked),
                          DITTO_FAST("masked_backward", py_masked_backward),
                          DITTO_FAST("paged", py_paged),
                          DITTO_FAST("append", py_append),
                          DITTO_FAST("cache_free", py_cache_free),
                          DITTO_FAST("cache_fork", py_cache_fork),
                          DITTO_FAST("cache_compact", py_cache_compact),
                          {"bind_masked", py_bind_masked, METH_VARARGS, nullptr},
                          {"plan", py_plan, METH_VARARGS, nullptr},
                          {"bind", py_bind, METH_VARARGS, nullptr},
                          {"status", py_status, METH_VARARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&kModule); }
