// The layer-level entry points of sglang_amd as one native call each.
//
// What bounds a decode step here is not the GPU: a block-FP8 linear at M = 1 is 13 us of kernels, and its pass through
// Python (argument checks, two dispatcher calls into Python implementations, four allocations, ctypes with twenty arguments)
// took 38 us; the fused expert layer took 130 us.  A function of this module checks the operands, takes all its scratch from
// torch's caching allocator in one piece and makes the C ABI calls back to back: 5 to 8 us for a linear.
//
// Every function returns None, before anything has been launched, for operands that it does not take as they are: tensors of
// a mode or a subclass (of the dispatcher's - tracing, fake tensors - or with a __torch_function__), inputs that want gradients, unusual types and layouts, and everything
// that is an error.  The Python caller then goes through the dispatcher ops, which know all cases and word the errors.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <map>
#include <mutex>
#include <vector>

#include "../../include/fp8k.h"

namespace {

using at::Tensor;
using c10::DispatchKey;
using c10::DispatchKeySet;
using c10::ScalarType;

constexpr float kEps = 1e-10f;

PyObject* g_has_torch_function = nullptr;  // torch.overrides.has_torch_function_unary
PyObject* g_workspaces = nullptr;     // sgl_kernel._workspaces: (device index, stream) -> the buffer of that stream
PyObject* g_grow_workspace = nullptr; // sgl_kernel._workspace

// ---------------------------------------------------------------------------------------------- operands
// A mode is active that has to see the ops: a torch function mode, or one of the dispatcher (tracing, fake tensors,
// functionalisation, vmap).
bool modes_active() {
  if (at::impl::torch_function_mode_enabled()) return true;
  constexpr DispatchKeySet modes({DispatchKey::Python, DispatchKey::PythonTLSSnapshot, DispatchKey::Functionalize,
                                  DispatchKey::FuncTorchDynamicLayerFrontMode, DispatchKey::FuncTorchBatched,
                                  DispatchKey::Tracer});
  return c10::impl::tls_local_dispatch_key_set().included_.has_any(modes);
}

// A strided GPU tensor with nothing between it and its memory, on the device of the call.
bool plain(const Tensor& t, int device) {
  constexpr DispatchKeySet odd({DispatchKey::Python, DispatchKey::PythonTLSSnapshot, DispatchKey::Functionalize,
                                DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper, DispatchKey::Conjugate,
                                DispatchKey::Negative, DispatchKey::ZeroTensor});
  if (!t.defined() || t.key_set().has_any(odd) || t.is_nested()) return false;
  if (!t.is_cuda() || t.layout() != c10::kStrided || t.get_device() != device) return false;
  return !(t.requires_grad() && at::GradMode::is_enabled());
}

// a tensor whose class has no say in what is done with it: a subclass may have a __torch_function__ without being a dispatcher
// subclass; parameters and subclasses that switch theirs off have none
bool tensor_arg(PyObject* o, Tensor& t) {
  if (!THPVariable_CheckExact(o)) {  // neither a Tensor nor a Parameter
    if (!THPVariable_Check(o)) return false;
    PyObject* const has = PyObject_CallFunctionObjArgs(g_has_torch_function, o, nullptr);
    if (!has) throw python_error();
    Py_DECREF(has);  // True or False
    if (has != Py_False) return false;
  }
  t = THPVariable_Unpack(o);
  return true;
}

bool truth(PyObject* o) {
  if (o == Py_True || o == Py_False) return o == Py_True;
  const int is = PyObject_IsTrue(o);
  if (is < 0) throw python_error();
  return is == 1;
}

bool is_fp8(const Tensor& t) { return t.scalar_type() == ScalarType::Float8_e4m3fn; }
bool is_half(ScalarType t) { return t == ScalarType::BFloat16 || t == ScalarType::Half; }

int code(ScalarType t) {
  return t == ScalarType::BFloat16 ? FP8K_BF16 : t == ScalarType::Half ? FP8K_F16 : FP8K_F32;
}

bool non_negative_strides(const Tensor& t) {
  for (int64_t s : t.strides())
    if (s < 0) return false;
  return true;
}

bool is_128x128(PyObject* o) {
  if (!PyList_Check(o) && !PyTuple_Check(o)) return false;
  if (PySequence_Fast_GET_SIZE(o) != 2) return false;
  for (int i = 0; i < 2; ++i) {
    PyObject* v = PySequence_Fast_GET_ITEM(o, i);
    if (!PyLong_CheckExact(v) || PyLong_AsLong(v) != 128) return false;
  }
  return true;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t ceil_to(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// a weight with its 128 x 128 block scales: w e4m3fn [N, K] contiguous, scale float32 [ceil(N/128), ceil(K/128)]
bool block_weight(const Tensor& w, const Tensor& s, int64_t K, int device) {
  if (!plain(w, device) || !plain(s, device) || !is_fp8(w) || w.dim() != 2 || w.size(1) != K || !w.is_contiguous()) return false;
  if (s.scalar_type() != ScalarType::Float || s.dim() != 2 || !non_negative_strides(s)) return false;
  const int64_t N = w.size(0);
  return N > 0 && N % 8 == 0 && s.size(0) == ceil_div(N, 128) && s.size(1) == ceil_div(K, 128);
}

void check(int status) {
  if (status != 0) {
    const char* msg = fp8k_last_error();
    throw std::runtime_error(msg && *msg ? msg : "fp8k error");
  }
}

// ---------------------------------------------------------------------------------------------- memory
Tensor empty(at::IntArrayRef size, ScalarType t, const at::Device& d) {
  return Tensor(at::detail::empty_cuda(size, t, d, std::nullopt));
}

// [rows, cols] with strides (1, ld): column-major, every column padded to ld entries
Tensor empty_column_major(int64_t rows, int64_t cols, int64_t ld, ScalarType t, const at::Device& d) {
  Tensor out = empty({cols * ld}, t, d);
  out.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({rows, cols}), at::IntArrayRef({(int64_t)1, ld}));
  return out;
}

// The scratch of one call: one block of torch's caching allocator on the call's stream, cut into 256-byte aligned pieces.  It
// goes back when the call returns; the allocator hands it out again on the same stream only (or, under graph capture, inside
// the capture's pool), so launches that are still queued keep it to themselves, whatever other threads and streams do.
class Scratch {
 public:
  Scratch(size_t bytes, hipStream_t st) {
    if (bytes) base_ = static_cast<char*>(c10::hip::HIPCachingAllocator::raw_alloc_with_stream(bytes, st));
  }
  ~Scratch() {
    if (base_) c10::hip::HIPCachingAllocator::raw_delete(base_);
  }
  Scratch(const Scratch&) = delete;
  Scratch& operator=(const Scratch&) = delete;
  static size_t room(int64_t bytes) { return (size_t)ceil_to(bytes, 256); }
  template <class T = void>
  T* take(int64_t bytes) {
    char* p = base_ + used_;
    used_ += room(bytes);
    return reinterpret_cast<T*>(p);
  }

 private:
  char* base_ = nullptr;
  size_t used_ = 0;
};

// What allocates or launches runs without the interpreter lock: a launch into a full queue and an allocation that has to free
// cached blocks wait for the device, and other Python threads, one of which the device may be waiting for, must not wait with it.
class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }
  WithoutGil(const WithoutGil&) = delete;
  WithoutGil& operator=(const WithoutGil&) = delete;

 private:
  PyThreadState* state_;
};

// the part of a call that works on the device: no interpreter lock, the call's device made current, and its stream
struct Call {
  explicit Call(const Tensor& t)
      : guard(t.device()), device(t.get_device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
  WithoutGil unlocked;  // first: taken back last
  c10::DeviceGuard guard;
  int device;
  hipStream_t stream;
};

// the GEMM workspace of the current stream (sgl_kernel._workspace): nullptr and false when the Python side raised.  Asked for
// with the interpreter lock; what it returns is never released.
bool stream_workspace(const Tensor& like, int64_t need, void*& p, int64_t& bytes) {
  p = nullptr;
  bytes = 0;
  if (need <= 0) return true;
  const hipStream_t st = c10::hip::getCurrentHIPStream(like.get_device()).stream();
  PyObject* key = Py_BuildValue("(iK)", (int)like.get_device(), (unsigned long long)(uintptr_t)st);
  if (!key) return false;
  PyObject* buf = PyDict_GetItem(g_workspaces, key);  // borrowed
  Py_DECREF(key);
  if (buf && THPVariable_Check(buf)) {
    const Tensor& t = THPVariable_Unpack(buf);
    if (t.numel() >= need) {
      p = t.data_ptr();
      bytes = t.numel();
      return true;
    }
  }
  PyObject* device = THPDevice_New(like.device());
  PyObject* got = device ? PyObject_CallFunction(g_grow_workspace, "OL", device, (long long)need) : nullptr;
  Py_XDECREF(device);
  if (!got) return false;
  const Tensor& t = THPVariable_Unpack(got);
  p = t.data_ptr();
  bytes = t.numel();
  Py_DECREF(got);  // the registry keeps it
  return true;
}

// Threads that share a stream share its workspace: the launches of one product (copy of the scales, GEMM, reduction) go onto the
// stream together.  One lock per workspace, so a thread waits for launches onto its own stream only; taken without the interpreter lock.
std::mutex& workspace_lock(const void* workspace) {
  static std::mutex mutex;
  static auto* const locks = new std::map<const void*, std::mutex>;  // as many as there are workspaces; both live as long as the process
  std::lock_guard<std::mutex> lock(mutex);
  return (*locks)[workspace];
}

// A record of the call for torch's profiler and other observers, as the dispatcher keeps one of an op: for the rest of the scope.
#define OBSERVED(name, ...) RECORD_FUNCTION("fp8k::" name, (std::vector<c10::IValue>{__VA_ARGS__}))

// an argument that did not convert is the dispatcher path's to word as well
#define DECLINE     \
  do {              \
    PyErr_Clear();  \
    Py_RETURN_NONE; \
  } while (0)

// ---------------------------------------------------------------------------------------------- group quant
// group_quant(x, group_size, eps, column_major, tma_aligned, ue8m0, fuse_silu) -> (q, scales) or None
PyObject* group_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x;
  if (n != 7 || !tensor_arg(a[0], x) || modes_active() || !x.is_cuda() || !plain(x, x.get_device())) DECLINE;
  if (!PyLong_Check(a[1]) || !PyFloat_Check(a[2])) DECLINE;
  const int64_t group = PyLong_AsLongLong(a[1]);
  const float eps = (float)PyFloat_AS_DOUBLE(a[2]);
  const bool column = truth(a[3]), tma = truth(a[4]), ue8m0 = truth(a[5]), fuse = truth(a[6]);
  const ScalarType dt = x.scalar_type();
  if (!(is_half(dt) || dt == ScalarType::Float) || x.dim() < 1 || x.numel() == 0 || !x.is_contiguous()) DECLINE;
  if ((column || ue8m0) && x.dim() != 2) DECLINE;
  if (ue8m0 && !(column && tma && group == 128)) DECLINE;
  const int64_t width = x.size(-1);
  const int64_t K = fuse ? width / 2 : width;
  if (group <= 0 || width % group != 0 || K % group != 0 || K == 0 || (fuse && (width % 2 != 0 || group != 128))) DECLINE;
  const int64_t M = x.numel() / width, G = K / group;

  Tensor q, s;
  {
    Call c(x);
    OBSERVED("group_quant", x);
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = K;
    q = empty(shape, ScalarType::Float8_e4m3fn, x.device());
    int64_t sm, sg;
    if (ue8m0) {
      sm = 1;
      sg = ceil_to(M, 4);
      s = empty_column_major(M, ceil_div(G, 4), sg, ScalarType::Int, x.device());
    } else if (column) {
      sm = 1;
      sg = tma ? ceil_to(M, 4) : M;
      s = empty_column_major(M, G, sg, ScalarType::Float, x.device());
    } else {
      shape.back() = G;
      s = empty(shape, ScalarType::Float, x.device());
      sm = G;
      sg = 1;
    }
    check((fuse ? fp8k_silu_mul_group_quant : fp8k_group_quant)(
        x.data_ptr(), q.data_ptr(), s.data_ptr(), M, K, group, eps, -448.f, 448.f, code(dt), sm, sg,
        ue8m0 ? FP8K_SCALE_UE8M0_PACKED : FP8K_SCALE_F32, c.stream));
  }
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(s)));
  return out;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- block-FP8 GEMM
// block_linear(x, weight, block_size, weight_scale, bias) -> output or None: group quant, GEMM, bias
PyObject* block_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w, ws, bias;
  if (n != 5 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], w) || !is_128x128(a[2]) || !tensor_arg(a[3], ws)) DECLINE;
  if (!x.is_cuda()) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !is_half(dt) || x.dim() < 1 || x.numel() == 0 || !x.is_contiguous()) DECLINE;
  const int64_t K = x.size(-1), M = x.numel() / K;
  if (K % 128 != 0 || !block_weight(w, ws, K, dev)) DECLINE;
  const int64_t N = w.size(0);
  if (a[4] != Py_None) {
    if (!tensor_arg(a[4], bias) || !plain(bias, dev) || bias.dim() != 1 || bias.size(0) != N || bias.scalar_type() != dt || !bias.is_contiguous()) DECLINE;
  }

  Tensor out;
  {
    Call c(x);
    OBSERVED("block_linear", x, w, ws, bias);
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    out = empty(shape, dt, x.device());
    const int64_t wsb = fp8k_linear_workspace_bytes(M, N, K, 1);
    Scratch mem(wsb, c.stream);
    check(fp8k_block_linear(x.data_ptr(), w.data_ptr(), ws.data_ptr<float>(), bias.defined() ? bias.data_ptr() : nullptr, out.data_ptr(), M,
                            N, K, K, ws.stride(0), ws.stride(1), N, kEps, code(dt), wsb ? mem.take(wsb) : nullptr, wsb, c.stream));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// block_matmul(A, B, As, Bs, block_size, out_dtype, scales_pow2) -> C or None: the GEMM on quantised activations, with
// float32 activation scales or, where the weight scales are known to be powers of two, packed UE8M0 ones
PyObject* block_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w, xs, ws;
  if (n != 7 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], w) || !tensor_arg(a[2], xs) || !tensor_arg(a[3], ws))
    DECLINE;
  if (!is_128x128(a[4]) || !THPDtype_Check(a[5]) || !x.is_cuda()) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  const bool pow2 = truth(a[6]);
  if (!plain(x, dev) || !is_fp8(x) || x.dim() != 2 || x.numel() == 0 || !x.is_contiguous() || !is_half(dt)) DECLINE;
  const int64_t M = x.size(0), K = x.size(1), kb = ceil_div(K, 128);
  if (K % 16 != 0 || !block_weight(w, ws, K, dev)) DECLINE;
  const int64_t N = w.size(0);
  if (!plain(xs, dev) || xs.dim() != 2 || xs.size(0) != M || !non_negative_strides(xs)) DECLINE;
  const bool packed = xs.scalar_type() == ScalarType::Int;
  if (packed) {
    // the matrix core applies the exponents in the tile kernels only (above 128 rows)
    if (!pow2 || M <= 128 || K % 128 != 0 || xs.size(1) != ceil_div(kb, 4)) DECLINE;
  } else if (xs.scalar_type() != ScalarType::Float || xs.size(1) != kb) {
    DECLINE;
  }

  void* work;
  int64_t bytes;
  if (!stream_workspace(x, fp8k_block_gemm_workspace_bytes(M, N, K), work, bytes)) return nullptr;
  Tensor out;
  {
    Call c(x);
    OBSERVED("block_matmul", x, w, xs, ws);
    out = empty({M, N}, dt, x.device());
    std::unique_lock<std::mutex> together;
    if (work) together = std::unique_lock<std::mutex>(workspace_lock(work));
    if (packed)
      check(fp8k_block_gemm_ue8m0(x.data_ptr(), w.data_ptr(), xs.data_ptr<int32_t>(), ws.data_ptr<float>(), out.data_ptr(), M, N, K, K,
                                  K, xs.stride(0), xs.stride(1), ws.stride(0), ws.stride(1), N, code(dt), work, bytes, c.stream));
    else
      check(fp8k_block_gemm(x.data_ptr(), w.data_ptr(), xs.data_ptr<float>(), ws.data_ptr<float>(), out.data_ptr(), M, N, K, K, K,
                            xs.stride(0), xs.stride(1), ws.stride(0), ws.stride(1), N, code(dt), work, bytes, c.stream));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- per-token linear
// token_linear(x, weight, weight_scale, bias, per_token) -> output or None: dynamic per-token quant, row-scaled GEMM, bias.
// per_token: the caller asked for per-token scales; without it only a per-channel weight scale implies them.
PyObject* token_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w, ws, bias;
  if (n != 5 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], w) || !tensor_arg(a[2], ws) || !x.is_cuda()) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !is_half(dt) || x.dim() < 1 || x.numel() == 0 || !x.is_contiguous()) DECLINE;
  const int64_t K = x.size(-1), M = x.numel() / K;
  if (!plain(w, dev) || !is_fp8(w) || w.dim() != 2 || w.size(0) != K || K % 16 != 0 || K <= 1) DECLINE;
  const int64_t N = w.size(1);
  if (N <= 0 || N % 8 != 0 || w.stride(0) != 1 || (N > 1 && w.stride(1) < K)) DECLINE;
  if (!plain(ws, dev) || ws.scalar_type() != ScalarType::Float || !ws.is_contiguous()) DECLINE;
  if (ws.numel() != N && !(ws.numel() == 1 && truth(a[4]))) DECLINE;
  if (a[3] != Py_None) {
    if (!tensor_arg(a[3], bias) || !plain(bias, dev) || bias.numel() != N || !bias.is_contiguous()) DECLINE;
    if (bias.scalar_type() != dt && bias.scalar_type() != ScalarType::Float) DECLINE;
  }

  Tensor out;
  {
    Call c(x);
    OBSERVED("token_linear", x, w, ws, bias);
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    out = empty(shape, dt, x.device());
    const int64_t wsb = fp8k_linear_workspace_bytes(M, N, K, 0);
    Scratch mem(wsb, c.stream);
    check(fp8k_token_linear(x.data_ptr(), w.data_ptr(), ws.data_ptr<float>(), ws.numel() == 1 ? 0 : 1, bias.defined() ? bias.data_ptr() : nullptr,
                            bias.defined() ? code(bias.scalar_type()) : FP8K_F32, out.data_ptr(), M, N, K, N > 1 ? w.stride(1) : K, N, code(dt),
                            wsb ? mem.take(wsb) : nullptr, wsb, c.stream));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- absorbed products
// Three zeroed int32 per (device, stream) for fp8k_tensor_quant_mla_sync, made on first use and kept: at most kMaxSync of them.  What
// makes one stream of a handle are torch's own streams, which live as long as the process.  A stream that came in from outside (its
// id is its handle) may be destroyed and its handle given to another while launches are queued, and hipStreamPerThread is one handle
// for a stream of every thread.  Those get none and take the two launches, as do calls under graph capture, whose replays may
// run on any stream.
constexpr size_t kMaxSync = 64;
int32_t* stream_sync(const Tensor& like, const c10::hip::HIPStream& stream) {
  const hipStream_t st = stream.stream();
  if (st && (uint64_t)stream.id() == (uint64_t)(uintptr_t)st) return nullptr;
  hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(st, &capturing) != hipSuccess) {
    (void)hipGetLastError();  // the launches report what is wrong with the stream, not this question
    return nullptr;
  }
  if (capturing != hipStreamCaptureStatusNone) return nullptr;
  static std::mutex mutex;
  static auto* const words = new std::map<std::pair<int, hipStream_t>, Tensor>;  // lives as long as the process
  const auto key = std::make_pair((int)like.get_device(), st);
  {
    std::lock_guard<std::mutex> lock(mutex);
    const auto it = words->find(key);
    if (it != words->end()) return it->second.data_ptr<int32_t>();
    if (words->size() >= kMaxSync) return nullptr;
  }
  // outside the lock, as it may wait for the device; of two threads on one stream the first to come back decides
  Tensor fresh = at::zeros({3}, like.options().dtype(ScalarType::Int));  // on the current stream, which is st
  std::lock_guard<std::mutex> lock(mutex);
  return words->emplace(key, std::move(fresh)).first->second.data_ptr<int32_t>();
}

// mla_quant(x, x_s, eps) -> x_q or None
PyObject* mla_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, s;
  if (n != 3 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], s) || !PyFloat_Check(a[2]) || !x.is_cuda()) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !plain(s, dev) || x.dim() != 3 || x.stride(2) != 1 || x.numel() == 0) DECLINE;
  if (!(is_half(dt) || dt == ScalarType::Float) || s.scalar_type() != ScalarType::Float || s.dim() != 1 || s.size(0) != 1) DECLINE;
  const float eps = (float)PyFloat_AS_DOUBLE(a[2]);
  Tensor q;
  {
    Call c(x);
    OBSERVED("mla_quant", x, s);
    q = empty(x.sizes(), ScalarType::Float8_e4m3fn, x.device());
    int32_t* const sync = fp8k_tensor_quant_mla_takes_sync(x.numel()) ? stream_sync(x, c10::hip::getCurrentHIPStream(dev)) : nullptr;
    check(fp8k_tensor_quant_mla_sync(x.data_ptr(), q.data_ptr(), s.data_ptr<float>(), x.size(0), x.size(1), x.size(2), x.stride(0),
                                     x.stride(1), eps, code(dt), sync, c.stream));
  }
  return THPVariable_Wrap(std::move(q));
  END_HANDLE_TH_ERRORS
}

// bmm(A, B, A_scale, B_scale, dtype) -> [b, m, n] or None
PyObject* bmm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor A, B, as, bs;
  if (n != 5 || modes_active() || !tensor_arg(a[0], A) || !tensor_arg(a[1], B) || !tensor_arg(a[2], as) || !tensor_arg(a[3], bs))
    DECLINE;
  if (!THPDtype_Check(a[4]) || !A.is_cuda()) DECLINE;
  const int dev = A.get_device();
  const ScalarType dt = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  if (!plain(A, dev) || !plain(B, dev) || !plain(as, dev) || !plain(bs, dev) || !is_half(dt) || !is_fp8(A) || !is_fp8(B)) DECLINE;
  if (A.dim() != 3 || B.dim() != 3 || A.size(0) != B.size(0) || A.size(2) != B.size(1) || A.numel() == 0 || B.numel() == 0) DECLINE;
  const int64_t b = A.size(0), m = A.size(1), k = A.size(2), nn = B.size(2);
  if (A.stride(2) != 1 || B.stride(1) != 1 || k % 128 != 0 || nn % 8 != 0) DECLINE;
  if (as.numel() != 1 || bs.numel() != 1 || as.scalar_type() != ScalarType::Float || bs.scalar_type() != ScalarType::Float) DECLINE;
  Tensor out;
  {
    Call c(A);
    OBSERVED("bmm", A, B, as, bs);
    out = empty({b, m, nn}, dt, A.device());
    check(fp8k_bmm_fp8_tensor_scales(A.data_ptr(), B.data_ptr(), as.data_ptr<float>(), bs.data_ptr<float>(), out.data_ptr(), b, m, nn, k,
                       b > 1 ? A.stride(0) : m * k, m > 1 ? A.stride(1) : k, b > 1 ? B.stride(0) : nn * k, nn > 1 ? B.stride(2) : k,
                       m * nn, nn, code(dt), c.stream));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- experts
// fused_gate(logits, bias, groups, topk_group, topk, shared_experts, scaling, scale_output) -> (weights, ids) or None
PyObject* fused_gate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, bias;
  if (n != 8 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], bias) || !x.is_cuda()) DECLINE;
  for (int i = 2; i < 6; ++i)
    if (!PyLong_Check(a[i])) DECLINE;
  if (!PyFloat_Check(a[6])) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !plain(bias, dev) || x.dim() != 2 || bias.dim() != 1 || bias.size(0) != x.size(1) || x.size(0) == 0) DECLINE;
  if (bias.scalar_type() != dt || !(is_half(dt) || dt == ScalarType::Float) || !x.is_contiguous() || !bias.is_contiguous()) DECLINE;
  const int64_t rows = x.size(0), groups = PyLong_AsLongLong(a[2]), topk_group = PyLong_AsLongLong(a[3]);
  const int64_t topk = PyLong_AsLongLong(a[4]), shared = PyLong_AsLongLong(a[5]);
  const double scaling = PyFloat_AS_DOUBLE(a[6]);
  const bool scale_output = truth(a[7]);
  if (topk <= 0 || PyErr_Occurred()) DECLINE;
  Tensor w, ids;
  {
    Call c(x);
    OBSERVED("fused_gate", x, bias);
    w = empty({rows, topk}, ScalarType::Float, x.device());
    ids = empty({rows, topk}, ScalarType::Int, x.device());
    check(fp8k_moe_fused_gate(x.data_ptr(), bias.data_ptr(), w.data_ptr<float>(), ids.data_ptr<int32_t>(), rows, x.size(1), groups,
                              topk_group, topk, shared, scaling, scale_output ? 1 : 0, code(dt), c.stream));
  }
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(w)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(ids)));
  return out;
  END_HANDLE_TH_ERRORS
}

// expert weights: w e4m3fn [E, rows, K] contiguous, scale float32 [E, ceil(rows/128), K/128]
bool expert_weight(const Tensor& w, const Tensor& s, int dev) {
  if (!plain(w, dev) || !plain(s, dev) || !is_fp8(w) || w.dim() != 3 || !w.is_contiguous() || w.numel() == 0) return false;
  return s.scalar_type() == ScalarType::Float && s.dim() == 3 && non_negative_strides(s) && s.size(0) == w.size(0) &&
         s.size(1) == ceil_div(w.size(1), 128) && s.size(2) == ceil_div(w.size(2), 128) && w.size(2) % 128 == 0;
}

// fused_experts(x, w13, w2, w13_scale, w2_scale, topk_weights, topk_ids, block_m, balanced, fuse_gemm1, weight_on_input,
//               scaling, inplace) -> output or None: the gated silu experts of fused_moe.fused_experts_impl in one call.  The
// decisions (block_m, balanced, fuse_gemm1) are the Python side's.
PyObject* fused_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w13, w2, s13, s2, tw, ids;
  if (n != 13 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], w13) || !tensor_arg(a[2], w2) || !tensor_arg(a[3], s13) ||
      !tensor_arg(a[4], s2) || !tensor_arg(a[5], tw) || !tensor_arg(a[6], ids) || !x.is_cuda())
    DECLINE;
  if (!PyLong_Check(a[7]) || !PyFloat_Check(a[11])) DECLINE;
  const int64_t bm = PyLong_AsLongLong(a[7]);
  const bool balanced = truth(a[8]), fuse = truth(a[9]), on_input = truth(a[10]), inplace = truth(a[12]);
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !is_half(dt) || x.dim() != 2 || x.numel() == 0 || !x.is_contiguous()) DECLINE;
  if (!expert_weight(w13, s13, dev) || !expert_weight(w2, s2, dev)) DECLINE;
  const int64_t T = x.size(0), H = x.size(1), E = w13.size(0), N = w13.size(1), I = N / 2;
  if (w13.size(2) != H || w2.size(0) != E || w2.size(1) != H || w2.size(2) != I || N % 256 != 0 || H % 128 != 0) DECLINE;
  if (!plain(tw, dev) || !plain(ids, dev) || tw.dim() != 2 || ids.dim() != 2 || tw.sizes() != ids.sizes() || ids.size(0) != T) DECLINE;
  if (tw.scalar_type() != ScalarType::Float || !tw.is_contiguous() || !ids.is_contiguous()) DECLINE;
  const bool ids64 = ids.scalar_type() == ScalarType::Long;
  if (!ids64 && ids.scalar_type() != ScalarType::Int) DECLINE;
  const int64_t topk = ids.size(1), slots = T * topk;
  if (topk <= 0 || bm <= 0 || (fuse && (bm != 256 || on_input)) || (balanced && bm != 256)) DECLINE;

  const int64_t cap = slots + (E + 1) * (bm - 1), blocks = ceil_div(cap, bm);
  // what of the table can be in use (a block holds at least one slot, and only an expert's last is not full): the launches
  // are sized by it, 7168 workgroups less for 2 tokens of 128 experts
  const int64_t cap_used = std::min(cap, bm * std::min(slots, E + 1 + slots / bm));
  const int64_t kb1 = H / 128, kb2 = I / 128;
  const bool act_gemm2 = !fuse && fp8k_moe_act_block_gemm_takes(bm, H, I, I);  // silu_and_mul and requantisation inside GEMM 2
  const bool sorted = bm >= 64;  // blocks of 64 slots and more read their activation scales in slot order
  const float scaling = (float)PyFloat_AS_DOUBLE(a[11]);
  Tensor out;
  {
    Call c(x);
    OBSERVED("fused_experts", x, w13, w2, s13, s2, tw, ids);
    out = inplace ? x : empty(x.sizes(), dt, x.device());
    const int64_t b_ids = cap * 4, b_q1 = T * H, b_s1 = T * kb1 * 4, b_ss1 = cap * kb1 * 4, b_mid = slots * N * 2, b_q2 = slots * I,
                  b_s2 = slots * kb2 * 4, b_ss2 = cap * kb2 * 4, b_out = slots * H * 2;
    using S = Scratch;
    Scratch mem(2 * S::room(b_ids) + S::room(blocks * 4) + S::room(4) + S::room((E + 2) * 4) + S::room(b_q1) + S::room(b_s1) +
                    (sorted ? S::room(b_ss1) + S::room(b_ss2) : 0) + (fuse ? 0 : S::room(b_mid) + S::room(b_s2)) + S::room(b_q2) +
                    S::room(b_out),
                c.stream);
    int32_t* sorted_ids = mem.take<int32_t>(b_ids);
    int32_t* even_ids = mem.take<int32_t>(b_ids);
    int32_t* block_expert = mem.take<int32_t>(blocks * 4);
    int32_t* padded = mem.take<int32_t>(4);
    int32_t* cumsum = mem.take<int32_t>((E + 2) * 4);
    void* q1 = mem.take(b_q1);
    float* s1 = mem.take<float>(b_s1);
    void* q2 = mem.take(b_q2);
    void* down = mem.take(b_out);
    float* ss1 = sorted ? mem.take<float>(b_ss1) : nullptr;
    float* ss2 = sorted ? mem.take<float>(b_ss2) : nullptr;
    void* mid = fuse ? nullptr : mem.take(b_mid);
    float* sm2 = fuse ? nullptr : mem.take<float>(b_s2);
    const int dc = code(dt);
    const float* twp = tw.data_ptr<float>();
    void* st = c.stream;

    // small blocks read their scales column-major per token, large ones get them gathered into slot order
    check(fp8k_moe_align_quant(ids.data_ptr(), ids64, slots, E + 1, bm, sorted_ids, cap, block_expert, blocks, padded, cumsum, x.data_ptr(), q1,
                               s1, T, H, kEps, dc, sorted ? kb1 : 1, sorted ? 1 : T, st));
    if (balanced) {
      check(fp8k_moe_balance_blocks(sorted_ids, block_expert, padded, cap, bm, slots, E, even_ids, st));
      sorted_ids = even_ids;
    }
    if (sorted) check(fp8k_moe_sort_scales(s1, ss1, sorted_ids, padded, cap, kb1, topk, slots, kb1, 1, st));
    auto gemm = [&](const void* A, const Tensor& W, const Tensor& Ws, const float* As, int64_t as_m, int64_t as_k, void* C, bool weigh,
                    int64_t per_row) {
      check(fp8k_moe_block_gemm(A, W.data_ptr(), As, Ws.data_ptr<float>(), C, sorted_ids, block_expert, padded, weigh ? twp : nullptr, cap_used,
                                bm, slots, per_row, E, W.size(1), W.size(2), W.size(2), as_m, as_k, W.stride(0), W.stride(1), Ws.stride(0),
                                Ws.stride(1), Ws.stride(2), W.size(1), dc, (sorted ? 1 : 0) | (balanced ? 2 : 0), st));
    };
    if (fuse) {
      check(fp8k_moe_block_gemm_silu_quant(q1, w13.data_ptr(), ss1, s13.data_ptr<float>(), q2, ss2, sorted_ids, block_expert, padded, cap,
                                           slots, topk, E, N, H, H, cap, w13.stride(0), w13.stride(1), s13.stride(0), s13.stride(1),
                                           s13.stride(2), I, cap, kEps, dc, balanced ? 1 : 0, st));
    } else {
      gemm(q1, w13, s13, sorted ? ss1 : s1, 1, sorted ? cap : T, mid, on_input, topk);
    }
    if (act_gemm2) {
      check(fp8k_moe_act_block_gemm(mid, w2.data_ptr(), s2.data_ptr<float>(), down, sorted_ids, block_expert, padded, on_input ? nullptr : twp,
                                    cap_used, bm, slots, E, H, I, N, w2.stride(0), I, s2.stride(0), s2.stride(1), s2.stride(2), H, kEps, dc, st));
    } else if (!fuse) {
      check(fp8k_silu_mul_group_quant(mid, q2, sm2, slots, I, 128, kEps, -448.f, 448.f, dc, sorted ? kb2 : 1, sorted ? 1 : slots,
                                      FP8K_SCALE_F32, st));
      if (sorted) check(fp8k_moe_sort_scales(sm2, ss2, sorted_ids, padded, cap, kb2, 1, slots, kb2, 1, st));
    }
    if (!act_gemm2) gemm(q2, w2, s2, sorted ? ss2 : sm2, 1, sorted ? cap : slots, down, !on_input, 1);
    check(fp8k_moe_sum_reduce(down, out.data_ptr(), T, topk, H, topk * H, H, H, scaling, dc, st));
  }
  if (inplace) {
    Py_INCREF(a[0]);
    return a[0];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- MXFP4
// codes uint8 [.., rows, K/2] with contiguous, 16-byte aligned rows, and their int32 scale words [.., rows, ceil(K/128)]
bool mx_operand(const Tensor& q, const Tensor& s, int64_t dim, int device) {
  if (!plain(q, device) || !plain(s, device) || q.scalar_type() != ScalarType::Byte || s.scalar_type() != ScalarType::Int) return false;
  if (q.dim() != dim || s.dim() != dim || q.numel() == 0 || q.stride(-1) != 1 || q.size(-1) % 16 != 0 || !non_negative_strides(s)) return false;
  if ((uintptr_t)q.data_ptr() % 16 != 0 || s.size(-1) != ceil_div(q.size(-1), 64)) return false;
  for (int64_t d = 0; d + 1 < dim; ++d)
    if (s.size(d) != q.size(d) || q.stride(d) % 16 != 0 || q.stride(d) < 0) return false;
  return q.size(-2) == 1 || q.stride(-2) >= q.size(-1);  // rows that overlap (an expanded one) are the dispatcher path's to copy
}

// rows of 16-bit or 32-bit activations that the kernels read as they lie in memory
bool mx_rows(const Tensor& x) {
  return x.dim() == 2 && x.numel() > 0 && x.stride(1) == 1 && (uintptr_t)x.data_ptr() % 16 == 0 &&
         (x.size(0) == 1 || (x.stride(0) >= x.size(1) && x.stride(0) % 8 == 0));
}
int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

bool mx_bias(const Tensor& bias, int64_t N, ScalarType dt, int device) {
  return plain(bias, device) && bias.numel() == N && bias.is_contiguous() && (bias.scalar_type() == dt || bias.scalar_type() == ScalarType::Float);
}

// mx_quant(x, fuse_silu_and_mul) -> (codes, scales) or None
PyObject* mx_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x;
  if (n != 2 || modes_active() || !tensor_arg(a[0], x) || !x.is_cuda() || !plain(x, x.get_device())) DECLINE;
  const bool fuse = truth(a[1]);
  const ScalarType dt = x.scalar_type();
  if (!(is_half(dt) || dt == ScalarType::Float) || !mx_rows(x)) DECLINE;
  const int64_t M = x.size(0), width = x.size(1), K = fuse ? width / 2 : width;
  if (K == 0 || K % 32 != 0 || (fuse && width % 2 != 0)) DECLINE;
  Tensor q, s;
  {
    Call c(x);
    OBSERVED("mx_quant", x);
    const int64_t ld = ceil_to(M, 4);
    q = empty({M, K / 2}, ScalarType::Byte, x.device());
    s = empty_column_major(M, ceil_div(K, 128), ld, ScalarType::Int, x.device());
    check(fp8k_mxfp4_quant(x.data_ptr(), q.data_ptr(), s.data_ptr(), M, K, row_stride(x), 1, ld, code(dt), fuse ? 1 : 0, c.stream));
  }
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(s)));
  return out;
  END_HANDLE_TH_ERRORS
}

// mx_dequant(q, s, dtype) -> values or None
PyObject* mx_dequant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, s;
  if (n != 3 || modes_active() || !tensor_arg(a[0], q) || !tensor_arg(a[1], s) || !THPDtype_Check(a[2]) || !q.is_cuda()) DECLINE;
  const ScalarType dt = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
  if (!(is_half(dt) || dt == ScalarType::Float) || (q.dim() != 2 && q.dim() != 3)) DECLINE;
  if (!mx_operand(q, s, q.dim(), q.get_device()) || !q.is_contiguous()) DECLINE;
  const int64_t E = q.dim() == 3 ? q.size(0) : 1, N = q.size(-2), K = q.size(-1) * 2;
  Tensor out;
  {
    Call c(q);
    OBSERVED("mx_dequant", q, s);
    c10::SmallVector<int64_t, 5> shape(q.sizes().begin(), q.sizes().end());
    shape.back() = K;
    out = empty(shape, dt, q.device());
    check(fp8k_mxfp4_dequant(q.data_ptr(), s.data_ptr(), out.data_ptr(), E, N, K, q.dim() == 3 ? s.stride(0) : 0, s.stride(-2), s.stride(-1),
                             code(dt), c.stream));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// mx_matmul(A, B, As, Bs, out_dtype, bias) -> C or None
PyObject* mx_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w, xs, ws, bias;
  if (n != 6 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], w) || !tensor_arg(a[2], xs) || !tensor_arg(a[3], ws)) DECLINE;
  if (!THPDtype_Check(a[4]) || !x.is_cuda()) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  if (!is_half(dt) || !mx_operand(x, xs, 2, dev) || !mx_operand(w, ws, 2, dev) || x.size(1) != w.size(1) || w.size(0) % 8 != 0) DECLINE;
  const int64_t M = x.size(0), N = w.size(0), K = x.size(1) * 2;
  if (a[5] != Py_None && (!tensor_arg(a[5], bias) || !mx_bias(bias, N, dt, dev))) DECLINE;
  Tensor out;
  {
    Call c(x);
    OBSERVED("mx_matmul", x, w, xs, ws, bias);
    out = empty({M, N}, dt, x.device());
    check(fp8k_mxfp4_gemm(x.data_ptr(), w.data_ptr(), xs.data_ptr(), ws.data_ptr(), bias.defined() ? bias.data_ptr() : nullptr, out.data_ptr(),
                          M, N, K, row_stride(x), row_stride(w), xs.stride(0), xs.stride(1), ws.stride(0), ws.stride(1), N, code(dt),
                          bias.defined() ? code(bias.scalar_type()) : FP8K_F32, c.stream));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// mx_linear(x, weight, weight_scale, bias) -> output or None: quantisation, product, bias
PyObject* mx_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w, ws, bias;
  if (n != 4 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], w) || !tensor_arg(a[2], ws) || !x.is_cuda()) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !is_half(dt) || x.dim() < 1 || x.numel() == 0) DECLINE;
  if (!(x.is_contiguous() || x.dim() == 2) || (x.dim() == 2 ? !mx_rows(x) : (uintptr_t)x.data_ptr() % 16 != 0)) DECLINE;
  if (!mx_operand(w, ws, 2, dev) || w.size(1) * 2 != x.size(-1) || w.size(0) % 8 != 0) DECLINE;
  const int64_t K = x.size(-1), M = x.numel() / K, N = w.size(0);
  if (a[3] != Py_None && (!tensor_arg(a[3], bias) || !mx_bias(bias, N, dt, dev))) DECLINE;
  Tensor out;
  {
    Call c(x);
    OBSERVED("mx_linear", x, w, ws, bias);
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    out = empty(shape, dt, x.device());
    const int64_t wsb = fp8k_mxfp4_linear_workspace_bytes(M, N, K);
    Scratch mem(wsb, c.stream);
    check(fp8k_mxfp4_linear(x.data_ptr(), w.data_ptr(), ws.data_ptr(), bias.defined() ? bias.data_ptr() : nullptr, out.data_ptr(), M, N, K,
                            x.dim() == 2 ? row_stride(x) : K, row_stride(w), ws.stride(0), ws.stride(1), N, code(dt),
                            bias.defined() ? code(bias.scalar_type()) : FP8K_F32, wsb ? mem.take(wsb) : nullptr, wsb, c.stream));
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// mx_experts(x, w1, w2, topk_weights, topk_ids, s1, s2, gelu, weight_on_input, scaling, inplace) -> output or None
PyObject* mx_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, w1, w2, tw, ids, s1, s2;
  if (n != 11 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], w1) || !tensor_arg(a[2], w2) || !tensor_arg(a[3], tw) ||
      !tensor_arg(a[4], ids) || !tensor_arg(a[5], s1) || !tensor_arg(a[6], s2) || !x.is_cuda() || !PyFloat_Check(a[9]))
    DECLINE;
  const bool gelu = truth(a[7]), on_input = truth(a[8]), inplace = truth(a[10]);
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !is_half(dt) || !mx_rows(x) || (inplace && !x.is_contiguous())) DECLINE;
  if (!mx_operand(w1, s1, 3, dev) || !mx_operand(w2, s2, 3, dev) || !w1.is_contiguous() || !w2.is_contiguous()) DECLINE;
  const int64_t T = x.size(0), H = x.size(1), E = w1.size(0), I = w1.size(1) / 2;
  if (w1.size(2) * 2 != H || w1.size(1) % 2 != 0 || w2.size(0) != E || w2.size(1) != H || w2.size(2) * 2 != I) DECLINE;
  if (!plain(tw, dev) || !plain(ids, dev) || tw.dim() != 2 || ids.dim() != 2 || tw.sizes() != ids.sizes() || ids.size(0) != T) DECLINE;
  if (tw.scalar_type() != ScalarType::Float || !tw.is_contiguous() || !ids.is_contiguous()) DECLINE;
  const bool ids64 = ids.scalar_type() == ScalarType::Long;
  if ((!ids64 && ids.scalar_type() != ScalarType::Int) || ids.size(1) == 0) DECLINE;
  const int64_t topk = ids.size(1);
  const float scaling = (float)PyFloat_AS_DOUBLE(a[9]);
  Tensor out;
  {
    Call c(x);
    OBSERVED("mx_experts", x, w1, w2, tw, ids, s1, s2);
    out = inplace ? x : empty({T, H}, dt, x.device());
    const int64_t wsb = fp8k_mxfp4_experts_workspace_bytes(T, topk, I);
    Scratch mem(wsb, c.stream);
    check(fp8k_mxfp4_experts(x.data_ptr(), w1.data_ptr(), w2.data_ptr(), s1.data_ptr(), s2.data_ptr(), tw.data_ptr<float>(), ids.data_ptr(), ids64,
                             out.data_ptr(), T, topk, E, H, I, row_stride(x), w1.stride(0), w2.stride(0), s1.stride(0), s1.stride(1), s1.stride(2),
                             s2.stride(0), s2.stride(1), s2.stride(2), gelu ? FP8K_ACT_GELU : FP8K_ACT_SILU, on_input, scaling, code(dt),
                             mem.take(wsb), wsb, c.stream));
  }
  if (inplace) {
    Py_INCREF(a[0]);
    return a[0];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- latent attention
constexpr int64_t kMlaLatent = 512, kMlaRope = 64, kMlaRow = kMlaLatent + kMlaRope, kMlaNope = 128, kMlaValue = 128;

bool aligned16(const Tensor& t) { return (uintptr_t)t.data_ptr() % 16 == 0; }

// rows that the kernels read as they lie: a contiguous last dimension, the others at multiples of 16 bytes
bool mla_rows(const Tensor& t, int64_t dim, int64_t last, ScalarType dt, int device) {
  if (!plain(t, device) || t.dim() != dim || t.scalar_type() != dt || t.size(-1) != last || t.stride(-1) != 1 || !aligned16(t)) return false;
  for (int64_t d = 0; d + 1 < dim; ++d)
    if (t.stride(d) % 8 != 0 || t.stride(d) < 0) return false;
  return true;
}

// a cache [pages, page_size, 576], and one float32 or nothing for its scale
bool mla_cache(const Tensor& cache, PyObject* so, Tensor& scale, ScalarType dt, int device) {
  if (!plain(cache, device) || cache.dim() != 3 || cache.size(2) != kMlaRow || cache.numel() == 0 || !cache.is_contiguous() || !aligned16(cache)) return false;
  if (cache.scalar_type() != dt && !is_fp8(cache)) return false;
  if (so == Py_None) return true;
  return is_fp8(cache) && tensor_arg(so, scale) && plain(scale, device) && scale.scalar_type() == ScalarType::Float && scale.numel() == 1;
}

bool ints(const Tensor& t, int64_t n, int device) {
  return plain(t, device) && t.dim() == 1 && t.size(0) == n && t.scalar_type() == ScalarType::Int && t.is_contiguous();
}
bool int_or_long(const Tensor& t, int64_t n, int device) {
  return plain(t, device) && t.dim() == 1 && t.size(0) == n && t.is_contiguous() && (t.scalar_type() == ScalarType::Int || t.scalar_type() == ScalarType::Long);
}
bool mla_table(const Tensor& t, int64_t rows, int device) {
  return plain(t, device) && t.dim() == 2 && t.size(0) == rows && t.scalar_type() == ScalarType::Int && t.size(1) > 0 && t.stride(1) == 1 && t.stride(0) >= 0;
}

float* float_or_null(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

PyObject* pair(PyObject* first, PyObject* second) {  // takes both
  PyObject* const out = first && second ? PyTuple_New(2) : nullptr;
  if (!out) {
    Py_XDECREF(first);
    Py_XDECREF(second);
    return nullptr;
  }
  PyTuple_SET_ITEM(out, 0, first);
  PyTuple_SET_ITEM(out, 1, second);
  return out;
}
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// mla_write(latent, cache, slots, norm_weight, eps, cos_sin, positions, neox, q_pe, scale, q_out) -> (done, rotated queries or None)
PyObject* mla_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
#define NOT_DONE                                    \
  do {                                              \
    PyErr_Clear();                                  \
    return pair(same(Py_False), same(Py_None));     \
  } while (0)
  Tensor x, cache, slots, weight, table, pos, q, scale, qo;
  if (n != 11 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], cache) || !tensor_arg(a[2], slots) || !PyFloat_Check(a[4]) || !x.is_cuda()) NOT_DONE;
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!is_half(dt) || !mla_rows(x, 2, kMlaRow, dt, dev) || x.size(0) == 0 || !mla_cache(cache, a[9], scale, dt, dev)) NOT_DONE;
  const int64_t T = x.size(0);
  if ((T > 1 && x.stride(0) < kMlaRow) || !int_or_long(slots, T, dev)) NOT_DONE;
  if (a[3] != Py_None) {
    if (!tensor_arg(a[3], weight) || !plain(weight, dev) || weight.dim() != 1 || weight.size(0) != kMlaLatent || !weight.is_contiguous() ||
        !aligned16(weight) || (weight.scalar_type() != dt && weight.scalar_type() != ScalarType::Float))
      NOT_DONE;
  }
  int64_t H = 0;
  if (a[5] != Py_None) {
    if (!tensor_arg(a[5], table) || !plain(table, dev) || table.scalar_type() != ScalarType::Float || table.dim() != 2 || table.size(0) == 0 ||
        table.size(1) != kMlaRope || !table.is_contiguous() || !aligned16(table) || !tensor_arg(a[6], pos) || !int_or_long(pos, T, dev))
      NOT_DONE;
    if (a[8] != Py_None) {
      if (!tensor_arg(a[8], q) || !mla_rows(q, 3, kMlaRope, dt, dev) || q.size(0) != T || q.size(1) == 0) NOT_DONE;
      if (a[10] != Py_None && (!tensor_arg(a[10], qo) || !mla_rows(qo, 3, kMlaRope, dt, dev) || qo.sizes() != q.sizes())) NOT_DONE;
      H = q.size(1);
    } else if (a[10] != Py_None) NOT_DONE;
  } else if (a[6] != Py_None || a[8] != Py_None || a[10] != Py_None) NOT_DONE;
#undef NOT_DONE
  const float eps = (float)PyFloat_AS_DOUBLE(a[4]);
  const bool neox = truth(a[7]), fresh = H > 0 && !qo.defined();
  {
    Call c(x);
    OBSERVED("mla_write", x, cache, slots, weight, table, pos, q);
    if (fresh) qo = empty(q.sizes(), dt, x.device());
    check(fp8k_mla_write_cache(x.data_ptr(), T > 1 ? x.stride(0) : kMlaRow, cache.data_ptr(), slots.data_ptr(), slots.scalar_type() == ScalarType::Long,
                               weight.defined() ? weight.data_ptr() : nullptr, weight.defined() ? code(weight.scalar_type()) : FP8K_F32, eps,
                               float_or_null(table), table.defined() ? table.size(0) : 0, pos.defined() ? pos.data_ptr() : nullptr,
                               pos.defined() && pos.scalar_type() == ScalarType::Long, neox, H ? q.data_ptr() : nullptr, H ? q.stride(0) : 0,
                               H ? q.stride(1) : 0, H ? qo.data_ptr() : nullptr, H ? qo.stride(0) : 0, H ? qo.stride(1) : 0, float_or_null(scale), T,
                               H, cache.numel() / kMlaRow, code(dt), is_fp8(cache), c.stream));
  }
  return pair(same(Py_True), H == 0 ? same(Py_None) : fresh ? THPVariable_Wrap(std::move(qo)) : same(a[10]));
  END_HANDLE_TH_ERRORS
}

// mla_gather(cache, page_table, cu_seqlens, num_tokens, starts, dtype, scale, out) -> rows or None
PyObject* mla_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor cache, table, cu, starts, scale, out;
  if (n != 8 || modes_active() || !tensor_arg(a[0], cache) || !tensor_arg(a[1], table) || !tensor_arg(a[2], cu) || !PyLong_Check(a[3]) ||
      !THPDtype_Check(a[5]) || !cache.is_cuda())
    DECLINE;
  const int dev = cache.get_device();
  const ScalarType dt = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  const int64_t tokens = PyLong_AsLongLong(a[3]);
  if (PyErr_Occurred() || tokens <= 0 || !is_half(dt) || !mla_cache(cache, a[6], scale, dt, dev) || cu.dim() != 1 || cu.size(0) < 2) DECLINE;
  const int64_t B = cu.size(0) - 1;
  if (!ints(cu, B + 1, dev) || !mla_table(table, B, dev)) DECLINE;
  if (a[4] != Py_None && (!tensor_arg(a[4], starts) || !ints(starts, B, dev))) DECLINE;
  const bool fresh = a[7] == Py_None;
  if (!fresh && (!tensor_arg(a[7], out) || !mla_rows(out, 2, kMlaRow, dt, dev) || out.size(0) != tokens || (tokens > 1 && out.stride(0) < kMlaRow))) DECLINE;
  {
    Call c(cache);
    OBSERVED("mla_gather", cache, table, cu);
    if (fresh) out = empty({tokens, kMlaRow}, dt, cache.device());
    check(fp8k_mla_gather_cache(cache.data_ptr(), table.data_ptr<int32_t>(), table.stride(0), table.size(1), cu.data_ptr<int32_t>(),
                                starts.defined() ? starts.data_ptr<int32_t>() : nullptr, float_or_null(scale), out.data_ptr(),
                                tokens > 1 ? out.stride(0) : kMlaRow, B, tokens, cache.size(0), cache.size(1), code(dt), is_fp8(cache), c.stream));
  }
  return fresh ? THPVariable_Wrap(std::move(out)) : same(a[7]);
  END_HANDLE_TH_ERRORS
}

// mla_decode(q_nope, q_pe, cache, page_table, seq_lens, sm_scale, scale, return_lse, out) -> output, (output, lse) or None
PyObject* mla_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, qp, cache, table, lens, scale, out, lse;
  if (n != 9 || modes_active() || !tensor_arg(a[0], q) || !tensor_arg(a[1], qp) || !tensor_arg(a[2], cache) || !tensor_arg(a[3], table) ||
      !tensor_arg(a[4], lens) || !PyFloat_Check(a[5]) || !q.is_cuda())
    DECLINE;
  const int dev = q.get_device();
  const ScalarType dt = q.scalar_type();
  const int64_t dim = q.dim();
  if (!is_half(dt) || (dim != 3 && dim != 4) || !mla_rows(q, dim, kMlaLatent, dt, dev) || !mla_rows(qp, dim, kMlaRope, dt, dev) || q.numel() == 0) DECLINE;
  const int64_t B = q.size(0), N = dim == 4 ? q.size(1) : 1, H = q.size(dim - 2);
  if (qp.size(0) != B || qp.size(dim - 2) != H || (dim == 4 && qp.size(1) != N)) DECLINE;
  if (!mla_cache(cache, a[6], scale, dt, dev) || !mla_table(table, B, dev) || !ints(lens, B, dev)) DECLINE;
  const double sm_scale = PyFloat_AS_DOUBLE(a[5]);
  if (!((float)sm_scale > 0.0f)) DECLINE;
  const bool want_lse = truth(a[7]), fresh = a[8] == Py_None;
  if (!fresh && (!tensor_arg(a[8], out) || !plain(out, dev) || out.scalar_type() != dt || out.sizes() != q.sizes() || !out.is_contiguous() || !aligned16(out))) DECLINE;
  {
    Call c(q);
    OBSERVED("mla_decode", q, qp, cache, table, lens);
    if (fresh) out = empty(q.sizes(), dt, q.device());
    if (want_lse) lse = empty(q.sizes().slice(0, dim - 1), ScalarType::Float, q.device());
    const int64_t wsb = fp8k_mla_decode_workspace_bytes(B, N, H, table.size(1) * cache.size(1));
    Scratch mem(wsb, c.stream);
    check(fp8k_mla_decode(q.data_ptr(), q.stride(0), dim == 4 ? q.stride(1) : 0, q.stride(dim - 2), qp.data_ptr(), qp.stride(0),
                          dim == 4 ? qp.stride(1) : 0, qp.stride(dim - 2), cache.data_ptr(), table.data_ptr<int32_t>(), table.stride(0), table.size(1),
                          lens.data_ptr<int32_t>(), float_or_null(scale), out.data_ptr(), float_or_null(lse), B, N, H, cache.size(0), cache.size(1),
                          (float)sm_scale, code(dt), is_fp8(cache), mem.take(wsb), wsb, c.stream));
  }
  PyObject* const result = fresh ? THPVariable_Wrap(std::move(out)) : same(a[8]);
  return want_lse ? pair(result, THPVariable_Wrap(std::move(lse))) : result;
  END_HANDLE_TH_ERRORS
}

// mla_prefill(q, k_nope, k_pe, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, sm_scale, causal, return_lse, out) -> output, (output, lse) or None
PyObject* mla_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, kn, kp, v, cu_q, cu_k, out, lse;
  if (n != 11 || modes_active() || !tensor_arg(a[0], q) || !tensor_arg(a[1], kn) || !tensor_arg(a[2], kp) || !tensor_arg(a[3], v) ||
      !tensor_arg(a[4], cu_q) || !tensor_arg(a[5], cu_k) || !PyLong_Check(a[6]) || !PyFloat_Check(a[7]) || !q.is_cuda())
    DECLINE;
  const int dev = q.get_device();
  const ScalarType dt = q.scalar_type();
  if (!is_half(dt) || !mla_rows(q, 3, kMlaNope + kMlaRope, dt, dev) || q.numel() == 0 || !mla_rows(kn, 3, kMlaNope, dt, dev) ||
      !mla_rows(v, 3, kMlaValue, dt, dev) || !mla_rows(kp, 2, kMlaRope, dt, dev))
    DECLINE;
  const int64_t Tq = q.size(0), H = q.size(1), Tk = kn.size(0);
  if (Tk == 0 || kn.size(1) != H || v.size(0) != Tk || v.size(1) != H || kp.size(0) != Tk || cu_q.dim() != 1 || cu_q.size(0) < 2) DECLINE;
  const int64_t B = cu_q.size(0) - 1, most = PyLong_AsLongLong(a[6]);
  if (PyErr_Occurred() || most < 0 || !ints(cu_q, B + 1, dev) || !ints(cu_k, B + 1, dev)) DECLINE;
  const double sm_scale = PyFloat_AS_DOUBLE(a[7]);
  if (!((float)sm_scale > 0.0f)) DECLINE;
  const bool causal = truth(a[8]), want_lse = truth(a[9]), fresh = a[10] == Py_None;
  if (!fresh && (!tensor_arg(a[10], out) || !plain(out, dev) || out.scalar_type() != dt || out.dim() != 3 || out.size(0) != Tq || out.size(1) != H ||
                 out.size(2) != kMlaValue || !out.is_contiguous() || !aligned16(out)))
    DECLINE;
  {
    Call c(q);
    OBSERVED("mla_prefill", q, kn, kp, v, cu_q, cu_k);
    if (fresh) out = empty({Tq, H, kMlaValue}, dt, q.device());
    if (want_lse) lse = empty({Tq, H}, ScalarType::Float, q.device());
    const int64_t wsb = fp8k_mla_prefill_workspace_bytes(B, H, Tq, Tk, most);
    Scratch mem(wsb, c.stream);
    check(fp8k_mla_prefill(q.data_ptr(), q.stride(0), q.stride(1), kn.data_ptr(), kn.stride(0), kn.stride(1), kp.data_ptr(), kp.stride(0), v.data_ptr(),
                           v.stride(0), v.stride(1), cu_q.data_ptr<int32_t>(), cu_k.data_ptr<int32_t>(), out.data_ptr(), float_or_null(lse), B, H, Tq,
                           Tk, most, (float)sm_scale, causal, code(dt), wsb ? mem.take(wsb) : nullptr, wsb, c.stream));
  }
  PyObject* const result = fresh ? THPVariable_Wrap(std::move(out)) : same(a[10]);
  return want_lse ? pair(result, THPVariable_Wrap(std::move(lse))) : result;
  END_HANDLE_TH_ERRORS
}

// merge_states(out_a, lse_a, out_b, lse_b) -> (out, lse) or None
PyObject* merge_states(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, sx, y, sy, out, lse;
  if (n != 4 || modes_active() || !tensor_arg(a[0], x) || !tensor_arg(a[1], sx) || !tensor_arg(a[2], y) || !tensor_arg(a[3], sy) || !x.is_cuda()) DECLINE;
  const int dev = x.get_device();
  const ScalarType dt = x.scalar_type();
  if (!plain(x, dev) || !plain(y, dev) || !(is_half(dt) || dt == ScalarType::Float) || y.scalar_type() != dt || x.dim() < 1 || x.numel() == 0 ||
      x.sizes() != y.sizes() || !x.is_contiguous() || !y.is_contiguous() || !aligned16(x) || !aligned16(y) || x.size(-1) % 8 != 0)
    DECLINE;
  for (const Tensor* s : {&sx, &sy})
    if (!plain(*s, dev) || s->scalar_type() != ScalarType::Float || !s->is_contiguous() || s->sizes() != x.sizes().slice(0, x.dim() - 1)) DECLINE;
  {
    Call c(x);
    OBSERVED("merge_states", x, sx, y, sy);
    out = empty(x.sizes(), dt, x.device());
    lse = empty(sx.sizes(), ScalarType::Float, x.device());
    check(fp8k_merge_attention_states(x.data_ptr(), sx.data_ptr<float>(), y.data_ptr(), sy.data_ptr<float>(), out.data_ptr(), lse.data_ptr<float>(),
                                      sx.numel(), x.size(-1), code(dt), c.stream));
  }
  return pair(THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
  END_HANDLE_TH_ERRORS
}

// set_workspace(registry, grow): the per-stream GEMM workspaces of sgl_kernel
PyObject* set_workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2 || !PyDict_Check(a[0]) || !PyCallable_Check(a[1])) {
    PyErr_SetString(PyExc_TypeError, "set_workspace(dict, callable)");
    return nullptr;
  }
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  g_workspaces = a[0];
  g_grow_workspace = a[1];
  Py_RETURN_NONE;
}

#define FN(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FN(group_quant), FN(block_linear), FN(block_matmul), FN(token_linear), FN(mla_quant),     FN(bmm),
                         FN(fused_gate),  FN(fused_experts), FN(mx_quant),     FN(mx_dequant),   FN(mx_matmul),
                         FN(mx_linear),   FN(mx_experts),    FN(mla_write),    FN(mla_gather),    FN(mla_decode),
                         FN(mla_prefill), FN(merge_states),  FN(set_workspace), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "native calls of the layer-level entry points", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
  PyObject* const overrides = PyImport_ImportModule("torch.overrides");
  if (!overrides) return nullptr;
  g_has_torch_function = PyObject_GetAttrString(overrides, "has_torch_function_unary");
  Py_DECREF(overrides);
  if (!g_has_torch_function) return nullptr;
  PyObject* const m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch", FP8K_TORCH_MARK) < 0) return nullptr;
  return m;
}
