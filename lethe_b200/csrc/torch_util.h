// What the PyTorch bindings share: errors, status words, tensors as the kernels read them.
#pragma once
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <mutex>
#include <string>
#include <vector>

#include "../../include/lethe_gdn.h"

namespace lethe_torch {

using at::Tensor;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int kMaxDevices = 64;

// ---------------------------------------------------------------------------------------------
// errors: lethe_b200.ops.GdnError, from threads with and without the interpreter lock
// ---------------------------------------------------------------------------------------------
inline PyObject* g_error_type = nullptr;

[[noreturn]] inline void fail(const std::string& msg, PyObject* type = g_error_type) {
  python_error e;
  {
    pybind11::gil_scoped_acquire gil;
    PyErr_SetString(type ? type : PyExc_RuntimeError, ("lethe_gdn: " + msg).c_str());
    e.persist();
  }
  throw e;
}
inline void check(int rc) {
  if (rc != 0) fail(std::string(lethe_gdn_strerror(rc)) + " (code " + std::to_string(rc) + ")");
}
// what a bound function throws has to be a Python error while the interpreter lock is held
template <typename F>
auto guarded(F&& f) -> decltype(f()) {
  try {
    return f();
  } catch (python_error& e) {
    e.restore();
    throw pybind11::error_already_set();
  }
}

// ---------------------------------------------------------------------------------------------
// Status words.  A device-side wait that gives up writes its code through `status` (host memory the GPU can write to,
// one word per device): nothing is copied, no event is recorded, and the host reads it at every later call.  An error
// therefore surfaces at a later call, as any asynchronous error does; the word is cleared when it has been reported.
// ---------------------------------------------------------------------------------------------
struct HostWords {
  volatile int32_t* status = nullptr;      // [kMaxDevices]
};
inline HostWords& host_words() {
  static HostWords w = [] {
    HostWords h;
    void* p = nullptr;
    if (cudaHostAlloc(&p, kMaxDevices * sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess)
      fail("no pinned host memory for the status words");
    memset(p, 0, kMaxDevices * sizeof(int32_t));
    h.status = static_cast<volatile int32_t*>(p);
    return h;
  }();
  return w;
}
inline int32_t* status_word(int dev) {
  TORCH_CHECK(dev >= 0 && dev < kMaxDevices);
  volatile int32_t* w = host_words().status + dev;
  const int32_t code = *w;
  if (code != 0) {
    *w = 0;
    if (code < 100)
      fail(std::string(lethe_gdn_strerror(code)) + " in an earlier call; the rows it was given for are not valid (code " + std::to_string(code) + ")");
    fail("a device-side wait of an earlier call timed out at site " + std::to_string(code) +
         "; the results of that call are invalid");
  }
  return const_cast<int32_t*>(w);
}

// ---------------------------------------------------------------------------------------------
// tensors
// ---------------------------------------------------------------------------------------------
// memory that does not hold the values: a negated view, a tensor of zeros without storage
inline bool lazy(const Tensor& t) { return t.is_neg() || t._is_zerotensor(); }
inline Tensor as(const Tensor& t, at::ScalarType dt) {
  if (t.scalar_type() != dt) return t.to(dt).contiguous();      // (writes them out)
  return lazy(t) ? t.clone().contiguous() : t.contiguous();
}
inline Tensor as32(const Tensor& t) { return t.defined() ? as(t, at::kFloat) : t; }
// a gate per channel is read through a tensor map, which wants its start on a 16-byte boundary
inline Tensor as_gate(const Tensor& t) {
  const Tensor r = as32(t);
  return r.defined() && (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) ? r.clone() : r;
}
inline Tensor opt(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
inline Tensor cast_back(const Tensor& t, at::ScalarType dt) { return t.scalar_type() == dt ? t : t.to(dt); }
template <typename T = void>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// Byte buffer for a workspace.  The library wants its start on a 1024-byte boundary, the allocator gives 512: the tensor
// is cut to the part that begins there.
constexpr int64_t kWorkspaceAlign = 1024;
inline bool workspace_aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % kWorkspaceAlign == 0; }
inline Tensor workspace(size_t bytes, const at::TensorOptions& o) {
  const int64_t n = static_cast<int64_t>(bytes);
  Tensor t = at::empty({n + kWorkspaceAlign}, o.dtype(at::kByte));
  const auto past = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr()) % kWorkspaceAlign);
  t.unsafeGetTensorImpl()->set_storage_offset(past ? kWorkspaceAlign - past : 0);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

inline cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

inline void need_shape(bool ok, const char* what) {
  if (!ok) fail(std::string("shapes do not match: ") + what);
}
// a pointer from somewhere else would fault in a kernel
template <typename... T>
void need_device(const Tensor& like, const T&... ts) {
  auto one = [&](const Tensor& t) {
    if (t.defined() && t.device() != like.device())
      fail("all inputs must live on one CUDA device (" + like.device().str() + " and " + t.device().str() + ")");
  };
  (one(ts), ...);
}

// the kernels would return the value without its tangent
inline void refuse_tangents(std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
      fail("forward-mode differentiation is not implemented", PyExc_NotImplementedError);
}

inline void need_cuda(const Tensor& t) {
  if (!t.is_cuda()) fail("inputs must live on a CUDA device (there is no CPU path)");
}
inline bool known(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
inline int32_t code(at::ScalarType t) { return t == at::kFloat ? LETHE_F32 : t == at::kBFloat16 ? LETHE_BF16 : LETHE_F16; }
inline void need_type(const Tensor& t, const char* name) {
  if (!known(t.scalar_type())) fail(std::string(name) + " must be fp32, bf16 or fp16");
}
inline void need_float(const Tensor& t, const char* name) {
  if (t.defined() && !at::isFloatingType(t.scalar_type())) fail(std::string(name) + " must be a real floating-point tensor");
}
// whether dimensions [from, end) of t lie in memory as one contiguous piece per index of those in front
inline bool packed_from(const Tensor& t, int64_t from) {
  int64_t want = 1;
  for (int64_t i = t.dim() - 1; i >= from; --i) {
    if (t.size(i) != 1 && t.stride(i) != want) return false;
    want *= t.size(i);
  }
  return true;
}
// stride of a dimension; one of a single index is never gone by, and its stride says nothing
inline int64_t step_of(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// places of tensors' memory from first to last byte, and whether two of them meet: by addresses, since two storages can stand for the same memory
inline std::pair<const char*, const char*> span_of(const Tensor& t) {
  const char* p = static_cast<const char*>(t.data_ptr());
  if (t.numel() == 0) return {p, p};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {p, p + (last + 1) * t.element_size()};
}
inline bool spans(const Tensor& a, const Tensor& b) {
  const auto x = span_of(a), y = span_of(b);
  return x.first < y.second && y.first < x.second;
}
// Several results in one allocation: bytes first, then tensors that are parts of them.  (An allocation costs the host about a microsecond.)
struct Parts {
  int64_t bytes = 0;
  Tensor whole;
  int64_t reserve(int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 15) / 16 * 16;
    return at;
  }
  void make(const Tensor& like) { whole = at::empty({bytes}, like.options().dtype(at::kByte)); }
  Tensor part(int64_t at, at::IntArrayRef sizes, at::ScalarType dt) const {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), c10::scalarTypeToTypeMeta(dt));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(c10::elementSize(dt)));
    return t;
  }
};
inline void need_index(const Tensor& t, const char* name) {
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) fail(std::string(name) + " must be int32 or int64");
}

void bind_block(pybind11::module_& m);      // torch_block.cpp
void bind_beam(pybind11::module_& m);       // torch_beam.cpp

}  // namespace lethe_torch
