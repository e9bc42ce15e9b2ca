// What the host side of all operators shares: argument checks, device-side errors through a mailbox in mapped memory, and
// what every call does around its launches.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime_api.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <exception>
#include <mutex>
#include <optional>
#include <string>
#include <vector>

#include "../../include/fastlstm_b200.h"

namespace blstm_host {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// (A std::exception, because backward runs in a thread of the autograd engine, which carries those over to the caller.)
struct DeviceError : std::exception {
  int code;
  std::string where, text;
  DeviceError(int c, std::string w) : code(c), where(std::move(w)) {
    text = "fastlstm_b200 " + where + ": [" + std::to_string(code) + "] " + blstm_strerror(code);
    if (code == BLSTM_E_CUDA) text += std::string(": ") + blstm_last_cuda_error();
  }
  const char* what() const noexcept override { return text.c_str(); }
};

inline int g_flags = 0;              // BLSTM_FLAG_FORCE_GENERIC or 0
inline int g_wait_limit_us = 0;
inline bool g_sync_check = false;
inline PyObject* g_error_class = nullptr;

// One mailbox per device, kept for the life of the process.  [1] code, [2..3] detail.
constexpr int kMaxDevices = 64;
inline std::array<std::atomic<int32_t*>, kMaxDevices> g_mail{};
inline std::mutex g_mail_mutex;

inline void cuda_ok(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e));
}

inline int32_t* mailbox(int dev) {
  TORCH_CHECK(dev >= 0 && dev < kMaxDevices, "device index out of range");
  int32_t* m = g_mail[dev].load(std::memory_order_acquire);
  if (m) return m;
  std::lock_guard<std::mutex> lock(g_mail_mutex);
  m = g_mail[dev].load(std::memory_order_acquire);
  if (!m) {
    void* p = nullptr;
    cuda_ok(cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable), "cudaHostAlloc");
    m = static_cast<int32_t*>(p);
    for (int i = 0; i < 16; ++i) m[i] = 0;
    g_mail[dev].store(m, std::memory_order_release);
  }
  return m;
}

// Throws when a finished launch of this device has left an error.
inline void poll(int dev) {
  volatile int32_t* m = mailbox(dev);
  if (__builtin_expect(m[1] == 0, 1)) return;
  const int code = m[1], d0 = m[2], d1 = m[3];
  m[1] = 0;
  if (code == BLSTM_E_TOKEN) throw DeviceError{code, "token " + std::to_string(d1) + " at position " + std::to_string((uint32_t)d0)};
  if (code == BLSTM_E_PARENT) throw DeviceError{code, "parent " + std::to_string(d1) + " at position " + std::to_string((uint32_t)d0)};
  throw DeviceError{code, "recurrence (step " + std::to_string(d0) + ", batch tile " + std::to_string(d1) + ")"};
}

inline void check(int rc, const char* where) {
  if (rc != BLSTM_OK) throw DeviceError{rc, where};
}

inline int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return BLSTM_F32;
  if (t == at::kHalf) return BLSTM_F16;
  if (t == at::kBFloat16) return BLSTM_BF16;
  throw py::value_error(std::string("unsupported dtype ") + c10::toString(t) + "; expected float32, float16 or bfloat16");
}

inline std::string shape_str(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

inline void require(const Tensor& t, const char* name) {
  if (!t.is_cuda()) throw py::value_error(std::string(name) + " must be a CUDA tensor (there is no CPU path)");
  if (!t.is_contiguous()) throw py::value_error(std::string(name) + " must be contiguous");
}
inline void require(const Tensor& t, const char* name, at::ScalarType dt, const at::Device& dev, at::IntArrayRef shape) {
  require(t, name);
  if (t.scalar_type() != dt)
    throw py::value_error(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(dt));
  if (t.device() != dev) throw py::value_error(std::string(name) + " is on " + t.device().str() + ", expected " + dev.str());
  if (t.sizes() != shape) throw py::value_error(std::string(name) + " has shape " + shape_str(t.sizes()) + ", expected " + shape_str(shape));
}
inline void require(const OptTensor& t, const char* name, at::ScalarType dt, const at::Device& dev, at::IntArrayRef shape) {
  if (t) require(*t, name, dt, dev, shape);
}

inline const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
inline const void* ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }

// What every call does around its launches.  (`listen`: whether it throws what an earlier launch has left; not in the middle of several.)
struct Call {
  c10::cuda::CUDAGuard guard;
  int dev;
  void* stream;
  explicit Call(const at::Device& d, bool listen = true) : guard(d), dev(d.index()), stream(at::cuda::getCurrentCUDAStream(d.index()).stream()) {
    if (listen) poll(dev);
    blstm_set_mailbox(mailbox(dev));
  }
  ~Call() { blstm_set_mailbox(nullptr); }
  void done(const Tensor& ws, const char* where) {
    if (g_sync_check && ws.defined()) check(blstm_read_status(ws.const_data_ptr(), nullptr, stream), where);
  }
};

void bind_language(py::module_& m);   // host_language.cpp
void bind_norm(py::module_& m);       // host_norm.cpp
void bind_adamw(py::module_& m);      // host_adamw.cpp
void bind_beam(py::module_& m);       // host_beam.cpp

}  // namespace blstm_host
