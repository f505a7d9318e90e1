// Host-side helpers of the language-model operators.
#pragma once

#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAException.h>
#include <cuda_runtime.h>
#include <torch/extension.h>

#include <atomic>
#include <string>
#include <vector>

namespace lm {

// Message text without iostreams: where the linker finds only the static C++
// library, a string stream of this extension and the one of torch's libraries
// do not share a locale, and formatting an error message ends the process.
inline std::string text(const char* s) { return s; }
inline std::string text(int64_t v) { return std::to_string(v); }
inline std::string text(int v) { return std::to_string(v); }
inline std::string text(double v) { return std::to_string(v); }
inline std::string text(const c10::Device& d) { return d.str(); }
inline std::string text(c10::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}
template <typename... A>
std::string message(const A&... parts) {
  std::string s;
  ((s += text(parts)), ...);
  return s;
}
// Raises ValueError in Python.
#define LM_CHECK_VALUE(cond, ...) TORCH_CHECK_VALUE(cond, ::lm::message(__VA_ARGS__))

// Whether `t` carries a derivative of forward-mode differentiation (which
// neither requires_grad nor the gradient mode tells).
inline bool has_tangent(const torch::Tensor& t) {
  return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined();
}
inline bool has_tangent(const c10::optional<torch::Tensor>& t) { return t && has_tangent(*t); }
// Raises NotImplementedError in Python.
#define LM_CHECK_NO_TANGENT(name, ...) \
  TORCH_CHECK_NOT_IMPLEMENTED(!::lm::any_tangent(__VA_ARGS__), name " has no forward-mode derivative")
template <typename... T>
bool any_tangent(const T&... t) {
  return (has_tangent(t) || ...);
}

// Kernels launched by the operators whose autograd lives in this extension;
// utils/launches.py adds it to its own count.
inline std::atomic<int64_t>& launch_counter() {
  static std::atomic<int64_t> n{0};
  return n;
}
inline void count_launches(int n) { launch_counter().fetch_add(n, std::memory_order_relaxed); }

// SMs of the current device.
inline int sm_count() {
  static std::atomic<int> counts[64];
  int dev = 0;
  TORCH_CHECK(cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64, "device query failed");
  int n = counts[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    TORCH_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess, "device query failed");
    counts[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// rows [R, n] with x's leading dimensions in place of R (a view).
inline torch::Tensor from_rows(const torch::Tensor& rows, const torch::Tensor& x) {
  if (x.dim() == 2) return rows;
  auto sizes = x.sizes().vec();
  sizes.back() = rows.size(1);
  std::vector<int64_t> strides(sizes.size(), 1);
  int64_t s = rows.stride(0);
  for (int i = (int)sizes.size() - 2; i >= 0; --i) {
    strides[i] = s;
    s *= sizes[i];
  }
  return rows.as_strided(sizes, strides);
}

}  // namespace lm
