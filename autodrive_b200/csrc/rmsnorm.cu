// Root-mean-square norm of rows with the residual's addition, its backward,
// and the form whose output is 8-bit with a scale for each 128 columns.
//
//   h = round(x + residual)            (the new residual stream; x alone without one)
//   y = h * rstd * w                   rstd = 1 / sqrt(mean(h^2) + eps)
//   dh = rstd (dy w - n c) + dh_out    n = h rstd, c = mean(dy w n)
//   dw = sum over rows of dy n
//
// The norm is taken of the rounded h, the value that is stored and that the
// backward reads again. Sums, rstd and the products are fp32; y, h and dh are
// rounded once to the rows' type.
//
// Bound by memory: every element is read and written once. A row is held in
// registers between the sum and the scaling, by as many threads as give each
// about 16 elements (32 lanes up to 512 columns, 1024 threads from 8193 on);
// CTAs are persistent, so that the weight is loaded once for many rows and
// the backward sums the weight's gradient in registers, one partial row for
// each CTA, added up in a fixed order by a second kernel.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "lm_vec.h"

namespace py = pybind11;

namespace {

constexpr int64_t kMaxWidth = 32768;

struct WeightPtr {
  const void* p;
  int kind;   // 0 fp32, 1 bf16, 2 fp16
  __device__ __forceinline__ float at(int c) const {
    if (kind == 0) return reinterpret_cast<const float*>(p)[c];
    if (kind == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[c]);
    return __half2float(reinterpret_cast<const __half*>(p)[c]);
  }
};

struct FwdArgs {
  const void* x;
  const void* res;      // null without a residual
  WeightPtr w;
  void* y;              // null in the 8-bit form
  void* h;              // null without a residual
  float* rstd;          // null when no backward follows
  uint8_t* q;           // the 8-bit form's values [rows][ldq]
  float* scale;         // [rows][groups]
  int64_t rows, ldx, ldres, ldq;
  int d, groups;
  float eps;
};

// Sum over the row's TPR threads; every thread gets it. `red` holds one value
// per warp, twice, so that one barrier per row is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float s, float* red, int buf) {
  s = lm::warp_sum(s);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* r = red + buf * 32;
    if (lane == 0) r[warp] = s;
    __syncthreads();
    const int first = warp / W * W;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += r[first + i];
  }
  return s;
}

constexpr int rows_per_cta(int tpr) { return tpr >= 256 ? 1 : 256 / tpr; }

template <typename T, bool VEC, bool FP8, int TPR, int NV>
__global__ void __launch_bounds__(TPR * rows_per_cta(TPR))
rms_fwd_kernel(const FwdArgs a) {
  constexpr int RPB = rows_per_cta(TPR), W = TPR / 32;
  __shared__ float red[64];
  const int lane = threadIdx.x & 31, part = (threadIdx.x >> 5) % W;   // this warp's part of the row
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* res = reinterpret_cast<const T*>(a.res);
  float w[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = lm::slice_col<VEC>(i * W + part, lane, e);
      w[i][e] = c < a.d ? a.w.at(c) : 0.f;
    }
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB, buf ^= 1) {
    const int64_t r = r0 + threadIdx.x / TPR;
    const bool live = r < a.rows;
    float v[NV][8];
    float s = 0.f;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) lm::load_slice<T, VEC>(x + r * a.ldx, i * W + part, lane, a.d, v[i]);
      if (res) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float u[8];
          lm::load_slice<T, VEC>(res + r * a.ldres, i * W + part, lane, a.d, u);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = lm::to_f<T>(lm::from_f<T>(v[i][e] + u[e]));
          lm::store_slice<T, VEC>(reinterpret_cast<T*>(a.h) + r * a.d, i * W + part, lane, a.d, v[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[i][e] * v[i][e];
    }
    s = row_sum<TPR>(s, red, buf);
    const float rstd = __frsqrt_rn(s / (float)a.d + a.eps);
    if (!live) continue;
    if (a.rstd && threadIdx.x % TPR == 0) a.rstd[r] = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * rstd * w[i][e];
      if constexpr (!FP8) {
        lm::store_slice<T, VEC>(reinterpret_cast<T*>(a.y) + r * a.d, i * W + part, lane, a.d, v[i]);
      } else {
        const int chunk = i * W + part;
        if (chunk * 256 >= a.d) break;   // the same for the whole warp
        uint8_t* q = a.q + r * a.ldq;
        float* sc = a.scale + r * a.groups + chunk * 2;
        if constexpr (VEC) {
          // a group is 16 neighbouring lanes
          uint32_t m = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) m = max(m, lm::abs_bits(v[i][e]));
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          const float gs = lm::group_scale(m);
          const lm::Divisor dv = lm::divisor(gs);
          const int c = lm::slice_col<true>(chunk, lane, 0);
          if (c < a.d) {
            *reinterpret_cast<uint2*>(q + c) = lm::quantize8(v[i], dv);
            if ((lane & 15) == 0) sc[lane >> 4] = gs;
          }
        } else {
          // the chunk's two groups are the elements 0-3 and 4-7 of all lanes
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) m = max(m, lm::abs_bits(v[i][4 * g + e]));
            m = __reduce_max_sync(0xffffffffu, m);
            if (chunk * 256 + g * 128 >= a.d) continue;
            const float gs = lm::group_scale(m);
            const lm::Divisor dv = lm::divisor(gs);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int c = lm::slice_col<false>(chunk, lane, 4 * g + e);
              if (c < a.d) q[c] = (uint8_t)(lm::e4m3x2(lm::quotient_to_odd(v[i][4 * g + e], dv), 0.f) & 0xff);
            }
            if (lane == 0) sc[g] = gs;
          }
        }
      }
    }
  }
}

struct BwdArgs {
  const void* dy;
  const void* h;
  const void* dh_out;   // null without a residual (or when nothing flows into h)
  WeightPtr w;
  const float* rstd;
  void* dx;
  float* part;          // [gridDim.x][d] partial weight gradients
  int64_t rows, ldh;
  int d;
};

template <typename T, bool VEC, int TPR, int NV>
__global__ void __launch_bounds__(TPR * rows_per_cta(TPR))
rms_bwd_kernel(const BwdArgs a) {
  constexpr int RPB = rows_per_cta(TPR), W = TPR / 32;
  __shared__ float red[64];
  __shared__ float cols[RPB > 1 ? RPB * TPR * NV * 8 : 1];
  const int lane = threadIdx.x & 31, part = (threadIdx.x >> 5) % W;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = lm::slice_col<VEC>(i * W + part, lane, e);
      w[i][e] = c < a.d ? a.w.at(c) : 0.f;
      dw[i][e] = 0.f;
    }
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB, buf ^= 1) {
    const int64_t r = r0 + threadIdx.x / TPR;
    const bool live = r < a.rows;
    float g[NV][8], n[NV][8];
    float s = 0.f, rstd = 0.f;
    if (live) {
      rstd = a.rstd[r];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        lm::load_slice<T, VEC>(reinterpret_cast<const T*>(a.dy) + r * a.d, i * W + part, lane, a.d, g[i]);
        lm::load_slice<T, VEC>(reinterpret_cast<const T*>(a.h) + r * a.ldh, i * W + part, lane, a.d, n[i]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          n[i][e] *= rstd;
          dw[i][e] += g[i][e] * n[i][e];
          g[i][e] *= w[i][e];
          s += g[i][e] * n[i][e];
        }
    }
    s = row_sum<TPR>(s, red, buf) / (float)a.d;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[i][e] = rstd * (g[i][e] - n[i][e] * s);
      if (a.dh_out) {
        float u[8];
        lm::load_slice<T, VEC>(reinterpret_cast<const T*>(a.dh_out) + r * a.d, i * W + part, lane, a.d, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[i][e] += u[e];
      }
      lm::store_slice<T, VEC>(reinterpret_cast<T*>(a.dx) + r * a.d, i * W + part, lane, a.d, g[i]);
    }
  }
  // one partial row for each CTA: the rows' shares are added in a fixed order
  float* out = a.part + (int64_t)blockIdx.x * a.d;
  if constexpr (RPB > 1) {
    constexpr int C = TPR * NV * 8;
    const int slot = threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) cols[slot * C + lm::slice_col<VEC>(i * W + part, lane, e)] = dw[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += TPR * RPB) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < RPB; ++k) s += cols[k * C + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = lm::slice_col<VEC>(i * W + part, lane, e);
        if (c < a.d) out[c] = dw[i][e];
      }
  }
}

// dw[c] = sum of the partial rows: 32 columns per CTA, 32 threads down each.
template <typename W>
__global__ void __launch_bounds__(1024) rms_dw_kernel(const float* part, int parts, int d, W* dw) {
  __shared__ float red[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < d)
    for (int p = threadIdx.y; p < parts; p += 32) s += part[(int64_t)p * d + c];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = lm::warp_sum(red[threadIdx.x][threadIdx.y]);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < d) dw[col] = lm::from_f<W>(s);
}

int sm_count() {
  int dev = 0, sms = 0;
  TORCH_CHECK(cudaGetDevice(&dev) == cudaSuccess &&
                  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess,
              "rms_norm: device query failed");
  return sms;
}

// Persistent CTAs: as many as fit on the SMs at once (2048 threads each).
int grid_for(int64_t rows, int tpr) {
  const int rpb = rows_per_cta(tpr), threads = tpr * rpb;
  const int64_t want = (rows + rpb - 1) / rpb;
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (int64_t)sm_count() * std::max(1, 1024 / threads)));
}

// Threads and 256-column chunks per row (see the file's comment).
template <typename F>
void for_width(int64_t d, F&& f) {
  const int64_t chunks = (d + 255) / 256;
  if (chunks <= 1) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  else if (chunks <= 2) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 2>{});
  else if (chunks <= 4) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  else if (chunks <= 8) f(std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{});
  else if (chunks <= 16) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  else if (chunks <= 32) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
  else if (chunks <= 64) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
}

template <typename F>
void for_type(torch::ScalarType t, F&& f) {
  if (t == torch::kFloat32) f(float{});
  else if (t == torch::kBFloat16) f(__nv_bfloat16{});
  else f(__half{});
}

bool known_type(torch::ScalarType t) {
  return t == torch::kFloat32 || t == torch::kBFloat16 || t == torch::kHalf;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

void check_rows(const torch::Tensor& t, const torch::Tensor& x, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), "rms_norm: ", name, " must be on x's device");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), "rms_norm: ", name, " must have x's dtype");
  TORCH_CHECK(t.dim() == 2 && t.sizes() == x.sizes(), "rms_norm: ", name, " must have x's shape");
  TORCH_CHECK(t.numel() == 0 || t.size(1) == 1 || t.stride(1) == 1, "rms_norm: ", name, "'s columns must be contiguous");
}

WeightPtr check_weight(const torch::Tensor& w, const torch::Tensor& x) {
  TORCH_CHECK(w.is_cuda() && w.device() == x.device(), "rms_norm: weight must be on x's device");
  TORCH_CHECK(known_type(w.scalar_type()) && w.dim() == 1 && w.size(0) == x.size(1) && w.is_contiguous(),
              "rms_norm: weight must be a contiguous fp32, bf16 or fp16 [D]");
  const int kind = w.scalar_type() == torch::kFloat32 ? 0 : (w.scalar_type() == torch::kBFloat16 ? 1 : 2);
  return WeightPtr{w.data_ptr(), kind};
}

void check_x(const torch::Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && known_type(x.scalar_type()),
              "rms_norm: x must be a CUDA fp32, bf16 or fp16 [rows, D] tensor");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= kMaxWidth, "rms_norm: D must be in 1..", kMaxWidth);
}

// Returns {y or q, h or undefined, rstd or undefined, scale or undefined}.
std::vector<c10::optional<torch::Tensor>> rms_norm_fwd(torch::Tensor x, c10::optional<torch::Tensor> residual,
                                                       torch::Tensor weight, double eps, bool fp8, bool keep_rstd) {
  check_x(x);
  check_rows(x, x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), d = x.size(1);
  FwdArgs a{};
  a.x = x.data_ptr();
  a.rows = rows;
  a.d = (int)d;
  a.ldx = rows > 1 ? x.stride(0) : d;
  a.w = check_weight(weight, x);
  a.eps = (float)eps;
  a.groups = (int)((d + 127) / 128);
  c10::optional<torch::Tensor> out, h, rstd, scale;
  bool vec = d % 8 == 0 && a.ldx % 8 == 0 && aligned(a.x);
  if (residual) {
    check_rows(*residual, x, "residual");
    a.res = residual->data_ptr();
    a.ldres = rows > 1 ? residual->stride(0) : d;
    h = torch::empty({rows, d}, x.options());
    a.h = h->data_ptr();
    vec = vec && a.ldres % 8 == 0 && aligned(a.res);
  }
  if (keep_rstd) {
    rstd = torch::empty({rows}, x.options().dtype(torch::kFloat32));
    a.rstd = rstd->data_ptr<float>();
  }
  if (fp8) {
    a.ldq = (d + 15) / 16 * 16;
    out = torch::empty({rows, a.ldq}, x.options().dtype(torch::kFloat8_e4m3fn)).narrow(1, 0, d);
    scale = torch::empty({rows, (int64_t)a.groups}, x.options().dtype(torch::kFloat32));
    a.q = reinterpret_cast<uint8_t*>(out->data_ptr());
    a.scale = scale->data_ptr<float>();
  } else {
    out = torch::empty({rows, d}, x.options());
    a.y = out->data_ptr();
  }
  if (rows > 0) {
    auto st = c10::cuda::getCurrentCUDAStream().stream();
    for_type(x.scalar_type(), [&](auto t) {
      using T = decltype(t);
      for_width(d, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        const int grid = grid_for(rows, TPR), threads = TPR * rows_per_cta(TPR);
        if (vec && fp8) rms_fwd_kernel<T, true, true, TPR, NV><<<grid, threads, 0, st>>>(a);
        else if (vec) rms_fwd_kernel<T, true, false, TPR, NV><<<grid, threads, 0, st>>>(a);
        else if (fp8) rms_fwd_kernel<T, false, true, TPR, NV><<<grid, threads, 0, st>>>(a);
        else rms_fwd_kernel<T, false, false, TPR, NV><<<grid, threads, 0, st>>>(a);
      });
    });
    TORCH_CHECK(cudaGetLastError() == cudaSuccess, "rms_norm forward launch failed");
  }
  return {out, h, rstd, scale};
}

// Returns {dx, dweight}.
std::vector<torch::Tensor> rms_norm_bwd(torch::Tensor dy, c10::optional<torch::Tensor> dh, torch::Tensor h,
                                        torch::Tensor weight, torch::Tensor rstd) {
  check_x(h);
  check_rows(h, h, "h");
  check_rows(dy, h, "dy");
  TORCH_CHECK(dy.is_contiguous(), "rms_norm: dy must be contiguous");
  TORCH_CHECK(rstd.is_cuda() && rstd.device() == h.device() && rstd.scalar_type() == torch::kFloat32 &&
                  rstd.numel() == h.size(0) && rstd.is_contiguous(), "rms_norm: rstd must be fp32 [rows]");
  const c10::cuda::CUDAGuard guard(h.device());
  const int64_t rows = h.size(0), d = h.size(1);
  BwdArgs a{};
  a.dy = dy.data_ptr();
  a.h = h.data_ptr();
  a.w = check_weight(weight, h);
  a.rstd = rstd.data_ptr<float>();
  a.rows = rows;
  a.ldh = rows > 1 ? h.stride(0) : d;
  a.d = (int)d;
  bool vec = d % 8 == 0 && a.ldh % 8 == 0 && aligned(a.h) && aligned(a.dy);
  if (dh) {
    check_rows(*dh, h, "dh");
    TORCH_CHECK(dh->is_contiguous(), "rms_norm: dh must be contiguous");
    a.dh_out = dh->data_ptr();
    vec = vec && aligned(a.dh_out);
  }
  auto dx = torch::empty({rows, d}, h.options());
  auto dw = rows > 0 ? torch::empty_like(weight) : torch::zeros_like(weight);
  if (rows == 0) return {dx, dw};
  a.dx = dx.data_ptr();
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  torch::Tensor part;
  int grid = 0;
  for_type(h.scalar_type(), [&](auto t) {
    using T = decltype(t);
    for_width(d, [&](auto tpr, auto nv) {
      constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
      grid = grid_for(rows, TPR);
      part = torch::empty({grid, d}, h.options().dtype(torch::kFloat32));
      a.part = part.data_ptr<float>();
      const int threads = TPR * rows_per_cta(TPR);
      if (vec) rms_bwd_kernel<T, true, TPR, NV><<<grid, threads, 0, st>>>(a);
      else rms_bwd_kernel<T, false, TPR, NV><<<grid, threads, 0, st>>>(a);
    });
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "rms_norm backward launch failed");
  for_type(weight.scalar_type(), [&](auto t) {
    using W = decltype(t);
    rms_dw_kernel<W><<<(int)((d + 31) / 32), dim3(32, 32), 0, st>>>(part.data_ptr<float>(), grid, (int)d,
                                                                  reinterpret_cast<W*>(dw.data_ptr()));
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "rms_norm weight gradient launch failed");
  return {dx, dw};
}

}  // namespace

void register_rmsnorm_ops(py::module& m) {
  m.def("rms_norm_fwd", &rms_norm_fwd,
        "RMS norm forward with the residual's addition: y (or 8-bit values), h, rstd, scales",
        py::arg("x"), py::arg("residual"), py::arg("weight"), py::arg("eps"), py::arg("fp8"), py::arg("keep_rstd"));
  m.def("rms_norm_bwd", &rms_norm_bwd, "RMS norm backward: dx, dweight", py::arg("dy"), py::arg("dh"), py::arg("h"),
        py::arg("weight"), py::arg("rstd"));
  m.attr("RMS_NORM_MAX_WIDTH") = kMaxWidth;
}
