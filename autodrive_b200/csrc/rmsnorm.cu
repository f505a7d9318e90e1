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
// CTAs are persistent, so that the weight is loaded once for many rows, the
// next row's loads are in flight while a row is worked on, and the backward
// sums the weight's gradient in registers, one partial row for each CTA, added
// up in a fixed order by a second kernel.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>
#include <vector>

#include "lm_host.h"
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

// Warps of a row: TPR / 32, but of wide rows as many as the row needs.
template <int TPR>
__device__ __forceinline__ int row_warps() { return TPR >= 512 ? blockDim.x >> 5 : TPR / 32; }

// Sum over the row's threads; every thread gets it. `red` holds one value per
// warp, twice, so that one barrier per row is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float s, float* red, int buf) {
  s = lm::warp_sum(s);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;   // a row's share of `red`: zeros where it has fewer warps
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* r = red + buf * 32;
    if (lane == 0) r[warp] = s;
    __syncthreads();
    const int first = TPR >= 256 ? 0 : warp / W * W;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += r[first + i];
  }
  return s;
}

constexpr int rows_per_cta(int tpr) { return tpr >= 256 ? 1 : 256 / tpr; }

// Aligned 16-bit rows fit three CTAs of 256 threads an SM, in 80 registers a
// thread, which spills none at 256 threads a row and at most 24 bytes at fewer
// (16384 x 4096 to 8 bits: 97 us with two, 88 with three).
template <typename T, bool VEC, bool FP8, int TPR, int NV>
__global__ void __launch_bounds__(TPR * rows_per_cta(TPR), VEC && sizeof(T) == 2 && TPR <= 256 ? 3 : 1)
rms_fwd_kernel(const FwdArgs a) {
  constexpr int RPB = rows_per_cta(TPR);
  __shared__ __align__(16) float red[64];
  if (threadIdx.x < 32) red[threadIdx.x] = red[threadIdx.x + 32] = 0.f;
  __syncthreads();
  const int W = row_warps<TPR>();
  const int lane = threadIdx.x & 31, part = TPR >= 256 ? threadIdx.x >> 5 : (threadIdx.x >> 5) % W;   // of the row
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
  // the next row is loaded while this one is worked on
  lm::RawSlice<T, VEC> next_x[NV], next_r[NV];
  const auto load = [&](int64_t r) {
    if (r >= a.rows) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) next_x[i].load(x + r * a.ldx, i * W + part, lane, a.d);
    if (res) {
#pragma unroll
      for (int i = 0; i < NV; ++i) next_r[i].load(res + r * a.ldres, i * W + part, lane, a.d);
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  load((int64_t)blockIdx.x * RPB + threadIdx.x / TPR);
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += step, buf ^= 1) {
    const int64_t r = r0 + threadIdx.x / TPR;
    const bool live = r < a.rows;
    float v[NV][8];
    float s = 0.f;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) next_x[i].get(v[i]);
      if (res) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float u[8];
          next_r[i].get(u);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = lm::to_f<T>(lm::from_f<T>(v[i][e] + u[e]));
        }
      }
      load(r + step);
      if (res) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          lm::store_slice<T, VEC>(reinterpret_cast<T*>(a.h) + r * a.d, i * W + part, lane, a.d, v[i]);
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
              if (c < a.d) q[c] = (uint8_t)(lm::e4m3x2(lm::e4m3_quotient(v[i][4 * g + e], dv), 0.f) & 0xff);
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
  constexpr int RPB = rows_per_cta(TPR);
  __shared__ __align__(16) float red[64];
  if (threadIdx.x < 32) red[threadIdx.x] = red[threadIdx.x + 32] = 0.f;
  __syncthreads();
  __shared__ float cols[RPB > 1 ? RPB * TPR * NV * 8 : 1];
  const int W = row_warps<TPR>();
  const int lane = threadIdx.x & 31, part = TPR >= 256 ? threadIdx.x >> 5 : (threadIdx.x >> 5) % W;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = lm::slice_col<VEC>(i * W + part, lane, e);
      w[i][e] = c < a.d ? a.w.at(c) : 0.f;
      dw[i][e] = 0.f;
    }
  // aligned rows are loaded one ahead; element by element that would cost too many registers
  lm::RawSlice<T, VEC> next_g[NV], next_h[NV], next_u[NV];
  float next_rstd = 0.f;
  const auto load = [&](int64_t r) {
    if (r >= a.rows) return;
    next_rstd = a.rstd[r];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      next_g[i].load(reinterpret_cast<const T*>(a.dy) + r * a.d, i * W + part, lane, a.d);
      next_h[i].load(reinterpret_cast<const T*>(a.h) + r * a.ldh, i * W + part, lane, a.d);
    }
    if (a.dh_out) {
#pragma unroll
      for (int i = 0; i < NV; ++i) next_u[i].load(reinterpret_cast<const T*>(a.dh_out) + r * a.d, i * W + part, lane, a.d);
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  if (VEC) load((int64_t)blockIdx.x * RPB + threadIdx.x / TPR);
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += step, buf ^= 1) {
    const int64_t r = r0 + threadIdx.x / TPR;
    const bool live = r < a.rows;
    float g[NV][8], n[NV][8];
    lm::RawSlice<T, VEC> u[NV];
    float s = 0.f, rstd = 0.f;
    if (live) {
      if (!VEC) load(r);
      rstd = next_rstd;
#pragma unroll
      for (int i = 0; i < NV; ++i) next_g[i].get(g[i]), next_h[i].get(n[i]), u[i] = next_u[i];
      if (VEC) load(r + step);
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
        float f[8];
        u[i].get(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[i][e] += f[e];
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

// Persistent CTAs: as many as fit on the SMs at once, so that none waits for a
// second round.
template <typename T, auto... V, typename K>
int grid_for(K* kernel, int64_t rows, int rpb, int threads) {
  static std::atomic<int> fits[64][33];   // of each kernel (T and V are its template arguments): by device and warps
  int dev = 0;
  TORCH_CHECK(cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64, "rms_norm: device query failed");
  auto& fit = fits[dev][threads / 32];
  int n = fit.load(std::memory_order_relaxed);
  if (n == 0) {
    TORCH_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) == cudaSuccess,
                "rms_norm: occupancy query failed");
    n = std::max(1, n);
    fit.store(n, std::memory_order_relaxed);
  }
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + rpb - 1) / rpb, (int64_t)lm::sm_count() * n));
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

// A CTA's threads: for wide rows no more warps than the row has chunks for.
int threads_for(int tpr, int nv, int64_t d) {
  return tpr < 512 ? tpr * rows_per_cta(tpr) : 32 * (int)(((d + 255) / 256 + nv - 1) / nv);
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

// `t` as rows of x's width: a view where its layout allows one.
torch::Tensor as_rows(const torch::Tensor& t) {
  const int64_t d = t.size(-1);
  torch::Tensor y = t.dim() == 2 ? t : t.reshape({t.numel() / d, d});
  const bool ok = y.numel() == 0 || ((d == 1 || y.stride(1) == 1) && (y.size(0) == 1 || y.stride(0) >= d));
  return ok ? y : y.contiguous();
}

void check_args(const torch::Tensor& x, const torch::Tensor& weight, const c10::optional<torch::Tensor>& residual) {
  LM_CHECK_VALUE(x.is_cuda() && x.dim() >= 1 && known_type(x.scalar_type()),
                    "rms_norm takes fp32, bf16 or fp16 rows");
  const int64_t d = x.size(-1);
  LM_CHECK_VALUE(d >= 1 && d <= kMaxWidth, "rms_norm rows are 1 to ", kMaxWidth, " wide, not ", d);
  LM_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == d && known_type(weight.scalar_type()) &&
                        weight.device() == x.device(),
                    "rms_norm needs an fp32, bf16 or fp16 weight [", d, "] on ", x.device());
  if (residual)
    LM_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() &&
                          residual->device() == x.device(),
                      "rms_norm needs a residual of x's shape, dtype and device");
}

WeightPtr weight_ptr(const torch::Tensor& w) {
  return WeightPtr{w.data_ptr(), w.scalar_type() == torch::kFloat32 ? 0 : (w.scalar_type() == torch::kBFloat16 ? 1 : 2)};
}

struct Forward {
  torch::Tensor y, h, rstd, q, scale;   // undefined where not asked for
};

// x [rows, D] and the residual are rows as as_rows() gives them; a contiguous weight.
Forward forward(const torch::Tensor& x, const torch::Tensor& residual, const torch::Tensor& weight, double eps, bool fp8,
                bool keep_rstd) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), d = x.size(1);
  Forward out;
  FwdArgs a{};
  a.x = x.data_ptr();
  a.rows = rows;
  a.d = (int)d;
  a.ldx = rows > 1 ? x.stride(0) : d;
  a.w = weight_ptr(weight);
  a.eps = (float)eps;
  a.groups = (int)((d + 127) / 128);
  bool vec = d % 8 == 0 && a.ldx % 8 == 0 && aligned(a.x);
  if (residual.defined()) {
    a.res = residual.data_ptr();
    a.ldres = rows > 1 ? residual.stride(0) : d;
    out.h = torch::empty({rows, d}, x.options());
    a.h = out.h.data_ptr();
    vec = vec && a.ldres % 8 == 0 && aligned(a.res);
  }
  if (keep_rstd) {
    out.rstd = torch::empty({rows}, x.options().dtype(torch::kFloat32));
    a.rstd = out.rstd.data_ptr<float>();
  }
  if (fp8) {
    a.ldq = (d + 15) / 16 * 16;
    out.q = torch::empty({rows, a.ldq}, x.options().dtype(torch::kFloat8_e4m3fn));
    if (a.ldq != d) out.q = out.q.narrow(1, 0, d);
    out.scale = torch::empty({rows, (int64_t)a.groups}, x.options().dtype(torch::kFloat32));
    a.q = reinterpret_cast<uint8_t*>(out.q.data_ptr());
    a.scale = out.scale.data_ptr<float>();
  } else {
    out.y = torch::empty({rows, d}, x.options());
    a.y = out.y.data_ptr();
  }
  if (rows == 0) return out;
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  for_type(x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    for_width(d, [&](auto tpr, auto nv) {
      constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
      const auto launch = [&](auto v8, auto q8) {
        constexpr bool VEC = decltype(v8)::value, FP8 = decltype(q8)::value;
        const int threads = threads_for(TPR, NV, d);
        const int grid = grid_for<T, VEC, FP8, TPR, NV>(rms_fwd_kernel<T, VEC, FP8, TPR, NV>, rows, rows_per_cta(TPR), threads);
        rms_fwd_kernel<T, VEC, FP8, TPR, NV><<<grid, threads, 0, st>>>(a);
      };
      if (vec && fp8) launch(std::true_type{}, std::true_type{});
      else if (vec) launch(std::true_type{}, std::false_type{});
      else if (fp8) launch(std::false_type{}, std::true_type{});
      else launch(std::false_type{}, std::false_type{});
    });
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "rms_norm forward launch failed");
  lm::count_launches(1);
  return out;
}

// {dx, dweight} of contiguous gradients; an undefined dh is zero.
std::pair<torch::Tensor, torch::Tensor> backward(const torch::Tensor& dy, const torch::Tensor& dh, const torch::Tensor& h,
                                                 const torch::Tensor& weight, const torch::Tensor& rstd) {
  const c10::cuda::CUDAGuard guard(h.device());
  const int64_t rows = h.size(0), d = h.size(1);
  auto dx = torch::empty({rows, d}, h.options());
  auto dw = rows > 0 ? torch::empty_like(weight) : torch::zeros_like(weight);
  if (rows == 0) return {dx, dw};
  BwdArgs a{};
  a.dy = dy.data_ptr();
  a.h = h.data_ptr();
  a.w = weight_ptr(weight);
  a.rstd = rstd.data_ptr<float>();
  a.rows = rows;
  a.ldh = rows > 1 ? h.stride(0) : d;
  a.d = (int)d;
  bool vec = d % 8 == 0 && a.ldh % 8 == 0 && aligned(a.h) && aligned(a.dy);
  if (dh.defined()) {
    a.dh_out = dh.data_ptr();
    vec = vec && aligned(a.dh_out);
  }
  a.dx = dx.data_ptr();
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  torch::Tensor part;
  int grid = 0;
  for_type(h.scalar_type(), [&](auto t) {
    using T = decltype(t);
    for_width(d, [&](auto tpr, auto nv) {
      constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
      const auto launch = [&](auto v8) {
        constexpr bool VEC = decltype(v8)::value;
        const int threads = threads_for(TPR, NV, d);
        grid = grid_for<T, VEC, TPR, NV>(rms_bwd_kernel<T, VEC, TPR, NV>, rows, rows_per_cta(TPR), threads);
        part = torch::empty({grid, d}, h.options().dtype(torch::kFloat32));
        a.part = part.data_ptr<float>();
        rms_bwd_kernel<T, VEC, TPR, NV><<<grid, threads, 0, st>>>(a);
      };
      if (vec) launch(std::true_type{});
      else launch(std::false_type{});
    });
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "rms_norm backward launch failed");
  for_type(weight.scalar_type(), [&](auto t) {
    using W = decltype(t);
    lm::sum_parts_kernel<W><<<(int)((d + lm::kSumColumns - 1) / lm::kSumColumns), 64 * lm::kSumColumns, 0, st>>>(part.data_ptr<float>(), grid, (int)d,
                                                                         reinterpret_cast<W*>(dw.data_ptr()));
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "rms_norm weight gradient launch failed");
  lm::count_launches(2);
  return {dx, dw};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct RmsNormFn : torch::autograd::Function<RmsNormFn> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& weight,
                               const c10::optional<torch::Tensor>& res, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const torch::Tensor residual = res ? *res : torch::Tensor();
    const auto x2 = as_rows(x), w = weight.contiguous();
    const Forward f = ::forward(x2, residual.defined() ? as_rows(residual) : residual, w, eps, false, true);
    ctx->set_materialize_grads(false);
    const auto y = f.y.view(x.sizes());
    // What the backward reads again is saved as the very tensor that the caller
    // holds (x, or the returned h), so that a change of it in place is noticed.
    if (!residual.defined()) {
      ctx->save_for_backward({x2.is_alias_of(x) ? x : x2, w, f.rstd});
      return {y};
    }
    const auto h = f.h.view(x.sizes());
    ctx->save_for_backward({h, w, f.rstd});
    return {y, h};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm has no second derivative (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const auto h = as_rows(saved[0]);
    const auto& dy = grads[0];
    const torch::Tensor dh = grads.size() > 1 ? grads[1] : torch::Tensor();
    const bool has_residual = grads.size() > 1;
    torch::Tensor dx, dw;
    if (dy.defined()) {
      const auto rows = [&](const torch::Tensor& g) { return g.reshape(h.sizes()).to(h.scalar_type()).contiguous(); };
      std::tie(dx, dw) = ::backward(rows(dy), dh.defined() ? rows(dh) : dh, h, saved[1], saved[2]);
      dx = dx.view(dy.sizes());
    } else {
      dx = dh;   // only the residual stream was used, or nothing at all
    }
    return {dx, dw, has_residual ? dx : torch::Tensor(), torch::Tensor()};
  }
};

// y, or (y, h) with a residual.
py::object rms_norm(torch::Tensor x, torch::Tensor weight, c10::optional<torch::Tensor> residual, double eps) {
  check_args(x, weight, residual);
  LM_CHECK_NO_TANGENT("rms_norm", x, weight, residual);
  const torch::Tensor res = residual ? *residual : torch::Tensor();
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (res.defined() && res.requires_grad()))) {
    const auto out = RmsNormFn::apply(x, weight, residual, eps);
    return residual ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
  }
  const Forward f = forward(as_rows(x), res.defined() ? as_rows(res) : res, weight.contiguous(), eps, false, false);
  const auto y = x.dim() == 2 ? f.y : f.y.view(x.sizes());
  if (!residual) return py::cast(y);
  return py::make_tuple(y, x.dim() == 2 ? f.h : f.h.view(x.sizes()));
}

// (q, scale), or (q, scale, h) with a residual.
py::tuple rms_norm_fp8(torch::Tensor x, torch::Tensor weight, c10::optional<torch::Tensor> residual, double eps) {
  check_args(x, weight, residual);
  LM_CHECK_VALUE(!lm::any_tangent(x, weight, residual) &&
                     !(at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() ||
                                                      (residual && residual->requires_grad()))),
                    "rms_norm_fp8 has no gradient: call it under torch.no_grad()");
  const Forward f = forward(as_rows(x), residual ? as_rows(*residual) : torch::Tensor(), weight.contiguous(), eps, true,
                            false);
  const auto q = lm::from_rows(f.q, x), scale = lm::from_rows(f.scale, x);
  if (!residual) return py::make_tuple(q, scale);
  return py::make_tuple(q, scale, f.h.view(x.sizes()));
}

}  // namespace

void register_rmsnorm_ops(py::module& m) {
  m.def("rms_norm", &rms_norm, "RMS norm of the last dimension with the residual's addition: y or (y, h), with autograd",
        py::arg("x"), py::arg("weight"), py::arg("residual"), py::arg("eps"));
  m.def("rms_norm_fp8", &rms_norm_fp8, "RMS norm with an e4m3 result: (q, scale) or (q, scale, h)", py::arg("x"),
        py::arg("weight"), py::arg("residual"), py::arg("eps"));
}
