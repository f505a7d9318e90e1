// Quantisation to e4m3 with fp32 scales for the 8-bit product: rows with one
// scale for each 128 columns (activations and gradients), and matrices with
// one scale for each 128 x 128 block (weights), optionally with the transposed
// copy that the input gradient's product reads.
//
// The values are exactly rounded (lm_vec.h), so a quantised tensor depends on
// its input's values alone, not on the kernel's order of operations. Bound by
// memory: one read of each element, one byte written (two with the
// transposed copy).
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <vector>

#include "fp8.h"
#include "lm_host.h"
#include "lm_vec.h"

namespace py = pybind11;

namespace {

// A warp takes 256 columns of a row, eight a lane: two groups of 128, the
// halves of the warp for aligned rows, the halves of every lane's columns
// otherwise. gridDim.y splits long rows between the CTAs.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
quant_rows_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                  int64_t rows, int k, int groups) {
  const int lane = threadIdx.x & 31, chunks = (groups + 1) / 2;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const T* row = x + r * ldx;
    uint8_t* out = q + r * ldq;
    float* sc = scale + r * groups;
    lm::RawSlice<T, VEC> next;
    next.load(row, blockIdx.y, lane, k);
    for (int chunk = blockIdx.y; chunk < chunks; chunk += gridDim.y) {
      float v[8];
      next.get(v);
      next.load(row, chunk + gridDim.y, lane, k);   // beyond the row: zeros
      if constexpr (VEC) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, lm::abs_bits(v[e]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = lm::group_scale(m);
        const int c = lm::slice_col<true>(chunk, lane, 0);
        if (c < k) {
          *reinterpret_cast<uint2*>(out + c) = lm::quantize8(v, lm::divisor(s));
          if ((lane & 15) == 0) sc[2 * chunk + (lane >> 4)] = s;
        }
      } else {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t m = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) m = max(m, lm::abs_bits(v[4 * g + e]));
          m = __reduce_max_sync(0xffffffffu, m);
          if (2 * chunk + g >= groups) continue;
          const float s = lm::group_scale(m);
          const lm::Divisor dv = lm::divisor(s);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = lm::slice_col<false>(chunk, lane, 4 * g + e);
            if (c < k) out[c] = (uint8_t)(lm::e4m3x2(lm::e4m3_quotient(v[4 * g + e], dv), 0.f) & 0xff);
          }
          if (lane == 0) sc[2 * chunk + g] = s;
        }
      }
    }
  }
}

// One CTA per 128 x 128 block, held in registers: warp w has the rows 8 i + w,
// 32 neighbouring columns an access. The values go out through shared memory,
// the transposed copy read down its columns.
template <typename T>
__global__ void __launch_bounds__(256)
quant_blocks_kernel(const T* __restrict__ w, int64_t ldw, uint8_t* __restrict__ q, int64_t ldq,
                    uint8_t* __restrict__ qt, int64_t ldqt, float* __restrict__ scale, float* __restrict__ scale_t,
                    int n, int k) {
  __shared__ uint8_t tile[128][132];
  __shared__ uint32_t red[8];
  const int bn = blockIdx.y, bk = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float v[16][4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = bn * 128 + i * 8 + warp;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = bk * 128 + j * 32 + lane;
      v[i][j] = row < n && col < k ? lm::to_f<T>(w[(int64_t)row * ldw + col]) : 0.f;
      m = max(m, lm::abs_bits(v[i][j]));
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  const float s = lm::group_scale(m);
  const lm::Divisor dv = lm::divisor(s);
  if (threadIdx.x == 0) {
    scale[bn * gridDim.x + bk] = s;
    if (scale_t) scale_t[bk * gridDim.y + bn] = s;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      tile[i * 8 + warp][j * 32 + lane] = (uint8_t)(lm::e4m3x2(lm::e4m3_quotient(v[i][j], dv), 0.f) & 0xff);
  __syncthreads();
  // four columns per thread and store; the last store of a row may run into its padding (rows are 16 bytes apart)
  for (int e = threadIdx.x; e < 128 * 32; e += 256) {
    const int r = e >> 5, c = (e & 31) * 4;
    if (bn * 128 + r < n && bk * 128 + c < k)
      *reinterpret_cast<uint32_t*>(q + (int64_t)(bn * 128 + r) * ldq + bk * 128 + c) =
          *reinterpret_cast<const uint32_t*>(&tile[r][c]);
  }
  if (!qt) return;
  for (int e = threadIdx.x; e < 128 * 32; e += 256) {
    const int r = e >> 5, c = (e & 31) * 4;   // row r of the transposed block is column r of the tile
    if (bk * 128 + r < k && bn * 128 + c < n) {
      const uint32_t u = tile[c][r] | (uint32_t)tile[c + 1][r] << 8 | (uint32_t)tile[c + 2][r] << 16 |
                         (uint32_t)tile[c + 3][r] << 24;
      *reinterpret_cast<uint32_t*>(qt + (int64_t)(bk * 128 + r) * ldqt + bn * 128 + c) = u;
    }
  }
}

// Partial column sums: a CTA takes 256 columns and every gridDim.y-th group of
// eight rows, one row a warp.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
column_sums_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int d, float* __restrict__ part) {
  __shared__ float red[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float acc[8] = {};
  const int64_t step = (int64_t)gridDim.y * 8;
  for (int64_t r = (int64_t)blockIdx.y * 8 + warp; r < rows; r += 4 * step) {
    lm::RawSlice<T, VEC> s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (r + j * step < rows) s[j].load(x + (r + j * step) * ldx, blockIdx.x, lane, d);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (r + j * step >= rows) continue;
      float v[8];
      s[j].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[warp][lm::slice_col<VEC>(0, lane, e)] = acc[e];
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += red[w][threadIdx.x];
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < d) part[(int64_t)blockIdx.y * d + c] = t;
}

template <typename F>
void for_type(torch::ScalarType t, F&& f) {
  if (t == torch::kFloat32) f(float{});
  else if (t == torch::kBFloat16) f(__nv_bfloat16{});
  else f(__half{});
}

// e4m3 [rows][cols] whose rows start 16 bytes apart, as the TMA unit reads them.
torch::Tensor empty_q(int64_t rows, int64_t cols, const torch::Tensor& like) {
  const int64_t ld = (cols + 15) / 16 * 16;
  auto q = torch::empty({rows, ld}, like.options().dtype(torch::kFloat8_e4m3fn));
  return ld == cols ? q : q.narrow(1, 0, cols);
}

void check_input(const torch::Tensor& x, int64_t dims, const char* what) {
  LM_CHECK_VALUE(x.is_cuda() && fp8::known_type(x.scalar_type()) && x.dim() >= dims, what,
                    " takes fp32, bf16 or fp16 tensors of at least ", dims, " dimension(s)");
  LM_CHECK_VALUE(x.size(-1) < (1ll << 30), what, ": too many columns");
}

}  // namespace

namespace fp8 {

bool known_type(torch::ScalarType t) {
  return t == torch::kFloat32 || t == torch::kBFloat16 || t == torch::kHalf;
}

torch::Tensor as_matrix(const torch::Tensor& t) {
  const int64_t k = t.size(-1);
  const auto y = t.dim() == 2 ? t : t.reshape({c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)), k});
  const bool ok = y.numel() == 0 || ((k == 1 || y.stride(1) == 1) && (y.size(0) == 1 || y.stride(0) >= k));
  return ok ? y : y.contiguous();
}

std::pair<torch::Tensor, torch::Tensor> quantize_rows(const torch::Tensor& x) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), k = x.size(1), groups = (k + 127) / 128;
  auto q = empty_q(rows, k, x);
  auto scale = torch::empty({rows, groups}, x.options().dtype(torch::kFloat32));
  if (rows == 0 || k == 0) return {q, scale};
  const int64_t ldx = rows > 1 ? x.stride(0) : k;
  const bool vec = k % 8 == 0 && ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  // eight warps a CTA, one row each; few rows are split between CTAs
  const int64_t ctas = (rows + 7) / 8, chunks = (groups + 1) / 2, room = (int64_t)lm::sm_count() * 8;
  const dim3 grid((unsigned)std::min<int64_t>(ctas, room),
                  (unsigned)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(chunks, 65535), room / ctas)));
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  for_type(x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    auto* out = reinterpret_cast<uint8_t*>(q.data_ptr());
    const T* in = reinterpret_cast<const T*>(x.data_ptr());
    const auto kernel = vec ? quant_rows_kernel<T, true> : quant_rows_kernel<T, false>;
    kernel<<<grid, 256, 0, st>>>(in, ldx, out, q.stride(0), scale.data_ptr<float>(), rows, (int)k, (int)groups);
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "quantize_rows launch failed");
  lm::count_launches(1);
  return {q, scale};
}

torch::Tensor column_sums(const torch::Tensor& x, torch::ScalarType out_type) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), d = x.size(1);
  auto out = torch::empty({d}, x.options().dtype(out_type));
  if (d == 0) return out;
  if (rows == 0) return out.zero_();
  const int64_t blocks = (d + 255) / 256;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>((rows + 31) / 32, 4 * lm::sm_count() / blocks));
  const int64_t ldx = rows > 1 ? x.stride(0) : d;
  const bool vec = d % 8 == 0 && ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  auto part = torch::empty({parts, d}, x.options().dtype(torch::kFloat32));
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  for_type(x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    const auto kernel = vec ? column_sums_kernel<T, true> : column_sums_kernel<T, false>;
    kernel<<<dim3((unsigned)blocks, (unsigned)parts), 256, 0, st>>>(reinterpret_cast<const T*>(x.data_ptr()), ldx, rows,
                                                                   (int)d, part.data_ptr<float>());
  });
  for_type(out_type, [&](auto t) {
    using W = decltype(t);
    lm::sum_parts_kernel<W><<<(unsigned)((d + lm::kSumColumns - 1) / lm::kSumColumns), 64 * lm::kSumColumns, 0, st>>>(
        part.data_ptr<float>(), (int)parts, (int)d, reinterpret_cast<W*>(out.data_ptr()));
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "column_sums launch failed");
  lm::count_launches(2);
  return out;
}

std::vector<torch::Tensor> quantize_blocks(const torch::Tensor& w, bool transposed) {
  const c10::cuda::CUDAGuard guard(w.device());
  const int64_t n = w.size(0), k = w.size(1), bn = (n + 127) / 128, bk = (k + 127) / 128;
  LM_CHECK_VALUE(n < (1ll << 22), "quantize_blocks: too many rows");   // grid.y holds n / 128
  auto q = empty_q(n, k, w);
  auto scale = torch::empty({bn, bk}, w.options().dtype(torch::kFloat32));
  std::vector<torch::Tensor> out = {q, scale};
  if (transposed) {
    out.push_back(empty_q(k, n, w));
    out.push_back(torch::empty({bk, bn}, scale.options()));
  }
  if (n == 0 || k == 0) return out;
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  for_type(w.scalar_type(), [&](auto t) {
    using T = decltype(t);
    quant_blocks_kernel<T><<<dim3((unsigned)bk, (unsigned)bn), 256, 0, st>>>(
        reinterpret_cast<const T*>(w.data_ptr()), n > 1 ? w.stride(0) : k, reinterpret_cast<uint8_t*>(q.data_ptr()),
        q.stride(0), transposed ? reinterpret_cast<uint8_t*>(out[2].data_ptr()) : nullptr,
        transposed ? out[2].stride(0) : 0, scale.data_ptr<float>(), transposed ? out[3].data_ptr<float>() : nullptr,
        (int)n, (int)k);
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "quantize_blocks launch failed");
  lm::count_launches(1);
  return out;
}

}  // namespace fp8

void register_fp8_quant_ops(py::module& m) {
  m.def("quantize_rows",
        [](torch::Tensor x) {
          check_input(x, 1, "quantize_rows");
          const auto r = fp8::quantize_rows(fp8::as_matrix(x.detach()));
          return py::make_tuple(lm::from_rows(r.first, x), lm::from_rows(r.second, x));
        },
        "e4m3 rows with a scale for each 128 columns: (q, scale)", py::arg("x"));
  m.def("quantize_blocks",
        [](torch::Tensor w, bool transposed) {
          check_input(w, 2, "quantize_blocks");
          LM_CHECK_VALUE(w.dim() == 2, "quantize_blocks takes a matrix");
          return py::tuple(py::cast(fp8::quantize_blocks(fp8::as_matrix(w.detach()), transposed)));
        },
        "e4m3 matrix with a scale for each 128 x 128 block: (q, scale), with its transpose (q, scale, q^T, scale^T)",
        py::arg("w"), py::arg("transposed"));
}
