// Matrix product of e4m3 operands with a scale for each block of 128:
//
//   C[m,n] = sum_g a_scale[m,g] b_scale[n/128,g] sum_{k in group g} A[m,k] B[n,k]  (+ bias[n])
//
// A [M,K] has one fp32 scale for each row and 128 columns, B [N,K] one for
// each 128 x 128 block. The tensor cores (tcgen05 kind::f8f6f4) multiply one
// group of 128 columns into TMEM; the scales differ from group to group, so
// each group's tile is read back and added, scaled, to fp32 sums in registers
// while the next group's products run into another TMEM buffer.
//
// Persistent kernel, one CTA per SM, 320 threads:
//   warp 0     TMA producer: the 128-byte wide A and B tiles of each group into
//              a shared-memory ring that runs on across output tiles;
//   warp 1     allocates TMEM; one lane issues the four K = 32 products of a
//              group into the next buffer, then commits the stage back to the
//              producer and the buffer to the epilogue;
//   warps 2-9  two per TMEM lane quadrant: thread = one row, half the columns.
// Waits are bounded and reported as in the bf16 GEMM (tc_gemm.cu), with the
// same status bits and the same drains before the CTA gives up its TMEM.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "fp8.h"
#include "lm_host.h"
#include "lm_vec.h"
#include "smem_opt_in.h"
#include "tc_sm100.h"
#include "tma_map.h"

namespace py = pybind11;

namespace {

constexpr int kBM = 128, kGroup = 128;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr uint64_t kDrainNs = 200000000ull;

struct Args {
  int M, N, groups;
  const float* a_scale;   // [M][groups]
  const float* b_scale;   // [ceil(N / 128)][groups]
  const float* bias;      // [N] or null
  void* c;
  int64_t ldc;
  int out_kind;           // 0 fp32, 1 bf16, 2 fp16
  int* status;
  uint64_t wait_ns;
};

template <int BN> struct Config {
  static constexpr int stages = BN == 128 ? 6 : 4;
  static constexpr uint32_t a_bytes = kBM * kGroup, stage_bytes = a_bytes + BN * kGroup;
  static constexpr uint32_t smem_bytes = stages * stage_bytes + 1024 + 256;
  static constexpr int buffers = 512 / BN;   // TMEM has 512 columns
};

template <typename T>
__device__ __forceinline__ void store32(T* dst, const float (&v)[32], int n, bool vec) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = v[8 * j + i];
      lm::store8(dst + 8 * j, u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) dst[i] = lm::from_f<T>(v[i]);
  }
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const Args g) {
  using C = Config<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* misc = smem + C::stages * C::stage_bytes;
  const uint32_t full0 = tc::smem_u32(misc);                    // stage loaded
  const uint32_t empty0 = full0 + 8 * C::stages;                // stage consumed
  const uint32_t tfull0 = empty0 + 8 * C::stages;               // TMEM buffer complete
  const uint32_t tempty0 = tfull0 + 8 * C::buffers;             // TMEM buffer read out
  const uint32_t drain = tempty0 + 8 * C::buffers;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(misc + 8 * (2 * C::stages + 2 * C::buffers + 1));
  int* s_fail = reinterpret_cast<int*>(s_tmem + 1);
  volatile int* fail = s_fail;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_n = (g.N + BN - 1) / BN, tiles_m = (g.M + kBM - 1) / kBM;
  const int total = tiles_n * tiles_m, G = g.groups;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::stages; ++s) {
      tc::mbar_init(full0 + 8 * s, 1);
      tc::mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < C::buffers; ++b) {
      tc::mbar_init(tfull0 + 8 * b, 1);
      tc::mbar_init(tempty0 + 8 * b, 32 * kEpiWarps);
    }
    tc::mbar_init(drain, 1);
    tc::mbar_init_fence();
    *s_fail = 0;
  }
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_u32(s_tmem), 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp == 0 && lane == 0) {
    uint32_t it = 0;
    for (int w = blockIdx.x; w < total && !*fail; w += gridDim.x) {
      const int n0 = (w % tiles_n) * BN, m0 = (w / tiles_n) * kBM;
      for (int kb = 0; kb < G; ++kb, ++it) {
        const uint32_t s = it % C::stages;
        if (it >= C::stages && !tc::mbar_wait(empty0 + 8 * s, ((it / C::stages) - 1) & 1, g.wait_ns)) {
          atomicOr(g.status, 1);
          atomicExch(s_fail, 1);
        }
        if (*fail) break;
        const uint32_t sa = tc::smem_u32(smem + s * C::stage_bytes), full = full0 + 8 * s;
        tc::mbar_arrive_expect_tx(full, C::stage_bytes);
        tc::tma_load_2d(sa, &ta, kb * kGroup, m0, full);
        tc::tma_load_2d(sa + C::a_bytes, &tb, kb * kGroup, n0, full);
      }
    }
    if (*fail) {   // every stage's latest load may still be in flight
      for (uint32_t i = it > (uint32_t)C::stages ? it - C::stages : 0u; i < it; ++i)
        if (!tc::mbar_wait(full0 + 8 * (i % C::stages), (i / C::stages) & 1, kDrainNs)) atomicOr(g.status, 16);
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t id = tc::idesc_e4m3(kBM, BN);
    uint32_t it = 0;
    for (int w = blockIdx.x; w < total && !*fail; w += gridDim.x) {
      for (int kb = 0; kb < G; ++kb, ++it) {
        const uint32_t s = it % C::stages, b = it % C::buffers;
        if (it >= C::buffers && !tc::mbar_wait(tempty0 + 8 * b, ((it / C::buffers) - 1) & 1, g.wait_ns)) {
          atomicOr(g.status, 8);
          atomicExch(s_fail, 1);
        } else if (!tc::mbar_wait(full0 + 8 * s, (it / C::stages) & 1, g.wait_ns)) {
          atomicOr(g.status, 2);
          atomicExch(s_fail, 1);
        }
        if (*fail) break;
        tc::tc_fence_after();
        const uint32_t sa = tc::smem_u32(smem + s * C::stage_bytes), sb = sa + C::a_bytes;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          tc::mma_e4m3(tmem + b * BN, tc::sw128_desc(sa + 32 * ks, 16, 1024), tc::sw128_desc(sb + 32 * ks, 16, 1024),
                       id, ks > 0);
        tc::mma_commit(empty0 + 8 * s);
        tc::mma_commit(tfull0 + 8 * b);
      }
    }
    if (*fail) {   // products issued so far may still read shared memory and write TMEM
      tc::mma_commit(drain);
      if (!tc::mbar_wait(drain, 0, kDrainNs)) atomicOr(g.status, 32);
    }
  }

  if (warp >= 2) {
    constexpr int kChunks = BN / 64;   // 32-column chunks per warp
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint32_t it = 0;
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
      const int n0 = (w % tiles_n) * BN + half * (BN / 2), row = (w / tiles_n) * kBM + 32 * q + lane;
      float acc[kChunks][32];
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[c][i] = 0.f;
      // this half of the tile lies inside one block of 128 rows of B
      const float* as = g.a_scale + (int64_t)min(row, g.M - 1) * G;
      const float* bs = g.b_scale + (int64_t)min(n0 / kGroup, (g.N - 1) / kGroup) * G;
      for (int kb = 0; kb < G; ++kb, ++it) {
        const uint32_t b = it % C::buffers;
        const float sc = as[kb] * bs[kb];
        if (!tc::mbar_wait(tfull0 + 8 * b, (it / C::buffers) & 1, g.wait_ns)) {
          atomicOr(g.status, 4);
          atomicExch(s_fail, 1);
        }
        if (__any_sync(0xffffffffu, *fail)) break;   // the loads below are whole-warp
        tc::tc_fence_after();
        const uint32_t base = tmem + b * BN + half * (BN / 2) + ((uint32_t)(32 * q) << 16);
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          float v[2][32];
          tc::tmem_ld32_issue(base + 32 * c, v[0]);
          tc::tmem_ld32_issue(base + 32 * (c + 1), v[1]);
          tc::tmem_ld_wait();
          tc::tmem_regs_ready(v[0]);
          tc::tmem_regs_ready(v[1]);
          if (c + 2 >= kChunks) {
            tc::tc_fence_before();
            tc::mbar_arrive(tempty0 + 8 * b);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c + j][i] = fmaf(v[j][i], sc, acc[c + j][i]);
        }
      }
      if (__any_sync(0xffffffffu, *fail)) break;
      if (row < g.M) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int col = n0 + 32 * c, n = g.N - col;
          if (n <= 0) continue;
          if (g.bias) {
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c][i] += i < n ? g.bias[col + i] : 0.f;
          }
          const int64_t off = (int64_t)row * g.ldc + col;
          const bool vec = n >= 32 && g.ldc % 8 == 0;   // the output's base is 16-byte aligned (host)
          if (g.out_kind == 0) store32(reinterpret_cast<float*>(g.c) + off, acc[c], n, vec);
          else if (g.out_kind == 1) store32(reinterpret_cast<__nv_bfloat16*>(g.c) + off, acc[c], n, vec);
          else store32(reinterpret_cast<__half*>(g.c) + off, acc[c], n, vec);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

template <int BN>
void launch(const CUtensorMap& ta, const CUtensorMap& tb, const Args& g, cudaStream_t st) {
  static size_t configured[dynsmem::kMaxDevices] = {};
  TORCH_CHECK(dynsmem::opt_in(fp8_gemm_kernel<BN>, Config<BN>::smem_bytes, configured) == cudaSuccess,
              "fp8_matmul shared-memory attribute");
  const int64_t total = (int64_t)((g.N + BN - 1) / BN) * ((g.M + kBM - 1) / kBM);
  TORCH_CHECK(total < (1ll << 31), "fp8_matmul: too many output tiles");
  fp8_gemm_kernel<BN><<<(int)std::min<int64_t>(total, lm::sm_count()), kThreads, Config<BN>::smem_bytes, st>>>(ta, tb, g);
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "fp8_matmul launch failed");
}

// `q` as the TMA unit reads it: rows that start 16 bytes apart on a 16-byte
// aligned base (a copy only where they do not).
torch::Tensor operand(const torch::Tensor& q) {
  const int64_t rows = q.size(0), k = q.size(1);
  const bool ok = (k <= 1 || q.stride(1) == 1) && (rows <= 1 || (q.stride(0) % 16 == 0 && q.stride(0) >= k)) &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
  if (ok || q.numel() == 0) return q;
  auto buf = torch::empty({rows, (k + 15) / 16 * 16}, q.options()).narrow(1, 0, k);
  buf.view(torch::kUInt8).copy_(q.view(torch::kUInt8));
  return buf;
}

}  // namespace

namespace fp8 {

torch::Tensor matmul(const torch::Tensor& a, const torch::Tensor& a_scale, const torch::Tensor& b,
                     const torch::Tensor& b_scale, const torch::Tensor& bias, torch::ScalarType out_dtype,
                     const torch::Tensor& status, int64_t wait_ns) {
  const c10::cuda::CUDAGuard guard(a.device());
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
  auto c = torch::empty({M, N}, a.options().dtype(out_dtype));
  if (M == 0 || N == 0) return c;
  if (K == 0) {
    c.zero_();
    if (bias.defined()) c.add_(bias);
    return c;
  }
  LM_CHECK_VALUE(M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30), "fp8_matmul: too large");
  Args g{};
  g.M = (int)M;
  g.N = (int)N;
  g.groups = (int)((K + kGroup - 1) / kGroup);
  g.a_scale = a_scale.data_ptr<float>();
  g.b_scale = b_scale.data_ptr<float>();
  g.bias = bias.defined() ? bias.data_ptr<float>() : nullptr;
  g.c = c.data_ptr();
  g.ldc = N;
  g.out_kind = out_dtype == torch::kFloat32 ? 0 : (out_dtype == torch::kBFloat16 ? 1 : 2);
  g.status = status.data_ptr<int>();
  g.wait_ns = (uint64_t)wait_ns;
  constexpr int BN = 128;
  const int64_t one_row = (K + 15) / 16 * 16;   // a single row's stride says nothing
  const CUtensorMap ta = tma::u8_sw128(a.data_ptr(), M, K, M > 1 ? a.stride(0) : one_row, kBM);
  const CUtensorMap tb = tma::u8_sw128(b.data_ptr(), N, K, N > 1 ? b.stride(0) : one_row, BN);
  launch<BN>(ta, tb, g, c10::cuda::getCurrentCUDAStream().stream());
  lm::count_launches(1);
  return c;
}

}  // namespace fp8

namespace {

torch::Tensor fp8_matmul(torch::Tensor a, torch::Tensor a_scale, torch::Tensor b, torch::Tensor b_scale,
                         c10::optional<torch::Tensor> bias, py::object dtype, torch::Tensor status, int64_t wait_ns) {
  const auto out_dtype = torch::python::detail::py_object_to_dtype(dtype);
  LM_CHECK_VALUE(a.is_cuda() && a.scalar_type() == torch::kFloat8_e4m3fn && a.dim() >= 1 &&
                        b.scalar_type() == torch::kFloat8_e4m3fn && b.dim() == 2,
                    "fp8_matmul takes e4m3 rows [..., K] and an e4m3 matrix [N, K]");
  const int64_t K = a.size(-1), N = b.size(0), groups = (K + kGroup - 1) / kGroup;
  LM_CHECK_VALUE(b.size(1) == K, "fp8_matmul: a has ", K, " columns and b ", b.size(1));
  auto want = a.sizes().vec();
  want.back() = groups;
  LM_CHECK_VALUE(a_scale.sizes() == c10::IntArrayRef(want) && b_scale.dim() == 2 &&
                        b_scale.size(0) == (N + kGroup - 1) / kGroup && b_scale.size(1) == groups,
                    "fp8_matmul needs scales ", c10::IntArrayRef(want), " and [", (N + kGroup - 1) / kGroup, ", ", groups,
                    "], not ", a_scale.sizes(), " and ", b_scale.sizes());
  LM_CHECK_VALUE(a_scale.scalar_type() == torch::kFloat32 && b_scale.scalar_type() == torch::kFloat32,
                    "fp8_matmul needs fp32 scales");
  LM_CHECK_VALUE(!bias || (bias->dim() == 1 && bias->size(0) == N && fp8::known_type(bias->scalar_type())),
                    "fp8_matmul needs a bias [", N, "]");
  LM_CHECK_VALUE(fp8::known_type(out_dtype), "fp8_matmul gives fp32, bf16 or fp16");
  for (const auto* t : {&a_scale, &b, &b_scale, &status})
    LM_CHECK_VALUE(t->device() == a.device(), "fp8_matmul needs all of its tensors on one device");
  LM_CHECK_VALUE(!bias || bias->device() == a.device(), "fp8_matmul needs all of its tensors on one device");
  TORCH_CHECK(status.scalar_type() == torch::kInt32, "fp8_matmul: status must be int32");
  LM_CHECK_VALUE(wait_ns >= 0, "wait_ns must not be negative");
  LM_CHECK_VALUE(!(at::GradMode::is_enabled() &&
                      (a_scale.requires_grad() || b_scale.requires_grad() || (bias && bias->requires_grad()))),
                    "fp8_matmul has no gradient: use fp8_linear, or call it under torch.no_grad()");
  const int64_t rows = c10::multiply_integers(a.sizes().slice(0, a.dim() - 1));
  const auto a2 = a.dim() == 2 ? a : a.reshape({rows, K});
  const auto s2 = a_scale.dim() == 2 ? a_scale : a_scale.reshape({rows, groups});
  torch::Tensor bf;
  if (bias) bf = (bias->scalar_type() == torch::kFloat32 ? *bias : bias->to(torch::kFloat32)).contiguous();
  const auto y = fp8::matmul(operand(a2), s2.contiguous(), operand(b), b_scale.contiguous(), bf, out_dtype, status, wait_ns);
  return a.dim() == 2 ? y : lm::from_rows(y, a);
}

}  // namespace

void register_fp8_gemm_ops(py::module& m) {
  m.def("fp8_matmul", &fp8_matmul, "e4m3 x e4m3 product with a scale for each block of 128 (+ bias): fp32, bf16 or fp16",
        py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("bias"), py::arg("out_dtype"),
        py::arg("status"), py::arg("wait_ns") = fp8::kWaitNs);
}
