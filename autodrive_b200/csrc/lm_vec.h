// Shared device helpers of the language-model operators: conversion between
// fp32 and the 16-bit types, a row slice of eight elements per thread, warp
// reductions, and the exactly rounded e4m3 quotient of the 8-bit quantisers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace lm {

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// Eight consecutive elements, 16-byte aligned (32 bytes for fp32, as two
// 16-byte accesses).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f<T>(e[i]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 u;
    uint32_t* w = &u.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // two at a time
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// A row is cut into chunks of 256 columns, one warp each; a lane owns eight
// columns of a chunk. With VEC (widths and strides that are multiples of
// eight, 16-byte aligned bases) they are consecutive and move as 16-byte
// accesses; otherwise they lie 32 apart, so that the lanes of every 2- or
// 4-byte access are neighbours whatever the row's alignment.
template <bool VEC>
__device__ __forceinline__ int slice_col(int chunk, int lane, int e) {
  return chunk * 256 + (VEC ? lane * 8 + e : e * 32 + lane);
}

// A slice as it lies in memory, to be loaded a row ahead.
template <typename T, bool VEC>
struct RawSlice {
  alignas(16) T e[8];
  __device__ __forceinline__ void load(const T* row, int chunk, int lane, int d) {
    if constexpr (VEC) {
      constexpr int kVectors = sizeof(T) * 8 / 16;
      const int c = slice_col<true>(chunk, lane, 0);
      uint4* u = reinterpret_cast<uint4*>(e);
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
        u[j] = c < d ? reinterpret_cast<const uint4*>(row + c)[j] : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = slice_col<false>(chunk, lane, i);
        e[i] = from_f<T>(0.f);
        if (c < d) e[i] = row[c];
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f<T>(e[i]);
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void store_slice(T* row, int chunk, int lane, int d, const float (&v)[8]) {
  if constexpr (VEC) {
    const int c = slice_col<true>(chunk, lane, 0);
    if (c < d) store8(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = slice_col<false>(chunk, lane, e);
      if (c < d) row[c] = from_f<T>(v[e]);
    }
  }
}

__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// out[c] = sum of the rows of part [parts][d]: eight columns per CTA (a sector
// of each row), 64 threads down each, in an order that depends on the sizes
// alone.
constexpr int kSumColumns = 8;
template <typename W>
__global__ void __launch_bounds__(64 * kSumColumns) sum_parts_kernel(const float* part, int parts, int d, W* out) {
  __shared__ float red[64][kSumColumns + 1];
  const int tx = threadIdx.x % kSumColumns, ty = threadIdx.x / kSumColumns, c = blockIdx.x * kSumColumns + tx;
  float s = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int p = ty; p < parts; p += 64) s += part[(int64_t)p * d + c];
  }
  red[ty][tx] = s;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp >= kSumColumns) return;
  s = warp_sum(red[lane][warp] + red[lane + 32][warp]);
  const int col = blockIdx.x * kSumColumns + warp;
  if (lane == 0 && col < d) out[col] = from_f<W>(s);
}

// ---- 8-bit quantisation ---------------------------------------------------------
// A group's scale is max(amax, 448 * 2^-126) / 448, rounded to fp32 once: the
// largest value becomes 448, the largest e4m3 number, and a group of zeros
// (or of values near the end of fp32's range) gets the smallest normal scale.
// amax is carried as the bits of |x|, which order like the values and put NaN
// above infinity: a NaN makes the group's scale NaN, an infinity makes it
// infinite, and in both cases the group's values NaN.
constexpr uint32_t kMinAmaxBits = 0x04e00000u;   // 448 * 2^-126

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float mul_nf(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fma_nf(float a, float b, float c) {
  float r;
  asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// amax / 448, correctly rounded by one correction of the product with the
// rounded reciprocal (Markstein, "Computation of elementary functions on the IBM
// RISC System/6000 processor", 1990): the remainder is exact in an fma.
__device__ __forceinline__ float group_scale(uint32_t amax_bits) {
  constexpr float r = 1.f / 448.f;
  const float a = __uint_as_float(max(amax_bits, kMinAmaxBits));
  const float q = mul_nf(a, r);
  const float s = fma_nf(fma_nf(-q, 448.f, a), r, q);
  return amax_bits < 0x7f800000u ? s : a;
}

// x / scale rounded to e4m3 once. A quotient rounded to fp32 first can land
// on the middle between two e4m3 numbers, or on its wrong side, and then be
// rounded to the wrong one. x times the reciprocal is within three units in
// the last place, so only values within four of a middle (the last 20 bits
// tell, among e4m3's normal numbers) and those below them take the exact way:
// there the quotient is rounded to odd (truncated, with the last bit set when
// the remainder is not zero; Boldo & Melquiond, "When double rounding is odd",
// 2005), from which the conversion rounds as if from the exact quotient. The
// remainder of the quotient's correction step is exact in an fma; `lift` (a
// power of two) keeps it out of the subnormal range for tiny scales. Written
// without the flush-to-zero that the compiler's fast-math mode adds, so
// subnormal inputs keep their value.
struct Divisor {
  float scale, inv, lift, direct;   // scale and 1 / scale, lifted; 1 / scale
};
__device__ __forceinline__ Divisor divisor(float scale) {
  Divisor d;
  d.lift = scale < 0x1p-60f ? 0x1p64f : 1.f;
  d.scale = scale * d.lift;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d.inv) : "f"(d.scale));   // within one unit in the last place
  d.direct = scale < __uint_as_float(0x7f800000u) ? d.inv * d.lift : __uint_as_float(0x7fffffffu);   // inf, NaN: NaN
  return d;
}
__device__ __forceinline__ float quotient_to_odd(float x, const Divisor& d) {
  float y;
  asm volatile("mul.rn.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(d.lift));   // volatile: a branch, not computed for all
  const float q0 = mul_nf(y, d.inv);
  const float q = fma_nf(fma_nf(-q0, d.scale, y), d.inv, q0);
  const float rem = fma_nf(-q, d.scale, y);                  // exact; its sign says on which side q lies
  uint32_t b = __float_as_uint(q);
  const uint32_t r = __float_as_uint(rem);
  if ((r << 1) != 0u) {                                      // inexact
    if ((int32_t)(b ^ r) < 0) b -= 1u;                       // |q| above the quotient: truncate
    b |= 1u;
  }
  return __uint_as_float(b);
}
// A number that converts to e4m3 as the exact quotient would.
__device__ __forceinline__ float e4m3_quotient(float x, const Divisor& d) {
  const float q = mul_nf(x, d.direct);
  const uint32_t u = __float_as_uint(q);
  const bool middle = (u & 0xfffffu) - 0x7fffcu <= 8u;
  const bool below = (u << 1) - 1u < (0x3c800000u << 1) - 1u;   // 0 < |q| < 2^-6
  return middle || below ? quotient_to_odd(x, d) : q;
}
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], const Divisor& d) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = e4m3x2(e4m3_quotient(v[2 * i], d), e4m3_quotient(v[2 * i + 1], d));
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

}  // namespace lm
