// AdamW over a list of tensors in one launch, the moments in fp32 or in 8 bits.
//
//   c = min(1, max_norm / (|g| + 1e-6))            where gradients are clipped, |g| over all tensors
//   m = b1 m + (1 - b1) c g,   v = b2 v + (1 - b2) (c g)^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Moments in 8 bits: m and r = sqrt(v) are e4m3 numbers times a scale for each
// 256 elements of a tensor (largest magnitude / 448). The root is held, not v:
// e4m3 spans 2^18, so v may span 2^36 in a block. A step moves v by a
// thousandth and e4m3's numbers lie a sixteenth apart, so rounding to the
// nearest one would never let a moment move: 16 random bits are added below
// the last bit that stays and the rest is cut off, which moves a moment by the
// right amount on average. The bits are mixed from (seed, step, element), so a
// step gives the same numbers again. A root that is not zero never becomes
// zero, as it is divided by; m and r of the step itself enter p unrounded.
// A block with a NaN or an infinity among its new moments becomes NaN.
//
// Layout: 256 elements (a block) are a warp's work, 8 to a lane; warps walk the
// blocks of all tensors with the stride of the grid, from the last to the first
// (the gradients' end is what the norm's pass left in L2). The tensors'
// addresses are the kernel's parameters, so no table is copied to the device.
#include <cuda_runtime.h>

#include "adamw.h"
#include "lm_vec.h"

namespace adamw {
namespace {

constexpr int kThreads = kWarps * 32;

// Kernel parameters: up to 4 KB travel with a launch at no cost; longer lists use the larger table.
template <int CAP>
struct Table {
  Header h;
  Entry e[CAP];
};
constexpr int kSmall = 58, kLarge = kMaxTensors;
static_assert(sizeof(Table<kSmall>) <= 4096 && sizeof(Table<kLarge>) <= 32764, "kernel parameter space");

__device__ __forceinline__ void load_f8(const float* p, float (&v)[8]) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void store_f8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// A lane's elements of a block: eight consecutive ones, or (`vec` unset, or at a tensor's end) 32 apart.
template <typename T>
__device__ __forceinline__ void load_lane(const T* p, int lane, int n, bool whole, float (&v)[8]) {
  if (whole) {
    if constexpr (sizeof(T) == 4) load_f8(p + lane * 8, v);
    else lm::load8(p + lane * 8, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i * 32 + lane < n ? lm::to_f<T>(p[i * 32 + lane]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_lane(T* p, int lane, int n, bool whole, const float (&v)[8]) {
  if (whole) {
    if constexpr (sizeof(T) == 4) store_f8(p + lane * 8, v);
    else lm::store8(p + lane * 8, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < n) p[i * 32 + lane] = lm::from_f<T>(v[i]);
  }
}
__device__ __forceinline__ void load_any(const void* p, int type, int64_t at, int lane, int n, bool whole, float (&v)[8]) {
  if (type == 0) load_lane(static_cast<const float*>(p) + at, lane, n, whole, v);
  else if (type == 1) load_lane(static_cast<const __nv_bfloat16*>(p) + at, lane, n, whole, v);
  else load_lane(static_cast<const __half*>(p) + at, lane, n, whole, v);
}
__device__ __forceinline__ void store_any(void* p, int type, int64_t at, int lane, int n, bool whole, const float (&v)[8]) {
  if (type == 0) store_lane(static_cast<float*>(p) + at, lane, n, whole, v);
  else if (type == 1) store_lane(static_cast<__nv_bfloat16*>(p) + at, lane, n, whole, v);
  else store_lane(static_cast<__half*>(p) + at, lane, n, whole, v);
}

// Two e4m3 numbers as fp32.
__device__ __forceinline__ float2 from_e4m3x2(uint16_t q) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(q));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ void load_codes(const uint8_t* p, int lane, int n, bool whole, float (&v)[8]) {
  uint2 u = make_uint2(0, 0);
  if (whole) {
    u = *reinterpret_cast<const uint2*>(p + lane * 8);
  } else {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < n) w[i / 4] |= (uint32_t)p[i * 32 + lane] << (8 * (i % 4));
    u = make_uint2(w[0], w[1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = from_e4m3x2((uint16_t)((i < 2 ? u.x : u.y) >> (16 * (i % 2))));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// `v`: numbers that e4m3 holds, or NaN.
__device__ __forceinline__ void store_codes(uint8_t* p, int lane, int n, bool whole, const float (&v)[8]) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = lm::e4m3x2(v[2 * i], v[2 * i + 1]);
  const uint2 u = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
  if (whole) {
    *reinterpret_cast<uint2*>(p + lane * 8) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < n) p[i * 32 + lane] = (uint8_t)((i < 4 ? u.x : u.y) >> (8 * (i % 4)));
  }
}

// The magnitude t, at most 448 and a rounding, as an e4m3 number at or below
// it, or the next one with the probability of its distance. Below 2^-6 the
// numbers lie 2^-9 apart: 2^-6 is added first, where the spacing is the same.
__device__ __forceinline__ float dithered(float t, uint32_t bits16) {
  const float off = t < 0x1p-6f ? 0x1p-6f : 0.f;
  const uint32_t u = (__float_as_uint(t + off) + (bits16 << 4)) & 0xfff00000u;
  return fminf(__uint_as_float(u) - off, 448.f);
}

__device__ __forceinline__ uint32_t warp_max(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

// Scale of a block with the largest magnitude `amax` (as bits) and what a magnitude is multiplied with.
__device__ __forceinline__ float2 scale_of(uint32_t amax) {
  const float s = lm::group_scale(amax);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  return make_float2(s, amax < 0x7f800000u ? inv : __uint_as_float(0x7fffffffu));
}

// Walks the blocks of the launch that belong to this warp, last to first:
// enter(tensor) before the first block of each tensor, f(tensor, block) for each.
template <typename TABLE, typename E, typename F>
__device__ __forceinline__ void for_blocks(const TABLE& t, E&& enter, F&& f) {
  const uint32_t warp = (threadIdx.x >> 5) * gridDim.x + blockIdx.x, warps = gridDim.x * kWarps;
  if (warp >= t.h.blocks) return;
  uint32_t b = t.h.blocks - 1 - warp;
  int lo = 0, hi = t.h.tensors - 1;   // the last tensor whose first block is at or before b
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= b) lo = mid;
    else hi = mid - 1;
  }
  enter(t.e[lo]);
  for (;;) {
    f(t.e[lo], b);
    if (b < warps) return;
    b -= warps;
    if (t.e[lo].first > b) {
      do --lo;
      while (t.e[lo].first > b);
      enter(t.e[lo]);
    }
  }
}

// parts[CTA] = sum of the gradients' squares, in fp64.
template <int CAP>
__global__ void __launch_bounds__(kThreads) square_sums_kernel(const __grid_constant__ Table<CAP> t, double* parts) {
  const int lane = threadIdx.x & 31;
  double s = 0.;
  for_blocks(t, [](const Entry&) {}, [&](const Entry& e, uint32_t b) {
    const int64_t at = (int64_t)(b - e.first) * kBlock;
    const int n = (int)min((int64_t)kBlock, (int64_t)e.n - at);
    float g[8];
    load_any(e.g, e.g_type, at, lane, n, e.vec && n == kBlock, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += (double)g[i] * (double)g[i];
  });
  __shared__ double red[kWarps];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) s += red[w];
    parts[blockIdx.x] = s;
  }
}

template <bool BITS8, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<CAP> t) {
  const int lane = threadIdx.x & 31;
  __shared__ double red[kWarps];
  __shared__ float clip_at;
  const Header& h = t.h;
  double s = 0.;
  for (int i = threadIdx.x; i < h.nparts; i += kThreads) s += h.parts[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) s += red[w];
    float c = 1.f;
    if (h.parts) {
      const double norm = sqrt(s), f = h.max_norm / (norm + 1e-6);
      c = f < 1. || f != f ? (float)f : 1.f;
      if (blockIdx.x == 0 && h.norm_out) *h.norm_out = (float)norm;
    }
    clip_at = c;
  }
  __syncthreads();
  const float clip = clip_at;
  float rate = 0.f, root_scale = 0.f;
  uint32_t key = 0;
  const auto enter = [&](const Entry& e) {
    const int64_t step = h.step_at ? *h.step_at : (int64_t)e.step;
    rate = h.lr / -expm1f((float)step * h.log_b1);
    root_scale = rsqrtf(-expm1f((float)step * h.log_b2));
    key = mix(h.seed ^ (uint32_t)step);
  };
  for_blocks(t, enter, [&](const Entry& e, uint32_t b) {
    const int64_t at = (int64_t)(b - e.first) * kBlock;
    const int n = (int)min((int64_t)kBlock, (int64_t)e.n - at);
    const bool whole = e.vec && n == kBlock;
    float p[8], g[8], m[8], v[8];
    load_any(e.p, e.p_type, at, lane, n, whole, p);
    load_any(e.g, e.g_type, at, lane, n, whole, g);
    if constexpr (BITS8) {
      load_codes(static_cast<const uint8_t*>(e.m) + at, lane, n, whole, m);
      load_codes(static_cast<const uint8_t*>(e.v) + at, lane, n, whole, v);
      const float ms = e.m_scale[b - e.first], vs = e.v_scale[b - e.first];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m[i] *= ms;
        v[i] *= vs;
        v[i] *= v[i];
      }
    } else {
      load_lane(static_cast<const float*>(e.m) + at, lane, n, whole, m);
      load_lane(static_cast<const float*>(e.v) + at, lane, n, whole, v);
    }
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float gi = g[i] * clip;
      m[i] = h.b1 * m[i] + h.c1 * gi;
      v[i] = h.b2 * v[i] + h.c2 * gi * gi;
      r[i] = sqrtf(v[i]);
      p[i] = p[i] * h.decay - rate * (m[i] / (r[i] * root_scale + h.eps));
    }
    store_any(e.p, e.p_type, at, lane, n, whole, p);
    if constexpr (BITS8) {
      uint32_t am = 0, ar = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        am = max(am, lm::abs_bits(m[i]));
        ar = max(ar, lm::abs_bits(r[i]));
      }
      const float2 sm = scale_of(warp_max(am)), sr = scale_of(warp_max(ar));
      const uint32_t number = (h.block0 + b) * kBlock + key;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t bits = mix(number + (whole ? lane * 8 + i : i * 32 + lane));
        const float q = dithered(fabsf(m[i]) * sm.y, bits & 0xffffu);
        m[i] = sm.y == sm.y ? copysignf(q, m[i]) : sm.y;
        const float z = dithered(r[i] * sr.y, bits >> 16);
        r[i] = sr.y == sr.y ? fmaxf(z, r[i] > 0.f ? 0x1p-9f : 0.f) : sr.y;
      }
      store_codes(static_cast<uint8_t*>(e.m) + at, lane, n, whole, m);
      store_codes(static_cast<uint8_t*>(e.v) + at, lane, n, whole, r);
      if (lane == 0) {
        e.m_scale[b - e.first] = sm.x;
        e.v_scale[b - e.first] = sr.x;
      }
    } else {
      store_lane(static_cast<float*>(e.m) + at, lane, n, whole, m);
      store_lane(static_cast<float*>(e.v) + at, lane, n, whole, v);
    }
  });
}

template <typename F>
cudaError_t with_table(const Header& h, const Entry* entries, F&& f) {
  const auto fill = [&](auto& table) {
    table.h = h;
    for (int i = 0; i < h.tensors; ++i) table.e[i] = entries[i];
    f(table);
    return cudaGetLastError();
  };
  if (h.tensors <= kSmall) {
    Table<kSmall> table;
    return fill(table);
  }
  Table<kLarge> table;
  return fill(table);
}

}  // namespace

cudaError_t launch_square_sums(const Header& h, const Entry* entries, double* parts, int grid, cudaStream_t st) {
  return with_table(h, entries, [&](const auto& table) { square_sums_kernel<<<grid, kThreads, 0, st>>>(table, parts); });
}

cudaError_t launch_step(const Header& h, const Entry* entries, bool bits8, int grid, cudaStream_t st) {
  return with_table(h, entries, [&](const auto& table) {
    if (bits8) adamw_kernel<true><<<grid, kThreads, 0, st>>>(table);
    else adamw_kernel<false><<<grid, kThreads, 0, st>>>(table);
  });
}

}  // namespace adamw
