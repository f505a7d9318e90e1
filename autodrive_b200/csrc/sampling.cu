// Sampling from rows of logits, with temperature, top-k, top-p and min-p, by
// given uniform numbers.
//
//   w_i = exp((l_i - max) / T)          over the valid entries
//   order: by l descending, equal ones by their index
//   stay: w_i >= min_p; of these the first k of the order; of these the
//         shortest prefix of the order whose sum is at least top_p times theirs
//   token: the first entry that stays, by index, at which the running sum of
//          the staying w exceeds u times their sum
//
// Which entry that is hangs on a sum's last bits: of 131072 entries one in
// fifty rows would come out otherwise with 32-bit sums. Weights and sums are
// fp64 (the device has half as many fp64 units as fp32 ones), added in an order
// that the sizes alone give. Entries further than 44 T below the largest (they
// hold less than 10^-13 of any row's sum) count as zero.
#include <cuda_runtime.h>

#include "lm_vec.h"
#include "sampling.h"

namespace sampling {
namespace {

constexpr float kRange = 44.f;   // in units of T below the largest logit

__device__ __forceinline__ uint32_t key_of(float l) {   // orders like l; both zeros alike
  const uint32_t b = __float_as_uint(l + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ double real_at(const Real& r, int64_t row) { return r.each ? (double)r.each[row] : r.all; }
__device__ __forceinline__ int64_t whole_at(const Whole& w, int64_t row) {
  if (!w.each) return w.all;
  return w.bytes == 4 ? (int64_t) static_cast<const int32_t*>(w.each)[row] : static_cast<const int64_t*>(w.each)[row];
}

// A row's numbers.
struct Row {
  double t, top_p, min_p, u;
  int64_t k;
  bool good;      // its parameters are usable
  __device__ __forceinline__ Row(const Args& a, int64_t row) {
    t = real_at(a.temperature, row);
    top_p = real_at(a.top_p, row);
    min_p = real_at(a.min_p, row);
    k = whole_at(a.top_k, row);
    u = a.u_double ? static_cast<const double*>(a.uniforms)[row] : (double)static_cast<const float*>(a.uniforms)[row];
    good = (t == 0. || (t >= 1e-30 && t <= 1e30)) && top_p == top_p && min_p <= 1. && k >= 0 && u == u;
    if (t == 0.) k = 1;
  }
};

// Weights relative to the row's largest logit.
struct Weights {
  double top, inv;        // 1 / T
  float top32, inv32, far;
  double least;
  __device__ __forceinline__ void set(float m, const Row& r) {
    top = m;
    top32 = m;
    inv = r.t == 0. ? 0. : 1. / r.t;
    inv32 = (float)inv;
    least = r.min_p;
    far = least > 0. ? fminf(kRange, -(float)log(least)) : kRange;
  }
  __device__ __forceinline__ double of(float l) const { return exp(((double)l - top) * inv); }
  // Whether an entry stays before the cut-offs by order: told in fp32 but next to the border.
  __device__ __forceinline__ bool in(float l) const {
    const float d = (top32 - l) * inv32;
    if (!(d <= far + 1e-3f)) return false;
    if (d < far - 1e-3f) return true;
    return least > 0. && far < kRange ? of(l) >= least : d <= far;
  }
};

template <typename T>
__device__ __forceinline__ float logit(const Args& a, int64_t row, int64_t i) {
  if (a.mask && !a.mask[row * a.mask_row + i * a.mask_col]) return -INFINITY;
  return lm::to_f<T>(static_cast<const T*>(a.logits)[row * a.ld + i]);
}

__device__ __forceinline__ void answer(const Args& a, int64_t row, int64_t token, float log_prob) {
  a.token[row] = token;
  a.log_prob[row] = log_prob;
}

__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ double block_sum(double s, double* red) {
  s = warp_sum(s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) s += red[w];
  return s;
}

// A CTA for a row.
template <typename T>
__global__ void __launch_bounds__(1024) row_kernel(const __grid_constant__ Args a) {
  __shared__ double red[32];
  __shared__ double parts[1024];
  __shared__ int ties[1024];
  __shared__ int64_t found;
  const int64_t row = blockIdx.x;
  const int n = blockDim.x, tid = threadIdx.x;
  const Row r(a, row);
  // the largest entry; a NaN or +inf
  float m = -INFINITY;
  bool bad = false;
  for (int64_t i = tid; i < a.v; i += n) {
    const float l = logit<T>(a, row, i);
    bad |= !(l < INFINITY);
    m = fmaxf(m, l);
  }
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < n / 32; ++w) m = fmaxf(m, (float)red[w]);
  __syncthreads();
  if (bad || !r.good || m == -INFINITY) {
    if (tid == 0) answer(a, row, -1, bad || !r.good ? __uint_as_float(0x7fc00000u) : -INFINITY);
    return;
  }
  Weights w;
  w.set(m, r);
  if (r.t == 0.) w.inv32 = w.far = 0.f, w.inv = 0.;
  const auto stays = [&](float l) { return r.t == 0. ? l == m : w.in(l); };
  // entries above `border`, and the first `most` of those on it, stay
  uint32_t border = 0;
  int64_t most = 0;
  const auto count_from = [&](uint32_t key) {
    int64_t c = 0;
    for (int64_t i = tid; i < a.v; i += n) {
      const float l = logit<T>(a, row, i);
      c += key_of(l) >= key && stays(l);
    }
    return (int64_t)block_sum((double)c, red);
  };
  if (r.k > 0 && count_from(0) > r.k) {
    uint32_t lo = 0, hi = key_of(m);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (count_from(mid) >= r.k) lo = mid;
      else hi = mid - 1;
    }
    border = lo;
    most = r.k - (border == key_of(m) ? 0 : count_from(border + 1));
  }
  // the sum of the staying entries from a key on (above the border)
  const auto sum_from = [&](uint32_t key) {
    double s = 0.;
    for (int64_t i = tid; i < a.v; i += n) {
      const float l = logit<T>(a, row, i);
      const uint32_t q = key_of(l);
      if (q >= key && q > border && stays(l)) s += w.of(l);
    }
    return block_sum(s, red);
  };
  if (r.top_p < 1.) {
    const double on = most ? (double)most * w.of(value_of(border)) : 0.;
    const double target = r.top_p * (sum_from(0) + on);
    uint32_t lo = border, hi = key_of(m);
    while (lo < hi) {   // the largest key from which on the sum reaches the target
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (sum_from(mid) >= target) lo = mid;
      else hi = mid - 1;
    }
    const double above = lo == key_of(m) ? 0. : sum_from(lo + 1), each = w.of(value_of(lo));
    int64_t have = lo == border ? most : 0;
    if (lo != border || !most) {
      int64_t c = 0;
      for (int64_t i = tid; i < a.v; i += n) {
        const float l = logit<T>(a, row, i);
        c += key_of(l) == lo && stays(l);
      }
      have = (int64_t)block_sum((double)c, red);
    }
    int64_t need = (int64_t)fmin((target - above) / each, (double)have);
    if (need < 1) need = 1;
    while (need > 1 && above + (double)(need - 1) * each >= target) --need;
    while (need < have && above + (double)need * each < target) ++need;
    border = lo;
    most = need;
  }
  // each thread's stretch of the row: its sum above the border, its entries on the border
  const int64_t per = (a.v + n - 1) / n, from = min(a.v, per * tid), to = min(a.v, from + per);
  double above = 0.;
  int on = 0;
  for (int64_t i = from; i < to; ++i) {
    const float l = logit<T>(a, row, i);
    if (!stays(l)) continue;
    const uint32_t q = key_of(l);
    if (q > border || (border == 0 && !most)) above += w.of(l);
    else if (q == border) ++on;
  }
  parts[tid] = above;
  ties[tid] = on;
  __syncthreads();
  const double each = most ? w.of(value_of(border)) : 0.;
  if (tid == 0) {
    // the running sum at each stretch's start, and the first border entry that counts there
    double total = 0.;
    int64_t seen = 0;
    int last = 0;
    for (int t = 0; t < n; ++t) {
      const int64_t here = max((int64_t)0, min((int64_t)ties[t], most - seen));
      const double s = parts[t] + (double)here * each;
      if (s > 0.) last = t;
      parts[t] = total;
      total += s;
      const int64_t start = seen;
      seen += ties[t];
      ties[t] = (int)min(start, (int64_t)INT32_MAX);
    }
    red[0] = total;
    const double target = r.u * total;
    int t = last;
    while (t > 0 && parts[t] > target) --t;
    found = t;
  }
  __syncthreads();
  if (tid == found) {
    const double total = red[0], target = r.u * total;
    double s = parts[tid];
    int64_t seen = ties[tid], token = -1;
    float at = m;
    for (int64_t i = from; i < to; ++i) {
      const float l = logit<T>(a, row, i);
      if (!stays(l)) continue;
      const uint32_t q = key_of(l);
      const bool tie = q == border && most;
      if (tie && seen++ >= most) continue;
      if (!tie && q < border) continue;
      s += w.of(l);
      token = i;
      at = l;
      if (s > target) break;
    }
    answer(a, row, token, (float)(((double)at - w.top) * w.inv - log(total)));
  }
}

}  // namespace

cudaError_t launch(const Args& a, int sms, cudaStream_t st) {
  const int threads = a.v >= 16384 ? 1024 : a.v >= 1024 ? 256 : 64;
  if (a.type == 0) row_kernel<float><<<(unsigned)a.rows, threads, 0, st>>>(a);
  else if (a.type == 1) row_kernel<__nv_bfloat16><<<(unsigned)a.rows, threads, 0, st>>>(a);
  else row_kernel<__half><<<(unsigned)a.rows, threads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace sampling
