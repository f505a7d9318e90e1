// Group norm with an activation over channels-last memory, forward and backward.
//
//   x^ = (x - mean_ng) rstd_ng,   z = x^ w_c + b_c,   y = act(z)
//   dz = dy act'(z),   P_nc = sum of dz,   Q_nc = sum of dz x^   (over a sample's pixels)
//   A_ng = sum of w_c P_nc,   B_ng = sum of w_c Q_nc   (over the group's channels)
//   dx = rstd (w dz - (A + x^ B) / m),   dw = sum over n of Q,   db = sum over n of P
//
// with m values in a group. Sums are fp32; the variance is that of the values
// less their mean, in a pass of its own (a sum of squares less the mean's
// square loses everything where the mean is large).
//
// A sample is one stretch of memory, cut into vectors of up to 16 bytes. After
// `cols` vectors the channels repeat, so threads that step by a multiple of
// `cols` keep their channels: their parameters and partial sums stay in
// registers, whatever the number of channels. A thread reads each of its
// vectors once from memory and keeps it in a slot of shared memory that no
// other thread reads, so only the sums need barriers.
//
// A cluster of CTAs holds a whole sample and joins its sums through
// distributed shared memory: one read and one write of each value. Samples too
// large for that take a pass for the sums and one that reads the values again.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <numeric>
#include <type_traits>

#include "groupnorm.h"
#include "lm_vec.h"

namespace cg = cooperative_groups;

namespace groupnorm {
namespace {

constexpr int kStages = 4;            // waits among a thread's loads

struct Args {
  const void *x, *dy;
  void *y;                            // y or dx
  Affine a;
  const float *mean_in, *rstd_in;
  float *mean, *rstd;
  float *ws;                          // partial sums of the samples' parts
  float *sums;                        // backward: [n][2][c] sums P and Q, or null
  int64_t pixels, vectors;            // of a sample
  int64_t n;
  int64_t chunk;
  int c, groups, cols, rows, iterations, act;
  float eps;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
  __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = lm::to_f<T>(e[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = lm::from_f<T>(f[i]);
  }
};

// One vector from memory into this thread's slot.
template <typename T, int V>
__device__ __forceinline__ void fetch(Vec<T, V>* slot, const Vec<T, V>* from) {
  if constexpr (sizeof(Vec<T, V>) >= 4) {
    const unsigned to = (unsigned)__cvta_generic_to_shared(slot);
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" :: "r"(to), "l"(from), "n"(sizeof(Vec<T, V>)) : "memory");
  } else {
    *slot = *from;
  }
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_for(int left) {
  switch (left) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
  }
}

__device__ __forceinline__ float parameter(const void* p, int type, int c, float otherwise) {
  if (!p) return otherwise;
  return type == 0 ? static_cast<const float*>(p)[c]
                   : type == 1 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c])
                               : __half2float(static_cast<const __half*>(p)[c]);
}

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }

template <int V>
__device__ __forceinline__ void activate(int act, float (&z)[V]) {
  if (act == kSilu) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] *= sigmoid(z[i]);
  } else if (act == kRelu) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] < 0.f ? 0.f : z[i];
  } else if (act == kGelu) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] *= normcdff(z[i]);
  }
}
// dy times the activation's slope at z.
template <int V>
__device__ __forceinline__ void slope(int act, const float (&z)[V], float (&d)[V]) {
  if (act == kSilu) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float s = sigmoid(z[i]);
      d[i] *= s * (1.f + z[i] * (1.f - s));
    }
  } else if (act == kRelu) {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = z[i] > 0.f ? d[i] : z[i] <= 0.f ? 0.f : z[i];
  } else if (act == kGelu) {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] *= normcdff(z[i]) + z[i] * .3989422804f * __expf(-.5f * z[i] * z[i]);
  }
}

// What the threads of a CTA share.
struct Shared {
  float *red;       // [threads * V] (twice for the backward)
  float *channel;   // [c] (twice)
  float *group;     // [2][groups]
  float *mean, *rstd;   // [groups]
};

template <int V, bool BWD>
__host__ __device__ inline int shared_floats(int threads, int c, int groups) {
  return (BWD ? 2 : 1) * (threads * V + c) + 4 * groups;
}
template <int V, bool BWD>
__device__ __forceinline__ Shared carve(float* at, int threads, int c, int groups) {
  Shared s;
  s.red = at;
  at += (BWD ? 2 : 1) * threads * V;
  s.channel = at;
  at += (BWD ? 2 : 1) * c;
  s.group = at;
  s.mean = at + 2 * groups;
  s.rstd = at + 3 * groups;
  return s;
}

// A thread's place: its column of the channels' pattern and its row, for the tile of columns from c0.
struct Place {
  int row, col, tile_cols, tile_rows;
  bool active;
};
__device__ __forceinline__ Place place_of(const Args& a, int c0) {
  Place p;
  p.tile_cols = min(a.cols - c0, (int)blockDim.x);
  p.tile_rows = a.cols <= (int)blockDim.x ? a.rows : 1;
  p.row = threadIdx.x / p.tile_cols;
  p.col = threadIdx.x - p.row * p.tile_cols;
  p.active = p.row < p.tile_rows;
  return p;
}

// Adds up v over the CTA's rows: channel[c] += the sum of the tile's values of channel c.
template <int V>
__device__ void join_rows(const Args& a, const Place& p, int c0, const float (&v)[V], float* red, float* channel) {
  if (p.active) {
#pragma unroll
    for (int i = 0; i < V; ++i) red[(p.row * p.tile_cols + p.col) * V + i] = v[i];
  }
  __syncthreads();
  const int width = p.tile_cols * V;
  for (int left = p.tile_rows; left > 1;) {
    const int half = (left + 1) >> 1;
    for (int i = threadIdx.x; i < (left - half) * width; i += blockDim.x) red[i] += red[i + half * width];
    left = half;
    __syncthreads();
  }
  const int from = c0 * V;
  for (int c = threadIdx.x; c < a.c; c += blockDim.x) {
    float s = channel[c];
    for (int q = c; q < from + width; q += a.c)
      if (q >= from) s += red[q - from];
    channel[c] = s;
  }
  __syncthreads();
}

// out[g] = the sum of channel[c] (times w_c) over the group's channels: a warp for each group.
__device__ __forceinline__ void join_channels(const Args& a, const float* channel, bool weighted, float* out) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = a.c / a.groups;
  for (int g = warp; g < a.groups; g += blockDim.x >> 5) {
    float s = 0.f;
    for (int i = lane; i < per; i += 32) {
      const int c = g * per + i;
      s += channel[c] * (weighted ? parameter(a.a.w, a.a.w_type, c, 1.f) : 1.f);
    }
    s = lm::warp_sum(s);
    if (lane == 0) out[g] = s;
  }
}

template <int V>
__device__ __forceinline__ int channel_of(const Args& a, int c0, int col, int i) {
  return (int)(((int64_t)(c0 + col) * V + i) % a.c);
}

// A CTA's part of a sample: vectors [begin, begin + count) and the first address.
struct Part {
  int64_t sample, begin, count;
};
__device__ __forceinline__ Part part_of(const Args& a, int ctas) {
  Part p;
  p.sample = blockIdx.x / ctas;
  p.begin = (int64_t)(blockIdx.x - p.sample * ctas) * a.chunk;
  p.count = max((int64_t)0, min(a.chunk, a.vectors - p.begin));
  return p;
}

// f(k, i) for this thread's vectors i of its part in the tile of columns from c0, k counting its slots over all tiles.
template <typename F>
__device__ __forceinline__ void for_vectors(const Args& a, const Place& p, int c0, int64_t count, F&& f) {
  if (!p.active) return;
  const int64_t step = (int64_t)p.tile_rows * a.cols;
  int k = c0 / (int)blockDim.x * a.iterations;
  for (int64_t i = (int64_t)p.row * a.cols + c0 + p.col; i < count; i += step, ++k) f(k, i);
}

// Sums `v` of the group over the cluster's CTAs, in the order of their ranks.
__device__ __forceinline__ void join_cluster(cg::cluster_group& cluster, float* mine, float* out, int n) {
  cluster.sync();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    float s = 0.f;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) s += cluster.map_shared_rank(mine, r)[i];
    out[i] = s;
  }
  __syncthreads();
}

// Forward. FULL: the cluster holds the sample and writes y. Otherwise a CTA
// writes its part's (sum, sum of squares less its own mean's) of each group.
template <typename T, int V, bool FULL>
__global__ void __launch_bounds__(512) forward_kernel(const __grid_constant__ Args a) {
  using Vector = Vec<T, V>;
  extern __shared__ __align__(16) unsigned char raw[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = FULL ? (int)cluster.num_blocks() : (int)gridDim.x / (int)a.n;
  const Part part = part_of(a, ctas);
  const int tiles = (a.cols + blockDim.x - 1) / blockDim.x;
  Vector* slots = reinterpret_cast<Vector*>(raw);
  const Shared s = carve<V, false>(reinterpret_cast<float*>(raw + sizeof(Vector) * blockDim.x * a.iterations * tiles),
                                   blockDim.x, a.c, a.groups);
  const Vector* x = static_cast<const Vector*>(a.x) + part.sample * a.vectors + part.begin;
  const int per = a.c / a.groups;
  // all loads are under way before the first is waited for
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    for_vectors(a, p, c0, part.count, [&](int k, int64_t i) { fetch(slots + k * blockDim.x + threadIdx.x, x + i); });
  }
  commit();
  for (int c = threadIdx.x; c < a.c; c += blockDim.x) s.channel[c] = 0.f;
  __syncthreads();
  wait_for(0);
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    float sum[V] = {};
    for_vectors(a, p, c0, part.count, [&](int k, int64_t) {
      float v[V];
      slots[k * blockDim.x + threadIdx.x].get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) sum[e] += v[e];
    });
    join_rows(a, p, c0, sum, s.red, s.channel);
  }
  join_channels(a, s.channel, false, s.group);
  __syncthreads();
  const float values = FULL ? (float)a.pixels * per : (float)((double)part.count * V / a.groups);
  if (FULL) {
    join_cluster(cluster, s.group, s.mean, a.groups);
  } else {
    for (int g = threadIdx.x; g < a.groups; g += blockDim.x) s.mean[g] = s.group[g];
    __syncthreads();
  }
  for (int g = threadIdx.x; g < a.groups; g += blockDim.x) s.mean[g] = values > 0.f ? s.mean[g] / values : 0.f;
  for (int c = threadIdx.x; c < a.c; c += blockDim.x) s.channel[c] = 0.f;
  __syncthreads();
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    float sum[V] = {}, mean[V];
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = p.active ? s.mean[channel_of<V>(a, c0, p.col, e) / per] : 0.f;
    for_vectors(a, p, c0, part.count, [&](int k, int64_t) {
      float v[V];
      slots[k * blockDim.x + threadIdx.x].get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) sum[e] += (v[e] - mean[e]) * (v[e] - mean[e]);
    });
    join_rows(a, p, c0, sum, s.red, s.channel);
  }
  join_channels(a, s.channel, false, s.group + a.groups);
  __syncthreads();
  if (!FULL) {
    float* to = a.ws + blockIdx.x * (int64_t)a.groups * 2;
    for (int g = threadIdx.x; g < a.groups; g += blockDim.x) {
      to[2 * g] = s.mean[g];
      to[2 * g + 1] = s.group[a.groups + g];
    }
    return;
  }
  join_cluster(cluster, s.group + a.groups, s.rstd, a.groups);
  for (int g = threadIdx.x; g < a.groups; g += blockDim.x) {
    s.rstd[g] = rsqrtf(s.rstd[g] / values + a.eps);
    if (a.mean && cluster.block_rank() == 0) {
      a.mean[part.sample * a.groups + g] = s.mean[g];
      a.rstd[part.sample * a.groups + g] = s.rstd[g];
    }
  }
  __syncthreads();
  Vector* y = static_cast<Vector*>(a.y) + part.sample * a.vectors + part.begin;
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    float mean[V], scale[V], shift[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = p.active ? channel_of<V>(a, c0, p.col, e) : 0;
      mean[e] = s.mean[c / per];
      scale[e] = s.rstd[c / per] * parameter(a.a.w, a.a.w_type, c, 1.f);
      shift[e] = parameter(a.a.b, a.a.b_type, c, 0.f);
    }
    for_vectors(a, p, c0, part.count, [&](int k, int64_t i) {
      float v[V];
      slots[k * blockDim.x + threadIdx.x].get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = (v[e] - mean[e]) * scale[e] + shift[e];
      activate(a.act, v);
      Vector o;
      o.set(v);
      y[i] = o;
    });
  }
  cluster.sync();   // no CTA ends while another reads its sums
}

// Means and deviations of the samples from their parts' (Chan, Golub & LeVeque, 1979): a warp for each (sample, group).
__global__ void merge_kernel(const __grid_constant__ Args a, int ctas, int vec) {
  const int64_t at = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (at >= a.n * a.groups) return;
  const int lane = threadIdx.x & 31, g = (int)(at % a.groups);
  const float* from = a.ws + at / a.groups * ctas * a.groups * 2 + 2 * g;
  const auto count = [&](int i) {
    return (float)((double)max((int64_t)0, min(a.chunk, a.vectors - i * a.chunk)) * vec / a.groups);
  };
  const float all = (float)a.pixels * (float)(a.c / a.groups);
  float s = 0.f;
  for (int i = lane; i < ctas; i += 32) s += from[(int64_t)i * a.groups * 2] * (count(i) / all);
  const float mean = lm::warp_sum(s);
  s = 0.f;
  for (int i = lane; i < ctas; i += 32) {
    const float d = from[(int64_t)i * a.groups * 2] - mean;
    s += from[(int64_t)i * a.groups * 2 + 1] + d * d * count(i);
  }
  const float var = lm::warp_sum(s) / all;
  if (lane == 0) {
    a.mean[at] = mean;
    a.rstd[at] = rsqrtf(var + a.eps);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(512) apply_kernel(const __grid_constant__ Args a) {
  using Vector = Vec<T, V>;
  const Part part = part_of(a, (int)gridDim.x / (int)a.n);
  const int per = a.c / a.groups;
  const Vector* x = static_cast<const Vector*>(a.x) + part.sample * a.vectors + part.begin;
  Vector* y = static_cast<Vector*>(a.y) + part.sample * a.vectors + part.begin;
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    float mean[V], scale[V], shift[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = p.active ? channel_of<V>(a, c0, p.col, e) : 0;
      const int64_t g = part.sample * a.groups + c / per;
      mean[e] = a.mean[g];
      scale[e] = a.rstd[g] * parameter(a.a.w, a.a.w_type, c, 1.f);
      shift[e] = parameter(a.a.b, a.a.b_type, c, 0.f);
    }
    for_vectors(a, p, c0, part.count, [&](int, int64_t i) {
      const Vector in = x[i];
      float v[V];
      in.get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = (v[e] - mean[e]) * scale[e] + shift[e];
      activate(a.act, v);
      Vector o;
      o.set(v);
      y[i] = o;
    });
  }
}

// A thread's parameters of its channels in the backward.
template <int V>
struct Channels {
  float mean[V], rstd[V], w[V], b[V];
  int c[V];
  __device__ __forceinline__ Channels(const Args& a, const Place& p, int c0, int64_t sample) {
    const int per = a.c / a.groups;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      c[e] = p.active ? channel_of<V>(a, c0, p.col, e) : 0;
      const int64_t g = sample * a.groups + c[e] / per;
      mean[e] = a.mean_in[g];
      rstd[e] = a.rstd_in[g];
      w[e] = parameter(a.a.w, a.a.w_type, c[e], 1.f);
      b[e] = parameter(a.a.b, a.a.b_type, c[e], 0.f);
    }
  }
  // x becomes x^, d (the gradient of y) becomes dz
  __device__ __forceinline__ void derive(int act, float (&x)[V], float (&d)[V]) const {
    float z[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      x[e] = (x[e] - mean[e]) * rstd[e];
      z[e] = x[e] * w[e] + b[e];
    }
    slope(act, z, d);
  }
};

// dx of a vector from its x^ and dz and the group's A / m and B / m.
template <int V>
__device__ __forceinline__ void input_gradient(const Channels<V>& ch, const float (&ga)[V], const float (&gb)[V],
                                               const float (&x)[V], float (&d)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) d[e] = ch.rstd[e] * (ch.w[e] * d[e] - (ga[e] + x[e] * gb[e]));
}

// Backward. FULL: the cluster holds the sample's x and dy and writes dx.
// Otherwise a CTA writes its part's P and Q of each channel.
template <typename T, int V, bool FULL>
__global__ void __launch_bounds__(512) backward_kernel(const __grid_constant__ Args a) {
  using Vector = Vec<T, V>;
  extern __shared__ __align__(16) unsigned char raw[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = FULL ? (int)cluster.num_blocks() : (int)gridDim.x / (int)a.n;
  const Part part = part_of(a, ctas);
  const int tiles = (a.cols + blockDim.x - 1) / blockDim.x;
  const int held = FULL ? blockDim.x * a.iterations * tiles : 0;
  Vector* slots = reinterpret_cast<Vector*>(raw);
  const Shared s = carve<V, true>(reinterpret_cast<float*>(raw + 2 * sizeof(Vector) * held), blockDim.x, a.c, a.groups);
  const Vector* x = static_cast<const Vector*>(a.x) + part.sample * a.vectors + part.begin;
  const Vector* dy = static_cast<const Vector*>(a.dy) + part.sample * a.vectors + part.begin;
  const int per = a.c / a.groups;
  if (FULL) {
    for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
      const Place p = place_of(a, c0);
      for_vectors(a, p, c0, part.count, [&](int k, int64_t i) {
        fetch(slots + k * blockDim.x + threadIdx.x, x + i);
        fetch(slots + held + k * blockDim.x + threadIdx.x, dy + i);
      });
    }
    commit();
  }
  for (int c = threadIdx.x; c < 2 * a.c; c += blockDim.x) s.channel[c] = 0.f;
  __syncthreads();
  if (FULL) wait_for(0);
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    const Channels<V> ch(a, p, c0, part.sample);
    float sp[V] = {}, sq[V] = {};
    for_vectors(a, p, c0, part.count, [&](int k, int64_t i) {
      float v[V], d[V];
      const Vector vx = FULL ? slots[k * blockDim.x + threadIdx.x] : x[i];
      const Vector vd = FULL ? slots[held + k * blockDim.x + threadIdx.x] : dy[i];
      vx.get(v);
      vd.get(d);
      ch.derive(a.act, v, d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sp[e] += d[e];
        sq[e] += d[e] * v[e];
      }
    });
    join_rows(a, p, c0, sp, s.red, s.channel);
    join_rows(a, p, c0, sq, s.red, s.channel + a.c);
  }
  if (!FULL) {
    float* to = a.ws + blockIdx.x * (int64_t)a.c * 2;
    for (int c = threadIdx.x; c < 2 * a.c; c += blockDim.x) to[c] = s.channel[c];
    return;
  }
  join_channels(a, s.channel, true, s.group);
  join_channels(a, s.channel + a.c, true, s.group + a.groups);
  __syncthreads();
  join_cluster(cluster, s.group, s.mean, 2 * a.groups);   // A and B lie where mean and rstd would
  if (a.sums) {   // this CTA's share of the channels
    for (int c = cluster.block_rank() * blockDim.x + threadIdx.x; c < 2 * a.c; c += cluster.num_blocks() * blockDim.x) {
      float v = 0.f;
      for (unsigned r = 0; r < cluster.num_blocks(); ++r) v += cluster.map_shared_rank(s.channel, r)[c];
      a.sums[part.sample * 2 * a.c + c] = v;
    }
  }
  const float inv = 1.f / ((float)a.pixels * per);
  Vector* dx = static_cast<Vector*>(a.y) + part.sample * a.vectors + part.begin;
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    const Channels<V> ch(a, p, c0, part.sample);
    float ga[V], gb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      ga[e] = s.mean[ch.c[e] / per] * inv;
      gb[e] = s.rstd[ch.c[e] / per] * inv;
    }
    for_vectors(a, p, c0, part.count, [&](int k, int64_t i) {
      float v[V], d[V];
      slots[k * blockDim.x + threadIdx.x].get(v);
      slots[held + k * blockDim.x + threadIdx.x].get(d);
      ch.derive(a.act, v, d);
      input_gradient(ch, ga, gb, v, d);
      Vector o;
      o.set(d);
      dx[i] = o;
    });
  }
  cluster.sync();   // no CTA ends while another reads its sums
}

// sums[n][2][c] = the sum of the sample's parts, in their order.
__global__ void join_parts_kernel(const __grid_constant__ Args a, int ctas) {
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (at >= a.n * 2 * a.c) return;
  const int64_t n = at / (2 * a.c), c = at - n * 2 * a.c;
  const float* from = a.ws + n * ctas * 2 * a.c + c;
  float s = 0.f;
  for (int i = 0; i < ctas; ++i) s += from[(int64_t)i * 2 * a.c];
  a.sums[at] = s;
}

template <typename T, int V>
__global__ void __launch_bounds__(512) input_gradient_kernel(const __grid_constant__ Args a) {
  using Vector = Vec<T, V>;
  extern __shared__ __align__(16) unsigned char raw[];
  float* group = reinterpret_cast<float*>(raw);   // [2][groups]
  const Part part = part_of(a, (int)gridDim.x / (int)a.n);
  const int per = a.c / a.groups;
  join_channels(a, a.sums + part.sample * 2 * a.c, true, group);
  join_channels(a, a.sums + part.sample * 2 * a.c + a.c, true, group + a.groups);
  __syncthreads();
  const float inv = 1.f / ((float)a.pixels * per);
  const Vector* x = static_cast<const Vector*>(a.x) + part.sample * a.vectors + part.begin;
  const Vector* dy = static_cast<const Vector*>(a.dy) + part.sample * a.vectors + part.begin;
  Vector* dx = static_cast<Vector*>(a.y) + part.sample * a.vectors + part.begin;
  for (int c0 = 0; c0 < a.cols; c0 += blockDim.x) {
    const Place p = place_of(a, c0);
    const Channels<V> ch(a, p, c0, part.sample);
    float ga[V], gb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      ga[e] = group[ch.c[e] / per] * inv;
      gb[e] = group[a.groups + ch.c[e] / per] * inv;
    }
    for_vectors(a, p, c0, part.count, [&](int, int64_t i) {
      float v[V], d[V];
      const Vector vx = x[i], vd = dy[i];
      vx.get(v);
      vd.get(d);
      ch.derive(a.act, v, d);
      input_gradient(ch, ga, gb, v, d);
      Vector o;
      o.set(d);
      dx[i] = o;
    });
  }
}

// dw and db: sums of the samples' Q and P, 64 threads down each column, in an order that the sizes alone give.
__device__ __forceinline__ void put(void* p, int type, int at, float v) {
  if (type == 0) static_cast<float*>(p)[at] = v;
  else if (type == 1) static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[at] = __float2half_rn(v);
}
__global__ void __launch_bounds__(512) parameters_kernel(const float* sums, int64_t n, int c, void* dw, int w_type, void* db,
                                                         int b_type) {
  __shared__ float red[64][9];
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3, col = blockIdx.x * 8 + tx;
  float s = 0.f;
  if (col < 2 * c) {
#pragma unroll 4
    for (int64_t i = ty; i < n; i += 64) s += sums[i * 2 * c + col];
  }
  red[ty][tx] = s;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, out = blockIdx.x * 8 + warp;
  if (warp >= 8) return;
  s = lm::warp_sum(red[lane][warp] + red[lane + 32][warp]);
  if (lane == 0 && out < 2 * c) {
    if (out < c) {
      if (db) put(db, b_type, out, s);
    } else if (dw) {
      put(dw, w_type, out - c, s);
    }
  }
}

template <typename F>
void with_vector(const Shape& s, const Plan& p, F&& f) {
  const auto by = [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2)
      if (p.vec == 8) return f(t, std::integral_constant<int, 8>{});
    if (p.vec == 4) return f(t, std::integral_constant<int, 4>{});
    return f(t, std::integral_constant<int, 1>{});
  };
  if (s.type == 0) by(float{});
  else if (s.type == 1) by(__nv_bfloat16{});
  else by(__half{});
}

Args args_of(const Shape& s, const Plan& p) {
  Args a{};
  a.pixels = s.pixels;
  a.vectors = s.pixels * s.c / p.vec;
  a.n = s.n;
  a.chunk = p.chunk;
  a.c = s.c;
  a.groups = s.groups;
  a.cols = p.cols;
  a.rows = p.rows;
  a.iterations = p.iterations;
  return a;
}

template <typename... A>
cudaError_t run(void (*kernel)(A...), int64_t grid, int threads, int cluster, int smem, cudaStream_t st, A... args) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

constexpr int kMostSmem = 200 * 1024;   // of a CTA
constexpr int kMostCtas = 8;            // of a cluster

int shared_bytes(const Shape& s, int vec, int threads, bool backward) {
  const int f = vec == 8 ? (backward ? shared_floats<8, true>(threads, s.c, s.groups) : shared_floats<8, false>(threads, s.c, s.groups))
              : vec == 4 ? (backward ? shared_floats<4, true>(threads, s.c, s.groups) : shared_floats<4, false>(threads, s.c, s.groups))
                         : (backward ? shared_floats<1, true>(threads, s.c, s.groups) : shared_floats<1, false>(threads, s.c, s.groups));
  return f * 4;
}

}  // namespace

Plan plan(const Shape& s, bool backward, bool aligned, int sms) {
  Plan p{};
  const int size = s.type == 0 ? 4 : 2, most = 16 / size;
  const int64_t values = s.pixels * s.c;
  p.vec = aligned && values % most == 0 ? most : aligned && values % 4 == 0 ? 4 : 1;
  p.cols = s.c / std::gcd(s.c, p.vec);
  // threads: as few as possible without a row
  p.threads = 256;
  if (p.cols < 512) {
    double best = 0.;
    for (int t = 256; t <= 512; t += 32) {
      const double used = (double)(t / p.cols * p.cols) / t;
      if (used > best + .02) best = used, p.threads = t;
    }
  }
  p.rows = std::max(1, p.threads / p.cols);
  const int tiles = (p.cols + p.threads - 1) / p.threads;
  const int64_t vectors = values / p.vec;
  const int64_t all_rows = (vectors + p.cols - 1) / p.cols;   // the last may be cut
  const int fixed = shared_bytes(s, p.vec, p.threads, backward);
  const auto cut = [&](int ctas) {
    p.ctas = ctas;
    const int64_t rows = (all_rows + ctas - 1) / ctas;
    p.iterations = (int)std::min<int64_t>((rows + p.rows - 1) / p.rows, 1 << 30);
    p.chunk = rows * p.cols;
    return (int64_t)(backward ? 2 : 1) * p.vec * size * p.threads * p.iterations * tiles + fixed;
  };
  for (int ctas = 1; ctas <= kMostCtas; ctas *= 2) {
    const int64_t bytes = cut(ctas);
    const bool last = ctas == kMostCtas;
    if (bytes <= (last ? kMostSmem : 72 * 1024) && (last || s.n * ctas >= 2 * sms || bytes < 16 * 1024)) {
      p.resident = true;
      p.smem = (int)bytes;
      return p;
    }
  }
  // parts that are read again: enough of them for all SMs, of at least 16 iterations
  const int64_t most_ctas = std::max<int64_t>(1, all_rows / (p.rows * 16));
  const int64_t fits = (kMostSmem / 2 - fixed) / ((int64_t)p.vec * size * p.threads * tiles);   // iterations that the forward's sums hold
  const int64_t least = (all_rows + fits * p.rows - 1) / (fits * p.rows);
  cut((int)std::max<int64_t>(least, std::min<int64_t>(most_ctas, (8 * sms + s.n - 1) / s.n)));
  p.resident = false;
  p.smem = backward ? fixed : (int)((int64_t)p.vec * size * p.threads * p.iterations * tiles + fixed);
  return p;
}

int64_t forward_workspace(const Shape& s, const Plan& p) { return p.resident ? 0 : s.n * p.ctas * s.groups * 2; }
int64_t backward_workspace(const Shape& s, const Plan& p) {
  return s.n * 2 * s.c * (p.resident ? 1 : 1 + (int64_t)p.ctas);
}

cudaError_t forward(const Shape& s, const Plan& p, const void* x, const Affine& affine, float eps, Activation act, void* y,
                    float* mean, float* rstd, float* workspace, cudaStream_t st) {
  Args a = args_of(s, p);
  a.x = x;
  a.y = y;
  a.a = affine;
  a.eps = eps;
  a.act = act;
  a.mean = mean;
  a.rstd = rstd;
  a.ws = workspace;
  cudaError_t e = cudaSuccess;
  with_vector(s, p, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    if (p.resident) {
      e = run(forward_kernel<T, V, true>, s.n * p.ctas, p.threads, p.ctas, p.smem, st, a);
      return;
    }
    e = run(forward_kernel<T, V, false>, s.n * p.ctas, p.threads, 1, p.smem, st, a);
    if (e == cudaSuccess) e = run(merge_kernel, (s.n * s.groups + 7) / 8, 256, 1, 0, st, a, p.ctas, p.vec);
    if (e == cudaSuccess) e = run(apply_kernel<T, V>, s.n * p.ctas, p.threads, 1, 0, st, a);
  });
  return e;
}

cudaError_t backward(const Shape& s, const Plan& p, const void* dy, const void* x, const Affine& affine, const float* mean,
                     const float* rstd, Activation act, void* dx, void* dw, void* db, float* workspace, cudaStream_t st) {
  Args a = args_of(s, p);
  a.x = x;
  a.dy = dy;
  a.y = dx;
  a.a = affine;
  a.act = act;
  a.mean_in = mean;
  a.rstd_in = rstd;
  a.sums = workspace;
  a.ws = workspace + s.n * 2 * s.c;
  cudaError_t e = cudaSuccess;
  with_vector(s, p, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    if (p.resident) {
      e = run(backward_kernel<T, V, true>, s.n * p.ctas, p.threads, p.ctas, p.smem, st, a);
      return;
    }
    e = run(backward_kernel<T, V, false>, s.n * p.ctas, p.threads, 1, p.smem, st, a);
    if (e == cudaSuccess) e = run(join_parts_kernel, (s.n * 2 * s.c + 255) / 256, 256, 1, 0, st, a, p.ctas);
    if (e == cudaSuccess) e = run(input_gradient_kernel<T, V>, s.n * p.ctas, p.threads, 1, s.groups * 8, st, a);
  });
  if (e == cudaSuccess && (dw || db))
    e = run(parameters_kernel, (2 * s.c + 7) / 8, 512, 1, 0, st, (const float*)workspace, s.n, s.c, dw, affine.w_type, db,
            affine.b_type);
  return e;
}

int launches(const Plan& p, bool backward, bool parameters) {
  return (p.resident ? 1 : 3) + (backward && parameters ? 1 : 0);
}

}  // namespace groupnorm
