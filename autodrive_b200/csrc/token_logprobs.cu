// Log-probabilities of given tokens under masked logits, with the entropy of
// each row's distribution, its most probable alternatives, and the gradient.
//
//   z = x / T over the valid entries      lse = log sum exp z
//   log_prob = z[token] - lse             entropy = -sum p log p
//   dx_j = (g_l ([j = token] - p_j) - g_e p_j (log p_j + entropy)) / T
//
// The forward reads the logits once: every thread keeps a running maximum m,
// s = sum e and t = sum e (x - m), e = exp((x - m) / T), of its share of a row,
// and rescales s and t when m grows; the shares are joined with the same rule.
// Then lse = m / T + log s and entropy = log s - t / (T s), both terms of which
// are positive, so nothing cancels. The row's m, log s and entropy are kept for
// the backward, which reads the logits once more and writes the gradient.
// Masked entries are never used, whatever they hold; entries that are -inf have
// no probability. A row without any entry left has log_prob -inf, entropy 0 and
// no gradient; a NaN or +inf among its entries makes a row's results NaN.
//
// Alternatives (the `top` largest logits, equal ones by their index): at least
// `top` entries are as large as the top-th largest of the maxima of groups of
// threads, so only the few threads whose maximum reaches that bound have their
// entries looked at again, and the entries that reach it are ranked.
//
// Bound by memory for long rows. Rows of up to 1024 entries are held in the
// registers of one warp or of a part of one; longer ones take a CTA each, or a
// cluster of CTAs where there are few rows.
#include <torch/extension.h>
#include <ATen/ExpandUtils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "lm_host.h"
#include "lm_vec.h"

namespace py = pybind11;

namespace {

constexpr int kMaxTop = 64;
constexpr int kSmall = 1024;        // longest row held in one warp's registers
constexpr int kThreads = 256;       // threads of a long row's CTA
constexpr int kAhead = 4;           // vectors of eight that a thread loads before it uses the first
constexpr int kMaxSplits = 8;       // CTAs of a cluster that share a row
constexpr int kCandidates = 1024;   // entries ranked in shared memory
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* x;
  const uint8_t* mask;     // null without one
  const int64_t* tokens;
  int64_t rows, ldx, ldm;
  int v, top;
  float inv_t;             // 1 / T
  int splits;              // CTAs that share a long row
  float* log_prob;
  float* entropy;
  float* top_value;        // [rows][top]
  int64_t* top_token;      // [rows][top]
  float* stats;            // [rows][3]: m, log s, entropy; null when no backward follows
};

// Running maximum, sum and first moment of a set of entries.
struct Stat {
  float m, s, t;
};
__device__ __forceinline__ Stat empty_stat() { return Stat{-INFINITY, 0.f, 0.f}; }

// The sums of `a` for the maximum m >= a.m.
__device__ __forceinline__ Stat rescaled(const Stat& a, float m, float c) {
  if (a.s == 0.f) return Stat{m, 0.f, 0.f};
  const float d = a.m - m;
  if (!(d < 0.f)) return Stat{m, a.s, a.t};   // the same maximum (NaN sums stay NaN)
  const float f = exp2f(d * c);
  const float s = a.s * f;                    // a NaN stays one, even times zero
  return Stat{m, s, f > 0.f ? (a.t + a.s * d) * f : s};
}
__device__ __forceinline__ Stat joined(const Stat& a, const Stat& b, float c) {
  const float m = fmaxf(a.m, b.m);
  const Stat p = rescaled(a, m, c), q = rescaled(b, m, c);
  return Stat{m, p.s + q.s, p.t + q.t};
}
// Adds an entry that is at most st.m. The difference is kept finite, so that an
// entry without weight adds 0 times a number; NaN passes through.
__device__ __forceinline__ void add_entry(Stat& st, float x, float c) {
  float d = x - st.m;
  asm("max.NaN.f32 %0, %0, 0fFF000000;" : "+f"(d));   // -2^127
  const float e = exp2f(d * c);
  st.s += e;
  st.t = fmaf(e, d, st.t);
}

template <int G>
__device__ __forceinline__ Stat group_join(Stat st, float c) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    Stat u;
    u.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    u.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    u.t = __shfl_xor_sync(0xffffffffu, st.t, o);
    st = joined(st, u, c);
  }
  return st;
}

// Bits that order like the values. Both zeros, and subnormal values (which the
// compiler's fast-math mode compares as zeros), are one value. Not for NaN.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = fabsf(x) < 0x1p-126f ? 0u : __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order_bits(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Larger values first, then smaller indices; 0 is "none".
__device__ __forceinline__ uint64_t entry_key(float x, int idx) {
  return (uint64_t)order_bits(x) << 32 | (uint32_t)~(uint32_t)idx;
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

// Whether an entry can be an alternative: it has a probability.
__device__ __forceinline__ bool ranked(float x) { return x > -INFINITY; }

template <int G>
__device__ __forceinline__ uint64_t group_max(uint64_t k) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(0xffffffffu, k, o);
    k = u > k ? u : k;
  }
  return k;
}

// log s of a sum s >= 1, within 6 * 2^-24 of itself. The logarithm of the
// compiler's fast-math mode is off by up to 2^-21.4 next to s = 1, which for a
// peaked row is the whole log-probability. s = 2^k m with m within a factor of
// sqrt(2) of 1, and log m = 2 atanh(f) = 2 (f + f^3/3 + f^5/5 + ...), f =
// (m - 1) / (m + 1), |f| < 0.172: what follows f^9 is below 2^-28 of it. Over
// 65536 rows of 8 this takes 0.4 us of 5.9, a 64-bit logarithm 1.4.
__device__ __forceinline__ float log_sum(const Stat& st) {
  if (st.m == -INFINITY) return 0.f;
  const uint32_t u = __float_as_uint(st.s);
  if (u >= 0x7f800000u) return st.s;                              // NaN
  const int k = ((int)u - 0x3f3504f3) >> 23;                      // 0x3f3504f3: sqrt(1/2)
  const float m = __uint_as_float(u - ((uint32_t)k << 23));
  const float a = m - 1.f, b = m + 1.f, inv = __fdividef(1.f, b), f0 = a * inv;
  const float f = fmaf(fmaf(-f0, b, a), inv, f0), q = f * f;      // the quotient, corrected by its remainder
  const float p = fmaf(fmaf(fmaf(q, 1.f / 9.f, 1.f / 7.f), q, 1.f / 5.f), q, 1.f / 3.f);
  const float r = 2.f * fmaf(f * q, p, f);
  return fmaf((float)k, 0.693147181f, r);
}

// The row's results, by one thread.
__device__ __forceinline__ void write_row(const Args& a, int64_t r, const Stat& st, float logs, float logit, bool valid) {
  const bool none = st.m == -INFINITY;
  const float ent = none ? 0.f : logs - st.t / st.s * a.inv_t;
  const int64_t tok = a.tokens[r];
  float lp;
  if (tok < 0) lp = 0.f;                                        // ignored
  else if (tok >= a.v) lp = __uint_as_float(0x7fffffffu);       // no such token
  else if (none || !valid) lp = -INFINITY;
  else lp = (logit - st.m) * a.inv_t - logs;
  a.log_prob[r] = lp;
  a.entropy[r] = ent;
  if (a.stats) {
    a.stats[3 * r] = st.m;
    a.stats[3 * r + 1] = logs;
    a.stats[3 * r + 2] = ent;
  }
}

__device__ __forceinline__ void write_top(const Args& a, int64_t r, int place, uint64_t key, const Stat& st,
                                          float logs) {
  const bool none = key == 0;
  a.top_token[r * a.top + place] = none ? -1 : key_index(key);
  a.top_value[r * a.top + place] =
      none ? -INFINITY : (from_order_bits((uint32_t)(key >> 32)) - st.m) * a.inv_t - logs;
}

// ---- short rows: G lanes per row, E entries per lane, 32 / G rows per warp ----
template <typename T, int G, int E>
__global__ void __launch_bounds__(256) small_fwd_kernel(const Args a) {
  const int lane = threadIdx.x & 31, sub = lane % G;
  const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
  const bool live = r < a.rows;
  const float c = a.inv_t * kLog2e;
  const T* row = reinterpret_cast<const T*>(a.x) + (live ? r : 0) * a.ldx;
  const uint8_t* mrow = a.mask ? a.mask + (live ? r : 0) * a.ldm : nullptr;
  float x[E];
  uint32_t ok = 0;
  Stat st = empty_stat();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int col = e * G + sub;
    const bool in = live && col < a.v && (!mrow || mrow[col]);
    x[e] = in ? lm::to_f<T>(row[col]) : -INFINITY;
    if (in) ok |= 1u << e;
    st.m = fmaxf(st.m, x[e]);
    if (x[e] != x[e]) st.t = x[e];   // a NaN makes the row NaN (fmaxf passes it over)
  }
  if (st.m != -INFINITY) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (ok >> e & 1) add_entry(st, x[e], c);
  } else if (st.t != st.t) {
    st = Stat{0.f, st.t, st.t};
  }
  st = group_join<G>(st, c);
  const int64_t tok = live ? a.tokens[r] : -1;
  // the taken token's logit, from the lane that has it
  float logit = 0.f;
  bool valid = false;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (tok == e * G + sub) logit = x[e], valid = ok >> e & 1;
  const int src = (lane & ~(G - 1)) + (tok < 0 ? 0 : (int)(tok % G));
  logit = __shfl_sync(0xffffffffu, logit, src);
  valid = __shfl_sync(0xffffffffu, (int)valid, src) != 0;
  const float logs = sub == 0 ? log_sum(st) : 0.f;
  if (live && sub == 0) write_row(a, r, st, logs, logit, valid);
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (ok >> e & 1 && ranked(x[e])) {
        const uint64_t key = entry_key(x[e], e * G + sub);
        best = key > best ? key : best;
      }
    best = group_max<G>(best);
#pragma unroll
    for (int e = 0; e < E; ++e)   // taken
      if (best && key_index(best) == e * G + sub) ok &= ~(1u << e);
    if (live && sub == 0) write_top(a, r, k, best, st, logs);
  }
}

template <typename T, int G, int E>
__global__ void __launch_bounds__(256)
small_bwd_kernel(const Args a, const float* __restrict__ g_lp, const float* __restrict__ g_ent, T* __restrict__ dx) {
  const int sub = threadIdx.x % G;
  const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
  if (r >= a.rows) return;
  const T* row = reinterpret_cast<const T*>(a.x) + r * a.ldx;
  const uint8_t* mrow = a.mask ? a.mask + r * a.ldm : nullptr;
  const float m = a.stats[3 * r], logs = a.stats[3 * r + 1], ent = a.stats[3 * r + 2];
  const int64_t tok = a.tokens[r];
  const float gl = g_lp && tok >= 0 && tok < a.v ? g_lp[r] : 0.f, ge = g_ent ? g_ent[r] : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int col = e * G + sub;
    if (col >= a.v) break;
    float d = 0.f;
    if ((!mrow || mrow[col]) && m != -INFINITY) {
      const float lp = (lm::to_f<T>(row[col]) - m) * a.inv_t - logs;
      const float p = exp2f(lp * kLog2e);
      d = p == 0.f ? 0.f : p * (-gl - ge * (lp + ent));
      if (col == tok) d += gl;
      d *= a.inv_t;
    }
    dx[r * a.v + col] = lm::from_f<T>(d);
  }
}

// ---- long rows ---------------------------------------------------------------
// A row is read in vectors of eight entries on 16-byte boundaries, whatever the
// boundary it starts on: vector i covers the columns 8 i - shift .. + 7, where
// `shift` entries lie before the row between the boundary and its start. The
// first and the last vector may run out of the row and are read one by one.
template <typename T>
struct Raw {   // eight entries as they lie in memory
  alignas(16) T e[8];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(T) / 2); ++j) reinterpret_cast<uint4*>(e)[j] = reinterpret_cast<const uint4*>(p)[j];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = lm::to_f<T>(e[i]);
  }
};

template <typename T>
struct RowView {
  const T* row;
  const uint8_t* mask;
  int v, shift, vectors;
  bool mask_aligned;   // the mask's bytes of a vector lie on an 8-byte boundary
  __device__ __forceinline__ RowView(const Args& a, int64_t r) {
    row = reinterpret_cast<const T*>(a.x) + r * a.ldx;
    mask = a.mask ? a.mask + r * a.ldm : nullptr;
    v = a.v;
    shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    vectors = (v + shift + 7) / 8;
    mask_aligned = mask && ((reinterpret_cast<uintptr_t>(mask) - shift) & 7) == 0;
  }
  // Vectors from..to - 1 lie wholly inside the row and have no masked entries.
  __device__ __forceinline__ int plain_from() const { return shift ? 1 : 0; }
  __device__ __forceinline__ int plain_to() const { return mask ? 0 : (v + shift) / 8; }
  // The entries of vector i and which of them are valid (bit e).
  __device__ __forceinline__ uint32_t load(int i, float (&x)[8]) const {
    const int c0 = 8 * i - shift;
    uint32_t ok = 0xff;
    if (c0 >= 0 && c0 + 8 <= v) {
      lm::load8(row + c0, x);
      if (mask) {
        if (mask_aligned) {
          const uint2 b = *reinterpret_cast<const uint2*>(mask + c0);
          ok = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ok |= (b.x >> 8 * e & 0xff ? 1u : 0u) << e;
            ok |= (b.y >> 8 * e & 0xff ? 1u : 0u) << (e + 4);
          }
        } else {
          ok = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) ok |= (mask[c0 + e] ? 1u : 0u) << e;
        }
      }
    } else {
      ok = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = c0 + e;
        x[e] = 0.f;
        if (c >= 0 && c < v && (!mask || mask[c])) {
          x[e] = lm::to_f<T>(row[c]);
          ok |= 1u << e;
        }
      }
    }
    return ok;
  }
};

// One vector's entries into the running sums.
__device__ __forceinline__ void add_vector(Stat& st, int& first, int i, uint32_t ok, float (&x)[8], float c) {
  if (ok != 0xff) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!(ok >> e & 1)) x[e] = -INFINITY;
  }
  float m = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) m = fmaxf(m, x[e]);
  if (m > st.m) {
    st = rescaled(st, m, c);
    first = i;
  }
  if (st.m != -INFINITY) {
#pragma unroll
    for (int e = 0; e < 8; ++e) add_entry(st, x[e], c);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (x[e] != x[e]) st.s = x[e];   // NaN and nothing else so far: the row is NaN
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same shared variable in the cluster's CTA `rank`.
template <typename V>
__device__ __forceinline__ const V* cluster_peer(const V* p, int rank) {
  uint64_t r;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(p), "r"(rank));
  return reinterpret_cast<const V*>(r);
}

// The `top` largest of `count` different keys, in order, into out (0: none).
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int count, int top, uint64_t* out) {
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const uint64_t key = keys[i];
    if (!key) continue;
    int place = 0;   // the number of keys above it
    for (int j = 0; j < count; ++j) place += keys[j] > key;
    if (place < top) out[place] = key;
  }
}

// A cluster of a.splits CTAs takes one row, each CTA an equal part of its vectors.
template <typename T>
__global__ void __launch_bounds__(kThreads) long_fwd_kernel(const Args a) {
  constexpr int W = kThreads / 32;
  __shared__ Stat red[W], part_s, part_s2;
  __shared__ uint64_t keys[kThreads], cand[kCandidates], found[kMaxTop];
  __shared__ uint64_t bound_s;
  __shared__ int count_s, owners_s;
  __shared__ uint16_t owners[kThreads];
  const int64_t r = blockIdx.x / a.splits;
  const int rank = a.splits > 1 ? (int)cluster_rank() : 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float c = a.inv_t * kLog2e;
  const RowView<T> view(a, r);
  const int share = (view.vectors + a.splits - 1) / a.splits, i0 = rank * share, i1 = min(view.vectors, i0 + share);
  Stat st = empty_stat();
  int first = 0;   // the vector in which this thread's maximum was first met
  int i = i0 + threadIdx.x;
  const int plain0 = view.plain_from(), plain1 = min(i1, view.plain_to());
  if (i < plain0) {   // the row's first vector, where the row starts inside it
    float x[8];
    const uint32_t ok = view.load(i, x);
    add_vector(st, first, i, ok, x, c);
    i += kThreads;
  }
  const T* base = view.row - view.shift;
  for (; i + (kAhead - 1) * kThreads < plain1; i += kAhead * kThreads) {
    Raw<T> raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) raw[j].load(base + 8 * (int64_t)(i + j * kThreads));
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      float x[8];
      raw[j].get(x);
      add_vector(st, first, i + j * kThreads, 0xffu, x, c);
    }
  }
  for (; i < i1; i += kThreads) {
    float x[8];
    const uint32_t ok = view.load(i, x);
    add_vector(st, first, i, ok, x, c);
  }
  // NaN alone: any finite maximum carries it through the joining
  const bool nan_only = st.m == -INFINITY && st.s != st.s;
  Stat mine = nan_only ? Stat{0.f, st.s, st.s} : st;
  mine = group_join<32>(mine, c);
  if (lane == 0) red[warp] = mine;
  if (a.top) {
    keys[threadIdx.x] = st.m == -INFINITY ? 0 : entry_key(st.m, first);
    if (threadIdx.x == 0) count_s = owners_s = 0, bound_s = 0;
    for (int k = threadIdx.x; k < a.top; k += kThreads) found[k] = 0;
  }
  __syncthreads();
  if (warp == 0) {
    const Stat s = group_join<W>(lane < W ? red[lane] : empty_stat(), c);
    if (lane == 0) part_s = s;
  }
  if (a.top) {
    // the top-th largest maximum of groups of threads, at least `top` of them
    int lanes = 32;
    while (kThreads / lanes < a.top) lanes /= 2;
    uint64_t best = keys[threadIdx.x];
    for (int o = lanes / 2; o > 0; o >>= 1) {
      const uint64_t u = __shfl_xor_sync(0xffffffffu, best, o);
      best = u > best ? u : best;
    }
    if (lane % lanes == 0) cand[threadIdx.x / lanes] = best;
    __syncthreads();
    if (threadIdx.x < kThreads / lanes) {
      const uint64_t own = cand[threadIdx.x];
      int place = 0;
      for (int j = 0; j < kThreads / lanes; ++j) place += cand[j] > own;
      if (own && place == a.top - 1) bound_s = own;
    }
    const uint64_t own = keys[threadIdx.x];
    __syncthreads();
    const uint64_t bound = bound_s;   // 0: fewer than `top` groups have an entry, so every entry counts
    if (own && own >= bound) owners[atomicAdd(&owners_s, 1)] = threadIdx.x;
    __syncthreads();
    // the owners' entries at or above the bound: a larger value, or the same value in no later vector
    const int per = (i1 - i0 + kThreads - 1) / kThreads, items = owners_s * per;
    for (int item = threadIdx.x; item < items; item += kThreads) {
      const int v = i0 + owners[item / per] + item % per * kThreads;
      if (v >= i1) continue;
      float x[8];
      const uint32_t ok = view.load(v, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!(ok >> e & 1) || !ranked(x[e])) continue;
        if (entry_key(x[e], v) < bound) continue;
        const int at = atomicAdd(&count_s, 1);
        if (at < kCandidates) cand[at] = entry_key(x[e], 8 * v - view.shift + e);
      }
    }
    __syncthreads();
    const int count = count_s;
    if (count <= kCandidates) {
      rank_keys(cand, count, a.top, found);
    } else {
      // too many for shared memory (many equal or clustered maxima): one pass over the row for each place
      uint64_t last = ~0ull;
      for (int n = 0; n < a.top; ++n) {
        uint64_t best = 0;
        for (int v = i0 + threadIdx.x; v < i1; v += kThreads) {
          float x[8];
          const uint32_t ok = view.load(v, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (!(ok >> e & 1) || !ranked(x[e])) continue;
            const uint64_t key = entry_key(x[e], 8 * v - view.shift + e);
            if (key < last && key > best) best = key;
          }
        }
        best = group_max<32>(best);
        __syncthreads();
        if (lane == 0) cand[warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) best = cand[w] > best ? cand[w] : best;
        last = best;
        if (threadIdx.x == 0) found[n] = best;
      }
    }
  }
  const uint64_t* list = found;
  if (a.splits > 1) {
    __syncthreads();
    cluster_sync();
    if (rank == 0) {
      // join the parts, and rank their lists once more
      if (warp == 0) {
        const Stat s = group_join<kMaxSplits>(lane < a.splits ? *cluster_peer(&part_s, lane) : empty_stat(), c);
        if (lane == 0) part_s2 = s;
      }
      const int n = a.splits * a.top;   // at most 8 x 64
      for (int k = threadIdx.x; k < n; k += kThreads) cand[k] = cluster_peer(found, k / a.top)[k % a.top];
      for (int k = threadIdx.x; k < a.top; k += kThreads) keys[k] = 0;
      __syncthreads();
      rank_keys(cand, n, a.top, keys);
      list = keys;
    }
    __syncthreads();
    cluster_sync();   // the parts stay until they have been read
    if (rank != 0) return;
  }
  __syncthreads();
  const Stat all = a.splits > 1 ? part_s2 : part_s;
  const float logs = threadIdx.x < max(1, a.top) ? log_sum(all) : 0.f;
  for (int k = threadIdx.x; k < a.top; k += kThreads) write_top(a, r, k, list[k], all, logs);
  if (threadIdx.x == 0) {
    const int64_t tok = a.tokens[r];
    float logit = 0.f;
    bool valid = false;
    if (tok >= 0 && tok < a.v) {
      valid = !view.mask || view.mask[tok];
      if (valid) logit = lm::to_f<T>(view.row[tok]);
    }
    write_row(a, r, all, logs, logit, valid);
  }
}

// The gradient: a CTA takes 256 x kBwdVectors vectors of one row.
constexpr int kBwdVectors = 4;

template <typename T>
__global__ void __launch_bounds__(256)
long_bwd_kernel(const Args a, const float* __restrict__ g_lp, const float* __restrict__ g_ent, T* __restrict__ dx,
                int parts) {
  const int64_t r = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - r * parts);
  const RowView<T> view(a, r);
  const float m = a.stats[3 * r], logs = a.stats[3 * r + 1], ent = a.stats[3 * r + 2];
  const int64_t tok = a.tokens[r];
  const float gl = g_lp && tok >= 0 && tok < a.v ? g_lp[r] : 0.f, ge = g_ent ? g_ent[r] : 0.f;
  const bool none = m == -INFINITY;
  T* out = dx + r * a.v;
  const bool same = ((reinterpret_cast<uintptr_t>(out) - view.shift * sizeof(T)) & 15) == 0;
  // d = p (k0 + k1 log p), plus `hot` at the token; without weight 0 times a finite number
  const float k0 = (-gl - ge * ent) * a.inv_t, k1 = -ge * a.inv_t, hot = gl * a.inv_t;
  const auto entry = [&](float x) {
    float lp = fmaf(x - m, a.inv_t, -logs);
    asm("max.NaN.f32 %0, %0, 0fC3480000;" : "+f"(lp));   // -200: the weight is zero from -88 on
    return exp2f(lp * kLog2e) * fmaf(k1, lp, k0);
  };
  const int first = part * kBwdVectors * 256 + threadIdx.x, hot_vector = (int)((tok + view.shift) >> 3);
  if (same && !none && part * kBwdVectors * 256 >= view.plain_from() &&
      (part + 1) * kBwdVectors * 256 <= view.plain_to()) {   // the whole CTA's vectors are plain
    Raw<T> raw[kBwdVectors];
    const T* in = view.row - view.shift;
#pragma unroll
    for (int j = 0; j < kBwdVectors; ++j) raw[j].load(in + 8 * (int64_t)(first + j * 256));
#pragma unroll
    for (int j = 0; j < kBwdVectors; ++j) {
      const int i = first + j * 256;
      float x[8];
      raw[j].get(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = entry(x[e]);
      if (i == hot_vector && hot != 0.f) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * i - view.shift + e == tok) x[e] += hot;
      }
      lm::store8(out + 8 * (int64_t)i - view.shift, x);
    }
    return;
  }
#pragma unroll 1
  for (int j = 0; j < kBwdVectors; ++j) {
    const int i = first + j * 256;
    if (i >= view.vectors) return;
    float x[8];
    const uint32_t ok = view.load(i, x);
    const int c0 = 8 * i - view.shift;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float d = 0.f;
      if (ok >> e & 1 && !none) {
        d = entry(x[e]);
        if (c0 + e == tok) d += hot;
      }
      x[e] = d;
    }
    if (same && c0 >= 0 && c0 + 8 <= a.v) {
      lm::store8(out + c0, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e >= 0 && c0 + e < a.v) out[c0 + e] = lm::from_f<T>(x[e]);
    }
  }
}

template <typename F>
void for_type(torch::ScalarType t, F&& f) {
  if (t == torch::kFloat32) f(float{});
  else if (t == torch::kBFloat16) f(__nv_bfloat16{});
  else f(__half{});
}

// Lanes per row and entries per lane of a short row.
template <typename F>
void for_small(int v, F&& f) {
  auto go = [&](auto g, auto e) { f(g, e); };
  using std::integral_constant;
  if (v <= 8) go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  else if (v <= 32) go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  else if (v <= 128) go(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  else if (v <= 512) go(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  else go(integral_constant<int, 32>{}, integral_constant<int, 32>{});
}

// Logits [rows, V] and mask (bool, or undefined) with contiguous rows.
Args common_args(const torch::Tensor& x, const torch::Tensor& tokens, const torch::Tensor& mask, double temperature) {
  Args a{};
  a.x = x.data_ptr();
  a.rows = x.size(0);
  a.v = (int)x.size(1);
  a.ldx = a.rows > 1 ? x.stride(0) : a.v;
  if (mask.defined()) {
    a.mask = reinterpret_cast<const uint8_t*>(mask.data_ptr());
    a.ldm = a.rows > 1 ? mask.stride(0) : a.v;
  }
  a.tokens = tokens.data_ptr<int64_t>();
  a.inv_t = (float)(1. / temperature);
  return a;
}

struct Results {
  torch::Tensor lp, ent, tv, tt, stats;   // stats only where a backward follows
};

Results forward(const torch::Tensor& x, const torch::Tensor& tokens, const torch::Tensor& mask, double temperature,
                int64_t top, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  Args a = common_args(x, tokens, mask, temperature);
  const auto f32 = x.options().dtype(torch::kFloat32);
  Results r;
  r.lp = torch::empty({a.rows}, f32);
  r.ent = torch::empty({a.rows}, f32);
  r.tv = torch::empty({a.rows, top}, f32);
  r.tt = torch::empty({a.rows, top}, x.options().dtype(torch::kInt64));
  if (keep) r.stats = torch::empty({a.rows, 3}, f32);
  if (a.rows == 0) return r;
  a.top = (int)top;
  a.log_prob = r.lp.data_ptr<float>();
  a.entropy = r.ent.data_ptr<float>();
  a.top_value = r.tv.data_ptr<float>();
  a.top_token = r.tt.data_ptr<int64_t>();
  a.stats = keep ? r.stats.data_ptr<float>() : nullptr;
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  for_type(x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    if (a.v <= kSmall) {
      for_small(a.v, [&](auto g, auto e) {
        constexpr int G = decltype(g)::value, E = decltype(e)::value;
        small_fwd_kernel<T, G, E><<<(unsigned)((a.rows * G + 255) / 256), 256, 0, st>>>(a);
      });
    } else {
      // few rows: as many CTAs for each as give the SMs two, with a vector at least for every thread
      a.splits = 1;
      while (a.splits < kMaxSplits && a.rows * a.splits <= lm::sm_count() && a.v / 8 >= 2 * a.splits * kThreads)
        a.splits *= 2;
      TORCH_CHECK(a.rows * a.splits < (1ll << 31), "token_log_probs: too many rows");
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(a.rows * a.splits));
      cfg.blockDim = dim3(kThreads);
      cfg.stream = st;
      cudaLaunchAttribute attr = {};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = a.splits;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      TORCH_CHECK(cudaLaunchKernelEx(&cfg, long_fwd_kernel<T>, a) == cudaSuccess, "token_log_probs launch failed");
    }
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "token_log_probs launch failed");
  lm::count_launches(1);
  return r;
}

torch::Tensor backward(const torch::Tensor& x, const torch::Tensor& tokens, const torch::Tensor& mask, double temperature,
                       const torch::Tensor& stats, const torch::Tensor& g_lp, const torch::Tensor& g_ent) {
  const c10::cuda::CUDAGuard guard(x.device());
  Args a = common_args(x, tokens, mask, temperature);
  auto dx = torch::empty({a.rows, (int64_t)a.v}, x.options());
  if (a.rows == 0) return dx;
  a.stats = stats.data_ptr<float>();
  const float* gl = g_lp.defined() ? g_lp.data_ptr<float>() : nullptr;
  const float* ge = g_ent.defined() ? g_ent.data_ptr<float>() : nullptr;
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  for_type(x.scalar_type(), [&](auto t) {
    using T = decltype(t);
    T* out = reinterpret_cast<T*>(dx.data_ptr());
    if (a.v <= kSmall) {
      for_small(a.v, [&](auto g, auto e) {
        constexpr int G = decltype(g)::value, E = decltype(e)::value;
        small_bwd_kernel<T, G, E><<<(unsigned)((a.rows * G + 255) / 256), 256, 0, st>>>(a, gl, ge, out);
      });
    } else {
      const int parts = (int)(((int64_t)a.v + 14) / 8 / (256 * kBwdVectors) + 1);   // a row may start inside a vector
      TORCH_CHECK(a.rows * parts < (1ll << 31), "token_log_probs: too many logits");
      long_bwd_kernel<T><<<(unsigned)(a.rows * parts), 256, 0, st>>>(a, gl, ge, out, parts);
    }
  });
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "token_log_probs backward launch failed");
  lm::count_launches(1);
  return dx;
}

// `t` as [rows, V] whose rows are contiguous (a row may be repeated).
torch::Tensor as_rows(const torch::Tensor& t) {
  const int64_t v = t.size(-1);
  const auto y = t.dim() == 2 ? t : t.reshape({t.numel() / v, v});
  return y.numel() == 0 || v == 1 || y.stride(1) == 1 ? y : y.contiguous();
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct TokenLogProbsFn : torch::autograd::Function<TokenLogProbsFn> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logits, const torch::Tensor& tokens,
                               const c10::optional<torch::Tensor>& m, double temperature, int64_t top) {
    at::AutoDispatchBelowADInplaceOrView below;
    const torch::Tensor mask = m ? *m : torch::Tensor();
    const auto x = as_rows(logits);
    const Results r = ::forward(x, tokens, mask, temperature, top, true);
    // saved as the caller's tensors where they are read again, so that a change in place is noticed
    ctx->save_for_backward({x.is_alias_of(logits) ? logits : x, tokens, mask, r.stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["sizes"] = logits.sizes().vec();
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r.tv, r.tt});
    return {r.lp, r.ent, r.tv, r.tt};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "token_log_probs has no second derivative (create_graph)");
    variable_list out(5);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto f32 = [](const torch::Tensor& g) {
      return g.defined() ? g.to(torch::kFloat32).contiguous() : g;
    };
    out[0] = ::backward(as_rows(saved[0]), saved[1], saved[2], ctx->saved_data["temperature"].toDouble(), saved[3],
                        f32(grads[0]), f32(grads[1])).view(ctx->saved_data["sizes"].toIntVector());
    return out;
  }
};

// (log_prob, entropy, top_log_prob, top_token).
py::tuple token_log_probs(torch::Tensor logits, torch::Tensor tokens, c10::optional<torch::Tensor> mask,
                          double temperature, int64_t top) {
  const auto type = logits.scalar_type();
  LM_CHECK_VALUE(logits.is_cuda() && logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) < (1ll << 30) &&
                        (type == torch::kFloat32 || type == torch::kBFloat16 || type == torch::kHalf),
                    "token_log_probs takes fp32, bf16 or fp16 logits [..., V]");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  LM_CHECK_VALUE(tokens.sizes() == lead && tokens.device() == logits.device() &&
                        (tokens.scalar_type() == torch::kInt64 || tokens.scalar_type() == torch::kInt32),
                    "token_log_probs needs integer tokens ", lead, " on ", logits.device());
  LM_CHECK_VALUE(tokens.numel() < (1ll << 31) - 1, "token_log_probs: too many rows");
  // far enough inside fp32's range for 1 / T, and for the difference of any two logits over T to be told from zero
  LM_CHECK_VALUE(temperature >= 1e-30 && temperature <= 1e30, "the temperature must be in 1e-30..1e30, not ", temperature);
  LM_CHECK_VALUE(top >= 0 && top <= kMaxTop, "top must be in 0..", kMaxTop, ", not ", top);
  LM_CHECK_NO_TANGENT("token_log_probs", logits);
  torch::Tensor m, t = tokens;
  if (mask) {
    LM_CHECK_VALUE(mask->scalar_type() == torch::kBool && mask->device() == logits.device(),
                      "the mask must be boolean (true: valid) on the logits' device");
    m = *mask;
    if (m.sizes() != logits.sizes()) {
      LM_CHECK_VALUE(at::is_expandable_to(m.sizes(), logits.sizes()), "the mask ", m.sizes(),
                        " does not broadcast to ", logits.sizes());
      m = m.expand(logits.sizes());
    }
    m = as_rows(m);
  }
  if (t.dim() != 1) t = t.reshape({t.numel()});
  if (t.scalar_type() != torch::kInt64) t = t.to(torch::kInt64);
  t = t.contiguous();
  Results r;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const auto o = TokenLogProbsFn::apply(logits, t, mask ? c10::optional<torch::Tensor>(m) : c10::nullopt, temperature, top);
    r = Results{o[0], o[1], o[2], o[3], {}};
  } else {
    r = forward(as_rows(logits), t, m, temperature, top, false);
  }
  if (lead.size() == 1) return py::make_tuple(r.lp, r.ent, r.tv, r.tt);
  auto sizes = lead.vec();
  const auto lp = r.lp.view(sizes), ent = r.ent.view(sizes);
  sizes.push_back(top);
  return py::make_tuple(lp, ent, r.tv.view(sizes), r.tt.view(sizes));
}

}  // namespace

void register_token_logprobs_ops(py::module& m) {
  m.def("token_log_probs", &token_log_probs,
        "log-probabilities of given tokens, with autograd: (log_prob, entropy, top_log_prob, top_token)",
        py::arg("logits"), py::arg("tokens"), py::arg("mask"), py::arg("temperature"), py::arg("top"));
}
