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
// Three kernels, chosen by the sizes (matmul() below): this one for as many 128
// x 128 tiles as the SMs hold at once, one for few rows and one by pairs of
// CTAs for more. A CTA has one tile, or, in a cluster, a part of one tile's
// groups; 320 threads:
//   warp 0     TMA producer: the 128-byte wide A and B tiles of each group into
//              a shared-memory ring;
//   warp 1     allocates TMEM; one lane issues the four K = 32 products of a
//              group into the next buffer and commits them to one barrier, on
//              which the producer waits for the stage and the epilogue for the
//              buffer (there are more stages than buffers, so neither can be
//              a whole round behind);
//   warps 2-9  two per TMEM lane quadrant: thread = one row, half the columns.
// Waits are bounded and reported as in the bf16 GEMM (tc_gemm.cu), with the
// same status bits; whichever wait runs out, the producer sees its loads land and
// the product thread its last products complete before the CTA gives up its
// shared memory and TMEM.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

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
  int splits;             // CTAs of a cluster that share one tile's groups (1: none do); 16 bits: parts of the rows
  int64_t part;           // 16 bits: elements between the results of two parts
  int half;               // 16 bits: fp16 operands, not bf16
  int* status;
  uint64_t wait_ns;
};

// A place in a ring of N slots and the parity of its current round.
template <int N> struct Ring {
  uint32_t slot = 0, round = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) slot = 0, round ^= 1;
  }
};

// 128 x 128 tiles: the ring, the epilogue's stores and the barriers; TMEM has 512 columns.
constexpr int kBN = 128, kStages = 6, kBuffers = 512 / kBN;
constexpr uint32_t kTileA = kBM * kGroup, kTileStage = kTileA + kBN * kGroup;
constexpr uint32_t kSmem = kStages * kTileStage + kEpiWarps * 4096 + 1024 + 256;

// The sums of a CTA's rows over one group: acc += sc * TMEM, `CHUNKS` times 32
// columns from `base`. Two chunks are loaded at a time, and the next ones into
// the registers of those that are added already. The buffer is handed back
// (release()) once its last chunks are in registers.
template <int CHUNKS, typename F>
__device__ __forceinline__ void add_group(uint32_t base, float sc, float (&acc)[CHUNKS][32], F&& release) {
  static_assert(CHUNKS % 2 == 0, "chunks are loaded in pairs");
  float v[2][32];
  tc::tmem_ld32_issue(base, v[0]);
  tc::tmem_ld32_issue(base + 32, v[1]);
#pragma unroll
  for (int c = 0; c < CHUNKS; c += 2) {
    tc::tmem_ld_wait();
    tc::tmem_regs_ready(v[0]);
    tc::tmem_regs_ready(v[1]);
    if (c + 2 >= CHUNKS) release();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 32; ++i) acc[c + j][i] = fmaf(v[j][i], sc, acc[c + j][i]);
      if (c + 2 < CHUNKS) tc::tmem_ld32_issue(base + 32 * (c + 2 + j), v[j]);
    }
  }
}

// The scales of one row of A and one row block of B, loaded four groups ahead
// and multiplied only when they are used: a load has four groups' time to
// arrive. A row's scales come as one load of four or two of two where its
// length and start are multiples of that: the lanes' rows lie apart, and with
// single loads their accesses took 150 cycles of a group's 1190.
struct Scales {
  const float* a;
  const float* b;
  int groups, width;
  float cur[4], na[4], nb[4];
  __device__ __forceinline__ void load(int kb) {
    if (width == 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(a + kb));
      na[0] = v.x, na[1] = v.y, na[2] = v.z, na[3] = v.w;
    } else if (width == 2) {
      const float2 v = __ldg(reinterpret_cast<const float2*>(a + kb));
      const float2 u = __ldg(reinterpret_cast<const float2*>(a + min(kb + 2, groups - 2)));
      na[0] = v.x, na[1] = v.y, na[2] = u.x, na[3] = u.y;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) na[j] = __ldg(a + min(kb + j, groups - 1));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) nb[j] = __ldg(b + min(kb + j, groups - 1));
  }
  // `stride`: groups of a whole row; `groups`: of the part that starts at pa.
  __device__ __forceinline__ Scales(const float* pa, const float* pb, int g, int stride) : a(pa), b(pb), groups(g) {
    const int bits = stride | g | (int)(reinterpret_cast<uintptr_t>(pa) >> 2);
    width = bits & 1 ? 1 : (bits & 2 ? 2 : 4);
    if (a && g > 0) load(0);
  }
  // Call for kb = 0, 1, 2, ...
  __device__ __forceinline__ float at(int kb) {
    if ((kb & 3) == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) cur[j] = na[j] * nb[j];
      if (kb + 4 < groups) load(kb + 4);
    }
    const float lo = kb & 1 ? cur[1] : cur[0], hi = kb & 1 ? cur[3] : cur[2];
    return kb & 2 ? hi : lo;
  }
};

// The store of 32 columns of a warp's 32 rows, one row a lane. Full columns of
// aligned rows go through `stage` (4 KB of the warp's own), from where
// neighbouring lanes write neighbouring 16 bytes of a row; with each lane
// writing its own row a 128 x 256 tile took twice as long to store. 16-byte
// pieces of a row are swapped by its number, so that neither side's accesses
// share banks.
template <typename T>
__device__ __forceinline__ void store32(const Args& g, const float (&v)[32], int row0, int col, uint8_t* stage) {
  constexpr int kPieces = 32 * sizeof(T) / 16, kShift = sizeof(T) == 4 ? 0 : 1, kRows = 32 / kPieces;
  const int lane = threadIdx.x & 31, n = g.N - col;
  T* c = reinterpret_cast<T*>(g.c);
  if (n >= 32 && g.ldc % 8 == 0) {   // the output's base is 16-byte aligned (host)
    uint4* s = reinterpret_cast<uint4*>(stage);
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      alignas(16) T e[16 / sizeof(T)];
#pragma unroll
      for (int i = 0; i < (int)(16 / sizeof(T)); ++i) e[i] = lm::from_f<T>(v[p * (16 / sizeof(T)) + i]);
      s[lane * kPieces + (p ^ ((lane >> kShift) & (kPieces - 1)))] = *reinterpret_cast<const uint4*>(e);
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int r = k * kRows + lane / kPieces, p = lane % kPieces;
      if (row0 + r < g.M)
        *reinterpret_cast<uint4*>(c + (int64_t)(row0 + r) * g.ldc + col + p * (16 / sizeof(T))) =
            s[r * kPieces + (p ^ ((r >> kShift) & (kPieces - 1)))];
    }
    __syncwarp();
  } else if (row0 + lane < g.M) {
    T* dst = c + (int64_t)(row0 + lane) * g.ldc + col;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) dst[i] = lm::from_f<T>(v[i]);
  }
}

// bias and the store of `acc`, `CHUNKS` times 32 columns from n0 of the warp's rows.
constexpr uint32_t kStoreStage = 4096;
template <int CHUNKS>
__device__ __forceinline__ void store_rows(const Args& g, float (&acc)[CHUNKS][32], int row0, int n0, uint8_t* stage) {
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int col = n0 + 32 * c, n = g.N - col;
    if (n <= 0) break;
    if (g.bias) {
#pragma unroll
      for (int i = 0; i < 32; ++i) acc[c][i] += i < n ? __ldg(g.bias + col + i) : 0.f;
    }
    if (g.out_kind == 0) store32<float>(g, acc[c], row0, col, stage);
    else if (g.out_kind == 1) store32<__nv_bfloat16>(g, acc[c], row0, col, stage);
    else store32<__half>(g, acc[c], row0, col, stage);
  }
}

// An epilogue warp: TMEM lanes 32 q .. + 31 and half of the tile's COLS columns,
// which lie inside one block of 128 rows of B. `walk` calls tile(first row,
// first column, first group, last group) for one of the CTA's tiles after the
// other; sink(sums, row, first column) gets each tile's sums. `tempty0` may
// lie in another CTA (a mapped address).
template <int STAGES, int BUFFERS, int COLS, bool SCALED = true, typename F, typename S>
__device__ __forceinline__ void epilogue(const Args& g, uint32_t tmem, uint32_t done0, uint32_t tempty0,
                                         int q, int half, F&& walk, S&& sink) {
  constexpr int kChunks = COLS / 64;   // 32-column chunks per warp
  const int lane = threadIdx.x & 31, G = g.groups;
  const uint32_t lanes = tmem + half * (COLS / 2) + ((uint32_t)(32 * q) << 16);
  Ring<STAGES> st;
  Ring<BUFFERS> buf;
  walk([&](int m0, int n0, int kb0, int kb1) {
    const int row = m0 + 32 * q + lane;
    n0 += half * (COLS / 2);
    float acc[kChunks][32];
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 32; ++i) acc[c][i] = 0.f;
    Scales sc(SCALED ? g.a_scale + (int64_t)min(row, g.M - 1) * G + kb0 : nullptr,
              SCALED ? g.b_scale + (int64_t)min(n0 / kGroup, (g.N - 1) / kGroup) * G + kb0 : nullptr, kb1 - kb0, G);
    for (int kb = kb0; kb < kb1; ++kb) {
      const float scale = SCALED ? sc.at(kb - kb0) : 1.f;
      const bool got = tc::mbar_wait(done0 + 8 * st.slot, st.round, g.wait_ns);
      if (!__all_sync(0xffffffffu, got)) {   // the loads below are whole-warp
        atomicOr(g.status, 4);
        return false;
      }
      tc::tc_fence_after();
      add_group<kChunks>(lanes + buf.slot * COLS, scale, acc, [&] {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tempty0 + 8 * buf.slot);
      });
      st.next();
      buf.next();
    }
    sink(acc, row, n0);
    return true;
  });
}

// ---- tiles whose groups are shared by a cluster --------------------------------
// Few tiles leave most SMs idle, so the CTAs of a cluster take a part of one
// tile's groups each, leave their sums in shared memory, and after a cluster
// barrier each adds up, in the order of the ranks, an equal part of the rows.
constexpr int kMaxSplits = 8;

__device__ __forceinline__ float4 load_cluster(uint32_t mapped) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapped) : "memory");
  return v;
}

// Row strides of the sums in shared memory: 16 bytes more than the row, so that
// the lanes' 16-byte accesses of neighbouring rows fall on different banks.
__host__ __device__ constexpr int sum_stride(int cols) { return cols + 4; }

template <int CHUNKS>
__device__ __forceinline__ void keep_sums(float* sums, int stride, const float (&acc)[CHUNKS][32], int row, int col) {
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      *reinterpret_cast<float4*>(sums + row * stride + col + 32 * c + i) =
          make_float4(acc[c][i], acc[c][i + 1], acc[c][i + 2], acc[c][i + 3]);
}

// Sums of four columns of one row over the cluster's CTAs.
__device__ __forceinline__ float4 cluster_sum(uint32_t sums, int stride, int splits, int row, int col) {
  const uint32_t at = sums + 4 * (row * stride + col);
  float4 s = load_cluster(tc::cluster_map(at, 0));
  for (int r = 1; r < splits; ++r) {
    const float4 v = load_cluster(tc::cluster_map(at, r));
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  return s;
}

__device__ __forceinline__ void store_one(const Args& g, int row, int col, float v) {
  if (g.bias) v += g.bias[col];
  const int64_t off = (int64_t)row * g.ldc + col;
  if (g.out_kind == 0) reinterpret_cast<float*>(g.c)[off] = v;
  else if (g.out_kind == 1) reinterpret_cast<__nv_bfloat16*>(g.c)[off] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(g.c)[off] = __float2half_rn(v);
}

// Where the second CTA of a pair leaves, in the first, the number of groups whose tiles it has asked for.
struct PairLink {
  uint32_t rank;
  uint32_t* issued;   // of the second CTA
  uint32_t through;   // barrier: it asks for no more
};

// The producer's thread: `walk` calls load(k, row of A, row of B) for one
// group's tiles after the other, until it answers false. Before it returns,
// every load has landed and the products of every stage are complete: the
// CTA's shared memory must not be given away before.
//
// In a pair both CTAs' loads complete on the first CTA's barriers, each round
// armed by both, and the first CTA sees to the landing of all of them (neither
// ends before the other). Where a wait ran out, one CTA may have armed up to a
// ring's rounds that the other has not: the first CTA arms those in its place.
template <int STAGES, bool PAIR = false, bool WIDE = false, typename F>
__device__ __forceinline__ void produce(const Args& g, const CUtensorMap* ta, const CUtensorMap* tb, uint32_t smem0,
                                        uint32_t stage_bytes, uint32_t a_bytes, uint32_t full0, uint32_t done0,
                                        const PairLink& link, F&& walk) {
  static_assert(PAIR || !WIDE, "16-bit tiles are the pairs' alone");
  const uint32_t armed0 = PAIR ? tc::cluster_map(full0, 0) : full0;
  const auto tile = [](uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (PAIR) tc::tma_load_2d_pair(dst, map, x, y, bar);
    else tc::tma_load_2d(dst, map, x, y, bar);
  };
  Ring<STAGES> st;
  uint32_t issued = 0;
  bool ok = true;
  walk([&](int k, int row_a, int row_b) {
    if (issued >= STAGES && !tc::mbar_wait(done0 + 8 * st.slot, st.round ^ 1, g.wait_ns)) {
      atomicOr(g.status, 1);
      return ok = false;
    }
    const uint32_t sa = smem0 + st.slot * stage_bytes, full = armed0 + 8 * st.slot;
    if constexpr (PAIR) tc::mbar_arrive_expect_tx_cluster(full, stage_bytes);
    else tc::mbar_arrive_expect_tx(full, stage_bytes);
    if constexpr (WIDE) {   // 64 rows by 128 columns, as two boxes of 64 columns
      tile(sa, ta, row_a, k, full);
      tile(sa + 8192, ta, row_a + 64, k, full);
      tile(sa + a_bytes, tb, row_b, k, full);
      tile(sa + a_bytes + 8192, tb, row_b + 64, k, full);
    } else {
      tile(sa, ta, k, row_a, full);
      tile(sa + a_bytes, tb, k, row_b, full);
    }
    st.next();
    ++issued;
    return true;
  });
  if (PAIR && link.rank == 1) {
    tc::publish_cluster(tc::cluster_map(tc::smem_u32(link.issued), 0), issued, tc::cluster_map(link.through, 0));
    return;
  }
  for (uint32_t i = issued > (uint32_t)STAGES ? issued - STAGES : 0u; ok && i < issued; ++i)
    if (!tc::mbar_wait(done0 + 8 * (i % STAGES), (i / STAGES) & 1, g.wait_ns)) {
      atomicOr(g.status, 1);
      ok = false;
    }
  if (ok) return;
  uint32_t end = issued;   // of the groups that have been asked for
  if constexpr (PAIR) {
    if (!tc::mbar_wait_cluster(link.through, 0, g.wait_ns + kDrainNs)) atomicOr(g.status, 16);
    const uint32_t other = *(volatile uint32_t*)link.issued;
    end = max(issued, other);
    for (uint32_t i = min(issued, other); i < end; ++i) tc::mbar_arrive(full0 + 8 * (i % STAGES));
  }
  for (uint32_t i = end > (uint32_t)STAGES ? end - STAGES : 0u; i < end; ++i)
    if (!tc::mbar_wait(full0 + 8 * (i % STAGES), (i / STAGES) & 1, kDrainNs)) atomicOr(g.status, 16);
}

// The product thread: for each of `count` groups, once its tiles are loaded (in
// both CTAs of a pair) and the TMEM buffer is read out, issue its four products
// and one commit, for the producer and the epilogue alike. Products take 48
// cycles to issue, commits 59 and successful waits 40, one after the other, so
// the next group's barriers are looked at between the products. Before it
// returns, its last products are complete.
template <int STAGES, int BUFFERS, int COLS, bool PAIR, bool WIDE = false>
__device__ __forceinline__ void multiply(const Args& g, uint32_t count, uint32_t smem0, uint32_t stage_bytes,
                                         uint32_t a_bytes, uint32_t tmem, uint32_t full0,
                                         uint32_t done0, uint32_t tempty0) {
  static_assert(!WIDE || PAIR, "16-bit tiles are the pairs' alone");
  uint32_t id = tc::idesc_e4m3(PAIR ? 256 : 128, COLS);
  if (WIDE) id = g.half ? tc::idesc_f16(256, COLS, true, true) : tc::idesc_bf16(256, COLS, true, true);
  const uint32_t lo = WIDE ? tc::mnmajor64_desc_lo(smem0) : tc::kmajor_desc_lo(smem0);
  Ring<STAGES> st, last;
  Ring<BUFFERS> buf;
  uint32_t issued = 0;
  bool loaded = false, read = true;   // the buffers' first round needs no waiting
  for (uint32_t it = 0; it < count; ++it) {
    if (!read && !tc::mbar_wait(tempty0 + 8 * buf.slot, buf.round ^ 1, g.wait_ns)) {
      atomicOr(g.status, 8);
      break;
    }
    if (!loaded && !tc::mbar_wait(full0 + 8 * st.slot, st.round, g.wait_ns)) {
      atomicOr(g.status, 2);
      break;
    }
    tc::tc_fence_after();
    const uint32_t la = lo + st.slot * (stage_bytes >> 4), lb = la + (a_bytes >> 4), d = tmem + buf.slot * COLS;
    const uint32_t done = done0 + 8 * st.slot;
    last = st;
    ++issued;
    st.next();
    buf.next();
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if constexpr (WIDE)
        tc::mma_16bit_pair(d, tc::kmajor_desc(la + 128 * ks), tc::kmajor_desc(lb + 128 * ks), id, ks > 0);
      else if constexpr (PAIR) tc::mma_e4m3_pair(d, tc::kmajor_desc(la + 2 * ks), tc::kmajor_desc(lb + 2 * ks), id, ks > 0);
      else tc::mma_e4m3(d, tc::kmajor_desc(la + 2 * ks), tc::kmajor_desc(lb + 2 * ks), id, ks > 0);
      if (ks == 1) {
        read = it + 1 < (uint32_t)BUFFERS || tc::mbar_try_wait(tempty0 + 8 * buf.slot, buf.round ^ 1);
        loaded = tc::mbar_try_wait(full0 + 8 * st.slot, st.round);
      }
    }
    if constexpr (PAIR) tc::mma_commit_pair(done);
    else tc::mma_commit(done);
  }
  // The last commit covers all products: whoever's wait has run out or runs out yet, they are through with shared
  // memory and TMEM before the CTA gives those up.
  if (issued && !tc::mbar_wait(done0 + 8 * last.slot, last.round, kDrainNs)) atomicOr(g.status, 32);
}

__global__ void __launch_bounds__(kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stage0 = smem + kStages * kTileStage;
  uint8_t* misc = stage0 + kEpiWarps * kStoreStage;
  const uint32_t full0 = tc::smem_u32(misc);             // stage loaded
  const uint32_t done0 = full0 + 8 * kStages;            // stage's products complete
  const uint32_t tempty0 = done0 + 8 * kStages;          // TMEM buffer read out
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(misc + 8 * (2 * kStages + kBuffers));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tc::tma_prefetch_map(&ta);
    tc::tma_prefetch_map(&tb);
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(full0 + 8 * s, 1);
      tc::mbar_init(done0 + 8 * s, 1);
    }
    for (int b = 0; b < kBuffers; ++b) tc::mbar_init(tempty0 + 8 * b, kEpiWarps);   // one lane of every epilogue warp
    tc::mbar_init_fence();
  }
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_u32(s_tmem), 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *s_tmem, smem0 = tc::smem_u32(smem);

  // this CTA's tile, and its part of the tile's groups
  const int tiles_n = (g.N + kBN - 1) / kBN, G = g.groups;
  const int splits = g.splits, rank = splits > 1 ? (int)tc::cluster_rank() : 0, tile = blockIdx.x / splits;
  const int m0 = (tile / tiles_n) * kBM, n0 = (tile % tiles_n) * kBN;
  const int part = (G + splits - 1) / splits, kb0 = min(G, rank * part), kb1 = min(G, kb0 + part);
  float* sums = reinterpret_cast<float*>(smem);   // the stages, once the part of a shared tile is done
  constexpr int kStride = sum_stride(kBN);
  static_assert(kBM * kStride * 4 <= kStages * kTileStage, "the sums take the stages' place");

  if (warp == 0 && lane == 0) {
    produce<kStages>(g, &ta, &tb, smem0, kTileStage, kTileA, full0, done0, PairLink{}, [&](auto&& load) {
      for (int kb = kb0; kb < kb1; ++kb)
        if (!load(kb * kGroup, m0, n0)) return;
    });
  } else if (warp == 1 && lane == 0) {
    multiply<kStages, kBuffers, kBN, false>(g, kb1 - kb0, smem0, kTileStage, kTileA, tmem, full0, done0, tempty0);
  } else if (warp >= 2) {
    const int q = warp & 3, half = (warp - 2) >> 2;
    epilogue<kStages, kBuffers, kBN>(
        g, tmem, done0, tempty0, q, half, [&](auto&& sum) { sum(m0, n0, kb0, kb1); },
        [&](auto& acc, int row, int col) {
          if (splits > 1) keep_sums<kBN / 64>(sums, kStride, acc, 32 * q + lane, half * (kBN / 2));
          else store_rows<kBN / 64>(g, acc, row - lane, col, stage0 + (warp - 2) * kStoreStage);
        });
  }
  if (splits > 1) {
    __syncwarp();
    tc::cluster_sync();
    const int rows = kBM / splits;
    for (int e = threadIdx.x; e < rows * (kBN / 4); e += kThreads) {
      const int r = rank * rows + e / (kBN / 4), c = (e % (kBN / 4)) * 4;
      if (m0 + r >= g.M || n0 + c >= g.N) continue;
      const float4 v = cluster_sum(smem0, kStride, splits, r, c);
      store_one(g, m0 + r, n0 + c, v.x);
      if (n0 + c + 1 < g.N) store_one(g, m0 + r, n0 + c + 1, v.y);
      if (n0 + c + 2 < g.N) store_one(g, m0 + r, n0 + c + 2, v.z);
      if (n0 + c + 3 < g.N) store_one(g, m0 + r, n0 + c + 3, v.w);
    }
    __syncwarp();
    tc::cluster_sync();   // the sums stay until every CTA has read them
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// ---- few rows --------------------------------------------------------------------
// Up to 32 rows of A: bound by reading B. The operands change places, 128 rows
// of B against COLS = 16 or 32 rows of A, so that no tensor work is spent
// on rows that are not there, and a cluster shares a tile's groups. A thread's
// sums are one row of B against all rows of A, with a scale for each: the
// products of the scales of the CTA's groups lie in shared memory.
//   warp 0  producer, warp 1  products (as above), warps 2-5  epilogue
constexpr int kRowsThreads = 192, kRowsStages = 8, kRowsBuffers = 4, kRowsScales = 8192;
template <int COLS> __host__ __device__ constexpr uint32_t rows_stage_bytes() { return kBM * kGroup + COLS * kGroup; }
template <int COLS> __host__ __device__ constexpr uint32_t rows_smem_bytes() {
  return kRowsStages * rows_stage_bytes<COLS>() + 1024 + 256 + 4 * kRowsScales;
}

template <int COLS>
__global__ void __launch_bounds__(kRowsThreads, 1)
fp8_gemm_rows_kernel(const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap ta, const Args g) {
  constexpr uint32_t kStage = rows_stage_bytes<COLS>();
  constexpr int kStride = sum_stride(COLS), kTmem = kRowsBuffers * COLS;
  static_assert(kBM * kStride * 4 <= kRowsStages * kStage, "the sums take the stages' place");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scales = reinterpret_cast<float*>(smem + kRowsStages * kStage);   // [group][COLS]
  uint8_t* misc = reinterpret_cast<uint8_t*>(scales + kRowsScales);
  const uint32_t full0 = tc::smem_u32(misc), done0 = full0 + 8 * kRowsStages, tempty0 = done0 + 8 * kRowsStages;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(misc + 8 * (2 * kRowsStages + kRowsBuffers));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = g.groups;
  const int splits = g.splits, rank = splits > 1 ? (int)tc::cluster_rank() : 0, n0 = (blockIdx.x / splits) * kBM;
  const int part = (G + splits - 1) / splits, kb0 = min(G, rank * part), kb1 = min(G, kb0 + part);

  if (threadIdx.x == 0) {
    tc::tma_prefetch_map(&ta);
    tc::tma_prefetch_map(&tb);
    for (int s = 0; s < kRowsStages; ++s) {
      tc::mbar_init(full0 + 8 * s, 1);
      tc::mbar_init(done0 + 8 * s, 1);
    }
    for (int b = 0; b < kRowsBuffers; ++b) tc::mbar_init(tempty0 + 8 * b, 4);
    tc::mbar_init_fence();
  }
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_u32(s_tmem), kTmem);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *s_tmem, smem0 = tc::smem_u32(smem);
  float* sums = reinterpret_cast<float*>(smem);

  if (warp == 0 && lane == 0) {
    produce<kRowsStages>(g, &tb, &ta, smem0, kStage, kBM * kGroup, full0, done0, PairLink{}, [&](auto&& load) {
      for (int kb = kb0; kb < kb1; ++kb)
        if (!load(kb * kGroup, n0, 0)) return;
    });
  } else if (warp == 1 && lane == 0) {
    multiply<kRowsStages, kRowsBuffers, COLS, false>(g, kb1 - kb0, smem0, kStage, kBM * kGroup, tmem, full0, done0,
                                                     tempty0);
  } else if (warp >= 2) {
    const int q = warp & 3;
    const float* bs = g.b_scale + (int64_t)(n0 / kGroup) * G;
    for (int e = threadIdx.x - 64; e < (kb1 - kb0) * COLS; e += 128) {
      // neighbouring threads read neighbouring groups of one row
      const int j = e / (kb1 - kb0), kb = kb0 + e - j * (kb1 - kb0);
      scales[(kb - kb0) * COLS + j] = j < g.M ? g.a_scale[(int64_t)j * G + kb] * bs[kb] : 0.f;
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");   // the four epilogue warps
    float acc[COLS / 16][16];
#pragma unroll
    for (int c = 0; c < COLS / 16; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][i] = 0.f;
    Ring<kRowsStages> st;
    Ring<kRowsBuffers> buf;
    for (int kb = kb0; kb < kb1; ++kb) {
      const bool got = tc::mbar_wait(done0 + 8 * st.slot, st.round, g.wait_ns);
      if (!__all_sync(0xffffffffu, got)) {
        atomicOr(g.status, 4);
        break;
      }
      tc::tc_fence_after();
      const uint32_t base = tmem + buf.slot * COLS + ((uint32_t)(32 * q) << 16);
      const float4* sc = reinterpret_cast<const float4*>(scales + (kb - kb0) * COLS);
      float v[COLS / 16][16];
#pragma unroll
      for (int c = 0; c < COLS / 16; ++c) tc::tmem_ld16_issue(base + 16 * c, v[c]);
      tc::tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < COLS / 16; ++c) tc::tmem_regs_ready16(v[c]);
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(tempty0 + 8 * buf.slot);
#pragma unroll
      for (int c = 0; c < COLS / 16; ++c)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 f = sc[c * 4 + i / 4];
          acc[c][i] = fmaf(v[c][i], f.x, acc[c][i]);
          acc[c][i + 1] = fmaf(v[c][i + 1], f.y, acc[c][i + 1]);
          acc[c][i + 2] = fmaf(v[c][i + 2], f.z, acc[c][i + 2]);
          acc[c][i + 3] = fmaf(v[c][i + 3], f.w, acc[c][i + 3]);
        }
      st.next();
      buf.next();
    }
    // every stage is read by now: the sums take the stages' place
#pragma unroll
    for (int c = 0; c < COLS / 16; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(sums + (32 * q + lane) * kStride + 16 * c + i) =
            make_float4(acc[c][i], acc[c][i + 1], acc[c][i + 2], acc[c][i + 3]);
  }
  __syncwarp();
  tc::cluster_sync();
  const int rows = kBM / splits, quads = (min(g.M, COLS) + 3) / 4;
  for (int e = threadIdx.x; e < rows * quads; e += kRowsThreads) {
    const int r = rank * rows + e % rows, m = (e / rows) * 4;   // neighbouring threads: neighbouring columns of C
    if (n0 + r >= g.N) continue;
    const float4 v = cluster_sum(smem0, kStride, splits, r, m);
    store_one(g, m, n0 + r, v.x);
    if (m + 1 < g.M) store_one(g, m + 1, n0 + r, v.y);
    if (m + 2 < g.M) store_one(g, m + 2, n0 + r, v.z);
    if (m + 3 < g.M) store_one(g, m + 3, n0 + r, v.w);
  }
  __syncwarp();
  tc::tc_fence_before();
  tc::cluster_sync();   // the sums stay until every CTA has read them
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmem);
  }
}

// ---- 256 x 256 tiles by pairs of CTAs ------------------------------------------
// Each CTA loads 128 rows of A and 128 rows of B a group and keeps 128 x 256
// sums; the pair's tensor cores share B, so that shared memory moves 64 KB per
// 128 x 256 x 128 products instead of 96 KB for one CTA with such a tile, or
// 128 KB with two of 128 x 128.
//   warp 0      producer of the CTA's own tiles, into its own ring;
//   warp 1      first CTA: issues the pair's products once both CTAs' tiles are
//               there, for which it waits on one barrier of its own, as the
//               loads of both complete on that;
//   warps 4-11  epilogue, as above; warps 2 and 3 only complete the warpgroup
//               that gives up its registers to the epilogue's 128 sums a thread.
// The first CTA waits for the loads of both before it ends, and both meet at a
// cluster barrier before either frees its TMEM or shared memory.
constexpr int kPairThreads = 384, kPairStages = 6, kPairBuffers = 2;
constexpr uint32_t kPairTile = 128 * kGroup, kPairStage = 2 * kPairTile;
constexpr uint32_t kPairSmem = kPairStages * kPairStage + kEpiWarps * kStoreStage + 1024 + 256;

// WIDE: the weight gradient's product instead, C = A^T B in fp32 of A [K,M]
// and B [K,N] in bf16 or fp16. A stage holds 64 rows of both (as many bytes), read down
// their columns by the tensor cores, and without scales the epilogue adds up
// every 64 rows in fp32 with round-to-nearest, which the tensor cores' own long
// sums do not; g.splits parts of the rows give as many partial results, `part`
// elements apart.
template <bool WIDE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
gemm_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stage0 = smem + kPairStages * kPairStage;
  uint8_t* misc = stage0 + kEpiWarps * kStoreStage;
  const uint32_t full0 = tc::smem_u32(misc);                  // first CTA: both CTAs' tiles loaded
  const uint32_t done0 = full0 + 8 * kPairStages;             // stage's products complete
  const uint32_t tempty0 = done0 + 8 * kPairStages;           // first CTA: TMEM buffer read out by both
  const uint32_t through = tempty0 + 8 * kPairBuffers;         // first CTA: the second one's producer is through
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(misc + 8 * (2 * kPairStages + kPairBuffers + 1));
  uint32_t* s_issued = s_tmem + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles_n = (g.N + 255) / 256, tiles_m = (g.M + 255) / 256;
  const int tiles = tiles_n * tiles_m, splits = WIDE ? g.splits : 1, total = tiles * splits, G = g.groups;
  const int share = (G + splits - 1) / splits;                // groups of a part of the rows
  const auto range = [&](int w) {
    const int kb0 = WIDE ? w / tiles * share : 0;
    return make_int2(min(G, kb0), min(G, kb0 + share));
  };
  uint32_t count = 0;                                         // of this pair's groups
  for (int w = pair; w < total; w += pairs) count += range(w).y - range(w).x;

  if (threadIdx.x == 0) {
    tc::tma_prefetch_map(&ta);
    tc::tma_prefetch_map(&tb);
    for (int s = 0; s < kPairStages; ++s) {
      tc::mbar_init(full0 + 8 * s, 2);   // both producers
      tc::mbar_init(done0 + 8 * s, 1);
    }
    for (int b = 0; b < kPairBuffers; ++b)
      tc::mbar_init(tempty0 + 8 * b, 2 * kEpiWarps);   // one lane of every epilogue warp of both CTAs
    tc::mbar_init(through, 1);
    tc::mbar_init_fence();
    *s_issued = 0;
  }
  if (warp == 1) {
    tc::tmem_alloc_pair(tc::smem_u32(s_tmem), 512);
    tc::tmem_relinquish_pair();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = *s_tmem, smem0 = tc::smem_u32(smem);

  if (warp < 4) {
    tc::regs_dec<40>();
    if (warp == 0 && lane == 0) {
      const PairLink link{rank, s_issued, through};
      produce<kPairStages, true, WIDE>(g, &ta, &tb, smem0, kPairStage, kPairTile, full0, done0, link, [&](auto&& load) {
        for (int w = pair; w < total; w += pairs) {
          const int2 kb = range(w);
          const int m0 = (w % tiles / tiles_n) * 256 + (int)rank * 128, n0 = (w % tiles_n) * 256 + (int)rank * 128;
          for (int k = kb.x; k < kb.y; ++k)
            if (!load(k * (WIDE ? 64 : kGroup), m0, n0)) return;
        }
      });
    } else if (warp == 1 && lane == 0 && rank == 0) {
      multiply<kPairStages, kPairBuffers, 256, true, WIDE>(g, count, smem0, kPairStage, kPairTile, tmem, full0, done0,
                                                           tempty0);
    }
    __syncwarp();
  } else {
    tc::regs_inc<216>();
    Args out = g;
    epilogue<kPairStages, kPairBuffers, 256, !WIDE>(
        g, tmem, done0, tc::cluster_map(tempty0, 0), warp & 3, (warp - 4) >> 2,
        [&](auto&& tile) {
          for (int w = pair; w < total; w += pairs) {
            const int2 kb = range(w);
            if (WIDE) out.c = reinterpret_cast<float*>(g.c) + (int64_t)(w / tiles) * g.part;
            if (!tile((w % tiles / tiles_n) * 256 + (int)rank * 128, (w % tiles_n) * 256, kb.x, kb.y)) return;
          }
        },
        [&](auto& acc, int row, int n0) {
          store_rows<4>(out, acc, row - lane, n0, stage0 + (warp - 4) * kStoreStage);
        });
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc_pair(tmem, 512);
  }
}

// out = sum of `splits` slices of `count` elements, in their order.
template <typename T>
__global__ void __launch_bounds__(256)
sum_slices_kernel(const float* __restrict__ parts, int splits, int64_t count, T* __restrict__ out) {
  const int64_t step = (int64_t)gridDim.x * 1024;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += step) {
    if (i + 4 <= count && count % 4 == 0) {
      float4 s = *reinterpret_cast<const float4*>(parts + i);
      for (int k = 1; k < splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(parts + k * count + i);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      out[i] = lm::from_f<T>(s.x), out[i + 1] = lm::from_f<T>(s.y);
      out[i + 2] = lm::from_f<T>(s.z), out[i + 3] = lm::from_f<T>(s.w);
    } else {
      for (int64_t j = i; j < min(count, i + 4); ++j) {
        float s = 0.f;
        for (int k = 0; k < splits; ++k) s += parts[k * count + j];
        out[j] = lm::from_f<T>(s);
      }
    }
  }
}

template <typename K>
cudaLaunchConfig_t cluster_config(K* kernel, int grid, int threads, size_t smem, int cluster, cudaStream_t st,
                                  cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = cluster;
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// CTAs that share a tile: the largest power of two (it divides a tile's rows)
// with which all clusters run at once and a CTA's part has at least two groups.
// How many clusters fit is asked of the device, whose SMs come in groups that
// clusters do not cross: 15 of eight, 33 of four and 74 of two on 148 SMs. One
// cluster too many costs a second round: at 16 rows and K = 8192, 15 tiles take
// 7.4 us in clusters of eight, and 16 tiles 13.5, against 9.4 in clusters of four.
// `KERNEL` has opted in to its shared memory.
template <auto* KERNEL>
int splits_for(int64_t tiles, int groups, int threads, size_t smem) {
  static std::atomic<int> fits[64][4];   // by device and cluster size
  int dev = 0;
  TORCH_CHECK(cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64, "fp8_matmul: device query failed");
  int s = 1;
  for (int i = 1; 2 * s <= kMaxSplits && groups >= 4 * s; ++i, s *= 2) {
    int n = fits[dev][i].load(std::memory_order_relaxed);
    if (n == 0) {
      cudaLaunchAttribute attr = {};
      const auto cfg = cluster_config(KERNEL, 2 * s, threads, smem, 2 * s, nullptr, &attr);
      TORCH_CHECK(cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) == cudaSuccess, "fp8_matmul: occupancy query failed");
      fits[dev][i].store(n, std::memory_order_relaxed);
    }
    if (tiles > n) break;
  }
  return s;
}

template <typename K, typename... A>
void launch_cluster(K* kernel, int grid, int threads, size_t smem, int cluster, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute attr = {};
  const auto cfg = cluster_config(kernel, grid, threads, smem, cluster, st, &attr);
  TORCH_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess, "fp8_matmul launch failed");
}

// At most as many tiles as SMs.
void launch_tiles(const CUtensorMap& ta, const CUtensorMap& tb, Args g, int tiles, cudaStream_t st) {
  static size_t configured[dynsmem::kMaxDevices] = {};
  TORCH_CHECK(dynsmem::opt_in(fp8_gemm_kernel, kSmem, configured) == cudaSuccess, "fp8_matmul shared-memory attribute");
  g.splits = splits_for<fp8_gemm_kernel>(tiles, g.groups, kThreads, kSmem);
  launch_cluster(fp8_gemm_kernel, tiles * g.splits, kThreads, kSmem, g.splits, st, ta, tb, g);
}

// Up to COLS rows of A; false where the scales of a CTA's groups do not fit into its shared memory.
template <int COLS>
bool launch_rows(const CUtensorMap& tb, const torch::Tensor& a, int64_t lda, Args g, cudaStream_t st) {
  static size_t configured[dynsmem::kMaxDevices] = {};
  TORCH_CHECK(dynsmem::opt_in(fp8_gemm_rows_kernel<COLS>, rows_smem_bytes<COLS>(), configured) == cudaSuccess,
              "fp8_matmul shared-memory attribute");
  const int tiles = (g.N + kBM - 1) / kBM;
  g.splits = splits_for<fp8_gemm_rows_kernel<COLS>>(tiles, g.groups, kRowsThreads, rows_smem_bytes<COLS>());
  if ((g.groups + g.splits - 1) / g.splits * COLS > kRowsScales) return false;
  const CUtensorMap ta = tma::u8_sw128(a.data_ptr(), a.size(0), a.size(1), lda, COLS);
  launch_cluster(fp8_gemm_rows_kernel<COLS>, tiles * g.splits, kRowsThreads, rows_smem_bytes<COLS>(), g.splits, st, tb, ta,
                 g);
  return true;
}

template <bool WIDE>
void launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const Args& g, int64_t tiles, cudaStream_t st) {
  static size_t configured[dynsmem::kMaxDevices] = {};
  TORCH_CHECK(dynsmem::opt_in(gemm_pair_kernel<WIDE>, kPairSmem, configured) == cudaSuccess,
              "fp8_matmul shared-memory attribute");
  TORCH_CHECK(tiles < (1ll << 31), "fp8_matmul: too many output tiles");
  gemm_pair_kernel<WIDE><<<2 * (int)std::min<int64_t>(tiles, lm::sm_count() / 2), kPairThreads, kPairSmem, st>>>(ta, tb, g);
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
  const int64_t one_row = (K + 15) / 16 * 16;   // a single row's stride says nothing
  const int64_t lda = M > 1 ? a.stride(0) : one_row;
  const CUtensorMap tb = tma::u8_sw128(b.data_ptr(), N, K, N > 1 ? b.stride(0) : one_row, 128);
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  // By sizes alone (us measured at N = K = 4096 unless said):
  //  * up to 32 rows the few-row kernel, 7.0 against 9.7 with 128 x 128 tiles at 16 rows, 9.4 against 12.6 for one row
  //    of 1408 x 16640, 8.7 against 9.7 at 32 rows;
  //  * 128 x 128 tiles, or parts of them, while one round of CTAs has them all: 17.8 against 23.2 with pairs for
  //    1024 x 2048, where pairs leave half of the SMs idle;
  //  * pairs of CTAs beyond: 24.4 against 33.2 for 2048 x 2048, 82.9 against 128 for 9472 x 2048.
  const bool few = M <= 16 ? launch_rows<16>(tb, a, lda, g, st) : M <= 32 && launch_rows<32>(tb, a, lda, g, st);
  if (!few) {
    const CUtensorMap ta = tma::u8_sw128(a.data_ptr(), M, K, lda, kBM);
    const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128);
    if (tiles > lm::sm_count()) launch_pair<false>(ta, tb, g, ((M + 255) / 256) * ((N + 255) / 256), st);
    else launch_tiles(ta, tb, g, (int)tiles, st);
  }
  lm::count_launches(1);
  return c;
}

torch::Tensor weight_gradient(const torch::Tensor& a, const torch::Tensor& b, torch::ScalarType out_type,
                              const torch::Tensor& status) {
  const c10::cuda::CUDAGuard guard(a.device());
  const int64_t K = a.size(0), M = a.size(1), N = b.size(1);
  auto out = torch::empty({M, N}, a.options().dtype(out_type));
  if (M == 0 || N == 0) return out;
  if (K == 0) return out.zero_();
  LM_CHECK_VALUE(M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30), "weight gradient: too large");
  Args g{};
  g.M = (int)M;
  g.N = (int)N;
  g.groups = (int)((K + 63) / 64);
  g.ldc = N;
  g.status = status.data_ptr<int>();
  g.wait_ns = kWaitNs;
  // Few tiles over many rows: as many parts of the rows as the SM pairs have room for, four stages each at least.
  const int64_t tiles = ((M + 255) / 256) * ((N + 255) / 256), pairs = lm::sm_count() / 2;
  g.splits = (int)std::max<int64_t>(1, std::min<int64_t>(pairs / tiles, g.groups / 4));
  g.part = M * N;
  const bool direct = g.splits == 1 && out_type == torch::kFloat32;
  torch::Tensor parts = direct ? out : torch::empty({g.splits, M, N}, a.options().dtype(torch::kFloat32));
  g.c = parts.data_ptr();
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), "weight gradient: operands of one type");
  g.half = a.scalar_type() == torch::kHalf;
  const auto type = g.half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMap ta = tma::bf16_sw128(a.data_ptr(), K, M, a.stride(0), 64, type);
  const CUtensorMap tb = tma::bf16_sw128(b.data_ptr(), K, N, b.stride(0), 64, type);
  auto st = c10::cuda::getCurrentCUDAStream().stream();
  launch_pair<true>(ta, tb, g, tiles * g.splits, st);
  lm::count_launches(1);
  if (direct) return out;
  const auto sum = [&](auto t) {
    using T = decltype(t);
    sum_slices_kernel<T><<<(unsigned)std::min<int64_t>((M * N + 1023) / 1024, lm::sm_count() * 16), 256, 0, st>>>(
        parts.data_ptr<float>(), g.splits, M * N, reinterpret_cast<T*>(out.data_ptr()));
  };
  if (out_type == torch::kFloat32) sum(float{});
  else if (out_type == torch::kBFloat16) sum(__nv_bfloat16{});
  else sum(__half{});
  TORCH_CHECK(cudaGetLastError() == cudaSuccess, "weight gradient launch failed");
  lm::count_launches(1);
  return out;
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
  LM_CHECK_VALUE(!lm::any_tangent(a, a_scale, b, b_scale, bias) &&
                     !(at::GradMode::is_enabled() &&
                       (a.requires_grad() || a_scale.requires_grad() || b.requires_grad() || b_scale.requires_grad() ||
                        (bias && bias->requires_grad()))),
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
