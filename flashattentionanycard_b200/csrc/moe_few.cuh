// The MoE layer of moe_decode.cuh for a handful of tokens (at most 16, and 64
// assignments): two kernels whose boundary takes the place of the persistent kernel's counters.
//
// With few tokens and small experts the layer is a chain of latencies, not a
// stream: route, first weights, reduce, hand h over, reduce, combine.  So here
//   * both kernels route by themselves (every CTA picks all tokens' experts: a
//     microsecond, no launch, no list in memory);
//   * a tile's K is split over a thread-block cluster and its partial sums meet
//     in distributed shared memory (one cluster barrier instead of a round trip
//     of partials, counter and reload through L2);
//   * moe_few_down starts beside moe_few_up (both fit an SM together), routes and
//     fills its ring with w_down while h is still being made.
// moe_few_up    h[row] = silu(x Wg) * (x Wu), 128 + 128 columns a cluster
// moe_few_down  out: 128 columns a cluster; its k-steps run over the experts in
//               use, each with 16 accumulator columns of its own; a CTA weighs
//               its rows by their gates before the cluster's sum.
// Both sums run in rank order.  Measured against the persistent kernel (us a
// call): 8 experts x [1024, 2 x 2048], top 2: one token 13.2 and 22.7, four 25
// and 33, sixteen 33 and 35; 128 x [2048, 2 x 768], top 8: one token 24 and 40,
// four 58 and 67; 16 x [4096, 2 x 14336], top 2: one token 122 and 123.  16 tokens
// are what one box of x and 16 accumulator columns an expert hold; a form for
// more was slower where it was measured (37 tokens of 12 experts: 45 and 35, every
// CTA routes all tokens).
#pragma once

#include "moe_decode.cuh"

namespace bokt {

constexpr int kFewTokens = 16;
constexpr int kFewRows = 64;  // assignments
constexpr int kFewThreads = 256;
constexpr int kFewStages = 3;
constexpr int kFewTmemCols = 256;                  // moe_few_down: 16 experts a CTA
constexpr int kFewExperts = kFewTmemCols / 16;
constexpr int kFewUpStage = kMdStageW + 16 * 128;
constexpr int kFewDownStage = kMdStageW + 2 * 16 * 128;

struct MoeFewArgs {
  const void* logits;
  int logits_dtype, renormalize;
  int tokens, experts, k, inner, topk;
  int cluster;
  uint32_t idesc;  // M = 128, N = 16
  void* h;         // [tokens * topk][inner], rows by expert
  void* out;       // [tokens][k]
};

// Every CTA's own routing: experts in use in the order of their first
// assignment, rows packed by expert and, inside one, in assignment order.
struct FewRoute {
  int active;
  int id[kFewRows];      // expert of assignment t * topk + j
  float gate[kFewRows];
  int expert[kFewRows];  // of the a-th expert in use
  int off[kFewRows + 1]; // its first row
  int place[kFewRows];   // a of an assignment
  int row[kFewRows];     // row of an assignment
  int token[kFewRows];   // token of a row
  int warp_leads[2];
};

template <int V>
__device__ __forceinline__ void few_route(const MoeFewArgs& args, FewRoute& r) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int k = args.topk, A = args.tokens * k;
  for (int t = warp; t < args.tokens; t += kFewThreads / 32) {
    float gate;
    const int id = md_pick<V>(args.logits, args.logits_dtype, t, args.experts, k, args.renormalize, lane, &gate);
    if (lane < k) {
      r.id[t * k + lane] = id;
      r.gate[t * k + lane] = gate;
    }
  }
  __syncthreads();
  // Assignment i leads its expert if none before it has it.
  int before = 0;  // assignments of the same expert before this one
  bool leads = false;
  unsigned votes = 0;
  if (tid < kFewRows) {
    if (tid < A) {
      for (int j = 0; j < tid; ++j) before += r.id[j] == r.id[tid] ? 1 : 0;
      leads = before == 0;
    }
    votes = __ballot_sync(0xffffffffu, leads);
    if (lane == 0) r.warp_leads[warp] = __popc(votes);
  }
  __syncthreads();
  if (tid < kFewRows) {
    int a = __popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) a += r.warp_leads[w];
    if (leads) {
      r.expert[a] = r.id[tid];
      r.place[tid] = a;
    }
    if (tid == 0) r.active = r.warp_leads[0] + r.warp_leads[1];
  }
  __syncthreads();
  if (tid < A && !leads) {
    int a = 0;
    while (r.expert[a] != r.id[tid]) ++a;
    r.place[tid] = a;
  }
  __syncthreads();
  if (tid < A) {
    int row = before;
    for (int j = 0; j < A; ++j) row += r.place[j] < r.place[tid] ? 1 : 0;
    r.row[tid] = row;
    r.token[row] = tid / k;
    if (leads) r.off[r.place[tid]] = row;
  }
  if (tid == 0) r.off[r.active] = A;
  __syncthreads();
}

__host__ __device__ inline int moe_few_smem_bytes(int stage) {
  return 1024 + kFewStages * stage + (2 * kFewStages + 1) * 8 + 16;
}

// After a given-up wait: let copies in flight land before the memory is reused.
__device__ __forceinline__ void few_settle(volatile int* abort_flag) {
  if (*abort_flag && threadIdx.x == 0) {
    const uint64_t start = globaltimer_ns();
    while (globaltimer_ns() - start < 2000000ull) {
    }
  }
}

__device__ __forceinline__ void st_cluster_f1(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Shared front of both kernels: barriers, TMEM, cluster start.
struct FewRing {
  uint8_t* base;
  uint64_t *full, *empty, *tfull;
  uint32_t* tmem_holder;
  volatile int* abort_flag;
};

__device__ __forceinline__ FewRing few_ring(uint8_t* raw, int stage_bytes) {
  FewRing r;
  r.base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  r.full = reinterpret_cast<uint64_t*>(r.base + kFewStages * stage_bytes);
  r.empty = r.full + kFewStages;
  r.tfull = r.empty + kFewStages;
  r.tmem_holder = reinterpret_cast<uint32_t*>(r.tfull + 1);
  r.abort_flag = reinterpret_cast<volatile int*>(r.tmem_holder + 1);
  return r;
}

__device__ __forceinline__ void few_start(const FewRing& r, int warp, uint32_t tmem_cols) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&r.full[s], 2);  // weight and token producers
      mbar_init(&r.empty[s], 1);
    }
    mbar_init(r.tfull, 1);
    *r.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 3) {
    tmem_alloc(r.tmem_holder, tmem_cols);
    tmem_relinquish();
  }
  cluster_sync();  // every CTA runs before another writes its shared memory
}

// Cluster (expert a, column block nb); CTA r of it runs its share of K.
template <typename T, int V>
__global__ void __launch_bounds__(kFewThreads, 1)
    moe_few_up_kernel(const __grid_constant__ CUtensorMap tm_gu,
                      const __grid_constant__ CUtensorMap tm_x, const MoeFewArgs args) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ FewRoute route;
  const FewRing ring = few_ring(smem_raw, kFewUpStage);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int C = args.cluster, rank = static_cast<int>(cluster_ctarank());
  const int tiles = (args.inner + 127) / 128;
  const int ci = static_cast<int>(blockIdx.x) / C;
  const int a = ci / tiles, nb = ci - a * tiles;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_gu);
    tma_prefetch_desc(&tm_x);
  }
  few_start(ring, warp, 32);
  pdl_wait();
  pdl_allow_next();  // after the wait: moe_few_down reads logits and weights without one
  few_route<V>(args, route);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *ring.tmem_holder;
  const bool live = a < route.active;  // the same in the whole cluster
  const int ksteps = (args.k + 63) / 64;
  const int kb0 = rank * ksteps / C, kb1 = (rank + 1) * ksteps / C;
  if (live) {
    if (warp == 0) {
      if (elect_one()) {
        const int e = route.expert[a], c0 = nb * 128, c1 = args.inner + c0;
        int stage = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&ring.empty[stage], phase ^ 1u, ring.abort_flag, 81)) break;
          uint8_t* w = ring.base + stage * kFewUpStage;
          mbar_arrive_expect_tx(&ring.full[stage], kMdStageW);
          tma_load_3d(w, &tm_gu, &ring.full[stage], c0, kb * 64, e);
          tma_load_3d(w + 8192, &tm_gu, &ring.full[stage], c0 + 64, kb * 64, e);
          tma_load_3d(w + 16384, &tm_gu, &ring.full[stage], c1, kb * 64, e);
          tma_load_3d(w + 24576, &tm_gu, &ring.full[stage], c1 + 64, kb * 64, e);
          if (++stage == kFewStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == 2) {
      if (elect_one()) {
        int stage = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&ring.empty[stage], phase ^ 1u, ring.abort_flag, 82)) break;
          mbar_arrive_expect_tx(&ring.full[stage], 16 * 128);
          tma_load_2d(ring.base + stage * kFewUpStage + kMdStageW, &tm_x, &ring.full[stage], kb * 64, 0);
          if (++stage == kFewStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == 1) {
      if (elect_one()) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = mbar_wait(&ring.full[stage], phase, ring.abort_flag, 83))) break;
          tc_fence_after();
          const uint32_t w = smem_addr(ring.base + stage * kFewUpStage), b = w + kMdStageW;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t bd = smem_desc_sw128(b + k * 32, 16, 1024);
            const uint32_t on = (kb != kb0 || k != 0) ? 1u : 0u;
            umma_f16_ss(tmem_base, smem_desc_sw128(w + k * 2048, 8192, 1024), bd, args.idesc, on);
            umma_f16_ss(tmem_base + 16, smem_desc_sw128(w + 16384 + k * 2048, 8192, 1024), bd, args.idesc, on);
          }
          umma_commit(&ring.empty[stage]);
          if (++stage == kFewStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit(ring.tfull);
      }
    }
    __syncwarp();
    const bool ok = mbar_wait(ring.tfull, 0, ring.abort_flag, 84);
    few_settle(ring.abort_flag);
    __syncthreads();
    cluster_sync();  // every CTA of the cluster has consumed its ring
    // [C sources][rows of the expert][gate, up][128 / C columns], in the ring
    float* recv = reinterpret_cast<float*>(ring.base);
    const int m0 = route.off[a], m = route.off[a + 1] - m0, own = 128 / C;
    if (warp >= 4 && __all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      const int q = warp & 3, lcol = q * 32 + lane, to = lcol / own;
      const uint32_t d = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
      const uint32_t at = map_shared(smem_addr(recv + rank * m * 2 * own + lcol - to * own), to);
      for (int r0 = 0; r0 < m; r0 += 8) {
        uint32_t g[8], u[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint32_t t = route.token[m0 + min(r0 + r, m - 1)];
          g[r] = tmem_ld_x1(d + t);
          u[r] = tmem_ld_x1(d + 16 + t);
        }
        tmem_ld_wait();
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r0 + r < m) {
            st_cluster_f1(at + (r0 + r) * 2 * own * 4, __uint_as_float(g[r]));
            st_cluster_f1(at + ((r0 + r) * 2 + 1) * own * 4, __uint_as_float(u[r]));
          }
      }
      tc_fence_before();
    }
    cluster_sync();
    T* h = static_cast<T*>(args.h);
    for (int i = threadIdx.x; i < m * own; i += kFewThreads) {
      const int r = i / own, c = i - r * own, col = nb * 128 + rank * own + c;
      if (col >= args.inner) continue;
      float g = 0.f, u = 0.f;
      for (int s = 0; s < C; ++s) {
        g += recv[((s * m + r) * 2) * own + c];
        u += recv[((s * m + r) * 2 + 1) * own + c];
      }
      h[static_cast<size_t>(m0 + r) * args.inner + col] = Pack2<T>::from_float(g / (1.f + expf(-g)) * u);
    }
  }
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 32);
  }
}

// Cluster: one block of 128 columns.  Its k-steps (128 deep) run over the rows
// of w_down of the experts in use, one after the other; CTA r takes a
// contiguous run, which touches at most kFewExperts of them.
template <typename T, int V>
__global__ void __launch_bounds__(kFewThreads, 1)
    moe_few_down_kernel(const __grid_constant__ CUtensorMap tm_down,
                        const __grid_constant__ CUtensorMap tm_h, const MoeFewArgs args) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ FewRoute route;
  const FewRing ring = few_ring(smem_raw, kFewDownStage);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int C = args.cluster, rank = static_cast<int>(cluster_ctarank());
  const int n0 = static_cast<int>(blockIdx.x) / C * 128;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_down);
    tma_prefetch_desc(&tm_h);
  }
  few_start(ring, warp, kFewTmemCols);
  pdl_allow_next();
  few_route<V>(args, route);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *ring.tmem_holder;
  const int steps = (args.inner + 127) / 128, units = route.active * steps;
  const int u0 = rank * units / C, u1 = (rank + 1) * units / C;
  const int a0 = u0 / steps;  // the first expert this CTA touches
  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int u = u0; u < u1; ++u) {
        if (!mbar_wait(&ring.empty[stage], phase ^ 1u, ring.abort_flag, 85)) break;
        const int a = u / steps, kb = (u - a * steps) * 128, e = route.expert[a];
        uint8_t* w = ring.base + stage * kFewDownStage;
        mbar_arrive_expect_tx(&ring.full[stage], kMdStageW);
        tma_load_3d(w, &tm_down, &ring.full[stage], n0, kb, e);
        tma_load_3d(w + 8192, &tm_down, &ring.full[stage], n0 + 64, kb, e);
        tma_load_3d(w + 16384, &tm_down, &ring.full[stage], n0, kb + 64, e);
        tma_load_3d(w + 24576, &tm_down, &ring.full[stage], n0 + 64, kb + 64, e);
        if (++stage == kFewStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 2) {
    if (elect_one()) {
      pdl_wait();               // h is complete
      fence_proxy_async_all();  // and was stored by ordinary stores
      int stage = 0;
      uint32_t phase = 0;
      for (int u = u0; u < u1; ++u) {
        if (!mbar_wait(&ring.empty[stage], phase ^ 1u, ring.abort_flag, 86)) break;
        const int a = u / steps, kb = (u - a * steps) * 128;
        uint8_t* b = ring.base + stage * kFewDownStage + kMdStageW;
        mbar_arrive_expect_tx(&ring.full[stage], 2 * 16 * 128);
        tma_load_2d(b, &tm_h, &ring.full[stage], kb, route.off[a]);
        tma_load_2d(b + 16 * 128, &tm_h, &ring.full[stage], kb + 64, route.off[a]);
        if (++stage == kFewStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = u0; u < u1; ++u) {
        if (!(ok = mbar_wait(&ring.full[stage], phase, ring.abort_flag, 87))) break;
        tc_fence_after();
        const int a = u / steps;
        const uint32_t d = tmem_base + (a - a0) * 16;
        const bool fresh = u == u0 || u == a * steps;  // this CTA's first k-step of the expert
        const uint32_t w = smem_addr(ring.base + stage * kFewDownStage), b = w + kMdStageW;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16_ss(d, smem_desc_sw128(w + (k >> 2) * 16384 + (k & 3) * 2048, 8192, 1024),
                      smem_desc_sw128(b + (k >> 2) * 2048 + (k & 3) * 32, 16, 1024), args.idesc,
                      fresh && k == 0 ? 0u : 1u);
        umma_commit(&ring.empty[stage]);
        if (++stage == kFewStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) umma_commit(ring.tfull);
    }
  }
  __syncwarp();
  const bool ok = mbar_wait(ring.tfull, 0, ring.abort_flag, 88);
  pdl_wait();
  few_settle(ring.abort_flag);
  __syncthreads();
  cluster_sync();  // every CTA of the cluster has consumed its ring
  // [C sources][tokens][128 / C columns], in the ring
  float* recv = reinterpret_cast<float*>(ring.base);
  const int own = 128 / C, topk = args.topk;
  if (warp >= 4 && __all_sync(0xffffffffu, ok)) {
    tc_fence_after();
    const int q = warp & 3, lcol = q * 32 + lane, to = lcol / own;
    const uint32_t d = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t at = map_shared(smem_addr(recv + rank * args.tokens * own + lcol - to * own), to);
    const int a1 = u1 > u0 ? (u1 - 1) / steps : a0 - 1;  // the last expert touched
    for (int t = 0; t < args.tokens; ++t) {
      uint32_t v[kMdMaxTopk];
#pragma unroll
      for (int j = 0; j < kMdMaxTopk; ++j) {
        const int i = t * topk + min(j, topk - 1), a = route.place[i];
        const int col = a >= a0 && a <= a1 ? (a - a0) * 16 + route.row[i] - route.off[a] : 0;
        v[j] = tmem_ld_x1(d + col);
      }
      tmem_ld_wait();
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < kMdMaxTopk; ++j) {
        const int i = t * topk + min(j, topk - 1), a = route.place[i];
        if (j < topk && a >= a0 && a <= a1) sum = fmaf(route.gate[i], __uint_as_float(v[j]), sum);
      }
      st_cluster_f1(at + t * own * 4, sum);
    }
    tc_fence_before();
  }
  cluster_sync();
  T* out = static_cast<T*>(args.out);
  for (int i = threadIdx.x; i < args.tokens * own / 2; i += kFewThreads) {
    const int t = i / (own / 2), c = (i - t * (own / 2)) * 2, col = n0 + rank * own + c;
    if (col >= args.k) continue;
    float2 sum = make_float2(0.f, 0.f);
    for (int s = 0; s < C; ++s) {
      const float2 v = *reinterpret_cast<const float2*>(recv + (s * args.tokens + t) * own + c);
      sum.x += v.x;
      sum.y += v.y;
    }
    *reinterpret_cast<uint32_t*>(out + static_cast<size_t>(t) * args.k + col) = Pack2<T>::pack(sum.x, sum.y);
  }
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kFewTmemCols);
  }
}

}  // namespace bokt
