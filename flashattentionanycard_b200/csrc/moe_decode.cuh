// A whole mixture-of-experts layer for a few tokens (at most 128), two kernels
// (sm_100a).  Per token t with router logits z[t, :]:
//   p = softmax(z[t]),  e_1..e_k = the k largest p (ties: lower index),
//   g_j = p[e_j] (/ their sum),
//   out[t] = sum_j g_j (silu(x[t] Wg_j) * (x[t] Wu_j)) Wd_j
// with [Wg | Wu] = w_gate_up[e] ([K, 2 I]) and Wd = w_down[e] ([I, K]).
//
// Bound by HBM: the weights of every expert in use are read once, 3 K I values
// each, and meet few tokens.  So the roles of the tensor-core operands are
// swapped against the GEMM's: a weight tile is the 128-row operand (its columns
// become accumulator lanes) and the tokens are the narrow operand (N = 16..128
// accumulator columns); whatever N is, the tcgen05 time stays below the time
// the weights take to arrive, and the kernel is a stream of TMA tile loads
// through a deep shared-memory ring.
//
//   moe_decode_gate_kernel   one cluster: softmax, top-k, rows sorted by expert
//   moe_decode_kernel        everything else, persistent, one CTA per SM:
//     phase 1  h[row] = silu(gate) * up per assignment, 128 + 128 columns a
//              tile; tokens are read in place (all T of them; the epilogue picks
//              the columns of those routed to the tile's expert).  h is phase
//              2's tensor-core operand, so it is rounded to the element type
//              (in fp16 within 65,504): the layer's error against fp64 is 0.0023
//              of its norm in bf16, where one rounding of the result gives 0.0017
//     phase 2  y[row] = h[row] Wd, 256 columns a tile
//     phase 3  out = gate-weighted sum of y (fp32, slot order)
//
// Work: a phase's k-steps (64 deep), tile-major, are cut into one contiguous
// run ("share") per CTA, so every SM streams the same number of bytes whatever
// the number of experts and tiles.  A tile cut by a share's end is summed from
// fp32 partials: in phase 1 by the last warp to arrive, in phase 3 with the sum
// over experts; both in share order, so the result does not depend on timing.
// Shares are claimed in order (phase 1 first) from a counter, so a CTA that
// waits for phase 1 to finish knows that every phase-1 share is held by a
// running CTA: no assumption on how many CTAs are resident.  The weight
// producer runs ahead across the phase boundary by the depth of the ring, so
// HBM stays busy while h is completed.
//
// Warps: 0 weight producer (and claims), 1 MMA issuer, 2 token producer, 3 TMEM
// owner, 4-7 epilogue (one TMEM lane quadrant each, independent of each other:
// no barrier across warps after the prologue, so an aborted wait strands none).
#pragma once

#include "bokt_device.cuh"
#include "splitk.cuh"

namespace bokt {

constexpr int kMdThreads = 256;
constexpr int kMdMaxTokens = 128;
constexpr int kMdMaxTopk = 8;
constexpr int kMdMaxExperts = 1024;
constexpr int kMdStageW = 32768;  // 4 boxes of 64 columns x 64 k
constexpr int kMdQueue = 4;
constexpr int kMdMaxStages = 8;
// Fewest k-steps of a share: below that a tile's partial sums cost more than the
// spreading saves.  With 1, 2, 4, 8 (us in a graph, weights not in L2): 17 tokens
// of 2 experts x [8192, 2 x 72] 49, 45, 36, 32; 20 of 4 x [4096, 2 x 136] 37, 37,
// 32, 31; 30 of 20 x [512, 2 x 512], top 2, 27, 27, 25, 23; 37 of 12 x [1032,
// 2 x 1000], top 3, 35, 35, 35, 33; 32 of 16 x [4096, 2 x 14336] and 64 of 128 x
// [2048, 2 x 768] the same within 0.3%.  8 is the better of the last two here.
constexpr int kMdMinSteps = 4;
// Phase 1 cuts tiles only where that shortens the longest share by more k-steps
// than the cut tiles' way through memory takes.  With 0, 6, 12, 24 and never: 37
// of 12 x [1032, 2 x 1000] 42, 35, 35, 35, 35; 64 of 8 x [4096, 2 x 2048] 100,
// 101, 85, 85, 85; 48 of 8 x [2048, 2 x 1024] 46, 46, 46, 38, 38; 20 of 4 x [4096,
// 2 x 136] 32, 32, 32, 32, 43; 17 of 2 x [8192, 2 x 72] 36, 36, 36, 36, 65.  So
// cutting is needed where few tiles are long, and 24 is the better limit here.
constexpr int kMdSplitSteps = 12;

// Header words of the workspace.
constexpr int kMdClaim = 0, kMdDone1 = 32, kMdDone2 = 64, kMdActive = 96, kMdCount1 = 128;

struct MoeDecodeArgs {
  int tokens, experts, k, inner, topk;
  int nt;      // token columns of phase 1 (tokens rounded up to 16)
  int stages;
  int shares;  // = gridDim.x
  uint32_t idesc;  // M = 128, N field 0
  uint32_t* header;
  int* act_e;      // [min(E, A)] experts in use, ascending
  int* act_off;    // [.. + 1] their first packed row
  int* row_token;  // [A] token of a packed row
  int* row_of;     // [A] packed row of assignment t * topk + j
  int* act_of;     // [A] its index in act_e
  float* gates;    // [A]
  void* h;         // [A][inner]
  float* y;        // [A][k]
  float* part;     // [2 * shares][tokens * 256]
  void* out;       // [tokens][k]
};

// Logits as integers of the same order (-0 as 0).  A NaN sorts below everything
// (its token's gates are NaN whatever is picked) and comes back as a NaN; 0
// marks a taken expert.
__device__ __forceinline__ uint32_t md_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  const uint32_t key = b & 0x80000000u ? ~b : b | 0x80000000u;
  return v == v ? key : 1u;
}
__device__ __forceinline__ float md_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

__device__ __forceinline__ float md_logit(const void* logits, int dtype, size_t at) {
  if (dtype == 2) return static_cast<const float*>(logits)[at];
  if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(logits)[at]);
  return __half2float(static_cast<const __half*>(logits)[at]);
}

// The top k of one token's softmax, one warp, V logits per lane (V * 32 >= E):
// lane j < k returns the j-th expert and its gate.  dtype: BOKT_FP16/BF16/FP32.
template <int V>
__device__ __forceinline__ int md_pick(const void* logits, int dtype, int t, int E, int k,
                                       int renormalize, int lane, float* gate_out) {
  uint32_t key[V], best = 0;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    key[i] = e < E ? md_key(md_logit(logits, dtype, static_cast<size_t>(t) * E + e)) : 0u;
    best = max(best, key[i]);
  }
  const float mx = md_value(__reduce_max_sync(0xffffffffu, best));
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i * 32 + lane < E) sum += expf(md_value(key[i]) - mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  int mine = 0;
  uint32_t mine_key = 0;
  for (int j = 0; j < k; ++j) {
    best = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) best = max(best, key[i]);
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    int at = 0x7fffffff;
#pragma unroll
    for (int i = V - 1; i >= 0; --i)
      if (key[i] == top) at = i * 32 + lane;
    at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * 32 + lane == at) key[i] = 0u;
    if (lane == j) {
      mine = at;
      mine_key = top;
    }
  }
  const float gate = lane < k ? expf(md_value(mine_key) - mx) / sum : 0.f;
  float picked = gate;
#pragma unroll
  for (int o = kMdMaxTopk / 2; o > 0; o >>= 1) picked += __shfl_xor_sync(0xffffffffu, picked, o);
  *gate_out = renormalize ? gate / picked : gate;
  return mine;
}

constexpr int kMdGateThreads = 512;
constexpr int kMdGateCtas = 8;

// One cluster of up to eight CTAs, a warp per token, V logits per lane.  Rank 0
// gathers the picked ids through distributed shared memory and sorts the
// assignments by expert.  The order of one expert's rows follows the atomics
// and decides nothing: a row's arithmetic does not depend on its place.
// Latency bound; few warps per SM pick faster than many (64 tokens of 128
// experts, top 8, on two CTAs of 32 warps: 4.3 us).
template <int V>
__global__ void __launch_bounds__(kMdGateThreads)
    moe_decode_gate_kernel(const void* __restrict__ logits, int logits_dtype, int renormalize,
                           const MoeDecodeArgs args) {
  __shared__ int s_id[kMdMaxTokens * kMdMaxTopk];
  __shared__ int s_pos[kMdMaxTokens * kMdMaxTopk];
  __shared__ int s_cnt[kMdMaxExperts];
  __shared__ int s_scan[kMdMaxExperts];  // first row | place among the experts in use << 16
  __shared__ int s_warp[kMdGateThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int E = args.experts, k = args.topk, T = args.tokens, A = T * k;
  const int rank = static_cast<int>(cluster_ctarank());
  for (int e = tid; e < E; e += kMdGateThreads) s_cnt[e] = 0;
  cluster_sync();  // every CTA runs before another writes its shared memory
  pdl_allow_next();
  pdl_wait();
  const int per = (T + gridDim.x - 1) / gridDim.x;  // tokens per CTA, at most 16
  const int t = rank * per + warp;
  if (warp < per && t < T) {
    float gate;
    const int mine = md_pick<V>(logits, logits_dtype, t, E, k, renormalize, lane, &gate);
    if (lane < k) {
      args.gates[t * k + lane] = gate;
      const uint32_t dst = map_shared(smem_addr(&s_id[t * k + lane]), 0);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(mine) : "memory");
    }
  }
  if (rank == 0) {
    for (int i = tid; i < kMdCount1 + args.shares * 4; i += kMdGateThreads) args.header[i] = 0u;
  }
  cluster_sync();
  if (rank != 0) return;
  for (int i = tid; i < A; i += kMdGateThreads) s_pos[i] = atomicAdd(&s_cnt[s_id[i]], 1);
  __syncthreads();
  // Exclusive scan over experts of (rows, in use), packed 16 + 16 bits; two
  // neighbouring experts per thread.
  static_assert(kMdMaxExperts == 2 * kMdGateThreads, "two experts per thread");
  int c[2], v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c[i] = 2 * tid + i < E ? s_cnt[2 * tid + i] : 0;
    v[i] = c[i] | (c[i] > 0 ? 1 << 16 : 0);
  }
  int incl = v[0] + v[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int excl = incl - v[0] - v[1], total = 0;
#pragma unroll
  for (int w = 0; w < kMdGateThreads / 32; ++w) {
    if (w < warp) excl += s_warp[w];
    total += s_warp[w];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (2 * tid + i < E) s_scan[2 * tid + i] = excl;
    if (c[i] > 0) {
      args.act_e[excl >> 16] = 2 * tid + i;
      args.act_off[excl >> 16] = excl & 0xffff;
    }
    excl += v[i];
  }
  if (tid == 0) {
    const int active = total >> 16;
    args.header[kMdActive] = static_cast<uint32_t>(active);
    args.act_off[active] = A;
  }
  __syncthreads();
  for (int i = tid; i < A; i += kMdGateThreads) {
    const int at = s_scan[s_id[i]], row = (at & 0xffff) + s_pos[i];
    args.row_token[row] = i / k;
    args.row_of[i] = row;
    args.act_of[i] = at >> 16;
  }
}

__device__ __forceinline__ void fence_proxy_async_all() {
  asm volatile("fence.proxy.async;" ::: "memory");
}

// Bounded wait for a device counter to reach `target`.
__device__ __forceinline__ bool md_wait_counter(const uint32_t* p, uint32_t target,
                                                volatile int* abort_flag, int where) {
  if (ld_acquire_gpu(p) >= target) return true;
  const uint64_t start = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (ld_acquire_gpu(p) >= target) return true;
    if ((it & 31u) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - start > kWaitTimeoutNs) {
        *abort_flag = 1;
        report_status(kStatusWaitTimeout, where);
        return false;
      }
    }
  }
}

__device__ __forceinline__ uint32_t tmem_ld_x1(uint32_t taddr) {
  uint32_t v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr));
  return v;
}

// The k-steps [u0, u1) of a phase, one tile's stretch ("segment") at a time.
struct MdSegments {
  int u, u1, steps;  // next k-step, end, k-steps per tile
  int tile, kb0, kb1;
  __device__ __forceinline__ bool next() {
    if (u >= u1) return false;
    tile = u / steps;
    kb0 = u - tile * steps;
    kb1 = min(steps, kb0 + u1 - u);
    u += kb1 - kb0;
    return true;
  }
};

__device__ __forceinline__ int md_share_begin(int share, int units, int shares) {
  return static_cast<int>(static_cast<long long>(share) * units / shares);
}
// The share that holds k-step u: the largest g with md_share_begin(g) <= u.
__device__ __forceinline__ int md_share_of(int u, int units, int shares) {
  return static_cast<int>(((static_cast<long long>(u) + 1) * shares - 1) / units);
}

struct MdPlan {
  int active;                          // experts in use
  int tiles1, steps1, units1, shares1;  // per expert: tiles1 of 128 + 128 columns
  int tiles2, steps2, units2, shares2;  // tiles2 column blocks of 256, experts inside
  int whole1;                          // phase 1 shares end at tile ends
  int claims;                          // of all phases
  const int* act_e;
  const int* act_off;
  const int* row_token;
};

// Phase (0, 1, 2) of a claim; *share: its share of that phase.
__device__ __forceinline__ int md_phase(const MdPlan& p, int claim, int* share) {
  if (claim < p.shares1) {
    *share = claim;
    return 0;
  }
  claim -= p.shares1;
  const int phase = claim < p.shares2 ? 1 : 2;
  *share = phase == 1 ? claim : claim - p.shares2;
  return phase;
}

__device__ __forceinline__ MdSegments md_segments(const MdPlan& p, int phase, int share) {
  MdSegments s;
  const int units = phase == 0 ? p.units1 : p.units2;
  const int shares = phase == 0 ? p.shares1 : p.shares2;
  s.steps = phase == 0 ? p.steps1 : p.steps2;
  if (phase == 0 && p.whole1) {
    s.u = md_share_begin(share, units / s.steps, shares) * s.steps;
    s.u1 = md_share_begin(share + 1, units / s.steps, shares) * s.steps;
  } else {
    s.u = md_share_begin(share, units, shares);
    s.u1 = md_share_begin(share + 1, units, shares);
  }
  return s;
}

__host__ __device__ inline int moe_decode_smem_bytes(int nt, int stages, int experts_max, int rows) {
  return 1024 + stages * (kMdStageW + nt * 128) + (2 * stages + 4 + 2 * kMdQueue) * 8 +
         (kMdQueue + 4) * 4 + (2 * experts_max + 1 + rows) * 4 + 16;
}

// CPL neighbouring fp32 columns of one lane.
template <int CPL>
struct MdCols {
  float f[CPL];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < CPL; ++i) f[i] = 0.f;
  }
  __device__ __forceinline__ void load(const float* p) {  // past L1: other SMs wrote it
    if constexpr (CPL == 2) {
      const float2 a = __ldcg(reinterpret_cast<const float2*>(p));
      f[0] = a.x, f[1] = a.y;
    } else {
#pragma unroll
      for (int i = 0; i < CPL; i += 4) {
        const float4 a = __ldcg(reinterpret_cast<const float4*>(p + i));
        f[i] = a.x, f[i + 1] = a.y, f[i + 2] = a.z, f[i + 3] = a.w;
      }
    }
  }
  __device__ __forceinline__ void add(const MdCols& o) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) f[i] += o.f[i];
  }
  __device__ __forceinline__ void fma(float g, const MdCols& o) {
#pragma unroll
    for (int i = 0; i < CPL; ++i) f[i] = fmaf(g, o.f[i], f[i]);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (CPL == 2) {
      *reinterpret_cast<uint32_t*>(p) = Pack2<T>::pack(f[0], f[1]);
    } else {
      static_assert(CPL == 8, "16-byte stores");
      *reinterpret_cast<uint4*>(p) =
          make_uint4(Pack2<T>::pack(f[0], f[1]), Pack2<T>::pack(f[2], f[3]),
                     Pack2<T>::pack(f[4], f[5]), Pack2<T>::pack(f[6], f[7]));
    }
  }
};

// What lane j knows of a token's j-th expert for one column block of phase 3.
struct MdSlot {
  int row = 0, base = 0;  // packed row, and its place among its expert's rows
  int g0 = 0, g1 = -1;    // shares that begin inside its tile: partials to add
  float gate = 0.f;
  __device__ __forceinline__ void load(const MoeDecodeArgs& args, const MdPlan& plan, int t, int nb,
                                       int lane) {
    if (lane >= args.topk) return;
    const int as = t * args.topk + lane;
    row = args.row_of[as];
    gate = args.gates[as];
    const int a = args.act_of[as];
    base = row - plan.act_off[a];
    const int u = (nb * plan.active + a) * plan.steps2;
    g0 = md_share_of(u, plan.units2, plan.shares2) + 1;
    g1 = md_share_of(u + plan.steps2 - 1, plan.units2, plan.shares2);
  }
};

// Items first, first + stride, ... of phase 3: the gate-weighted sum of one
// token's rows of y over 32 CPL columns, each row completed by the partials of
// the shares that begin inside its tile.  All rows are loaded before the first
// is used; the sum runs in slot order.  The first item's slots are read before
// the wait for phase 2.
template <typename T, int CPL>
__device__ __forceinline__ bool md_combine(const MoeDecodeArgs& args, const MdPlan& plan, int first,
                                           int stride, int lane, volatile int* abort_flag) {
  const int K = args.k, topk = args.topk;
  const int blocks = (K + 32 * CPL - 1) / (32 * CPL);
  const size_t slot_floats = static_cast<size_t>(args.tokens) * 256;
  using Vec = MdCols<CPL>;
  bool waited = false;
  for (int it = first; it < args.tokens * blocks; it += stride) {
    const int t = it / blocks, col = (it - t * blocks) * 32 * CPL + lane * CPL;
    MdSlot slot;
    slot.load(args, plan, t, (it - t * blocks) * 32 * CPL / 256, lane);
    if (!waited) {
      const bool ok = lane != 0 || md_wait_counter(args.header + kMdDone2,
                                                   4u * static_cast<uint32_t>(plan.units2), abort_flag, 40);
      if (!__all_sync(0xffffffffu, ok)) return false;
      __threadfence();
      waited = true;
    }
    const bool in = col < K;
    const int c = col & 255;
    Vec v[kMdMaxTopk], first_part[kMdMaxTopk];
#pragma unroll
    for (int j = 0; j < kMdMaxTopk; ++j) {
      const int r = __shfl_sync(0xffffffffu, slot.row, j), b = __shfl_sync(0xffffffffu, slot.base, j);
      const int s0 = __shfl_sync(0xffffffffu, slot.g0, j), s1 = __shfl_sync(0xffffffffu, slot.g1, j);
      v[j].zero();
      first_part[j].zero();
      if (j < topk && in) v[j].load(args.y + static_cast<size_t>(r) * K + col);
      if (j < topk && s0 <= s1) first_part[j].load(args.part + 2 * s0 * slot_floats + b * 256 + c);
    }
#pragma unroll
    for (int j = 0; j < kMdMaxTopk; ++j) {
      if (j >= topk) break;
      const int b = __shfl_sync(0xffffffffu, slot.base, j);
      const int s0 = __shfl_sync(0xffffffffu, slot.g0, j), s1 = __shfl_sync(0xffffffffu, slot.g1, j);
      v[j].add(first_part[j]);
      for (int s = s0 + 1; s <= s1; s += 4) {
        Vec w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i].zero();
          if (s + i <= s1) w[i].load(args.part + 2 * (s + i) * slot_floats + b * 256 + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j].add(w[i]);
      }
    }
    Vec sum;
    sum.zero();
#pragma unroll
    for (int j = 0; j < kMdMaxTopk; ++j) {
      const float g = __shfl_sync(0xffffffffu, slot.gate, j);
      if (j < topk) sum.fma(g, v[j]);
    }
    if (in) sum.template store<T>(static_cast<T*>(args.out) + static_cast<size_t>(t) * K + col);
  }
  return true;
}

template <typename T>
__global__ void __launch_bounds__(kMdThreads, 1)
    moe_decode_kernel(const __grid_constant__ CUtensorMap tm_gu,
                      const __grid_constant__ CUtensorMap tm_down,
                      const __grid_constant__ CUtensorMap tm_x,
                      const __grid_constant__ CUtensorMap tm_h, const MoeDecodeArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stages = args.stages, nt = args.nt;
  const int stage_b = nt * 128;
  uint8_t* sW = smem;
  uint8_t* sB = sW + stages * kMdStageW;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + stages * stage_b);
  uint64_t* empty = full + stages;
  uint64_t* tfull = empty + stages;
  uint64_t* tempty = tfull + 2;
  uint64_t* qfull = tempty + 2;
  uint64_t* qempty = qfull + kMdQueue;
  volatile int* queue = reinterpret_cast<volatile int*>(qempty + kMdQueue);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(qempty + kMdQueue) + kMdQueue;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* s_active = reinterpret_cast<int*>(tmem_holder + 2);
  int* s_claim = s_active + 1;
  int* s_act_e = reinterpret_cast<int*>(tmem_holder + 4);
  const int A = args.tokens * args.topk;
  const int emax = min(args.experts, A);
  int* s_act_off = s_act_e + emax;
  int* s_row_token = s_act_off + emax + 1;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  uint32_t tmem_cols = 32;
  while (tmem_cols < 4u * nt) tmem_cols *= 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 2);  // weight and token producers
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4);
    }
    for (int i = 0; i < kMdQueue; ++i) {
      mbar_init(&qfull[i], 1);
      mbar_init(&qempty[i], 6);  // MMA issuer, token producer, four epilogue warps
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_gu);
    tma_prefetch_desc(&tm_down);
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_h);
  }
  if (warp == 3) {
    tmem_alloc(tmem_holder, tmem_cols);
    tmem_relinquish();
  }
  pdl_allow_next();
  pdl_wait();
  if (threadIdx.x == 0) *s_claim = static_cast<int>(atomicAdd(args.header + kMdClaim, 1u));
  if (threadIdx.x == 32) *s_active = static_cast<int>(args.header[kMdActive]);
  for (int i = threadIdx.x; i < emax + 1; i += kMdThreads) {
    if (i < emax) s_act_e[i] = args.act_e[i];
    s_act_off[i] = args.act_off[i];
  }
  for (int i = threadIdx.x; i < A; i += kMdThreads) s_row_token[i] = args.row_token[i];
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  MdPlan plan;
  plan.active = *s_active;
  plan.tiles1 = (args.inner + 127) / 128;
  plan.steps1 = (args.k + 63) / 64;
  plan.units1 = plan.active * plan.tiles1 * plan.steps1;
  plan.tiles2 = (args.k + 255) / 256;
  plan.steps2 = (args.inner + 63) / 64;
  plan.units2 = plan.active * plan.tiles2 * plan.steps2;
  plan.act_e = s_act_e;
  plan.act_off = s_act_off;
  plan.row_token = s_row_token;
  const int shares = args.shares;
  const int tiles = plan.active * plan.tiles1;
  plan.whole1 = (tiles + shares - 1) / shares * plan.steps1 <= plan.units1 / shares + kMdSplitSteps;
  plan.shares1 = plan.whole1 ? min(shares, tiles) : max(1, min(shares, plan.units1 / kMdMinSteps));
  plan.shares2 = max(1, min(shares, plan.units2 / kMdMinSteps));
  plan.claims = plan.shares1 + plan.shares2 + shares;

  if (warp == 0) {
    // ------------------------------------------------------- weights, claims
    if (elect_one()) {
      int stage = 0, claim = *s_claim;
      uint32_t phase = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int slot = n % kMdQueue;
        if (!mbar_wait(&qempty[slot], ((n / kMdQueue) & 1) ^ 1, abort_flag, 31)) break;
        queue[slot] = claim;
        mbar_arrive(&qfull[slot]);
        if (claim >= plan.claims) break;
        int share;
        const int ph = md_phase(plan, claim, &share);
        if (ph < 2) {
          MdSegments sg = md_segments(plan, ph, share);
          while (ok && sg.next()) {
            const int a = ph == 0 ? sg.tile / plan.tiles1 : sg.tile % plan.active;
            const int nb = ph == 0 ? sg.tile % plan.tiles1 : sg.tile / plan.active;
            const int e = plan.act_e[a];
            const CUtensorMap* map = ph == 0 ? &tm_gu : &tm_down;
            const int c0 = ph == 0 ? nb * 128 : nb * 256;
            const int c1 = ph == 0 ? args.inner + c0 : c0 + 128;
            for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
              if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 32)) {
                ok = false;
                break;
              }
              uint8_t* w = sW + stage * kMdStageW;
              mbar_arrive_expect_tx(&full[stage], kMdStageW);
              tma_load_3d(w, map, &full[stage], c0, kb * 64, e);
              tma_load_3d(w + 8192, map, &full[stage], c0 + 64, kb * 64, e);
              tma_load_3d(w + 16384, map, &full[stage], c1, kb * 64, e);
              tma_load_3d(w + 24576, map, &full[stage], c1 + 64, kb * 64, e);
              if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
              }
            }
          }
        }
        // A phase-3 share loads nothing here: claim the next when this one is done.
        if (ph == 2)
          ok = ok && mbar_wait(&qempty[slot], (n / kMdQueue) & 1, abort_flag, 42);
        if (ok) claim = static_cast<int>(atomicAdd(args.header + kMdClaim, 1u));
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------- token operand
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, ready = false;
      for (int n = 0; ok; ++n) {
        const int slot = n % kMdQueue;
        if (!mbar_wait(&qfull[slot], (n / kMdQueue) & 1, abort_flag, 33)) break;
        const int claim = queue[slot];
        mbar_arrive(&qempty[slot]);
        if (claim >= plan.claims) break;
        int share;
        const int ph = md_phase(plan, claim, &share);
        if (ph == 2) continue;
        MdSegments sg = md_segments(plan, ph, share);
        while (ok && sg.next()) {
          if (ph == 1 && !ready) {
            // Every warp of phase 1 has stored its h (generic stores, read
            // below through the async proxy).
            ok = md_wait_counter(args.header + kMdDone1,
                                 4u * static_cast<uint32_t>(plan.active * plan.tiles1), abort_flag, 34);
            if (!ok) break;
            fence_proxy_async_all();
            ready = true;
          }
          const int a = ph == 0 ? 0 : sg.tile % plan.active;
          const int row0 = ph == 0 ? 0 : plan.act_off[a];
          const int rows = ph == 0 ? nt : (plan.act_off[a + 1] - row0 + 15) & ~15;
          for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
            if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 35)) {
              ok = false;
              break;
            }
            uint8_t* b = sB + stage * stage_b;
            mbar_arrive_expect_tx(&full[stage], rows * 128);
            if (ph == 0) {
              tma_load_2d(b, &tm_x, &full[stage], kb * 64, 0);
            } else {
              for (int r = 0; r < rows; r += 16)
                tma_load_2d(b + r * 128, &tm_h, &full[stage], kb * 64, row0 + r);
            }
            if (++stage == stages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------- MMA issuer
    if (elect_one()) {
      int stage = 0, i = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int slot = n % kMdQueue;
        if (!mbar_wait(&qfull[slot], (n / kMdQueue) & 1, abort_flag, 36)) break;
        const int claim = queue[slot];
        mbar_arrive(&qempty[slot]);
        if (claim >= plan.claims) break;
        int share;
        const int ph = md_phase(plan, claim, &share);
        if (ph == 2) continue;
        MdSegments sg = md_segments(plan, ph, share);
        for (; ok && sg.next(); ++i) {
          int cols = nt;
          if (ph == 1) {
            const int a = sg.tile % plan.active;
            cols = (plan.act_off[a + 1] - plan.act_off[a] + 15) & ~15;
          }
          const uint32_t idesc = args.idesc | (static_cast<uint32_t>(cols >> 3) << 17);
          const int acc = i & 1;
          if (!mbar_wait(&tempty[acc], ((i >> 1) & 1) ^ 1, abort_flag, 37)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d0 = tmem_base + static_cast<uint32_t>(acc * 2 * nt);
          for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
            if (!mbar_wait(&full[stage], phase, abort_flag, 38)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t w = smem_addr(sW + stage * kMdStageW);
            const uint32_t b = smem_addr(sB + stage * stage_b);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t bd = smem_desc_sw128(b + k * 32, 16, 1024);
              const uint32_t on = (kb != sg.kb0 || k != 0) ? 1u : 0u;
              umma_f16_ss(d0, smem_desc_sw128(w + k * 2048, 8192, 1024), bd, idesc, on);
              umma_f16_ss(d0 + nt, smem_desc_sw128(w + 16384 + k * 2048, 8192, 1024), bd, idesc, on);
            }
            umma_commit(&empty[stage]);
            if (++stage == stages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) umma_commit(&tfull[acc]);
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------- epilogue
    const int q = warp & 3;
    const int lcol = q * 32 + lane;  // column inside a 128-column tile half
    const size_t slot_floats = static_cast<size_t>(args.tokens) * 256;
    const int I = args.inner, K = args.k;
    T* h = static_cast<T*>(args.h);
    int i = 0;
    for (int n = 0;; ++n) {
      const int qslot = n % kMdQueue;
      bool ok = mbar_wait(&qfull[qslot], (n / kMdQueue) & 1, abort_flag, 39);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int claim = queue[qslot];
      __syncwarp();
      if (claim >= plan.claims) break;
      int share;
      const int ph = md_phase(plan, claim, &share);
      if (ph == 2) {
        // One warp per item of one token and 32 CPL columns: two columns a lane
        // where every item has a warp of the grid to itself, else eight.
        ok = args.tokens * ((K + 63) / 64) > 4 * shares
                 ? md_combine<T, 8>(args, plan, 4 * share + q, 4 * shares, lane, abort_flag)
                 : md_combine<T, 2>(args, plan, 4 * share + q, 4 * shares, lane, abort_flag);
        if (!ok) break;
        if (lane == 0) mbar_arrive(&qempty[qslot]);
        continue;
      }
      if (lane == 0) mbar_arrive(&qempty[qslot]);
      MdSegments sg = md_segments(plan, ph, share);
      bool stop = false;
      for (; sg.next(); ++i) {
        const int acc = i & 1;
        ok = mbar_wait(&tfull[acc], (i >> 1) & 1, abort_flag, 41);
        if (!__all_sync(0xffffffffu, ok)) {
          stop = true;
          break;
        }
        tc_fence_after();
        const uint32_t d0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                            static_cast<uint32_t>(acc * 2 * nt);
        const int a = ph == 0 ? sg.tile / plan.tiles1 : sg.tile % plan.active;
        const int row0 = plan.act_off[a], m = plan.act_off[a + 1] - row0;
        if (ph == 0) {
          const int col = (sg.tile % plan.tiles1) * 128 + lcol;
          const bool whole = sg.kb0 == 0 && sg.kb1 == plan.steps1;
          // A share's first segment, if it starts inside its tile, has slot 2 g;
          // its last, if the tile goes on after it, slot 2 g + 1.
          float* part = args.part + (2 * share + (sg.kb0 == 0)) * slot_floats;
          for (int r0 = 0; r0 < m; r0 += 8) {
            uint32_t gv[8], uv[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const uint32_t d = d0 + plan.row_token[row0 + min(r0 + r, m - 1)];
              gv[r] = tmem_ld_x1(d);
              uv[r] = tmem_ld_x1(d + nt);
            }
            tmem_ld_wait();
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const float g = __uint_as_float(gv[r]), u = __uint_as_float(uv[r]);
              if (r0 + r >= m) continue;
              if (whole) {
                if (col < I)
                  h[static_cast<size_t>(row0 + r0 + r) * I + col] =
                      Pack2<T>::from_float(g / (1.f + expf(-g)) * u);
              } else {
                part[(r0 + r) * 256 + lcol] = g;
                part[(r0 + r) * 256 + 128 + lcol] = u;
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[acc]);
          bool done = whole;
          if (!whole) {
            const int u = sg.tile * plan.steps1;
            const int s0 = md_share_of(u, plan.units1, plan.shares1);
            const int s1 = md_share_of(u + plan.steps1 - 1, plan.units1, plan.shares1);
            uint32_t seen = 0;
            __threadfence();
            __syncwarp();
            if (lane == 0)
              seen = atomicAdd(args.header + kMdCount1 + s0 * 4 + q,
                               static_cast<uint32_t>(sg.kb1 - sg.kb0)) + (sg.kb1 - sg.kb0);
            seen = __shfl_sync(0xffffffffu, seen, 0);
            if (seen == static_cast<uint32_t>(plan.steps1)) {
              done = true;
              __threadfence();
              // Share s0 starts at or before the tile: slot 2 s0 + 1; the others
              // 2 s.  32 loads in flight: one row of sixteen shares, or eight
              // rows of two.
              const float* from = args.part + lcol;
              auto slot_of = [&](int s) { return from + (2 * s + (s == s0)) * slot_floats; };
              auto finish = [&](int r, float g, float u) {
                if (col < I)
                  h[static_cast<size_t>(row0 + r) * I + col] =
                      Pack2<T>::from_float(g / (1.f + expf(-g)) * u);
              };
              if (m <= 2) {
                for (int r = 0; r < m; ++r) {
                  float g = 0.f, uu = 0.f;
                  for (int s = s0; s <= s1; s += 16) {
                    float v[16][2];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                      v[i][0] = s + i <= s1 ? __ldcg(slot_of(s + i) + r * 256) : 0.f;
                      v[i][1] = s + i <= s1 ? __ldcg(slot_of(s + i) + r * 256 + 128) : 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                      if (s + i <= s1) {
                        g += v[i][0];
                        uu += v[i][1];
                      }
                  }
                  finish(r, g, uu);
                }
              } else {
                for (int r0 = 0; r0 < m; r0 += 8) {
                  float g[8] = {}, uu[8] = {};
                  for (int s = s0; s <= s1; s += 2) {
                    const float* p0 = slot_of(s);
                    const float* p1 = slot_of(min(s + 1, s1));
                    float v[8][4];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                      const int at = min(r0 + r, m - 1) * 256;
                      v[r][0] = __ldcg(p0 + at);
                      v[r][1] = __ldcg(p0 + at + 128);
                      v[r][2] = __ldcg(p1 + at);
                      v[r][3] = __ldcg(p1 + at + 128);
                    }
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                      g[r] += v[r][0];
                      uu[r] += v[r][1];
                      if (s < s1) {
                        g[r] += v[r][2];
                        uu[r] += v[r][3];
                      }
                    }
                  }
#pragma unroll
                  for (int r = 0; r < 8; ++r)
                    if (r0 + r < m) finish(r0 + r, g[r], uu[r]);
                }
              }
            }
          }
          if (done) {
            __threadfence();
            fence_proxy_async_all();
            __syncwarp();
            if (lane == 0) atomicAdd(args.header + kMdDone1, 1u);
          }
        } else {
          // Rows m of y, 256 columns: the segment that starts the tile writes y,
          // a later one (always its share's first) slot 2 g.
          const int nb = sg.tile / plan.active;
          const bool owner = sg.kb0 == 0;
          const size_t step = owner ? static_cast<size_t>(K) : 256;
          float* dst = owner ? args.y + static_cast<size_t>(row0) * K + nb * 256
                             : args.part + 2 * share * slot_floats;
          const int left = owner ? K - nb * 256 : 256;  // columns of the block inside K
          for (int r0 = 0; r0 < m; r0 += 8) {
            uint32_t v0[8], v1[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const uint32_t d = d0 + min(r0 + r, m - 1);
              v0[r] = tmem_ld_x1(d);
              v1[r] = tmem_ld_x1(d + nt);
            }
            tmem_ld_wait();
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              if (r0 + r >= m) continue;
              float* p = dst + (r0 + r) * step + lcol;
              if (lcol < left) p[0] = __uint_as_float(v0[r]);
              if (lcol + 128 < left) p[128] = __uint_as_float(v1[r]);
            }
          }
          tc_fence_before();
          __threadfence();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&tempty[acc]);
            atomicAdd(args.header + kMdDone2, static_cast<uint32_t>(sg.kb1 - sg.kb0));
          }
        }
      }
      if (stop) break;
    }
  }

  // ------------------------------------------------------------ teardown
  if (warp == 0 && lane == 0 && *abort_flag) {
    // After a given-up wait: let copies in flight land before the CTA leaves.
    const uint64_t start = globaltimer_ns();
    while (globaltimer_ns() - start < 2000000ull) {
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

}  // namespace bokt
