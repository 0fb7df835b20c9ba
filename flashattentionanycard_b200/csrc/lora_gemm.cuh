// A shared projection with one low-rank adapter per token (sm_100a):
//   out[t] = x[t] W + s_a (x[t] A_a^T) B_a,   a = ids[t]  (a = -1: x[t] W alone)
// x [M, K], W [K, N], A [slots, R, K], B [slots, R, N], R the bank's padded rank.
//
// The adapters' second product joins the projection's own K loop: with
//   H_j[t] = s_a (x[t] A_a^T) where ids[t] = a_j, else 0
// for the adapters a_j of a row tile, the tile is x W + sum_j H_j B_{a_j}: the
// tile's accumulator runs R more k-values per adapter in use, 64 / R adapters to
// a 64-deep step, and nothing is read back or rounded in between.  H is rounded to the element type (it is a
// tensor-core operand).  The zeros of H_j meet B of other tokens' adapters, so
// B must be finite; the bank refuses adapters that are not.
//
//   lora_shrink_kernel  H (and each row tile's list of adapters) for few tokens.
//       Latency bound; a cluster per (row tile, adapter), its tokens gathered 16
//       at a time, K split over warps and CTAs; warp-level mma.sync on fragments
//       loaded straight from global memory (few flops: a 128-row tcgen05 tile
//       would idle on an adapter's handful of tokens).
//   lora_shrink_tc_kernel  the same for many tokens: bound by reading x; 128
//       tokens a cluster of four CTAs that split K, TMA ring and tcgen05.
//   lora_stream_kernel  few tokens, or few tiles (row tiles of up to 128): bound
//       by reading W.  W tiles are the 128-row operand and the tokens the narrow
//       one; a cluster of C CTAs splits K and reduces through distributed shared
//       memory.
//   lora_tc2_kernel     many tokens: the CTA-pair GEMM's 256 x 256 tiles.
// Both products start on x and W while the shrink kernel still runs (the stream
// on the SMs that hold a CTA of each, see kLoraShrinkSmem): it lets its
// dependents go only after its own wait, so everything before it is complete by
// then; they wait for it before the first H.
// Held in 16 bits: H.  Its scale is applied in fp32 before that rounding; in fp16
// the bank keeps both in range.  Scratch: H for min(slots, tile rows) adapters a
// row tile, whichever of them the batch uses.
// lora_shrink_kernel spills 8 bytes at rank 64 (128 registers for two CTAs an SM).
#pragma once

#include "bokt_device.cuh"
#include "gemm_tc2.cuh"
#include "moe_decode.cuh"

namespace bokt {

constexpr int kStatusBadAdapter = 6;
constexpr int kLoraMaxSlots = 1024;
constexpr int kLoraThreads = 256;
constexpr int kLoraPairRows = 256;  // row tile of lora_tc2_kernel

struct LoraArgs {
  int M, N, K, slots, rank;  // rank: padded (16, 32, 64 or 128)
  int tile_rows;             // row tile of the product: token columns, or 256
  int smax;                  // list entries per row tile (min(slots, tile_rows))
  const int32_t* ids;
  const int32_t* ranks;   // [slots], 0: empty slot
  const float* scales;    // [slots]
  int32_t* count;         // [row tiles] adapters in use
  int32_t* list;          // [row tiles][smax]
  void* h;                // [row tiles][gmax][tile_rows][64]: entry j's R columns start at
                          // column j R of the tile's gmax x 64
  void* out;
  int gmax;               // 64-wide groups of columns per row tile
  int walkers;            // shrink: clusters per row tile, each walking every walkers-th entry
  int cluster;            // CTAs per cluster of the kernel at hand
  int stages, group_m, chunks;
  int shrink_rows;        // lora_shrink_tc_kernel: tokens per cluster (at most 128, whole in a row tile)
  uint32_t idesc;
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1,
                                                         uint32_t a2, uint32_t a3, uint32_t b0,
                                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1,
                                                  uint32_t a2, uint32_t a3, uint32_t b0,
                                                  uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u32x4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                                 uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}

template <int RN>
__host__ __device__ constexpr int lora_shrink_smem_bytes() {
  return (8 + 1) * 16 * RN * 8 * 4;  // a partial per warp, their sum
}

// Cluster (row tile, w) takes the tile's list entries w, w + walkers, ...: for
// adapter a_j all rows of H_j, the products of its own tokens and zeros for the
// others.  The tokens are walked in groups of 16; kc CTAs of the cluster
// share a group and split its K (all of them for one group, one each for as
// many groups as CTAs).  A lane's 16-byte loads hold 8 neighbouring k-values of
// one row; two mma.sync take them as their k-fragments (the same k-order on
// both sides, so the dot products are whole).  Partial sums meet over the warps
// in shared memory and over the CTAs through distributed shared memory, in
// order.
template <typename T, int RN>
__global__ void __launch_bounds__(kLoraThreads, 2)
    lora_shrink_kernel(const T* x, const T* lora_a, const LoraArgs args) {
  constexpr int kTok = 16, kCols = RN * 8, NW = 8, kThreads = kLoraThreads;
  constexpr int kVotes = kLoraMaxSlots / kThreads;  // slots per lane
  extern __shared__ float sm[];
  float* part = sm;                      // [NW][kTok][kCols]
  float* local = sm + NW * kTok * kCols;  // [kTok][kCols]
  __shared__ int s_flag[kLoraMaxSlots];
  __shared__ int s_list[kLoraPairRows], s_id[kLoraPairRows], s_rows[kLoraPairRows], s_warp[NW];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = args.cluster;
  const int rank = static_cast<int>(cluster_ctarank());
  const int cluster = static_cast<int>(blockIdx.x) / C;
  const int mt = cluster / args.walkers, walker = cluster - mt * args.walkers;
  const int m0 = mt * args.tile_rows;
  const int rows = min(args.tile_rows, args.M - m0);  // at most 256, one per thread
  for (int i = tid; i < args.slots; i += kThreads) s_flag[i] = 0;
  cluster_sync();  // every CTA runs before another reads its shared memory
  pdl_wait();
  pdl_allow_next();
  // Which adapters the row tile uses, in slot order.
  int my_id = -1;
  if (tid < rows) {
    const int id = args.ids[m0 + tid];
    if (id >= 0 && id < args.slots && args.ranks[id] > 0) {
      my_id = id;
      s_flag[id] = 1;
    } else if (id != -1) {
      report_status(kStatusBadAdapter, m0 + tid);
    }
  }
  if (tid < kLoraPairRows) s_id[tid] = my_id;
  __syncthreads();
  int used[kVotes], mine = 0;
#pragma unroll
  for (int i = 0; i < kVotes; ++i) {
    const int slot = warp * 32 * kVotes + i * 32 + lane;
    const unsigned b = __ballot_sync(0xffffffffu, slot < args.slots && s_flag[slot]);
    used[i] = b >> lane & 1u ? mine + __popc(b & ((1u << lane) - 1u)) : -1;
    mine += __popc(b);
  }
  if (lane == 0) s_warp[warp] = mine;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    before += w < warp ? s_warp[w] : 0;
    total += s_warp[w];
  }
  const bool writes_list = rank == 0 && walker == 0;
  if (writes_list && tid == 0) args.count[mt] = total;
#pragma unroll
  for (int i = 0; i < kVotes; ++i)
    if (used[i] >= 0) {
      const int slot = warp * 32 * kVotes + i * 32 + lane;
      s_list[before + used[i]] = slot;
      if (writes_list) args.list[mt * args.smax + before + used[i]] = slot;
    }
  __syncthreads();

  const int g = lane >> 2, q = lane & 3;
  const T* xt = x + static_cast<size_t>(m0) * args.K;
  for (int j = walker; j < total; j += args.walkers) {
    const int id = s_list[j];
    T* h = static_cast<T*>(args.h) +
           (static_cast<size_t>(mt) * args.gmax + j * args.rank / 64) * args.tile_rows * 64 +
           j * args.rank % 64;  // column 0 of the entry; 64 columns on: the next group
    const size_t group = static_cast<size_t>(args.tile_rows) * 64;
    // The adapter's tokens, in row order.
    const bool own = my_id == id;
    const unsigned b = __ballot_sync(0xffffffffu, own);
    if (lane == 0) s_warp[warp] = __popc(b);
    __syncthreads();
    int at = __popc(b & ((1u << lane) - 1u)), tokens = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      at += w < warp ? s_warp[w] : 0;
      tokens += s_warp[w];
    }
    if (own) s_rows[at] = tid;
    __syncthreads();
    const int groups = (tokens + kTok - 1) / kTok;
    int kc = C;
    while (kc > 1 && C / kc < groups) kc >>= 1;
    const int sub = rank % kc, lead = rank - sub, stride = C / kc;
    const int own_rank = args.ranks[id];
    const float scale = args.scales[id];
    for (int r0 = 0; r0 < args.rank; r0 += 64) {
      const T* ar = lora_a + (static_cast<size_t>(id) * args.rank + r0 + g) * args.K + q * 8;
      for (int it = 0; it * stride < groups; ++it) {
        const int t0 = (it * stride + rank / kc) * kTok;
        const T* xr[2];  // rows g, g + 8, ... of the group (past its end: dropped below)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          xr[i] = xt + static_cast<size_t>(s_rows[t0 + 8 * i + g < tokens ? t0 + 8 * i + g : 0]) * args.K + q * 8;
        float acc[RN][4] = {};
        if (t0 < tokens) {
#pragma unroll 2
          for (int k = (sub * NW + warp) * 32; k < args.K; k += kc * NW * 32) {
            const bool in = k + q * 8 < args.K;  // K is a multiple of 8
            uint4 xa[2], bv[RN];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              xa[i] = in ? *reinterpret_cast<const uint4*>(xr[i] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int n = 0; n < RN; ++n)
              bv[n] = in ? *reinterpret_cast<const uint4*>(ar + static_cast<size_t>(n) * 8 * args.K + k)
                         : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int n = 0; n < RN; ++n) {
              mma_16816<T>(acc[n], xa[0].x, xa[1].x, xa[0].y, xa[1].y, bv[n].x, bv[n].y);
              mma_16816<T>(acc[n], xa[0].z, xa[1].z, xa[0].w, xa[1].w, bv[n].z, bv[n].w);
            }
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int n = 0; n < RN; ++n)
            *reinterpret_cast<float2*>(part + (warp * kTok + 8 * half + g) * kCols + n * 8 + 2 * q) =
                make_float2(acc[n][2 * half], acc[n][2 * half + 1]);
        __syncthreads();
        for (int i = tid; i < kTok * kCols; i += kThreads) {
          const int row = i / kCols, c = i % kCols;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < NW; ++w) sum += part[(w * kTok + row) * kCols + c];
          local[row * kCols + c] = sum;
        }
        if (kc > 1) cluster_sync();
        else __syncthreads();
        for (int i = sub * kThreads + tid; i < kTok * kCols / 2; i += kc * kThreads) {
          const int row = i / (kCols / 2), c = i % (kCols / 2) * 2;
          if (t0 + row >= tokens) continue;
          float2 sum = make_float2(0.f, 0.f);
          if (kc > 1) {
            const uint32_t a = smem_addr(local + row * kCols + c);
            for (int p = 0; p < kc; ++p) {
              const float2 v = ld_cluster_f32x2(map_shared(a, lead + p));
              sum.x += v.x;
              sum.y += v.y;
            }
          } else {
            sum = *reinterpret_cast<const float2*>(local + row * kCols + c);
          }
          // Past the adapter's own rank H is 0 whatever x holds.
          sum.x = r0 + c < own_rank ? sum.x * scale : 0.f;
          sum.y = r0 + c + 1 < own_rank ? sum.y * scale : 0.f;
          *reinterpret_cast<uint32_t*>(h + r0 / 64 * group + s_rows[t0 + row] * 64 + c) =
              Pack2<T>::pack(sum.x, sum.y);
        }
        // The sums are read before the next ones overwrite them, or the CTA leaves.
        if (kc > 1) cluster_sync();
        else __syncthreads();
      }
    }
    // Zeros where the tile's other tokens meet this adapter.
    const int vecs = args.rank / 8;
    for (int i = rank * kThreads + tid; i < rows * vecs; i += C * kThreads) {
      const int row = i / vecs, c = (i - row * vecs) * 8;
      if (s_id[row] != id)
        *reinterpret_cast<uint4*>(h + c / 64 * group + row * 64 + c % 64) = make_uint4(0, 0, 0, 0);
    }
  }
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

constexpr int kLoraShrinkRows = 128, kLoraShrinkSplit = 4;  // tokens and CTAs of a cluster
constexpr int kLoraShrinkCols = 128;                        // accumulator columns of a pass
constexpr int kLoraShrinkStage = (kLoraShrinkRows + kLoraShrinkCols) * 128;

__host__ __device__ inline int lora_shrink_tc_smem_bytes(int stages, int rank) {
  return 1024 + stages * kLoraShrinkStage + kLoraShrinkSplit * 32 * rank * 4 + (2 * stages + 4) * 8 + 16;
}

// H and the lists, many tokens.  A cluster takes shrink_rows tokens (a row tile,
// or half a pair's); CTA r runs a quarter of K: x as the 128-row operand, the A
// rows of the adapters that these tokens use as the narrow one, 128 columns
// (128 / R adapters) a pass, two accumulators.  A token keeps the columns of its
// own adapter, so all passes fill one [tokens][R] buffer in distributed shared
// memory: CTA r collects the quarters of tokens [32 r, +32), and after one
// cluster barrier sums them in rank order.
template <typename T>
__global__ void __launch_bounds__(kLoraThreads, 1)
    lora_shrink_tc_kernel(const __grid_constant__ CUtensorMap tm_x,
                          const __grid_constant__ CUtensorMap tm_a, const LoraArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stages = args.stages;
  const int R = args.rank, rs = min(R, 64);
  float* recv = reinterpret_cast<float*>(smem + stages * kLoraShrinkStage);  // [4][32][R]
  uint64_t* full = reinterpret_cast<uint64_t*>(recv + kLoraShrinkSplit * 32 * R);
  uint64_t* empty = full + stages;
  uint64_t* tfull = empty + stages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  __shared__ int s_flag[kLoraMaxSlots];  // 1 used by the row tile, 3 also by these tokens; then the place
  __shared__ int s_slot[kLoraShrinkRows];  // the adapters of these tokens
  __shared__ int s_id[kLoraShrinkRows], s_own[kLoraShrinkRows], s_warp[8], s_mine[8];
  __shared__ float s_scale[kLoraShrinkRows];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int rank = static_cast<int>(cluster_ctarank());
  const int per = args.shrink_rows;
  const int t0 = static_cast<int>(blockIdx.x) / kLoraShrinkSplit * per;
  const int mt = t0 / args.tile_rows, m0 = mt * args.tile_rows;
  const int nkb = (args.K + 63) / 64;
  const int kb0 = rank * nkb / kLoraShrinkSplit, kb1 = (rank + 1) * nkb / kLoraShrinkSplit;

  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_a);
  }
  if (warp == 3) {
    tmem_alloc(tmem_holder, 2 * kLoraShrinkCols);
    tmem_relinquish();
  }
  for (int i = tid; i < args.slots; i += kLoraThreads) s_flag[i] = 0;
  cluster_sync();  // every CTA runs before another writes its shared memory
  pdl_wait();
  pdl_allow_next();
  // Adapters of the row tile (at most 256 rows, one per thread) and of these tokens.
  int my_id = -1;
  const bool here = m0 + tid >= t0 && m0 + tid < t0 + per;
  if (tid < args.tile_rows && m0 + tid < args.M) {
    const int id = args.ids[m0 + tid];
    const int own_rank = id >= 0 && id < args.slots ? args.ranks[id] : 0;
    if (own_rank > 0) {
      my_id = id;
      atomicOr(&s_flag[id], here ? 3 : 1);
      if (here) {
        s_own[m0 + tid - t0] = own_rank;
        s_scale[m0 + tid - t0] = args.scales[id];
      }
    } else if (id != -1 && here && rank == 0) {
      report_status(kStatusBadAdapter, m0 + tid);
    }
  }
  if (here) s_id[m0 + tid - t0] = my_id;
  if (tid >= per && tid < kLoraShrinkRows) s_id[tid] = -1;
  __syncthreads();
  int place[4], mine[4], used = 0, own = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = warp * 128 + i * 32 + lane;
    const int f = slot < args.slots ? s_flag[slot] : 0;
    const unsigned b = __ballot_sync(0xffffffffu, f != 0), c = __ballot_sync(0xffffffffu, f == 3);
    const unsigned below = (1u << lane) - 1u;
    place[i] = f != 0 ? used + __popc(b & below) : -1;
    mine[i] = f == 3 ? own + __popc(c & below) : -1;
    used += __popc(b);
    own += __popc(c);
  }
  if (lane == 0) {
    s_warp[warp] = used;
    s_mine[warp] = own;
  }
  __syncthreads();
  int before = 0, total = 0, before_own = 0, adapters = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    before += w < warp ? s_warp[w] : 0;
    before_own += w < warp ? s_mine[w] : 0;
    total += s_warp[w];
    adapters += s_mine[w];
  }
  const bool writes_list = rank == 0 && t0 == m0;
  if (writes_list && tid == 0) args.count[mt] = total;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = warp * 128 + i * 32 + lane;
    if (place[i] < 0) continue;
    s_flag[slot] = before + place[i];
    if (writes_list) args.list[mt * args.smax + before + place[i]] = slot;
    if (mine[i] >= 0) s_slot[before_own + mine[i]] = slot;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  T* h = static_cast<T*>(args.h) + static_cast<size_t>(mt) * args.gmax * args.tile_rows * 64;
  const size_t group = static_cast<size_t>(args.tile_rows) * 64;
  const int per_pass = kLoraShrinkCols / R;
  const int passes = kb1 > kb0 ? (adapters + per_pass - 1) / per_pass : 0;
  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int p = 0; p < passes; ++p) {
        const int p0 = p * per_pass, cols = min(per_pass, adapters - p0) * R;
        for (int kb = kb0; ok && kb < kb1; ++kb) {
          if (!(ok = mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 71))) break;
          uint8_t* b = smem + stage * kLoraShrinkStage;
          mbar_arrive_expect_tx(&full[stage], per * 128 + cols * 128);
          tma_load_2d(b, &tm_x, &full[stage], kb * 64, t0);
          b += kLoraShrinkRows * 128;
          for (int c = 0; c < cols; c += rs)
            tma_load_2d(b + c * 128, &tm_a, &full[stage], kb * 64, s_slot[p0 + c / R] * R + c % R);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int p = 0; ok && p < passes; ++p) {
        const int cols = min(per_pass, adapters - p * per_pass) * R;
        const uint32_t idesc = args.idesc | (static_cast<uint32_t>(cols >> 3) << 17);
        if (!(ok = mbar_wait(&tempty[p & 1], (p >> 1 & 1) ^ 1, abort_flag, 74))) break;
        tc_fence_after();
        const uint32_t d = tmem_base + (p & 1) * kLoraShrinkCols;
        for (int kb = kb0; ok && kb < kb1; ++kb) {
          if (!(ok = mbar_wait(&full[stage], phase, abort_flag, 72))) break;
          tc_fence_after();
          const uint32_t a = smem_addr(smem + stage * kLoraShrinkStage);
          const uint32_t b = a + kLoraShrinkRows * 128;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ss(d, smem_desc_sw128(a + k * 32, 16, 1024), smem_desc_sw128(b + k * 32, 16, 1024),
                        idesc, kb != kb0 || k != 0 ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit(&tfull[p & 1]);
      }
    }
  } else if (warp >= 4) {
    // Warp q holds tokens [32 q, +32), a lane each; their sums go to CTA q.
    const int q = warp & 3;
    const int id = s_id[q * 32 + lane];
    const uint32_t at = map_shared(smem_addr(recv + (rank * 32 + lane) * R), q);
    if (kb1 == kb0 && id >= 0)  // without k-steps this CTA's part of the sum is 0
      for (int c = 0; c < R; c += 4) st_cluster_u32x4(at + c * 4, 0u, 0u, 0u, 0u);
    for (int p = 0; p < passes; ++p) {
      const int p0 = p * per_pass, na = min(per_pass, adapters - p0);
      const bool done = mbar_wait(&tfull[p & 1], p >> 1 & 1, abort_flag, 73);
      if (!__all_sync(0xffffffffu, done)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + (p & 1) * kLoraShrinkCols;
      for (int e = 0; e < na; ++e) {
        const bool is_mine = s_slot[p0 + e] == id;
        if (!__any_sync(0xffffffffu, is_mine)) continue;
        for (int c = 0; c < R; c += 16) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(d + e * R + c, v);
          tmem_ld_wait();
          if (is_mine) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              st_cluster_u32x4(at + (c + j) * 4, v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[p & 1]);
    }
  }
  __syncwarp();
  cluster_sync();  // all quarters of this CTA's tokens are here
  for (int i = tid; i < 32 * R / 2; i += kLoraThreads) {
    const int tok = i / (R / 2), c = i % (R / 2) * 2, row = rank * 32 + tok;
    const int id = s_id[row];
    if (id < 0) continue;
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int s = 0; s < kLoraShrinkSplit; ++s) {
      const float2 v = *reinterpret_cast<const float2*>(recv + (s * 32 + tok) * R + c);
      sum.x += v.x;
      sum.y += v.y;
    }
    // Past the adapter's own rank H is 0 whatever x holds.
    sum.x = c < s_own[row] ? sum.x * s_scale[row] : 0.f;
    sum.y = c + 1 < s_own[row] ? sum.y * s_scale[row] : 0.f;
    const int col = s_flag[id] * R + c;
    *reinterpret_cast<uint32_t*>(h + col / 64 * group + (t0 - m0 + row) * 64 + col % 64) =
        Pack2<T>::pack(sum.x, sum.y);
  }
  // Zeros where a token meets another adapter of its row tile.
  const int vecs = R / 8;
  for (int i = tid; i < 32 * total * vecs; i += kLoraThreads) {
    const int v = i % vecs, e = i / vecs % total, tok = rank * 32 + i / (vecs * total);
    if (tok >= per || t0 + tok >= args.M || (s_id[tok] >= 0 && s_flag[s_id[tok]] == e)) continue;
    const int col = e * R + v * 8;
    *reinterpret_cast<uint4*>(h + col / 64 * group + (t0 - m0 + tok) * 64 + col % 64) = make_uint4(0, 0, 0, 0);
  }
  if (*abort_flag && tid == 0) {
    // After a given-up wait: let copies in flight land before the CTA leaves.
    const uint64_t start = globaltimer_ns();
    while (globaltimer_ns() - start < 2000000ull) {
    }
  }
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * kLoraShrinkCols);
  }
}

__host__ __device__ inline int lora_stream_smem_bytes(int nt, int stages) {
  return 1024 + stages * (kMdStageW + nt * 256) + (2 * stages + 3) * 8 + 16 + kLoraPairRows * 4;
}

// 128 columns x tile_rows tokens per cluster of C CTAs.  CTA r runs the k-steps
// (128 deep: four 64 x 64 boxes of W, two of x) and the list entries of its
// share of both, and the accumulators are reduce-scattered over the tokens
// through distributed shared memory (the ring's, free by then), summed in rank
// order.  The ring holds 100-190 KB of loads in flight per SM.
template <typename T>
__global__ void __launch_bounds__(kLoraThreads, 1)
    lora_stream_kernel(const __grid_constant__ CUtensorMap tm_w,
                       const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ CUtensorMap tm_b,
                       const __grid_constant__ CUtensorMap tm_h, const LoraArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stages = args.stages, nt = args.tile_rows, C = args.cluster;
  const int stage_b = nt * 256;
  uint8_t* sW = smem;
  uint8_t* sB = sW + stages * kMdStageW;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + stages * stage_b);
  uint64_t* empty = full + stages;
  uint64_t* tfull = empty + stages;
  uint64_t* listed = tfull + 1;
  uint64_t* issued = listed + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(issued + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile int* s_width = reinterpret_cast<volatile int*>(tmem_holder + 2);
  volatile int* s_slot = reinterpret_cast<volatile int*>(tmem_holder + 4);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / C;
  const int chunk = tile % args.chunks, n0 = tile / args.chunks * 128;
  const int ksteps = (args.K + 127) / 128;
  const int kb0 = rank * ksteps / C, kb1 = (rank + 1) * ksteps / C;
  const int R = args.rank, rs = min(R, 64);  // rs: rows of B in one box
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(nt)) tmem_cols *= 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_init(listed, 1);
    mbar_init(issued, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_b);
    tma_prefetch_desc(&tm_h);
  }
  if (warp == 3) {
    tmem_alloc(tmem_holder, tmem_cols);
    tmem_relinquish();
  }
  pdl_allow_next();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  // This CTA's share of the row tile's list, known once the shrink kernel is
  // done: warp 3 brings the slots into shared memory in one round of loads.
  if (warp == 3) {
    pdl_wait();
    const int n = __ldcg(args.count + chunk);
    for (int i = lane; i < n; i += 32) s_slot[i] = __ldcg(args.list + chunk * args.smax + i);
    if (lane == 0) *s_width = n * R;
    __syncwarp();
    if (lane == 0) mbar_arrive(listed);
  }
  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 51))) break;
        uint8_t* w = sW + stage * kMdStageW;
        mbar_arrive_expect_tx(&full[stage], kMdStageW);
        tma_load_2d(w, &tm_w, &full[stage], n0, kb * 128);
        tma_load_2d(w + 8192, &tm_w, &full[stage], n0 + 64, kb * 128);
        tma_load_2d(w + 16384, &tm_w, &full[stage], n0, kb * 128 + 64);
        tma_load_2d(w + 24576, &tm_w, &full[stage], n0 + 64, kb * 128 + 64);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) {
        mbar_arrive(issued);
        ok = mbar_wait(listed, 0, abort_flag, 57);
      }
      const int cols = ok ? *s_width : 0, groups = (cols + 63) / 64;
      for (int i = rank * groups / C; i < (rank + 1) * groups / C; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 52)) break;
        mbar_arrive_expect_tx(&full[stage], min(64, cols - i * 64) * 256);  // from warps 4-7
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 2) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 53))) break;
        uint8_t* b = sB + stage * stage_b;
        mbar_arrive_expect_tx(&full[stage], nt * 256);
        tma_load_2d(b, &tm_x, &full[stage], kb * 128, chunk * nt);
        tma_load_2d(b + nt * 128, &tm_x, &full[stage], kb * 128 + 64, chunk * nt);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) ok = mbar_wait(listed, 0, abort_flag, 58);
      const int cols = ok ? *s_width : 0, groups = (cols + 63) / 64;
      pdl_wait();
      fence_proxy_async_all();  // H was stored by ordinary stores
      for (int i = rank * groups / C; i < (rank + 1) * groups / C; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 54)) break;
        mbar_arrive_expect_tx(&full[stage], nt * 128);
        tma_load_2d(sB + stage * stage_b, &tm_h, &full[stage], 0, (chunk * args.gmax + i) * nt);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0, on = 0;
      bool ok = true;
      // ksub 16-deep MMAs on one filled stage.
      auto step = [&](int ksub) {
        if (!mbar_wait(&full[stage], phase, abort_flag, 55)) return false;
        tc_fence_after();
        const uint32_t w = smem_addr(sW + stage * kMdStageW);
        const uint32_t b = smem_addr(sB + stage * stage_b);
        for (int k = 0; k < ksub; ++k) {
          const uint32_t wk = w + (k >> 2) * 16384 + (k & 3) * 2048;
          const uint32_t bk = b + (k >> 2) * nt * 128 + (k & 3) * 32;
          umma_f16_ss(tmem_base, smem_desc_sw128(wk, 8192, 1024), smem_desc_sw128(bk, 16, 1024),
                      args.idesc, on);
          on = 1;
        }
        umma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
        return true;
      };
      for (int kb = kb0; ok && kb < kb1; ++kb) ok = step(8);
      if (ok) ok = mbar_wait(listed, 0, abort_flag, 59);
      const int cols = ok ? *s_width : 0, groups = (cols + 63) / 64;
      for (int i = rank * groups / C; ok && i < (rank + 1) * groups / C; ++i)
        ok = step(min(64, cols - i * 64) / 16);
      if (ok) umma_commit(tfull);
    }
  }
  if (warp >= 4) {
    // The B rows of a 64-deep step: up to four adapters of two boxes each, one
    // adapter per warp (issued by one thread they take longer than to arrive).
    // A parity wait tells neighbouring uses of a stage apart only, so these
    // start when warp 0 has issued, and so waited for, every k-step before them.
    if (elect_one() && mbar_wait(listed, 0, abort_flag, 60) && mbar_wait(issued, 0, abort_flag, 62)) {
      const int cols = *s_width, groups = (cols + 63) / 64;
      const int g0 = rank * groups / C, g1 = (rank + 1) * groups / C;
      for (int i = g0; i < g1; ++i) {
        const int c = i * 64 + (warp - 4) * rs;
        if ((warp - 4) * rs >= 64 || c >= cols) break;
        const int step = kb1 - kb0 + i - g0, stage = step % stages;
        if (!mbar_wait(&empty[stage], (step / stages & 1) ^ 1, abort_flag, 61)) break;
        uint8_t* w = sW + stage * kMdStageW + (warp - 4) * rs * 128;
        const int slot = s_slot[c / R];
        tma_load_3d(w, &tm_b, &full[stage], n0, c % R, slot);
        tma_load_3d(w + 8192, &tm_b, &full[stage], n0 + 64, c % R, slot);
      }
    }
  }
  __syncwarp();
  const bool ok = mbar_wait(tfull, 0, abort_flag, 56);
  pdl_wait();
  if (*abort_flag && threadIdx.x == 0) {
    // After a given-up wait: let copies in flight land before the memory is reused.
    const uint64_t start = globaltimer_ns();
    while (globaltimer_ns() - start < 2000000ull) {
    }
  }
  __syncthreads();
  cluster_sync();  // every CTA of the cluster has consumed its ring
  // [C sources][tokens of this rank / 4][128 columns][4 tokens]
  float* recv = reinterpret_cast<float*>(sW);
  const int own = nt / C;
  if (warp >= 4 && __all_sync(0xffffffffu, ok)) {
    tc_fence_after();
    const int q = warp & 3;
    const uint32_t mine = smem_addr(recv + rank * own * 128 + (q * 32 + lane) * 4);
    uint32_t to = 0, at = map_shared(mine, 0), left = own;
    for (int c = 0; c < nt; c += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        st_cluster_u32x4(at, v[j], v[j + 1], v[j + 2], v[j + 3]);
        at += 4 * 128 * 4;
        left -= 4;
        if (left == 0 && c + j + 4 < nt) {
          at = map_shared(mine, ++to);
          left = own;
        }
      }
    }
    tc_fence_before();
  }
  cluster_sync();
  T* out = static_cast<T*>(args.out);
  const int row0 = chunk * nt + rank * own;
  for (int i = threadIdx.x; i < own * 16; i += kLoraThreads) {
    const int tok = (i >> 6) * 4, c = (i & 63) * 2;
    if (row0 + tok >= args.M || n0 + c >= args.N) continue;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;  // four tokens of columns c, c + 1
    for (int s = 0; s < C; ++s) {
      const float4* p = reinterpret_cast<const float4*>(recv + (s * own + tok) * 128 + c * 4);
      const float4 va = p[0], vb = p[1];
      a.x += va.x, a.y += va.y, a.z += va.z, a.w += va.w;
      b.x += vb.x, b.y += vb.y, b.z += vb.z, b.w += vb.w;
    }
    const uint32_t pk[4] = {Pack2<T>::pack(a.x, b.x), Pack2<T>::pack(a.y, b.y),
                            Pack2<T>::pack(a.z, b.z), Pack2<T>::pack(a.w, b.w)};
    T* o = out + static_cast<size_t>(row0 + tok) * args.N + n0 + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (row0 + tok + j < args.M) *reinterpret_cast<uint32_t*>(o + static_cast<size_t>(j) * args.N) = pk[j];
  }
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

__host__ __device__ inline int lora_tc2_smem_bytes(int stages) {
  return 1024 + stages * GemmTc2Shape<256>::kStageBytes + kEpiBytes + (2 * stages + 4) * 8 + 16;
}

// The dense CTA-pair GEMM (gemm_tc2.cuh: 256 x 256 pair tiles, GROUP_M raster,
// two accumulators) with the row tile's adapters appended to each tile's K
// loop: per 64 columns of H, 128 of its rows and 64 rows of B per CTA.  Tensor
// bound: an adapter costs R / 64 of a k-step.
template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
    lora_tc2_kernel(const __grid_constant__ CUtensorMap tm_x,
                    const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_h,
                    const __grid_constant__ CUtensorMap tm_b, const LoraArgs args) {
  constexpr int BN = 256;
  using Shape = GemmTc2Shape<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stages = args.stages;
  uint8_t* sA = smem;
  uint8_t* sB = smem + stages * kGemmABytes;
  uint8_t* sEpi = sB + stages * Shape::kBBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sEpi + kEpiBytes);
  uint64_t* empty = full + stages;
  uint64_t* tfull = empty + stages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int M = args.M, N = args.N;
  const int nm = (M + kLoraPairRows - 1) / kLoraPairRows, nn = (N + BN - 1) / BN;
  const int ntiles = nm * nn;
  const int nkb = (args.K + kGemmBK - 1) / kGemmBK;
  const int R = args.rank, rs = min(R, 64);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_h);
    tma_prefetch_desc(&tm_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, Shape::kTmemCols);
    tmem_relinquish_pair();
  }
  pdl_allow_next();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  auto tile_at = [&](int t, int* pm, int* n0) {
    const int per_group = args.group_m * nn;
    const int group = t / per_group;
    const int first_m = group * args.group_m;
    const int gm = min(nm - first_m, args.group_m);
    const int local = t - group * per_group;
    *pm = first_m + local % gm;
    *n0 = local / gm * BN;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producers (both CTAs)
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0, t = pair; ok && t < ntiles; ++i, t += npairs) {
        int pm, n0;
        tile_at(t, &pm, &n0);
        const int row = pm * kLoraPairRows + rank * kGemmBM;
        const int col = n0 + rank * Shape::kBHalf;
        for (int kk = 0; kk < nkb; ++kk) {
          const int kb = (i & 1) ? nkb - 1 - kk : kk;  // odd waves walk K downwards (L2 reuse)
          if (!(ok = mbar_wait_cluster(&empty[stage], phase ^ 1u, abort_flag, 61))) break;
          const uint32_t bar = map_shared(smem_addr(&full[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * Shape::kStageBytes);
          tma_load_2d_pair(sA + stage * kGemmABytes, &tm_x, bar, kb * kGemmBK, row);
          tma_load_2d_pair(sB + stage * Shape::kBBytes, &tm_w, bar, col, kb * kGemmBK);
          tma_load_2d_pair(sB + stage * Shape::kBBytes + 8192, &tm_w, bar, col + 64, kb * kGemmBK);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (i == 0) {
          pdl_wait();
          fence_proxy_async_all();  // H was stored by ordinary stores
        }
        const int cols = __ldcg(args.count + pm) * R;
        int next = __ldcg(args.list + pm * args.smax);
        for (int c0 = 0; c0 < cols; c0 += 64) {
          if (!(ok = mbar_wait_cluster(&empty[stage], phase ^ 1u, abort_flag, 62))) break;
          const uint32_t bar = map_shared(smem_addr(&full[stage]), 0);
          const int c1 = min(cols, c0 + 64);
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * (kGemmABytes + (c1 - c0) * 256));
          tma_load_2d_pair(sA + stage * kGemmABytes, &tm_h, bar, 0,
                           (pm * args.gmax + c0 / 64) * kLoraPairRows + rank * kGemmBM);
          uint8_t* b = sB + stage * Shape::kBBytes;
          for (int c = c0; c < c1; c += rs, b += rs * 128) {
            const int slot = next;
            if (c + rs < cols) next = __ldcg(args.list + pm * args.smax + (c + rs) / R);
            tma_load_3d_pair(b, &tm_b, bar, col, c % R, slot);
            tma_load_3d_pair(b + 8192, &tm_b, bar, col + 64, c % R, slot);
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0, t = pair; ok && t < ntiles; ++i, t += npairs) {
        int pm, n0;
        tile_at(t, &pm, &n0);
        const int acc = i & 1;
        if (!mbar_wait_cluster(&tempty[acc], ((i >> 1) & 1) ^ 1, abort_flag, 63)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
        auto step = [&](int ksub, bool first) {
          if (!mbar_wait_cluster(&full[stage], phase, abort_flag, 64)) return false;
          tc_fence_after();
          const uint32_t a = smem_addr(sA + stage * kGemmABytes);
          const uint32_t b = smem_addr(sB + stage * Shape::kBBytes);
          for (int k = 0; k < ksub; ++k)
            umma_f16_ss_pair(d, smem_desc_sw128(a + k * 32, 16, 1024),
                             smem_desc_sw128(b + k * 2048, 8192, 1024), args.idesc,
                             first && k == 0 ? 0u : 1u);
          umma_commit_both(&empty[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
          return true;
        };
        for (int kb = 0; ok && kb < nkb; ++kb) ok = step(4, kb == 0);
        if (!ok) break;
        if (i == 0) pdl_wait();
        const int cols = __ldcg(args.count + pm) * R;
        for (int c = 0; ok && c < cols; c += 64) ok = step(min(64, cols - c) / 16, false);
        if (ok) umma_commit_both(&tfull[acc]);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;
    T* C = static_cast<T*>(args.out);
    uint8_t* stage = sEpi + (warp - 2) * kEpiStageBytes;
    T** rowptr = reinterpret_cast<T**>(sEpi + kEpiWarps * kEpiStageBytes) + (warp - 2) * 32;
    for (int i = 0, t = pair; t < ntiles; ++i, t += npairs) {
      int pm, n0;
      tile_at(t, &pm, &n0);
      const int acc = i & 1;
      const bool ok = mbar_wait_cluster(&tfull[acc], (i >> 1) & 1, abort_flag, 65);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (i == 0) pdl_wait();
      tc_fence_after();
      const uint32_t taddr =
          tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN);
      const int row = pm * kLoraPairRows + rank * kGemmBM + q * 32 + lane;
      rowptr[lane] = row < M ? C + static_cast<size_t>(row) * N + n0 : nullptr;
      __syncwarp();
      epilogue_store_tile<BN, T>(taddr, stage, rowptr, n0, N, lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(map_shared(smem_addr(&tempty[acc]), 0));
    }
  }

  // ---------------------------------------------------------------- teardown
  __syncwarp();
  pdl_wait();
  if (*abort_flag && threadIdx.x == 0) {
    // After a given-up wait: let copies in flight land before the CTA leaves.
    const uint64_t start = globaltimer_ns();
    while (globaltimer_ns() - start < 2000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still signal its barriers
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, Shape::kTmemCols);
  }
}

}  // namespace bokt
