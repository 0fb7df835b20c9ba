// A shared projection with one low-rank adapter per token (sm_100a):
//   out[t] = x[t] W + s_a (x[t] A_a^T) B_a,   a = ids[t]  (a = -1: x[t] W alone)
// x [M, K], W [K, N], A [slots, R, K], B [slots, R, N], R the bank's padded rank.
//
// The adapters' second product joins the projection's own K loop: with
//   H_j[t] = s_a (x[t] A_a^T) where ids[t] = a_j, else 0
// for the adapters a_j of a row tile, the tile is x W + sum_j H_j B_{a_j}: the
// tile's accumulator runs R more k-values per adapter in use, and nothing is
// read back or rounded in between.  H is rounded to the element type (it is a
// tensor-core operand).  The zeros of H_j meet B of other tokens' adapters, so
// B must be finite; the bank refuses adapters that are not.
//
//   lora_shrink_kernel  H (and each row tile's list of adapters).  HBM / latency
//       bound; 16 or 32 tokens a cluster, K split over its warps and CTAs,
//       warp-level mma.sync on fragments loaded straight from global memory
//       (few flops: a tcgen05 tile would idle on 16 columns).
//   lora_stream_kernel  few tokens (row tiles of up to 128): bound by reading W.
//       W tiles are the 128-row operand and the tokens the narrow one; a cluster
//       of C CTAs splits K and reduces through distributed shared memory.
//   lora_tc2_kernel     many tokens: the CTA-pair GEMM's 256 x 256 tiles.
// Both products start on x and W while the shrink kernel still runs: it lets
// its dependents go only after its own wait, so everything before it is
// complete by then; they wait for it before the first H.
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
  void* h;                // [row tiles][smax][tile_rows][64 * parts]
  void* out;
  int parts;              // 64-wide parts of a row of H (1 or 2)
  int cluster;            // CTAs per cluster of the kernel at hand
  int stages, group_m, chunks;
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

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <int MT>
__host__ __device__ constexpr int lora_shrink_smem_bytes() {
  return (8 + 1) * 16 * MT * 64 * 4;  // one partial per warp, their sum
}

// One cluster per 16 MT tokens.  A lane's 16-byte loads hold 8 neighbouring
// k-values of one row; two mma.sync take them as their k-fragments (the same
// k-order on both sides, so the dot products are whole).  Only the rows of the
// adapter at hand are kept, so the partials of all adapters of the tile share
// one [tokens][64] buffer per warp and are reduced once: over the warps in
// shared memory, over the cluster through distributed shared memory, in order.
template <typename T, int MT, int RN>
__global__ void __launch_bounds__(kLoraThreads) lora_shrink_kernel(const T* x, const T* lora_a,
                                                                   const LoraArgs args) {
  constexpr int kTok = 16 * MT;
  extern __shared__ float sm[];
  float* part = sm;                  // [8][kTok][64]
  float* local = sm + 8 * kTok * 64;  // [kTok][64]
  __shared__ int s_flag[kLoraMaxSlots];  // 1: in use; then its place in the list
  __shared__ int s_id[kTok], s_uniq[kTok], s_warp[8], s_nuniq;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = args.cluster;
  const int rank = static_cast<int>(cluster_ctarank());
  const int t0 = static_cast<int>(blockIdx.x) / C * kTok;
  const int mt = t0 / args.tile_rows, m0 = mt * args.tile_rows;
  for (int i = tid; i < args.slots; i += kLoraThreads) s_flag[i] = 0;
  cluster_sync();  // every CTA runs before another reads its shared memory
  pdl_wait();
  pdl_allow_next();
  // The product's row tile: which adapters it uses, in slot order.
  for (int i = tid; i < args.tile_rows && m0 + i < args.M; i += kLoraThreads) {
    const int id = args.ids[m0 + i];
    const bool ok = id >= 0 && id < args.slots && args.ranks[id] > 0;
    if (ok) s_flag[id] = 1;
    else if (id != -1 && m0 + i >= t0 && m0 + i < t0 + kTok) report_status(kStatusBadAdapter, m0 + i);
    if (m0 + i >= t0 && m0 + i < t0 + kTok) s_id[m0 + i - t0] = ok ? id : -1;
  }
  for (int i = tid; i < kTok; i += kLoraThreads)
    if (t0 + i >= args.M) s_id[i] = -1;
  __syncthreads();
  int used[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = warp * 128 + i * 32 + lane;
    const unsigned b = __ballot_sync(0xffffffffu, slot < args.slots && s_flag[slot]);
    used[i] = b >> lane & 1u ? mine + __popc(b & ((1u << lane) - 1u)) : -1;
    mine += __popc(b);
  }
  if (lane == 0) s_warp[warp] = mine;
  if (warp == 0) {  // distinct adapters of this cluster's tokens
    const int id = lane < kTok ? s_id[lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    const bool first = id >= 0 && (same & ((1u << lane) - 1u)) == 0;
    const unsigned b = __ballot_sync(0xffffffffu, first);
    if (first) s_uniq[__popc(b & ((1u << lane) - 1u))] = id;
    if (lane == 0) s_nuniq = __popc(b);
  }
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    before += w < warp ? s_warp[w] : 0;
    total += s_warp[w];
  }
  const bool writes_list = rank == 0 && t0 == m0;
  if (writes_list && tid == 0) args.count[mt] = total;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (used[i] >= 0) {
      const int slot = warp * 128 + i * 32 + lane;
      s_flag[slot] = before + used[i];
      if (writes_list) args.list[mt * args.smax + before + used[i]] = slot;
    }
  __syncthreads();

  const int g = lane >> 2, q = lane & 3;
  const int width = 64 * args.parts;
  T* h = static_cast<T*>(args.h) + static_cast<size_t>(mt) * args.smax * args.tile_rows * width;
  const T* xr[2 * MT];  // rows g, g + 8, ... of the tile (past M: row 0, dropped below)
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i)
    xr[i] = x + static_cast<size_t>(t0 + 8 * i + g < args.M ? t0 + 8 * i + g : t0) * args.K + q * 8;
  for (int r0 = 0; r0 < args.rank; r0 += 64) {
    for (int u = 0; u < s_nuniq; ++u) {
      const int id = s_uniq[u];
      const T* ar = lora_a + (static_cast<size_t>(id) * args.rank + r0 + g) * args.K + q * 8;
      float acc[MT][RN][4] = {};
#pragma unroll 2
      for (int k = (rank * 8 + warp) * 32; k < args.K; k += C * 8 * 32) {
        const bool in = k + q * 8 < args.K;  // K is a multiple of 8
        uint4 xa[2 * MT], bv[RN];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
          xa[i] = in ? *reinterpret_cast<const uint4*>(xr[i] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < RN; ++n)
          bv[n] = in ? *reinterpret_cast<const uint4*>(ar + static_cast<size_t>(n) * 8 * args.K + k)
                     : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < RN; ++n) {
            mma_16816<T>(acc[m][n], xa[2 * m].x, xa[2 * m + 1].x, xa[2 * m].y, xa[2 * m + 1].y,
                         bv[n].x, bv[n].y);
            mma_16816<T>(acc[m][n], xa[2 * m].z, xa[2 * m + 1].z, xa[2 * m].w, xa[2 * m + 1].w,
                         bv[n].z, bv[n].w);
          }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = 16 * m + 8 * half + g;
          if (s_id[row] != id) continue;
#pragma unroll
          for (int n = 0; n < RN; ++n)
            *reinterpret_cast<float2*>(part + (warp * kTok + row) * 64 + n * 8 + 2 * q) =
                make_float2(acc[m][n][2 * half], acc[m][n][2 * half + 1]);
        }
    }
    __syncthreads();
    constexpr int kCols = RN * 8;
    for (int i = tid; i < kTok * kCols; i += kLoraThreads) {
      const int row = i / kCols, c = i % kCols;
      float sum = 0.f;
      if (s_id[row] >= 0) {
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += part[(w * kTok + row) * 64 + c];
      }
      local[row * 64 + c] = sum;
    }
    cluster_sync();
    for (int i = rank * kLoraThreads + tid; i < kTok * kCols; i += C * kLoraThreads) {
      const int row = i / kCols, c = i % kCols;
      const int id = s_id[row];
      if (id < 0) continue;
      const uint32_t at = smem_addr(local + row * 64 + c);
      float sum = 0.f;
      for (int p = 0; p < C; ++p) sum += ld_cluster_f32(map_shared(at, p));
      // Past the adapter's own rank H is 0 whatever x holds.
      const float v = r0 + c < args.ranks[id] ? sum * args.scales[id] : 0.f;
      h[(static_cast<size_t>(s_flag[id]) * args.tile_rows + t0 - m0 + row) * width + r0 + c] =
          Pack2<T>::from_float(v);
    }
    cluster_sync();  // sums read before the next part overwrites them, or the CTA leaves
  }
  // Zeros where a token meets another adapter of its row tile.
  const int vecs = args.rank / 8;
  for (int i = rank * kLoraThreads + tid; i < kTok * total * vecs; i += C * kLoraThreads) {
    const int v = i % vecs, e = i / vecs % total, row = i / (vecs * total);
    if (t0 + row >= args.M || (s_id[row] >= 0 && s_flag[s_id[row]] == e)) continue;
    *reinterpret_cast<uint4*>(
        h + (static_cast<size_t>(e) * args.tile_rows + t0 - m0 + row) * width + v * 8) =
        make_uint4(0, 0, 0, 0);
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

__host__ __device__ inline int lora_stream_smem_bytes(int nt, int stages) {
  return 1024 + stages * (kMdStageW + nt * 256) + (2 * stages + 1) * 8 + 16;
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
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tfull + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / C;
  const int chunk = tile % args.chunks, n0 = tile / args.chunks * 128;
  const int ksteps = (args.K + 127) / 128;
  const int kb0 = rank * ksteps / C, kb1 = (rank + 1) * ksteps / C;
  const int rs = min(args.rank, 64);  // k-values of one list step
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(nt)) tmem_cols *= 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
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

  // The entries of this CTA's share of the row tile's list: known once the
  // shrink kernel is done.
  auto entries = [&](int* e0) {
    pdl_wait();
    const int n = __ldcg(args.count + chunk);
    *e0 = rank * n / C;
    return (rank + 1) * n / C;
  };

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
      int e0, e1 = 0;
      if (ok) e1 = entries(&e0);
      for (int i = ok ? e0 * args.parts : 0; i < e1 * args.parts; ++i) {
        const int slot = __ldcg(args.list + chunk * args.smax + i / args.parts);
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 52)) break;
        uint8_t* w = sW + stage * kMdStageW;
        const int row = i % args.parts * 64;
        mbar_arrive_expect_tx(&full[stage], 2 * rs * 128);
        tma_load_3d(w, &tm_b, &full[stage], n0, row, slot);
        tma_load_3d(w + 8192, &tm_b, &full[stage], n0 + 64, row, slot);
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
      int e0, e1 = 0;
      if (ok) e1 = entries(&e0);
      fence_proxy_async_all();  // H was stored by ordinary stores
      for (int i = ok ? e0 * args.parts : 0; i < e1 * args.parts; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, 54)) break;
        mbar_arrive_expect_tx(&full[stage], nt * 128);
        tma_load_2d(sB + stage * stage_b, &tm_h, &full[stage], i % args.parts * 64,
                    (chunk * args.smax + i / args.parts) * nt);
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
      int e0, e1 = 0;
      if (ok) e1 = entries(&e0);
      for (int i = ok ? e0 * args.parts : 0; ok && i < e1 * args.parts; ++i) ok = step(rs / 16);
      if (ok) umma_commit(tfull);
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
  float* recv = reinterpret_cast<float*>(sW);  // [C sources][tokens of this rank][128]
  const int own = nt / C;
  if (warp >= 4 && __all_sync(0xffffffffu, ok)) {
    tc_fence_after();
    const int q = warp & 3;
    for (int c = 0; c < nt; c += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int to = (c + j) / own;
        const uint32_t at = smem_addr(recv + (rank * own + (c + j - to * own)) * 128 + q * 32 + lane);
        st_cluster_f32(map_shared(at, to), __uint_as_float(v[j]));
      }
    }
    tc_fence_before();
  }
  cluster_sync();
  T* out = static_cast<T*>(args.out);
  const int row0 = chunk * nt + rank * own;
  for (int i = threadIdx.x; i < own * 64; i += kLoraThreads) {
    const int tok = i >> 6, c = (i & 63) * 2;
    if (row0 + tok >= args.M || n0 + c >= args.N) continue;
    float2 sum = make_float2(0.f, 0.f);
    for (int s = 0; s < C; ++s) {
      const float2 v = *reinterpret_cast<const float2*>(recv + (s * own + tok) * 128 + c);
      sum.x += v.x;
      sum.y += v.y;
    }
    *reinterpret_cast<uint32_t*>(out + static_cast<size_t>(row0 + tok) * args.N + n0 + c) =
        Pack2<T>::pack(sum.x, sum.y);
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
// loop: per list entry, 128 rows of H and `rank` rows of B per CTA.  Tensor
// bound: an entry costs rank / 64 of a k-step.
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
  const int rs = min(args.rank, 64);

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
        const int steps = __ldcg(args.count + pm) * args.parts;
        for (int e = 0; e < steps; ++e) {
          const int entry = pm * args.smax + e / args.parts;
          const int slot = __ldcg(args.list + entry), part = e % args.parts * 64;
          if (!(ok = mbar_wait_cluster(&empty[stage], phase ^ 1u, abort_flag, 62))) break;
          const uint32_t bar = map_shared(smem_addr(&full[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * (kGemmABytes + 2 * rs * 128));
          tma_load_2d_pair(sA + stage * kGemmABytes, &tm_h, bar, part,
                           entry * kLoraPairRows + rank * kGemmBM);
          tma_load_3d_pair(sB + stage * Shape::kBBytes, &tm_b, bar, col, part, slot);
          tma_load_3d_pair(sB + stage * Shape::kBBytes + 8192, &tm_b, bar, col + 64, part, slot);
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
        const int steps = __ldcg(args.count + pm) * args.parts;
        for (int e = 0; ok && e < steps; ++e) ok = step(rs / 16, false);
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
