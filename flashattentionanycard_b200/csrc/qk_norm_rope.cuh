// RMSNorm of every query and key head and the rotary position rotation, in one
// pass, forward and backward (sm_100a).
//
// Per token t and head h, with x = q[t, h, :] (or k[t, h, :]), head size D, and
// c_i, s_i the table's cosine and sine of token t's position:
//   n = x * rsqrt(mean(x^2) + eps),   y = n * w                        (fp32)
//   out[a_i] = y[a_i] c_i - y[b_i] s_i,  out[b_i] = y[b_i] c_i + y[a_i] s_i
// for i < rot / 2, with (a_i, b_i) = (i, i + rot / 2), or (2 i, 2 i + 1) when
// the pairs are interleaved; out = y past rot.  One rounding, on store.
// Backward, with g the incoming gradient turned back by the same angle:
//   dw = sum over tokens and heads of g n          (fp32, fixed order)
//   dx = r (g w - n mean(g w n)),   r = rsqrt(mean(x^2) + eps)
// The statistics are recomputed from x, so nothing is saved by the forward pass.
//
// HBM bound: x in and out once (backward: x, the gradient, dx).  A head row is
// D / 8 lanes of one warp, 16 bytes each (L = 8, 16 or 32 lanes, the smallest
// that holds D), so the row lives in registers, its mean takes log2(L)
// shuffles, and a rotation partner is another lane's register.  A warp takes
// 32 / L x R x loops heads of one token: the token's angles are loaded once
// into 16 registers and serve all of them, and R row loads are in flight per
// lane.  Measured at (32 + 8) heads x 128 bf16: forward of 16384 tokens 62-63 us
// back to back in a graph, 5.4 TB/s with the table, 67-70 in single calls (without
// overlap of launches: one loop of R = 4 77 us, two 68, four 64; R = 2 70-82);
// backward of 8192 tokens 58 us, 4.4 TB/s (one loop 64, two 57, four 58; R = 2
// 58-83; 24 warps an SM instead of 16: 62).  The forward kernel of R = 4 spills 4-32
// bytes under its 64 registers (32 warps an SM), but for neighbours that all turn;
// the backward kernel none.
// The strided kernel below (other head sizes, rotations and alignments) is not
// tuned: one warp a row, 2-byte loads, at most 8 warps an SM.  Forward and backward
// in us: 4096 tokens of (32 + 8) x 512 924 and 1057 (0.37 and 0.48 TB/s), 16384 of
// 96 with rot 24 924 and 1124, 16384 of 128 off 16 bytes 1184 and 1335.
#pragma once

#include "bokt_device.cuh"

namespace bokt {

constexpr int kStatusBadPosition = 5;
constexpr int kQkThreads = 256;
constexpr int kQkWarps = kQkThreads / 32;
constexpr int kQkMaxVecDim = 256;
constexpr int kQkMaxDim = 1024;

// One of the two operands (queries or keys); strides in elements.
struct QkSide {
  const void* x;
  const void* g;  // backward: gradient of the output
  const void* w;  // [D]
  void* out;      // forward: result, backward: gradient of x
  int64_t x_row, x_head, g_row, g_head, out_row, out_head;
  int heads;
};

struct QkArgs {
  QkSide side[2];
  const void* positions;
  int positions_i64;
  const float* cos_sin;  // [table_rows][rot]: rot / 2 cosines, then rot / 2 sines
  int table_rows;
  int tokens, dim, rot;
  float eps;
  int loops;        // head units: loops x R rows per lane group share one load of the angles
  float* partials;  // backward: [gridDim.x][2][dim]
};

__device__ __forceinline__ long long qk_position(const QkArgs& a, int t) {
  return a.positions_i64 ? reinterpret_cast<const long long*>(a.positions)[t]
                         : static_cast<long long>(reinterpret_cast<const int32_t*>(a.positions)[t]);
}

// Two fp32 operations per instruction (sm_100's packed f32x2 arithmetic, each
// half rounded like the scalar form): both kernels issue more arithmetic per
// byte than a copy, so this is what keeps them near the memory rate.
__device__ __forceinline__ unsigned long long qk_bits(float2 a) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 qk_pair(unsigned long long r) {
  float2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
  return a;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(qk_bits(a)), "l"(qk_bits(b)), "l"(qk_bits(c)));
  return qk_pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(qk_bits(a)), "l"(qk_bits(b)));
  return qk_pair(r);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

template <typename T>
__device__ __forceinline__ void qk_unpack(const uint4& v, float2 (&f)[4]) {
  f[0] = Pack2<T>::unpack(v.x);
  f[1] = Pack2<T>::unpack(v.y);
  f[2] = Pack2<T>::unpack(v.z);
  f[3] = Pack2<T>::unpack(v.w);
}

template <typename T>
__device__ __forceinline__ uint4 qk_pack(const float2 (&f)[4]) {
  return make_uint4(Pack2<T>::pack(f[0].x, f[0].y), Pack2<T>::pack(f[1].x, f[1].y),
                    Pack2<T>::pack(f[2].x, f[2].y), Pack2<T>::pack(f[3].x, f[3].y));
}

template <int L>
__device__ __forceinline__ float qk_row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The angles of one token as this lane needs them: element j of the lane turns
// with c[j] and its partner enters with s[j] (the sign of the forward rotation
// is in s).
struct QkAngles {
  float2 c[4], s[4];
  __device__ __forceinline__ QkAngles() {
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = both(1.f), s[j] = both(0.f);
  }
};

template <bool PAIRS>
__device__ __forceinline__ void qk_load_angles(const float* row, int rot, int i, QkAngles& a) {
  if constexpr (PAIRS) {
    const float4 c = *reinterpret_cast<const float4*>(row + i / 2);
    const float4 s = *reinterpret_cast<const float4*>(row + rot / 2 + i / 2);
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a.c[j] = both(cc[j]);
      a.s[j] = make_float2(-ss[j], ss[j]);
    }
  } else {
    const bool low = i < rot / 2;
    const int f = low ? i : i - rot / 2;
    const float2 sign = both(low ? -1.f : 1.f);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 c = *reinterpret_cast<const float4*>(row + f + 4 * h);
      const float4 s = *reinterpret_cast<const float4*>(row + rot / 2 + f + 4 * h);
      a.c[2 * h] = make_float2(c.x, c.y), a.c[2 * h + 1] = make_float2(c.z, c.w);
      a.s[2 * h] = mul2(make_float2(s.x, s.y), sign);
      a.s[2 * h + 1] = mul2(make_float2(s.z, s.w), sign);
    }
  }
}

// The 8 elements that turn with this lane's: the partner lane's row bits (four
// shuffles of packed pairs), or the neighbours of the lane's own pairs; zeros
// for a lane that does not turn (its s is 0, but 0 times an infinity is not).
template <typename T, bool PAIRS>
__device__ __forceinline__ void qk_partner(const uint4& raw, const float2 (&v)[4], int partner,
                                           bool turns, float2 (&o)[4]) {
  if constexpr (PAIRS) {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = turns ? make_float2(v[j].y, v[j].x) : both(0.f);
  } else {
    uint4 p;
    p.x = __shfl_sync(0xffffffffu, raw.x, partner);
    p.y = __shfl_sync(0xffffffffu, raw.y, partner);
    p.z = __shfl_sync(0xffffffffu, raw.z, partner);
    p.w = __shfl_sync(0xffffffffu, raw.w, partner);
    qk_unpack<T>(turns ? p : make_uint4(0, 0, 0, 0), o);
  }
}

// Head units: unit u covers heads [chunk * HPU, +HPU) of token u / chunks.
// PART: rot is less than the head size.  A rotation of whole heads leaves the
// zeros of qk_partner out, which for neighbours are eight selects a row
// ((32 + 8) heads x 128, forward of 16384 tokens 57.9 us without and 60.9 with
// them, backward of 8192 54.8 and 56.2; halves within 0.3 either way: always PART).
template <typename T, int L, bool PAIRS, bool PART, int R>
__global__ void __launch_bounds__(kQkThreads, 4) qk_norm_rope_kernel(const QkArgs args) {
  constexpr int S = 32 / L;
  pdl_allow_next();
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L;
  const int i = l * 8;
  const float inv_dim = 1.f / args.dim;
  const bool active = i < args.dim;
  const bool turns = i < args.rot;
  const int half = args.rot / 16;
  const int partner = PAIRS || !turns ? lane : (i < args.rot / 2 ? lane + half : lane - half);
  const int hpu = S * R * args.loops;
  const int chunks0 = (args.side[0].heads + hpu - 1) / hpu;
  const int chunks1 = (args.side[1].heads + hpu - 1) / hpu;
  const int units0 = args.tokens * chunks0;
  int u = blockIdx.x * kQkWarps + (threadIdx.x >> 5);
  if (u >= units0 + args.tokens * chunks1) return;
  const QkSide& sd = args.side[u >= units0];
  const int chunks = u >= units0 ? chunks1 : chunks0;
  if (u >= units0) u -= units0;
  const int t = u / chunks;
  int h0 = (u - t * chunks) * hpu + sub;
  const int hend = min(sd.heads, (u - t * chunks + 1) * hpu);
  pdl_wait();
  const long long pos = qk_position(args, t);
  const T* x = static_cast<const T*>(sd.x) + t * sd.x_row + i;
  uint4 raw[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int h = h0 + r * S;
    raw[r] = active && h < hend ? *reinterpret_cast<const uint4*>(x + h * sd.x_head)
                                : make_uint4(0, 0, 0, 0);
  }
  // The weights join the angles: with wc = w c and ws = (partner's w) s, a row
  // costs one product and one FMA per element, times its rsqrt.
  const uint4 wraw = active ? *reinterpret_cast<const uint4*>(static_cast<const T*>(sd.w) + i)
                            : make_uint4(0, 0, 0, 0);
  if (pos < 0 || pos >= args.table_rows) {
    if (lane == 0) report_status(kStatusBadPosition, t);
    return;
  }
  QkAngles ang;
  if (turns) qk_load_angles<PAIRS>(args.cos_sin + pos * args.rot, args.rot, i, ang);
  {
    float2 w[4], pw[4];
    qk_unpack<T>(wraw, w);
    qk_partner<T, PAIRS>(wraw, w, partner, !PART || turns, pw);
#pragma unroll
    for (int j = 0; j < 4; ++j) ang.c[j] = mul2(ang.c[j], w[j]), ang.s[j] = mul2(ang.s[j], pw[j]);
  }
  T* out = static_cast<T*>(sd.out) + t * sd.out_row + i;
  for (;;) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int h = h0 + r * S;
      float2 v[4], o[4], ss = both(0.f);
      qk_unpack<T>(raw[r], v);
      // Past rot a lane of halves is its own partner: an infinity there is NaN as
      // it is (its row's rsqrt is 0), so only neighbours need the zeros.
      qk_partner<T, PAIRS>(raw[r], v, partner, !PAIRS || !PART || turns, o);
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = fma2(v[j], v[j], ss);
      const float2 rs = both(rsqrtf(fmaf(qk_row_sum<L>(ss.x + ss.y), inv_dim, args.eps)));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = mul2(fma2(v[j], ang.c[j], mul2(o[j], ang.s[j])), rs);
      if (active && h < hend) *reinterpret_cast<uint4*>(out + h * sd.out_head) = qk_pack<T>(v);
    }
    h0 += R * S;
    if (h0 - sub >= hend) break;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int h = h0 + r * S;
      raw[r] = active && h < hend ? *reinterpret_cast<const uint4*>(x + h * sd.x_head)
                                  : make_uint4(0, 0, 0, 0);
    }
  }
}

// 16 bytes to shared memory without passing through registers; zeros where the
// lane has nothing to read.
__device__ __forceinline__ void qk_copy_async(uint4* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}

// Rows of one warp's walk over the units of both sides (a token's query units,
// then its key units): batches of R heads per lane group, unit after unit.
struct QkWalk {
  int u, t, h0, hend, side;
  __device__ __forceinline__ void enter(const QkArgs& args, int unit, int chunks0, int chunks, int hpu,
                                        int sub) {
    u = unit;
    t = unit / chunks;
    int chunk = unit - t * chunks;
    side = chunk >= chunks0;
    if (side) chunk -= chunks0;
    h0 = chunk * hpu + sub;
    hend = min(args.side[side].heads, (chunk + 1) * hpu);
  }
};

constexpr int kQkRing = 2;  // batches in flight or in use per warp (3 or 4 measured no faster)

// Shared memory of the backward kernel: a ring of R rows of x and of the
// gradient per lane, and the block's sums.
template <int L, int R>
__host__ __device__ constexpr int qk_grad_smem_bytes() {
  const int ring = kQkThreads * kQkRing * R * 2 * 16;
  const int sums = kQkWarps * (32 / L) * (L * 8 + 1) * 4;
  return ring > sums ? ring : sums;
}

// Backward: persistent warps walk the units of all tokens.  The next batches'
// rows arrive by cp.async while one is computed (each lane reads back what it
// copied itself: no barrier); the weight gradients stay in 8 registers a side
// and lane until the end, are summed over the block's rows in shared memory and
// leave as one partial row per block and side, which
// qk_norm_rope_dweight_kernel adds in block order.
template <typename T, int L, bool PAIRS, bool PART, int R>
__global__ void __launch_bounds__(kQkThreads, 2) qk_norm_rope_grad_kernel(const QkArgs args) {
  constexpr int S = 32 / L;
  extern __shared__ uint4 qk_ring[];
  pdl_allow_next();
  const int lane = threadIdx.x & 31, l = lane % L, sub = lane / L, warp = threadIdx.x >> 5;
  const int i = l * 8;
  const float inv_dim = 1.f / args.dim;
  const bool active = i < args.dim;
  const bool turns = i < args.rot;
  const int half = args.rot / 16;
  const int partner = PAIRS || !turns ? lane : (i < args.rot / 2 ? lane + half : lane - half);
  uint4* ring = qk_ring + threadIdx.x;  // [slot][row][x, gradient][thread]
  const int stride = gridDim.x * kQkWarps;
  const int hpu = S * R * args.loops;
  const int chunks0 = (args.side[0].heads + hpu - 1) / hpu;
  const int chunks = chunks0 + (args.side[1].heads + hpu - 1) / hpu;
  const int units = args.tokens * chunks;
  pdl_wait();
  float2 dwq[4] = {}, dwk[4] = {};
  QkWalk in = {}, at = {};  // the batch to copy next, the batch to compute
  in.u = at.u = blockIdx.x * kQkWarps + warp;
  if (in.u < units) in.enter(args, in.u, chunks0, chunks, hpu, sub);
  int slot_in = 0, slot = 0;
  auto copy = [&] {
    if (in.u < units) {
      const QkSide& sd = args.side[in.side];
      const T* x = static_cast<const T*>(sd.x) + in.t * sd.x_row + i;
      const T* g = static_cast<const T*>(sd.g) + in.t * sd.g_row + i;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int h = in.h0 + r * S;
        const bool have = active && h < in.hend;
        uint4* dst = ring + (slot_in * R + r) * 2 * kQkThreads;
        qk_copy_async(dst, have ? x + h * sd.x_head : sd.x, have);
        qk_copy_async(dst + kQkThreads, have ? g + h * sd.g_head : sd.g, have);
      }
      slot_in = slot_in + 1 == kQkRing ? 0 : slot_in + 1;
      in.h0 += S * R;
      if (in.h0 - sub >= in.hend) {
        in.u += stride;
        if (in.u < units) in.enter(args, in.u, chunks0, chunks, hpu, sub);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < kQkRing - 1; ++s) copy();
  long long next = at.u < units ? qk_position(args, at.u / chunks) : 0;
#pragma unroll 1
  for (; at.u < units; at.u += stride) {
    at.enter(args, at.u, chunks0, chunks, hpu, sub);
    const QkSide& sd = args.side[at.side];
    const long long pos = next;
    if (at.u + stride < units) next = qk_position(args, (at.u + stride) / chunks);
    const bool known = pos >= 0 && pos < args.table_rows;
    if (!known && lane == 0) report_status(kStatusBadPosition, at.t);
    QkAngles ang;
    if (turns && known) {
      qk_load_angles<PAIRS>(args.cos_sin + pos * args.rot, args.rot, i, ang);
#pragma unroll
      for (int j = 0; j < 4; ++j) ang.s[j] = make_float2(-ang.s[j].x, -ang.s[j].y);  // backwards
    }
    const uint4 wraw = active ? *reinterpret_cast<const uint4*>(static_cast<const T*>(sd.w) + i)
                              : make_uint4(0, 0, 0, 0);
    T* out = static_cast<T*>(sd.out) + at.t * sd.out_row + i;
#pragma unroll 1
    for (; at.h0 - sub < at.hend; at.h0 += S * R) {
      copy();
      asm volatile("cp.async.wait_group %0;" ::"n"(kQkRing - 1) : "memory");
      const uint4* row = ring + slot * R * 2 * kQkThreads;
      slot = slot + 1 == kQkRing ? 0 : slot + 1;
      if (!known) continue;  // its rows stay unwritten and add nothing
      float2 dw[4] = {};
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int h = at.h0 + r * S;
        const uint4 xr = row[r * 2 * kQkThreads], gr = row[(r * 2 + 1) * kQkThreads];
        float2 v[4], gv[4], o[4], w[4], ss = both(0.f), dot = both(0.f);
        qk_unpack<T>(xr, v);
        qk_unpack<T>(gr, gv);
        qk_unpack<T>(wraw, w);
        qk_partner<T, PAIRS>(gr, gv, partner, !PART || turns, o);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          gv[j] = fma2(gv[j], ang.c[j], mul2(o[j], ang.s[j]));  // turned back
          o[j] = mul2(gv[j], v[j]);
          gv[j] = mul2(gv[j], w[j]);
          ss = fma2(v[j], v[j], ss);
          dot = fma2(gv[j], v[j], dot);
        }
        // Both sums at once; with n = x r: mean(g w n) = r dot / D.
        // Rows past the unit's heads are zeros: r = 0, or eps = 0 would make them NaN.
        const float r0 = rsqrtf(fmaf(qk_row_sum<L>(ss.x + ss.y), inv_dim, args.eps));
        const float r1 = h < at.hend ? r0 : 0.f;
        const float2 rs = both(r1), mean = both(-r1 * inv_dim * qk_row_sum<L>(dot.x + dot.y));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dw[j] = fma2(o[j], rs, dw[j]);
          gv[j] = mul2(fma2(mul2(v[j], rs), mean, gv[j]), rs);
        }
        if (active && h < at.hend) *reinterpret_cast<uint4*>(out + h * sd.out_head) = qk_pack<T>(gv);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2& to = at.side ? dwk[j] : dwq[j];
        to.x += dw[j].x;
        to.y += dw[j].y;
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the ring turns into the sums
  float* sums = reinterpret_cast<float*>(qk_ring);
  constexpr int kRow = L * 8 + 1;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 d = side ? dwk[j / 2] : dwq[j / 2];
      sums[(warp * S + sub) * kRow + i + j] = j & 1 ? d.y : d.x;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < args.dim; d += kQkThreads) {
      float total = 0.f;
#pragma unroll
      for (int r = 0; r < kQkWarps * S; ++r) total += sums[r * kRow + d];
      args.partials[(static_cast<size_t>(blockIdx.x) * 2 + side) * args.dim + d] = total;
    }
    __syncthreads();
  }
}

// Any head size up to kQkMaxDim, any even rot, any strides: one warp per head
// row, the row staged in shared memory in fp32.  Blocks are persistent in both
// directions; the weight gradient is accumulated per warp in shared memory
// (each lane owns its columns).
template <typename T, bool PAIRS, bool GRAD>
__global__ void __launch_bounds__(128) qk_norm_rope_any_kernel(const QkArgs args) {
  extern __shared__ float rows[];  // [4 warps][3][dim]: x, gradient, weight gradient
  pdl_allow_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int D = args.dim, hr = args.rot / 2;
  const float inv_dim = 1.f / D;
  float* v = rows + static_cast<size_t>(warp) * 3 * D;
  float* gv = v + D;
  float* dw = gv + D;
  pdl_wait();
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const QkSide& sd = args.side[side];
    const T* w = static_cast<const T*>(sd.w);
    const int units = args.tokens * sd.heads;
    if (GRAD)
      for (int d = lane; d < D; d += 32) dw[d] = 0.f;
    for (int u = blockIdx.x * 4 + warp; u < units; u += gridDim.x * 4) {
      const int t = u / sd.heads, h = u - t * sd.heads;
      const long long pos = qk_position(args, t);
      if (pos < 0 || pos >= args.table_rows) {
        if (lane == 0) report_status(kStatusBadPosition, t);
        continue;
      }
      const float* cs = args.cos_sin + pos * args.rot;
      const T* x = static_cast<const T*>(sd.x) + t * sd.x_row + h * sd.x_head;
      T* out = static_cast<T*>(sd.out) + t * sd.out_row + h * sd.out_head;
      float ss = 0.f;
      for (int d = lane; d < D; d += 32) {
        const float f = Pack2<T>::to_float(x[d]);
        v[d] = f;
        ss = fmaf(f, f, ss);
        if (GRAD)
          gv[d] = Pack2<T>::to_float(static_cast<const T*>(sd.g)[t * sd.g_row + h * sd.g_head + d]);
      }
      const float rs = rsqrtf(fmaf(qk_row_sum<32>(ss), inv_dim, args.eps));
      __syncwarp();
      if (!GRAD) {
        for (int d = lane; d < D; d += 32) v[d] = v[d] * rs * Pack2<T>::to_float(w[d]);
        __syncwarp();
      }
      float* y = GRAD ? gv : v;
      for (int p = lane; p < hr; p += 32) {
        const int a = PAIRS ? 2 * p : p, b = PAIRS ? 2 * p + 1 : p + hr;
        const float c = cs[p], s = GRAD ? -cs[hr + p] : cs[hr + p];
        const float ya = y[a], yb = y[b];
        y[a] = fmaf(ya, c, -(yb * s));
        y[b] = fmaf(yb, c, ya * s);
      }
      __syncwarp();
      if (GRAD) {
        float dot = 0.f;
        for (int d = lane; d < D; d += 32) {
          const float n = v[d] * rs, g = gv[d];
          dw[d] = fmaf(g, n, dw[d]);
          dot = fmaf(g * Pack2<T>::to_float(w[d]), n, dot);
        }
        const float mean = qk_row_sum<32>(dot) * inv_dim;
        for (int d = lane; d < D; d += 32)
          out[d] = Pack2<T>::from_float(
              rs * (gv[d] * Pack2<T>::to_float(w[d]) - v[d] * rs * mean));
      } else {
        for (int d = lane; d < D; d += 32) out[d] = Pack2<T>::from_float(v[d]);
      }
      __syncwarp();
    }
    if (GRAD) {
      __syncthreads();
      for (int d = threadIdx.x; d < D; d += 128) {
        float total = 0.f;
        for (int r = 0; r < 4; ++r) total += rows[(r * 3 + 2) * static_cast<size_t>(D) + d];
        args.partials[(static_cast<size_t>(blockIdx.x) * 2 + side) * D + d] = total;
      }
      __syncthreads();
    }
  }
}

// dw[side][d] = sum over blocks of the partial rows, in a fixed order: thread
// (x, y) adds blocks y, y + 32, ..., then the 32 sums of a column are added in
// y order.
__global__ void __launch_bounds__(1024) qk_norm_rope_dweight_kernel(const float* partials,
                                                                    int blocks, int dim,
                                                                    float* dqw, float* dkw) {
  __shared__ float part[32][33];
  pdl_allow_next();
  pdl_wait();
  const int side = blockIdx.y, d = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (d < dim)
    for (int b = threadIdx.y; b < blocks; b += 32)
      sum += partials[(static_cast<size_t>(b) * 2 + side) * dim + d];
  part[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && d < dim) {
    float total = 0.f;
#pragma unroll
    for (int y = 0; y < 32; ++y) total += part[y][threadIdx.x];
    (side ? dkw : dqw)[d] = total;
  }
}

// cos_sin[p][i] = cos(p base^(-2 i / rot)), cos_sin[p][rot / 2 + i] = its sine;
// angles in 64 bits (fp32 has no correct digit of the sine left once the angle
// passes 2^24), rounded once to fp32.
__global__ void __launch_bounds__(256) rope_table_kernel(float* cos_sin, int rows, int rot,
                                                         double base) {
  pdl_allow_next();
  pdl_wait();
  const int hr = rot / 2;
  const int64_t n = static_cast<int64_t>(rows) * hr;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
    const int64_t p = e / hr;
    const int i = static_cast<int>(e - p * hr);
    double sn, cn;
    sincos(static_cast<double>(p) * pow(base, -2.0 * i / rot), &sn, &cn);
    cos_sin[p * rot + i] = static_cast<float>(cn);
    cos_sin[p * rot + hr + i] = static_cast<float>(sn);
  }
}

}  // namespace bokt
