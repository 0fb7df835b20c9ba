// C ABI of the sm_100a kernel library (declarations and reference citations in
// include/bokt.h).  Host side: argument checks, path selection, TMA tensor-map
// encoding, launch configuration.  No allocation, no synchronisation and no
// host read-back on any compute entry point.
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <numeric>

#include "../../include/bokt.h"
#include "bokt_device.cuh"
#include "ep_sync.cuh"
#include "gemm_edge.cuh"
#include "gemm_tc.cuh"
#include "gemm_tc2.cuh"
#include "lora_gemm.cuh"
#include "moe_decode.cuh"
#include "moe_few.cuh"
#include "moe_route.cuh"
#include "norm_gemm.cuh"
#include "qk_norm_rope.cuh"
#include "rmsnorm.cuh"

namespace {

thread_local char g_err[1024] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int cuda_fail(cudaError_t e, const char* what) {
  return fail(BOKT_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int param_or(int v, int dflt) { return v > 0 ? v : dflt; }

// Programmatic dependent launch for every kernel (each kernel waits with
// griddepcontrol.wait before touching global memory).  BOKT_DISABLE_PDL=1
// turns the attribute off, e.g. to compare timings.
bool pdl_enabled() {
  static const bool on = [] {
    const char* v = getenv("BOKT_DISABLE_PDL");
    return !(v && v[0] && v[0] != '0');
  }();
  return on;
}

cudaLaunchConfig_t launch_config(dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                                 cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cfg;
}

// Typed launch: kernel<<<grid, block, smem, s>>>(args...) with PDL.
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                   Args... args) {
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_config(grid, block, smem, s, attr);
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// Untyped launch through a kernel pointer and an argument array, with PDL.
cudaError_t launch_ptr(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                       void** args) {
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_config(grid, block, smem, s, attr);
  return cudaLaunchKernelExC(&cfg, fn, args);
}

// ----------------------------------------------------------------- device info
struct DeviceInfo {
  int sm_count = 0;
  int smem_optin = 0;
};
constexpr int kMaxDevices = 64;
DeviceInfo g_dev[kMaxDevices];
std::mutex g_dev_mu;

int device_info(DeviceInfo* out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(BOKT_ERR_UNSUPPORTED, "device index %d", dev);
  std::lock_guard<std::mutex> lock(g_dev_mu);
  DeviceInfo& d = g_dev[dev];
  if (d.sm_count == 0) {
    int major = 0;
    e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    if (major != 10)
      return fail(BOKT_ERR_UNSUPPORTED, "library built for sm_100a; device %d is sm_%d.x", dev,
                  major);
    e = cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    e = cudaDeviceGetAttribute(&d.smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
  }
  *out = d;
  return BOKT_OK;
}

// Raise a kernel's dynamic shared-memory limit once per (device, kernel, size).
// The first call for a configuration happens outside graph capture (warm-up).
struct SmemAttr {
  int dev;
  const void* fn;
  int bytes;
};
SmemAttr g_smem_attr[512];
int g_smem_attr_n = 0;
std::mutex g_smem_mu;

int ensure_smem(const void* fn, int bytes) {
  if (bytes <= 48 * 1024) return BOKT_OK;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(g_smem_mu);
  for (int i = 0; i < g_smem_attr_n; ++i)
    if (g_smem_attr[i].dev == dev && g_smem_attr[i].fn == fn && g_smem_attr[i].bytes >= bytes)
      return BOKT_OK;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(MaxDynamicSharedMemorySize)");
  if (g_smem_attr_n < 512) g_smem_attr[g_smem_attr_n++] = {dev, fn, bytes};
  return BOKT_OK;
}

// Ask for the largest shared-memory carve-out for a small kernel whose successor
// is launched while it runs: the successor's CTAs only join an SM whose carve-out
// already holds them.  Once per (device, kernel).
int ensure_carveout(const void* fn) {
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(g_smem_mu);
  for (int i = 0; i < g_smem_attr_n; ++i)
    if (g_smem_attr[i].dev == dev && g_smem_attr[i].fn == fn && g_smem_attr[i].bytes == -1)
      return BOKT_OK;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                                       cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(PreferredSharedMemoryCarveout)");
  if (g_smem_attr_n < 512) g_smem_attr[g_smem_attr_n++] = {dev, fn, -1};
  return BOKT_OK;
}

// ----------------------------------------------------------------- tensor maps
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

int get_encoder() {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (!g_encode) return fail(BOKT_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  return BOKT_OK;
}

// Row-major [outer..., rows, cols] 16-bit tensor, box {64 cols, box_rows, 1...},
// 128-byte swizzle, zero fill outside the tensor.
int encode_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
               const uint64_t* strides_bytes, const uint32_t* box, bool fp16) {
  (void)fp16;
  int rc = get_encoder();
  if (rc) return rc;
  uint32_t elem_strides[3] = {1, 1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, const_cast<void*>(base), dims,
                        strides_bytes, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(BOKT_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));
  return BOKT_OK;
}

// ----------------------------------------------------------------- GEMM dispatch
using bokt::GemmTcArgs;

template <int BN, bool GROUPED, typename T, bool SCATTER, bool ROWSCALE = false>
const void* tc_kernel_ptr() {
  return reinterpret_cast<const void*>(&bokt::gemm_tc_kernel<BN, GROUPED, T, SCATTER, ROWSCALE>);
}

template <bool GROUPED, typename T, bool SCATTER, bool ROWSCALE = false>
const void* tc_kernel_for(int bn) {
  switch (bn) {
    case 64: return tc_kernel_ptr<64, GROUPED, T, SCATTER, ROWSCALE>();
    case 128: return tc_kernel_ptr<128, GROUPED, T, SCATTER, ROWSCALE>();
    case 256: return tc_kernel_ptr<256, GROUPED, T, SCATTER, ROWSCALE>();
  }
  return nullptr;
}

const void* tc_kernel(bool grouped, int dtype, int bn, bool scatter = false,
                      bool rowscale = false) {
  if (rowscale)
    return dtype == BOKT_BF16 ? tc_kernel_for<false, __nv_bfloat16, false, true>(bn)
                              : tc_kernel_for<false, __half, false, true>(bn);
  if (scatter)
    return dtype == BOKT_BF16 ? tc_kernel_for<true, __nv_bfloat16, true>(bn)
                              : tc_kernel_for<true, __half, true>(bn);
  if (grouped)
    return dtype == BOKT_BF16 ? tc_kernel_for<true, __nv_bfloat16, false>(bn)
                              : tc_kernel_for<true, __half, false>(bn);
  return dtype == BOKT_BF16 ? tc_kernel_for<false, __nv_bfloat16, false>(bn)
                            : tc_kernel_for<false, __half, false>(bn);
}

struct TcConfig {
  int bn, stages, group_m, smem, cta_group, raster, split_k;
};

int resolve_tc_config(const bokt_params* p, bool grouped, int experts, int smem_optin,
                      TcConfig* out) {
  const bokt_params zero = {};
  if (!p) p = &zero;
  const int bm = param_or(p->block_m, 128);
  const int bk = param_or(p->block_k, 64);
  const int bn = param_or(p->block_n, 256);
  const int warps = param_or(p->num_warps, 6);
  if (bm != 128) return fail(BOKT_ERR_CONFIG, "block_m must be 128 (tcgen05 cta_group::1 M)");
  if (bk != 64) return fail(BOKT_ERR_CONFIG, "block_k must be 64 (one 128-byte swizzle row)");
  if (bn != 64 && bn != 128 && bn != 256)
    return fail(BOKT_ERR_CONFIG, "block_n must be 64, 128 or 256 (got %d)", bn);
  if (warps != 6) return fail(BOKT_ERR_CONFIG, "num_warps must be 6 (TMA, MMA, 4 epilogue)");
  const int split_k = param_or(p->split_k, 1);
  if (split_k < 1 || split_k > bokt::kSplitKMax)
    return fail(BOKT_ERR_CONFIG, "split_k must be in [1, %d] (got %d)", bokt::kSplitKMax, split_k);
  const int cta_group = param_or(p->cta_group, 1);
  if (cta_group != 1 && cta_group != 2) return fail(BOKT_ERR_CONFIG, "cta_group must be 1 or 2");
  if (split_k > 1 && cta_group == 2 && grouped)
    return fail(BOKT_ERR_CONFIG,
                "split_k > 1 applies to the dense GEMM (single CTAs or pairs) and the "
                "single-CTA grouped GEMM, not to grouped CTA pairs");
  if (cta_group == 2 && bn == 64)
    return fail(BOKT_ERR_CONFIG, "cta_group 2 needs block_n 128 or 256");
  const int raster = param_or(p->raster, bokt::kRasterExpert);
  if (raster != bokt::kRasterExpert && raster != bokt::kRasterBalanced)
    return fail(BOKT_ERR_CONFIG, "raster must be 1 (expert order) or 2 (balanced)");
  if (raster == bokt::kRasterBalanced && !grouped)
    return fail(BOKT_ERR_CONFIG, "raster 2 applies to the grouped GEMM (dense: group_m)");
  const int stages = param_or(p->stages, cta_group == 2 ? (bn == 256 ? 6 : 8) : (bn == 256 ? 4 : 6));
  if (stages < 2 || stages > 8) return fail(BOKT_ERR_CONFIG, "stages must be in [2, 8]");
  int smem = cta_group == 2 ? bokt::gemm_tc2_smem_bytes(bn, stages, grouped ? experts : 0)
                            : bokt::gemm_tc_smem_bytes(bn, stages, grouped, experts);
  if (smem > smem_optin)
    return fail(BOKT_ERR_CONFIG, "block_n=%d stages=%d needs %d bytes of shared memory (max %d)",
                bn, stages, smem, smem_optin);
  // One CTA per SM: the persistent schedule assumes it and two CTAs would
  // contend for the 512 TMEM columns.
  const int one_per_sm = smem_optin / 2 + 1024;
  if (smem < one_per_sm) smem = one_per_sm;
  out->bn = bn;
  out->stages = stages;
  out->group_m = param_or(p->group_m, 8);
  out->smem = smem;
  out->cta_group = cta_group;
  out->raster = raster;
  out->split_k = split_k;
  return BOKT_OK;
}

// Split-K workspace of the current device: one slot per SM (no launch of a
// split-K kernel uses more CTAs), sized for the configuration's BN.
int64_t splitk_bytes_for(const DeviceInfo& dev, int bn) {
  return bokt::splitk_workspace_bytes(dev.sm_count, bn);
}

// Attach the workspace to `args` for a split-K launch; checks size and alignment.
int attach_splitk(const TcConfig& cfg, const DeviceInfo& dev, int nkb, void* ws, int64_t ws_bytes,
                  GemmTcArgs* args) {
  int split = cfg.split_k < nkb ? cfg.split_k : nkb;
  if (split < 1) split = 1;
  args->split_k = split;
  if (split == 1) return BOKT_OK;
  const int64_t need = splitk_bytes_for(dev, cfg.bn);
  if (!ws)
    return fail(BOKT_ERR_INVALID,
                "split_k > 1 needs a workspace of %lld bytes (zero-filled once when allocated); "
                "pass it to the _ex entry point", (long long)need);
  if (ws_bytes < need)
    return fail(BOKT_ERR_INVALID, "split-K workspace too small: %lld bytes, need %lld",
                (long long)ws_bytes, (long long)need);
  if ((reinterpret_cast<uintptr_t>(ws) & 255u) != 0)
    return fail(BOKT_ERR_INVALID, "split-K workspace must be 256-byte aligned");
  args->splitk_ws = ws;
  args->splitk_slots = dev.sm_count;
  return BOKT_OK;
}

template <typename T, bool ROWSCALE, bool GROUPED, bool SCATTER = false>
const void* tc2_kernel_for(int bn) {
  return bn == 256
             ? reinterpret_cast<const void*>(&bokt::gemm_tc2_kernel<256, T, ROWSCALE, GROUPED, SCATTER>)
             : reinterpret_cast<const void*>(&bokt::gemm_tc2_kernel<128, T, ROWSCALE, GROUPED, SCATTER>);
}

const void* tc2_kernel(int dtype, int bn, bool rowscale = false, bool grouped = false,
                       bool scatter = false) {
  const bool bf = dtype == BOKT_BF16;
  if (scatter)
    return bf ? tc2_kernel_for<__nv_bfloat16, false, true, true>(bn)
              : tc2_kernel_for<__half, false, true, true>(bn);
  if (grouped)
    return bf ? tc2_kernel_for<__nv_bfloat16, false, true>(bn)
              : tc2_kernel_for<__half, false, true>(bn);
  if (rowscale)
    return bf ? tc2_kernel_for<__nv_bfloat16, true, false>(bn)
              : tc2_kernel_for<__half, true, false>(bn);
  return bf ? tc2_kernel_for<__nv_bfloat16, false, false>(bn)
            : tc2_kernel_for<__half, false, false>(bn);
}

// Dense GEMM on CTA pairs: cluster of 2 along x, PDL as every other launch.
int launch_tc2(int dtype, const TcConfig& cfg, const CUtensorMap& ma, const CUtensorMap& mb,
               const GemmTcArgs& args, int pairs, cudaStream_t s, bool grouped = false,
               bool scatter = false, const CUtensorMap* ma64 = nullptr) {
  const void* fn = tc2_kernel(dtype, cfg.bn, args.row_scale != nullptr, grouped, scatter);
  int rc = ensure_smem(fn, cfg.smem);
  if (rc) return rc;
  // Third map: 64-row A boxes for grouped half-height tiles (unused by dense launches).
  void* kargs[] = {const_cast<CUtensorMap*>(&ma), const_cast<CUtensorMap*>(&mb),
                   const_cast<CUtensorMap*>(ma64 ? ma64 : &ma), const_cast<GemmTcArgs*>(&args)};
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t lc = launch_config(
      dim3(2 * pairs), dim3(bokt::kGemmThreads), cfg.smem, s,
      attr);
  attr[lc.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[lc.numAttrs].val.clusterDim.x = 2;
  attr[lc.numAttrs].val.clusterDim.y = 1;
  attr[lc.numAttrs].val.clusterDim.z = 1;
  lc.numAttrs += 1;
  cudaError_t e = cudaLaunchKernelExC(&lc, fn, kargs);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_tc2 launch");
  return BOKT_OK;
}

int launch_tc(bool grouped, int dtype, const TcConfig& cfg, const CUtensorMap& ma,
              const CUtensorMap& mb, const GemmTcArgs& args, int grid, cudaStream_t s,
              bool scatter = false) {
  const void* fn = tc_kernel(grouped, dtype, cfg.bn, scatter, args.row_scale != nullptr);
  int rc = ensure_smem(fn, cfg.smem);
  if (rc) return rc;
  void* kargs[] = {const_cast<CUtensorMap*>(&ma), const_cast<CUtensorMap*>(&mb),
                   const_cast<GemmTcArgs*>(&args)};
  cudaError_t e = launch_ptr(fn, dim3(grid), dim3(bokt::kGemmThreads), cfg.smem, s, kargs);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_tc launch");
  return BOKT_OK;
}

// Edge shapes (row strides TMA cannot describe): the tcgen05 edge kernel, one
// CTA per 128 x 64 tile.  Dense: experts == 0, rows = M; grouped: rows = T.
template <typename T>
int launch_edge(const void* A, const void* B, void* C, int rows, int N, int K,
                const void* offsets, int offsets_i64, int experts, int dtype, cudaStream_t s) {
  const long long nn = (N + bokt::kEdgeBN - 1) / bokt::kEdgeBN;
  const long long mtiles = (rows + bokt::kEdgeBM - 1) / bokt::kEdgeBM + (experts > 0 ? experts : 0);
  const long long tiles = mtiles * nn;
  if (tiles > 0x7fffffffLL) return fail(BOKT_ERR_UNSUPPORTED, "edge path: too many tiles");
  const uint32_t idesc = bokt::make_idesc_f16(uint32_t(dtype), bokt::kEdgeBM, bokt::kEdgeBN);
  cudaError_t e = launch(bokt::gemm_tc_edge_kernel<T>, dim3(unsigned(tiles)),
                         dim3(bokt::kEdgeThreads), bokt::kEdgeSmemBytes, s,
                         static_cast<const T*>(A), static_cast<const T*>(B), static_cast<T*>(C),
                         rows, N, K, offsets, offsets_i64, experts, idesc);
  if (e != cudaSuccess) return cuda_fail(e, "gemm_tc_edge launch");
  return BOKT_OK;
}

// The separate split-K reduction after a dense launch with args.splitk_reduce
// set: one CTA per (tile, CTA row half, 8 / lanes column groups of 4),
// 128 rows x `lanes` worker lanes; lanes grows with the workers one tile can
// span (about four partials per lane, at most 8 lanes).
int launch_splitk_reduce(int dtype, const TcConfig& cfg, const GemmTcArgs& args, int launched,
                         bool pair, cudaStream_t s) {
  const int tile_rows = pair ? 256 : 128;
  const long long nt = (long long)((args.M + tile_rows - 1) / tile_rows) *
                       ((args.N + cfg.bn - 1) / cfg.bn);
  const int ntiles = int(nt);
  const int workers = bokt::splitk_workers(launched, ntiles, args.split_k);
  const int span = (workers + ntiles - 1) / ntiles + 1;  // workers one tile can touch
  int lanes = 1;
  while (lanes * 4 < span && lanes < 8) lanes *= 2;
  const long long blocks = nt * (pair ? 2 : 1) * (cfg.bn / (32 / lanes));
  if (blocks > 0x7fffffffLL) return fail(BOKT_ERR_UNSUPPORTED, "split-K reduction: too many tiles");
  const float* partials = reinterpret_cast<const float*>(
      static_cast<const uint8_t*>(args.splitk_ws) + bokt::kSplitKHeaderBytes +
      bokt::splitk_flags_bytes(args.splitk_slots));
  const int p = pair ? 1 : 0;
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kernel, auto* c) {
    e = launch(kernel, dim3(unsigned(blocks)), dim3(128 * lanes), 0, s, partials, c, args.M,
               args.N, args.split_k, workers, ntiles, p, cfg.bn, args.group_m);
  };
  if (dtype == BOKT_BF16) {
    auto* c = static_cast<__nv_bfloat16*>(args.C);
    if (lanes == 1) go(bokt::splitk_reduce_kernel<__nv_bfloat16, 1>, c);
    else if (lanes == 2) go(bokt::splitk_reduce_kernel<__nv_bfloat16, 2>, c);
    else if (lanes == 4) go(bokt::splitk_reduce_kernel<__nv_bfloat16, 4>, c);
    else go(bokt::splitk_reduce_kernel<__nv_bfloat16, 8>, c);
  } else {
    auto* c = static_cast<__half*>(args.C);
    if (lanes == 1) go(bokt::splitk_reduce_kernel<__half, 1>, c);
    else if (lanes == 2) go(bokt::splitk_reduce_kernel<__half, 2>, c);
    else if (lanes == 4) go(bokt::splitk_reduce_kernel<__half, 4>, c);
    else go(bokt::splitk_reduce_kernel<__half, 8>, c);
  }
  if (e != cudaSuccess) return cuda_fail(e, "splitk_reduce launch");
  return BOKT_OK;
}

bool tc_eligible(const void* A, const void* B, const void* C, int N, int K) {
  return K > 0 && (K % 8) == 0 && (N % 8) == 0 && aligned16(A) && aligned16(B) && aligned16(C);
}

// Dense GEMM entry body.  row_scale != nullptr scales C row m by row_scale[m]
// in the epilogue (the fused RMSNorm -> GEMM; tcgen05 path only).
int dense_gemm_impl(const void* A, const void* B, void* C, int M, int N, int K, int dtype,
                    const bokt_params* params, void* stream, const float* row_scale,
                    void* workspace = nullptr, int64_t workspace_bytes = 0) {
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (M < 0 || N < 0 || K < 0) return fail(BOKT_ERR_INVALID, "negative size");
  if (M == 0 || N == 0) return BOKT_OK;
  if (!A || !B || !C) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  if (!tc_eligible(A, B, C, N, K)) {
    if (row_scale)
      return fail(BOKT_ERR_UNSUPPORTED,
                  "fused RMSNorm-GEMM needs K > 0, K and N multiples of 8 and 16-byte aligned "
                  "operands (got M=%d N=%d K=%d)", M, N, K);
    return dtype == BOKT_BF16
               ? launch_edge<__nv_bfloat16>(A, B, C, M, N, K, nullptr, 0, 0, dtype, s)
               : launch_edge<__half>(A, B, C, M, N, K, nullptr, 0, 0, dtype, s);
  }
  TcConfig cfg;
  rc = resolve_tc_config(params, false, 0, dev.smem_optin, &cfg);
  if (rc) return rc;
  CUtensorMap ma, mb;
  const uint64_t da[2] = {uint64_t(K), uint64_t(M)};
  const uint64_t sa[1] = {uint64_t(K) * 2};
  const uint32_t ba[2] = {64, 128};
  rc = encode_map(&ma, A, 2, da, sa, ba, dtype == BOKT_FP16);
  if (rc) return rc;
  const uint64_t db[2] = {uint64_t(N), uint64_t(K)};
  const uint64_t sb[1] = {uint64_t(N) * 2};
  const uint32_t bb[2] = {64, 64};
  rc = encode_map(&mb, B, 2, db, sb, bb, dtype == BOKT_FP16);
  if (rc) return rc;
  GemmTcArgs args = {};
  args.C = C;
  args.M = M;
  args.N = N;
  args.K = K;
  args.group_m = cfg.group_m;
  args.stages = cfg.stages;
  args.row_scale = row_scale;
  rc = attach_splitk(cfg, dev, (K + bokt::kGemmBK - 1) / bokt::kGemmBK, workspace,
                     workspace_bytes, &args);
  if (rc) return rc;
  const long long split = args.split_k;
  // Many slices per tile: partials summed by a separate, fully parallel
  // kernel instead of the owner's serial fix-up (not with the fused row scale,
  // which the owner's epilogue applies).
  args.splitk_reduce = split >= bokt::kSplitKReduceMin && !row_scale ? 1 : 0;
  if (cfg.cta_group == 2) {
    args.idesc = bokt::make_idesc_f16(uint32_t(dtype), 256, uint32_t(cfg.bn));
    const long long units = (long long)((M + 255) / 256) * ((N + cfg.bn - 1) / cfg.bn) * split;
    const long long max_pairs = dev.sm_count / 2;
    const int pairs = int(units < max_pairs ? units : max_pairs);
    rc = launch_tc2(dtype, cfg, ma, mb, args, pairs, s);
    if (rc || !args.splitk_reduce) return rc;
    return launch_splitk_reduce(dtype, cfg, args, pairs, true, s);
  }
  args.idesc = bokt::make_idesc_f16(uint32_t(dtype), 128, uint32_t(cfg.bn));
  const long long units = (long long)((M + 127) / 128) * ((N + cfg.bn - 1) / cfg.bn) * split;
  const int grid = int(units < dev.sm_count ? units : dev.sm_count);
  rc = launch_tc(false, dtype, cfg, ma, mb, args, grid, s);
  if (rc || !args.splitk_reduce) return rc;
  return launch_splitk_reduce(dtype, cfg, args, grid, false, s);
}

// ----------------------------------------------------------------- RMSNorm dispatch
struct NormConfig {
  int rows_per_cta, threads, tpr_log2, vpt;  // vpt 0 = generic kernel
  int ring_slots;                            // > 0: persistent TMA-staged ring kernel
};

int resolve_norm_config(const bokt_params* p, int N, bool vec_ok, NormConfig* out) {
  const bokt_params zero = {};
  if (!p) p = &zero;
  const int rows = param_or(p->rows_per_cta, 1);
  const int warps = param_or(p->num_warps, 4);
  if (warps != 1 && warps != 2 && warps != 4 && warps != 8 && warps != 16 && warps != 32)
    return fail(BOKT_ERR_CONFIG, "num_warps must be a power of two <= 32 (got %d)", warps);
  if (rows != 1 && rows != 2 && rows != 4 && rows != 8 && rows != 16)
    return fail(BOKT_ERR_CONFIG, "rows_per_cta must be 1, 2, 4, 8 or 16 (got %d)", rows);
  const int threads = warps * 32;
  if (rows > threads) return fail(BOKT_ERR_CONFIG, "rows_per_cta exceeds threads per CTA");
  const int tpr = threads / rows;
  int lg = 0;
  while ((1 << lg) < tpr) ++lg;
  int vpt = 0;
  if (vec_ok) {
    const int nvec = N / 8;
    const int need = (nvec + tpr - 1) / tpr;
    int v = 1;
    while (v < need) v <<= 1;
    if (v <= 16) vpt = v;
  }
  const int stages = param_or(p->stages, 1);
  if (stages < 1 || stages > 32) return fail(BOKT_ERR_CONFIG, "stages must be in [1, 32]");
  // The ring kernel streams whole rows with cp.async.bulk (16-byte multiples,
  // 16-byte aligned); odd or unaligned rows take the per-row kernels instead,
  // as odd GEMM shapes take the edge GEMM kernel.
  int ring = 0;
  if (stages == 2 && vec_ok && rows == 1 && vpt > 0 && vpt <= 8) {
    // Two register buffers: the persistent software-pipelined kernel (one row
    // per CTA at a time).  Other shapes keep the per-row kernels.
    *out = {rows, threads, lg, vpt, -1};
    return BOKT_OK;
  }
  if (stages >= 4 && vec_ok) {
    if (warps > 31) return fail(BOKT_ERR_CONFIG, "ring kernel: num_warps must be <= 31");
    if (stages % warps != 0)
      return fail(BOKT_ERR_CONFIG,
                  "ring kernel: stages (%d) must be a multiple of num_warps (%d) so each ring "
                  "slot is consumed by one warp",
                  stages, warps);
    ring = stages;
  }
  *out = {rows, threads, lg, vpt, ring};
  return BOKT_OK;
}

// The three routing launches, scratch = ceil(A / 4096) * E int32 words.
int launch_route(const int32_t* ids, int A, int E, int32_t* scratch, int32_t* counts,
                 int32_t* offsets, int64_t* offsets64, int32_t* perm, int32_t* inv_perm,
                 cudaStream_t s, const char* what) {
  const int chunks = (A + bokt::kRouteChunk - 1) / bokt::kRouteChunk;
  cudaError_t e = cudaSuccess;
  if (chunks > 0)
    e = launch(bokt::route_count_kernel, dim3(chunks), dim3(bokt::kRouteThreads), 0, s, ids, A, E,
               scratch);
  if (e == cudaSuccess)
    e = launch(bokt::route_scan_kernel, dim3(1), dim3(1024), 0, s, scratch, chunks, E, counts,
               offsets, reinterpret_cast<long long*>(offsets64));
  if (e == cudaSuccess && chunks > 0)
    e = launch(bokt::route_scatter_kernel, dim3(chunks), dim3(bokt::kRouteThreads), 0, s, ids, A,
               E, static_cast<const int32_t*>(scratch), perm, inv_perm);
  if (e != cudaSuccess) return cuda_fail(e, what);
  return BOKT_OK;
}

template <typename T>
const void* pipe_kernel(int vpt) {
  switch (vpt) {
    case 1: return reinterpret_cast<const void*>(&bokt::rmsnorm_pipe_kernel<T, 1>);
    case 2: return reinterpret_cast<const void*>(&bokt::rmsnorm_pipe_kernel<T, 2>);
    case 4: return reinterpret_cast<const void*>(&bokt::rmsnorm_pipe_kernel<T, 4>);
    case 8: return reinterpret_cast<const void*>(&bokt::rmsnorm_pipe_kernel<T, 8>);
  }
  return nullptr;
}

template <typename T>
const void* norm_kernel(int vpt) {
  switch (vpt) {
    case 0: return reinterpret_cast<const void*>(&bokt::rmsnorm_generic_kernel<T>);
    case 1: return reinterpret_cast<const void*>(&bokt::rmsnorm_vec_kernel<T, 1>);
    case 2: return reinterpret_cast<const void*>(&bokt::rmsnorm_vec_kernel<T, 2>);
    case 4: return reinterpret_cast<const void*>(&bokt::rmsnorm_vec_kernel<T, 4>);
    case 8: return reinterpret_cast<const void*>(&bokt::rmsnorm_vec_kernel<T, 8>);
    case 16: return reinterpret_cast<const void*>(&bokt::rmsnorm_vec_kernel<T, 16>);
  }
  return nullptr;
}

}  // namespace

// =================================================================== C ABI
extern "C" {

int bokt_abi_version(void) { return BOKT_ABI_VERSION; }

int bokt_built_sm(void) { return 100; }

const char* bokt_last_error(void) { return g_err; }

int bokt_gemm(const void* A, const void* B, void* C, int M, int N, int K, int dtype,
              const bokt_params* params, void* stream) {
  g_err[0] = 0;
  return dense_gemm_impl(A, B, C, M, N, K, dtype, params, stream, nullptr);
}

int bokt_gemm_ex(const void* A, const void* B, void* C, int M, int N, int K, int dtype,
                 const bokt_params* params, void* workspace, int64_t workspace_bytes,
                 void* stream) {
  g_err[0] = 0;
  return dense_gemm_impl(A, B, C, M, N, K, dtype, params, stream, nullptr, workspace,
                         workspace_bytes);
}

int64_t bokt_gemm_workspace_bytes(int kernel, const bokt_params* params) {
  g_err[0] = 0;
  if (kernel != BOKT_KERNEL_GEMM && kernel != BOKT_KERNEL_MOE_GROUPED_GEMM) return 0;
  const bokt_params zero = {};
  const bokt_params* p = params ? params : &zero;
  if (param_or(p->split_k, 1) <= 1) return 0;
  DeviceInfo dev;
  if (device_info(&dev)) return -1;
  return splitk_bytes_for(dev, param_or(p->block_n, 256));
}

int bokt_rmsnorm_fold_weight(const void* norm_weight, const void* B, void* B_folded, int K, int N,
                             int dtype, void* stream) {
  g_err[0] = 0;
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (K < 0 || N < 0) return fail(BOKT_ERR_INVALID, "negative size");
  if (K == 0 || N == 0) return BOKT_OK;
  if (!norm_weight || !B || !B_folded) return fail(BOKT_ERR_INVALID, "null pointer");
  if (N % 8 != 0 || !aligned16(B) || !aligned16(B_folded))
    return fail(BOKT_ERR_UNSUPPORTED, "fold needs N %% 8 == 0 and 16-byte aligned B, B_folded");
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  const long long vecs = (long long)K * (N / 8);
  long long blocks = (vecs + 255) / 256;
  if (blocks > 8LL * dev.sm_count) blocks = 8LL * dev.sm_count;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = dtype == BOKT_BF16
      ? launch(bokt::fold_norm_weight_kernel<__nv_bfloat16>, dim3(unsigned(blocks)), dim3(256), 0, s,
               static_cast<const __nv_bfloat16*>(norm_weight),
               static_cast<const __nv_bfloat16*>(B), static_cast<__nv_bfloat16*>(B_folded), K, N)
      : launch(bokt::fold_norm_weight_kernel<__half>, dim3(unsigned(blocks)), dim3(256), 0, s,
               static_cast<const __half*>(norm_weight), static_cast<const __half*>(B),
               static_cast<__half*>(B_folded), K, N);
  if (e != cudaSuccess) return cuda_fail(e, "fold_norm_weight launch");
  return BOKT_OK;
}

int bokt_rmsnorm_row_scale(const void* X, float* scale, int M, int K, float eps, int dtype,
                           void* stream) {
  g_err[0] = 0;
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (M < 0 || K <= 0) return fail(BOKT_ERR_INVALID, "bad size");
  if (M == 0) return BOKT_OK;
  if (!X || !scale) return fail(BOKT_ERR_INVALID, "null pointer");
  if (!(eps >= 0.f) || !(eps < 3.0e38f)) return fail(BOKT_ERR_INVALID, "eps must be finite >= 0");
  if (K % 8 != 0 || !aligned16(X))
    return fail(BOKT_ERR_UNSUPPORTED, "row scale needs K %% 8 == 0 and a 16-byte aligned X");
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  const int warps = bokt::kRowScaleThreads / 32;
  long long blocks = ((long long)M + warps - 1) / warps;
  if (blocks > 16LL * dev.sm_count) blocks = 16LL * dev.sm_count;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = dtype == BOKT_BF16
      ? launch(bokt::rmsnorm_row_scale_kernel<__nv_bfloat16>, dim3(unsigned(blocks)),
               dim3(bokt::kRowScaleThreads), 0, s, static_cast<const __nv_bfloat16*>(X), scale, M,
               K, eps)
      : launch(bokt::rmsnorm_row_scale_kernel<__half>, dim3(unsigned(blocks)),
               dim3(bokt::kRowScaleThreads), 0, s, static_cast<const __half*>(X), scale, M, K, eps);
  if (e != cudaSuccess) return cuda_fail(e, "rmsnorm_row_scale launch");
  return BOKT_OK;
}

int bokt_gemm_row_scaled(const void* A, const void* B, void* C, const float* row_scale, int M,
                         int N, int K, int dtype, const bokt_params* params, void* stream) {
  g_err[0] = 0;
  if (!row_scale) return fail(BOKT_ERR_INVALID, "null row_scale");
  return dense_gemm_impl(A, B, C, M, N, K, dtype, params, stream, row_scale);
}

int bokt_rmsnorm_gemm(const void* X, const void* B_folded, void* C, float* row_scale, int M,
                      int N, int K, float eps, int dtype, const bokt_params* params,
                      void* stream) {
  g_err[0] = 0;
  if (!row_scale) return fail(BOKT_ERR_INVALID, "null row_scale workspace");
  if (M > 0 && N > 0 && !tc_eligible(X, B_folded, C, N, K))
    return fail(BOKT_ERR_UNSUPPORTED,
                "fused RMSNorm-GEMM needs K > 0, K and N multiples of 8 and 16-byte aligned "
                "operands (got M=%d N=%d K=%d)", M, N, K);
  int rc = bokt_rmsnorm_row_scale(X, row_scale, M, K, eps, dtype, stream);
  if (rc) return rc;
  return dense_gemm_impl(X, B_folded, C, M, N, K, dtype, params, stream, row_scale);
}

}  // extern "C"

namespace {

// Shared body of the grouped GEMM entry points; scatter != nullptr selects the
// expert-parallel epilogue that sends each packed row to its owner's buffer.
struct ScatterArgs {
  const int32_t* rowmap;
  void* const* out_ptrs;
  int rows_per_owner;
  int owners;
};

int grouped_gemm_impl(const void* X, const void* W, const void* offsets, int offsets_is_i64,
                      void* Y, int T, int E, int N, int K, int dtype, int sm_count,
                      const bokt_params* params, void* stream, const ScatterArgs* scatter,
                      void* workspace = nullptr, int64_t workspace_bytes = 0) {
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (T < 0 || E < 0 || N < 0 || K < 0) return fail(BOKT_ERR_INVALID, "negative size");
  if (E > bokt::kGemmMaxExperts)
    return fail(BOKT_ERR_UNSUPPORTED, "at most %d experts", bokt::kGemmMaxExperts);
  if (T == 0 || E == 0 || N == 0) return BOKT_OK;
  if (!X || !W || !Y || !offsets) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  if (!tc_eligible(X, W, Y, N, K)) {
    if (scatter)
      return fail(BOKT_ERR_UNSUPPORTED,
                  "scatter epilogue needs the tcgen05 path (K, N multiples of 8, aligned)");
    return dtype == BOKT_BF16
               ? launch_edge<__nv_bfloat16>(X, W, Y, T, N, K, offsets, offsets_is_i64, E, dtype, s)
               : launch_edge<__half>(X, W, Y, T, N, K, offsets, offsets_is_i64, E, dtype, s);
  }
  const bokt_params zero = {};
  TcConfig cfg;
  rc = resolve_tc_config(params, true, E, dev.smem_optin, &cfg);
  if (rc) return rc;
  CUtensorMap ma, mb;
  const uint64_t da[2] = {uint64_t(K), uint64_t(T)};
  const uint64_t sa[1] = {uint64_t(K) * 2};
  const uint32_t ba[2] = {64, 128};
  rc = encode_map(&ma, X, 2, da, sa, ba, dtype == BOKT_FP16);
  if (rc) return rc;
  const uint64_t db[3] = {uint64_t(N), uint64_t(K), uint64_t(E)};
  const uint64_t sb[2] = {uint64_t(N) * 2, uint64_t(K) * uint64_t(N) * 2};
  const uint32_t bb[3] = {64, 64, 1};
  rc = encode_map(&mb, W, 3, db, sb, bb, dtype == BOKT_FP16);
  if (rc) return rc;
  GemmTcArgs args = {};
  args.C = Y;
  args.M = T;
  args.N = N;
  args.K = K;
  args.group_m = 1;
  args.stages = cfg.stages;
  args.idesc = bokt::make_idesc_f16(uint32_t(dtype), 128, uint32_t(cfg.bn));
  args.offsets = offsets;
  args.offsets_i64 = offsets_is_i64 ? 1 : 0;
  args.E = E;
  args.raster = cfg.raster;
  if (scatter) {
    args.rowmap = scatter->rowmap;
    args.out_ptrs = scatter->out_ptrs;
    args.rows_per_owner = scatter->rows_per_owner;
    args.owners = scatter->owners;
  }
  const int mult = param_or((params ? params : &zero)->cta_multiplier, 1);
  const int sms = sm_count > 0 ? sm_count : dev.sm_count;
  const long long nn = (N + cfg.bn - 1) / cfg.bn;
  if (cfg.cta_group == 2) {
    // CTA pairs: 256-row tiles per expert, a last block of <= 128 rows as a
    // half-height tile (M = 128, 64 rows per CTA, A boxes of 64 rows).
    CUtensorMap ma64;
    const uint32_t ba64[2] = {64, 64};
    rc = encode_map(&ma64, X, 2, da, sa, ba64, dtype == BOKT_FP16);
    if (rc) return rc;
    GemmTcArgs pa = args;
    pa.idesc = bokt::make_idesc_f16(uint32_t(dtype), 256, uint32_t(cfg.bn));
    pa.idesc_half = bokt::make_idesc_f16(uint32_t(dtype), 128, uint32_t(cfg.bn));
    const long long max_pair_tiles = ((long long)(T + 255) / 256 + E) * nn;
    long long pairs = sms / 2;
    if (pairs > max_pair_tiles) pairs = max_pair_tiles;
    if (pairs < 1) pairs = 1;
    return launch_tc2(dtype, cfg, ma, mb, pa, int(pairs), s, /*grouped=*/true, scatter != nullptr,
                      &ma64);
  }
  rc = attach_splitk(cfg, dev, (K + bokt::kGemmBK - 1) / bokt::kGemmBK, workspace,
                     workspace_bytes, &args);
  if (rc) return rc;
  // Upper bound on tiles without reading offsets: sum_e cdiv(c_e, 128) <= cdiv(T, 128) + E.
  const long long max_tiles = ((long long)(T + 127) / 128 + E) * nn;
  long long grid = (long long)sms * mult;
  if (args.split_k > 1 && grid > dev.sm_count) grid = dev.sm_count;  // one slot per CTA
  if (grid > max_tiles * args.split_k) grid = max_tiles * args.split_k;
  if (grid < 1) grid = 1;
  return launch_tc(true, dtype, cfg, ma, mb, args, int(grid), s, scatter != nullptr);
}

}  // namespace

extern "C" {

int bokt_moe_grouped_gemm(const void* X, const void* W, const void* offsets, int offsets_is_i64,
                          void* Y, int T, int E, int N, int K, int dtype, int sm_count,
                          const bokt_params* params, void* stream) {
  g_err[0] = 0;
  return grouped_gemm_impl(X, W, offsets, offsets_is_i64, Y, T, E, N, K, dtype, sm_count, params,
                           stream, nullptr);
}

int bokt_moe_grouped_gemm_ex(const void* X, const void* W, const void* offsets,
                             int offsets_is_i64, void* Y, int T, int E, int N, int K, int dtype,
                             int sm_count, const bokt_params* params, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  return grouped_gemm_impl(X, W, offsets, offsets_is_i64, Y, T, E, N, K, dtype, sm_count, params,
                           stream, nullptr, workspace, workspace_bytes);
}

int bokt_moe_grouped_gemm_scatter(const void* X, const void* W, const void* offsets,
                                  int offsets_is_i64, int T, int E, int N, int K, int dtype,
                                  int sm_count, const int32_t* rowmap, void* const* out_ptrs,
                                  int rows_per_owner, int owners, const bokt_params* params,
                                  void* stream) {
  g_err[0] = 0;
  if (!rowmap || !out_ptrs || rows_per_owner <= 0 || owners <= 0)
    return fail(BOKT_ERR_INVALID, "scatter needs rowmap, out_ptrs, rows_per_owner, owners");
  const ScatterArgs sc = {rowmap, out_ptrs, rows_per_owner, owners};
  // Y is unused by the scatter epilogue; any valid aligned pointer satisfies the path checks.
  return grouped_gemm_impl(X, W, offsets, offsets_is_i64, const_cast<void*>(X), T, E, N, K,
                           dtype, sm_count, params, stream, &sc);
}

int bokt_ep_plan(const int32_t* counts, const int32_t* offsets, const int32_t* replicas, int E,
                 const int32_t* v_rank, int V, int world, int me, const int32_t* capacity,
                 int32_t* v_plo, int32_t* v_size, int32_t* v_lbase, int32_t* loffs,
                 int32_t* rank_rows, void* stream) {
  g_err[0] = 0;
  if (E <= 0 || V <= 0 || world <= 0 || me < 0 || me >= world)
    return fail(BOKT_ERR_INVALID, "bad size");
  if (!counts || !offsets || !replicas || !v_rank || !capacity || !v_plo || !v_size ||
      !v_lbase || !loffs || !rank_rows)
    return fail(BOKT_ERR_INVALID, "null pointer");
  const int smem = bokt::ep_plan_smem_bytes(E, V, world);
  if (smem > 200 * 1024) return fail(BOKT_ERR_UNSUPPORTED, "ep_plan: E, V or world too large");
  int rc = ensure_smem(reinterpret_cast<const void*>(&bokt::ep_plan_kernel), smem);
  if (rc) return rc;
  cudaError_t e = launch(bokt::ep_plan_kernel, dim3(1), dim3(256), smem,
                         static_cast<cudaStream_t>(stream), counts, offsets, replicas, E, v_rank,
                         V, world, me, capacity, v_plo, v_size, v_lbase, loffs, rank_rows);
  if (e != cudaSuccess) return cuda_fail(e, "ep_plan launch");
  return BOKT_OK;
}

int bokt_ep_dispatch(const void* x_local, int cols, int elem_bytes, const int32_t* ids,
                     const int32_t* inv_perm, const int32_t* offsets, const int32_t* counts,
                     const int32_t* replicas, const int32_t* vbase, const int32_t* v_rank,
                     const int32_t* v_plo, const int32_t* v_lbase, void* const* xpk_ptrs,
                     const int32_t* capacity, int a_local, int topk, int me, int E,
                     void* stream) {
  g_err[0] = 0;
  if (cols <= 0 || elem_bytes <= 0 || a_local < 0 || topk <= 0 || me < 0 || E <= 0)
    return fail(BOKT_ERR_INVALID, "bad size");
  if (a_local == 0) return BOKT_OK;
  const long long row_bytes = (long long)cols * elem_bytes;
  if (row_bytes % 16 != 0 || !aligned16(x_local))
    return fail(BOKT_ERR_UNSUPPORTED, "dispatch rows must be 16-byte multiples, 16-byte aligned");
  if (!ids || !inv_perm || !offsets || !counts || !replicas || !vbase || !v_rank || !v_plo ||
      !v_lbase || !xpk_ptrs || !capacity)
    return fail(BOKT_ERR_INVALID, "null pointer");
  const int warps_per_block = 8;
  int grid = (a_local + warps_per_block - 1) / warps_per_block;
  if (grid > 148 * 16) grid = 148 * 16;
  cudaError_t e = launch(bokt::ep_dispatch_kernel, dim3(grid), dim3(32 * warps_per_block), 0,
                         static_cast<cudaStream_t>(stream), static_cast<const uint4*>(x_local),
                         int(row_bytes / 16), ids, inv_perm, offsets, counts, replicas, vbase,
                         v_rank, v_plo, v_lbase, reinterpret_cast<uint4* const*>(xpk_ptrs),
                         capacity, a_local, topk, me, E);
  if (e != cudaSuccess) return cuda_fail(e, "ep_dispatch launch");
  return BOKT_OK;
}

int bokt_ep_put(const void* src, int64_t bytes, void* const* dst_ptrs, int64_t dst_offset_bytes,
                int world, void* stream) {
  g_err[0] = 0;
  if (bytes < 0 || dst_offset_bytes < 0 || world <= 0 || world > bokt::kEpMaxWorld)
    return fail(BOKT_ERR_INVALID, "bad size");
  if (bytes == 0) return BOKT_OK;
  if (!src || !dst_ptrs) return fail(BOKT_ERR_INVALID, "null pointer");
  if (bytes % 16 != 0 || dst_offset_bytes % 16 != 0 || !aligned16(src))
    return fail(BOKT_ERR_UNSUPPORTED, "put needs 16-byte aligned source, size and offset");
  const long long vecs = bytes / 16;
  long long grid = (vecs + 255) / 256;
  if (grid > 148 * 4) grid = 148 * 4;
  cudaError_t e = launch(bokt::ep_put_kernel, dim3(unsigned(grid)), dim3(256), 0,
                         static_cast<cudaStream_t>(stream), static_cast<const uint4*>(src),
                         (long long)vecs, reinterpret_cast<uint4* const*>(dst_ptrs),
                         (long long)(dst_offset_bytes / 16), world);
  if (e != cudaSuccess) return cuda_fail(e, "ep_put launch");
  return BOKT_OK;
}

int bokt_ep_barrier(int32_t* const* flag_ptrs, int32_t* epoch, int world, int me,
                    int64_t timeout_ns, void* stream) {
  g_err[0] = 0;
  if (world <= 0 || world > bokt::kEpMaxWorld || me < 0 || me >= world)
    return fail(BOKT_ERR_INVALID, "bad world/rank");
  if (timeout_ns <= 0 || timeout_ns > 60000000000ll)
    return fail(BOKT_ERR_INVALID, "timeout must be in (0, 60 s]");
  if (!flag_ptrs || !epoch) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaError_t e = launch(bokt::ep_barrier_kernel, dim3(1), dim3(32), 0,
                         static_cast<cudaStream_t>(stream), flag_ptrs, epoch, world, me,
                         (long long)timeout_ns);
  if (e != cudaSuccess) return cuda_fail(e, "ep_barrier launch");
  return BOKT_OK;
}

int bokt_ep_barrier_combine(int32_t* const* flag_ptrs, int32_t* epoch, int world, int me,
                            int64_t timeout_ns, const void* y, const float* gates, void* out,
                            int tokens, int k, int N, int dtype, void* stream) {
  g_err[0] = 0;
  if (world <= 0 || world > bokt::kEpMaxWorld || me < 0 || me >= world)
    return fail(BOKT_ERR_INVALID, "bad world/rank");
  if (timeout_ns <= 0 || timeout_ns > 60000000000ll)
    return fail(BOKT_ERR_INVALID, "timeout must be in (0, 60 s]");
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (tokens < 0 || k <= 0 || N <= 0) return fail(BOKT_ERR_INVALID, "bad size");
  if (!flag_ptrs || !epoch || (tokens > 0 && (!y || !gates || !out)))
    return fail(BOKT_ERR_INVALID, "null pointer");
  if (N % 8 != 0 || (tokens > 0 && (!aligned16(y) || !aligned16(out))))
    return fail(BOKT_ERR_UNSUPPORTED, "combine needs N %% 8 == 0 and 16-byte aligned rows");
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  // Every CTA waits for the peers, so keep the grid within one wave.
  long long grid = tokens < 1 ? 1 : tokens;
  if (grid > 4LL * dev.sm_count) grid = 4LL * dev.sm_count;
  const int threads = N / 8 < 256 ? ((N / 8 + 31) / 32) * 32 : 256;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long y_rows = (long long)tokens * k;
  cudaError_t e =
      dtype == BOKT_BF16
          ? launch(bokt::ep_barrier_combine_kernel<__nv_bfloat16>, dim3(unsigned(grid)),
                   dim3(threads), 0, s, flag_ptrs, epoch, world, me, (long long)timeout_ns,
                   static_cast<const __nv_bfloat16*>(y), y_rows, gates,
                   static_cast<__nv_bfloat16*>(out), tokens, k, N)
          : launch(bokt::ep_barrier_combine_kernel<__half>, dim3(unsigned(grid)), dim3(threads),
                   0, s, flag_ptrs, epoch, world, me, (long long)timeout_ns,
                   static_cast<const __half*>(y), y_rows, gates, static_cast<__half*>(out),
                   tokens, k, N);
  if (e != cudaSuccess) return cuda_fail(e, "ep_barrier_combine launch");
  return BOKT_OK;
}

int bokt_ep_rowmap(const int32_t* perm, const int32_t* ids, const int32_t* offsets,
                   const int32_t* counts, const int32_t* replicas, const int32_t* vbase,
                   const int32_t* v_rank, const int32_t* v_plo, const int32_t* v_lbase, int A,
                   int E, int me, int capacity, int32_t* rowmap, void* stream) {
  g_err[0] = 0;
  if (A < 0 || E <= 0 || me < 0 || capacity < 0) return fail(BOKT_ERR_INVALID, "bad size");
  if (A == 0) return BOKT_OK;
  if (!perm || !ids || !offsets || !counts || !replicas || !vbase || !v_rank || !v_plo ||
      !v_lbase || !rowmap)
    return fail(BOKT_ERR_INVALID, "null pointer");
  const int grid = (A + 255) / 256 < 4096 ? (A + 255) / 256 : 4096;
  cudaError_t e = launch(bokt::ep_rowmap_kernel, dim3(grid), dim3(256), 0,
                         static_cast<cudaStream_t>(stream), perm, ids, offsets, counts, replicas,
                         vbase, v_rank, v_plo, v_lbase, A, E, me, capacity, rowmap);
  if (e != cudaSuccess) return cuda_fail(e, "ep_rowmap launch");
  return BOKT_OK;
}

int bokt_rmsnorm(const void* X, const void* W, void* Y, int M, int N, float eps, int dtype,
                 const bokt_params* params, void* stream) {
  g_err[0] = 0;
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (M < 0 || N < 0) return fail(BOKT_ERR_INVALID, "negative size");
  if (M == 0 || N == 0) return BOKT_OK;
  if (!X || !W || !Y) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool vec_ok = (N % 8) == 0 && aligned16(X) && aligned16(W) && aligned16(Y);
  NormConfig cfg;
  int rc = resolve_norm_config(params, N, vec_ok, &cfg);
  if (rc) return rc;
  if (cfg.ring_slots < 0) {
    DeviceInfo dev;
    rc = device_info(&dev);
    if (rc) return rc;
    const void* pfn = dtype == BOKT_BF16 ? pipe_kernel<__nv_bfloat16>(cfg.vpt)
                                         : pipe_kernel<__half>(cfg.vpt);
    int per_sm = 0;
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, pfn, cfg.threads, 0);
    if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
    if (per_sm < 1) per_sm = 1;
    long long grid = (long long)dev.sm_count * per_sm;
    if (grid > M) grid = M;
    void* pargs[] = {const_cast<void**>(&X), const_cast<void**>(&W), &Y, &M, &N, &eps,
                     &cfg.tpr_log2};
    e = launch_ptr(pfn, dim3(unsigned(grid)), dim3(cfg.threads), 0, s, pargs);
    if (e != cudaSuccess) return cuda_fail(e, "rmsnorm pipe launch");
    return BOKT_OK;
  }
  if (cfg.ring_slots > 0) {
    DeviceInfo dev;
    rc = device_info(&dev);
    if (rc) return rc;
    const int smem = bokt::rmsnorm_ring_smem_bytes(N, 2, cfg.ring_slots);
    if (smem > dev.smem_optin)
      return fail(BOKT_ERR_CONFIG, "ring kernel: %d slots of %d-element rows need %d bytes of "
                                   "shared memory (max %d)", cfg.ring_slots, N, smem,
                  dev.smem_optin);
    const void* rfn = dtype == BOKT_BF16
                          ? reinterpret_cast<const void*>(&bokt::rmsnorm_ring_kernel<__nv_bfloat16>)
                          : reinterpret_cast<const void*>(&bokt::rmsnorm_ring_kernel<__half>);
    rc = ensure_smem(rfn, smem);
    if (rc) return rc;
    int per_sm = (228 * 1024) / (smem + 1024);
    if (per_sm < 1) per_sm = 1;
    if (per_sm > 4) per_sm = 4;
    long long grid = (long long)dev.sm_count * per_sm;
    if (grid > M) grid = M;
    int slots = cfg.ring_slots;
    void* rargs[] = {const_cast<void**>(&X), const_cast<void**>(&W), &Y, &M, &N, &eps, &slots};
    cudaError_t e = launch_ptr(rfn, dim3(unsigned(grid)), dim3(cfg.threads + 32), smem, s, rargs);
    if (e != cudaSuccess) return cuda_fail(e, "rmsnorm ring launch");
    return BOKT_OK;
  }
  const int grid = (M + cfg.rows_per_cta - 1) / cfg.rows_per_cta;
  const void* fn = dtype == BOKT_BF16 ? norm_kernel<__nv_bfloat16>(cfg.vpt)
                                      : norm_kernel<__half>(cfg.vpt);
  void* kargs[] = {const_cast<void**>(&X), const_cast<void**>(&W), &Y, &M, &N, &eps,
                   &cfg.rows_per_cta, &cfg.tpr_log2};
  cudaError_t e = launch_ptr(fn, dim3(grid), dim3(cfg.threads), 0, s, kargs);
  if (e != cudaSuccess) return cuda_fail(e, "rmsnorm launch");
  return BOKT_OK;
}

int64_t bokt_moe_route_workspace_bytes(int A, int E) {
  if (A < 0 || E <= 0) return 0;
  const int64_t chunks = (A + bokt::kRouteChunk - 1) / bokt::kRouteChunk;
  return (chunks > 0 ? chunks : 1) * int64_t(E) * 4;
}

int bokt_moe_route(const int32_t* expert_ids, int A, int E, int32_t* counts, int32_t* offsets,
                   int64_t* offsets64, int32_t* perm, int32_t* inv_perm, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (A < 0 || E <= 0) return fail(BOKT_ERR_INVALID, "need A >= 0 and E > 0");
  if (E > bokt::kRouteMaxExperts)
    return fail(BOKT_ERR_UNSUPPORTED, "at most %d experts", bokt::kRouteMaxExperts);
  if (!counts || !offsets || (A > 0 && (!expert_ids || !perm || !inv_perm)))
    return fail(BOKT_ERR_INVALID, "null pointer");
  if (workspace_bytes < bokt_moe_route_workspace_bytes(A, E) || !workspace)
    return fail(BOKT_ERR_INVALID, "workspace too small: need %lld bytes",
                (long long)bokt_moe_route_workspace_bytes(A, E));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int32_t* ws = static_cast<int32_t*>(workspace);
  return launch_route(expert_ids, A, E, ws, counts, offsets, offsets64, perm, inv_perm, s,
                      "moe_route launch");
}

int bokt_gather_rows(const void* src, int64_t src_rows, void* dst, const int32_t* index, int rows,
                     int cols, int elem_bytes, int divisor, void* stream) {
  g_err[0] = 0;
  if (rows < 0 || cols < 0 || src_rows < 0 || divisor <= 0 || elem_bytes <= 0)
    return fail(BOKT_ERR_INVALID, "bad size");
  if (rows == 0 || cols == 0) return BOKT_OK;
  if (!src || !dst || !index) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long row_bytes = (long long)cols * elem_bytes;
  const int grid = rows < 65535 * 4 ? rows : 65535 * 4;
  cudaError_t e;
  if (row_bytes % 16 == 0 && aligned16(src) && aligned16(dst)) {
    const int vecs = int(row_bytes / 16);
    e = launch(bokt::gather_rows_kernel<uint4>, dim3(grid), dim3(128), 0, s,
               static_cast<const uint4*>(src), (long long)src_rows, static_cast<uint4*>(dst), index,
               rows, vecs, divisor);
  } else {
    e = launch(bokt::gather_rows_kernel<uint8_t>, dim3(grid), dim3(128), 0, s,
               static_cast<const uint8_t*>(src), (long long)src_rows, static_cast<uint8_t*>(dst),
               index, rows, int(row_bytes), divisor);
  }
  if (e != cudaSuccess) return cuda_fail(e, "gather_rows launch");
  return BOKT_OK;
}

int bokt_gather_rows_indirect(const void* src, int64_t src_rows, void* dst, const int32_t* inner,
                               int64_t inner_len, const int32_t* outer, int rows, int cols,
                               int elem_bytes, int divisor, int64_t base, void* stream) {
  g_err[0] = 0;
  if (rows < 0 || cols < 0 || src_rows < 0 || divisor <= 0 || elem_bytes <= 0 || inner_len < 0)
    return fail(BOKT_ERR_INVALID, "bad size");
  if (rows == 0 || cols == 0) return BOKT_OK;
  if (!src || !dst || !inner) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long row_bytes = (long long)cols * elem_bytes;
  const int grid = rows < 65535 * 4 ? rows : 65535 * 4;
  cudaError_t e;
  if (row_bytes % 16 == 0 && aligned16(src) && aligned16(dst)) {
    e = launch(bokt::gather_rows_indirect_kernel<uint4>, dim3(grid), dim3(128), 0, s,
               static_cast<const uint4*>(src), (long long)src_rows, static_cast<uint4*>(dst),
               inner, outer, (long long)inner_len, rows, int(row_bytes / 16), divisor,
               (long long)base);
  } else {
    e = launch(bokt::gather_rows_indirect_kernel<uint8_t>, dim3(grid), dim3(128), 0, s,
               static_cast<const uint8_t*>(src), (long long)src_rows, static_cast<uint8_t*>(dst),
               inner, outer, (long long)inner_len, rows, int(row_bytes), divisor,
               (long long)base);
  }
  if (e != cudaSuccess) return cuda_fail(e, "gather_rows_indirect launch");
  return BOKT_OK;
}

int bokt_ep_keys(const int32_t* perm, const int32_t* ids, const int32_t* offsets,
                 const int32_t* counts, const int32_t* replicas, const int32_t* vbase,
                 const int32_t* v_rank, const int32_t* v_local, int A, int E, int topk,
                 int tokens_per_rank, int me, int world, int n_local, int32_t* key_send,
                 int32_t* key_recv, int32_t* key_local, void* stream) {
  g_err[0] = 0;
  if (A < 0 || E <= 0 || topk <= 0 || tokens_per_rank <= 0 || world <= 0 || me < 0 ||
      me >= world || n_local < 0)
    return fail(BOKT_ERR_INVALID, "bad size");
  if (A == 0) return BOKT_OK;
  if (!perm || !ids || !offsets || !counts || !replicas || !vbase || !v_rank || !v_local ||
      !key_send || !key_recv || !key_local)
    return fail(BOKT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = (A + 255) / 256 < 4096 ? (A + 255) / 256 : 4096;
  cudaError_t e = launch(bokt::ep_keys_kernel, dim3(grid), dim3(256), 0, s, perm, ids, offsets,
                         counts, replicas, vbase, v_rank, v_local, A, E, topk, tokens_per_rank,
                         me, world, n_local, key_send, key_recv, key_local);
  if (e != cudaSuccess) return cuda_fail(e, "ep_keys launch");
  return BOKT_OK;
}

int bokt_check_counts(const int32_t* counts, const int32_t* expected, int n, int tag,
                      void* stream) {
  g_err[0] = 0;
  if (n < 0) return fail(BOKT_ERR_INVALID, "bad size");
  if (n == 0) return BOKT_OK;
  if (!counts || !expected) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaError_t e = launch(bokt::check_counts_kernel, dim3(1), dim3(256), 0,
                         static_cast<cudaStream_t>(stream), counts, expected, n, tag);
  if (e != cudaSuccess) return cuda_fail(e, "check_counts launch");
  return BOKT_OK;
}

int bokt_ipc_export(const void* ptr, void* handle_out, int64_t* offset_out) {
  g_err[0] = 0;
  if (!ptr || !handle_out || !offset_out) return fail(BOKT_ERR_INVALID, "null pointer");
  static PFN_cuMemGetAddressRange_v3020 get_range = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &fn, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      get_range = reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(fn);
  });
  if (!get_range) return fail(BOKT_ERR_CUDA, "cuMemGetAddressRange entry point unavailable");
  CUdeviceptr base = 0;
  size_t size = 0;
  CUresult r = get_range(&base, &size, reinterpret_cast<CUdeviceptr>(ptr));
  if (r != CUDA_SUCCESS) return fail(BOKT_ERR_CUDA, "cuMemGetAddressRange failed (%d)", int(r));
  cudaIpcMemHandle_t h;
  cudaError_t e = cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base));
  if (e != cudaSuccess) return cuda_fail(e, "cudaIpcGetMemHandle");
  memcpy(handle_out, &h, sizeof(h));
  *offset_out = int64_t(reinterpret_cast<uintptr_t>(ptr) - uintptr_t(base));
  return BOKT_OK;
}

int bokt_ipc_import(const void* handle, int64_t offset, void** base_out, void** ptr_out) {
  g_err[0] = 0;
  if (!handle || !base_out || !ptr_out || offset < 0) return fail(BOKT_ERR_INVALID, "bad argument");
  cudaIpcMemHandle_t h;
  memcpy(&h, handle, sizeof(h));
  void* base = nullptr;
  cudaError_t e = cudaIpcOpenMemHandle(&base, h, cudaIpcMemLazyEnablePeerAccess);
  if (e != cudaSuccess) return cuda_fail(e, "cudaIpcOpenMemHandle");
  *base_out = base;
  *ptr_out = static_cast<char*>(base) + offset;
  return BOKT_OK;
}

int bokt_ipc_close(void* base) {
  g_err[0] = 0;
  if (!base) return BOKT_OK;
  cudaError_t e = cudaIpcCloseMemHandle(base);
  if (e != cudaSuccess) return cuda_fail(e, "cudaIpcCloseMemHandle");
  return BOKT_OK;
}

int bokt_moe_topk_gate(const void* logits, int logits_dtype, int tokens, int E, int k,
                       int renormalize, int32_t* ids, float* gates, void* stream) {
  g_err[0] = 0;
  if (tokens < 0 || E <= 0 || k <= 0) return fail(BOKT_ERR_INVALID, "bad size");
  if (k > bokt::kTopkMax || k > E)
    return fail(BOKT_ERR_UNSUPPORTED, "k must be <= %d and <= E", bokt::kTopkMax);
  if (E > bokt::kGateMaxExperts)
    return fail(BOKT_ERR_UNSUPPORTED, "at most %d experts", bokt::kGateMaxExperts);
  if (tokens == 0) return BOKT_OK;
  if (!logits || !ids || !gates) return fail(BOKT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int grid = (tokens + 7) / 8;
  if (grid > 148 * 32) grid = 148 * 32;
  cudaError_t e;
  if (logits_dtype == BOKT_BF16)
    e = launch(bokt::moe_topk_gate_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, s,
               static_cast<const __nv_bfloat16*>(logits), tokens, E, k, renormalize, ids, gates);
  else if (logits_dtype == BOKT_FP16)
    e = launch(bokt::moe_topk_gate_kernel<__half>, dim3(grid), dim3(256), 0, s,
               static_cast<const __half*>(logits), tokens, E, k, renormalize, ids, gates);
  else if (logits_dtype == BOKT_FP32)
    e = launch(bokt::moe_topk_gate_kernel<float>, dim3(grid), dim3(256), 0, s,
               static_cast<const float*>(logits), tokens, E, k, renormalize, ids, gates);
  else
    return fail(BOKT_ERR_INVALID, "logits dtype %d", logits_dtype);
  if (e != cudaSuccess) return cuda_fail(e, "moe_topk_gate launch");
  return BOKT_OK;
}

int bokt_moe_combine(const void* y, int64_t y_rows, const int32_t* rows, const float* gates,
                     void* out, int tokens, int k, int N, int dtype, void* stream) {
  g_err[0] = 0;
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (tokens < 0 || k <= 0 || N < 0 || y_rows < 0) return fail(BOKT_ERR_INVALID, "bad size");
  if (tokens == 0 || N == 0) return BOKT_OK;
  if (!y || !gates || !out) return fail(BOKT_ERR_INVALID, "null pointer");
  if (N % 8 != 0 || !aligned16(y) || !aligned16(out))
    return fail(BOKT_ERR_UNSUPPORTED, "combine needs N %% 8 == 0 and 16-byte aligned rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = tokens < 148 * 64 ? tokens : 148 * 64;
  const int threads = N / 8 < 256 ? ((N / 8 + 31) / 32) * 32 : 256;
  cudaError_t e =
      dtype == BOKT_BF16
          ? launch(bokt::moe_combine_kernel<__nv_bfloat16>, dim3(grid), dim3(threads), 0, s,
                   static_cast<const __nv_bfloat16*>(y), (long long)y_rows, rows, gates,
                   static_cast<__nv_bfloat16*>(out), tokens, k, N)
          : launch(bokt::moe_combine_kernel<__half>, dim3(grid), dim3(threads), 0, s,
                   static_cast<const __half*>(y), (long long)y_rows, rows, gates,
                   static_cast<__half*>(out), tokens, k, N);
  if (e != cudaSuccess) return cuda_fail(e, "moe_combine launch");
  return BOKT_OK;
}

int bokt_selftest_bounded_wait(int64_t timeout_ns, int* gave_up, void* stream) {
  g_err[0] = 0;
  if (timeout_ns <= 0 || timeout_ns > 10000000000ll || !gave_up)
    return fail(BOKT_ERR_INVALID, "timeout must be in (0, 10 s] and gave_up non-null");
  cudaError_t e = launch(bokt::selftest_bounded_wait_kernel, dim3(1), dim3(32), 0,
                         static_cast<cudaStream_t>(stream), uint64_t(timeout_ns), gave_up);
  if (e != cudaSuccess) return cuda_fail(e, "selftest launch");
  return BOKT_OK;
}

int bokt_kernel_attrs(int kernel, int dtype, int n, int k, const bokt_params* params,
                      bokt_attrs* out) {
  g_err[0] = 0;
  if (!out) return fail(BOKT_ERR_INVALID, "null output");
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  const void* fn = nullptr;
  int dyn = 0, threads = 0, path = 0;
  if (kernel == BOKT_KERNEL_GEMM || kernel == BOKT_KERNEL_MOE_GROUPED_GEMM ||
      kernel == BOKT_KERNEL_RMSNORM_GEMM) {
    const bool grouped = kernel == BOKT_KERNEL_MOE_GROUPED_GEMM;
    const bool norm = kernel == BOKT_KERNEL_RMSNORM_GEMM;
    if ((n % 8) == 0 && (k % 8) == 0 && k > 0) {
      TcConfig cfg;
      rc = resolve_tc_config(params, grouped, grouped ? 64 : 0, dev.smem_optin, &cfg);
      if (rc) return rc;
      fn = cfg.cta_group == 2 ? tc2_kernel(dtype, cfg.bn, norm, grouped)
                              : tc_kernel(grouped, dtype, cfg.bn, false, norm);
      dyn = cfg.smem;
      threads = bokt::kGemmThreads;
      path = 0;
    } else if (norm) {
      return fail(BOKT_ERR_UNSUPPORTED, "fused RMSNorm-GEMM needs K and N multiples of 8");
    } else {
      fn = dtype == BOKT_BF16
               ? reinterpret_cast<const void*>(&bokt::gemm_tc_edge_kernel<__nv_bfloat16>)
               : reinterpret_cast<const void*>(&bokt::gemm_tc_edge_kernel<__half>);
      threads = bokt::kEdgeThreads;
      dyn = bokt::kEdgeSmemBytes;
      path = 1;
    }
  } else if (kernel == BOKT_KERNEL_RMSNORM) {
    NormConfig cfg;
    rc = resolve_norm_config(params, n, (n % 8) == 0, &cfg);
    if (rc) return rc;
    if (cfg.ring_slots < 0) {
      fn = dtype == BOKT_BF16 ? pipe_kernel<__nv_bfloat16>(cfg.vpt) : pipe_kernel<__half>(cfg.vpt);
      threads = cfg.threads;
      path = 5;
    } else if (cfg.ring_slots > 0) {
      fn = dtype == BOKT_BF16
               ? reinterpret_cast<const void*>(&bokt::rmsnorm_ring_kernel<__nv_bfloat16>)
               : reinterpret_cast<const void*>(&bokt::rmsnorm_ring_kernel<__half>);
      threads = cfg.threads + 32;
      dyn = bokt::rmsnorm_ring_smem_bytes(n, 2, cfg.ring_slots);
      path = 4;
    } else {
      fn = dtype == BOKT_BF16 ? norm_kernel<__nv_bfloat16>(cfg.vpt) : norm_kernel<__half>(cfg.vpt);
      threads = cfg.threads;
      path = cfg.vpt ? 2 : 3;
    }
  } else {
    return fail(BOKT_ERR_INVALID, "unknown kernel id %d", kernel);
  }
  cudaFuncAttributes a;
  cudaError_t e = cudaFuncGetAttributes(&a, fn);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes");
  out->shared_bytes = int(a.sharedSizeBytes) + dyn;
  out->registers = a.numRegs;
  out->local_bytes = int(a.localSizeBytes);
  out->threads = threads;
  out->max_threads = a.maxThreadsPerBlock;
  out->path = path;
  return BOKT_OK;
}

int bokt_splitk_schedule(int ntiles, int split_k, int nkb, int launched, int32_t* out,
                         int capacity) {
  g_err[0] = 0;
  if (ntiles < 0 || split_k < 1 || nkb < 1 || launched < 1 || capacity < 0 || (!out && capacity))
    return -fail(BOKT_ERR_INVALID, "bad argument");
  const int split = split_k < nkb ? split_k : nkb;
  const int workers = bokt::splitk_workers(launched, ntiles, split);
  int n = 0;
  for (int w = 0; w < launched; ++w) {
    bokt::SegmentCursor cur = bokt::segment_cursor(w, workers, ntiles, split);
    bokt::Segment sg;
    while (bokt::segment_next(cur, split, nkb, sg)) {
      int first = 0, count = 0;
      if (split > 1 && sg.kb0 == 0 && sg.kb1 < nkb)
        count = bokt::splitk_contributors(w, workers, ntiles, split, sg.tile, &first);
      if (n < capacity) {
        int32_t* r = out + 6 * static_cast<int64_t>(n);
        r[0] = w;
        r[1] = sg.tile;
        r[2] = sg.kb0;
        r[3] = sg.kb1;
        r[4] = first;
        r[5] = count;
      }
      ++n;
    }
  }
  return n;
}

int bokt_splitk_reduce_sources(int ntiles, int split_k, int nkb, int launched, int32_t* out,
                               int capacity) {
  g_err[0] = 0;
  if (ntiles < 0 || split_k < 1 || nkb < 1 || launched < 1 || capacity < 0 || (!out && capacity))
    return -fail(BOKT_ERR_INVALID, "bad argument");
  const int split = split_k < nkb ? split_k : nkb;
  if (split <= 1) return 0;
  const int workers = bokt::splitk_workers(launched, ntiles, split);
  int n = 0;
  for (int t = 0; t < ntiles; ++t) {
    int wa, wb, first_which;
    bokt::splitk_tile_workers(t, split, workers, ntiles, &wa, &wb, &first_which);
    if (wb - wa < 2) continue;
    for (int w = wa; w < wb; ++w, ++n) {
      if (n >= capacity) continue;
      int32_t* r = out + 3 * static_cast<int64_t>(n);
      r[0] = t;
      r[1] = w;
      r[2] = w == wa ? first_which : 0;
    }
  }
  return n;
}

int bokt_device_status(int* code, int* detail, int reset) {
  g_err[0] = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceSynchronize");
  int h[2] = {0, 0};
  e = cudaMemcpyFromSymbol(h, bokt::g_status, sizeof(h));
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyFromSymbol(status)");
  if (code) *code = h[0];
  if (detail) *detail = h[1];
  if (reset) {
    const int z[2] = {0, 0};
    e = cudaMemcpyToSymbol(bokt::g_status, z, sizeof(z));
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyToSymbol(status)");
  }
  return BOKT_OK;
}

}  // extern "C"

// =================================================================== allocation-free routing
// bokt_moe_route_noalloc: the routing front end for callers that cannot call
// cudaMalloc (or any allocator) at all.  The per-chunk expert table that
// bokt_moe_route keeps in a caller-provided workspace lives here in a fixed
// device array instead, which every GPU that loads this library holds until
// the process exits.  Host code never dereferences or passes the array's name
// to a kernel: in host code that name is only a host-side stand-in, so the
// device address is looked up with cudaGetSymbolAddress once per device.
namespace {

// chunks * experts int32 words, chunks = ceil(assignments / 4096).
constexpr int64_t kRouteScratchWords = 64 * 1024;  // 256 KiB

static __device__ __align__(256) int32_t g_route_scratch[kRouteScratchWords];

// Resolved device address per device, with the context it was resolved in: a
// different current context (after cudaDeviceReset, or a user-created
// context) loads its own copy of the module, so the address is looked up
// again rather than reusing one from a context that may be gone.
struct ScratchAddr {
  CUcontext ctx;
  int32_t* ptr;
};
ScratchAddr g_route_scratch_addr[kMaxDevices] = {};
std::mutex g_route_scratch_mu;
PFN_cuCtxGetCurrent_v4000 g_ctx_current = nullptr;
std::once_flag g_ctx_current_once;

// Device address of g_route_scratch in the current device's current context,
// resolved on the first call in that context (that first call must not be
// inside stream capture).
int route_scratch(int32_t** out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(BOKT_ERR_UNSUPPORTED, "device index %d", dev);
  std::call_once(g_ctx_current_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_ctx_current = reinterpret_cast<PFN_cuCtxGetCurrent_v4000>(fn);
  });
  if (!g_ctx_current) return fail(BOKT_ERR_CUDA, "cuCtxGetCurrent entry point unavailable");
  CUcontext ctx = nullptr;
  if (g_ctx_current(&ctx) != CUDA_SUCCESS) return fail(BOKT_ERR_CUDA, "cuCtxGetCurrent failed");
  std::lock_guard<std::mutex> lock(g_route_scratch_mu);
  ScratchAddr& slot = g_route_scratch_addr[dev];
  if (!ctx || !slot.ptr || slot.ctx != ctx) {
    // Also makes the device's primary context current when none is yet.
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_route_scratch);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetSymbolAddress(g_route_scratch)");
    if (g_ctx_current(&ctx) != CUDA_SUCCESS || !ctx)
      return fail(BOKT_ERR_CUDA, "no current CUDA context");
    slot.ctx = ctx;
    slot.ptr = static_cast<int32_t*>(p);
  }
  *out = slot.ptr;
  return BOKT_OK;
}

}  // namespace

extern "C" int64_t bokt_moe_route_noalloc_max_words(void) { return kRouteScratchWords; }

extern "C" int bokt_moe_route_noalloc(const int32_t* expert_ids, int A, int E, int32_t* counts,
                                      int32_t* offsets, int64_t* offsets64, int32_t* perm,
                                      int32_t* inv_perm, void* stream) {
  g_err[0] = 0;
  if (A < 0 || E <= 0) return fail(BOKT_ERR_INVALID, "need A >= 0 and E > 0");
  if (E > bokt::kRouteMaxExperts)
    return fail(BOKT_ERR_UNSUPPORTED, "at most %d experts", bokt::kRouteMaxExperts);
  if (!counts || !offsets || (A > 0 && (!expert_ids || !perm || !inv_perm)))
    return fail(BOKT_ERR_INVALID, "null pointer");
  const int64_t words = bokt_moe_route_workspace_bytes(A, E) / 4;
  if (words > kRouteScratchWords)
    return fail(BOKT_ERR_UNSUPPORTED,
                "bokt_moe_route_noalloc: ceil(A/4096) * E = %lld scratch words exceeds the fixed "
                "%lld-word device array (A=%d, E=%d); use bokt_moe_route with a workspace",
                (long long)words, (long long)kRouteScratchWords, A, E);
  int32_t* scratch = nullptr;
  int rc = route_scratch(&scratch);
  if (rc) return rc;
  // Same kernels as bokt_moe_route.  route_count overwrites every scratch word
  // the later launches read, so no clearing is needed between calls.
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launch_route(expert_ids, A, E, scratch, counts, offsets, offsets64, perm, inv_perm, s,
                      "moe_route_noalloc launch");
}

// ----------------------------------------------------------------- query/key norm + rotation
namespace {

// Blocks per SM of the persistent backward kernel (its partial rows are sized by this).
constexpr int kQkGradBlocksPerSm = 2;

bool qk_strides_vec(const bokt::QkSide& s) {
  return ((s.x_row | s.x_head | s.g_row | s.g_head | s.out_row | s.out_head) & 7) == 0 &&
         aligned16(s.x) && aligned16(s.g) && aligned16(s.out) && aligned16(s.w);
}

template <typename T, bool PAIRS, bool GRAD>
cudaError_t launch_qk_any(const bokt::QkArgs& a, int sm_count, int* blocks, cudaStream_t s) {
  const long long rows = (long long)a.tokens * max(a.side[0].heads, a.side[1].heads);
  long long grid = (rows + 3) / 4;
  if (grid > (long long)kQkGradBlocksPerSm * sm_count) grid = (long long)kQkGradBlocksPerSm * sm_count;
  *blocks = int(grid);
  return launch(bokt::qk_norm_rope_any_kernel<T, PAIRS, GRAD>, dim3(unsigned(grid)), dim3(128),
                size_t(4) * 3 * a.dim * 4, s, a);
}

template <typename T, int L, bool PAIRS, bool PART, int R, bool GRAD>
cudaError_t launch_qk_vec(bokt::QkArgs a, int sm_count, int* blocks, cudaStream_t s) {
  // As many rows behind one load of the angles as leave every SM two rounds
  // of 32 warps, up to the measured best (four loops forward, two backward).
  const long long rows = (long long)a.tokens * (a.side[0].heads + a.side[1].heads);
  a.loops = 1;
  while (R > 1 && a.loops < (GRAD ? 2 : 4) && rows / (32 / L * R * 2 * a.loops) >= 64ll * sm_count)
    a.loops *= 2;
  const int hpu = 32 / L * R * a.loops;
  const long long u0 = (long long)a.tokens * ((a.side[0].heads + hpu - 1) / hpu);
  const long long u1 = (long long)a.tokens * ((a.side[1].heads + hpu - 1) / hpu);
  if constexpr (GRAD) {
    long long grid = (u0 + u1 + bokt::kQkWarps - 1) / bokt::kQkWarps;
    if (grid > (long long)kQkGradBlocksPerSm * sm_count)
      grid = (long long)kQkGradBlocksPerSm * sm_count;
    *blocks = int(grid);
    auto* kernel = bokt::qk_norm_rope_grad_kernel<T, L, PAIRS, PART, R>;
    const int smem = bokt::qk_grad_smem_bytes<L, R>();
    if (ensure_smem(reinterpret_cast<const void*>(kernel), smem)) return cudaErrorInvalidValue;
    return launch(kernel, dim3(unsigned(grid)), dim3(bokt::kQkThreads), smem, s, a);
  } else {
    *blocks = 0;
    return launch(bokt::qk_norm_rope_kernel<T, L, PAIRS, PART, R>,
                  dim3(unsigned((u0 + u1 + bokt::kQkWarps - 1) / bokt::kQkWarps)),
                  dim3(bokt::kQkThreads), 0, s, a);
  }
}

template <typename T, bool PAIRS, bool GRAD>
cudaError_t launch_qk(const bokt::QkArgs& a, bool vec, int sm_count, int* blocks, cudaStream_t s) {
  if (!vec) return launch_qk_any<T, PAIRS, GRAD>(a, sm_count, blocks, s);
  // Few head rows: one row per lane group, so that the call spreads over the
  // SMs; many: four loads in flight per lane.
  const bool few = (long long)a.tokens * (a.side[0].heads + a.side[1].heads) < 64ll * sm_count;
#define BOKT_QK_PART(L, PART) \
  (few ? launch_qk_vec<T, L, PAIRS, PART, 1, GRAD>(a, sm_count, blocks, s) \
       : launch_qk_vec<T, L, PAIRS, PART, 4, GRAD>(a, sm_count, blocks, s))
  // PART, but for neighbours that all turn (see the kernel).
#define BOKT_QK(L) (!PAIRS || a.rot < a.dim ? BOKT_QK_PART(L, true) : BOKT_QK_PART(L, !PAIRS))
  if (a.dim <= 64) return BOKT_QK(8);
  if (a.dim <= 128) return BOKT_QK(16);
  return BOKT_QK(32);
#undef BOKT_QK
#undef BOKT_QK_PART
}

// Memory of one operand of T x H head rows, in bytes.
struct QkSpan {
  const char* p;
  int64_t row, head, width;
  int T, H;
};

QkSpan qk_span(const void* p, int64_t row, int64_t head, const bokt::QkArgs& a, int heads) {
  QkSpan s = {static_cast<const char*>(p), 2 * row, 2 * head, 2 * (int64_t)a.dim, a.tokens, heads};
  if (s.T <= 1) s.row = 0;  // a stride that nothing takes
  if (s.H <= 1) s.head = 0;
  if (s.row < 0) s.p += (s.T - 1) * s.row, s.row = -s.row;
  if (s.head < 0) s.p += (s.H - 1) * s.head, s.head = -s.head;
  return s;
}

bool qk_same(const QkSpan& a, const QkSpan& b) { return a.p == b.p && a.row == b.row && a.head == b.head; }

// Whether the two share no byte: separate ranges, or blocks that never meet
// modulo a stride they have in common (heads beside each other in every token's
// row, token rows beside each other in every head, or all strides' divisor).
// False also where none of these shows it.
bool qk_apart(const QkSpan& a, const QkSpan& b) {
  if (!a.T || !a.H || !b.T || !b.H) return true;
  using wide = __int128;
  const wide gap = (wide) reinterpret_cast<intptr_t>(b.p) - reinterpret_cast<intptr_t>(a.p);
  auto row_block = [](const QkSpan& s) { return (wide)(s.H - 1) * s.head + s.width; };
  auto head_block = [](const QkSpan& s) { return (wide)(s.T - 1) * s.row + s.width; };
  auto end = [&](const QkSpan& s) { return (wide)(s.T - 1) * s.row + row_block(s); };
  if (gap >= end(a) || -gap >= end(b)) return true;
  auto beside = [&](wide period, wide ea, wide eb) {
    if (period <= 0) return false;
    const wide at = (gap % period + period) % period;
    return at >= ea && at + eb <= period;
  };
  // A span of one token (or head) may be taken to step like the other.
  if (a.row == b.row || a.T == 1 || b.T == 1)
    if (beside(std::max(a.row, b.row), row_block(a), row_block(b))) return true;
  if (a.head == b.head || a.H == 1 || b.H == 1)
    if (beside(std::max(a.head, b.head), head_block(a), head_block(b))) return true;
  return beside(std::gcd(std::gcd(a.row, b.row), std::gcd(a.head, b.head)), a.width, b.width);
}

// Outputs are written while other rows are still read: they share no memory
// with each other or with an input, but for each side's own inputs, whole (a
// row is read and written by one warp).  dw: the weights' gradients, or null.
int qk_check_overlap(const bokt::QkArgs& a, bool grad, const float* const* dw) {
  const char* const outs[2] = {grad ? "dq" : "q_out", grad ? "dk" : "k_out"};
  const char* const ins[4] = {"q", "k", "dq_out", "dk_out"};
  QkSpan out[2], in[4];
  for (int i = 0; i < 2; ++i) {
    const bokt::QkSide& s = a.side[i];
    out[i] = qk_span(s.out, s.out_row, s.out_head, a, s.heads);
    in[i] = qk_span(s.x, s.x_row, s.x_head, a, s.heads);
    in[2 + i] = qk_span(s.g, s.g_row, s.g_head, a, grad ? s.heads : 0);
  }
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 4; ++j)
      if (!((j & 1) == i && qk_same(out[i], in[j])) && !qk_apart(out[i], in[j]))
        return fail(BOKT_ERR_OVERLAP, "%s must not overlap %s%s", outs[i], ins[j],
                    (j & 1) == i ? " (unless it is the same view)" : "");
  if (!qk_apart(out[0], out[1])) return fail(BOKT_ERR_OVERLAP, "%s must not overlap %s", outs[0], outs[1]);
  if (!dw) return BOKT_OK;
  const char* const dws[2] = {"dq_weight", "dk_weight"};
  QkSpan w[2];
  for (int i = 0; i < 2; ++i) w[i] = {reinterpret_cast<const char*>(dw[i]), 0, 0, 4 * (int64_t)a.dim, 1, 1};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if (!qk_apart(w[i], out[j])) return fail(BOKT_ERR_OVERLAP, "%s must not overlap %s", dws[i], outs[j]);
  if (!qk_apart(w[0], w[1])) return fail(BOKT_ERR_OVERLAP, "dq_weight must not overlap dk_weight");
  return BOKT_OK;
}

int qk_norm_rope_impl(bokt::QkArgs* a, const int64_t* strides, int interleaved, int dtype,
                      const float* const* dw, void* stream, int* blocks, DeviceInfo* dev) {
  const bool grad = dw != nullptr;
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (a->tokens < 0 || a->side[0].heads < 0 || a->side[1].heads < 0 || a->table_rows < 0)
    return fail(BOKT_ERR_INVALID, "negative size");
  if (a->dim < 2 || a->dim > bokt::kQkMaxDim)
    return fail(BOKT_ERR_UNSUPPORTED, "head size must be in [2, %d] (got %d)", bokt::kQkMaxDim, a->dim);
  if (a->rot < 2 || a->rot > a->dim || (a->rot & 1))
    return fail(BOKT_ERR_INVALID, "rot must be even and in [2, head size] (got %d)", a->rot);
  if (!(a->eps >= 0.f) || !(a->eps < 3.0e38f))
    return fail(BOKT_ERR_INVALID, "eps must be finite >= 0");
  // Persistent warps step past the last row by up to a grid: leave the counter room.
  if ((long long)a->tokens * ((long long)a->side[0].heads + a->side[1].heads) > 0x7fff0000LL)
    return fail(BOKT_ERR_UNSUPPORTED, "more than 2^31 - 2^16 head rows");
  const bool empty = a->tokens == 0 || a->side[0].heads + a->side[1].heads == 0;
  bool vec = a->dim % 8 == 0 && a->dim <= bokt::kQkMaxVecDim && a->rot % (interleaved ? 8 : 16) == 0 &&
             aligned16(a->cos_sin);
  int rc;
  if (!empty) {
    // A table without rows has no memory: every position is outside it.
    if (!strides || !a->positions || (!a->cos_sin && a->table_rows > 0))
      return fail(BOKT_ERR_INVALID, "null pointer");
    for (int i = 0; i < 2; ++i) {
      bokt::QkSide& s = a->side[i];
      if (s.heads && (!s.x || !s.w || !s.out || (grad && !s.g)))
        return fail(BOKT_ERR_INVALID, "null pointer");
      const int64_t* st = strides + (grad ? 6 : 4) * i;
      s.x_row = st[0], s.x_head = st[1];
      s.out_row = st[2], s.out_head = st[3];
      if (grad) s.g_row = st[4], s.g_head = st[5];
      vec = vec && (s.heads == 0 || qk_strides_vec(s));
    }
  }
  if ((rc = qk_check_overlap(*a, grad, dw))) return rc;
  *blocks = 0;
  if ((rc = device_info(dev))) return rc;
  if (empty) return BOKT_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define BOKT_QK(T, P) \
  (grad ? launch_qk<T, P, true>(*a, vec, dev->sm_count, blocks, s) \
        : launch_qk<T, P, false>(*a, vec, dev->sm_count, blocks, s))
  if (dtype == BOKT_BF16)
    e = interleaved ? BOKT_QK(__nv_bfloat16, true) : BOKT_QK(__nv_bfloat16, false);
  else
    e = interleaved ? BOKT_QK(__half, true) : BOKT_QK(__half, false);
#undef BOKT_QK
  if (e != cudaSuccess) return cuda_fail(e, "qk_norm_rope launch");
  return BOKT_OK;
}

}  // namespace

extern "C" {

int bokt_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight,
                      const void* positions, int positions_i64, const float* cos_sin,
                      int table_rows, void* q_out, void* k_out, int tokens, int heads,
                      int kv_heads, int dim, int rot, const int64_t* strides, int interleaved,
                      float eps, int dtype, void* stream) {
  g_err[0] = 0;
  bokt::QkArgs a = {};
  a.side[0].x = q, a.side[0].w = q_weight, a.side[0].out = q_out, a.side[0].heads = heads;
  a.side[1].x = k, a.side[1].w = k_weight, a.side[1].out = k_out, a.side[1].heads = kv_heads;
  a.positions = positions, a.positions_i64 = positions_i64;
  a.cos_sin = cos_sin, a.table_rows = table_rows;
  a.tokens = tokens, a.dim = dim, a.rot = rot, a.eps = eps;
  int blocks;
  DeviceInfo dev;
  return qk_norm_rope_impl(&a, strides, interleaved, dtype, nullptr, stream, &blocks, &dev);
}

int64_t bokt_qk_norm_rope_workspace_bytes(int dim) {
  g_err[0] = 0;
  DeviceInfo dev;
  if (device_info(&dev)) return -1;
  return (int64_t)kQkGradBlocksPerSm * dev.sm_count * 2 * dim * 4;
}

int bokt_qk_norm_rope_backward(const void* dq_out, const void* dk_out, const void* q,
                               const void* k, const void* q_weight, const void* k_weight,
                               const void* positions, int positions_i64, const float* cos_sin,
                               int table_rows, void* dq, void* dk, float* dq_weight,
                               float* dk_weight, int tokens, int heads, int kv_heads, int dim,
                               int rot, const int64_t* strides, int interleaved, float eps,
                               int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  bokt::QkArgs a = {};
  a.side[0].x = q, a.side[0].g = dq_out, a.side[0].w = q_weight, a.side[0].out = dq;
  a.side[1].x = k, a.side[1].g = dk_out, a.side[1].w = k_weight, a.side[1].out = dk;
  a.side[0].heads = heads, a.side[1].heads = kv_heads;
  a.positions = positions, a.positions_i64 = positions_i64;
  a.cos_sin = cos_sin, a.table_rows = table_rows;
  a.tokens = tokens, a.dim = dim, a.rot = rot, a.eps = eps;
  a.partials = static_cast<float*>(workspace);
  if (!dq_weight || !dk_weight || !workspace) return fail(BOKT_ERR_INVALID, "null pointer");
  DeviceInfo dev;
  int blocks;
  const float* const dw[2] = {dq_weight, dk_weight};
  int rc = device_info(&dev);
  if (rc == BOKT_OK && workspace_bytes < (int64_t)kQkGradBlocksPerSm * dev.sm_count * 2 * dim * 4)
    return fail(BOKT_ERR_INVALID, "workspace too small (%lld bytes)", (long long)workspace_bytes);
  // Without a device the sizes and the overlaps are still looked at first.
  rc = qk_norm_rope_impl(&a, strides, interleaved, dtype, dw, stream, &blocks, &dev);
  if (rc) return rc;
  // No rows: the weight gradients are zero.
  cudaError_t e = launch(bokt::qk_norm_rope_dweight_kernel, dim3(unsigned((dim + 31) / 32), 2),
                         dim3(32, 32), 0, static_cast<cudaStream_t>(stream), a.partials, blocks,
                         dim, dq_weight, dk_weight);
  if (e != cudaSuccess) return cuda_fail(e, "qk_norm_rope_dweight launch");
  return BOKT_OK;
}

int bokt_rope_table(float* cos_sin, int rows, int rot, double base, void* stream) {
  g_err[0] = 0;
  if (rows < 0 || rot < 2 || (rot & 1)) return fail(BOKT_ERR_INVALID, "bad size");
  if (!(base > 0.0) || !(base < 1e300)) return fail(BOKT_ERR_INVALID, "base must be finite > 0");
  if (rows == 0) return BOKT_OK;
  if (!cos_sin) return fail(BOKT_ERR_INVALID, "null pointer");
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  const long long n = (long long)rows * (rot / 2);
  long long blocks = (n + 255) / 256;
  if (blocks > 8LL * dev.sm_count) blocks = 8LL * dev.sm_count;
  cudaError_t e = launch(bokt::rope_table_kernel, dim3(unsigned(blocks)), dim3(256), 0,
                         static_cast<cudaStream_t>(stream), cos_sin, rows, rot, base);
  if (e != cudaSuccess) return cuda_fail(e, "rope_table launch");
  return BOKT_OK;
}

}  // extern "C"

// ----------------------------------------------------------------- MoE layer for a few tokens
namespace {

cudaError_t launch_cluster(const void* fn, int grid, int threads, int smem, int cluster,
                           cudaStream_t s, void** kargs) {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t lc = launch_config(dim3(unsigned(grid)), dim3(unsigned(threads)), smem, s, attr);
  attr[lc.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[lc.numAttrs].val.clusterDim.x = unsigned(cluster);
  attr[lc.numAttrs].val.clusterDim.y = 1;
  attr[lc.numAttrs].val.clusterDim.z = 1;
  lc.numAttrs += 1;
  return cudaLaunchKernelExC(&lc, fn, kargs);
}


// Byte offsets of the workspace's parts, each 256-byte aligned.
struct MoeDecodeLayout {
  int shares;
  int64_t act_e, act_off, row_token, row_of, act_of, gates, h, y, part, total;
};

int moe_decode_layout(int tokens, int E, int K, int I, int topk, const DeviceInfo& dev,
                      MoeDecodeLayout* l) {
  if (tokens < 0 || E <= 0 || K <= 0 || I <= 0 || topk <= 0)
    return fail(BOKT_ERR_INVALID, "need tokens >= 0 and positive sizes");
  if (topk > E) return fail(BOKT_ERR_INVALID, "topk %d exceeds the %d experts", topk, E);
  if (tokens > bokt::kMdMaxTokens || topk > bokt::kMdMaxTopk || E > bokt::kMdMaxExperts)
    return fail(BOKT_ERR_UNSUPPORTED,
                "at most %d tokens, top-%d and %d experts (got %d, %d, %d); route more tokens "
                "through bokt_moe_route and bokt_moe_grouped_gemm", bokt::kMdMaxTokens,
                bokt::kMdMaxTopk, bokt::kMdMaxExperts, tokens, topk, E);
  if (K % 8 != 0 || I % 8 != 0 || K > 65536 || I > 65536)
    return fail(BOKT_ERR_UNSUPPORTED, "K and I must be multiples of 8 up to 65536 (got %d, %d)", K, I);
  const int64_t g = dev.sm_count;
  l->shares = dev.sm_count;
  const int64_t A = (int64_t)tokens * topk, em = E < A ? E : A;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  take((bokt::kMdCount1 + 4 * g) * 4);
  l->act_e = take(em * 4);
  l->act_off = take((em + 1) * 4);
  l->row_token = take(A * 4);
  l->row_of = take(A * 4);
  l->act_of = take(A * 4);
  l->gates = take(A * 4);
  l->h = take(A * I * 2);
  l->y = take(A * K * 4);
  l->part = take(2 * g * tokens * 256 * 4);
  l->total = at;
  return BOKT_OK;
}

const void* moe_decode_gate_ptr(int E) {
  if (E <= 32) return reinterpret_cast<const void*>(&bokt::moe_decode_gate_kernel<1>);
  if (E <= 128) return reinterpret_cast<const void*>(&bokt::moe_decode_gate_kernel<4>);
  if (E <= 256) return reinterpret_cast<const void*>(&bokt::moe_decode_gate_kernel<8>);
  return reinterpret_cast<const void*>(&bokt::moe_decode_gate_kernel<32>);
}

template <typename T>
const void* moe_few_ptr(bool down, int E) {
  if (down)
    return E <= 128 ? reinterpret_cast<const void*>(&bokt::moe_few_down_kernel<T, 4>)
                    : reinterpret_cast<const void*>(&bokt::moe_few_down_kernel<T, 32>);
  return E <= 128 ? reinterpret_cast<const void*>(&bokt::moe_few_up_kernel<T, 4>)
                  : reinterpret_cast<const void*>(&bokt::moe_few_up_kernel<T, 32>);
}

// Cluster sizes of the two kernels for a handful of tokens, or false: the
// persistent kernel's case.
bool moe_few_plan(int tokens, int E, int K, int I, int topk, const DeviceInfo& dev, int* up, int* down) {
  if (tokens > bokt::kFewTokens || tokens * topk > bokt::kFewRows) return false;
  const long long active = E < tokens * topk ? E : tokens * topk;  // at most
  const long long tiles1 = active * ((I + 127) / 128), tiles2 = (K + 127) / 128;
  const int ksteps = (K + 63) / 64, steps2 = (I + 127) / 128;
  *up = *down = 1;
  while (*up < 8 && tiles1 * *up * 2 <= dev.sm_count && ksteps >= *up * 2) *up *= 2;
  while (*down < 8 && tiles2 * *down * 2 <= dev.sm_count && topk * steps2 >= *down * 2) *down *= 2;
  // The second kernel has one cluster per 128 columns of out: with few of them
  // and long runs the persistent kernel's even shares are faster (16 tokens of
  // 64 experts x [1024, 2 x 1024], 64 steps a CTA: 58 us, here 74).
  if (tiles2 * *down * 2 < dev.sm_count && active * steps2 > 32 * *down) return false;
  // A CTA of the second kernel keeps an accumulator for every expert of its run.
  return (active + *down - 1) / *down + 1 <= bokt::kFewExperts;
}

}  // namespace

extern "C" {

int64_t bokt_moe_decode_workspace_bytes(int tokens, int E, int K, int I, int topk) {
  g_err[0] = 0;
  DeviceInfo dev;
  MoeDecodeLayout l;
  if (device_info(&dev) || moe_decode_layout(tokens, E, K, I, topk, dev, &l)) return -1;
  return l.total;
}

int bokt_moe_decode(const void* x, const void* logits, int logits_dtype, const void* w_gate_up,
                    const void* w_down, void* out, int tokens, int E, int K, int I, int topk,
                    int renormalize, int dtype, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  g_err[0] = 0;
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  if (logits_dtype != BOKT_FP16 && logits_dtype != BOKT_BF16 && logits_dtype != BOKT_FP32)
    return fail(BOKT_ERR_INVALID, "logits dtype %d", logits_dtype);
  DeviceInfo dev = {};
  MoeDecodeLayout l;
  int rc = moe_decode_layout(tokens, E, K, I, topk, dev, &l);  // sizes, before any device call
  if (rc) return rc;
  if (tokens == 0) return BOKT_OK;
  if (!x || !logits || !w_gate_up || !w_down || !out || !workspace)
    return fail(BOKT_ERR_INVALID, "null pointer");
  if (!aligned16(x) || !aligned16(w_gate_up) || !aligned16(w_down) || !aligned16(out))
    return fail(BOKT_ERR_UNSUPPORTED, "x, weights and out must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return fail(BOKT_ERR_INVALID, "workspace must be 256-byte aligned");
  rc = device_info(&dev);
  if (rc) return rc;
  rc = moe_decode_layout(tokens, E, K, I, topk, dev, &l);
  if (rc) return rc;
  if (workspace_bytes < l.total)
    return fail(BOKT_ERR_INVALID, "workspace too small: %lld bytes, need %lld",
                (long long)workspace_bytes, (long long)l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int A = tokens * topk;
  bokt::MoeDecodeArgs a = {};
  a.tokens = tokens, a.experts = E, a.k = K, a.inner = I, a.topk = topk;
  a.nt = (tokens + 15) & ~15;
  a.shares = l.shares;
  a.idesc = bokt::make_idesc_f16_swapped(uint32_t(dtype), 0);
  a.header = reinterpret_cast<uint32_t*>(ws);
  a.act_e = reinterpret_cast<int*>(ws + l.act_e);
  a.act_off = reinterpret_cast<int*>(ws + l.act_off);
  a.row_token = reinterpret_cast<int*>(ws + l.row_token);
  a.row_of = reinterpret_cast<int*>(ws + l.row_of);
  a.act_of = reinterpret_cast<int*>(ws + l.act_of);
  a.gates = reinterpret_cast<float*>(ws + l.gates);
  a.h = ws + l.h;
  a.y = reinterpret_cast<float*>(ws + l.y);
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.out = out;
  const int emax = E < A ? E : A;
  a.stages = bokt::kMdMaxStages;
  while (a.stages > 2 && bokt::moe_decode_smem_bytes(a.nt, a.stages, emax, A) > dev.smem_optin)
    --a.stages;
  int smem = bokt::moe_decode_smem_bytes(a.nt, a.stages, emax, A);
  if (smem > dev.smem_optin) return fail(BOKT_ERR_UNSUPPORTED, "needs %d bytes of shared memory", smem);
  // One CTA per SM (its TMEM may be all 512 columns).
  if (smem < dev.smem_optin / 2 + 1024) smem = dev.smem_optin / 2 + 1024;

  const bool fp16 = dtype == BOKT_FP16;
  CUtensorMap mg, md, mx, mh;
  {
    const uint64_t d[3] = {uint64_t(2) * I, uint64_t(K), uint64_t(E)};
    const uint64_t st[2] = {uint64_t(I) * 4, uint64_t(I) * 4 * K};
    const uint32_t b[3] = {64, 64, 1};
    if ((rc = encode_map(&mg, w_gate_up, 3, d, st, b, fp16))) return rc;
  }
  {
    const uint64_t d[3] = {uint64_t(K), uint64_t(I), uint64_t(E)};
    const uint64_t st[2] = {uint64_t(K) * 2, uint64_t(K) * 2 * I};
    const uint32_t b[3] = {64, 64, 1};
    if ((rc = encode_map(&md, w_down, 3, d, st, b, fp16))) return rc;
  }
  {
    const uint64_t d[2] = {uint64_t(K), uint64_t(tokens)};
    const uint64_t st[1] = {uint64_t(K) * 2};
    const uint32_t b[2] = {64, uint32_t(a.nt)};
    if ((rc = encode_map(&mx, x, 2, d, st, b, fp16))) return rc;
  }
  {
    const uint64_t d[2] = {uint64_t(I), uint64_t(A)};
    const uint64_t st[1] = {uint64_t(I) * 2};
    const uint32_t b[2] = {64, 16};
    if ((rc = encode_map(&mh, a.h, 2, d, st, b, fp16))) return rc;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int up = 1, down = 1;
  if (moe_few_plan(tokens, E, K, I, topk, dev, &up, &down)) {
    bokt::MoeFewArgs f = {};
    f.logits = logits, f.logits_dtype = logits_dtype, f.renormalize = renormalize ? 1 : 0;
    f.tokens = tokens, f.experts = E, f.k = K, f.inner = I, f.topk = topk;
    f.idesc = bokt::make_idesc_f16_swapped(uint32_t(dtype), 16);
    f.h = a.h, f.out = out;
    const long long active = E < A ? E : A;
    for (int i = 0; i < 2; ++i) {
      const void* fn = fp16 ? moe_few_ptr<__half>(i, E) : moe_few_ptr<__nv_bfloat16>(i, E);
      const int smem_few = bokt::moe_few_smem_bytes(i ? bokt::kFewDownStage : bokt::kFewUpStage);
      if ((rc = ensure_smem(fn, smem_few)) || (rc = ensure_carveout(fn))) return rc;
      f.cluster = i ? down : up;
      const long long grid = f.cluster * (i ? (K + 127) / 128 : active * ((I + 127) / 128));
      void* up_args[] = {&mg, &mx, &f};
      void* down_args[] = {&md, &mh, &f};
      cudaError_t e = launch_cluster(fn, int(grid), bokt::kFewThreads, smem_few, f.cluster, s,
                                     i ? down_args : up_args);
      if (e != cudaSuccess) return cuda_fail(e, "moe_few launch");
    }
    return BOKT_OK;
  }
  {
    const void* fn = moe_decode_gate_ptr(E);
    // At least eight tokens to a CTA, at most its sixteen warps.
    const unsigned ctas = unsigned(tokens >= 8 * bokt::kMdGateCtas ? bokt::kMdGateCtas : (tokens + 7) / 8);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t lc = launch_config(dim3(ctas), dim3(bokt::kMdGateThreads), 0, s, attr);
    attr[lc.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[lc.numAttrs].val.clusterDim.x = ctas;
    attr[lc.numAttrs].val.clusterDim.y = 1;
    attr[lc.numAttrs].val.clusterDim.z = 1;
    lc.numAttrs += 1;
    if ((rc = ensure_carveout(fn))) return rc;
    int renorm = renormalize ? 1 : 0;
    void* kargs[] = {&logits, &logits_dtype, &renorm, &a};
    cudaError_t e = cudaLaunchKernelExC(&lc, fn, kargs);
    if (e != cudaSuccess) return cuda_fail(e, "moe_decode_gate launch");
  }
  const void* fn = dtype == BOKT_BF16
                       ? reinterpret_cast<const void*>(&bokt::moe_decode_kernel<__nv_bfloat16>)
                       : reinterpret_cast<const void*>(&bokt::moe_decode_kernel<__half>);
  if ((rc = ensure_smem(fn, smem))) return rc;
  void* kargs[] = {&mg, &md, &mx, &mh, &a};
  cudaError_t e = launch_ptr(fn, dim3(unsigned(a.shares)), dim3(bokt::kMdThreads), smem, s, kargs);
  if (e != cudaSuccess) return cuda_fail(e, "moe_decode launch");
  return BOKT_OK;
}

}  // extern "C"

// ----------------------------------------------------------------- projection with adapters
namespace {

// Rows up to which W is always streamed, beside the shrink of few rows.
constexpr int kLoraFewRows = 256;
// Rows up to which W is streamed while the tiles are one wave.
constexpr int kLoraStreamRows = 1024;
// Sizes whose tile arithmetic stays in 32 bits.
constexpr int kLoraMaxSize = 1 << 30;
// Shared memory left beside the W stream: a shrink CTA of rank 16 (9 KB of
// partials, 7 KB of lists, 1 KB of the system's).  Rank 32 takes 26 KB and rank 64
// or more 44 KB, which only what the stream's whole stages leave over may hold:
// beside tiles of 32 rows neither, of 64 and 128 rows rank 32, of the others both.
// Where they do not fit, the stream's CTA starts when the shrink's leaves its SM.
constexpr int kLoraShrinkSmem = 20 * 1024;

struct LoraPlan {
  bool stream, shrink_tc;
  int tile_rows, tiles, smax, gmax, cluster, stages;
  int shrink_cluster, walkers;
  int64_t count, list, h, total;
};

// Clusters of `cluster` stream-kernel CTAs (one per SM) that the current device
// holds at once: a cluster keeps to one GPC, so fewer than sm_count / cluster.
int lora_cluster_room(const DeviceInfo& dev, int cluster) {
  if (dev.sm_count == 0) return 0;
  static int room[kMaxDevices][4];
  static std::mutex mu;
  int d = 0;
  cudaGetDevice(&d);
  const int at = cluster == 2 ? 0 : cluster == 4 ? 1 : 2;
  std::lock_guard<std::mutex> lock(mu);
  if (room[d][at] == 0) {
    const void* fn = reinterpret_cast<const void*>(&bokt::lora_stream_kernel<__nv_bfloat16>);
    if (ensure_smem(fn, dev.smem_optin)) return 0;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(unsigned(dev.sm_count / cluster * cluster));
    lc.blockDim = dim3(bokt::kLoraThreads);
    lc.dynamicSmemBytes = dev.smem_optin;
    lc.attrs = attr;
    lc.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &lc) != cudaSuccess) n = 0;
    room[d][at] = n > 0 ? n : -1;
  }
  return room[d][at];
}

int lora_plan(int M, int N, int K, int slots, int rank, const DeviceInfo& dev, LoraPlan* p) {
  if (M < 0 || N <= 0 || K <= 0 || slots <= 0)
    return fail(BOKT_ERR_INVALID, "need M >= 0 and positive N, K and slots");
  if (rank != 16 && rank != 32 && rank != 64 && rank != 128)
    return fail(BOKT_ERR_INVALID, "padded rank must be 16, 32, 64 or 128 (got %d)", rank);
  if (slots > bokt::kLoraMaxSlots)
    return fail(BOKT_ERR_UNSUPPORTED, "at most %d slots (got %d)", bokt::kLoraMaxSlots, slots);
  if (K % 8 != 0 || N % 8 != 0)
    return fail(BOKT_ERR_UNSUPPORTED, "K and N must be multiples of 8 (got %d, %d)", K, N);
  if (M > kLoraMaxSize || N > kLoraMaxSize || K > kLoraMaxSize)
    return fail(BOKT_ERR_UNSUPPORTED, "M, N and K must be at most 2^30 (got %d, %d, %d)", M, N, K);
  *p = {};
  // Few rows stream W; so do up to 1024 while their 128 x 128 tiles are one wave
  // (K = 4096, streamed and on pair tiles: 512 x 4096 22 and 26 us, 768 x 2048 20.5
  // and 26, 1024 x 1024 21 and 26; 1024 x 2048 equal; 1000 -> 2056 at 1024 rows
  // 20.7 and 19.0).  Two waves lose (768 x 4096: 39 and 27), as do 2048 rows of
  // 1024 columns (28 and 26).  The shrink of many rows is faster from 257 on with
  // a few adapters a row tile (512 rows of 9 of rank 32: 27 and 34 us), and slower
  // up to 700 rows with many (512 rows of 16 of rank 64: 59 and 41).
  const long long small_tiles = (long long)((M + 127) / 128) * ((N + 127) / 128);
  p->stream = M <= kLoraFewRows || (M <= kLoraStreamRows && small_tiles <= dev.sm_count);
  p->shrink_tc = M > kLoraFewRows;
  if (p->stream) {
    const int chunks = (M + 127) / 128;
    p->tiles = chunks;
    // Split K over a cluster while that fills SMs (all clusters resident at
    // once) and leaves each CTA a k-step.
    const long long ctas = (long long)chunks * ((N + 127) / 128);
    const int ksteps = (K + 127) / 128;
    p->cluster = 1;
    while (p->cluster < 8 && ctas <= lora_cluster_room(dev, p->cluster * 2) &&
           ksteps >= p->cluster * 2)
      p->cluster *= 2;
    // Each CTA of a cluster finishes its own quads of tokens.
    const int unit = 4 * p->cluster > 16 ? 4 * p->cluster : 16;
    p->tile_rows = chunks ? ((M + chunks - 1) / chunks + unit - 1) / unit * unit : 16;
    // Leave room beside the shrink kernel's CTAs, so that the W stream starts
    // while they run.
    p->stages = 8;
    while (p->stages > 2 &&
           bokt::lora_stream_smem_bytes(p->tile_rows, p->stages) > dev.smem_optin - kLoraShrinkSmem)
      --p->stages;
  } else {
    p->tile_rows = bokt::kLoraPairRows;
    p->tiles = (M + bokt::kLoraPairRows - 1) / bokt::kLoraPairRows;
    p->cluster = 2;
    p->stages = 6;
  }
  p->smax = slots < p->tile_rows ? slots : p->tile_rows;
  if (M < p->smax && M > 0) p->smax = M;
  // The shrink of few tokens splits K as far as there are SMs.
  p->shrink_cluster = 8;
  while (p->shrink_cluster > 1 && ((long long)p->tiles * p->smax * p->shrink_cluster > dev.sm_count ||
                                   K < p->shrink_cluster * 256))
    p->shrink_cluster /= 2;
  const long long want = dev.sm_count / ((long long)p->shrink_cluster * (p->tiles ? p->tiles : 1));
  p->walkers = int(want < 1 ? 1 : (want < p->smax ? want : p->smax));
  p->gmax = (p->smax * rank + 63) / 64;
  const int64_t entries = (int64_t)p->tiles * p->smax, groups = (int64_t)p->tiles * p->gmax;
  if (groups * p->tile_rows > 0x7fffffffLL)
    return fail(BOKT_ERR_UNSUPPORTED, "too many rows and adapters (M=%d, slots=%d)", M, slots);
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  p->count = 0;
  p->list = up((int64_t)p->tiles * 4);
  p->h = p->list + up(entries * 4);
  p->total = p->h + up(groups * p->tile_rows * 64 * 2);
  if (p->total < 256) p->total = 256;
  return BOKT_OK;
}

template <typename T>
const void* lora_shrink_ptr(int rank, int* smem) {
  if (rank == 16) {
    *smem = bokt::lora_shrink_smem_bytes<2>();
    return reinterpret_cast<const void*>(&bokt::lora_shrink_kernel<T, 2>);
  }
  if (rank == 32) {
    *smem = bokt::lora_shrink_smem_bytes<4>();
    return reinterpret_cast<const void*>(&bokt::lora_shrink_kernel<T, 4>);
  }
  *smem = bokt::lora_shrink_smem_bytes<8>();
  return reinterpret_cast<const void*>(&bokt::lora_shrink_kernel<T, 8>);
}

}  // namespace

extern "C" {

int64_t bokt_lora_gemm_workspace_bytes(int M, int N, int K, int slots, int rank) {
  g_err[0] = 0;
  DeviceInfo dev;
  LoraPlan p;
  if (device_info(&dev) || lora_plan(M, N, K, slots, rank, dev, &p)) return -1;
  return p.total;
}

int bokt_lora_gemm(const void* x, const void* W, const void* lora_a, const void* lora_b,
                   const float* scales, const int32_t* ranks, const int32_t* ids, void* out, int M,
                   int N, int K, int slots, int rank, int dtype, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (dtype != BOKT_FP16 && dtype != BOKT_BF16) return fail(BOKT_ERR_INVALID, "dtype %d", dtype);
  DeviceInfo dev = {};
  LoraPlan p;
  int rc = lora_plan(M, N, K, slots, rank, dev, &p);  // sizes, before any device call
  if (rc) return rc;
  if (M == 0) return BOKT_OK;
  if (!x || !W || !lora_a || !lora_b || !scales || !ranks || !ids || !out || !workspace)
    return fail(BOKT_ERR_INVALID, "null pointer");
  if (!aligned16(x) || !aligned16(W) || !aligned16(lora_a) || !aligned16(lora_b) || !aligned16(out))
    return fail(BOKT_ERR_UNSUPPORTED, "x, W, the adapters and out must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return fail(BOKT_ERR_INVALID, "workspace must be 256-byte aligned");
  rc = device_info(&dev);
  if (rc) return rc;
  rc = lora_plan(M, N, K, slots, rank, dev, &p);
  if (rc) return rc;
  if (workspace_bytes < p.total)
    return fail(BOKT_ERR_INVALID, "workspace too small: %lld bytes, need %lld",
                (long long)workspace_bytes, (long long)p.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  bokt::LoraArgs a = {};
  a.M = M, a.N = N, a.K = K, a.slots = slots, a.rank = rank;
  a.tile_rows = p.tile_rows, a.smax = p.smax, a.gmax = p.gmax;
  a.ids = ids, a.ranks = ranks, a.scales = scales;
  a.count = reinterpret_cast<int32_t*>(ws + p.count);
  a.list = reinterpret_cast<int32_t*>(ws + p.list);
  a.h = ws + p.h;
  a.out = out;
  a.chunks = p.tiles;
  const bool fp16 = dtype == BOKT_FP16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  CUtensorMap mx, mw, mh, mb;
  const uint32_t rs = uint32_t(rank < 64 ? rank : 64);
  {
    const uint64_t d[2] = {uint64_t(K), uint64_t(M)};
    const uint64_t st[1] = {uint64_t(K) * 2};
    const uint32_t b[2] = {64, p.stream ? uint32_t(p.tile_rows) : 128u};
    if ((rc = encode_map(&mx, x, 2, d, st, b, fp16))) return rc;
  }
  {
    const uint64_t d[2] = {uint64_t(N), uint64_t(K)};
    const uint64_t st[1] = {uint64_t(N) * 2};
    const uint32_t b[2] = {64, 64};
    if ((rc = encode_map(&mw, W, 2, d, st, b, fp16))) return rc;
  }
  {
    const uint64_t d[2] = {64, uint64_t(p.tiles) * p.gmax * p.tile_rows};
    const uint64_t st[1] = {128};
    const uint32_t b[2] = {64, p.stream ? uint32_t(p.tile_rows) : 128u};
    if ((rc = encode_map(&mh, a.h, 2, d, st, b, fp16))) return rc;
  }
  {
    const uint64_t d[3] = {uint64_t(N), uint64_t(rank), uint64_t(slots)};
    const uint64_t st[2] = {uint64_t(N) * 2, uint64_t(N) * 2 * rank};
    const uint32_t b[3] = {64, rs, 1};
    if ((rc = encode_map(&mb, lora_b, 3, d, st, b, fp16))) return rc;
  }
  cudaError_t e;
  if (!p.shrink_tc) {
    int smem = 0;
    const void* fn = fp16 ? lora_shrink_ptr<__half>(rank, &smem) : lora_shrink_ptr<__nv_bfloat16>(rank, &smem);
    if ((rc = ensure_smem(fn, smem)) || (rc = ensure_carveout(fn))) return rc;
    a.cluster = p.shrink_cluster;
    a.walkers = p.walkers;
    void* kargs[] = {&x, &lora_a, &a};
    e = launch_cluster(fn, p.tiles * p.walkers * a.cluster, bokt::kLoraThreads, smem, a.cluster, s, kargs);
  } else {
    CUtensorMap ma;
    const uint64_t d[2] = {uint64_t(K), uint64_t(slots) * rank};
    const uint64_t st[1] = {uint64_t(K) * 2};
    const uint32_t b[2] = {64, rs};
    if ((rc = encode_map(&ma, lora_a, 2, d, st, b, fp16))) return rc;
    a.idesc = bokt::make_idesc_f16_kk(uint32_t(dtype), 0);
    a.stages = 5;
    while (a.stages > 2 && bokt::lora_shrink_tc_smem_bytes(a.stages, rank) + 8192 > dev.smem_optin) --a.stages;
    const int smem = bokt::lora_shrink_tc_smem_bytes(a.stages, rank);
    const void* fn = fp16 ? reinterpret_cast<const void*>(&bokt::lora_shrink_tc_kernel<__half>)
                          : reinterpret_cast<const void*>(&bokt::lora_shrink_tc_kernel<__nv_bfloat16>);
    if ((rc = ensure_smem(fn, smem))) return rc;
    a.shrink_rows = p.tile_rows < bokt::kLoraShrinkRows ? p.tile_rows : bokt::kLoraShrinkRows;
    const int clusters = (M + a.shrink_rows - 1) / a.shrink_rows;
    void* kargs[] = {&mx, &ma, &a};
    e = launch_cluster(fn, clusters * bokt::kLoraShrinkSplit, bokt::kLoraThreads, smem,
                       bokt::kLoraShrinkSplit, s, kargs);
  }
  if (e != cudaSuccess) return cuda_fail(e, "lora_shrink launch");
  a.cluster = p.cluster;
  a.stages = p.stages;
  if (p.stream) {
    a.idesc = bokt::make_idesc_f16_swapped(uint32_t(dtype), uint32_t(p.tile_rows));
    const void* fn = fp16 ? reinterpret_cast<const void*>(&bokt::lora_stream_kernel<__half>)
                          : reinterpret_cast<const void*>(&bokt::lora_stream_kernel<__nv_bfloat16>);
    int smem = bokt::lora_stream_smem_bytes(p.tile_rows, p.stages);
    if (smem < dev.smem_optin / 2 + 1024) smem = dev.smem_optin / 2 + 1024;  // one CTA per SM
    if ((rc = ensure_smem(fn, smem))) return rc;
    const long long grid = (long long)p.tiles * ((N + 127) / 128) * p.cluster;
    if (grid > 0x7fffffffLL) return fail(BOKT_ERR_UNSUPPORTED, "too many tiles");
    void* kargs[] = {&mw, &mx, &mb, &mh, &a};
    e = launch_cluster(fn, int(grid), bokt::kLoraThreads, smem, p.cluster, s, kargs);
  } else {
    a.idesc = bokt::make_idesc_f16(uint32_t(dtype), 256, 256);
    a.group_m = 8;
    const void* fn = fp16 ? reinterpret_cast<const void*>(&bokt::lora_tc2_kernel<__half>)
                          : reinterpret_cast<const void*>(&bokt::lora_tc2_kernel<__nv_bfloat16>);
    const int smem = bokt::lora_tc2_smem_bytes(p.stages);
    if (smem > dev.smem_optin) return fail(BOKT_ERR_UNSUPPORTED, "needs %d bytes of shared memory", smem);
    if ((rc = ensure_smem(fn, smem))) return rc;
    const long long tiles = (long long)p.tiles * ((N + 255) / 256);
    if (tiles > 0x7fffffffLL) return fail(BOKT_ERR_UNSUPPORTED, "too many tiles");
    const int pairs = int(tiles < dev.sm_count / 2 ? tiles : dev.sm_count / 2);
    void* kargs[] = {&mx, &mw, &mh, &mb, &a};
    e = launch_cluster(fn, 2 * pairs, bokt::kGemmThreads, smem, 2, s, kargs);
  }
  if (e != cudaSuccess) return cuda_fail(e, "lora product launch");
  return BOKT_OK;
}

}  // extern "C"
