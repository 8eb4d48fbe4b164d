// Parts of the int8 matrix product: parameters, tensor-core and mbarrier wrappers, the epilogue.
#pragma once

#include <cuda.h>  // CUtensorMap (types only: the encoder is looked up at run time)
#include <cuda_bf16.h>

#include <mutex>

#include "mgv_common.cuh"

namespace mgv {

struct GemmI8Params {
  alignas(64) CUtensorMap w_map;  // weights: boxes of 128 bytes (K) x 128 rows, 128-byte swizzle
  alignas(64) CUtensorMap x_map;  // activations: boxes of 128 bytes x the rows one block copies
  const float *x_scale;
  const void *w_scale, *bias;
  void *out;
  int64_t ldd;
  int *err;        // device error word of bounded waits
  int M, N, K;
  int scale_dtype;
  int wide;        // two neighbouring features can be stored as one aligned word
  int bt;          // activation rows of a tile
  int stages;      // ring slots
  int split;       // blocks of a cluster that share a tile's K range
  int n_tiles, m_tiles;
  uint32_t idesc;  // instruction descriptor of the matrix instruction
  uint32_t tmem_cols;
};

constexpr int kGemmRows = 128;             // weight rows (output features) a block owns of a tile
constexpr int kGemmK = 128;                // K of a ring slot: one 128-byte swizzle row
constexpr int kGemmABytes = kGemmRows * kGemmK;
constexpr int kGemmThreads = 192;          // producer warp, matrix warp, four epilogue warps
constexpr int kGemmMaxStages = 16;
constexpr int kGemmTimeout = 0x100;        // bit of the device error word

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGated = 3 };

#if defined(__CUDACC__)

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 q, [%1], %2;\n\tselp.b32 %0, 1, 0, q;\n\t}"
               : "=r"(ok)
               : "r"(bar), "r"(parity)
               : "memory");
  return ok;
}
// Waits for the phase of the given parity, for at most about a second; false (and the device error
// word set) when it gave up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int *err) {
  for (int i = 0; i < 1024; ++i)
    if (bar_try(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  do {
    for (int i = 0; i < 256; ++i)
      if (bar_try(bar, parity)) return true;
  } while (global_timer_ns() - t0 < 1000000000ull);
  atomicOr(err, kGemmTimeout);
  return false;
}

// One box of a tensor map into shared memory of this block; bytes are counted on bar.
__device__ __forceinline__ void box_load(uint32_t dst, const CUtensorMap *map, int k, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(k), "r"(row), "r"(bar)
               : "memory");
}

// The same from one block of a pair that works on a common tile: bytes are counted on a barrier of
// either block (an address in the cluster's window).
__device__ __forceinline__ void box_load_pair(uint32_t dst, const CUtensorMap *map, int k, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(k), "r"(row), "r"(bar)
               : "memory");
}

// Shared-memory operand descriptor: rows of 128 bytes along K in the 128-byte swizzle, groups of
// eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return (uint64_t(addr & 0x3ffff) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// 16 accumulator columns of the warp's 32 lanes.
__device__ __forceinline__ void tmem_load16(uint32_t addr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address, in the cluster's window, of what `addr` is in this block's shared memory, in block `rank`.
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_in_block(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrives at the barrier `bar` of both blocks of a pair when the matrix instructions issued so far have completed.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(uint16_t(3))
               : "memory");
}
__device__ __forceinline__ int load_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float load_as_float(const void *p, int64_t i, int dtype) {
  if (dtype == MGV_DTYPE_F16) return __half2float(static_cast<const __half *>(p)[i]);
  if (dtype == MGV_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  return static_cast<const float *>(p)[i];
}

// v / (1 + exp(-v)); exp and the quotient err by a few steps of fp32, far below the 16-bit output
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }

template <bool BF16>
__device__ __forceinline__ uint16_t round_out(float v) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// What a lane of the epilogue knows of its output feature (one lane per weight row).
struct Feature {
  int n;
  bool inside;
  float scale, bias;
};
template <bool BF16>
__device__ __forceinline__ Feature load_feature(const GemmI8Params &p, int n) {
  Feature f = {n, n < p.N, 0.0f, 0.0f};
  if (f.inside) {
    f.scale = load_as_float(p.w_scale, n, p.scale_dtype);
    if (p.bias) f.bias = load_as_float(p.bias, n, BF16 ? MGV_DTYPE_BF16 : MGV_DTYPE_F16);
  }
  return f;
}

// Sums of two neighbouring rows m, m + 1 of the activations for the lane's feature, scaled,
// activated and stored.  Lanes 2i and 2i + 1 swap one value each, so that the even lane holds both
// features of row m and the odd lane both of row m + 1: one 32-bit store, or gate and up together.
// All 32 lanes call it.
template <int ACT, bool BF16>
__device__ __forceinline__ void finish_pair(const GemmI8Params &p, const Feature &f, int m, int a0, int a1, float s0, float s1) {
  float v0 = fmaf(float(a0), f.scale * s0, f.bias), v1 = fmaf(float(a1), f.scale * s1, f.bias);
  if (ACT == kActRelu) v0 = v0 < 0.0f ? 0.0f : v0, v1 = v1 < 0.0f ? 0.0f : v1;
  if (ACT == kActSilu) v0 = silu(v0), v1 = silu(v1);
  const bool odd = f.n & 1;
  uint16_t *out = static_cast<uint16_t *>(p.out);
  if (ACT == kActGated || p.wide) {
    const float got = __shfl_xor_sync(~0u, odd ? v0 : v1, 1);
    const float lo = odd ? got : v0, hi = odd ? v1 : got;
    const int row = m + (odd ? 1 : 0);
    if (row >= p.M) return;
    if (ACT == kActGated) {
      if (f.inside) out[int64_t(row) * p.ldd + (f.n >> 1)] = round_out<BF16>(silu(lo) * hi);
      return;
    }
    const int n = f.n & ~1;
    uint16_t *at = out + int64_t(row) * p.ldd + n;
    if (n + 1 < p.N) *reinterpret_cast<uint32_t *>(at) = uint32_t(round_out<BF16>(lo)) | uint32_t(round_out<BF16>(hi)) << 16;
    else if (n < p.N) *at = round_out<BF16>(lo);
    return;
  }
  if (!f.inside) return;
  if (m < p.M) out[int64_t(m) * p.ldd + f.n] = round_out<BF16>(v0);
  if (m + 1 < p.M) out[int64_t(m + 1) * p.ldd + f.n] = round_out<BF16>(v1);
}

#endif  // __CUDACC__

// ---- host side, shared by the translation units ----

struct GemmI8Plan {
  GemmI8Params p;
  int device = 0, grid = 0, smem = 0, cluster = 1, act = 0, bf16 = 0, flags = 0;
  int pair = 0;  // the kernel of block pairs takes the call
};

// Launches KERN as the plan says; its first launch on a device lifts its shared-memory limit.
template <auto KERN>
mgv_status launch_gemm(const GemmI8Plan &pl, cudaStream_t s) {
  static bool configured[64];
  static std::mutex mu;
  if (pl.device < 0 || pl.device >= 64) return fail(MGV_STATUS_UNSUPPORTED, "gemm_i8: device index %d beyond 63", pl.device);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!configured[pl.device]) {
      int optin = 0;
      cudaFuncAttributes fa;
      MGV_CUDA_TRY(cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, pl.device));
      MGV_CUDA_TRY(cudaFuncGetAttributes(&fa, KERN));
      MGV_CUDA_TRY(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, optin - int(fa.sharedSizeBytes)));
      configured[pl.device] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.grid);
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  int n = 0;
  if (pl.cluster > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = unsigned(pl.cluster);
    attrs[n].val.clusterDim.y = attrs[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pl.flags & MGV_FLAG_PDL) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = n;
  MGV_CUDA_TRY(cudaLaunchKernelEx(&cfg, KERN, pl.p));
  return MGV_STATUS_OK;
}

// The kernel of block pairs (mgv_gemm_pair.cu).
mgv_status launch_gemm_pair(const GemmI8Plan &pl, cudaStream_t s);

}  // namespace mgv
