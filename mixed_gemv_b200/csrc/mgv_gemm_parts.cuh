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
  alignas(64) CUtensorMap x_half_map;  // ... x half of them, for halved tiles
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
  int split;       // blocks, or pairs of blocks, of a cluster that share a tile's K range
  int n_tiles, m_tiles;
  int sums_off;    // split: where the sums arrive in dynamic shared memory; 0: in the ring, once it is free
  int halved;      // pairs: tiles from this one on, in the order of work, come in two halves of their rows
  uint32_t idesc, half_idesc;  // instruction descriptors of the matrix instruction, for whole and halved tiles
  uint32_t tmem_cols;
};

constexpr int kGemmRows = 128;             // weight rows (output features) a block owns of a tile
constexpr int kGemmK = 128;                // K of a ring slot: one 128-byte swizzle row
constexpr int kGemmABytes = kGemmRows * kGemmK;
constexpr int kGemmEpilogue = 256;         // threads of the epilogue: two warps for each 32 lanes of tensor memory
constexpr int kGemmThreads = 64 + kGemmEpilogue;  // ... behind the producer warp and the matrix warp
constexpr int kGemmBlocksPerSm = 3;        // of the single-block kernel, by its registers
constexpr int kGemmMaxStages = 16;
constexpr int kGemmAlign = 1024;           // of the ring; dynamic shared memory lost to it at most
constexpr int kGemmReserved = 1024;        // shared memory the system takes for each block
constexpr int kGemmSmShared = 228 * 1024;  // of an SM
constexpr int kGemmTimeout = 0x100;        // bit of the device error word

// Static shared memory of the two kernels.
struct GemmBlockShared {
  alignas(16) float x_scale[256];
  uint64_t full[kGemmMaxStages], empty[kGemmMaxStages], done, sums;
  uint32_t tmem_base;
  int failed;
};
struct GemmPairShared {
  alignas(16) float x_scale[2][256];
  uint64_t full[kGemmMaxStages], empty[kGemmMaxStages], ready[2], drained[2], sums;
  uint32_t tmem_base;
};

constexpr int kQuadBytes = kGemmRows * 16;  // sums of 128 features x 4 columns

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGated = 3 };

#if defined(__CUDACC__)

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One lane of a converged warp.  The roles below are whole warps with one lane elected for the
// instructions that a single thread issues: with operands and control flow the same for the warp, a
// matrix instruction takes 40 cycles to issue and a slot's wait, four instructions and commit 265;
// the same by a lone thread in a branch of its own, with waits of cluster scope, took 640.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(one));
  return one;
}
template <bool CLUSTER>
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if (CLUSTER)
    asm volatile("{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 q, [%1], %2;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred q;\n\tmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
  return ok;
}
template <bool CLUSTER>
__device__ __noinline__ bool bar_wait_long(uint32_t bar, uint32_t parity, int *err) {
  bool ok = false;
  for (int i = 0; i < 1024 && !ok; ++i) ok = bar_try<CLUSTER>(bar, parity);
  const uint64_t t0 = global_timer_ns();
  while (!ok && global_timer_ns() - t0 < 1000000000ull)
    for (int i = 0; i < 256 && !ok; ++i) ok = bar_try<CLUSTER>(bar, parity);
  if (!ok) atomicOr(err, kGemmTimeout);
  return __all_sync(~0u, ok);
}
// A warp waits for the phase of the given parity, for at most about a second; false, for all its lanes
// and with the device error word set, when it gave up.  CLUSTER: threads of another block arrive here.
template <bool CLUSTER = false>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int *err) {
  return __all_sync(~0u, bar_try<CLUSTER>(bar, parity)) || bar_wait_long<CLUSTER>(bar, parity, err);
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

// D (tensor memory) = or += A (rows x 32) * B (columns x 32)^T of int8 operands, by one SM or a pair
template <int SMS>
__device__ __forceinline__ void multiply_add(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  if (SMS == 1)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, q;\n\t}" ::"r"(d), "l"(a),
        "l"(b), "r"(idesc), "r"(add)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, q;\n\t}" ::"r"(d), "l"(a),
        "l"(b), "r"(idesc), "r"(add)
        : "memory");
}

// 16 accumulator columns of the warp's 32 lanes; the registers hold them behind tmem_wait only.
__device__ __forceinline__ void tmem_load16(uint32_t addr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait(int (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::"memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <bool RELEASE>  // whether what the block wrote before has to be seen behind the wait
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  if (RELEASE) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  else asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
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
// Arrives at the barrier `bar` of both blocks of a pair, the first of which has rank `lead`, when the matrix
// instructions issued so far have completed.
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t lead) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(uint16_t(3u << lead))
               : "memory");
}
// 16 bytes into the shared memory of a block of the cluster, counted on that block's barrier `bar`
// (both addresses in the cluster's window)
__device__ __forceinline__ void send16(uint32_t addr, uint32_t bar, int a, int b, int c, int d) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%2,%3,%4,%5}, [%1];" ::"r"(addr), "r"(bar), "r"(a),
               "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ int4 load_shared(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float load_as_float(const void *p, int64_t i, int dtype) {
  if (dtype == MGV_DTYPE_F16) return __half2float(static_cast<const __half *>(p)[i]);
  if (dtype == MGV_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  return static_cast<const float *>(p)[i];
}

// v / (1 + exp(-v)) = v m^2 / (1 + h^2) with h = exp(-|v| / 2) and m = h below zero, 1 above: neither the exponential nor the
// denominator, which is in 1..2, leaves fp32's normal numbers before the result does, so a bf16 gate far below zero keeps its
// value (v / (1 + exp(-v)) itself is 0 from -88 on).  The argument of 2^x errs by |v| steps of 2^-24, the square by twice as much:
// 2^-16 of the value at -100, far below the 16-bit output.  The approximate instructions on normal numbers need no care
// around them: 4096 x 8192 x 1024 gated 48.0 us, with __expf and __fdividef 57.0, with v / (1 + __expf(-v)) 51.7.
__device__ __forceinline__ float silu(float v) {
  float h, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(v) * -0.72134752f));  // log2(e) / 2
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.0f)));
  const float m = v > 0.0f ? 1.0f : h;
  return v * m * (m * r);
}

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

// Sums of C neighbouring activation rows from m on for the lane's feature -- `rows` of them exist --
// scaled, activated and stored.  The sum takes the feature's scale first: the two scales' product may be beyond fp32
// (infinite, or short of bits) where the value is not; a sum times a weight's scale below 2^96 is not, and a sum of zero
// stays zero.  Lanes 2i and 2i + 1 swap half of their values, so that the even lane holds both features of the even rows
// and the odd lane both of the odd rows: one 32-bit store for two features, or gate and up together.  All 32 lanes call it;
// x_scale is 16-byte aligned.
template <int ACT, bool BF16, int C>
__device__ __forceinline__ void finish(const GemmI8Params &p, const Feature &f, int m, int rows, const int (&v)[C], const float *x_scale) {
  float y[C];
#pragma unroll
  for (int i = 0; i < C; i += 4) {
    const float4 s = *reinterpret_cast<const float4 *>(x_scale + i);
    y[i] = fmaf(float(v[i]) * f.scale, s.x, f.bias);
    y[i + 1] = fmaf(float(v[i + 1]) * f.scale, s.y, f.bias);
    y[i + 2] = fmaf(float(v[i + 2]) * f.scale, s.z, f.bias);
    y[i + 3] = fmaf(float(v[i + 3]) * f.scale, s.w, f.bias);
  }
  if (ACT == kActRelu || ACT == kActSilu) {
#pragma unroll
    for (int i = 0; i < C; ++i) y[i] = ACT == kActSilu ? silu(y[i]) : y[i] < 0.0f ? 0.0f : y[i];
  }
  const int odd = f.n & 1;
  uint16_t *out = static_cast<uint16_t *>(p.out);
  if (ACT == kActGated || p.wide) {
    float got[C / 2];
#pragma unroll
    for (int i = 0; i < C / 2; ++i) got[i] = __shfl_xor_sync(~0u, odd ? y[2 * i] : y[2 * i + 1], 1);
    if (ACT == kActGated) {
      uint16_t *at = out + int64_t(m + odd) * p.ldd + (f.n >> 1);
#pragma unroll
      for (int i = 0; i < C / 2; ++i) {
        const float gate = odd ? got[i] : y[2 * i], up = odd ? y[2 * i + 1] : got[i];
        if (f.inside && 2 * i + odd < rows) *at = round_out<BF16>(silu(gate) * up);
        at += 2 * p.ldd;
      }
    } else {
      const bool both = (f.n | 1) < p.N, one = !both && (f.n & ~1) < p.N;  // the last feature of an odd N stands alone
      uint16_t *at = out + int64_t(m + odd) * p.ldd + (f.n & ~1);
#pragma unroll
      for (int i = 0; i < C / 2; ++i) {
        const uint32_t lo = round_out<BF16>(odd ? got[i] : y[2 * i]), hi = round_out<BF16>(odd ? y[2 * i + 1] : got[i]);
        if (both && 2 * i + odd < rows) *reinterpret_cast<uint32_t *>(at) = lo | hi << 16;
        if (one && 2 * i + odd < rows) *at = uint16_t(lo);
        at += 2 * p.ldd;
      }
    }
    return;
  }
  uint16_t *at = out + int64_t(m) * p.ldd + f.n;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    if (f.inside && i < rows) *at = round_out<BF16>(y[i]);
    at += p.ldd;
  }
}

// The 16-column groups at c, c + 32, ... of a tile from row m0 on, out of the warp's lanes of tensor
// memory.  (Fetching the next group while one is finished gained nothing and took 30 registers more.)
template <int ACT, bool BF16>
__device__ __forceinline__ void finish_columns(const GemmI8Params &p, const Feature &f, uint32_t lanes, int m0, int c, int columns, const float *x_scale) {
  for (; c < columns; c += 32) {
    int v[16];
    __syncwarp();
    tmem_load16(lanes + c, v);
    tmem_wait(v);
    finish<ACT, BF16>(p, f, m0 + c, columns - c, v, x_scale + c);
  }
}

#endif  // __CUDACC__

// ---- host side, shared by the translation units ----

struct GemmI8Plan {
  GemmI8Params p;
  int device = 0, grid = 0, smem = 0, cluster = 1, act = 0, bf16 = 0, flags = 0;
  int pair = 0;     // the kernel of block pairs takes the call
  double cost = 0;  // estimated cycles
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
