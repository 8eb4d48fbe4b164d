// int8 matrix product with a scale for each row and each output feature: entry points, plan and kernels.
#include <algorithm>
#include <mutex>
#include <new>

#include "mgv_gemm_parts.cuh"

namespace mgv {

// One tile -- 128 output features x p.bt activation rows -- per cluster of p.split blocks, each with
// its share of K.  The weights are the matrix instruction's 128-row operand and the activations its
// column operand, whose width goes from 16 up: one token costs a sixteen-column tile, not 128 rows.
// Weights and activations reach a ring of shared-memory slots by tiled bulk copies, one thread issues
// the matrix instructions, accumulators are 32-bit integers in tensor memory: lane = feature, column =
// row of the activations.  With split > 1 every block sends each other one its sums of that block's share of the columns, and
// adds and finishes its own share; integer sums, so the result does not depend on the split.
template <int ACT, bool BF16>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_i8_block_kernel(const __grid_constant__ GemmI8Params p) {
  extern __shared__ uint8_t dynamic[];
  __shared__ GemmBlockShared sh;
  const uint32_t ring = (smem_u32(dynamic) + 1023) & ~1023u;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t rank = p.split > 1 ? cluster_rank() : 0;
  const uint32_t tile = blockIdx.x / uint32_t(p.split);
  const int n0 = int(tile % uint32_t(p.n_tiles)) * kGemmRows, m0 = int(tile / uint32_t(p.n_tiles)) * p.bt;
  const int slices = (p.K + kGemmK - 1) / kGemmK;
  const int first = int(int64_t(slices) * rank / p.split), count = int(int64_t(slices) * (rank + 1) / p.split) - first;
  const uint32_t slot_bytes = kGemmABytes + p.bt * kGemmK;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) bar_init(smem_u32(&sh.full[i]), 1), bar_init(smem_u32(&sh.empty[i]), 1);
    bar_init(smem_u32(&sh.done), 1);
    sh.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, sh.tmem_base, 0);
  // only now: a dependent kernel that starts on this SM may hold tensor memory while it waits for this one to end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    // weights of the first ring fill before the wait for the previous kernel, its output (x) after it
    const bool one = elect_one();
    const int ahead = min(count, p.stages);
    if (one) {
      for (int i = 0; i < ahead; ++i) {
        bar_expect(smem_u32(&sh.full[i]), slot_bytes);
        box_load(ring + i * slot_bytes, &p.w_map, (first + i) * kGemmK, n0, smem_u32(&sh.full[i]));
      }
    }
    asm volatile("griddepcontrol.wait;\n\tfence.proxy.async.global;" ::: "memory");
    if (one)
      for (int i = 0; i < ahead; ++i)
        box_load(ring + i * slot_bytes + kGemmABytes, &p.x_map, (first + i) * kGemmK, m0, smem_u32(&sh.full[i]));
    int slot = 0, issued = ahead;
    uint32_t phase = 0;
    for (int i = ahead; i < count; ++i, ++issued) {
      if (!bar_wait(smem_u32(&sh.empty[slot]), phase, p.err)) break;
      if (one) {
        const uint32_t bar = smem_u32(&sh.full[slot]), dst = ring + slot * slot_bytes;
        bar_expect(bar, slot_bytes);
        box_load(dst, &p.w_map, (first + i) * kGemmK, n0, bar);
        box_load(dst + kGemmABytes, &p.x_map, (first + i) * kGemmK, m0, bar);
      }
      if (++slot == p.stages) slot = 0, phase ^= 1;
    }
    // no copy may be in flight when the block ends: the last ones are waited for, whoever else gave up
    for (int i = max(0, issued - p.stages); i < issued; ++i)
      if (!bar_wait(smem_u32(&sh.full[i % p.stages]), (i / p.stages) & 1, p.err)) break;
  } else if (warp == 1) {
    const bool one = elect_one();
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < count; ++i) {
      ok = bar_wait(smem_u32(&sh.full[slot]), phase, p.err);
      if (!ok) break;
      tmem_fence_after();
      const uint64_t a = operand_desc(ring + slot * slot_bytes), b = operand_desc(ring + slot * slot_bytes + kGemmABytes);
      if (one) {
#pragma unroll
        for (int k = 0; k < kGemmK / 32; ++k)  // 32 bytes of K per instruction: two 16-byte steps of the descriptors
          multiply_add<1>(tmem, a + 2 * k, b + 2 * k, p.idesc, i + k > 0);
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&sh.empty[slot])) : "memory");
      }
      __syncwarp();
      if (++slot == p.stages) slot = 0, phase ^= 1;
    }
    if (one) {
      if (!ok) *static_cast<volatile int *>(&sh.failed) = 1;
      asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&sh.done)) : "memory");
    }
  }

  // tensor memory: a warp reads the 32 lanes of its number modulo 4
  const int quarter = warp % 4, row = quarter * 32 + lane;
  const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
  bool good = true;
  Feature f = {};
  if (warp >= 2) {
    f = load_feature<BF16>(p, n0 + row);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = threadIdx.x - 64; i < p.bt; i += 128) sh.x_scale[i] = m0 + i < p.M ? p.x_scale[m0 + i] : 0.0f;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    good = bar_wait(smem_u32(&sh.done), 0, p.err) && !*static_cast<volatile int *>(&sh.failed);
    tmem_fence_after();
    if (p.split == 1 && good) {
      const int columns = min(p.bt, p.M - m0);
      for (int c = 0; c < columns; c += 16) {
        int v[16];
        __syncwarp();
        tmem_load16(lanes + c, v);
        tmem_wait_load();
        finish16<ACT, BF16>(p, f, m0 + c, columns - c, v, sh.x_scale + c);
      }
    }
  }
  if (p.split > 1) {
    // Every copy of the cluster has landed and every matrix instruction has read its slot: the rings'
    // memory is free for the sums.  Block r finishes the 16-column groups r, r + split, ...; of each it
    // gets, from each block, [4 quads of columns][128 features][4 columns].
    cluster_sync();
    const int groups = (min(p.bt, p.M - m0) + 15) / 16;
    constexpr int kQuad = kGemmRows * 16, kGroup = 4 * kQuad;
    if (warp >= 2) {
      for (int g = 0; g < groups; ++g) {
        int v[16];
        __syncwarp();
        tmem_load16(lanes + 16 * g, v);
        tmem_wait_load();
        const uint32_t to = in_block(ring, g % p.split) + ((g / p.split) * p.split + rank) * kGroup + row * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) store_cluster(to + i * kQuad, v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
      tmem_fence_before();
    }
    cluster_sync();
    if (warp >= 2 && good) {
      for (int g = int(rank); g < groups; g += p.split) {
        const uint32_t from = ring + (g / p.split) * p.split * kGroup + row * 16;
        int v[16] = {};
        for (int b = 0; b < p.split; ++b) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int4 u = load_shared(from + b * kGroup + i * kQuad);
            v[4 * i] += u.x, v[4 * i + 1] += u.y, v[4 * i + 2] += u.z, v[4 * i + 3] += u.w;
          }
        }
        finish16<ACT, BF16>(p, f, m0 + 16 * g, p.M - m0 - 16 * g, v, sh.x_scale + 16 * g);
      }
    }
  } else {
    tmem_fence_before();
    __syncwarp();
    __syncthreads();
  }
  if (warp == 1) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
  }
}

static mgv_status check_args(const mgv_gemm_i8_args *a) {
  if (!a || a->struct_size != int32_t(sizeof(*a))) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: args null or of another version");
  if (a->M < 0 || a->M > (1 << 30)) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: M=%lld outside 0..2^30", (long long)a->M);
  if (a->N < 1 || a->N > (1 << 30)) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: N=%d outside 1..2^30", a->N);
  if (a->K < 1 || a->K > 131071) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: K=%d outside 1..131071", a->K);
  if (a->out_dtype != MGV_DTYPE_F16 && a->out_dtype != MGV_DTYPE_BF16)
    return fail(MGV_STATUS_UNSUPPORTED, "gemm_i8: out_dtype %d is neither F16 nor BF16", a->out_dtype);
  if (a->scale_dtype < MGV_DTYPE_F16 || a->scale_dtype > MGV_DTYPE_F32)
    return fail(MGV_STATUS_UNSUPPORTED, "gemm_i8: scale_dtype %d is unknown", a->scale_dtype);
  const int acts = MGV_FLAG_ACT_RELU | MGV_FLAG_ACT_SILU | MGV_FLAG_GATED_SILU, act = a->flags & acts;
  if (a->flags & ~(acts | MGV_FLAG_PDL)) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: flags %d do not apply", a->flags);
  if (act & (act - 1)) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: one activation at most (flags %d)", a->flags);
  const bool gated = act == MGV_FLAG_GATED_SILU;
  if (gated && a->N % 2) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: a gated layer needs an even N (%d)", a->N);
  if (a->reserved) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: reserved must be 0");
  if (a->M == 0) return MGV_STATUS_OK;
  if (!a->x || !a->weights || !a->x_scale || !a->weight_scale || !a->out) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: null operand");
  if (a->ldx < a->K || a->ldw < a->K || a->ldd < (gated ? a->N / 2 : a->N))
    return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: a leading dimension is shorter than its row (ldx %lld, ldw %lld, ldd %lld)",
                (long long)a->ldx, (long long)a->ldw, (long long)a->ldd);
  if (a->ldx >= (int64_t(1) << 40) || a->ldw >= (int64_t(1) << 40) || a->ldd >= (int64_t(1) << 40))
    return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: leading dimension too large");
  if (a->ldx % 16 || a->ldw % 16 || reinterpret_cast<uintptr_t>(a->x) % 16 || reinterpret_cast<uintptr_t>(a->weights) % 16)
    return fail(MGV_STATUS_MISALIGNED, "gemm_i8: rows of x and weights must start at multiples of 16 bytes (ldx %lld, ldw %lld)",
                (long long)a->ldx, (long long)a->ldw);
  const int scale_bytes = a->scale_dtype == MGV_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->x_scale) % 4 || reinterpret_cast<uintptr_t>(a->weight_scale) % scale_bytes ||
      reinterpret_cast<uintptr_t>(a->bias) % 2 || reinterpret_cast<uintptr_t>(a->out) % 2)
    return fail(MGV_STATUS_MISALIGNED, "gemm_i8: scales, bias and out must be aligned to their elements");
  return MGV_STATUS_OK;
}

}  // namespace mgv

using namespace mgv;

struct mgv_gemm_i8_plan : GemmI8Plan {};


// A dense int8 matrix [rows][ld] as boxes of 128 bytes of K x box_rows rows, in the 128-byte swizzle
// that the matrix instruction reads; what lies beyond K or the last row arrives as zeros.
static mgv_status encode_rows(CUtensorMap *map, const void *ptr, int64_t rows, int K, int64_t ld, int box_rows) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  static std::mutex mu;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!encode) {
      void *fn = nullptr;
      cudaDriverEntryPointQueryResult q;
      MGV_CUDA_TRY(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
      if (q != cudaDriverEntryPointSuccess || !fn) return fail(MGV_STATUS_CUDA_ERROR, "gemm_i8: the driver has no cuTensorMapEncodeTiled");
      encode = reinterpret_cast<Encode>(fn);
    }
  }
  const cuuint64_t dims[2] = {cuuint64_t(K), cuuint64_t(rows)}, strides[1] = {cuuint64_t(ld)};
  const cuuint32_t box[2] = {kGemmK, cuuint32_t(box_rows)}, elem[2] = {1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(ptr), dims, strides, box, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MGV_STATUS_CUDA_ERROR, "gemm_i8: cuTensorMapEncodeTiled failed (%d)", int(r));
  return MGV_STATUS_OK;
}

// Instruction descriptor: 32-bit integer sums (2 at bit 4), signed operands (1 at bits 7 and 10),
// columns / 8 at bit 17, rows / 16 at bit 24.
static uint32_t instruction(int rows, int columns) { return 2u << 4 | 1u << 7 | 1u << 10 | uint32_t(columns / 8) << 17 | uint32_t(rows / 16) << 24; }

// bt, split: 0 where the plan is free to choose.
static mgv_status plan_block(GemmI8Plan &pl, int64_t M, int bt, int split, int sms, int most) {
  GemmI8Params &p = pl.p;
  // columns of the matrix instruction: 16, or a multiple of 32 up to 256
  p.bt = bt ? bt : M <= 16 ? 16 : int(std::min<int64_t>(256, (M + 31) / 32 * 32));
  p.n_tiles = (p.N + kGemmRows - 1) / kGemmRows;
  const int64_t tiles = p.n_tiles * ((M + p.bt - 1) / p.bt);
  const int slices = (p.K + kGemmK - 1) / kGemmK;
  p.split = 1;
  while (p.split < 8 && 2 * p.split <= slices && tiles * p.split < sms * 7 / 8) p.split *= 2;
  if (split) p.split = split;
  p.split = std::min(p.split, slices);
  const int64_t grid = tiles * p.split;
  if (grid > 0x7fffffff) return fail(MGV_STATUS_UNSUPPORTED, "gemm_i8: too many tiles (M=%lld N=%d)", (long long)M, p.N);
  pl.grid = int(grid);
  pl.cluster = p.split;
  p.tmem_cols = 32;
  while (int(p.tmem_cols) < p.bt) p.tmem_cols *= 2;
  // Shared memory of a block: its share of an SM by the number of blocks an SM gets.  Blocks that fit an SM by
  // their shared memory must fit it by their tensor memory too (512 columns), or one would wait in its
  // allocation for another to end: at least the same fraction of both.
  const int slot = kGemmABytes + p.bt * kGemmK, share = (slices + p.split - 1) / p.split;
  const int fixed = kGemmReserved + int(sizeof(GemmBlockShared));  // beside the dynamic part; kGemmAlign of that goes to alignment
  const int64_t wanted = std::min<int64_t>((grid + sms - 1) / sms, 512 / p.tmem_cols);
  int per_sm = int(std::max<int64_t>(1, wanted));
  while (per_sm > 1 && (kGemmSmShared / per_sm - fixed - kGemmAlign) / slot < std::min(3, share)) --per_sm;
  const int room = std::min(kGemmSmShared / per_sm - fixed, most - int(sizeof(GemmBlockShared))) - kGemmAlign;
  p.stages = std::min(std::min(share, kGemmMaxStages), room / slot);
  int smem = p.stages * slot;
  if (p.split > 1) smem = std::max(smem, (p.bt / 16 + p.split - 1) / p.split * p.split * kGemmRows * 64);  // the sums of a split tile
  smem = std::max(smem + kGemmAlign, int(int64_t(kGemmSmShared) * p.tmem_cols / 512) - fixed);
  pl.smem = smem;
  p.idesc = instruction(kGemmRows, p.bt);
  return MGV_STATUS_OK;
}

static void plan_pair(GemmI8Plan &pl, int64_t M, int bt, int sms, int most) {
  GemmI8Params &p = pl.p;
  p.bt = bt ? bt : int(std::min<int64_t>(256, (M + 31) / 32 * 32));
  p.n_tiles = (p.N + 2 * kGemmRows - 1) / (2 * kGemmRows);
  p.m_tiles = int((M + p.bt - 1) / p.bt);
  p.split = 1;
  const int64_t tiles = int64_t(p.n_tiles) * p.m_tiles;
  pl.grid = int(2 * std::min<int64_t>(tiles, sms / 2));
  pl.cluster = 2;
  p.tmem_cols = 64;  // two accumulators
  while (int(p.tmem_cols) < 2 * p.bt) p.tmem_cols *= 2;
  const int slot = kGemmABytes + p.bt / 2 * kGemmK, room = most - int(sizeof(GemmPairShared));
  p.stages = std::min(kGemmMaxStages, (room - kGemmAlign) / slot);
  pl.smem = room;  // one block per SM: it may hold all of the tensor memory
  p.idesc = instruction(2 * kGemmRows, p.bt);
}

static mgv_status prepare(const mgv_gemm_i8_args *a, mgv_gemm_i8_plan &pl) {
  mgv_status st = check_args(a);
  if (st != MGV_STATUS_OK) return st;
  GemmI8Params &p = pl.p;
  p = GemmI8Params{};
  pl.flags = a->flags;
  MGV_CUDA_TRY(cudaGetDevice(&pl.device));
  if (a->M == 0) return MGV_STATUS_OK;
  int sms = 0, most = 0;
  MGV_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, pl.device));
  MGV_CUDA_TRY(cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, pl.device));
  p.x_scale = static_cast<const float *>(a->x_scale);
  p.w_scale = a->weight_scale; p.bias = a->bias; p.out = a->out; p.ldd = a->ldd;
  p.M = int(a->M); p.N = a->N; p.K = a->K; p.scale_dtype = a->scale_dtype;
  p.wide = reinterpret_cast<uintptr_t>(a->out) % 4 == 0 && a->ldd % 2 == 0;
  p.err = device_error_word();
  if (!p.err) return fail(MGV_STATUS_CUDA_ERROR, "gemm_i8: no device error word");
  pl.act = a->flags & MGV_FLAG_ACT_RELU ? kActRelu : a->flags & MGV_FLAG_ACT_SILU ? kActSilu : a->flags & MGV_FLAG_GATED_SILU ? kActGated : kActNone;
  pl.bf16 = a->out_dtype == MGV_DTYPE_BF16;

  const int want = (a->hints >> 8) & 31;
  pl.pair = a->hints & MGV_GEMM_HINT_PAIR || (!(a->hints & MGV_GEMM_HINT_BLOCK) && a->M > 256);
  if (pl.pair) plan_pair(pl, a->M, want ? std::min(256, (want + 1) / 2 * 32) : 0, sms, most);
  else if ((st = plan_block(pl, a->M, want == 1 ? 16 : std::min(256, (want + 1) / 2 * 32), want ? (a->hints & 7) + 1 : 0, sms, most)) != MGV_STATUS_OK) return st;
  if ((st = encode_rows(&p.w_map, a->weights, a->N, a->K, a->ldw, kGemmRows)) != MGV_STATUS_OK) return st;
  return encode_rows(&p.x_map, a->x, a->M, a->K, a->ldx, pl.pair ? p.bt / 2 : p.bt);
}

template <int ACT>
static mgv_status launch_act(const GemmI8Plan &pl, cudaStream_t s) {
  return pl.bf16 ? launch_gemm<gemm_i8_block_kernel<ACT, true>>(pl, s) : launch_gemm<gemm_i8_block_kernel<ACT, false>>(pl, s);
}

static mgv_status launch(const GemmI8Plan &pl, cudaStream_t s) {
  if (pl.p.M == 0) return MGV_STATUS_OK;
  if (pl.pair) return launch_gemm_pair(pl, s);
  switch (pl.act) {
    case kActRelu: return launch_act<kActRelu>(pl, s);
    case kActSilu: return launch_act<kActSilu>(pl, s);
    case kActGated: return launch_act<kActGated>(pl, s);
    default: return launch_act<kActNone>(pl, s);
  }
}

extern "C" void mgv_gemm_i8_args_init(mgv_gemm_i8_args *a) {
  if (!a) return;
  *a = mgv_gemm_i8_args{};
  a->struct_size = int32_t(sizeof(*a));
}

extern "C" mgv_status mgv_gemm_i8(const mgv_gemm_i8_args *a, mgv_stream_t s) {
  mgv_gemm_i8_plan pl;
  const mgv_status st = prepare(a, pl);
  return st == MGV_STATUS_OK ? launch(pl, s) : st;
}

extern "C" mgv_status mgv_gemm_i8_plan_create(const mgv_gemm_i8_args *a, mgv_gemm_i8_plan **plan) {
  if (!plan) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8_plan_create: null plan pointer");
  *plan = nullptr;
  mgv_gemm_i8_plan *pl = new (std::nothrow) mgv_gemm_i8_plan;
  if (!pl) return fail(MGV_STATUS_CUDA_ERROR, "gemm_i8_plan_create: out of host memory");
  const mgv_status st = prepare(a, *pl);
  if (st != MGV_STATUS_OK) {
    delete pl;
    return st;
  }
  *plan = pl;
  return MGV_STATUS_OK;
}

extern "C" mgv_status mgv_gemm_i8_plan_run(const mgv_gemm_i8_plan *pl, mgv_stream_t s) {
  if (!pl) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8_plan_run: null plan");
  int dev = 0;
  MGV_CUDA_TRY(cudaGetDevice(&dev));
  if (dev != pl->device) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8_plan_run: the plan was made on device %d, current is %d", pl->device, dev);
  return launch(*pl, s);
}

extern "C" void mgv_gemm_i8_plan_destroy(mgv_gemm_i8_plan *pl) { delete pl; }
