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
// row of the activations.  With split > 1 every block finishes a share of the columns, out of the sums that all
// blocks of the cluster send it; integer sums, so the result does not depend on the split.
// Bound by HBM (weights), and by a call's start, first fetch and exchange, some 3 us, where there is little of those: B200,
// dependent launches, 1 x 4096 x 4096 5.2 us, 16 x 22016 x 4096 gated 17.5 us (0.79 of the copy bandwidth).
template <int ACT, bool BF16>
__global__ void __launch_bounds__(kGemmThreads, kGemmBlocksPerSm) gemm_i8_block_kernel(const __grid_constant__ GemmI8Params p) {
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

  const bool one = elect_one();
  const int ahead = min(count, p.stages);  // slots of the first ring fill
  if (warp == 0 && one) {
    for (int i = 0; i < p.stages; ++i) bar_init(smem_u32(&sh.full[i]), 1), bar_init(smem_u32(&sh.empty[i]), 1);
    bar_init(smem_u32(&sh.done), 1);
    bar_init(smem_u32(&sh.sums), 1);
    sh.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async;" ::: "memory");
    // the weights first of all: before the rest of the set-up, and before the wait for the previous kernel
    for (int i = 0; i < ahead; ++i) {
      bar_expect(smem_u32(&sh.full[i]), slot_bytes);
      box_load(ring + i * slot_bytes, &p.w_map, (first + i) * kGemmK, n0, smem_u32(&sh.full[i]));
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tmem_fence_before();
  __syncwarp();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, sh.tmem_base, 0);
  const int columns = min(p.bt, p.M - m0), quads = (columns + 3) / 4;
  const int mine = p.split > 1 ? (quads - int(rank) + p.split - 1) / p.split : 0;  // column quads this block finishes of a split tile
  if (p.split > 1 && p.sums_off) cluster_arrive<true>();  // this block can be sent to: its barriers are set up

  if (warp == 0) {
    // A dependent kernel may start only now: behind the wait, so that it runs beside no kernel but this one, and
    // behind the allocation of tensor memory, of which it may hold some while it waits for this one.
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;\n\tfence.proxy.async.global;" ::: "memory");
    if (one) {
      for (int i = 0; i < ahead; ++i)
        box_load(ring + i * slot_bytes + kGemmABytes, &p.x_map, (first + i) * kGemmK, m0, smem_u32(&sh.full[i]));
      if (mine > 0) bar_expect(smem_u32(&sh.sums), mine * p.split * kQuadBytes);
    }
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
    // its wait for the first slot is limited, and the slot's activations are asked for behind the wait above: what the
    // previous kernel still takes is not to count
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
  const int quarter = warp % 4, half = warp >= 6, row = quarter * 32 + lane;
  const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
  bool good = true;
  Feature f = {};
  if (warp >= 2) {
    f = load_feature<BF16>(p, n0 + row);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (const int i = threadIdx.x - 64; i < p.bt) sh.x_scale[i] = m0 + i < p.M ? p.x_scale[m0 + i] : 0.0f;
    asm volatile("bar.sync 1, %0;" ::"n"(kGemmEpilogue) : "memory");
    good = bar_wait(smem_u32(&sh.done), 0, p.err) && !*static_cast<volatile int *>(&sh.failed);
    tmem_fence_after();
    if (p.split == 1 && good) finish_columns<ACT, BF16>(p, f, lanes, m0, half * 16, columns, sh.x_scale);
  }
  if (p.split > 1) {
    // Block r finishes the column quads r, r + split, ...; of each it gets [128 features][4 columns] from
    // every block, itself among them.  Where that goes into the ring, every copy of the cluster has to have
    // landed and every matrix instruction to have read its slot.
    if (!p.sums_off) cluster_arrive<true>();
    cluster_wait();
    const uint32_t sums = p.sums_off ? smem_u32(dynamic) + p.sums_off : ring;
    if (warp >= 2) {
      for (int c = half * 16; c < columns && good; c += 32) {
        int v[16];
        __syncwarp();
        tmem_load16(lanes + c, v);
        tmem_wait(v);
        int owner = c / 4 % p.split, at = c / 4 - owner + int(rank);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (c / 4 + i < quads)
            send16(in_block(sums + at * kQuadBytes + row * 16, owner), in_block(smem_u32(&sh.sums), owner), v[4 * i], v[4 * i + 1],
                   v[4 * i + 2], v[4 * i + 3]);
          if (++owner == p.split) owner = 0, at += p.split;
        }
      }
      tmem_fence_before();
    }
    cluster_arrive<false>();
    // Only blocks that finish columns are sent anything, and they wait for all of it: after that none of
    // them is written to.  Where the wait gave up, the block stays until all others have sent what they will.
    if (mine > 0) {
      if (!bar_wait<true>(smem_u32(&sh.sums), 0, p.err)) {
        cluster_wait();
      } else if (warp >= 2 && good) {
        for (int quad = int(rank) + half * p.split; quad < quads; quad += 2 * p.split) {
          const uint32_t from = sums + quad / p.split * p.split * kQuadBytes + row * 16;
          int v[4] = {};
          for (int b = 0; b < p.split; ++b) {
            const int4 u = load_shared(from + b * kQuadBytes);
            v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
          }
          finish<ACT, BF16>(p, f, m0 + 4 * quad, columns - 4 * quad, v, sh.x_scale + 4 * quad);
        }
      }
    }
    __syncwarp();
    __syncthreads();
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
  constexpr int hints = 7 | MGV_GEMM_HINT_BLOCK | MGV_GEMM_HINT_PAIR | 31 << 8;
  if (a->hints & ~hints) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: unknown bits in hints %d", a->hints);
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

// The estimate that tilings are compared by, in cycles.  Measured on B200 (4096-deep reductions, 1.9 GHz): an
// SM alone takes in 96 bytes a cycle from L2, all SMs together 7500 as single blocks and 9400 as pairs; a slice of
// 128 K keeps the issuing warp for 330 cycles at least and the matrix unit for the time of its four
// instructions (taken as half a cycle a column each, 40 at least; measured 127 at 256 columns); HBM delivers 3260 bytes a cycle but for the start and end of a block's row of slices; 16
// columns of an epilogue take 320 cycles; a split tile's exchange takes 1500 and, a column, 30 and
// 5 for each part beside the next call's start.
// (Of 20 shapes from 1 x 4096 x 4096 to 4096 x 4096 x 4096 -- rows x features x K -- the choice was within 8 % of the best
// tiling on 17 and 13 % off at most.)
constexpr double kSmBytes = 96, kBlockBytes = 7500, kPairBytes = 9400, kHbmBytes = 3260, kIssue = 330, kColumn16 = 320, kStart = 4500;

// chain: of the slices that one block works through; fed: to get all operands from L2 to the SMs
static double estimate(double chain, double fed, double weights, double tail) {
  return kStart + std::max(std::max(chain, fed), weights / kHbmBytes + 0.4 * chain) + tail;
}

static double exchange(int bt, int split) { return 1500 + bt * (30.0 + 5 * split); }

static int rounded_columns(int want) { return want == 1 ? 16 : std::min(256, (want + 1) / 2 * 32); }

static void plan_block(GemmI8Plan &pl, int64_t M, int bt, int split, int sms, int most) {
  GemmI8Params &p = pl.p;
  p.bt = bt;
  p.split = split;
  p.n_tiles = (p.N + kGemmRows - 1) / kGemmRows;
  p.m_tiles = int((M + bt - 1) / bt);
  p.sums_off = 0;
  p.tmem_cols = 32;
  while (int(p.tmem_cols) < bt) p.tmem_cols *= 2;
  p.idesc = instruction(kGemmRows, bt);
  const int64_t grid = int64_t(p.n_tiles) * p.m_tiles * split;
  const int slices = (p.K + kGemmK - 1) / kGemmK, share = (slices + split - 1) / split, slot = kGemmABytes + bt * kGemmK;
  // Shared memory of a block: its share of an SM by the number of blocks an SM gets, and half of it at most
  // for narrow tiles, so that the next call's blocks can start fetching weights beside it.  Blocks that fit an
  // SM by their shared memory must fit it by their tensor memory too (512 columns), or one would wait in
  // its allocation for another to end: at least the same fraction of both.
  const int fixed = kGemmReserved + int(sizeof(GemmBlockShared));  // beside the dynamic part; kGemmAlign of that goes to alignment
  const int64_t on_sm = (grid + sms - 1) / sms;
  int per_sm = int(std::max<int64_t>(bt <= 64 ? 2 : 1, std::min<int64_t>(std::min<int64_t>(on_sm, kGemmBlocksPerSm), 512 / p.tmem_cols)));
  while (per_sm > 1 && (kGemmSmShared / per_sm - fixed - kGemmAlign) / slot < std::min(3, share)) --per_sm;
  const int room = std::min(kGemmSmShared / per_sm - fixed, most - int(sizeof(GemmBlockShared))) - kGemmAlign;
  p.stages = std::min(std::min(share, kGemmMaxStages), room / slot);
  int smem = p.stages * slot + kGemmAlign;
  if (split > 1) {  // the sums of a split tile: beside the ring where they fit, which saves a wait, else in it
    const int sums = (bt / 4 + split - 1) / split * split * kQuadBytes;
    if (smem + sums <= room + kGemmAlign) {
      p.sums_off = smem;
      smem += sums;
    } else {
      smem = std::max(smem, sums + kGemmAlign);
    }
  }
  smem = std::max(smem, int(int64_t(kGemmSmShared) * p.tmem_cols / 512) - fixed);
  pl.pair = 0;
  pl.smem = smem;
  pl.grid = int(std::min<int64_t>(grid, 0x7fffffff));
  pl.cluster = split;
  const int64_t at_once = std::max(1, std::min(std::min(kGemmSmShared / (smem + fixed), int(512 / p.tmem_cols)), kGemmBlocksPerSm));
  const double slice = std::max(slot / kSmBytes, 4 * std::max(40.0, bt / 2.0));  // of the SM's time
  const double tail = split > 1 ? exchange(bt, split) : kColumn16 * ((bt + 15) / 16);
  const int64_t rounds = (on_sm + at_once - 1) / at_once;  // blocks that follow one another: each starts and ends alone
  const double chain = rounds * share * std::max(kIssue, slice) + (rounds - 1) * (2500 + tail);
  const double fed = std::max(double(on_sm) * share * slice, double(grid) * share * slot / kBlockBytes);
  pl.cost = estimate(chain, fed, double(p.N) * p.K, tail);
}

static void plan_pair(GemmI8Plan &pl, int64_t M, int bt, int split, int sms, int most) {
  GemmI8Params &p = pl.p;
  p.bt = bt;
  p.split = split;
  p.n_tiles = (p.N + 2 * kGemmRows - 1) / (2 * kGemmRows);
  p.m_tiles = int((M + bt - 1) / bt);
  p.tmem_cols = 64;  // two accumulators
  while (int(p.tmem_cols) < 2 * bt) p.tmem_cols *= 2;
  p.idesc = instruction(2 * kGemmRows, bt);
  const int64_t tiles = int64_t(p.n_tiles) * p.m_tiles, pairs = std::min<int64_t>(tiles, sms / 2);
  const int slices = ((p.K + kGemmK - 1) / kGemmK + split - 1) / split, slot = kGemmABytes + bt / 2 * kGemmK, room = most - int(sizeof(GemmPairShared));
  p.stages = std::min(kGemmMaxStages, (room - kGemmAlign) / slot);
  // the last round's tiles in halves where those are enough for no more than a round of their own
  const int64_t rounds = tiles / pairs, rest = tiles % pairs;
  const bool halve = split == 1 && rounds > 0 && rest > 0 && 2 * rest <= pairs && bt % 64 == 0;
  p.halved = int(halve ? tiles - rest : tiles);
  p.half_idesc = instruction(2 * kGemmRows, halve ? bt / 2 : bt);
  pl.pair = 1;
  pl.smem = room;  // one block per SM: it may hold all of the tensor memory
  pl.grid = int(2 * std::min<int64_t>(split > 1 ? tiles * split : pairs, 1 << 28));
  pl.cluster = 2 * split;
  auto round = [&](int rows) {  // a tile's epilogue runs beside the next tile
    const double slice = std::max(std::max((kGemmABytes + rows / 2 * kGemmK) / kSmBytes, kIssue), 2.0 * rows);
    return std::max(slices * slice, kColumn16 * (rows / 16));
  };
  const double tail = split > 1 ? exchange(bt, split) : kColumn16 * ((halve ? bt / 2 : bt) / 16);
  const double chain = rounds * round(bt) + (halve ? round(bt / 2) : rest ? round(bt) : 0);
  pl.cost = estimate(chain, 2.0 * tiles * split * slices * slot / kPairBytes, double(p.N) * p.K, tail);
}

// The tiling of least estimated cost, of those that the hints leave.
static mgv_status plan(GemmI8Plan &pl, const mgv_gemm_i8_args *a, int sms, int most) {
  const int rows = (a->hints >> 8) & 31, slices = (a->K + kGemmK - 1) / kGemmK;
  const int widest = int(std::min<int64_t>(256, (a->M + 31) / 32 * 32));
  GemmI8Plan best;
  best.cost = 0;
  auto keep = [&](const GemmI8Plan &one) {
    if (best.cost == 0 || one.cost < best.cost) best = one;
  };
  if (!(a->hints & MGV_GEMM_HINT_PAIR)) {
    for (int bt = 16; bt <= 256; bt += bt == 16 ? 16 : 32) {
      if (rows ? bt != rounded_columns(rows) : (a->M <= 16 ? bt > 16 : bt == 16 || bt > widest)) continue;
      // clusters of 3, 5, 6 or 7 blocks leave SMs of a GPC empty: 131 x 12288 x 4096 in threes takes 20 us, in ones 13
      for (int split = 1; split <= std::min(8, slices); split = rows ? split + 1 : 2 * split) {
        if (rows && split != std::min((a->hints & 7) + 1, slices)) continue;
        plan_block(pl, a->M, bt, split, sms, most);
        keep(pl);
      }
    }
  }
  if (!(a->hints & MGV_GEMM_HINT_BLOCK)) {
    for (int bt = 32; bt <= 256; bt += 32) {
      if (rows ? bt != std::max(32, rounded_columns(rows)) : bt > widest) continue;
      // pairs share a tile where all clusters fit the GPU at once (of 4 or 8 blocks, 32 or 16 find room in its GPCs)
      const int64_t tiles = int64_t((a->N + 2 * kGemmRows - 1) / (2 * kGemmRows)) * ((a->M + bt - 1) / bt);
      for (int split = 1; split <= std::min(4, slices); split *= 2) {
        if (rows ? 2 * split <= std::min((a->hints & 7) + 1, std::min(4, slices)) : split > 1 && tiles * split > 64) continue;
        if (rows && split > (a->hints & 7) + 1) break;
        plan_pair(pl, a->M, bt, split, sms, most);
        keep(pl);
      }
    }
  }
  if (best.cost == 0) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: hints %d leave no kernel", a->hints);
  pl = best;
  const int64_t blocks = int64_t(pl.p.n_tiles) * pl.p.m_tiles * pl.p.split;
  if (blocks > 0x7fffffff) return fail(MGV_STATUS_UNSUPPORTED, "gemm_i8: too many tiles (M=%lld N=%d)", (long long)a->M, a->N);
  return MGV_STATUS_OK;
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

  if ((st = plan(pl, a, sms, most)) != MGV_STATUS_OK) return st;
  if ((st = encode_rows(&p.w_map, a->weights, a->N, a->K, a->ldw, kGemmRows)) != MGV_STATUS_OK) return st;
  if (pl.pair && p.halved < p.n_tiles * p.m_tiles && (st = encode_rows(&p.x_half_map, a->x, a->M, a->K, a->ldx, p.bt / 4)) != MGV_STATUS_OK) return st;
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
