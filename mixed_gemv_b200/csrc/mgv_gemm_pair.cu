// int8 matrix product, the kernel of block pairs: prompts.
#include "mgv_gemm_parts.cuh"

namespace mgv {

// Tiles are ordered so that the pairs at work at one time share operands in L2: kGemmBand tiles of
// activation rows against one tile of features, then the next features, then the next band.
constexpr int kGemmBand = 8;

struct TileAt {
  int n0, m0, rows;
};
// The item of that number in the order of work: a tile, or half the rows of one.
__device__ __forceinline__ TileAt tile_at(const GemmI8Params &p, uint32_t item) {
  const uint32_t whole = uint32_t(p.halved), tile = item < whole ? item : whole + (item - whole) / 2;
  const uint32_t per_band = uint32_t(kGemmBand) * p.n_tiles, band = tile / per_band, in = tile % per_band;
  const uint32_t height = min(uint32_t(kGemmBand), uint32_t(p.m_tiles) - band * kGemmBand);
  const int n0 = int(in / height) * 2 * kGemmRows, m0 = int(band * kGemmBand + in % height) * p.bt;
  if (item < whole) return {n0, m0, p.bt};
  return {n0, m0 + int((item - whole) % 2) * (p.bt / 2), p.bt / 2};
}

// Persistent: a pair of blocks (two SMs) per tile of 256 output features x p.bt activation rows.  Each
// block holds 128 of the features and copies half of the rows; one thread of the first block issues
// matrix instructions for both.  Two accumulators in tensor memory: the epilogue of a tile runs
// beside the next tile's products.  Tiles too few for the GPU are shared by the p.split pairs of a cluster.  Where the last round of tiles would leave half of the pairs or more without
// one, its tiles are halved: 2048 x 8192 features at 256 rows are 3.46 tiles to a pair, in 3.5 rounds instead of 4.
// Bound by the matrix unit (508 cycles for a slice of a 256-row tile: four instructions of 127) and, over more than a
// few milliseconds, by the power limit: B200, 4096 x 4096 x 4096 43.9 us (3.13 POP/s at 1.9 GHz), 4096 x 57344 x 8192 gated
// 1.28 ms (3.00 POP/s at 1.2 - 1.3 GHz); 256 x 4096 x 11008 as 32 tiles of two pairs each 15.2 us, one pair each 17.4.
template <int ACT, bool BF16>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_i8_pair_kernel(const __grid_constant__ GemmI8Params p) {
  extern __shared__ uint8_t dynamic[];
  __shared__ GemmPairShared sh;
  const uint32_t ring = (smem_u32(dynamic) + 1023) & ~1023u;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  // A cluster is a pair, or the p.split pairs that share a tile's K range; `lead` is the pair's first block.
  const uint32_t cluster_at = cluster_rank(), rank = cluster_at % 2, lead = cluster_at - rank, part = cluster_at / 2;
  const uint32_t pairs = gridDim.x / (2 * p.split), pair = blockIdx.x / (2 * p.split);
  const uint32_t items = 2 * uint32_t(p.n_tiles) * uint32_t(p.m_tiles) - uint32_t(p.halved);
  const int all_slices = (p.K + kGemmK - 1) / kGemmK, first = int(int64_t(all_slices) * part / p.split);
  const int slices = int(int64_t(all_slices) * (part + 1) / p.split) - first;
  const uint32_t slot_bytes = kGemmABytes + p.bt / 2 * kGemmK;  // of whole tiles

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) bar_init(smem_u32(&sh.full[i]), 1), bar_init(smem_u32(&sh.empty[i]), 1);
    for (int i = 0; i < 2; ++i) bar_init(smem_u32(&sh.ready[i]), 1), bar_init(smem_u32(&sh.drained[i]), 2 * kGemmEpilogue / 32);
    bar_init(smem_u32(&sh.sums), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n\tfence.proxy.async;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tmem_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_sync();
  tmem_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, sh.tmem_base, 0);
  bool good = true;

  if (warp == 0) {
    // both blocks' copies count on the first block's barriers; each block waits on its own for a free slot
    const bool one = elect_one();
    TileAt at = tile_at(p, pair);
    const int ahead = min(slices, p.stages);
    if (one) {
      for (int i = 0; i < ahead; ++i) {
        if (rank == 0) bar_expect(smem_u32(&sh.full[i]), 2 * kGemmABytes + at.rows * kGemmK);
        box_load_pair(ring + i * slot_bytes, &p.w_map, (first + i) * kGemmK, at.n0 + int(rank) * kGemmRows, in_block(smem_u32(&sh.full[i]), lead));
      }
    }
    // as in the kernel of single blocks: dependents start behind the wait and the allocation
    asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;\n\tfence.proxy.async.global;" ::: "memory");
    if (one)
      for (int i = 0; i < ahead; ++i)
        box_load_pair(ring + i * slot_bytes + kGemmABytes, at.rows == p.bt ? &p.x_map : &p.x_half_map, (first + i) * kGemmK, at.m0 + int(rank) * at.rows / 2, in_block(smem_u32(&sh.full[i]), lead));
    int slot = ahead % p.stages;
    uint32_t issued = ahead, phase = 0;  // phase: of `empty` once the ring is full
    bool ok = true;
    for (uint32_t tile = pair; tile < items && ok; tile += pairs) {
      at = tile_at(p, tile);
      for (int i = tile == pair ? ahead : 0; i < slices; ++i) {
        if (issued >= uint32_t(p.stages)) {
          ok = bar_wait(smem_u32(&sh.empty[slot]), phase, p.err);
          if (!ok) break;
          if (slot == p.stages - 1) phase ^= 1;
        }
        if (one) {
          const uint32_t bar = in_block(smem_u32(&sh.full[slot]), lead), dst = ring + slot * slot_bytes;
          if (rank == 0) bar_expect(smem_u32(&sh.full[slot]), 2 * kGemmABytes + at.rows * kGemmK);
          box_load_pair(dst, &p.w_map, (first + i) * kGemmK, at.n0 + int(rank) * kGemmRows, bar);
          box_load_pair(dst + kGemmABytes, at.rows == p.bt ? &p.x_map : &p.x_half_map, (first + i) * kGemmK, at.m0 + int(rank) * at.rows / 2, bar);
        }
        if (++slot == p.stages) slot = 0;
        ++issued;
      }
    }
    // The blocks end only when their slots have been read (and so filled): every slot's last release is
    // waited for.  If the matrix warp gave up, the first block waits for the copies of both instead.
    for (uint32_t i = issued > uint32_t(p.stages) ? issued - p.stages : 0; i < issued && ok; ++i)
      ok = bar_wait(smem_u32(&sh.empty[i % p.stages]), (i / p.stages) & 1, p.err);
    if (!ok && rank == 0)
      for (uint32_t i = issued > uint32_t(p.stages) ? issued - p.stages : 0; i < issued; ++i)
        if (!bar_wait(smem_u32(&sh.full[i % p.stages]), (i / p.stages) & 1, p.err)) break;
  } else if (warp == 1 && rank == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // its limited waits count from the previous kernel's end
    const bool one = elect_one();
    int slot = 0;
    uint32_t phase = 0, turn = 0;
    bool ok = true;
    for (uint32_t tile = pair; tile < items && ok; tile += pairs, ++turn) {
      const uint32_t buf = turn & 1, acc = tmem + buf * (p.tmem_cols / 2), idesc = tile < uint32_t(p.halved) ? p.idesc : p.half_idesc;
      if (turn >= 2) ok = bar_wait<true>(smem_u32(&sh.drained[buf]), ((turn >> 1) - 1) & 1, p.err);
      tmem_fence_after();
      for (int i = 0; i < slices && ok; ++i) {
        ok = bar_wait(smem_u32(&sh.full[slot]), phase, p.err);
        if (!ok) break;
        tmem_fence_after();
        const uint64_t a = operand_desc(ring + slot * slot_bytes), b = operand_desc(ring + slot * slot_bytes + kGemmABytes);
        if (one) {
#pragma unroll
          for (int k = 0; k < kGemmK / 32; ++k) multiply_add<2>(acc, a + 2 * k, b + 2 * k, idesc, i + k > 0);
          commit_pair(smem_u32(&sh.empty[slot]), lead);
        }
        __syncwarp();
        if (++slot == p.stages) slot = 0, phase ^= 1;
      }
      if (ok && one) commit_pair(smem_u32(&sh.ready[buf]), lead);
      __syncwarp();
    }
  } else if (warp >= 2) {
    const int quarter = warp % 4, half = warp >= 6, row = int(rank) * kGemmRows + quarter * 32 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint32_t turn = 0;
    for (uint32_t tile = pair; tile < items; tile += pairs, ++turn) {
      const TileAt at = tile_at(p, tile);
      const uint32_t buf = turn & 1, lanes = tmem + buf * (p.tmem_cols / 2) + (uint32_t(quarter * 32) << 16);
      const Feature f = load_feature<BF16>(p, at.n0 + row);
      // the buffer's last readers have passed the barrier of the tile between
      if (const int i = threadIdx.x - 64; i < at.rows) sh.x_scale[buf][i] = at.m0 + i < p.M ? p.x_scale[at.m0 + i] : 0.0f;
      asm volatile("bar.sync 1, %0;" ::"n"(kGemmEpilogue) : "memory");
      good = good && bar_wait(smem_u32(&sh.ready[buf]), (turn >> 1) & 1, p.err);
      if (!good) continue;  // on to the barrier that the other warps wait at
      tmem_fence_after();
      const int columns = min(at.rows, p.M - at.m0);
      if (p.split > 1) break;  // one tile, finished below
      finish_columns<ACT, BF16>(p, f, lanes, at.m0, half * 16, columns, sh.x_scale[buf]);
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) arrive_in_block(in_block(smem_u32(&sh.drained[buf]), lead));
    }
  }
  if (p.split > 1) {
    // Pairs of a cluster share the tile: block by block, those of the same features send each other their sums.  Part
    // r finishes the 16-column groups r, r + split, ...; what the others send of them goes into the ring, which is
    // free once all copies of the cluster have landed and been read.
    const TileAt at = tile_at(p, pair);
    const int groups = (min(at.rows, p.M - at.m0) + 15) / 16, mine = (groups - int(part) + p.split - 1) / p.split;
    constexpr int kGroup = 4 * kQuadBytes;
    if (threadIdx.x == 0 && mine > 0) bar_expect(smem_u32(&sh.sums), mine * (p.split - 1) * kGroup);
    cluster_sync();
    if (warp >= 2 && good) {
      const int quarter = warp % 4, half = warp >= 6, row = quarter * 32 + lane;
      const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16), ours = ring + row * 16;
      for (int g = half; g < groups; g += 2) {
        const int owner = g % p.split;
        if (owner == int(part)) continue;
        int v[16];
        __syncwarp();
        tmem_load16(lanes + 16 * g, v);
        tmem_wait(v);
        const int at_group = g / p.split * (p.split - 1) + int(part) - (int(part) > owner ? 1 : 0);
        const uint32_t to = in_block(ours + at_group * kGroup, 2 * owner + rank), bar = in_block(smem_u32(&sh.sums), 2 * owner + rank);
#pragma unroll
        for (int i = 0; i < 4; ++i) send16(to + i * kQuadBytes, bar, v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
      const Feature f = load_feature<BF16>(p, at.n0 + int(rank) * kGemmRows + row);
      if (mine > 0 && bar_wait<true>(smem_u32(&sh.sums), 0, p.err)) {
        for (int j = half; j < mine; j += 2) {
          const int g = j * p.split + int(part);
          int v[16];
          __syncwarp();
          tmem_load16(lanes + 16 * g, v);
          tmem_wait(v);
          for (int s = 0; s < p.split - 1; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int4 u = load_shared(ours + (j * (p.split - 1) + s) * kGroup + i * kQuadBytes);
              v[4 * i] += u.x, v[4 * i + 1] += u.y, v[4 * i + 2] += u.z, v[4 * i + 3] += u.w;
            }
          }
          finish<ACT, BF16>(p, f, at.m0 + 16 * g, p.M - at.m0 - 16 * g, v, sh.x_scale[0] + 16 * g);
        }
      }
      tmem_fence_before();
    }
  }
  __syncwarp();
  cluster_sync();
  if (warp == 1) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
  }
}

template <int ACT>
static mgv_status launch_act(const GemmI8Plan &pl, cudaStream_t s) {
  return pl.bf16 ? launch_gemm<gemm_i8_pair_kernel<ACT, true>>(pl, s) : launch_gemm<gemm_i8_pair_kernel<ACT, false>>(pl, s);
}

mgv_status launch_gemm_pair(const GemmI8Plan &pl, cudaStream_t s) {
  switch (pl.act) {
    case kActRelu: return launch_act<kActRelu>(pl, s);
    case kActSilu: return launch_act<kActSilu>(pl, s);
    case kActGated: return launch_act<kActGated>(pl, s);
    default: return launch_act<kActNone>(pl, s);
  }
}

}  // namespace mgv
