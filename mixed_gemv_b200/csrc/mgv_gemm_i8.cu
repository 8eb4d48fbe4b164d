// int8 matrix product with a scale for each row and each output feature: entry points, plan and kernel.
#include <cuda_bf16.h>

#include <new>

#include "mgv_common.cuh"

namespace mgv {

struct GemmI8Params {
  const int8_t *x, *w;
  const float *x_scale;
  const void *w_scale, *bias;
  void *out;
  int64_t ldx, ldw, ldd;
  int M, N, K, out_dtype, scale_dtype, flags;
};

__device__ __forceinline__ float load_as_float(const void *p, int64_t i, int dtype) {
  if (dtype == MGV_DTYPE_F16) return __half2float(static_cast<const __half *>(p)[i]);
  if (dtype == MGV_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  return static_cast<const float *>(p)[i];
}

__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }

constexpr int kSimpleTile = 64, kSimpleK = 16;  // 64 x 64 outputs, 16 words (64 values) of K at a time

// 64 x 64 outputs per block through shared memory, four-way int8 dot products.
__global__ void __launch_bounds__(256) gemm_i8_simple_kernel(GemmI8Params p) {
  __shared__ int xs[kSimpleK][kSimpleTile + 1], ws[kSimpleK][kSimpleTile + 1];
  const int n0 = blockIdx.x * kSimpleTile, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t m0 = int64_t(blockIdx.y) * kSimpleTile; m0 < p.M; m0 += int64_t(gridDim.y) * kSimpleTile) {
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 4 * kSimpleK) {
      for (int i = threadIdx.x; i < kSimpleTile * kSimpleK; i += 256) {
        const int row = i / kSimpleK, kw = i % kSimpleK, k = k0 + 4 * kw;
        int xv = 0, wv = 0;
        for (int b = 0; b < 4; ++b) {
          if (k + b >= p.K) break;
          if (m0 + row < p.M) xv |= int(uint8_t(p.x[(m0 + row) * p.ldx + k + b])) << (8 * b);
          if (n0 + row < p.N) wv |= int(uint8_t(p.w[int64_t(n0 + row) * p.ldw + k + b])) << (8 * b);
        }
        xs[kw][row] = xv;
        ws[kw][row] = wv;
      }
      __syncthreads();
      for (int kw = 0; kw < kSimpleK; ++kw)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(xs[kw][ty * 4 + i], ws[kw][tx * 4 + j], acc[i][j]);
      __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + ty * 4 + i;
      if (m >= p.M) continue;
      const float sx = p.x_scale[m];
      float v[4];
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx * 4 + j;
        v[j] = 0.0f;
        if (n >= p.N) continue;
        v[j] = float(acc[i][j]) * (sx * load_as_float(p.w_scale, n, p.scale_dtype));
        if (p.bias) v[j] += load_as_float(p.bias, n, p.out_dtype);
        if (p.flags & MGV_FLAG_ACT_RELU) v[j] = v[j] < 0.0f ? 0.0f : v[j];
        if (p.flags & MGV_FLAG_ACT_SILU) v[j] = silu(v[j]);
      }
      const bool gated = p.flags & MGV_FLAG_GATED_SILU;
      for (int j = 0; j < 4; j += gated ? 2 : 1) {
        const int n = n0 + tx * 4 + j;
        if (n >= p.N) continue;
        const float y = gated ? silu(v[j]) * v[j + 1] : v[j];
        const int64_t at = m * p.ldd + (gated ? n / 2 : n);
        if (p.out_dtype == MGV_DTYPE_F16) static_cast<__half *>(p.out)[at] = __float2half_rn(y);
        else static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(y);
      }
    }
  }
}

static mgv_status check_args(const mgv_gemm_i8_args *a) {
  if (!a || a->struct_size != int32_t(sizeof(*a))) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: args null or of another version");
  if (a->M < 0 || a->M > 0x7fffffff) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: M=%lld outside 0..2^31-1", (long long)a->M);
  if (a->N < 1) return fail(MGV_STATUS_INVALID_ARGUMENT, "gemm_i8: N=%d must be at least 1", a->N);
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

struct mgv_gemm_i8_plan {
  GemmI8Params p;
  int device = 0;
};

static mgv_status prepare(const mgv_gemm_i8_args *a, mgv_gemm_i8_plan &pl) {
  const mgv_status st = check_args(a);
  if (st != MGV_STATUS_OK) return st;
  MGV_CUDA_TRY(cudaGetDevice(&pl.device));
  pl.p = {static_cast<const int8_t *>(a->x), static_cast<const int8_t *>(a->weights), static_cast<const float *>(a->x_scale),
          a->weight_scale, a->bias, a->out, a->ldx, a->ldw, a->ldd, int(a->M), a->N, a->K, a->out_dtype, a->scale_dtype, a->flags};
  return MGV_STATUS_OK;
}

static mgv_status launch(const mgv_gemm_i8_plan &pl, cudaStream_t s) {
  if (pl.p.M == 0) return MGV_STATUS_OK;
  cudaLaunchConfig_t cfg = {};
  const int64_t mt = (int64_t(pl.p.M) + kSimpleTile - 1) / kSimpleTile;
  cfg.gridDim = dim3((unsigned(pl.p.N) + kSimpleTile - 1) / kSimpleTile, unsigned(mt < 65535 ? mt : 65535));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (pl.p.flags & MGV_FLAG_PDL) ? 1 : 0;
  MGV_CUDA_TRY(cudaLaunchKernelEx(&cfg, gemm_i8_simple_kernel, pl.p));
  return MGV_STATUS_OK;
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
