// Rows of 16-bit activations into int8 with one scale each, plain and behind a root-mean-square
// norm with the residual's addition, and the way back.
#include <cuda_bf16.h>

#include <cfloat>
#include <cmath>

#include "mgv_common.cuh"

namespace mgv {

struct RowParams {
  const void *x, *residual, *weight;
  void *residual_out;
  int8_t *q;
  float *scale;
  int64_t M, ldx, ldr, ldro, ldq;
  int K;
  float eps;
};

constexpr int kRowThreads = 256;

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename V>
__device__ __forceinline__ V block_reduce(V v, V (*op)(V, V), V *buf) {
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(~0u, v, o));
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < kRowThreads / 32; ++i) v = op(v, buf[i]);
  __syncthreads();
  return v;
}

// One block per row, two passes.  Double precision throughout: right for every finite row,
// whatever its magnitude.
template <typename T, bool NORM>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(RowParams p) {
  __shared__ double buf[kRowThreads / 32];
  const int64_t m = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + m * p.ldx;
  const T *r = p.residual ? static_cast<const T *>(p.residual) + m * p.ldr : nullptr;
  T *ro = p.residual ? static_cast<T *>(p.residual_out) + m * p.ldro : nullptr;
  const T *w = static_cast<const T *>(p.weight);
  int8_t *q = p.q + m * p.ldq;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double ss = 0, top = 0;
  bool bad = false;
  for (int k = threadIdx.x; k < p.K; k += kRowThreads) {
    float h = to_f(x[k]);
    if (NORM && r) {
      const T t = from_f<T>(h + to_f(r[k]));
      ro[k] = t;
      h = to_f(t);
    }
    const double v = NORM ? double(h) * double(to_f(w[k])) : double(h);
    bad |= !(fabs(v) <= DBL_MAX);
    ss += double(h) * double(h);
    top = fmax(top, fabs(v));
  }
  auto add = [](double a, double b) { return a + b; };
  auto larger = [](double a, double b) { return fmax(a, b); };
  if (NORM) ss = block_reduce<double>(ss, add, buf);
  top = block_reduce<double>(top, larger, buf);
  bad = block_reduce<double>(bad ? 1.0 : 0.0, larger, buf) != 0.0;
  const double inv = top > 0 ? 127.0 / top : 0.0;
  if (threadIdx.x == 0) {
    double s = top / 127.0;
    if (NORM && top > 0) s /= sqrt(ss / p.K + double(p.eps));
    p.scale[m] = bad ? NAN : float(s);
  }
  const T *again = NORM && r ? ro : x;
  for (int k = threadIdx.x; k < p.K; k += kRowThreads) {
    const double v = NORM ? double(to_f(again[k])) * double(to_f(w[k])) : double(to_f(again[k]));
    q[k] = bad ? 0 : int8_t(rint(v * inv));
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) back_kernel(T *out, const int8_t *q, const float *scale, int K, int64_t ldo, int64_t ldq) {
  const int64_t m = blockIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float s = scale[m];
  for (int k = threadIdx.x; k < K; k += kRowThreads) out[m * ldo + k] = from_f<T>(float(q[m * ldq + k]) * s);
}

template <typename... P, typename... A>
static mgv_status launch_rows(void (*kern)(P...), int64_t rows, int flags, cudaStream_t s, A... a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & MGV_FLAG_PDL) ? 1 : 0;
  MGV_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a...));
  return MGV_STATUS_OK;
}

// What the three entry points check alike; `what` names the call in the message.
static mgv_status check_rows(const char *what, int dtype, int64_t M, int32_t K, int flags) {
  if (dtype != MGV_DTYPE_F16 && dtype != MGV_DTYPE_BF16)
    return fail(MGV_STATUS_UNSUPPORTED, "%s: dtype %d is neither F16 nor BF16", what, dtype);
  if (M < 0 || M > 0x7fffffff) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: M=%lld outside 0..2^31-1", what, (long long)M);
  if (K < 1) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: K=%d must be at least 1", what, K);
  if (flags & ~MGV_FLAG_PDL) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: only MGV_FLAG_PDL applies (flags %d)", what, flags);
  return MGV_STATUS_OK;
}

static mgv_status check_operand(const char *what, const char *name, const void *ptr, int64_t ld, int32_t K, int elem) {
  if (!ptr) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: %s is null", what, name);
  if (ld < K) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: leading dimension %lld of %s is below K=%d", what, (long long)ld, name, K);
  if (ld > (int64_t(1) << 40)) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: leading dimension of %s too large", what, name);
  if (reinterpret_cast<uintptr_t>(ptr) % elem) return fail(MGV_STATUS_MISALIGNED, "%s: %s must be %d-byte aligned", what, name, elem);
  return MGV_STATUS_OK;
}

#define MGV_CHECK(expr)                    \
  do {                                     \
    const mgv_status st__ = (expr);        \
    if (st__ != MGV_STATUS_OK) return st__; \
  } while (0)

}  // namespace mgv

using namespace mgv;

extern "C" mgv_status mgv_quantize_rows(void *q, void *scale, const void *x, int dtype, int64_t M, int32_t K, int64_t ldq,
                                        int64_t ldx, int flags, mgv_stream_t s) {
  MGV_CHECK(check_rows("quantize_rows", dtype, M, K, flags));
  if (M == 0) return MGV_STATUS_OK;
  MGV_CHECK(check_operand("quantize_rows", "x", x, ldx, K, 2));
  MGV_CHECK(check_operand("quantize_rows", "q", q, ldq, K, 1));
  MGV_CHECK(check_operand("quantize_rows", "scale", scale, K, K, 4));
  RowParams p = {};
  p.x = x; p.q = static_cast<int8_t *>(q); p.scale = static_cast<float *>(scale);
  p.M = M; p.K = K; p.ldx = ldx; p.ldq = ldq;
  return dtype == MGV_DTYPE_F16 ? launch_rows(rows_kernel<__half, false>, M, flags, s, p)
                                : launch_rows(rows_kernel<__nv_bfloat16, false>, M, flags, s, p);
}

extern "C" mgv_status mgv_dequantize_rows(void *out, const void *q, const void *scale, int dtype, int64_t M, int32_t K,
                                          int64_t ldo, int64_t ldq, int flags, mgv_stream_t s) {
  MGV_CHECK(check_rows("dequantize_rows", dtype, M, K, flags));
  if (M == 0) return MGV_STATUS_OK;
  MGV_CHECK(check_operand("dequantize_rows", "out", out, ldo, K, 2));
  MGV_CHECK(check_operand("dequantize_rows", "q", q, ldq, K, 1));
  MGV_CHECK(check_operand("dequantize_rows", "scale", scale, K, K, 4));
  const int8_t *qp = static_cast<const int8_t *>(q);
  const float *sp = static_cast<const float *>(scale);
  return dtype == MGV_DTYPE_F16 ? launch_rows(back_kernel<__half>, M, flags, s, static_cast<__half *>(out), qp, sp, K, ldo, ldq)
                                : launch_rows(back_kernel<__nv_bfloat16>, M, flags, s, static_cast<__nv_bfloat16 *>(out), qp, sp, K, ldo, ldq);
}

extern "C" void mgv_rmsnorm_args_init(mgv_rmsnorm_args *a) {
  if (!a) return;
  *a = mgv_rmsnorm_args{};
  a->struct_size = int32_t(sizeof(*a));
  a->eps = 1e-5f;
}

extern "C" mgv_status mgv_rmsnorm_quantize(const mgv_rmsnorm_args *a, mgv_stream_t s) {
  if (!a || a->struct_size != int32_t(sizeof(*a))) return fail(MGV_STATUS_INVALID_ARGUMENT, "rmsnorm_quantize: args null or of another version");
  MGV_CHECK(check_rows("rmsnorm_quantize", a->dtype, a->M, a->K, a->flags));
  if (!(a->eps >= 0.0f) || !std::isfinite(a->eps)) return fail(MGV_STATUS_INVALID_ARGUMENT, "rmsnorm_quantize: eps must be finite and not negative");
  if ((a->residual == nullptr) != (a->residual_out == nullptr))
    return fail(MGV_STATUS_INVALID_ARGUMENT, "rmsnorm_quantize: residual and residual_out are given together or not at all");
  if (a->M == 0) return MGV_STATUS_OK;
  MGV_CHECK(check_operand("rmsnorm_quantize", "x", a->x, a->ldx, a->K, 2));
  MGV_CHECK(check_operand("rmsnorm_quantize", "weight", a->weight, a->K, a->K, 2));
  MGV_CHECK(check_operand("rmsnorm_quantize", "q", a->q, a->ldq, a->K, 1));
  MGV_CHECK(check_operand("rmsnorm_quantize", "scale", a->scale, a->K, a->K, 4));
  if (a->residual) {
    MGV_CHECK(check_operand("rmsnorm_quantize", "residual", a->residual, a->ldr, a->K, 2));
    MGV_CHECK(check_operand("rmsnorm_quantize", "residual_out", a->residual_out, a->ldro, a->K, 2));
    if ((a->residual_out == a->residual && a->M > 1 && a->ldro != a->ldr) || (a->residual_out == a->x && a->M > 1 && a->ldro != a->ldx))
      return fail(MGV_STATUS_INVALID_ARGUMENT, "rmsnorm_quantize: residual_out in place needs the leading dimension of what it replaces");
  }
  RowParams p = {};
  p.x = a->x; p.residual = a->residual; p.weight = a->weight; p.residual_out = a->residual_out;
  p.q = static_cast<int8_t *>(a->q); p.scale = static_cast<float *>(a->scale);
  p.M = a->M; p.K = a->K; p.ldx = a->ldx; p.ldr = a->ldr; p.ldro = a->ldro; p.ldq = a->ldq; p.eps = a->eps;
  return a->dtype == MGV_DTYPE_F16 ? launch_rows(rows_kernel<__half, true>, a->M, a->flags, s, p)
                                   : launch_rows(rows_kernel<__nv_bfloat16, true>, a->M, a->flags, s, p);
}
