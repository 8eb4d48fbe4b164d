// Rows of 16-bit activations into int8 with one scale each, plain and behind a root-mean-square
// norm with the residual's addition, and the way back.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "mgv_common.cuh"

namespace mgv {

// Waits for the stream's previous kernel (dependent launches), and only then lets the next one start: so what
// follows these kernels runs beside its direct predecessor only, and what it touches before its own wait only
// has to be older than that.  (Behind a kernel that lets its dependents start before its own wait, as the GEMV and the
// wait for partials do, it has to be older than what that one waits for too.)
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

struct RowParams {
  const void *x, *residual, *weight;
  void *residual_out;
  int8_t *q;
  float *scale;
  int64_t M, ldx, ldr, ldro, ldq;
  int K;
  float eps;
};

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two values of a 32-bit word, and back (each rounded to T).
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// What a thread holds of a row at a time: eight neighbouring 16-bit values in four words (V = 8, one
// 16-byte access), or one value, the low half of a word whose high half is zero (V = 1).
template <int V>
struct Piece {
  uint32_t u[V == 8 ? 4 : 1];
};
// Of a piece at `at`, `n` values belong to the row: what is behind its end is neither read (it counts
// as zero) nor written.
template <int V>
__device__ __forceinline__ Piece<V> load_piece(const void *row, int k, int n) {
  const uint16_t *at = static_cast<const uint16_t *>(row) + k;
  Piece<V> r;
  if constexpr (V == 1) {
    r.u[0] = *at;
  } else if (n >= 8) {
    const uint4 v = *reinterpret_cast<const uint4 *>(at);
    r.u[0] = v.x, r.u[1] = v.y, r.u[2] = v.z, r.u[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.u[j] = (2 * j < n ? uint32_t(at[2 * j]) : 0u) | (2 * j + 1 < n ? uint32_t(at[2 * j + 1]) << 16 : 0u);
  }
  return r;
}
template <int V>
__device__ __forceinline__ void store_piece(void *row, int k, const Piece<V> &v, int n) {
  uint16_t *at = static_cast<uint16_t *>(row) + k;
  if constexpr (V == 1) {
    *at = uint16_t(v.u[0]);
  } else if (n >= 8) {
    *reinterpret_cast<uint4 *>(at) = make_uint4(v.u[0], v.u[1], v.u[2], v.u[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) at[j] = uint16_t(v.u[j / 2] >> (j % 2 * 16));
  }
}

// Four fp32 values in [-127, 127], each added to 1.5 * 2^23 (so rounded to an integer, ties to even):
// the low bytes are the integers.
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const uint32_t ab = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
  const uint32_t cd = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}
constexpr float kRoundMagic = 12582912.0f;

__device__ __forceinline__ double block_reduce_double(double v, bool largest, double *buf) {
  for (int o = 16; o; o >>= 1) {
    const double w = __shfl_xor_sync(~0u, v, o);
    v = largest ? fmax(v, w) : v + w;
  }
  __syncthreads();
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < int(blockDim.x / 32); ++i) v = largest ? fmax(v, buf[i]) : v + buf[i];
  return v;
}

// One row in double precision, by `step` threads from `t`: right for whatever magnitude its values
// have.  The kernels come here for a row that has no finite fp32 statistics (an infinity or a NaN
// among the values, squares or products beyond fp32, or all of them near its smallest), and re-read
// the row, with the residual already added.
template <typename T, bool NORM, bool WARP_ROW>
__device__ __noinline__ void row_in_double(const RowParams &p, int64_t m, int t, int step, double *buf) {
  const T *h = p.residual ? static_cast<const T *>(p.residual_out) + m * p.ldro : static_cast<const T *>(p.x) + m * p.ldx;
  const T *w = static_cast<const T *>(p.weight);
  int8_t *q = p.q + m * p.ldq;
  if (WARP_ROW) __syncwarp();
  else __syncthreads();  // the row's threads have stored their part of residual_out, and read the mark in scale
  double ss = 0, top = 0, bad = 0;
  for (int k = t; k < p.K; k += step) {
    const double v = to_f(h[k]), y = NORM ? v * double(to_f(w[k])) : v;
    if (!(fabs(y) <= DBL_MAX)) bad = 1;
    ss += v * v;
    top = fmax(top, fabs(y));
  }
  if (WARP_ROW) {
    for (int o = 16; o; o >>= 1) {
      ss += __shfl_xor_sync(~0u, ss, o);
      top = fmax(top, __shfl_xor_sync(~0u, top, o));
      bad = fmax(bad, __shfl_xor_sync(~0u, bad, o));
    }
  } else {
    ss = block_reduce_double(ss, false, buf);
    top = block_reduce_double(top, true, buf);
    bad = block_reduce_double(bad, true, buf);
  }
  if (t == 0) {
    double s = top / 127.0;
    if (NORM && top > 0) s /= sqrt(ss / p.K + double(p.eps));
    p.scale[m] = bad != 0 ? NAN : float(s);
  }
  for (int k = t; k < p.K; k += step) {
    const double v = to_f(h[k]), y = NORM ? v * double(to_f(w[k])) : v;
    q[k] = bad != 0 || top == 0 ? 0 : int8_t(rint(y * 127.0 / top));  // y has 24 bits at most: the product is exact, and so is a tie
  }
}

// Statistics of a row: the sum of squares of h, and the largest |h w| as the bits of a float (whose
// order as integers is that of the magnitudes, with infinities and NaN above every number).
struct RowStats {
  float ss;
  uint32_t top;
};
// The fp32 statistics serve: squares, products and their quotients are numbers well inside fp32.
template <bool NORM>
__device__ __forceinline__ bool row_is_tame(const RowStats &s, float mean) {
  const bool sum_ok = !NORM || (mean >= 1e-30f && mean <= FLT_MAX);
  return sum_ok && (s.top == 0 || (s.top >= __float_as_uint(1e-30f) && s.top < 0x7f800000u));
}
// Products, fused products and sums, and sums of two fp32 values at a time.
__device__ __forceinline__ uint64_t both(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 each(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return each(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(both(a)), "l"(both(b)), "l"(both(c)));
  return each(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return each(r);
}

// y * 127 / top as an integer, ties to even, in the low bits of the result.
//
// In two terms: 127 / top = inv + rest, and the quotient is rounded to fp32 once, out of more bits than fp32 has, and then
// to the integer.  A tie is a number of fp32, so the first rounding returns it and leaves the second to decide.  A
// quotient that is none stays off it: with a y of b bits it is 1 / (254 * 2^b) of itself away from the next tie, more than
// half a step of fp32 for b <= 16.  (Only the products of fp16 norms have more bits, up to 22: of those some within 2^-24
// of a tie are taken for one.)
//
// In one: y * inv, rounded to the integer at once, with the error of inv deciding at a tie.  Without a weight y and top have
// the 11 or 8 bits of their type, and no quotient but a tie is nearer to one than the error is large.  A tie is y / top = (2n + 1) / 254,
// so where 127 does not divide top's mantissa only y = +-top / 2 is one, 63.5, which goes to 64: as it does with
// an inv that is not below 127 / top.  Rows whose top has 127 in its mantissa (one in 127 of fp16 rows; of bf16 rows their
// inv is exact) take two terms.  (Tried on every pair of mantissas.)
//
// B200, 4096 x 8192 bf16: quantisation 16.8 us in one term, 18.3 in two (19.1 with one value an instruction); the norm with
// residual, in two, 38.7 (40.6).
struct RowFactors {
  float scale, inv, rest;  // inv + rest has 40 bits and more (28 for a top near fp32's largest, where rest is subnormal)
  bool two;
};
template <bool NORM>
__device__ __forceinline__ RowFactors row_factors(const RowStats &s, float mean) {
  const float top = __uint_as_float(s.top);
  RowFactors f;
  f.scale = top / 127.0f;  // first: the largest y itself may be beyond fp32
  if (NORM) f.scale *= rsqrtf(mean);
  f.inv = s.top ? 127.0f / top : 0.0f;
  const float over = fmaf(-f.inv, top, 127.0f);  // exact
  f.rest = over * (f.inv * (1.0f / 127.0f));
  f.two = NORM || (over != 0.0f && (s.top & 0x7fffffu | 0x800000u) % 127 == 0);
  if (!f.two && over > 0.0f && s.top) f.inv = __uint_as_float(__float_as_uint(f.inv) + 1);
  return f;
}
template <bool TWO>
__device__ __forceinline__ float2 level2(float2 y, const RowFactors &f) {
  const float2 inv = make_float2(f.inv, f.inv), magic = make_float2(kRoundMagic, kRoundMagic);
  return TWO ? add2(fma2(y, inv, mul2(y, make_float2(f.rest, f.rest))), magic) : fma2(y, inv, magic);
}
template <bool TWO>
__device__ __forceinline__ float level(float y, const RowFactors &f) {
  return TWO ? fmaf(y, f.inv, y * f.rest) + kRoundMagic : fmaf(y, f.inv, kRoundMagic);
}
__device__ __forceinline__ RowStats warp_stats(RowStats s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s.ss += __shfl_xor_sync(~0u, s.ss, o);
  s.top = __reduce_max_sync(~0u, s.top);
  return s;
}
__device__ __forceinline__ RowStats block_stats(RowStats s, RowStats *buf) {
  s = warp_stats(s);
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = s;
  __syncthreads();
  const int warps = blockDim.x / 32, lane = threadIdx.x % 32;
  RowStats r = {0.0f, 0u};
  if (lane < warps) r = buf[lane];
  return warp_stats(r);
}

constexpr int kLongThreads = 512;

// Marks, in its place in `scale`, a row that is left for row_in_double.
constexpr float kLeft = -1.0f;

// The rows in one pass.  A row's h stays in registers, 16 bits a value, between the statistics and the
// quantisation, and one reduction serves both: with y = h w r, r = 1 / sqrt(mean + eps), the scale is
// r max|h w| / 127 and q = h w 127 / max|h w|, in which r does not occur.  The sum of squares, the
// largest value and the scale are fp32.  A block takes a row (a warp, for short rows) with NV pieces of V
// values to a thread, then the next one; the norm's weights stay in registers over its rows where there is room.
// Bound by HBM: B200, 4096 x 8192 bf16 with residual 38.7 us (6.1 TB/s, 0.93 of the copy bandwidth), without norm 16.8 us.
// Two forms spill, at the 64 registers of a 1024-thread block: the norm with eight pieces a thread (44 bytes) and the norm value by value (16).
template <typename T, bool NORM, int V, int NV, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 128 : 1024, WARP_ROW ? 6 : 1) rows_kernel(const __grid_constant__ RowParams p) {
  constexpr bool kKeepWeight = NV <= 2 || (V == 1 && NV == 8);
  constexpr int kWords = V == 8 ? 4 : 1;
  using P = Piece<V>;
  __shared__ RowStats stats[2][32];
  __shared__ double buf[32];
  const int step = WARP_ROW ? 32 : blockDim.x, t = WARP_ROW ? threadIdx.x % 32 : threadIdx.x;
  const int per_block = WARP_ROW ? 4 : 1;
  const int64_t first = int64_t(blockIdx.x) * per_block + (WARP_ROW ? threadIdx.x / 32 : 0), stride = int64_t(gridDim.x) * per_block;
  P w[NORM && kKeepWeight ? NV : 1];
  if (NORM && kKeepWeight) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * step + t) * V;
      if (k < p.K) w[i] = load_piece<V>(p.weight, k, p.K - k);
    }
  }
  wait_for_previous();
  const bool add = NORM && p.residual;
  // Where registers allow it the next row is on its way while this one is reduced.
  constexpr bool kAhead = V == 8 && !WARP_ROW && NV <= (NORM ? 2 : 4);
  constexpr int kGroup = NV < 4 ? NV : 4;  // pieces of the residual in flight
  P h[NV], r[kGroup];
  auto load = [&](P *to, int count, int from, const void *rows, int64_t ld, int64_t m) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i >= count) break;
      const int k = ((from + i) * step + t) * V;
      if (k < p.K) to[i] = load_piece<V>(static_cast<const T *>(rows) + m * ld, k, p.K - k);
    }
  };
  if (kAhead && first < p.M) {
    load(h, NV, 0, p.x, p.ldx, first);
    if (add) load(r, kGroup, 0, p.residual, p.ldr, first);
  }
  int turn = 0;
  bool left = false;
  for (int64_t m = first; m < p.M; m += stride, turn ^= 1) {
    if (!kAhead) load(h, NV, 0, p.x, p.ldx, m);
    if (add) {
      T *ro = static_cast<T *>(p.residual_out) + m * p.ldro;
#pragma unroll
      for (int g = 0; g < NV; g += kGroup) {
        if (!kAhead) load(r, kGroup, g, p.residual, p.ldr, m);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const int k = ((g + i) * step + t) * V;
          if (k < p.K) {
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
              const float2 u = unpack2<T>(h[g + i].u[j]), v = unpack2<T>(r[i].u[j]);
              h[g + i].u[j] = pack2<T>(u.x + v.x, u.y + v.y);
            }
            store_piece<V>(ro, k, h[g + i], p.K - k);
          }
        }
      }
    }
    P next[kAhead ? NV : 1];
    if (kAhead && m + stride < p.M) {
      load(next, NV, 0, p.x, p.ldx, m + stride);
      if (add) load(r, kGroup, 0, p.residual, p.ldr, m + stride);
    }
    RowStats s = {0.0f, 0u};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * step + t) * V;
      if (k < p.K) {
        P wi = {};
        if (NORM) wi = kKeepWeight ? w[kKeepWeight ? i : 0] : load_piece<V>(p.weight, k, p.K - k);
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          const float2 v = unpack2<T>(h[i].u[j]);
          float2 y = v;
          if (NORM) {
            const float2 g = unpack2<T>(wi.u[j]);
            y = mul2(v, g);
            s.ss = fmaf(v.x, v.x, s.ss);
            s.ss = fmaf(v.y, v.y, s.ss);
          }
          s.top = max(s.top, max(__float_as_uint(y.x) & 0x7fffffffu, __float_as_uint(y.y) & 0x7fffffffu));
        }
      }
    }
    s = WARP_ROW ? warp_stats(s) : block_stats(s, stats[turn]);
    const float mean = s.ss / float(p.K) + p.eps;
    const bool tame = row_is_tame<NORM>(s, mean);
    if (!tame) {
      if (t == 0) p.scale[m] = kLeft;
      left = true;
    }
    const RowFactors f = row_factors<NORM>(s, mean);
    if (t == 0 && tame) p.scale[m] = f.scale;
    int8_t *q = p.q + m * p.ldq;
    auto quantise_row = [&](auto two) {
      constexpr bool kTwo = decltype(two)::value;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (i * step + t) * V;
        if (k < p.K) {
          P wi = {};
          if (NORM) wi = kKeepWeight ? w[kKeepWeight ? i : 0] : load_piece<V>(p.weight, k, p.K - k);
          if constexpr (V == 8) {
            float2 y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 v = unpack2<T>(h[i].u[j]);
              y[j] = level2<kTwo>(NORM ? mul2(v, unpack2<T>(wi.u[j])) : v, f);
            }
            const uint2 o = make_uint2(pack4(y[0].x, y[0].y, y[1].x, y[1].y), pack4(y[2].x, y[2].y, y[3].x, y[3].y));
            const int n = p.K - k;
            if (n >= 8) *reinterpret_cast<uint2 *>(q + k) = o;
            else
              for (int j = 0; j < n; ++j) q[k + j] = int8_t((j < 4 ? o.x : o.y) >> (j % 4 * 8));
          } else {
            const float v = unpack2<T>(h[i].u[0]).x;
            q[k] = int8_t(__float_as_uint(level<kTwo>(NORM ? v * unpack2<T>(wi.u[0]).x : v, f)) & 0xff);
          }
        }
      }
    };
    if (tame) {
      if (f.two) quantise_row(std::true_type());
      else quantise_row(std::false_type());
    }
    if (kAhead) {
#pragma unroll
      for (int i = 0; i < NV; ++i) h[i] = next[i];
    }
  }
  if (!left) return;  // the same for all threads of a row
  if (WARP_ROW) __syncwarp();
  else __syncthreads();
  for (int64_t m = first; m < p.M; m += stride)
    if (*static_cast<volatile float *>(p.scale + m) == kLeft) row_in_double<T, NORM, WARP_ROW>(p, m, t, step, buf);
}

// Rows too long for registers: a block per row, value by value, in two passes over it.  A thread adds the squares of up to
// kRun / kLongThreads = 96 of its values, and these sums with what each addition loses carried along (Kahan's sum): the error
// stays below 100 steps of fp32 and 10 more in the block's reduction, however long the row.  One running sum of a thread's
// K / 512 values was off by 1e-3 at K = 2^26.
template <typename T, bool NORM>
__global__ void __launch_bounds__(kLongThreads, 3) long_rows_kernel(const __grid_constant__ RowParams p) {
  __shared__ RowStats stats[32];
  __shared__ double buf[32];
  const int64_t m = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + m * p.ldx, *w = static_cast<const T *>(p.weight);
  const bool add = NORM && p.residual;
  const T *r = add ? static_cast<const T *>(p.residual) + m * p.ldr : nullptr;
  T *ro = add ? static_cast<T *>(p.residual_out) + m * p.ldro : nullptr;
  wait_for_previous();
  RowStats s = {0.0f, 0u};
  float ss = 0, lost = 0;
  constexpr int kBatch = 6;  // loads in flight of each operand (eight with a residual spill: 16.3 us for 12.9, 1000 x 5001)
  constexpr int kRun = 16 * kBatch * kLongThreads;
  auto fold = [&] {
    const float add_now = ss - lost, sum = s.ss + add_now;
    lost = (sum - s.ss) - add_now;
    s.ss = sum;
    ss = 0;
  };
  for (int k0 = threadIdx.x; k0 < p.K; k0 += kBatch * kLongThreads) {
    T h[kBatch], a[kBatch], g[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int k = k0 + j * kLongThreads;
      if (k < p.K) {
        h[j] = x[k];
        if (NORM) g[j] = w[k];
        if (add) a[j] = r[k];
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int k = k0 + j * kLongThreads;
      if (k < p.K) {
        if (add) ro[k] = h[j] = from_f<T>(to_f(h[j]) + to_f(a[j]));
        const float v = to_f(h[j]), y = NORM ? v * to_f(g[j]) : v;
        if (NORM) ss = fmaf(v, v, ss);
        s.top = max(s.top, __float_as_uint(y) & 0x7fffffffu);
      }
    }
    if (NORM && (k0 + kBatch * kLongThreads) % kRun < kLongThreads) fold();
  }
  if (NORM) fold();
  s = block_stats(s, stats);
  const float mean = s.ss / float(p.K) + p.eps;
  if (!row_is_tame<NORM>(s, mean)) {
    row_in_double<T, NORM, false>(p, m, threadIdx.x, kLongThreads, buf);
    return;
  }
  const RowFactors f = row_factors<NORM>(s, mean);
  if (threadIdx.x == 0) p.scale[m] = f.scale;
  const T *again = add ? ro : x;  // every thread reads back what it wrote
  int8_t *q = p.q + m * p.ldq;
  auto quantise_row = [&](auto two) {
    for (int k0 = threadIdx.x; k0 < p.K; k0 += kBatch * kLongThreads) {
      T h[kBatch], g[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k = k0 + j * kLongThreads;
        if (k < p.K) {
          h[j] = again[k];
          if (NORM) g[j] = w[k];
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int k = k0 + j * kLongThreads;
        if (k < p.K) {
          const float v = to_f(h[j]);
          q[k] = int8_t(__float_as_uint(level<decltype(two)::value>(NORM ? v * to_f(g[j]) : v, f)) & 0xff);
        }
      }
    }
  };
  if (f.two) quantise_row(std::true_type());
  else quantise_row(std::false_type());
}

struct BackParams {
  const int8_t *q;
  const float *scale;
  void *out;
  int64_t M, ldq, ldo;
  int K, lanes;  // lanes: threads of a block that share a row, a power of two
};

constexpr int kBackThreads = 256;

// Four int8 values of a word, as floats times s: q + 128 in the mantissa of 2^23 is exact, without a
// conversion instruction.
__device__ __forceinline__ float4 scaled4(uint32_t word, float s) {
  const uint32_t u = word ^ 0x80808080u;
  return make_float4((__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540)) - 8388736.0f) * s,
                     (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541)) - 8388736.0f) * s,
                     (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7542)) - 8388736.0f) * s,
                     (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7543)) - 8388736.0f) * s);
}
template <typename T>
__device__ __forceinline__ uint4 scaled8(uint32_t lo, uint32_t hi, float s) {
  const float4 f = scaled4(lo, s), g = scaled4(hi, s);
  return make_uint4(pack2<T>(f.x, f.y), pack2<T>(f.z, f.w), pack2<T>(g.x, g.y), pack2<T>(g.z, g.w));
}

// A block takes kBackThreads / lanes rows, a thread 16 neighbouring values of rows at 16-byte addresses (V = 16).
// Of other rows it takes the eight that one aligned 16-byte piece of the output holds (V = 8), out of the three words
// around their bytes; pieces that reach beyond the row go value by value.  Bound by HBM: B200, 4096 x 8192 bf16
// 16.6 us (6.1 TB/s).
template <typename T, int V>
__global__ void __launch_bounds__(kBackThreads) back_kernel(const BackParams p) {
  const int rows = kBackThreads / p.lanes, row = threadIdx.x / p.lanes, width = p.lanes * V;
  const uint32_t chunks = uint32_t((int64_t(p.K) + (V == 8 ? 7 : 0) + width - 1) / width);
  const uint32_t group = blockIdx.x / chunks, chunk = blockIdx.x - group * chunks;
  const int64_t m = int64_t(group) * rows + row;
  T *out = static_cast<T *>(p.out) + m * p.ldo;
  const int8_t *q = p.q + m * p.ldq;
  int k = int(chunk) * width + (threadIdx.x % p.lanes) * V;
  if (V == 8) k -= int(reinterpret_cast<uintptr_t>(out) / 2 % 8);
  wait_for_previous();
  if (m >= p.M || k >= p.K) return;
  const float s = p.scale[m];
  if (k >= 0 && k + V <= p.K) {
    if constexpr (V == 16) {
      const uint4 b = *reinterpret_cast<const uint4 *>(q + k);
      reinterpret_cast<uint4 *>(out + k)[0] = scaled8<T>(b.x, b.y, s);
      reinterpret_cast<uint4 *>(out + k)[1] = scaled8<T>(b.z, b.w, s);
    } else {
      const uintptr_t at = reinterpret_cast<uintptr_t>(q + k);
      const uint32_t *words = reinterpret_cast<const uint32_t *>(at & ~uintptr_t(3));
      const int shift = int(at & 3) * 8;
      const uint32_t w0 = words[0], w1 = words[1], w2 = shift ? words[2] : 0;
      *reinterpret_cast<uint4 *>(out + k) = scaled8<T>(__funnelshift_r(w0, w1, shift), __funnelshift_r(w1, w2, shift), s);
    }
  } else {
    for (int j = max(0, -k); j < V && k + j < p.K; ++j) out[k + j] = from_f<T>(float(q[k + j]) * s);
  }
}

template <typename... P, typename... A>
static mgv_status launch_rows(void (*kern)(P...), int64_t grid, int threads, int flags, cudaStream_t s, A... a) {
  if (grid > 0x7fffffff) return fail(MGV_STATUS_UNSUPPORTED, "row kernel: too many rows for one launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & MGV_FLAG_PDL) ? 1 : 0;
  MGV_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a...));
  return MGV_STATUS_OK;
}

static bool aligned_rows(const void *p, int64_t ld, int64_t elem, int64_t rows, unsigned to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && (rows <= 1 || ld * elem % to == 0);
}

static int sm_count() {
  static std::atomic<int> known[64];  // calls may come from several threads
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int count = known[dev].load(std::memory_order_relaxed);
  if (!count && cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
    known[dev].store(count, std::memory_order_relaxed);
  return count > 0 ? count : 148;
}

template <typename T, bool NORM>
static mgv_status quantise(const RowParams &p, int flags, cudaStream_t s) {
  const bool wide = aligned_rows(p.x, p.ldx, 2, p.M, 16) && aligned_rows(p.q, p.ldq, 1, p.M, 8) &&
                    (!NORM || (aligned_rows(p.weight, 0, 2, 1, 16) &&
                               (!p.residual || (aligned_rows(p.residual, p.ldr, 2, p.M, 16) && aligned_rows(p.residual_out, p.ldro, 2, p.M, 16)))));
  const int sms = sm_count();
  const int64_t few = 2 * int64_t(sms);
  if (wide && p.K <= 65536) {
    const int pieces = (p.K + 7) / 8;
    if (pieces <= 128 && p.M > few)
      return launch_rows(rows_kernel<T, NORM, 8, 4, true>, std::min<int64_t>((p.M + 3) / 4, int64_t(sms) * 16), 128, flags, s, p);
    // few rows: as many threads as a row has pieces, for the shortest chain of loads; many rows: more pieces a thread and
    // smaller blocks, so that several of an SM are at different points of their rows (norm of 4096 x 8192 with residual
    // 43.2 us with four pieces, 38.7 with two and the next row on its way; quantisation 18.9 us with two, 16.8 with four)
    int nv = 1;
    while (nv < 8 && pieces > 1024 * nv) nv *= 2;
    if (p.M > few) nv = std::max(nv, NORM ? 2 : 4);
    const int threads = std::max(32, ((pieces + nv - 1) / nv + 31) / 32 * 32);
    const int64_t grid = std::min<int64_t>(p.M, int64_t(sms) * std::max(1, 2048 / threads));
    switch (nv) {
      case 1: return launch_rows(rows_kernel<T, NORM, 8, 1, false>, grid, threads, flags, s, p);
      case 2: return launch_rows(rows_kernel<T, NORM, 8, 2, false>, grid, threads, flags, s, p);
      case 4: return launch_rows(rows_kernel<T, NORM, 8, 4, false>, grid, threads, flags, s, p);
      default: return launch_rows(rows_kernel<T, NORM, 8, 8, false>, grid, threads, flags, s, p);
    }
  }
  // Value by value: in registers where rows are short or few, else in two passes (the norm of 1000 rows of 5001:
  // 9.7 us against 12.3, with residual 13.0 against 16.4).
  if (p.K <= 2048 || (p.K <= 8192 && p.M <= few)) {
    const int threads = ((p.K + 7) / 8 + 31) / 32 * 32;
    return launch_rows(rows_kernel<T, NORM, 1, 8, false>, std::min<int64_t>(p.M, int64_t(sms) * (2048 / threads)), threads, flags, s, p);
  }
  return launch_rows(long_rows_kernel<T, NORM>, p.M, kLongThreads, flags, s, p);
}

template <typename T>
static mgv_status dequantise(BackParams p, int flags, cudaStream_t s) {
  const bool wide = aligned_rows(p.q, p.ldq, 1, p.M, 16) && aligned_rows(p.out, p.ldo, 2, p.M, 16);
  const int v = wide ? 16 : 8;
  const int64_t reach = int64_t(p.K) + (wide ? 0 : 7);  // a row may begin inside its first piece
  p.lanes = 1;
  while (p.lanes < kBackThreads && p.lanes * v < reach) p.lanes *= 2;
  const int rows = kBackThreads / p.lanes;
  const int64_t grid = (p.M + rows - 1) / rows * ((reach + p.lanes * v - 1) / (p.lanes * v));
  return wide ? launch_rows(back_kernel<T, 16>, grid, kBackThreads, flags, s, p) : launch_rows(back_kernel<T, 8>, grid, kBackThreads, flags, s, p);
}

// What the three entry points check alike; `what` names the call in the message.
static mgv_status check_rows(const char *what, int dtype, int64_t M, int32_t K, int flags) {
  if (dtype != MGV_DTYPE_F16 && dtype != MGV_DTYPE_BF16)
    return fail(MGV_STATUS_UNSUPPORTED, "%s: dtype %d is neither F16 nor BF16", what, dtype);
  if (M < 0 || M > 0x7fffffff) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: M=%lld outside 0..2^31-1", what, (long long)M);
  if (K < 1 || K > (1 << 30)) return fail(MGV_STATUS_INVALID_ARGUMENT, "%s: K=%d outside 1..2^30", what, K);
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
  return dtype == MGV_DTYPE_F16 ? quantise<__half, false>(p, flags, s) : quantise<__nv_bfloat16, false>(p, flags, s);
}

extern "C" mgv_status mgv_dequantize_rows(void *out, const void *q, const void *scale, int dtype, int64_t M, int32_t K,
                                          int64_t ldo, int64_t ldq, int flags, mgv_stream_t s) {
  MGV_CHECK(check_rows("dequantize_rows", dtype, M, K, flags));
  if (M == 0) return MGV_STATUS_OK;
  MGV_CHECK(check_operand("dequantize_rows", "out", out, ldo, K, 2));
  MGV_CHECK(check_operand("dequantize_rows", "q", q, ldq, K, 1));
  MGV_CHECK(check_operand("dequantize_rows", "scale", scale, K, K, 4));
  BackParams p = {};
  p.q = static_cast<const int8_t *>(q); p.scale = static_cast<const float *>(scale); p.out = out;
  p.M = M; p.K = K; p.ldq = ldq; p.ldo = ldo;
  return dtype == MGV_DTYPE_F16 ? dequantise<__half>(p, flags, s) : dequantise<__nv_bfloat16>(p, flags, s);
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
  return a->dtype == MGV_DTYPE_F16 ? quantise<__half, true>(p, a->flags, s) : quantise<__nv_bfloat16, true>(p, a->flags, s);
}
