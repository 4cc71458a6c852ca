// Row-group building blocks shared by the quantisation kernels (int8 and
// 4-bit): parameters, streaming loads, reductions over the threads that own a
// row, and the correctly rounded reciprocal square root of the RMSNorm.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.h"
#include "ptx.cuh"

namespace tmw {
namespace {

enum QuantMode : int {
  kDynamic = 0,    // per-row amax/127
  kStatic = 1,     // given per-tensor scale, q = x / s
  kWeight = 2,     // per-row amax/127 clamped at 1e-12, q = clamp(x / s, +-127)
  kModulate = 3,   // adaLN modulate, then dynamic
  kRmsModulate = 4,  // RMSNorm, adaLN modulate, then dynamic
  kResGateRmsModulate = 5,  // gated residual add, then as kRmsModulate
  kModulateRows = 6,  // kModulate with one table row per row (no index): tables loaded with x
  kRmsModulateRows = 7,         // kRmsModulate and kResGateRmsModulate with one table row
  kResGateRmsModulateRows = 8   // per row: tables asked for before they are used
};

// adaLN modulate without RMSNorm (indexed or per-row tables)
__host__ __device__ constexpr bool modulate_only(int mode) {
  return mode == kModulate || mode == kModulateRows;
}

struct QuantParams {
  const void* x;
  int64_t ldx;
  int8_t* q;          // [rows, cols], row stride cols
  float* scales;      // [rows]
  const float* static_scale;
  __nv_bfloat16* hidden_out;  // optional [rows, cols] bf16 (modulate modes)
  const __nv_bfloat16* shift;
  const __nv_bfloat16* mod_scale;
  const int64_t* index;
  int64_t table_stride;
  const __nv_bfloat16* norm_w;
  float eps;
  double inv_cols;  // 1 / cols, correctly rounded (RMSNorm modes)
  // kResGateRmsModulate: x is the residual stream; branch [rows, cols] and
  // the gate table (row stride table_stride) update it, and the updated
  // residual is written to residual_out [rows, cols]
  const __nv_bfloat16* branch;
  const __nv_bfloat16* gate;
  __nv_bfloat16* residual_out;
  int64_t rows;
  int64_t cols;
  int tpr_log2;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}

// Round-to-nearest-even through bf16 and back (identical to the reference's
// _round_bf16 for finite values, fused_kernels.py:57-61).
__device__ __forceinline__ float round_bf16(float v) {
  return __bfloat162float(__float2bfloat16_rn(v));
}

template <typename T>
struct VecTraits {
  static constexpr int kElems = 16 / sizeof(T);
};

// Unpack one 16-byte vector into floats.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& raw, float (&out)[VecTraits<T>::kElems]) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int j = 0; j < VecTraits<T>::kElems; ++j) out[j] = to_f32<T>(e[j]);
}

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// Read-only 16-byte load the compiler may schedule freely (not volatile):
// the adaLN tables and the gated branch are never written by the kernel, so
// an unrolled loop's loads can all be issued ahead of its stores instead of
// one L2 round trip per iteration.
__device__ __forceinline__ uint4 ld_nc16(const void* p) {
  uint4 r;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
      : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
      : "l"(p));
  return r;
}

__device__ __forceinline__ uint4 ld_cached16(const void* p) {
  return __ldg(reinterpret_cast<const uint4*>(p));
}

// Max / sum over the TPR threads of a row group.  Groups of <= 32 threads
// live inside one warp; wider groups combine per-warp partials through
// shared memory (every thread of the block reaches the __syncthreads).
template <bool kMax>
__device__ __forceinline__ float group_reduce(float v, int tpr, float* red) {
  const int lane_span = tpr < 32 ? tpr : 32;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    if (off < lane_span) {
      const float o = __shfl_xor_sync(0xffffffffu, v, off);
      v = kMax ? fmaxf(v, o) : v + o;
    }
  }
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    __syncthreads();  // protect `red` from the previous use
    if (lane == 0) red[warp] = v;
    __syncthreads();
    const int wpr = tpr >> 5;
    const int first = (warp / wpr) * wpr;
    float acc = red[first];
    for (int w = 1; w < wpr; ++w) acc = kMax ? fmaxf(acc, red[first + w]) : acc + red[first + w];
    v = acc;
  }
  return v;
}

// Sum of one double per thread over the row group (the RMSNorm sum of
// squares).  `red` must hold 8 doubles.
__device__ __forceinline__ double group_sum_f64(double v, int tpr, double* red) {
  const int lane_span = tpr < 32 ? tpr : 32;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    if (off < lane_span) v = __dadd_rn(v, __shfl_xor_sync(0xffffffffu, v, off));
  }
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    __syncthreads();  // protect `red` from the previous use
    if (lane == 0) red[warp] = v;
    __syncthreads();
    const int wpr = tpr >> 5;
    const int first = (warp / wpr) * wpr;
    double acc = red[first];
    for (int w = 1; w < wpr; ++w) acc = __dadd_rn(acc, red[first + w]);
    v = acc;
  }
  return v;
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack_bf16x2(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

// Correctly rounded fp32 square root and reciprocal without the library's
// division / square-root subroutines (whose slow-path calls make the caller
// save its live registers: the producers hold a whole row in registers).
// Method: a hardware approximation (rsqrt.approx / rcp.approx, about 2^-22
// relative), one Newton-Raphson step in fp64, rounding to fp32, then an exact
// rounding test against the two neighbouring midpoints (Tuckerman's test):
// a midpoint has at most 25 significant bits, so its square or its product
// with a 24-bit value is exact in fp64 and the comparisons decide the
// rounding exactly.  Exact midpoint ties cannot occur for either operation.
__device__ __forceinline__ float f32_next_up(float v) {
  return __uint_as_float(__float_as_uint(v) + 1u);  // v positive and finite
}
__device__ __forceinline__ float f32_next_down(float v) {
  return __uint_as_float(__float_as_uint(v) - 1u);  // v positive
}

// fp32(sqrt(v)) for v positive, finite and normal.
__device__ __forceinline__ float sqrt_rn_normal(float v) {
  float y0;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(y0) : "f"(v));
  const double vd = static_cast<double>(v);
  double y = static_cast<double>(y0);
  // y <- y (3 - v y^2) / 2: Newton-Raphson for 1 / sqrt(v)
  y = __dmul_rn(y, __fma_rn(-0.5 * vd, __dmul_rn(y, y), 1.5));
  float s = __double2float_rn(__dmul_rn(vd, y));
  const double hi = 0.5 * (static_cast<double>(s) + static_cast<double>(f32_next_up(s)));
  const double lo = 0.5 * (static_cast<double>(s) + static_cast<double>(f32_next_down(s)));
  if (vd >= __dmul_rn(hi, hi)) {
    s = f32_next_up(s);
  } else if (vd < __dmul_rn(lo, lo)) {
    s = f32_next_down(s);
  }
  return s;
}

// fp32(1 / fp32(sqrt(v))), IEEE semantics for v >= 0 (and NaN).
__device__ __forceinline__ float rsqrt_two_step_rn(float v) {
  if (!(v > 0.0f)) return v == 0.0f ? __int_as_float(0x7f800000) : v;  // +inf / NaN
  if (v == __int_as_float(0x7f800000)) return 0.0f;
  float s;
  if (v < 1.17549435e-38f) {  // subnormal: sqrt(v * 2^32) = sqrt(v) * 2^16, exactly
    s = __fmul_rn(sqrt_rn_normal(__fmul_rn(v, 4294967296.0f)), 1.52587890625e-05f);
  } else {
    s = sqrt_rn_normal(v);
  }
  // s is normal here (s >= sqrt of the smallest subnormal), and so is 1 / s
  float r0;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r0) : "f"(s));
  const double sd = static_cast<double>(s);
  double r = static_cast<double>(r0);
  r = __fma_rn(r, __fma_rn(-sd, r, 1.0), r);  // r <- r (2 - s r)
  float q = __double2float_rn(r);
  const double hi = 0.5 * (static_cast<double>(q) + static_cast<double>(f32_next_up(q)));
  const double lo = 0.5 * (static_cast<double>(q) + static_cast<double>(f32_next_down(q)));
  if (__dmul_rn(sd, hi) <= 1.0) {  // 1 / s >= hi
    q = f32_next_up(q);
  } else if (__dmul_rn(sd, lo) > 1.0) {  // 1 / s < lo
    q = f32_next_down(q);
  }
  return q;
}

}  // namespace
}  // namespace tmw
