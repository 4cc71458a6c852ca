// Pieces shared by the scaled GEMM kernels: the raster of output tiles and the
// epilogue's activations, conversions and TMA-store staging layout.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "common.h"
#include "ptx.cuh"

namespace tmw {
namespace {

constexpr int kGroupM = 16;  // M-blocks of a raster group

// Raster order of output tiles.  Concurrent tiles should share operand
// panels in L2.  Default: groups of kGroupM M-blocks, M fastest -- a wave
// shares kGroupM A panels and a few B panels.  With group_n > 0 (long K,
// where kGroupM A panels of K bytes per row would not stay in L2 beside B):
// groups of group_n N-blocks over all M-blocks, N fastest -- a wave shares
// a few A panels, each read from DRAM once, while the group's B panels stay
// resident for every M-block.
__device__ __forceinline__ void tile_coords(int tile, int num_m, int num_n, int& mb, int& nb,
                                            int m_owners, int mb_per_owner, int group_n = 0) {
  if (group_n > 0) {
    const int group_size = group_n * num_m;
    const int group = tile / group_size;
    const int first_n = group * group_n;
    const int gn = min(num_n - first_n, group_n);
    const int local = tile - group * group_size;
    nb = first_n + local % gn;
    mb = local / gn;
  } else {
    const int group_size = kGroupM * num_n;
    const int group = tile / group_size;
    const int first_m = group * kGroupM;
    const int gm = min(num_m - first_m, kGroupM);
    const int local = tile - group * group_size;
    mb = first_m + local % gm;
    nb = local / gm;
  }
  if (m_owners > 1) {  // num_m == m_owners x mb_per_owner
    const int owner = mb % m_owners;
    mb = owner * mb_per_owner + mb / m_owners;
  }
}

__device__ __forceinline__ float gelu_tanh(float x) {
  // 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))), every operation explicit
  // (no contraction left to the compiler), so each epilogue path that
  // inlines it computes the same bits
  // inner = x (beta + beta kappa x^2); result = 0.5 x + 0.5 x tanh(inner)
  const float k_beta = 0.7978845608028654f;          // sqrt(2 / pi)
  const float k_beta_kappa = 0.035677408136300125f;  // sqrt(2 / pi) * 0.044715
  const float inner = __fmul_rn(x, __fmaf_rn(k_beta_kappa, __fmul_rn(x, x), k_beta));
  const float h = __fmul_rn(0.5f, x);
  return __fmaf_rn(h, tanh_approx(inner), h);
}

template <typename OutT>
__device__ __forceinline__ float out_to_f32(OutT v);
template <>
__device__ __forceinline__ float out_to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float out_to_f32<__half>(__half v) {
  return __half2float(v);
}

template <typename OutT>
__device__ __forceinline__ OutT from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

template <typename OutT>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <typename OutT>
__device__ __forceinline__ float round_out(float v);
template <>
__device__ __forceinline__ float round_out<__nv_bfloat16>(float v) {
  return __bfloat162float(__float2bfloat16_rn(v));
}
template <>
__device__ __forceinline__ float round_out<__half>(float v) {
  return __half2float(__float2half_rn(v));
}

// Round two values to OutT and back with one paired conversion (the same
// bits as two round_out calls; the conversion unit, which bounds the
// epilogue's arithmetic, does half the work for bf16).
template <typename OutT>
__device__ __forceinline__ void round2_out(float& a, float& b);
template <>
__device__ __forceinline__ void round2_out<__nv_bfloat16>(float& a, float& b) {
  const uint32_t p = pack2<__nv_bfloat16>(a, b);  // a in the low half, b in the high half
  a = __uint_as_float(p << 16);
  b = __uint_as_float(p & 0xffff0000u);
}
template <>
__device__ __forceinline__ void round2_out<__half>(float& a, float& b) {
  a = round_out<__half>(a);
  b = round_out<__half>(b);
}

constexpr int kStage64Bytes = 32 * 64;  // a 32 x 32 tile of a 16-bit type, 64-byte swizzle

__device__ __forceinline__ uint4* stage64_slot(uint8_t* stage, int row, int chunk) {
  return reinterpret_cast<uint4*>(stage + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}

__device__ __forceinline__ float sigmoid_f32(float x) {
  return __fdividef(1.0f, __fadd_rn(1.0f, __expf(-x)));
}

// Raster choice (GemmArgs::group_n).  Once kGroupM A panels (rows_per_mb x K
// bytes each) pass kAGroupBudget they no longer stay in L2 next to the B
// panels a wave reads (the 480p fc2, K = 12288: 16 x 3 MiB of A), so the
// tiles switch to N-fastest groups whose B panels fit kBGroupBudget.
constexpr uint64_t kAGroupBudget = 24ull << 20;
constexpr uint64_t kBGroupBudget = 48ull << 20;

inline int choose_group_n(int num_n, int rows_per_mb, int bn, int k) {
  const uint64_t a_group = static_cast<uint64_t>(kGroupM) * rows_per_mb * static_cast<uint64_t>(k);
  if (a_group <= kAGroupBudget) return 0;
  const uint64_t b_panel = static_cast<uint64_t>(bn) * static_cast<uint64_t>(k);
  const uint64_t fit = b_panel > 0 ? kBGroupBudget / b_panel : 1;
  return static_cast<int>(fit < 1 ? 1 : (fit > static_cast<uint64_t>(num_n) ? num_n : fit));
}

}  // namespace
}  // namespace tmw
