// Block-scaled 4-bit GEMM on the 5th-generation tensor cores (sm_100a).
//
//   out[m, n] = act(sa[m] * (sb[n] * sum_k (a s_a)[m, k] (b s_b)[n, k]) + bias[n])
//
// a, b: e2m1 codes with a scale for each block of K (fp4.cuh); sa, sb: the
// fp32 outer scales of TM_FP4_NV.  The block scales are applied by the tensor
// cores (tcgen05.mma kind::mxf4nvf4), which accumulate in fp32; everything
// after the accumulator is fp32 and rounded once, on output.
//
// A k-block is 128 bytes (256 elements) of K: one swizzle row of codes, four
// MMAs of K = 64.  Its scales are 4 (TM_FP4_NV) or 2 (TM_FP4_MX) 512-byte tiles
// for each 128 rows; they travel by TMA beside the codes and are copied to TMEM
// by the MMA thread (tcgen05.cp, in order with its MMAs); the columns of a scale
// tile are written again only after the MMAs that read them have completed.
//
//   gemm_fp4_pair_kernel  persistent CTA pairs (clusters of 2), a 256 token x 256
//     weight row tile each: a CTA fetches 128 token rows and 128 weight rows, the
//     leader issues tcgen05.mma.cta_group::2 (M = 256, N = 256), and each CTA's
//     TMEM receives 128 x 256 sums.  Two such accumulators and the scales exceed
//     the 512 TMEM columns, so there is one: the epilogue takes it into registers
//     (128 columns a warp) and converts and stores while the next tile runs.
//   gemm_fp4_small_kernel  one CTA per (128 weight rows x TOK tokens, K slice).
//     The weight is the M operand (128 TMEM lanes), the tokens the N operand, so
//     one token costs a 32-column accumulator and the weight streams once.
//     Slices of K are the CTAs of a cluster; their partial sums meet in
//     distributed shared memory and are added in slice order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstring>
#include <type_traits>

#include "epilogue.cuh"
#include "fp4.cuh"

namespace tmw {
namespace {

constexpr int kRowBytes = 128;  // a k-block of one row of codes
constexpr int kKBlock = 256;    // elements
constexpr int kMmaK = 64;
constexpr int kTileRows = 128;

struct Fp4Args {
  const float* sa;  // NULL: 1
  const float* sb;
  int sa_per_row;
  int sb_per_col;
  const void* bias;  // NULL or [N] in the output type
  void* out;
  int64_t ldo;
  int M, N, K;
  int kblocks;
  int num_m, num_n;
  int group_n;
  int stages;
  bool wide;  // output rows start on 32-byte boundaries
  uint32_t epilogue;
  int* status;
};

// MMAs of k-block kb: the last one may hold fewer than 256 elements (the codes
// past K are zero; whole steps past K have no scales and are left out).
__device__ __forceinline__ int kblock_steps(int K, int kb) {
  const int left = K - kb * kKBlock;
  return left >= kKBlock ? kKBlock / kMmaK : (left + kMmaK - 1) / kMmaK;
}

template <int FORMAT>
struct ScaleGeom {
  static constexpr int kBlock = FORMAT == TM_FP4_NV ? 16 : 32;
  static constexpr int kTiles = kKBlock / kBlock / 4;       // per 128 rows and k-block
  static constexpr int kBytes = kTiles * 512;
  static constexpr int kStepsPerTile = 4 / kTiles;          // MMAs sharing a tile
  static constexpr bool kE8m0 = FORMAT == TM_FP4_MX;
};

__device__ __forceinline__ float swiglu(float g, float u) {
  return __fmul_rn(__fmul_rn(g, sigmoid_f32(g)), u);
}

// GELU (tanh form): 0.5 y (1 + tanh(u)) = y / (1 + exp(-2 u)) with
// u = sqrt(2/pi) (y + 0.044715 y^3), hence exp(-2 u) = 2^(-y (A + B y^2)).  The
// quotient has no cancellation: its error is (|2 u| + 2) 2^-22 of the value, far
// below the output's half step, where 1 + tanh(u) from the tanh instruction is off
// by 2^-11 absolute, more than the value itself from y = -3.5 on.  What lies below
// |y| 2^-126 becomes 0.  Two special-function instructions a value in place of one:
// 8192 x 12288 x 3072 141 us against 133 in a burst, 157 against 148 sustained;
// one reciprocal for two values (of the denominators' product) 143 and 159.
constexpr float kGeluA = 2.3022081985f;   // 2 sqrt(2/pi) log2(e)
constexpr float kGeluB = 0.10294323960f;  // 0.044715 A
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float gelu_quotient(float y) {
  const float x = __fmul_rn(y, __fmaf_rn(-kGeluB, __fmul_rn(y, y), -kGeluA));
  return __fmul_rn(y, rcp_approx(__fadd_rn(1.0f, ex2_approx(x))));
}
// The same bits for two values.  The pair kernel's form; in the small kernel, whose
// loops are short, the scalar one is faster (128 x 12288 x 3072: 8.8 against 9.2 us).
__device__ __forceinline__ uint64_t gelu_quotient_f32x2(uint64_t y) {
  const uint64_t x = mul_f32x2(
      y, fma_f32x2(f32x2(-kGeluB, -kGeluB), mul_f32x2(y, y), f32x2(-kGeluA, -kGeluA)));
  float a, b;
  f32x2_split(x, a, b);
  f32x2_split(add_f32x2(f32x2(ex2_approx(a), ex2_approx(b)), f32x2(1.0f, 1.0f)), a, b);
  return mul_f32x2(y, f32x2(rcp_approx(a), rcp_approx(b)));
}

__device__ __forceinline__ uint8_t* align1k(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) &
                                    ~static_cast<uintptr_t>(1023));
}

// ====================================================================== small
constexpr int kSmallThreads = 320;  // producer, MMA, eight epilogue warps
constexpr int kMaxStages = 8;

template <int TOK, int FORMAT>
struct SmallLayout {
  using S = ScaleGeom<FORMAT>;
  static constexpr int kWBytes = kTileRows * kRowBytes;
  static constexpr int kXBytes = TOK * kRowBytes;
  // codes first: swizzle atoms need 1 KiB alignment
  static constexpr int kStageBytes = kWBytes + kXBytes + 2 * S::kBytes;
  static_assert(kStageBytes % 1024 == 0, "stages stay aligned");
  static constexpr int kReduceBytes = kTileRows * TOK * 4;
  static constexpr int kBarBytes = 256 + kTileRows * 4;  // and the tokens' scales
  static constexpr int total(int stages, int splits) {
    return 1024 + stages * kStageBytes + kBarBytes + (splits > 1 ? kReduceBytes : 0);
  }
  // TMEM columns: the accumulator, then each stage's scale tiles (4 columns for
  // the weight rows and 4 for the tokens), written again after the stage's MMAs
  static constexpr int kTileCols = 8;
  static constexpr int kStageCols = kTileCols * S::kTiles;
  __host__ __device__ static constexpr int tmem_cols(int stages) {
    int cols = 64;
    while (cols < TOK + stages * kStageCols) cols *= 2;
    return cols;
  }
  static_assert(TOK + kMaxStages * kStageCols <= 512, "TMEM columns");
};

struct SmallBars {
  uint64_t* full;
  uint64_t* empty;
  uint64_t* acc;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
};

__device__ __forceinline__ SmallBars small_bars(uint8_t* base) {
  SmallBars b;
  b.full = reinterpret_cast<uint64_t*>(base);
  b.empty = b.full + kMaxStages;
  b.acc = b.empty + kMaxStages;
  b.tmem_slot = reinterpret_cast<uint32_t*>(b.acc + 1);
  b.abort_flag = reinterpret_cast<volatile int*>(b.tmem_slot + 1);
  return b;
}

__device__ __forceinline__ void st_cluster_f32x2(uint32_t addr, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}

// What a lane of an epilogue warp keeps: its weight row's constants.
struct RowConsts {
  int n;
  float sb, bias;
};

template <typename OutT>
__device__ __forceinline__ RowConsts row_consts(const Fp4Args& g, int n) {
  RowConsts c{n, 1.f, 0.f};
  if (n < g.N) {
    if (g.sb != nullptr) c.sb = ld_nc_f32(g.sb + (g.sb_per_col ? n : 0));
    if (g.bias != nullptr) c.bias = out_to_f32<OutT>(static_cast<const OutT*>(g.bias)[n]);
  }
  return c;
}

// Finish and store the sums of two tokens, a weight row per lane (the lanes of a
// warp are 32 consecutive output columns).  Neighbouring lanes exchange a value,
// so that each stores two columns of one token.  `left`: tokens from the first
// on (the stores alone depend on it, so the arithmetic of several pairs
// overlaps).  sa: the tokens' scales.  Called by the whole warp.
template <int EPI, typename OutT>
__device__ __forceinline__ void store_tokens(const Fp4Args& g, const RowConsts& c, int64_t m,
                                             int left, float2 sa, float acc0, float acc1) {
  const int lane = threadIdx.x & 31;
  float y0 = __fmaf_rn(sa.x, __fmul_rn(c.sb, acc0), c.bias);
  float y1 = __fmaf_rn(sa.y, __fmul_rn(c.sb, acc1), c.bias);
  int col = c.n;
  bool in = c.n < g.N;
  if constexpr (EPI == TM_EPI_GELU_TANH) {
    y0 = gelu_quotient(y0);
    y1 = gelu_quotient(y1);
  } else if constexpr (EPI == TM_EPI_SWIGLU) {
    // weight rows come as 16 gate rows, then the 16 matching up rows
    const float u0 = __shfl_down_sync(0xffffffffu, y0, 16);
    const float u1 = __shfl_down_sync(0xffffffffu, y1, 16);
    y0 = swiglu(y0, u0);
    y1 = swiglu(y1, u1);
    col = (c.n >> 5) * 16 + (c.n & 15);
    in = in && lane < 16;
  }
  const int odd = lane & 1;  // odd lanes take the second token
  const float got = __shfl_xor_sync(0xffffffffu, odd ? y0 : y1, 1);
  if (in && odd < left) {
    OutT* dst = static_cast<OutT*>(g.out) + (m + odd) * g.ldo + (col & ~1);
    *reinterpret_cast<uint32_t*>(dst) = odd ? pack2<OutT>(got, y1) : pack2<OutT>(y0, got);
  }
}

// The epilogue warps' work, in loops short enough to be fetched quickly: these
// kernels run their code once.  Warp half h (0, 1) takes every other group of
// eight tokens, or every other pair.
template <int EPI, typename OutT>
__device__ __forceinline__ void store_tile(const Fp4Args& g, const RowConsts& c, const float* sa,
                                           uint32_t t_row, int64_t m0, int tokens, int h) {
#pragma unroll 1
  for (int t = 8 * h; t < tokens; t += 16) {
    uint32_t r[8];
    tmem_ld_32x32b_x8(t_row + t, r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      store_tokens<EPI, OutT>(g, c, m0 + t + j, tokens - t - j,
                              *reinterpret_cast<const float2*>(sa + t + j), __uint_as_float(r[j]),
                              __uint_as_float(r[j + 1]));
  }
}

// Pairs of tokens are dealt out to the slices of the cluster: pair p is finished
// by slice p % splits, its sums at sums[slice][p / splits][weight row].
constexpr int kMaxSplits = 8;

__device__ __forceinline__ void send_sums(float2* sums, uint32_t t_row, int row, int tokens,
                                          int slice, int splits, int log_splits, int h, bool ok) {
  const int pairs = ((tokens + 1) / 2 + splits - 1) >> log_splits;  // of one slice
  const uint32_t mine = smem_u32(sums + slice * pairs * kTileRows + row);
#pragma unroll 1
  for (int t = 8 * h; t < tokens; t += 16) {
    uint32_t r[8];
    tmem_ld_32x32b_x8(t_row + t, r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const int p = (t + j) >> 1;
      const uint32_t at = mine + (p >> log_splits) * (kTileRows * 8);
      const float nan = __int_as_float(0x7fffffff);
      if (t + j < tokens)
        st_cluster_f32x2(map_to_cta(at, p & (splits - 1)), ok ? __uint_as_float(r[j]) : nan,
                         ok ? __uint_as_float(r[j + 1]) : nan);
    }
  }
}

template <int EPI, typename OutT>
__device__ __forceinline__ void store_reduced(const Fp4Args& g, const RowConsts& c, const float* sa,
                                              const float2* sums, int row, int64_t m0, int tokens,
                                              int slice, int splits, int log_splits, int h) {
  const int all = (tokens + 1) / 2;
  const int pairs = (all + splits - 1) >> log_splits;
#pragma unroll 1
  for (int l = h; l < pairs; l += 2) {
    const int p = (l << log_splits) + slice;
    if (p >= all) break;
    float2 part[kMaxSplits];
#pragma unroll
    for (int s = 0; s < kMaxSplits; ++s)
      part[s] = s < splits ? sums[(s * pairs + l) * kTileRows + row] : make_float2(0.f, 0.f);
    float a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int s = 0; s < kMaxSplits; ++s) {  // in slice order; the absent ones add 0
      a0 += part[s].x;
      a1 += part[s].y;
    }
    store_tokens<EPI, OutT>(g, c, m0 + 2 * p, tokens - 2 * p,
                            *reinterpret_cast<const float2*>(sa + 2 * p), a0, a1);
  }
}

template <int TOK, int FORMAT, typename OutT>
__global__ void __launch_bounds__(kSmallThreads)
    gemm_fp4_small_kernel(const __grid_constant__ CUtensorMap tm_w,
                          const __grid_constant__ CUtensorMap tm_x,
                          const __grid_constant__ CUtensorMap tm_ws,
                          const __grid_constant__ CUtensorMap tm_xs, const Fp4Args g,
                          const int splits) {
  using L = SmallLayout<TOK, FORMAT>;
  using S = ScaleGeom<FORMAT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1k(smem_raw);
  const SmallBars bar = small_bars(smem + g.stages * L::kStageBytes);
  float* token_sa = reinterpret_cast<float*>(smem + g.stages * L::kStageBytes + 256);
  float2* sums = reinterpret_cast<float2*>(smem + g.stages * L::kStageBytes + L::kBarBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int slice = blockIdx.x % splits;
  const int tile = blockIdx.x / splits;
  const int nb = tile % g.num_n;
  const int mb = tile / g.num_n;
  // even slices, none empty (splits <= kblocks)
  const int kb0 = static_cast<int>(static_cast<int64_t>(slice) * g.kblocks / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(slice + 1) * g.kblocks / splits);
  const uint32_t tmem_cols = L::tmem_cols(g.stages);

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(&bar.full[s], 1);
      mbar_init(&bar.empty[s], 1);
    }
    mbar_init(bar.acc, 1);
    *bar.abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_ws);
    tma_prefetch_desc(&tm_xs);
  }
  if (warp == 1) {
    tmem_alloc(bar.tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  if (splits > 1)
    cluster_sync();  // every slice is running before any writes to another's shared memory
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *bar.tmem_slot;
  // With one token tile the weight is read once: ask for this slice of it while
  // the previous kernel on the stream still runs (an L2 prefetch has no effect
  // on what is read later, whoever writes the weight).
  if (threadIdx.x == 64 && g.num_m == 1) {
    for (int kb = kb0; kb < kb1; ++kb) {
      tma_prefetch_l2_2d(&tm_w, kb * kRowBytes, nb * kTileRows);
      tma_prefetch_l2_2d(&tm_ws, kb * (S::kBytes / 8), nb);
    }
  }
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    uint32_t issued_mask = 0, issued_parity = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(&bar.empty[stage], phase ^ 1u, bar.abort_flag, g.status)) {
        ok = false;
        break;
      }
      issued_mask &= ~(1u << stage);
      if (elect_one()) {
        uint8_t* s = smem + stage * L::kStageBytes;
        mbar_arrive_expect_tx(&bar.full[stage], L::kStageBytes);
        tma_load_2d(&tm_w, &bar.full[stage], s, kb * kRowBytes, nb * kTileRows);
        tma_load_2d(&tm_ws, &bar.full[stage], s + L::kWBytes + L::kXBytes, kb * (S::kBytes / 8), nb);
        tma_load_2d(&tm_x, &bar.full[stage], s + L::kWBytes, kb * kRowBytes, mb * TOK);
        tma_load_2d(&tm_xs, &bar.full[stage], s + L::kWBytes + L::kXBytes + S::kBytes,
                    kb * (S::kBytes / 8), mb);  // TOK = 128, or a single token tile
      }
      __syncwarp();
      issued_mask |= 1u << stage;
      issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
      if (++stage == g.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok && lane == 0) {
      for (int s = 0; s < g.stages; ++s)
        if (issued_mask & (1u << s))
          mbar_wait_drain(&bar.full[s], (issued_parity >> s) & 1u, g.status);
    }
    __syncwarp();
  } else if (warp == 1) {
    // the whole warp runs the loop, one lane issues (see elect_one)
    const uint32_t tmem = __reduce_max_sync(0xffffffffu, tmem_base);
    const uint32_t smem0 = smem_u32(smem);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true, issued_any = false;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(&bar.full[stage], phase, bar.abort_flag, g.status)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t base = smem0 + stage * L::kStageBytes;
      const uint64_t w_desc = make_desc_kmajor_sw128(base);
      const uint64_t x_desc = make_desc_kmajor_sw128(base + L::kWBytes);
      const uint64_t ws_desc = make_desc_scale_tile(base + L::kWBytes + L::kXBytes);
      const uint64_t xs_desc = make_desc_scale_tile(base + L::kWBytes + L::kXBytes + S::kBytes);
      const uint32_t col = tmem + TOK + stage * L::kStageCols;
      const uint32_t more = kb != kb0 ? 1u : 0u;
      const int steps = kblock_steps(g.K, kb);
      // descriptors count 16-byte units
      const auto copy = [&](int t) {
        tmem_copy_scale_tile<false>(col + L::kTileCols * t, ws_desc + 32 * t);
        tmem_copy_scale_tile<false>(col + L::kTileCols * t + 4, xs_desc + 32 * t);
      };
      const auto multiply = [&](int k) {
        const int t = k / S::kStepsPerTile;
        umma_fp4<false, S::kBlock>(
            tmem, w_desc + 2 * k, x_desc + 2 * k,
            make_idesc_fp4(kTileRows, TOK, S::kE8m0, k % S::kStepsPerTile * 2),
            col + L::kTileCols * t, col + L::kTileCols * t + 4, k == 0 ? more : 1u);
      };
      if (steps == kKBlock / kMmaK) {
        if (elect_one()) {
#pragma unroll
          for (int t = 0; t < S::kTiles; ++t) copy(t);
#pragma unroll
          for (int k = 0; k < kKBlock / kMmaK; ++k) multiply(k);
          umma_commit(&bar.empty[stage]);
        }
      } else {  // the last k-block of a K that is not a multiple of 256
        if (elect_one()) {
          for (int t = 0; t * S::kStepsPerTile < steps; ++t) copy(t);
          for (int k = 0; k < steps; ++k) multiply(k);
          umma_commit(&bar.empty[stage]);
        }
      }
      __syncwarp();
      issued_any = true;
      if (++stage == g.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (ok) {
      if (elect_one()) umma_commit(bar.acc);
    } else if (issued_any) {  // the last commit: the tensor pipe has drained
      const int last = stage == 0 ? g.stages - 1 : stage - 1;
      mbar_wait_drain(&bar.empty[last], stage == 0 ? (phase ^ 1u) : phase, g.status);
    }
    __syncwarp();
  } else {
    const int h = (warp - 2) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int64_t m0 = static_cast<int64_t>(mb) * TOK;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(TOK), g.M - m0));
    const RowConsts c = row_consts<OutT>(g, nb * kTileRows + row);
    if (threadIdx.x - 64 < TOK) {
      const int t = threadIdx.x - 64;
      token_sa[t] = g.sa == nullptr || t >= tokens ? 1.f : ld_nc_f32(g.sa + (g.sa_per_row ? m0 + t : 0));
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the epilogue warps: token_sa is complete
    const bool ok = mbar_wait_warp(bar.acc, 0, bar.abort_flag, g.status);
    tc_fence_after();
    const int log_splits = 31 - __clz(splits);
    if (splits > 1) {
      send_sums(sums, t_row, row, tokens, slice, splits, log_splits, h, ok);
      tc_fence_before();
      cluster_sync();  // every slice's sums have arrived
      if (g.epilogue & TM_EPI_GELU_TANH)
        store_reduced<TM_EPI_GELU_TANH, OutT>(g, c, token_sa, sums, row, m0, tokens, slice, splits,
                                              log_splits, h);
      else if (g.epilogue & TM_EPI_SWIGLU)
        store_reduced<TM_EPI_SWIGLU, OutT>(g, c, token_sa, sums, row, m0, tokens, slice, splits,
                                           log_splits, h);
      else
        store_reduced<0, OutT>(g, c, token_sa, sums, row, m0, tokens, slice, splits, log_splits, h);
    } else if (ok) {
      if (g.epilogue & TM_EPI_GELU_TANH)
        store_tile<TM_EPI_GELU_TANH, OutT>(g, c, token_sa, t_row, m0, tokens, h);
      else if (g.epilogue & TM_EPI_SWIGLU)
        store_tile<TM_EPI_SWIGLU, OutT>(g, c, token_sa, t_row, m0, tokens, h);
      else
        store_tile<0, OutT>(g, c, token_sa, t_row, m0, tokens, h);
    }
  }

  tc_fence_before();
  if (splits > 1 && warp < 2) cluster_sync();  // the epilogue warps' barrier is for every thread
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

// ====================================================================== pair
constexpr int kPairThreads = 320;  // producer, MMA, eight epilogue warps
constexpr int kPairEpiWarps = 8;
constexpr int kPairRows = 256;     // tokens, and weight rows, of a tile
// per epilogue warp: 128 column scales and 128 bias values
constexpr int kPairBiasCache = 512;
constexpr int kPairRegion = 768;
// TMEM: the 256-column accumulator, then each stage's scale tiles (4 columns
// for the tokens and 8 for the weight rows): a stage's columns are written
// again when its shared memory has been refilled, hence after its MMAs.
constexpr uint32_t kScaleCol = 256;
constexpr int kTileCols = 12;

template <int FORMAT>
struct PairLayout {
  using S = ScaleGeom<FORMAT>;
  static constexpr int kHalfBytes = 128 * kRowBytes;
  static constexpr int kStageBytes = 2 * kHalfBytes + 3 * S::kBytes;  // per CTA
  static constexpr int kStages = FORMAT == TM_FP4_NV ? 5 : 6;
  static_assert(kScaleCol + kStages * S::kTiles * kTileCols <= 512, "TMEM columns");
  static constexpr int kBarOffset = kStages * kStageBytes;
  static constexpr int kEpiOffset = kBarOffset + 256;
  static constexpr int kTotal = kEpiOffset + kPairEpiWarps * kPairRegion + 1024;
  static_assert(kStageBytes % 1024 == 0, "stages stay aligned");
  static_assert(kTotal <= 227 * 1024, "shared memory budget");
};

struct PairBars {
  uint64_t* full;
  uint64_t* empty;
  uint64_t* acc_full;
  uint64_t* acc_free;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
};

__device__ __forceinline__ PairBars pair_bars(uint8_t* base) {
  PairBars b;
  b.full = reinterpret_cast<uint64_t*>(base);
  b.empty = b.full + kMaxStages;
  b.acc_full = b.empty + kMaxStages;
  b.acc_free = b.acc_full + 1;
  b.tmem_slot = reinterpret_cast<uint32_t*>(b.acc_free + 1);
  b.abort_flag = reinterpret_cast<volatile int*>(b.tmem_slot + 1);
  return b;
}

// A lane's share of a tile's constants: the scales and bias values of four of
// the warp's 128 columns, and its row's scale.
struct PairConsts {
  float sb[4];
  float bias[4];
  float sa;
};

template <int FORMAT, typename OutT>
__device__ __forceinline__ PairConsts pair_consts(const Fp4Args& g, int nb, int h, int64_t row,
                                                  int lane) {
  PairConsts c;
  const int col = nb * kPairRows + 128 * h + 4 * lane;
  const bool in = col < g.N;  // N % 8 == 0: all four or none
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c.sb[j] = FORMAT == TM_FP4_NV && in ? ld_nc_f32(g.sb + (g.sb_per_col ? col + j : 0)) : 0.f;
    c.bias[j] =
        g.bias != nullptr && in ? out_to_f32<OutT>(static_cast<const OutT*>(g.bias)[col + j]) : 0.f;
  }
  c.sa = FORMAT == TM_FP4_NV && row < g.M ? ld_nc_f32(g.sa + (g.sa_per_row ? row : 0)) : 1.f;
  return c;
}

template <int FORMAT, typename OutT>
__device__ __forceinline__ void pair_consts_store(uint8_t* region, const PairConsts& c, int lane) {
  if constexpr (FORMAT == TM_FP4_NV)
    *reinterpret_cast<float4*>(region + 16 * lane) =
        make_float4(c.sb[0], c.sb[1], c.sb[2], c.sb[3]);
  *reinterpret_cast<uint2*>(region + kPairBiasCache + 8 * lane) =
      make_uint2(pack2<OutT>(c.bias[0], c.bias[1]), pack2<OutT>(c.bias[2], c.bias[3]));
}

// Outer scales, bias and (GELU) activation on 16 accumulator columns, in place.
template <int FORMAT, int EPI, typename OutT>
__device__ __forceinline__ void pair_finish16(uint32_t* r, uint64_t sa2, bool has_bias,
                                              const float* sb, const OutT* bias) {
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    uint64_t y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      y[i] = f32x2(__uint_as_float(r[j + 2 * i]), __uint_as_float(r[j + 2 * i + 1]));
    if constexpr (FORMAT == TM_FP4_NV) {
      const float4 s = *reinterpret_cast<const float4*>(sb + j);
      y[0] = mul_f32x2(y[0], f32x2(s.x, s.y));
      y[1] = mul_f32x2(y[1], f32x2(s.z, s.w));
    }
    if (has_bias) {
      const uint2 b = *reinterpret_cast<const uint2*>(bias + j);
      const OutT* e = reinterpret_cast<const OutT*>(&b);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        y[i] = fma_f32x2(sa2, y[i],
                         f32x2(out_to_f32<OutT>(e[2 * i]), out_to_f32<OutT>(e[2 * i + 1])));
    } else if constexpr (FORMAT == TM_FP4_NV) {
#pragma unroll
      for (int i = 0; i < 2; ++i) y[i] = mul_f32x2(sa2, y[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (EPI == TM_EPI_GELU_TANH) y[i] = gelu_quotient_f32x2(y[i]);
      float lo, hi;
      f32x2_split(y[i], lo, hi);
      r[j + 2 * i] = __float_as_uint(lo);
      r[j + 2 * i + 1] = __float_as_uint(hi);
    }
  }
}

// Store 16 columns of this lane's row, as one 32-byte sector where the output
// allows it (`wide`: rows start on 32-byte boundaries).  8192 x 12288 x 3072
// nvfp4: two 16-byte stores in place of the one cost 154 against 130 us, with GELU
// 162 against 143; staged TMA stores (121 against 123 when they were tried), or full
// lines after an exchange between lanes (mxfp4 117 against 111), gain nothing: what
// remains is the output's share of the traffic.
// Not allocating in L1: 135 -> 130 us, with GELU 148 -> 143.
template <typename OutT>
__device__ __forceinline__ void pair_store16(OutT* row, const uint32_t* y, int col, int cols,
                                             bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = pack2<OutT>(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
  OutT* dst = row + col;
  if (wide && col + 16 <= cols) {
    asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {  // columns come in multiples of 8
    if (col + 8 <= cols) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    if (col + 16 <= cols) *reinterpret_cast<uint4*>(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// EPI: 0, TM_EPI_GELU_TANH or TM_EPI_SWIGLU.
template <int FORMAT, int EPI, typename OutT>
__global__ void __launch_bounds__(kPairThreads, 1)
    gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tm_a,
                         const __grid_constant__ CUtensorMap tm_b,
                         const __grid_constant__ CUtensorMap tm_as,
                         const __grid_constant__ CUtensorMap tm_bs, const Fp4Args g) {
  using L = PairLayout<FORMAT>;
  using S = ScaleGeom<FORMAT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1k(smem_raw);
  const PairBars bar = pair_bars(smem + L::kBarOffset);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1;  // in the cluster of 2; 0 = leader (issues the MMAs)
  const bool leader = rank == 0;
  const int tiles = g.num_m * g.num_n;
  const int pair = blockIdx.x >> 1;
  const int pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&bar.full[s], 1);
      mbar_init(&bar.empty[s], 1);
    }
    mbar_init(bar.acc_full, 1);
    mbar_init(bar.acc_free, 2 * kPairEpiWarps);  // both CTAs' epilogue warps
    *bar.abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
    tma_prefetch_desc(&tm_as);
    tma_prefetch_desc(&tm_bs);
  }
  if (warp == 1) {
    tmem_alloc_pair(bar.tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *bar.tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    uint32_t issued_mask = 0, issued_parity = 0;
    bool ok = true;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      int mb, nb;
      tile_coords(tile, g.num_m, g.num_n, mb, nb, 0, 0, g.group_n);
      for (int kb = 0; kb < g.kblocks; ++kb) {
        if (!mbar_wait_warp(&bar.empty[stage], phase ^ 1u, bar.abort_flag, g.status)) {
          ok = false;
          break;
        }
        issued_mask &= ~(1u << stage);
        if (elect_one()) {
          uint8_t* s = smem + stage * L::kStageBytes;
          uint8_t* scales = s + 2 * L::kHalfBytes;
          // the leader's `full` barrier counts the bytes landing in both CTAs
          if (leader) mbar_arrive_expect_tx(&bar.full[stage], 2 * L::kStageBytes);
          const uint32_t full = map_to_cta(smem_u32(&bar.full[stage]), 0);
          tma_load_2d_pair(&tm_a, full, s, kb * kRowBytes,
                           mb * kPairRows + static_cast<int>(rank) * 128);
          tma_load_2d_pair(&tm_b, full, s + L::kHalfBytes, kb * kRowBytes,
                           nb * kPairRows + static_cast<int>(rank) * 128);
          // own tokens' scales, and the whole tile's weight scales in both CTAs
          tma_load_2d_pair(&tm_as, full, scales, kb * (S::kBytes / 8),
                           mb * 2 + static_cast<int>(rank));
          tma_load_2d_pair(&tm_bs, full, scales + S::kBytes, kb * (S::kBytes / 8), nb * 2);
        }
        __syncwarp();
        issued_mask |= 1u << stage;
        issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (lane == 0) {
      if (!ok) {
        if (leader) {
          for (int s = 0; s < L::kStages; ++s)
            if (issued_mask & (1u << s))
              mbar_wait_drain(&bar.full[s], (issued_parity >> s) & 1u, g.status);
        } else {
          // this CTA's copies complete on the leader's barriers, which it cannot
          // poll; give any in-flight copy ample time to land
          const uint64_t t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // the whole warp runs the loop, one lane issues (see elect_one)
    if (leader) {
      const uint32_t tmem = __reduce_max_sync(0xffffffffu, tmem_base);
      const uint32_t smem0 = smem_u32(smem);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, issued_any = false;
      int i = 0;
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++i) {
        // the previous tile's sums are in the epilogue's registers
        if (i > 0 && !mbar_wait_warp(bar.acc_free, (i - 1) & 1, bar.abort_flag, g.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < g.kblocks; ++kb) {
          if (!mbar_wait_warp(&bar.full[stage], phase, bar.abort_flag, g.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem0 + stage * L::kStageBytes;
          const uint64_t a_desc = make_desc_kmajor_sw128(base);
          const uint64_t b_desc = make_desc_kmajor_sw128(base + L::kHalfBytes);
          const uint64_t as_desc = make_desc_scale_tile(base + 2 * L::kHalfBytes);
          const uint64_t bs_desc = make_desc_scale_tile(base + 2 * L::kHalfBytes + S::kBytes);
          const uint32_t col = tmem + kScaleCol + stage * (S::kTiles * kTileCols);
          const uint32_t more = kb != 0 ? 1u : 0u;
          const int steps = kblock_steps(g.K, kb);
          // descriptors count 16-byte units
          const auto copy = [&](int t) {
            tmem_copy_scale_tile<true>(col + kTileCols * t, as_desc + 32 * t);
            tmem_copy_scale_tile<true>(col + kTileCols * t + 4, bs_desc + 32 * t);
            tmem_copy_scale_tile<true>(col + kTileCols * t + 8, bs_desc + S::kBytes / 16 + 32 * t);
          };
          const auto multiply = [&](int k) {
            const int t = k / S::kStepsPerTile;
            umma_fp4<true, S::kBlock>(
                tmem, a_desc + 2 * k, b_desc + 2 * k,
                make_idesc_fp4(kPairRows, kPairRows, S::kE8m0, k % S::kStepsPerTile * 2),
                col + kTileCols * t, col + kTileCols * t + 4, k == 0 ? more : 1u);
          };
          if (steps == kKBlock / kMmaK) {
            if (elect_one()) {
#pragma unroll
              for (int t = 0; t < S::kTiles; ++t) copy(t);
#pragma unroll
              for (int k = 0; k < kKBlock / kMmaK; ++k) multiply(k);
              umma_commit_pair(&bar.empty[stage], 0x3);  // frees the stage in both CTAs
            }
          } else {  // the last k-block of a K that is not a multiple of 256
            if (elect_one()) {
              for (int t = 0; t * S::kStepsPerTile < steps; ++t) copy(t);
              for (int k = 0; k < steps; ++k) multiply(k);
              umma_commit_pair(&bar.empty[stage], 0x3);
            }
          }
          __syncwarp();
          issued_any = true;
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok && elect_one()) umma_commit_pair(bar.acc_full, 0x3);
        __syncwarp();
      }
      if (!ok && issued_any) {  // the last commit: the tensor pipe has drained
        const int last = stage == 0 ? L::kStages - 1 : stage - 1;
        mbar_wait_drain(&bar.empty[last], stage == 0 ? (phase ^ 1u) : phase, g.status);
      }
    }
    __syncwarp();
  } else {
    const uint32_t free_leader = map_to_cta(smem_u32(bar.acc_free), 0);
    uint8_t* region = smem + L::kEpiOffset + (warp - 2) * kPairRegion;
    const float* sb_s = reinterpret_cast<const float*>(region);
    const OutT* bias_s = reinterpret_cast<const OutT*>(region + kPairBiasCache);
    const int q = warp & 3;
    const int h = (warp - 2) >> 2;
    const int row_in_tile = static_cast<int>(rank) * 128 + q * 32;
    PairConsts next{};
    if (pair < tiles) {
      int mb, nb;
      tile_coords(pair, g.num_m, g.num_n, mb, nb, 0, 0, g.group_n);
      next = pair_consts<FORMAT, OutT>(g, nb, h, static_cast<int64_t>(mb) * kPairRows + row_in_tile + lane,
                                       lane);
    }
    int i = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++i) {
      int mb, nb;
      tile_coords(tile, g.num_m, g.num_n, mb, nb, 0, 0, g.group_n);
      __syncwarp();
      pair_consts_store<FORMAT, OutT>(region, next, lane);
      const float sa = next.sa;
      __syncwarp();
      if (tile + pairs < tiles) {  // the next tile's constants, a tile ahead
        int mb1, nb1;
        tile_coords(tile + pairs, g.num_m, g.num_n, mb1, nb1, 0, 0, g.group_n);
        next = pair_consts<FORMAT, OutT>(
            g, nb1, h, static_cast<int64_t>(mb1) * kPairRows + row_in_tile + lane, lane);
      }
      if (!mbar_wait(bar.acc_full, i & 1, bar.abort_flag, g.status)) break;
      tc_fence_after();
      const int64_t row = static_cast<int64_t>(mb) * kPairRows + row_in_tile + lane;
      const bool in_rows = row < g.M;
      const uint64_t sa2 = f32x2(sa, sa);
      OutT* out_row = static_cast<OutT*>(g.out) + row * g.ldo;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
      // the warp's 128 columns, then the accumulator belongs to the next tile
      uint32_t r[4][32];
#pragma unroll
      for (int k = 0; k < 4; ++k) tmem_ld_32x32b_x32(t_row + 128 * h + 32 * k, r[k]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(free_leader);
      const int col0 = nb * kPairRows + 128 * h;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < 32; j += 16) {
          pair_finish16<FORMAT, EPI, OutT>(r[k] + j, sa2, g.bias != nullptr, sb_s + 32 * k + j,
                                           bias_s + 32 * k + j);
          if (EPI != TM_EPI_SWIGLU && in_rows)
            pair_store16<OutT>(out_row, r[k] + j, col0 + 32 * k + j, g.N, g.wide);
        }
        if constexpr (EPI == TM_EPI_SWIGLU) {  // 16 gate columns, then the 16 up columns
#pragma unroll
          for (int j = 0; j < 16; ++j)
            r[k][j] = __float_as_uint(swiglu(__uint_as_float(r[k][j]), __uint_as_float(r[k][16 + j])));
          if (in_rows) pair_store16<OutT>(out_row, r[k], (col0 + 32 * k) / 2, g.N / 2, g.wide);
        }
      }
    }
  }

  tc_fence_before();
  cluster_sync();  // no CTA leaves while its peer may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ====================================================================== host
struct Fp4Device {
  int id, sms, max_pairs;
};

struct Fp4Operand {
  const uint8_t* codes;
  int64_t ld;  // bytes
  const uint8_t* blocks;
  int64_t rows;
};

bool encode_codes(CUtensorMap* map, const Fp4Operand& op, int64_t k, int box_rows) {
  return encode_tmap_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, op.codes, k / 2, op.rows, op.ld,
                        kRowBytes, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The scale tiles as 8-byte elements: a row is the tiles of 128 operand rows,
// a box the tiles of one k-block for `row_tiles` of them.
template <int FORMAT>
bool encode_scales(CUtensorMap* map, const Fp4Operand& op, int64_t k, int row_tiles) {
  const int64_t ktiles = round_up(k / fp4_block(FORMAT), 4) / 4;
  return encode_tmap_2d(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, op.blocks, ktiles * 64,
                        round_up(op.rows, 128) / 128, ktiles * 512,
                        ScaleGeom<FORMAT>::kBytes / 8, row_tiles, CU_TENSOR_MAP_SWIZZLE_NONE);
}

constexpr int kSmemBudget = 227 * 1024;

template <int TOK, int FORMAT, typename OutT>
int launch_small(const Fp4Operand& x, const Fp4Operand& w, Fp4Args args, int splits,
                 const Fp4Device& dev, cudaStream_t stream) {
  using L = SmallLayout<TOK, FORMAT>;
  args.num_m = (args.M + TOK - 1) / TOK;
  args.num_n = (args.N + kTileRows - 1) / kTileRows;
  if (splits > args.kblocks) return TM_ERR_UNSUPPORTED;
  const int longest = (args.kblocks + splits - 1) / splits;
  const int64_t ctas = static_cast<int64_t>(args.num_m) * args.num_n * splits;
  if (ctas > 0x7fffffffLL) return TM_ERR_TOO_LARGE;
  // two CTAs an SM (half the shared memory and TMEM each) once the grid has
  // more CTAs than SMs, else deeper rings
  const int budget = ctas > dev.sms ? kSmemBudget / 2 - 1024 : kSmemBudget;
  const int tmem_budget = ctas > dev.sms ? 256 : 512;
  int stages = kMaxStages;
  while (stages > 2 && (L::total(stages, splits) > budget || L::tmem_cols(stages) > tmem_budget))
    --stages;
  if (stages > longest) stages = longest < 2 ? 2 : longest;
  args.stages = stages;
  CUtensorMap tw, tx, tws, txs;
  if (!encode_codes(&tw, w, args.K, kTileRows) || !encode_codes(&tx, x, args.K, TOK) ||
      !encode_scales<FORMAT>(&tws, w, args.K, 1) || !encode_scales<FORMAT>(&txs, x, args.K, 1))
    return TM_ERR_CUDA;
  auto kernel = gemm_fp4_small_kernel<TOK, FORMAT, OutT>;
  const int smem = L::total(stages, splits);
  static std::atomic<bool> allowed[64] = {};
  if (!allow_smem(kernel, kSmemBudget, dev.id, allowed)) return TM_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  if (launch_with_pdl(cfg, attr, splits > 1 ? 1 : 0, kernel, tw, tx, tws, txs, args, splits) !=
      cudaSuccess)
    return TM_ERR_CUDA;
  return check_launch();
}

// Resident pairs of the pair kernel on a device (cached; its instances differ by
// a few KiB of shared memory only, one CTA an SM each).
int max_fp4_pairs(int device, int sms) {
  static std::atomic<int> known[64] = {};
  return known_per_device(known, device, [&] {
    auto kernel = gemm_fp4_pair_kernel<TM_FP4_NV, 0, __nv_bfloat16>;
    constexpr int smem = PairLayout<TM_FP4_NV>::kTotal;
    cudaError_t err =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(sms & ~1));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (err == cudaSuccess) err = cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg);
    if (err != cudaSuccess) {
      cudaGetLastError();  // a failed query must not poison later launches
      return 0;
    }
    return clusters;
  });
}

template <int FORMAT, int EPI, typename OutT>
int launch_pair_fp4(const Fp4Operand& x, const Fp4Operand& w, Fp4Args args, const Fp4Device& dev,
                    cudaStream_t stream) {
  using L = PairLayout<FORMAT>;
  if (dev.max_pairs <= 0) return TM_ERR_UNSUPPORTED;
  args.num_m = (args.M + kPairRows - 1) / kPairRows;
  args.num_n = (args.N + kPairRows - 1) / kPairRows;
  args.group_n = choose_group_n(args.num_n, kPairRows, kPairRows, args.K / 2);
  const int64_t tiles = static_cast<int64_t>(args.num_m) * args.num_n;
  if (tiles > 0x3fffffffLL) return TM_ERR_TOO_LARGE;
  args.wide = reinterpret_cast<uintptr_t>(args.out) % 32 == 0 && args.ldo % 16 == 0;
  CUtensorMap ta, tb, tas, tbs;
  if (!encode_codes(&ta, x, args.K, 128) || !encode_codes(&tb, w, args.K, 128) ||
      !encode_scales<FORMAT>(&tas, x, args.K, 1) || !encode_scales<FORMAT>(&tbs, w, args.K, 2))
    return TM_ERR_CUDA;
  auto kernel = gemm_fp4_pair_kernel<FORMAT, EPI, OutT>;
  static std::atomic<bool> allowed[64] = {};
  if (!allow_smem(kernel, L::kTotal, dev.id, allowed)) return TM_ERR_CUDA;
  const int pairs = static_cast<int>(tiles < dev.max_pairs ? tiles : dev.max_pairs);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = L::kTotal;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  if (launch_with_pdl(cfg, attr, 1, kernel, ta, tb, tas, tbs, args) != cudaSuccess)
    return TM_ERR_CUDA;
  return check_launch();
}

// Tile configurations: 32, 64, 128 = the small kernel with that many tokens a
// tile (32 and 64 only for M up to that); kPairTile = the pair kernel; 0 =
// chosen here.
constexpr int kPairTile = 1256;

struct Fp4Choice {
  int tile;
  int splits;
};

// Measured on a B200 (back to back, us): one wave of 128 x 128 tiles is ahead of
// the pair kernel (512 x 3072 x 3072: 7.6 against 8.9; 1003 x 1160 x 1376: 6.8
// against 9.6), two waves are behind (1024 x 3072 x 3072: 10.3 against 9.5; with GELU
// 256 x 12288 x 3072: 12.0 against 11.1, 512 x 12288 x 3072: 19.5 against 15.3), so
// more than 128 tokens take the small kernel only while its tiles fit the SMs at
// once.  Up to 128 tokens the weight is read once either way, by twice the CTAs (128 x
// 12288 x 3072: 7.9 against 9.5, with GELU 9.0 against 11.0).
//
// Slices of K: about 0.2 us a k-block, against 0.7 us and what grows with the
// slices and tokens for the partial sums; only while every slice has an SM of its
// own (1 x 3072 x 12288: 12.4, 7.6, 6.2 us with 1, 2, 4 slices; 48 x 3072 x 12288
// mxfp4: 12.5, 8.9, 7.0; 256 x 3072 x 3072: 7.1, 8.8, 13.7).
Fp4Choice pick_fp4(int64_t m, int64_t n, int kblocks, const Fp4Device& dev) {
  Fp4Choice c{m <= 32 ? 32 : m <= 64 ? 64 : 128, 1};
  const int64_t tiles = (m + c.tile - 1) / c.tile * ((n + kTileRows - 1) / kTileRows);
  if (m > 128 && tiles > dev.sms && dev.max_pairs > 0) return Fp4Choice{kPairTile, 1};
  const double tokens = static_cast<double>(m < c.tile ? m : c.tile);
  double best = 0.21 * kblocks;
  for (int s = 2; s <= kMaxSplits && s <= kblocks && tiles * s <= dev.sms; s *= 2) {
    const double t = 0.21 * ((kblocks + s - 1) / s) + 0.7 + 0.005 * tokens + 0.1 * s;
    if (t < best) {
      best = t;
      c.splits = s;
    }
  }
  return c;
}

template <int FORMAT, typename OutT>
int dispatch_fp4(const Fp4Operand& x, const Fp4Operand& w, const Fp4Args& args, Fp4Choice c,
                 const Fp4Device& dev, cudaStream_t stream) {
  switch (c.tile) {
    case 32: return launch_small<32, FORMAT, OutT>(x, w, args, c.splits, dev, stream);
    case 64: return launch_small<64, FORMAT, OutT>(x, w, args, c.splits, dev, stream);
    case 128: return launch_small<128, FORMAT, OutT>(x, w, args, c.splits, dev, stream);
    case kPairTile:
      if (args.epilogue & TM_EPI_GELU_TANH)
        return launch_pair_fp4<FORMAT, TM_EPI_GELU_TANH, OutT>(x, w, args, dev, stream);
      if (args.epilogue & TM_EPI_SWIGLU)
        return launch_pair_fp4<FORMAT, TM_EPI_SWIGLU, OutT>(x, w, args, dev, stream);
      return launch_pair_fp4<FORMAT, 0, OutT>(x, w, args, dev, stream);
    default: return TM_ERR_UNSUPPORTED;
  }
}

int scaled_mm_fp4_impl(void* out, int out_dtype, const uint8_t* a, const uint8_t* b,
                       const uint8_t* blocks_a, const uint8_t* blocks_b, const float* sa,
                       int64_t sa_numel, const float* sb, int64_t sb_numel, const void* bias,
                       int format, int64_t m, int64_t n, int64_t k, int64_t lda, int64_t ldb,
                       int64_t ldo, uint32_t epilogue, int tile, int splits, void* stream) {
  if (format != TM_FP4_NV && format != TM_FP4_MX) return TM_ERR_UNSUPPORTED;
  if (m < 0 || n <= 0 || k <= 0 || k % 32 != 0 || n % 8 != 0) return TM_ERR_SHAPE;
  if (lda < k / 2 || ldb < k / 2) return TM_ERR_SHAPE;
  if (epilogue & ~(TM_EPI_GELU_TANH | TM_EPI_SWIGLU)) return TM_ERR_UNSUPPORTED;
  if ((epilogue & TM_EPI_GELU_TANH) && (epilogue & TM_EPI_SWIGLU)) return TM_ERR_UNSUPPORTED;
  if ((epilogue & TM_EPI_SWIGLU) && n % 64 != 0) return TM_ERR_SHAPE;
  if (ldo < ((epilogue & TM_EPI_SWIGLU) ? n / 2 : n)) return TM_ERR_SHAPE;
  if (out_dtype != TM_DTYPE_BF16 && out_dtype != TM_DTYPE_FP16) return TM_ERR_DTYPE;
  if (m == 0) return TM_OK;
  if (m > 0x7fffffffLL - 256 || n > 0x7fffffffLL - 256 || k > (1ll << 30)) return TM_ERR_TOO_LARGE;
  if (!out || !a || !b || !blocks_a || !blocks_b) return TM_ERR_NULL_POINTER;
  if (sa && sa_numel != 1 && sa_numel != m) return TM_ERR_SHAPE;
  if (sb && sb_numel != 1 && sb_numel != n) return TM_ERR_SHAPE;
  if (format == TM_FP4_MX && (sa || sb)) return TM_ERR_UNSUPPORTED;
  if (format == TM_FP4_NV && (!sa || !sb)) return TM_ERR_NULL_POINTER;
  if (!aligned16(a) || !aligned16(b) || !aligned16(blocks_a) || !aligned16(blocks_b) ||
      !aligned16(out) || lda % 16 != 0 || ldb % 16 != 0 || ldo % 8 != 0)
    return TM_ERR_ALIGNMENT;
  const int device = current_device();
  const int sms = sm_count(device);
  if (device < 0 || sms <= 0) return TM_ERR_CUDA;
  Fp4Args args{};
  args.sa = sa;
  args.sb = sb;
  args.sa_per_row = sa_numel == m;
  args.sb_per_col = sb_numel == n;
  args.bias = bias;
  args.out = out;
  args.ldo = ldo;
  args.M = static_cast<int>(m);
  args.N = static_cast<int>(n);
  args.K = static_cast<int>(k);
  args.kblocks = static_cast<int>((k + kKBlock - 1) / kKBlock);
  args.epilogue = epilogue;
  args.status = device_status_ptr(device);
  const Fp4Device dev{device, sms, max_fp4_pairs(device, sms)};
  Fp4Choice c{tile, splits};
  if (tile == 0) {
    c = pick_fp4(m, n, args.kblocks, dev);
  } else {
    if (splits != 1 && splits != 2 && splits != 4 && splits != 8) return TM_ERR_UNSUPPORTED;
    if ((tile < 128 && m > tile) || (tile == kPairTile && splits != 1)) return TM_ERR_UNSUPPORTED;
  }
  const Fp4Operand x{a, lda, blocks_a, m}, w{b, ldb, blocks_b, n};
  const cudaStream_t st = as_stream(stream);
  const bool bf16 = out_dtype == TM_DTYPE_BF16;
  if (format == TM_FP4_NV)
    return bf16 ? dispatch_fp4<TM_FP4_NV, __nv_bfloat16>(x, w, args, c, dev, st)
                : dispatch_fp4<TM_FP4_NV, __half>(x, w, args, c, dev, st);
  return bf16 ? dispatch_fp4<TM_FP4_MX, __nv_bfloat16>(x, w, args, c, dev, st)
              : dispatch_fp4<TM_FP4_MX, __half>(x, w, args, c, dev, st);
}

}  // namespace
}  // namespace tmw

extern "C" {

int tm_scaled_mm_fp4(void* out, int out_dtype, const uint8_t* a, const uint8_t* b,
                     const uint8_t* block_scales_a, const uint8_t* block_scales_b,
                     const float* scale_a, int64_t scale_a_numel, const float* scale_b,
                     int64_t scale_b_numel, const void* bias, int format, int64_t m, int64_t n,
                     int64_t k, int64_t lda, int64_t ldb, int64_t ldo, uint32_t epilogue,
                     void* stream) {
  return tmw::scaled_mm_fp4_impl(out, out_dtype, a, b, block_scales_a, block_scales_b, scale_a,
                                 scale_a_numel, scale_b, scale_b_numel, bias, format, m, n, k, lda,
                                 ldb, ldo, epilogue, 0, 1, stream);
}

int tm_scaled_mm_fp4_tile(void* out, int out_dtype, const uint8_t* a, const uint8_t* b,
                          const uint8_t* block_scales_a, const uint8_t* block_scales_b,
                          const float* scale_a, int64_t scale_a_numel, const float* scale_b,
                          int64_t scale_b_numel, const void* bias, int format, int64_t m, int64_t n,
                          int64_t k, int64_t lda, int64_t ldb, int64_t ldo, uint32_t epilogue,
                          int tile, int splits, void* stream) {
  return tmw::scaled_mm_fp4_impl(out, out_dtype, a, b, block_scales_a, block_scales_b, scale_a,
                                 scale_a_numel, scale_b, scale_b_numel, bias, format, m, n, k, lda,
                                 ldb, ldo, epilogue, tile, splits, stream);
}

}  // extern "C"
