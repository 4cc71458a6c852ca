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
// by the MMA thread (tcgen05.cp, in order with its MMAs).  Two TMEM scale
// buffers alternate; one is written again only after the MMAs that read it
// have completed.
//
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

// The value of one output before rounding (SwiGLU pairs are combined by the caller).
__device__ __forceinline__ float activate(float y, uint32_t epilogue) {
  return (epilogue & TM_EPI_GELU_TANH) ? gelu_tanh(y) : y;
}

__device__ __forceinline__ float swiglu(float g, float u) {
  return __fmul_rn(__fmul_rn(g, sigmoid_f32(g)), u);
}

__device__ __forceinline__ uint8_t* align1k(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) &
                                    ~static_cast<uintptr_t>(1023));
}

// ====================================================================== small
constexpr int kSmallThreads = 192;  // producer, MMA, four epilogue warps
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
  static constexpr int kBarBytes = 256;
  static constexpr int total(int stages, int splits) {
    return 1024 + stages * kStageBytes + kBarBytes + (splits > 1 ? kReduceBytes : 0);
  }
  // TMEM columns: the accumulator, then two buffers of scale tiles (4 columns each)
  static constexpr uint32_t kScaleCol = TOK;
  static constexpr uint32_t kScaleBuf = 2 * 4 * S::kTiles;
  static constexpr uint32_t kTmemCols = TOK + 2 * kScaleBuf <= 128 ? 128 : 256;
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

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Store the outputs of token `m` held one weight row per lane: `n` is this
// lane's output row, y its value before the activation.
template <typename OutT>
__device__ __forceinline__ void store_token(const Fp4Args& g, int64_t m, int n, float y) {
  OutT* row = static_cast<OutT*>(g.out) + m * g.ldo;
  if (g.epilogue & TM_EPI_SWIGLU) {
    // weight rows come as 16 gate rows, then the 16 matching up rows
    const float u = __shfl_down_sync(0xffffffffu, y, 16);
    if ((threadIdx.x & 16) == 0 && n < g.N)
      row[(n >> 5) * 16 + (n & 15)] = from_f32<OutT>(swiglu(y, u));
  } else {
    if (n < g.N) row[n] = from_f32<OutT>(activate(y, g.epilogue));
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
  float* reduce = reinterpret_cast<float*>(smem + g.stages * L::kStageBytes + L::kBarBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int slice = blockIdx.x % splits;
  const int tile = blockIdx.x / splits;
  const int nb = tile % g.num_n;
  const int mb = tile / g.num_n;
  // even slices, none empty (splits <= kblocks)
  const int kb0 = static_cast<int>(static_cast<int64_t>(slice) * g.kblocks / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(slice + 1) * g.kblocks / splits);

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
    tmem_alloc(bar.tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  if (splits > 1)
    cluster_sync();  // every slice is running before any writes to another's shared memory
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *bar.tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued_mask = 0, issued_parity = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&bar.empty[stage], phase ^ 1u, bar.abort_flag, g.status)) {
          ok = false;
          break;
        }
        issued_mask &= ~(1u << stage);
        uint8_t* s = smem + stage * L::kStageBytes;
        mbar_arrive_expect_tx(&bar.full[stage], L::kStageBytes);
        tma_load_2d(&tm_w, &bar.full[stage], s, kb * kRowBytes, nb * kTileRows);
        tma_load_2d(&tm_ws, &bar.full[stage], s + L::kWBytes + L::kXBytes, kb * (S::kBytes / 8), nb);
        tma_load_2d(&tm_x, &bar.full[stage], s + L::kWBytes, kb * kRowBytes, mb * TOK);
        tma_load_2d(&tm_xs, &bar.full[stage], s + L::kWBytes + L::kXBytes + S::kBytes,
                    kb * (S::kBytes / 8), mb);  // TOK = 128, or a single token tile
        issued_mask |= 1u << stage;
        issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == g.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {
        for (int s = 0; s < g.stages; ++s)
          if (issued_mask & (1u << s))
            mbar_wait_drain(&bar.full[s], (issued_parity >> s) & 1u, g.status);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int last = -1, before = -1;  // stages of the previous k-block and of the one before it
      uint32_t last_phase = 0, before_phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        // the scale buffer was last read two k-blocks ago
        if (before >= 0 &&
            !mbar_wait(&bar.empty[before], before_phase, bar.abort_flag, g.status)) {
          ok = false;
          break;
        }
        if (!mbar_wait(&bar.full[stage], phase, bar.abort_flag, g.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t w_addr = smem_u32(smem + stage * L::kStageBytes);
        const uint32_t x_addr = w_addr + L::kWBytes;
        const uint32_t ws_addr = x_addr + L::kXBytes;
        const uint32_t xs_addr = ws_addr + S::kBytes;
        const uint32_t ws_col = tmem_base + L::kScaleCol + ((kb - kb0) & 1) * L::kScaleBuf;
        const uint32_t xs_col = ws_col + 4 * S::kTiles;
        const int steps = kblock_steps(g.K, kb);
        for (int t = 0; t * S::kStepsPerTile < steps; ++t) {
          tmem_copy_scale_tile<false>(ws_col + 4 * t, make_desc_scale_tile(ws_addr + 512 * t));
          tmem_copy_scale_tile<false>(xs_col + 4 * t, make_desc_scale_tile(xs_addr + 512 * t));
        }
        for (int k = 0; k < steps; ++k) {
          const int t = k / S::kStepsPerTile, id = k % S::kStepsPerTile * 2;
          umma_fp4<false, S::kBlock>(tmem_base, make_desc_kmajor_sw128(w_addr + k * 32),
                                     make_desc_kmajor_sw128(x_addr + k * 32),
                                     make_idesc_fp4(kTileRows, TOK, S::kE8m0, id), ws_col + 4 * t,
                                     xs_col + 4 * t, (kb > kb0 || k > 0) ? 1u : 0u);
        }
        umma_commit(&bar.empty[stage]);
        before = last;
        before_phase = last_phase;
        last = stage;
        last_phase = phase;
        if (++stage == g.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok)
        umma_commit(bar.acc);
      else if (last >= 0)
        mbar_wait_drain(&bar.empty[last], last_phase, g.status);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int n = nb * kTileRows + q * 32 + lane;  // this lane's weight row
    const float sb = n < g.N ? (g.sb == nullptr ? 1.f : __ldg(g.sb + (g.sb_per_col ? n : 0))) : 0.f;
    const float bias = (g.bias != nullptr && n < g.N)
                           ? out_to_f32<OutT>(static_cast<const OutT*>(g.bias)[n])
                           : 0.f;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const int tokens = min(TOK, g.M - mb * TOK);
    const bool ok = mbar_wait(bar.acc, 0, bar.abort_flag, g.status);
    tc_fence_after();
    const auto token_scale = [&](int64_t m) {
      return g.sa == nullptr ? 1.f : __ldg(g.sa + (g.sa_per_row ? m : 0));
    };
    if (splits == 1) {
      if (ok) {
#pragma unroll 1
        for (int c = 0; c < tokens; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t_row + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (c + j < tokens) {  // the same for the whole warp
              const int64_t m = static_cast<int64_t>(mb) * TOK + c + j;
              store_token<OutT>(g, m, n,
                                __fmaf_rn(token_scale(m), __fmul_rn(sb, __uint_as_float(r[j])), bias));
            }
          }
        }
      }
    } else {
      // Slice j of the cluster finishes tokens [j, j + 1) * per: send it this
      // slice's sums of those tokens, [slice][token][weight row].
      const int per = TOK / splits;
      const uint32_t mine = smem_u32(reduce);
#pragma unroll 1
      for (int c = 0; c < TOK; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_row + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int to = (c + j) / per, at = (c + j) % per;
          const uint32_t local = mine + ((slice * per + at) * kTileRows + q * 32 + lane) * 4;
          st_cluster_f32(map_to_cta(local, to), ok ? __uint_as_float(r[j]) : __int_as_float(0x7fffffff));
        }
      }
    }
  }

  tc_fence_before();
  if (splits > 1) {
    cluster_sync();  // every slice's sums have arrived
    if (warp >= 2) {
      const int q = warp & 3;
      const int row = q * 32 + lane;
      const int n = nb * kTileRows + row;
      const float sb = n < g.N ? (g.sb == nullptr ? 1.f : __ldg(g.sb + (g.sb_per_col ? n : 0))) : 0.f;
      const float bias = (g.bias != nullptr && n < g.N)
                             ? out_to_f32<OutT>(static_cast<const OutT*>(g.bias)[n])
                             : 0.f;
      const int per = TOK / splits;
      for (int at = 0; at < per; ++at) {
        const int64_t m = static_cast<int64_t>(mb) * TOK + slice * per + at;
        if (m >= g.M) break;
        float acc = 0.f;
        for (int s = 0; s < splits; ++s) acc += reduce[(s * per + at) * kTileRows + row];
        const float sa = g.sa == nullptr ? 1.f : __ldg(g.sa + (g.sa_per_row ? m : 0));
        store_token<OutT>(g, m, n, __fmaf_rn(sa, __fmul_rn(sb, acc), bias));
      }
    }
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

// ====================================================================== host
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
                 cudaStream_t stream) {
  using L = SmallLayout<TOK, FORMAT>;
  args.num_m = (args.M + TOK - 1) / TOK;
  args.num_n = (args.N + kTileRows - 1) / kTileRows;
  if (splits > args.kblocks) return TM_ERR_UNSUPPORTED;
  const int longest = (args.kblocks + splits - 1) / splits;
  const int64_t ctas = static_cast<int64_t>(args.num_m) * args.num_n * splits;
  if (ctas > 0x7fffffffLL) return TM_ERR_TOO_LARGE;
  // two CTAs an SM where that leaves each at least three stages
  int stages = kMaxStages;
  while (stages > 3 && L::total(stages, splits) > kSmemBudget / 2 - 1024) --stages;
  if (stages > longest) stages = longest < 2 ? 2 : longest;
  args.stages = stages;
  CUtensorMap tw, tx, tws, txs;
  if (!encode_codes(&tw, w, args.K, kTileRows) || !encode_codes(&tx, x, args.K, TOK) ||
      !encode_scales<FORMAT>(&tws, w, args.K, 1) || !encode_scales<FORMAT>(&txs, x, args.K, 1))
    return TM_ERR_CUDA;
  auto kernel = gemm_fp4_small_kernel<TOK, FORMAT, OutT>;
  const int smem = L::total(stages, splits);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget) !=
      cudaSuccess)
    return TM_ERR_CUDA;
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

// Tile configurations: 32, 64, 128 = the small kernel with that many tokens a
// tile (32 and 64 only for M up to that); 0 = chosen here.
struct Fp4Choice {
  int tile;
  int splits;
};

Fp4Choice pick_fp4(int64_t m, int64_t n, int kblocks, int sms) {
  Fp4Choice c{m <= 32 ? 32 : m <= 64 ? 64 : 128, 1};
  const int64_t tiles = (m + c.tile - 1) / c.tile * ((n + kTileRows - 1) / kTileRows);
  while (c.splits < 8 && tiles * c.splits * 2 <= 2 * sms && kblocks >= 4 * c.splits) c.splits *= 2;
  return c;
}

template <int FORMAT, typename OutT>
int dispatch_fp4(const Fp4Operand& x, const Fp4Operand& w, const Fp4Args& args, Fp4Choice c,
                 cudaStream_t stream) {
  switch (c.tile) {
    case 32: return launch_small<32, FORMAT, OutT>(x, w, args, c.splits, stream);
    case 64: return launch_small<64, FORMAT, OutT>(x, w, args, c.splits, stream);
    case 128: return launch_small<128, FORMAT, OutT>(x, w, args, c.splits, stream);
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
  if (m > 0x7fffffffLL - 256 || n > 0x7fffffffLL - 256 || k > 0x7fffffffLL) return TM_ERR_TOO_LARGE;
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
  Fp4Choice c{tile, splits};
  if (tile == 0) {
    c = pick_fp4(m, n, args.kblocks, sms);
  } else {
    if (splits != 1 && splits != 2 && splits != 4 && splits != 8) return TM_ERR_UNSUPPORTED;
    if (tile < 128 && m > tile) return TM_ERR_UNSUPPORTED;
  }
  const Fp4Operand x{a, lda, blocks_a, m}, w{b, ldb, blocks_b, n};
  const cudaStream_t st = as_stream(stream);
  const bool bf16 = out_dtype == TM_DTYPE_BF16;
  if (format == TM_FP4_NV)
    return bf16 ? dispatch_fp4<TM_FP4_NV, __nv_bfloat16>(x, w, args, c, st)
                : dispatch_fp4<TM_FP4_NV, __half>(x, w, args, c, st);
  return bf16 ? dispatch_fp4<TM_FP4_MX, __nv_bfloat16>(x, w, args, c, st)
              : dispatch_fp4<TM_FP4_MX, __half>(x, w, args, c, st);
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
