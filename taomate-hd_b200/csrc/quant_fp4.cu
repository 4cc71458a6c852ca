// Quantisation to the 4-bit block formats (fp4.cuh), its inverse, and the
// adaLN producers fused into it.
//
//   TM_FP4_NV  o = fp32(max(max |x|, 2^-100) / 2688) for the row (2688 = 448 x 6, the
//              largest e4m3 times the largest e2m1), or a given o;
//              s = e4m3(m / (6 o)) for the block maximum m, at most 448;
//              q = e2m1(x / (o s)), 0 where s = 0
//   TM_FP4_MX  s = 2^(floor(log2 m) - 2), at least 2^-127;  q = e2m1(x / s)
//
// Every quotient is rounded once, from its exact value, to nearest with ties
// to even.  For TM_FP4_MX that is free (s is a power of two).  For TM_FP4_NV
// the fp32 product y = x * (1 / (o s)) is off by up to 2^-22, and 16-bit data
// meets the borders between two codes, or passes them by less than that, once
// in a thousand elements or two.
//   16-bit rows with their own scale: were o exactly a / 2688, x / (o s) and a
// border t would be equal, or apart by at least 1 / (105 2^p) of t: they are
// 21 X 2^i and T S A 2^j with X, A below 2^p (p = 8 bf16, 11 fp16), S <= 15 and
// T <= 7 odd.  The rounding of o moves all the equal ones to the same side, by
// at most 2^-24, and the sign of a - 2688 o (one fma, exact) says which.  So y
// times 1 +- 2^-20 rounds to the right code: the factor outweighs the arithmetic
// (2^-22) and the shift, and is far below 1 / (105 2^11) = 2^-17.7.  The block
// scale's borders, 7 M 2^i against T A 2^j with T <= 31, are further apart still.
// Rows whose o is exact (true ties) take the general way.
//   In general y (1 - 2^-21) and y (1 + 2^-21) are both converted: where the
// codes agree no border lies between them and the code is right; where they
// differ the border t decides by the sign of x - (t s) o, which one fma gives
// exactly (t s has at most 7 bits, so the product is not rounded before the
// subtraction).  The scale's rounding is decided the same way, with its border
// t: m - (6 t) o.  Taken for every row, 20480 x
// 3072 bf16 needs 36 us in place of 30; with a given scale it is 33.
//
// The kernels are bound by HBM: 2 bytes read and 0.56 written per bf16 element.
// As in the int8 kernels a group of 32..256 threads owns a row and holds it in
// registers between the row maximum and the conversion; a thread's unit is 16
// elements (32 contiguous bytes of bf16), i.e. a whole TM_FP4_NV block and half
// a TM_FP4_MX one, so the block maximum needs no shuffle or one.  Maxima are
// taken on the bits of |x| as unsigned integers, which order NaN above inf
// above every finite value: one reduction finds the maximum and what is not
// finite.
#include "fp4.cuh"
#include "rows.cuh"

namespace tmw {
namespace {

enum Fp4Kind : int {
  kNvDynamic = 0,  // row scale from the row's maximum
  kNvGiven = 1,    // one given scale
  kMx = 2
};

struct Fp4Params : QuantParams {
  uint8_t* codes;       // [rows, cols / 2]
  uint8_t* blocks;      // tiles
  int64_t ktiles;       // tiles along a row
  int64_t padded_rows;  // rows, rounded up to whole tiles
};

constexpr uint32_t kInfBits = 0x7f800000u;

// Eight values -> eight e2m1 codes, v[0] in the low half of the first byte;
// to nearest, ties to even, at most 6.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Two values -> two e4m3 bytes, `lo` in the low one; at most 448.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Value of an e2m1 magnitude code 0..7.
__device__ __forceinline__ float e2m1_value(uint32_t c) {
  // codes 2..7 have the bits of an fp32 number's low exponent and top mantissa
  return c < 2 ? 0.5f * static_cast<float>(c)
               : __uint_as_float(((c >> 1) + 126u) << 23 | (c & 1u) << 22);
}

__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float kBelow = 1.0f - 4.76837158203125e-07f;  // 1 - 2^-21
constexpr float kAbove = 1.0f + 4.76837158203125e-07f;

// e4m3 scale byte of a block with maximum m under the outer scale o;
// inv6o is 1 / (6 o) to 2^-22.
__device__ __forceinline__ uint32_t nv_scale_byte(float m, float o, float inv6o) {
  const float z = __fmul_rn(m, inv6o);
  const uint32_t pair = e4m3x2(__fmul_rn(z, kBelow), __fmul_rn(z, kAbove));
  const uint32_t lo = pair & 0xffu, hi = pair >> 8;
  if (lo == hi) return lo;
  const float2 v = e4m3x2_to_f32(pair);
  const float d = __fmaf_rn(-3.0f * (v.x + v.y), o, m);  // m - 6 (lo + hi) / 2 o, exact sign
  return d > 0.0f || (d == 0.0f && (lo & 1u)) ? hi : lo;
}

// ---- a thread's 16 elements ----
template <typename T>
struct Unit {  // 16-bit types: 16 values in 32 bytes
  uint4 raw[2];
};
template <>
struct Unit<float> {
  uint4 raw[4];
};

// Value j (0..7) of a half unit, picked at run time without indexing memory.
template <typename T>
__device__ __forceinline__ float unit_value(const Unit<T>& u, int half, int j) {
  if constexpr (sizeof(T) == 2) {
    const uint4& r = u.raw[half];
    const uint32_t w = j < 4 ? (j < 2 ? r.x : r.y) : (j < 6 ? r.z : r.w);
    const uint16_t e = static_cast<uint16_t>(j & 1 ? w >> 16 : w);
    return to_f32<T>(*reinterpret_cast<const T*>(&e));
  } else {
    const uint4 &a = u.raw[2 * half], &b = u.raw[2 * half + 1];
    const uint32_t x = j < 4 ? a.x : b.x, y = j < 4 ? a.y : b.y;
    const uint32_t z = j < 4 ? a.z : b.z, w = j < 4 ? a.w : b.w;
    return __uint_as_float((j & 2) ? (j & 1 ? w : z) : (j & 1 ? y : x));
  }
}

// Decide the codes that differ between lo and hi (the conversions from just
// below and just above a value): the value lies within 2^-21 of a border.
template <typename T>
__device__ __forceinline__ uint32_t resolve8(uint32_t lo, uint32_t hi, const Unit<T>& u, int half,
                                             float s, float o) {
  uint32_t left = lo ^ hi;
  do {
    const int j = (__ffs(left) - 1) >> 2;
    const uint32_t a = (lo >> (4 * j)) & 7u, b = (hi >> (4 * j)) & 7u;
    const float ts = __fmul_rn(0.5f * (e2m1_value(a) + e2m1_value(b)), s);
    const float d = __fmaf_rn(-ts, o, fabsf(unit_value(u, half, j)));
    if (d > 0.0f || (d == 0.0f && (a & 1u))) lo = (lo & ~(7u << (4 * j))) | (b << (4 * j));
    left &= ~(15u << (4 * j));
  } while (left != 0u);
  return lo;
}

// Eight codes of a half unit under block scale s and outer scale o; inv = 1 / (o s).
template <typename T>
__device__ __forceinline__ uint32_t nv_codes8(const Unit<T>& u, int half, const float (&x)[8],
                                              float inv, float s, float o) {
  const uint64_t below = f32x2(__fmul_rn(inv, kBelow), __fmul_rn(inv, kBelow));
  const uint64_t above = f32x2(__fmul_rn(inv, kAbove), __fmul_rn(inv, kAbove));
  float a[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint64_t v = f32x2(x[j], x[j + 1]);
    f32x2_split(mul_f32x2(v, below), a[j], a[j + 1]);
    f32x2_split(mul_f32x2(v, above), b[j], b[j + 1]);
  }
  const uint32_t lo = e2m1x8(a), hi = e2m1x8(b);
  return lo == hi ? lo : resolve8(lo, hi, u, half, s, o);
}

// Eight codes of x * inv.
__device__ __forceinline__ uint32_t scaled_codes8(const float (&x)[8], float inv) {
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = __fmul_rn(x[j], inv);
  return e2m1x8(a);
}

__device__ __forceinline__ uint4 ld_nc_u32x4(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// 32 bytes that no kernel in flight writes; `wide`: the address is a multiple of
// 32 (one load), else of 16.  Volatile, so that it stays behind griddep_wait(); the
// loads of an unrolled loop are still issued ahead of its stores (timed: no difference).
__device__ __forceinline__ void ld_stream32(const void* p, bool wide, uint4& a, uint4& b) {
  if (wide) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z),
                   "=r"(b.w)
                 : "l"(p));
  } else {
    a = ld_nc_u32x4(p);
    b = ld_nc_u32x4(static_cast<const uint8_t*>(p) + 16);
  }
}

// 32 bytes of a table row that other rows may share: kept in L1.
__device__ __forceinline__ void ld_table32(const void* p, bool wide, uint4& a, uint4& b) {
  if (wide) {
    asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z),
                   "=r"(b.w)
                 : "l"(p));
  } else {
    a = ld_nc_u32x4(p);
    b = ld_nc_u32x4(static_cast<const uint8_t*>(p) + 16);
  }
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// 32 bytes to a multiple of 32.
__device__ __forceinline__ void st_global32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y),
               "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void load_unit(Unit<T>& u, const T* p, bool wide) {
#pragma unroll
  for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h)
    ld_stream32(reinterpret_cast<const uint8_t*>(p) + 32 * h, wide, u.raw[2 * h], u.raw[2 * h + 1]);
}

template <typename T>
__device__ __forceinline__ void clear_unit(Unit<T>& u) {
#pragma unroll
  for (int h = 0; h < static_cast<int>(sizeof(T)); ++h) u.raw[h] = make_uint4(0u, 0u, 0u, 0u);
}

// Element by element: any alignment (16 elements from p).
template <typename T>
__device__ __forceinline__ void load_unit_scalar(Unit<T>& u, const T* p) {
  T* e = reinterpret_cast<T*>(u.raw);
#pragma unroll
  for (int j = 0; j < 16; ++j) e[j] = p[j];
}

// Largest |x| of the unit as the bits of an fp32 number (NaN > inf > finite).
template <typename T>
__device__ __forceinline__ uint32_t unit_max_bits(const Unit<T>& u) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(u.raw);
  if constexpr (sizeof(T) == 2) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
    const uint16_t top = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
    return __float_as_uint(to_f32<T>(*reinterpret_cast<const T*>(&top))) & 0x7fffffffu;
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max(m, w[j] & 0x7fffffffu);
    return m;
  }
}

template <typename T>
__device__ __forceinline__ void unit_values(const Unit<T>& u, int half, float (&v)[8]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u.raw[half]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  } else {
    const T* e = reinterpret_cast<const T*>(u.raw) + 8 * half;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(e[j]);
  }
}

// Wait for the threads of this row's group (tpr <= 32: a warp, nothing to wait
// for).  A barrier of its own for each group: the rows of a block do not wait
// for one another.
__device__ __forceinline__ void group_sync(int tpr) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / tpr), "r"(tpr)
               : "memory");
}

// Shared words of a block's reductions: a slot per warp for each, written once.
struct GroupRed {
  double sum[2][8];
  uint32_t top[8];
};

// Largest of one value per thread over the row's group.
__device__ __forceinline__ uint32_t group_max_bits(uint32_t v, int tpr, GroupRed& red) {
  v = __reduce_max_sync(0xffffffffu, v);  // a group is whole warps
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5;
    const int wpr = tpr >> 5;
    const int first = warp / wpr * wpr;
    if ((threadIdx.x & 31) == 0) red.top[warp] = v;
    group_sync(tpr);
    v = red.top[first];
    for (int w = 1; w < wpr; ++w) v = max(v, red.top[first + w]);
  }
  return v;
}

// Sum of one double per thread over the row's group, the same bits in all of its
// threads; `slots` is red.sum[0] or, for a second sum, red.sum[1].
__device__ __forceinline__ double group_sum(double v, int tpr, double* slots) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5;
    const int wpr = tpr >> 5;
    const int first = warp / wpr * wpr;
    if ((threadIdx.x & 31) == 0) slots[warp] = v;
    group_sync(tpr);
    v = slots[first];
    for (int w = 1; w < wpr; ++w) v += slots[first + w];
  }
  return v;
}

// What a row's conversion needs.
struct RowScale {
  float o;      // outer scale (TM_FP4_NV)
  float inv6o;  // 1 / (6 o) to 2^-22
  float nudge;  // 1 +- 2^-20 (above); 0: the general way
  bool bad;     // the row holds an inf or a NaN (its own scale is NaN, blocks and codes 0);
                // or the given scale is out of range (block scales NaN, codes 0)
};

__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
  RowScale r;
  r.bad = max_bits >= kInfBits;
  const float a = fmaxf(__uint_as_float(max_bits), 7.888609052210118e-31f);  // 2^-100
  r.o = r.bad ? __int_as_float(0x7fffffff) : __fdiv_rn(a, 2688.0f);
  r.inv6o = rcp_approx(__fmul_rn(6.0f, r.o));
  const float d = __fmaf_rn(-2688.0f, r.o, a);  // o below (d > 0) or above a / 2688
  constexpr float kNudge = 9.5367431640625e-07f;  // 2^-20
  r.nudge = d > 0.0f ? 1.0f + kNudge : d < 0.0f ? 1.0f - kNudge : 0.0f;
  return r;
}

// From 2^-110 to 2^110 every product of o with a code, a block scale and a border is
// a normal fp32 number.  Others (a scale of 0, say, or a NaN) are refused where they
// can be seen without a copy to the host: here, by NaN for the whole tensor.
__device__ __forceinline__ RowScale given_scale(float o) {
  return RowScale{o, rcp_approx(__fmul_rn(6.0f, o)), 0.0f, !(o >= 0x1p-110f && o <= 0x1p110f)};
}

// Convert one unit (16 elements, block maximum `m_bits` as fp32 bits) and
// return its scale byte; codes to c[0..1].
template <typename T, int KIND>
__device__ __forceinline__ uint32_t convert_unit(const Unit<T>& u, uint32_t m_bits,
                                                 const RowScale& rs, uint32_t (&c)[2]) {
  c[0] = c[1] = 0u;
  float v[8];
  if constexpr (KIND == kMx) {
    if (m_bits >= kInfBits) return 0xffu;  // e8m0 NaN
    const int e = static_cast<int>(m_bits >> 23) - 2;  // an fp32 subnormal maximum: 2^-127
    const uint32_t byte = static_cast<uint32_t>(max(e, 0));
    // 2^(127 - byte); byte <= 252, so the factor is a normal number
    const float inv = __uint_as_float((254u - byte) << 23);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unit_values(u, h, v);
      c[h] = scaled_codes8(v, inv);  // exact products, or far below the first border
    }
    return byte;
  } else {
    if (KIND == kNvGiven && (m_bits >= kInfBits || rs.bad)) return 0x7fu;  // e4m3 NaN
    if (rs.bad) return 0u;
    if (KIND == kNvDynamic && sizeof(T) == 2 && rs.nudge != 0.0f) {  // the same for the whole row
      const float z = __fmul_rn(__uint_as_float(m_bits), __fmul_rn(rs.inv6o, rs.nudge));
      const uint32_t byte = e4m3x2(z, 0.0f) & 0xffu;
      if (byte == 0u) return 0u;
      const float s = e4m3x2_to_f32(byte).x;
      const float inv = __fmul_rn(rcp_approx(__fmul_rn(rs.o, s)), rs.nudge);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        unit_values(u, h, v);
        c[h] = scaled_codes8(v, inv);
      }
      return byte;
    }
    const uint32_t byte = nv_scale_byte(__uint_as_float(m_bits), rs.o, rs.inv6o);
    if (byte == 0u) return 0u;
    const float s = e4m3x2_to_f32(byte).x;
    const float inv = rcp_approx(__fmul_rn(rs.o, s));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unit_values(u, h, v);
      c[h] = nv_codes8(u, h, v, inv, s, rs.o);
    }
    return byte;
  }
}

// Where a row's results go: the row's part of every address.
struct RowOut {
  uint8_t* codes;
  uint8_t* blocks;
};

__device__ __forceinline__ RowOut row_out(const Fp4Params& p, int64_t row) {
  return RowOut{p.codes + row * (p.cols / 2), p.blocks + fp4_scale_offset(row, 0, p.ktiles)};
}

// Scale byte of a unit; TM_FP4_MX blocks span two units (adjacent lanes), the
// even one stores it.
template <int KIND>
__device__ __forceinline__ void store_scale(const RowOut& out, int unit, uint32_t byte) {
  const int block = KIND == kMx ? unit >> 1 : unit;
  if (KIND != kMx || (unit & 1) == 0)
    out.blocks[(block >> 2) * 512 + (block & 3)] = static_cast<uint8_t>(byte);
}

template <int KIND>
__device__ __forceinline__ void store_unit(const RowOut& out, int unit, const uint32_t (&c)[2],
                                           uint32_t byte) {
  *reinterpret_cast<uint2*>(out.codes + unit * 8) = make_uint2(c[0], c[1]);
  store_scale<KIND>(out, unit, byte);
}

// ---- adaLN producers on a row held as units of packed bf16 ----
// The steps of the int8 producers, each rounded to bf16, two values at a time.
// The bf16x2 multiply and add round the exact result once, which equals the
// fp32 operation followed by the rounding to bf16: products of two bf16 values
// are exact in fp32, and a sum either is exact there (24 bits hold two 8-bit
// significands up to 16 binades apart) or is too far from a bf16 midpoint for
// the first rounding to matter.
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                      *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bf2_add(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                      *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint64_t bf2_to_f32x2(uint32_t w) {
  return f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Word w (0..7) of a unit.
__device__ __forceinline__ uint32_t& unit_word(Unit<__nv_bfloat16>& u, int w) {
  return reinterpret_cast<uint32_t*>(u.raw)[w];
}

// 1 / sqrt(mean of squares + eps) of a row whose squares, or their sum, leave the
// range of fp32.  They are summed in fp64, where the square of any bf16 value is
// exact; where the mean itself leaves it, the row is scaled by a power of two
// (2^-64 or 2^100, in place) and the result belongs to the scaled row, so that the
// products x * result are those of the row as it was.  Of a row that large, what
// becomes subnormal is below 2^-125 after the norm.
template <int VPT>
__device__ __forceinline__ float row_rms_inverse_f64(const Fp4Params& p,
                                                     Unit<__nv_bfloat16> (&u)[VPT], bool small,
                                                     int tpr, GroupRed& red) {
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float2 x = unpack_bf16x2(unit_word(u[i], w));
      const double lo = x.x, hi = x.y;
      ss = __fma_rn(hi, hi, __fma_rn(lo, lo, ss));
    }
  }
  const double mean = __dmul_rn(group_sum(ss, tpr, red.sum[1]), p.inv_cols);
  const double v = mean + static_cast<double>(p.eps);
  if (v >= 0x1p-100 && v <= 0x1p126)
    return rsqrt_two_step_rn(__fadd_rn(__double2float_rn(mean), p.eps));
  const uint32_t factor = small ? 0x71807180u : 0x1f801f80u;  // 2^100, 2^-64 twice
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int w = 0; w < 8; ++w) unit_word(u[i], w) = bf2_mul(unit_word(u[i], w), factor);
  }
  return rsqrt_two_step_rn(__double2float_rn(__dmul_rn(v, small ? 0x1p200 : 0x1p-128)));
}

// 1 / sqrt(mean of squares + eps) of the row, as the int8 producers compute it:
// exact fp32 squares added in compensated fp32 chains (TwoSum: every rounding
// error is kept in a second word), the chains in fp64, then two correctly
// rounded fp32 steps.  The squares are exact, and no chain overflows, while their
// sum is 2^-90 to 2^126 (what vanishes below 2^-149 is then 2^-45 of it at most);
// a smaller sum beside an eps of 2^-60 or more does not count at all.
template <int VPT>
__device__ __forceinline__ float row_rms_inverse(const Fp4Params& p, Unit<__nv_bfloat16> (&u)[VPT],
                                                 int tpr, GroupRed& red) {
  uint64_t sum[2] = {0ull, 0ull}, err[2] = {0ull, 0ull};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint64_t x = bf2_to_f32x2(unit_word(u[i], w));
      const uint64_t sq = mul_f32x2(x, x);
      uint64_t &s = sum[w & 1], &e = err[w & 1];
      const uint64_t t = add_f32x2(s, sq);
      const uint64_t z = sub_f32x2(t, s);
      e = add_f32x2(e, add_f32x2(sub_f32x2(s, sub_f32x2(t, z)), sub_f32x2(sq, z)));
      s = t;
    }
  }
  double ss = 0.0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float s0, s1, e0, e1;
    f32x2_split(sum[j], s0, s1);
    f32x2_split(err[j], e0, e1);
    ss += (static_cast<double>(s0) + e0) + (static_cast<double>(s1) + e1);
  }
  ss = group_sum(ss, tpr, red.sum[0]);
  const bool small = ss < 0x1p-90;
  if ((small && p.eps < 0x1p-60f) || !(ss <= 0x1p126))  // overflow leaves an inf or a NaN
    return row_rms_inverse_f64(p, u, small, tpr, red);
  const float variance = __double2float_rn(__dmul_rn(ss, p.inv_cols));
  return rsqrt_two_step_rn(__fadd_rn(variance, p.eps));
}

__host__ __device__ constexpr bool has_residual(int mode) {
  return mode == kResGateRmsModulate || mode == kResGateRmsModulateRows;
}

// Producers with a norm whose rows have tables of their own.
__host__ __device__ constexpr bool norm_rows(int mode) {
  return mode == kRmsModulateRows || mode == kResGateRmsModulateRows;
}

// A producer applied to the row's units, in place; also writes the updated
// residual and the hidden state where there are such outputs.
template <int VPT, int MODE>
__device__ __forceinline__ void adaln_units(const Fp4Params& p, Unit<__nv_bfloat16> (&u)[VPT],
                                            int64_t row, int t, int tpr, int units, bool active,
                                            bool wide, GroupRed& red) {
  using U = Unit<__nv_bfloat16>;
  const int64_t trow = active ? (p.index ? p.index[row] : row) : 0;
  const auto unit_of = [&](int i) { return t + i * tpr; };
  // 32-byte table loads in the producers without a norm: 41 -> 39 us (nvfp4) and 37 -> 34
  // (mxfp4) at 20480 x 3072 with five tables; with a norm they change nothing (67, 61 us)
  // and cost with the residual (94 -> 97, 89 -> 92).
  const auto load = [&](U& v, const __nv_bfloat16* at, int unit) {
    ld_table32(at + unit * 16, wide && modulate_only(MODE), v.raw[0], v.raw[1]);
  };
  const auto store = [&](__nv_bfloat16* at, int unit, const U& v) {
    uint4* dst = reinterpret_cast<uint4*>(at + (row * p.cols + unit * 16));
    if (wide) {
      st_global32(dst, v.raw[0], v.raw[1]);
    } else {
      dst[0] = v.raw[0];
      dst[1] = v.raw[1];
    }
  };
  // per-row tables come from HBM like x: all of them are asked for at once
  U pre_sc[MODE == kModulateRows ? VPT : 1], pre_sh[MODE == kModulateRows ? VPT : 1];
  if constexpr (MODE == kModulateRows) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (active && unit_of(i) < units) {
        load(pre_sc[i], p.mod_scale + trow * p.table_stride, unit_of(i));
        load(pre_sh[i], p.shift + trow * p.table_stride, unit_of(i));
      }
  }
  if constexpr (has_residual(MODE)) {
    const __nv_bfloat16* branch = p.branch + row * p.cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (active && unit_of(i) < units) {
        U b, g;
        ld_stream32(branch + unit_of(i) * 16, wide, b.raw[0], b.raw[1]);
        load(g, p.gate + trow * p.table_stride, unit_of(i));
#pragma unroll
        for (int w = 0; w < 8; ++w)
          unit_word(u[i], w) =
              bf2_add(unit_word(u[i], w), bf2_mul(unit_word(g, w), unit_word(b, w)));
        store(p.residual_out, unit_of(i), u[i]);
      }
    }
  }
  // With a norm no registers are left to hold them: L2 fetches them during the row's sum.
  // 20480 x 3072, nvfp4 / mxfp4: RMSNorm 82 -> 75 / 76 -> 70 us, with the residual
  // 129 -> 121 / 124 -> 118; asked for before the residual's loads they gain nothing there.
  if constexpr (norm_rows(MODE)) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (active && unit_of(i) < units) {
        prefetch_l2(p.mod_scale + trow * p.table_stride + unit_of(i) * 16);
        prefetch_l2(p.shift + trow * p.table_stride + unit_of(i) * 16);
      }
  }
  uint64_t rinv2 = 0;
  if constexpr (!modulate_only(MODE)) {
    const float rinv = row_rms_inverse(p, u, tpr, red);
    rinv2 = f32x2(rinv, rinv);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (active && unit_of(i) < units) {
      U wt, sc, sh;
      if constexpr (!modulate_only(MODE)) load(wt, p.norm_w, unit_of(i));
      if constexpr (MODE == kModulateRows) {
        sc = pre_sc[i];
        sh = pre_sh[i];
      } else {
        load(sc, p.mod_scale + trow * p.table_stride, unit_of(i));
        load(sh, p.shift + trow * p.table_stride, unit_of(i));
      }
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        uint32_t x = unit_word(u[i], w);
        if constexpr (!modulate_only(MODE)) {
          const uint64_t v =
              mul_f32x2(mul_f32x2(bf2_to_f32x2(x), rinv2), bf2_to_f32x2(unit_word(wt, w)));
          float lo, hi;
          f32x2_split(v, lo, hi);
          x = pack_bf16x2(lo, hi);
        }
        x = bf2_mul(x, bf2_add(0x3f803f80u, unit_word(sc, w)));  // x (1 + scale)
        unit_word(u[i], w) = bf2_add(x, unit_word(sh, w));
      }
      if (p.hidden_out != nullptr) store(p.hidden_out, unit_of(i), u[i]);
    }
  }
}

// Blocks an SM must hold (a cap on registers): the loads of some rows overlap
// the reductions and the arithmetic of others.
template <typename T, int VPT, int MODE>
constexpr int fp4_min_blocks() {
  if (sizeof(T) == 4) return VPT <= 3 ? 3 : 1;
  if (MODE == kDynamic || MODE == kModulate) return VPT <= 3 ? 4 : 2;
  return VPT <= 3 ? 3 : 2;
}

// A row group per row, the row in registers.  MODE: an adaLN producer, or
// kDynamic for a plain row.
template <typename T, int VPT, int MODE, int KIND>
__global__ void __launch_bounds__(256, (fp4_min_blocks<T, VPT, MODE>())) quant_fp4_rows_kernel(const Fp4Params p, const bool wide) {
  griddep_wait();  // the rows may come from the previous kernel on the stream
  griddep_launch_dependents();
  __shared__ GroupRed red;
  const int tpr = 1 << p.tpr_log2;
  const int t = threadIdx.x & (tpr - 1);
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * (blockDim.x >> p.tpr_log2) + (threadIdx.x >> p.tpr_log2);
  const bool active = row < p.rows;
  const int units = static_cast<int>(p.cols / 16);
  const int pad_units = static_cast<int>(p.ktiles) * (KIND == kMx ? 8 : 4);
  const T* xr = static_cast<const T*>(p.x) + (active ? row : 0) * p.ldx;
  constexpr bool kAdaLN = MODE != kDynamic;

  Unit<T> u[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int unit = t + i * tpr;
    if (active && unit < units)
      load_unit(u[i], xr + unit * 16, wide);
    else
      clear_unit(u[i]);
  }
  if constexpr (kAdaLN) {
    static_assert(std::is_same<T, __nv_bfloat16>::value, "adaLN modes are bf16");
    adaln_units<VPT, MODE>(p, u, row, t, tpr, units, active, wide, red);
  }

  uint32_t m[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    m[i] = unit_max_bits(u[i]);
    if constexpr (KIND == kMx) m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 1));
  }
  RowScale rs{};
  if constexpr (KIND == kNvDynamic) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) top = max(top, m[i]);
    rs = row_scale(group_max_bits(top, tpr, red));
    if (active && t == 0) p.scales[row] = rs.o;
  } else if constexpr (KIND == kNvGiven) {
    rs = given_scale(ld_nc_f32(p.static_scale));
  }
  if (row >= p.padded_rows) return;
  const RowOut out = row_out(p, row);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int unit = t + i * tpr;
    if (active && unit < units) {
      uint32_t c[2];
      const uint32_t byte = convert_unit<T, KIND>(u[i], m[i], rs, c);
      store_unit<KIND>(out, unit, c, byte);
    } else if (unit < pad_units) {  // blocks that only pad a tile
      store_scale<KIND>(out, unit, 0u);
    }
  }
}

// Rows of any width and alignment: a block per row, the row read twice (once
// where no row maximum is needed), element by element.
template <typename T, int KIND>
__global__ void __launch_bounds__(256) quant_fp4_any_kernel(const Fp4Params p) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ GroupRed red;
  const int64_t row = blockIdx.x;
  const bool active = row < p.rows;
  const int units = static_cast<int>(p.cols / 16);
  const int pad_units = static_cast<int>(p.ktiles) * (KIND == kMx ? 8 : 4);
  const T* xr = static_cast<const T*>(p.x) + (active ? row : 0) * p.ldx;
  RowScale rs{};
  if constexpr (KIND == kNvDynamic) {
    uint32_t top = 0;
    if (active) {
      for (int unit = threadIdx.x; unit < units; unit += 256) {
        Unit<T> u;
        load_unit_scalar(u, xr + unit * 16ll);
        top = max(top, unit_max_bits(u));
      }
    }
    rs = row_scale(group_max_bits(top, 256, red));
    if (active && threadIdx.x == 0) p.scales[row] = rs.o;
  } else if constexpr (KIND == kNvGiven) {
    rs = given_scale(ld_nc_f32(p.static_scale));
  }
  const RowOut out = row_out(p, row);
  const int lane_units = (pad_units + 255) / 256 * 256;  // whole warps: shuffles below
  for (int unit = threadIdx.x; unit < lane_units; unit += 256) {
    Unit<T> u;
    const bool in = active && unit < units;
    if (in)
      load_unit_scalar(u, xr + unit * 16ll);
    else
      clear_unit(u);
    uint32_t m = unit_max_bits(u);
    if constexpr (KIND == kMx) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    if (in) {
      uint32_t c[2];
      const uint32_t byte = convert_unit<T, KIND>(u, m, rs, c);
      store_unit<KIND>(out, unit, c, byte);
    } else if (unit < pad_units) {  // blocks that only pad a tile
      store_scale<KIND>(out, unit, 0u);
    }
  }
}

// ------------------------------------------------------------------ inverse
struct DequantParams {
  void* out;  // [rows, cols]
  const uint8_t* codes;
  const uint8_t* blocks;
  const float* scales;  // NULL: 1
  bool per_row;
  int64_t rows, cols, ktiles;
  int tpr_log2;
  bool wide;  // out on a 32-byte boundary (its rows are multiples of 64 bytes)
};

// Two e2m1 codes -> two values.
__device__ __forceinline__ float2 e2m1x2_to_f32(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 b, z;\n\t"
      "mov.b16 {b, z}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
      : "=r"(h)
      : "h"(static_cast<uint16_t>(byte)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <typename T>
__device__ __forceinline__ void store16(T* out, const float (&v)[16], bool wide) {
  uint4 w[sizeof(T)];
  uint32_t* e = reinterpret_cast<uint32_t*>(w);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 16; ++j) e[j] = __float_as_uint(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        e[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        e[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < static_cast<int>(sizeof(T)); j += 2) {
    uint4* dst = reinterpret_cast<uint4*>(out) + j;
    if (wide) {
      st_global32(dst, w[j], w[j + 1]);
    } else {
      dst[0] = w[j];
      dst[1] = w[j + 1];
    }
  }
}

// value = (q * s) * o: q * s is exact in fp32, the product with o is rounded,
// and the result is rounded once more to a 16-bit output type.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(256) dequant_fp4_kernel(const DequantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int tpr = 1 << p.tpr_log2;
  // read-only loads, which the unrolled loop may issue ahead of its stores: every
  // address depends on a row that is only known behind the wait
  const int thread = behind_wait(static_cast<int>(threadIdx.x));
  const int t = thread & (tpr - 1);
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * (blockDim.x >> p.tpr_log2) + (thread >> p.tpr_log2);
  if (row >= p.rows) return;
  const int units = static_cast<int>(p.cols / 16);
  const uint8_t* blocks = p.blocks + fp4_scale_offset(row, 0, p.ktiles);
  const uint2* codes = reinterpret_cast<const uint2*>(p.codes + row * (p.cols / 2));
  const float o = p.scales == nullptr ? 1.0f : ld_nc_f32(p.scales + (p.per_row ? row : 0));
  T* out = static_cast<T*>(p.out) + row * p.cols;
#pragma unroll 4
  for (int unit = t; unit < units; unit += tpr) {
    const uint2 c = __ldg(codes + unit);
    const int block = FORMAT == TM_FP4_MX ? unit >> 1 : unit;
    const uint32_t byte = __ldg(blocks + (block >> 2) * 512 + (block & 3));
    float s;
    if constexpr (FORMAT == TM_FP4_MX)  // 2^(byte - 127); 0 is the subnormal 2^-127, 255 NaN
      s = __uint_as_float(byte == 255u ? 0x7fffffffu : byte == 0u ? 0x00400000u : byte << 23);
    else
      s = e4m3x2_to_f32(byte).x;
    float v[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 q = e2m1x2_to_f32(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 0xffu);
      v[2 * j] = __fmul_rn(__fmul_rn(q.x, s), o);
      v[2 * j + 1] = __fmul_rn(__fmul_rn(q.y, s), o);
    }
    store16(out + unit * 16, v, p.wide);
  }
}

// ------------------------------------------------------------------ host
template <typename T>
constexpr int max_units() {  // 16-element units a thread may hold in registers
  return sizeof(T) == 2 ? 8 : 4;
}

// Threads per row (32..256) and units per thread; false: the row does not fit.
// At most 4 units a thread while the group can still grow: 20480 x 3072 then
// runs on 64 threads a row.
template <typename T>
bool pick_fp4_layout(int64_t units, int* tpr_log2, int* vpt) {
  for (int l = 5; l <= 8; ++l) {
    const int64_t v = (units + (1 << l) - 1) >> l;
    if (v <= 4 || (l == 8 && v <= max_units<T>())) {
      *tpr_log2 = l;
      *vpt = static_cast<int>(v);
      return true;
    }
  }
  return false;
}

template <typename T, int MODE, int KIND>
int launch_rows(Fp4Params p, int tpr_log2, int vpt, bool wide, cudaStream_t stream) {
  p.tpr_log2 = tpr_log2;
  const int rpb = 256 >> tpr_log2;
  const int64_t grid = (p.padded_rows + rpb - 1) / rpb;
  if (grid > 0x7fffffffLL) return TM_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaError_t err = cudaErrorInvalidValue;
  const auto go = [&](auto tag) {
    err = launch_with_pdl(cfg, nullptr, 0, quant_fp4_rows_kernel<T, decltype(tag)::value, MODE, KIND>,
                          p, wide);
  };
  if (vpt <= 1) go(std::integral_constant<int, 1>{});
  else if (vpt <= 2) go(std::integral_constant<int, 2>{});
  else if (vpt <= 3) go(std::integral_constant<int, 3>{});
  else if (vpt <= 4) go(std::integral_constant<int, 4>{});
  else if constexpr (max_units<T>() > 4) {
    if (vpt <= 6) go(std::integral_constant<int, 6>{});
    else if (vpt <= 8) go(std::integral_constant<int, 8>{});
    else return TM_ERR_UNSUPPORTED;
  } else {
    return TM_ERR_UNSUPPORTED;
  }
  return err == cudaSuccess ? check_launch() : TM_ERR_CUDA;
}

inline bool multiple_of(const void* ptr, int64_t stride_bytes, int64_t n) {
  return reinterpret_cast<uintptr_t>(ptr) % n == 0 && stride_bytes % n == 0;
}

template <typename T, int KIND>
int launch_plain(const Fp4Params& p, cudaStream_t stream) {
  int tpr_log2 = 0, vpt = 0;
  const int64_t stride = p.ldx * static_cast<int64_t>(sizeof(T));
  if (multiple_of(p.x, stride, 16) && pick_fp4_layout<T>(p.cols / 16, &tpr_log2, &vpt))
    return launch_rows<T, kDynamic, KIND>(p, tpr_log2, vpt, multiple_of(p.x, stride, 32), stream);
  if (p.padded_rows > 0x7fffffffLL) return TM_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.padded_rows));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  if (launch_with_pdl(cfg, nullptr, 0, quant_fp4_any_kernel<T, KIND>, p) != cudaSuccess)
    return TM_ERR_CUDA;
  return check_launch();
}

template <int KIND>
int launch_typed(const Fp4Params& p, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case TM_DTYPE_BF16: return launch_plain<__nv_bfloat16, KIND>(p, stream);
    case TM_DTYPE_FP16: return launch_plain<__half, KIND>(p, stream);
    case TM_DTYPE_FP32: return launch_plain<float, KIND>(p, stream);
    default: return TM_ERR_DTYPE;
  }
}

// Shape checks of every quantising entry point, and the stored form's geometry.
int set_geometry(Fp4Params& p, int format, int64_t rows, int64_t cols, int64_t ld) {
  if (format != TM_FP4_NV && format != TM_FP4_MX) return TM_ERR_UNSUPPORTED;
  if (rows < 0 || cols <= 0 || cols % 32 != 0 || ld < cols) return TM_ERR_SHAPE;
  if (cols > (1ll << 30)) return TM_ERR_TOO_LARGE;  // positions within a row are 32-bit
  p.rows = rows;
  p.cols = cols;
  p.ldx = ld;
  p.padded_rows = round_up(rows, 128);
  p.ktiles = round_up(cols / fp4_block(format), 4) / 4;
  return TM_OK;
}

template <int MODE>
int launch_adaln(Fp4Params p, int format, cudaStream_t stream) {
  if (p.table_stride % 8 != 0 || !aligned16(p.x) || !aligned16(p.shift) ||
      !aligned16(p.mod_scale) || (p.hidden_out != nullptr && !aligned16(p.hidden_out)) ||
      (!modulate_only(MODE) && !aligned16(p.norm_w)) ||
      (has_residual(MODE) &&
       (!aligned16(p.branch) || !aligned16(p.gate) || !aligned16(p.residual_out))))
    return TM_ERR_ALIGNMENT;
  int tpr_log2 = 0, vpt = 0;
  if (!pick_fp4_layout<__nv_bfloat16>(p.cols / 16, &tpr_log2, &vpt)) return TM_ERR_TOO_LARGE;
  // rows are multiples of 64 bytes: 32-byte accesses wherever the tensors start on one
  const auto on32 = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 32 == 0; };
  bool wide = on32(p.x) && on32(p.hidden_out) && on32(p.branch) && on32(p.residual_out);
  if (modulate_only(MODE))
    wide = wide && on32(p.shift) && on32(p.mod_scale) && p.table_stride % 16 == 0;
  return format == TM_FP4_MX
             ? launch_rows<__nv_bfloat16, MODE, kMx>(p, tpr_log2, vpt, wide, stream)
             : launch_rows<__nv_bfloat16, MODE, kNvDynamic>(p, tpr_log2, vpt, wide, stream);
}

template <typename T>
int launch_dequant(const DequantParams& p, int format, cudaStream_t stream) {
  const int rpb = 256 >> p.tpr_log2;
  const int64_t grid = (p.rows + rpb - 1) / rpb;
  if (grid > 0x7fffffffLL) return TM_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  const cudaError_t err =
      format == TM_FP4_MX ? launch_with_pdl(cfg, nullptr, 0, dequant_fp4_kernel<T, TM_FP4_MX>, p)
                          : launch_with_pdl(cfg, nullptr, 0, dequant_fp4_kernel<T, TM_FP4_NV>, p);
  return err == cudaSuccess ? check_launch() : TM_ERR_CUDA;
}

// The adaLN arguments common to the producers.
int adaln_params(Fp4Params& p, uint8_t* q, uint8_t* block_scales, float* scales, void* hidden_out,
                 const void* x, const void* shift, const void* scale, const int64_t* index,
                 int64_t table_stride, int format, int64_t rows, int64_t cols) {
  if (int s = set_geometry(p, format, rows, cols, cols)) return s;
  if (table_stride < cols) return TM_ERR_SHAPE;
  if (rows == 0) return TM_OK;
  if (!q || !block_scales || !x || !shift || !scale || (format == TM_FP4_NV && !scales))
    return TM_ERR_NULL_POINTER;
  if (!aligned16(q)) return TM_ERR_ALIGNMENT;
  p.x = x;
  p.codes = q;
  p.blocks = block_scales;
  p.scales = scales;
  p.hidden_out = static_cast<__nv_bfloat16*>(hidden_out);
  p.shift = static_cast<const __nv_bfloat16*>(shift);
  p.mod_scale = static_cast<const __nv_bfloat16*>(scale);
  p.index = index;
  p.table_stride = table_stride;
  return TM_OK;
}

}  // namespace
}  // namespace tmw

extern "C" {

int tm_fp4_block_scales_size(int64_t rows, int64_t cols, int format, uint64_t* bytes) {
  if (!bytes) return TM_ERR_NULL_POINTER;
  tmw::Fp4Params p{};
  if (int s = tmw::set_geometry(p, format, rows, cols, cols)) return s;
  *bytes = static_cast<uint64_t>(p.padded_rows) * static_cast<uint64_t>(p.ktiles) * 4u;
  return TM_OK;
}

int tm_scaled_fp4_quant(uint8_t* q, uint8_t* block_scales, float* scales, const float* given_scale,
                        const void* input, int input_dtype, int format, int64_t rows, int64_t cols,
                        int64_t input_row_stride, void* stream) {
  tmw::Fp4Params p{};
  if (int s = tmw::set_geometry(p, format, rows, cols, input_row_stride)) return s;
  if (format == TM_FP4_MX && (given_scale || scales)) return TM_ERR_UNSUPPORTED;
  if (rows == 0) return TM_OK;
  if (!q || !block_scales || !input || (format == TM_FP4_NV && !scales == !given_scale))
    return TM_ERR_NULL_POINTER;  // TM_FP4_NV: one of the two scales
  if (!tmw::aligned16(q)) return TM_ERR_ALIGNMENT;
  p.x = input;
  p.codes = q;
  p.blocks = block_scales;
  p.scales = scales;
  p.static_scale = given_scale;
  const cudaStream_t st = tmw::as_stream(stream);
  if (format == TM_FP4_MX) return tmw::launch_typed<tmw::kMx>(p, input_dtype, st);
  return given_scale ? tmw::launch_typed<tmw::kNvGiven>(p, input_dtype, st)
                     : tmw::launch_typed<tmw::kNvDynamic>(p, input_dtype, st);
}

int tm_dequantize_fp4(void* out, int out_dtype, const uint8_t* q, const uint8_t* block_scales,
                      const float* scales, int64_t scales_numel, int format, int64_t rows,
                      int64_t cols, void* stream) {
  tmw::Fp4Params g{};
  if (int s = tmw::set_geometry(g, format, rows, cols, cols)) return s;
  if (scales && scales_numel != 1 && scales_numel != rows) return TM_ERR_SHAPE;
  if (rows == 0) return TM_OK;
  if (!out || !q || !block_scales) return TM_ERR_NULL_POINTER;
  if (!tmw::aligned16(out) || !tmw::aligned16(q)) return TM_ERR_ALIGNMENT;
  tmw::DequantParams p{};
  p.out = out;
  p.codes = q;
  p.blocks = block_scales;
  p.scales = scales;
  p.per_row = scales_numel == rows;
  p.rows = rows;
  p.cols = cols;
  p.ktiles = g.ktiles;
  p.wide = reinterpret_cast<uintptr_t>(out) % 32 == 0;
  p.tpr_log2 = 5;
  while (p.tpr_log2 < 8 && (cols / 16) > (4ll << p.tpr_log2)) ++p.tpr_log2;
  const cudaStream_t st = tmw::as_stream(stream);
  switch (out_dtype) {
    case TM_DTYPE_BF16: return tmw::launch_dequant<__nv_bfloat16>(p, format, st);
    case TM_DTYPE_FP16: return tmw::launch_dequant<__half>(p, format, st);
    case TM_DTYPE_FP32: return tmw::launch_dequant<float>(p, format, st);
    default: return TM_ERR_DTYPE;
  }
}

int tm_modulate_fp4_quant(uint8_t* q, uint8_t* block_scales, float* scales, void* hidden_out,
                          const void* x, const void* shift, const void* scale, const int64_t* index,
                          int64_t table_stride, int format, int64_t rows, int64_t cols,
                          void* stream) {
  tmw::Fp4Params p{};
  if (int s = tmw::adaln_params(p, q, block_scales, scales, hidden_out, x, shift, scale, index,
                                table_stride, format, rows, cols))
    return s;
  if (rows == 0) return TM_OK;
  const cudaStream_t st = tmw::as_stream(stream);
  return index == nullptr ? tmw::launch_adaln<tmw::kModulateRows>(p, format, st)
                          : tmw::launch_adaln<tmw::kModulate>(p, format, st);
}

int tm_rms_norm_modulate_fp4_quant(uint8_t* q, uint8_t* block_scales, float* scales,
                                   void* hidden_out, const void* x, const void* norm_weight,
                                   float eps, const void* shift, const void* scale,
                                   const int64_t* index, int64_t table_stride, int format,
                                   int64_t rows, int64_t cols, void* stream) {
  tmw::Fp4Params p{};
  if (int s = tmw::adaln_params(p, q, block_scales, scales, hidden_out, x, shift, scale, index,
                                table_stride, format, rows, cols))
    return s;
  if (rows == 0) return TM_OK;
  if (!norm_weight) return TM_ERR_NULL_POINTER;
  p.norm_w = static_cast<const __nv_bfloat16*>(norm_weight);
  p.eps = eps;
  p.inv_cols = 1.0 / static_cast<double>(cols);
  cudaStream_t st = tmw::as_stream(stream);
  return index == nullptr ? tmw::launch_adaln<tmw::kRmsModulateRows>(p, format, st)
                          : tmw::launch_adaln<tmw::kRmsModulate>(p, format, st);
}

int tm_residual_gate_rms_norm_modulate_fp4_quant(
    uint8_t* q, uint8_t* block_scales, float* scales, void* residual_out, void* hidden_out,
    const void* residual, const void* branch, const void* gate, const void* norm_weight, float eps,
    const void* shift, const void* scale, const int64_t* index, int64_t table_stride, int format,
    int64_t rows, int64_t cols, void* stream) {
  tmw::Fp4Params p{};
  if (int s = tmw::adaln_params(p, q, block_scales, scales, hidden_out, residual, shift, scale,
                                index, table_stride, format, rows, cols))
    return s;
  if (rows == 0) return TM_OK;
  if (!residual_out || !branch || !gate || !norm_weight) return TM_ERR_NULL_POINTER;
  p.norm_w = static_cast<const __nv_bfloat16*>(norm_weight);
  p.eps = eps;
  p.inv_cols = 1.0 / static_cast<double>(cols);
  p.branch = static_cast<const __nv_bfloat16*>(branch);
  p.gate = static_cast<const __nv_bfloat16*>(gate);
  p.residual_out = static_cast<__nv_bfloat16*>(residual_out);
  cudaStream_t st = tmw::as_stream(stream);
  return index == nullptr ? tmw::launch_adaln<tmw::kResGateRmsModulateRows>(p, format, st)
                          : tmw::launch_adaln<tmw::kResGateRmsModulate>(p, format, st);
}

}  // extern "C"
