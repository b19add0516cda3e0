// Weights held in 4 bits: the layout that mq_linear4 reads and its decoding in registers (gfx950 only).
//
// A weight [N, K] is cut into tiles of 16 rows x 128 columns, 1 KiB each, stored tile after tile along K.  Inside a tile
// lane l = 16 * kq + (n % 16) of a wave owns four dwords: dword j holds the eight codes k = 32 j + 8 kq + (0 .. 7) of row
// n -- exactly the B operand of the j-th v_mfma_f32_16x16x32 over that tile.  So a wave fetches a tile with one 16-byte
// load per lane (1 KiB in one piece) and feeds it to the matrix cores after decoding, with no exchange between lanes.
//
// Where a code's bits stand in its dword depends on how the kind is decoded; every route ends in one packed conversion per
// two weights, exact in float16 and bfloat16:
//   U4   unsigned integers 0 .. 15: code i < 4 in the low nibble of byte i, code 4 + i in the high one.  A byte 0 .. 15
//        read as fp8 e4m3 is the number byte * 2^-9 (subnormals, then the first binade: the same straight line), so
//        v_cvt_scalef32_pk_*_fp8 with the scale 2^9 returns the integer: 3 + 4 instructions per 8 weights.
//   S4   sign and magnitude, +-(0 .. 7): as U4, but the sign stands in bit 7 of the byte that the conversion reads: for the
//        low nibbles in place, for the high ones where a rotation by 4 brings it (bit 3 of the next byte): 3 + 4.
//   LUT  sixteen table values that are fp8 e4m3 numbers (every 3- / 4-bit list of the framework): bits as in S4; the low
//        three bits select from the two halves of the table with v_perm_b32, bit 7 chooses the half: 15 + 4.
//   FP4  the e2m1 grid times two (the framework's fp4 list 1, 2, 3, 4, 6, 8, 12): codes are e2m1 numbers, code 2 i in the
//        low nibble of byte i, 2 i + 1 in the high one, v_cvt_scalef32_pk_*_fp4 with the scale 2: 4 instructions.
#pragma once
#include "mq_common.h"

enum { W4_U4 = MQ_W4_INT_ASYM, W4_S4 = MQ_W4_INT_SYM, W4_LUT = MQ_W4_TABLE, W4_FP4 = MQ_W4_FP4 };

typedef _Float16 w4_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 w4_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 w4_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 w4_b8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float w4_f2 __attribute__((ext_vector_type(2)));

struct W4Lut {
  uint32_t w[4];  // sixteen e4m3 bytes, entry i = the value of code i (LUT)
};

// ---- scalars of the layout ------------------------------------------------------------------------
__host__ __device__ __forceinline__ int64_t w4_ntiles(int64_t n) { return (n + 15) / 16; }
__host__ __device__ __forceinline__ int64_t w4_ktiles(int64_t k) { return (k + 127) / 128; }

// Bit position of the low three bits / of the top bit of code i in its dword.
template <int KIND> __host__ __device__ __forceinline__ int w4_low_at(int i) {
  return KIND == W4_FP4 ? 4 * i : i < 4 ? 8 * i : 8 * (i - 4) + 4;
}
template <int KIND> __host__ __device__ __forceinline__ int w4_top_at(int i) {
  if (KIND == W4_U4 || KIND == W4_FP4) return w4_low_at<KIND>(i) + 3;
  return i < 4 ? 8 * i + 7 : (8 * (i - 4) + 11) & 31;
}
template <int KIND> __host__ __device__ __forceinline__ uint32_t w4_put(uint32_t code, int i) {
  return ((code & 7u) << w4_low_at<KIND>(i)) | ((code >> 3 & 1u) << w4_top_at<KIND>(i));
}
template <int KIND> __host__ __device__ __forceinline__ uint32_t w4_get(uint32_t d, int i) {
  return (d >> w4_low_at<KIND>(i) & 7u) | ((d >> w4_top_at<KIND>(i) & 1u) << 3);
}

// ---- decoding --------------------------------------------------------------------------------------
// Four codes in S4's byte form -> four e4m3 bytes of the table.
__device__ __forceinline__ uint32_t w4_lookup(uint32_t t, const W4Lut& lut) {
  const uint32_t sel = t & 0x07070707u, top = t & 0x80808080u;
  const uint32_t a = __builtin_amdgcn_perm(lut.w[1], lut.w[0], sel);
  const uint32_t b = __builtin_amdgcn_perm(lut.w[3], lut.w[2], sel);
  const uint32_t mask = (top << 1) - (top >> 7);  // 0xFF in every byte whose bit 7 is set (the carries cancel)
  return (b & mask) | (a & ~mask);
}
// Dword -> the e4m3 bytes of codes 0 .. 3 (lo) and 4 .. 7 (hi); not for FP4.
template <int KIND> __device__ __forceinline__ void w4_bytes(uint32_t d, const W4Lut& lut, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == W4_U4) {
    lo = d & 0x0F0F0F0Fu;
    hi = (d >> 4) & 0x0F0F0F0Fu;
  } else {
    lo = d & 0x87878787u;
    hi = __builtin_amdgcn_alignbit(d, d, 4) & 0x87878787u;
    if constexpr (KIND == W4_LUT) {
      lo = w4_lookup(lo, lut);
      hi = w4_lookup(hi, lut);
    }
  }
}
// What an e4m3 byte has to be multiplied by to be the code's value.
template <int KIND> constexpr float w4_byte_scale() { return KIND == W4_U4 || KIND == W4_S4 ? 512.0f : 1.0f; }

struct W4F16 {  // element traits: float16
  static constexpr bool kHalf = true;
  template <bool HI> static __device__ __forceinline__ uint32_t from_fp8(uint32_t v, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, s, HI));
  }
  template <int B> static __device__ __forceinline__ uint32_t from_fp4(uint32_t v) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 2.0f, B));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {  // two roundings to nearest
    w4_h2 r;
    r[0] = (_Float16)a;
    r[1] = (_Float16)b;
    return __builtin_bit_cast(uint32_t, r);
  }
  static __device__ __forceinline__ float to_f32(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t from_f32(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(w4_h8, a), __builtin_bit_cast(w4_h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(w4_h8, a), __builtin_bit_cast(w4_h8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kOnes = 0x3C003C00u;
};
struct W4BF16 {  // element traits: bfloat16
  static constexpr bool kHalf = false;
  template <bool HI> static __device__ __forceinline__ uint32_t from_fp8(uint32_t v, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, s, HI));
  }
  template <int B> static __device__ __forceinline__ uint32_t from_fp4(uint32_t v) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 2.0f, B));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    w4_b2 r;
    r[0] = (__bf16)a;
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
  }
  static __device__ __forceinline__ float to_f32(uint16_t v) { return f_from_bits((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t from_f32(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_b8, a), __builtin_bit_cast(w4_b8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(w4_b8, a), __builtin_bit_cast(w4_b8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kOnes = 0x3F803F80u;
};

// Dword -> its eight codes' values as four packed pairs of T, exact.
template <class T, int KIND> __device__ __forceinline__ u32x4 w4_decode(uint32_t d, const W4Lut& lut) {
  u32x4 r;
  if constexpr (KIND == W4_FP4) {
    r[0] = T::template from_fp4<0>(d);
    r[1] = T::template from_fp4<1>(d);
    r[2] = T::template from_fp4<2>(d);
    r[3] = T::template from_fp4<3>(d);
  } else {
    uint32_t lo, hi;
    w4_bytes<KIND>(d, lut, lo, hi);
    constexpr float s = w4_byte_scale<KIND>();
    r[0] = T::template from_fp8<false>(lo, s);
    r[1] = T::template from_fp8<true>(lo, s);
    r[2] = T::template from_fp8<false>(hi, s);
    r[3] = T::template from_fp8<true>(hi, s);
  }
  return r;
}
// Dword -> its eight codes' values in float32.
template <int KIND> __device__ __forceinline__ void w4_decode_f32(uint32_t d, const W4Lut& lut, float* f) {
  w4_f2 p[4];
  if constexpr (KIND == W4_FP4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 2.0f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 2.0f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 2.0f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 2.0f, 3);
  } else {
    uint32_t lo, hi;
    w4_bytes<KIND>(d, lut, lo, hi);
    constexpr float s = w4_byte_scale<KIND>();
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, s, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, s, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, s, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, s, true);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = p[i][0], f[2 * i + 1] = p[i][1];
}

__device__ __forceinline__ f32x16 w4_zero16() { return f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}; }

// ---- the arguments that all kernels share ------------------------------------------------------------
struct W4Args {
  const uint32_t* data;    // [E][NT][KT][64][4]
  const void* params;      // [E][NT][GP][16]: float16 scale, or (U4) float16 scale | float16 zero point << 16
  const float* norm;       // [E] power of two that brings the largest |weight| of an expert near 2^15
  const int32_t* counts;   // [E] rows of each expert, or NULL: all rows belong to the one weight
  int64_t experts, n, k, rows;
  int32_t nt, kt, gp;      // tiles along N and K, groups along the padded K
  int32_t gu;              // K-steps of 32 per group
  uint32_t gmagic;         // ceil(2^31 / gu): see w4_group
  W4Lut lut;
};
// Group of K-step s: floor(s / gu) = floor((2 s + 1) / (2 gu)) as the high half of (2 s + 1) * ceil(2^32 / (2 gu)).  The
// product is too large by (2 s + 1) * d / 2^32 with d < 2 gu, and the fraction leaves 1 / (2 gu) of room: exact for
// (2 s + 1) * 2 gu <= 2^32, and s, gu < 2^15 (columns <= 2^20).
__device__ __forceinline__ int w4_group(const W4Args& a, int step) { return (int)__umulhi((uint32_t)(2 * step + 1), a.gmagic); }

// Inclusive sum over the lanes of a wave, cut off at `top` (0 <= v <= top < 2^31), in the vector unit's own lane moves.
__device__ __forceinline__ uint32_t w4_scan(uint32_t v, uint32_t top) {
#define MQ_W4_SCAN_STEP(CTRL, ROWS)                                                             \
  {                                                                                             \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false); \
    v = v + o < top ? v + o : top;                                                              \
  }
  MQ_W4_SCAN_STEP(0x111, 0xF)  // one lane up within rows of 16, then two, four, eight
  MQ_W4_SCAN_STEP(0x112, 0xF)
  MQ_W4_SCAN_STEP(0x114, 0xF)
  MQ_W4_SCAN_STEP(0x118, 0xF)
  MQ_W4_SCAN_STEP(0x142, 0xA)  // lane 15 of a row to the next row (rows 1 and 3)
  MQ_W4_SCAN_STEP(0x143, 0xC)  // lane 31 to the upper half
#undef MQ_W4_SCAN_STEP
  return v;
}

// Row tile t -> (expert, first row, rows).  Experts without rows have no tiles; counts below zero stand for none and the
// sum stops at `rows`, whatever the array holds, so that every row is in bounds; the rows behind the last expert's form
// tiles of their own, expert = -1.  -> false when there is no tile t.  Called by whole waves.
__device__ __forceinline__ bool w4_find_tile(const W4Args& a, int bm, int t, int& expert, int64_t& row0, int& rows) {
  if (!a.counts) {
    row0 = (int64_t)t * bm;
    if (row0 >= a.rows) return false;
    expert = 0;
    rows = (int)(a.rows - row0 < bm ? a.rows - row0 : bm);
    return true;
  }
  const int lane = threadIdx.x & 63;
  const uint32_t all = (uint32_t)a.rows;
  uint32_t row_base = 0, tile_base = 0;
  for (int e0 = 0; e0 <= (int)a.experts; e0 += 64) {  // entry `experts` is what is left
    const int e = e0 + lane;
    uint32_t c = 0;
    if (e < (int)a.experts) {
      const int32_t v = a.counts[e];
      c = v > 0 ? ((uint32_t)v < all ? (uint32_t)v : all) : 0u;
    }
    if (e == (int)a.experts) c = all;
    const uint32_t up = w4_scan(c, all);
    const uint32_t end = row_base + up < all ? row_base + up : all;
    const uint32_t before = (uint32_t)__shfl_up((int)end, 1), start = lane ? before : row_base;
    const uint32_t tiles = (end - start + bm - 1) / (uint32_t)bm;
    const uint32_t last = tile_base + w4_scan(tiles, 0x7FFFFFFFu);
    const uint64_t who = __ballot((uint32_t)t < last);  // the first lane whose tiles reach beyond t
    if (who) {
      const int src = __builtin_ctzll(who);
      const uint32_t st = (uint32_t)__builtin_amdgcn_readlane((int)start, src), en = (uint32_t)__builtin_amdgcn_readlane((int)end, src);
      const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)(last - tiles), src);
      row0 = st + ((uint32_t)t - first) * bm;
      rows = (int)(en - (uint32_t)row0 < (uint32_t)bm ? en - (uint32_t)row0 : (uint32_t)bm);
      expert = e0 + src < (int)a.experts ? e0 + src : -1;
      return true;
    }
    row_base = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
    tile_base = (uint32_t)__builtin_amdgcn_readlane((int)last, 63);
  }
  return false;
}
