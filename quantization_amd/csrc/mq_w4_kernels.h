// The products of one element type and one kind of 4-bit codes: k_w4_rows (few rows: bound by reading the weight),
// k_w4_gemm (many rows: matrix cores) and their launchers.  Included by mq_linear4.hip once per (type, kind).
//
#pragma once
#include "mq_w4.h"

struct W4Product {
  const uint16_t* x;     // [rows][ldx], contraction index contiguous
  const uint32_t* b;     // packed operand: W4Args::data, or its transpose for the gradient
  const uint16_t* bias;  // [E][nc] or NULL
  uint16_t* y;           // [rows][nc]
  float* part;           // [splits][rows][16 * ct] partial sums, NULL when splits == 1
  float* xs;             // sums of x per window and row (k_w4_rowsum), for zero points in k_w4_gemm
  const void* ts;        // gradient: scales along the contraction, k_w4_turn's [E][GP][128 rb]
  const void* tz;        // ... and zero points (float16) or scale * zero (bfloat16)
  int64_t ldx, kc, nc;   // contraction length, output columns
  int32_t ct, rb;        // 16-column tiles of the output, 128-blocks of the contraction
  int32_t vec;           // rows of x are 16-byte aligned and kc % 8 == 0
  int32_t nblocks, mblocks, splits;
};

// Eight contraction-neighbours of a row of x, zeros behind the end.
__device__ __forceinline__ u32x4 w4_load8(const uint16_t* row, int64_t k, int64_t kc, bool vec) {
  u32x4 v = {0, 0, 0, 0};
  if (vec) {
    if (k < kc) v = *reinterpret_cast<const u32x4*>(row + k);
  } else {
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = k + i < kc ? row[k + i] : (uint16_t)0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
  }
  return v;
}

// Scales (and zero points) of the four output columns 4 * (lane / 16) .. + 3 of tile `tile` in group `grp`.
template <int KIND>
__device__ __forceinline__ void w4_params4(const W4Args& a, int64_t tile, int grp, int quad, f32x4& s, f32x4& sz) {
  const int64_t at = (tile * a.gp + grp) * 16 + quad * 4;
  if constexpr (KIND == W4_U4) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const uint32_t*>(a.params) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = (float)h_from_bits(v[i]);
      sz[i] = s[i] * (float)h_from_bits(v[i] >> 16);  // exact: 11 x 11 bits
    }
  } else {
    const u32x2 v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(a.params) + at);
    s[0] = (float)h_from_bits(v[0]);
    s[1] = (float)h_from_bits(v[0] >> 16);
    s[2] = (float)h_from_bits(v[1]);
    s[3] = (float)h_from_bits(v[1] >> 16);
  }
}

template <class T> __device__ __forceinline__ void w4_store4(uint16_t* y, int64_t nc, int64_t row, int64_t col, f32x4 v) {
  uint16_t* to = y + row * nc + col;
  if (nc % 4 == 0) {  // (y itself is 16-byte aligned)
    u32x2 o;
    o[0] = T::pack(v[0], v[1]);
    o[1] = T::pack(v[2], v[3]);
    *reinterpret_cast<u32x2*>(to) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < nc) to[i] = T::from_f32(v[i]);
  }
}
template <class T>
__device__ __forceinline__ f32x4 w4_bias4(const uint16_t* bias, int64_t nc, int expert, int64_t col, f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < nc) v[i] += T::to_f32(bias[expert * nc + col + i]);
  return v;
}

// ---- few rows --------------------------------------------------------------------------------------
// A workgroup owns NT column tiles and 16 * MT rows; its waves take the 128-blocks of the contraction in turn and their
// sums meet in LDS at the end, in the waves' order.  The weight is the matrix instruction's A operand, so a lane's four
// results are four neighbouring columns of one row and y is stored 8 bytes at a time.
template <class T, int KIND, int MT, int NT, int FS>
__global__ __launch_bounds__(512) void k_w4_rows(const W4Args a, const W4Product p) {
  extern __shared__ f32x4 w4_red[];
  constexpr int D = MT * NT >= 4 ? 1 : 2;  // 128-blocks in flight per wave
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int quad = lane >> 4;
  const int64_t tile0 = (int64_t)(blockIdx.x % p.nblocks) * NT;
  int expert, rows;
  int64_t row0;
  if (!w4_find_tile(a, 16 * MT, blockIdx.x / p.nblocks, expert, row0, rows)) return;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = {0, 0, 0, 0};

  if (expert >= 0) {
    int64_t tile[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) tile[n] = (int64_t)expert * a.nt + (tile0 + n < a.nt ? tile0 + n : a.nt - 1);
    const uint16_t* xr[MT];
    bool live[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = m * 16 + (lane & 15);
      live[m] = r < rows;
      xr[m] = p.x + (row0 + (live[m] ? r : 0)) * p.ldx;
    }
    for (int kb = w; kb < a.kt; kb += nw * D) {
      u32x4 wv[D][NT], xv[D][MT][4];
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int k0 = kb + d * nw;
        if (k0 < a.kt) {
#pragma unroll
          for (int n = 0; n < NT; ++n) wv[d][n] = *reinterpret_cast<const u32x4*>(p.b + (tile[n] * a.kt + k0) * 256 + lane * 4);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              xv[d][m][j] = {0, 0, 0, 0};
              if (live[m]) xv[d][m][j] = w4_load8(xr[m], (int64_t)k0 * 128 + j * 32 + quad * 8, p.kc, p.vec);
            }
        }
      }
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int k0 = kb + d * nw;
        if (k0 < a.kt) {
          f32x4 tmp[MT][NT], xs[MT];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j % FS == 0) {
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                xs[m] = {0, 0, 0, 0};
#pragma unroll
                for (int n = 0; n < NT; ++n) tmp[m][n] = {0, 0, 0, 0};
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const u32x4 v = w4_decode<T, KIND>(wv[d][n][j], a.lut);
#pragma unroll
              for (int m = 0; m < MT; ++m) tmp[m][n] = T::mfma(v, xv[d][m][j], tmp[m][n]);
            }
            if constexpr (KIND == W4_U4) {
              const u32x4 ones = {T::kOnes, T::kOnes, T::kOnes, T::kOnes};
#pragma unroll
              for (int m = 0; m < MT; ++m) xs[m] = T::mfma(ones, xv[d][m][j], xs[m]);
            }
            if ((j + 1) % FS == 0) {
              const int grp = w4_group(a, k0 * 4 + j);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                f32x4 s, sz;
                w4_params4<KIND>(a, tile[n], grp, quad, s, sz);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    acc[m][n][i] = __builtin_fmaf(s[i], tmp[m][n][i], acc[m][n][i]);
                    if constexpr (KIND == W4_U4) acc[m][n][i] = __builtin_fmaf(-sz[i], xs[m][i], acc[m][n][i]);
                  }
              }
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) w4_red[((w * MT + m) * NT + n) * 64 + lane] = acc[m][n];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * NT * 64; i += blockDim.x) {
    f32x4 v = w4_red[i];
    for (int o = 1; o < nw; ++o) v += w4_red[o * MT * NT * 64 + i];
    const int l = i & 63, n = (i >> 6) % NT, m = (i >> 6) / NT;
    const int r = m * 16 + (l & 15);
    const int64_t col = (tile0 + n) * 16 + (l >> 4) * 4;
    if (r < rows && col < p.nc) {
      if (p.bias && expert >= 0) v = w4_bias4<T>(p.bias, p.nc, expert, col, v);
      w4_store4<T>(p.y, p.nc, row0 + r, col, v);
    }
  }
}

// ---- the gradient's scaled weights ---------------------------------------------------------------------
// Eight weights of one column, scale * (q - zero) rounded once to T.  float16: the integer difference is exact, the
// product rounds (scales are held times the expert's norm, a power of two); bfloat16: one float32 fma, then the rounding.
template <class T, int KIND> struct W4Scales;
template <int KIND> struct W4Scales<W4F16, KIND> {
  u32x4 s, z;
  __device__ __forceinline__ void load(const W4Product& p, int64_t at) {
    s = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.ts) + at);
    if constexpr (KIND == W4_U4) z = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.tz) + at);
  }
  __device__ __forceinline__ u32x4 scaled(uint32_t d, const W4Lut& lut) const {
    u32x4 v = w4_decode<W4F16, KIND>(d, lut);
    // (whole vectors: the compiler takes a bit cast of one element of a vector for one of its first element)
    w4_h8 q = __builtin_bit_cast(w4_h8, v);
    if constexpr (KIND == W4_U4) q = q - __builtin_bit_cast(w4_h8, z);
    return __builtin_bit_cast(u32x4, q * __builtin_bit_cast(w4_h8, s));
  }
};
template <int KIND> struct W4Scales<W4BF16, KIND> {
  f32x4 s[2], z[2];
  __device__ __forceinline__ void load(const W4Product& p, int64_t at) {
    const f32x4* from = reinterpret_cast<const f32x4*>(static_cast<const float*>(p.ts) + at);
    s[0] = from[0], s[1] = from[1];
    if constexpr (KIND == W4_U4) {
      const f32x4* zero = reinterpret_cast<const f32x4*>(static_cast<const float*>(p.tz) + at);
      z[0] = zero[0], z[1] = zero[1];
    }
  }
  __device__ __forceinline__ u32x4 scaled(uint32_t d, const W4Lut& lut) const {
    float f[8];
    w4_decode_f32<KIND>(d, lut, f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = KIND == W4_U4 ? __builtin_fmaf(f[i], s[i / 4][i % 4], -z[i / 4][i % 4]) : f[i] * s[i / 4][i % 4];
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = W4BF16::pack(f[2 * i], f[2 * i + 1]);
    return v;
  }
};

// ---- many rows -------------------------------------------------------------------------------------
// A workgroup of WM x WN waves owns 32 MT WM rows and 32 NT WN columns, in tiles of v_mfma_f32_32x32x16 (which leaves six
// vector instructions per matrix instruction free; two 16x16x32 leave four).  Here the activations are the A operand, so
// that a lane's results belong to one column: one scale per tile and lane.  A 128-block of the rows is staged in LDS,
// 256 bytes a row, its sixteen 16-byte pieces permuted by the row (piece c stands at c ^ (row % 16)), so that rows are
// fetched in whole lines and neither the writes nor the operand reads meet in a bank.  The packed weight goes from memory
// straight into the registers of the wave that decodes it: lane l takes row l % 32 of the 32-row tile, the halves of its
// wave the eight columns 8 (l / 32) of every sixteen -- two of the layout's four dwords-quadruples.
// Rows are 16-byte aligned and a multiple of 128 long here: others are copied first (k_w4_pad).
// GRAD = false: sums run over exact code values; every FS steps of 32 they are scaled in float32 into the result.
// GRAD = true (dx = dy W, operand b transposed): scales change along the contraction, so they are multiplied into the
// weights, which are rounded once to T -- half a step of T per weight, as a weight stored in T has.
typedef __attribute__((address_space(1))) const void w4_global_t;
typedef __attribute__((address_space(3))) void w4_lds_t;

template <class T, int KIND, bool GRAD, int MT, int NT, int WM, int WN, int FS>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_w4_gemm(const W4Args a, const W4Product p) {
  constexpr int BM = 32 * MT * WM, NW = WM * WN, CH = BM / 4 / NW;  // 1 KiB pieces (4 rows) per wave
  static_assert(BM / 4 % NW == 0, "the rows of a block are dealt evenly");
  __shared__ u32x4 lds[2][BM * 16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, half = lane >> 5, l32 = lane & 31;
  const int wm = w % WM, wn = w / WM;
  const int64_t mb = blockIdx.x % p.mblocks;
  const int64_t tile0 = ((int64_t)(blockIdx.x / p.mblocks) * WN + wn) * NT;  // tiles of 32 columns
  int expert, rows;
  int64_t row0;
  if (!w4_find_tile(a, BM, mb, expert, row0, rows)) return;
  f32x16 acc[MT][NT];     // GRAD: the matrix instructions' own sums
  float sum[MT][NT][16];  // forward: the scaled sums (single registers: they are never a matrix operand)
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[m][n] = w4_zero16();
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[m][n][i] = 0;
    }

  if (expert >= 0) {
    // 16-row tile of this lane's row: tiles past the end repeat the last one (their results are not stored)
    const uint32_t* bp[NT];
    int64_t pt[NT];  // forward: this lane's column in the parameters of group 0
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      int64_t t = (tile0 + n) * 2 + (l32 >> 4);
      t = (int64_t)expert * p.ct + (t < p.ct ? t : p.ct - 1);
      bp[n] = p.b + t * p.rb * 256 + (half * 16 + (lane & 15)) * 4;
      pt[n] = t * a.gp * 16 + (lane & 15);
    }
    const uint16_t* xp[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int r = (w * CH + c) * 4 + (lane >> 4);
      xp[c] = p.x + (row0 + (r < rows ? r : rows - 1)) * p.ldx + (((lane & 15) ^ (r & 15)) * 8);
    }
    const int kb0 = (int)((int64_t)p.rb * blockIdx.y / p.splits), kb1 = (int)((int64_t)p.rb * (blockIdx.y + 1) / p.splits);
    int64_t st0[NT];  // gradient: this lane's first scale under column tile n
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t c = tile0 + n, last = (p.ct - 1) >> 1;
      st0[n] = ((int64_t)expert * a.gp + w4_group(a, (int)(c < last ? c : last))) * p.rb * 128 + half * 8;
    }
    u32x4 bn[NT][2];
    auto fetch = [&](int kb, int buf) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        __builtin_amdgcn_global_load_lds((w4_global_t*)(xp[c] + (int64_t)kb * 128), (w4_lds_t*)&lds[buf][(w * CH + c) * 64], 16, 0, 0);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) bn[n][h] = *reinterpret_cast<const u32x4*>(bp[n] + (int64_t)kb * 256 + h * 128);
    };
    if (kb0 < kb1) fetch(kb0, 0);
    __syncthreads();
    for (int kb = kb0; kb < kb1; ++kb) {
      const int buf = (kb - kb0) & 1;
      u32x4 bv[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) bv[n][0] = bn[n][0], bv[n][1] = bn[n][1];
      if (kb + 1 < kb1) fetch(kb + 1, buf ^ 1);
      const u32x4* xb = lds[buf] + (wm * MT * 32 + l32) * 16;
      const int turn = (l32 & 15) ^ half;
      if constexpr (!GRAD) {
        f32x16 tmp[MT][NT];
#pragma unroll
        for (int st = 0; st < 8; ++st) {
          u32x4 xv[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) xv[m] = xb[m * 512 + ((2 * st) ^ turn)];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const u32x4 v = w4_decode<T, KIND>(bv[n][st & 1][st >> 1], a.lut);
#pragma unroll
            for (int m = 0; m < MT; ++m) tmp[m][n] = T::mfma32(xv[m], v, st % (2 * FS) == 0 ? w4_zero16() : tmp[m][n]);
          }
          if ((st + 1) % (2 * FS) == 0) {
            const int grp = w4_group(a, kb * 4 + st / 2);
            float s[NT], sz[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (KIND == W4_U4) {
                const uint32_t v = static_cast<const uint32_t*>(a.params)[pt[n] + grp * 16];
                s[n] = (float)h_from_bits(v);
                sz[n] = -(s[n] * (float)h_from_bits(v >> 16));  // exact: 11 x 11 bits
              } else {
                s[n] = (float)h_from_bits(static_cast<const uint16_t*>(a.params)[pt[n] + grp * 16]);
              }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const float* xs = KIND == W4_U4 ? p.xs + (int64_t)(kb * (4 / FS) + st / (2 * FS)) * a.rows + row0 + (wm * MT + m) * 32 + half * 4 : nullptr;
#pragma unroll
              for (int q = 0; q < 4; ++q) {  // registers 4 q .. 4 q + 3: rows 8 q + 4 half + (0 .. 3) of the tile
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float x = KIND == W4_U4 ? xs[q * 8 + i] : 0.0f;
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    sum[m][n][4 * q + i] = __builtin_fmaf(s[n], tmp[m][n][4 * q + i], sum[m][n][4 * q + i]);
                    if constexpr (KIND == W4_U4) sum[m][n][4 * q + i] = __builtin_fmaf(sz[n], x, sum[m][n][4 * q + i]);
                  }
                }
              }
            }
            // one window's unscaled sums at a time: without this the scheduler keeps several in registers and spills
            if (FS < 4) __builtin_amdgcn_sched_barrier(0);
          }
        }
      } else {
        constexpr int SETS = FS == 1 ? NT : 1;  // groups under a wave's 32 NT columns
#pragma unroll
        for (int st = 0; st < 8; ++st) {
          W4Scales<T, KIND> sc[SETS];
#pragma unroll
          for (int g = 0; g < SETS; ++g) sc[g].load(p, st0[g] + kb * 128 + st * 16);
          u32x4 xv[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) xv[m] = xb[m * 512 + ((2 * st) ^ turn)];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const u32x4 v = sc[FS == 1 ? n : 0].scaled(bv[n][st & 1][st >> 1], a.lut);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][n] = T::mfma32(xv[m], v, acc[m][n]);
          }
        }
      }
      __syncthreads();
    }
    if constexpr (GRAD) {
      const float down = T::kHalf ? 1.0f / a.norm[expert] : 1.0f;  // (float16 weights are held times norm, a power of two)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[m][n][i] = acc[m][n][i] * down;
    }
  }
  // A lane holds one column; neighbours exchange half of their rows, so that each stores pairs of columns: the even lane
  // of a pair rows 0, 2, .. of its registers, the odd one rows 1, 3, ..
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t col = (tile0 + n) * 32 + (l32 & ~1);
    float b0 = 0, b1 = 0;
    if (p.bias && expert >= 0 && blockIdx.y == 0) {
      if (col < p.nc) b0 = T::to_f32(p.bias[expert * p.nc + col]);
      if (col + 1 < p.nc) b1 = T::to_f32(p.bias[expert * p.nc + col + 1]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const bool odd = lane & 1;
        const float mine = odd ? sum[m][n][i + 1] : sum[m][n][i], other = odd ? sum[m][n][i] : sum[m][n][i + 1];
        const float got = __shfl_xor(other, 1);
        const float v0 = (odd ? got : mine) + b0, v1 = (odd ? mine : got) + b1;
        const int r = (wm * MT + m) * 32 + (i >> 2) * 8 + half * 4 + (i & 3) + odd;
        if (r < rows && col < p.nc) {
          if (p.part) {
            float* to = p.part + ((int64_t)blockIdx.y * a.rows + row0 + r) * (p.ct * 16) + col;
            to[0] = v0;
            to[1] = v1;
          } else {
            uint16_t* to = p.y + (row0 + r) * p.nc + col;
            if (p.nc % 2 == 0) {
              *reinterpret_cast<uint32_t*>(to) = T::pack(v0, v1);
            } else {
              to[0] = T::from_f32(v0);
              if (col + 1 < p.nc) to[1] = T::from_f32(v1);
            }
          }
        }
      }
  }
}

// Sums of x over the windows of 32 FS columns that k_w4_gemm scales at a time: xs[window][row], for the zero points.
// A wave takes four rows x 128 columns.
template <class T, int FS> __global__ __launch_bounds__(256) void k_w4_rowsum(const W4Product p, int64_t rows, float* xs) {
  const int lane = threadIdx.x & 63;
  const int64_t r = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4 + (lane >> 4);
  const int kb = blockIdx.y;
  const u32x4 v = w4_load8(p.x + (r < rows ? r : rows - 1) * p.ldx, (int64_t)kb * 128 + (lane & 15) * 8, p.kc, p.vec);
  float s = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += T::to_f32((uint16_t)v[i]) + T::to_f32((uint16_t)(v[i] >> 16));
#pragma unroll
  for (int d = 1; d < 4 * FS; d <<= 1) s += __shfl_xor(s, d);
  if (r < rows && (lane & (4 * FS - 1)) == 0) xs[((int64_t)kb * (4 / FS) + (lane & 15) / (4 * FS)) * rows + r] = s;
}

// The splits' partial sums, added in their order.
template <class T> __global__ __launch_bounds__(256) void k_w4_join(const W4Product p, int64_t rows) {
  const int64_t quads = (int64_t)p.ct * 4, total = rows * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads, col = (i % quads) * 4;
    if (col >= p.nc) continue;
    const f32x4* from = reinterpret_cast<const f32x4*>(p.part) + i;
    f32x4 v = from[0];
    for (int s = 1; s < p.splits; ++s) v += from[s * total];
    w4_store4<T>(p.y, p.nc, row, col, v);
  }
}

// ---- launchers: one set per (type, kind) -------------------------------------------------------------
struct W4Plan {
  int mt, nt, waves;  // k_w4_rows
  int bm, bn;         // k_w4_gemm (bm = 0: k_w4_rows)
  int fs;
};

template <class T, int KIND, int MT, int NT>
static void w4_rows_go(const W4Args& a, const W4Product& p, const W4Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.nblocks * p.mblocks)), block(64 * pl.waves);
  const size_t lds = (size_t)pl.waves * MT * NT * 1024;
  if (pl.fs == 4)
    hipLaunchKernelGGL((k_w4_rows<T, KIND, MT, NT, 4>), grid, block, lds, st, a, p);
  else if (pl.fs == 2)
    hipLaunchKernelGGL((k_w4_rows<T, KIND, MT, NT, 2>), grid, block, lds, st, a, p);
  else
    hipLaunchKernelGGL((k_w4_rows<T, KIND, MT, NT, 1>), grid, block, lds, st, a, p);
}
template <class T, int KIND, bool GRAD, int MT, int NT, int WM, int WN>
static void w4_gemm_go(const W4Args& a, const W4Product& p, const W4Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.nblocks * p.mblocks), p.splits), block(64 * WM * WN);
  const dim3 sums((unsigned)((a.rows + 15) / 16), p.rb);
  constexpr bool xs = KIND == W4_U4 && !GRAD;
  if (GRAD ? pl.fs >= 2 : pl.fs == 4) {
    if (xs) hipLaunchKernelGGL((k_w4_rowsum<T, 4>), sums, dim3(256), 0, st, p, a.rows, p.xs);
    hipLaunchKernelGGL((k_w4_gemm<T, KIND, GRAD, MT, NT, WM, WN, 4>), grid, block, 0, st, a, p);
  } else if (!GRAD && pl.fs == 2) {
    if (xs) hipLaunchKernelGGL((k_w4_rowsum<T, 2>), sums, dim3(256), 0, st, p, a.rows, p.xs);
    hipLaunchKernelGGL((k_w4_gemm<T, KIND, GRAD, MT, NT, WM, WN, GRAD ? 4 : 2>), grid, block, 0, st, a, p);
  } else {
    if (xs) hipLaunchKernelGGL((k_w4_rowsum<T, 1>), sums, dim3(256), 0, st, p, a.rows, p.xs);
    hipLaunchKernelGGL((k_w4_gemm<T, KIND, GRAD, MT, NT, WM, WN, 1>), grid, block, 0, st, a, p);
  }
}

template <class T, int KIND>
hipError_t w4_launch(const W4Args& a, const W4Product& p, const W4Plan& pl, bool grad, hipStream_t st) {
  if (!pl.bm) {
    if (pl.mt == 1 && pl.nt == 1) w4_rows_go<T, KIND, 1, 1>(a, p, pl, st);
    else if (pl.mt == 1) w4_rows_go<T, KIND, 1, 4>(a, p, pl, st);
    else if (pl.nt == 1) w4_rows_go<T, KIND, 2, 1>(a, p, pl, st);
    else w4_rows_go<T, KIND, 2, 4>(a, p, pl, st);
  } else if (grad) {
    if (pl.bm == 64) w4_gemm_go<T, KIND, true, 1, 2, 2, 2>(a, p, pl, st);
    else if (pl.bn == 256) w4_gemm_go<T, KIND, true, 4, 2, 1, 4>(a, p, pl, st);
    else w4_gemm_go<T, KIND, true, 2, 2, 2, 2>(a, p, pl, st);
  } else {
    if (pl.bm == 64) w4_gemm_go<T, KIND, false, 1, 2, 2, 2>(a, p, pl, st);
    else w4_gemm_go<T, KIND, false, 2, 2, 2, 2>(a, p, pl, st);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.part) return e;
  const int64_t work = (a.rows * p.ct * 4 + 255) / 256;
  hipLaunchKernelGGL((k_w4_join<T>), dim3((unsigned)(work < 2048 ? work : 2048)), dim3(256), 0, st, p, a.rows);
  return hipGetLastError();
}

// The eight instances live in objects of their own (mq_linear4.hip with MQ_W4_PART = 1 .. 8).
#define MQ_W4_LAUNCHER(NAME) hipError_t NAME(const W4Args& a, const W4Product& p, const W4Plan& pl, bool grad, hipStream_t st)
MQ_W4_LAUNCHER(w4_launch_1);
MQ_W4_LAUNCHER(w4_launch_2);
MQ_W4_LAUNCHER(w4_launch_3);
MQ_W4_LAUNCHER(w4_launch_4);
MQ_W4_LAUNCHER(w4_launch_5);
MQ_W4_LAUNCHER(w4_launch_6);
MQ_W4_LAUNCHER(w4_launch_7);
MQ_W4_LAUNCHER(w4_launch_8);
