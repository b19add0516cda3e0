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
  const uint16_t* ts;    // gradient: scales along the contraction times norm, k_w4_turn's [E][GP][128 rb]
  const uint16_t* tz;    // ... and zero points
  const float* down;     // gradient of bfloat16: what w4_half_row's rows have to be multiplied by
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
// ---- few rows --------------------------------------------------------------------------------------
// y = sum over groups of scale * (sum q x - zero sum x), in tiles of v_mfma_f32_16x16x32 with x as the A operand; the sums
// of x are a product with ones.  A workgroup owns NT column tiles and 16 * MT rows; its waves take the 128-blocks of the
// contraction in turn and their sums meet in LDS at the end, in the waves' order.  Everything is in registers on its way: a
// wave keeps D blocks in flight while it works on the D before them.  Rows that are not there repeat the tile's last one
// (their loads fall into the same lines, their results are not stored; masking them off measured slower).  Rows are 16-byte
// aligned and a multiple of 128 long (k_w4_pad).
// Bound by reading the weight: 5 rows through 128256 x 4096 (280 MB) 48 us, 5.8 TB/s (a stream of reads alone reaches 7.0);
// one row through 14336 x 4096 with zero points (31 MB) 9.3 us alone, 8.5 among others, 3.7 TB/s; 2048 x 2048 4.0 us, which
// is the latency of a launch and of two blocks.
template <class T, int KIND, int MT, int NT, int FS, int D> struct W4RowsStage {
  u32x4 w[D][NT], x[D][MT][4];
  uint32_t s[D][NT];  // lane 16 v + c: the scale (and zero point) of column c in window v of the block's 4 / FS
};
template <class T, int KIND, int MT, int NT, int FS>
__global__ __launch_bounds__(MT * NT == 1 ? 1024 : 512) void k_w4_rows(const W4Args a, const W4Product p) {
  extern __shared__ f32x4 w4_red[];
  constexpr int D = MT * NT >= 4 ? 1 : 2, W = 4 / FS;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int quad = lane >> 4, l16 = lane & 15;
  const int tile0 = (int)(blockIdx.x % (uint32_t)p.nblocks) * NT;
  int expert, rows;
  int64_t row0;
  if (!w4_find_tile(a, 16 * MT, (int)(blockIdx.x / (uint32_t)p.nblocks), expert, row0, rows)) return;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = {0, 0, 0, 0};

  if (expert >= 0) {
    const uint32_t* wp[NT];
    int64_t sp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t tile = (int64_t)expert * a.nt + (tile0 + n < a.nt ? tile0 + n : a.nt - 1);
      wp[n] = p.b + tile * a.kt * 256;
      sp[n] = tile * a.gp * 16;
    }
    const uint16_t* xp = p.x + row0 * p.ldx;
    uint32_t xo[MT];  // (rows of a tile lie within 2^31 bytes: others are copied first)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = m * 16 + l16;
      xo[m] = (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)p.ldx + quad * 8;
    }
    typedef W4RowsStage<T, KIND, MT, NT, FS, D> Stage;
    auto load = [&](Stage& g, int kb, int n_blocks) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (d < n_blocks) {
          const int k0 = kb + d * nw;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            g.w[d][n] = *reinterpret_cast<const u32x4*>(wp[n] + (int64_t)k0 * 256 + lane * 4);
            // one load for all windows of the block: it would take as long as a load of the weight for each
            const int64_t at = sp[n] + l16 + (W == 1 ? w4_group(a, k0 * 4) : w4_group(a, k0 * 4 + (quad & (W - 1)) * FS)) * 16;
            if constexpr (KIND == W4_U4)
              g.s[d][n] = static_cast<const uint32_t*>(a.params)[at];
            else
              g.s[d][n] = static_cast<const uint16_t*>(a.params)[at];
          }
        }
      }
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (d < n_blocks) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              g.x[d][m][j] = *reinterpret_cast<const u32x4*>(xp + (int64_t)(kb + d * nw) * 128 + j * 32 + xo[m]);
        }
    };
    auto work = [&](const Stage& g, int n_blocks) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (d < n_blocks) {
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
              const u32x4 v = w4_decode<T, KIND>(g.w[d][n][j], a.lut);
#pragma unroll
              for (int m = 0; m < MT; ++m) tmp[m][n] = T::mfma(g.x[d][m][j], v, tmp[m][n]);
            }
            if constexpr (KIND == W4_U4) {  // sums of x, in the layout of the results
              const u32x4 ones = {T::kOnes, T::kOnes, T::kOnes, T::kOnes};
#pragma unroll
              for (int m = 0; m < MT; ++m) xs[m] = T::mfma(g.x[d][m][j], ones, xs[m]);
            }
            if ((j + 1) % FS == 0) {
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint32_t sv = W == 1 ? g.s[d][n] : (uint32_t)__builtin_amdgcn_ds_bpermute((j / FS * 16 + l16) * 4, (int)g.s[d][n]);
                const float s = (float)h_from_bits(sv);
                const float sz = KIND == W4_U4 ? -(s * (float)h_from_bits(sv >> 16)) : 0.0f;  // exact: 11 x 11 bits
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    acc[m][n][i] = __builtin_fmaf(s, tmp[m][n][i], acc[m][n][i]);
                    if constexpr (KIND == W4_U4) acc[m][n][i] = __builtin_fmaf(sz, xs[m][i], acc[m][n][i]);
                  }
              }
            }
          }
        }
      }
    };
    const int first = (int)((int64_t)a.kt * blockIdx.y / p.splits), last = (int)((int64_t)a.kt * (blockIdx.y + 1) / p.splits);
    int left = (last - first - w + nw - 1) / nw;  // this wave's blocks
    int kb = first + w;
    Stage g0, g1;
    if (left >= D) load(g0, kb, D);
    while (left >= D) {
      left -= D;
      kb += D * nw;
      const bool more = left >= D;
      if (more) load(g1, kb, D);
      work(g0, D);
      if (!more) break;
      left -= D;
      kb += D * nw;
      if (left >= D) load(g0, kb, D);
      work(g1, D);
    }
    if (D > 1 && left > 0) {  // D is at most 2: one block
      load(g0, kb, 1);
      work(g0, 1);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (m * 16 + quad * 4 < rows) w4_red[((w * MT + m) * NT + n) * 64 + lane] = acc[m][n];
  __syncthreads();
  // one thread per result; column 16 n + c of row r: lane 16 (r % 16 / 4) + c, component r % 4
  const float* red = reinterpret_cast<const float*>(w4_red);
  for (int i = threadIdx.x; i < rows * NT * 16; i += blockDim.x) {
    const int c = i % (NT * 16), r = i / (NT * 16);
    const int64_t col = (int64_t)tile0 * 16 + c;
    const float* from = red + ((((r >> 4) * NT + (c >> 4)) * 64 + ((r & 15) >> 2) * 16 + (c & 15)) << 2) + (r & 3);
    float v = from[0];
#pragma unroll 4
    for (int o = 1; o < nw; ++o) v += from[o * MT * NT * 256];
    if (col < p.nc) {
      if (p.bias && expert >= 0 && blockIdx.y == 0) v += T::to_f32(p.bias[expert * p.nc + col]);
      if (p.part)
        p.part[((int64_t)blockIdx.y * a.rows + row0 + r) * (p.ct * 16) + col] = v;
      else
        p.y[(row0 + r) * p.nc + col] = T::from_f32(v);
    }
  }
}

// ---- the gradient's scaled weights ---------------------------------------------------------------------
// Eight weights of one column in float16, scale * (q - zero) times the expert's norm (a power of two): the difference is
// exact for whole zero points up to 2048 (others round it by 2^-11 of itself, as the quantizers' dequantization does), the
// product rounds once: by 2^-11 of the weight, or 2^-25 where it is below 2^-14, 2^-28 or less of what the expert's largest
// scale can make.
template <int KIND> struct W4Scales {
  u32x4 s, z;
  __device__ __forceinline__ u32x4 scaled(uint32_t d, const W4Lut& lut) const {
    const u32x4 v = w4_decode<W4F16, KIND>(d, lut);
    // (whole vectors: the compiler takes a bit cast of one element of a vector for one of its first element)
    w4_h8 q = __builtin_bit_cast(w4_h8, v);
    if constexpr (KIND == W4_U4) q = q - __builtin_bit_cast(w4_h8, z);
    return __builtin_bit_cast(u32x4, q * __builtin_bit_cast(w4_h8, s));
  }
};

// ---- many rows -------------------------------------------------------------------------------------
// A workgroup of WM x WN waves owns 32 MT WM rows and 32 NT WN columns, in tiles of v_mfma_f32_32x32x16 (which leaves six
// vector instructions per matrix instruction free; two 16x16x32 leave four).  Here the activations are the A operand, so
// that a lane's results belong to one column: one scale per tile and lane.  A 128-block of the rows is staged in LDS,
// 256 bytes a row, its sixteen 16-byte pieces permuted by the row (piece c stands at c ^ (row % 16)), so that rows are
// fetched in whole lines and neither the writes nor the operand reads meet in a bank.  The packed weight goes from memory
// straight into the registers of the wave that decodes it: lane l takes row l % 32 of the 32-row tile, the halves of its
// wave the eight columns 8 (l / 32) of every sixteen -- two of the layout's four dwords-quadruples.  Waves stand side by
// side along the columns (WM = 1): no two of them decode the same weights, at the price of reading all rows from LDS each
// (384 rows, 4096 x 14336 with zero points: 91 us, 105 with two by two waves).
// WK = 2: two sets of waves with buffers of their own take the blocks of the contraction in turn, for tiles of 64 rows and
// where a compute unit has only one tile: one wave per SIMD would wait for its own decoding.  Four sets gave nothing more.
// Rows are 16-byte aligned and a multiple of 128 long here: others are copied first (k_w4_pad).
//
// GRAD = false: sums run over exact code values; every FS steps of 32 they are scaled in float32 into the result.  The row
// tiles are taken in two halves, first with the decoding, then with the decoded operands once more, and the scaling of one
// half is dealt out between the products of the other: in one piece it left the matrix cores idle (2000 x 14336 x 4096:
// 232 us).  The second half has the higher priority in the SIMD, so that its products run while another wave decodes (223
// to 218).  Zero points: minus (scale * zero)[column] * (sum of x)[row] per window of FS steps, a float32 product on the
// matrix cores with a contraction over the windows (v_mfma_f32_32x32x2_f32): the vector units took as many instructions
// for it as for the scaling (2048 x 4096 x 4096, groups of 64: 106 us, 100 with the product).
// 2000 rows through 14336 x 4096: 199 to 214 us a call, by the card, 1.10 to 1.18 PFLOP/s (the times of the steps above are
// launches kept apart by a profiler, 206 to 218 us now).  The matrix cores are busy in 0.58 of the cycles, 168 vector
// instructions stand beside every 32 products, and under this load the clock falls to 1.8 GHz: the steps above took 11 % of
// the cycles away and 4 % of the time.
//
// GRAD = true (dx = dy W, operand b transposed): scales change along the contraction, so they are multiplied into the
// weights, which are rounded once to float16 (W4Scales).  It runs in float16 for both types: rows of bfloat16 are brought
// into its range by a power of two each (w4_half_row), where they lose nothing, while weights rounded to bfloat16 would add
// as much error as the rounding of the result (2.4e-3 of the norm against 1.7e-3) and take more instructions to make.  The
// scales along the contraction come with the block's rows through LDS, two to a lane (4096 x 4096 x 4096: 131 us, 149 with
// loads between the products).  2048 rows through 4096 x 4096, one tile to a compute unit: 83 us with zero points, the matrix
// cores busy in 0.35 of the cycles, the waves waiting in 0.33; 4096 rows without: 1.05 PFLOP/s, turning included.  What bounds
// that tile of 128 x 256 are its instructions: with zero points 386 vector ones stand beside every 64 products (float16 rows),
// the subtraction q - zero being compiled value by value, 12 instructions where 4 would do; and for rows of bfloat16 (475) the
// compiler does not see that the tile's place is the same in all lanes, keeps the buffer descriptors in vector registers and
// puts each of the block's 14 to 16 loads into a loop over their values.  With two sets of waves 76 bytes a lane are spilled,
// outside the loop.
template <int NT, int W> struct W4Ahead {  // what a wave holds of a block that is on its way
  u32x4 b[NT][2];
  uint32_t s[NT][W];
};
#ifdef __HIP_DEVICE_COMPILE__
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_buffer(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000);  // raw 32-bit data
}
#endif
typedef __attribute__((address_space(3))) void w4_lds_t;

template <class T, class TO, int KIND, bool GRAD, int MT, int NT, int WM, int WN, int WK, int FS>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void k_w4_gemm(const W4Args a, const W4Product p) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass has no buffer descriptors; it needs the kernel's name only)
  constexpr int BM = 32 * MT * WM, NW = WM * WN, CH = BM / 4 / NW;  // 1 KiB pieces (4 rows) per wave
  constexpr int W = 4 / FS;                                         // windows of a block with a scale each
  constexpr bool XS = KIND == W4_U4 && !GRAD;                       // zero points, taken away through the rows' sums
  constexpr int PAIRS = W == 4 ? 2 : 1;
  static_assert(BM / 4 % NW == 0 && BM % 64 == 0, "the rows of a block are dealt evenly");
  constexpr int SETS = FS == 1 ? NT : 1;          // gradient: groups under a wave's 32 NT columns
  constexpr int SZ = KIND == W4_U4 ? 2 : 1;       // scales, and zero points
  // One array for the rows' blocks [WK][2][BM * 16] and the gradient's scales [WK * NW][2][SETS][SZ][16]: of two arrays the
  // compiler would order every read behind all loads on their way into LDS, those of the other buffer among them.
  constexpr int ROWS = WK * 2 * BM * 16, SCALES = GRAD ? WK * NW * 2 * SETS * SZ * 16 : 0;
  __shared__ u32x4 lds_all[ROWS + SCALES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l32 = lane & 31;
  const int w = wave % NW, wk = wave / NW, wm = w % WM, wn = w / WM;
  u32x4* const lds = lds_all + wk * 2 * BM * 16;
  u32x4* const lds_sc = lds_all + ROWS + wave * 2 * SETS * SZ * 16;  // of this wave alone
  // Workgroups go to the eight chiplets in turn: row tile 8 i + c belongs to chiplet c, whose L2 then holds its rows for all
  // columns; the row tiles behind the last eight are dealt out by columns.
  const uint32_t whole = (uint32_t)p.mblocks / 8 * (uint32_t)p.nblocks * 8, id = blockIdx.x;
  const uint32_t rows8 = id < whole ? (uint32_t)p.mblocks / 8 : (uint32_t)p.mblocks % 8;
  const uint32_t at = id < whole ? id / 8 : id - whole;
  const int mb = (int)(id < whole ? at % rows8 * 8 + id % 8 : (uint32_t)p.mblocks / 8 * 8 + at % rows8);
  const int64_t tile0 = ((int64_t)(at / rows8) * WN + wn) * NT;  // tiles of 32 columns
  int expert, rows;
  int64_t row0;
  if (!w4_find_tile(a, BM, mb, expert, row0, rows)) return;
  f32x16 acc[MT][NT];     // GRAD, zero points: the matrix instructions' own sums
  float sum[MT][NT][16];  // forward: the scaled sums (single registers, where they are no matrix operand)
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
    // The loads go through buffer descriptors: one offset per lane for the whole loop, the block's in a scalar register.  (The
    // descriptors are scalar too but in the gradient's large tile with a bfloat16 result: see above.)
    const int64_t bt0 = (tile0 - wn * NT) * 2 < p.ct ? (tile0 - wn * NT) * 2 : p.ct - 1;  // the workgroup's first 16-row tile
    const auto bsrc = w4_buffer(p.b + ((int64_t)expert * p.ct + bt0) * p.rb * 256, (uint32_t)(WN * NT * 2) * (uint32_t)p.rb * 1024u);
    const auto xsrc = w4_buffer(p.x + row0 * p.ldx, (uint32_t)(((int64_t)(rows - 1) * p.ldx + (int64_t)p.rb * 128) * 2));
    uint32_t bo[NT];
    int64_t pt[NT];  // forward: this lane's column in the parameters of group 0
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      int64_t t = (tile0 + n) * 2 + (l32 >> 4);
      t = t < p.ct ? t : p.ct - 1;
      bo[n] = (uint32_t)(t - bt0) * (uint32_t)p.rb * 1024u + (half * 16 + (lane & 15)) * 16;
      pt[n] = ((int64_t)expert * p.ct + t) * a.gp * 16 + (lane & 15);
    }
    uint32_t xo[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int r = (w * CH + c) * 4 + (lane >> 4);
      xo[c] = (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)p.ldx * 2u + (((lane & 15) ^ (r & 15)) * 16);
    }
    const int kb0 = (int)((int64_t)p.rb * blockIdx.y / p.splits), kb1 = (int)((int64_t)p.rb * (blockIdx.y + 1) / p.splits);
    // gradient: the wave's scales (and zero points) along the contraction, two to a lane
    __amdgpu_buffer_rsrc_t ssrc[GRAD ? SETS : 1][SZ];
    if constexpr (GRAD) {
#pragma unroll
      for (int g = 0; g < SETS; ++g) {
        const int64_t c = tile0 + g, last = (p.ct - 1) >> 1;
        const int64_t from = ((int64_t)expert * a.gp + w4_group(a, (int)(c < last ? c : last))) * p.rb * 128;
        ssrc[g][0] = w4_buffer(p.ts + from, (uint32_t)p.rb * 256u);
        if constexpr (SZ == 2) ssrc[g][SZ - 1] = w4_buffer(p.tz + from, (uint32_t)p.rb * 256u);
      }
    }
    W4Ahead<NT, GRAD ? 1 : W> next;
    auto fetch = [&](int kb, int buf, W4Ahead<NT, GRAD ? 1 : W>& to) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xsrc, (w4_lds_t*)(lds + buf * BM * 16 + (w * CH + c) * 64), 16, xo[c], kb * 256, 0, 0);
      if constexpr (GRAD) {
#pragma unroll
        for (int g = 0; g < SETS; ++g) {
#pragma unroll
          for (int z = 0; z < SZ; ++z)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ssrc[g][z], (w4_lds_t*)(lds_sc + ((buf * SETS + g) * SZ + z) * 16), 4, lane * 4, kb * 256, 0, 0);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) to.b[n][h] = __builtin_amdgcn_raw_buffer_load_b128(bsrc, bo[n] + h * 512, kb * 1024, 0);
        if constexpr (!GRAD) {
#pragma unroll
          for (int v = 0; v < W; ++v)
            to.s[n][v] = static_cast<const uint16_t*>(a.params)[(pt[n] + w4_group(a, kb * 4 + v * FS) * 16) * (KIND == W4_U4 ? 2 : 1)];
        }
      }
    };
    // forward: the row tiles' halves.  `hi` holds the second half's unscaled sums until the next window's first products,
    // sh their scales.
    constexpr int MH = MT / 2;
    static_assert(GRAD || MT % 2 == 0, "two halves");
    f32x16 hi[GRAD ? 1 : MH][NT];
    float sh[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      sh[n] = 0;
#pragma unroll
      for (int m = 0; m < (GRAD ? 1 : MH); ++m) hi[m][n] = w4_zero16();
    }
    // the share of product step `step` in scaling a half's sums: none behind the first step, while they are on their way
    auto add = [&](const f32x16 (&from)[GRAD ? 1 : MH][NT], const float (&by)[NT], int m0, int step) {
      constexpr int ALL = MH * NT * 16, S = 2 * FS - 1;
#pragma unroll
      for (int i = 0; i < ALL; ++i) {
        if (step == 0 || i < ALL * (step - 1) / S || i >= ALL * step / S) continue;
        const int m = i / (16 * NT), n = i / 16 % NT, r = i % 16;
        if constexpr (XS)
          acc[m0 + m][n][r] = __builtin_fmaf(by[n], from[m][n][r], acc[m0 + m][n][r]);
        else
          sum[m0 + m][n][r] = __builtin_fmaf(by[n], from[m][n][r], sum[m0 + m][n][r]);
      }
    };
    if (kb0 + wk < kb1) fetch(kb0 + wk, 0, next);
    __syncthreads();
    for (int it = 0; kb0 + it * WK < kb1; ++it) {
      const int kb = kb0 + it * WK + wk, buf = it & 1;
      const W4Ahead<NT, GRAD ? 1 : W> cur = next;
      if (kb + WK < kb1) fetch(kb + WK, buf ^ 1, next);
      const u32x4* xb = lds + buf * BM * 16 + (wm * MT * 32 + l32) * 16;
      const int turn = (l32 & 15) ^ half;
      if (WK > 1 && kb >= kb1) {
        // the other waves' last block: nothing for this half
      } else if constexpr (!GRAD) {
        // What the zero points take away of two windows at a time -- of this block, or (one window to a block) of every
        // second block and the one before it: the lanes' halves hold a window each.
        const bool pair_now = W > 1 || buf || kb + WK >= kb1, there = W > 1 || buf || !half;
        float zx[PAIRS][MT], zz[PAIRS][NT];
        uint32_t zq[PAIRS][NT];
        auto scaled_zeros = [&]() {
#pragma unroll
          for (int v = 0; v < PAIRS; ++v)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              zz[v][n] = there ? -(float)h_from_bits(zq[v][n]) * (float)h_from_bits(zq[v][n] >> 16) : 0.0f;  // exact: 11 x 11 bits
        };
        if constexpr (XS) {
          if (pair_now) {
#pragma unroll
            for (int v = 0; v < PAIRS; ++v) {
              const int win = W > 1 ? kb * W + 2 * v + half : buf && !half ? kb - WK : kb;
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const int r = (wm * MT + m) * 32 + l32;
                zx[v][m] = p.xs[(int64_t)win * a.rows + row0 + (r < rows ? r : rows - 1)];
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) zq[v][n] = static_cast<const uint32_t*>(a.params)[pt[n] + w4_group(a, win * FS) * 16];
            }
            // Two sets of waves, a compute unit's only tile, must not wait here for what they have just asked for (384 rows,
            // 4096 x 14336: 84 us, 92 with this line for both); other tiles hide that and gain registers (2048 x 4096 x
            // 4096: 88.5, 91 without).
            if (WK == 1) scaled_zeros();
          }
        }
        f32x16 lo[MH][NT];
        u32x4 xv[2][MH];
        // operands of product step t = 4 FS window + 2 FS half + step, read from LDS a step ahead
        auto rows_of = [&](int t) {
#pragma unroll
          for (int m = 0; m < MH; ++m) {
            const int st = t / (4 * FS) * 2 * FS + t % (2 * FS), first = t / (2 * FS) % 2 * MH;
            if (t < 16) xv[t & 1][m] = xb[(first + m) * 512 + ((2 * st) ^ turn)];
          }
        };
        rows_of(0);
#pragma unroll
        for (int v = 0; v < W; ++v) {
          float s[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            s[n] = (float)h_from_bits(cur.s[n][v]);
            asm("" : "+v"(s[n]));  // a float32 register: v_fmac_f32 issues faster than the mixed fma the compiler would choose
          }
          // (each step is fixed in its place: left alone, the scheduler gathers the scaling behind the products)
          u32x4 q[2 * FS][NT];
#pragma unroll
          for (int i = 0; i < 2 * FS; ++i) {  // the first half of the row tiles; the second's sums of the window before
            const int st = v * 2 * FS + i, t = v * 4 * FS + i;
            rows_of(t + 1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              q[i][n] = w4_decode<T, KIND>(cur.b[n][st & 1][st >> 1], a.lut);
#pragma unroll
              for (int m = 0; m < MH; ++m)
                lo[m][n] = T::mfma32(xv[t & 1][m], q[i][n], i == 0 ? w4_zero16() : lo[m][n]);
            }
            add(hi, sh, MH, i);
            __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int i = 0; i < 2 * FS; ++i) {
            const int t = v * 4 * FS + 2 * FS + i;
            rows_of(t + 1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int m = 0; m < MH; ++m)
                hi[m][n] = T::mfma32(xv[t & 1][m], q[i][n], i == 0 ? w4_zero16() : hi[m][n]);
            add(lo, s, 0, i);
            __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_s_setprio(0);
#pragma unroll
          for (int n = 0; n < NT; ++n) sh[n] = s[n];
        }
        if constexpr (XS) {
          if (pair_now) {
            if (WK > 1) scaled_zeros();
#pragma unroll
            for (int v = 0; v < PAIRS; ++v)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(zx[v][m], zz[v][n], acc[m][n], 0, 0, 0);
          }
        }
      } else {
        // Two products to a step hide no LDS load: the operands of the whole block at once.
        constexpr bool ALL = MT * NT <= 2;
        u32x4 xa[ALL ? MT : 1][ALL ? 8 : 1];
        if constexpr (ALL) {
#pragma unroll
          for (int st = 0; st < 8; ++st)
#pragma unroll
            for (int m = 0; m < MT; ++m) xa[m][st] = xb[m * 512 + ((2 * st) ^ turn)];
        }
#pragma unroll
        for (int st = 0; st < 8; ++st) {
          W4Scales<KIND> sc[SETS];
#pragma unroll
          for (int g = 0; g < SETS; ++g) {
            sc[g].s = lds_sc[(buf * SETS + g) * SZ * 16 + st * 2 + half];
            if constexpr (SZ == 2) sc[g].z = lds_sc[((buf * SETS + g) * SZ + 1) * 16 + st * 2 + half];
          }
          u32x4 xv[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) xv[m] = ALL ? xa[ALL ? m : 0][ALL ? st : 0] : xb[m * 512 + ((2 * st) ^ turn)];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const u32x4 v = sc[FS == 1 ? n : 0].scaled(cur.b[n][st & 1][st >> 1], a.lut);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][n] = T::mfma32(xv[m], v, acc[m][n]);
          }
        }
      }
      __syncthreads();
    }
    if constexpr (!GRAD) {
#pragma unroll
      for (int i = 1; i < 2 * FS; ++i) add(hi, sh, MH, i);
    }
    if constexpr (XS) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[m][n][i] = acc[m][n][i];
    }
    if constexpr (GRAD) {
      const float down = 1.0f / a.norm[expert];  // a power of two, as are the rows' factors
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = (wm * MT + m) * 32 + q * 8 + half * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float row = TO::kHalf ? 1.0f : p.down[row0 + (r + i < rows ? r + i : rows - 1)];
#pragma unroll
            for (int n = 0; n < NT; ++n) sum[m][n][4 * q + i] = acc[m][n][4 * q + i] * down * row;
          }
        }
    }
  }
  if constexpr (WK > 1) {  // the halves' sums, through the buffers that nobody reads any more
    float* red = reinterpret_cast<float*>(lds_all) + (w * MT * NT * 16) * 64 + lane;
    static_assert(WK == 2 && sizeof(lds_all) >= NW * MT * NT * 16 * 64 * 4, "the sums of one half fit");
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (wk) red[((m * NT + n) * 16 + i) * 64] = sum[m][n][i];
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[m][n][i] += red[((m * NT + n) * 16 + i) * 64];
  }
  // A lane holds one column; neighbours exchange half of their rows, so that each stores pairs of columns: the even lane
  // of a pair rows 0, 2, .. of its registers, the odd one rows 1, 3, ..
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t col = (tile0 + n) * 32 + (l32 & ~1);
    float b0 = 0, b1 = 0;
    if (p.bias && expert >= 0 && blockIdx.y == 0) {
      if (col < p.nc) b0 = TO::to_f32(p.bias[expert * p.nc + col]);
      if (col + 1 < p.nc) b1 = TO::to_f32(p.bias[expert * p.nc + col + 1]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const bool odd = lane & 1;
        const float mine = odd ? sum[m][n][i + 1] : sum[m][n][i], other = odd ? sum[m][n][i] : sum[m][n][i + 1];
        const float got = f_from_bits((uint32_t)__builtin_amdgcn_mov_dpp((int)__builtin_bit_cast(uint32_t, other), 0xB1, 0xF, 0xF, true));  // lane ^ 1
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
              *reinterpret_cast<uint32_t*>(to) = TO::pack(v0, v1);
            } else {
              to[0] = TO::from_f32(v0);
              if (col + 1 < p.nc) to[1] = TO::from_f32(v1);
            }
          }
        }
      }
  }
#endif
}

// Sums of x over the windows of 32 FS columns that k_w4_gemm scales at a time: xs[window][row], for the zero points.
// A wave takes four rows x 128 columns.  Bound by reading x (2048 x 4096, 16 MB: 5.4 us, 3.1 TB/s); every column tile of
// the product would have to add them up again.
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

// The splits' partial sums, added in their order.  Bound by a launch and by the sums' bytes, which the caches hold (77 x
// 5632, two splits, 3.5 MB: 4 us of which the launch is 2).
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
  int bm, bn, wk;     // k_w4_gemm (bm = 0: k_w4_rows)
  int fs;
};

template <class T, int KIND, int MT, int NT>
static void w4_rows_go(const W4Args& a, const W4Product& p, const W4Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.nblocks * p.mblocks), p.splits), block(64 * pl.waves);
  const size_t lds = (size_t)pl.waves * MT * NT * 1024;
  if (pl.fs == 4)
    hipLaunchKernelGGL((k_w4_rows<T, KIND, MT, NT, 4>), grid, block, lds, st, a, p);
  else if (pl.fs == 2)
    hipLaunchKernelGGL((k_w4_rows<T, KIND, MT, NT, 2>), grid, block, lds, st, a, p);
  else
    hipLaunchKernelGGL((k_w4_rows<T, KIND, MT, NT, 1>), grid, block, lds, st, a, p);
}
template <class T, class TO, int KIND, bool GRAD, int MT, int NT, int WM, int WN, int WK>
static void w4_gemm_go(const W4Args& a, const W4Product& p, const W4Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.nblocks * p.mblocks), p.splits), block(64 * WM * WN * WK);
  const dim3 sums((unsigned)((a.rows + 15) / 16), p.rb);
  constexpr bool xs = KIND == W4_U4 && !GRAD;
  if (GRAD ? pl.fs >= 2 : pl.fs == 4) {
    if (xs) hipLaunchKernelGGL((k_w4_rowsum<T, 4>), sums, dim3(256), 0, st, p, a.rows, p.xs);
    hipLaunchKernelGGL((k_w4_gemm<T, TO, KIND, GRAD, MT, NT, WM, WN, WK, 4>), grid, block, 0, st, a, p);
  } else if (!GRAD && pl.fs == 2) {
    if (xs) hipLaunchKernelGGL((k_w4_rowsum<T, 2>), sums, dim3(256), 0, st, p, a.rows, p.xs);
    hipLaunchKernelGGL((k_w4_gemm<T, TO, KIND, GRAD, MT, NT, WM, WN, WK, GRAD ? 4 : 2>), grid, block, 0, st, a, p);
  } else {
    if (xs) hipLaunchKernelGGL((k_w4_rowsum<T, 1>), sums, dim3(256), 0, st, p, a.rows, p.xs);
    hipLaunchKernelGGL((k_w4_gemm<T, TO, KIND, GRAD, MT, NT, WM, WN, WK, 1>), grid, block, 0, st, a, p);
  }
}

template <class T, int KIND>
hipError_t w4_launch(const W4Args& a, const W4Product& p, const W4Plan& pl, bool grad, hipStream_t st) {
  if (!pl.bm) {
    if (pl.mt == 1 && pl.nt == 1) w4_rows_go<T, KIND, 1, 1>(a, p, pl, st);
    else if (pl.mt == 1 && pl.nt == 2) w4_rows_go<T, KIND, 1, 2>(a, p, pl, st);
    else if (pl.mt == 1) w4_rows_go<T, KIND, 1, 4>(a, p, pl, st);
    else if (pl.nt == 1) w4_rows_go<T, KIND, 2, 1>(a, p, pl, st);
    else if (pl.nt == 2) w4_rows_go<T, KIND, 2, 2>(a, p, pl, st);
    else w4_rows_go<T, KIND, 2, 4>(a, p, pl, st);
  } else if (grad) {
    if (pl.bm == 64) w4_gemm_go<W4F16, T, KIND, true, 2, 1, 1, 4, 2>(a, p, pl, st);
    else if (pl.wk == 2) w4_gemm_go<W4F16, T, KIND, true, 4, 2, 1, 4, 2>(a, p, pl, st);
    else w4_gemm_go<W4F16, T, KIND, true, 4, 2, 1, 4, 1>(a, p, pl, st);
  } else {
    if (pl.bm == 64) w4_gemm_go<T, T, KIND, false, 2, 1, 1, 4, 2>(a, p, pl, st);
    else if (pl.wk == 2) w4_gemm_go<T, T, KIND, false, 4, 1, 1, 4, 2>(a, p, pl, st);
    else w4_gemm_go<T, T, KIND, false, 4, 1, 1, 4, 1>(a, p, pl, st);
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
