// Products with weights held in 4 bits (mq_linear4, mq_linear4_grad), their packing and unpacking, and the bias's
// gradient.  Layout and decoding: mq_w4.h; the product kernels: mq_w4_kernels.h.
//
// MQ_W4_PART = 0: host side and the small kernels; 1 .. 8: the product kernels of one element type and kind of codes.
#include "mq_w4_kernels.h"

#ifndef MQ_W4_PART
#define MQ_W4_PART 0
#endif

#if MQ_W4_PART == 1
MQ_W4_LAUNCHER(w4_launch_1) { return w4_launch<W4F16, W4_S4>(a, p, pl, grad, st); }
#elif MQ_W4_PART == 2
MQ_W4_LAUNCHER(w4_launch_2) { return w4_launch<W4F16, W4_U4>(a, p, pl, grad, st); }
#elif MQ_W4_PART == 3
MQ_W4_LAUNCHER(w4_launch_3) { return w4_launch<W4F16, W4_LUT>(a, p, pl, grad, st); }
#elif MQ_W4_PART == 4
MQ_W4_LAUNCHER(w4_launch_4) { return w4_launch<W4F16, W4_FP4>(a, p, pl, grad, st); }
#elif MQ_W4_PART == 5
MQ_W4_LAUNCHER(w4_launch_5) { return w4_launch<W4BF16, W4_S4>(a, p, pl, grad, st); }
#elif MQ_W4_PART == 6
MQ_W4_LAUNCHER(w4_launch_6) { return w4_launch<W4BF16, W4_U4>(a, p, pl, grad, st); }
#elif MQ_W4_PART == 7
MQ_W4_LAUNCHER(w4_launch_7) { return w4_launch<W4BF16, W4_LUT>(a, p, pl, grad, st); }
#elif MQ_W4_PART == 8
MQ_W4_LAUNCHER(w4_launch_8) { return w4_launch<W4BF16, W4_FP4>(a, p, pl, grad, st); }
#else

// ---- packing ---------------------------------------------------------------------------------------
struct PackArgs {
  const void* codes;   // [E][N][K]: bytes, or float16 table values
  const uint16_t* scale;
  const uint16_t* zero;
  uint32_t* data;
  void* params;
  int64_t n, k;
  int32_t nt, kt, g, gp;  // g: groups that the scales have per row
  float values[16];
};

// One thread per dword: eight codes of one row.  Consecutive threads take consecutive octets of a row, so that a wave
// reads four rows' 128 bytes each.  Runs once per weight; its byte loads bound it (14336 x 4096: 39 us, 2.3 TB/s).
template <int KIND> __global__ __launch_bounds__(256) void k_w4_pack(const PackArgs p) {
  const int t = threadIdx.x, octet = t & 15, r = t >> 4;
  const int64_t n = (int64_t)blockIdx.y * 16 + r, k0 = (int64_t)blockIdx.x * 128 + octet * 8;
  const int64_t e = blockIdx.z;
  uint32_t d = 0;
  if (n < p.n) {
    const int64_t at = (e * p.n + n) * p.k;
    for (int i = 0; i < 8; ++i) {
      if (k0 + i >= p.k) break;
      uint32_t c = 0;
      if constexpr (KIND == W4_U4) {
        c = static_cast<const uint8_t*>(p.codes)[at + k0 + i];
        c = c < 15 ? c : 15;
      } else if constexpr (KIND == W4_S4) {
        const int v = static_cast<const int8_t*>(p.codes)[at + k0 + i];
        const int m = v < 0 ? -v : v;
        c = (uint32_t)(m < 7 ? m : 7) | (v < 0 ? 8u : 0u);
      } else {
        const float v = (float)static_cast<const half_t*>(p.codes)[at + k0 + i];
        for (int q = 1; q < 16; ++q)
          if (p.values[q] == v && v != 0.0f) c = q;
      }
      d |= w4_put<KIND>(c, i);
    }
  }
  const int lane = (octet & 3) * 16 + r, j = octet >> 2;
  p.data[((e * p.nt + blockIdx.y) * p.kt + blockIdx.x) * 256 + lane * 4 + j] = d;
}
__global__ __launch_bounds__(256) void k_w4_params(const PackArgs p, int64_t total) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t grp = (i >> 4) % p.gp, tile = (i >> 4) / p.gp, e = tile / p.nt, n = (tile % p.nt) * 16 + (i & 15);
    uint32_t s = 0, z = 0;
    if (n < p.n && grp < p.g) {
      const int64_t at = (e * p.n + n) * p.g + grp;
      s = p.scale[at];
      if (p.zero) z = p.zero[at];
    }
    if (p.zero)
      static_cast<uint32_t*>(p.params)[i] = s | (z << 16);
    else
      static_cast<uint16_t*>(p.params)[i] = (uint16_t)s;
  }
}

// The float16 weight: h(h(q - zero) * scale), the arithmetic of the quantizers' dequantization, eight values to a thread.
// Bound by its bytes.
template <int KIND> __global__ __launch_bounds__(256) void k_w4_unpack(const W4Args a, uint16_t* out) {
  const int t = threadIdx.x, octet = t & 15, r = t >> 4;
  const int64_t n = (int64_t)blockIdx.y * 16 + r, k0 = (int64_t)blockIdx.x * 128 + octet * 8, e = blockIdx.z;
  if (n >= a.n || k0 >= a.k) return;
  const int64_t tile = e * a.nt + blockIdx.y;
  const uint32_t d = a.data[(tile * a.kt + blockIdx.x) * 256 + ((octet & 3) * 16 + r) * 4 + (octet >> 2)];
  float f[8];
  w4_decode_f32<KIND>(d, a.lut, f);
  const int64_t at = (tile * a.gp + w4_group(a, (int)(k0 >> 5))) * 16 + r;
  float s, z = 0;
  if constexpr (KIND == W4_U4) {
    const uint32_t v = static_cast<const uint32_t*>(a.params)[at];
    s = (float)h_from_bits(v);
    z = (float)h_from_bits(v >> 16);
  } else {
    s = (float)h_from_bits(static_cast<const uint16_t*>(a.params)[at]);
  }
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float q = f[i];
    if constexpr (KIND == W4_U4) q = (float)h_from_bits(f2h_bits(q - z));
    h[i] = f2h_bits(q * s) & 0xFFFFu;
  }
  uint16_t* to = out + (e * a.n + n) * a.k + k0;
  if (a.k % 8 == 0 && (uintptr_t)out % 16 == 0) {
    *reinterpret_cast<u32x4*>(to) = u32x4{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < a.k) to[i] = (uint16_t)h[i];
  }
}

// ---- rows that the products cannot read as they are -------------------------------------------------
// Rows of any stride, alignment and length -> rows of 128 rb elements, zeros behind the end.  A copy before the products
// keeps the bounds of rows out of their loops; its element loads bound it (2048 rows of 4096 at an odd address: 12 us, 2.7 TB/s).
__global__ __launch_bounds__(256) void k_w4_pad(const W4Product p, int64_t rows, uint16_t* to) {
  const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), k = (int64_t)blockIdx.y * 128 + (threadIdx.x & 15) * 8;
  if (r < rows) *reinterpret_cast<u32x4*>(to + r * p.rb * 128 + k) = w4_load8(p.x + r * p.ldx, k, p.kc, p.vec);
}

// Rows of bfloat16 -> rows of float16 times a power of two each, which brings a row's largest value into [2^14, 2^15):
// eight significant bits fit float16's eleven, so nothing is lost but of values more than 2^28 below the largest.
// down[row]: the inverse factor.  A row that holds an infinity or NaN keeps its scale (its results are not finite anyway).
// One wave to a row; the second pass finds the row in the caches.  It shares k_w4_turn's launch, which leaves compute units
// free: 2048 rows of 4096 beside the turning of 4096 x 4096 take 11.4 us, the turning alone 7.7.
__device__ __forceinline__ void w4_half_row(const W4Product& p, int64_t row, uint16_t* to, float* down) {
  const int lane = threadIdx.x & 63;
  const uint16_t* from = p.x + row * p.ldx;
  uint32_t m = 0;
#pragma unroll 4
  for (int64_t k = lane * 8; k < p.kc; k += 512) {
    const u32x4 v = w4_load8(from, k, p.kc, p.vec);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = v[i] & 0x7FFFu, hi = v[i] >> 16 & 0x7FFFu;
      m = m > lo ? m : lo;
      m = m > hi ? m : hi;
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
    m = m > o ? m : o;
  }
  const int e = (int)(m >> 7);
  int shift = e == 255 ? 0 : 141 - (e ? e : 1);
  if (shift > 126) shift = 126;
  const float up = f_from_bits((uint32_t)(127 + shift) << 23);
  if (lane == 0) down[row] = f_from_bits((uint32_t)(127 - shift) << 23);
#pragma unroll 4
  for (int64_t k = lane * 8; k < (int64_t)p.rb * 128; k += 512) {
    u32x4 v = w4_load8(from, k, p.kc, p.vec);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = W4F16::pack(f_from_bits(v[i] << 16) * up, f_from_bits(v[i] & 0xFFFF0000u) * up);
    *reinterpret_cast<u32x4*>(to + row * p.rb * 128 + k) = v;
  }
}

// ---- the transposed operand of the gradient ----------------------------------------------------------
// dx = dy W contracts over the weight's rows: the same codes in the same layout with the roles of rows and columns
// exchanged.  A wave turns 128 rows x 128 columns, a thread 8 rows x 32 columns: it
// reads four dwords of each row at once (8 x 16 contiguous bytes) and turns four blocks of 8 x 8 nibbles in registers, by
// exchanging nibbles, bytes and halves between pairs of dwords (32 instructions a block).  The turned dwords go through
// LDS, so that whole tiles are stored.  Bound by its bytes, half a byte read and written per weight: 32 experts of
// 2048 x 2048 (134 MB) with 4096 rows of bfloat16 beside them 36 us, 3.7 TB/s.  One wave to a workgroup: nobody waits for
// another's loads.
// It also writes the scales (and zero points) along the contraction, in the form that W4Scales loads.
struct TurnArgs {
  uint32_t* out;  // [E][ct][rb][64][4]
  uint16_t* ts;   // [E][GP][128 rb]
  uint16_t* tz;
  int32_t ct, rb;
  uint32_t blocks;   // workgroups that turn; the others bring rows of bfloat16 to float16
  uint16_t* half;
  float* down;
};
// Nibble r of b[c] = nibble c of a[r].
__device__ __forceinline__ void w4_turn8(uint32_t* a) {
#pragma unroll
  for (int r = 0; r < 8; r += 2) {
    const uint32_t x = a[r], y = a[r + 1];
    a[r] = (x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u);
    a[r + 1] = ((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (i & 1) + (i >> 1) * 4;
    const uint32_t x = a[r], y = a[r + 2];
    a[r] = __builtin_amdgcn_perm(y, x, 0x06020400u);
    a[r + 2] = __builtin_amdgcn_perm(y, x, 0x07030501u);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t x = a[r], y = a[r + 4];
    a[r] = __builtin_amdgcn_perm(y, x, 0x05040100u);
    a[r + 4] = __builtin_amdgcn_perm(y, x, 0x07060302u);
  }
}
template <int KIND> __global__ __launch_bounds__(64) void k_w4_turn(const W4Args a, const TurnArgs t, const W4Product p) {
  __shared__ u32x4 lds[512];
  if (blockIdx.x >= t.blocks) {
    for (int64_t row = blockIdx.x - t.blocks; row < a.rows; row += gridDim.x - t.blocks) w4_half_row(p, row, t.half, t.down);
    return;
  }
  const int lane = threadIdx.x, kq = lane & 3, nb = lane >> 2;
  const uint32_t kt = blockIdx.x % (uint32_t)a.kt, rt = blockIdx.x / (uint32_t)a.kt % (uint32_t)t.rb;
  const int64_t e = blockIdx.x / (uint32_t)a.kt / (uint32_t)t.rb;
  if (a.counts && a.counts[e] <= 0) return;
  const int64_t nt = (int64_t)rt * 8 + (nb >> 1);
  u32x4 in[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    in[i] = {0, 0, 0, 0};
    if (nt < a.nt)
      in[i] = *reinterpret_cast<const u32x4*>(a.data + ((e * a.nt + nt) * a.kt + kt) * 256 + (kq * 16 + (nb & 1) * 8 + i) * 4);
  }
  uint32_t* flat = reinterpret_cast<uint32_t*>(lds);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // the code at slot i of a dword stands in nibble at(i); rows and columns are both taken in the order of the nibbles
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = KIND == W4_FP4 ? i : i < 4 ? 2 * i : 2 * (i - 4) + 1;
      uint32_t d = in[i][j];
      if constexpr (KIND == W4_S4 || KIND == W4_LUT) d = (d & 0x77777777u) | (__builtin_amdgcn_alignbit(d, d, 4) & 0x88888888u);
      b[at] = d;
    }
    w4_turn8(b);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int at = KIND == W4_FP4 ? q : q < 4 ? 2 * q : 2 * (q - 4) + 1;
      uint32_t d = b[at];
      if constexpr (KIND == W4_S4 || KIND == W4_LUT) d = (d & 0x77777777u) | (__builtin_amdgcn_alignbit(d, d, 28) & 0x88888888u);
      const int k = j * 32 + kq * 8 + q;  // column in the block; n = 8 nb + i: dword nb / 4 of lane 16 (nb % 4) + k % 16
      const int pos = (k >> 4) * 256 + ((nb & 3) * 16 + (k & 15)) * 4 + (nb >> 2);
      flat[pos ^ (((pos >> 6 & 3) | (pos >> 8 & 1) << 2) << 2)] = d;  // (spread over the banks)
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t tile = (int64_t)kt * 8 + i;
    if (tile < t.ct) {
      const int pos = i * 64 + lane;
      reinterpret_cast<u32x4*>(t.out)[((e * t.ct + tile) * t.rb + rt) * 64 + lane] = lds[pos ^ ((pos >> 4 & 3) | (pos >> 6 & 1) << 2)];
    }
  }
  // scales of the groups that begin in this block of columns
  const float up = a.norm[e];
  for (int j = 0; j < 4; ++j) {
    const int step = kt * 4 + j, grp = w4_group(a, step);
    if (grp * a.gu != step || grp >= a.gp) continue;
    for (int i = lane; i < 128; i += 64) {
      const int64_t n = (int64_t)rt * 128 + i, tile = n >> 4;
      float s = 0, z = 0;
      if (tile < a.nt) {
        const int64_t at = ((e * a.nt + tile) * a.gp + grp) * 16 + (n & 15);
        if constexpr (KIND == W4_U4) {
          const uint32_t v = static_cast<const uint32_t*>(a.params)[at];
          s = (float)h_from_bits(v);
          z = (float)h_from_bits(v >> 16);
        } else {
          s = (float)h_from_bits(static_cast<const uint16_t*>(a.params)[at]);
        }
      }
      const int64_t to = (e * a.gp + grp) * t.rb * 128 + n;
      t.ts[to] = W4F16::from_f32(s * up);  // exact down to 2^-14, off by 2^-25 at most below
      if constexpr (KIND == W4_U4) t.tz[to] = W4F16::from_f32(z);
    }
  }
}

// ---- the bias's gradient -----------------------------------------------------------------------------
// Sums of dy's rows per expert in float32: 64 columns to a workgroup, whose sixteen waves take the rows in turn; where an
// expert has many rows they are cut into runs, whose sums a second launch adds in order.  Bound by reading dy once more,
// which the caches mostly hold, and by a launch (509 x 2048: 5.4 us).  No atomics: the order of the sum is fixed.
struct BiasArgs {
  const uint16_t* dy;
  const int32_t* counts;
  float* part;  // [splits][E][N], NULL when splits == 1
  uint16_t* db;
  int64_t rows, n, ldy, experts;
  int32_t splits;
};
template <class T> __global__ __launch_bounds__(1024) void k_w4_bias(const BiasArgs p) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane, e = blockIdx.z;
  int64_t start = 0, count = p.rows;
  if (p.counts) {
    int64_t before = 0;
    for (int64_t i = lane; i < e; i += 64) before += p.counts[i] > 0 ? p.counts[i] : 0;
    for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off);
    const int64_t c = p.counts[e] > 0 ? p.counts[e] : 0;
    start = before < p.rows ? before : p.rows;
    count = before + c < p.rows ? before + c - start : p.rows - start;
  }
  const int64_t r0 = start + count * blockIdx.y / p.splits, r1 = start + count * (blockIdx.y + 1) / p.splits;
  float s = 0;
  if (col < p.n) {
    const uint16_t* from = p.dy + col;
#pragma unroll 8
    for (int64_t r = r0 + w; r < r1; r += 16) s += T::to_f32(from[r * p.ldy]);
  }
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && col < p.n) {
    float v = red[0][lane];
#pragma unroll
    for (int i = 1; i < 16; ++i) v += red[i][lane];
    if (p.part)
      p.part[((int64_t)blockIdx.y * p.experts + e) * p.n + col] = v;
    else
      p.db[e * p.n + col] = T::from_f32(v);
  }
}
template <class T> __global__ __launch_bounds__(256) void k_w4_bias_join(const BiasArgs p) {
  const int64_t total = p.experts * p.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float s = p.part[i];
    for (int o = 1; o < p.splits; ++o) s += p.part[o * total + i];
    p.db[i] = T::from_f32(s);
  }
}

// ---- host side -----------------------------------------------------------------------------------------
namespace {

constexpr int64_t kMaxK = 1 << 20, kMaxN = 1 << 22, kMaxExperts = 4096, kMaxRows = (int64_t)1 << 27;
constexpr int64_t kMaxStride = 1 << 23;  // elements between rows that the kernels address in 32 bits

uint8_t e4m3_of(float v, bool* ok) {  // exact, or *ok = false
  for (int b = 0; b < 256; ++b) {
    if ((b & 0x7F) == 0x7F) continue;
    const int e = b >> 3 & 15, m = b & 7;
    float f = e ? (8 + m) * 0.125f : m * 0.125f;
    for (int i = (e ? e : 1); i < 7; ++i) f *= 0.5f;
    for (int i = 7; i < e; ++i) f *= 2.0f;
    if ((b & 0x80 ? -f : f) == v && !(b == 0x80)) return (uint8_t)b;
  }
  *ok = false;
  return 0;
}

int check_w4(const mq_w4* w) {
  if (!w) return MQ_ERR_ARG;
  if (w->experts < 1 || w->n < 1 || w->k < 1 || w->kind < 0 || w->kind > 3) return MQ_ERR_ARG;
  if (w->experts > kMaxExperts || w->n > kMaxN || w->k > kMaxK) return MQ_ERR_TOO_LARGE;
  if (w->group < 0) return MQ_ERR_ARG;
  if (w->group > 0 && w->k % w->group) return MQ_ERR_GROUP;
  if (w->group > 0 && w->group % 32) return MQ_ERR_UNSUPPORTED;
  if (w->kind == W4_LUT && w->values[0] != 0.0f) return MQ_ERR_UNSUPPORTED;  // (padding is code 0)
  return MQ_OK;
}
int32_t steps_of_group(const mq_w4* w) { return (int32_t)(w->group > 0 ? w->group / 32 : w4_ktiles(w->k) * 4); }
int32_t groups_padded(const mq_w4* w) {
  const int64_t steps = w4_ktiles(w->k) * 4, gu = steps_of_group(w);
  return (int32_t)((steps + gu - 1) / gu);
}

int fill_args(const mq_w4* w, const int32_t* counts, int64_t rows, W4Args* a) {
  if (!w->data || !w->params || !w->norm) return MQ_ERR_ARG;
  if ((uintptr_t)w->data % 16 || (uintptr_t)w->params % 16 || (uintptr_t)w->norm % 4 || (uintptr_t)counts % 4) return MQ_ERR_ALIGN;
  *a = W4Args{};
  a->data = static_cast<const uint32_t*>(w->data);
  a->params = w->params;
  a->norm = w->norm;
  a->counts = counts;
  a->experts = w->experts;
  a->n = w->n;
  a->k = w->k;
  a->rows = rows;
  a->nt = (int32_t)w4_ntiles(w->n);
  a->kt = (int32_t)w4_ktiles(w->k);
  a->gu = steps_of_group(w);
  a->gp = groups_padded(w);
  a->gmagic = (uint32_t)((((uint64_t)1 << 31) + a->gu - 1) / a->gu);
  if (w->kind == W4_LUT) {
    bool ok = true;
    for (int i = 0; i < 16; ++i) a->lut.w[i / 4] |= (uint32_t)e4m3_of(w->values[i], &ok) << (8 * (i % 4));
    if (!ok) return MQ_ERR_UNSUPPORTED;
  }
  return MQ_OK;
}

// Which kernel and launch shape.  Everything goes by sizes; times are microseconds per call in a graph, launch included.
W4Plan plan_of(const mq_w4* w, int64_t rows, bool grad, bool counted, W4Product* p) {
  W4Plan pl = {};
  const int32_t gu = steps_of_group(w);
  pl.fs = gu % 4 == 0 ? 4 : gu % 2 == 0 ? 2 : 1;
  p->kc = grad ? w->n : w->k;
  p->nc = grad ? w->k : w->n;
  p->ct = (int32_t)w4_ntiles(p->nc);
  p->rb = (int32_t)w4_ktiles(p->kc);
  p->splits = 1;
  const int64_t per = counted ? (rows + w->experts - 1) / w->experts : rows;  // rows of an expert, on average
  const int64_t busy = counted ? (rows < w->experts ? rows : w->experts) : 1;  // experts that have rows, at most
  auto row_blocks = [&](int bm) {
    if (!counted) return (rows + bm - 1) / bm;
    return rows / bm + (rows < w->experts + 1 ? rows : w->experts + 1);  // every expert may end inside a tile
  };
  if (!grad && per <= 32) {
    // Up to 32 rows k_w4_rows reads the weight at most twice; from 33 on the tiles of k_w4_gemm share it (4096 x 4096:
    // 32 rows 10.5 against 13.5, 64 rows 17 against 15).
    pl.mt = per <= 16 ? 1 : 2;
    p->mblocks = (int32_t)row_blocks(16 * pl.mt);
    const int64_t tiles = p->ct * busy;  // 16-column tiles that have rows
    // Four column tiles to a workgroup read x a quarter as often, if enough workgroups are left (14336 x 4096, one row:
    // 11.9, 11.0, 9.5 with one, two, four; 4096 x 4096: 4.7, 5.2, 6.8).
    pl.nt = tiles >= 800 ? 4 : tiles >= 400 ? 2 : 1;
    if (pl.nt < 4 && per > 4 && p->rb >= 64 && !counted) {
      // many rows over a long contraction: reading x costs more than a second launch that joins pieces of the
      // contraction (4096 x 14336, 16 rows: 18.0 against 14.6; one row: 11.6 against 12.8)
      pl.nt = 4;
      while (p->splits < 8 && tiles * p->splits < 800 && p->rb >= 16 * p->splits) p->splits *= 2;
    }
    p->nblocks = (p->ct + pl.nt - 1) / pl.nt;
    const int64_t blocks = p->nblocks * busy * p->splits;
    // waves share a workgroup's contraction: more of them only where there are few workgroups (32000 x 4096: 15.8 with
    // four, 16.9 with eight; 14336 x 4096: 10.3 and 9.5)
    pl.waves = blocks >= 384 ? 4 : pl.nt == 1 && pl.mt == 1 && p->rb >= 64 ? 16 : 8;
    while (pl.waves > 1 && pl.waves * p->splits > p->rb) pl.waves /= 2;
    return pl;
  }
  // Tile height and cuts of the contraction (pieces of at least 4 blocks of 128, joined by a second launch): the cheapest
  // by what was measured on 4096 x 4096, microseconds per block of 128 for a compute unit with one tile (two sets of waves
  // in it), with two, and for an odd one behind pairs.  64 x 128 (always two sets): 0.65, 1.3, 0.55 (gradient 0.75, 1.2,
  // 0.6), 128 x 128: 1.05, 1.85, 1.2, the gradient's 128 x 256: 2.1, 3.6, 1.75 (one tile with one set of waves: forward
  // 1.1, gradient the same without zero points and 2.4 with them; pairs with two sets: 2.15 and 4.1).  A tile begins and ends
  // in 1.5; a join takes 3 and moves its sums at about 4 MB per microsecond.  Measured with integer codes and taken for all
  // kinds (a table's decoding takes 19 instructions, an integer's 7).
  static const double kTime[2][2][3] = {{{0.65, 1.3, 0.55}, {1.05, 1.85, 1.2}}, {{0.75, 1.2, 0.6}, {2.1, 3.6, 1.75}}};
  double best = 0;
  for (int tall = 0; tall < 2; ++tall) {
    const int bm = tall ? 128 : 64, bn = tall && grad ? 256 : 128;
    const int64_t nblocks = (p->ct * 16 + bn - 1) / bn;
    // (the last tile of an expert is half full on average)
    const int64_t tiles = (counted ? rows / bm + (busy + 1) / 2 : (rows + bm - 1) / bm) * nblocks;
    const double* time = kTime[grad][tall];
    for (int s = 1; s <= 8 && (s == 1 || p->rb >= 4 * s); s *= 2) {
      const int64_t each = (tiles * s + 255) / 256;  // tiles of a compute unit
      const double t = (each == 1 ? time[0] : each / 2 * time[1] + each % 2 * time[2]) * p->rb / s + 1.5 * each +
                       (s > 1 ? 3 + 8e-6 * s * rows * p->ct * 16 / 4 : 0);
      if (pl.bm && t >= best) continue;
      best = t;
      pl.bm = bm;
      pl.bn = bn;
      pl.wk = each == 1 ? 2 : 1;
      p->splits = s;
      p->nblocks = (int32_t)nblocks;
    }
  }
  p->mblocks = (int32_t)row_blocks(pl.bm);
  return pl;
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }
size_t turned_bytes(const mq_w4* w) { return up256((size_t)w->experts * w4_ntiles(w->k) * w4_ktiles(w->n) * 1024); }
size_t turned_params_bytes(const mq_w4* w) {  // of one of the two arrays
  return up256((size_t)w->experts * groups_padded(w) * w4_ktiles(w->n) * 128 * 2);
}
size_t turn_bytes(const mq_w4* w) { return turned_bytes(w) + 2 * turned_params_bytes(w); }
size_t part_bytes(const W4Product& p, int64_t rows) {
  return p.splits > 1 ? up256((size_t)p.splits * rows * p.ct * 16 * 4) : 0;
}
// the row sums for the zero points (k_w4_rowsum)
size_t sums_bytes(const mq_w4* w, const W4Plan& pl, const W4Product& p, int64_t rows, bool grad) {
  return pl.bm && !grad && w->kind == W4_U4 ? up256((size_t)p.rb * (4 / pl.fs) * rows * 4) : 0;
}

int32_t bias_splits(int64_t rows, int64_t experts) {
  const int64_t per = rows / experts;  // up to 512 rows in one run: a second launch costs as much as reading them
  return (int32_t)(per <= 512 ? 1 : per / 256 < 32 ? per / 256 : 32);
}
size_t bias_bytes(const mq_w4* w, int64_t rows) {
  const int32_t s = bias_splits(rows, w->experts);
  return s > 1 ? up256((size_t)s * w->experts * w->n * 4) : 0;
}
template <class T> hipError_t bias_launch(const BiasArgs& p, hipStream_t st) {
  hipLaunchKernelGGL((k_w4_bias<T>), dim3((unsigned)((p.n + 63) / 64), p.splits, (unsigned)p.experts), dim3(1024), 0, st, p);
  const int64_t join = (p.experts * p.n + 255) / 256;
  if (p.part) hipLaunchKernelGGL((k_w4_bias_join<T>), dim3((unsigned)(join < 4096 ? join : 4096)), dim3(256), 0, st, p);
  return hipGetLastError();
}

int product(const mq_w4* w, const void* x, int32_t dtype, int64_t rows, int64_t ldx, const void* bias,
            const int32_t* counts, void* y, void* ws, size_t ws_bytes, void* stream, bool grad) {
  int rc = check_w4(w);
  if (rc != MQ_OK) return rc;
  if (dtype != MQ_F16 && dtype != MQ_BF16) return MQ_ERR_UNSUPPORTED;
  if (rows < 0 || (!counts && w->experts != 1)) return MQ_ERR_ARG;
  if (rows > kMaxRows) return MQ_ERR_TOO_LARGE;
  if (rows == 0) return MQ_OK;
  const int64_t kc = grad ? w->n : w->k;
  if (!x || !y || ldx < 0 || (ldx < kc && ldx != 0 && rows > 1)) return MQ_ERR_ARG;
  if ((uintptr_t)x % 2 || (uintptr_t)y % 16 || (uintptr_t)bias % 2) return MQ_ERR_ALIGN;
  W4Args a;
  rc = fill_args(w, counts, rows, &a);
  if (rc != MQ_OK) return rc;
  W4Product p = {};
  const W4Plan pl = plan_of(w, rows, grad, counts != nullptr, &p);
  // (a launch counts its threads in 32 bits)
  if ((int64_t)p.nblocks * p.mblocks * (pl.bm ? 512 : 64 * pl.waves) >= (int64_t)1 << 32) return MQ_ERR_TOO_LARGE;
  p.vec = (uintptr_t)x % 16 == 0 && (ldx % 8 == 0 || rows == 1) && kc % 8 == 0;
  const bool halved = grad && dtype == MQ_BF16;
  // workspace: the turned operand (gradient) or the row sums, the splits' partial sums, the padded or halved rows and the
  // factors of the latter
  const size_t sums = sums_bytes(w, pl, p, rows, grad), turned = grad ? turn_bytes(w) : sums;
  const size_t padded = halved || !p.vec || kc % 128 || (ldx > kMaxStride && rows > 1) ? (size_t)rows * p.rb * 256 : 0;
  const size_t need = turned + part_bytes(p, rows) + padded + (halved ? (size_t)rows * 4 : 0);
  if (need && (!ws || ws_bytes < need)) return MQ_ERR_WORKSPACE;
  if ((uintptr_t)ws % 16) return MQ_ERR_ALIGN;
  p.x = static_cast<const uint16_t*>(x);
  p.ldx = ldx;
  p.b = a.data;
  p.bias = static_cast<const uint16_t*>(bias);
  p.y = static_cast<uint16_t*>(y);
  p.part = p.splits > 1 ? reinterpret_cast<float*>(static_cast<char*>(ws) + turned) : nullptr;
  p.xs = sums ? static_cast<float*>(ws) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint16_t* copy = nullptr;  // the rows that the product reads instead of x
  if (padded) {
    uint16_t* to = reinterpret_cast<uint16_t*>(static_cast<char*>(ws) + turned + part_bytes(p, rows));
    if (!halved) {
      hipLaunchKernelGGL(k_w4_pad, dim3((unsigned)((rows + 15) / 16), p.rb), dim3(256), 0, st, p, rows, to);
      MQ_HIP(hipGetLastError());
    }
    copy = to;
  }
  if (grad) {
    char* at = static_cast<char*>(ws);
    uint16_t* scales = reinterpret_cast<uint16_t*>(at + turned_bytes(w));
    TurnArgs t = {reinterpret_cast<uint32_t*>(at), scales, scales + turned_params_bytes(w) / 2, p.ct, p.rb, 0, nullptr, nullptr};
    const int64_t blocks = (int64_t)a.kt * p.rb * w->experts, more = halved ? (rows < 65536 ? rows : 65536) : 0;
    if ((blocks + more) * 64 >= (int64_t)1 << 32) return MQ_ERR_TOO_LARGE;
    t.blocks = (uint32_t)blocks;
    if (halved) {
      t.half = copy;
      t.down = reinterpret_cast<float*>(reinterpret_cast<char*>(copy) + padded);
      p.down = t.down;
    }
    const dim3 grid((unsigned)(blocks + more));
    switch (w->kind) {
      case W4_U4: hipLaunchKernelGGL((k_w4_turn<W4_U4>), grid, dim3(64), 0, st, a, t, p); break;
      case W4_S4: hipLaunchKernelGGL((k_w4_turn<W4_S4>), grid, dim3(64), 0, st, a, t, p); break;
      case W4_LUT: hipLaunchKernelGGL((k_w4_turn<W4_LUT>), grid, dim3(64), 0, st, a, t, p); break;
      default: hipLaunchKernelGGL((k_w4_turn<W4_FP4>), grid, dim3(64), 0, st, a, t, p); break;
    }
    MQ_HIP(hipGetLastError());
    p.b = t.out;
    p.ts = t.ts;
    p.tz = t.tz;
  }
  if (copy) {
    p.x = copy;
    p.ldx = (int64_t)p.rb * 128;
    p.kc = p.ldx;
    p.vec = 1;
  }
  const bool h = dtype == MQ_F16;
  hipError_t e;
  switch (w->kind) {
    case W4_S4: e = (h ? w4_launch_1 : w4_launch_5)(a, p, pl, grad, st); break;
    case W4_U4: e = (h ? w4_launch_2 : w4_launch_6)(a, p, pl, grad, st); break;
    case W4_LUT: e = (h ? w4_launch_3 : w4_launch_7)(a, p, pl, grad, st); break;
    default: e = (h ? w4_launch_4 : w4_launch_8)(a, p, pl, grad, st); break;
  }
  if (e != hipSuccess) {
    mq_set_hip_error(e, "mq_linear4");
    return MQ_ERR_HIP;
  }
  return MQ_OK;
}

}  // namespace

extern "C" size_t mq_w4_data_bytes(int64_t experts, int64_t n, int64_t k) {
  if (experts < 1 || n < 1 || k < 1 || experts > kMaxExperts || n > kMaxN || k > kMaxK) return 0;
  return (size_t)experts * w4_ntiles(n) * w4_ktiles(k) * 1024;
}
extern "C" size_t mq_w4_params_bytes(const mq_w4* w) {
  if (check_w4(w) != MQ_OK) return 0;
  return (size_t)w->experts * w4_ntiles(w->n) * groups_padded(w) * 16 * (w->kind == W4_U4 ? 4 : 2);
}
extern "C" int mq_w4_pack(const mq_w4* w, const void* codes, const void* scale, const void* zero, void* hip_stream) {
  const int rc = check_w4(w);
  if (rc != MQ_OK) return rc;
  if (!codes || !scale || !w->data || !w->params || (zero != nullptr) != (w->kind == W4_U4)) return MQ_ERR_ARG;
  if ((uintptr_t)w->data % 16 || (uintptr_t)w->params % 16 || (uintptr_t)scale % 2 || (uintptr_t)zero % 2 ||
      (w->kind >= W4_LUT && (uintptr_t)codes % 2))
    return MQ_ERR_ALIGN;
  PackArgs p = {};
  p.codes = codes;
  p.scale = static_cast<const uint16_t*>(scale);
  p.zero = static_cast<const uint16_t*>(zero);
  p.data = static_cast<uint32_t*>(const_cast<void*>(w->data));
  p.params = const_cast<void*>(w->params);
  p.n = w->n;
  p.k = w->k;
  p.nt = (int32_t)w4_ntiles(w->n);
  p.kt = (int32_t)w4_ktiles(w->k);
  p.g = (int32_t)(w->group > 0 ? w->k / w->group : 1);
  p.gp = groups_padded(w);
  static const float fp4[16] = {0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12};
  for (int i = 0; i < 16; ++i) p.values[i] = w->kind == W4_FP4 ? fp4[i] : w->values[i];
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  for (int64_t t0 = 0; t0 < p.nt; t0 += 65535) {  // grid.y holds 65535 row tiles
    const int64_t cnt = p.nt - t0 < 65535 ? p.nt - t0 : 65535;
    if (cnt != p.nt && w->experts != 1) return MQ_ERR_TOO_LARGE;
    PackArgs q = p;
    if (cnt != p.nt) {  // one expert: a run of row tiles is a weight of its own
      q.codes = static_cast<const char*>(codes) + t0 * 16 * p.k * (w->kind >= W4_LUT ? 2 : 1);
      q.data = p.data + t0 * p.kt * 256;
      q.n = p.n - t0 * 16;
    }
    const dim3 grid(p.kt, (unsigned)cnt, (unsigned)w->experts);
    switch (w->kind) {
      case W4_U4: hipLaunchKernelGGL((k_w4_pack<W4_U4>), grid, dim3(256), 0, st, q); break;
      case W4_S4: hipLaunchKernelGGL((k_w4_pack<W4_S4>), grid, dim3(256), 0, st, q); break;
      case W4_LUT: hipLaunchKernelGGL((k_w4_pack<W4_LUT>), grid, dim3(256), 0, st, q); break;
      default: hipLaunchKernelGGL((k_w4_pack<W4_FP4>), grid, dim3(256), 0, st, q); break;
    }
    MQ_HIP(hipGetLastError());
  }
  const int64_t total = w->experts * p.nt * p.gp * 16, blocks = (total + 255) / 256;
  hipLaunchKernelGGL(k_w4_params, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, p, total);
  MQ_HIP(hipGetLastError());
  return MQ_OK;
}
extern "C" int mq_w4_unpack(const mq_w4* w, void* deq, void* hip_stream) {
  int rc = check_w4(w);
  if (rc != MQ_OK) return rc;
  if (!deq) return MQ_ERR_ARG;
  if ((uintptr_t)deq % 2) return MQ_ERR_ALIGN;
  W4Args a;
  rc = fill_args(w, nullptr, 0, &a);
  if (rc != MQ_OK) return rc;
  if (a.nt > 65535 && w->experts != 1) return MQ_ERR_TOO_LARGE;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  for (int64_t t0 = 0; t0 < a.nt; t0 += 65535) {
    const int64_t cnt = a.nt - t0 < 65535 ? a.nt - t0 : 65535;
    W4Args b = a;
    uint16_t* out = static_cast<uint16_t*>(deq) + t0 * 16 * a.k;
    b.data += t0 * a.kt * 256;
    b.params = static_cast<const char*>(a.params) + t0 * a.gp * 16 * (w->kind == W4_U4 ? 4 : 2);
    if (w->experts == 1) b.n = a.n - t0 * 16;
    const dim3 grid(a.kt, (unsigned)cnt, (unsigned)w->experts);
    switch (w->kind) {
      case W4_U4: hipLaunchKernelGGL((k_w4_unpack<W4_U4>), grid, dim3(256), 0, st, b, out); break;
      case W4_S4: hipLaunchKernelGGL((k_w4_unpack<W4_S4>), grid, dim3(256), 0, st, b, out); break;
      case W4_LUT: hipLaunchKernelGGL((k_w4_unpack<W4_LUT>), grid, dim3(256), 0, st, b, out); break;
      default: hipLaunchKernelGGL((k_w4_unpack<W4_FP4>), grid, dim3(256), 0, st, b, out); break;
    }
    MQ_HIP(hipGetLastError());
  }
  return MQ_OK;
}
extern "C" size_t mq_linear4_workspace_bytes(const mq_w4* w, int32_t dtype, int64_t rows, int32_t aligned, int32_t counted,
                                             int32_t grad) {
  if (check_w4(w) != MQ_OK || rows < 1 || rows > kMaxRows) return 0;
  size_t need = grad & 2 ? bias_bytes(w, rows) : 0;
  if (grad == 2) return need;
  W4Product p = {};
  const W4Plan pl = plan_of(w, rows, grad != 0, counted != 0, &p);
  need += (grad ? turn_bytes(w) : sums_bytes(w, pl, p, rows, false)) + part_bytes(p, rows);
  const bool halved = grad && dtype == MQ_BF16;
  return need + (halved || !aligned || p.kc % 128 ? (size_t)rows * p.rb * 256 : 0) + (halved ? (size_t)rows * 4 : 0);
}
extern "C" int mq_linear4(const mq_w4* w, const void* x, int32_t dtype, int64_t rows, int64_t ldx, const void* bias,
                          const int32_t* counts, void* y, void* workspace, size_t workspace_bytes, void* hip_stream) {
  return product(w, x, dtype, rows, ldx, bias, counts, y, workspace, workspace_bytes, hip_stream, false);
}
extern "C" int mq_linear4_grad(const mq_w4* w, const void* dy, int32_t dtype, int64_t rows, int64_t ldy,
                               const int32_t* counts, void* dx, void* db, void* workspace, size_t workspace_bytes,
                               void* hip_stream) {
  int rc = check_w4(w);
  if (rc != MQ_OK) return rc;
  if (!dx && !db) return MQ_ERR_ARG;
  size_t used = 0;
  if (db) {
    if (dtype != MQ_F16 && dtype != MQ_BF16) return MQ_ERR_UNSUPPORTED;
    if (rows < 0 || ldy < 0 || (rows > 0 && !dy) || (!counts && w->experts != 1)) return MQ_ERR_ARG;
    if (rows > kMaxRows) return MQ_ERR_TOO_LARGE;
    if ((uintptr_t)dy % 2 || (uintptr_t)db % 2 || (uintptr_t)counts % 4 || (uintptr_t)workspace % 16) return MQ_ERR_ALIGN;
    used = bias_bytes(w, rows);
    if (used && (!workspace || workspace_bytes < used)) return MQ_ERR_WORKSPACE;
  }
  if (dx) {
    rc = product(w, dy, dtype, rows, ldy, nullptr, counts, dx, static_cast<char*>(workspace) + used, workspace_bytes - used,
                 hip_stream, true);
    if (rc != MQ_OK) return rc;
  }
  if (db) {
    const BiasArgs p = {static_cast<const uint16_t*>(dy), counts, used ? static_cast<float*>(workspace) : nullptr,
                        static_cast<uint16_t*>(db), rows, w->n, ldy, w->experts, bias_splits(rows, w->experts)};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    MQ_HIP(dtype == MQ_F16 ? bias_launch<W4F16>(p, st) : bias_launch<W4BF16>(p, st));
  }
  return MQ_OK;
}
#endif
