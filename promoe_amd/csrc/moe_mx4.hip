// Microscaled 4-bit floating point (gfx950): rows quantised and back, and the products of dense layers and of experts with weights
// in that form.  A value is a code (sign, two bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times the power of two of
// its block of 32 columns, 2^(byte - 127); byte 255 makes the block NaN.
//   y = act(x W^T + b) + residual,   y = act(x Wg^T + bg) * (x Wu^T + bu)
// x in the same form: both operands go into the scaled matrix products as they are.  x in bf16 or fp16: the weights become bf16 in
// registers, exactly; an fp16 value is the sum of two bf16 (11 bits of mantissa), so that nothing of it is lost either.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "moe_common.h"
#include "moe_kernels.h"
#include "moe_device.h"
#include "moe_linear.h"

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// ---- rows into codes and back ---------------------------------------------------------------------------------------------------
// Scales lie in blocks of 32 rows by 8 bytes (256 columns, a slab of the products below), so that what 32 rows need of a slab is 256 bytes
// in one piece: byte kb of row r at ((r / 32) slabs + kb / 8) 256 + (r % 32) 8 + kb % 8.  Row by row, as they are exchanged, every row would
// cost the products a cache line for 8 bytes, by count as much traffic as the codes (not timed by itself).
static __host__ __device__ __forceinline__ int mx_slabs(int K) { return (K + 255) >> 8; }
static __device__ __forceinline__ long long mx_scale_row(long long r, int slabs) { return (r >> 5) * (slabs * 256ll) + (r & 31) * 8; }
struct QuantArgs {
  const char *x;              // the rows that are read: values, or codes
  char *y;                    // the rows that are written: codes, or values
  uint8_t *scales;
  long long ldx, ldc;         // elements between rows of values, bytes between rows of codes
  long long next_x, next_c, next_s;  // between matrices: elements, bytes, bytes
  u32 n;                      // pieces of 8 values of a matrix
  u32 per, magic, shift;      // pieces of a row; i / per = (mulhi(i, magic) + i) >> shift for i < 2^31
  int slabs;
};
struct Place { long long x, c, s; };
static __device__ __forceinline__ Place place_of(const QuantArgs &a, u32 i) {
  const u32 row = (__umulhi(i, a.magic) + i) >> a.shift, col = i - row * a.per;
  return Place{blockIdx.y * a.next_x + row * a.ldx + 8ll * col, blockIdx.y * a.next_c + row * a.ldc + 4ll * col,
               blockIdx.y * a.next_s + mx_scale_row(row, a.slabs) + (col >> 5) * 256 + (col >> 2 & 7)};
}
// the largest of the four lanes of a block
static __device__ __forceinline__ u32 quad_max(u32 v) {
  v = max(v, (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  return max(v, (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}
// Exponent byte of the scale of a block from the bits of its largest magnitude as fp32: floor(log2) - 2, at least 0; 255 (NaN) where a
// value is none or infinite
static __device__ __forceinline__ u32 scale_byte(u32 top) {
  const u32 e = top >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// Four lanes a block, eight values each: one 16-byte load (two of fp32) and four bytes of codes, side by side over the lanes.  The
// hardware's conversion divides by the scale, rounds to the nearest (ties to the even code) and goes no further than 6.
// Bound by memory: 4096 x 14336 in bf16 25 to 27 us (5.9 TB/s, the last cache helps), back 22 to 25.
#define QT_U 4  // pieces of a lane, all of them on their way at once
template <int DT>
__global__ __launch_bounds__(256) void k_mx4_quantize(const QuantArgs a) {
  const u32 first = blockIdx.x * (256 * QT_U) + threadIdx.x;
  u32x4_t v[QT_U][DT == MOE_DT_FP32 ? 2 : 1];
#pragma unroll
  for (int u = 0; u < QT_U; ++u) {
    const u32 i = min(first + 256 * u, a.n - 1);  // (no condition around a load)
    const char *p = a.x + place_of(a, i).x * (DT == MOE_DT_FP32 ? 4 : 2);
    v[u][0] = *(const u32x4_t *)p;
    if constexpr (DT == MOE_DT_FP32) v[u][1] = *(const u32x4_t *)(p + 16);
  }
#pragma unroll
  for (int u = 0; u < QT_U; ++u) {
    const u32 i = first + 256 * u;
    if (i >= a.n) break;
    u32 top = 0;
    if constexpr (DT == MOE_DT_FP32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, v[u][e >> 2][e & 3] & 0x7fffffffu);
    } else {  // (magnitudes compare as whole numbers, two at a time)
      u16x2_t m{0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, v[u][0][e] & 0x7fff7fffu));
      top = max(m[0], m[1]);
    }
    top = quad_max(top);
    if constexpr (DT == MOE_DT_BF16) top <<= 16;
    if constexpr (DT == MOE_DT_FP16) top = __float_as_uint(half_bits_to_f32((uint16_t)top));
    const u32 byte = scale_byte(top);
    const float s = __uint_as_float(byte << 23);        // (the conversion takes the exponent field alone: 0 is 2^-127)
    u32 c = 0;
    lt_each<4>([&](auto j_) {
      constexpr int J = decltype(j_)::value;
      if constexpr (DT == MOE_DT_FP32) {
        const u32 p = v[u][DT == MOE_DT_FP32 ? J / 2 : 0][2 * (J & 1)], q = v[u][DT == MOE_DT_FP32 ? J / 2 : 0][2 * (J & 1) + 1];
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(p), __uint_as_float(q), s, J);
      } else {
        const u32 p = v[u][0][J];                       // (a value of its own: bit_cast of a vector's element takes the first one)
        if constexpr (DT == MOE_DT_BF16) c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p), s, J);
        else c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, p), s, J);
      }
    });
    const Place at = place_of(a, i);
    *(u32 *)(a.y + at.c) = c;
    if ((threadIdx.x & 3) == 0) a.scales[at.s] = (uint8_t)byte;
  }
}
template <int DT>
__global__ __launch_bounds__(256) void k_mx4_dequantize(const QuantArgs a) {
  const u32 first = blockIdx.x * (256 * QT_U) + threadIdx.x;
  u32 c[QT_U], b[QT_U];
#pragma unroll
  for (int u = 0; u < QT_U; ++u) {
    const Place at = place_of(a, min(first + 256 * u, a.n - 1));
    c[u] = *(const u32 *)(a.x + at.c);
    b[u] = a.scales[at.s];
  }
#pragma unroll
  for (int u = 0; u < QT_U; ++u) {
    const u32 i = first + 256 * u;
    if (i >= a.n) break;
    const float s = __uint_as_float(b[u] << 23);
    char *p = a.y + place_of(a, i).x * (DT == MOE_DT_FP32 ? 4 : 2);
    f32x2_t f[4];
    f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 0);
    f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 1);
    f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 2);
    f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 3);
    if constexpr (DT == MOE_DT_FP32) {
      *(f32x4_t *)p = f32x4_t{f[0][0], f[0][1], f[1][0], f[1][1]};
      *(f32x4_t *)(p + 16) = f32x4_t{f[2][0], f[2][1], f[3][0], f[3][1]};
    } else {
      const float v[8] = {f[0][0], f[0][1], f[1][0], f[1][1], f[2][0], f[2][1], f[3][0], f[3][1]};
      *(u32x4_t *)p = lin_pack<DT == MOE_DT_FP16>(v);
    }
  }
}

// ---- products -------------------------------------------------------------------------------------------------------------------
struct MxArgs {
  const void *x;
  const uint8_t *xs;                         // scales of x, NULL: x has 16 bits
  const uint8_t *w[2], *ws[2];               // codes and scales of the matrices; [1]: the second one of a gated pair
  const uint16_t *bias[2], *res;
  void *y;
  long long ldx, ldw, ew, ews;               // bytes between rows; ew, ews: between the matrices (scales) of consecutive experts
  long long ldr, ldy;                        // elements
  int M, N, K, act, y32;                     // M: rows of y
  int nm, nn, splits, ldp, slabs, extra;     // as in the products of 16-bit matrices
  float *part;
  // products by expert
  const int *counts, *offsets, *tok;         // rows of each expert, its first; tok: the row of x of each row of y (NULL: the same)
  const moe_unit *units;
  int E;
};
enum { X_MX4 = 0, X_BF16 = 1, X_FP16 = 2 };   // what x is
static __device__ __forceinline__ f32x4_t mx_mfma16(u32x4_t a, u32x4_t b, f32x4_t c, u32 sa, u32 sb) {
  const i32x8_t a8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, b8{(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, (int)sa, 0, (int)sb);
}
// eight codes as bf16, exactly
static __device__ __forceinline__ u32x4_t mx_bf16(u32 c, float s) {
  return u32x4_t{__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}
// the same as fp16, exactly where the scale is between 2^-23 and 2^13 (mx_fits_f16)
static __device__ __forceinline__ u32x4_t mx_f16(u32 c, float s) {
  return u32x4_t{__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 0)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 1)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 2)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 3))};
}
static __device__ __forceinline__ bool mx_fits_f16(u32 byte) { return byte - 104u <= 36u; }
// eight fp16 values as the sums of two bf16: the first to the nearest, the second what is left (at most 4 bits)
static __device__ __forceinline__ void mx_split(u32x4_t x, u32x4_t &hi, u32x4_t &lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = half_bits_to_f32((uint16_t)x[i]), b = half_bits_to_f32((uint16_t)(x[i] >> 16));
    const u32 h = lin_bits<false>(a) | (u32)lin_bits<false>(b) << 16;
    const float c = a - bf16lo(h), d = b - bf16hi(h);   // (of an infinite value NaN: the second part is 0 then)
    hi[i] = h;
    lo[i] = (c == c ? lin_bits<false>(c) : 0u) | (u32)(d == d ? lin_bits<false>(d) : 0u) << 16;
  }
}

// ---- few rows of x: the matrix streams past them --------------------------------------------------------------------------------
// A workgroup of four or eight waves takes NB sets of R = 16 / SH rows of W (gated: of both matrices), its waves the pieces of K in turn;
// their sums meet in LDS.  A lane's load is one block, 32 columns of a row: with SH = 1 the 16 rows of the operand are 16 rows of W, with few rows of x
// (at most 16 / SH) R rows of W by SH pieces of K: row s R + r and column s R + m hold piece s of both, and the products of unlike
// pieces are left unread.  By expert the second dimension of the grid is a unit of the dispatch; more than 16 rows go in turn.
// NB: sets of R rows a workgroup takes, all against the same operand of x; U: loads of a set in flight per wave, twice.  Four waves, U = 1:
// what counts is how soon a workgroup's trip to memory begins and ends (us, U = 1 / 2: 1 x 14336 x 4096 gated 17.9 / 19.1; waves 4 / 8: 17.9 / 18.8).
// Bound by memory where it is long enough: 20 tokens of 64 experts, 1408 x 2048 gated, 35 to 38 us (4.4 TB/s and more); 1 x 2048 x 10944, 6.6 us
// (floor 2.3), is three trips to memory one behind the other for each wave, and the join.
template <int X, bool F16, bool GATED, int SH, int NB, int U, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_mx4_rows(const MxArgs a) {
  constexpr int MATS = GATED ? 2 : 1, NM = MATS * NB, R = 16 / SH, STEP = 4 * SH * U, SPAN = STEP * WAVES, NX = X == X_MX4 ? 1 : 4;
  __shared__ f32x4_t red[WAVES][NM][64];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = (lane & 15) % R, s = (lane & 15) / R, n0 = blockIdx.x * (R * NB), blocks = a.K >> 5, slabs = mx_slabs(a.K);
  int e = 0, first = 0, rows = a.M;
  if (a.units) {
    const moe_unit u = a.units[blockIdx.y];
    e = __builtin_amdgcn_readfirstlane(u.expert); first = __builtin_amdgcn_readfirstlane(u.row0); rows = __builtin_amdgcn_readfirstlane(u.m);
    if ((unsigned)e >= (unsigned)a.E) return;
  }
  MxArgs o = a;                                                  // what the epilogue goes by
  if (o.bias[0]) o.bias[0] += (long long)e * a.N;
  if (GATED && o.bias[1]) o.bias[1] += (long long)e * a.N;
  const int k0 = (lane >> 4) * SH + s;                           // the lane's block among 4 SH
  rsrc_t rw[MATS], rs[MATS];
  int vw[NB], vs[NB];
#pragma unroll
  for (int i = 0; i < MATS; ++i) {
    rw[i] = make_rsrc(a.w[i] + e * a.ew + n0 * a.ldw, LT_OUT);
    rs[i] = make_rsrc(a.ws[i] + e * a.ews + mx_scale_row(n0 & ~31, slabs), LT_OUT);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int row = min(n0 + b * R + r, a.N - 1) - n0;
    vw[b] = row * (int)a.ldw;
    vs[b] = (int)mx_scale_row(row + (n0 & 31), slabs);
  }
  for (int m0 = 0; m0 < rows; m0 += R) {
    const int m = first + m0 + min(r, rows - 1 - m0);
    const long long xrow = a.tok ? a.tok[m] : m, x0 = a.tok ? 0 : first + m0;  // (rows side by side from the block's first on)
    const rsrc_t rx = make_rsrc((const char *)a.x + x0 * a.ldx, LT_OUT), rxs = make_rsrc(X == X_MX4 ? a.xs + mx_scale_row(x0 & ~31, slabs) : (const uint8_t *)a.x, LT_OUT);
    const int vx = (int)((xrow - x0) * a.ldx), vxs = (int)mx_scale_row(xrow - (x0 & ~31), slabs);
    f32x4_t acc[NM] = {};
    uint4 fw[2][NM][U], fx[2][U][NX];
    u32 sw[2][NM][U], sx[2][U];
    auto load = [&](int p, int base) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = base + 4 * SH * u + k0;
        const bool in = k < blocks;                              // past the end: zeros on both sides
        const int ks = (k >> 3) * 256 + (k & 7);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          fw[p][i][u] = bload16(rw[i % MATS], in ? vw[i / MATS] + 16 * k : LT_OUT, 0);
          const u32 b = bload1(rs[i % MATS], in ? vs[i / MATS] + ks : LT_OUT, 0);
          sw[p][i][u] = X == X_FP16 && !in ? 127u : b;           // (of zeros any scale will do)
        }
        if constexpr (X == X_MX4) {
          fx[p][u][0] = bload16(rx, in ? vx + 16 * k : LT_OUT, 0);
          sx[p][u] = bload1(rxs, in ? vxs + ks : LT_OUT, 0);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) fx[p][u][j] = bload16(rx, in ? vx + 64 * k + 16 * j : LT_OUT, 0);
        }
      }
    };
    auto use = [&](int p) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if constexpr (X == X_MX4) {
#pragma unroll
          for (int i = 0; i < NM; ++i)
            acc[i] = mx_mfma16(__builtin_bit_cast(u32x4_t, fw[p][i][u]), __builtin_bit_cast(u32x4_t, fx[p][u][0]), acc[i], sw[p][i][u], sx[p][u]);
        } else {
          if constexpr (X == X_FP16) {  // weights in fp16 where the whole wave's can be
            bool fits = true;
#pragma unroll
            for (int i = 0; i < NM; ++i) fits = fits && mx_fits_f16(sw[p][i][u]);
            if (__all(fits)) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < NM; ++i)
                  acc[i] = lin_mfma16<true>(mx_f16(__builtin_bit_cast(u32x4_t, fw[p][i][u])[j], __uint_as_float(sw[p][i][u] << 23)),
                                            __builtin_bit_cast(u32x4_t, fx[p][u][j]), acc[i]);
              continue;
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            u32x4_t x = __builtin_bit_cast(u32x4_t, fx[p][u][j]), lo;
            if constexpr (X == X_FP16) mx_split(x, x, lo);
#pragma unroll
            for (int i = 0; i < NM; ++i) {
              const u32x4_t v = mx_bf16(__builtin_bit_cast(u32x4_t, fw[p][i][u])[j], __uint_as_float(sw[p][i][u] << 23));
              acc[i] = lin_mfma16<false>(v, x, acc[i]);
              if constexpr (X == X_FP16) acc[i] = lin_mfma16<false>(v, lo, acc[i]);
            }
          }
        }
      }
    };
    load(0, w * STEP);
    for (int base = w * STEP; base < blocks; base += 2 * SPAN) {
      load(1, base + SPAN);
      use(0);
      load(0, base + 2 * SPAN);
      use(1);
    }
#pragma unroll
    for (int i = 0; i < NM; ++i) red[w][i][lane] = acc[i];
    __syncthreads();
    // result (m, n): element n' % 4 of lane 16 (n' / 4) + m', n' = s R + n and m' = s R + m, over the pieces and the waves in order
    const int cnt = min(R, rows - m0);
    for (int t = tid; t < R * NB * cnt; t += 64 * WAVES) {
      const int n = t % R, b = t / R % NB, i_m = t / (R * NB);
      if (n0 + b * R + n >= a.N) continue;
      float sum[MATS];
#pragma unroll
      for (int i = 0; i < MATS; ++i) {
        sum[i] = 0.f;
#pragma unroll
        for (int p = 0; p < SH; ++p) {
          const int at = p * R + n;
#pragma unroll
          for (int v = 0; v < WAVES; ++v) sum[i] += ((const float *)&red[v][b * MATS + i][16 * (at >> 2) + p * R + i_m])[at & 3];
        }
      }
      lin_store<F16, GATED>(o, first + m0 + i_m, n0 + b * R + n, sum[0], sum[MATS - 1]);
    }
    __syncthreads();
  }
}

// ---- tiles ----------------------------------------------------------------------------------------------------------------------
// Where a workgroup works.  Dense: tile (mt, nt) of rows and columns and a piece of K.  By expert: the tiles of an expert's rows by nt; the
// counts of all experts are added up by every wave, the host does not know them.  Workgroup i runs on XCD i % 8: each XCD takes a
// contiguous run of tiles, four rows of tiles wide.
struct MxTile { int m0, m_end, n0, e, split, kt0, nk; };  // rows m0 .. m_end - 1 of y at most; slabs kt0 .. nk - 1
template <int BM, int NC>
struct MxTiles {
  // by expert: lane l has experts per l .. per l + per - 1, their tiles, those up to them, the first row and how many there are
  int total, per, mine, upto, first, have;
  __device__ __forceinline__ MxTiles(const MxArgs &a) : per(0), mine(0), upto(0), first(0), have(0) {
    total = a.nm * a.nn * a.splits;
    if (a.units) {
      const int lane = threadIdx.x & 63;
      per = (a.E + 63) >> 6;
      for (int i = 0; i < per; ++i) {
        const int x = per * lane + i;
        const int c = x < a.E ? a.counts[x] : 0;
        mine += (c + BM - 1) / BM;
        have += c;
      }
      first = a.offsets[min(per * lane, a.E)];
      upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
      }
      total = __builtin_amdgcn_readlane(upto, 63) * a.nn;
    }
  }
  // the run of this workgroup's XCD: its first tile, the end, and the workgroups that share it
  __device__ __forceinline__ int begin() const { return ((int)blockIdx.x & 7) * ((total + 7) >> 3) + ((int)blockIdx.x >> 3); }
  __device__ __forceinline__ int end() const { return min(total, (((int)blockIdx.x & 7) + 1) * ((total + 7) >> 3)); }
  __device__ __forceinline__ MxTile at(const MxArgs &a, int v) const {
    MxTile t{};
    int nm = a.nm, r, e = 0, row0 = 0, rows = a.M;
    if (!a.units) {
      const int tiles = nm * a.nn;
      t.split = v / tiles;
      r = v - t.split * tiles;
    } else {
      const int row = v / a.nn;  // (tiles come expert by expert: one of its rows of tiles, whichever)
      const int l = (int)__builtin_ctzll(__ballot(upto > row) | 1ull << 63);
      int before = __builtin_amdgcn_readlane(upto - mine, l);
      e = per * l;
      row0 = __builtin_amdgcn_readlane(first, l);
      rows = __builtin_amdgcn_readlane(have, l);
      nm = (rows + BM - 1) / BM;
      if (per > 1)                 // (a lane's experts one after the other)
        for (;; ++e) {
          rows = a.counts[e];
          nm = (rows + BM - 1) / BM;
          if (before + nm > row || e + 1 >= min(a.E, per * (l + 1))) break;
          before += nm;
          row0 += rows;
        }
      r = v - before * a.nn;
    }
    const int group = r / (4 * a.nn), in = r - group * 4 * a.nn, wide = min(4, nm - 4 * group);
    const int nt = in / wide, mt = 4 * group + in - nt * wide;
    // (scalars, whatever the divisions are made of)
    t.m0 = __builtin_amdgcn_readfirstlane(row0 + mt * BM);
    t.m_end = __builtin_amdgcn_readfirstlane(row0 + rows);
    t.n0 = __builtin_amdgcn_readfirstlane(nt * NC);
    t.e = __builtin_amdgcn_readfirstlane(e);
    t.split = __builtin_amdgcn_readfirstlane(t.split);
    t.kt0 = t.split * a.slabs + min(t.split, a.extra);
    t.nk = t.kt0 + a.slabs + (t.split < a.extra);
    return t;
  }
};
// Rows of x that a lane's transfers read, behind xbase: all lookups of a gathered x on their way at once
template <int N, class F>
static __device__ __forceinline__ void mx_rows_of_x(const MxArgs &a, const MxTile &t, int (&row)[N], const F &of) {
#pragma unroll
  for (int i = 0; i < N; ++i) row[i] = min(t.m0 + of(i), t.m_end - 1);
  if (a.tok) {
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] = a.tok[row[i]];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] -= t.m0;
  }
}
// what the epilogue of a tile goes by
static __device__ __forceinline__ MxArgs mx_out(const MxArgs &a, const MxTile &t) {
  MxArgs o = a;
  if (o.bias[0]) o.bias[0] += (long long)t.e * a.N;
  if (o.bias[1]) o.bias[1] += (long long)t.e * a.N;
  o.M = t.m_end;
  return o;
}
// The end of a tile of 2 x 2 waves with WM x WN blocks of 32 x 32 each (a gated pair's W blocks alternate between the matrices): the sums of
// rows from m0 and columns from n0 on, through the LDS that `ring` is.
template <bool F16, bool GATED, int WM, int WN>
static __device__ __forceinline__ void mx_tile_out(const MxArgs &a, const f32x16_t (&acc)[WM][WN], unsigned char *ring, int m0, int n0, int split) {
  constexpr int NC = GATED ? 32 * WN : 64 * WN;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w & 1, wn = w >> 1;
  const int fr = lane & 31, q = lane >> 5;
  // The sums leave through LDS, 32 rows of the wave at a time, so that a lane then has 8 adjacent columns of a row and the rest is
  // one loop of whole lines.  Element e of a lane: column 8 (e / 4) + 4 q + e % 4 of W's block, row fr of x's.
  LT_VM(0);
  __syncthreads();
  constexpr int LDE = 32 * WN + 4;                       // floats between rows: 16 lanes that write 16 bytes each fall on all banks
  constexpr int LPR = NC / 16, RPP = 64 / LPR;           // lanes of a row (8 columns each), rows of a pass
  float *buf = (float *)ring + w * 32 * LDE;
  const int col = 8 * (lane % LPR), n = n0 + wn * (NC / 2) + col;
  const int at = GATED ? (col >> 5) * 64 + (col & 31) : col;
  const LinColumns<F16, GATED> c(a, n);
  constexpr int NP = 32 / RPP;
  // eight columns of row r of the block, from column k of the wave's sums on: gated the second eight of the second matrix
  auto fetch = [&](int r, int k, float (&s0)[8], float (&s1)[8]) {
#pragma unroll
    for (int h = 0; h < (GATED ? 4 : 2); ++h) {
      const f32x4_t f = *(const f32x4_t *)(buf + r * LDE + k + (h & 1) * 4 + (h >> 1) * 32);
#pragma unroll
      for (int e = 0; e < 4; ++e) (h >> 1 ? s1 : s0)[4 * (h & 1) + e] = f[e];
    }
  };
  // all rows of a block: every load of a residual in front of the sums' way through LDS, the activation chosen once
  auto plain = [&](int first, const u32x4_t (&res)[NP], auto act_) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float s0[8], s1[8];
      fetch(lane / LPR + p * RPP, at, s0, s1);
      c.template finish<decltype(act_)::value>(s0, s1);
      if (!GATED && a.res) lin_add<F16>(s0, res[p]);
      const int m = first + p * RPP;
      if (m < a.M && c.count == 8) {
        if (a.y32) {
          float *y = (float *)a.y + m * a.ldy + n;
          *(f32x4_any *)y = f32x4_t{s0[0], s0[1], s0[2], s0[3]};
          *(f32x4_any *)(y + 4) = f32x4_t{s0[4], s0[5], s0[6], s0[7]};
        } else {
          *(u32x4_any *)((uint16_t *)a.y + m * a.ldy + n) = lin_pack<F16>(s0);
        }
      }
    }
  };
  // fewer than eight columns at the end of a row: a row a lane
  const int tail = (a.N & 7) ? (a.N & ~7) - (n0 + wn * (NC / 2)) : -1;  // where they begin among the wave's
  // (one copy of the loop for all blocks: code that runs once a tile waits for its instructions, line by line)
#pragma clang loop unroll(disable)
  for (int i = 0; i < WM; ++i) {
    if (m0 + 32 * (2 * i + wm) >= a.M) break;
    const int first = m0 + 32 * (2 * i + wm) + lane / LPR;
    u32x4_t res[NP];
    if (!GATED && a.res && !a.part && c.count == 8)
#pragma unroll
      for (int p = 0; p < NP; ++p) res[p] = *(const u32x4_any *)(a.res + (long long)min(first + p * RPP, a.M - 1) * a.ldr + n);
    lt_each<WM>([&](auto i_) {
      if (i == decltype(i_)::value) {
#pragma unroll
        for (int b = 0; b < WN; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x16_t &s = acc[decltype(i_)::value][b];
            *(f32x4_t *)(buf + fr * LDE + 32 * b + 8 * e + 4 * q) = f32x4_t{s[4 * e], s[4 * e + 1], s[4 * e + 2], s[4 * e + 3]};
          }
        __asm__ volatile("; %0" :: "i"(decltype(i_)::value));  // (or the compiler makes one copy of them, over registers chosen by i)
      }
    });
    __builtin_amdgcn_wave_barrier();
    switch (a.part ? -1 : a.act) {
      case MOE_ACT_NONE: plain(first, res, std::integral_constant<int, MOE_ACT_NONE>()); break;
      case MOE_ACT_SILU: plain(first, res, std::integral_constant<int, MOE_ACT_SILU>()); break;
      case MOE_ACT_GELU: plain(first, res, std::integral_constant<int, MOE_ACT_GELU>()); break;
      case MOE_ACT_GELU_TANH: plain(first, res, std::integral_constant<int, MOE_ACT_GELU_TANH>()); break;
      case MOE_ACT_RELU: plain(first, res, std::integral_constant<int, MOE_ACT_RELU>()); break;
      case MOE_ACT_RELU2: plain(first, res, std::integral_constant<int, MOE_ACT_RELU2>()); break;
      default:
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          float s0[8], s1[8];
          fetch(lane / LPR + p * RPP, at, s0, s1);
          if (first + p * RPP < a.M) c.partial(a, split, first + p * RPP, s0, s1);
        }
    }
    if (!a.part && tail >= 0 && tail < NC / 2 && lane < 32) {
      const int m = first - lane / LPR + lane;
      float s0[8], s1[8];
      fetch(lane, GATED ? (tail >> 5) * 64 + (tail & 31) : tail, s0, s1);
      if (m < a.M) LinColumns<F16, GATED>(a, a.N & ~7).store(a, m, s0, s1, u32x4_t{0, 0, 0, 0});
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The pieces of K added in their order, then what a tile kernel does behind its sums: eight columns a thread of 256
template <bool F16, bool GATED>
__global__ __launch_bounds__(256) void k_mx4_join(const MxArgs a) {
  const int per = a.ldp >> 3;
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(t / per), n = (int)(t - (long long)m * per) * 8;
  if (m >= a.M) return;
  float s[2][8] = {};
  constexpr int NM = GATED ? 2 : 1;
  const long long step = (long long)a.M * a.ldp;
  for (int p = 0; p < a.splits; ++p)
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const float *q = a.part + (p * NM + i) * step + (long long)m * a.ldp + n;
      const f32x4_t u = *(const f32x4_t *)q, v = *(const f32x4_t *)(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { s[i][e] += u[e]; s[i][4 + e] += v[e]; }
    }
  const LinColumns<F16, GATED> c(a, n);
  c.store(a, m, s[0], s[1], c.residual(a, m));
}

// x in 4 bits.  Four waves (2 x 2), wave (wm, wn) on WM x WN blocks of 32 x 32: a tile of 64 WM rows of x (block i of wave wm: rows 32 (2 i +
// wm) ..) by 64 WN rows of W.  A gated
// pair's W blocks alternate between the two matrices (block b: matrix b & 1, its columns 32 (b >> 1) ..), so that a lane holds both sums
// of a column.  K advances 256 at a time (a slab: 128 bytes of codes and 8 of scales a row); slabs go global -> LDS directly, RING of them
// in LDS.  A lane's operand of a product is one block of 32 columns: half q of the wave takes the blocks 4 q .. 4 q + 3 of a slab, so that
// the scales of a fragment's four steps are one word, a byte a step.  Where K is short two workgroups a compute unit (RING 2) do
// better than one with a longer ring: 2048 tokens of 64 experts, WM 1, WN 2, RING 4 / 2: 139 / 94 us (k_mx4_wide, which the plan takes there: 79).
#define M4_K 256
static __device__ __forceinline__ void mx_dma16(unsigned at, int off, lt_rsrc_t rs, int soff) {
  // (assembly: told that a load writes LDS, the compiler would wait for all of them in front of every barrier and LDS read; the waits
  // stand by hand)
  __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                   :: "s"(at), "v"(off), "s"(rs), "s"(soff) : "memory", "m0");
}
static __device__ __forceinline__ void mx_dma4(unsigned at, int off, lt_rsrc_t rs, int soff) {
  __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                   :: "s"(at), "v"(off), "s"(rs), "s"(soff) : "memory", "m0");
}
typedef __attribute__((address_space(3))) const u32x4_t lds_u4;
typedef __attribute__((address_space(3))) const u32 lds_u1;
template <int S>
static __device__ __forceinline__ f32x16_t mx_mfma32(u32x4_t a, u32x4_t b, f32x16_t c, u32 sa, u32 sb) {
  const i32x8_t a8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, b8{(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, S, (int)sa, S, (int)sb);
}
// the bytes of a word of scales that stand for blocks in front of the last, `left` of them; what lies behind may be anything, NaN too
static __device__ __forceinline__ u32 mx_mask(int left) { return left >= 4 ? ~0u : left <= 0 ? 0u : (1u << 8 * left) - 1u; }

template <bool F16, bool GATED, int WM, int WN, int RING>
__global__ __launch_bounds__(256, RING * (WM + WN) * 64 * 136 > 80 * 1024 ? 1 : 2) void k_mx4_tile(const MxArgs a) {
  constexpr int BM = 64 * WM, BN = 64 * WN, NX = 2 * WM, NW = 2 * WN, NS = (WM + WN + 1) / 2, NG = WM * WN, NT = NX + NW + NS;
  constexpr int CODES = (BM + BN) * 128, SLAB = CODES + NS * 1024, NC = GATED ? BN / 2 : BN;
  __shared__ __align__(1024) unsigned char s_ring[RING * SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w & 1, wn = w >> 1;
  const int fr = lane & 31, q = lane >> 5;
  const MxTiles<BM, NC> tiles(a);
  const int v = tiles.begin();
  if (v >= tiles.end()) return;
  const MxTile t = tiles.at(a, v);
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)s_ring;
  const uint8_t *w0 = a.w[0] + t.e * a.ew + t.n0 * a.ldw, *w1 = a.w[GATED ? 1 : 0] + t.e * a.ew + t.n0 * a.ldw;
  const int slabs = mx_slabs(a.K);
  const uint8_t *ws0 = a.ws[0] + t.e * a.ews + mx_scale_row(t.n0, slabs), *ws1 = a.ws[GATED ? 1 : 0] + t.e * a.ews + mx_scale_row(t.n0, slabs);
  const long long xbase = a.tok ? 0 : t.m0;
  const lt_rsrc_t rx = lt_rsrc((const uint8_t *)a.x + xbase * a.ldx), rxs = lt_rsrc(a.xs + mx_scale_row(xbase & ~31ll, slabs));
  const lt_rsrc_t rw0 = lt_rsrc(w0), rw1 = lt_rsrc(w1), rs0 = lt_rsrc(ws0), rs1 = lt_rsrc(ws1);
  auto wrow = [&](int i) { return min(t.n0 + i, a.N - 1) - t.n0; };
  // transfer i of wave w: rows 32 i + 8 w .. + 7, eight lanes a row; the lanes choose the chunk that belongs in their slot (chunk c of row
  // r in slot c ^ ((r >> 1) & 7)).  Scales: 32 rows a transfer, a word for each half of the wave, transfer 4 i + w of x's blocks and then W's.
  const int tr = 8 * w + (lane >> 3), chunk = (lane & 7) ^ ((tr >> 1) & 7);
  int vx[NX], vw[NW], vs[NS], row[NX + NS];
  mx_rows_of_x(a, t, row, [&](int i) { return i < NX ? 32 * i + tr : 32 * min(4 * (i - NX) + w, NX - 1) + (lane >> 1); });
#pragma unroll
  for (int i = 0; i < NX; ++i) vx[i] = row[i] * (int)a.ldx + 16 * chunk;
#pragma unroll
  for (int i = 0; i < NW; ++i) vw[i] = wrow(32 * (GATED ? i >> 1 : i) + tr) * (int)a.ldw + 16 * chunk;
  lt_rsrc_t rsc[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int b = 4 * i + w, bw = b - NX;
    if (b < NX) { vs[i] = (int)mx_scale_row(row[NX + i] + (xbase & 31), slabs) + 4 * (lane & 1); rsc[i] = rxs; }
    else {
      vs[i] = b < NX + NW ? (int)mx_scale_row(wrow(32 * (GATED ? bw >> 1 : bw) + (lane >> 1)), slabs) + 4 * (lane & 1) : LT_OUT;
      rsc[i] = GATED && (bw & 1) ? rs1 : rs0;
    }
  }
  const int kt0 = t.kt0, nk = t.nk, blocks = min(a.K >> 5, nk * (M4_K / 32));  // (past the last block: zeros)
  auto dma = [&](int i, int kt, int place) {
    if (i < NX + NW) {
      const bool in = kt * 8 + chunk < blocks;
      mx_dma16(lds + (unsigned)(place + (i * 32 + 8 * w) * 128), in ? (i < NX ? vx[i < NX ? i : 0] : vw[i < NX ? 0 : i - NX]) : LT_OUT,
               i < NX ? rx : (GATED && ((i - NX) & 1)) ? rw1 : rw0, kt * (M4_K / 2));
    } else {
      const int s = i - NX - NW;
      const bool in = kt * 8 + 4 * (lane & 1) < blocks;
      mx_dma4(lds + (unsigned)(place + CODES + (4 * s + w) * 256), in ? vs[s] : LT_OUT, rsc[s], kt * 256);
    }
  };
  unsigned ax[4], aw[4];  // LDS address of the lane's fragment of step j in block 0, of rows that begin where the ring does
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned c = (unsigned)(((4 * q + j) ^ ((fr >> 1) & 7)) * 16);
    ax[j] = lds + (unsigned)((wm * 32 + fr) * 128) + c;
    aw[j] = lds + (unsigned)((BM + wn * WN * 32 + fr) * 128) + c;
  }
  const unsigned asx = lds + CODES + (unsigned)((wm * 32 + fr) * 8 + 4 * q), asw = lds + CODES + (unsigned)((BM + wn * WN * 32 + fr) * 8 + 4 * q);
  f32x16_t acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int b = 0; b < WN; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][b][e] = 0.f;
  // A slab's products are short, a step of them shorter than an LDS read: the fragments of the whole next slab are read between this
  // one's.  At the barrier everybody has this slab's fragments, so its slot is free, and the next has landed.
#pragma unroll
  for (int i = 0; i < RING; ++i)
#pragma unroll
    for (int d = 0; d < NT; ++d) dma(d, kt0 + i, i * SLAB);
  LT_VM((RING - 1) * NT);
  __builtin_amdgcn_s_barrier();
  u32x4_t fx[2][4][WM], fw[2][4][WN];
  u32 sx[2][WM], sw[2][WN];
  auto read = [&](int p, int r, unsigned place) {  // fragment r of a slab: scales, then step by step
    if (r < WM) sx[p][r] = *(lds_u1 *)(uintptr_t)(asx + place + (unsigned)(r * 512));
    else if (r < WM + WN) sw[p][r - WM] = *(lds_u1 *)(uintptr_t)(asw + place + (unsigned)((r - WM) * 256));
    else {
      const int s = r - WM - WN, j = s / (WM + WN), i = s % (WM + WN);
      if (i < WM) fx[p][j][i] = *(lds_u4 *)(uintptr_t)(ax[j] + place + (unsigned)(i * 64 * 128));
      else fw[p][j][i - WM] = *(lds_u4 *)(uintptr_t)(aw[j] + place + (unsigned)((i - WM) * 32 * 128));
    }
  };
  constexpr int NR = 5 * (WM + WN), NP = 4 * NG;
#pragma unroll
  for (int r = 0; r < NR; ++r) read(0, r, 0);
  int slot = 0;
  auto step = [&](auto p_, int kt) {
    constexpr int p = decltype(p_)::value;
    const int next = slot + 1 < RING ? slot + 1 : 0;
    LT_LGKM0();
    LT_VM((RING - 2) * NT);
    __builtin_amdgcn_s_barrier();
    const u32 mask = mx_mask(blocks - kt * 8 - 4 * q);
#pragma unroll
    for (int i = 0; i < WM; ++i) sx[p][i] &= mask;
#pragma unroll
    for (int i = 0; i < WN; ++i) sw[p][i] &= mask;
    __builtin_amdgcn_sched_barrier(0);
    lt_each<NP>([&](auto g_) {
      constexpr int g = decltype(g_)::value, j = g / NG, i = g % NG / WN, b = g % WN;
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r * NP / NR == g) read(p ^ 1, r, (unsigned)(next * SLAB));
#pragma unroll
      for (int d = 0; d < NT; ++d)
        if (d * NP / NT == g) dma(d, kt + RING, slot * SLAB);
      __builtin_amdgcn_sched_barrier(0);
      acc[i][b] = mx_mfma32<j>(fw[p][j][b], fx[p][j][i], acc[i][b], sw[p][b], sx[p][i]);
      __builtin_amdgcn_sched_barrier(0);
    });
    slot = next;
  };
  // (always a pair of slabs: one past the end is zeros)
  for (int kt = kt0; kt < nk; kt += 2) {
    step(std::integral_constant<int, 0>(), kt);
    step(std::integral_constant<int, 1>(), kt + 1);
  }
  static_assert(4 * 32 * (32 * WN + 4) * 4 <= RING * SLAB, "the sums of four waves fit the ring");
  mx_tile_out<F16, GATED, WM, WN>(mx_out(a, t), acc, s_ring, t.m0, t.n0, t.split);
}

// ---- wide tiles, x in 4 bits: 256 x 256 -------------------------------------------------------------------------------------------
// The same four waves, each on 4 x 4 blocks of 32 x 32: a step (a quarter of a slab) is 16 products, which last many times an LDS read, so that
// fragments are read step by step.  Two slabs in LDS.  The fragments of a whole slab fit the registers (four steps of eight), and they are
// read as early as the slab is there: in the middle of its step 1 everybody has all of it, so its place takes the slab after next from
// then on, more than a slab's time in front of the first read of that.
// 4096 x 4096 x 14336 108 to 124 us (3.9 to 4.5 PFLOP/s).  4096 x 4096, one round of tiles, K 1024 / 2048 / 4096 / 8192 / 11264 / 14336: 20.9 / 27.4 / 41.4 /
// 71.3 / 90.4 / 111.2 us, so 1.7 us a slab (2048 cycles of products, which are 0.85 us at 2.4 GHz) and 14 us of start and write-out, which nothing
// hides.  Why a slab takes twice its products' cycles is not separated: the clock under this load, LDS and waits all have a part.
template <bool F16, bool GATED>
__global__ __launch_bounds__(256, 1) void k_mx4_wide(const MxArgs a) {
  constexpr int B = 256, NB = 4, NX = 8, NW = 8, NS = 4, NT = NX + NW + NS;
  constexpr int CODES = 2 * B * 128, SLAB = CODES + NS * 1024, NC = GATED ? B / 2 : B;
  constexpr int FREE = 28, SENT = 60;  // product (of 64) in front of which a slab's place is free; the last that a transfer goes with
  __shared__ __align__(1024) unsigned char s_ring[2 * SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w & 1, wn = w >> 1;
  const int fr = lane & 31, q = lane >> 5;
  const MxTiles<B, NC> tiles(a);
  const int v = tiles.begin();
  if (v >= tiles.end()) return;
  const MxTile t = tiles.at(a, v);
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)s_ring;
  const int slabs = mx_slabs(a.K);
  const long long xbase = a.tok ? 0 : t.m0;
  const lt_rsrc_t rx = lt_rsrc((const uint8_t *)a.x + xbase * a.ldx), rxs = lt_rsrc(a.xs + mx_scale_row(xbase & ~31ll, slabs));
  const lt_rsrc_t rw0 = lt_rsrc(a.w[0] + t.e * a.ew + t.n0 * a.ldw), rw1 = lt_rsrc(a.w[GATED ? 1 : 0] + t.e * a.ew + t.n0 * a.ldw);
  const lt_rsrc_t rs0 = lt_rsrc(a.ws[0] + t.e * a.ews + mx_scale_row(t.n0, slabs)), rs1 = lt_rsrc(a.ws[GATED ? 1 : 0] + t.e * a.ews + mx_scale_row(t.n0, slabs));
  auto wrow = [&](int i) { return min(t.n0 + i, a.N - 1) - t.n0; };
  // transfers as in k_mx4_tile; scales: transfers 0 and 1 x's blocks w and 4 + w, 2 and 3 W's
  const int tr = 8 * w + (lane >> 3), chunk = (lane & 7) ^ ((tr >> 1) & 7);
  int vx[NX], vw[NW], vs[NS], row[NX + 2];
  mx_rows_of_x(a, t, row, [&](int i) { return i < NX ? 32 * i + tr : 32 * (4 * (i - NX) + w) + (lane >> 1); });
#pragma unroll
  for (int i = 0; i < NX; ++i) vx[i] = t.m0 + 32 * i < t.m_end ? row[i] * (int)a.ldx + 16 * chunk : LT_OUT;  // (blocks without a row: zeros)
#pragma unroll
  for (int i = 0; i < NW; ++i) vw[i] = wrow(32 * (GATED ? i >> 1 : i) + tr) * (int)a.ldw + 16 * chunk;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 4 * i + w;
    vs[i] = (int)mx_scale_row(row[NX + i] + (xbase & 31), slabs) + 4 * (lane & 1);
    vs[2 + i] = (int)mx_scale_row(wrow(32 * (GATED ? b >> 1 : b) + (lane >> 1)), slabs) + 4 * (lane & 1);
  }
  const lt_rsrc_t rsw = GATED && (w & 1) ? rs1 : rs0;
  const int kt0 = t.kt0, nk = t.nk, blocks = min(a.K >> 5, nk * (M4_K / 32));
  auto dma = [&](int i, int kt, int place) {
    if (i < NX + NW) {
      const bool in = kt * 8 + chunk < blocks;
      mx_dma16(lds + (unsigned)(place + (i * 32 + 8 * w) * 128), in ? (i < NX ? vx[i < NX ? i : 0] : vw[i < NX || i >= NX + NW ? 0 : i - NX]) : LT_OUT,
               i < NX ? rx : (GATED && (i & 1)) ? rw1 : rw0, kt * (M4_K / 2));
    } else {
      const int s = i - NX - NW;
      const bool in = kt * 8 + 4 * (lane & 1) < blocks;
      mx_dma4(lds + (unsigned)(place + CODES + (4 * s + w) * 256), in ? vs[s] : LT_OUT, s < 2 ? rxs : rsw, kt * 256);
    }
  };
  unsigned ax[4], aw[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned c = (unsigned)(((4 * q + j) ^ ((fr >> 1) & 7)) * 16);
    ax[j] = lds + (unsigned)((wm * 32 + fr) * 128) + c;
    aw[j] = lds + (unsigned)((B + wn * 128 + fr) * 128) + c;
  }
  const unsigned asx = lds + CODES + (unsigned)((wm * 32 + fr) * 8 + 4 * q), asw = lds + CODES + (unsigned)((B + wn * 128 + fr) * 8 + 4 * q);
  f32x16_t acc[NB][NB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][b][e] = 0.f;
  u32x4_t fx[4][NB], fw[4][NB];
  u32 sx[2][NB], sw[2][NB];
  auto read = [&](int j, int r, unsigned place) {  // fragment r of step j in the order of need: W's first, then x's
    if (r < NB) fw[j][r & 3] = *(lds_u4 *)(uintptr_t)(aw[j] + place + (unsigned)((r & 3) * 32 * 128));
    else fx[j][r & 3] = *(lds_u4 *)(uintptr_t)(ax[j] + place + (unsigned)((r & 3) * 64 * 128));
  };
  auto read_s = [&](int p, int r, unsigned place) {
    if (r < NB) sw[p][r & 3] = *(lds_u1 *)(uintptr_t)(asw + place + (unsigned)((r & 3) * 256));
    else sx[p][r & 3] = *(lds_u1 *)(uintptr_t)(asx + place + (unsigned)((r & 3) * 512));
  };
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int d = 0; d < NT; ++d) dma(d, kt0 + i, i * SLAB);
  LT_VM(NT);
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int r = 0; r < 2 * NB; ++r) { read_s(0, r, 0); read(0, r, 0); }
  // slab kt in place p; transfers that are sent in front of product g of the slab's 64: those of slab kt + 2, from FREE on
  auto sent = [](int g) { return g < FREE ? 0 : g >= SENT ? NT : (g - FREE) * NT / (SENT - FREE); };
  auto slab = [&](auto p_, auto ni_, int kt) {
    constexpr int p = decltype(p_)::value, NI = decltype(ni_)::value;
    constexpr int PLACE = p * SLAB, NEXT = (p ^ 1) * SLAB;
    const u32 mask = mx_mask(blocks - kt * 8 - 4 * q);
    LT_LGKM0();
#pragma unroll
    for (int i = 0; i < NB; ++i) { sx[p][i] &= mask; sw[p][i] &= mask; }
    __builtin_amdgcn_sched_barrier(0);
    lt_each<64>([&](auto g_) {
      constexpr int g = decltype(g_)::value, j = g / 16, i = g % 16 / NB, b = g % NB;
      if constexpr (g < 24 && g % 8 < NB + NI) read(1 + g / 8, g % 8, PLACE);                     // (as fast as LDS gives them to four waves)
      if constexpr (g == FREE) {
        LT_LGKM0();
        __builtin_amdgcn_s_barrier();
      }
      if constexpr (g == 48) {                                                 // the next slab has landed
        LT_VM(sent(48));
        __builtin_amdgcn_s_barrier();
      }
      if constexpr (g >= 48 && g < 52 + NI) { read_s(p ^ 1, g - 48, NEXT); read(0, g - 48, NEXT); }
#pragma unroll
      for (int d = 0; d < NT; ++d)
        if (d >= sent(g) && d < sent(g + 1)) dma(d, kt + 2, PLACE);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i < NI) acc[i][b] = mx_mfma32<j>(fw[j][b], fx[j][i], acc[i][b], sw[p][b], sx[p][i]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto run = [&](auto ni) {
    for (int kt = kt0; kt < nk; kt += 2) {  // (always a pair of slabs: one past the end is zeros)
      slab(std::integral_constant<int, 0>(), ni, kt);
      slab(std::integral_constant<int, 1>(), ni, kt + 1);
    }
  };
  // an expert's last rows: a wave leaves out the products of blocks that have none (the waits and barriers are the same for all)
  switch (min(NB, ((t.m_end - t.m0 + 31) / 32 - wm + 1) / 2)) {
    case 4: run(std::integral_constant<int, 4>()); break;
    case 3: run(std::integral_constant<int, 3>()); break;
    case 2: run(std::integral_constant<int, 2>()); break;
    case 1: run(std::integral_constant<int, 1>()); break;
    default: run(std::integral_constant<int, 0>()); break;
  }
  static_assert(4 * 32 * (32 * NB + 4) * 4 <= 2 * SLAB, "the sums of four waves fit the ring");
  mx_tile_out<F16, GATED, NB, NB>(mx_out(a, t), acc, s_ring, t.m0, t.n0, t.split);
}

static __device__ __forceinline__ f32x16_t mx_mfma32_bf16(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// x in 16 bits: the same tile, K 128 at a time (256 bytes of a row of x, 64 of codes, one word of scales).  Half q of the wave takes the
// columns 64 q .. 64 q + 63 of a slab, eight a step: blocks 2 q and 2 q + 1 of W, which become bf16 in front of their products.
// Chunk c (16 bytes) of row r of x stands in slot c ^ (r & 15), of W in slot c ^ ((r >> 2) & 3).  Bound by LDS, which x fills: wide tiles are the
// better ones (2048 tokens of 64 experts, us: 64 x 256 166, 128 x 128 209).  4096 x 4096 x 14336 374 to 441 us (1090 to 1290 TFLOP/s);
// past 2048 rows (fp16: 1024) weights expanded by k_mx4_dequantize and the product of 16-bit matrices are mostly faster (327 together).
#define M16_K 128
template <int X, bool GATED, int WM, int WN, int RING>
__global__ __launch_bounds__(256, RING * (WM * 64 * 256 + WN * 64 * 64 + 1024) > 80 * 1024 ? 1 : 2) void k_mx4_tile16(const MxArgs a) {
  constexpr bool F16 = X == X_FP16;
  constexpr int BM = 64 * WM, BN = 64 * WN, NX = 4 * WM, NW = WN, NG = WM * WN, NT = NX + NW + 1;
  constexpr int XS = BM * 256, CODES = XS + BN * 64, SLAB = CODES + 1024, NC = GATED ? BN / 2 : BN;
  __shared__ __align__(1024) unsigned char s_ring[RING * SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w & 1, wn = w >> 1;
  const int fr = lane & 31, q = lane >> 5;
  const MxTiles<BM, NC> tiles(a);
  const int v = tiles.begin();
  if (v >= tiles.end()) return;
  const MxTile t = tiles.at(a, v);
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)s_ring;
  const long long xbase = a.tok ? 0 : t.m0;
  const lt_rsrc_t rx = lt_rsrc((const uint8_t *)a.x + xbase * a.ldx);
  const lt_rsrc_t rw0 = lt_rsrc(a.w[0] + t.e * a.ew + t.n0 * a.ldw), rw1 = lt_rsrc(a.w[GATED ? 1 : 0] + t.e * a.ew + t.n0 * a.ldw);
  const int slabs = mx_slabs(a.K);
  const lt_rsrc_t rs0 = lt_rsrc(a.ws[0] + t.e * a.ews + mx_scale_row(t.n0, slabs)), rs1 = lt_rsrc(a.ws[GATED ? 1 : 0] + t.e * a.ews + mx_scale_row(t.n0, slabs));
  // transfer i of wave w: four rows of x from 16 i + 4 w on, sixteen lanes a row; sixteen rows of W from 64 i + 16 w on, four lanes a row.
  // Scales: wave w (w < WN) 64 rows of W.
  const int xr = 4 * w + (lane >> 4), xc = (lane & 15) ^ xr, wr = 16 * w + (lane >> 2), wc = (lane & 3) ^ ((wr >> 2) & 3);
  auto wrow = [&](int i) {  // row i of the tile in its matrix, from n0 on
    const int n = GATED ? 32 * (i >> 6) + (i & 31) : i;
    return min(t.n0 + n, a.N - 1) - t.n0;
  };
  int vx[NX], vw[NW];
  mx_rows_of_x(a, t, vx, [&](int i) { return 16 * i + xr; });
#pragma unroll
  for (int i = 0; i < NX; ++i) vx[i] = vx[i] * (int)a.ldx + 16 * xc;
#pragma unroll
  for (int i = 0; i < NW; ++i) vw[i] = wrow(64 * i + wr) * (int)a.ldw + 16 * wc;
  // a gated pair's matrices change every 32 rows of the tile, so with the wave; its scales stand one matrix behind the other, 64 rows a wave
  const lt_rsrc_t rw = GATED && (w & 2) ? rw1 : rw0, rs = GATED && w >= WN / 2 ? rs1 : rs0;
  const int vs = w < WN ? (int)mx_scale_row(min(t.n0 + 64 * (GATED ? w % ((WN + 1) / 2) : w) + lane, a.N - 1) - t.n0, slabs) : LT_OUT;
  const int kt0 = t.kt0, nk = t.nk, blocks = min(a.K >> 5, nk * (M16_K / 32));  // (past the last block: zeros)
  auto dma = [&](int i, int kt, int place) {
    if (i < NX) {
      const bool in = kt * 4 + (xc >> 2) < blocks;
      mx_dma16(lds + (unsigned)(place + (i * 16 + 4 * w) * 256), in ? vx[i < NX ? i : 0] : LT_OUT, rx, kt * (M16_K * 2));
    } else if (i < NX + NW) {
      const bool in = kt * 4 + wc < blocks;
      mx_dma16(lds + (unsigned)(place + XS + ((i - NX) * 64 + 16 * w) * 64), in ? vw[i < NX || i >= NX + NW ? 0 : i - NX] : LT_OUT, rw, kt * (M16_K / 2));
    } else {
      mx_dma4(lds + (unsigned)(place + CODES + w * 256), kt * 4 < blocks ? vs : LT_OUT, rs, (kt >> 1) * 256 + (kt & 1) * 4);
    }
  };
  unsigned ax[8], aw[2], as[WN];  // LDS address of the lane's fragments in block 0 (scales: every block), of rows that begin where the ring does
#pragma unroll
  for (int j = 0; j < 8; ++j) ax[j] = lds + (unsigned)((wm * 32 + fr) * 256 + ((8 * q + j) ^ (fr & 15)) * 16);
#pragma unroll
  for (int h = 0; h < 2; ++h) aw[h] = lds + (unsigned)(XS + (wn * WN * 32 + fr) * 64 + ((2 * q + h) ^ ((fr >> 2) & 3)) * 16);
#pragma unroll
  for (int b = 0; b < WN; ++b) {
    const int block = wn * WN + b;
    as[b] = lds + (unsigned)(CODES + (GATED ? (block & 1) * NC + 32 * (block >> 1) + fr : 32 * block + fr) * 4);
  }
  f32x16_t acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int b = 0; b < WN; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][b][e] = 0.f;
#pragma unroll
  for (int i = 0; i < RING; ++i)
#pragma unroll
    for (int d = 0; d < NT; ++d) dma(d, kt0 + i, i * SLAB);
  // fp16: can all weights of this wave be fp16?  Decided by all of their scales (a sixteenth of the codes' bytes) while the ring fills.
  // One scale outside of 104 .. 140, such as the 0 of a block of zeros, sends the wave's rows of W through the split form for all of K:
  // 4096 x 4096 x 14336 with such a block in every 32 rows 958 us (without 435), 379 x 1409 x 2048 28.8 (9.8).
  bool fits = false;
  if constexpr (F16) {
    u16x2_t least{127, 127}, most{127, 127};
    for (int b = 0; b < WN; ++b) {
      const int block = wn * WN + b, row0 = t.n0 + 32 * (GATED ? block >> 1 : block);
      const uint8_t *base = a.ws[GATED ? block & 1 : 0] + t.e * a.ews + mx_scale_row(row0, slabs);
      if (row0 < a.N)
        for (int i = lane; i < slabs * 16; i += 64) {  // 16 bytes: two rows of a slab
          const u32x4_t v = *(const u32x4_t *)(base + 16 * i);
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const u32 mask = row0 + 2 * (i & 15) + (d >> 1) < a.N ? mx_mask((a.K >> 5) - 8 * (i >> 4) - 4 * (d & 1)) : 0u;
            const u32 w4 = (v[d] & mask) | (0x7f7f7f7fu & ~mask);
            const u16x2_t even = __builtin_bit_cast(u16x2_t, w4 & 0x00ff00ffu), odd = __builtin_bit_cast(u16x2_t, w4 >> 8 & 0x00ff00ffu);
            least = __builtin_elementwise_min(least, __builtin_elementwise_min(even, odd));
            most = __builtin_elementwise_max(most, __builtin_elementwise_max(even, odd));
          }
        }
    }
    fits = __all(mx_fits_f16(min(least[0], least[1])) && mx_fits_f16(max(most[0], most[1])));
  }
  LT_VM((RING - 1) * NT);
  __builtin_amdgcn_s_barrier();
  u32x4_t fx[2][8][WM], fw[2][2][WN];
  u32 fs[2][WN];
  auto read = [&](int p, int r, unsigned place) {  // fragment r of a slab: scales and W, then x step by step
    if (r < WN) fs[p][r] = *(lds_u1 *)(uintptr_t)(as[r < WN ? r : 0] + place);
    else if (r < 3 * WN) {
      const int h = (r - WN) / WN, b = (r - WN) % WN;
      fw[p][h & 1][b] = *(lds_u4 *)(uintptr_t)(aw[h & 1] + place + (unsigned)(b * 32 * 64));
    } else {
      const int j = (r - 3 * WN) / WM, i = (r - 3 * WN) % WM;
      fx[p][j][i] = *(lds_u4 *)(uintptr_t)(ax[j] + place + (unsigned)(i * 64 * 256));
    }
  };
  constexpr int NR = 3 * WN + 8 * WM, NP = 8 * NG;
  // operands of a step, made during the step before.  FAST (fp16): the weights become fp16 and x stays as it is; otherwise x is two
  // bf16 and the products are twice as many.
  u32x4_t cw[2][WN], hi[2][WM], lo[2][WM];
  float sv[WN][2];
  constexpr int NC2 = WN + (F16 ? WM : 0);
  auto make = [&](auto fast_, int m, int j, int p, int kt) {
    constexpr bool FAST = decltype(fast_)::value;
    if (m < WN) {
      const int b = m < WN ? m : 0;
      if (j == 0) {
        const u32 two = (fs[p][b] & mx_mask(blocks - kt * 4)) >> (16 * q);
        sv[b][0] = __uint_as_float((two & 255u) << 23);
        sv[b][1] = __uint_as_float((two >> 8 & 255u) << 23);
      }
      cw[j & 1][b] = FAST ? mx_f16(fw[p][j >> 2][b][j & 3], sv[b][j >> 2]) : mx_bf16(fw[p][j >> 2][b][j & 3], sv[b][j >> 2]);
    } else if constexpr (F16 && !FAST) {
      const int i = m < WN ? 0 : m - WN;
      mx_split(fx[p][j][i], hi[j & 1][i], lo[j & 1][i]);
    }
  };
  int slot = 0;
  auto step = [&](auto p_, auto fast_, int kt) __attribute__((always_inline)) {
    constexpr int p = decltype(p_)::value;
    constexpr bool FAST = decltype(fast_)::value;
    const int next = slot + 1 < RING ? slot + 1 : 0;
    LT_LGKM0();
    LT_VM((RING - 2) * NT);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    lt_each<NP>([&](auto g_) {
      constexpr int g = decltype(g_)::value, j = g / NG, i = g % NG / WN, b = g % WN, in = g % NG;
      // (the next slab's fragments are all there in front of the last step, which makes the first operands of them)
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r * (NP - NG) / NR == g) read(p ^ 1, r, (unsigned)(next * SLAB));
#pragma unroll
      for (int d = 0; d < NT; ++d)
        if (d * NP / NT == g) dma(d, kt + RING, slot * SLAB);
#pragma unroll
      for (int m = 0; m < NC2; ++m)
        if (m * NG / NC2 == in) make(fast_, m, (j + 1) & 7, j == 7 ? p ^ 1 : p, j == 7 ? kt + 1 : kt);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (FAST) {
        acc[i][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, cw[j & 1][b]), __builtin_bit_cast(f16x8_t, fx[p][j][i]), acc[i][b], 0, 0, 0);
      } else {
        acc[i][b] = mx_mfma32_bf16(cw[j & 1][b], F16 ? hi[j & 1][i] : fx[p][j][i], acc[i][b]);
        if constexpr (F16) acc[i][b] = mx_mfma32_bf16(cw[j & 1][b], lo[j & 1][i], acc[i][b]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    slot = next;
  };
  auto run = [&](auto fast) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < NR; ++r) read(0, r, 0);
#pragma unroll
    for (int m = 0; m < NC2; ++m) make(fast, m, 0, 0, kt0);
    for (int kt = kt0; kt < nk; kt += 2) {  // (always a pair of slabs: one past the end is zeros)
      step(std::integral_constant<int, 0>(), fast, kt);
      step(std::integral_constant<int, 1>(), fast, kt + 1);
    }
  };
  if constexpr (F16) {
    if (fits) run(std::true_type());
    else run(std::false_type());
  } else {
    run(std::false_type());
  }
  static_assert(4 * 32 * (32 * WN + 4) * 4 <= RING * SLAB, "the sums of four waves fit the ring");
  mx_tile_out<F16, GATED, WM, WN>(mx_out(a, t), acc, s_ring, t.m0, t.n0, t.split);
}

// ---- entry points -------------------------------------------------------------------------------------------------------------
// Do na rows of len_a bytes, la apart, share a byte with nb rows of len_b bytes, lb apart?  (Rows side by side in one buffer, the same
// distance apart, do not; rows of different distances whose ranges meet are taken to.)
static bool mx_meet(const void *a, int64_t na, int64_t la, int64_t len_a, const void *b, int64_t nb, int64_t lb, int64_t len_b) {
  const char *p = (const char *)a, *q = (const char *)b;
  if (!p || !q || na <= 0 || nb <= 0 || len_a <= 0 || len_b <= 0 || p >= q + (nb - 1) * lb + len_b || q >= p + (na - 1) * la + len_a) return false;
  if (la != lb || la <= 0) return true;
  const int64_t d = ((p - q) % lb + lb) % lb;
  return d < len_b || d + len_a > lb;
}
extern "C" int64_t moe_mx4_scale_bytes(int64_t rows, int K) {
  return rows <= 0 || K <= 0 ? 0 : (rows + 31) / 32 * mx_slabs(K) * 256;
}
static int quant_run(const char *who, const void *v, int64_t ldv, int64_t next_v, int dtype, int E, int M, int K, const moe_mx4 *q, bool back,
                     hipStream_t s) {
  const int size = dtype == MOE_DT_FP32 ? 4 : 2;
  const bool one = E <= 1;
  if (!q || E < 0 || M < 0 || K < 0 || K % 32 || dtype < MOE_DT_BF16 || dtype > MOE_DT_FP32 || E > 65535 || ldv < K || ldv >= 1ll << 40 ||
      q->ldc < K / 2 || q->ldc % 16 || q->ldc >= 1ll << 40 || ldv * size % 16 ||
      (!one && (next_v < 0 || next_v * size % 16 || q->next_c < 0 || q->next_c % 16 || q->next_s < 0))) {
    moe_set_error("%s: bad shape (E=%d M=%d K=%d dtype=%d, rows %lld and %lld apart)", who, E, M, K, dtype, (long long)ldv,
                  q ? (long long)q->ldc : 0);
    return MOE_EINVAL;
  }
  if (!E || !M || !K) return MOE_OK;
  if (!v || !q->codes || !q->scales || (((uintptr_t)v | (uintptr_t)q->codes) & 15)) {
    moe_set_error("%s: rows of values and of codes must be present and on 16-byte boundaries", who);
    return MOE_EINVAL;
  }
  const int64_t n = (int64_t)M * (K / 8);
  if (n >= 1ll << 31) {
    moe_set_error("%s: %d x %d values are too many for one matrix", who, M, K);
    return MOE_EINVAL;
  }
  const int64_t nv = one ? 0 : next_v * size, nc = one ? 0 : q->next_c, ns = one ? 0 : q->next_s;
  const int64_t all_v = (E - 1) * nv + (M - 1) * ldv * size + (int64_t)K * size, all_c = (E - 1) * nc + (M - 1) * q->ldc + K / 2;
  const int64_t all_s = (E - 1) * ns + moe_mx4_scale_bytes(M, K);
  if (mx_meet(v, 1, 0, all_v, q->codes, 1, 0, all_c) || mx_meet(v, 1, 0, all_v, q->scales, 1, 0, all_s) ||
      mx_meet(q->codes, 1, 0, all_c, q->scales, 1, 0, all_s)) {
    moe_set_error("%s: values, codes and scales overlap", who);
    return MOE_EINVAL;
  }
  QuantArgs a{(const char *)(back ? q->codes : v), (char *)(back ? v : q->codes), (uint8_t *)q->scales, ldv, q->ldc, one ? 0 : next_v, nc, ns,
              (u32)n, (u32)K / 8, 0, 0, mx_slabs(K)};
  while ((1ull << a.shift) < a.per) ++a.shift;
  a.magic = (u32)((((1ull << a.shift) - a.per) << 32) / a.per + 1);
  const dim3 grid((unsigned)((n + 256 * QT_U - 1) / (256 * QT_U)), E);
  switch (dtype * 2 + (back ? 1 : 0)) {
    case 0: hipLaunchKernelGGL(k_mx4_quantize<MOE_DT_BF16>, grid, dim3(256), 0, s, a); break;
    case 1: hipLaunchKernelGGL(k_mx4_dequantize<MOE_DT_BF16>, grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL(k_mx4_quantize<MOE_DT_FP16>, grid, dim3(256), 0, s, a); break;
    case 3: hipLaunchKernelGGL(k_mx4_dequantize<MOE_DT_FP16>, grid, dim3(256), 0, s, a); break;
    case 4: hipLaunchKernelGGL(k_mx4_quantize<MOE_DT_FP32>, grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL(k_mx4_dequantize<MOE_DT_FP32>, grid, dim3(256), 0, s, a); break;
  }
  return moe_check_launch(back ? "k_mx4_dequantize" : "k_mx4_quantize");
}
extern "C" int moe_mx4_quantize(const void *x, int64_t ldx, int64_t next_x, int dtype, int E, int M, int K, const moe_mx4 *q, void *stream) {
  return quant_run("moe_mx4_quantize", x, ldx, next_x, dtype, E, M, K, q, false, (hipStream_t)stream);
}
extern "C" int moe_mx4_dequantize(const moe_mx4 *q, int E, int M, int K, void *y, int64_t ldy, int64_t next_y, int dtype, void *stream) {
  return quant_run("moe_mx4_dequantize", y, ldy, next_y, dtype, E, M, K, q, true, (hipStream_t)stream);
}

// What the products of both kinds check; xrows: rows of x, experts: matrices
static int mx_check(const char *who, const MxArgs &a, int xkind, int64_t xrows, int experts, int dtype, bool gated) {
  const int64_t xlen = xkind == X_MX4 ? a.K / 2 : a.K * 2ll, wlen = a.K / 2;
  const bool empty = a.M == 0 || a.N == 0;
  if (a.M < 0 || a.N < 0 || a.K <= 0 || a.K % 32 || (dtype != MOE_DT_BF16 && dtype != MOE_DT_FP16) || a.act < MOE_ACT_NONE ||
      a.act > MOE_ACT_RELU2 || a.ldx < xlen || a.ldx % 16 || a.ldx >= 1 << 22 || a.ldw < wlen || a.ldw % 16 || a.ldw >= 1 << 22 ||
      a.ew < 0 || a.ews < 0 || a.ew % 16 || a.ews % 4 || a.ldy < a.N || (a.res && a.ldr < a.N) || a.M > 1 << 26 || a.N > 1 << 26) {
    moe_set_error("%s: bad shape (M=%d N=%d K=%d dtype=%d act=%d, rows %lld %lld %lld %lld apart)", who, a.M, a.N, a.K, dtype,
                  a.act, a.ldx, a.ldw, a.res ? a.ldr : 0, a.ldy);
    return MOE_EINVAL;
  }
  if (empty) return MOE_OK;
  uintptr_t low = (uintptr_t)a.x, low4 = (uintptr_t)a.xs;
  bool there = a.x && a.y && (xkind != X_MX4 || a.xs);
  for (int i = 0; i < (gated ? 2 : 1); ++i) {
    there = there && a.w[i] && a.ws[i];
    low |= (uintptr_t)a.w[i];
    low4 |= (uintptr_t)a.ws[i];
  }
  if (!there || (low & 15) || (low4 & 3)) {
    moe_set_error("%s: operands must be present, x and codes on 16-byte boundaries, scales on 4-byte ones", who);
    return MOE_EINVAL;
  }
  const int64_t e = a.y32 ? 4 : 2, ylen = a.N * e, yld = a.ldy * e;
  auto meets = [&](const void *p, int64_t rows, int64_t ld, int64_t len) { return mx_meet(a.y, a.M, yld, ylen, p, rows, ld, len); };
  bool shares = meets(a.x, xrows, a.ldx, xlen) || (xkind == X_MX4 && meets(a.xs, 1, 0, moe_mx4_scale_bytes(xrows, a.K)));
  for (int i = 0; i < (gated ? 2 : 1); ++i) {
    shares = shares || (experts == 1 ? meets(a.w[i], a.N, a.ldw, wlen) : meets(a.w[i], 1, 0, (experts - 1) * a.ew + (a.N - 1) * a.ldw + wlen)) ||
             meets(a.ws[i], 1, 0, (experts - 1) * a.ews + moe_mx4_scale_bytes(a.N, a.K)) || meets(a.bias[i], 1, 0, 2ll * experts * a.N);
  }
  const bool in_place = a.res == a.y && !a.y32 && (a.ldr == a.ldy || a.M == 1);
  if (shares || (!in_place && meets(a.res, a.M, a.ldr * 2, a.N * 2ll))) {
    moe_set_error("%s: the result overlaps an operand (only a residual may be the result itself)", who);
    return MOE_EINVAL;
  }
  return MOE_OK;
}
// Which kernel a product takes: few rows (wm 0), or tiles of 64 wm x 64 wn with `ring` slabs in LDS (4 x 4: the wide kernel), dense ones
// with K in `splits` pieces.  The plan of the least time after a model of one launch, us, fitted to measured times of dense products (12 matrices, 286
// products of 17 to 4096 rows for each kind of x, 12000 times in all; the chosen plan is 2.4 % (16-bit x 2.1 %) slower than the best of all
// on average, 31 % (20 %) at worst).  By expert it is an estimate from the average rows of an expert, not fitted:
//   start + rounds x (slabs x (c0 + c1 x share of the compute units in use) + f),  with pieces j0 + j1 a piece + j2 per MB of partial sums
// c0, c1: a slab of a workgroup on an idle chip, and what the others' traffic adds; f: first slab and epilogue.
struct MxPlan { int wm, wn, ring, splits; float us; };
struct MxTileKind { int wm, wn, ring, per_cu; float c0, c1, f; };
struct MxModel { MxTileKind tile[7]; int tiles; float start, j0, j1, j2; };
static const MxModel MX_MODEL4 = {{{1, 1, 4, 2, .163f, .111f, 2.46f}, {1, 2, 2, 2, .484f, .114f, 1.94f}, {1, 2, 4, 1, .284f, .133f, 2.59f},
                                   {2, 2, 2, 2, .534f, .307f, 2.32f}, {2, 2, 3, 1, .374f, .259f, 2.97f}, {2, 4, 3, 1, .680f, .397f, 3.98f},
                                   {4, 4, 2, 1, 1.072f, .633f, 3.98f}}, 7, 3.43f, 3.50f, .161f, .166f};
static const MxModel MX_MODEL16 = {{{1, 1, 3, 2, .264f, .118f, 2.32f}, {1, 2, 3, 2, .401f, .227f, 2.63f}, {1, 4, 2, 2, .742f, .386f, 2.49f},
                                    {2, 2, 3, 1, .633f, .222f, 3.08f}, {2, 4, 3, 1, 1.146f, .333f, 4.13f}}, 5, 3.62f, 2.90f, .217f, .174f};
// rows of all `units` products together; units 0: a dense one
static MxPlan mx_plan(int xkind, long long rows, int units, int N, int K, bool gated) {
  const long long each = units ? rows / units : rows;
  if (each <= (xkind == X_MX4 ? 8 : 16)) return MxPlan{0, 0, 0, 1, 0.f};
  static const int pieces[] = {1, 2, 3, 4, 6, 8, 12};
  const MxModel &model = xkind == X_MX4 ? MX_MODEL4 : MX_MODEL16;
  const int slab = xkind == X_MX4 ? M4_K : M16_K;
  const long long slabs = (K + slab - 1) / slab;
  MxPlan best{2, 2, 3, 1, 1e30f};
  for (int i = 0; i < model.tiles; ++i) {
    const MxTileKind &t = model.tile[i];
    if (gated && t.wn == 1) continue;  // (a pair needs both matrices' blocks in a wave)
    const int bm = 64 * t.wm, cols = 64 * t.wn / (gated ? 2 : 1);
    // by expert the last tile of each is half full on average (the counts are not known here), and the wide kernel leaves its empty blocks out
    const float full = (float)each / (float)bm;
    const float down = !units ? (float)((rows + bm - 1) / bm) : (float)units * (full >= 1.f ? full + .5f : 1.f + std::max(0.f, full - .7f) * 1.67f);
    const float fill = units && t.wm == 4 ? .3f + .7f * (float)rows / (down * (float)bm) : 1.f;
    const long long n = (long long)(down * (float)((N + cols - 1) / cols));
    for (int s : pieces) {
      if (s > slabs || (s > 1 && (units || n * s > 640))) break;
      const long long wgs = n * s, at_once = 256 * t.per_cu;
      const float use = wgs > 256 ? (float)t.per_cu : (float)wgs / 256.f;
      // (by expert rounds end at different times)
      const float rounds = units && wgs > at_once ? (float)wgs / (float)at_once + .25f : (float)((wgs + at_once - 1) / at_once);
      float us = model.start + rounds * ((float)((slabs + s - 1) / s) * (t.c0 + t.c1 * use) * fill + t.f);
      if (s > 1) us += model.j0 + model.j1 * (float)s + model.j2 * 8e-6f * (float)s * (gated ? 2.f : 1.f) * (float)rows * (float)N;
      if (us < best.us) best = MxPlan{t.wm, t.wn, t.ring, s, us};
    }
  }
  return best;
}
extern "C" int64_t moe_mx4_linear_workspace_bytes(int M, int N, int K, int x_mx4, int gated) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const MxPlan p = mx_plan(x_mx4 ? X_MX4 : X_BF16, M, 0, N, K, gated != 0);
  return p.splits > 1 ? (int64_t)p.splits * (gated ? 2 : 1) * M * ((N + 7) & ~7) * 4 : 0;
}
extern "C" int moe_mx4_plan(int64_t rows, int units, int N, int K, int x_mx4, int gated, int *plan) {
  if (rows <= 0 || units < 0 || N <= 0 || K <= 0 || !plan) {
    moe_set_error("moe_mx4_plan: bad argument (rows=%lld units=%d N=%d K=%d)", (long long)rows, units, N, K);
    return MOE_EINVAL;
  }
  const MxPlan p = mx_plan(x_mx4 ? X_MX4 : X_BF16, rows, units, N, K, gated != 0);
  plan[0] = 64 * p.wm; plan[1] = 64 * p.wn; plan[2] = p.ring; plan[3] = p.splits;
  return MOE_OK;
}
template <int X, bool F16, bool GATED>
static int mx_launch(const MxArgs &a, int units, int most, float *ws, hipStream_t s) {  // most: rows that one expert (or the product) can have
  const MxPlan pl = mx_plan(X, a.M, a.units ? units : 0, a.N, a.K, GATED);
  if (pl.wm == 0) {
#define MR_LAUNCH(SH_, NB_, W_)                                                                                                      \
  hipLaunchKernelGGL(HIP_KERNEL_NAME(k_mx4_rows<X, F16, GATED, SH_, NB_, 1, W_>), dim3((a.N + 16 / SH_ * NB_ - 1) / (16 / SH_ * NB_), units), \
                     dim3(64 * W_), 0, s, a)
    // Two blocks a workgroup share one operand of x where enough workgroups are left (16-bit x, us, NB 2 / 1: gated 8 x 14336 x 4096, SH 1,
    // 19.1 / 23.5); with few sets eight waves on one block shorten each wave's part of K (1 x 2048 x 10944, NB 1 and 8 waves / NB 2 and 4:
    // 8.1 / 8.8; 1 x 14336 x 4096 gated, NB 2, 8 / 4: 18.8 / 17.9).
    const long long sets = (a.N + 15) / 16 * (long long)units;  // of 16 rows of W
    if (most <= 8) {
      if (sets >= 256) MR_LAUNCH(2, 2, 4);
      else MR_LAUNCH(2, 1, 8);
    } else {
      if (sets >= 512) MR_LAUNCH(1, 2, 4);
      else MR_LAUNCH(1, 1, 4);
    }
#undef MR_LAUNCH
    return moe_check_launch("k_mx4_rows");
  }
  MxArgs t = a;
  const int bm = 64 * pl.wm, nc = 64 * pl.wn / (GATED ? 2 : 1);
  t.nm = a.units ? 0 : (a.M + bm - 1) / bm;
  t.nn = (a.N + nc - 1) / nc;
  // (by expert: whole tiles, and one that is not for each expert at most)
  const long long tiles = (a.units ? a.M / bm + units : t.nm) * (long long)t.nn * pl.splits;
  if (tiles >= 1 << 24) {
    moe_set_error("moe_mx4: %d x %d results are too many for one launch", a.M, a.N);
    return MOE_EINVAL;
  }
  t.splits = pl.splits;
  t.ldp = (a.N + 7) & ~7;
  t.part = pl.splits > 1 ? ws : nullptr;
  constexpr int SLAB_K = X == X_MX4 ? M4_K : M16_K;
  const int slabs = (a.K + SLAB_K - 1) / SLAB_K;
  t.slabs = slabs / pl.splits;
  t.extra = slabs % pl.splits;
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8));
#define MT_LAUNCH(WM_, WN_, RING_)                                                                                                 \
  if constexpr (X == X_MX4) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_mx4_tile<F16, GATED, WM_, WN_, RING_>), grid, dim3(256), 0, s, t); \
  else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_mx4_tile16<X, GATED, WM_, WN_, RING_>), grid, dim3(256), 0, s, t)
  switch (pl.wm * 100 + pl.wn * 10 + pl.ring) {
    case 114: if constexpr (X == X_MX4 && !GATED) { MT_LAUNCH(1, 1, 4); } break;
    case 113: if constexpr (X != X_MX4 && !GATED) { MT_LAUNCH(1, 1, 3); } break;
    case 124: if constexpr (X == X_MX4) { MT_LAUNCH(1, 2, 4); } break;
    case 123: if constexpr (X != X_MX4) { MT_LAUNCH(1, 2, 3); } break;
    case 122: if constexpr (X == X_MX4) { MT_LAUNCH(1, 2, 2); } break;
    case 142: if constexpr (X != X_MX4) { MT_LAUNCH(1, 4, 2); } break;
    case 223: MT_LAUNCH(2, 2, 3); break;
    case 222: if constexpr (X == X_MX4) { MT_LAUNCH(2, 2, 2); } break;
    case 243: MT_LAUNCH(2, 4, 3); break;
    case 442: if constexpr (X == X_MX4) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_mx4_wide<F16, GATED>), grid, dim3(256), 0, s, t); break;
    default: moe_set_error("moe_mx4: no tile %d x %d", pl.wm, pl.wn); return MOE_EINVAL;
  }
#undef MT_LAUNCH
  if (int rc = moe_check_launch("k_mx4_tile")) return rc;
  if (!t.part) return MOE_OK;
  const long long pieces = (long long)a.M * (t.ldp >> 3);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(k_mx4_join<F16, GATED>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, t);
  return moe_check_launch("k_mx4_join");
}
static int mx_run(const MxArgs &a, int xkind, int dtype, bool gated, int units, int most, float *ws, hipStream_t s) {
  const bool f16 = dtype == MOE_DT_FP16;
  switch ((xkind == X_MX4 ? 0 : 4) + (f16 ? 2 : 0) + (gated ? 1 : 0)) {
    case 0: return mx_launch<X_MX4, false, false>(a, units, most, ws, s);
    case 1: return mx_launch<X_MX4, false, true>(a, units, most, ws, s);
    case 2: return mx_launch<X_MX4, true, false>(a, units, most, ws, s);
    case 3: return mx_launch<X_MX4, true, true>(a, units, most, ws, s);
    case 4: return mx_launch<X_BF16, false, false>(a, units, most, ws, s);
    case 5: return mx_launch<X_BF16, false, true>(a, units, most, ws, s);
    case 6: return mx_launch<X_FP16, true, false>(a, units, most, ws, s);
    default: return mx_launch<X_FP16, true, true>(a, units, most, ws, s);
  }
}
static MxArgs mx_args(const void *x, int64_t ldx, const moe_mx4 *xq, const moe_mx4 *w, const moe_mx4 *w_up, const void *bias,
                      const void *bias_up, const void *residual, int64_t ldr, void *y, int64_t ldy, int M, int N, int K, int act, int y_fp32) {
  MxArgs a{};
  a.x = xq ? xq->codes : x;
  a.xs = xq ? (const uint8_t *)xq->scales : nullptr;
  a.ldx = xq ? xq->ldc : ldx < 1ll << 40 ? ldx * 2 : ldx;
  a.w[0] = (const uint8_t *)w->codes; a.ws[0] = (const uint8_t *)w->scales;
  if (w_up) { a.w[1] = (const uint8_t *)w_up->codes; a.ws[1] = (const uint8_t *)w_up->scales; }
  a.ldw = w->ldc; a.ew = w->next_c; a.ews = w->next_s;
  a.bias[0] = (const uint16_t *)bias; a.bias[1] = (const uint16_t *)bias_up; a.res = (const uint16_t *)residual;
  a.y = y; a.ldr = ldr; a.ldy = ldy; a.M = M; a.N = N; a.K = K; a.act = act; a.y32 = y_fp32 != 0;
  return a;
}
// the descriptions themselves
static int mx_described(const char *who, const void *x, const moe_mx4 *xq, const moe_mx4 *w, const moe_mx4 *w_up) {
  if (!w || (x && xq) || (w_up && (w_up->ldc != w->ldc || w_up->next_c != w->next_c || w_up->next_s != w->next_s))) {
    moe_set_error("%s: one x, a matrix, and for a pair a second one laid out like the first", who);
    return MOE_EINVAL;
  }
  return MOE_OK;
}

extern "C" int moe_mx4_linear(const void *x, int64_t ldx, const moe_mx4 *xq, const moe_mx4 *w, const moe_mx4 *w_up, const void *bias,
                              const void *bias_up, const void *residual, int64_t ldr, void *y, int64_t ldy, int M, int N, int K, int dtype,
                              int act, int y_fp32, void *ws, int64_t ws_bytes, void *stream) {
  if (int rc = mx_described("moe_mx4_linear", x, xq, w, w_up)) return rc;
  const MxArgs a = mx_args(x, ldx, xq, w, w_up, bias, bias_up, residual, ldr, y, ldy, M, N, K, act, y_fp32);
  const int xkind = xq ? X_MX4 : dtype == MOE_DT_FP16 ? X_FP16 : X_BF16;
  if (int rc = mx_check("moe_mx4_linear", a, xkind, M, 1, dtype, w_up != nullptr)) return rc;
  if (!M || !N) return MOE_OK;
  const int64_t need = moe_mx4_linear_workspace_bytes(M, N, K, xq != nullptr, w_up != nullptr);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) {
    moe_set_error("moe_mx4_linear: a workspace of %lld bytes on a 16-byte boundary is needed", (long long)need);
    return MOE_EINVAL;
  }
  auto meets = [&](const void *p, int64_t rows, int64_t ld, int64_t len) { return mx_meet(ws, 1, 0, need, p, rows, ld, len); };
  bool shares = meets(y, M, ldy * (a.y32 ? 4 : 2), N * (a.y32 ? 4ll : 2ll)) || meets(a.x, M, a.ldx, xq ? K / 2 : K * 2ll) ||
                meets(residual, M, ldr * 2, N * 2ll) || (xq && meets(a.xs, 1, 0, moe_mx4_scale_bytes(M, K)));
  for (int i = 0; i < (w_up ? 2 : 1); ++i)
    shares = shares || meets(a.w[i], N, a.ldw, K / 2) || meets(a.ws[i], 1, 0, moe_mx4_scale_bytes(N, K)) || meets(a.bias[i], 1, 0, 2ll * N);
  if (shares) {
    moe_set_error("moe_mx4_linear: the workspace overlaps an operand or the result");
    return MOE_EINVAL;
  }
  return mx_run(a, xkind, dtype, w_up != nullptr, 1, M, (float *)ws, (hipStream_t)stream);
}

extern "C" int moe_mx4_experts(const void *x, int64_t ldx, const moe_mx4 *xq, const moe_mx4 *w, const moe_mx4 *w_up, const void *bias,
                               const void *bias_up, void *y, int64_t ldy, const int *counts, const int *offsets, const moe_unit *units,
                               int max_units, const int *sorted_tok, int T, int P, int E, int N, int K, int dtype, int act, int y_fp32,
                               void *stream) {
  if (int rc = mx_described("moe_mx4_experts", x, xq, w, w_up)) return rc;
  MxArgs a = mx_args(x, ldx, xq, w, w_up, bias, bias_up, nullptr, 0, y, ldy, P, N, K, act, y_fp32);
  a.counts = counts; a.offsets = offsets; a.units = units; a.tok = sorted_tok; a.E = E;
  const int xkind = xq ? X_MX4 : dtype == MOE_DT_FP16 ? X_FP16 : X_BF16;
  if (E < 1 || E > 1024 || max_units < (E < P ? E : P) || T < 0 || (P && !T) || (P && N && (!counts || !offsets || !units))) {
    moe_set_error("moe_mx4_experts: bad argument (E=%d T=%d P=%d max_units=%d)", E, T, P, max_units);
    return MOE_EINVAL;
  }
  if (int rc = mx_check("moe_mx4_experts", a, xkind, sorted_tok ? T : P, E, dtype, w_up != nullptr)) return rc;
  auto meets = [&](const void *p, int64_t bytes) { return mx_meet(y, P, ldy * (a.y32 ? 4 : 2), N * (a.y32 ? 4ll : 2ll), p, 1, 0, bytes); };
  if (meets(counts, 4ll * E) || meets(offsets, 4ll * E + 4) || meets(units, (int64_t)sizeof(moe_unit) * max_units) || meets(sorted_tok, 4ll * P)) {
    moe_set_error("moe_mx4_experts: the result overlaps the dispatch");
    return MOE_EINVAL;
  }
  if (sorted_tok && T * a.ldx > LT_OUT) {  // (offsets of gathered rows are those of a buffer resource)
    moe_set_error("moe_mx4_experts: %d rows of tokens %lld bytes apart (less than 2 GiB are needed)", T, a.ldx);
    return MOE_EINVAL;
  }
  if (!P || !N) return MOE_OK;
  return mx_run(a, xkind, dtype, w_up != nullptr, E < P ? E : P, T, nullptr, (hipStream_t)stream);
}
