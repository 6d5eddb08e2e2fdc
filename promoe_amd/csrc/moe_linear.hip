// Products of dense layers (gfx950): y = act(x W^T + b) + residual, and the gated pair y = act(x Wg^T + bg) * (x Wu^T + bu).
// x [M, K], W [N, K] row-major in bf16 or fp16, sums in fp32; bias, activation, product and residual are applied to the
// fp32 sums, which are rounded once, to the type of y.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <type_traits>

#include "moe_common.h"
#include "moe_kernels.h"
#include "moe_device.h"
#include "moe_linear.h"

struct LinArgs {
  const uint16_t *x, *w[2], *bias[2], *res;  // w[1]: the second matrix of a gated pair
  void *y;
  long long ldx, ldw, ldr, ldy;              // elements
  int M, N, K, act, y32;
  int nm, nn;                                // tiles
  int splits, ldp;                           // pieces of K, columns of a row of partial sums
  int slabs, extra;                          // slabs of a piece; the first `extra` pieces have one more
  float *part;                               // partial sums [splits][1 or 2 matrices][M][ldp], NULL: the tile kernel finishes
};

// ---- few rows of x: the matrix streams past them --------------------------------------------------------------------------------
// A workgroup of eight waves takes R = 16 / SH rows of W (gated: of both matrices), its waves the pieces of K in turn; their sums meet
// in LDS.  Weights go from memory into the matrix core's operands: one v_mfma_f32_16x16x32 per 1 KiB.  With SH = 1 the 16 rows of
// the operand are 16 rows of W; with few rows of x (M <= 16 / SH) the operand is R rows of W by SH pieces of K, row s R + r and column
// s R + m hold piece s of both, and the products of unlike pieces are left unread: a smaller unit of work (more workgroups for a
// short matrix) and longer runs of a row per load.
// Bound by HBM: 1 x 2048 x 10944 (45 MB) 10.5 us, 4.3 TB/s; gated 1 x 10944 x 2048 (90 MB) 20.4 us, 4.4 TB/s (a large copy: 5.2).  Twice the
// loads in flight, 16 waves or non-temporal loads are no faster.
#define LR_WAVES 8
#define LR_U 4  // loads of a matrix in flight per wave, twice
template <bool F16, bool GATED, int SH>
__global__ __launch_bounds__(64 * LR_WAVES) void k_linear_rows(const LinArgs a) {
  constexpr int NM = GATED ? 2 : 1, R = 16 / SH, STEP = 32 * SH * LR_U, SPAN = STEP * LR_WAVES;
  __shared__ f32x4_t red[LR_WAVES][NM][64];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = (lane & 15) % R, s = (lane & 15) / R, n0 = blockIdx.x * R;
  const int k0 = 8 * ((lane >> 4) * SH + s);                    // the lane's columns inside 32 SH
  const rsrc_t rx = make_rsrc(a.x, LT_OUT), rw0 = make_rsrc(a.w[0] + n0 * a.ldw, LT_OUT), rw1 = make_rsrc(a.w[GATED ? 1 : 0] + n0 * a.ldw, LT_OUT);
  const int vw = (min(n0 + r, a.N - 1) - n0) * (int)a.ldw * 2;
  const int vx = min(r, a.M - 1) * (int)a.ldx * 2;
  f32x4_t acc[NM] = {};
  uint4 fw[2][NM][LR_U], fx[2][LR_U];
  auto load = [&](int p, int base) {
#pragma unroll
    for (int u = 0; u < LR_U; ++u) {
      const int k = base + 32 * SH * u + k0;
      const bool in = k < a.K;                                  // past the end: zeros on both sides
      fw[p][0][u] = bload16(rw0, in ? vw + 2 * k : LT_OUT, 0);
      if constexpr (GATED) fw[p][1][u] = bload16(rw1, in ? vw + 2 * k : LT_OUT, 0);
      fx[p][u] = bload16(rx, in ? vx + 2 * k : LT_OUT, 0);
    }
  };
  auto use = [&](int p) {
#pragma unroll
    for (int u = 0; u < LR_U; ++u)
#pragma unroll
      for (int i = 0; i < NM; ++i)
        acc[i] = lin_mfma16<F16>(__builtin_bit_cast(u32x4_t, fw[p][i][u]), __builtin_bit_cast(u32x4_t, fx[p][u]), acc[i]);
  };
  load(0, w * STEP);
  for (int base = w * STEP; base < a.K; base += 2 * SPAN) {
    load(1, base + SPAN);
    use(0);
    load(0, base + 2 * SPAN);
    use(1);
  }
#pragma unroll
  for (int i = 0; i < NM; ++i) red[w][i][lane] = acc[i];
  __syncthreads();
  // result (m, n): element n' % 4 of lane 16 (n' / 4) + m', n' = s R + n and m' = s R + m, over the pieces and the waves in order
  for (int t = tid; t < R * a.M; t += 64 * LR_WAVES) {
    const int n = t % R, m = t / R;
    if (n0 + n >= a.N) continue;
    float sum[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      sum[i] = 0.f;
#pragma unroll
      for (int p = 0; p < SH; ++p) {
        const int row = p * R + n;
#pragma unroll
        for (int v = 0; v < LR_WAVES; ++v) sum[i] += ((const float *)&red[v][i][16 * (row >> 2) + p * R + m])[row & 3];
      }
    }
    lin_store<F16, GATED>(a, m, n0 + n, sum[0], sum[NM - 1]);
  }
}

// ---- tile kernel --------------------------------------------------------------------------------------------------------------
// Four waves (2 x 2), wave (wm, wn) on WM x WN blocks of 32 x 32: a tile of 64 WM rows of x by 64 WN rows of W.  A gated pair's W
// blocks alternate between the two matrices (block b: matrix b & 1, its columns 32 (b >> 1) ..), so that a lane holds both sums
// of a column.  K advances 64 at a time (a slab); slabs go global -> LDS directly, RING of them in LDS.
// A slab costs 192 (WM + WN) cycles of LDS for 128 WM WN of products; with few workgroups about half of the time is that, the rest the
// launch's start, the ring's fill, a barrier a slab and the epilogue: 24 x 4096 x 4096 9.9 us and 3.8 for the join; with matrices from the last cache 512 x 4096 x 4096 25.0 (687 TFLOP/s), gated 251 x 2560 x 3584 19.1 (482), 1024 x 4096 x 4096 38.1 (902);
// from memory 31.6, 28.6 and 44.1.
#define LT_K 64
#define LT_ROW 128  // bytes of a row of a slab: 8 chunks of 16, chunk c of row r in slot c ^ ((r >> 1) & 7)
template <bool F16>
static __device__ __forceinline__ f32x16_t lin_mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <bool F16, bool GATED, int WM, int WN, int RING>
__global__ __launch_bounds__(256, RING * (WM + WN) * 64 * LT_ROW > 80 * 1024 ? 1 : 2) void k_linear_tile(const LinArgs a) {
  constexpr int BM = 64 * WM, BN = 64 * WN, NX = 2 * WM, NW = 2 * WN, SLAB = (BM + BN) * LT_ROW, NG = WM * WN;
  __shared__ __align__(128) unsigned char s_ring[RING * SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w & 1, wn = w >> 1;
  const int fr = lane & 31, q = lane >> 5;
  int mt, nt, split;
  {  // workgroup i runs on XCD i % 8: each XCD takes a contiguous run of tiles, four rows of tiles wide
    const int per = (int)gridDim.x >> 3;
    int b = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (b >= a.nm * a.nn * a.splits) return;
    split = b / (a.nm * a.nn);
    b -= split * a.nm * a.nn;
    const int group = b / (4 * a.nn), r = b - group * 4 * a.nn, rows = min(4, a.nm - 4 * group);
    mt = 4 * group + r % rows;
    nt = r / rows;
  }
  constexpr int NC = GATED ? BN / 2 : BN;  // columns of the result
  const int m0 = mt * BM, n0 = nt * NC;
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)s_ring;
  // transfer t of wave w: rows 32 t + 8 w .. + 7, eight lanes a row; the lanes choose the chunk that belongs in their slot
  const int tr = 8 * w + (lane >> 3), chunk = (lane & 7) ^ ((tr >> 1) & 7);
  const lt_rsrc_t rx = lt_rsrc(a.x + m0 * a.ldx), rw0 = lt_rsrc(a.w[0] + n0 * a.ldw), rw1 = lt_rsrc(a.w[GATED ? 1 : 0] + n0 * a.ldw);
  int vx[NX], vw[NW];
#pragma unroll
  for (int t = 0; t < NX; ++t) vx[t] = (min(m0 + 32 * t + tr, a.M - 1) - m0) * (int)a.ldx * 2 + 16 * chunk;
#pragma unroll
  for (int t = 0; t < NW; ++t) vw[t] = (min(n0 + 32 * (GATED ? t >> 1 : t) + tr, a.N - 1) - n0) * (int)a.ldw * 2 + 16 * chunk;
  const int kt0 = split * a.slabs + min(split, a.extra), nk = kt0 + a.slabs + (split < a.extra);
  const int k_end = min(a.K, nk * LT_K);
  auto dma = [&](int t, int kt, int place) {  // place: where in the ring the rows of x (t < NX), of W, begin
    // (assembly: told that a load writes LDS, the compiler would wait for all of them in front of every barrier and LDS read;
    // the waits stand by hand.  Columns past the end, slabs past the last among them, are out of the resource's range: zeros.)
    const bool in = kt * LT_K + 8 * chunk < k_end;
    const unsigned at = lds + (unsigned)(place + ((t < NX ? t : t - NX) * 32 + 8 * w) * LT_ROW);
    const int off = in ? (t < NX ? vx[t < NX ? t : 0] : vw[t < NX ? 0 : t - NX]) : LT_OUT;
    const lt_rsrc_t rs = t < NX ? rx : (GATED && ((t - NX) & 1)) ? rw1 : rw0;
    __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :: "s"(at), "v"(off), "s"(rs), "s"(kt * (LT_K * 2)) : "memory", "m0");
  };
  unsigned ax[4], aw[4];  // LDS address of the lane's fragment of step j in block 0, of rows that begin where the ring does
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned c = (unsigned)(((4 * q + j) ^ ((fr >> 1) & 7)) * 16);
    ax[j] = lds + (unsigned)((wm * WM * 32 + fr) * LT_ROW) + c;
    aw[j] = lds + (unsigned)((wn * WN * 32 + fr) * LT_ROW) + c;
  }
  typedef __attribute__((address_space(3))) const u32x4_t lds_u4;
  unsigned cx[4], cw[4];  // and of the current slab
  auto use = [&](int place_x, int place_w) {
#pragma unroll
    for (int j = 0; j < 4; ++j) { cx[j] = ax[j] + (unsigned)place_x; cw[j] = aw[j] + (unsigned)place_w; }
  };
  auto read_x = [&](int j, int i) { return *(lds_u4 *)(uintptr_t)(cx[j] + (unsigned)(i * 32 * LT_ROW)); };
  auto read_w = [&](int j, int i) { return *(lds_u4 *)(uintptr_t)(cw[j] + (unsigned)(i * 32 * LT_ROW)); };
  f32x16_t acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int b = 0; b < WN; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][b][e] = 0.f;
  // A slab's products are short here, a step of them shorter than an LDS read: the fragments of the whole next slab are read
  // between this one's.  At the barrier everybody has this slab's fragments, so its slot is free, and the next has landed.
#pragma unroll
  for (int i = 0; i < RING; ++i)
#pragma unroll
    for (int t = 0; t < NX + NW; ++t) dma(t, kt0 + i, i * SLAB + (t < NX ? 0 : BM * LT_ROW));
  LT_VM((RING - 1) * (NX + NW));
  __builtin_amdgcn_s_barrier();
  use(0, BM * LT_ROW);
  u32x4_t fx[2][4][WM], fw[2][4][WN];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int i = 0; i < WM; ++i) fx[0][j][i] = read_x(j, i);
#pragma unroll
    for (int i = 0; i < WN; ++i) fw[0][j][i] = read_w(j, i);
  }
  int slot = 0;
  auto step = [&](const u32x4_t(&x)[4][WM], const u32x4_t(&v)[4][WN], u32x4_t(&xn)[4][WM], u32x4_t(&vn)[4][WN], int kt) {
    const int next = slot + 1 < RING ? slot + 1 : 0;
    LT_LGKM0();
    LT_VM((RING - 2) * (NX + NW));
    __builtin_amdgcn_s_barrier();
    use(next * SLAB, next * SLAB + BM * LT_ROW);
    __builtin_amdgcn_sched_barrier(0);
    constexpr int NP = 4 * NG, NR = 4 * (WM + WN), ND = NX + NW;
#pragma unroll
    for (int g = 0; g < NP; ++g) {
      const int j = g / NG, i = g % NG / WN, b = g % WN;
#pragma unroll
      for (int r = 0; r < NR; ++r)
        if (r * NP / NR == g) {
          const int rj = r / (WM + WN), ri = r % (WM + WN);
          if (ri < WM) xn[rj][ri] = read_x(rj, ri);
          else vn[rj][ri - WM] = read_w(rj, ri - WM);
        }
#pragma unroll
      for (int t = 0; t < ND; ++t)
        if (t * NP / ND == g) dma(t, kt + RING, slot * SLAB + (t < NX ? 0 : BM * LT_ROW));
      __builtin_amdgcn_sched_barrier(0);
      acc[i][b] = lin_mfma32<F16>(v[j][b], x[j][i], acc[i][b]);
      __builtin_amdgcn_sched_barrier(0);
    }
    slot = next;
  };
  // (always a pair of slabs: one past the end is zeros)
  for (int kt = kt0; kt < nk; kt += 2) {
    step(fx[0], fw[0], fx[1], fw[1], kt);
    step(fx[1], fw[1], fx[0], fw[0], kt + 1);
  }
  // The sums leave through LDS, 32 rows of the wave at a time, so that a lane then has 8 adjacent columns of a row and the rest is
  // one loop of whole lines.  Element e of a lane: column 8 (e / 4) + 4 q + e % 4 of W's block, row fr of x's.
  LT_VM(0);
  __syncthreads();
  constexpr int LDE = 32 * WN + 4;                       // floats between rows: 16 lanes that write 16 bytes each fall on all banks
  constexpr int LPR = NC / 16, RPP = 64 / LPR;           // lanes of a row (8 columns each), rows of a pass
  static_assert(4 * 32 * LDE * 4 <= RING * SLAB, "the sums of four waves fit the ring");
  float *buf = (float *)s_ring + w * 32 * LDE;
  const int col = 8 * (lane % LPR), n = n0 + wn * (NC / 2) + col;
  const int at = GATED ? (col >> 5) * 64 + (col & 31) : col;
  const LinColumns<F16, GATED> c(a, n);
  // (one copy of the loop for all blocks: code that runs once a tile waits for its instructions, line by line)
#pragma clang loop unroll(disable)
  for (int i = 0; i < WM; ++i) {
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
    const int first = m0 + 32 * (wm * WM + i) + lane / LPR;
    u32x4_t res = c.residual(a, first);
#pragma clang loop unroll(disable)
    for (int r = lane / LPR; r < 32; r += RPP) {
      const int m = first - lane / LPR + r;
      const u32x4_t ahead = c.residual(a, r + RPP < 32 ? m + RPP : a.M);
      if (m < a.M) {
        if (a.part) c.partial(a, split, m, buf + r * LDE + at, buf + r * LDE + at + 32);
        else c.store(a, m, buf + r * LDE + at, buf + r * LDE + at + 32, res);
      }
      res = ahead;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- wide tiles: 256 x 256, one workgroup per compute unit that goes from tile to tile -------------------------------------------------
// Four waves (2 x 2), each on 8 x 8 blocks of 16 x 16.  A slab (64 columns) is two steps of 64 products v_mfma_f32_16x16x32: a step covers
// an LDS read many times, so the fragments of the next step are read between its products.  (At this size the card is at its power
// limit, and what counts is the energy of a product: the 32 x 32 x 16 form reads and writes twice the sums per product of two values.)
// LDS has room for two slabs and a half: a ring of five halves, x and W of a slab in turn (half h of the run in place h % 5).  The loop
// turns at a barrier in front of step 1 of slab g - 1, whose fragments are that slab's last: everybody has read slab g - 1 then, and
// slab g has landed.  In that step the wave's transfers of W of slab g + 1 go out (where x of slab g - 1 was), in step 0 of slab g those
// of x of slab g + 2 (where its W was).  Evenly, since 64 bytes per cycle and compute unit is all that the path takes, half of the time
// that the products of a slab need: all 16 of a wave at once stopped the products for as long again (59 % busy matrix cores, then 74).
// The run of slabs goes on from tile to tile: the next tile's first slab and the W half behind it land under the last products, and the
// sums leave through the one place that nothing else needs then.
// Bound by power: 4096 x 4096 x 14336 328 to 350 us on different cards (1370 to 1470 TFLOP/s, 73 % busy matrix cores at 1.75 to 1.9 GHz; the
// library's product 305 - 315), gated 4096 x 14336 x 4096 657 to 707 us (the library's of both matrices, no gate, 622 - 640); the first launches
// after a pause up to 408 and 730.
template <bool F16, bool GATED>
__global__ __launch_bounds__(256, 1) void k_linear_wide(const LinArgs a) {
  constexpr int B = 256, NT = 8, HALF = B * LT_ROW, NC = GATED ? B / 2 : B;
  __shared__ __align__(1024) unsigned char s_ring[5 * HALF];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w & 1, wn = w >> 1;
  const int fr = lane & 15, q = lane >> 4;
  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)s_ring;
  // workgroup i runs on XCD i % 8: each XCD takes a contiguous run of tiles, four rows of tiles wide
  const int tiles = a.nm * a.nn, stride = (int)gridDim.x >> 3;
  const int per = (tiles * a.splits + 7) >> 3, last = min(tiles * a.splits, ((int)(blockIdx.x & 7) + 1) * per);
  struct Tile { int m0, n0, split, kt0, kt1; };  // kt1 0: none
  auto tile_of = [&](int v) {
    if (v >= last) return Tile{0, 0, 0, 0, 0};
    const int split = v / tiles, b = v - split * tiles, group = b / (4 * a.nn), r = b - group * 4 * a.nn, rows = min(4, a.nm - 4 * group);
    const int nt = r / rows, mt = 4 * group + r - nt * rows, kt0 = split * a.slabs + min(split, a.extra);
    // (scalars, whatever the divisions are made of)
    return Tile{__builtin_amdgcn_readfirstlane(mt) * B, __builtin_amdgcn_readfirstlane(nt) * NC, __builtin_amdgcn_readfirstlane(split),
                __builtin_amdgcn_readfirstlane(kt0), __builtin_amdgcn_readfirstlane(kt0 + a.slabs + (split < a.extra))};
  };
  int v = (int)(blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (v >= last) return;
  Tile cur = tile_of(v), nxt = tile_of(v + stride);
  // transfer t of wave w: rows 32 t + 8 w .. + 7, eight lanes a row; the lanes choose the chunk that belongs in their slot
  const int tr = 8 * w + (lane >> 3), chunk = (lane & 7) ^ ((tr >> 1) & 7);
  // x and W each have a cursor: the slab that their next transfers bring, of this tile or of the next.  A tile has at least two slabs.
  // Columns past K, and everything past the last tile, are out of the resource's range: zeros.
  int vx[NT], vw[NT], kx, kw, end_x, end_w;
  lt_rsrc_t rx, rw0, rw1{};
  auto start_x = [&](const Tile &t) {
    kx = t.kt0; end_x = t.kt1;
    rx = lt_rsrc(a.x + t.m0 * a.ldx);
#pragma unroll
    for (int i = 0; i < NT; ++i) vx[i] = (min(t.m0 + 32 * i + tr, a.M - 1) - t.m0) * (int)a.ldx * 2 + 16 * chunk;
  };
  auto start_w = [&](const Tile &t) {
    kw = t.kt0; end_w = t.kt1;
    rw0 = lt_rsrc(a.w[0] + t.n0 * a.ldw);
    if constexpr (GATED) rw1 = lt_rsrc(a.w[1] + t.n0 * a.ldw);
#pragma unroll
    for (int i = 0; i < NT; ++i) vw[i] = (min(t.n0 + 32 * (GATED ? i >> 1 : i) + tr, a.N - 1) - t.n0) * (int)a.ldw * 2 + 16 * chunk;
  };
  // what a slab's transfers need beyond the slab before: the next tile's rows, or the lanes past K left out (a slab that ends past K is its
  // tile's last)
  auto leave_out = [&](int (&o)[NT], bool all, int k) {
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = all || k * LT_K + 8 * chunk >= a.K ? LT_OUT : o[i];
  };
  auto turn_x = [&]() {
    if (kx == end_x) { if (nxt.kt1) start_x(nxt); else { end_x = 0; leave_out(vx, true, 0); } }
    if (kx * LT_K + LT_K > a.K) leave_out(vx, false, kx);
  };
  auto turn_w = [&]() {
    if (kw == end_w) { if (nxt.kt1) start_w(nxt); else { end_w = 0; leave_out(vw, true, 0); } }
    if (kw * LT_K + LT_K > a.K) leave_out(vw, false, kw);
  };
  // (assembly: see k_linear_tile)
  auto send = [&](int off, const lt_rsrc_t rs, int kt, int to, auto t) {
    __asm__ volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :: "s"(to), "v"(off), "s"(rs), "s"(kt * (LT_K * 2)), "i"(decltype(t)::value * 32 * LT_ROW)
                     : "memory", "m0", "scc");
  };
  const int mine = (int)lds + 8 * w * LT_ROW;  // the wave's rows in a half
  auto send_x = [&](auto t, int h) { send(vx[t], rx, kx, mine + h * HALF, t); };
  auto send_w = [&](auto t, int h) { send(vw[t], GATED && (t & 1) ? rw1 : rw0, kw, mine + h * HALF, t); };
  unsigned ax[2], aw[2], cx[2], cw[2];  // LDS address of the lane's fragment of step j in block 0: in place 0, and of the slab in use
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const unsigned c = (unsigned)(((4 * j + q) ^ ((fr >> 1) & 7)) * 16);
    ax[j] = lds + (unsigned)((wm * 128 + fr) * LT_ROW) + c;
    aw[j] = lds + (unsigned)((wn * 128 + fr) * LT_ROW) + c;
  }
  auto use = [&](int hx, int hw) {
    int px = hx * HALF, pw = hw * HALF;
    __asm__ volatile("" : "+s"(px), "+s"(pw));  // (here, and not in front of the slab's first product)
#pragma unroll
    for (int j = 0; j < 2; ++j) { cx[j] = ax[j] + (unsigned)px; cw[j] = aw[j] + (unsigned)pw; }
  };
  typedef __attribute__((address_space(3))) u32x4_t lds_u4;
  f32x4_t acc[8][8];
  u32x4_t fx[2][8], fw[2][8];
  // fragment r of a step in the order of need: x's first block, W's, the rest of x's
  auto read = [&](int r, int j) {
    if (r == 0) fx[j][0] = *(lds_u4 *)(uintptr_t)cx[j];
    else if (r <= 8) fw[j][r - 1] = *(lds_u4 *)(uintptr_t)(cw[j] + (unsigned)((r - 1) * 16 * LT_ROW));
    else fx[j][r - 8] = *(lds_u4 *)(uintptr_t)(cx[j] + (unsigned)((r - 8) * 16 * LT_ROW));
  };
  start_x(cur);
  start_w(cur);
  lt_each<NT>([&](auto t) { send_x(t, 0); });
  ++kx;
  lt_each<NT>([&](auto t) { send_w(t, 1); });
  ++kw;
  turn_x();
  lt_each<NT>([&](auto t) { send_x(t, 2); });
  ++kx;
  use(0, 1);
  int h = 3;  // place of W of the next slab
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < 64; ++i) acc[i >> 3][i & 7] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  };
  // products of step j; between them the reads of the other step and eight transfers
  auto step = [&](auto j_, auto transfer) {
    constexpr int j = decltype(j_)::value;
    __builtin_amdgcn_sched_barrier(0);
    lt_each<64>([&](auto g_) {
      constexpr int g = decltype(g_)::value;
      acc[g >> 3][g & 7] = lin_mfma16<F16>(fw[j][g & 7], fx[j][g >> 3], acc[g >> 3][g & 7]);
      __builtin_amdgcn_sched_barrier(0);
      // (in front of the barrier the reads have to be over: those of step 1 come in the first half of step 0)
      if constexpr (j == 0) { if constexpr (g % 2 == 0 && g < 32) read(g / 2, 1); }
      else if constexpr (g % 4 == 0) read(g / 4, 0);
      if constexpr (g % 8 == 3) transfer(std::integral_constant<int, g / 8>());
      if constexpr (j == 0 && g == 36) use(h >= 1 ? h - 1 : 4, h);  // the next slab's addresses, behind this one's last read
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  clear();
#pragma unroll
  for (int i = 0; i < 8; ++i) fx[1][i] = fw[1][i] = u32x4_t{0, 0, 0, 0};  // (step 1 in front of the first slab: products of zeros)
  int left = cur.kt1 - cur.kt0;  // slabs of the tile ahead
  for (;;) {
    turn_w();
    LT_LGKM0();
    LT_VM(NT);  // (x of the slab after next may be on its way)
    __builtin_amdgcn_s_barrier();
    step(std::integral_constant<int, 1>(), [&](auto t) { send_w(t, h); });
    ++kw;
    const int h1 = h + 1 < 5 ? h + 1 : 0;
    if (left == 0) {
      // 16 rows of the wave at a time through the kilobytes of place h1 that its own transfers will fill, so that a lane then has 8
      // adjacent columns of a row and the rest works on whole lines.  Element e of a lane: column 4 q + e of W's block, row fr of x's;
      // chunk c (four columns) of row r stands in place c ^ r of the row's 512 bytes.
      constexpr int LPR = NC / 16, RPP = 64 / LPR, NP = 16 / RPP;  // lanes of a row (8 columns each), rows of a pass, passes
      const int lr = lane / LPR, col = 8 * (lane % LPR), at = GATED ? (col >> 5) * 16 + ((col & 31) >> 2) : col >> 2;
      unsigned put = (unsigned)(mine + h1 * HALF + (fr >> 1) * 32 * LT_ROW + (fr & 1) * 512 + (q ^ fr) * 16);
      unsigned get = (unsigned)(mine + h1 * HALF + (lr >> 1) * 32 * LT_ROW + (lr & 1) * 512 + (at ^ lr) * 16);
      // pass p of a lane: row lr + RPP p; chunk k of its four (two: columns, gated the second two: of the second matrix)
      auto fetch = [&](int p, float (&s0)[8], float (&s1)[8]) {
#pragma unroll
        for (int k = 0; k < (GATED ? 4 : 2); ++k) {
          const int x = (RPP * p) ^ (k & 1) ^ (k >> 1) * 8;
          const unsigned from = (get ^ (unsigned)(16 * x)) + (unsigned)(p * (RPP / 2) * 32 * LT_ROW);
          const f32x4_t f = __builtin_bit_cast(f32x4_t, *(lds_u4 *)(uintptr_t)from);
#pragma unroll
          for (int e = 0; e < 4; ++e) (k >> 1 ? s1 : s0)[4 * (k & 1) + e] = f[e];
        }
      };
      const int n = cur.n0 + wn * (NC / 2) + col, row0 = cur.m0 + wm * 128 + lr;
      const LinColumns<F16, GATED> c(a, n);
      // (one copy of the passes for all eight blocks: code that runs once a tile waits for its instructions, line by line)
      auto blocks = [&](auto rows) {
#pragma clang loop unroll(disable)
        for (int i = 0; i < 8; ++i) {
          __asm__ volatile("" : "+v"(put), "+v"(get));  // (the addresses that follow from them are not kept over the blocks)
          lt_each<8>([&](auto i_) {
            if (i == decltype(i_)::value) {
#pragma unroll
              for (int b = 0; b < 8; ++b)
                *(lds_u4 *)(uintptr_t)(put ^ (unsigned)(16 * 4 * b)) = __builtin_bit_cast(u32x4_t, acc[decltype(i_)::value][b]);
              __asm__ volatile("; %0" :: "i"(decltype(i_)::value));  // (or the compiler makes one copy of the eight, over registers chosen by i)
            }
          });
          __builtin_amdgcn_wave_barrier();
          rows(row0 + 16 * i);
          __builtin_amdgcn_wave_barrier();
        }
      };
      const bool inside = !a.y32 && !a.part && cur.m0 + B <= a.M && cur.n0 + NC <= a.N;
      // a tile inside the result: no conditions, addresses by addition, the activation chosen once
      auto plain = [&](int m, auto act_) {
        const uint16_t *pr = GATED || !a.res ? nullptr : a.res + m * a.ldr + n;
        uint16_t *py = (uint16_t *)a.y + m * a.ldy + n;
        u32x4_t res[NP];
        if (!GATED && a.res)
#pragma unroll
          for (int p = 0; p < NP; ++p) res[p] = *(const u32x4_any *)(pr + p * RPP * a.ldr);
        float s0[2][8], s1[2][8];
        fetch(0, s0[0], s1[0]);
#pragma unroll
        for (int p = 0; p < NP; ++p) {  // (one pass read ahead and no more: the compiler counts on registers that the sums have)
          __builtin_amdgcn_sched_barrier(0);
          if (p + 1 < NP) fetch(p + 1, s0[(p + 1) & 1], s1[(p + 1) & 1]);
          c.template finish<decltype(act_)::value>(s0[p & 1], s1[p & 1]);
          if (!GATED && a.res) lin_add<F16>(s0[p & 1], res[p]);
          *(u32x4_any *)(py + p * RPP * a.ldy) = lin_pack<F16>(s0[p & 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      blocks([&](int m) {
        switch (inside ? a.act : -1) {
          case MOE_ACT_NONE: plain(m, std::integral_constant<int, MOE_ACT_NONE>()); break;
          case MOE_ACT_SILU: plain(m, std::integral_constant<int, MOE_ACT_SILU>()); break;
          case MOE_ACT_GELU: plain(m, std::integral_constant<int, MOE_ACT_GELU>()); break;
          case MOE_ACT_GELU_TANH: plain(m, std::integral_constant<int, MOE_ACT_GELU_TANH>()); break;
          case MOE_ACT_RELU: plain(m, std::integral_constant<int, MOE_ACT_RELU>()); break;
          case MOE_ACT_RELU2: plain(m, std::integral_constant<int, MOE_ACT_RELU2>()); break;
          default: {
            LinColumns<F16, GATED> c1 = c;
            __asm__ volatile("" : "+v"(c1.n), "+v"(c1.count));  // (what follows from them is not kept in registers over the blocks)
            u32x4_t res = c1.residual(a, m);
#pragma clang loop unroll(disable)
            for (int p = 0; p < NP; ++p) {
              const u32x4_t ahead = c1.residual(a, p + 1 < NP ? m + (p + 1) * RPP : a.M);
              float s0[8], s1[8];
              fetch(p, s0, s1);
              if (m + p * RPP < a.M) {
                if (a.part) c1.partial(a, cur.split, m + p * RPP, s0, s1);
                else c1.store(a, m + p * RPP, s0, s1, res);
              }
              res = ahead;
            }
          }
        }
      });
      if (nxt.kt1 == 0) break;
      v += stride;
      cur = nxt;
      nxt = tile_of(v + stride);
      left = cur.kt1 - cur.kt0;
      LT_LGKM0();  // (the wave's reads of its places are over)
      clear();
    }
    turn_x();
    --left;
    step(std::integral_constant<int, 0>(), [&](auto t) { send_x(t, h1); });
    ++kx;
    h = h1 + 1 < 5 ? h1 + 1 : 0;
  }
  LT_VM(0);  // nothing of this workgroup's is on its way into LDS when it ends
}

// The pieces of K added in their order, then what the tile kernel does behind its sums
template <bool F16, bool GATED>
__global__ __launch_bounds__(256) void k_linear_join(const LinArgs a) {
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

// ---- entry points -------------------------------------------------------------------------------------------------------------
// Does the result share a byte with p's `rows` rows of `len` bytes, `ld` bytes apart?  (Rows side by side in one buffer do not; rows of
// different distances whose ranges meet are taken to.)
static bool lin_shares(const LinArgs &a, const void *p, long long rows, long long ld, long long len) {
  if (!p) return false;
  const long long e = a.y32 ? 4 : 2, ldy = a.ldy * e, ny = a.N * e;
  const intptr_t y = (intptr_t)a.y, q = (intptr_t)p;
  if (y + (a.M - 1) * ldy + ny <= q || q + (rows - 1) * ld + len <= y) return false;
  if (ldy != ld) return true;
  const long long d = ((y - q) % ld + ld) % ld;
  return d < len || d + ny > ld;
}
static int lin_check(const char *who, const LinArgs &a, int dtype, bool gated) {
  const bool empty = a.M == 0 || a.N == 0;
  if (a.M < 0 || a.N < 0 || a.K <= 0 || a.K % 8 || (dtype != MOE_DT_BF16 && dtype != MOE_DT_FP16) || a.act < MOE_ACT_NONE ||
      a.act > MOE_ACT_RELU2 || a.ldx < a.K || a.ldx % 8 || a.ldw < a.K || a.ldw % 8 || a.ldy < a.N || (a.res && a.ldr < a.N) ||
      a.ldx >= 1 << 21 || a.ldw >= 1 << 21 || a.M > 1 << 26 || a.N > 1 << 26) {
    moe_set_error("%s: bad shape (M=%d N=%d K=%d dtype=%d act=%d, rows %lld %lld %lld %lld elements apart)", who, a.M, a.N, a.K, dtype,
                  a.act, a.ldx, a.ldw, a.res ? a.ldr : 0, a.ldy);
    return MOE_EINVAL;
  }
  if (!empty && (!a.x || !a.w[0] || (gated && !a.w[1]) || !a.y || ((uintptr_t)a.x | (uintptr_t)a.w[0] | (uintptr_t)a.w[1]) & 15)) {
    moe_set_error("%s: operands must be present, x and the matrices on 16-byte boundaries", who);
    return MOE_EINVAL;
  }
  const bool in_place = a.res == a.y && !a.y32 && (a.ldr == a.ldy || a.M == 1);
  if (!empty && (lin_shares(a, a.x, a.M, a.ldx * 2, a.K * 2ll) || lin_shares(a, a.w[0], a.N, a.ldw * 2, a.K * 2ll) ||
                 lin_shares(a, a.w[1], a.N, a.ldw * 2, a.K * 2ll) || lin_shares(a, a.bias[0], 1, a.N * 2ll, a.N * 2ll) ||
                 lin_shares(a, a.bias[1], 1, a.N * 2ll, a.N * 2ll) || (!in_place && lin_shares(a, a.res, a.M, a.ldr * 2, a.N * 2ll)))) {
    moe_set_error("%s: the result overlaps an operand (only a residual may be the result itself)", who);
    return MOE_EINVAL;
  }
  return MOE_OK;
}

// Which kernel a product takes: few rows (wm 0), or tiles of 64 wm x 64 wn with `ring` slabs in LDS (4 x 4: the wide kernel) and K in
// `splits` pieces.  The plan of the least time after a model of one launch, us, fitted to 8758 measured times of 160 shapes (24 to 4096
// rows; matrices from memory and from the last cache; the chosen plan is 0.9 % slower than the best of all on average, 19 % at worst):
//   rounds x (slabs x (c0 + c1 x share of the compute units in use) + f),  with pieces 1.6 + 0.43 a piece + 0.15 per MB of partial sums
// c0, c1: a slab of a workgroup on an idle chip, and what the others' traffic adds; f: start and epilogue.  The narrow tiles are bound by
// LDS (192 (wm + wn) cycles a slab for 128 wm wn of products), the wide one by the matrix cores, at the power limit.
// us with matrices from memory, best other tile / chosen: 64 x 4096 x 4096 16.4 / 13.9 (64 x 64, 4 pieces), 512 x 4096 x 4096 32.8 / 31.6 (64 x 128), 1024 x 4096 x
// 4096 48.3 / 44.1 (128 x 128), 384 x 2048 x 10944 38.1 / 35.0 (128 x 128, 5 pieces), 2048 x 4096 x 4096 78.8 / 67.9 (128 x 256), 1536 x 2048 x
// 10944 90.4 / 81.5 (256 x 256, 5 pieces); gated 128 x 14336 x 4096 66.1 / 57.4 (128 x 128), 2048 x 10944 x 2048 205 / 166 (256 x 256).
// Few rows, us, k_linear_rows / best tile: 3 x 2048 x 10944 13.4 / 14.8, 8 x 4096 x 4096 11.2 / 11.5, 16 x 4096 x 4096 10.7 / 11.6, 8 x 2048 x
// 1408 4.9 / 7.4, 16 x 2048 x 1408 6.0 / 7.4; past 8 rows a long reduction is faster on tiles in pieces (every workgroup reads all of x,
// which no longer passes unnoticed beside the weights): 12 x 2048 x 10944 23.0 / 15.5, 16 x 4096 x 14336 37.7 / 27.9, and past 16 the tiles
// are in general: 24 x 4096 x 4096 13.3 / 12.0, 24 gated 14336 x 4096 69 / 51.
struct LinTile { int wm, wn, ring, per_cu; float c0, c1, f; };
static const LinTile LIN_TILES[] = {{1, 1, 4, 2, 0.173f, 0.129f, 0.13f}, {1, 2, 6, 1, 0.233f, 0.139f, 1.38f}, {2, 2, 4, 1, 0.380f, 0.245f, 2.27f},
                                    {2, 4, 3, 1, 0.636f, 0.221f, 4.34f}, {4, 4, 5, 1, 1.176f, 0.f, 9.52f}};
static float lin_us(const LinTile &t, int M, int N, int K, bool gated, long long n, int s) {
  const long long slabs = (K + LT_K - 1) / LT_K, wgs = n * s, rounds = (wgs + 256 * t.per_cu - 1) / (256 * t.per_cu);
  const float use = wgs > 256 ? (float)t.per_cu : (float)wgs / 256.f;  // (one compute unit with two workgroups is what a launch waits for)
  const float us = (float)rounds * ((float)((slabs + s - 1) / s) * (t.c0 + t.c1 * use) + t.f);
  return s == 1 ? us : us + 1.6f + 0.43f * (float)s + 0.151e-6f * 8.f * (float)s * (gated ? 2.f : 1.f) * (float)M * (float)N;
}
struct LinPlan { int wm, wn, ring, splits; float us; };
static LinPlan lin_plan(int M, int N, int K, bool gated) {
  if (M <= 8 || (M <= 16 && K <= 4096)) return LinPlan{0, 0, 0, 1, 2.5f + 0.6e-6f * (gated ? 2.f : 1.f) * (float)N * (float)K};
  static const int pieces[] = {1, 2, 3, 4, 5, 6, 8, 12, 16};
  const long long slabs = (K + LT_K - 1) / LT_K;
  LinPlan best{2, 2, 4, 1, 1e30f};
  for (const LinTile &t : LIN_TILES) {
    if (gated && t.wn == 1) continue;  // (a pair needs both matrices' blocks in a wave)
    const int cols = 64 * t.wn / (gated ? 2 : 1);
    const long long n = ((long long)M + 64 * t.wm - 1) / (64 * t.wm) * (((long long)N + cols - 1) / cols);
    for (int s : pieces) {
      if (s > slabs || (s > 1 && n * s > 640) || (t.wm == 4 && slabs < 2 * s)) break;
      const float us = lin_us(t, M, N, K, gated, n, s);
      if (us < best.us) best = LinPlan{t.wm, t.wn, t.ring, s, us};
    }
  }
  return best;
}
// Where a product is cut in two launches: the large tiles that fill the chip whole rounds through, and the columns (or rows) behind them
// on tiles of their own, instead of a last round of a few (3 us: the second launch).  us, one launch / two: 4097 x 4096 x 4096 174 / 117,
// 1184 x 13760 x 2112 111 / 85, gated 768 x 10944 x 2048 97 / 71, 1300 x 10944 x 2048 137 / 125, 768 x 14336 x 4096 183 / 167.
struct LinCut { int M, N; };  // size of the first part
static LinCut lin_cut(int M, int N, int K, bool gated) {
  LinCut cut{M, N};
  const int half = gated ? 2 : 1;
  if (((long long)M + 127) / 128 * (((long long)N + 256 / half - 1) / (256 / half)) <= 256) return cut;
  float least = lin_plan(M, N, K, gated).us;
  for (const LinTile &t : LIN_TILES) {
    if (t.wn != 4) continue;
    const int cols = 256 / half, rows = 64 * t.wm;
    const long long nm = ((long long)M + rows - 1) / rows, nn = ((long long)N + cols - 1) / cols, full = nm * nn / 256 * 256;
    if (full == 0 || full == nm * nn || (t.wm == 4 && K <= LT_K)) continue;
    auto consider = [&](long long am, long long an) {
      if (am < 1 || an < 1 || am > nm || an > nn || (am == nm && an == nn)) return;
      const int m = am == nm ? M : (int)am * rows, n = an == nn ? N : (int)an * cols;
      const float us = 3.f + lin_us(t, m, n, K, gated, am * an, 1) + lin_plan(m < M ? M - m : M, n < N ? N - n : N, K, gated).us;
      if (us < least) { least = us; cut = LinCut{m, n}; }
    };
    consider(nm, full / nm);
    consider(full / nn, nn);
  }
  return cut;
}

template <bool F16, bool GATED>
static int lin_launch(const LinArgs &a, float *ws, hipStream_t s) {
  constexpr int NM = GATED ? 2 : 1;
  LinArgs t = a;
  const LinPlan pl = lin_plan(a.M, a.N, a.K, GATED);
  if (pl.wm == 0) {
    // rows of x in the operand beside pieces of K: more workgroups where 16 rows of W each would be fewer than two per compute unit
    const int sh = a.N >= 16 * 512 ? 1 : a.M <= 4 ? 4 : a.M <= 8 ? 2 : 1;
    const dim3 grid((a.N + 16 / sh - 1) / (16 / sh));
#define LR_LAUNCH(SH_) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_linear_rows<F16, GATED, SH_>), grid, dim3(64 * LR_WAVES), 0, s, t)
    if (sh == 4) LR_LAUNCH(4);
    else if (sh == 2) LR_LAUNCH(2);
    else LR_LAUNCH(1);
#undef LR_LAUNCH
    return moe_check_launch("k_linear_rows");
  }
  t.nm = (a.M + 64 * pl.wm - 1) / (64 * pl.wm);
  t.nn = (a.N + 64 * pl.wn / NM - 1) / (64 * pl.wn / NM);
  if ((long long)t.nm * t.nn * pl.splits >= 1 << 24) {  // (a grid has fewer than 2^32 threads)
    moe_set_error("moe_linear: %d x %d results are too many for one launch", a.M, a.N);
    return MOE_EINVAL;
  }
  t.splits = pl.splits;
  t.ldp = (a.N + 7) & ~7;
  t.part = pl.splits > 1 ? ws : nullptr;
  t.slabs = (a.K + LT_K - 1) / LT_K / pl.splits;
  t.extra = (a.K + LT_K - 1) / LT_K % pl.splits;
  const dim3 grid((t.nm * t.nn * t.splits + 7) / 8 * 8);
#define LT_LAUNCH(WM_, WN_, RING_) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_linear_tile<F16, GATED, WM_, WN_, RING_>), grid, dim3(256), 0, s, t)
  switch (pl.wm * 100 + pl.wn * 10 + pl.ring) {
    case 445:
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_linear_wide<F16, GATED>), dim3(grid.x < 256 ? grid.x : 256), dim3(256), 0, s, t);
      break;
    case 224: LT_LAUNCH(2, 2, 4); break;
    case 126: LT_LAUNCH(1, 2, 6); break;
    case 114: if constexpr (!GATED) LT_LAUNCH(1, 1, 4); break;
    case 243: LT_LAUNCH(2, 4, 3); break;
    default: moe_set_error("moe_linear: no tile %d x %d", pl.wm, pl.wn); return MOE_EINVAL;
  }
#undef LT_LAUNCH
  if (int rc = moe_check_launch("k_linear_tile")) return rc;
  if (!t.part) return MOE_OK;
  const long long pieces = (long long)a.M * (t.ldp >> 3);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(k_linear_join<F16, GATED>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, t);
  return moe_check_launch("k_linear_join");
}
extern "C" int64_t moe_linear_workspace_bytes(int M, int N, int K, int gated) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  auto bytes = [&](int m, int n) -> int64_t {
    const LinPlan p = lin_plan(m, n, K, gated != 0);
    return p.splits > 1 ? (int64_t)p.splits * (gated ? 2 : 1) * m * ((n + 7) & ~7) * 4 : 0;
  };
  const LinCut c = lin_cut(M, N, K, gated != 0);
  if (c.M == M && c.N == N) return bytes(M, N);
  return std::max(bytes(c.M, c.N), bytes(c.M < M ? M - c.M : M, c.N < N ? N - c.N : N));
}

template <bool GATED>
static int lin_run(const char *who, const LinArgs &a, int dtype, void *ws, int64_t ws_bytes, hipStream_t s) {
  if (int rc = lin_check(who, a, dtype, GATED)) return rc;
  if (a.M == 0 || a.N == 0) return MOE_OK;
  const int64_t need = moe_linear_workspace_bytes(a.M, a.N, a.K, GATED);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) {
    moe_set_error("%s: a workspace of %lld bytes on a 16-byte boundary is needed", who, (long long)need);
    return MOE_EINVAL;
  }
  auto launch = [&](const LinArgs &p) {
    return dtype == MOE_DT_FP16 ? lin_launch<true, GATED>(p, (float *)ws, s) : lin_launch<false, GATED>(p, (float *)ws, s);
  };
  const LinCut c = lin_cut(a.M, a.N, a.K, GATED);
  if (c.M == a.M && c.N == a.N) return launch(a);
  LinArgs p = a;
  p.M = c.M;
  p.N = c.N;
  if (int rc = launch(p)) return rc;
  p = a;
  const long long m = c.M < a.M ? c.M : 0, n = c.N < a.N ? c.N : 0;
  p.M -= (int)m;
  p.N -= (int)n;
  p.x += m * a.ldx;
  for (int i = 0; i < (GATED ? 2 : 1); ++i) {
    p.w[i] += n * a.ldw;
    if (p.bias[i]) p.bias[i] += n;
  }
  if (p.res) p.res += m * a.ldr + n;
  p.y = (char *)a.y + (m * a.ldy + n) * (a.y32 ? 4 : 2);
  return launch(p);
}


extern "C" int moe_linear(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *residual, int64_t ldr,
                          void *y, int64_t ldy, int M, int N, int K, int dtype, int act, int y_fp32, void *ws, int64_t ws_bytes,
                          void *stream) {
  const LinArgs a{(const uint16_t *)x, {(const uint16_t *)w, nullptr}, {(const uint16_t *)bias, nullptr}, (const uint16_t *)residual,
                  y, ldx, ldw, ldr, ldy, M, N, K, act, y_fp32 != 0};
  return lin_run<false>("moe_linear", a, dtype, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int moe_linear_gated(const void *x, int64_t ldx, const void *w_gate, const void *w_up, int64_t ldw, const void *b_gate,
                                const void *b_up, void *y, int64_t ldy, int M, int N, int K, int dtype, int act, int y_fp32, void *ws,
                                int64_t ws_bytes, void *stream) {
  const LinArgs a{(const uint16_t *)x, {(const uint16_t *)w_gate, (const uint16_t *)w_up}, {(const uint16_t *)b_gate, (const uint16_t *)b_up},
                  nullptr, y, ldx, ldw, 0, ldy, M, N, K, act, y_fp32 != 0};
  return lin_run<true>("moe_linear_gated", a, dtype, ws, ws_bytes, (hipStream_t)stream);
}
