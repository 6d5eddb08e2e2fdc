// Rows of the tokens in the order of their experts, and the experts' rows back to the tokens (gfx950).
//   sort      y[p] = x[token of p]                      for the pairs p = pos(t, j) in the dispatch's order
//   unsort    y[t] = sum_j w(t, j) x[pos(t, j)]         w absent: 1 (which is the gradient of sort)
//   gradients of unsort: dx[p] = w(t, j) dy[t],  dw(t, j) = <dy[t], x[p]>
// All go by token: a token's row is read (or written) once, its k rows in the experts' order are written (read) whole, and each sum is one
// lane's, in the order of the choices: no atomics, the same bits every time.  A pair without a place (pos -1: its expert is not one of
// the E) takes no part; rows behind the last pair are zero in what is written in the experts' order.  Bound by memory: 4096 tokens of 2048
// bf16 columns, 6 choices: sort and unsort (117 MB) 24 us (4.9 TB/s) and 29 to 33 (3.6 to 4.1), the gradients of unsort (218 MB) 36 (6.0, the last cache helps).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_common.h"
#include "moe_kernels.h"
#include "moe_device.h"

struct MoveArgs {
  const char *x, *dy;
  char *y;
  const int *pos, *total;     // places of the pairs; number of pairs that have one
  const float *w;
  float *dw;
  long long ldx, ldy, ldd;    // bytes between rows of x, y, dy
  int T, k, H, units;         // units: 16-byte (or single-element) pieces of a row
  int cs;                     // lanes of a row: 1 << cs
};

// V elements of type DT as one load
template <int DT, int V> struct Unit;
template <int DT> struct Unit<DT, 8> { typedef u32x4_t type; };
template <int DT> struct Unit<DT, 4> { typedef u32x4_t type; };
template <> struct Unit<MOE_DT_FP32, 1> { typedef u32 type; };
template <> struct Unit<MOE_DT_BF16, 1> { typedef uint16_t type; };
template <> struct Unit<MOE_DT_FP16, 1> { typedef uint16_t type; };

template <int DT, int V>
static __device__ __forceinline__ void unpack(const typename Unit<DT, V>::type u, float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (DT == MOE_DT_FP32) v[0] = __uint_as_float(u);
    else v[0] = DT == MOE_DT_FP16 ? half_bits_to_f32(u) : __uint_as_float((u32)u << 16);
  } else if constexpr (DT == MOE_DT_FP32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = DT == MOE_DT_FP16 ? half_bits_to_f32((uint16_t)u[i]) : bf16lo(u[i]);
      v[2 * i + 1] = DT == MOE_DT_FP16 ? half_bits_to_f32((uint16_t)(u[i] >> 16)) : bf16hi(u[i]);
    }
  }
}
template <int DT>
static __device__ __forceinline__ u32 bits16(float f) {
  if constexpr (DT == MOE_DT_FP16) return __builtin_bit_cast(uint16_t, (_Float16)f);
  else return __builtin_bit_cast(uint16_t, (__bf16)f);
}
template <int DT, int V>
static __device__ __forceinline__ typename Unit<DT, V>::type pack(const float (&v)[V]) {
  if constexpr (V == 1) {
    if constexpr (DT == MOE_DT_FP32) return __float_as_uint(v[0]);
    else return (uint16_t)bits16<DT>(v[0]);
  } else if constexpr (DT == MOE_DT_FP32) {
    return u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  } else {
    u32x4_t u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = bits16<DT>(v[2 * i]) | bits16<DT>(v[2 * i + 1]) << 16;
    return u;
  }
}

// the lane's token and piece; a wave whose row is one token's has its places and weights by scalar loads
struct Spot { int t, c; bool in; };
static __device__ __forceinline__ Spot spot_of(const MoveArgs &a) {
  const int rows = 256 >> a.cs;
  int r = (int)threadIdx.x >> a.cs;
  if (a.cs >= 6) r = __builtin_amdgcn_readfirstlane(r);
  const int t = (int)blockIdx.x * rows + r, c = (int)(blockIdx.y << a.cs) + ((int)threadIdx.x & ((1 << a.cs) - 1));
  return Spot{t, c, t < a.T && c < a.units};
}

template <class U>
__global__ __launch_bounds__(256) void k_sort_rows(const MoveArgs a) {
  const Spot s = spot_of(a);
  if (!s.in) return;
  const int total = *a.total, P = a.T * a.k, p0 = s.t * a.k;
  const U u = *(const U *)(a.x + s.t * a.ldx + s.c * (long long)sizeof(U));
  for (int j = 0; j < a.k; ++j) {
    const int p = a.pos[p0 + j];
    if ((unsigned)p < (unsigned)P) *(U *)(a.y + p * a.ldy + s.c * (long long)sizeof(U)) = u;
    if (p0 + j >= total) *(U *)(a.y + (p0 + j) * a.ldy + s.c * (long long)sizeof(U)) = U{};
  }
}

// acc += the weighted rows of choices j .. j + N - 1
template <int DT, int V, int N>
static __device__ __forceinline__ void add_rows(const MoveArgs &a, const Spot &s, int j, float (&acc)[V]) {
  typedef typename Unit<DT, V>::type U;
  const int P = a.T * a.k, p0 = s.t * a.k + j;
  U u[N];
  bool in[N];
  float w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {  // (a pair without a place reads row 0 and drops it: no condition around a load)
    const int p = a.pos[p0 + i];
    in[i] = (unsigned)p < (unsigned)P;
    w[i] = a.w ? a.w[p0 + i] : 1.f;
    u[i] = *(const U *)(a.x + (in[i] ? p : 0) * a.ldx + s.c * (long long)sizeof(U));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float v[V];
    unpack<DT, V>(u[i], v);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = in[i] ? fmaf(w[i], v[e], acc[e]) : acc[e];
  }
}
// K: choices, 0 for any number
template <int DT, int V, int K>
__global__ __launch_bounds__(256) void k_unsort_rows(const MoveArgs a) {
  typedef typename Unit<DT, V>::type U;
  const Spot s = spot_of(a);
  if (!s.in) return;
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  if constexpr (K > 0) {
    add_rows<DT, V, K>(a, s, 0, acc);
  } else {
    int j = 0;
    for (; j + 8 <= a.k; j += 8) add_rows<DT, V, 8>(a, s, j, acc);
    for (; j < a.k; ++j) add_rows<DT, V, 1>(a, s, j, acc);
  }
  *(U *)(a.y + s.t * a.ldy + s.c * (long long)sizeof(U)) = pack<DT, V>(acc);
}

// A workgroup per token: its row of dy in registers, piece by piece, past the k rows of x.  The dots: lanes, then the four waves in order.
template <int DT, int V, int N>
static __device__ __forceinline__ void grad_rows(const MoveArgs &a, int t, int j0, float *red) {
  typedef typename Unit<DT, V>::type U;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = a.T * a.k, p0 = t * a.k + j0;
  int p[N];
  float w[N], dot[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = a.pos[p0 + i];
    w[i] = a.w[p0 + i];
    dot[i] = 0.f;
  }
  for (int c = tid; c < a.units; c += 256) {
    const long long at = c * (long long)sizeof(U);
    float g[V];
    U u[N];
    const U ug = *(const U *)(a.dy + t * a.ldd + at);
    if (a.dw)
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = *(const U *)(a.x + ((unsigned)p[i] < (unsigned)P ? p[i] : 0) * a.ldx + at);
    unpack<DT, V>(ug, g);
    if (a.dw)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float v[V];
        unpack<DT, V>(u[i], v);
#pragma unroll
        for (int e = 0; e < V; ++e) dot[i] = fmaf(g[e], v[e], dot[i]);
      }
    if (a.y)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((unsigned)p[i] < (unsigned)P) {
          float v[V];
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = w[i] * g[e];
          *(U *)(a.y + p[i] * a.ldy + at) = pack<DT, V>(v);
        }
  }
  if (!a.dw) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) dot[i] += __shfl_xor(dot[i], m, 64);
    if (lane == 0) red[wave * 8 + i] = dot[i];
  }
  __syncthreads();
  if (tid < N) {
    const int q = a.pos[p0 + tid];
    a.dw[p0 + tid] = (unsigned)q < (unsigned)P ? (red[tid] + red[8 + tid]) + (red[16 + tid] + red[24 + tid]) : 0.f;
  }
  __syncthreads();
}
template <int DT, int V, int K>
__global__ __launch_bounds__(256) void k_unsort_grad(const MoveArgs a) {
  typedef typename Unit<DT, V>::type U;
  __shared__ float red[32];
  const int t = blockIdx.x;
  if (a.y) {
    const int total = *a.total;
    for (int j = 0; j < a.k; ++j)
      if (t * a.k + j >= total)
        for (int c = threadIdx.x; c < a.units; c += 256) *(U *)(a.y + (t * a.k + j) * a.ldy + c * (long long)sizeof(U)) = U{};
  }
  if constexpr (K > 0) {
    grad_rows<DT, V, K>(a, t, 0, red);
  } else {
    int j = 0;
    for (; j + 8 <= a.k; j += 8) grad_rows<DT, V, 8>(a, t, j, red);
    for (; j < a.k; ++j) grad_rows<DT, V, 1>(a, t, j, red);
  }
}

// ---- entry points -------------------------------------------------------------------------------------------------------------
static int move_check(const char *who, int T, int k, int H, int dtype, int64_t ldt, int64_t ldp, bool present) {
  if (T < 0 || k < 1 || H < 0 || T >= 1 << 26 || (long long)T * k >= 1ll << 31 || H >= 1 << 24 || dtype < MOE_DT_BF16 || dtype > MOE_DT_FP32 ||
      ldt < H || ldp < H || ldt >= 1ll << 31 || ldp >= 1ll << 31) {
    moe_set_error("%s: bad shape (T=%d k=%d H=%d dtype=%d, rows %lld and %lld elements apart)", who, T, k, H, dtype, (long long)ldt,
                  (long long)ldp);
    return MOE_EINVAL;
  }
  if (T && H && !present) {
    moe_set_error("%s: a tensor is missing", who);
    return MOE_EINVAL;
  }
  return MOE_OK;
}
// From the first byte of an array to behind its last one (bytes 0: there is none)
struct Span { const char *at; int64_t bytes; };
static Span rows_span(const void *p, int64_t rows, int64_t ld, int64_t len) { return Span{(const char *)p, rows && len ? (rows - 1) * ld + len : 0}; }
static Span words_span(const void *p, int64_t n) { return Span{(const char *)p, 4 * n}; }
// Does a result share memory with one of the others?  (Spans that meet are taken to.)
template <class... S>
static bool move_shares(const Span &a, const S &...others) {
  auto meets = [&](const Span &b) { return a.at && b.at && a.bytes && b.bytes && a.at < b.at + b.bytes && b.at < a.at + a.bytes; };
  return (meets(others) || ...);
}
static bool move_wide(const void *p, int64_t ld) { return ((uintptr_t)p | (uintptr_t)ld) % 16 == 0; }
// pieces of a row, and the lanes it gets: a wave, or fewer where a row is shorter
static dim3 move_grid(MoveArgs &a) {
  a.cs = 6;
  while (a.cs > 0 && (1 << (a.cs - 1)) >= a.units) --a.cs;
  const int rows = 256 >> a.cs;
  return dim3((a.T + rows - 1) / rows, (a.units + (1 << a.cs) - 1) >> a.cs);
}

// (the second dimension of a grid ends at 65535: 64 pieces each)
static int move_pieces(const char *who, const MoveArgs &a, dim3 grid) {
  if (grid.y <= 65535) return MOE_OK;
  moe_set_error("%s: rows of %d elements are %d pieces (16 bytes each, single elements where rows are not on 16-byte boundaries), 4194240 at most",
                who, a.H, a.units);
  return MOE_EINVAL;
}

extern "C" int moe_sort_rows(const void *x, int64_t ldx, void *y, int64_t ldy, const int *pos_of_pair, const int *total, int T, int k,
                             int H, int dtype, void *stream) {
  if (int rc = move_check("moe_sort_rows", T, k, H, dtype, ldx, ldy, x && y && pos_of_pair && total)) return rc;
  if (!T || !H) return MOE_OK;
  const int size = dtype == MOE_DT_FP32 ? 4 : 2;
  ldx *= size; ldy *= size;
  const int64_t P = (int64_t)T * k, len = (int64_t)H * size;
  if (move_shares(rows_span(y, P, ldy, len), rows_span(x, T, ldx, len), words_span(pos_of_pair, P), words_span(total, 1))) {
    moe_set_error("moe_sort_rows: the result overlaps what is read");
    return MOE_EINVAL;
  }
  MoveArgs a{(const char *)x, nullptr, (char *)y, pos_of_pair, total, nullptr, nullptr, ldx, ldy, 0, T, k, H, 0, 0};
  const bool wide = move_wide(x, ldx) && move_wide(y, ldy) && (long long)H * size % 16 == 0;
  a.units = wide ? H * size / 16 : H;
  const dim3 grid = move_grid(a);
  if (int rc = move_pieces("moe_sort_rows", a, grid)) return rc;
  if (wide) hipLaunchKernelGGL(k_sort_rows<u32x4_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else if (size == 4) hipLaunchKernelGGL(k_sort_rows<u32>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(k_sort_rows<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
  return moe_check_launch("k_sort_rows");
}

template <int DT, int V>
static void unsort_launch(const MoveArgs &a, dim3 grid, hipStream_t s) {
#define MOVE_K(K_) case K_: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_unsort_rows<DT, V, K_>), grid, dim3(256), 0, s, a); return
  if constexpr (V > 1) switch (a.k) {
    MOVE_K(1); MOVE_K(2); MOVE_K(3); MOVE_K(4); MOVE_K(5); MOVE_K(6); MOVE_K(7); MOVE_K(8);
    default: break;
  }
#undef MOVE_K
  hipLaunchKernelGGL(HIP_KERNEL_NAME(k_unsort_rows<DT, V, 0>), grid, dim3(256), 0, s, a);
}
template <int DT, int V>
static void grad_launch(const MoveArgs &a, hipStream_t s) {
#define MOVE_K(K_) case K_: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_unsort_grad<DT, V, K_>), dim3(a.T), dim3(256), 0, s, a); return
  if constexpr (V > 1) switch (a.k) {
    MOVE_K(1); MOVE_K(2); MOVE_K(3); MOVE_K(4); MOVE_K(5); MOVE_K(6); MOVE_K(7); MOVE_K(8);
    default: break;
  }
#undef MOVE_K
  hipLaunchKernelGGL(HIP_KERNEL_NAME(k_unsort_grad<DT, V, 0>), dim3(a.T), dim3(256), 0, s, a);
}
#define MOVE_TYPES(F, WIDE, ...)                                              \
  switch (dtype) {                                                            \
    case MOE_DT_BF16: WIDE ? F<MOE_DT_BF16, 8>(__VA_ARGS__) : F<MOE_DT_BF16, 1>(__VA_ARGS__); break; \
    case MOE_DT_FP16: WIDE ? F<MOE_DT_FP16, 8>(__VA_ARGS__) : F<MOE_DT_FP16, 1>(__VA_ARGS__); break; \
    default: WIDE ? F<MOE_DT_FP32, 4>(__VA_ARGS__) : F<MOE_DT_FP32, 1>(__VA_ARGS__); break;          \
  }

extern "C" int moe_unsort_rows(const void *x, int64_t ldx, void *y, int64_t ldy, const int *pos_of_pair, const float *w, int T, int k,
                               int H, int dtype, void *stream) {
  if (int rc = move_check("moe_unsort_rows", T, k, H, dtype, ldy, ldx, x && y && pos_of_pair)) return rc;
  if (!T || !H) return MOE_OK;
  const int size = dtype == MOE_DT_FP32 ? 4 : 2;
  ldx *= size; ldy *= size;
  const int64_t P = (int64_t)T * k, len = (int64_t)H * size;
  if (move_shares(rows_span(y, T, ldy, len), rows_span(x, P, ldx, len), words_span(pos_of_pair, P), words_span(w, P))) {
    moe_set_error("moe_unsort_rows: the result overlaps what is read");
    return MOE_EINVAL;
  }
  MoveArgs a{(const char *)x, nullptr, (char *)y, pos_of_pair, nullptr, w, nullptr, ldx, ldy, 0, T, k, H, 0, 0};
  const bool wide = move_wide(x, ldx) && move_wide(y, ldy) && (long long)H * size % 16 == 0;
  a.units = wide ? H * size / 16 : H;
  const dim3 grid = move_grid(a);
  if (int rc = move_pieces("moe_unsort_rows", a, grid)) return rc;
  MOVE_TYPES(unsort_launch, wide, a, grid, (hipStream_t)stream)
  return moe_check_launch("k_unsort_rows");
}

extern "C" int moe_unsort_rows_grad(const void *dy, int64_t lddy, const void *x, int64_t ldx, const int *pos_of_pair, const float *w,
                                    const int *total, void *dx, int64_t lddx, float *dw, int T, int k, int H, int dtype, void *stream) {
  if (int rc = move_check("moe_unsort_rows_grad", T, k, H, dtype, lddy, dw ? ldx : lddx,
                          dy && pos_of_pair && w && (dx || dw) && (x || !dw) && (total || !dx))) return rc;
  if (int rc = move_check("moe_unsort_rows_grad", T, k, H, dtype, lddy, dx ? lddx : ldx, true)) return rc;
  if (!T || (!H && !dw)) return MOE_OK;
  if (!H) {  // dw is zero all the same, and no row of dx exists
    if (!pos_of_pair || !w) {
      moe_set_error("moe_unsort_rows_grad: a tensor is missing");
      return MOE_EINVAL;
    }
    dx = nullptr;
  }
  const int size = dtype == MOE_DT_FP32 ? 4 : 2;
  const int64_t P = (int64_t)T * k, len = (int64_t)H * size;
  lddy *= size; ldx *= size; lddx *= size;
  const Span sdx = rows_span(dx, P, lddx, len), sdw = words_span(dw, P), sx = dw ? rows_span(x, P, ldx, len) : Span{nullptr, 0};
  const Span sdy = rows_span(dy, T, lddy, len), spos = words_span(pos_of_pair, P), sw = words_span(w, P), sn = dx ? words_span(total, 1) : Span{nullptr, 0};
  if (move_shares(sdx, sdy, sx, spos, sw, sn, sdw) || move_shares(sdw, sdy, sx, spos, sw, sn)) {
    moe_set_error("moe_unsort_rows_grad: a gradient overlaps what is read, or the other gradient");
    return MOE_EINVAL;
  }
  MoveArgs a{(const char *)x, (const char *)dy, (char *)dx, pos_of_pair, total, w, dw, ldx, lddx, lddy, T, k, H, 0, 0};
  const bool wide = move_wide(dy, lddy) && (!dw || move_wide(x, ldx)) && (!dx || move_wide(dx, lddx)) && len % 16 == 0;
  a.units = wide ? H * size / 16 : H;
  MOVE_TYPES(grad_launch, wide, a, (hipStream_t)stream)
  return moe_check_launch("k_unsort_grad");
}
