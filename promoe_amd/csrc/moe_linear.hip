// Products of dense layers (gfx950): y = act(x W^T + b) + residual, and the gated pair y = act(x Wg^T + bg) * (x Wu^T + bu).
// x [M, K], W [N, K] row-major in bf16 or fp16, sums in fp32; bias, activation, product and residual are applied to the
// fp32 sums, which are rounded once, to the type of y.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_common.h"
#include "moe_kernels.h"
#include "moe_device.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct LinArgs {
  const uint16_t *x, *w[2], *bias[2], *res;  // w[1]: the second matrix of a gated pair
  void *y;
  long long ldx, ldw, ldr, ldy;              // elements
  int M, N, K, act, y32;
};

template <bool F16>
static __device__ __forceinline__ float lin_f32(uint16_t v) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, v);
  else return __uint_as_float((u32)v << 16);
}
template <bool F16>
static __device__ __forceinline__ uint16_t lin_bits(float v) {
  if constexpr (F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  else return __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <bool F16>
static __device__ __forceinline__ f32x4_t lin_mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// 1 / (1 + e^-v) with the hardware's 2^x and reciprocal (1 ulp each, and v log2 e rounded: |v| 2^-24 more)
static __device__ __forceinline__ float lin_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896f));
}
static __device__ __forceinline__ float lin_act(int act, float v) {
  switch (act) {
    case MOE_ACT_SILU: return v * lin_sigmoid(v);
    case MOE_ACT_GELU: return 0.5f * v * erfcf(v * -0.70710678118654752f);
    // (1 + tanh z) / 2 = 1 / (1 + e^-2z), z = sqrt(2 / pi) (v + 0.044715 v^3)
    case MOE_ACT_GELU_TANH: return v * lin_sigmoid(1.5957691216057308f * v * fmaf(0.044715f * v, v, 1.f));
    case MOE_ACT_RELU: return v <= 0.f ? 0.f : v;  // (a NaN stays one)
    case MOE_ACT_RELU2: return v <= 0.f ? 0.f : v * v;
    default: return v;
  }
}

// bias, activation, gate, residual and the one rounding of element (m, n)
template <bool F16, bool GATED>
static __device__ __forceinline__ void lin_store(const LinArgs &a, int m, int n, float s0, float s1) {
  if (a.bias[0]) s0 += lin_f32<F16>(a.bias[0][n]);
  float v = lin_act(a.act, s0);
  if constexpr (GATED) {
    if (a.bias[1]) s1 += lin_f32<F16>(a.bias[1][n]);
    v *= s1;
  }
  if (a.res) v += lin_f32<F16>(a.res[m * a.ldr + n]);
  if (a.y32) ((float *)a.y)[m * a.ldy + n] = v;
  else ((uint16_t *)a.y)[m * a.ldy + n] = lin_bits<F16>(v);
}

// A workgroup of four waves on a tile of 64 x 64 (gated: of both matrices), 32 columns of K at a time through LDS.  Rows past the
// end read the last one and are not stored; columns past K are zeros on both sides.
#define LN_T 64
#define LN_K 32
template <bool F16, bool GATED>
__global__ __launch_bounds__(256) void k_linear(const LinArgs a) {
  constexpr int NM = GATED ? 2 : 1;
  __shared__ u32x4_t sx[LN_T][5], sw[NM][LN_T][5];  // four of five 16-byte chunks in use: rows 80 bytes apart
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = lane & 15, q = lane >> 4;
  const int m0 = blockIdx.y * LN_T, n0 = blockIdx.x * LN_T, wm = (wv & 1) * 32, wn = (wv >> 1) * 32;
  f32x4_t acc[NM][2][2] = {};
  const int lr = tid >> 2, lc = tid & 3;  // the row and chunk this thread brings
  const uint16_t *px = a.x + min(m0 + lr, a.M - 1) * a.ldx + 8 * lc;
  const uint16_t *pw[NM];
#pragma unroll
  for (int i = 0; i < NM; ++i) pw[i] = a.w[i] + min(n0 + lr, a.N - 1) * a.ldw + 8 * lc;
  for (int k = 0; k < a.K; k += LN_K) {
    const bool in = k + 8 * lc < a.K;
    const u32x4_t zero = {0, 0, 0, 0};
    const u32x4_t vx = in ? *(const u32x4_t *)(px + k) : zero;
    u32x4_t vw[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) vw[i] = in ? *(const u32x4_t *)(pw[i] + k) : zero;
    __syncthreads();
    sx[lr][lc] = vx;
#pragma unroll
    for (int i = 0; i < NM; ++i) sw[i][lr][lc] = vw[i];
    __syncthreads();
#pragma unroll
    for (int bm = 0; bm < 2; ++bm) {
      const u32x4_t fx = sx[wm + 16 * bm + r][q];
#pragma unroll
      for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int bn = 0; bn < 2; ++bn) acc[i][bm][bn] = lin_mfma16<F16>(sw[i][wn + 16 * bn + r][q], fx, acc[i][bm][bn]);
    }
  }
  // element i of a lane: column 4 q + i of W's block, row r of x's
#pragma unroll
  for (int bm = 0; bm < 2; ++bm)
#pragma unroll
    for (int bn = 0; bn < 2; ++bn)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + wm + 16 * bm + r, n = n0 + wn + 16 * bn + 4 * q + i;
        if (m < a.M && n < a.N) lin_store<F16, GATED>(a, m, n, acc[0][bm][bn][i], acc[NM - 1][bm][bn][i]);
      }
}

// ---- entry points -------------------------------------------------------------------------------------------------------------
static int lin_check(const char *who, const LinArgs &a, int dtype, bool gated) {
  const bool empty = a.M == 0 || a.N == 0;
  if (a.M < 0 || a.N < 0 || a.K <= 0 || a.K % 8 || (dtype != MOE_DT_BF16 && dtype != MOE_DT_FP16) || a.act < MOE_ACT_NONE ||
      a.act > MOE_ACT_RELU2 || a.ldx < a.K || a.ldx % 8 || a.ldw < a.K || a.ldw % 8 || a.ldy < a.N || (a.res && a.ldr < a.N) ||
      a.ldx >= 1 << 21 || a.ldw >= 1 << 21) {
    moe_set_error("%s: bad shape (M=%d N=%d K=%d dtype=%d act=%d, rows %lld %lld %lld %lld elements apart)", who, a.M, a.N, a.K, dtype,
                  a.act, a.ldx, a.ldw, a.res ? a.ldr : 0, a.ldy);
    return MOE_EINVAL;
  }
  if (!empty && (!a.x || !a.w[0] || (gated && !a.w[1]) || !a.y || ((uintptr_t)a.x | (uintptr_t)a.w[0] | (uintptr_t)a.w[1]) & 15)) {
    moe_set_error("%s: operands must be present, x and the matrices on 16-byte boundaries", who);
    return MOE_EINVAL;
  }
  return MOE_OK;
}

template <bool F16, bool GATED>
static int lin_launch(const LinArgs &a, hipStream_t s) {
  const dim3 grid((a.N + LN_T - 1) / LN_T, (a.M + LN_T - 1) / LN_T);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(k_linear<F16, GATED>), grid, dim3(256), 0, s, a);
  return moe_check_launch("k_linear");
}
template <bool GATED>
static int lin_run(const char *who, const LinArgs &a, int dtype, hipStream_t s) {
  if (int rc = lin_check(who, a, dtype, GATED)) return rc;
  if (a.M == 0 || a.N == 0) return MOE_OK;
  return dtype == MOE_DT_FP16 ? lin_launch<true, GATED>(a, s) : lin_launch<false, GATED>(a, s);
}

extern "C" int64_t moe_linear_workspace_bytes(int M, int N, int K, int gated) { return 0; }

extern "C" int moe_linear(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *residual, int64_t ldr,
                          void *y, int64_t ldy, int M, int N, int K, int dtype, int act, int y_fp32, void *ws, int64_t ws_bytes,
                          void *stream) {
  const LinArgs a{(const uint16_t *)x, {(const uint16_t *)w, nullptr}, {(const uint16_t *)bias, nullptr}, (const uint16_t *)residual,
                  y, ldx, ldw, ldr, ldy, M, N, K, act, y_fp32 != 0};
  return lin_run<false>("moe_linear", a, dtype, (hipStream_t)stream);
}

extern "C" int moe_linear_gated(const void *x, int64_t ldx, const void *w_gate, const void *w_up, int64_t ldw, const void *b_gate,
                                const void *b_up, void *y, int64_t ldy, int M, int N, int K, int dtype, int act, int y_fp32, void *ws,
                                int64_t ws_bytes, void *stream) {
  const LinArgs a{(const uint16_t *)x, {(const uint16_t *)w_gate, (const uint16_t *)w_up}, {(const uint16_t *)b_gate, (const uint16_t *)b_up},
                  nullptr, y, ldx, ldw, 0, ldy, M, N, K, act, y_fp32 != 0};
  return lin_run<true>("moe_linear_gated", a, dtype, (hipStream_t)stream);
}
