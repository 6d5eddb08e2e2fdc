// What the kernels of dense products share (gfx950): operands from memory, waits, activations and the way of a sum to its result.
// A, where it is a template's class: a launch's arguments with bias[2], res, ldr, y, ldy, y32, act, M, N, part and ldp (LinArgs has them).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "moe_kernels.h"
#include "moe_device.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
#define LT_OUT 0x7fffff00  // length of the buffer resources; a load from there on reads zeros
typedef int lt_rsrc_t __attribute__((ext_vector_type(4)));
// raw buffer resource over the 2 GiB from p on, as four scalars for the assembly below
static __device__ __forceinline__ lt_rsrc_t lt_rsrc(const void *p) {
  const unsigned long long u = (unsigned long long)p;
  return lt_rsrc_t{(int)(u32)u, (int)(u32)(u >> 32), LT_OUT, 0x00020000};
}

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
// x y + the float of bits C, which stands in the instruction: from the compiler's hands constants go to scalar registers, and k_linear_wide,
// which has none left, moves others out of their way (gated 4096 x 14336 x 4096: 8 us of 663)
template <u32 C>
static __device__ __forceinline__ float lin_fma_k(float x, float y) {
  float r;
  __asm__("v_fmaak_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "n"(C));
  return r;
}
// erfc(a / sqrt 2) / 2 for a >= 0 as 2^-(a q(a) + 1): q, of degree 9, is fitted to -log2(erfc(a / sqrt 2)) / a over [0, 11] in the maximum
// norm (a linear programme), weighted so that v times the fit's error is 1.6e-8 at most, or 4e-3 of the tail; from there on it
// grows, so that nothing is left before the range of fp32 ends.  gelu comes out 3.4e-8 off on average over [-7, 7], with an erf correctly
// rounded to fp32 4.2e-8.  Twelve operations, one of them 2^x, without a branch, where the library's erf has three.
static __device__ __forceinline__ float lin_half_erfc(float a) {
  float q = 5.36956876e-09f;
#define LIN_STEP(C) q = lin_fma_k<__builtin_bit_cast(u32, C)>(q, a)
  LIN_STEP(-2.32354601e-07f); LIN_STEP(4.06335677e-06f); LIN_STEP(-3.57522085e-05f);
  LIN_STEP(1.39703061e-04f); LIN_STEP(2.88132411e-04f); LIN_STEP(-7.29801325e-03f);
  LIN_STEP(5.26819479e-02f); LIN_STEP(4.59138335e-01f); LIN_STEP(1.15111462f);
#undef LIN_STEP
  return __builtin_amdgcn_exp2f(fmaf(-a, q, -1.f));
}
template <int C>
static __device__ __forceinline__ void lin_act(int act, float (&v)[C]) {
  switch (act) {
    case MOE_ACT_SILU:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = v[i] * lin_sigmoid(v[i]);
      break;
    case MOE_ACT_GELU:
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float h = lin_half_erfc(fabsf(v[i]));
        v[i] *= v[i] > 0.f ? 1.f - h : h;
      }
      break;
    case MOE_ACT_GELU_TANH:  // (1 + tanh z) / 2 = 1 / (1 + e^-2z), z = sqrt(2 / pi) (v + 0.044715 v^3)
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = v[i] * lin_sigmoid(1.5957691216057308f * v[i] * fmaf(0.044715f * v[i], v[i], 1.f));
      break;
    case MOE_ACT_RELU:       // (a NaN stays one)
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = v[i] <= 0.f ? 0.f : v[i];
      break;
    case MOE_ACT_RELU2:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = v[i] <= 0.f ? 0.f : v[i] * v[i];
      break;
    default: break;
  }
}

// element (m, n): bias, activation, gate, residual and the one rounding
template <bool F16, bool GATED, class A>
static __device__ __forceinline__ void lin_store(const A &a, int m, int n, float s0, float s1) {
  float v[1] = {a.bias[0] ? s0 + lin_f32<F16>(a.bias[0][n]) : s0};
  lin_act(a.act, v);
  if constexpr (GATED) v[0] *= a.bias[1] ? s1 + lin_f32<F16>(a.bias[1][n]) : s1;
  if (a.res) v[0] += lin_f32<F16>(a.res[m * a.ldr + n]);
  if (a.y32) ((float *)a.y)[m * a.ldy + n] = v[0];
  else ((uint16_t *)a.y)[m * a.ldy + n] = lin_bits<F16>(v[0]);
}

template <bool F16>
static __device__ __forceinline__ void lin_add(float (&v)[8], const u32x4_t r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] += lin_f32<F16>((uint16_t)r[i]);
    v[2 * i + 1] += lin_f32<F16>((uint16_t)(r[i] >> 16));
  }
}
template <bool F16>
static __device__ __forceinline__ u32x4_t lin_pack(const float (&v)[8]) {
  u32x4_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = lin_bits<F16>(v[2 * i]) | (u32)lin_bits<F16>(v[2 * i + 1]) << 16;
  return o;
}

// Sixteen bytes of a result or residual, whose rows may start at any element: the hardware splits an access that crosses a line (us, the
// elements one by one / together: 379 x 1409 x 2048 12.9 / 10.7, 1000 x 1409 x 2048 18.6 / 15.7, of 1408 columns 15.4)
typedef u32x4_t u32x4_any __attribute__((aligned(2)));
typedef f32x4_t f32x4_any __attribute__((aligned(4)));
// Eight adjacent columns of the result from column n on (past N: left out): bias, activation, gate, residual and the one rounding
template <bool F16, bool GATED>
struct LinColumns {
  int n, count;
  float b0[8], b1[8];
  template <class A>
  __device__ __forceinline__ LinColumns(const A &a, int n_) : n(n_), count(min(8, a.N - n_)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b0[i] = b1[i] = 0.f;
    if (a.bias[0])  // (no condition around a load: all of them are on their way at once)
#pragma unroll
      for (int i = 0; i < 8; ++i) b0[i] = lin_f32<F16>(a.bias[0][min(n + i, a.N - 1)]);
    if (GATED && a.bias[1])
#pragma unroll
      for (int i = 0; i < 8; ++i) b1[i] = lin_f32<F16>(a.bias[1][min(n + i, a.N - 1)]);
  }
  // the residual of row m where all eight are there (asked for a row ahead: its trip to memory is longer than a row's work)
  template <class A>
  __device__ __forceinline__ u32x4_t residual(const A &a, int m) const {
    if (GATED || !a.res || count < 8 || m >= a.M) return u32x4_t{0, 0, 0, 0};
    return *(const u32x4_any *)(a.res + m * a.ldr + n);
  }
  // the sums alone, of one piece of K (the join has the rest); rows of a.ldp columns, a multiple of 8
  template <class A>
  __device__ __forceinline__ void partial(const A &a, int split, int m, const float *s0, const float *s1) const {
    if (count <= 0) return;
#pragma unroll
    for (int i = 0; i < (GATED ? 2 : 1); ++i) {
      float *p = a.part + (((long long)split * (GATED ? 2 : 1) + i) * a.M + m) * a.ldp + n;
      *(f32x4_t *)p = *(const f32x4_t *)(i ? s1 : s0);
      *(f32x4_t *)(p + 4) = *(const f32x4_t *)((i ? s1 : s0) + 4);
    }
  }
  // bias, a known activation and gate on the sums s0 (s1: of the second matrix), in place
  template <int ACT>
  __device__ __forceinline__ void finish(float (&s0)[8], const float (&s1)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) s0[i] += b0[i];
    lin_act(ACT, s0);
    if constexpr (GATED) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s0[i] *= s1[i] + b1[i];
    }
  }
  // s0, s1: the sums of row m (s1: of the second matrix); r: its residual
  template <class A>
  __device__ __forceinline__ void store(const A &a, int m, const float *s0, const float *s1, const u32x4_t r) const {
    if (count <= 0) return;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = s0[i] + b0[i];
    lin_act(a.act, v);
    if constexpr (GATED) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= s1[i] + b1[i];
    }
    if (count == 8) {
      if (!GATED && a.res) lin_add<F16>(v, r);
      if (a.y32) {
        float *y = (float *)a.y + m * a.ldy + n;
        *(f32x4_any *)y = f32x4_t{v[0], v[1], v[2], v[3]};
        *(f32x4_any *)(y + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
      } else {
        *(u32x4_any *)((uint16_t *)a.y + m * a.ldy + n) = lin_pack<F16>(v);
      }
      return;
    }
    if (!GATED && a.res) {
      uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = a.res[m * a.ldr + n + min(i, count - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += lin_f32<F16>(e[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) {
        if (a.y32) ((float *)a.y)[m * a.ldy + n + i] = v[i];
        else ((uint16_t *)a.y)[m * a.ldy + n + i] = lin_bits<F16>(v[i]);
      }
  }
};

// f(0), f(1), .. f(N - 1) with numbers known to the compiler
template <int N, int I = 0, class F>
static __device__ __forceinline__ void lt_each(const F &f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    lt_each<N, I + 1>(f);
  }
}

// s_waitcnt for all but the N latest vector-memory operations and nothing else; for all LDS operations and nothing else
#define LT_VM(N) __builtin_amdgcn_s_waitcnt(((N) & 15) | (7 << 4) | (15 << 8) | (((N) >> 4) << 14))
#define LT_LGKM0() __builtin_amdgcn_s_waitcnt(0xc07f)
