// Routing with groups of experts and a selection bias (gfx950).  One token:
//   s_e = sigmoid(l_e) or exp(l_e - max l) / sum exp(l - max l),   c_e = s_e + bias_e
//   v_g = the largest c of group g, or the sum of its two largest; the topk_group groups of largest v are kept
//   the k largest c in kept groups, descending, are chosen; w_j = s of choice j (/ their sum) * scale
// Equal values: the lower group, the lower expert.  Scores, group values and the comparisons are in 64 bits: with 256 experts
// two scores lie within a rounding of 32 bits of each other in one token of a few thousand, and the choice would then depend on
// whose exponential it is.
//
// A NaN logit counts as -inf (as in the routing without groups).  A NaN among the c (a bias, or a row with +inf under softmax) is
// ordered behind everything.  Whatever the values are, k different experts of kept groups come out: the dispatch counts on it.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "moe_common.h"
#include "moe_kernels.h"
#include "moe_device.h"

#define GR_MAXE 256
#define GR_MAXK 32
#define GR_MAXG 64

struct GroupRule {
  int E, k, G, size, keep, sigmoid, top2, renorm;
  float scale;
  // four tokens by a wave: 2^shift lanes of a token's 16 share a group (all groups kept: a lane is one), `per` experts a lane
  int shift, per;
};

static __device__ __forceinline__ double gr_shfl_xor(double x, int m) { return __shfl_xor(x, m, 64); }
static __device__ __forceinline__ double gr_wave_max(double x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x = fmax(x, gr_shfl_xor(x, m));
  return x;
}
static __device__ __forceinline__ double gr_wave_sum(double x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x += gr_shfl_xor(x, m);
  return x;
}
// NaN behind everything (a lane without an expert holds a NaN all the same: fmax passes over it and nothing equals it)
static __device__ __forceinline__ double gr_ordered(double c) { return fmax(c, -__builtin_inf()); }

// One token by one wave: lane l holds experts l, l + 64, ... (NR of them).  s_c: GR_MAXE doubles of LDS of this wave.
// s_idx, s_mask (LDS, optional): the choices again and as a bit mask [4 x 64] for a dispatch in the same kernel.
template <int NR>
static __device__ __forceinline__ void group_topk_token(const GroupRule &q, const float *__restrict__ row, const float *__restrict__ bias,
                                                        const int lane, double *s_c, int *__restrict__ idx, float *__restrict__ w,
                                                        int *s_idx, unsigned long long *s_mask) {
  double s[NR], c[NR];
  float l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int e = lane + 64 * r;
    l[r] = e < q.E ? fmaxf(row[e], -__builtin_inff()) : -__builtin_inff();
  }
  if (q.sigmoid) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      s[r] = 1.0 / (1.0 + exp(-(double)l[r]));
      __builtin_amdgcn_sched_barrier(0);  // (one after the other: in 64 registers)
    }
  } else {
    float m = l[0];
#pragma unroll
    for (int r = 1; r < NR; ++r) m = fmaxf(m, l[r]);
    m = wave_max_f32(m);
    double sum = 0.0;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      s[r] = lane + 64 * r < q.E ? exp((double)l[r] - (double)m) : 0.0;
      sum += s[r];
      __builtin_amdgcn_sched_barrier(0);
    }
    sum = gr_wave_sum(sum);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      s[r] = s[r] / sum;
      __builtin_amdgcn_sched_barrier(0);
    }
    if (m == -__builtin_inff()) {  // a row that its mask leaves nothing of: scores of zero
#pragma unroll
      for (int r = 0; r < NR; ++r) s[r] = 0.0;
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int e = lane + 64 * r;
    c[r] = e < q.E ? gr_ordered(bias ? s[r] + (double)bias[e] : s[r]) : __builtin_nan("");
  }
  if (q.keep < q.G) {
#pragma unroll
    for (int r = 0; r < NR; ++r) s_c[lane + 64 * r] = c[r];
    __builtin_amdgcn_wave_barrier();
    // lane g: group g's value and how many groups come before it
    double a = -__builtin_inf(), b = a;  // the two largest
    if (lane < q.G)
      for (int i = 0; i < q.size; ++i) {
        const double x = s_c[lane * q.size + i];
        b = fmax(b, fmin(a, x));
        a = fmax(a, x);
      }
    const double v = gr_ordered(q.top2 ? a + b : a);
    int before = 0;
    for (int h = 0; h < q.G; ++h) {
      const double o = __shfl(v, h, 64);
      before += o > v || (o == v && h < lane);
    }
    const unsigned long long kept = __ballot(lane < q.G && before < q.keep);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int e = lane + 64 * r;
      if (e < q.E && !((kept >> (e / q.size)) & 1ull)) c[r] = __builtin_nan("");
    }
    __builtin_amdgcn_wave_barrier();
  }
  unsigned long long msel[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) msel[r] = 0ull;
  double my_s = 0.0, total = 0.0;  // lane j: the j-th choice's score
  for (int j = 0; j < q.k; ++j) {
    double best = c[0];
#pragma unroll
    for (int r = 1; r < NR; ++r) best = fmax(best, c[r]);
    best = gr_wave_max(best);
    int wr = 0, wl = 0;
#pragma unroll
    for (int r = NR - 1; r >= 0; --r) {
      const unsigned long long m = __ballot(c[r] == best);
      if (m) { wr = r; wl = (int)__builtin_ctzll(m); }
    }
    double sc = 0.0;
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (r == wr) {
        sc = s[r];
        if (lane == wl) c[r] = __builtin_nan("");
        msel[r] |= 1ull << wl;
      }
    sc = __shfl(sc, wl, 64);
    total += sc;
    if (lane == j) {
      my_s = sc;
      idx[j] = wl + 64 * wr;
      if (s_idx) s_idx[j] = wl + 64 * wr;
    }
  }
  if (s_mask && lane == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) s_mask[r] = r < NR ? msel[r < NR ? r : 0] : 0ull;
  }
  if (lane < q.k) {
    double x = my_s;
    if (q.renorm) x = total == 0.0 ? 0.0 : x / total;
    w[lane] = (float)(x * (double)q.scale);
  }
}

// ---- four tokens by a wave, in 32 bits where that decides ---------------------------------------------------------------------------
// 16 lanes a token, a lane has a run of at most V experts of one group.  Scores, group values and the k + 1 largest c in 32 bits; a
// token whose every decision (the groups kept, the order of those choices) stands by more than 32 bits can be wrong goes out with these
// choices, and any other one again through group_topk_token: equal values, values next to a border (under 2 % of random tokens), rows of
// masks, infinities.  Without a bias (and sums of two) the logits themselves are ordered.  Weights are in 64 bits either way.
// What 32 bits can be wrong by: sigmoid s (1 - s) (|l| 2^-24 + 2^-23) for 2^x and 2^-23 for the reciprocal, together under 2^-22; softmax 2^-20 of the
// row's largest probability (nine additions one after the other, 2^x, the quotient); the bias added 2^-24 of the sum c; a group's
// value as a sum a + b of two such c 2^-24 (|a| + |b| + |a + b|), whatever cancels in it; the place in the lane's run, which the
// ordered value carries in its last bits, V 2^-23 of it.
// Bound by the vector unit: 32768 tokens over 256 experts in 8 groups, a bias and sums of two take 26.5 to 29 us (36 MB: 7 us at a copy's rate), 1230
// operations a wave of four.  A wave per token in 64 bits takes 67; experts dealt out one by one (16 r + lane), their indexes beside the
// values and the groups' values through LDS 36 (1900 operations); no fours in order 30; 82 registers instead of 64, which cost the exact
// form some in scratch, two waves fewer a SIMD and 2 us; waves that go on to
// further tokens, whose logits are on their way meanwhile, four a SIMD, 40.
template <int N>
static __device__ __forceinline__ float gr_ror(float x) {  // lane j: x of lane j - N within its 16
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, true));
}
static __device__ __forceinline__ float gr_max16(float x) {
  x = fmaxf(x, gr_ror<8>(x)); x = fmaxf(x, gr_ror<4>(x)); x = fmaxf(x, gr_ror<2>(x));
  return fmaxf(x, gr_ror<1>(x));
}
static __device__ __forceinline__ float gr_sum16(float x) {
  x += gr_ror<8>(x); x += gr_ror<4>(x); x += gr_ror<2>(x);
  return x + gr_ror<1>(x);
}
template <int N>
static __device__ __forceinline__ double gr_ror(double x) {
  const long long u = __builtin_bit_cast(long long, x);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)u, 0x120 + N, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), 0x120 + N, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (long long)(unsigned)lo | (long long)hi << 32);
}
static __device__ __forceinline__ double gr_sum16(double x) {
  x += gr_ror<8>(x); x += gr_ror<4>(x); x += gr_ror<2>(x);
  return x + gr_ror<1>(x);
}
// e^x for x <= 0 to about 2^-41: 2^n times the Taylor polynomial of 2^f, |f| <= 1/2, of degree 10 (next term 2.2e-13)
static __device__ __forceinline__ double gr_exp(double x) {
  x = fmax(x, -800.0);  // (zero from there on)
  const double y = x * 1.4426950408889634074, n = rint(y), z = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 3628800;
  p = fma(p, z, 1.0 / 362880); p = fma(p, z, 1.0 / 40320); p = fma(p, z, 1.0 / 5040); p = fma(p, z, 1.0 / 720); p = fma(p, z, 1.0 / 120);
  p = fma(p, z, 1.0 / 24); p = fma(p, z, 1.0 / 6); p = fma(p, z, 0.5); p = fma(p, z, 1.0); p = fma(p, z, 1.0);
  return ldexp(p, (int)n);
}

// a / b for b in the middle of the range: reciprocal and two of Newton's steps, the quotient corrected once
static __device__ __forceinline__ double gr_div(double a, double b) {
  double r = __builtin_amdgcn_rcp(b);
  r = fma(fma(-b, r, 1.0), r, r);
  r = fma(fma(-b, r, 1.0), r, r);
  const double x = a * r;
  return fma(fma(-b, x, a), r, x);
}
// floats as integers of the same order, and back
static __device__ __forceinline__ int gr_key(float x) {
  const int b = __builtin_bit_cast(int, x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
static __device__ __forceinline__ float gr_value(int k) { return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff)); }
template <int N>
static __device__ __forceinline__ int gr_ror_i(int x) { return __builtin_amdgcn_update_dpp(0, x, 0x120 + N, 0xf, 0xf, true); }
static __device__ __forceinline__ int gr_max16_i(int x) {
  x = max(x, gr_ror_i<8>(x)); x = max(x, gr_ror_i<4>(x)); x = max(x, gr_ror_i<2>(x));
  return max(x, gr_ror_i<1>(x));
}

union GroupLds {
  float v[4][16];          // the groups' values of four tokens
  double exact[GR_MAXE];
};
// tokens t0 .. t0 + 3 (those below T).  s_idx, s_mask as in group_topk_token, of token 0.
template <int V>
static __device__ __forceinline__ void group_topk_quad(const GroupRule &q, const float *__restrict__ logits, const int ldl, const int t0,
                                                       const int T, const float *__restrict__ bias, const int lane, GroupLds &m,
                                                       int *__restrict__ idx, float *__restrict__ w, int *s_idx, unsigned long long (*s_mask)[4]) {
  constexpr float INF = __builtin_inff();
  constexpr int NONE = (int)0x80000000;
  const int tok = lane >> 4, j = lane & 15, t = min(t0 + tok, T - 1);
  const bool by_logit = !bias && (!q.top2 || q.keep == q.G);
  // lane j's run of experts: in group j >> shift, part j & .. of it
  const int g = j >> q.shift, per = q.per, size = q.keep < q.G ? q.size : per, G = q.keep < q.G ? q.G : 16;
  const int part0 = (j - (g << q.shift)) * per, start = g * size + part0;
  const int count = g < G ? max(0, min(min(per, size - part0), q.E - start)) : 0;
  // (sixteen bytes from any float on; what a run does not hold is masked, and zeros behind the last row)
  const long long end = ((long long)(T - 1 - t0) * ldl + q.E) * 4;
  const rsrc_t rl = make_rsrc(logits + (size_t)t0 * ldl, (int)(end < 0x7fffff00ll ? end : 0x7fffff00ll)), rb = make_rsrc(bias, bias ? q.E * 4 : 0);
  const int at = ((t - t0) * ldl + start) * 4;
  float l[V], c[V];
#pragma unroll
  for (int r = 0; r < V; r += 4) {
    const float4 x = __builtin_bit_cast(float4, bload16(rl, r < count ? at + 4 * r : 0, 0));
    l[r] = x.x; l[r + 1] = x.y; l[r + 2] = x.z; l[r + 3] = x.w;
  }
  if (bias) {
#pragma unroll
    for (int r = 0; r < V; r += 4) {
      const float4 x = __builtin_bit_cast(float4, bload16(rb, r < count ? (start + r) * 4 : 0, 0));
      c[r] = x.x; c[r + 1] = x.y; c[r + 2] = x.z; c[r + 3] = x.w;
    }
  }
#pragma unroll
  for (int r = 0; r < V; ++r) l[r] = r < count ? fmaxf(l[r], -INF) : -INF;
  float top = l[0];
#pragma unroll
  for (int r = 1; r < V; ++r) top = fmaxf(top, l[r]);
  top = gr_max16(top);
  bool sure = top > -INF && top < INF;
  float unsure_abs = 9.3132257e-10f, unsure_rel = 0.f;  // values this close (2^-30; relative to both) may be in either order
  if (by_logit) {
#pragma unroll
    for (int r = 0; r < V; ++r) c[r] = l[r];
    if (q.sigmoid) sure = sure && top <= 15.f;  // (from about 34 on scores of different logits are equal in 64 bits)
  } else {
    float s[V];
    if (q.sigmoid) {
#pragma unroll
      for (int r = 0; r < V; ++r) s[r] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(l[r] * -1.44269504088896f));
      unsure_abs = 9.5367432e-7f;               // 2^-20
    } else {
      float sum[V];
#pragma unroll
      for (int r = 0; r < V; ++r) sum[r] = s[r] = __builtin_amdgcn_exp2f((l[r] - top) * 1.44269504088896f);
#pragma unroll
      for (int k = V / 2; k >= 1; k >>= 1)
#pragma unroll
        for (int r = 0; r < k; ++r) sum[r] += sum[r + k];
      const float most = 1.f / gr_sum16(sum[0]);
#pragma unroll
      for (int r = 0; r < V; ++r) s[r] *= most;
      unsure_abs = 3.8146973e-6f * most;        // 2^-18
    }
    unsure_rel = 9.5367432e-7f;
#pragma unroll
    for (int r = 0; r < V; ++r) c[r] = r < count ? fmaxf(bias ? s[r] + c[r] : s[r], -INF) : -INF;  // (a NaN counts as -inf)
  }
  bool mine_kept = true;
  if (q.keep < q.G) {
    float a = c[0], b = -INF;  // the two largest of the lane, of the group
#pragma unroll
    for (int r = 1; r < V; ++r) {
      if (q.top2) b = fmaxf(b, fminf(a, c[r]));
      a = fmaxf(a, c[r]);
    }
    for (int k = 1; k < 1 << q.shift; k <<= 1) {
      const float oa = __shfl_xor(a, k, 64), ob = __shfl_xor(b, k, 64);
      b = fmaxf(fminf(a, oa), fmaxf(b, ob));
      a = fmaxf(a, oa);
    }
    const float v = q.top2 ? a + b : a;
    float *sv = m.v[tok];
    __builtin_amdgcn_wave_barrier();
    if (part0 == 0) sv[g] = v;
    __builtin_amdgcn_wave_barrier();
    int before = 0;
    for (int k = 0; k < G; ++k) before += sv[k] > v;
    mine_kept = g < G && before < q.keep;
    const float least = -gr_max16(mine_kept ? -v : -INF), most = gr_max16(g < G && !mine_kept ? v : -INF);
    // (more groups than stay where those at the border are equal: each has fewer than `keep` in front of it)
    const unsigned heads = (unsigned)(__ballot(mine_kept && part0 == 0) >> (16 * tok)) & 0xffffu;
    sure = sure && __popc(heads) == q.keep;
    // (a sum of two is off by twice as much, and with a bias by a part of what it is the sum of, which can be far more than the sum:
    // 1000.4 - 999.8; NaN and two infinities are not sure)
    const float size_of = q.top2 && bias ? gr_max16(g < G ? fabsf(a) + fabsf(b) : 0.f) : fabsf(least) + fabsf(most);
    sure = sure && least - most > 2.f * unsure_abs + unsure_rel * size_of;
    if (by_logit) sure = sure && least > (q.sigmoid ? -700.f : top - 700.f);
  }
  // k + 1 rounds of the largest value; lane i keeps choice i (two of them past 16 choices).  The place in the run in the last bits.
  int key[V], at_lane = NONE;
#pragma unroll
  for (int r = 0; r < V; ++r) {
    const int x = (gr_key(c[r]) & -V) | r;
    key[r] = mine_kept & (c[r] > -1e38f) ? x : NONE;
  }
  // (fours in descending order: a round takes the first of one away)
#pragma unroll
  for (int r = 0; r < V; r += 4) {
    auto order = [&](int x, int y) {
      const int hi = max(key[r + x], key[r + y]);
      key[r + y] = min(key[r + x], key[r + y]);
      key[r + x] = hi;
    };
    order(0, 1); order(2, 3); order(0, 2); order(1, 3); order(1, 2);
    at_lane = max(at_lane, key[r]);
  }
  unsure_rel += (float)V * 1.3e-7f;
  const float floor = by_logit ? (q.sigmoid ? -700.f : top - 700.f) : -1e37f;
  const bool more = q.k < q.keep * q.size;
  float last = INF;
  int mine[2] = {0, 0};
  for (int i = 0; i < q.k + more; ++i) {
    const int best = gr_max16_i(at_lane);
    const unsigned who = (unsigned)(__ballot(at_lane == best) >> (16 * tok)) & 0xffffu;
    const float value = gr_value(best);
    // (a last round that finds none, and the first, have no border)
    sure &= (i == 0) | ((i == q.k) & (best == NONE)) | (last - value > unsure_abs + unsure_rel * (fabsf(last) + fabsf(value)));
    if (i == q.k) break;
    sure &= (best != NONE) & (value > floor) & ((who & (who - 1u)) == 0u);
    last = value;
    const int jw = __builtin_ctz(who | 0x10000u), gw = jw >> q.shift;
    const int e = gw * size + (jw - (gw << q.shift)) * per + (best & (V - 1));
    if ((i & 15) == j) mine[i >> 4] = sure ? e : 0;
    at_lane = NONE;
#pragma unroll
    for (int r = 0; r < V; r += 4) {
      const bool gone = key[r] == best;
      key[r] = gone ? key[r + 1] : key[r];
      key[r + 1] = gone ? key[r + 2] : key[r + 1];
      key[r + 2] = gone ? key[r + 3] : key[r + 2];
      key[r + 3] = gone ? NONE : key[r + 3];
      at_lane = max(at_lane, key[r]);
    }
  }
  // weights, in 64 bits: lane i those of its choices
  double den = 1.0;
  if (!q.sigmoid) {
    double s = 0.0;
#pragma unroll
    for (int r = 0; r < V; ++r) s += gr_exp((double)l[r] - (double)top);
    den = gr_sum16(s);
  }
  double s[2], total = 0.0;
  bool tiny = false;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s[h] = 0.0;
    if (h && q.k <= 16) break;
    const double x = (double)fmaxf(logits[(size_t)t * ldl + mine[h]], -INF), d = q.sigmoid ? -fabs(x) : x - (double)top, p = gr_exp(d);
    // (scores of few bits, and sigmoids that the exact form has as zero: the bias has chosen them, and in a sum of nothing else they count)
    tiny |= j + 16 * h < q.k && d < -700.0 && d > -750.0;
    s[h] = q.sigmoid ? gr_div(x < 0.0 ? p : 1.0, 1.0 + p) : gr_div(p, den);
    total += j + 16 * h < q.k ? s[h] : 0.0;
  }
  if (q.renorm) total = gr_sum16(total);
  sure = sure && ((unsigned)(__ballot(tiny) >> (16 * tok)) & 0xffffu) == 0u;
  const bool live = t0 + tok < T;
  if (live && sure) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = j + 16 * h;
      if (i >= q.k) break;
      const double x = q.renorm ? (total == 0.0 ? 0.0 : s[h] / total) : s[h];
      idx[(size_t)t * q.k + i] = mine[h];
      w[(size_t)t * q.k + i] = (float)(x * (double)q.scale);
      if (s_idx) s_idx[t * q.k + i] = mine[h];
    }
  }
  if (s_mask) {  // bit e of the token's mask
    if (live && sure && j < 4) s_mask[t][j] = 0ull;
    __builtin_amdgcn_wave_barrier();
    if (live && sure) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (j + 16 * h < q.k) atomicOr(&s_mask[t][mine[h] >> 6], 1ull << (mine[h] & 63));
    }
  }
  unsigned long long again = __ballot(live && !sure && j == 0);
  __builtin_amdgcn_wave_barrier();
  while (again) {
    const int k = (int)__builtin_ctzll(again) >> 4, tk = t0 + k;
    again &= again - 1ull;
    group_topk_token<4>(q, logits + (size_t)tk * ldl, bias, lane, m.exact, idx + (size_t)tk * q.k, w + (size_t)tk * q.k,
                        s_idx ? s_idx + tk * q.k : nullptr, s_mask ? s_mask[tk] : nullptr);
  }
}
// V 0: more groups than a token has lanes: 64-bit scores throughout, a token by a wave
template <int V>
static __device__ __forceinline__ void group_topk_four(const GroupRule &q, const float *__restrict__ logits, const int ldl, const int t0,
                                                       const int T, const float *__restrict__ bias, const int lane, GroupLds &m,
                                                       int *__restrict__ idx, float *__restrict__ w, int *s_idx, unsigned long long (*s_mask)[4]) {
  if constexpr (V == 0) {
    for (int t = t0; t < min(t0 + 4, T); ++t)
      group_topk_token<4>(q, logits + (size_t)t * ldl, bias, lane, m.exact, idx + (size_t)t * q.k, w + (size_t)t * q.k,
                          s_idx ? s_idx + t * q.k : nullptr, s_mask ? s_mask[t] : nullptr);
  } else {
    group_topk_quad<V>(q, logits, ldl, t0, T, bias, lane, m, idx, w, s_idx, s_mask);
  }
}
// f(V) for the form that a rule takes
template <class F>
static void gr_form(const GroupRule &q, const F &f) {
  if (q.per == 0) f(std::integral_constant<int, 0>());
  else if (q.per <= 4) f(std::integral_constant<int, 4>());
  else if (q.per <= 8) f(std::integral_constant<int, 8>());
  else if (q.per <= 16) f(std::integral_constant<int, 16>());
  else f(std::integral_constant<int, 32>());
}

template <int V>
__global__ __launch_bounds__(256, V == 32 ? 4 : 8) void k_group_topk(const GroupRule q, const float *__restrict__ logits, const int T, const int ldl,
                                                    const float *__restrict__ bias, int *__restrict__ idx, float *__restrict__ w) {
  __shared__ GroupLds s_m[4];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, t0 = __builtin_amdgcn_readfirstlane(4 * (blockIdx.x * 4 + wv));
  if (t0 < T) group_topk_four<V>(q, logits, ldl, t0, T, bias, lane, s_m[wv], idx, w, nullptr, nullptr);
}

// ---- with the stable dispatch of a decode batch in the same launch: one workgroup, a wave per four tokens -----------------------
// Latency: 1 token of 64 experts 4.8 us, 33 of 256 10.9 us.
#define GR_MAXT 64
#define GR_MAXP 512
struct GroupDispatch {
  int *counts, *offsets, *sorted_pair, *pos_of_pair, *sorted_tok;
  moe_unit *units;
  int *n_active;
  long long *active_ids;
  int max_units;
  moe_unit *host_units;
  int *host_n_active, *host_seq;
  int host_seq_val;
};

template <int NW, int V>
__global__ __launch_bounds__(64 * NW) void k_group_topk_dispatch(const GroupRule q, const float *__restrict__ logits, const int T,
                                                                 const int ldl, const float *__restrict__ bias, int *__restrict__ idx,
                                                                 float *__restrict__ w, const GroupDispatch d) {
  constexpr int NT = 64 * NW;
  __shared__ GroupLds s_m[NW];
  __shared__ int s_idx[GR_MAXP];
  __shared__ unsigned long long s_mask[GR_MAXT][4];
  __shared__ int s_off[GR_MAXE];
  __shared__ int s_rows[4], s_used[4], s_tot;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), E = q.E, k = q.k;
  if (4 * wv < T) group_topk_four<V>(q, logits, ldl, 4 * wv, T, bias, lane, s_m[wv], idx, w, s_idx, s_mask);  // (T <= 4 NW)
  __syncthreads();
  // A token holds an expert at most once: the pairs of an expert in stable order are its tokens in order, so the place of
  // (t, e) is the offset of e plus the tokens before t whose mask has e.  Thread e owns expert e (E <= 256 <= threads).
  int c = 0;
  if (tid < E)
    for (int t = 0; t < T; ++t) c += (int)((s_mask[t][wv] >> lane) & 1ull);
  int rows = c, used = c > 0;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const int a = __shfl_up(rows, i, 64), b = __shfl_up(used, i, 64);
    if (lane >= i) { rows += a; used += b; }
  }
  if (wv < 4 && lane == 63) { s_rows[wv] = rows; s_used[wv] = used; }
  __syncthreads();
  if (wv < 4) {
    for (int i = 0; i < wv; ++i) { rows += s_rows[i]; used += s_used[i]; }
    const int row0 = rows - c, u = used - 1;
    if (tid < E) {
      s_off[tid] = row0;
      d.counts[tid] = c;
      d.offsets[tid] = row0;
      if (c > 0 && u < d.max_units) {
        d.units[u] = moe_unit{tid, c, row0, 0};
        d.active_ids[u] = tid;
        if (d.host_units) host_store_unit(d.host_units, u, tid, c, row0);
      }
    }
    if (tid == E - 1) {
      const int n = used < d.max_units ? used : d.max_units;
      d.offsets[E] = rows;
      *d.n_active = n;
      if (d.host_units) host_store_i32(d.host_n_active, n);
      s_tot = used;
    }
  }
  __syncthreads();
  for (int u = s_tot + tid; u < d.max_units; u += NT) {
    d.units[u] = moe_unit{-1, 0, 0, 0};
    d.active_ids[u] = -1;
  }
  for (int p = tid; p < T * k; p += NT) {
    const int e = s_idx[p], t = p / k;
    int pos = s_off[e];
    for (int i = 0; i < t; ++i) pos += (int)((s_mask[i][e >> 6] >> (e & 63)) & 1ull);
    d.sorted_pair[pos] = p;
    d.pos_of_pair[p] = pos;
    d.sorted_tok[pos] = t;
  }
  if (d.host_units) {
    host_stores_done();
    __syncthreads();
    if (tid == 0) __hip_atomic_store(d.host_seq, d.host_seq_val, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  }
}

// ---- entry points -------------------------------------------------------------------------------------------------------------
static int rule_check(const char *who, const moe_route_rule *r, int E, int k) {
  if (!r || E <= 0 || E > GR_MAXE || k <= 0 || k > GR_MAXK || (r->scores != MOE_SCORES_SOFTMAX && r->scores != MOE_SCORES_SIGMOID) ||
      (r->group_value != MOE_GROUP_MAX && r->group_value != MOE_GROUP_TOP2) || r->n_group <= 0 || r->n_group > GR_MAXG ||
      E % r->n_group || r->topk_group <= 0 || r->topk_group > r->n_group || k > E / r->n_group * r->topk_group ||
      (r->group_value == MOE_GROUP_TOP2 && r->topk_group < r->n_group && E / r->n_group < 2)) {
    if (!r) moe_set_error("%s: no rule", who);
    else
      moe_set_error("%s: bad rule (E=%d k=%d scores=%d n_group=%d topk_group=%d group_value=%d)", who, E, k, r->scores, r->n_group,
                    r->topk_group, r->group_value);
    return MOE_EINVAL;
  }
  return MOE_OK;
}
static GroupRule rule_of(const moe_route_rule &r, int E, int k, int ldl) {
  GroupRule q{E, k, r.n_group, E / r.n_group, r.topk_group, r.scores == MOE_SCORES_SIGMOID, r.group_value == MOE_GROUP_TOP2,
              r.renorm != 0, r.scale, 0, 0};
  if (ldl > 1 << 26) return q;  // (four rows have to be in reach of 31 bits)
  if (q.keep == q.G) q.per = (E + 15) / 16;
  else if (q.G <= 16) {
    while ((q.G << (q.shift + 1)) <= 16) ++q.shift;
    q.per = (q.size + (1 << q.shift) - 1) >> q.shift;
  }
  return q;
}

extern "C" int moe_group_topk(const float *logits, int T, int E, int ldl, int k, const moe_route_rule *rule_host, const float *bias,
                              int *idx, float *w, void *stream) {
  if (int rc = rule_check("moe_group_topk", rule_host, E, k)) return rc;
  if (T < 0 || T > 1 << 27 || ldl < E || (T > 0 && (!logits || !idx || !w))) {
    moe_set_error("moe_group_topk: bad argument (T=%d E=%d ldl=%d)", T, E, ldl);
    return MOE_EINVAL;
  }
  if (T == 0) return MOE_OK;
  hipStream_t s = (hipStream_t)stream;
  moe_ktimer_begin(MOE_K_TOPK, s);
  const GroupRule q = rule_of(*rule_host, E, k, ldl);
  gr_form(q, [&](auto v) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_group_topk<decltype(v)::value>), dim3((T + 15) / 16), dim3(256), 0, s, q, logits, T, ldl, bias, idx, w);
  });
  moe_ktimer_end(MOE_K_TOPK, s);
  return moe_check_launch("k_group_topk");
}

extern "C" int moe_group_topk_dispatch(const float *logits, int T, int E, int ldl, int k, const moe_route_rule *rule_host,
                                       const float *bias, int *idx, float *w, int *counts, int *offsets, int *sorted_pair,
                                       int *pos_of_pair, int *sorted_tok, moe_unit *units, int *n_active, int64_t *active_ids,
                                       int max_units, moe_unit *units_host_out, int *n_active_host_out, int *seq_host_out,
                                       int seq_value, void *stream) {
  if (int rc = rule_check("moe_group_topk_dispatch", rule_host, E, k)) return rc;
  if (T <= 0 || T > GR_MAXT || T * k > GR_MAXP || ldl < E || !logits || !idx || !w || !counts || !offsets || !sorted_pair ||
      !pos_of_pair || !sorted_tok || !units || !n_active || !active_ids || max_units < 0 ||
      (units_host_out && (!n_active_host_out || !seq_host_out))) {
    moe_set_error("moe_group_topk_dispatch: bad argument (T=%d E=%d k=%d ldl=%d)", T, E, k, ldl);
    return MOE_EINVAL;
  }
  hipStream_t s = (hipStream_t)stream;
  const GroupDispatch d{counts, offsets, sorted_pair, pos_of_pair, sorted_tok, units, n_active, (long long *)active_ids, max_units,
                        units_host_out, n_active_host_out, seq_host_out, seq_value};
  const GroupRule q = rule_of(*rule_host, E, k, ldl);
  moe_ktimer_begin(MOE_K_TOPK, s);
  // (four tokens a wave: four waves for up to 16 tokens, whose barriers are cheaper; thread e also owns expert e)
  gr_form(q, [&](auto v) {
    constexpr int V = decltype(v)::value;
    if (T <= 16)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_group_topk_dispatch<4, V>), dim3(1), dim3(256), 0, s, q, logits, T, ldl, bias, idx, w, d);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_group_topk_dispatch<16, V>), dim3(1), dim3(1024), 0, s, q, logits, T, ldl, bias, idx, w, d);
  });
  moe_ktimer_end(MOE_K_TOPK, s);
  return moe_check_launch("k_group_topk_dispatch");
}
