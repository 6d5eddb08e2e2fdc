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

#include "moe_common.h"
#include "moe_kernels.h"
#include "moe_device.h"

#define GR_MAXE 256
#define GR_MAXK 32
#define GR_MAXG 64

struct GroupRule {
  int E, k, G, size, keep, sigmoid, top2, renorm;
  float scale;
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
    for (int r = 0; r < NR; ++r) s[r] = 1.0 / (1.0 + exp(-(double)l[r]));
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
    }
    sum = gr_wave_sum(sum);
#pragma unroll
    for (int r = 0; r < NR; ++r) s[r] = s[r] / sum;
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

__global__ __launch_bounds__(256) void k_group_topk(const GroupRule q, const float *__restrict__ logits, const int T, const int ldl,
                                                    const float *__restrict__ bias, int *__restrict__ idx, float *__restrict__ w) {
  __shared__ double s_c[4][GR_MAXE];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, t = blockIdx.x * 4 + wv;
  if (t >= T) return;
  const float *row = logits + (size_t)t * ldl;
  int *ir = idx + (size_t)t * q.k;
  float *wr = w + (size_t)t * q.k;
  if (q.E <= 64) group_topk_token<1>(q, row, bias, lane, s_c[wv], ir, wr, nullptr, nullptr);
  else if (q.E <= 128) group_topk_token<2>(q, row, bias, lane, s_c[wv], ir, wr, nullptr, nullptr);
  else group_topk_token<4>(q, row, bias, lane, s_c[wv], ir, wr, nullptr, nullptr);
}

// ---- with the stable dispatch of a decode batch in the same launch: one workgroup, a wave per token in turn --------------------
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

template <int NW>
__global__ __launch_bounds__(64 * NW) void k_group_topk_dispatch(const GroupRule q, const float *__restrict__ logits, const int T,
                                                                 const int ldl, const float *__restrict__ bias, int *__restrict__ idx,
                                                                 float *__restrict__ w, const GroupDispatch d) {
  constexpr int NT = 64 * NW;
  __shared__ double s_c[NW][GR_MAXE];
  __shared__ int s_idx[GR_MAXP];
  __shared__ unsigned long long s_mask[GR_MAXT][4];
  __shared__ int s_off[GR_MAXE];
  __shared__ int s_rows[4], s_used[4], s_tot;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, E = q.E, k = q.k;
  for (int t = wv; t < T; t += NW) {
    const float *row = logits + (size_t)t * ldl;
    int *ir = idx + (size_t)t * k;
    float *wr = w + (size_t)t * k;
    if (E <= 64) group_topk_token<1>(q, row, bias, lane, s_c[wv], ir, wr, s_idx + t * k, s_mask[t]);
    else if (E <= 128) group_topk_token<2>(q, row, bias, lane, s_c[wv], ir, wr, s_idx + t * k, s_mask[t]);
    else group_topk_token<4>(q, row, bias, lane, s_c[wv], ir, wr, s_idx + t * k, s_mask[t]);
  }
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
static GroupRule rule_of(const moe_route_rule &r, int E, int k) {
  return GroupRule{E, k, r.n_group, E / r.n_group, r.topk_group, r.scores == MOE_SCORES_SIGMOID, r.group_value == MOE_GROUP_TOP2,
                   r.renorm != 0, r.scale};
}

extern "C" int moe_group_topk(const float *logits, int T, int E, int ldl, int k, const moe_route_rule *rule_host, const float *bias,
                              int *idx, float *w, void *stream) {
  if (int rc = rule_check("moe_group_topk", rule_host, E, k)) return rc;
  if (T < 0 || ldl < E || (T > 0 && (!logits || !idx || !w))) {
    moe_set_error("moe_group_topk: bad argument (T=%d E=%d ldl=%d)", T, E, ldl);
    return MOE_EINVAL;
  }
  if (T == 0) return MOE_OK;
  hipStream_t s = (hipStream_t)stream;
  moe_ktimer_begin(MOE_K_TOPK, s);
  hipLaunchKernelGGL(k_group_topk, dim3((T + 3) / 4), dim3(256), 0, s, rule_of(*rule_host, E, k), logits, T, ldl, bias, idx, w);
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
  const GroupRule q = rule_of(*rule_host, E, k);
  moe_ktimer_begin(MOE_K_TOPK, s);
  // (a wave per token: four waves for few tokens, whose barriers are cheaper; thread e also owns expert e)
  if (T <= 4) hipLaunchKernelGGL(k_group_topk_dispatch<4>, dim3(1), dim3(256), 0, s, q, logits, T, ldl, bias, idx, w, d);
  else hipLaunchKernelGGL(k_group_topk_dispatch<16>, dim3(1), dim3(1024), 0, s, q, logits, T, ldl, bias, idx, w, d);
  moe_ktimer_end(MOE_K_TOPK, s);
  return moe_check_launch("k_group_topk_dispatch");
}
