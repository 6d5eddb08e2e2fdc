// moe_forward's host side for layers that route by a rule (moe_set_layer_routing), over the stand-ins of forward_slots.cpp: which
// routing launches a batch takes, with which rule and bias, and that one that is refused leaves nothing waiting.  (The launches that
// route by themselves are stubs here: a forward that took one would fail without any of these.)
#define main forward_slots_main
#include "forward_slots.cpp"
#undef main

static int g_topk = 0, g_dispatch = 0, g_topk_dispatch = 0, g_refuse_routing = 0;
static moe_route_rule g_rule;
static const float *g_bias = nullptr;

static void fill(int T, int max_units, moe_unit *units, int *n_active) {
  for (int u = 0; u < max_units; ++u) units[u] = moe_unit{u, T * K / max_units, u * (T * K / max_units), 0};
  *n_active = max_units;
}
extern "C" {
int moe_group_topk(const float *, int T, int, int, int, const moe_route_rule *rule, const float *bias, int *, float *, void *) {
  if (T == 0) return rule->n_group == 3 ? MOE_EINVAL : MOE_OK;  // (moe_set_layer_routing asks whether the rule is one)
  if (g_refuse_routing > 0) { --g_refuse_routing; return MOE_EINVAL; }
  ++g_topk;
  g_rule = *rule;
  g_bias = bias;
  return MOE_OK;
}
int moe_dispatch_ws(const int *, int T, int, int, int *, int *, int *, int *, int *, moe_unit *units, int *n_active, int64_t *, int max_units,
                    void *, int64_t, int *, void *) {
  ++g_dispatch;
  fill(T, max_units, units, n_active);
  return MOE_OK;
}
int moe_group_topk_dispatch(const float *, int T, int, int, int, const moe_route_rule *rule, const float *bias, int *, float *, int *, int *,
                            int *, int *, int *, moe_unit *units, int *n_active, int64_t *, int max_units, moe_unit *host_units,
                            int *host_n, int *host_seq, int seq, void *) {
  if (g_refuse_routing > 0) { --g_refuse_routing; return MOE_EINVAL; }
  ++g_topk_dispatch;
  g_rule = *rule;
  g_bias = bias;
  fill(T, max_units, units, n_active);
  if (host_units) {
    fill(T, max_units, host_units, host_n);
    *host_seq = seq;
  }
  return MOE_OK;
}
}

int main() {
  moe_cfg *cfg = moe_cfg_create(1, E);
  const char *names[1] = {"w"};
  CK(moe_cfg_set_params(cfg, names, 1));
  CK(moe_cfg_set(cfg, "num_expert_per_token", "2"));
  CK(moe_cfg_set(cfg, "cache_rate", "1.0"));
  CK(moe_cfg_set(cfg, "cache_policy", "lru"));
  setenv("SPARSE_CACHE_PHYSICAL_MEM_IMPL", "slab", 1);
  CK(moe_cfg_finalize(cfg));
  moe_engine *eng = nullptr;
  CK(moe_engine_create(cfg, MOE_BACKEND_HIP, g_compute, &eng));
  std::vector<std::vector<uint8_t>> bufs;
  for (int e = 0; e < E; ++e) {
    bufs.emplace_back(512, (uint8_t)e);
    CK(moe_register_param(eng, 0, e, 0, bufs.back().data(), bufs.back().size(), 0));
  }
  CK(moe_init_slots(eng));
  std::vector<uint16_t> gate((size_t)E * H), x((size_t)100 * H), y((size_t)100 * H);
  std::vector<float> bias(E);
  moe_layer_desc d;
  memset(&d, 0, sizeof d);
  d.H = H; d.I = I; d.top_k = K; d.fmt = MOE_FMT_BF16; d.gate_w = gate.data();
  CK(moe_set_layer(eng, 0, &d));
  moe_route_rule rule{MOE_SCORES_SIGMOID, 4, 2, MOE_GROUP_TOP2, 1, 2.5f}, bad = rule;
  bad.n_group = 3;
  if (moe_set_layer_routing(eng, 0, &bad, nullptr) != MOE_EINVAL) { printf("a bad rule was taken\n"); return 1; }
  CK(moe_set_layer_routing(eng, 0, &rule, bias.data()));
  CK(moe_forward_prepare(eng, 100));
  CK(moe_launch(eng));
  const int before = g_topk + g_topk_dispatch;
  auto routed = [&](const char *what, int fused, int apart) {
    const bool ok = g_topk_dispatch == fused && g_topk == apart && g_dispatch == apart &&
                    (fused + apart == 0 || (g_rule.n_group == 4 && g_rule.scale == 2.5f && g_bias == bias.data()));
    if (!ok) printf("%s: %d fused, %d + %d apart\n", what, g_topk_dispatch, g_topk, g_dispatch);
    g_topk_dispatch = g_topk = g_dispatch = 0;
    return ok;
  };
  if (before) { printf("a launch before the first forward\n"); return 1; }
  // prompts: group_topk and the dispatch, the first forward (experts missing) and later ones (all resident)
  for (int i = 0; i < 3; ++i) {
    CK(moe_forward(eng, 0, x.data(), 40, y.data()));
    if (!routed("40 tokens", 0, 1)) return 1;
  }
  CK(moe_drain(eng));
  // a refused routing launch fails the forward; the next ones go on at once
  const auto t0 = std::chrono::steady_clock::now();
  g_refuse_routing = 1;
  if (moe_forward(eng, 0, x.data(), 40, y.data()) == MOE_OK || g_refuse_routing) { printf("the refused launch was not met\n"); return 1; }
  if (!routed("refused", 0, 0)) return 1;
  for (int i = 0; i < 20; ++i) CK(moe_forward(eng, 0, x.data(), 40, y.data()));
  if (!routed("20 forwards", 0, 20)) return 1;
  // decode batches: the one launch, once in vain (the expert launch behind it is a stub that refuses)
  for (int T : {1, 2, 16, 32}) {
    moe_forward(eng, 0, x.data(), T, y.data());
    if (!routed("a decode batch", 1, 0)) { printf("%d tokens\n", T); return 1; }
  }
  CK(moe_forward(eng, 0, x.data(), 33, y.data()));
  if (!routed("33 tokens", 0, 1)) return 1;
  // without the rule, and after a new description
  CK(moe_set_layer_routing(eng, 0, nullptr, nullptr));
  CK(moe_forward(eng, 0, x.data(), 40, y.data()));
  if (!routed("no rule", 0, 0)) return 1;
  CK(moe_set_layer_routing(eng, 0, &rule, bias.data()));
  CK(moe_set_layer(eng, 0, &d));
  CK(moe_forward(eng, 0, x.data(), 40, y.data()));
  if (!routed("a new description", 0, 0)) return 1;
  CK(moe_drain(eng));
  const double s = std::chrono::duration<double>(std::chrono::steady_clock::now() - t0).count();
  printf("rule_slots ok, %.3f s\n", s);
  moe_engine_destroy(eng);
  moe_cfg_destroy(cfg);
  return s < 2.0 ? 0 : 1;
}
