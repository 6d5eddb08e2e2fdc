// Routers with groups of experts, sigmoid scores or a selection bias in moe_forward.
#include "engine_internal.h"

extern "C" int moe_set_layer_routing(moe_engine *eng, int layer, const moe_route_rule *rule_host, const float *bias) {
  if (!eng) { moe_set_error("moe_set_layer_routing: null engine"); return MOE_EINVAL; }
  if (layer < 0 || layer >= eng->cfg.num_layer) { moe_set_error("moe_set_layer_routing: bad layer %d", layer); return MOE_EINVAL; }
  const moe_layer_desc &d = eng->layer_desc[layer];
  if (!d.gate_w) { moe_set_error("moe_set_layer_routing: layer %d not described (moe_set_layer)", layer); return MOE_ESTATE; }
  LayerRouting r;
  if (rule_host) {
    const int E = eng->cfg.num_expert;
    if (int rc = moe_group_topk(nullptr, 0, E, E, d.top_k, rule_host, nullptr, nullptr, nullptr, nullptr)) return rc;  // checks the rule
    r.set = true;
    r.rule = *rule_host;
    r.bias = bias;
    r.topk = moe_group_topk;
    r.topk_dispatch = moe_group_topk_dispatch;
  }
  eng->layer_routing[layer] = r;
  return MOE_OK;
}
