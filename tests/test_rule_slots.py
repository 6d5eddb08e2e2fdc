"""moe_forward's host side for layers with a routing rule, on the CPU under the address and undefined-behaviour sanitizers
(tests/cpp/rule_slots.cpp)."""
import os
import subprocess

import pytest

from tests.test_forward_slots import CPP, HIPCC


@pytest.mark.skipif(HIPCC is None, reason="needs hipcc for the host-only build")
def test_layers_with_a_rule():
    """Decode batches take the routing with the dispatch in one launch, prompts the two launches, both with the layer's rule and bias; a
    refused routing launch fails its forward and no other."""
    r = subprocess.run(["make", "-C", CPP, "rule_slots_asan", "HIPCC=" + HIPCC], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1", UBSAN_OPTIONS="halt_on_error=1")
    r = subprocess.run([os.path.join(CPP, "rule_slots_asan")], capture_output=True, text=True, env=env, timeout=60)
    assert r.returncode == 0 and "rule_slots ok" in r.stdout, (r.returncode, r.stdout[-2000:], r.stderr[-2000:])
