"""A router and the matrices it is called with: compared at every call, and neither holds the other."""
import gc

import pytest
import torch

from vox_serve_b200 import ops

I32 = torch.int32


def _weights(experts=4, width=72, shared=0):
    n = experts * 64 + shared
    packed = lambda n, k, rows: ops.PackedWeight(torch.zeros(8, dtype=torch.uint8), n, k, rows)                                    # noqa: E731
    return ops.MoeWeights(packed(2 * n, width, 128), packed(width, n, 128), experts, width, 64, shared)


def test_a_router_does_not_hold_the_matrices():
    """gigabytes of experts stay alive otherwise, by a router that answers for another mixture next"""
    router, weights = ops.MoeRouter("softmax", 2, weight=torch.zeros(4, 72)), _weights()
    assert router._goes_with(weights)
    held = [o for o in gc.get_referrers(weights) if o is router]
    assert not held and not any(getattr(router, name, None) is weights for name in router.__slots__)


@pytest.mark.parametrize("router,experts,width,shared,goes", [
    ({"kind": "softmax", "weight": (4, 72)}, 4, 72, 0, True), ({"kind": "softmax", "weight": (5, 72)}, 4, 72, 0, False), ({"kind": "softmax", "weight": (4, 64)}, 4, 72, 0, False),
    ({"kind": "table", "table": (9, 3)}, 4, 72, 0, True), ({"kind": "table", "table": (9, 3)}, 2, 72, 0, False),
    ({"kind": "sigmoid", "weight": (4, 72), "shared_gate": (72,)}, 4, 72, 64, True), ({"kind": "sigmoid", "weight": (4, 72), "shared_gate": (72,)}, 4, 72, 0, False),
    ({"kind": "sigmoid", "weight": (4, 72), "shared_gate": (64,)}, 4, 72, 64, False), ({"kind": "sigmoid", "weight": (4, 72), "shared_gate": (0,)}, 4, 72, 64, False)])
def test_what_goes_together(router, experts, width, shared, goes):
    kw = {k: torch.zeros(v, dtype=I32 if k == "table" else torch.float32) for k, v in router.items() if k != "kind"}
    r, w = ops.MoeRouter(router["kind"], 3, **kw), _weights(experts, width, shared)
    assert r._goes_with(w) == goes
    assert r._goes_with(_weights(experts, width, shared)) == goes
