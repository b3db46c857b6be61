"""Few-row experts where they are for: steps of one row, alone and in a model's captured decode steps, every one of them compared."""
import pytest
import torch

from tests import test_gpu_moe_layer as L
from tests.test_gpu_row_weights_engines import _text_model

pytestmark = pytest.mark.gpu

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32

ONE = [(1024, 1024, 8, 2, 1024, "silu_glu", "softmax", 0, 0), (72, 70, 4, 4, 3, "clamped_glu", "softmax", 0, 0), (2048, 256, 8, 2, 256, "relu2", "table", 0, 0),
       (200, 64, 33, 3, 0, "gelu", "sigmoid", 0, 0), (136, 130, 64, 8, 0, "silu_glu", "softmax_all", 8, 3), (4096, 64, 6, 1, 0, "gelu_tanh", "softmax", 0, 0)]


@pytest.mark.parametrize("case", ONE, ids=lambda c: "-".join(map(str, c)))
def test_steps_of_one_row(case):
    """sixteen rows of one layer, a call each, against 64 bits together: two of them at most may hang on a tie of the router"""
    from vox_serve_b200 import ops
    h, ex, sh, router, w, ids = L._layer(16, *case, seed=case[0] + case[1])
    got = torch.cat([ops.moe_layer(h[t:t + 1], w, router, ids=None if ids is None else ids[t:t + 1]) for t in range(16)])
    L._check(got, h, ex, sh, router, ids, case[5])


@pytest.mark.parametrize("name", ["bobavik", "redalix", "razevik", "nadevik"])
def test_captured_decode_steps_are_the_eager_ones(name, monkeypatch):
    """tokens one at a time by replays of a captured step and by eager steps: the same bits; every eager step's layers against 64 bits on the rows that they were given"""
    from vox_serve_b200 import ops

    cfg, sd, O, T, up, kw = _text_model(name)
    steps = [[("a", 6)]] + [[("a", 1)]] * 16
    toks = T._tokens(22, cfg["vocab"], 9)
    w = T._worker(cfg, sd, BF16, **kw)
    w.engine.few_experts = True
    replayed = T._replay(w, {"a": toks}, steps)["a"]
    assert w.decode_graphs
    w = T._worker(cfg, sd, BF16, **kw)
    w.engine.few_experts, w.use_cuda_graph = True, False
    rows, real = {}, ops.moe_layer

    def kept(h, weights, router, ids=None, **k):
        out = real(h, weights, router, ids=ids, **k)
        if h.shape[0] == 1:
            rows.setdefault(id(weights), (router, [], [], []))[1].append(h.clone())
            rows[id(weights)][2].append(out.clone())
            rows[id(weights)][3].append(None if ids is None else ids.clone())
        return out
    monkeypatch.setattr(ops, "moe_layer", kept)
    eager = T._replay(w, {"a": toks}, steps)["a"]
    assert torch.equal(replayed, eager)
    layers = [(i, x) for i, x in enumerate(w.engine.w.layers) if up in x]
    assert len(rows) == len(layers) and all(len(r[1]) == 16 for r in rows.values())
    for i, x in layers:
        router, h, out, ids = rows[id(x["few"][0])]
        f = x["few"][0]
        monkeypatch.setattr(L, "LIMIT", f.limit)
        monkeypatch.setattr(L, "SLOPE", f.slope)
        gated = f.act.endswith("glu")
        mats = lambda e: [sd[f"l{i}.mlp.{e}.{m}"].to(device="cuda", dtype=BF16) if m != "gate" or gated else None for m in ("gate", "up", "down")]     # noqa: E731
        per = [mats(f"e{e}") for e in range(f.experts)]
        ex = [None if per[0][m] is None else torch.stack([p[m] for p in per]) for m in range(3)]
        L._check(torch.cat(out), torch.cat(h), ex, mats("shared") if f.shared_ff else None, router, None if ids[0] is None else torch.cat(ids), f.act)


@pytest.mark.parametrize("E,T", [(8, 1), (64, 9), (300, 17)])
def test_router_written_by_the_kernel_in_front(E, T):
    """the router's matrix and bias are changed in place right before a call: the call reads what was written"""
    from vox_serve_b200 import ops
    h, ex, sh, router, w, _ = L._layer(T, 512, 64, E, 2, 0, "silu_glu", "softmax", 0, 0, seed=E)
    rnd = L._rnd(E + 1)
    kept = [(rnd(E, 512, std=0.07), rnd(E, std=0.2)) for _ in range(4)]
    want = []
    for weight, bias in kept:
        torch.cuda.synchronize()
        want.append(ops.moe_layer(h, w, ops.MoeRouter("softmax", 2, weight=weight, bias=bias)))
    assert not torch.equal(want[0], want[1])
    got = []
    for turn in range(50):
        weight, bias = kept[turn % 4]
        router.bias.copy_(bias)
        router.weight.copy_(weight)
        got.append(ops.moe_layer(h, w, router))
        router.weight.copy_(weight)
        router.bias.copy_(bias)
        got.append(ops.moe_layer(h, w, router))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i // 2 % 4]) for i, g in enumerate(got))
