"""Refusals of the operators whose weights a row brings with it (adapters, experts of a decode step): raised on the host, before anything is launched."""
import pytest
import torch

from vox_serve_b200 import ops
from vox_serve_b200._lib import VoxB200Error

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.mark.parametrize("args", [(0, 64, (32,), 8), (1024, 64, (32,), 8), (2, 60, (32,), 8), (2, 0, (32,), 8), (2, 64, (), 8), (2, 64, (32,) * 5, 8), (2, 64, (36,), 8),
                                  (2, 64, (32, 0), 8), (2, 64, (32,), 0), (2, 64, (32,), 129)])
def test_bank_shapes(args):
    with pytest.raises(VoxB200Error):
        ops.LoraBank(*args, device="cpu")


def test_bank_loads_only_what_fits():
    bank = ops.LoraBank(2, 64, (32, 16), 8, device="cpu")
    a, b = torch.zeros(2, 8, 64, dtype=BF16), torch.zeros(48, 8, dtype=BF16)
    bank.load(1, a, b)
    for slot, x, y in ((2, a, b), (-1, a, b), (0, a[:1], b), (0, a[:, :, :56], b), (0, a, b[:40]), (0, a, b[:, :4]), (0, torch.zeros(2, 9, 64), torch.zeros(48, 9)),
                       (0, a[0], b), (0, a[:, :0], b[:, :0])):
        with pytest.raises(VoxB200Error):
            bank.load(slot, x, y)
    with pytest.raises(VoxB200Error):
        bank.clear(2)


def test_bank_order_of_values():
    """every value of A and B stands once in the bank, the rest is zero: the layout as index arithmetic"""
    K, widths, r = 72, (40, 8), 5
    bank = ops.LoraBank(1, K, widths, r, device="cpu")
    a = torch.arange(1, 2 * r * K + 1).view(2, r, K) % 251 + 1
    b = torch.arange(1, 48 * r + 1).view(48, r) % 241 + 1
    bank.load(0, a.float(), b.float(), 2.0)
    A, B, kb = bank.a[0].float(), bank.b[0].float(), (K + 63) // 64
    rp = bank.rank_pad
    seen = torch.zeros_like(A)
    for s in range(2):
        for j in range(r):
            for k in range(K):
                row = s * rp + j
                at = (k // 64 * 2 * rp + row) * 64 + (k % 64 // 8 ^ row % 8) * 8 + k % 8
                assert A[at] == a[s, j, k]
                seen[at] = 1
    assert not bool(A[seen == 0].any())
    seen = torch.zeros_like(B)
    starts, blocks = [0, 40], [0, 2]
    for n in range(48):
        s = int(n >= 40)
        c = n - starts[s]
        for j in range(r):
            block, lane_n, tile, e = blocks[s] + c // 32, c % 32 // 8, c % 8 // 2, c % 2
            lane = (lane_n * 2 + e) * 4 + j % 8 // 2
            at = (((block * (rp // 16) + j // 16) * 2 + tile // 2) * 32 + lane) * 8 + (tile % 2) * 4 + j % 16 // 8 * 2 + j % 2
            assert B[at] == b[n, j]
            seen[at] = 1
    assert not bool(B[seen == 0].any())
    assert float(bank.scale[0]) == 2.0


def test_plan_and_calls_need_the_device():
    with pytest.raises(VoxB200Error):
        ops.LoraPlan(0, 4, device="cpu")
    with pytest.raises(VoxB200Error):
        ops.LoraPlan(4, 1024, device="cpu")
    plan, bank = ops.LoraPlan(4, 2, device="cpu"), ops.LoraBank(2, 64, (32, 32), 8, device="cpu")
    x = torch.zeros(4, 64, dtype=BF16)
    for call in (lambda: ops.lora_plan(plan, torch.zeros(4, dtype=I32)), lambda: ops.lora(x, bank, plan),
                 lambda: ops.lora_gate_up(x, bank, plan, torch.zeros(1, 4, 64), 16)):
        with pytest.raises(VoxB200Error, match="current device"):
            call()


def _packed(n, k, rows):
    return ops.PackedWeight(torch.zeros(8, dtype=torch.uint8), n, k, rows)


@pytest.mark.parametrize("change", [{"act": "swish"}, {"act": "clamped_glu"}, {"act": "clamped_glu", "limit": float("nan")}, {"experts": 0}, {"experts": 1025}, {"width": 60},
                                    {"ff": 96}, {"ff": 0}, {"shared_ff": 32}, {"up": _packed(2 * 5 * 64, 72, 128)}, {"down": _packed(64, 72, 128)},
                                    {"up": _packed(2 * 4 * 64, 72, 48)}, {"down": _packed(72, 4 * 64, 64)}, {"act": "gelu"}])
def test_expert_matrices(change):
    good = {"up": _packed(2 * 4 * 64, 72, 128), "down": _packed(72, 4 * 64, 128), "experts": 4, "width": 72, "ff": 64}
    ops.MoeWeights(**good)
    with pytest.raises(VoxB200Error):
        ops.MoeWeights(**{**good, **change})


def test_expert_packing_checks_its_matrices():
    up, down = torch.zeros(4, 64, 72, dtype=BF16), torch.zeros(4, 72, 64, dtype=BF16)
    for args, kw in (((None, up, down), {}), ((up, up, down), {"act": "gelu"}), ((up, up, down), {})):       # (the last: not on a device)
        with pytest.raises(VoxB200Error):
            ops.MoeWeights.pack(*args, **kw)


@pytest.mark.parametrize("kw", [{"kind": "hash", "top": 2}, {"kind": "softmax", "top": 2}, {"kind": "softmax", "top": 0, "weight": torch.zeros(8, 16)},
                                {"kind": "softmax", "top": 33, "weight": torch.zeros(64, 16)}, {"kind": "softmax", "top": 9, "weight": torch.zeros(8, 16)},
                                {"kind": "softmax", "top": 2, "weight": torch.zeros(8, 16, dtype=BF16)}, {"kind": "table", "top": 2},
                                {"kind": "table", "top": 2, "table": torch.zeros(5, 3, dtype=I32)}, {"kind": "table", "top": 2, "table": torch.zeros(5, 2)},
                                {"kind": "softmax_all", "top": 2, "weight": torch.zeros(8, 16), "bias": torch.zeros(8)},
                                {"kind": "softmax", "top": 2, "weight": torch.zeros(8, 16), "bias": torch.zeros(7)},
                                {"kind": "softmax", "top": 2, "weight": torch.zeros(8, 16), "shared_gate": torch.zeros(16)},
                                {"kind": "softmax", "top": 2, "weight": torch.zeros(8, 16), "groups": 4, "keep": 2},
                                {"kind": "sigmoid", "top": 2, "weight": torch.zeros(8, 16), "groups": 3, "keep": 2},
                                {"kind": "sigmoid", "top": 5, "weight": torch.zeros(8, 16), "groups": 4, "keep": 2},
                                {"kind": "sigmoid", "top": 2, "weight": torch.zeros(8, 16), "groups": 4, "keep": 0}])
def test_routers(kw):
    with pytest.raises(VoxB200Error):
        ops.MoeRouter(**kw)


def test_layer_needs_the_device():
    w = ops.MoeWeights(_packed(2 * 4 * 64, 72, 128), _packed(72, 4 * 64, 128), 4, 72, 64)
    with pytest.raises(VoxB200Error, match="current device"):
        ops.moe_layer(torch.zeros(1, 72, dtype=BF16), w, ops.MoeRouter("softmax", 2, weight=torch.zeros(4, 72)))


def test_refused_adapters_leave_their_slot_as_it_was():
    from vox_serve_b200.engine import LlamaAdapters, LlamaDims

    rnd = torch.Generator().manual_seed(5)
    bank = LlamaAdapters(LlamaDims(128, 2, 2, 1, 64, 256, 100), 2, 8, device="cpu")
    key = "model.layers.%d.self_attn.q_proj.lora_%s.weight"
    good = {key % (0, "A"): torch.randn(4, 128, generator=rnd), key % (0, "B"): torch.randn(128, 4, generator=rnd)}
    bank.load(1, good, 2.0)
    banks = [b for layer in bank.layers for b in layer.values()]
    before = [(b.a.clone(), b.b.clone(), b.scale.clone()) for b in banks]
    assert any(a.any() for a, _, _ in before)
    other = {k: v + 1 for k, v in good.items()}
    for more in ({"model.layers.2.self_attn.q_proj.lora_A.weight": torch.zeros(4, 128)},                    # no such layer
                 {key % (1, "A"): torch.zeros(4, 128)},                                                     # an A without its B
                 {key % (1, "A"): torch.zeros(4, 64), key % (1, "B"): torch.zeros(128, 4)},
                 {key % (1, "A"): torch.zeros(9, 128), key % (1, "B"): torch.zeros(128, 9)}):               # a rank too many
        with pytest.raises(VoxB200Error):
            bank.load(1, {**other, **more}, 1.0)
        for b, (a0, b0, s0) in zip(banks, before):
            assert torch.equal(b.a, a0) and torch.equal(b.b, b0) and torch.equal(b.scale, s0)
    with pytest.raises(VoxB200Error):
        bank.load(2, good, 1.0)
