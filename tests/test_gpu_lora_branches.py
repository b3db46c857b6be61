"""Adapters of many requests: what v keeps on its way between the two products, in every form that a call may take.

A form is one launch (few rows, small adapters), two launches with tiles of 16 rows (at most 64 rows) or two launches with tiles of 64 rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32

FORMS = {"one launch": (64, 16, 1), "tiles of 16": (64, 128, 2), "tiles of 64": (130, 128, 2), "tiles of 64, few ranks": (130, 16, 2)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["rows", "gate_up"])
def test_v_between_the_products(form, kind):
    """Every row's v is one number just beside the middle between two bf16 values, so the result is rounded the wrong way if v loses that distance.  A and B select it:
    no sum has two terms.  Distances: 2^-20 of v in steps of at most 64 rows (v goes over whole), 2^-16 in larger ones (two parts, rounded: the second holds
    2^-8 - 2^-16 = 255 2^-16 and its like exactly)."""
    from vox_serve_b200 import ops
    T, rank, launches = FORMS[form]
    slots, K, W = 128, 72, 32
    side = 2.0 ** -20 if T <= 64 else 2.0 ** -16
    v = 1.0 + torch.arange(64, dtype=F64) * 3 % 128 * 2.0 ** -7 + 2.0 ** -8        # in the middle: odd multiples of 2^-8
    scale = torch.cat([v + side, v - side])
    assert torch.equal(scale.float().double(), scale)                             # (fp32 holds them)
    g = torch.Generator(device="cuda").manual_seed(1)
    bank = ops.LoraBank(slots, K, (W, W), rank)
    sign = torch.tensor([(-1.0) ** n * 2.0 ** (n % 5) for n in range(W)], dtype=F64)
    for s in range(slots):
        a, b = torch.zeros(2, rank, K, device="cuda"), torch.zeros(2 * W, rank, device="cuda")
        a[:, (7 * s) % rank, (5 * s) % K] = 1.0
        b[W:, (7 * s) % rank] = sign.to("cuda", F32)
        if kind == "rows":
            b[:W] = b[W:].flip(0)
        bank.load(s, a, b, float(scale[s]))
    ids = torch.randperm(slots, generator=torch.Generator().manual_seed(2))[:T]
    ids = torch.cat([ids, torch.full((T - ids.numel(),), -1)])
    x = torch.randn(T, K, generator=g, device="cuda").to(BF16)
    for t, s in enumerate(ids.tolist()):
        if s >= 0:
            x[t, (5 * s) % K] = 1.0
    plan = ops.lora_plan(ops.LoraPlan(T, slots), ids.to("cuda", I32))
    rows = torch.where(ids >= 0, scale[ids.clamp(min=0)], torch.zeros((), dtype=F64))[:, None]
    before = ops.launch_count()
    if kind == "rows":
        got = ops.lora(x, bank, plan, out=torch.empty(T, 2 * W, dtype=BF16, device="cuda"))
        want = rows * torch.cat([sign.flip(0), sign])
    else:
        planes = torch.zeros(1, T, 2, 2, 16, device="cuda")
        planes[:, :, :, 0] = 64.0                                                # silu(64) = 64 to 2^-24
        got = ops.lora_gate_up(x, bank, plan, planes.view(1, T, 2 * W), 32)
        want = 64.0 * rows * sign
    assert ops.launch_count() - before == launches
    assert torch.equal(want.float().double(), want)
    assert torch.equal(got.float().cpu(), want.float().to(BF16).float())


@pytest.mark.parametrize("T,K,rank", [(9, 65536, 128), (150, 65536, 128), (9, 65536, 16), (200, 65536, 16), (40, 28672, 64), (150, 28672, 64), (64, 14336, 128), (150, 14336, 128),
                                      (9, 32768, 16), (9, 8192, 128)])
def test_long_sums_of_fp32_results(T, K, rank):
    """Products of one sign, where every step of the matrix units that cuts its sum off makes it smaller.  A chain of the first product has at most 32 steps, whose sums grow evenly:
    cuts of 2^-22 of the sum so far (2^-23, twice that for the sums inside a step) are 33 / 2 of them at most.  Then up to 16 sums of a block and 8 blocks are added, each
    rounded (2^-24).  Second product: rank / 16 steps over v's first parts (the sums over the others are below 2^-7 of it), then one rounding."""
    from vox_serve_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(K + rank + T)
    rnd = lambda *s: torch.rand(*s, generator=g, device="cuda")                       # noqa: E731
    bank = ops.LoraBank(2, K, (64,), rank)
    a, b = (rnd(1, rank, K) / K).to(BF16), rnd(64, rank).to(BF16)
    bank.load(1, a, b, 0.75)
    x = rnd(T, K).to(BF16)
    ids = torch.ones(T, dtype=I32, device="cuda")
    ids[T // 2] = -1
    got = ops.lora(x, bank, ops.lora_plan(ops.LoraPlan(T, 2), ids))
    want = 0.75 * (x.double() @ a[0].double().t()) @ b.double().t()
    want[T // 2] = 0.0
    bound = 33 / 2 * 2.0 ** -22 + 24 * 2.0 ** -24 + (rank // 16 + 1) / 2 * 1.02 * 2.0 ** -22 + 4 * 2.0 ** -24
    assert bool(((got.double() - want).abs() <= bound * want).all()), float(((got.double() - want).abs() / want.clamp(min=1e-30)).max() / bound)
