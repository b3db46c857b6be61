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


def _delta64(x, a, b, scale, widths, ids, v_off):
    """(value, bound of its error) of B (scale A x) in 64 bits.  fp32 chains: K / 16 steps of the first product and 40 sums of warps and blocks, 3 rank / 16 + 4 of the second,
    2^-22 of the absolute sum a step (a step may cut off, 2^-23, twice that for the sums inside it); v_off: what v loses in between."""
    T, K = x.shape
    val = torch.zeros(T, sum(widths), dtype=F64, device="cuda")
    err = torch.zeros_like(val)
    for s in set(ids.tolist()):
        if not 0 <= s < len(a):
            continue
        rows = ids == s
        xs, n0 = x[rows].double(), 0
        d1, d2 = (K / 16 + 40) * 2.0 ** -22, (3 * a[s].shape[1] / 16 + 4) * 2.0 ** -22 + v_off
        out, bad = [], []
        for i, w in enumerate(widths):
            A, B = a[s][i].double(), b[s][n0:n0 + w].double()
            v, av = xs @ A.t() * scale[s], xs.abs() @ A.abs().t() * scale[s]
            out.append(v @ B.t())
            bad.append((d1 * av + d2 * v.abs()) @ B.abs().t())
            n0 += w
        val[rows], err[rows] = torch.cat(out, 1), torch.cat(bad, 1)
    return val, err


def _order(T, slots, order):
    if order == "runs":                                   # long runs, the last adapter's rows before those without one
        ids = [min(slots - 1, t * (slots + 1) // T) for t in range(T - min(3, T // 4))] + [-1] * min(3, T // 4)
    elif order == "turns":
        ids = [t % (slots + 1) - 1 for t in range(T)]
    else:                                                 # a run, then turns
        ids = [0] * (T // 2) + [t % (slots + 1) - 1 for t in range(T - T // 2)]
    return torch.tensor(ids, dtype=I32, device="cuda")


# T, K, widths, rank, slots: two launches each, by more than 128 columns of v, ranks beyond 64 or adapters beyond 3 MB
TWO = [(40, 264, (40, 72, 24), 64, 1), (64, 520, (136, 8, 40), 64, 2), (64, 40, (104,), 128, 3), (40, 8, (64,), 128, 1), (17, 72, (40, 200), 128, 2), (2, 264, (64, 64), 100, 1),
       (64, 8, (264,), 65, 1), (33, 12296, (320,), 128, 2), (64, 24584, (328,), 64, 3)]


def _case(T, K, widths, rank, slots, order):
    from vox_serve_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(13 * T + K + rank)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                      # noqa: E731
    bank = ops.LoraBank(slots, K, widths, rank)
    a, b = [(rnd(len(widths), rank, K) / K ** 0.5).to(BF16) for _ in range(slots)], [rnd(sum(widths), rank).to(BF16) for _ in range(slots)]
    scale = [0.5 + 0.375 * s for s in range(slots)]
    for s in range(slots):
        bank.load(s, a[s], b[s], scale[s])
    ids = _order(T, slots, order)
    return bank, a, b, scale, ids, rnd(T, K).to(BF16), ops.lora_plan(ops.LoraPlan(T, slots), ids), rnd


@pytest.mark.parametrize("order", ["runs", "turns", "both"])
@pytest.mark.parametrize("case", TWO, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("kind", ["plane", "plane_base", "rows", "rows_base"])
def test_two_launches_of_few_rows_against_64_bits(case, kind, order):
    """adapters of up to 64 rows, so of several tiles of 16, whose v the first launch leaves tile by tile"""
    from vox_serve_b200 import ops
    T, K, widths, rank, slots = case
    bank, a, b, scale, ids, x, plan, rnd = _case(*case, order)
    N, f32 = sum(widths), kind.startswith("plane")
    base = rnd(T, N).to(F32 if f32 else BF16) if kind.endswith("base") else None
    out = torch.full((T, N), float("nan"), dtype=F32 if f32 else BF16, device="cuda")
    before = ops.launch_count()
    got = ops.lora(x, bank, plan, out=out, base=base)
    assert ops.launch_count() - before == 2
    want, err = _delta64(x, a, b, scale, widths, ids, 0.0)
    if base is not None:
        want = want + base.double()
    tol = err + want.abs() * (2.0 ** -23 if f32 else 2.0 ** -8) + 1e-30
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("order", ["runs", "turns", "both"])
@pytest.mark.parametrize("T,K,ff,rank,slots,half,splits", [(40, 264, 88, 128, 1, 16, 2), (64, 520, 264, 65, 2, 48, 1), (64, 40, 1000, 128, 3, 64, 1), (17, 8, 72, 128, 2, 32, 3)])
def test_two_launches_of_few_rows_gate_up(T, K, ff, rank, slots, half, splits, order):
    from vox_serve_b200 import ops
    bank, a, b, scale, ids, x, plan, rnd = _case(T, K, (ff, ff), rank, slots, order)
    tiles = (ff + half - 1) // half
    planes = rnd(splits, T, 2 * tiles * half)
    before = ops.launch_count()
    got = ops.lora_gate_up(x, bank, plan, planes, half)
    assert ops.launch_count() - before == 2
    d, err = _delta64(x, a, b, scale, (ff, ff), ids, 0.0)
    p = planes.double().view(splits, T, tiles, half // 16, 2, 16)
    split = lambda v: (v[:, :, :, 0].reshape(T, -1)[:, :ff], v[:, :, :, 1].reshape(T, -1)[:, :ff])   # noqa: E731
    (pg, pu), (ag, au) = split(p.sum(0)), split(p.abs().sum(0))
    gate, up = pg + d[:, :ff], pu + d[:, ff:]
    eg = err[:, :ff] + (splits + 1) * 2.0 ** -23 * (ag + d[:, :ff].abs())
    eu = err[:, ff:] + (splits + 1) * 2.0 ** -23 * (au + d[:, ff:].abs())
    silu = gate * torch.sigmoid(gate)
    want = silu * up
    # |silu'| < 1.1; the exponential of an argument that is rounded, 1.5 |g| 2^-24, itself, the reciprocal and two products: below 2^-20
    tol = 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + want.abs() * (2.0 ** -8 + 2.0 ** -20 + gate.abs() * 2.0 ** -23) + 1e-30
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("K", [8, 40])
@pytest.mark.parametrize("order", ["runs", "turns", "both"])
def test_inputs_narrower_than_a_box(K, order):
    """large steps of fewer inputs than a box of x has columns; x as columns of a wider matrix whose others are NaN"""
    from vox_serve_b200 import ops
    T, widths, rank, slots = 200, (72, 40), 24, 2
    bank, a, b, scale, ids, x, plan, rnd = _case(T, K, widths, rank, slots, order)
    wide = torch.full((T + 70, K + 72), float("nan"), dtype=BF16, device="cuda")
    wide[:T, 8:8 + K] = x
    got = ops.lora(wide[:T, 8:8 + K], bank, plan)
    want, err = _delta64(x, a, b, scale, widths, ids, 0.0)
    assert bool(((got.double() - want).abs() <= err + want.abs() * 2.0 ** -23 + 1e-30).all())


@pytest.mark.parametrize("T,rank,others", [(16, 16, (17, 40, 15, 200)), (16, 128, (17, 130, 9)), (130, 16, (129, 16, 300)), (130, 128, (64, 131))])
def test_captured_steps_behind_another_step_s_plan(T, rank, others):
    """A captured plane and gate | up, then the plan is made for a step of other rows: the replay writes nothing and the host learns of it; behind a plan of its own rows it
    is as before.  So is a plan that was never made, and one of other slots."""
    from vox_serve_b200 import ops
    slots, K, ff = 4, 136, 72
    bank, a, b, scale, ids, x, plan, rnd = _case(T, K, (ff, ff), rank, slots, "turns")
    room = ops.LoraPlan(300, slots)
    planes = rnd(1, T, 2 * 2 * 48)
    outs = torch.zeros(T, 2 * ff, device="cuda"), torch.zeros(T, ff, dtype=BF16, device="cuda")
    ops.check_waits()

    def step():
        ops.lora(x, bank, room, out=outs[0])
        ops.lora_gate_up(x, bank, room, planes, 48, out=outs[1])
    ops.lora_plan(room, ids)
    step()
    want = [o.clone() for o in outs]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        step()

    def replay(whole):
        for o in outs:
            o.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        if whole:
            ops.check_waits()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))
        else:
            with pytest.raises(ops.VoxB200Error, match="a plan of adapters"):
                ops.check_waits()
            assert all(bool((o == 7.0).all()) for o in outs)
    replay(True)
    for n in others:
        ops.lora_plan(room, _order(n, slots, "both"))
        replay(False)
        ops.lora_plan(room, ids)
        replay(True)
    room.tiles.zero_()
    replay(False)
    few = ops.LoraPlan(T, slots - 1)
    ops.lora_plan(few, ids.clamp(max=slots - 2))
    room.tiles[:few.tiles.numel()].copy_(few.tiles)
    replay(False)
    ops.lora_plan(room, ids)
    replay(True)


def test_the_most_rows_and_offsets_past_32_bits():
    """2^21 rows, the most that a plan takes, into results whose last rows stand past 2^31 elements; sampled rows against 64 bits, and rows without an adapter are their base"""
    from vox_serve_b200 import ops
    T, K, N, slots = 2 ** 21, 8, 64, 3
    g = torch.Generator(device="cuda").manual_seed(4)
    bank = ops.LoraBank(slots, K, (N,), 16)
    a, b = [], []
    for s in range(slots):
        a.append(torch.randn(1, 16, K, generator=g, device="cuda").to(BF16))
        b.append(torch.randn(N, 16, generator=g, device="cuda").to(BF16))
        bank.load(s, a[s], b[s], 0.5)
    ids = torch.randint(-1, slots, (T,), generator=g, device="cuda").to(I32)
    ids[:T // 2] = 1                                      # half of the rows in a run
    x = torch.randn(T, K, generator=g, device="cuda").to(BF16)
    plan = ops.lora_plan(ops.LoraPlan(T, slots), ids)
    wide = torch.zeros(T, 1032, dtype=BF16, device="cuda")[:, 512:512 + N]
    assert T * wide.stride(0) > 2 ** 31
    wide.copy_(torch.randn(T, N, generator=g, device="cuda"))
    at = torch.cat([torch.randint(0, T, (3000,), generator=g, device="cuda"), torch.arange(T - 200, T, device="cuda"), torch.arange(T // 2 - 70, T // 2 + 70, device="cuda")])
    base = wide[at].double()
    assert ops.lora(x, bank, plan, out=wide, base=wide) is wide
    d, err = _delta64(x[at], a, b, [0.5] * slots, (N,), ids[at], 2.0 ** -17)
    want = base + d
    got = wide[at].double()
    assert bool(((got - want).abs() <= err + want.abs() * 2.0 ** -8 + 1e-30).all())
    assert bool((got[ids[at] < 0] == base[ids[at] < 0]).all())
    with pytest.raises(ops.VoxB200Error):
        ops.LoraPlan(T + 1, slots)


@pytest.mark.parametrize("rank", [16, 128])
def test_beside_a_vocoder_on_another_stream(rank):
    """Large steps of adapters while a vocoder decodes on another stream, as a serving step has them: kernels of both keep tensor memory and meet in clusters, and a block
    gives its own back before it waits for another.  Both streams' results are those of each alone, to the bit."""
    from oracle import mimi as omimi
    from tests.test_gpu_mimi import _decoder
    from vox_serve_b200 import ops
    cfg = omimi.MimiConfig()
    dec, _ = _decoder(cfg, 5)
    codes = torch.randint(0, cfg.bins, (2, 32, 10), generator=torch.Generator().manual_seed(1)).cuda()
    bank, a, b, scale, ids, x, plan, rnd = _case(600, 2048, (512, 64), rank, 5, "runs")
    wav, want = dec.decode(codes).clone(), ops.lora(x, bank, plan)
    torch.cuda.synchronize()
    side, main = torch.cuda.Stream(), torch.cuda.Stream()
    got, heard = [], []
    for _ in range(10):
        with torch.cuda.stream(side):
            heard.append(dec.decode(codes).clone())
        with torch.cuda.stream(main):
            got += [ops.lora(x, bank, plan) for _ in range(20)]
    torch.cuda.synchronize()
    ops.check_waits()
    assert all(torch.equal(h, wav) for h in heard) and all(torch.equal(o, want) for o in got)
