"""Adapters of many requests (ops.lora, ops.lora_gate_up) against their formula in 64 bits.

Tolerances, derived: inputs are bf16 and exact in both.  A chain of fp32 sums of depth d over products whose absolute sum is S is off by at most d 2^-22 S (a
step of the matrix units may cut off instead of rounding: 2^-23, twice that leaves room for the sums inside a step).  First product: a step takes 16 k, the
warps' and pieces' sums follow, so d <= K / 16 + 40.  Second: v enters in exact parts (fp32 results: 3 rank / 16 + 4 steps) or cut off by 2^-15 (bf16
results).  A rounding to bf16 is off by 2^-8 of the value at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def _inputs(T, K, widths, rank, slots, seed, rank_of=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                      # noqa: E731
    from vox_serve_b200 import ops
    bank = ops.LoraBank(slots, K, widths, rank)
    a, b, scale = [], [], []
    for s in range(slots):
        r = rank if rank_of is None else rank_of[s % len(rank_of)]
        a.append((rnd(len(widths), r, K) / K ** 0.5).to(BF16))
        b.append(rnd(sum(widths), r).to(BF16))
        scale.append(0.5 + 0.25 * (s % 5))
        bank.load(s, a[s], b[s], scale[s])
    ids = torch.randint(-1, slots, (T,), generator=g, device="cuda").to(I32)
    x = rnd(T, K).to(BF16)
    return bank, a, b, scale, ids, x


def _delta64(x, a, b, scale, widths, ids, parts_cut):
    """(value, bound of its error) of B (scale A x) in 64 bits"""
    T, K = x.shape
    val = torch.zeros(T, sum(widths), dtype=F64, device="cuda")
    err = torch.zeros_like(val)
    for t, s in enumerate(ids.tolist()):
        if not 0 <= s < len(a):
            continue
        xt, n0 = x[t].double(), 0
        d1, d2 = (K / 16 + 40) * 2.0 ** -22, (3 * a[s].shape[1] / 16 + 4) * 2.0 ** -22 + parts_cut
        for i, w in enumerate(widths):
            A, B = a[s][i].double(), b[s][n0:n0 + w].double()
            v, av = A @ xt * scale[s], A.abs() @ xt.abs() * scale[s]
            val[t, n0:n0 + w] = B @ v
            err[t, n0:n0 + w] = B.abs() @ (d1 * av + d2 * v.abs())
            n0 += w
    return val, err


def _plan(ids, slots):
    from vox_serve_b200 import ops
    return ops.lora_plan(ops.LoraPlan(max(1, ids.numel()), slots), ids)


CASES = [(1, 8, (8,), 1, 1), (1, 896, (896,), 8, 4), (2, 40, (40, 8, 24), 3, 2), (16, 264, (128,), 16, 5), (17, 1000, (64, 8), 17, 3),
         (64, 2048, (2048, 256, 256), 16, 40), (65, 520, (72, 40), 32, 3), (130, 96, (200,), 64, 2), (200, 1504, (104, 96, 8, 16), 100, 1),
         (333, 640, (352,), 40, 64), (1, 4096, (4096,), 128, 2)]


@pytest.mark.parametrize("T,K,widths,rank,slots", CASES)
@pytest.mark.parametrize("kind", ["plane", "plane_base", "rows", "rows_base"])
def test_lora_against_64_bits(T, K, widths, rank, slots, kind):
    from vox_serve_b200 import ops
    bank, a, b, scale, ids, x = _inputs(T, K, widths, rank, slots, 7 * T + K, rank_of=[rank, max(1, rank // 2)])
    N = sum(widths)
    f32 = kind.startswith("plane")
    base = torch.randn(T, N, device="cuda").to(F32 if f32 else BF16) if kind.endswith("base") else None
    out = None if kind != "rows" else torch.full((T, N), float("nan"), dtype=BF16, device="cuda")
    got = ops.lora(x, bank, _plan(ids, slots), out=out, base=base)
    assert got.dtype == (F32 if f32 else BF16) and tuple(got.shape) == (T, N)
    want, err = _delta64(x, a, b, scale, widths, ids, 0.0 if f32 else 2.0 ** -15)
    if base is not None:
        want = want + base.double()
    tol = err + want.abs() * (2.0 ** -23 if f32 else 2.0 ** -8) + 1e-30
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("T,K,ff,rank,slots,half,splits", [(1, 8, 8, 1, 1, 64, 1), (17, 896, 488, 16, 5, 48, 1), (33, 200, 1000, 24, 3, 16, 2),
                                                          (70, 512, 264, 64, 2, 32, 3), (129, 72, 72, 128, 4, 64, 1), (64, 256, 2048, 32, 70, 64, 1)])
@pytest.mark.parametrize("tiled", [False, True])
def test_lora_gate_up_against_64_bits(T, K, ff, rank, slots, half, splits, tiled):
    from vox_serve_b200 import ops
    bank, a, b, scale, ids, x = _inputs(T, K, (ff, ff), rank, slots, 11 * T + ff)
    tiles = (ff + half - 1) // half
    planes = torch.randn(splits, T, 2 * tiles * half, device="cuda")
    out = ops.TiledAct(T, ff, "cuda") if tiled else None
    got = ops.lora_gate_up(x, bank, _plan(ids, slots), planes, half, out=out)
    got = got.to_rows() if tiled else got
    assert got.dtype == BF16 and tuple(got.shape) == (T, ff)
    d, err = _delta64(x, a, b, scale, (ff, ff), ids, 2.0 ** -15)
    p = planes.double().view(splits, T, tiles, half // 16, 2, 16)
    pa = p.abs().sum(0)
    split = lambda v: (v[:, :, :, 0].reshape(T, -1)[:, :ff], v[:, :, :, 1].reshape(T, -1)[:, :ff])   # noqa: E731
    (pg, pu), (ag, au) = split(p.sum(0)), split(pa)
    gate, up = pg + d[:, :ff], pu + d[:, ff:]
    eg = err[:, :ff] + (splits + 1) * 2.0 ** -23 * (ag + d[:, :ff].abs())
    eu = err[:, ff:] + (splits + 1) * 2.0 ** -23 * (au + d[:, ff:].abs())
    silu = gate * torch.sigmoid(gate)
    want = silu * up
    # |silu'| < 1.1; the exponential, the quotient and the product: a few units of 2^-23 each
    tol = 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + want.abs() * (2.0 ** -8 + 2.0 ** -19) + 1e-30
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


def test_lora_ids_outside_have_no_adapter():
    from vox_serve_b200 import ops
    bank, a, b, scale, _, x = _inputs(70, 64, (32,), 8, 3, 1)
    ids = torch.randint(0, 3, (70,), device="cuda").to(I32)
    ids[::7], ids[3], ids[5] = -1, 3, 2 ** 31 - 1
    ids[8] = -2 ** 31
    base = torch.randn(70, 32, device="cuda")
    got = ops.lora(x, bank, _plan(ids, 3), base=base)
    none = (ids < 0) | (ids > 2)
    assert torch.equal(got[none], base[none]) and bool((got[~none] != base[~none]).any(1).all())


def test_lora_strides_in_place_and_rows_behind():
    from vox_serve_b200 import ops
    bank, a, b, scale, ids, x = _inputs(37, 128, (64, 32), 16, 4, 2)
    wide = torch.zeros(40, 136, dtype=BF16, device="cuda")
    wide[:37, 8:] = x
    plan = _plan(ids, 4)
    want = ops.lora(x, bank, plan)
    buf = torch.full((41, 200), 5.0, device="cuda")
    ops.lora(wide[:37, 8:], bank, plan, out=buf[:37, 4:100])
    assert torch.equal(buf[:37, 4:100], want)
    buf[:37, 4:100] = 5.0
    assert bool((buf == 5.0).all())                       # nothing beside or behind
    rows = torch.randn(37, 96, device="cuda").to(BF16)
    into = rows.clone()
    assert ops.lora(x, bank, plan, out=into, base=into) is into
    assert torch.equal(into, ops.lora(x, bank, plan, base=rows))


def test_lora_rows_do_not_depend_on_their_company():
    """a row's result is the same alone, in another order and in a tile of another height"""
    from vox_serve_b200 import ops
    bank, a, b, scale, ids, x = _inputs(150, 512, (96,), 16, 6, 3)
    got = ops.lora(x, bank, _plan(ids, 6))
    perm = torch.randperm(150, device="cuda")
    assert torch.equal(ops.lora(x[perm].contiguous(), bank, _plan(ids[perm].contiguous(), 6)), got[perm])
    want, err = _delta64(x, a, b, scale, (96,), ids, 0.0)
    for t in (0, 77, 149):
        one = ops.lora(x[t:t + 1], bank, _plan(ids[t:t + 1], 6))
        assert bool(((one[0].double() - want[t]).abs() <= err[t] + want[t].abs() * 2.0 ** -23 + 1e-30).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_lora_non_finite_rows_stay_among_themselves(bad):
    from vox_serve_b200 import ops
    bank, a, b, scale, ids, x = _inputs(40, 256, (64,), 16, 2, 4)
    ids.fill_(1)
    plan = _plan(ids, 2)
    want = ops.lora(x, bank, plan)
    x[13, 100] = bad
    got = ops.lora(x, bank, plan)
    rest = torch.arange(40, device="cuda") != 13
    assert torch.equal(got[rest], want[rest]) and not bool(torch.isfinite(got[13]).any())
    # an adapter whose values are not finite reaches its own rows only
    ids[::2] = 0
    bank.load(0, torch.full((16, 256), bad, dtype=BF16, device="cuda"), b[0], 1.0)
    x[13] = 1.0
    got = ops.lora(x, bank, _plan(ids, 2), base=torch.ones(40, 64, device="cuda"))
    assert bool(torch.isfinite(got[1::2]).all()) and not bool(torch.isfinite(got[::2]).any())


def test_lora_bank_slots_are_replaced_and_cleared():
    from vox_serve_b200 import ops
    bank, a, b, scale, ids, x = _inputs(9, 64, (40,), 32, 2, 5)
    ids.fill_(1)
    plan = _plan(ids, 2)
    bank.load(1, a[0][:, :4], b[0][:, :4], 3.0)           # a smaller rank over a larger one
    want, err = _delta64(x, [None, a[0][:, :4]], [None, b[0][:, :4]], [0, 3.0], (40,), ids, 0.0)
    got = ops.lora(x, bank, plan)
    assert bool(((got.double() - want).abs() <= err + want.abs() * 2.0 ** -23 + 1e-30).all())
    bank.clear(1)
    assert not bool(ops.lora(x, bank, plan).any())


def test_lora_captured_and_on_another_stream():
    """one graph of plan, plane and gate | up replayed over changing rows, beside calls on another stream"""
    from vox_serve_b200 import ops
    T, K, ff = 48, 256, 136
    bank, a, b, scale, ids, x = _inputs(T, K, (ff, ff), 16, 5, 6)
    plan, planes = ops.LoraPlan(T, 5), torch.randn(1, T, 2 * 3 * 48, device="cuda")
    sx, sid = x.clone(), ids.clone()

    def step():
        ops.lora_plan(plan, sid)
        return ops.lora(sx, bank, plan), ops.lora_gate_up(sx, bank, plan, planes, 48)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in (1, 2, 3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        sx.copy_(torch.randn(T, K, generator=gen, device="cuda").to(BF16))
        sid.copy_(torch.randint(-1, 5, (T,), generator=gen, device="cuda").to(I32))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            p2 = ops.lora_plan(ops.LoraPlan(T, 5), sid)
            want = ops.lora(sx, bank, p2), ops.lora_gate_up(sx, bank, p2, planes, 48)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_lora_no_rows():
    from vox_serve_b200 import ops
    bank = ops.LoraBank(2, 64, (32, 32), 8)
    plan = ops.lora_plan(ops.LoraPlan(4, 2), torch.zeros(0, dtype=I32, device="cuda"))
    x = torch.zeros(0, 64, dtype=BF16, device="cuda")
    assert tuple(ops.lora(x, bank, plan).shape) == (0, 64)
    assert tuple(ops.lora_gate_up(x, bank, plan, torch.zeros(1, 0, 64, device="cuda"), 16).shape) == (0, 32)


def test_lora_many_adapters_and_rows():
    """every slot of a large bank in one step, rows of a slot far apart"""
    from vox_serve_b200 import ops
    slots, T = 1023, 2500
    bank, a, b, scale, _, x = _inputs(T, 64, (40,), 4, slots, 8)
    ids = (torch.arange(T, device="cuda") * 7 % (slots + 1) - 1).to(I32)
    got = ops.lora(x, bank, _plan(ids, slots))
    want, err = _delta64(x, a, b, scale, (40,), ids, 0.0)
    assert bool(((got.double() - want).abs() <= err + want.abs() * 2.0 ** -23 + 1e-30).all())


@pytest.mark.parametrize("T,K,rank,launches", [(9, 256, 16, 1), (9, 1024, 128, 2), (70, 256, 16, 2)])
def test_lora_counts_its_launches(T, K, rank, launches):
    """a step of few rows whose adapters are small is one launch, every other two (128 x 3 columns of v are more than the one launch takes)"""
    from vox_serve_b200 import ops

    widths = (128, 64, 64) if rank == 128 else (256,)
    bank = ops.LoraBank(2, K, widths, rank)
    plan = ops.lora_plan(ops.LoraPlan(T, 2), torch.zeros(T, dtype=I32, device="cuda"))
    x = torch.zeros(T, K, dtype=BF16, device="cuda")
    before = ops.launch_count()
    ops.lora(x, bank, plan)
    assert ops.launch_count() - before == launches


@pytest.mark.parametrize("K,widths,rank", [(200, (264,), 16), (72, (40, 72), 128), (1032, (136, 8, 24), 64), (320, (64,), 24)])
@pytest.mark.parametrize("order", ["prompts", "turns", "both"])
def test_lora_rows_in_a_row_and_apart(K, widths, rank, order):
    """rows of an adapter that follow one another in x (fetched as boxes, which reach past the adapter's rows and, for the last, past x), rows that alternate, and
    both; x as columns of a wider matrix whose others, and whose rows behind the step's, are NaN"""
    from vox_serve_b200 import ops

    T, slots = 333, 4
    runs = [0] * 129 + [3] * 70 + [-1] * 3 + [1] * 131
    ids = runs if order == "prompts" else [t % 5 - 1 for t in range(T)] if order == "turns" else runs[:202] + [t % 5 - 1 for t in range(T - 202)]
    bank, a, b, scale, _, x = _inputs(T, K, widths, rank, slots, seed=K + rank)
    ids = torch.tensor(ids, dtype=I32, device="cuda")
    wide = torch.full((T + 40, K + 48), float("nan"), dtype=BF16, device="cuda")
    wide[:T, 16:16 + K] = x
    plan = _plan(ids, slots)
    got = ops.lora(wide[:T, 16:16 + K], bank, plan)
    want, err = _delta64(x, a, b, scale, widths, ids, 0.0)
    assert bool(((got.double() - want).abs() <= err + want.abs() * 2.0 ** -23 + 1e-30).all())
    assert bool((got[ids < 0] == 0).all())
    again = ops.lora(x, bank, _plan(ids, slots))            # the order of a step's rows is kept: the same sums
    assert torch.equal(got, again)


@pytest.mark.parametrize("T,rank", [(150, 16), (150, 128), (64, 128)])
def test_lora_two_launch_steps_captured_and_at_once(T, rank):
    """steps of two launches: one graph of plan, plane and gate | up replayed over changing rows and adapters, the same calls on two streams at once: the same bits"""
    from vox_serve_b200 import ops
    K, ff, slots = 328, 136, 3
    bank, a, b, scale, _, x = _inputs(T, K, (ff, ff), rank, slots, 11)
    planes = torch.randn(1, T, 2 * 3 * 48, device="cuda")
    sx, sid, plan = x.clone(), torch.zeros(T, dtype=I32, device="cuda"), ops.LoraPlan(T, slots)

    def step(rows, ids, plan):
        ops.lora_plan(plan, ids)
        before = ops.launch_count()
        out = ops.lora(rows, bank, plan), ops.lora_gate_up(rows, bank, plan, planes, 48)
        assert ops.launch_count() - before == 4
        return out
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    streams[0].wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams[0]):
        step(sx, sid, plan)
    torch.cuda.current_stream().wait_stream(streams[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(sx, sid, plan)
    cases = []
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        ids = torch.randint(-1, slots, (T,), generator=gen, device="cuda").to(I32)
        cases.append((torch.randn(T, K, generator=gen, device="cuda").to(BF16), ids if seed % 2 else ids.sort().values.contiguous()))
    want = [step(xs, ids, ops.LoraPlan(T, slots)) for xs, ids in cases]
    torch.cuda.synchronize()
    plans, at_once = [ops.LoraPlan(T, slots) for _ in cases], [None] * len(cases)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, (xs, ids) in enumerate(cases):
            with torch.cuda.stream(streams[i % 2]):
                at_once[i] = step(xs, ids, plans[i])
    torch.cuda.synchronize()
    for (xs, ids), w, o in zip(cases, want, at_once):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
        sx.copy_(xs)
        sid.copy_(ids)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
