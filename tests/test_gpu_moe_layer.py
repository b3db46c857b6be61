"""A mixture-of-experts layer for the rows of a decode step (ops.moe_layer) against its formula in 64 bits.

Tolerances, derived: h and the matrices are bf16 and exact in both.  A chain of fp32 sums of depth d over products whose absolute sum is S is off by at most
d 2^-22 S (a step of the matrix units, 16 products, may cut off instead of rounding).  Up: width / 16 steps and 8 sums.  The activation: a few units of 2^-23 and
its slope (at most 1.2, times the other factor of a gated form; 2 u of the squared form) times the error of its argument.  It enters the second product in exact parts.
Down: three steps per 16 of ff, then sums over warps, blocks and experts.  Routing weights: exponentials and sums of at most 128 scores whose
arguments are off by (width / 32 + 40) 2^-23 of their absolute sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
LIMIT, SLOPE = 3.0, 1.702


def _rnd(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s, std=1.0: torch.randn(*s, generator=g, device="cuda") * std


def _experts(rnd, n, ff, W, act):
    m = lambda *s, std: rnd(*s, std=std).to(BF16)                                     # noqa: E731
    return (m(n, ff, W, std=W ** -0.5) if act.endswith("glu") else None, m(n, ff, W, std=W ** -0.5), m(n, W, ff, std=ff ** -0.5))


def _layer(T, W, ff, E, top, sff, act, kind, groups, keep, seed):
    from vox_serve_b200 import ops
    rnd = _rnd(seed)
    h = rnd(T, W).to(BF16)
    ex = _experts(rnd, E, ff, W, act)
    sh = tuple(None if m is None else m[0] for m in _experts(rnd, 1, sff, W, act)) if sff else None
    kw, ids = {}, None
    if kind == "table":
        kw["table"] = torch.stack([torch.randperm(E, device="cuda")[:top] for _ in range(50)]).to(I32).contiguous()
        ids = torch.randint(0, 50, (T,), device="cuda").to(I32)
    else:
        kw["weight"] = rnd(E, W, std=1.5 * W ** -0.5)
        if kind != "softmax_all":
            kw["bias"] = rnd(E, std=0.2)
        kw["groups"], kw["keep"] = groups, keep
    if sff and kind in ("sigmoid", "table"):
        kw["shared_gate"] = rnd(W, std=W ** -0.5)
    router = ops.MoeRouter(kind, top, **kw)
    w = ops.MoeWeights.pack(*ex, shared=sh, act=act, **({"limit": LIMIT, "slope": SLOPE} if act == "clamped_glu" else {}))
    return h, ex, sh, router, w, ids


def _act64(name, g, u):
    """(value, |d/dg| bound, |d/du| bound)"""
    if name == "silu_glu":
        s = g * torch.sigmoid(g)
        return s * u, 1.1 * u.abs(), s.abs()
    if name == "clamped_glu":
        gc, uc = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        s = gc * torch.sigmoid(SLOPE * gc)
        return s * (uc + 1), 1.2 * (uc + 1).abs(), s.abs()
    if name == "relu2":
        return u.clamp(min=0) ** 2, torch.zeros_like(u), 2 * u.abs()
    return torch.nn.functional.gelu(u, approximate="none" if name == "gelu" else "tanh"), torch.zeros_like(u), torch.full_like(u, 1.2)


def _expert64(ex, e, x, act, depth_sums):
    """down(act(up x)) of one row: (value, bound of its error)"""
    gate, up, down = (None if m is None else m[e].double() for m in ex)
    W, ff = up.shape[1], up.shape[0]
    d1 = (W / 16 + 16) * 2.0 ** -22
    g, eg = (None, 0.0) if gate is None else (gate @ x, d1 * (gate.abs() @ x.abs()))
    u, eu = up @ x, d1 * (up.abs() @ x.abs())
    a, dg, du = _act64(act, g, u)
    ea = dg * eg + du * eu + 1.2 * eg * eu + a.abs() * 2.0 ** -19 + u.abs() * 2.0 ** -22 + 1e-30
    if act == "relu2":
        ea = ea + eu * eu
    return down @ a, down.abs() @ ea + (3 * ff / 16 + depth_sums) * 2.0 ** -22 * (down.abs() @ (a.abs() + ea))


def _route64(router, h, ids, t):
    """the chosen experts of row t and their weights, with the smallest distance of a choice to the next best"""
    top = router.top
    if router.kind == "table":
        return router.table[int(ids[t])].tolist(), [1.0 / top] * top, math.inf, 0.0
    x = h[t].double()
    z = router.weight.double() @ x
    noise = float((h.shape[1] / 32 + 40) * 2.0 ** -23 * (router.weight.double().abs() @ x.abs()).max())
    E = z.numel()
    bias = router.bias.double() if router.bias is not None else torch.zeros_like(z)
    if router.kind == "softmax":
        z = z + bias
        pick = score = z
    elif router.kind == "sigmoid":
        score = torch.sigmoid(z)
        pick = score + bias
    else:
        score = torch.softmax(z, 0)
        pick = z
    gap = math.inf
    pick = pick.clone()
    if router.groups > 1:
        by = pick.view(router.groups, -1)
        rank = by.topk(min(2, by.shape[1]), 1)[0].sum(1) if router.kind == "sigmoid" else by.max(1)[0]
        order = torch.sort(rank, descending=True, stable=True)
        if router.keep < router.groups:
            gap = float(order[0][router.keep - 1] - order[0][router.keep])
        keep = set(order[1][:router.keep].tolist())
        for g in range(router.groups):
            if g not in keep:
                by[g] = -math.inf
    v, order = torch.sort(pick, descending=True, stable=True)
    if top < E:
        gap = min(gap, float(v[top - 1] - v[top]))
    idx = order[:top].tolist()
    s = score[order[:top]]
    if router.kind == "softmax":
        w = torch.softmax(s, 0)
    elif router.kind == "sigmoid":
        w = s / s.sum()
    else:
        w = s
    # exponentials and quotients of arguments that are off by `noise`, and the same again for the sum
    return idx, w.tolist(), gap, noise


def _check(got, h, ex, sh, router, ids, act, sums=150):
    """rows whose choice hangs on less than what rounding may change are left to the kernel (there are hardly any)"""
    skipped = 0
    for t in range(h.shape[0]):
        idx, ws, gap, noise = _route64(router, h, ids, t)
        if gap < 4 * noise:
            skipped += 1
            continue
        x = h[t].double()
        want, err = torch.zeros_like(x), torch.zeros_like(x)
        for e, w in zip(idx, ws):
            y, ey = _expert64(ex, e, x, act, sums)
            want += w * y
            err += w * ey + w * (2 * noise + 2.0 ** -17) * (y.abs() + ey)
        if sh is not None:
            y, ey = _expert64([None if m is None else m[None] for m in sh], 0, x, act, sums)
            gate = 1.0 if router.shared_gate is None else float(torch.sigmoid(router.shared_gate.double() @ x))
            want += gate * y
            err += ey + (2 * noise + 2.0 ** -17 + (h.shape[1] / 32 + 40) * 2.0 ** -23 * 3) * y.abs()
        bad = (got[t].double() - want).abs() / (err + 1e-30)
        assert bool((bad <= 1.0).all()), (t, float(bad.max()))
    assert skipped <= max(1, h.shape[0] // 8)


CASES = [  # T, W, ff, E, top, shared, act, router, groups, keep
    (1, 1024, 1024, 8, 2, 1024, "silu_glu", "softmax", 0, 0), (1, 8, 1, 1, 1, 0, "silu_glu", "softmax", 0, 0), (2, 72, 70, 4, 4, 3, "clamped_glu", "softmax", 0, 0),
    (5, 2048, 256, 8, 2, 256, "relu2", "table", 0, 0), (8, 200, 64, 33, 3, 0, "gelu", "sigmoid", 0, 0), (9, 1032, 200, 16, 4, 96, "gelu_tanh", "sigmoid", 4, 2),
    (16, 136, 130, 64, 8, 0, "silu_glu", "softmax_all", 8, 3), (17, 264, 320, 5, 2, 64, "relu2", "table", 0, 0), (33, 520, 100, 128, 8, 40, "silu_glu", "sigmoid", 0, 0),
    (64, 256, 64, 4, 4, 128, "gelu", "softmax", 0, 0), (64, 128, 192, 256, 6, 0, "clamped_glu", "softmax_all", 16, 4), (40, 96, 64, 1024, 32, 64, "silu_glu", "softmax", 0, 0),
    (31, 4096, 64, 6, 1, 0, "gelu_tanh", "softmax", 0, 0)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_layer_against_64_bits(case):
    from vox_serve_b200 import ops
    T, W, ff, E, top, sff, act, kind, groups, keep = case
    h, ex, sh, router, w, ids = _layer(*case, seed=T + W)
    got = ops.moe_layer(h, w, router, ids=ids)
    assert got.dtype == F32 and tuple(got.shape) == (T, W)
    _check(got, h, ex, sh, router, ids, act)


def test_layer_writes_its_rows_only_and_rows_stand_alone():
    from vox_serve_b200 import ops
    h, ex, sh, router, w, ids = _layer(21, 264, 128, 16, 3, 64, "silu_glu", "sigmoid", 4, 2, seed=3)
    want = ops.moe_layer(h, w, router)
    buf = torch.full((23, 300), 7.0, device="cuda")
    assert ops.moe_layer(h, w, router, out=buf[:21, 5:269]).data_ptr() == buf[:, 5:].data_ptr()
    assert torch.equal(buf[:21, 5:269], want)
    buf[:21, 5:269] = 7.0
    assert bool((buf == 7.0).all())
    perm = torch.randperm(21, device="cuda")
    assert torch.equal(ops.moe_layer(h[perm].contiguous(), w, router), want[perm])
    assert torch.equal(ops.moe_layer(h, w, router), want)                # and from run to run


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("kind", ["softmax", "sigmoid", "softmax_all"])
def test_layer_non_finite_rows_stay_among_themselves(bad, kind):
    from vox_serve_b200 import ops
    groups, keep = (0, 0) if kind == "softmax" else (4, 2)
    h, ex, sh, router, w, ids = _layer(12, 136, 64, 8, 2, 64, "silu_glu", kind, groups, keep, seed=4)
    h[5, 17] = bad
    got = ops.moe_layer(h, w, router)
    rest = torch.arange(12, device="cuda") != 5
    # (not bit for bit: the row's experts change, and sums are grouped by the step's experts; the bound holds for any grouping)
    _check(got[rest], h[rest], ex, sh, router, ids, "silu_glu")
    assert bool(got[5].isnan().any())


def test_layer_table_names_experts_twice_and_out_of_range():
    from vox_serve_b200 import ops
    rnd = _rnd(5)
    ex, W = _experts(rnd, 6, 64, 72, "relu2"), 72
    h = rnd(4, W).to(BF16)
    w = ops.MoeWeights.pack(*ex, act="relu2")
    table = torch.tensor([[2, 2, 5], [1, 7, -3], [0, 4, 0], [9, 9, 9]], dtype=I32, device="cuda")
    ids = torch.arange(4, dtype=I32, device="cuda")
    got = ops.moe_layer(h, w, ops.MoeRouter("table", 3, table=table), ids=ids)
    for t, terms in enumerate([{2: 2, 5: 1}, {1: 1}, {0: 2, 4: 1}, {}]):
        want, err = torch.zeros(W, dtype=F64, device="cuda"), torch.full((W,), 1e-30, dtype=F64, device="cuda")
        for e, n in terms.items():
            y, ey = _expert64(ex, e, h[t].double(), "relu2", 100)
            want += y * n / 3
            err += ey * n / 3 + 2.0 ** -20 * y.abs()
        assert bool(((got[t].double() - want).abs() <= err).all())


def test_layer_infinite_and_nan_matrices_reach_their_rows_only():
    from vox_serve_b200 import ops
    rnd = _rnd(6)
    gate, up, down = _experts(rnd, 4, 64, 72, "silu_glu")
    h = rnd(6, 72).to(BF16)
    table = torch.tensor([[0], [1], [2], [3], [0], [1]], dtype=I32, device="cuda")
    ids = torch.arange(6, dtype=I32, device="cuda")
    router = ops.MoeRouter("table", 1, table=table)
    want = ops.moe_layer(h, ops.MoeWeights.pack(gate, up, down), router, ids=ids)
    up[2, 5], down[3, 7] = float("nan"), float("inf")
    got = ops.moe_layer(h, ops.MoeWeights.pack(gate, up, down), router, ids=ids)
    assert torch.equal(got[[0, 1, 4, 5]], want[[0, 1, 4, 5]])
    assert bool(got[2].isnan().all()) and not bool(torch.isfinite(got[3, 7])) and torch.equal(got[3, :7], want[3, :7])


def test_layer_no_rows_and_too_many():
    from vox_serve_b200 import ops
    h, ex, sh, router, w, ids = _layer(3, 72, 64, 4, 2, 0, "silu_glu", "softmax", 0, 0, seed=7)
    assert tuple(ops.moe_layer(h[:0], w, router).shape) == (0, 72)
    for args, kw in (((torch.zeros(65, 72, dtype=BF16, device="cuda"), w, router), {}), ((h.float(), w, router), {}), ((h[:, :64], w, router), {}),
                     ((h, w, router), {"ids": torch.zeros(3, dtype=I32, device="cuda")}), ((h, w, router), {"out": torch.zeros(3, 72, dtype=BF16, device="cuda")}),
                     ((h, w, ops.MoeRouter("softmax", 2, weight=torch.zeros(5, 72, device="cuda"))), {}),
                     ((h, w, ops.MoeRouter("sigmoid", 2, weight=router.weight, shared_gate=torch.zeros(72, device="cuda"))), {})):
        with pytest.raises(ops.VoxB200Error):
            ops.moe_layer(*args, **kw)


def test_layer_captured_and_on_another_stream():
    """two graphs of one layer's weights, replayed in turn over changing rows, beside calls on another stream"""
    from vox_serve_b200 import ops
    T = 11
    h, ex, sh, router, w, ids = _layer(T, 264, 192, 16, 3, 128, "silu_glu", "softmax", 0, 0, seed=8)
    side = torch.cuda.Stream()
    graphs = []
    for n in (T, 4):
        x = h[:n].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.moe_layer(x, w, router)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.moe_layer(x, w, router)
        graphs.append((g, x, y))
    for seed in (1, 2, 3):
        rnd = _rnd(seed)
        for _, x, _ in graphs:
            x.copy_(rnd(*x.shape).to(BF16))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [ops.moe_layer(x, w, router) for _, x, _ in graphs]
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, v) for (_, _, y), v in zip(graphs, want))
