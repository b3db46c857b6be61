"""A step of a beam search (ops.beam_select) and the states that follow it (ops.beam_reorder) against plain forms in 64 bits.

Tolerance of a total, derived: a row's sum of exponentials has terms off by 2^-22 (the special function unit) and by half a step of their exponent, at most 40 * 2^-24 for
terms that count, and passes 20 additions; together under 2^-18 of the sum, which is the error of its logarithm.  The total is rounded once (half a step: 2^-24 of it).
Within a beam nothing is rounded that orders candidates: its tokens have to be the first of its logits' order, equal ones by number."""
import math

import pytest
import torch

from vox_serve_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
INF, NAN = math.inf, math.nan


def _plain(logits, scores, weight=None, ended=None, end=None):
    """(totals, ranks) [B, W * V] in 64 bits on the CPU, -inf: no candidate"""
    B, W = scores.shape
    z = logits.detach().cpu().to(F64).view(B, W, -1).clone()
    z[~torch.isfinite(z)] = -INF
    s = scores.cpu().to(F64)[:, :, None]
    top = z.max(2, keepdim=True)[0]
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    total = s + ((z - top) - torch.log(torch.exp(z - top).sum(2, keepdim=True)))      # (a row of lowest values alone: x - top first)
    w = torch.ones(B, W, 1, dtype=F64) if weight is None else weight.cpu().to(F64)[:, :, None]
    alive = torch.isfinite(s) & torch.isfinite(w) & (w > 0) & torch.isfinite(z).any(2, keepdim=True)
    if ended is not None:
        over = ended.cpu()[:, :, None]
        alive = torch.isfinite(s) & torch.isfinite(w) & (w > 0) & (over | torch.isfinite(z).any(2, keepdim=True))
        only = torch.full_like(total, -INF)
        only[:, :, end] = s[:, :, 0]
        total = torch.where(over, only, total)
    total = torch.where(alive & (total > -INF), total, torch.full_like(total, -INF))
    rank = torch.where(total > -INF, total * torch.where(alive, w, torch.ones_like(w)), total)
    return total.view(B, -1), rank.view(B, -1)


def _check(step, logits, scores, n, weight=None, ended=None, end=None, exact=False):
    B, W = scores.shape
    V = logits.shape[1]
    total, rank = _plain(logits, scores, weight, ended, end)
    got_s, got_p, got_t = step.scores.cpu().to(F64), step.parent.cpu().long(), step.token.cpu()
    assert got_s.shape == got_p.shape == got_t.shape == (B, n)
    want_rank, want = torch.sort(rank, dim=1, descending=True, stable=True)
    z = logits.detach().cpu().to(F64).view(B, W, V).clone()
    z[~torch.isfinite(z)] = -INF
    for b in range(B):
        have = min(n, int((rank[b] > -INF).sum()))
        assert (got_p[b, have:] == -1).all() and (got_t[b, have:] == -1).all() and (got_s[b, have:] == -INF).all()
        at = got_p[b, :have] * V + got_t[b, :have]
        assert (got_p[b, :have] >= 0).all() and (got_t[b, :have] >= 0).all() and len(set(at.tolist())) == have
        tol = 2.0 ** -18 + 2.0 ** -23 * total[b][at].abs()
        assert ((got_s[b, :have] - total[b][at]).abs() <= tol).all()
        if exact:
            assert torch.equal(at, want[b, :have])
        big = 1.0 if weight is None else float(weight[b][torch.isfinite(weight[b]) & (weight[b] > 0)].max())
        slack = 2 * big * (2.0 ** -18) + 2.0 ** -50 * want_rank[b, :have].abs()
        assert (rank[b][at] >= want_rank[b, :have] - slack).all()
        for w in range(W):
            mine = got_t[b, :have][got_p[b, :have] == w]
            if ended is not None and bool(ended[b, w]):
                assert mine.tolist() in ([], [end])
            else:
                assert torch.equal(mine, torch.sort(z[b, w], descending=True, stable=True)[1][:len(mine)])
        if step.ended is not None:
            over = torch.zeros(W, dtype=torch.bool) if ended is None else ended[b].cpu()
            assert torch.equal(step.ended[b, :have].cpu(), over[got_p[b, :have]] | (got_t[b, :have] == end)) and bool(step.ended[b, have:].all())


def _inputs(B, W, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * V + W)
    z = (torch.randn(B * W, V, generator=g, device="cuda") * spread).to(dtype)
    s = -30.0 * torch.rand(B, W, generator=g, device="cuda")
    return z, s


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,W,V,n", [(1, 1, 1, 1), (1, 1, 2, 4), (1, 2, 7, 4), (3, 4, 33, 8), (2, 5, 1000, 10), (1, 3, 8191, 6), (2, 2, 8192, 16), (1, 4, 8193, 17), (2, 8, 2051, 64),
                                     (1, 32, 1025, 64), (5, 1, 50000, 33), (1, 16, 32003, 32), (1, 2, 156940, 64), (40, 3, 515, 2)])
def test_select(B, W, V, n, dtype):
    z, s = _inputs(B, W, V, dtype)
    _check(ops.beam_select(z, s, n), z, s, n)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("first,stride", [(0, 1003), (1, 1000), (3, 1005), (5, 1016), (7, 999), (2, 2000)])
def test_rows_at_any_element(first, stride, dtype):
    """strides and offsets of every alignment; a beam's result does not hang on them, to the bit"""
    V = 999 - first % 2
    z, s = _inputs(2, 3, V, dtype)
    big = torch.full((6 * stride + 16,), NAN, dtype=dtype, device="cuda")
    view = torch.as_strided(big, (6, V), (stride, 1), first)
    view.copy_(z)
    a, b = ops.beam_select(view, s, 12), ops.beam_select(z, s, 12)
    _check(a, z, s, 12)
    assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3]))


def test_one_row_read_by_all():
    """a row stride of zero: beams of one distribution"""
    z, _ = _inputs(1, 1, 2051, BF16)
    s = torch.tensor([[-1.0, -2.0, -1.0]], device="cuda")
    _check(ops.beam_select(z.expand(3, 2051), s, 9), z.repeat(3, 1), s, 9, exact=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [5, 700, 9001, 40001])
def test_equal_logits(V, dtype):
    """ties everywhere: the lowest beam and token come first"""
    s = torch.zeros(2, 4, device="cuda")
    z = torch.zeros(8, V, dtype=dtype, device="cuda")
    z[:, ::2] = -0.0
    _check(ops.beam_select(z, s, 20), z, s, 20, exact=True)
    z[:, V // 2:] = 1.0
    _check(ops.beam_select(z, s, 64), z, s, 64, exact=True)


@pytest.mark.parametrize("V", [3001, 20000])
def test_equal_beams(V):
    """beams that hold the same are equal in rank: their order is the beams', whatever address their rows begin at"""
    z, _ = _inputs(1, 1, V, BF16)
    s = torch.full((1, 6), -3.5, device="cuda")
    z = z.repeat(6, 1)
    _check(ops.beam_select(z, s, 40), z, s, 40, exact=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 5, 16, 64])
def test_long_runs(n, dtype):
    """orders that a slice's first cut is worst at: rising, falling, all but a stretch masked or lowest"""
    V = 30011
    ramp = torch.linspace(-50.0, 50.0, V, device="cuda")
    low = torch.finfo(dtype).min
    rows = [ramp, ramp.flip(0), torch.where(torch.arange(V, device="cuda") < 12000, ramp, torch.full_like(ramp, -INF)),
            torch.where((torch.arange(V, device="cuda") > 9000) & (torch.arange(V, device="cuda") < 9100), ramp, torch.full_like(ramp, low)),
            torch.where(torch.arange(V, device="cuda") == 17, ramp, torch.full_like(ramp, -INF)), torch.full_like(ramp, low)]
    z = torch.stack(rows).clamp(min=-INF).to(dtype)
    z[3] = torch.where(rows[3] == low, torch.full_like(z[3], low), z[3])
    z[5] = low
    s = torch.tensor([[-1.0, -1.25, -2.5, -0.5, -40.0, -3.0]], device="cuda")
    _check(ops.beam_select(z, s, n), z, s, n)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masks(dtype):
    """-inf, +inf and NaN are masked, the type's lowest value is a value; rows without any candidate"""
    V, n = 517, 24
    z, s = _inputs(4, 3, V, dtype)
    low, top = torch.finfo(dtype).min, torch.finfo(dtype).max
    z[0] = -INF
    z[1, 5:] = -INF
    z[2, ::3] = NAN
    z[3] = NAN
    z[4, 100] = INF
    z[4, 200] = top
    z[5] = low
    z[6, :500] = low
    z[7] = top
    z[9] = -INF
    z[10] = NAN
    z[11] = INF
    _check(ops.beam_select(z, s, n), z, s, n)
    z[:, :] = -INF
    _check(ops.beam_select(z, s, n), z, s, n)


def test_scores_without_a_number():
    z, s = _inputs(3, 4, 900, BF16)
    s[0, 1:] = -INF                                        # the first step
    s[1] = torch.tensor([NAN, INF, -3.0, -INF])
    s[2] = -INF                                            # a request that is over
    _check(ops.beam_select(z, s, 10), z, s, 10)
    w = torch.full((3, 4), 0.5, device="cuda")
    w[0, 0], w[1, 2] = 0.0, NAN
    _check(ops.beam_select(z, s, 10, weight=w), z, s, 10, weight=w)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_weights(dtype):
    z, s = _inputs(4, 6, 3000, dtype)
    w = torch.rand(4, 6, device="cuda") + 0.05
    w[1, 0], w[1, 1], w[2, 3] = -1.0, INF, 1e-30
    _check(ops.beam_select(z, s, 12, weight=w), z, s, 12, weight=w)


@pytest.mark.parametrize("end", [0, 13, 1999])
def test_ended(end):
    z, s = _inputs(3, 5, 2000, BF16)
    z[:, end] += 12.0
    over = torch.zeros(3, 5, dtype=torch.bool, device="cuda")
    over[0, 1] = over[0, 4] = over[1, :] = True
    z[0 * 5 + 1] = NAN                                     # (not read)
    s[0, 4] = -INF                                         # ended, but dead
    w = torch.rand(3, 5, device="cuda") + 0.5
    for weight in (None, w):
        _check(ops.beam_select(z, s, 10, weight=weight, ended=over, end_token=end), z, s, 10, weight=weight, ended=over, end=end)
    step = ops.beam_select(z, s, 10, end_token=end)
    z2 = z.clone()
    _check(step, z2, s, 10, end=end)


def test_same_bits_on_every_run():
    z, s = _inputs(4, 8, 40000, BF16, spread=0.01)
    a = ops.beam_select(z, s, 64)
    for _ in range(5):
        assert all(torch.equal(x, y) for x, y in zip(a[:3], ops.beam_select(z, s, 64)[:3]))


def test_captured_and_on_two_streams():
    z, s = _inputs(4, 4, 30000, BF16)
    z2, s2 = _inputs(4, 4, 30000, BF16, seed=9)
    graphs = []
    for _ in range(2):
        ops.beam_select(z, s, 8)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.beam_select(z, s, 8)
        graphs.append((g, out))
    z.copy_(z2)
    s.copy_(s2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            _check(out, z2, s2, 8)


# ---- states ----------------------------------------------------------------------------------------------------------------------
def _reordered(states, parent, slots):
    out = [t.clone() for t in states]
    B, W = parent.shape
    p, sl = parent.tolist(), slots.tolist()
    for b in range(B):
        for i in range(W):
            j = p[b][i]
            if 0 <= j < W:
                for o, t in zip(out, states):
                    o[sl[b][i]] = t[sl[b][j]]
    return out


@pytest.mark.parametrize("B,W", [(1, 1), (1, 2), (2, 4), (3, 5), (2, 8), (1, 9), (2, 16), (1, 17), (2, 32)])
@pytest.mark.parametrize("own_slots", [False, True])
def test_reorder(B, W, own_slots):
    g = torch.Generator(device="cuda").manual_seed(B * 100 + W)
    S = B * W + 5
    states = [torch.randn(S, 4, 33, generator=g, device="cuda"), torch.randn(S, 903, generator=g, device="cuda").to(BF16), torch.randn(S, 2048, generator=g, device="cuda"),
              torch.randint(0, 100, (S, 3), generator=g, device="cuda").to(torch.uint8), torch.randint(0, 9, (S,), generator=g, device="cuda"),
              torch.randint(0, 9, (S,), generator=g, device="cuda").to(I32), torch.randn(S, 6, generator=g, device="cuda").to(BF16), torch.rand(S, 17, generator=g, device="cuda") > 0.5]
    slots = (torch.randperm(S, generator=g, device="cuda")[:B * W] if own_slots else torch.arange(B * W, device="cuda")).to(I32).view(B, W)
    for parent in (torch.randint(-1, W, (B, W), generator=g, device="cuda"), torch.arange(W - 1, -1, -1, device="cuda").expand(B, W), torch.arange(W, device="cuda").roll(1).expand(B, W),
                   torch.zeros(B, W, device="cuda"), torch.full((B, W), W, device="cuda"), torch.arange(W, device="cuda").expand(B, W)):
        parent = parent.to(I32).contiguous()
        want = _reordered(states, parent, slots)
        ops.beam_reorder(states, parent, slots if own_slots else None)
        for a, b in zip(states, want):
            assert torch.equal(a, b)


def test_reorder_of_many_states_and_unaligned_rows():
    g = torch.Generator(device="cuda").manual_seed(3)
    base = [torch.randn(7 * k + 8, generator=g, device="cuda") for k in range(1, 151)]
    states = [t[k % 4:k % 4 + 7 * (k + 1)].view(7, k + 1) for k, t in enumerate(base)]
    parent = torch.tensor([[2, 0, 1], [0, 0, 2]], dtype=I32, device="cuda")
    slots = torch.tensor([[6, 0, 3], [1, 5, 2]], dtype=I32, device="cuda")
    want = _reordered(states, parent, slots)
    before = ops.launch_count()
    ops.beam_reorder(states, parent, slots)
    assert ops.launch_count() - before == 3
    for a, b in zip(states, want):
        assert torch.equal(a, b)


def test_reorder_skips_slots_that_are_none():
    t = torch.arange(12.0, device="cuda").view(6, 2)
    want = t.clone()
    want[1] = t[0]
    ops.beam_reorder([t], torch.tensor([[0, 0, 0, 3]], dtype=I32, device="cuda"), torch.tensor([[0, 1, 6, -1]], dtype=I32, device="cuda"))
    assert torch.equal(t, want)
    ops.beam_reorder([t], torch.tensor([[2, 3, 0, 0]], dtype=I32, device="cuda"), torch.tensor([[0, 1, 6, -1]], dtype=I32, device="cuda"))
    assert torch.equal(t, want)


def test_reorder_of_a_large_state():
    """rows beyond 2^31 bytes from the first"""
    t = torch.zeros(12, 60_000_000, dtype=torch.int32, device="cuda")      # 2.9 GB
    t[:, -1] = torch.arange(12, device="cuda", dtype=torch.int32)
    t[:, 0] = 100 + torch.arange(12, device="cuda", dtype=torch.int32)
    ops.beam_reorder([t], torch.tensor([[3, 0, 1, 2]], dtype=I32, device="cuda"), torch.tensor([[11, 10, 1, 0]], dtype=I32, device="cuda"))
    assert t[:, -1].tolist() == [1, 10, 2, 3, 4, 5, 6, 7, 8, 9, 11, 0] and t[:, 0].tolist() == [101, 110, 102, 103, 104, 105, 106, 107, 108, 109, 111, 100]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_largest_vocabulary(dtype):
    z, s = _inputs(1, 1, 1 << 24, dtype)
    _check(ops.beam_select(z, s, 3), z, s, 3)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [9, 40, 12345])
def test_everything_at_once(V, dtype):
    """weights, beams that ended, dead ones, masks, rows apart, requests with fewer candidates than are asked for, one with none"""
    B, W, n, end = 4, 6, 50, 3
    z, s = _inputs(B, W, V + 5, dtype, seed=3)
    z = z[:, 2:2 + V]
    weight = torch.rand(B, W, device="cuda") + 0.2
    ended = torch.zeros(B, W, dtype=torch.bool, device="cuda")
    ended[0, 1] = ended[1, 2] = ended[1, 5] = True
    s[0, 3], s[2, 1:], s[3, :] = -INF, -INF, -INF
    ended[2, 4] = True                                       # (dead: its ended bit does not wake it)
    weight[1, 0], weight[0, 5] = 0.0, NAN
    z[W + 3] = -INF
    z[::2, V // 2:] = torch.finfo(dtype).min
    z[1::2, :V // 3] = -INF
    _check(ops.beam_select(z, s, n, weight=weight, ended=ended, end_token=end), z, s, n, weight, ended, end)


def _row_of_top(top, V, dtype, kind):
    """fp32 row whose largest value is ``top``: alone in its thread's share of the row, everywhere, or above values that 64 bits tell apart beside it"""
    t = torch.tensor(top, dtype=F32, device="cuda")
    if kind == "alone":
        z = torch.full((V,), -INF, device="cuda")
        z[V // 3] = t
    elif kind == "equal":
        z = torch.full((V,), top, device="cuda")
    else:
        z = t - t.abs() * (torch.arange(V, device="cuda").roll(V // 2) % 977) / 1024
    return z.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["alone", "equal", "lower"])
def test_large_logits(kind, dtype):
    """a maximum whose product with log2 e is rounded by up to 2^127: no term is lost, of either sign, at any size"""
    V, n = 2500, 12
    tops = [1600008448.0, 2000003840.0, 2500027136.0, 4000063488.0, 1073741760.0, 1073741824.0, 1488522240.0, 1.4e9] + [float(10 ** k) for k in range(3, 37)]
    tops = [x for t in tops for x in (t, -t)]
    z = torch.stack([_row_of_top(t, V, dtype, kind) for t in tops])
    s = torch.full((len(tops) // 2, 2), -1.5, device="cuda")
    s[:, 1] = -2.0
    step = ops.beam_select(z, s, n)
    _check(step, z, s, n)
    one = s.view(-1, 1)                                     # each row as a request of its own
    step = ops.beam_select(z, one, n)
    _check(step, z, one, n)
    assert bool((step.parent[:, 0] == 0).all())


def test_every_size_of_a_single_logit():
    """one open token a row: its total is the row's score, whatever the logit"""
    g = torch.Generator(device="cuda").manual_seed(5)
    e = torch.rand(20000, generator=g, device="cuda", dtype=F64) * 126 * (1 - 2 * (torch.arange(20000, device="cuda") % 2))
    x = torch.exp2(e).to(F32) * torch.where(torch.rand(20000, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    near = torch.exp2(29.5 + 5.0 * torch.rand(20000, generator=g, device="cuda", dtype=F64)).to(F32)
    x = torch.cat([x, near, -near])
    s = -40.0 * torch.rand(x.numel(), 1, generator=g, device="cuda")
    z = torch.full((x.numel(), 9), -INF, device="cuda")
    z[:, 4] = x
    step = ops.beam_select(z, s, 1)
    assert bool((step.token == 4).all()) and bool((step.parent == 0).all())
    assert bool(((step.scores - s).abs() <= 2.0 ** -18 + 2.0 ** -23 * s.abs()).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,W,V,n", [(64, 4, 32003, 8), (74, 8, 2051, 16), (300, 8, 515, 5), (148, 1, 20000, 2), (700, 1, 33, 3), (222, 2, 9000, 4), (5000, 2, 12, 4)])
def test_many_requests(B, W, V, n, dtype):
    """more requests than run at once as clusters, and as many as do: a workspace in the first case, none in the second, the same choices"""
    z, s = _inputs(B, W, V, dtype)
    s[::3, W - 1] = -INF
    _check(ops.beam_select(z, s, n), z, s, n)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_launch_only_where_all_requests_run_at_once(dtype):
    """the workspace grows from none to some with the requests, and never back; one request is one launch up to eight parts"""
    f32 = dtype is F32
    for W, V in ((1, 2051), (2, 2051), (4, 2051), (8, 2051), (3, 500)):
        none = [ops._beam_ws(B, W, V, 4, f32) == 0 for B in (1, 2, 8, 32, 60, 200, 400, 800, 2000)]
        assert none[0] and not none[-1] and none == sorted(none, reverse=True)
    z, s = _inputs(3, 4, 700, dtype)
    for B, launches in ((3, 1), (900, 2)):
        zz, ss = z.repeat(B // 3, 1), s.repeat(B // 3, 1)
        before = ops.launch_count()
        step = ops.beam_select(zz, ss, 5)
        assert ops.launch_count() - before == launches
        _check(step, zz, ss, 5)


def test_reorder_of_a_slot_named_twice():
    """in a request: the last of its beams that move, in every column"""
    t = torch.arange(6.0, device="cuda")[:, None].repeat(1, 5000).contiguous()
    ops.beam_reorder([t], torch.tensor([[2, 3, 2, 3]], dtype=I32, device="cuda"), torch.tensor([[4, 4, 1, 0]], dtype=I32, device="cuda"))
    assert bool((t[4] == 0).all()) and bool((t[[0, 1, 2, 3, 5]] == torch.tensor([0.0, 1, 2, 3, 5], device="cuda")[:, None]).all())
    ops.beam_reorder([t], torch.tensor([[2, 1, 2, 3]], dtype=I32, device="cuda"), torch.tensor([[4, 4, 1, 0]], dtype=I32, device="cuda"))
    assert bool((t[4] == 1).all())
