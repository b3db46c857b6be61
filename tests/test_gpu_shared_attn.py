"""Attention of one new token a row over pages that rows share (ops.shared_plan, ops.shared_attn) against softmax attention in 64 bits.

Tolerance, derived: q, k, v are bf16 and exact in both.  A score is a sum of D products in fp32 (a step of the matrix units may cut off: 2^-23 of the absolute sum a step, D / 16 steps), so
its exponent is off by dS = (D / 16 + 4) 2^-22 * scale * sum |q k|, and a weight by 2 dS + 2^-21 of itself (the special function unit, the rescaling).  The weights enter as two
bf16 parts (2^-17).  The output is sum of weight |v| times those, sums of at most tokens / 16 steps a warp and a few joins (2^-20 of the absolute sum here), and one rounding to bf16,
half a step: 2^-9 (the step of bf16 is 2^-8 of the value's power of two at most 2^-8 of the value)."""
import math

import pytest
import torch

from vox_serve_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
INF, NAN = math.inf, math.nan


def _exact(q, kv, table, tokens, scale):
    """(output, bound of its error before the rounding) in 64 bits; kv [pages, 2, P, H, D]"""
    R, Hq, D = q.shape
    P, H = kv.shape[2], kv.shape[3]
    out = torch.zeros(R, Hq, D, dtype=F64, device="cuda")
    err = torch.zeros_like(out)
    for r, n in enumerate(tokens.tolist()):
        if n <= 0:
            continue
        pages = table[r, :-(-n // P)].long()
        k, v = (kv[pages, i].to(F64).reshape(-1, H, D)[:n].repeat_interleave(Hq // H, 1) for i in (0, 1))
        qq = q[r].to(F64)
        s = torch.einsum("hd,nhd->hn", qq, k) * scale
        p = torch.softmax(s, 1)
        ds = (D / 16 + 4) * 2.0 ** -22 * abs(scale) * torch.einsum("hd,nhd->hn", qq.abs(), k.abs())
        out[r] = torch.einsum("hn,nhd->hd", p, v)
        rel = 2 * ds.max(1)[0] + 2.0 ** -21 + 2.0 ** -17 + 2.0 ** -20
        err[r] = 2 * rel[:, None] * torch.einsum("hn,nhd->hd", p, v.abs())
    return out, err


def _check(out, q, kv, table, tokens, scale=None):
    want, err = _exact(q, kv, table, tokens, q.shape[2] ** -0.5 if scale is None else scale)
    far = (out.to(F64) - want).abs()
    assert bool((far <= err + 2.0 ** -8 * want.abs() + 1e-30).all()), float((far - err - 2.0 ** -8 * want.abs()).max())
    assert not bool(out[tokens <= 0].any())


def _tree(B, W, prompt, new, P, seed, spare=2, dead=0):
    """requests of W rows: whole pages of the prompt are shared, behind them rows part; (table, tokens, pages)"""
    g = torch.Generator().manual_seed(seed)
    rows, n_pages = [], 0
    tokens = []
    for b in range(B):
        p = max(1, prompt - 7 * b)
        shared = p // P
        for w in range(W):
            n = p + int(torch.randint(0, new + 1, (1,), generator=g)) if new else p
            if w >= W - dead:
                rows.append([]), tokens.append(0)
                continue
            rows.append([("s", b, c) if c < shared else ("h", b, c, w // 2) if c == shared and n >= (c + 1) * P else ("o", b, c, w) for c in range(-(-n // P))])
            tokens.append(n)
    names = {}
    for t in rows:
        for x in t:
            names.setdefault(x, len(names))
    n_pages = len(names) + spare
    perm = torch.randperm(n_pages, generator=g).tolist()
    cols = max(1, max(len(t) for t in rows))
    table = torch.full((B * W, cols), -1, dtype=I32)
    for r, t in enumerate(rows):
        table[r, :len(t)] = torch.tensor([perm[names[x]] for x in t], dtype=I32)
    return table.cuda(), torch.tensor(tokens, dtype=I32).cuda(), n_pages


def _data(pages, P, R, Hq, H, D, seed, layers=1, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = torch.randn(layers, pages, 2, P, H, D, generator=g, device="cuda").to(BF16)
    return kv, (std * torch.randn(R, Hq, D, generator=g, device="cuda")).to(BF16)


def _run(q, kv, base, table, tokens, W, **kw):
    R, Hq, D = q.shape
    plan = ops.SharedPlan(R, W, table.shape[1], kv.shape[-3], Hq, kv.shape[-2], D)
    ops.shared_plan(plan, table, tokens, kv.shape[-5])
    return ops.shared_attn(q, kv, base, plan, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,W,Hq,H,P,prompt,new", [
    (1, 1, 1, 1, 16, 1, 0), (1, 1, 8, 8, 16, 15, 0), (1, 2, 4, 2, 16, 16, 1), (1, 4, 14, 2, 16, 150, 21), (2, 3, 6, 2, 48, 100, 60), (3, 8, 16, 8, 128, 700, 300),
    (2, 5, 32, 2, 48, 1000, 97), (1, 16, 4, 4, 32, 333, 33), (1, 32, 2, 1, 64, 65, 130), (2, 33, 3, 3, 16, 40, 17), (1, 7, 64, 1, 16, 90, 10), (4, 2, 24, 8, 64, 511, 2),
    (1, 3, 9, 1, 80, 161, 5), (1, 1, 64, 1, 4096, 5000, 0), (30, 4, 8, 4, 16, 60, 50)])
def test_against_64_bits(B, W, Hq, H, P, prompt, new, D):
    table, tokens, pages = _tree(B, W, prompt, new, P, seed=B + W + P)
    kv, q = _data(pages, P, B * W, Hq, H, D, seed=P + D)
    _check(_run(q, kv, 0, table, tokens, W), q, kv[0], table, tokens)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_without_tokens(D):
    """dead rows between living ones, a request without any, all without any: zeros, whatever the table holds"""
    table, tokens, pages = _tree(4, 4, 70, 20, 16, seed=1)
    tokens[5] = tokens[0] = 0
    tokens[8:12] = 0
    tokens[13] = -4
    kv, q = _data(pages, 16, 16, 4, 2, D, seed=2)
    out = torch.full_like(q, NAN)
    _check(_run(q, kv, 0, table, tokens, 4, out=out), q, kv[0], table, tokens)
    out.fill_(NAN)
    tokens.zero_()
    assert not bool(_run(q, kv, 0, table, tokens, 4, out=out).any())


@pytest.mark.parametrize("G", [1, 4, 8])
def test_peaked_and_shifted_scores(G):
    """scores of some hundred, either sign; other scales"""
    table, tokens, pages = _tree(2, 4, 300, 40, 32, seed=5)
    kv, q = _data(pages, 32, 8, 2 * G, 2, 64, seed=6, std=30.0)
    for scale in (None, -0.125, 0.0, 0.5):
        _check(_run(q, kv, 0, table, tokens, 4, sm_scale=scale), q, kv[0], table, tokens, scale)


@pytest.mark.parametrize("W,G", [(4, 1), (4, 4), (8, 8)])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_what_is_not_finite_stays_with_its_rows(bad, W, G):
    """behind a row's tokens, in free pages, and in a page of one row: the other rows' bits are those without it"""
    P, D = 16, 64
    table, tokens, pages = _tree(2, W, 75, 30, P, seed=11)
    kv, q = _data(pages, P, 2 * W, 2 * G, 2, D, seed=12)
    clean = _run(q, kv, 0, table, tokens, W).clone()
    _check(clean, q, kv[0], table, tokens)
    on = torch.zeros(pages, P, dtype=torch.bool)
    for r, n in enumerate(tokens.tolist()):
        for t in range(n):
            on[int(table[r, t // P]), t % P] = True
    on = on.cuda()
    dirty = torch.where(on[None, :, None, :, None, None], kv, torch.full_like(kv, bad))
    assert torch.equal(_run(q, dirty, 0, table, tokens, W), clean)
    r = 1                                                   # row 1's last page is its own
    page = int(table[r, (int(tokens[r]) - 1) // P])
    own = [i for i in range(2 * W) if page in table[i, :-(-int(tokens[i]) // P)].tolist()]
    dirty[0, page, 1, (int(tokens[r]) - 1) % P] = bad
    out = _run(q, dirty, 0, table, tokens, W)
    assert not bool(torch.isfinite(out[own]).any())
    rest = [i for i in range(2 * W) if i not in own]
    _check(out[rest], q[rest], kv[0], table[rest], tokens[rest])


def test_lengths_that_part_within_a_page():
    """rows that hold one page and see different numbers of its tokens"""
    P = 64
    kv, q = _data(5, P, 4, 4, 2, 128, seed=3)
    table = torch.tensor([[2, 4], [2, 4], [2, -1], [2, -1]], dtype=I32, device="cuda")
    tokens = torch.tensor([65, 128, 33, 64], dtype=I32, device="cuda")
    kv[0, 2, 1, 33:] *= 3
    _check(_run(q, kv, 0, table, tokens, 4), q, kv[0], table, tokens)
    kv[0, 2, 1, 40, 0, 5] = INF                              # row 2 does not see it
    out = _run(q, kv, 0, table, tokens, 4)
    _check(out[2:3], q[2:3], kv[0].clone().nan_to_num_(posinf=1.0), table[2:3], tokens[2:3])
    assert not bool(torch.isfinite(out[[0, 1, 3], :2, 5]).any())


def test_tables_that_name_no_pages():
    """such a column counts as no tokens"""
    P = 16
    kv, q = _data(6, P, 2, 2, 2, 64, seed=4)
    table = torch.tensor([[1, 99, 2], [1, -5, 1 << 27]], dtype=I32, device="cuda")
    tokens = torch.tensor([40, 48], dtype=I32, device="cuda")
    out = _run(q, kv, 0, table, tokens, 2)
    t2 = torch.tensor([[1, 2], [1, -1]], dtype=I32, device="cuda")
    _check(out, q, kv[0], t2, torch.tensor([24, 16], dtype=I32, device="cuda"))


def test_pages_behind_the_cache_are_zeros():
    """a plan that was made for any cache, a table that names a page this one has not: keys and values of zero, also where values are looked over again"""
    P = 16
    kv, q = _data(4, P, 2, 2, 2, 64, seed=6)
    table = torch.tensor([[1, 1 << 20], [1, 2]], dtype=I32, device="cuda")
    tokens = torch.tensor([30, 20], dtype=I32, device="cuda")
    plan = ops.SharedPlan(2, 2, 2, P, 2, 2, 64)
    padded = torch.cat([kv[0], torch.zeros_like(kv[0, :1])])
    for bad in (0.0, NAN):
        kv[0, 2, 1, 3] += bad                                # (row 1's)
        out = ops.shared_attn(q, kv, 0, ops.shared_plan(plan, table, tokens))
        _check(out[:1], q[:1], padded, torch.tensor([[1, 4]], dtype=I32, device="cuda"), tokens[:1])
    assert not bool(torch.isfinite(out[1]).any())


def test_layers_and_one_layer():
    table, tokens, pages = _tree(2, 3, 90, 9, 16, seed=8)
    kv, q = _data(pages, 16, 6, 6, 3, 64, seed=9, layers=3)
    for layer in range(3):
        out = _run(q, kv, layer * pages, table, tokens, 3)
        _check(out, q, kv[layer], table, tokens)
        assert torch.equal(out, _run(q, kv[layer], 0, table, tokens, 3))


def test_tiled_output():
    table, tokens, pages = _tree(2, 4, 90, 9, 16, seed=8)
    kv, q = _data(pages, 16, 8, 8, 4, 64, seed=9)
    rows = _run(q, kv, 0, table, tokens, 4)
    tiled = _run(q, kv, 0, table, tokens, 4, out=ops.TiledAct(8, 8 * 64, "cuda"))
    assert torch.equal(tiled.to_rows().view(8, 8, 64), rows)


def test_a_cache_beyond_32_bits():
    P, pages = 128, 17000
    kv = torch.zeros(1, pages, 2, P, 8, 128, dtype=BF16, device="cuda")      # 8.9 GB
    ids = [16999, 3, 16384, 8192, 12000]
    small, q = _data(5, P, 2, 16, 8, 128, seed=1)
    kv[0, ids] = small[0]
    table = torch.tensor([ids, ids[:4] + [7]], dtype=I32, device="cuda")
    tokens = torch.tensor([600, 500], dtype=I32, device="cuda")
    _check(_run(q, kv, 0, table, tokens, 2), q, kv[0], table, tokens)


def test_long_rows():
    """sums over 200,000 tokens in small pages"""
    P, D, n = 16, 64, 200_003
    cols = -(-n // P)
    kv, q = _data(cols + 1, P, 2, 2, 1, D, seed=21, std=0.5)
    table = torch.arange(cols, dtype=I32, device="cuda").repeat(2, 1)
    table[1, -1] = cols
    tokens = torch.tensor([n, n], dtype=I32, device="cuda")
    _check(_run(q, kv, 0, table, tokens, 2), q, kv[0], table, tokens)


def test_same_bits_on_every_run_and_with_or_without_sharing():
    """a plan that is made again, and rows that come one to a request, agree to rounding; the same call to the bit"""
    table, tokens, pages = _tree(3, 4, 200, 30, 16, seed=31)
    kv, q = _data(pages, 16, 12, 8, 4, 128, seed=32)
    a = _run(q, kv, 0, table, tokens, 4)
    for _ in range(4):
        assert torch.equal(a, _run(q, kv, 0, table, tokens, 4))
    _check(_run(q, kv, 0, table, tokens, 1), q, kv[0], table, tokens)
    _check(_run(q, kv, 0, table, tokens, 12), q, kv[0], table, tokens)


def test_captured_with_its_plan_and_on_two_streams():
    steps = []
    for seed in (41, 43):
        table, tokens, pages = _tree(2, 4, 200, 0, 16, seed=seed)
        kv, q = _data(pages, 16, 8, 8, 4, 64, seed=seed)
        plan = ops.SharedPlan(8, 4, table.shape[1], 16, 8, 4, 64)
        out = torch.empty_like(q)
        ops.shared_attn(q, kv, 0, ops.shared_plan(plan, table, tokens, pages), out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.shared_plan(plan, table, tokens, pages)
            ops.shared_attn(q, kv, 0, plan, out=out)
        steps.append((g, q, kv, table, tokens, out, torch.cuda.Stream()))
    for n in (200, 131, 16, 1):
        for s in steps:
            s[4].fill_(n)
            s[5].fill_(NAN)
        torch.cuda.synchronize()
        for s in steps:
            with torch.cuda.stream(s[6]):
                s[0].replay()
        torch.cuda.synchronize()
        for _, q, kv, table, tokens, out, _ in steps:
            _check(out, q, kv[0], table, tokens)


@pytest.mark.parametrize("bad", [NAN, INF])
def test_what_is_not_finite_where_blocks_walk_on(bad):
    """more groups and heads than blocks: a block goes on from one to the next, a second time where values are not finite"""
    B, W, G, H, P, D = 41, 2, 2, 8, 16, 64
    table, tokens, pages = _tree(B, W, 330, 25, P, seed=17)
    tokens[10:12] = 0
    kv, q = _data(pages, P, B * W, G * H, H, D, seed=18)
    clean = _run(q, kv, 0, table, tokens, W).clone()
    _check(clean, q, kv[0], table, tokens)
    on = torch.zeros(pages, P, dtype=torch.bool)
    for r, n in enumerate(tokens.tolist()):
        for t in range(n):
            on[int(table[r, t // P]), t % P] = True
    dirty = torch.where(on.cuda()[None, :, None, :, None, None], kv, torch.full_like(kv, bad))
    assert torch.equal(_run(q, dirty, 0, table, tokens, W), clean)
    own = []
    for r in (1, 30, 67):                                   # one value of a row's last token, in one head
        dirty[0, table[r, (int(tokens[r]) - 1) // P].long(), 1, (int(tokens[r]) - 1) % P, r % H, 7] = bad
        own += [i for i in range(B * W) if int(table[r, (int(tokens[r]) - 1) // P]) in table[i, :-(-int(tokens[i]) // P)].tolist()]
    out = _run(q, dirty, 0, table, tokens, W)
    rest = [i for i in range(B * W) if i not in own]
    assert torch.equal(out[rest], clean[rest])
    for r in (1, 30, 67):
        hit = out[r, r % H * G:(r % H + 1) * G]
        assert not bool(torch.isfinite(hit[:, 7]).any()) and bool(torch.isfinite(out[r].view(H, G, D)[[h for h in range(H) if h != r % H]]).all())


@pytest.mark.parametrize("rows,columns", [(8, 300), (3, 1100), (32, 140)])
def test_rows_that_share_nothing_in_their_columns(rows, columns):
    """every row its own pages, and pages that stand in several columns, of one row or of several"""
    P, D = 16, 64
    g = torch.Generator().manual_seed(rows)
    table = torch.randperm(rows * columns, generator=g).to(I32).view(rows, columns)
    table[0, 5:9] = table[0, 3]
    table[1] = table[0].roll(1)
    table[2, ::2] = table[1, ::2]
    table = table.cuda()
    tokens = torch.randint(columns * P // 2, columns * P + 1, (rows,), generator=g).to(I32).cuda()
    tokens[0] = columns * P
    kv, q = _data(rows * columns, P, rows, 2, 1, D, seed=3)
    _check(_run(q, kv, 0, table, tokens, rows), q, kv[0], table, tokens)


def test_output_over_the_queries():
    table, tokens, pages = _tree(2, 3, 200, 30, 16, seed=9)
    kv, q = _data(pages, 16, 6, 6, 3, 128, seed=10)
    want = _run(q, kv, 0, table, tokens, 3).clone()
    assert torch.equal(_run(q, kv, 0, table, tokens, 3, out=q), want)


@pytest.mark.parametrize("G", [2, 16])
def test_masked_tiles_one_behind_the_other(G):
    """every tile has its own pieces and masks, which one warp writes and four read while the next tiles are fetched: the same bits on every run, in line with 64 bits"""
    B, W, H, P, D, cols = 3, 8, 2, 16, 128, 90
    g = torch.Generator().manual_seed(2)
    table = torch.randperm(B * W * cols, generator=g).to(I32).view(B * W, cols)
    for b in range(B):                                       # every other page is held by a changing half of the rows
        for c in range(0, cols, 2):
            half = torch.randperm(W, generator=g)[:W // 2] + b * W
            table[half, c] = table[b * W, c].clone()
    table = table.cuda()
    tokens = torch.randint(cols * P - 300, cols * P + 1, (B * W,), generator=g).to(I32).cuda()
    kv, q = _data(B * W * cols, P, B * W, G * H, H, D, seed=13)
    a = _run(q, kv, 0, table, tokens, W)
    _check(a, q, kv[0], table, tokens)
    for _ in range(40):
        assert torch.equal(a, _run(q, kv, 0, table, tokens, W))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,W", [(1, 4), (3, 4), (70, 2)])
def test_a_plan_of_other_lengths(B, W, D):
    """rows for which the plan has other lengths than the step come out as zeros and the host is told; the others' bits are what they are without lengths"""
    table, tokens, pages = _tree(B, W, 200, 30, 16, seed=51)
    R = B * W
    kv, q = _data(pages, 16, R, 8, 4, D, seed=52)
    tokens[1] = -2
    plan = ops.SharedPlan(R, W, table.shape[1], 16, 8, 4, D)
    ops.shared_plan(plan, table, tokens, pages)
    want = ops.shared_attn(q, kv, 0, plan)
    assert torch.equal(ops.shared_attn(q, kv, 0, plan, tokens=tokens), want)
    torch.cuda.synchronize()
    ops.check_waits()
    step = tokens.clone()
    step[0] += 1
    step[1] = 0                                              # (none, as -2 is)
    step[R - 1] = 0
    out = ops.shared_attn(q, kv, 0, plan, tokens=step, out=torch.full_like(q, NAN))
    torch.cuda.synchronize()
    with pytest.raises(ops.VoxB200Error, match="shared pages"):
        ops.check_waits()
    ops.check_waits()
    assert not bool(out[[0, R - 1]].any()) and torch.equal(out[1:R - 1], want[1:R - 1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.shared_plan(plan, table, step, pages)
        ops.shared_attn(q, kv, 0, plan, tokens=step, out=out)
    step.copy_(tokens)
    g.replay()
    torch.cuda.synchronize()
    ops.check_waits()
    assert torch.equal(out, want)
