"""Page tables on the device (ops.fork_pages, ops.compact_pages) against the same steps in Python lists.  Everything is whole numbers or moved bytes: equal, or wrong."""
import random

import pytest
import torch

from vox_serve_b200 import ops
from vox_serve_b200._lib import VoxB200Error

pytestmark = pytest.mark.gpu

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


class Plain:
    """tables as lists; caches as tensors on the CPU"""

    def __init__(self, pages, P, rows, columns, caches):
        self.pages, self.P, self.rows, self.columns = pages, P, rows, columns
        self.table = [[] for _ in range(rows)]
        self.tokens = [0] * rows
        self.caches = caches

    def refs(self):
        r = [0] * self.pages
        for t in self.table:
            for p in t:
                r[p] += 1
        return r

    def step(self, src, grow):
        """False: nothing changed"""
        P = self.P
        table = [list(self.table[s]) if 0 <= s < self.rows else [] for s in src]
        tokens = [self.tokens[s] if 0 <= s < self.rows else 0 for s in src]
        keeper = {}
        for i, (t, n) in enumerate(zip(table, tokens)):
            if n % P:
                keeper.setdefault(t[n // P], i)
        held = {p for t in table for p in t}
        free = iter([p for p in range(self.pages) if p not in held])
        copies, ok = [], True
        for i, (t, n) in enumerate(zip(table, tokens)):
            if not 0 <= src[i] < self.rows:
                continue
            want = -(-(n + max(grow[i], 0)) // P)
            ok = ok and want <= self.columns
            try:
                if n % P and keeper[t[n // P]] != i:
                    new = next(free)
                    copies.append((t[n // P], new, n % P))
                    t[n // P] = new
                while len(t) < min(want, self.columns):
                    t.append(next(free))
            except StopIteration:
                ok = False
            tokens[i] = n + max(grow[i], 0)
        if not ok:
            return False
        for a, b, n in copies:
            for c, kind in self.caches:
                if kind == "kv":
                    c[:, b, :, :n] = c[:, a, :, :n].clone()
                elif kind == "layer":
                    c[b, :, :n] = c[a, :, :n].clone()
                elif kind == "tokens":
                    c[b, :n] = c[a, :n].clone()
                else:
                    c[b] = c[a].clone()
        self.table, self.tokens = table, tokens
        return True

    def compact(self):
        refs = self.refs()
        used = sum(r > 0 for r in refs)
        holes = [p for p in range(used) if not refs[p]]
        movers = [p for p in range(used, self.pages) if refs[p]]
        new = [p if r else -1 for p, r in enumerate(refs)]
        for a, b in zip(movers, holes):
            new[a] = b
            for c, kind in self.caches:
                if kind == "kv":
                    c[:, b] = c[:, a].clone()
                else:
                    c[b] = c[a].clone()
        self.table = [[new[p] for p in t] for t in self.table]
        return new, used

    def same_as(self, pool, caches):
        want = [t + [-1] * (self.columns - len(t)) for t in self.table]
        assert pool.table.cpu().tolist() == want
        assert pool.tokens.tolist() == self.tokens
        assert pool.refs.tolist() == self.refs()
        for (c, _), t in zip(self.caches, caches):
            assert torch.equal(c, t.cpu())


def _make(pages, P, rows, columns, seed=0, kinds=("kv", "tokens", "layer", "page")):
    g = torch.Generator().manual_seed(seed)
    shapes = {"kv": (3, pages, 2, P, 2, 8), "tokens": (pages, P, 1, 24), "layer": (pages, 2, P, 1, 8), "page": (pages, 3, 2, 4)}
    host = [(torch.randn(shapes[k], generator=g).to(F32 if k == "page" else BF16), k) for k in kinds]
    return Plain(pages, P, rows, columns, host), ops.PagePool(pages, P, rows, columns), [c.cuda() for c, _ in host]


def _i32(v):
    return torch.tensor(v, dtype=I32, device="cuda")


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("P", [1, 5, 16, 64])
@pytest.mark.parametrize("rows", [1, 6, 33])
def test_a_life_of_steps(rows, P, apart):
    """prompts, forks, exchanges, rows that leave and come back, in place and from one pool to another"""
    rng = random.Random(rows * 100 + P)
    pages, columns = rows * 8 + 3, 12
    plain, pool, caches = _make(pages, P, rows, columns, seed=P)
    other = ops.PagePool(pages, P, rows, columns)
    for step in range(30):
        src = [rng.choice([i, i, rng.randrange(-1, rows), rng.randrange(rows)]) for i in range(rows)] if step else list(range(rows))
        grow = [rng.choice([0, 1, 1, P, 2 * P + 1, -3]) if step else rng.randrange(0, 3 * P) for _ in range(rows)]
        out = other if apart else pool
        before = (pool.table.clone(), pool.tokens.clone(), pool.refs.clone())
        ok = plain.step(src, grow)
        ops.fork_pages(pool, _i32(src), _i32(grow), caches=caches, out=out)
        if ok:
            out.check()
        else:
            with pytest.raises(VoxB200Error):
                out.check()
            assert torch.equal(out.table, before[0]) and torch.equal(out.tokens, before[1]) and torch.equal(out.refs, before[2])
        plain.same_as(out, caches)
        if apart:
            assert torch.equal(pool.table, before[0]) and torch.equal(pool.refs, before[2])
            pool, other = other, pool
        if step % 7 == 5:
            new, used = plain.compact()
            out = other if apart else pool
            ops.compact_pages(pool, caches=caches, out=out)
            plain.same_as(out, caches)
            assert out.moved.tolist() == new and int(out.status[3]) == used
            if apart:
                pool, other = other, pool


def test_groups_and_one_number():
    plain, pool, caches = _make(40, 16, 6, 5)
    assert plain.step(list(range(6)), [37] * 6)
    ops.fork_pages(pool, grow=37)
    plain.same_as(pool, caches)
    parent = [[2, 0, 0], [1, 1, -1]]
    assert plain.step([2, 0, 0, 4, 4, -1], [1] * 6)
    ops.fork_pages(pool, _i32(parent), 1, caches=caches)
    pool.check()
    plain.same_as(pool, caches)
    assert plain.step([1, 2, 0, 3, 4, -1], [0] * 6)
    ops.fork_pages(pool, _i32([1, 2, 0, 0, 1, 3]), caches=caches, group=3)      # (3 is outside its group: none)
    plain.same_as(pool, caches)
    assert plain.step([-1] * 6, [5] * 6)
    ops.fork_pages(pool, _i32([-1, 6, 7, 1 << 30, -5, 9]), 5)
    plain.same_as(pool, caches)


def test_short_of_pages_changes_nothing():
    plain, pool, caches = _make(10, 16, 4, 8)
    assert plain.step([0, 1, 2, 3], [20, 32, 0, 0])
    ops.fork_pages(pool, grow=_i32([20, 32, 0, 0]))
    state = [t.clone() for t in (pool.table, pool.tokens, pool.refs)]
    kept = [c.clone() for c in caches]
    ops.fork_pages(pool, _i32([0, 0, 0, 0]), _i32([40, 40, 40, 40]), caches=caches)      # 3 copies and 8 pages, of which 8 are free
    with pytest.raises(VoxB200Error, match="3 pages are missing"):
        pool.check()
    for a, b in zip(state, (pool.table, pool.tokens, pool.refs)):
        assert torch.equal(a, b)
    for a, b in zip(kept, caches):
        assert torch.equal(a, b)
    ops.fork_pages(pool, grow=_i32([0, 97, 0, 0]))
    with pytest.raises(VoxB200Error, match="1 rows grew past 8 pages"):
        pool.check()
    ops.fork_pages(pool, grow=0x3fffffff)
    with pytest.raises(VoxB200Error):
        pool.check()
    for a, b in zip(state, (pool.table, pool.tokens, pool.refs)):
        assert torch.equal(a, b)
    assert plain.step([0, 0, 0, 0], [28, 0, 0, 0])
    ops.fork_pages(pool, _i32([0, 0, 0, 0]), _i32([28, 0, 0, 0]), caches=caches)
    pool.check()
    plain.same_as(pool, caches)


@pytest.mark.parametrize("rows,columns,P", [(64, 700, 16), (300, 90, 2), (4096, 3, 4), (4096, 2, 7), (4096, 1, 9), (2, 5000, 1), (1, 8000, 3), (33, 33, 64)])
def test_large_tables(rows, columns, P):
    """tables that several blocks share, pools that are searched in steps"""
    rng = random.Random(rows)
    pages = rows * columns + 10
    plain, pool, caches = _make(pages, P, rows, columns, kinds=())
    grow = [rng.randrange(0, columns * P // 3) for _ in range(rows)]
    assert plain.step(list(range(rows)), grow)
    ops.fork_pages(pool, grow=_i32(grow))
    plain.same_as(pool, caches)
    for _ in range(3):
        src = [rng.randrange(-1, rows) for _ in range(rows)]
        grow = [rng.randrange(0, max(1, columns * P // 10) + 1) for _ in range(rows)]
        assert plain.step(src, grow)
        ops.fork_pages(pool, _i32(src), _i32(grow))
        pool.check()
        plain.same_as(pool, caches)
    new, used = plain.compact()
    ops.compact_pages(pool)
    plain.same_as(pool, caches)
    assert pool.moved.tolist() == new and int(pool.status[3]) == used


@pytest.mark.parametrize("pages,held", [(1, []), (1, [0]), (9, []), (9, [8]), (9, list(range(9))), (6000, [5999, 0, 4100, 4095, 4096])])
def test_compact_ends(pages, held):
    plain, pool, caches = _make(pages, 16, 2, max(1, len(held)), kinds=("kv",))
    plain.table[1], plain.tokens[1] = list(held), 16 * len(held)
    table = torch.full((2, max(1, len(held))), -1, dtype=I32)
    table[1, :len(held)] = torch.tensor(held, dtype=I32)
    pool.load(table.cuda(), _i32([0, 16 * len(held)]))
    new, used = plain.compact()
    ops.compact_pages(pool, caches=caches)
    plain.same_as(pool, caches)
    assert pool.moved.tolist() == new and int(pool.status[3]) == used


def test_tables_that_name_no_pages():
    """numbers outside the pool are passed over: nothing is read or written through them"""
    pool = ops.PagePool(6, 16, 4, 3)
    pool.table.copy_(_i32([[0, 99, -7], [1 << 30, 2, -1], [-(1 << 31), -1, -1], [5, -1, -1]]))
    pool.tokens.copy_(_i32([40, 20, 3, 1 << 30]))
    pool.refs.copy_(_i32([1, 0, 1, 0, 0, 1]))
    kv = torch.randn(1, 6, 2, 16, 2, 8, device="cuda").to(BF16)
    before = kv.clone()
    ops.fork_pages(pool, _i32([1, 0, 2, -1]), 0, caches=[kv])
    torch.cuda.synchronize()
    assert torch.equal(kv, before)
    assert pool.table[0].tolist() == [1 << 30, 2, -1] and pool.table[1].tolist() == [0, 99, -7] and pool.refs.tolist() == [1, 0, 1, 0, 0, 0]
    ops.compact_pages(pool, caches=[kv])
    torch.cuda.synchronize()
    assert pool.table[1].tolist() == [0, 99, -7] and pool.table[0].tolist() == [1 << 30, 1, -1] and torch.equal(kv[:, 1], before[:, 2])


def test_many_caches_in_one_step():
    P, pages = 16, 12
    plain, pool, _ = _make(pages, P, 4, 3, kinds=())
    caches = [torch.randn(pages, P, 1, 8 * (1 + i % 3), device="cuda").to(BF16) for i in range(70)]
    plain.caches = [(c.cpu().clone(), "tokens") for c in caches]
    assert plain.step([0, 1, 2, 3], [21, 0, 0, 0])
    ops.fork_pages(pool, grow=_i32([21, 0, 0, 0]))
    assert plain.step([0, 0, 0, 0], [1, 1, 1, 1])
    before = ops.launch_count()
    ops.fork_pages(pool, _i32([0, 0, 0, 0]), 1, caches=caches)
    assert ops.launch_count() - before == 4
    plain.same_as(pool, caches)


def test_a_cache_beyond_32_bits():
    """pages whose bytes stand beyond 2^32 from the first; the last tokens of a page and nothing behind them"""
    P, pages = 16, 33000
    kv = torch.zeros(1, pages, 2, P, 8, 256, dtype=BF16, device="cuda")      # 4.3 GB
    pool = ops.PagePool(pages, P, 3, 2)
    pool.load(_i32([[32999, -1], [-1, -1], [-1, -1]]), _i32([7, 0, 0]))
    pool.refs[:32990] = 1
    kv[0, 32999] = torch.randn(2, P, 8, 256, device="cuda").to(BF16)
    ops.fork_pages(pool, _i32([0, 0, -1]), 0, caches=[kv])
    pool.check()
    assert pool.table[1].tolist() == [32990, -1]
    assert torch.equal(kv[0, 32990, :, :7], kv[0, 32999, :, :7]) and not bool(kv[0, 32990, :, 7:].any())
    pool.refs[:32990] = 0
    ops.compact_pages(pool, caches=[kv])
    assert pool.table[:2, 0].tolist() == [1, 0] and torch.equal(kv[0, 1], kv[0, 32999]) and torch.equal(kv[0, 0], kv[0, 32990])


def test_captured_steps():
    plain, pool, caches = _make(60, 16, 6, 8, kinds=("kv",))
    src, grow = _i32(list(range(6))), _i32([30] * 6)
    with torch.cuda.stream(torch.cuda.Stream()):
        g = torch.cuda.CUDAGraph()
        ops.fork_pages(pool, src, grow, caches=caches)
        torch.cuda.synchronize()
        assert plain.step(list(range(6)), [30] * 6)
        with torch.cuda.graph(g):
            ops.fork_pages(pool, src, grow, caches=caches)
        rng = random.Random(5)
        for _ in range(12):
            s, n = [rng.randrange(6) for _ in range(6)], [1] * 6
            src.copy_(_i32(s))
            grow.copy_(_i32(n))
            g.replay()
            torch.cuda.synchronize()
            assert plain.step(s, n)
            plain.same_as(pool, caches)


@pytest.mark.parametrize("apart", [False, True])
def test_a_shortage_stays_until_it_is_asked_for(apart):
    """steps behind one that ran short change nothing, though they could go on; rows have no tokens to see meanwhile; compacting does not forget it"""
    plain, pool, caches = _make(10, 16, 4, 8)
    other = ops.PagePool(10, 16, 4, 8)

    def turn(f):
        nonlocal pool, other
        out = f(pool, other if apart else pool)
        if apart:
            pool, other = other, pool
        return out
    assert plain.step([0, 1, 2, 3], [20, 32, 5, 0])
    turn(lambda a, out: ops.fork_pages(a, grow=_i32([20, 32, 5, 0]), out=out))
    assert torch.equal(pool.live, pool.tokens)
    for src, grow in (([0, 0, 0, 0], [40] * 4), ([0, 1, 2, 3], [1] * 4), ([0, 1, -1, -1], [0] * 4), ([0, 1, 2, 3], [8 * 16 + 1, 0, 0, 0])):
        turn(lambda a, out: ops.fork_pages(a, _i32(src), _i32(grow), caches=caches, out=out))
        plain.same_as(pool, caches)
        assert pool.status[:3].tolist() == [3, 0, 0] and not bool(pool.live.any())      # 3 copies and 8 pages, of which 8 are free
    plain.compact()
    turn(lambda a, out: ops.compact_pages(a, caches, out=out))
    plain.same_as(pool, caches)
    assert not bool(pool.live.any())
    with pytest.raises(VoxB200Error, match="3 pages are missing"):
        pool.check()
    assert torch.equal(pool.live, pool.tokens)
    pool.check()
    assert plain.step([0, 1, 1, -1], [1] * 4)
    turn(lambda a, out: ops.fork_pages(a, _i32([0, 1, 1, -1]), 1, caches=caches, out=out))
    pool.check()
    plain.same_as(pool, caches)
    assert torch.equal(pool.live, pool.tokens)
    # rows that outgrow their columns stay said too
    turn(lambda a, out: ops.fork_pages(a, grow=_i32([0, 8 * 16, 0, 0]), out=out))
    turn(lambda a, out: ops.fork_pages(a, grow=_i32([0, 0, 0, 0]), out=out))
    with pytest.raises(VoxB200Error, match="1 rows grew past 8 pages"):
        pool.check()
    plain.same_as(pool, caches)
    # other tables begin anew
    turn(lambda a, out: ops.fork_pages(a, grow=4000, out=out))
    pool.load(pool.table.clone(), pool.tokens.clone())
    pool.check()
    assert torch.equal(pool.live, pool.tokens)


@pytest.mark.parametrize("rows,columns,pages", [(64, 700, 9000), (300, 90, 400)])
def test_live_rows_of_large_tables(rows, columns, pages):
    """several blocks, counts in shared memory and not: live is tokens, and 0 everywhere once a step has run short"""
    plain, pool, caches = _make(pages, 2, rows, columns, kinds=())
    grow = [(i * 7) % 3 for i in range(rows)]
    assert plain.step(list(range(rows)), grow)
    ops.fork_pages(pool, grow=_i32(grow))
    assert pool.live.tolist() == plain.tokens
    ops.fork_pages(pool, grow=columns * 2)
    ops.fork_pages(pool, grow=0)
    plain.same_as(pool, caches)
    assert not bool(pool.live.any())
    with pytest.raises(VoxB200Error):
        pool.check()


def test_pools_of_a_c_caller_without_live_rows():
    import ctypes

    from vox_serve_b200 import _lib
    plain, pool, caches = _make(10, 16, 4, 8, kinds=())
    s = _lib.PagePoolStruct.from_buffer_copy(pool._struct)
    s.d_live = None
    pool.live.fill_(77)
    ops.call("vb_fork_pages", ctypes.addressof(s), ctypes.addressof(s), None, 0, None, 5, None, 0, torch.cuda.current_stream().cuda_stream)
    ops.call("vb_compact_pages", ctypes.addressof(s), ctypes.addressof(s), None, 0, torch.cuda.current_stream().cuda_stream)
    assert plain.step([0, 1, 2, 3], [5] * 4)
    plain.same_as(pool, caches)
    assert bool((pool.live == 77).all())


@pytest.mark.parametrize("first", [0, 1])
def test_a_layer_beside_the_stack_it_begins(first):
    """all layers follow, whichever of the two stands in front"""
    plain, pool, caches = _make(20, 16, 4, 3, kinds=("kv",))
    both = [caches[0], caches[0][0]] if first else [caches[0][0], caches[0]]
    assert plain.step([0, 1, 2, 3], [21, 3, 0, 40])
    ops.fork_pages(pool, grow=_i32([21, 3, 0, 40]))
    assert plain.step([0, 0, 1, -1], [1] * 4)
    ops.fork_pages(pool, _i32([0, 0, 1, -1]), 1, caches=both)
    plain.same_as(pool, caches)
    assert plain.step([-1, 1, 2, -1], [0] * 4)
    ops.fork_pages(pool, _i32([-1, 1, 2, -1]), 0, caches=both)
    plain.compact()
    ops.compact_pages(pool, caches=both)
    plain.same_as(pool, caches)


def test_load_refuses_shared_partial_pages_and_is_captured():
    pool = ops.PagePool(6, 4, 3, 3)
    table, tokens = _i32([[5, 1, -1], [5, 2, -1], [-1, -1, -1]]), _i32([5, 7, 0])
    pool.load(table, tokens)
    with pytest.raises(VoxB200Error, match="2 rows share a page"):
        pool.load(_i32([[5, 1, -1], [5, 1, -1], [-1, -1, -1]]), tokens)
    assert pool.refs.tolist() == [0, 1, 1, 0, 0, 2]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.load(table, tokens)
        ops.fork_pages(pool, torch.zeros(3, dtype=I32, device="cuda"), 1)
    table.copy_(_i32([[0, 3, -1], [0, 4, -1], [0, -1, -1]]))
    tokens.copy_(_i32([6, 8, 4]))
    g.replay()
    pool.check()
    assert pool.tokens.tolist() == [7, 7, 7] and pool.table.tolist() == [[0, 3, -1], [0, 1, -1], [0, 2, -1]] and pool.refs.tolist() == [3, 1, 1, 1, 0, 0]
