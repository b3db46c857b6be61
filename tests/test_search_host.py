"""Refusals of the operators of a search over several continuations, raised on the host before anything is launched (the launch is replaced by a record of it)."""
import ctypes

import pytest
import torch

from vox_serve_b200 import _lib, ops
from vox_serve_b200._lib import VoxB200Error

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "_need_here", lambda who, *ts: None)
    monkeypatch.setattr(ops, "_device_index", lambda: 0)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "call", lambda name, *a: calls.append(name))
    return calls


def test_cpu_tensors_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_device_index", lambda: 0)
    with pytest.raises(VoxB200Error):
        ops.beam_select(torch.zeros(2, 8), torch.zeros(1, 2), 2)
    with pytest.raises(VoxB200Error):
        ops.beam_reorder([torch.zeros(2, 8)], torch.zeros(1, 2, dtype=I32))
    with pytest.raises(VoxB200Error):
        ops.fork_pages(ops.PagePool(4, 16, 2, 2, device="cpu"))
    with pytest.raises(VoxB200Error):
        ops.compact_pages(ops.PagePool(4, 16, 2, 2, device="cpu"))
    plan = ops.SharedPlan(2, 2, 2, 16, 2, 1, 64, device="cpu")
    with pytest.raises(VoxB200Error):
        ops.shared_plan(plan, torch.zeros(2, 2, dtype=I32), torch.zeros(2, dtype=I32))
    with pytest.raises(VoxB200Error):
        ops.shared_attn(torch.zeros(2, 2, 64, dtype=BF16), torch.zeros(4, 2, 16, 1, 64, dtype=BF16), 0, plan)


def _select(logits=(6, 40), dtype=BF16, scores=(2, 3), n=4, **k):
    return ops.beam_select(torch.zeros(*logits, dtype=dtype), torch.zeros(*scores), n, **k)


def test_select_takes(launched):
    for kw in ({}, {"dtype": F32}, {"n": 1}, {"n": 64}, {"weight": torch.ones(2, 3)}, {"end_token": 39}, {"ended": torch.zeros(2, 3, dtype=torch.bool), "end_token": 0},
               {"logits": (64, 7), "scores": (2, 32)}):
        step = _select(**kw)
        n = kw.get("n", 4)
        assert step.scores.shape == step.parent.shape == step.token.shape == (2, n) and (step.ended is None) == ("end_token" not in kw)
    assert launched == ["vb_beam_select"] * 8


@pytest.mark.parametrize("kw", [{"logits": (5, 40)}, {"logits": (6, 0)}, {"dtype": torch.float16}, {"dtype": torch.int32}, {"n": 0}, {"n": 65}, {"scores": (6,)}, {"scores": (0, 3), "logits": (0, 40)},
                                {"scores": (2, 33), "logits": (66, 40)}, {"weight": torch.ones(6)}, {"weight": torch.ones(2, 3, dtype=BF16)},
                                {"ended": torch.zeros(2, 3, dtype=torch.bool)}, {"ended": torch.zeros(2, 3), "end_token": 1}, {"end_token": 40}, {"end_token": -1},
                                {"weight": torch.ones(3, 2).t()}])
def test_select_refuses(launched, kw):
    with pytest.raises(VoxB200Error):
        _select(**kw)
    assert launched == []


def test_select_refuses_columns_apart(launched):
    with pytest.raises(VoxB200Error):
        ops.beam_select(torch.zeros(40, 6).t(), torch.zeros(2, 3), 4)
    ops.beam_select(torch.zeros(6, 80)[:, 1:40], torch.zeros(2, 3), 4)
    assert launched == ["vb_beam_select"]


def test_reorder(launched):
    par = torch.zeros(2, 3, dtype=I32)
    a, b = torch.zeros(8, 4, 5), torch.zeros(8, 3, dtype=BF16)
    ops.beam_reorder([a, b], par)
    ops.beam_reorder([a, b], par, slots=par)
    ops.beam_reorder([], par)
    assert launched == ["vb_beam_reorder"] * 2
    for states, p, s in (([a], par.long(), None), ([a], par.view(-1), None), ([a], par[:, ::2], None), ([a, torch.zeros(7, 2)], par, None), ([a, a], par, None),
                         ([a.transpose(0, 1)], par, None), ([torch.zeros(5, 4)], par, None), ([a], par, par[:1]), ([a], par, par.long()),
                         ([torch.zeros(8, 0)], par, None), ([torch.zeros(())], par, None), ([torch.zeros(200, 1)], torch.zeros(1, 33, dtype=I32), None)):
        with pytest.raises(VoxB200Error):
            ops.beam_reorder(states, p, s)
    assert len(launched) == 2


@pytest.mark.parametrize("args", [(0, 16, 2, 2), (4, 0, 2, 2), (4, 16, 0, 2), (4, 16, 4097, 2), (4, 16, 2, 0), (4, 1 << 20, 2, 1 << 11), (4, 1, 4096, 1 << 20)])
def test_pool_sizes(args):
    with pytest.raises(VoxB200Error):
        ops.PagePool(*args, device="cpu")


def test_pool_counts_what_it_loads():
    pool = ops.PagePool(6, 4, 3, 3, device="cpu")
    assert bool((pool.table == -1).all()) and not bool(pool.refs.any()) and pool.indptr.tolist() == [0, 3, 6, 9]
    pool.load(torch.tensor([[5, 1, 3], [5, 2, 9], [-1, 0, 0]], dtype=I32), torch.tensor([5, 12, 0], dtype=I32))
    assert pool.refs.tolist() == [0, 1, 1, 0, 0, 2]
    assert pool.table.tolist() == [[5, 1, -1], [5, 2, -1], [-1, -1, -1]]
    with pytest.raises(VoxB200Error):
        pool.load(torch.zeros(3, 2, dtype=I32), torch.zeros(3, dtype=I32))
    pool.status[0] = 2
    with pytest.raises(VoxB200Error, match="2 pages are missing"):
        pool.check()
    pool.status[0], pool.status[1] = 0, 1
    with pytest.raises(VoxB200Error, match="1 rows grew past"):
        pool.check()


def _pool(**kw):
    pool = ops.PagePool(kw.get("pages", 6), 16, kw.get("rows", 4), kw.get("columns", 3), device="cpu")
    pool._device = 0
    return pool


def test_fork(launched):
    pool, other = _pool(), _pool()
    kv = torch.zeros(2, 6, 2, 16, 2, 8, dtype=BF16)
    four = torch.zeros(4, dtype=I32)
    for kw in ({}, {"grow": 3}, {"grow": four}, {"src": four}, {"src": four.view(2, 2)}, {"src": four, "group": 2}, {"src": four.view(2, 2), "group": 2}, {"out": other},
               {"caches": [kv, kv[0], torch.zeros(6, 16, 1, 8), torch.zeros(6, 3, 4), torch.zeros(6, 2, 16, 2, 8, dtype=BF16)]}):
        assert ops.fork_pages(pool, **kw) is kw.get("out", pool)
    n = len(launched)
    assert n == 9
    for kw in ({"grow": -1}, {"grow": 1 << 30}, {"grow": four[:2]}, {"grow": four.long()}, {"src": four.long()}, {"src": four[:3]}, {"src": four.view(2, 2, 1)}, {"src": four, "group": 3},
               {"src": four, "group": 0}, {"src": four.view(2, 2), "group": 4}, {"out": _pool(pages=7)}, {"out": _pool(rows=5)}, {"caches": [kv.transpose(4, 5)]},
               {"caches": [torch.zeros(5, 16, 8)]}, {"caches": [torch.zeros(6)]}, {"caches": [torch.zeros(6, 16, 3)]}, {"caches": [torch.zeros(6, 16, 0)]},
               {"caches": [torch.zeros(6 * 64 + 1)[1:].view(6, 16, 4)]}):
        with pytest.raises(VoxB200Error):
            ops.fork_pages(pool, **kw)
    with pytest.raises(VoxB200Error):
        ops.compact_pages(pool, out=_pool(columns=4))
    assert len(launched) == n
    ops.compact_pages(pool, caches=[kv], out=other)
    assert launched[n:] == ["vb_compact_pages"]


def test_caches_are_described(launched):
    pool = _pool()
    kv, k, pooled = torch.zeros(3, 6, 2, 16, 2, 8, dtype=BF16), torch.zeros(6, 16, 1, 40, dtype=BF16), torch.zeros(6, 4, 2, 8)
    c, n = ops._page_caches("fork_pages", [kv, k, k, pooled], pool)
    assert n == 3      # (a cache that is both keys and values stands once)
    got = [(s.data, s.slot_bytes, s.layers, s.parts, s.slots) for s in c]
    assert got == [(kv.data_ptr(), 32, 3, 2, 16), (k.data_ptr(), 80, 1, 1, 16), (pooled.data_ptr(), 64, 1, 1, 4)]


@pytest.mark.parametrize("args", [(0, 1, 4, 16, 2, 1, 64), (6, 4, 4, 16, 2, 1, 64), (6, 3, 0, 16, 2, 1, 64), (6, 3, 16385, 16, 2, 1, 64), (6, 3, 4, 24, 2, 1, 64), (6, 3, 4, 0, 2, 1, 64),
                                  (6, 3, 4, 4112, 2, 1, 64), (6, 3, 4, 16, 3, 2, 64), (6, 3, 4, 16, 129, 1, 64), (6, 3, 4, 16, 2, 1, 96), (6, 3, 4, 16, 2, 0, 64),
                                  (30000, 3, 16384, 64, 8, 8, 64)])
def test_plan_sizes(args):
    with pytest.raises(VoxB200Error):
        ops.SharedPlan(*args, device="cpu")


def test_attn(launched):
    plan = ops.SharedPlan(6, 3, 4, 16, 4, 2, 64, device="cpu")
    table, tokens = torch.zeros(6, 4, dtype=I32), torch.zeros(6, dtype=I32)
    ops.shared_plan(plan, table, tokens, 5)
    q, kv = torch.zeros(6, 4, 64, dtype=BF16), torch.zeros(3, 5, 2, 16, 2, 64, dtype=BF16)
    plan._device = -1                                  # (what a tensor of no GPU says)
    ops.shared_attn(q, kv, 10, plan)
    ops.shared_attn(q, kv[1], 0, plan, out=torch.empty_like(q), sm_scale=0.3)
    n = len(launched)
    assert n == 3
    for args, kw in (((q.float(), kv, 0, plan), {}), ((q[:5], kv, 0, plan), {}), ((q, kv.float(), 0, plan), {}), ((q, kv[:, :, :, :, :1], 0, plan), {}),
                     ((q, torch.zeros(3, 5, 2, 16, 3, 64, dtype=BF16), 0, plan), {}), ((q, kv, 15, plan), {}), ((q, kv, -5, plan), {}), ((q, kv, 3, plan), {}),
                     ((q, torch.zeros(4, 2, 16, 2, 64, dtype=BF16), 0, plan), {}), ((q, kv, 0, plan), {"out": q.float()}), ((q, kv, 0, plan), {"out": q[:, :2]}),
                     ((q.transpose(0, 1), kv, 0, plan), {})):
        with pytest.raises(VoxB200Error):
            ops.shared_attn(*args, **kw)
    for t, k, p in ((table.long(), tokens, 5), (table[:, :3], tokens, 5), (table, tokens[:5], 5), (table, tokens.long(), 5), (table, tokens, -1), (table, tokens, 1 << 30)):
        with pytest.raises(VoxB200Error):
            ops.shared_plan(plan, t, k, p)
    assert len(launched) == n


def test_plan_cuts_requests_evenly():
    """rows times query heads of a key head: at most 128 to a group, and 32 rows, which the buffer's size shows through its groups"""
    lib = _lib.load()

    def size(width, G):
        s = _lib.SharedPlanStruct(None, width, width, 1, 16, G, 1, 64, 1)
        return lib.vb_shared_plan_bytes(ctypes.addressof(s))

    def expect(rows, sub, groups, mpad):
        segments = 1 + groups
        return 16 * groups * sub + 128 + segments * mpad * (64 * 4 + 8) + 8 * groups + 4 * (3 * groups + 1 + rows)
    assert size(9, 16) == expect(9, 5, 2, 80)          # 8 rows would fit: 5 and 4
    assert size(16, 8) == expect(16, 16, 1, 128)
    assert size(17, 8) == expect(17, 9, 2, 80)
    assert size(33, 1) == expect(33, 17, 2, 32)
    assert size(8, 2) == expect(8, 8, 1, 16)
    assert size(1, 128) == expect(1, 1, 1, 128)


def test_entry_points_check_by_themselves():
    """the C ABI refuses without a device what it would not survive"""
    lib = _lib.load()
    assert lib.vb_beam_select_workspace_bytes(2, 5, 8193, 4, 0) == 2 * 5 * 2 * (8 + 32) and lib.vb_beam_select_workspace_bytes(2, 4, 8193, 4, 0) == 0
    assert lib.vb_beam_select(None, None, None, None, None, 0, 0, None, None, None, 1, 1, 8, 1, -1, None, 0, None) != 0 and b"null" in lib.vb_last_error()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    for B, W, V, n, end, ended in ((0, 1, 8, 1, -1, None), (1, 33, 8, 1, -1, None), (1, 1, 0, 1, -1, None), (1, 1, (1 << 24) + 1, 1, -1, None), (1, 1, 8, 65, -1, None),
                                   (1, 1, 8, 1, 8, at), (1, 1, 8, 1, -1, at), (1, 32, 1 << 20, 64, -1, None)):
        assert lib.vb_beam_select(at, at, at, None, at, 8, 0, at, None, ended, B, W, V, n, end, at, 512, None) != 0
    one, size = (ctypes.c_void_p * 1)(at), (ctypes.c_int64 * 1)(16)
    for k, slots, B, W in ((0, 4, 1, 2), (1, 0, 1, 2), (1, 4, 65536, 1), (1, 4, 1, 33), (1, 4, 3, 2)):
        assert lib.vb_beam_reorder(one, size, k, slots, at, None, B, W, None) != 0
    pool = _lib.PagePoolStruct(at, at, at, at, at, at, at, 4, 16, 2, 2)
    null = _lib.PagePoolStruct(at, None, at, at, at, at, at, 4, 16, 2, 2)
    cache = _lib.PageCacheStruct(at, 24, 1, 2, 16, 0)
    p, z, c = ctypes.addressof(pool), ctypes.addressof(null), ctypes.addressof(cache)
    assert lib.vb_fork_pages(p, z, None, 0, None, 0, None, 0, None) != 0 and lib.vb_compact_pages(z, p, None, 0, None) != 0
    assert lib.vb_fork_pages(p, p, None, 0, None, 0, c, 1, None) != 0 and b"24 bytes" in lib.vb_last_error()
    assert lib.vb_fork_pages(p, p, None, 3, None, 0, None, 0, None) != 0
    shared = _lib.PagePoolStruct(at, at + 64, at, at, at, at, at, 4, 16, 2, 2)
    assert lib.vb_fork_pages(p, ctypes.addressof(shared), None, 0, None, 0, None, 0, None) != 0 and b"share" in lib.vb_last_error()


def test_a_shortage_is_said_once():
    pool = ops.PagePool(6, 4, 3, 3, device="cpu")
    assert pool.live.shape == (3,) and not bool(pool.live.any())
    pool.load(torch.tensor([[5, 1, -1], [2, -1, -1], [-1, -1, -1]], dtype=I32), torch.tensor([5, 4, 0], dtype=I32))
    assert pool.live.tolist() == [5, 4, 0]
    pool.status[0], pool.status[2] = 2, 7
    pool.live.zero_()
    with pytest.raises(VoxB200Error, match="2 pages are missing"):
        pool.check()
    assert pool.status.tolist() == [0, 0, 7, 0] and pool.live.tolist() == [5, 4, 0]
    pool.check()
    pool.status[1] = 1
    pool.load(pool.table.clone(), pool.tokens.clone())
    pool.check()


def test_caches_that_begin_at_one_address(launched):
    """the same cache twice is one; one that is longer, or has other slots, is another, whichever comes first"""
    pool = _pool()
    kv = torch.zeros(3, 6, 2, 16, 2, 8, dtype=BF16)
    flat = kv.view(3, 6, 32, 16)[0]
    for caches in ([kv, kv[0], flat], [flat, kv[0], kv], [kv[0], kv, flat, kv, kv[0], flat]):
        c, n = ops._page_caches("compact_pages", caches, pool)
        got = [(s.data, s.slot_bytes, s.layers, s.parts, s.slots) for s in c[:n]]
        assert n == 3 and set(got) == {(kv.data_ptr(), 32, 3, 2, 16), (kv.data_ptr(), 32, 1, 2, 16), (kv.data_ptr(), 32, 1, 1, 32)}


def test_attn_needs_a_plan_that_was_made(launched):
    plan = ops.SharedPlan(6, 3, 4, 16, 4, 2, 64, device="cpu")
    plan._device = -1
    q, kv = torch.zeros(6, 4, 64, dtype=BF16), torch.zeros(5, 2, 16, 2, 64, dtype=BF16)
    table, tokens = torch.zeros(6, 4, dtype=I32), torch.zeros(6, dtype=I32)
    with pytest.raises(VoxB200Error, match="never made"):
        ops.shared_attn(q, kv, 0, plan)
    assert launched == []
    ops.shared_plan(plan, table, tokens, 5)
    ops.shared_attn(q, kv, 0, plan)
    assert not plan._struct.d_row_tokens
    ops.shared_attn(q, kv, 0, plan, tokens=tokens)
    assert plan._struct.d_row_tokens == tokens.data_ptr()
    ops.shared_attn(q, kv, 0, plan)
    assert not plan._struct.d_row_tokens
    n = len(launched)
    for bad in (tokens.long(), tokens[:5], tokens.view(2, 3), torch.zeros(12, dtype=I32)[::2]):
        with pytest.raises(VoxB200Error, match="int32 tokens"):
            ops.shared_attn(q, kv, 0, plan, tokens=bad)
    assert len(launched) == n


@pytest.mark.parametrize("table,tokens,rows", [
    ([[5, 1, -1], [5, 1, -1], [-1, -1, -1]], [5, 5, 0], 2),       # both go on in page 1
    ([[5, 1, -1], [5, 1, -1], [-1, -1, -1]], [5, 8, 0], 1),       # row 1 has filled it, row 0 would write over it
    ([[5, 1, -1], [0, 2, 1], [3, 4, -1]], [6, 9, 8], 2),
    ([[1, 1, -1], [-1, -1, -1], [-1, -1, -1]], [5, 0, 0], 1)])    # a row that holds it twice
def test_tables_that_share_a_page_that_is_not_full(table, tokens, rows):
    pool = ops.PagePool(6, 4, 3, 3, device="cpu")
    pool.load(torch.tensor([[0, 1, 2], [0, 3, -1], [-1, -1, -1]], dtype=I32), torch.tensor([12, 8, 0], dtype=I32))
    before = pool._buf.clone()
    with pytest.raises(VoxB200Error, match=f"{rows} rows share a page"):
        pool.load(torch.tensor(table, dtype=I32), torch.tensor(tokens, dtype=I32))
    assert torch.equal(pool._buf, before)


def test_tables_that_may_be_loaded():
    """full pages are shared, partial ones are not; what stands behind a row's tokens, numbers that are no page, rows longer than their columns and rows of less than none are passed over"""
    pool = ops.PagePool(6, 4, 3, 3, device="cpu")
    for table, tokens, refs in (([[5, 1, -1], [5, 2, 1], [5, 0, -1]], [7, 8, 4], [0, 1, 1, 0, 0, 3]), ([[5, 9, 0], [5, 9, 0], [9, 9, -3]], [6, 6, 3], [0, 0, 0, 0, 0, 2]),
                                ([[0, 1, 2], [0, 1, 2], [0, -1, -1]], [13, 12, -3], [2, 2, 2, 0, 0, 0]), ([[0, 1, 2], [3, 3, 3], [4, 0, 0]], [9, 0, 1], [1, 1, 1, 0, 1, 0])):
        pool.load(torch.tensor(table), torch.tensor(tokens))
        assert pool.refs.tolist() == refs and pool.tokens.tolist() == tokens
