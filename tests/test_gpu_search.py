"""A beam search on a decoder stack, as a program runs it: prompts once, then steps of beam_select, fork_pages, beam_reorder of what else belongs to a row (here its tokens),
shared_plan and LlamaEngine.forward(shared=), without the host between them.

Tolerances: the engine rounds to bf16 behind every projection, norm, rotation and attention; that of its own tests holds (logits within 2e-2 of the largest)."""
import pytest
import torch

from oracle import orpheus as oorph

pytestmark = pytest.mark.gpu

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
PAGE, PAGES, COLS, WIDTH = 16, 96, 8, 4


def _i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


class Search:
    """two requests of four beams"""

    def __init__(self, mode="unfused", dims=None, end_token=None, weighted=False):
        from vox_serve_b200 import ops
        from vox_serve_b200.engine import LlamaDims, LlamaEngine, LlamaWeights
        self.ops = ops
        self.d = d = dims or oorph.OrpheusDims.tiny()
        ld = LlamaDims(d.hidden_size, d.num_hidden_layers, d.num_attention_heads, d.num_key_value_heads, d.head_dim, d.intermediate_size, d.vocab_size, d.rms_norm_eps,
                       d.rope_theta, d.rope_factor, d.low_freq_factor, d.high_freq_factor, d.old_context_len)
        self.weights = LlamaWeights.from_state_dict(oorph.synth_weights(d, seed=7), ld)
        self.kv = torch.zeros(d.num_hidden_layers, PAGES, 2, PAGE, d.num_key_value_heads, d.head_dim, dtype=BF16, device="cuda")
        self.eng = LlamaEngine(self.weights, self.kv, PAGE, max_rows=128)
        self.eng.force_unfused = mode == "unfused"
        self.teacher = LlamaEngine(self.weights, torch.zeros_like(self.kv), PAGE, max_rows=128)
        g = torch.Generator().manual_seed(3)
        self.prompts = [torch.randint(10, d.vocab_size, (n,), generator=g).tolist() for n in (37, 21)]
        self.rows = len(self.prompts) * WIDTH
        self.pool = ops.PagePool(PAGES, PAGE, self.rows, COLS)
        self.plan = ops.SharedPlan(self.rows, WIDTH, COLS, PAGE, d.num_attention_heads, d.num_key_value_heads, d.head_dim)
        self.history = torch.zeros(self.rows, 32, dtype=I32, device="cuda")
        self.scores = torch.full((2, WIDTH), -float("inf"), device="cuda")
        self.ended = torch.zeros(2, WIDTH, dtype=torch.bool, device="cuda") if end_token is not None else None
        self.end_token, self.weighted, self.t = end_token, weighted, 0
        self.weight = torch.ones(2, WIDTH, device="cuda") if weighted else None
        self.ids = torch.zeros(self.rows, dtype=I32, device="cuda")
        self.at = torch.zeros(1, dtype=torch.int64, device="cuda")      # the history's next place

    def prompt_logits(self, eng, tables, tokens, rows):
        """logits of the last token of every prompt in ``tokens``; its pages: a row of ``tables``"""
        ops = self.ops
        qo = [0]
        for t in tokens:
            qo.append(qo[-1] + len(t))
        ops.plan_rows(eng.plan, _i32(qo), _i32([r * tables.shape[1] for r in rows] + [tables.numel()]), tables.view(-1), None, len(tokens), qo[-1], PAGE, eng.chunk,
                      kv_len=_i32([len(t) for t in tokens]))
        pos = torch.cat([torch.arange(len(t), dtype=I32) for t in tokens]).cuda()
        return eng.forward(_i32([x for t in tokens for x in t]), pos, qo[-1], last_rows=_i32([q - 1 for q in qo[1:]])).clone()

    def start(self):
        self.ops.fork_pages(self.pool, grow=_i32([37, 0, 0, 0, 21, 0, 0, 0]))
        self.pool.check()
        logits = self.prompt_logits(self.eng, self.pool.table, self.prompts, [0, WIDTH])
        self.scores[:, 0] = 0.0
        self.choose(logits.repeat_interleave(WIDTH, 0))

    def choose(self, logits):
        ops = self.ops
        step = ops.beam_select(logits, self.scores, WIDTH, weight=self.weight, ended=self.ended, end_token=self.end_token)
        ops.beam_reorder([self.history], step.parent)
        self.history.index_copy_(1, self.at, step.token.to(I32).view(-1, 1))
        self.at += 1
        ops.fork_pages(self.pool, step.parent, 1, [self.kv])
        self.scores.copy_(step.scores)
        if self.ended is not None:
            self.ended.copy_(step.ended)
        self.ids.copy_(step.token.view(-1))

    def forward(self, shared=True):
        ops = self.ops
        ops.plan_rows(self.eng.plan, None, self.pool.indptr, self.pool.table.view(-1), None, self.rows, self.rows, PAGE, self.eng.chunk, kv_len=self.pool.tokens)
        if shared:
            ops.shared_plan(self.plan, self.pool.table, self.pool.tokens, PAGES)
        return self.eng.forward(self.ids, self.pool.tokens - 1, self.rows, shared=self.plan if shared else None)

    def step(self):
        self.choose(self.forward())

    def sequences(self):
        n = int(self.at)
        return [self.prompts[r // WIDTH] + self.history[r, :n].tolist() for r in range(self.rows)]

    def taught(self):
        """logits behind every row's whole sequence, each read as one prompt"""
        seq = self.sequences()
        tables = torch.arange(4 * 8, dtype=I32, device="cuda").view(4, 8)
        return torch.cat([self.prompt_logits(self.teacher, tables[:1], [s], [0]) for s in seq])


@pytest.mark.parametrize("mode", ["unfused", "fused"])
def test_rows_know_their_own_sequences(mode):
    """every step's logits are those of the row's sequence read from its start, and those of one stream a row on the same tables"""
    s = Search(mode)
    s.start()
    held = []
    for _ in range(18):
        want = s.taught()
        got = s.forward().clone()
        alone = s.forward(shared=False).clone()
        tol = 2e-2 * want.float().abs().max()
        assert bool(((got.float() - want.float()).abs() <= tol).all())
        assert bool(((got.float() - alone.float()).abs() <= tol).all())
        s.pool.check()
        held.append(int((s.pool.refs > 0).sum()))
        s.choose(got)
    # shared pages of prompts are held once, pages of beams that died come back
    refs = s.pool.refs.tolist()
    counted = [0] * PAGES
    for row in s.pool.table.tolist():
        for p in row:
            if p >= 0:
                counted[p] += 1
    assert refs == counted and s.pool.tokens.tolist() == [37 + 19] * 4 + [21 + 19] * 4
    assert max(held) < sum(-(-n // PAGE) for n in s.pool.tokens.tolist())
    # scores are in order, and the sum of what the steps gave
    assert bool((s.scores[:, :-1] >= s.scores[:, 1:]).all())
    # moved to the front of the cache, the same rows see the same
    before = s.forward().clone()
    s.ops.compact_pages(s.pool, [s.kv])
    assert s.pool.refs[:int(s.pool.status[3])].min() > 0 and not bool(s.pool.refs[int(s.pool.status[3]):].any())
    assert torch.equal(s.forward(), before)


def test_beams_that_end_and_die():
    """an end token that is likely: beams end and keep their place by their weighted scores; nothing is missing or left over"""
    s = Search(end_token=11, weighted=True)
    s.start()
    total = s.scores.clone()
    for k in range(12):
        s.weight.copy_(torch.where(s.ended, s.weight, torch.full_like(s.weight, (k + 2) ** -0.7)))
        logits = s.forward().clone()
        logits[:, 11] += 4.0
        was, old = s.ended.clone(), s.scores.clone()
        s.choose(logits)
        s.pool.check()
        for b in range(2):
            for w in range(WIDTH):
                if bool(was[b, w]):                        # an ended beam's score comes back as it was, if it comes back
                    same = (s.scores[b] == old[b, w]) & s.ended[b]
                    assert int(same.sum()) <= int((old[b] == old[b, w]).sum())
        total = s.scores
    assert bool(s.ended.any()) and bool(torch.isfinite(total).all())


def test_a_captured_step():
    """the whole step as one graph: the same bits as step by step"""
    runs = []
    for captured in (False, True):
        s = Search()
        s.start()
        s.step()
        if captured:
            state = [s.kv, s.pool._buf, s.history, s.scores, s.ids, s.at]
            kept = [t.clone() for t in state]
            g = torch.cuda.CUDAGraph()
            s.step()
            torch.cuda.synchronize()
            with torch.cuda.graph(g):
                s.step()
            for t, k in zip(state, kept):
                t.copy_(k)
        for _ in range(10):
            g.replay() if captured else s.step()
        torch.cuda.synchronize()
        s.pool.check()
        runs.append((s.sequences(), s.scores.clone(), s.pool.table.clone(), s.pool.refs.clone(), s.kv.clone()))
    assert runs[0][0] == runs[1][0]
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1:], runs[1][1:]))


def test_plans_of_other_steps_are_refused():
    s = Search()
    s.start()
    ops, d = s.ops, s.d
    s.ops.plan_rows(s.eng.plan, None, s.pool.indptr, s.pool.table.view(-1), None, 8, 8, PAGE, s.eng.chunk, kv_len=s.pool.tokens)
    for other in (ops.SharedPlan(4, 4, COLS, PAGE, d.num_attention_heads, d.num_key_value_heads, d.head_dim), ops.SharedPlan(8, 4, COLS, 32, d.num_attention_heads, d.num_key_value_heads, d.head_dim),
                  ops.SharedPlan(8, 4, COLS, PAGE, 2 * d.num_attention_heads, d.num_key_value_heads, d.head_dim), ops.SharedPlan(8, 4, COLS, PAGE, d.num_attention_heads, d.num_key_value_heads, 64)):
        with pytest.raises(ops.VoxB200Error):
            s.eng.forward(s.ids, s.pool.tokens - 1, 8, shared=other)
    ops.plan_rows(s.eng.plan, _i32([0, 4, 8]), s.pool.indptr, s.pool.table.view(-1), None, 2, 8, PAGE, s.eng.chunk, kv_len=s.pool.tokens)
    with pytest.raises(ops.VoxB200Error, match="decode steps"):
        s.eng.forward(s.ids, s.pool.tokens - 1, 8, shared=s.plan)


@pytest.mark.parametrize("mode", ["unfused", "fused"])
def test_a_request_that_leaves(mode):
    """its rows stay in the step without a token: positions of -1, token -1, no page is written for them, and the others' logits are those of their sequences"""
    s = Search(mode)
    s.start()
    for _ in range(3):
        s.step()
    s.ops.fork_pages(s.pool, _i32([0, 1, 2, 3, -1, -1, -1, -1]))
    s.pool.check()
    assert s.pool.tokens.tolist() == [37 + 4] * 4 + [0] * 4
    s.ids[4:] = -1
    for shared in (True, False):
        before = s.kv.clone()
        got = s.forward(shared).clone()
        want = s.taught()
        assert bool(((got[:4].float() - want[:4].float()).abs() <= 2e-2 * want.float().abs().max()).all())
        own = s.pool.refs > 0
        assert torch.equal(before[:, ~own], s.kv[:, ~own])


def test_rows_without_a_token_have_no_place():
    """plan_rows of kv_len 0: no page, whatever the table holds, and the row in front is not looked at"""
    from vox_serve_b200 import ops
    for page in (1, 16):
        plan = ops.RowPlan(4, "cuda")
        table = _i32([7, 3, 5, 2, 9, 9, 9, 9])
        ops.plan_rows(plan, None, _i32([0, 2, 4, 6, 8]), table, None, 4, 4, page, page, kv_len=_i32([0, 1, 0, 2]))
        assert plan.row_page[:4].tolist() == [-1, 5, -1, 9] and plan.row_kvlen[:4].tolist() == [0, 1, 0, 2]
        assert plan.row_slot[:4].tolist() == [0, 0, 0, 1 % page]


def test_with_adapters():
    """rows with adapters of their own read shared pages as others do"""
    from vox_serve_b200.engine import LlamaAdapters
    s = Search()
    s.start()
    for _ in range(2):
        s.step()
    bank = LlamaAdapters(s.weights.dims, 2, 8)
    g = torch.Generator().manual_seed(1)
    state = {}
    for i in range(s.d.num_hidden_layers):
        for short, module in (("q", "self_attn.q_proj"), ("o", "self_attn.o_proj"), ("down", "mlp.down_proj")):
            n, k = oorph.synth_weights(s.d, seed=7)[oorph.layer_names(i)[short]].shape
            state[f"model.layers.{i}.{module}.lora_A.weight"] = (torch.randn(4, k, generator=g) / k ** 0.5).to(BF16)
            state[f"model.layers.{i}.{module}.lora_B.weight"] = (torch.randn(n, 4, generator=g) * 0.1).to(BF16)
    bank.load(1, state, 2.0)
    s.eng.set_adapters(bank)
    plan = s.ops.LoraPlan(s.rows, 2)
    s.ops.lora_plan(plan, _i32([1, -1, 1, 0, -1, 1, 1, -1]))
    logits = []
    for shared in (True, False):
        s.ops.plan_rows(s.eng.plan, None, s.pool.indptr, s.pool.table.view(-1), None, s.rows, s.rows, PAGE, s.eng.chunk, kv_len=s.pool.tokens)
        s.ops.shared_plan(s.plan, s.pool.table, s.pool.tokens, PAGES)
        logits.append(s.eng.forward(s.ids, s.pool.tokens - 1, s.rows, adapters=plan, shared=s.plan if shared else None).float().clone())
    assert bool(((logits[0] - logits[1]).abs() <= 2e-2 * logits[1].abs().max()).all())
    bare = s.forward().float()
    assert float((bare[0] - logits[0][0]).abs().max()) > float((bare[1] - logits[0][1]).abs().max())      # (the adapter of row 0 is there)


class LiveSearch(Search):
    """lengths of a step from the pool's live rows"""

    def forward(self, shared=True):
        ops, live = self.ops, self.pool.live
        ops.plan_rows(self.eng.plan, None, self.pool.indptr, self.pool.table.view(-1), None, self.rows, self.rows, PAGE, self.eng.chunk, kv_len=live)
        if shared:
            ops.shared_plan(self.plan, self.pool.table, live, PAGES)
        return self.eng.forward(self.ids, live - 1, self.rows, shared=self.plan if shared else None)


@pytest.mark.parametrize("shared", [True, False])
def test_a_captured_loop_that_runs_short_in_the_middle(shared):
    """from the step on that found too few pages, tables and cache hold what they held, though pages come free again behind it; and it is said at the end"""
    s = LiveSearch()
    s.start()
    s.choose(s.forward(shared))
    g = torch.cuda.CUDAGraph()
    s.choose(s.forward(shared))
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        s.choose(s.forward(shared))
    s.pool.check()
    others = s.pool.refs == 0
    others[torch.nonzero(others)[:3].view(-1)] = False      # three pages are left, the others somebody else's
    s.pool.refs[others] = 1
    kept = None
    for k in range(26):
        g.replay()
        torch.cuda.synchronize()
        if kept is None and bool(s.pool.status[:2].any()):
            kept = [t.clone() for t in (s.kv, s.pool.table, s.pool.tokens)]
            s.pool.refs[others] = 0                          # (pages come free: the next step would find enough)
            assert 2 < k < 20
    assert kept is not None and not bool(s.pool.live.any())
    for t, was in zip((s.kv, s.pool.table, s.pool.tokens), kept):
        assert torch.equal(t, was)
    with pytest.raises(s.ops.VoxB200Error, match="pages are missing"):
        s.pool.check()
    s.ops.check_waits()
    g.replay()                                               # (asked for: it goes on)
    torch.cuda.synchronize()
    s.pool.check()
    assert torch.equal(s.pool.tokens, kept[2] + 1) and torch.equal(s.pool.live, s.pool.tokens)


class KeptSearch(Search):
    """keeps what a step chose"""

    def choose(self, logits):
        ops = self.ops
        self.last = step = ops.beam_select(logits, self.scores, WIDTH, weight=self.weight, ended=self.ended, end_token=self.end_token)
        ops.fork_pages(self.pool, step.parent, 1, [self.kv])
        ops.beam_reorder([self.history], step.parent)
        self.history.index_copy_(1, self.at, step.token.to(I32).view(-1, 1))
        self.at += 1
        self.scores.copy_(step.scores)
        self.ended.copy_(step.ended)
        self.ids.copy_(step.token.view(-1))


def test_ended_beams_keep_their_scores():
    """an ended beam comes back once at most, under its end token and at its own score to the bit; it is there wherever its rank is above the last chosen one by more than a
    sum's error (2^-18 of a total, both sides); every total of a step is a number"""
    s = KeptSearch(end_token=11, weighted=True)
    s.start()
    carried = 0
    for k in range(14):
        s.weight.copy_(torch.where(s.ended, s.weight, torch.full_like(s.weight, (k + 2) ** -0.7)))
        logits = s.forward().clone()
        logits[:, 11] += 4.0
        was, old, weight = s.ended.cpu(), s.scores.cpu(), s.weight.cpu()
        s.choose(logits)
        s.pool.check()
        parent, token, score, over = (t.cpu() for t in (s.last.parent, s.last.token, s.last.scores, s.last.ended))
        assert bool(torch.isfinite(score).all()) and bool((parent >= 0).all())
        for b in range(2):
            ranks = [float(score[b, i].double() * weight[b, parent[b, i]].double()) for i in range(WIDTH)]
            slack = 4 * 2.0 ** -18 * float(weight[b].max()) + 2.0 ** -22 * max(abs(r) for r in ranks)
            assert all(x >= y - slack for x, y in zip(ranks, ranks[1:]))
            for w in range(WIDTH):
                mine = torch.nonzero(parent[b] == w).view(-1).tolist()
                if not bool(was[b, w]):
                    assert all(bool(over[b, i]) == (int(token[b, i]) == 11) for i in mine)
                    continue
                assert len(mine) <= 1
                for i in mine:
                    assert float(score[b, i]) == float(old[b, w]) and int(token[b, i]) == 11 and bool(over[b, i])
                    carried += 1
                if not mine:
                    assert float(old[b, w].double() * weight[b, w].double()) <= ranks[-1] + slack
    assert carried > 0


@pytest.mark.parametrize("mode", ["unfused", "fused"])
def test_a_plan_that_is_not_the_steps(mode):
    """one that was never made is refused before anything is written; one of the step before gives no logits that go unnoticed"""
    s = Search(mode)
    s.start()
    ops = s.ops

    def rows():
        ops.plan_rows(s.eng.plan, None, s.pool.indptr, s.pool.table.view(-1), None, s.rows, s.rows, PAGE, s.eng.chunk, kv_len=s.pool.tokens)
    rows()
    before = s.kv.clone()
    with pytest.raises(ops.VoxB200Error, match="never made"):
        s.eng.forward(s.ids, s.pool.tokens - 1, s.rows, shared=s.plan)
    assert torch.equal(s.kv, before)
    s.choose(s.forward())
    torch.cuda.synchronize()
    ops.check_waits()
    rows()
    with pytest.raises(ops.VoxB200Error, match="shared pages"):      # (by a launch of a later layer, or at the end)
        s.eng.forward(s.ids, s.pool.tokens - 1, s.rows, shared=s.plan)
        torch.cuda.synchronize()
        ops.check_waits()
    torch.cuda.synchronize()
    try:                                                     # (layers that were on their way when the first one raised)
        ops.check_waits()
    except ops.VoxB200Error:
        pass
    assert bool(torch.isfinite(s.forward()).all())
    torch.cuda.synchronize()
    ops.check_waits()
