"""Adapters and few-row experts where the engines call them: a decoder stack whose requests bring adapters of their own, mixture-of-experts models whose decode
steps run ops.moe_layer, and both behind one another as a block's second half has them.

Tolerances: the engines round to bf16 behind every projection, norm, rotation and attention; those of the engines' own tests against the same oracles hold
(logits of the decoder stack within 2e-2 of the largest, of the text models 8e-2 of their rms)."""
from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

from oracle import lm_ops, orpheus as oorph

pytestmark = pytest.mark.gpu

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def _i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


class Adapted:
    """a projection of the oracle with an adapter beside it"""

    def __init__(self, w, a, b, scale):
        self.w, self.a, self.b, self.scale = w, a, b, scale

    @staticmethod
    def linear(x, w):
        if not isinstance(w, Adapted):
            return F.linear(x, w)
        y = x.float() @ w.w.float().t() + w.scale * (x.float() @ w.a.float().t()) @ w.b.float().t()
        return y.to(x.dtype)


MODULES = {"q": "self_attn.q_proj", "k": "self_attn.k_proj", "v": "self_attn.v_proj", "o": "self_attn.o_proj", "gate": "mlp.gate_proj", "up": "mlp.up_proj",
           "down": "mlp.down_proj"}


def _adapter(weights, dims, rank, seed, only=None):
    """(checkpoint of an adapter, the oracle's weights with it)"""
    g = torch.Generator().manual_seed(seed)
    state, merged, scale = {}, dict(weights), 2.0
    for i in range(dims.num_hidden_layers):
        for short, module in MODULES.items():
            if only is not None and short not in only:
                continue
            name = oorph.layer_names(i)[short]
            n, k = weights[name].shape
            a, b = (torch.randn(rank, k, generator=g) / k ** 0.5).to(BF16), (torch.randn(n, rank, generator=g) * 0.2 / rank ** 0.5).to(BF16)
            state[f"model.layers.{i}.{module}.lora_A.weight"], state[f"model.layers.{i}.{module}.lora_B.weight"] = a, b
            merged[name] = Adapted(weights[name], a, b, scale)
    return state, merged, scale


@pytest.mark.parametrize("gu_half", [None, 48])
def test_decoder_stack_with_adapters_of_many_requests(monkeypatch, gu_half):
    """prompts of four requests (three adapters of different ranks and modules, one without) in one step, then decode steps with all of them, one step captured; against
    the oracle with the adapters beside its projections; and the step without adapters as it was"""
    from vox_serve_b200 import ops
    from vox_serve_b200.engine import LlamaAdapters, LlamaDims, LlamaEngine, LlamaWeights

    if gu_half:
        monkeypatch.setattr(ops, "gate_up_tile_half", lambda I, sms=None: gu_half)
    monkeypatch.setattr(oorph, "F", SimpleNamespace(linear=Adapted.linear, embedding=F.embedding, silu=F.silu))
    dims = oorph.OrpheusDims.tiny()
    base = oorph.synth_weights(dims, seed=5)
    specs = [_adapter(base, dims, 16, 1), _adapter(base, dims, 5, 2, only=("q", "v")), _adapter(base, dims, 40, 3, only=("o", "gate", "up", "down"))]
    ld = LlamaDims(dims.hidden_size, dims.num_hidden_layers, dims.num_attention_heads, dims.num_key_value_heads, dims.head_dim, dims.intermediate_size, dims.vocab_size,
                   dims.rms_norm_eps, dims.rope_theta, dims.rope_factor, dims.low_freq_factor, dims.high_freq_factor, dims.old_context_len)
    page, pages, slots = 16, 32, 5
    kv = torch.zeros(dims.num_hidden_layers, pages, 2, page, dims.num_key_value_heads, dims.head_dim, dtype=BF16, device="cuda")
    eng = LlamaEngine(LlamaWeights.from_state_dict(base, ld), kv, page, max_rows=256)
    bank = LlamaAdapters(ld, slots, 40)
    for slot, (state, _, scale) in zip((3, 0, 4), specs):
        bank.load(slot, state, scale)
    with pytest.raises(ops.VoxB200Error):
        eng.forward(_i32([1]), _i32([0]), 1, adapters=ops.LoraPlan(4, slots))
    eng.set_adapters(bank)
    g = torch.Generator().manual_seed(9)
    lens, who, ws = [37, 5, 70, 12], [3, 0, -1, 4], [specs[0][1], specs[1][1], base, specs[2][1]]
    tokens = [torch.randint(10, dims.vocab_size, (n + 3,), generator=g) for n in lens]
    table = [list(range(8 * i, 8 * i + 8)) for i in range(4)]

    def oracle(i, n):
        cache = torch.zeros(dims.num_hidden_layers, pages, 2, page, dims.num_key_value_heads, dims.head_dim, dtype=BF16)
        wrap = lm_ops.PagedWrapperCPU("prefill", page)
        np_ = (n + page - 1) // page
        wrap.plan([0, n], [0, np_], table[i][:np_], [n - (np_ - 1) * page])
        return oorph.lm_forward(ws[i], dims, tokens[i][:n], torch.arange(n, dtype=I32), wrap, cache)

    def plan_step(cur, qo):
        counts = [(n + page - 1) // page for n in cur]
        indptr = [0]
        for c in counts:
            indptr.append(indptr[-1] + c)
        return _i32(indptr), _i32([p for t, c in zip(table, counts) for p in t[:c]]), _i32([n - (c - 1) * page for n, c in zip(cur, counts)]), qo

    def check(logits, cur):
        for i, n in enumerate(cur):
            ref = oracle(i, n)[-1].float()
            err = (logits[i].float().cpu() - ref).abs().max().item()
            assert err < 2e-2 * ref.abs().max().item(), (i, n, err)

    # prompts
    qo = [0]
    for n in lens:
        qo.append(qo[-1] + n)
    R = qo[-1]
    lora = ops.LoraPlan(256, slots)
    ops.lora_plan(lora, _i32([a for n, a in zip(lens, who) for _ in range(n)]))
    indptr, indices, last, q = plan_step(lens, _i32(qo))
    ops.plan_rows(eng.plan, q, indptr, indices, last, 4, R, page, eng.chunk)
    ids = torch.cat([t[:n] for t, n in zip(tokens, lens)]).to(I32).cuda()
    pos = torch.cat([torch.arange(n, dtype=I32) for n in lens]).cuda()
    got = eng.forward(ids, pos, R, last_rows=_i32([x - 1 for x in qo[1:]]), adapters=lora).clone()
    check(got, lens)
    # the adapters move the logits by more than rounding does
    plain = oorph.lm_forward(base, dims, tokens[0][:37], torch.arange(37, dtype=I32), _prefill(37, table[0], page), torch.zeros_like(kv, device="cpu"))[-1].float()
    assert (got[0].float().cpu() - plain).abs().max().item() > 0.1 * plain.abs().max().item()
    # decode steps
    step_ids, step_pos = torch.zeros(4, dtype=I32, device="cuda"), torch.zeros(4, dtype=I32, device="cuda")
    graph = None
    for k in range(2):
        cur = [n + k + 1 for n in lens]
        indptr, indices, last, _ = plan_step(cur, None)
        ops.plan_rows(eng.plan, None, indptr, indices, last, 4, 4, page, eng.chunk)
        ops.lora_plan(lora, _i32(who))
        step_ids.copy_(torch.stack([t[n - 1] for t, n in zip(tokens, cur)]).to(I32))
        step_pos.copy_(_i32([n - 1 for n in cur]))
        if graph is None:
            check(eng.forward(step_ids, step_pos, 4, adapters=lora).clone(), cur)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = eng.forward(step_ids, step_pos, 4, adapters=lora)
        else:
            graph.replay()
            torch.cuda.synchronize()
            check(out.clone(), cur)
    # no adapters: the path as it was, whatever has been set
    other = LlamaEngine(eng.w, kv.clone(), page, max_rows=256)
    ops.plan_rows(other.plan, None, indptr, indices, last, 4, 4, page, other.chunk)
    assert torch.equal(eng.forward(step_ids, step_pos, 4), other.forward(step_ids, step_pos, 4))


def _prefill(n, pages, page):
    wrap = lm_ops.PagedWrapperCPU("prefill", page)
    c = (n + page - 1) // page
    wrap.plan([0, n], [0, c], pages[:c], [n - (c - 1) * page])
    return wrap


def test_adapter_checkpoints_that_do_not_fit():
    from vox_serve_b200.engine import LlamaAdapters, LlamaDims
    from vox_serve_b200 import ops

    dims = LlamaDims(128, 1, 2, 1, 64, 256, 100)
    bank = LlamaAdapters(dims, 2, 8)
    a, b = torch.zeros(4, 128), torch.zeros(128, 4)
    key = "model.layers.0.self_attn.q_proj.lora_%s.weight"
    bank.load(1, {key % "A": a, key % "B": b}, 1.0)
    for state in ({key % "A": a}, {key % "A": a[:, :64], key % "B": b}, {key % "A": a, key % "B": b[:64]}, {"model.layers.1.self_attn.q_proj.lora_A.weight": a},
                  {key % "A": torch.zeros(9, 128), key % "B": torch.zeros(128, 9)}):
        with pytest.raises(ops.VoxB200Error):
            bank.load(0, state, 1.0)


def _text_model(name):
    if name == "bobavik":
        from tests import bobavik_oracle as O, test_gpu_bobavik as T
        cfg = O.make_config(width=64, layers=("attention", "lightning"), ff=64, shared_ff=128, experts=4, top=2, dim=16, vdim=16, window=40)
        return cfg, O.random_weights(cfg, 23), O, T, "gu_all", {"pages": 40, "page_size": 8}
    if name == "redalix":
        from tests import redalix_oracle as O, test_gpu_redalix as T
        cfg = O.make_config(layers=("mamba:moe", "pair:moe", "attn:moe"), **T.TC)
        return cfg, O.make_weights(cfg, 21), O, T, "up_all", {"slots": 2, "pages": 24, "page_size": 64}
    if name == "razevik":
        from tests import razevik_oracle as O, test_gpu_razevik as T
        cfg = O.make_config(width=64, ff=64, shared_ff=64, experts=8, top=2, groups=(4, 2))
        return cfg, O.random_weights(cfg, 7), O, T, "up_all", {"pages": 40, "page_size": 8}
    from tests import nadevik_oracle as O, test_gpu_nadevik as T
    cfg = O.make_config(width=64, ff=64, s_inner=64, experts=6, top=2, groups=(3, 2))
    return cfg, O.make_weights(cfg, 3, calm=True), O, T, "gu_all", {"pages": 40, "page_size": 8}


@pytest.mark.parametrize("name", ["bobavik", "redalix", "razevik", "nadevik"])
def test_text_models_decode_with_few_row_experts(name, monkeypatch):
    """every kind of router and expert on its model: token by token and in batches with ops.moe_layer, against the oracle and against the stacked form"""
    from vox_serve_b200 import ops

    cfg, sd, O, T, up, kw = _text_model(name)
    w = T._worker(cfg, sd, BF16, **kw)
    layers = [L for L in w.engine.w.layers if up in L]
    assert layers and all("few" in L for L in layers)
    calls, prompt = [], []
    real = ops.moe_layer

    def counted(h, weights, router, **k):
        out = real(h, weights, router, **k)
        calls.append(h.shape[0])
        if h.shape[0] == 30:                             # (the prompt's step is not captured)
            prompt.append((h.clone(), router, out.clone()))
        return out
    monkeypatch.setattr(ops, "moe_layer", counted)
    toks = T._tokens(40, cfg["vocab"], 9)
    ref = O.forward(cfg, sd, toks)
    ref = ref[0] if isinstance(ref, tuple) else ref
    steps = [[("a", 30)]] + [[("a", 1)]] * 10
    err = T._err50 if name == "nadevik" else T._err
    stacked = T._replay(w, {"a": toks}, steps)["a"]
    assert not calls                                     # off: the path as it was
    w = T._worker(cfg, sd, BF16, **kw)                   # (decode steps are captured once: a worker of its own)
    w.engine.few_experts = True
    few = T._replay(w, {"a": toks}, steps)["a"]
    assert calls.count(30) == len(layers) and calls.count(1) >= len(layers) and calls.count(1) % len(layers) == 0
    if name == "nadevik":
        # (at this size bfloat16 elsewhere in the model moves the logits by more than the bound whichever way the experts run, 0.11 with the stacked form: judged
        # are the layers themselves, each on the rows that it was given)
        from tests import test_gpu_moe_layer as L
        monkeypatch.setattr(L, "LIMIT", cfg["layers"][0]["mlp"]["expert"]["limit"])
        at = [i for i, c in enumerate(cfg["layers"]) if c["mlp"]]
        assert len(prompt) == len(at)
        for i, (h, router, out) in zip(at, prompt):
            ex = [torch.stack([sd[f"l{i}.mlp.e{e}.{m}"] for e in range(6)]).to(device="cuda", dtype=BF16) for m in ("gate", "up", "down")]
            L._check(out, h, ex, None, router, None, "clamped_glu")
        return
    assert err(few, ref) < T.TOL[BF16] and err(stacked, ref) < T.TOL[BF16] and err(few, stacked.double()) < T.TOL[BF16]
    both = T._replay(w, {"a": toks, "b": toks[:12]}, [[("a", 25), ("b", 2)]] + [[("a", 1), ("b", 1)]] * 10 + [[("a", 1)]] * 5)
    assert err(both["a"], ref) < T.TOL[BF16] and err(both["b"], ref[:12]) < T.TOL[BF16]


def test_second_half_of_a_block():
    """output projection with the rows' adapters as one more plane, residual and norm, then a mixture-of-experts layer: the kernels as a decode step has them behind one
    another, captured and replayed over other adapters, against 64 bits with the same two roundings (the stream and its norm)"""
    from vox_serve_b200 import ops

    T, H, E, top, ff = 13, 512, 16, 3, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std)                     # noqa: E731
    attn, wo, res, ln = rnd(T, H).to(BF16), rnd(H, H, std=H ** -0.5).to(BF16), rnd(T, H).to(BF16), (1 + rnd(H, std=0.1)).to(BF16)
    a, b = rnd(4, 1, 16, H, std=H ** -0.5).to(BF16), rnd(4, H, 16, std=0.25).to(BF16)
    gate, up, down = (rnd(E, ff, H, std=H ** -0.5).to(BF16), rnd(E, ff, H, std=H ** -0.5).to(BF16), rnd(E, H, ff, std=ff ** -0.5).to(BF16))
    router = ops.MoeRouter("softmax", top, weight=rnd(E, H, std=2 * H ** -0.5))
    bank, experts, packed = ops.LoraBank(4, H, (H,), 16), ops.MoeWeights.pack(gate, up, down), ops.pack_weight(wo)
    for s in range(4):
        bank.load(s, a[s], b[s], 0.5)
    plan, ids = ops.LoraPlan(T, 4), torch.zeros(T, dtype=I32, device="cuda")
    planes = torch.zeros(3, T, H, device="cuda")

    def step():
        ops.lora_plan(plan, ids)
        ops.gemm(attn, packed, mode=1, split_k=2, out=planes[:2])
        ops.lora(attn, bank, plan, out=planes[2])
        hidden, normed = ops.reduce_residual_rmsnorm(planes, res, ln, 1e-5)
        return hidden, normed, ops.moe_layer(normed, experts, router)
    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        ids.copy_(torch.randint(-1, 4, (T,), generator=torch.Generator().manual_seed(seed)).to(I32))
        graph.replay()
        torch.cuda.synchronize()
        hidden, normed, y = (t.double() for t in out)
        d = torch.stack([torch.zeros(H, dtype=torch.float64, device="cuda") if s < 0 else 0.5 * b[s].double() @ (a[s, 0].double() @ attn[t].double())
                         for t, s in enumerate(ids.tolist())])
        proj = attn.double() @ wo.double().t() + d
        # the projection's result is rounded to bf16, then the sum with the stream: half a step each, and the sums' error far below
        want = proj + res.double()
        assert bool(((hidden - want).abs() <= 2.0 ** -8 * (proj.abs() + want.abs()) + 1e-3 * 2.0 ** -8).all())
        norm = hidden / (hidden.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * ln.double()
        assert bool(((normed - norm).abs() <= (2.0 ** -8 + 2.0 ** -18) * norm.abs()).all())
        z = normed @ router.weight.double().t()
        v, idx = torch.sort(z, dim=1, descending=True, stable=True)
        w = torch.softmax(v[:, :top], 1)
        for t in range(T):
            if float(v[t, top - 1] - v[t, top]) < 1e-4:            # (a choice within the router's rounding)
                continue
            ref = torch.zeros(H, dtype=torch.float64, device="cuda")
            size = torch.zeros_like(ref)
            for c in range(top):
                e = int(idx[t, c])
                gt, ut = gate[e].double() @ normed[t], up[e].double() @ normed[t]
                act = gt * torch.sigmoid(gt) * ut
                ref += w[t, c] * (down[e].double() @ act)
                size += w[t, c] * (down[e].double().abs() @ (gt.abs() * ut.abs() + act.abs() + 1.1 * (gate[e].double().abs() @ normed[t].abs()) * ut.abs()
                                                             + gt.abs() * (up[e].double().abs() @ normed[t].abs())))
            # (sums of at most 32 steps of the matrix units, three parts of eight steps and the warps' sums: below 100 2^-22 of the terms' sizes; weights 2^-17)
            assert bool(((y[t] - ref).abs() <= (100 * 2.0 ** -22 + 2.0 ** -16) * size + 1e-30).all())
