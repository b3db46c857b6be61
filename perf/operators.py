"""Operators whose weights a row brings with it, as cases that can be timed and checked.

Kinds:

  lora         low-rank adapters of many requests beside a shared projection: out[t] = base[t] + B_a(scale_a A_a x_t), the adapter a being row t's
               (none: the base alone).  ``plane``: fp32, no base -- one more split-K plane of the projection; else bf16 rows with a base
  lora_glu     the same beside the gated MLP: silu(gate + its adapter) * (up + its adapter) from the projection's fp32 planes
  moe          a whole mixture-of-experts layer for the rows of a decode step: router, the chosen experts, shared expert, weighted sum

``run`` computes them in their plain form, or (``own``) through vox_serve_b200.ops.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def _device():
    return torch.device("cuda", torch.cuda.current_device())


# ---- the cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one stream of a small speech LM with a small adapter on its output projection: nothing but latency
        {"name": "lora_one", "kind": "lora", "prompts": 0, "prompt_rows": 0, "riders": 1, "slots": 4, "used": 1, "bare": 0, "K": 896, "slices": "896",
         "rank": 8, "plane": True},
        # a full decode batch, every stream with a voice of its own
        {"name": "lora_decode_32", "kind": "lora", "prompts": 0, "prompt_rows": 0, "riders": 32, "slots": 64, "used": 32, "bare": 0, "K": 2048,
         "slices": "2048", "rank": 16, "plane": True},
        # 64 streams on a dozen voices, some on the base model; q | k | v of a model with two key heads
        {"name": "lora_decode_qkv_64", "kind": "lora", "prompts": 0, "prompt_rows": 0, "riders": 64, "slots": 32, "used": 12, "bare": 5, "K": 4096,
         "slices": "4096,256,256", "rank": 32, "plane": True},
        # one prompt joins a running batch
        {"name": "lora_join", "kind": "lora", "prompts": 1, "prompt_rows": 435, "riders": 31, "slots": 32, "used": 19, "bare": 7, "K": 2048,
         "slices": "2048,512,512", "rank": 16, "plane": True},
        # a large prompt step: ragged prompts of several voices through a down projection, bf16 rows with their base
        {"name": "lora_prompts", "kind": "lora", "prompts": 9, "prompt_rows": 4096, "riders": 0, "slots": 16, "used": 6, "bare": 0, "K": 8192,
         "slices": "2048", "rank": 64, "plane": False},
        # the gated MLP of a decode batch of odd size
        {"name": "glu_decode_17", "kind": "lora_glu", "prompts": 0, "prompt_rows": 0, "riders": 17, "slots": 24, "used": 11, "bare": 6, "K": 896, "ff": 4864,
         "half": 48, "splits": 1, "rank": 16},
        # ... of a prompt step
        {"name": "glu_prompts", "kind": "lora_glu", "prompts": 3, "prompt_rows": 1000, "riders": 0, "slots": 8, "used": 2, "bare": 0, "K": 2048, "ff": 8192,
         "half": 64, "splits": 1, "rank": 32},
        # one stream of a small mixture: two of eight experts beside a shared one
        {"name": "moe_one", "kind": "moe", "rows": 1, "W": 1024, "ff": 1024, "experts": 8, "top": 2, "shared": 1024, "act": "silu_glu", "router": "softmax",
         "groups": 0, "keep": 0},
        # table-routed experts of the form down(relu(up h)^2) with a gated shared expert, a batch of odd size
        {"name": "moe_table_5", "kind": "moe", "rows": 5, "W": 2048, "ff": 2048, "experts": 8, "top": 2, "shared": 2048, "act": "relu2", "router": "table",
         "groups": 0, "keep": 0},
        # many small experts, chosen among the best groups
        {"name": "moe_8", "kind": "moe", "rows": 8, "W": 2048, "ff": 1024, "experts": 64, "top": 6, "shared": 0, "act": "silu_glu", "router": "softmax_all",
         "groups": 8, "keep": 4},
        # clamped gates, an expert width that is no multiple of a tile
        {"name": "moe_clamped_16", "kind": "moe", "rows": 16, "W": 1536, "ff": 1000, "experts": 32, "top": 4, "shared": 0, "act": "clamped_glu",
         "router": "softmax", "groups": 0, "keep": 0},
        # a full decode batch that touches nearly every expert
        {"name": "moe_64", "kind": "moe", "rows": 64, "W": 2048, "ff": 768, "experts": 128, "top": 8, "shared": 768, "act": "silu_glu", "router": "sigmoid",
         "groups": 0, "keep": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("lora", "lora_glu", "moe"))
    if kind == "moe":
        while True:
            E = _log(rng, 4, 128)
            top = rng.randint(1, min(8, E))
            W, ff = 8 * _log(rng, 32, 512), _log(rng, 64, 2048)
            if E * W * ff <= 128 * 2048 * 768:
                break
        router = rng.choice(("softmax", "sigmoid", "softmax_all", "table"))
        act = rng.choice(("silu_glu", "clamped_glu", "relu2", "gelu", "gelu_tanh"))
        groups = keep = 0
        if router in ("sigmoid", "softmax_all") and rng.random() < 0.5:
            fit = [g for g in (2, 4, 8) if E % g == 0 and E // g >= 2]
            if fit:
                groups = rng.choice(fit)
                keep = rng.randint(-(-top // (E // groups)), groups)
        return {"kind": "moe", "rows": _log(rng, 1, 64), "W": W, "ff": ff, "experts": E, "top": top, "shared": rng.choice((0, 0, ff, _log(rng, 64, 2048))),
                "act": act, "router": router, "groups": groups, "keep": keep}
    prompts = rng.choice((0, 0, 1, rng.randint(2, 9)))
    rows = max(prompts * 2, _log(rng, 16, 4096)) if prompts else 0
    riders = _log(rng, 1, 64) if not prompts or rng.random() < 0.5 else 0
    slots = _log(rng, 1, 64)
    case = {"kind": kind, "prompts": prompts, "prompt_rows": rows, "riders": riders, "slots": slots, "used": rng.randint(1, slots),
            "bare": rng.choice((0, 0, 2, 5)), "K": 8 * _log(rng, 32, 1024), "rank": rng.choice((1, 4, 8, 16, 16, 24, 32, 40, 64))}
    if kind == "lora":
        case["slices"] = ",".join(str(8 * _log(rng, 8, 512)) for _ in range(rng.choice((1, 1, 2, 3))))
        case["plane"] = rng.random() < 0.5
    else:
        case["ff"], case["half"], case["splits"] = 8 * _log(rng, 32, 1024), rng.choice((16, 32, 48, 64)), rng.choice((1, 1, 2))
    return case


# ---- what a user's program has in hand ---------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    return g


def _rand(g, *shape, std=1.0, dtype=BF16):
    out = torch.empty(shape, dtype=dtype, device=_device())
    return out.normal_(0.0, std, generator=g)


def _activations(g, T, W):
    """rows behind a norm: channels of unequal size, a few of them large"""
    gain = torch.exp(_rand(g, W, std=0.4, dtype=F32))
    gain[torch.randperm(W, generator=g, device=_device())[:max(1, W // 256)]] *= 6.0
    return (_rand(g, T, W, dtype=F32) * gain).to(BF16)


def _requests(case):
    """rows of every request: the prompts (uneven), then the riders of one row"""
    n = case["prompts"]
    total, weights = case["prompt_rows"], [i + 1 for i in range(n)]
    lens = [max(1, total * w // sum(weights)) for w in weights]
    if n:
        lens[-1] += total - sum(lens)
    return lens + [1] * case["riders"]


def _adapters_of(case, perm):
    """adapter of every request (-1: none)"""
    bare = case["bare"]
    return [-1 if bare and i % bare == bare - 1 else perm[i % case["used"]] for i in range(len(_requests(case)))]


def _widths(case):
    return [int(w) for w in case["slices"].split(",")] if case["kind"] == "lora" else [case["ff"], case["ff"]]


def _prepare_lora(case, seed):
    g = _gen(seed)
    lens, widths = _requests(case), _widths(case)
    T, K, N, S, r, slots = sum(lens), case["K"], sum(widths), len(widths), case["rank"], case["slots"]
    perm = torch.randperm(slots, generator=g, device=_device()).tolist()
    ids = [a for n, a in zip(lens, _adapters_of(case, perm)) for _ in range(n)]
    x = _activations(g, T, K)
    a = _rand(g, slots, S, r, K, std=1.0 / math.sqrt(K))
    b = _rand(g, slots, N, r, std=0.3 / math.sqrt(r))
    scale = [0.25 * (1 + s % 7) for s in range(slots)]
    rows = {}
    for t, s in enumerate(ids):
        rows.setdefault(s, []).append(t)
    st = {"case": case, "x": x, "a": a, "b": b, "scale": scale, "widths": widths,
          "rows": [(s, torch.tensor(t, device=_device())) for s, t in sorted(rows.items())]}
    if case["kind"] == "lora":
        st["base"] = None if case["plane"] else _rand(g, T, N)
    else:
        tiles = -(-case["ff"] // case["half"])
        st["planes"] = _rand(g, case["splits"], T, 2 * tiles * case["half"], dtype=F32)
    if own:
        from vox_serve_b200 import ops
        bank = ops.LoraBank(slots, K, widths, r, _device())
        for s in range(slots):
            bank.load(s, a[s], b[s], scale[s])
        st["bank"] = bank
        # the plan of a step: made once, read by every projection of every layer
        st["plan"] = ops.lora_plan(ops.LoraPlan(T, slots, _device()), torch.tensor(ids, dtype=I32, device=_device()))
    return st


def _prepare_moe(case, seed):
    g = _gen(seed)
    T, W, ff, E, top, sff = case["rows"], case["W"], case["ff"], case["experts"], case["top"], case["shared"]
    gated = case["act"].endswith("glu")
    st = {"case": case, "h": _activations(g, T, W)}

    def experts(n, width):
        return {"gate": _rand(g, n, width, W, std=1.0 / math.sqrt(W)) if gated else None, "up": _rand(g, n, width, W, std=1.0 / math.sqrt(W)),
                "down": _rand(g, n, W, width, std=1.0 / math.sqrt(width))}
    st["experts"] = experts(E, ff)
    st["shared"] = experts(1, sff) if sff else None
    st["router"] = st["bias"] = st["table"] = st["ids"] = st["shared_gate"] = None
    if case["router"] == "table":
        vocab = 4096
        st["table"] = torch.argsort(torch.rand(vocab, E, generator=g, device=_device()), 1)[:, :top].to(I32).contiguous()
        st["ids"] = torch.randint(0, vocab, (T,), generator=g, device=_device()).to(I32)
    else:
        st["router"] = _rand(g, E, W, std=1.0 / math.sqrt(W), dtype=F32)
        if case["router"] != "softmax_all":
            st["bias"] = _rand(g, E, std=0.1, dtype=F32)
    if sff and case["router"] in ("sigmoid", "table"):
        st["shared_gate"] = _rand(g, W, std=1.0 / math.sqrt(W), dtype=F32)
    if own:
        from vox_serve_b200 import ops
        ex, sh = st["experts"], st["shared"]
        limit = {"limit": LIMIT, "slope": SLOPE} if case["act"] == "clamped_glu" else {}
        st["weights"] = ops.MoeWeights.pack(ex["gate"], ex["up"], ex["down"], shared=None if sh is None else (None if sh["gate"] is None else sh["gate"][0],
                                            sh["up"][0], sh["down"][0]), act=case["act"], **limit)
        st["plan"] = ops.MoeRouter(case["router"], top, weight=st["router"], bias=st["bias"], groups=case["groups"], keep=case["keep"],
                                   shared_gate=st["shared_gate"], table=st["table"])
    return st


def prepare(case, seed):
    return _prepare_moe(case, seed) if case["kind"] == "moe" else _prepare_lora(case, seed)


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def _delta(st):
    """B (scale A x) of every row, fp32 [T, N]; zeros where a row has no adapter"""
    x, widths = st["x"], st["widths"]
    out = torch.zeros(x.shape[0], sum(widths), dtype=F32, device=x.device)
    for s, rows in st["rows"]:
        if s < 0:
            continue
        xs, n0, parts = x[rows].float(), 0, []
        for i, n in enumerate(widths):
            v = (xs @ st["a"][s, i].float().t()) * st["scale"][s]
            parts.append(v @ st["b"][s, n0:n0 + n].float().t())
            n0 += n
        out[rows] = torch.cat(parts, 1)
    return out


def _packed_columns(ff, half, device):
    """where the gate value of column i stands in a row of planes (its up value: 16 further)"""
    i = torch.arange(ff, device=device)
    tile, j = i // half, i % half
    return tile * 2 * half + j // 16 * 32 + j % 16


LIMIT, SLOPE = 7.0, 1.702


def _act(name, g, u):
    """g: gate (None for the plain forms), u: up"""
    if name == "silu_glu":
        return g / (1.0 + torch.exp(-g)) * u
    if name == "clamped_glu":
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g / (1.0 + torch.exp(-SLOPE * g)) * (u + 1.0)
    if name == "relu2":
        return u.clamp(min=0.0) ** 2
    if name == "gelu":
        return 0.5 * u * (1.0 + torch.erf(u * math.sqrt(0.5)))
    return 0.5 * u * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (u + 0.044715 * u ** 3)))


def _route(st):
    """routing weight of every expert for every row, fp32 [T, E] (0: not chosen); scores in 64 bits, since a choice may hang on their last digits"""
    case, h = st["case"], st["h"]
    T, E, top = h.shape[0], case["experts"], case["top"]
    comb = torch.zeros(T, E, dtype=F32, device=h.device)
    if case["router"] == "table":
        return comb.scatter_(1, st["table"][st["ids"].long()].long(), 1.0 / top)
    z = h.double() @ st["router"].double().t()
    if case["router"] == "softmax":
        z = z + st["bias"].double()
        idx = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :top]
        w = torch.softmax(z.gather(1, idx), 1)
        return comb.scatter_(1, idx, w.float())
    score = torch.softmax(z, 1) if case["router"] == "softmax_all" else 1.0 / (1.0 + torch.exp(-z))
    pick = score if st["bias"] is None else score + st["bias"].double()
    if case["groups"] > 1:
        by = pick.view(T, case["groups"], -1)
        rank = by.max(2)[0] if case["router"] == "softmax_all" else torch.sort(by, dim=2, descending=True)[0][:, :, :2].sum(2)
        kept = torch.sort(rank, dim=1, descending=True, stable=True)[1][:, :case["keep"]]
        mask = torch.zeros_like(rank, dtype=torch.bool).scatter_(1, kept, True)
        pick = torch.where(mask[:, :, None], by, torch.full_like(by, -math.inf)).view(T, E)
    idx = torch.sort(pick, dim=1, descending=True, stable=True)[1][:, :top]
    w = score.gather(1, idx)
    if case["router"] == "sigmoid":
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return comb.scatter_(1, idx, w.float())


def _expert_rows(name, h, ex):
    """every expert on every row, fp32 [E, T, W]"""
    g = None if ex["gate"] is None else torch.matmul(h, ex["gate"].float().transpose(1, 2))
    return torch.matmul(_act(name, g, torch.matmul(h, ex["up"].float().transpose(1, 2))), ex["down"].float().transpose(1, 2))


def run(state):
    case = state["case"]
    if case["kind"] == "moe":
        if own:
            from vox_serve_b200 import ops
            return {"out": ops.moe_layer(state["h"], state["weights"], state["plan"], ids=state["ids"])}
        h = state["h"].float()
        comb = _route(state)
        y = _expert_rows(case["act"], h, state["experts"])
        out = (torch.where(comb.t()[:, :, None] != 0, y, torch.zeros_like(y)) * comb.t()[:, :, None]).sum(0)
        if state["shared"] is not None:
            s = _expert_rows(case["act"], h, state["shared"])[0]
            if state["shared_gate"] is not None:
                s = s / (1.0 + torch.exp(-(h @ state["shared_gate"])))[:, None]
            out = out + s
        return {"out": out}
    if case["kind"] == "lora":
        if own:
            from vox_serve_b200 import ops
            return {"out": ops.lora(state["x"], state["bank"], state["plan"], base=state["base"])}
        d = _delta(state)
        return {"out": d if state["base"] is None else (state["base"].float() + d).to(BF16)}
    if own:
        from vox_serve_b200 import ops
        return {"act": ops.lora_gate_up(state["x"], state["bank"], state["plan"], state["planes"], case["half"])}
    d, ff = _delta(state), case["ff"]
    p = state["planes"].sum(0)
    at = _packed_columns(ff, case["half"], p.device)
    return {"act": _act("silu_glu", p[:, at] + d[:, :ff], p[:, at + 16] + d[:, ff:]).to(BF16)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "moe":
        T, W, ff, E, top, sff = case["rows"], case["W"], case["ff"], case["experts"], case["top"], case["shared"]
        mats = 3 if case["act"].endswith("glu") else 2
        chosen = E * (1.0 - (1.0 - top / E) ** T)               # distinct experts, expected
        router = 0 if case["router"] == "table" else E * W * 4
        return {"bytes": int(mats * W * 2 * (chosen * ff + sff) + router + T * W * (2 + 4)),
                "flops": int(2 * T * W * (mats * (top * ff + sff) + (E if router else 0)))}
    lens, widths = _requests(case), _widths(case)
    T, K, N, S, r = sum(lens), case["K"], sum(widths), len(widths), case["rank"]
    adapters = _adapters_of(case, list(range(case["slots"])))
    used, rows = len({a for a in adapters if a >= 0}), sum(n for n, a in zip(lens, adapters) if a >= 0)
    nbytes = rows * K * 2 + used * (S * K + N) * r * 2
    nbytes += T * N * (4 if case["plane"] else 2 + 2) if case["kind"] == "lora" else T * N * 4 * case["splits"] + T * case["ff"] * 2
    return {"bytes": int(nbytes), "flops": int(2 * rows * r * (S * K + N))}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------
def _silu64(z):
    return z * torch.sigmoid(z)


def _act64(name, g, u):
    if name == "silu_glu":
        return _silu64(g) * u
    if name == "clamped_glu":
        g, u = torch.minimum(g, torch.full_like(g, LIMIT)), torch.clamp(u, min=-LIMIT, max=LIMIT)
        return _silu64(SLOPE * g) / SLOPE * (u + 1.0)
    if name == "relu2":
        return torch.relu(u) * torch.relu(u)
    return torch.nn.functional.gelu(u, approximate="none" if name == "gelu" else "tanh")


def _exact_moe(st):
    case, h = st["case"], st["h"].to(F64)
    T, E, top = h.shape[0], case["experts"], case["top"]
    out = torch.zeros_like(h)

    def expert(ex, e, row):
        g = None if ex["gate"] is None else ex["gate"][e].to(F64) @ row
        return ex["down"][e].to(F64) @ _act64(case["act"], g, ex["up"][e].to(F64) @ row)
    for t in range(T):
        if case["router"] == "table":
            chosen = [(int(e), 1.0 / top) for e in st["table"][int(st["ids"][t])].tolist()]
        else:
            z = (st["router"].to(F64) @ h[t]).tolist()
            bias = [0.0] * E if st["bias"] is None else st["bias"].to(F64).tolist()
            if case["router"] == "softmax":
                z = [a + b for a, b in zip(z, bias)]
                score = pick = z
            else:
                if case["router"] == "softmax_all":
                    big = max(z)
                    total = math.fsum(math.exp(v - big) for v in z)
                    score = [math.exp(v - big) / total for v in z]
                else:
                    score = [1.0 / (1.0 + math.exp(-v)) for v in z]
                pick = [a + b for a, b in zip(score, bias)]
            open_ = list(range(E))
            if case["groups"] > 1:
                size = E // case["groups"]
                best = [sorted(pick[i * size:(i + 1) * size], reverse=True) for i in range(case["groups"])]
                rank = [v[0] if case["router"] == "softmax_all" else sum(v[:2]) for v in best]
                kept = sorted(range(case["groups"]), key=lambda i: (-rank[i], i))[:case["keep"]]
                open_ = [e for e in open_ if e // size in kept]
            first = sorted(open_, key=lambda e: (-pick[e], e))[:top]
            if case["router"] == "softmax":
                ws = [math.exp(z[e] - z[first[0]]) for e in first]
            else:
                ws = [score[e] for e in first]
            total = 1.0 if case["router"] == "softmax_all" else math.fsum(ws) + (1e-20 if case["router"] == "sigmoid" else 0.0)
            chosen = [(e, w / total) for e, w in zip(first, ws)]
        for e, w in chosen:
            out[t] += w * expert(st["experts"], e, h[t])
        if st["shared"] is not None:
            gate = 1.0 if st["shared_gate"] is None else torch.sigmoid(st["shared_gate"].to(F64) @ h[t])
            out[t] += gate * expert(st["shared"], 0, h[t])
    return {"out": out}


def exact(case, seed):
    global own
    was, own = own, False                # inputs only
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "moe":
        return _exact_moe(st)
    x = st["x"].to(F64)
    T, widths = x.shape[0], st["widths"]
    d = x.new_zeros(T, sum(widths))
    for s, rows in st["rows"]:
        if s >= 0:
            low = torch.einsum("tk,srk->tsr", x[rows], st["a"][s].to(F64)) * st["scale"][s]
            cols = torch.split(st["b"][s].to(F64), widths)
            d[rows] = torch.cat([torch.einsum("tr,nr->tn", low[:, i], c) for i, c in enumerate(cols)], 1)
    if case["kind"] == "lora":
        return {"out": d if st["base"] is None else d + st["base"].to(F64)}
    ff, half = case["ff"], case["half"]
    p = st["planes"].to(F64).sum(0)
    tiles = p.shape[1] // (2 * half)
    p = p.view(T, tiles, half // 16, 2, 16)
    gate, up = p[:, :, :, 0].reshape(T, -1)[:, :ff], p[:, :, :, 1].reshape(T, -1)[:, :ff]
    return {"act": _silu64(gate + d[:, :ff]) * (up + d[:, ff:])}
