"""Operators of a search over several continuations of a prompt, as cases that can be timed and checked.

Kinds:

  select   one step of a beam search: of the continuations of every beam by every token of the vocabulary the n best of a request, with the beam each came from
  reorder  the recurrent states of beams follow them: row i of a request becomes what row parent[i] was, in place, for all layers
  fork     page tables of a paged cache follow the beams: tables and counts of holders, pages for the next token, copies of pages that two rows would write to
  compact  pages in use move to the front of a cache, tables with them
  attn     attention of one new token a row over a paged cache in which rows of a request share pages

``run`` computes them in their plain form, or (``own``) through vox_serve_b200.ops.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64


def _device():
    return torch.device("cuda", torch.cuda.current_device())


# ---- the cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the first step of one small search over a codebook: only the first beam is alive
        {"name": "select_first", "kind": "select", "groups": 1, "width": 2, "n": 4, "vocab": 2051, "dtype": "bf16", "masked": 0.0, "alive": 1, "ended": 0,
         "weight": False},
        # a text model of odd vocabulary, fp32 logits, beams that have ended, ranked by length
        {"name": "select_text_5", "kind": "select", "groups": 16, "width": 5, "n": 10, "vocab": 32003, "dtype": "f32", "masked": 0.0, "alive": 5, "ended": 1,
         "weight": True},
        # a speech model's whole vocabulary, of which a step allows the audio tokens
        {"name": "select_speech_16", "kind": "select", "groups": 16, "width": 16, "n": 32, "vocab": 156940, "dtype": "bf16", "masked": 0.8, "alive": 16, "ended": 0,
         "weight": False},
        # one request of a small recurrent model: nothing but latency
        {"name": "reorder_one", "kind": "reorder", "groups": 1, "width": 4, "kept": 2, "layers": 6, "state": 1000, "conv": 903, "dtype": "bf16"},
        # eight requests on state-space layers: a megabyte of state a row and layer beside the last inputs of a short convolution
        {"name": "reorder_states_8", "kind": "reorder", "groups": 8, "width": 8, "kept": 3, "layers": 12, "state": 262144, "conv": 6912, "dtype": "f32"},
        # the step of a search on eight prompts: rows take over their parents' pages and get room for a token
        {"name": "fork_step_8", "kind": "fork", "groups": 8, "width": 8, "kept": 5, "dead": 0, "prompt": 700, "new": 90, "page": 64, "layers": 16, "heads": 8,
         "dim": 64, "spare": 160},
        # sixteen continuations of one long prompt in small pages
        {"name": "fork_prompt_16", "kind": "fork", "groups": 1, "width": 16, "kept": 1, "dead": 0, "prompt": 8005, "new": 0, "page": 16, "layers": 24, "heads": 2,
         "dim": 64, "spare": 40},
        # a cache after many requests came and went, half of it in use
        {"name": "compact_half", "kind": "compact", "groups": 24, "width": 1, "dead": 0, "prompt": 1100, "new": 33, "page": 64, "layers": 16, "heads": 8, "dim": 64,
         "spare": 300, "moved": 140},
        # a small pool in small pages: a handful of pages to move
        {"name": "compact_few", "kind": "compact", "groups": 3, "width": 4, "dead": 1, "prompt": 131, "new": 17, "page": 16, "layers": 5, "heads": 2, "dim": 64,
         "spare": 21, "moved": 9},
        # one search on a short prompt
        {"name": "attn_one_4", "kind": "attn", "groups": 1, "width": 4, "dead": 0, "prompt": 150, "new": 21, "page": 16, "q_heads": 14, "heads": 2, "dim": 64,
         "spare": 3},
        # eight searches on prompts of some thousand tokens
        {"name": "attn_prompts_8", "kind": "attn", "groups": 8, "width": 8, "dead": 1, "prompt": 4050, "new": 300, "page": 128, "q_heads": 16, "heads": 8, "dim": 128,
         "spare": 0},
        # a long document, many query heads on few key heads
        {"name": "attn_document_5", "kind": "attn", "groups": 2, "width": 5, "dead": 0, "prompt": 61007, "new": 97, "page": 48, "q_heads": 32, "heads": 2, "dim": 128,
         "spare": 5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng, kind):
    G, W = _log(rng, 1, 32), rng.randint(1, 16)
    if kind == "select":
        return {"kind": kind, "groups": G, "width": W, "n": rng.randint(1, 2 * W), "vocab": _log(rng, 300, 170000), "dtype": rng.choice(("bf16", "f32")),
                "masked": rng.choice((0.0, 0.0, 0.3, 0.9)), "alive": rng.choice((1, W, W, W)), "ended": rng.choice((0, 0, 1, W // 3)), "weight": rng.random() < 0.4}
    if kind == "reorder":
        W = max(W, 2)
        return {"kind": kind, "groups": G, "width": W, "kept": rng.randint(1, W - 1), "layers": rng.randint(1, 24), "state": _log(rng, 64, 262144),
                "conv": _log(rng, 64, 16384), "dtype": rng.choice(("bf16", "f32"))}
    case = {"kind": kind, "groups": G, "width": W, "dead": rng.choice((0, 0, 1 if W > 1 else 0)), "prompt": _log(rng, 1, 60000), "new": _log(rng, 1, 600),
            "page": rng.choice((16, 32, 48, 64, 128)), "heads": rng.choice((1, 2, 3, 4, 8)), "dim": rng.choice((64, 128)), "spare": _log(rng, 1, 300)}
    if kind == "attn":
        case["q_heads"] = case["heads"] * rng.choice((1, 2, 3, 4, 7, 8, 16))
        return case
    case["layers"] = rng.randint(1, 28)
    if kind == "fork":
        case["kept"] = rng.randint(1, W - case["dead"])
        case["spare"] += G * W * (2 + 1)
    else:
        case["moved"] = -1                                     # set once the number of pages is known
    return case


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("select", "reorder", "fork", "compact", "attn"))
    top = max(_size(c) for c in listed() if c["kind"] == kind)
    while True:
        case = _draw_once(rng, kind)
        if _size(case) <= top:
            break
    if kind == "compact":
        used = _pages_used(case)
        case["moved"] = rng.randint(0, min(used, case["spare"]))
    return case


def _size(case):
    """what bounds a draw: bytes that a state holds or a pass reads"""
    kind = case["kind"]
    if kind == "select":
        return case["groups"] * case["width"] * case["vocab"] * (2 if case["dtype"] == "bf16" else 4)
    if kind == "reorder":
        return case["groups"] * case["width"] * case["layers"] * (case["state"] * 4 + case["conv"] * 4)
    page = case["page"] * case["heads"] * case["dim"] * 4
    if kind == "attn":                                         # (the plain form gathers every row's keys by itself)
        return case["groups"] * case["width"] * (case["prompt"] + case["new"]) * case["heads"] * case["dim"]
    return (_pages_used(case) + case["spare"]) * page * case["layers"]


# ---- rows of a paged cache ------------------------------------------------------------------------------------------------------
def _tokens(case, g):
    """prompt tokens and tokens of a row of request g (uneven: the last request has the longest prompt)"""
    G = case["groups"]
    p = max(1, case["prompt"] * (G + g + 1) // (2 * G))
    return p, p + case["new"]


def _classes(case, g):
    """pages of request g: for every column the number of different pages that its rows hold there.  Whole pages of the prompt are held by all rows; behind
    them the rows part, more with every page; the last page is every row's own"""
    W, P = case["width"] - case["dead"], case["page"]
    p, n = _tokens(case, g)
    cols, whole = -(-n // P), p // P
    if case["kind"] == "fork" and case["new"] == 0:            # one row has read the prompt, the others are still empty
        return [1] * cols
    return [1 if c < whole and c < cols - 1 else W if c == cols - 1 else min(W, 2 << min(c - whole, 20)) for c in range(cols)]


def _pages_used(case):
    return sum(sum(_classes(case, g)) for g in range(case["groups"]))


def _columns(case):
    return max(len(_classes(case, g)) for g in range(case["groups"])) + 1


def _held(case):
    """(page numbers [rows, columns] with pages counted in the order of requests, columns and rows, -1: none; tokens of every row)"""
    W, alive, cols = case["width"], case["width"] - case["dead"], _columns(case)
    if case["kind"] == "fork" and case["new"] == 0:
        alive = 1
    tables, tokens, used = [], [], 0
    row = torch.arange(alive)
    for g in range(case["groups"]):
        classes = torch.tensor(_classes(case, g))
        first = used + torch.cumsum(classes, 0) - classes
        t = torch.full((W, cols), -1, dtype=I64)
        t[:alive, :len(classes)] = first[None] + row[:, None] * classes[None] // alive
        tables.append(t)
        tokens += [_tokens(case, g)[1]] * alive + [0] * (W - alive)
        used += int(classes.sum())
    return torch.cat(tables), torch.tensor(tokens, dtype=I32), used


def _parents(case, g):
    """row that every row of a request continues: ``kept`` rows go on where they are, the others start again as copies of these in turn; dead rows stay
    dead.  (Taken once or twice the step leaves the same rows.)"""
    W = case["width"]
    alive = W - case.get("dead", 0)
    order = torch.randperm(alive, generator=g, device=_device()).cpu() if case.get("new", 1) else torch.arange(alive)
    parent = torch.full((W,), -1, dtype=I32)
    kept, rest = order[:case["kept"]], order[case["kept"]:]
    parent[kept] = kept.to(I32)
    parent[rest] = kept[torch.arange(len(rest)) % len(kept)].to(I32)
    return parent


# ---- what a user's program has in hand ---------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    return g


def _rand(g, *shape, std=1.0, dtype=BF16):
    out = torch.empty(shape, dtype=dtype, device=_device())
    return out.normal_(0.0, std, generator=g)


def _prepare_select(case, seed):
    g = _gen(seed)
    B, W, V = case["groups"], case["width"], case["vocab"]
    # a few likely tokens over a broad rest, as a language model's output has them
    z = _rand(g, B * W, V, std=2.0, dtype=F32)
    z += 9.0 * torch.exp(_rand(g, B * W, V, dtype=F32) - 3.0)
    if case["masked"]:
        open_ = max(1, int(V * (1.0 - case["masked"])))
        z[:, :V - open_] = -math.inf                           # audio tokens stand behind the text's
    st = {"case": case, "logits": z.to(BF16 if case["dtype"] == "bf16" else F32)}
    scores = -25.0 * torch.rand(B, W, generator=g, device=_device()) - 5.0
    scores = torch.sort(scores, 1, descending=True)[0]
    scores[:, case["alive"]:] = -math.inf
    st["scores"] = scores
    st["ended"] = st["weight"] = None
    st["end"] = V - 1
    if case["ended"]:
        st["ended"] = torch.zeros(B, W, dtype=torch.bool, device=_device())
        st["ended"][:, :case["ended"]] = torch.rand(B, case["ended"], generator=g, device=_device()) < 0.7
    if case["weight"]:
        lens = torch.randint(10, 90, (B, W), generator=g, device=_device()).to(F32)
        st["weight"] = lens ** -0.8
    return st


def _prepare_reorder(case, seed):
    g = _gen(seed)
    B, W, L = case["groups"], case["width"], case["layers"]
    conv = BF16 if case["dtype"] == "bf16" else F32
    st = {"case": case, "parent": torch.stack([_parents(case, g) for _ in range(B)]).to(_device())}
    # a pool of slots, of which the requests have these
    slots = B * W + 3
    st["slots"] = torch.randperm(slots, generator=g, device=_device())[:B * W].to(I32).view(B, W)
    st["states"] = [t for _ in range(L) for t in (_rand(g, slots, case["state"], dtype=F32), _rand(g, slots, case["conv"], dtype=conv))]
    return st


def _prepare_pages(case, seed):
    g = _gen(seed)
    W, P, H, D, L = case["width"], case["page"], case["heads"], case["dim"], case.get("layers", 1)
    held, tokens, used = _held(case)
    pages = used + case["spare"]
    if case["kind"] == "compact":                              # ``moved`` of the pages in use stand behind the first ``used``
        low = torch.randperm(used, generator=g, device=_device())[:used - case["moved"]]
        high = used + torch.randperm(case["spare"], generator=g, device=_device())[:case["moved"]]
        ids = torch.cat([low, high])
        ids = ids[torch.randperm(used, generator=g, device=_device())]
    else:
        ids = torch.randperm(pages, generator=g, device=_device())[:used]
    held = held.to(_device())
    table = torch.where(held >= 0, ids[held.clamp(min=0)], held).to(I32)
    st = {"case": case, "table": table, "tokens": tokens.to(_device()), "cache": _rand(g, L, pages, 2, P, H, D)}
    st["refs"] = torch.bincount(table[table >= 0].long(), minlength=pages).to(I32)
    if case["kind"] == "fork":
        st["src"] = torch.stack([_parents(case, g) for _ in range(case["groups"])]).to(_device())
    if case["kind"] == "attn":
        st["q"] = _rand(g, table.shape[0], case["q_heads"], D, std=1.5)
        if own:
            from vox_serve_b200 import ops
            # a step's list of pages: made once, read by every layer
            plan = ops.SharedPlan(table.shape[0], W, table.shape[1], P, case["q_heads"], H, D, _device())
            st["plan"] = ops.shared_plan(plan, table, st["tokens"])
    elif own:
        from vox_serve_b200 import ops
        # the tables that a step reads and the ones it leaves
        st["pool"], st["next"] = (ops.PagePool(pages, P, table.shape[0], table.shape[1], _device()) for _ in range(2))
        st["pool"].load(table, st["tokens"])
    return st


def prepare(case, seed):
    return {"select": _prepare_select, "reorder": _prepare_reorder}.get(case["kind"], _prepare_pages)(case, seed)


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def _plain_select(st):
    """64 bits: a choice may hang on the last digits of a sum"""
    case, z = st["case"], st["logits"].to(F64)
    B, W, V, n = case["groups"], case["width"], case["vocab"], case["n"]
    score = st["scores"].to(F64).view(B * W, 1)
    top = z.max(1, keepdim=True)[0]
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    total = score + (z - top - torch.log(torch.exp(z - top).sum(1, keepdim=True)))
    if st["ended"] is not None:                                # an ended beam goes on as it is, under the end token
        over = st["ended"].view(B * W, 1)
        total = torch.where(over, torch.full_like(total, -math.inf), total)
        total[:, st["end"]] = torch.where(over[:, 0], score[:, 0], total[:, st["end"]])
    rank = total if st["weight"] is None else total * st["weight"].to(F64).view(B * W, 1)
    rank, token = torch.sort(rank, dim=1, descending=True, stable=True)
    k = min(n, V)
    total = total.gather(1, token[:, :k]).view(B, W * k)
    token = token[:, :k].reshape(B, W * k)
    rank, at = torch.sort(rank[:, :k].reshape(B, W * k), dim=1, descending=True, stable=True)
    short = n - min(n, W * k)
    rank, at = rank[:, :n], at[:, :n]
    none = rank == -math.inf
    out = [total.gather(1, at).to(F32), torch.where(none, torch.full_like(at, -1), at // k).to(I32),
           torch.where(none, torch.full_like(at, -1), token.gather(1, at))]
    fill = (-math.inf, -1, -1)
    return [torch.nn.functional.pad(t, (0, short), value=f) for t, f in zip(out, fill)]


def _plain_reorder(st):
    parent, slots = st["parent"].long(), st["slots"].long()
    B, W = parent.shape
    src = torch.where(parent >= 0, parent, torch.arange(W, device=parent.device))
    rows = slots.gather(1, src).view(-1)
    return [t.index_copy_(0, slots.view(-1), t[rows]) for t in st["states"]]


def _move(cache, src, dst, slots):
    """the first slots[i] tokens of page src[i] to page dst[i], in every layer"""
    keep = torch.arange(cache.shape[3], device=cache.device)[None] < slots[:, None]
    cache[:, dst] = torch.where(keep[None, :, None, :, None, None], cache[:, src], cache[:, dst])


def _plain_fork(st):
    case, cache, P = st["case"], st["cache"], st["case"]["page"]
    R, cols = st["table"].shape
    src = (st["src"].long() + torch.arange(case["groups"], device=cache.device)[:, None] * case["width"]).view(-1)
    gone = st["src"].view(-1) < 0
    src = src.clamp(min=0)
    tokens = torch.where(gone, torch.zeros_like(src), st["tokens"].long()[src])
    table = torch.where(gone[:, None], torch.full_like(st["table"], -1), st["table"][src]).long()
    pages = cache.shape[1]
    row = torch.arange(R, device=cache.device)

    def holders(t):
        return torch.zeros(pages + 1, dtype=I64, device=t.device).index_add_(0, torch.where(t >= 0, t, pages).view(-1), torch.ones_like(t).view(-1))[:pages]
    # a page that is not full yet belongs to one row: the first that holds it keeps it, the others get copies
    part = tokens % P
    tail = table.gather(1, (tokens // P)[:, None])[:, 0]
    at = torch.where(part > 0, tail, torch.full_like(tail, pages))
    first = torch.full((pages + 1,), R, device=cache.device).scatter_reduce_(0, at, row, "amin")
    copy = (part > 0) & (first[at] != row)
    grown = torch.where(gone, tokens, tokens + 1)
    have, want = (tokens + P - 1) // P, (grown + P - 1) // P
    need = copy.long() + want - have
    base = torch.cumsum(need, 0) - need
    free = torch.sort((holders(table) > 0).long(), stable=True)[1]          # the lowest numbers first
    col = torch.arange(cols, device=cache.device)[None]
    table = torch.where((col >= have[:, None]) & (col < want[:, None]), free[(base + copy.long())[:, None] + (col - have[:, None]).clamp(min=0)], table)
    table = torch.where((col == (tokens // P)[:, None]) & copy[:, None], free[base][:, None], table)
    _move(cache, tail[copy], free[base][copy], part[copy])
    return {"table": table.to(I32), "tokens": grown.to(I32), "refs": holders(table).to(I32), "cache": cache}


def _plain_compact(st):
    cache, refs = st["cache"], st["refs"]
    page = torch.arange(refs.shape[0], device=cache.device)
    used = refs > 0
    total = used.sum()
    out, hole = used & (page >= total), ~used & (page < total)
    src, dst = page[out], page[hole]
    new = torch.where(used, page, torch.full_like(page, -1))
    new[src] = dst
    cache[:, dst] = cache[:, src]
    table = torch.where(st["table"] >= 0, new[st["table"].clamp(min=0).long()], st["table"].long())
    after = torch.zeros_like(refs)
    after[new[used]] = refs[used]
    return {"table": table.to(I32), "tokens": st["tokens"], "refs": after, "moved": new.to(I32), "cache": cache}


def _plain_attn(st):
    case, q = st["case"], st["q"].float()
    R, Hq, D = q.shape
    H, P = case["heads"], case["page"]
    kv = st["cache"][0][st["table"].clamp(min=0).long()]       # [rows, columns, 2, P, H, D]
    k, v = (kv[:, :, i].reshape(R, -1, H, D).permute(0, 2, 1, 3).float() for i in (0, 1))
    s = torch.matmul(q.view(R, H, Hq // H, D), k.transpose(2, 3)) / math.sqrt(D)
    seen = (torch.arange(k.shape[2], device=q.device)[None] < st["tokens"][:, None])[:, None, None]
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.max(3, keepdim=True)[0].clamp(min=-1e30)
    e = torch.exp(s - top)
    total = e.sum(3, keepdim=True)
    out = torch.matmul(e, torch.where(seen.view(R, 1, -1, 1), v, torch.zeros_like(v))) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(R, Hq, D).to(BF16)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "select":
            score, parent, token = _plain_select(state)
            return {"score": score, "parent": parent, "token": token}
        return {"reorder": _plain_reorder, "fork": _plain_fork, "compact": _plain_compact, "attn": _plain_attn}[kind](state)
    from vox_serve_b200 import ops
    if kind == "select":
        step = ops.beam_select(state["logits"], state["scores"], case["n"], weight=state["weight"], ended=state["ended"], end_token=state["end"])
        return {"score": step.scores, "parent": step.parent, "token": step.token}
    if kind == "reorder":
        return ops.beam_reorder(state["states"], state["parent"], state["slots"])
    if kind == "fork":
        pool = ops.fork_pages(state["pool"], state["src"], grow=1, caches=[state["cache"]], out=state["next"])
        return {"table": pool.table, "tokens": pool.tokens, "refs": pool.refs, "cache": state["cache"]}
    if kind == "compact":
        pool = ops.compact_pages(state["pool"], caches=[state["cache"]], out=state["next"])
        return {"table": pool.table, "tokens": pool.tokens, "refs": pool.refs, "moved": pool.moved, "cache": state["cache"]}
    return ops.shared_attn(state["q"], state["cache"], 0, state["plan"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    kind, B, W = case["kind"], case["groups"], case["width"]
    if kind == "select":
        rows = B * min(case["alive"], W)
        each = 2 if case["dtype"] == "bf16" else 4
        rows -= B * min(case["ended"], case["alive"]) * 0.7            # (expected: their logits need not be read)
        return {"bytes": int(rows * case["vocab"] * each + B * W * 4 + B * case["n"] * 16), "flops": int(3 * rows * case["vocab"])}
    if kind == "reorder":
        moved, read = W - case["kept"], min(case["kept"], W - case["kept"])
        row = case["layers"] * (case["state"] * 4 + case["conv"] * (2 if case["dtype"] == "bf16" else 4))
        return {"bytes": int(B * (moved + read) * row + B * W * 8), "flops": 0}
    P, H, D, L = case["page"], case["heads"], case["dim"], case.get("layers", 1)
    token = 2 * H * D * 2
    used, cols = _pages_used(case), _columns(case)
    tables = 2 * (B * W * cols + B * W + used + case["spare"]) * 4
    if kind == "fork":
        alive = W - case["dead"]
        filled = copied = 0
        for g in range(B):
            part = _tokens(case, g)[1] % P
            copied += part * (alive - case["kept"])
            filled += part * min(case["kept"], alive - case["kept"])
        return {"bytes": int(tables + (copied + filled) * token * L), "flops": 0}
    if kind == "compact":
        return {"bytes": int(tables + 2 * case["moved"] * P * token * L), "flops": 0}
    alive, read, flops = W - case["dead"], 0, 0
    for g in range(B):
        n, classes = _tokens(case, g)[1], _classes(case, g)
        read += sum(c * min(P, n - i * P) for i, c in enumerate(classes))
        flops += 4 * alive * n * case["q_heads"] * D
    return {"bytes": int(read * token + 2 * B * W * case["q_heads"] * D * 2 + B * W * cols * 4), "flops": int(flops)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------
def _exact_select(st):
    case = st["case"]
    B, W, V, n = case["groups"], case["width"], case["vocab"], case["n"]
    score = torch.full((B, n), -math.inf, dtype=F64)
    parent, token = torch.full((B, n), -1, dtype=I32), torch.full((B, n), -1, dtype=I64)
    z = st["logits"].to(F64).view(B, W, V)
    for b in range(B):
        found = []
        for w in range(W):
            s, by = float(st["scores"][b, w]), 1.0 if st["weight"] is None else float(st["weight"][b, w])
            if s == -math.inf:
                continue
            if st["ended"] is not None and bool(st["ended"][b, w]):
                found.append((-s * by, w, st["end"], s))
                continue
            p = s + torch.log_softmax(z[b, w], 0)
            edge = torch.topk(p, min(n, V))[0][-1]
            for v in torch.nonzero((p >= edge) & (p > -math.inf)).view(-1).tolist() if edge > -math.inf else torch.nonzero(p > -math.inf).view(-1).tolist():
                found.append((-float(p[v]) * by, w, v, float(p[v])))
        for i, (_, w, v, s) in enumerate(sorted(found)[:n]):
            score[b, i], parent[b, i], token[b, i] = s, w, v
    return {"score": score, "parent": parent, "token": token}


def _exact_attn(st):
    case, q = st["case"], st["q"].to(F64)
    R, Hq, D = q.shape
    H, P = case["heads"], case["page"]
    out = torch.zeros_like(q)
    for r, n in enumerate(st["tokens"].tolist()):
        if n:
            pages = st["table"][r, :-(-n // P)].long()
            kv = st["cache"][0, pages].to(F64).transpose(0, 1).reshape(2, -1, H, D)[:, :n].repeat_interleave(Hq // H, 2)
            p = torch.softmax(torch.einsum("hd,nhd->hn", q[r], kv[0]) * D ** -0.5, 1)
            out[r] = torch.einsum("hn,nhd->hd", p, kv[1])
    return out


def exact(case, seed):
    global own
    was, own = own, False                # inputs only
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "select":
        return _exact_select(st)
    if case["kind"] == "attn":
        return _exact_attn(st)
    return None                          # (nothing is computed: states, pages and tables move)
