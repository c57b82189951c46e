"""Measured calls of the paged serving operators: block tables and slot maps from request
lengths, the cache write through the slot map, attention of a chunk of new tokens over the paged
cache, and the verification of drafted tokens.

A batch is ragged and token-major: request b brings rows `starts[b]` to `starts[b + 1]` of the
step's T rows, behind `past[b]` tokens that its cache holds. A row's slot is its place in the
cache: block · block size + offset. Whole numbers are u32 in the framework and int32 with the same
bits here; −1 is "none".

With `own` false a pass computes the operators in plain torch operations; with `own` true it calls
the framework: a program prepared once per shape (`HipDevice.prepare`), as a serving loop keeps it,
and run by `Executable.execute_static` on the caller's tensors.

Kinds:
  tables   block tables, slots and positions of a step from the requests' lengths
  write    the step's new K and V rows into the paged cache
  attn     causal attention of the step's rows over the cache, optionally a sliding window
  verify   drafted tokens against the target's probabilities, from given random numbers
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ── the cases ────────────────────────────────────────────────────────────────

def listed():
    return [
        # one decode step of a small batch: most requests stay inside the block they have
        {"name": "tables_8", "kind": "tables", "b": 8, "ctx": 2048, "new": 1, "mix": "same", "block": 16, "pad": 0},
        # a large batch with prompts of all lengths among its decodes, padded rows behind it
        {"name": "tables_512", "kind": "tables", "b": 512, "ctx": 16384, "new": 512, "mix": "ragged", "block": 16, "pad": 777},
        # the rows of a decode batch of eight, the widths of the shipped decode step
        {"name": "write_8", "kind": "write", "b": 8, "ctx": 2048, "new": 1, "mix": "same", "nkv": 8, "hd": 64, "block": 16,
         "rows": "f32", "cache": "bf16", "pad": 0},
        # the rows of prompt chunks, heads of 128
        {"name": "write_4096", "kind": "write", "b": 8, "ctx": 4096, "new": 512, "mix": "same", "nkv": 8, "hd": 128, "block": 64,
         "rows": "bf16", "cache": "bf16", "pad": 100},
        # one token of one request over the shipped step's 2048-entry cache: latency
        {"name": "attn_1", "kind": "attn", "b": 1, "ctx": 2048, "new": 1, "mix": "same", "nkv": 8, "rep": 4, "hd": 64, "block": 16,
         "window": 0, "type": "bf16", "pad": 0},
        # a decode batch of uneven lengths: the cache's bytes
        {"name": "attn_64", "kind": "attn", "b": 64, "ctx": 8000, "new": 1, "mix": "same", "nkv": 8, "rep": 4, "hd": 128, "block": 16,
         "window": 0, "type": "bf16", "pad": 0},
        # drafts being verified: five rows a request, more queries than one matrix tile holds
        {"name": "attn_draft_24", "kind": "attn", "b": 24, "ctx": 5000, "new": 5, "mix": "same", "nkv": 8, "rep": 4, "hd": 64, "block": 32,
         "window": 0, "type": "f16", "pad": 0},
        # a prompt's chunk beside the decodes of 40 other requests, some of them idle, in padded rows
        {"name": "attn_mixed", "kind": "attn", "b": 41, "ctx": 6000, "new": 1500, "mix": "one", "nkv": 8, "rep": 4, "hd": 64, "block": 16,
         "window": 1024, "type": "bf16", "pad": 36},
        # a long prompt's chunk over what was prefilled before it: the matrix cores
        {"name": "attn_4096", "kind": "attn", "b": 1, "ctx": 12288, "new": 4096, "mix": "same", "nkv": 8, "rep": 4, "hd": 128, "block": 64,
         "window": 0, "type": "bf16", "pad": 0},
        # one request's four drafts over the shipped vocabulary: latency
        {"name": "verify_1", "kind": "verify", "b": 1, "drafts": 4, "vocab": 128256, "type": "f32", "draft": True},
        # a batch of drafts of uneven numbers, the draft model's probabilities given
        {"name": "verify_64", "kind": "verify", "b": 64, "drafts": 7, "vocab": 128256, "type": "f32", "draft": True},
        # drafts that were looked up, so that they have no probabilities, over a small vocabulary in bf16
        {"name": "verify_200", "kind": "verify", "b": 200, "drafts": 3, "vocab": 32003, "type": "bf16", "draft": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "write", "attn", "attn", "attn", "verify"])
    if kind == "tables":
        return {"kind": kind, "b": _log(rng, 1, 1024), "ctx": _log(rng, 16, 32768), "new": _log(rng, 1, 512),
                "mix": rng.choice(["same", "ragged", "one"]) if rng.random() < 0.5 else "ragged",
                "block": rng.choice([8, 16, 16, 24, 32, 64, 128]), "pad": rng.choice([0, _log(rng, 1, 300)])}
    if kind == "write":
        return {"kind": kind, "b": _log(rng, 1, 64), "ctx": _log(rng, 16, 4096), "new": _log(rng, 1, 128),
                "mix": rng.choice(["same", "ragged"]), "nkv": rng.choice([1, 2, 4, 8]), "hd": rng.choice([64, 64, 80, 96, 128, 128]),
                "block": rng.choice([8, 16, 16, 24, 32, 64]), "rows": rng.choice(["f32", "bf16"]), "cache": "bf16",
                "pad": rng.choice([0, _log(rng, 1, 60)])}
    if kind == "attn":
        c = {"kind": kind, "b": _log(rng, 1, 64), "ctx": _log(rng, 16, 16384), "nkv": rng.choice([1, 2, 4, 8, 8]),
             "rep": rng.choice([1, 2, 4, 4, 4, 7, 8]), "hd": rng.choice([64, 64, 128, 128, 96, 80]),
             "block": rng.choice([16, 16, 32, 64, 128, 24]), "window": 0 if rng.random() < 0.7 else _log(rng, 64, 4096),
             "type": rng.choice(["bf16", "bf16", "f16"]), "pad": rng.choice([0, _log(rng, 1, 60)])}
        c["mix"], c["new"] = rng.choice([("same", 1), ("same", 1), ("same", _log(rng, 2, 9)), ("ragged", _log(rng, 8, 600)),
                                         ("one", _log(rng, 30, 3000))])
        while work(c)["flops"] > 6e11 or work(c)["bytes"] > 2.5e9:
            c["ctx"], c["new"] = max(1, c["ctx"] * 2 // 3), max(1, c["new"] * 3 // 4)
        return c
    vocab, drafts = _log(rng, 500, 160000), _log(rng, 1, 9)
    return {"kind": kind, "b": min(_log(rng, 1, 128), max(1, 512 * 128256 // (vocab * (drafts + 1)))), "drafts": drafts, "vocab": vocab,
            "type": rng.choice(["f32", "f32", "bf16", "f16"]), "draft": rng.random() < 0.7}


def _lengths(case):
    """(past, new) of every request: part of the case, not of its seed."""
    r = random.Random("%(b)d %(ctx)d %(new)d %(mix)s" % case)
    past, new = [], []
    for i in range(case["b"]):
        past.append(case["ctx"] if i == 0 else int(case["ctx"] * r.uniform(0.15, 1.0)))
        if case["mix"] == "same":
            new.append(case["new"])
        elif case["mix"] == "one":
            # a chunk among decodes; now and then a request has nothing this step
            new.append(case["new"] if i == case["b"] // 2 else int(r.random() < 0.9))
        else:
            new.append(0 if r.random() < 0.06 else _log(r, 1, case["new"]) if r.random() < 0.7 else 1)
    if sum(new) == 0:
        new[0] = 1
    return past, new


def _drafts(case):
    """Rows of every request: its last token's and one for each draft."""
    r = random.Random("%(b)d %(drafts)d %(vocab)d" % case)
    return [case["drafts"] + 1 if i == 0 or r.random() < 0.7 else r.randint(1, case["drafts"] + 1) for i in range(case["b"])]


def _ceil(a, b):
    return -(-a // b)


def _prefix(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


# ── inputs ───────────────────────────────────────────────────────────────────

def _normal(g, shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=g).to(dtype)


def _ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _pages(case, g, lens):
    """Tables of requests of these lengths over blocks in no order: (tables, number of blocks, width)."""
    have = [_ceil(n, case["block"]) for n in lens]
    blocks = sum(have) + 3
    width = max(have) + 2
    order = torch.randperm(blocks, generator=g, device="cuda", dtype=torch.int32)
    flat = torch.full((case["b"] * width,), -1, device="cuda", dtype=torch.int32)
    at = torch.cat([torch.arange(b * width, b * width + n) for b, n in enumerate(have)]).cuda()
    flat[at] = order[:at.numel()]
    return flat.view(case["b"], width), blocks, width


def _inputs(case, seed):
    """The case's tensors by name, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    if kind == "verify":
        return _verify_inputs(case, g)
    past, new = _lengths(case)
    rows = sum(new) + case["pad"]
    t = {"past": _ints(past), "starts": _ints(_prefix(new))}
    if kind == "tables":
        block = case["block"]
        # what the requests hold: their blocks, now and then one more, left over from rejected drafts
        more = random.Random(seed)
        held = [_ceil(p, block) + int(more.random() < 0.1) for p in past]
        taken = 5
        width = max(_ceil(p + n, block) for p, n in zip(past, new)) + 2
        spare = sum(_ceil(p, block) + 1 for p in past)
        free = taken + 9 + sum(_ceil(p + n, block) - _ceil(p, block) for p, n in zip(past, new))
        order = torch.randperm(spare + free, generator=g, device="cuda", dtype=torch.int32)
        tables = torch.full((case["b"] * width,), -1, device="cuda", dtype=torch.int32)
        at = torch.cat([torch.arange(b * width, b * width + n) for b, n in enumerate(held)]).cuda()
        tables[at] = order[:at.numel()]
        t.update(new=_ints(new), held=_ints(held + [taken]), free=order[spare:].contiguous(), tables=tables.view(case["b"], width))
        del t["starts"]
        for name, shape in (("starts", case["b"] + 1), ("slots", rows), ("positions", rows), ("held_next", case["b"] + 1)):
            t[name] = torch.zeros(shape, device="cuda", dtype=torch.int32)
        return t
    lens = [p + n for p, n in zip(past, new)]
    t["tables"], blocks, _ = _pages(case, g, lens)
    shape = (blocks, case["nkv"], case["block"], case["hd"])
    if kind == "write":
        cache = _TYPES[case["cache"]]
        t["k_cache"], t["v_cache"] = _normal(g, shape, dtype=cache), _normal(g, shape, dtype=cache)
        for name in ("k", "v"):
            t[name] = _normal(g, (rows, case["nkv"], case["hd"]), dtype=_TYPES[case["rows"]])
        block = case["block"]
        req = _ints([b for b, n in enumerate(new) for _ in range(n)]).long()
        pos = _ints([p + i for p, n in zip(past, new) for i in range(n)]).long()
        slots = t["tables"][req, pos // block] * block + (pos % block).int()
        # the padded rows hold what an earlier, longer step left there
        t["slots"] = torch.cat((slots, torch.zeros(case["pad"], device="cuda", dtype=torch.int32)))
        return t
    typ = _TYPES[case["type"]]
    t["q"] = _normal(g, (rows, case["nkv"] * case["rep"], case["hd"]), dtype=typ)
    t["k_cache"], t["v_cache"] = _normal(g, shape, dtype=typ), _normal(g, shape, dtype=typ)
    t["o"] = torch.zeros_like(t["q"])
    return t


def _verify_inputs(case, g):
    counts = _drafts(case)
    rows, vocab, typ = sum(counts), case["vocab"], _TYPES[case["type"]]
    logits = _normal(g, (rows, vocab), 3.0)
    p = torch.softmax(logits, -1).to(typ)
    t = {"p": p, "starts": _ints(_prefix(counts))}
    # a draft model that agrees with the target in part, and draws its tokens from its own probabilities
    q = torch.softmax(logits.add_(_normal(g, (rows, vocab), 0.7)), -1)
    if case["draft"]:
        t["q"] = q.to(typ)
    noise = torch.empty_like(q).exponential_(generator=g)
    drawn = q.div_(noise).argmax(-1).int()
    first = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    # row r + 1 holds the token drawn behind row r; a request's first row its last token
    t["tokens"] = torch.cat((first[:1], drawn[:-1]))
    t["u"] = torch.rand((rows,), generator=g, device="cuda")
    t["draw"] = torch.rand((case["b"],), generator=g, device="cuda")
    t["out"] = torch.zeros(rows, device="cuda", dtype=torch.int32)
    t["accepted"] = torch.zeros(case["b"], device="cuda", dtype=torch.int32)
    return t


_device = None
_prepared = {}


def _program(case, t):
    """The case's program and the names its buffers go by, built once per shape as a server does."""
    from sanic_amd import ir
    from sanic_amd.program import Program
    ty = {torch.bfloat16: ir.BF16, torch.float16: ir.F16, torch.float32: ir.F32, torch.int32: ir.U32}
    prog = Program()
    kind = case["kind"]

    def node(name):
        return prog.input(name, t[name].shape, ty[t[name].dtype])

    def state(name):
        return prog.state(name, t[name].shape, ty[t[name].dtype])

    if kind == "tables":
        state("tables")
        prog.block_tables("plan", node("past"), node("new"), node("held"), node("free"), "tables", block=case["block"],
                          rows=t["slots"].numel())
        return prog, {"plan.starts": "starts", "plan.slots": "slots", "plan.positions": "positions", "plan.held": "held_next"}
    if kind == "write":
        state("k_cache"), state("v_cache")
        prog.cache_write("write", node("k"), node("v"), node("slots"), node("starts"), "k_cache", "v_cache")
        return prog, {}
    if kind == "attn":
        prog.paged_attention("o", node("q"), node("k_cache"), node("v_cache"), node("tables"), node("starts"), node("past"),
                             window=case["window"], out_dtype=ty[t["q"].dtype])
        return prog, {}
    prog.verify_drafts("check", node("p"), node("q") if case["draft"] else None, node("tokens"), node("starts"), node("u"), node("draw"))
    return prog, {"check.tokens": "out", "check.accepted": "accepted"}


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if case["kind"] != "verify":
        state["lengths"] = _lengths(case)
    else:
        state["counts"] = _drafts(case)
    if own:
        global _device
        from sanic_amd.backend import HipDevice
        if _device is None:
            torch.cuda.init()
            _device = HipDevice(0)
        key = tuple(sorted((k, tuple(v.shape), str(v.dtype)) for k, v in t.items())) + (case.get("block"), case.get("window"))
        if key not in _prepared:
            prog, names = _program(case, t)
            _prepared[key] = (_device.prepare(prog), [b.name for b in prog.buffers if b.role != 3], names)
        exe, buffers, names = _prepared[key]
        state["exe"] = exe
        state["binds"] = {n: _device.wrap(t[names.get(n, n)].data_ptr(), t[names.get(n, n)].numel() * t[names.get(n, n)].element_size())
                          for n in buffers}
    torch.cuda.synchronize()
    return state


_OUTPUTS = {"tables": ("starts", "slots", "positions", "held_next", "tables"), "write": ("k_cache", "v_cache"), "attn": ("o",),
            "verify": ("out", "accepted")}


def run(state):
    case, t = state["case"], state["t"]
    if own:
        state["exe"].execute_static(state["binds"])
    else:
        {"tables": _plain_tables, "write": _plain_write, "attn": _plain_attn, "verify": _plain_verify}[case["kind"]](state, case, t)
    return {n: t[n] for n in _OUTPUTS[case["kind"]]}


# ── the plain forms ──────────────────────────────────────────────────────────

def _plain_tables(state, case, t):
    block, b = case["block"], case["b"]
    rows, width = t["slots"].numel(), t["tables"].shape[1]
    past, held, taken = t["past"].long(), t["held"][:b].long(), t["held"][b].long()
    ends = torch.cumsum(t["new"].long(), 0).clamp(max=rows)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    new = starts[1:] - starts[:-1]
    want = ((past + new + block - 1) // block).clamp(max=width) - held
    want = torch.where(new > 0, want.clamp(min=0), torch.zeros_like(want))
    before = torch.cumsum(want, 0) - want
    got = torch.minimum((t["free"].numel() - taken - before).clamp(min=0), want)
    j = torch.arange(width, device="cuda")[None, :]
    fresh = (j >= held[:, None]) & (j < (held + got)[:, None])
    at = (taken + before - held)[:, None] + j
    tables = torch.where(fresh, t["free"][at.clamp(0, t["free"].numel() - 1)], t["tables"])
    r = torch.arange(rows, device="cuda")
    live = r < starts[b]
    req = (r[:, None] >= starts[None, 1:]).sum(1).clamp(max=b - 1)
    pos = past[req] + r - starts[req]
    page = pos // block
    slot = tables[req, page.clamp(max=width - 1)].long() * block + pos % block
    slot = torch.where(page < (held + got)[req], slot, torch.full_like(slot, -1))
    t["slots"].copy_(torch.where(live, slot.int(), t["slots"]))
    t["positions"].copy_(torch.where(live, pos.int(), t["positions"]))
    t["starts"].copy_(starts)
    t["held_next"].copy_(torch.cat((held + got, (taken + got.sum())[None])))
    t["tables"].copy_(tables)


def _plain_write(state, case, t):
    # the host knows how many rows the step has
    n = sum(state["lengths"][1])
    slots = t["slots"][:n].long()
    block, offset = slots // case["block"], slots % case["block"]
    for src, dst in (("k", "k_cache"), ("v", "v_cache")):
        t[dst][block, :, offset] = t[src][:n].to(t[dst].dtype)


def _plain_attn(state, case, t):
    """Requests with about as many rows go together, padded to the largest of them."""
    nkv, rep = case["nkv"], case["rep"]
    past, new = state["lengths"]
    starts = _prefix(new)
    groups = {}
    for b, n in enumerate(new):
        if n:
            groups.setdefault(n.bit_length(), []).append(b)
    for bs in groups.values():
        rows, keys = max(new[b] for b in bs), max(past[b] + new[b] for b in bs)
        # as many requests at a time as leave the scores at 2 GiB, and a long prompt by its key heads
        some = max(1, (1 << 29) // (nkv * rep * rows * keys))
        heads = 1 if nkv * rep * rows * keys > 1 << 29 else nkv
        for i in range(0, len(bs), some):
            for h in range(0, nkv, heads):
                _plain_group(case, t, [(past[b], new[b], starts[b], b) for b in bs[i:i + some]], slice(h, h + heads))


def _plain_group(case, t, reqs, heads):
    rep, hd, block = case["rep"], case["hd"], case["block"]
    past, new, start, b = (torch.tensor(x).cuda() for x in zip(*reqs))
    rows, keys = max(r[1] for r in reqs), max(r[0] + r[1] for r in reqs)
    pages = t["tables"][b, :_ceil(keys, block)].clamp(min=0).long()
    k, v = (t[n][:, heads][pages].transpose(1, 2).reshape(len(reqs), -1, pages.shape[1] * block, hd)[:, :, :keys].float()
            for n in ("k_cache", "v_cache"))
    i = torch.arange(rows, device="cuda")
    live = i < new[:, None]
    at = (start[:, None] + i).clamp(max=t["q"].shape[0] - 1)
    nkv = k.shape[1]
    q = t["q"].view(t["q"].shape[0], case["nkv"], rep, hd)[at][:, :, heads].permute(0, 2, 3, 1, 4).reshape(len(reqs), nkv, rep * rows, hd).float()
    s = (q @ k.transpose(2, 3).contiguous() * (1.0 / math.sqrt(hd))).view(len(reqs), nkv, rep, rows, keys)
    pos, key = (past[:, None] + i)[:, None, None, :, None], torch.arange(keys, device="cuda")
    hidden = key > pos
    if case["window"]:
        hidden = hidden | (key <= pos - case["window"])
    s.masked_fill_(hidden, -math.inf)
    w = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    o = (w.view(len(reqs), nkv, rep * rows, keys) @ v).view(s.shape[:4] + (hd,)) / w.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4)[live].to(t["o"].dtype)
    t["o"].view(t["o"].shape[0], case["nkv"], rep, hd)[at[live], heads] = o


def _plain_verify(state, case, t):
    b = case["b"]
    starts, p, tokens = t["starts"].long(), t["p"], t["tokens"].long()
    rows, vocab = p.shape
    drafts = starts[1:] - starts[:-1] - 1
    # row r tests the token of row r + 1, but in a request's last row
    r = torch.arange(rows, device="cuda")
    x = tokens[(r + 1).clamp(max=rows - 1)]
    px = p[r, x].double()
    qx = t["q"][r, x].double() if case["draft"] else torch.ones_like(px)
    fine = t["u"].double() * qx < px
    k = torch.arange(case["drafts"] + 1, device="cuda")[None, :]
    at = (starts[:-1, None] + k).clamp(max=rows - 1)
    stop = ~fine[at] | (k >= drafts[:, None])
    accepted = (torch.cumsum(stop, 1) == 0).sum(1)
    row = starts[:-1] + accepted
    left = p[row].double()
    rejected = (accepted < drafts)[:, None]
    if case["draft"]:
        rest = (left - t["q"][row].double()).clamp(min=0)
    else:
        rest = left * (torch.arange(vocab, device="cuda")[None, :] != tokens[(row + 1).clamp(max=rows - 1)][:, None])
    weight = torch.where(rejected & (rest.sum(1, keepdim=True) > 0), rest, left)
    sums = torch.cumsum(weight, 1)
    drawn = (sums <= t["draw"].double()[:, None] * sums[:, -1:]).sum(1)
    last = torch.where(weight > 0, torch.arange(vocab, device="cuda")[None, :], 0).amax(1)
    drawn = torch.minimum(drawn, last)
    own_row = (r[:, None] >= starts[None, 1:]).sum(1)
    i = r - starts[own_row]
    out = torch.where(i < accepted[own_row], x, torch.where(i == accepted[own_row], drawn[own_row], torch.full_like(x, -1)))
    t["out"].copy_(out)
    t["accepted"].copy_(accepted)


# ── what a pass cannot do without ────────────────────────────────────────────

_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def work(case):
    kind, b = case["kind"], case["b"]
    if kind == "verify":
        counts, size = _drafts(case), _SIZE[case["type"]]
        # the row that the last token is drawn from, of the target and as a rule of the draft
        return {"bytes": size * case["vocab"] * b * (2 if case["draft"] else 1) + 16 * sum(counts) + 8 * b,
                "flops": 3 * case["vocab"] * b}
    past, new = _lengths(case)
    rows = sum(new)
    if kind == "tables":
        grown = sum(max(0, _ceil(p + n, case["block"]) - _ceil(p, case["block"])) for p, n in zip(past, new))
        # lengths and held counts in, starts and held counts out, two words a row, two a new block
        return {"bytes": 4 * (5 * b + 3 + 2 * rows + 2 * grown), "flops": 0}
    width = case["nkv"] * case["hd"]
    if kind == "write":
        return {"bytes": rows * (4 + 2 * width * (_SIZE[case["rows"]] + _SIZE[case["cache"]])), "flops": 0}
    w = case["window"]
    pairs = keys = 0
    for p, n in zip(past, new):
        if n == 0:
            continue
        first = max(0, p + 1 - w) if w else 0
        keys += p + n - first
        full = n * p + n * (n + 1) // 2
        if w:
            # what the window hides of the causal triangle: max(0, position + 1 − w) keys a row
            lo, hi = max(0, p + 1 - w), max(0, p + n - w)
            full -= (hi * (hi + 1) - (lo - 1) * lo) // 2 if hi else 0
        pairs += full
    return {"bytes": _SIZE[case["type"]] * (2 * keys * width + 2 * rows * width * case["rep"]) + 4 * _ceil(keys, case["block"]),
            "flops": 4 * pairs * width * case["rep"]}


# ── the same in 64 bits, from the definitions ────────────────────────────────

def exact(case, seed):
    t = _inputs(case, seed)
    return {"tables": _exact_tables, "write": _exact_write, "attn": _exact_attn, "verify": _exact_verify}[case["kind"]](case, t)


def _exact_tables(case, t):
    """The step's bookkeeping request by request, on the host."""
    block, rows = case["block"], t["slots"].numel()
    past, new, held, free = (t[n].tolist() for n in ("past", "new", "held", "free"))
    tables, slots, positions = t["tables"].cpu(), [0] * rows, [0] * rows
    taken, at, starts = held[-1], 0, [0]
    for b in range(case["b"]):
        n = min(new[b], rows - at)
        while n and held[b] * block < past[b] + n and held[b] < tables.shape[1] and taken < len(free):
            tables[b, held[b]] = free[taken]
            held[b] += 1
            taken += 1
        line = tables[b].tolist()
        for i in range(n):
            pos = past[b] + i
            slots[at + i] = line[pos // block] * block + pos % block if pos // block < held[b] else -1
            positions[at + i] = pos
        at += n
        starts.append(at)
    held[-1] = taken
    return {"starts": _ints(starts), "slots": _ints(slots), "positions": _ints(positions), "held_next": _ints(held), "tables": tables}


def _exact_write(case, t):
    out = {}
    slots = t["slots"][:sum(_lengths(case)[1])].long()
    for src, dst in (("k", "k_cache"), ("v", "v_cache")):
        # token-major, so that a slot is a row
        flat = t[dst].double().transpose(1, 2).reshape(-1, case["nkv"], case["hd"]).contiguous()
        flat[slots] = t[src][:slots.numel()].double()
        out[dst] = flat.view(-1, case["block"], case["nkv"], case["hd"]).transpose(1, 2).contiguous()
    return out


def _exact_attn(case, t):
    out = t["o"].double()
    past, new = _lengths(case)
    starts = _prefix(new)
    for b, (p, n) in enumerate(zip(past, new)):
        where = torch.arange(p + n, device="cuda")
        page, offset = t["tables"][b].long()[where // case["block"]], where % case["block"]
        for h in range(case["nkv"]):
            k, v = t["k_cache"][page, h, offset].double(), t["v_cache"][page, h, offset].double()
            for g in range(h * case["rep"], (h + 1) * case["rep"]):
                # rows a block at a time, so that the scores stay small
                for r0 in range(0, n, 1024):
                    r1 = min(n, r0 + 1024)
                    at = torch.arange(p + r0, p + r1, device="cuda")[:, None]
                    seen = where[None, :] <= at
                    if case["window"]:
                        seen &= where[None, :] > at - case["window"]
                    s = t["q"][starts[b] + r0:starts[b] + r1, g].double() @ k.t().contiguous() * case["hd"] ** -0.5
                    w = torch.where(seen, torch.exp(s - torch.where(seen, s, -math.inf).amax(1, keepdim=True)), 0.0)
                    out[starts[b] + r0:starts[b] + r1, g] = w @ v / w.sum(1, keepdim=True)
    return {"o": out}


def _exact_verify(case, t):
    starts, tokens = t["starts"].tolist(), t["tokens"].tolist()
    u, draws = t["u"].double().tolist(), t["draw"].double().tolist()
    out, accepted = [], []
    for b in range(case["b"]):
        r, end, n = starts[b], starts[b + 1], 0
        weight = None
        while r + 1 < end:
            p, x = t["p"][r].double(), tokens[r + 1]
            q = t["q"][r].double() if case["draft"] else torch.zeros_like(p).index_fill_(0, torch.tensor([x], device="cuda"), 1.0)
            if u[r] * q[x].item() < p[x].item():
                out.append(x)
                n, r = n + 1, r + 1
                continue
            weight = (p - q).clamp(min=0)
            if not case["draft"]:
                weight[x] = 0.0
            if weight.sum().item() == 0:
                weight = p
            break
        if weight is None:
            weight = t["p"][r].double()
        line = torch.cumsum(weight, 0)
        over = (line > draws[b] * line[-1]) & (weight > 0)
        i = int(over.int().argmax()) if bool(over.any()) else int(weight.nonzero()[-1])
        out += [i] + [-1] * (end - r - 1)
        accepted.append(n)
    return {"out": _ints(out), "accepted": _ints(accepted)}
