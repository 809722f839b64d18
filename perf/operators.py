"""Performance cases of the paged-cache operators: rotary positions, what writes the cache, reads it and cuts it.

A case is one call as a serving program makes it between its layers' matrix products. Its sizes:

  op        "rope": rotation of a step's queries and keys; "append": a step's keys (rotated) and values into their pages;
            "attend": attention of a step's rows over the pages; "weigh": the attention each cached position gets, added
            up; "evict": the cache cut back to a budget of positions
  heads, kv_heads, dim   attention heads, cached heads, their width
  type      the values' type (the cache's, and the rows' unless "rows_type" says otherwise)
  seqs      sequences of the step
  rows      new token rows per sequence (the most of one)
  length    positions cached before them (the most of one)
  page      positions per page
  ragged    whether the sequences differ in rows and length
  layout, n_rot, scaling   the rotation
  budget, first, recent    what a cut keeps: positions in all, of the start, of the end (0 where the case cuts nothing)
"""
from __future__ import annotations

import math

import torch

from jetsonfabric_amd.configs import CONFIGS

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BASE, FACTOR, CONTEXT = 1.0e6, 4.0, 32768  # rotation base; context extension by 4 over the trained 32768 positions
BETA_FAST, BETA_SLOW = 32.0, 1.0


def _heads(name):
    m = CONFIGS[name].model
    return {"heads": m.n_head, "kv_heads": m.n_head_kv, "dim": m.head_dim}


H_1_5B, H_7B = _heads("qwen2.5-1.5b-q4k"), _heads("qwen2.5-7b-q4k")
H_14B, H_32B = _heads("qwen2.5-14b-q4k"), _heads("qwen2.5-32b-q2k")


def _case(op, heads, seqs, rows, length, **more):
    c = {"op": op, **heads, "type": "f16", "rows_type": "", "seqs": seqs, "rows": rows, "length": length, "page": 16,
         "ragged": False, "layout": "half", "n_rot": heads["dim"], "scaling": "yarn", "budget": 0, "first": 0, "recent": 0}
    c.update(more)
    c["rows_type"] = c["rows_type"] or c["type"]
    return c


def listed():
    cases = {
        # the next token of two requests far beyond the trained context
        "rope-decode-7b-x2": _case("rope", H_7B, 2, 1, 100000, page=1),
        # a whole prompt's queries and keys
        "rope-prompt-14b": _case("rope", H_14B, 1, 4096, 0, type="bf16", page=1),
        # two requests' drafts of 8, rows as the products leave them
        "append-verify-14b-x2": _case("append", H_14B, 2, 9, 4096, rows_type="f32"),
        # prompts of several requests, different lengths, in one chunk
        "append-prompt-7b-x3": _case("append", H_7B, 3, 2048, 2048, type="bf16", page=64, ragged=True),
        # one short request's next token: launches and latency
        "attend-decode-1.5b": _case("attend", H_1_5B, 1, 1, 256),
        # eight requests at long, different contexts
        "attend-decode-32b-x8": _case("attend", H_32B, 8, 1, 32700, type="bf16", page=64, ragged=True),
        # two requests' drafts of 8
        "attend-verify-14b-x2": _case("attend", H_14B, 2, 9, 4096),
        # a chunk of a long prompt behind its cached part
        "attend-chunk-7b": _case("attend", H_7B, 1, 2048, 6144, page=32),
        # after each step of eight requests
        "weigh-decode-32b-x8": _case("weigh", H_32B, 8, 1, 2176, page=64),
        # once after a prompt's last chunk
        "weigh-prompt-7b": _case("weigh", H_7B, 1, 1777, 2222, type="bf16", page=32),
        # eight requests whose caches are full: a new token each, and one position goes
        "evict-step-7b-x8": _case("evict", H_7B, 8, 1, 4096, budget=4096, first=4, recent=256),
        # two long prompts cut once, before their answers begin
        "evict-prompt-14b-x2": _case("evict", H_14B, 2, 0, 16384, type="bf16", page=64, budget=2048, first=4, recent=512),
    }
    return [{"name": name, **c} for name, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = listed()
    most = {k: max(work(c)[k] for c in most) for k in ("bytes", "flops")}
    while True:
        heads = rng.choice([H_1_5B, H_7B, H_14B, H_32B, {"heads": 8, "kv_heads": 2, "dim": 64},
                            {"heads": 6, "kv_heads": 6, "dim": 96}, {"heads": 4, "kv_heads": 1, "dim": 256}])
        op = rng.choice(["rope", "append", "attend", "attend", "weigh", "evict"])
        c = _case(op, heads, rng.choice([1, 1, 2, 3, 5, 8]), 1, _log(rng, 20, 32768), type=rng.choice(["f16", "bf16"]),
                  page=rng.choice([1, 8, 16, 16, 32, 64, 256]), ragged=rng.random() < 0.5,
                  layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                  n_rot=heads["dim"] // rng.choice([1, 1, 2]))
        c["rows"] = rng.choice([1, rng.randint(2, 9), _log(rng, 10, 2048)])
        if op in ("rope", "append"):
            c["rows_type"] = rng.choice(["f32", c["type"]])
        if op == "rope":
            c["type"] = c["rows_type"]
        if op == "evict":
            c["rows"] = rng.choice([0, 1, rng.randint(2, 9)])
            c["first"], c["recent"] = rng.choice([0, 4]), rng.randint(1, max(1, c["length"] // 8))
            c["budget"] = c["length"] if c["rows"] else max(c["first"] + c["recent"] + 1, _log(rng, 1 + c["length"] // 16, c["length"]))
        w = work(c)
        pairs = c["seqs"] * c["heads"] * c["rows"] * (c["length"] + c["rows"])
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and (op not in ("attend", "weigh") or pairs < 6e8):
            return c


# ---------------------------------------------------------------- inputs

def _counts(case):
    """Rows and slots in use (the new rows included) of each sequence."""
    rows, lens = [], []
    for s in range(case["seqs"]):
        part = (case["seqs"] - s) / case["seqs"] if case["ragged"] else 1.0
        r = max(min(case["rows"], 1), int(case["rows"] * part))
        rows.append(r)
        lens.append(max(1, int(case["length"] * part)) + r)
    return rows, lens


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows, lens = _counts(case)
    total, most = sum(rows), max(lens)
    t, rt = TYPES[case["type"]], TYPES[case["rows_type"]]

    def normal(*size, std=1.0):
        return torch.randn(*size, generator=g, device="cuda") * std

    x = {"starts": _ints([sum(rows[:s]) for s in range(len(rows) + 1)]), "lengths": _ints(lens),
         "positions": torch.cat([torch.arange(n - r, n, dtype=torch.int32, device="cuda") for r, n in zip(rows, lens)])}
    if case["op"] in ("rope", "append"):
        # the rows of a fused product: queries, keys, values side by side
        x["qkv"] = normal(total, heads + 2 * kv, dim, std=1.5).to(rt)
    if case["op"] == "rope":
        x["out"] = torch.zeros(total, heads + kv, dim, dtype=t, device="cuda")
        return x
    pages = -(-most // page)
    count = len(rows) * pages + 3
    x["table"] = torch.randperm(count, generator=g, device="cuda")[:len(rows) * pages].to(torch.int32).reshape(len(rows), pages)
    x["k"] = normal(count, kv, page, dim, std=1.2).to(t)
    x["v"] = normal(count, kv, page, dim).to(t)
    if case["op"] in ("attend", "weigh"):
        x["q"] = normal(total, heads, dim, std=1.5).to(t)
    if case["op"] == "attend":
        x["out"] = torch.zeros(total, heads, dim, dtype=t, device="cuda")
        return x
    # attention gathers on few positions: weights over several powers of ten
    x["weights"] = torch.exp(normal(count, kv, page, std=2.0)) * 0.1
    if case["op"] == "weigh":
        size = torch.logsumexp(normal(total, heads, 64) * 2, -1)  # of the order of what attention of these rows gives
        x["lse"] = size + math.log(most / 64.0)
        return x
    x["slots"] = torch.zeros(count, kv, page, dtype=torch.int32, device="cuda")
    at = torch.arange(pages * page, dtype=torch.int32, device="cuda").reshape(pages, 1, page).expand(pages, kv, page)
    for s in range(len(rows)):
        x["slots"][x["table"][s].long()] = at
    if case["op"] == "evict":
        x["lengths"] -= _ints(rows)
        if case["rows"]:
            x["new"] = normal(total, 2 * kv, dim, std=1.2).to(t)
            x["step"] = _ints(rows)
            x["positions"] -= x["step"].repeat_interleave(x["step"].long())
        else:
            x["saved"] = [x[n].clone() for n in ("lengths", "weights", "slots")]
    return x


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["op"] == "evict" and case["rows"]:
        state["advance"] = state["step"].repeat_interleave(state["step"].long())
    rows, lens = _counts(case)
    state["max_rows"], state["max_length"] = max(rows), max(lens)
    return state


# ---------------------------------------------------------------- plain forms

def _scale(case):
    return case["dim"] ** -0.5


def _frequencies(case, device):
    """Angle per position of each pair, and the size of the rotated values, in 64 bits."""
    n, s = case["n_rot"], FACTOR
    i = torch.arange(n // 2, dtype=torch.float64, device=device)
    if case["scaling"] == "ntk":
        return (BASE * s ** (n / (n - 2))) ** (-2 * i / n), 1.0
    f = BASE ** (-2 * i / n)
    if case["scaling"] == "none":
        return f, 1.0
    if case["scaling"] == "linear":
        return f / s, 1.0

    def pair(turns):  # the pair that turns so often over the trained context
        return n * math.log(CONTEXT / (turns * 2 * math.pi)) / (2 * math.log(BASE))

    lo, hi = max(math.floor(pair(BETA_FAST)), 0), min(math.ceil(pair(BETA_SLOW)), n - 1)
    far = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f * (1 - far) + f / s * far, 0.1 * math.log(s) + 1


def _rotated(case, x, positions):
    """x [rows, heads, dim], rotated, in 32 bits."""
    f, size = _frequencies(case, x.device)
    angle = positions.double()[:, None] * f
    cos, sin = (angle.cos() * size).float()[:, None], (angle.sin() * size).float()[:, None]
    x, n = x.float(), case["n_rot"]
    if case["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([y, x[..., n:]], -1)


def _where(state, rows):
    """Sequence of each row, its number within it, and its slot."""
    starts = state["starts"].long()
    r = torch.arange(rows, device=starts.device)
    seq = torch.searchsorted(starts, r, right=True) - 1
    local = r - starts[seq]
    return seq, local, state["lengths"].long()[seq] - (starts[seq + 1] - starts[seq]) + local


def _append(state, k, v, rotate):
    case = state["case"]
    seq, _, slot = _where(state, len(k))
    page, at = state["table"].long()[seq, slot // case["page"]], slot % case["page"]
    kr = _rotated(case, k, state["positions"]) if rotate else k.float()
    state["k"][page, :, at] = kr.to(state["k"].dtype)
    state["v"][page, :, at] = v.to(state["v"].dtype)
    state["weights"][page, :, at] = 0.0
    state["slots"][page, :, at] = state["positions"][:, None].expand(-1, case["kv_heads"])


def _pages(state, x):
    """The sequences' pages behind one another: [seqs, kv heads, slots, ...]."""
    y = x[state["table"].long()].transpose(1, 2)
    return y.reshape(*y.shape[:2], -1, *y.shape[4:])


def _scores(state):
    """Scores of the rows by sequence, [seqs, kv heads, rows, heads of one, slots], what each row sees, and where a row is."""
    case, q = state["case"], state["q"]
    kv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    most = state["max_rows"]
    starts, lens = state["starts"].long(), state["lengths"].long()
    r = torch.arange(most, device=q.device)
    row = (starts[:-1, None] + r).clamp(max=len(q) - 1)
    x = q[row].float().reshape(len(lens), most, kv, group, -1).permute(0, 2, 1, 3, 4)
    keys = _pages(state, state["k"]).float()
    s = (x.reshape(len(lens), kv, most * group, -1) @ keys.transpose(-1, -2)) * _scale(case)
    s = s.reshape(len(lens), kv, most, group, -1)
    end = (lens - starts.diff())[:, None] + r + 1
    sees = (torch.arange(s.shape[-1], device=q.device) < end[..., None]) & (r < starts.diff()[:, None])[..., None]
    return s, sees[:, None, :, None], _where(state, len(q))[:2]


def _attend(state):
    case = state["case"]
    s, sees, (seq, local) = _scores(state)
    s = s.masked_fill_(~sees, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    values = _pages(state, state["v"]).float()
    o = (p.reshape(*p.shape[:2], -1, p.shape[-1]) @ values).reshape(*p.shape[:-1], -1) / total
    lse = (top + total.log()).squeeze(-1)
    o, lse = o.transpose(1, 2)[seq, local], lse.transpose(1, 2)[seq, local]
    state["out"].copy_(o.reshape(state["out"].shape))
    return [state["out"], lse.reshape(len(seq), case["heads"])]


def _weigh(state):
    case = state["case"]
    s, sees, _ = _scores(state)
    kv, group, most = case["kv_heads"], case["heads"] // case["kv_heads"], state["max_rows"]
    row = (state["starts"].long()[:-1, None] + torch.arange(most, device=s.device)).clamp(max=len(state["q"]) - 1)
    lse = state["lse"][row].reshape(len(row), most, kv, group).permute(0, 2, 1, 3).unsqueeze(-1)
    got = s.sub_(lse).exp_().masked_fill_(~sees, 0.0).sum((2, 3))  # [seqs, kv heads, slots]
    got = got.reshape(*got.shape[:2], -1, case["page"]).transpose(1, 2)
    state["weights"][state["table"].long()] += got
    return [state["weights"]]


def _evict(state):
    case, budget, page = state["case"], state["case"]["budget"], state["case"]["page"]
    w, pos, lens = _pages(state, state["weights"]), _pages(state, state["slots"]), state["lengths"].long()
    slot = torch.arange(w.shape[-1], device=w.device)
    used = (slot < lens[:, None])[:, None].expand_as(w)
    newest = pos.masked_fill(~used, -1).amax(-1, keepdim=True)
    kind = torch.where((pos < case["first"]) | (pos > newest - case["recent"]), 2, 1).masked_fill(~used, 0)
    order = w.argsort(dim=-1, descending=True, stable=True)  # by kind, then weight, then slot
    order = order.gather(-1, kind.gather(-1, order).argsort(dim=-1, descending=True, stable=True))
    kept = torch.zeros_like(used).scatter(-1, order[..., :budget], True) & used
    inside = slot < budget
    hole, mover = ~kept & inside & (lens > budget)[:, None, None], kept & ~inside
    movers = (~mover).to(torch.int8).argsort(dim=-1, stable=True)[..., :budget]  # moving slots first, ascending
    rank = hole[..., :budget].cumsum(-1) - 1
    source = torch.where(hole[..., :budget], movers.gather(-1, rank.clamp(min=0)), slot[:budget])
    table, h = state["table"].long()[:, None], torch.arange(case["kv_heads"], device=w.device)[None, :, None]
    to = (table.expand(-1, len(h[0]), -1)[..., slot[:budget] // page], h, (slot[:budget] % page).expand_as(source))
    at = (table.expand(-1, len(h[0]), -1).gather(-1, source // page), h, source % page)
    for name in ("k", "v", "weights", "slots"):
        state[name][to] = state[name][at]
    state["lengths"].clamp_(max=budget)
    return [state["k"], state["v"], state["weights"], state["slots"], state["lengths"]]


# ---------------------------------------------------------------- a pass

def _handles(state):
    """What a program makes once for its cache and its step's shape."""
    import jetsonfabric_amd as jf

    case = state["case"]
    if "rope" not in state:
        state["rope"] = jf.Rope(case["n_rot"], base=BASE, layout=case["layout"], scaling=case["scaling"], factor=FACTOR,
                                original_context=CONTEXT, beta_fast=BETA_FAST, beta_slow=BETA_SLOW)
        if "k" in state:
            state["cache"] = jf.PagedCache(state["k"], state["v"], state.get("weights"), state.get("slots"))
            state["batch"] = jf.PagedBatch(state["table"], state["lengths"], state["starts"], state["max_rows"],
                                           state["max_length"])
    return state["rope"], state.get("cache"), state.get("batch")


def run(state):
    case = state["case"]
    op, heads, kv = case["op"], case["heads"], case["kv_heads"]
    rope, cache, batch = _handles(state) if own else (None, None, None)
    if op == "rope":
        x = state["qkv"][:, :heads + kv]
        if own:
            return [rope.rotate(x, state["positions"], out=state["out"])]
        return [state["out"].copy_(_rotated(case, x, state["positions"]))]
    if op == "append":
        k, v = state["qkv"][:, heads:heads + kv], state["qkv"][:, heads + kv:]
        if own:
            cache.append(batch, k, v, state["positions"], rope)
        else:
            _append(state, k, v, True)
        return [state["k"], state["v"], state["weights"], state["slots"]]
    if op == "attend":
        return list(cache.attend(batch, state["q"], _scale(case), out=state["out"])) if own else _attend(state)
    if op == "weigh":
        if not own:
            return _weigh(state)
        cache.weigh(batch, state["q"], state["lse"], _scale(case))
        return [state["weights"]]
    if case["rows"]:  # the step of a full cache: a row more per sequence, and as many positions less
        state["lengths"].add_(state["step"])
        state["positions"].add_(state["advance"])
        k, v = state["new"][:, :kv], state["new"][:, kv:]
        if own:
            cache.append(batch, k, v, state["positions"], rope)
        else:
            _append(state, k, v, True)
    else:  # every pass cuts the same full cache: what the last one cut is taken back
        for name, saved in zip(("lengths", "weights", "slots"), state["saved"]):
            state[name].copy_(saved)
    if not own:
        return _evict(state)
    cache.evict(batch, case["budget"], case["first"], case["recent"])
    return [state["k"], state["v"], state["weights"], state["slots"], state["lengths"]]


def work(case):
    rows, lens = _counts(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    b, rb = size[case["type"]], size[case["rows_type"]]
    n = sum(rows)
    seen = sum(sum(range(t - r + 1, t + 1)) for r, t in zip(rows, lens))  # (row, slot) pairs
    if case["op"] == "rope":
        return {"bytes": n * ((heads + kv) * dim * (rb + b) + 4), "flops": 3.0 * n * (heads + kv) * case["n_rot"]}
    write = n * (2 * kv * dim * (rb + b) + 8 * kv + 4)
    if case["op"] == "append":
        return {"bytes": write, "flops": 3.0 * n * kv * case["n_rot"]}
    if case["op"] == "attend":
        return {"bytes": n * heads * (2 * dim * b + 4) + sum(lens) * kv * 2 * dim * b, "flops": 4.0 * dim * heads * seen}
    if case["op"] == "weigh":
        return {"bytes": n * heads * (dim * b + 4) + sum(lens) * kv * (dim * b + 8), "flops": 2.0 * dim * heads * seen}
    # weights and positions of every slot; what moves is read and written
    byte = write if case["rows"] else 0
    for r, t in zip(rows, lens):
        over = max(0, t - case["budget"])
        if over:
            held = min(case["budget"], case["first"] + case["recent"])
            moved = min(over, case["recent"] + (case["budget"] - held) * max(0, over - case["recent"]) / max(1, t - held))
            byte += kv * (8 * t + moved * 2 * (2 * dim * b + 8))
    return {"bytes": max(byte, 8 * kv * sum(lens)), "flops": 0.0}


# ---------------------------------------------------------------- in 64 bits

def _turn(case, x, positions):
    """The rotation as a product of complex numbers."""
    n = case["n_rot"]
    d = torch.arange(0, n, 2, dtype=torch.float64, device=x.device)
    base = BASE * FACTOR ** (n / (n - 2)) if case["scaling"] == "ntk" else BASE
    step, size = torch.exp(-d / n * math.log(base)), 1.0
    if case["scaling"] == "linear":
        step = step / FACTOR
    if case["scaling"] == "yarn":
        edge = [n / 2 * math.log(CONTEXT / (2 * math.pi * t)) / math.log(BASE) for t in (BETA_FAST, BETA_SLOW)]
        lo, hi = max(0, math.floor(edge[0])), min(n - 1, math.ceil(edge[1]))
        keep = 1 - torch.clamp((d / 2 - lo) / (hi - lo if hi > lo else 1e-3), 0, 1)
        step, size = step * (keep + (1 - keep) / FACTOR), 1 + math.log(FACTOR) / 10
    turn = torch.polar(torch.full((len(x), n // 2), size, dtype=torch.float64, device=x.device),
                       positions.double()[:, None] * step[None])[:, None]
    y = x.double().clone()
    if case["layout"] == "half":
        z = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * turn
        y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
    else:
        z = torch.view_as_complex(y[..., :n].reshape(*y.shape[:2], n // 2, 2).contiguous()) * turn
        y[..., :n] = torch.view_as_real(z).flatten(-2)
    return y


def exact(case, seed):
    x = _inputs(case, seed)
    heads, kv, page = case["heads"], case["kv_heads"], case["page"]
    group = heads // kv
    if case["op"] == "rope":
        return [_turn(case, x["qkv"][:, :heads + kv], x["positions"])]
    starts, lens, table = x["starts"].tolist(), x["lengths"].tolist(), x["table"].long()
    k, v = x["k"].double(), x["v"].double()

    def flat(s):  # page and place of every slot of a sequence
        slot = torch.arange(table.shape[1] * page, device=table.device)
        return table[s][slot // page], slot % page

    def write(kn, vn, positions):
        kn = _turn(case, kn, positions)
        for s in range(len(lens)):
            r0, r1 = starts[s], starts[s + 1]
            p, i = (u[lens[s] - (r1 - r0):lens[s]] for u in flat(s))
            k[p, :, i], v[p, :, i] = kn[r0:r1], vn[r0:r1].double()
            x["weights"][p, :, i] = 0.0
            x["slots"][p, :, i] = positions[r0:r1, None].expand(-1, kv)

    if case["op"] == "append":
        write(x["qkv"][:, heads:heads + kv], x["qkv"][:, heads + kv:], x["positions"])
        return [k, v, x["weights"], x["slots"]]
    if case["op"] in ("attend", "weigh"):
        q = x["q"].double()
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
        weights = x["weights"].double() if case["op"] == "weigh" else None
        for s in range(len(lens)):
            r0, r1, n = starts[s], starts[s + 1], lens[s]
            p, i = (u[:n] for u in flat(s))
            sees = torch.arange(n, device=q.device) <= torch.arange(n - (r1 - r0), n, device=q.device)[:, None]
            for h in range(heads):
                a = (q[r0:r1, h] @ k[p, h // group, i].T) / math.sqrt(case["dim"])
                if case["op"] == "weigh":
                    got = torch.exp(a - x["lse"][r0:r1, h].double()[:, None])
                    weights[p, h // group, i] += torch.where(sees, got, 0.0).sum(0)
                    continue
                a.masked_fill_(~sees, -math.inf)
                lse[r0:r1, h] = torch.logsumexp(a, -1)
                out[r0:r1, h] = torch.softmax(a, -1) @ v[p, h // group, i]
        return [weights] if case["op"] == "weigh" else [out, lse]
    if case["rows"]:
        lens = (x["lengths"] + x["step"]).tolist()
        write(x["new"][:, :kv], x["new"][:, kv:], x["positions"] + x["step"].repeat_interleave(x["step"].long()))
    budget = case["budget"]
    for s in range(len(lens)):
        n = lens[s]
        if n <= budget:
            continue
        p, i = (u[:n] for u in flat(s))
        for h in range(kv):
            w, pos = x["weights"][p, h, i], x["slots"][p, h, i]
            safe = (pos < case["first"]) | (pos > pos.max() - case["recent"])
            # protected first, then the heavier, then the lower slot
            rank = torch.argsort(torch.where(safe, 0, 1) * 4.0e9 + torch.argsort(torch.argsort(-w.double(), stable=True)).double(), stable=True)
            keep = torch.zeros(n, dtype=torch.bool, device=w.device)
            keep[rank[:budget]] = True
            to, at = torch.nonzero(~keep[:budget])[:, 0], budget + torch.nonzero(keep[budget:])[:, 0]
            for u in (k, v, x["weights"], x["slots"]):
                u[p[to], h, i[to]] = u[p[at], h, i[at]]
        lens[s] = budget
    return [k, v, x["weights"], x["slots"], _ints(lens)]
