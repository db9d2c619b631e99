"""The attention half of a speculative decode step: rotary positions, attention of a tree of drafted tokens over a paged
cache, verification of the drafted tokens, and the append of the accepted rows.  What is measured, in plain form and
through the framework."""
import math
import random

import torch

own = False

HALF, INTERLEAVED = "half", "interleaved"
_backends = {}


def listed():
    return [
        # one token's fused q|k|v row (5120 + 2 x 1024 columns) of a decode step: latency
        {"name": "rope_token", "op": "rope", "rows": 1, "q_heads": 40, "kv_heads": 8, "dim": 128, "rot": 128, "layout": HALF,
         "src": "f32", "dst": "bf16", "factor": 1.0, "base": 5000},
        # a prefill chunk with an odd length, a quarter of the head rotated, positions far beyond the trained context
        {"name": "rope_chunk", "op": "rope", "rows": 4099, "q_heads": 24, "kv_heads": 4, "dim": 256, "rot": 64, "layout": INTERLEAVED,
         "src": "bf16", "dst": "bf16", "factor": 8.0, "base": 900000},
        # the backward pass of the rotation over a training chunk
        {"name": "rope_back", "op": "rope", "rows": 2047, "q_heads": 40, "kv_heads": 8, "dim": 128, "rot": 128, "layout": HALF,
         "src": "f32", "dst": "f32", "factor": 4.0, "base": 0, "back": True},
        # the accepted rows of a served batch go behind the cached ones
        {"name": "append_accepted", "op": "append", "batch": 32, "rows": 16, "len": 700, "page": 16, "kv_heads": 8, "dim": 128,
         "src": "bf16", "select": True},
        # a prompt's rows, straight from the projections
        {"name": "append_prompt", "op": "append", "batch": 3, "rows": 4001, "len": 130, "page": 64, "kv_heads": 4, "dim": 256,
         "src": "f32", "select": False},
        # one token, short context: latency
        {"name": "attend_token_short", "op": "attention", "batch": 1, "nodes": 1, "len": 333, "ragged": False, "page": 16,
         "q_heads": 40, "kv_heads": 8, "dim": 128, "type": "bf16", "width": 1},
        # a served batch of ordinary decode steps, lengths from half to the whole of 8191
        {"name": "attend_token_batch", "op": "attention", "batch": 32, "nodes": 1, "len": 8191, "ragged": True, "page": 64,
         "q_heads": 40, "kv_heads": 8, "dim": 128, "type": "bf16", "width": 1},
        # one token of one user over a very long context, activations in 32 bits as the projections leave them
        {"name": "attend_token_long", "op": "attention", "batch": 1, "nodes": 1, "len": 120001, "ragged": False, "page": 256,
         "q_heads": 24, "kv_heads": 4, "dim": 256, "type": "f32", "width": 1},
        # small trees of a served batch
        {"name": "attend_tree", "op": "attention", "batch": 8, "nodes": 13, "len": 4000, "ragged": True, "page": 16,
         "q_heads": 40, "kv_heads": 8, "dim": 128, "type": "f32", "width": 3},
        # the largest tree over a long context
        {"name": "attend_tree_wide", "op": "attention", "batch": 4, "nodes": 64, "len": 16384, "ragged": False, "page": 64,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "width": 6},
        # a chain of four drafts for one user over the whole vocabulary
        {"name": "verify_chain", "op": "verify", "batch": 1, "nodes": 5, "vocab": 248320, "type": "f32", "width": 1, "sampled": True,
         "greedy": 0},
        # trees of a served batch, an odd vocabulary, some of the users greedy
        {"name": "verify_trees", "op": "verify", "batch": 16, "nodes": 24, "vocab": 100003, "type": "bf16", "width": 4, "sampled": True,
         "greedy": 3},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention", "attention", "verify", "verify"])
    dim = rng.choice([64, 80, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 3, 4, 5, 8])
    if op == "rope":
        return {"op": op, "rows": _spread(rng, 1, 2500), "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "layout": rng.choice([HALF, INTERLEAVED]), "src": rng.choice(["f32", "bf16"]),
                "dst": rng.choice(["f32", "bf16"]), "factor": rng.choice([1.0, 4.0, 32.0]), "base": _spread(rng, 1, 1000000),
                "back": rng.random() < 0.3}
    if op == "append":
        rows = _spread(rng, 1, 3000)
        return {"op": op, "batch": _spread(rng, 1, max(1, min(64, 4000 // rows))), "rows": rows, "len": _spread(rng, 1, 600),
                "page": rng.choice([5, 16, 24, 64, 256]), "kv_heads": kv_heads, "dim": dim, "src": rng.choice(["f32", "bf16"]),
                "select": rng.random() < 0.5}
    if op == "attention":
        nodes = rng.choice([1, 1, _spread(rng, 2, 64)])
        batch = _spread(rng, 1, 64)
        # no more than the largest listed ones read (about half a gigabyte) and compute
        most = int(min(4e8 / (batch * kv_heads * dim * 4), 5e10 / (batch * nodes * kv_heads * group * dim * 4)))
        return {"op": op, "batch": batch, "nodes": nodes, "len": _spread(rng, 1, max(2, min(100000, most))), "ragged": rng.random() < 0.5,
                "page": rng.choice([5, 16, 24, 64, 256]), "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "type": rng.choice(["f32", "bf16"]), "width": _spread(rng, 1, 8)}
    batch, nodes = _spread(rng, 1, 32), rng.choice([1, _spread(rng, 2, 12), _spread(rng, 2, 64)])
    return {"op": op, "batch": batch, "nodes": nodes, "vocab": min(_spread(rng, 50, 260000), 38000000 // (batch * nodes)),
            "type": rng.choice(["f32", "bf16"]), "width": _spread(rng, 1, 8), "sampled": rng.random() < 0.7, "greedy": rng.choice([0, 0, 2])}


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _lengths(case):
    """Committed tokens of each sequence: all of `len`, or spread evenly from `len` down to half of it."""
    b, n = case["batch"], case["len"]
    return [n - (i * n) // (2 * b) for i in range(b)] if case.get("ragged", True) else [n] * b


def _path_rows(case):
    """Nodes that a verification visits, about: a draft is accepted two times in three."""
    depth = int(2 * (case["nodes"] - 1) / (1 + case["width"]))
    return sum(0.67 ** i for i in range(depth + 1))


def work(case):
    if case["op"] == "rope":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        size = lambda t: 4 if t == "f32" else 2  # noqa: E731
        return {"bytes": case["rows"] * (heads * case["dim"] * (size(case["src"]) + size(case["dst"])) + 4),
                "flops": case["rows"] * (heads - case["kv_heads"]) * case["rot"] * 3}
    if case["op"] == "append":
        rows = case["batch"] * case["rows"] * (0.5 if case["select"] else 1.0)
        return {"bytes": rows * 2 * case["kv_heads"] * case["dim"] * ((4 if case["src"] == "f32" else 2) + 2), "flops": 0}
    if case["op"] == "attention":
        keys = sum(n + case["nodes"] for n in _lengths(case))
        act = case["batch"] * case["nodes"] * case["q_heads"] * case["dim"] * (4 if case["type"] == "f32" else 2)
        return {"bytes": keys * case["kv_heads"] * case["dim"] * 4 + 2 * act, "flops": 4 * keys * case["nodes"] * case["q_heads"] * case["dim"]}
    rows = case["batch"] * _path_rows(case)
    return {"bytes": rows * case["vocab"] * (4 if case["type"] == "f32" else 2) * (2 if case["sampled"] else 1), "flops": rows * case["vocab"] * 4}


def _parents(case, gen, dev):
    """[batch, nodes]: each node hangs on one of the `width` nodes before it; node 0 is the root."""
    b, t = case["batch"], case["nodes"]
    at = torch.arange(t, device=dev)
    back = (torch.rand(b, t, generator=gen, device=dev) * at.clamp(max=case["width"])).long()
    return (at - 1 - back).clamp(min=-1).to(torch.int32)


def _frequencies(case):
    """Radians a position of each pair, in 64 bits: plain, or with the low frequencies stretched by `factor`
    (a ramp over the pairs that turn 32 to 1 times in 4096 positions); and the factor of the rotated values."""
    half, theta, factor = case["rot"] // 2, 1e6, case["factor"]
    f = [theta ** (-i / half) for i in range(half)]
    if factor == 1.0:
        return f, 1.0
    turn = lambda turns: half * math.log(4096 / (turns * 2 * math.pi)) / math.log(theta)  # noqa: E731
    low, high = max(math.floor(turn(32)), 0), min(math.ceil(turn(1)), half - 1)
    keep = [1 - min(max((i - low) / max(high - low, 0.001), 0), 1) for i in range(half)]
    return [v / factor * (1 - k) + v * k for v, k in zip(f, keep)], 0.1 * math.log(factor) + 1


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape, t=torch.float32: torch.randn(*shape, generator=gen, device=dev, dtype=t)  # noqa: E731
    s = {"case": case}
    if case["op"] == "rope":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        s["x"] = normal(case["rows"], heads * case["dim"]).to(_type(case["src"])).view(case["rows"], heads, case["dim"])
        s["positions"] = (case["base"] + torch.arange(case["rows"], device=dev)).to(torch.int32)
        f, s["scale"] = _frequencies(case)
        s["freq"] = torch.tensor(f, dtype=torch.float64, device=dev)
        return s
    if case["op"] == "verify":
        b, t, v = case["batch"], case["nodes"], case["vocab"]
        target = normal(b, t, v).mul_(3)
        draft = target + 0.8 * normal(b, t, v)
        s["parents"] = _parents(case, gen, dev) if case["width"] > 1 else None
        par = s["parents"] if s["parents"] is not None else torch.arange(-1, t - 1, device=dev).expand(b, t)
        s["target"], s["draft"] = target.to(_type(case["type"])), draft.to(_type(case["type"])) if case["sampled"] else None
        s["temperature"] = 0.6 + 0.4 * torch.rand(b, generator=gen, device=dev)
        # each node's token is drawn from the draft's distribution behind its parent
        noise = -torch.log(-torch.log(torch.rand(b, t, v, generator=gen, device=dev).clamp(1e-30, 1 - 1e-7)))
        of_parent = torch.take_along_dim(draft, par.clamp(min=0).long()[..., None], 1)
        s["tokens"] = (of_parent / s["temperature"][:, None, None] + noise).argmax(-1).to(torch.int32)
        s["temperature"][:case["greedy"]] = 0
        s["uniforms"] = torch.rand(b, t, generator=gen, device=dev)
        return s
    b, d, h, page = case["batch"], case["dim"], case["kv_heads"], case["page"]
    lens = _lengths(case)
    rows = case["rows"] if case["op"] == "append" else 0
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    table = -(-(max(lens) + rows + page) // page)
    s["table"] = torch.randperm(b * table, generator=gen, device=dev).to(torch.int32).view(b, table)
    s["k_cache"] = normal(b * table, page, h, d, t=torch.bfloat16)
    s["v_cache"] = normal(b * table, page, h, d, t=torch.bfloat16)
    if case["op"] == "append":
        fused = normal(b, rows, 2 * h, d).to(_type(case["src"]))            # k|v of one projection
        s["k"], s["v"] = fused[:, :, :h], fused[:, :, h:]
        s["counts"] = s["index"] = None
        if case["select"]:
            s["counts"] = torch.randint(0, rows + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
            s["index"] = torch.rand(b, rows, generator=gen, device=dev).argsort(-1).to(torch.int32)
            live = torch.arange(rows, device=dev) < s["counts"][:, None]    # the accepted ones in rising order, -1 behind them
            s["index"] = torch.where(live, s["index"], rows).sort(-1).values.to(torch.int32)
            s["index"] = torch.where(live, s["index"], -1).to(torch.int32)
        return s
    t = case["nodes"]
    s["q"] = (2 * normal(b, t, case["q_heads"], d)).to(_type(case["type"]))
    s["k"], s["v"] = normal(b, t, h, d, t=torch.bfloat16), normal(b, t, h, d, t=torch.bfloat16)
    s["parents"] = _parents(case, gen, dev) if case["width"] > 1 and t > 1 else None
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------


def _pairs(x, rot, layout):
    """The two halves of every rotated pair, as views of x."""
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if layout == INTERLEAVED else (x[..., :rot // 2], x[..., rot // 2:rot])


def _plain_rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["freq"]
    sign = -s["scale"] if c.get("back") else s["scale"]
    cos, sin = (angle.cos() * s["scale"]).float()[:, None], (angle.sin() * sign).float()[:, None]
    q, k, v = s["x"].float().split([c["q_heads"], c["kv_heads"], c["kv_heads"]], 1)

    def turned(x):
        x1, x2 = _pairs(x, c["rot"], c["layout"])
        y = x.clone()
        y1, y2 = _pairs(y, c["rot"], c["layout"])
        y1.copy_(x1 * cos - x2 * sin)
        y2.copy_(x1 * sin + x2 * cos)
        return y.to(_type(c["dst"]))

    return turned(q), turned(k), v.to(_type(c["dst"]))


def _plain_append(s):
    b, rows = s["k"].shape[:2]
    dev, page = s["k"].device, s["case"]["page"]
    at = torch.arange(rows, device=dev)
    slot = s["lens"].long()[:, None] + at
    where = torch.gather(s["table"].long(), 1, slot // page) * page + slot % page
    counts = s["counts"] if s["counts"] is not None else torch.full((b,), rows, dtype=torch.int32, device=dev)
    live = at < counts[:, None]
    source = s["index"].long().clamp(min=0) if s["index"] is not None else at.expand(b, rows)
    seq = torch.arange(b, device=dev)[:, None].expand(b, rows)
    for cache, x in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        cache.view(-1, *cache.shape[2:])[where[live]] = x[seq[live], source[live]].to(torch.bfloat16)
    return s["k_cache"], s["v_cache"], s["lens"] + counts


def _plain_attention(s):
    c, q = s["case"], s["q"]
    b, t, heads, d = q.shape
    h = c["kv_heads"]
    dev = q.device
    slots = (s["table"].long()[:, :, None] * c["page"] + torch.arange(c["page"], device=dev)).view(b, -1)

    def keys(cache, rows):                                                   # [b, h, slots + t, d], zero behind the length
        x = torch.cat([cache.view(-1, h, d)[slots], rows], 1).float()
        return x.permute(0, 2, 1, 3)

    parents = s["parents"] if s["parents"] is not None else torch.arange(-1, t - 1, device=dev).expand(b, t)
    step = (torch.arange(t, device=dev) == parents[..., None]).float() + torch.eye(t, device=dev)
    tree = torch.linalg.matrix_power(step, t) > 0                            # [b, t, t]: itself and its ancestors
    seen = (torch.arange(slots.shape[1], device=dev) < s["lens"][:, None])[:, None].expand(b, t, -1)
    seen = torch.cat([seen, tree], 2)[:, None, :, None]                      # [b, 1, t, 1, keys]
    x = q.float().view(b, t, h, heads // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    score = (x @ keys(s["k_cache"], s["k"]).transpose(2, 3)).mul_(d ** -0.5).view(b, h, t, heads // h, -1)
    score = score.masked_fill_(~seen, -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True))
    total = score.sum(-1).view(b, h, -1, 1)
    out = score.view(b, h, t * (heads // h), -1) @ keys(s["v_cache"], s["v"]) / total
    return out.view(b, h, t, heads // h, d).permute(0, 2, 1, 3, 4).reshape(b, t, heads, d).to(q.dtype)


def _first(mask):
    """The lowest index where the last axis of `mask` is true."""
    n = mask.shape[-1]
    return torch.where(mask, torch.arange(n, device=mask.device), n).amin(-1)


def _plain_verify(s):
    c = s["case"]
    b, t, v = s["target"].shape
    dev = s["target"].device
    rows = torch.arange(b, device=dev)
    parents = s["parents"] if s["parents"] is not None else torch.arange(-1, t - 1, device=dev).expand(b, t)
    greedy = s["temperature"] == 0
    tau = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]

    def dist(logits, cur):                                                   # in 64 bits: decisions lie next to borders
        x = logits[rows, cur].double()
        x = (x - x.amax(-1, keepdim=True)) / tau
        x = x.exp()
        return x / x.sum(-1, keepdim=True)

    def state(cur):
        p = dist(s["target"], cur)
        raw = s["target"][rows, cur]
        return p, dist(s["draft"], cur) if c["sampled"] else torch.zeros_like(p), _first(raw == raw.amax(-1, keepdim=True))

    cur = torch.zeros(b, dtype=torch.long, device=dev)
    p, q, best = state(cur)
    a, z = torch.zeros(b, dtype=torch.float64, device=dev), torch.ones(b, dtype=torch.float64, device=dev)
    gone = torch.zeros(b, v, dtype=torch.bool, device=dev)                   # certain drafts: refused tokens of this node
    path = torch.full((b, t), -1, dtype=torch.int32, device=dev)
    path[:, 0], count = 0, torch.ones(b, dtype=torch.int32, device=dev)
    for child in range(1, t):                                                # each decision needs the ones before it
        tried = parents[:, child] == cur
        token = s["tokens"][:, child].long()
        u = s["uniforms"][:, child].double()
        pt, qt = p[rows, token], q[rows, token]
        if c["sampled"]:
            ok = u * qt * z < (pt - a * qt).clamp(min=0)
        else:
            ok = (u * z < pt) & ~gone[rows, token]
        ok = torch.where(greedy, token == best, ok)
        yes, no = tried & ok, tried & ~ok
        path[rows, count.long().clamp(max=t - 1)] = torch.where(yes, child, path[rows, count.long().clamp(max=t - 1)])
        count, cur = count + yes, torch.where(yes, child, cur)
        if c["sampled"]:
            a = torch.where(no, a + z, a)
            z = torch.where(no, (p - a[:, None] * q).clamp(min=0).sum(-1), z)
        else:
            z = torch.where(no & ~gone[rows, token], z - pt, z)
            gone[rows, token] |= no
        p, q, best = state(cur)
        a, z = torch.where(yes, 0.0, a), torch.where(yes, 1.0, z)
        gone &= ~yes[:, None]
    w = (p - a[:, None] * q).clamp(min=0).masked_fill(gone, 0)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p)
    total = w.cumsum(-1)
    border = s["uniforms"][:, 0].double() * total[:, -1]
    last = v - 1 - _first((w > 0).flip(-1))
    token = torch.where(greedy, best, torch.minimum(_first(total > border[:, None]), last))
    return path, count, token.to(torch.int32)


# ---- the framework's calls ---------------------------------------------------------------------------------------


def _backend(device):
    if device not in _backends:
        from lattice_b200 import CudaQ4Backend
        _backends[device] = CudaQ4Backend(device)
    return _backends[device]


def _own(s):
    from lattice_b200 import KvCache, RopeTable
    c = s["case"]
    if c["op"] == "rope":
        be = _backend(s["x"].device.index)
        q, k, v = s["x"].split([c["q_heads"], c["kv_heads"], c["kv_heads"]], 1)
        table = RopeTable(s["freq"], c["layout"], s["scale"])
        turn = -1 if c.get("back") else 1
        return tuple(be.rope_rows([(q, turn), (k, turn), (v, 0)], s["positions"], table, out_dtype=_type(c["dst"])))
    if c["op"] == "verify":
        be = _backend(s["target"].device.index)
        return be.verify_draft(s["target"], s["tokens"], s["uniforms"], draft_logits=s["draft"], parents=s["parents"],
                               temperature=s["temperature"])
    be = _backend(s["k"].device.index)
    cache = KvCache(s["k_cache"], s["v_cache"], s["table"])
    if c["op"] == "append":
        lens = be.kv_append(cache, s["k"], s["v"], s["lens"], counts=s["counts"], index=s["index"])
        return s["k_cache"], s["v_cache"], lens
    return be.tree_attention(s["q"], s["k"], s["v"], cache, s["lens"], parents=s["parents"])


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}[state["case"]["op"]](state)


# ---- in 64 bits, by the definitions ------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "verify":
        return None                                                          # whole numbers only
    s = prepare(case, seed)
    if case["op"] == "rope":
        # a pair is a complex number, its position a turn
        turn = torch.polar(torch.full_like(s["freq"], s["scale"]).expand(case["rows"], -1).contiguous(),
                           s["positions"].double()[:, None] * s["freq"])
        turn = turn.conj() if case.get("back") else turn
        x = s["x"].double()
        r = case["rot"]
        z = x[..., :r].unflatten(-1, (r // 2, 2)) if case["layout"] == INTERLEAVED else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn[:, None])
        z = z if case["layout"] == INTERLEAVED else z.transpose(-1, -2)
        y = torch.cat([z.flatten(-2), x[..., r:]], -1)
        n, m = case["q_heads"], case["kv_heads"]
        return y[:, :n], y[:, n:n + m], x[:, n + m:]
    lens, table, page = s["lens"].tolist(), s["table"].tolist(), case["page"]
    if case["op"] == "append":
        out = [s["k_cache"].double(), s["v_cache"].double()]
        b, rows = s["k"].shape[:2]
        counts = s["counts"].tolist() if s["counts"] is not None else [rows] * b
        for i in range(b):
            source = s["index"][i, :counts[i]].long() if s["index"] is not None else torch.arange(rows, device=s["k"].device)
            to = [table[i][j // page] * page + j % page for j in range(lens[i], lens[i] + counts[i])]
            for x, rows_of in zip(out, (s["k"], s["v"])):
                x.view(-1, *x.shape[2:])[torch.tensor(to, dtype=torch.long, device=x.device)] = rows_of[i, source].double()
        return out[0], out[1], None
    t, heads, h = case["nodes"], case["q_heads"], case["kv_heads"]
    parents = s["parents"].tolist() if s["parents"] is not None else [list(range(-1, t - 1))] * case["batch"]
    outs = []
    for i in range(case["batch"]):
        pages = s["table"][i].long()
        k = torch.cat([s["k_cache"][pages].flatten(0, 1)[:lens[i]], s["k"][i]]).double()
        v = torch.cat([s["v_cache"][pages].flatten(0, 1)[:lens[i]], s["v"][i]]).double()
        mask = torch.zeros(t, lens[i] + t, dtype=torch.bool)
        mask[:, :lens[i]] = True
        for j in range(t):
            at = j
            while at >= 0:
                mask[j, lens[i] + at] = True
                at = parents[i][at]
        mask = mask.to(k.device)
        per_head = []
        for g in range(h):
            x = s["q"][i, :, g * (heads // h):(g + 1) * (heads // h)].double()
            w = torch.einsum("tgd,nd->tgn", x, k[:, g]) / math.sqrt(case["dim"])
            w = torch.softmax(w.masked_fill(~mask[:, None], -math.inf), -1)
            per_head.append(torch.einsum("tgn,nd->tgd", w, v[:, g]))
        outs.append(torch.cat(per_head, 1))
    return torch.stack(outs)
