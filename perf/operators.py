"""Timed cases of the latent-cache attention operators: rotary positions, the cache append, attention of drafted
token trees, accumulated attention weight, and eviction by it.

`run` makes the framework's calls where `own` is true (loki_b200.attention) and computes the same formulas with
elementary torch operations in 32 bits where it is false.  One cached row is 576 values: a 512-wide latent, which
is both key and value, and 64 rotated key values.  The query of one (token, head) row has the same 576 values.
"""
import math

import torch

own = False

LATENT, ROPE, ROW = 512, 64, 576
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
YARN = dict(base=10000.0, factor=40.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0)


def listed():
    return [
        # the query heads of one 8-row decode pass, whole heads of 192 of which the last 64 rotate
        {"name": "rope decode 8 rows", "op": "rope", "tokens": 8, "heads": 128, "head_dim": 192, "rot_offset": 128, "rot_dim": 64,
         "layout": "interleaved", "grad": False, "dtype": "bf16", "max_pos": 40960, "scaled": True},
        # the gradient of the same rotation over a long training or tuning chunk, in the other layout
        {"name": "rope gradient 4096 rows", "op": "rope", "tokens": 4096, "heads": 128, "head_dim": 192, "rot_offset": 128, "rot_dim": 64,
         "layout": "half", "grad": True, "dtype": "f32", "max_pos": 163840, "scaled": True},
        # the rows of a prefill batch written to the paged cache
        {"name": "append 8 x 1024", "op": "append", "seqs": 8, "n_min": 1000, "n_max": 1024, "len_min": 0, "len_max": 9000,
         "page": 64, "layout": "interleaved", "dtype": "bf16", "max_pos": 40960},
        # one token of one sequence on a few heads with a short context: launch latency
        {"name": "tree 1 token short", "op": "tree", "seqs": 1, "n_min": 1, "n_max": 1, "len_min": 77, "len_max": 77, "heads": 20,
         "page": 16, "dtype": "f16"},
        # ordinary single-token decode of one sequence, all heads
        {"name": "tree 1 token", "op": "tree", "seqs": 1, "n_min": 1, "n_max": 1, "len_min": 30011, "len_max": 30011, "heads": 128,
         "page": 64, "dtype": "bf16"},
        # one sequence verifying a small drafted tree (the 8-row decode pass)
        {"name": "tree 8 nodes", "op": "tree", "seqs": 1, "n_min": 8, "n_max": 8, "len_min": 16384, "len_max": 16384, "heads": 128,
         "page": 128, "dtype": "bf16"},
        # a ragged batch with trees of different sizes, on the head shard of a 4-way split
        {"name": "tree ragged batch", "op": "tree", "seqs": 16, "n_min": 3, "n_max": 17, "len_min": 501, "len_max": 12007, "heads": 32,
         "page": 32, "dtype": "f16"},
        # the widest tree over a long context
        {"name": "tree 64 nodes long", "op": "tree", "seqs": 1, "n_min": 64, "n_max": 64, "len_min": 65000, "len_max": 65000,
         "heads": 128, "page": 64, "dtype": "bf16"},
        # weight of one decoded token added to every cached row
        {"name": "mass 1 token", "op": "mass", "seqs": 1, "n_min": 1, "n_max": 1, "len_min": 8191, "len_max": 8191, "heads": 128,
         "page": 64, "dtype": "bf16", "decay": 1.0},
        # weights of the accepted nodes of four sequences' trees
        {"name": "mass 4 x 12 nodes", "op": "mass", "seqs": 4, "n_min": 12, "n_max": 12, "len_min": 10000, "len_max": 30000,
         "heads": 128, "page": 64, "dtype": "bf16", "decay": 0.99},
        # one sequence that has grown a little over its budget
        {"name": "evict 1 sequence", "op": "evict", "seqs": 1, "len_min": 1200, "len_max": 1200, "budget": 1024, "sinks": 4,
         "recent": 128, "page": 64, "dtype": "bf16"},
        # a batch cut down to its budget after long prefills
        {"name": "evict 16 sequences", "op": "evict", "seqs": 16, "len_min": 6000, "len_max": 40000, "budget": 8192, "sinks": 4,
         "recent": 1024, "page": 64, "dtype": "bf16"},
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["rope", "append", "tree", "tree", "tree", "mass", "evict"])
    if op == "rope":
        rot = rng.choice([32, 64, 128])
        off = rng.choice([0, 64, 128])
        return {"op": op, "tokens": _logint(rng, 1, 4096), "heads": _logint(rng, 1, 128), "head_dim": off + rot + rng.choice([0, 0, 32]),
                "rot_offset": off, "rot_dim": rot, "layout": rng.choice(["interleaved", "half"]), "grad": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "max_pos": 40960, "scaled": rng.random() < 0.5}
    seqs = _logint(rng, 1, 16)
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["bf16", "f16"])
    hi = _logint(rng, 1, 65536)
    lo = hi if rng.random() < 0.3 else rng.randint(0, hi)
    if op == "append":
        n = _logint(rng, 1, 1024)
        return {"op": op, "seqs": seqs, "n_min": max(1, n // 2), "n_max": n, "len_min": min(lo, 8192), "len_max": min(hi, 16384),
                "page": page, "layout": rng.choice(["interleaved", "half"]), "dtype": dtype, "max_pos": 40960}
    if op == "evict":
        hi = max(hi, 64)
        return {"op": op, "seqs": seqs, "len_min": min(lo, 40000), "len_max": min(hi, 40000), "budget": _logint(rng, max(1, hi // 16), hi), "sinks": rng.randint(0, 8),
                "recent": rng.choice([0, 16, 128]), "page": page, "dtype": dtype}
    n = _logint(rng, 1, 64)
    c = {"op": op, "seqs": seqs, "n_min": rng.randint(1, n), "n_max": n, "len_min": lo, "len_max": hi,
         "heads": rng.choice([8, 20, 32, 64, 128]), "page": page, "dtype": dtype}
    if op == "mass":
        c["decay"] = rng.choice([1.0, 0.95])
    return c


def _cost(case):
    w = work(case)
    pad = 0.0
    if case["op"] in ("tree", "mass"):      # the plain form pads every sequence to the longest
        pad = case["seqs"] * case["n_max"] * case["heads"] * (case["len_max"] + case["n_max"]) * 2176.0
    return w["bytes"] / 6e12 + max(w["flops"], pad) / 50e12


_most = None


def draw(rng):
    global _most
    if _most is None:
        _most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= _most:
            return c


def _spread(lo, hi, n, down=False):
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
    return v[::-1] if down else v


def _sizes(case):
    """Context lengths and new rows of every sequence."""
    lens = _spread(case["len_min"], case["len_max"], case["seqs"])
    new = _spread(case["n_min"], case["n_max"], case["seqs"], down=True) if "n_min" in case else [0] * case["seqs"]
    return lens, new


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["head_dim"] * e, "flops": 3 * n * case["rot_dim"]}
    lens, new = _sizes(case)
    if case["op"] == "append":
        return {"bytes": sum(new) * (2 * ROW * e + 256 + 12), "flops": 3 * sum(new) * ROPE}
    if case["op"] == "evict":
        over = [max(0, n - case["budget"]) for n in lens]
        kept = [o * min(n, case["budget"]) // max(1, n) for o, n in zip(over, lens)]
        return {"bytes": sum(8 * n for n, o in zip(lens, over) if o) + sum(kept) * 2 * (ROW * e + 8) + 4 * len(lens), "flops": 0}
    H = case["heads"]
    rows = sum(new) * H
    pairs = sum(H * (n * l + n * (n + 1) // 2) for l, n in zip(lens, new))
    cache = sum(l + n for l, n in zip(lens, new)) * ROW * e
    if case["op"] == "tree":
        return {"bytes": cache + rows * ((ROW + LATENT) * e + 4), "flops": 2 * pairs * (ROW + LATENT)}
    return {"bytes": cache + rows * (ROW * e + 4) + 8 * sum(l + n for l, n in zip(lens, new)), "flops": 2 * pairs * ROW}


def _freqs(rot_dim, scaled, device="cpu"):
    """Rotation frequencies in 64 bits; scaled: interpolated where a turn is longer than the original context."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64, device=device)
    f = YARN["base"] ** (-2.0 * i / rot_dim)
    if not scaled:
        return f
    at = lambda turns: rot_dim * math.log(YARN["orig_ctx"] / (turns * 2 * math.pi)) / (2 * math.log(YARN["base"]))
    lo, hi = max(0, math.floor(at(YARN["beta_fast"]))), min(rot_dim - 1, math.ceil(at(YARN["beta_slow"])))
    r = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f * (1 - r) + f / YARN["factor"] * r


def _mscale(scaled):
    return 0.1 * math.log(YARN["factor"]) + 1.0 if scaled else 1.0


def _table(max_pos, rot_dim, scaled):
    """cos and sin of every position in 32 bits, as a program keeps them: [max_pos][rot_dim / 2][2]."""
    a = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * _freqs(rot_dim, scaled, DEV)
    return (torch.stack([a.cos(), a.sin()], -1) * _mscale(scaled)).float()


def _pages(case, g, lens, new):
    """A shuffled block table for lens + new rows and the pool's number of pages."""
    page = case["page"]
    need = [(l + n + page - 1) // page for l, n in zip(lens, new)]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=g, device=DEV).int()
    width = max(1, max(need))
    table = torch.zeros(len(lens), width, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def _trees(case, seed, new):
    """One random tree per sequence: bit j of a node's mask is set for its ancestors and itself."""
    import random
    r = random.Random(seed * 7919 + 13)
    masks = []
    for n in new:
        m = []
        for j in range(n):
            p = r.randint(max(-1, j - 4), j - 1)
            v = (m[p] if p >= 0 else 0) | (1 << j)
            m.append(v)
        masks += m
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in masks], dtype=torch.int64, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)
    st = {"case": case, "seed": seed}
    if own:
        from loki_b200 import attention as A
        st["A"] = A
    if case["op"] == "rope":
        T = case["tokens"]
        st["x"] = randn(T, case["heads"], case["head_dim"]).to(dt)
        first = int(torch.randint(0, case["max_pos"] - T + 1, (1,), generator=g, device=DEV))
        st["pos"] = torch.arange(first, first + T, dtype=torch.int32, device=DEV)
        if own:
            st["ctx"] = A.AttnContext(0)
            st["rope"] = A.RopeTable(case["max_pos"], case["rot_dim"], mscale=_mscale(case["scaled"]), device=DEV,
                                     **(YARN if case["scaled"] else {"base": YARN["base"]}))
        else:
            st["table"] = _table(case["max_pos"], case["rot_dim"], case["scaled"])
        return st
    lens, new = _sizes(case)
    B, T = case["seqs"], sum(new)
    bt, n_pages = _pages(case, g, lens, new)
    slots = n_pages * case["page"]
    rows = torch.empty(slots, ROW, dtype=dt, device=DEV)
    for at in range(0, slots, 65536):
        rows[at:at + 65536] = randn(min(65536, slots - at), ROW).to(dt)
    st["rows"], st["block_table"] = rows, bt
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["starts"] = torch.tensor([sum(new[:i]) for i in range(B + 1)], dtype=torch.int32, device=DEV)
    st["mass"] = torch.rand(slots, generator=g, device=DEV).pow(8) * 16
    st["pos"] = torch.zeros(slots, dtype=torch.int32, device=DEV)
    if case["op"] == "append":
        st["latent"], st["k_rope"] = randn(T, LATENT).to(dt), randn(T, ROPE).to(dt)
        st["new_pos"] = torch.cat([torch.arange(l, l + n, dtype=torch.int32, device=DEV) for l, n in zip(lens, new)])
        if own:
            st["rope"] = A.RopeTable(case["max_pos"], ROPE, mscale=_mscale(True), device=DEV, **YARN)
        else:
            st["table"] = _table(case["max_pos"], ROPE, True)
    elif case["op"] == "evict":
        L = max(lens)
        order = torch.arange(L, device=DEV)
        real = order[None, :] < st["lens"][:, None]
        st["pos"][_slots(st, order[None, :].expand(B, L))[real]] = order.int()[None, :].expand(B, L)[real]
        st["mass"][torch.rand(slots, generator=g, device=DEV) < 0.02] = 0.0      # rows that nothing attended to
        st["next_pos"] = st["lens"].clone()
    else:
        st["q"] = randn(T, case["heads"], ROW).to(dt)
        st["tree"] = _trees(case, seed, new)
        st["scale"] = 192 ** -0.5
        if case["op"] == "mass":
            st["weight"] = (torch.rand(T, generator=g, device=DEV) < 0.6).float()      # accepted nodes
            st["weight"][st["starts"][:-1].long()] = 1.0
            st["lse"] = torch.logsumexp(_scores(st)[0], -1)[_tokens(st)].contiguous()
    if own:
        st["ctx"] = A.AttnContext(0, max_seqs=B, max_tokens=max(T, 1))
        st["cache"] = A.KvCache(rows, case["page"], bt, st["lens"], mass=st["mass"], pos=st["pos"])
    return st


def _slots(st, i):
    """Pool row of row i [B][n] of every sequence."""
    page = st["case"]["page"]
    page_id = torch.gather(st["block_table"].long(), 1, (i // page).clamp(max=st["block_table"].shape[1] - 1))
    return page_id * page + i % page


def _tokens(st):
    """(sequence, node) index of every token in the padded [B][n_max] order."""
    n = st["starts"].diff().long()
    N = max(_sizes(st["case"])[1])
    j = torch.arange(N, device=DEV)[None, :].expand(len(n), N)
    return torch.nonzero(j < n[:, None], as_tuple=True)


def _rotate(x, cs, layout, grad):
    """x [T][...][R] rotated by cs [T][R / 2][2]."""
    cs = cs.reshape(cs.shape[0], *[1] * (x.dim() - 2), *cs.shape[1:])
    c, s = cs[..., 0], -cs[..., 1] if grad else cs[..., 1]
    if layout == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _scores(st):
    """Masked scores [B][n_max][H][L] of the padded batch in 32 bits, with the padded keys [B][L][ROW]."""
    lens, n = st["lens"].long(), st["starts"].diff().long()
    all_lens, new = _sizes(st["case"])
    L, N, B = max(a + b for a, b in zip(all_lens, new)), max(new), len(new)
    b, j = _tokens(st)
    q = torch.zeros(B, N, st["q"].shape[1], ROW, device=DEV)
    q[b, j] = st["q"].float()
    tree = torch.zeros(B, N, dtype=torch.int64, device=DEV)
    tree[b, j] = st["tree"]
    i = torch.arange(L, device=DEV)[None, :].expand(B, L)
    keys = st["rows"][_slots(st, i)].float()
    node = i - lens[:, None]
    keys = torch.where((node < n[:, None])[..., None], keys, 0.0)
    seen = (tree[:, :, None] >> node[:, None, :].clamp(0, 63)) & 1
    ok = (node[:, None, :] < 0) | ((node < n[:, None])[:, None, :] & (seen == 1))
    s = torch.matmul(q.flatten(1, 2), keys.transpose(1, 2)).view(B, N, -1, L) * st["scale"]
    return s.masked_fill_(~ok[:, :, None, :], -math.inf), keys, i


def _plain_tree(st):
    s, keys, _ = _scores(st)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(1, 2), keys[..., :LATENT]).view(*p.shape[:3], LATENT)
    o = torch.where(l > 0, o / l, 0.0)
    lse = (m + l.log()).squeeze(-1)
    at = _tokens(st)
    return o[at].to(st["rows"].dtype), lse[at]


def _plain_mass(st):
    s, _, i = _scores(st)
    b, j = _tokens(st)
    lse = torch.full(s.shape[:3], math.inf, device=DEV)
    lse[b, j] = st["lse"]
    w = torch.zeros(s.shape[:2], device=DEV)
    w[b, j] = st["weight"]
    add = (s.sub_(lse[..., None]).exp_() * w[:, :, None, None]).sum((1, 2))
    real = i < (st["lens"] + st["starts"].diff())[:, None]
    at = _slots(st, i)[real]
    st["mass"][at] = st["case"]["decay"] * st["mass"][at] + add[real]
    return st["mass"]


def _plain_evict(st):
    c, lens = st["case"], st["lens"].long()
    L, B = max(_sizes(c)[0]), c["seqs"]
    i = torch.arange(L, device=DEV)[None, :].expand(B, L)
    at, real = _slots(st, i), i < lens[:, None]
    mass, pos = st["mass"][at], st["pos"][at].long()
    safe = (pos < c["sinks"]) | (pos >= st["next_pos"].long()[:, None] - c["recent"])
    key = torch.where(safe, math.inf, mass.nan_to_num(nan=-1e30))
    key = torch.where(real, key, -math.inf)
    rank = torch.sort(key, dim=1, descending=True, stable=True).indices
    new = lens.clamp(max=c["budget"])
    keep = torch.zeros(B, L, dtype=torch.bool, device=DEV).scatter_(1, rank, i < new[:, None])
    dst, src = at[(i < new[:, None]) & ~keep], at[(i >= new[:, None]) & keep]
    for t in (st["rows"], st["mass"], st["pos"]):
        t[dst] = t[src]
    return new.int(), st["rows"], st["mass"], st["pos"]


def _plain_append(st):
    i = st["lens"].long()[:, None] + torch.arange(max(_sizes(st["case"])[1]), device=DEV)[None, :]
    at = _slots(st, i)[_tokens(st)]
    k = _rotate(st["k_rope"].float(), st["table"][st["new_pos"].long()], st["case"]["layout"], False)
    st["rows"][at] = torch.cat([st["latent"].float(), k], -1).to(st["rows"].dtype)
    st["mass"][at] = 0.0
    st["pos"][at] = st["new_pos"]
    return st["rows"], st["mass"], st["pos"]


def run(state):
    c = state["case"]
    op = c["op"]
    if own:
        ctx = state["ctx"]
        if op == "rope":
            return ctx.rope(state["x"], state["pos"], state["rope"], rot_offset=c["rot_offset"], layout=c["layout"], grad=c["grad"])
        cache = state["cache"]
        if op == "append":
            ctx.append(cache, state["latent"], state["k_rope"], state["starts"], state["new_pos"], state["rope"], layout=c["layout"])
            return state["rows"], state["mass"], state["pos"]
        if op == "tree":
            return ctx.tree(state["q"], cache, state["starts"], state["tree"], state["scale"])
        if op == "mass":
            ctx.mass(state["q"], state["lse"], cache, state["starts"], state["tree"], state["scale"], weight=state["weight"],
                     decay=c["decay"])
            return state["mass"]
        new = ctx.evict(cache, c["budget"], state["next_pos"], sinks=c["sinks"], recent=c["recent"])
        return new, state["rows"], state["mass"], state["pos"]
    if op == "rope":
        x = state["x"].float()
        a, r = c["rot_offset"], c["rot_dim"]
        y = _rotate(x[..., a:a + r], state["table"][state["pos"].long()], c["layout"], c["grad"])
        return torch.cat([x[..., :a], y, x[..., a + r:]], -1).to(state["x"].dtype)
    return {"append": _plain_append, "tree": _plain_tree, "mass": _plain_mass, "evict": _plain_evict}[op](state)


# ---- the definitions in 64 bits, one sequence and one slab of rows at a time

def _exact_turn(x, pos, rot_dim, scaled, layout, sign):
    z = torch.polar(torch.full((1,), _mscale(scaled), dtype=torch.float64, device=DEV),
                    sign * pos.double()[:, None] * _freqs(rot_dim, scaled, DEV))
    x = x.double()
    h = rot_dim // 2
    v = torch.complex(*((x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :h], x[..., h:])))
    v = v * (z[:, None, :] if x.dim() == 3 else z)
    return torch.view_as_real(v).flatten(-2) if layout == "interleaved" else torch.cat([v.real, v.imag], -1)


def _exact_rows(st, b, n):
    page = st["case"]["page"]
    i = torch.arange(n, device=DEV)
    return st["block_table"][b].long()[i // page] * page + i % page


def exact(case, seed):
    if case["op"] == "evict":        # rows are chosen and moved, nothing is computed
        return None
    global own
    was, own = own, False
    st = prepare(case, seed)
    own = was
    if case["op"] == "rope":
        a, r = case["rot_offset"], case["rot_dim"]
        y = st["x"].double()
        y[..., a:a + r] = _exact_turn(st["x"][..., a:a + r], st["pos"], r, case["scaled"], case["layout"], -1.0 if case["grad"] else 1.0)
        return y
    lens, new = _sizes(case)
    if case["op"] == "append":
        rows = st["rows"].double()
        k = _exact_turn(st["k_rope"], st["new_pos"], ROPE, True, case["layout"], 1.0)
        at = torch.cat([_exact_rows(st, b, l + n)[l:] for b, (l, n) in enumerate(zip(lens, new))])
        rows[at, :LATENT], rows[at, LATENT:] = st["latent"].double(), k
        return rows, None, None
    H = case["heads"]
    out = torch.zeros(sum(new), H, LATENT, dtype=torch.float64, device=DEV)
    lse = torch.full((sum(new), H), -math.inf, dtype=torch.float64, device=DEV)
    mass = st["mass"].double()
    t = 0
    for b, (l, n) in enumerate(zip(lens, new)):
        at = _exact_rows(st, b, l + n)
        k = st["rows"][at].double()
        bits = torch.arange(n, device=DEV)
        add = torch.zeros(l + n, dtype=torch.float64, device=DEV)
        for j in range(n):
            s = st["scale"] * (st["q"][t].double() @ k.T)
            s[:, l:][:, (st["tree"][t] >> bits) & 1 == 0] = -math.inf
            if case["op"] == "tree":
                lse[t] = torch.logsumexp(s, -1)
                out[t] = torch.exp(s - lse[t][:, None]) @ k[:, :LATENT]
            else:
                add += float(st["weight"][t]) * torch.exp(s - st["lse"][t].double()[:, None]).sum(0)
            t += 1
        if case["op"] == "mass":
            mass[at] = case["decay"] * mass[at] + add
    return (out, lse) if case["op"] == "tree" else mass
