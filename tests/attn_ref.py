"""Plain 64-bit (CPU) forms of the latent-cache attention operators, and the cases that their tests build."""
import math

import numpy as np
import torch

LATENT, ROPE, ROW = 512, 64, 576
# unit roundoff of each type (half a unit in the last place of 1)
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def freqs(rot_dim, base=10000.0, factor=1.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0):
    out = []
    for i in range(rot_dim // 2):
        f = base ** (-2.0 * i / rot_dim)
        if factor > 1:
            at = [rot_dim * math.log(orig_ctx / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (beta_fast, beta_slow)]
            lo, hi = max(0, math.floor(at[0])), min(rot_dim - 1, math.ceil(at[1]))
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            f = f * (1 - r) + f / factor * r
        out.append(f)
    return np.array(out)


def rope(x, pos, f, off, layout, grad=False, mscale=1.0):
    """x [T][H][D] float64 -> the rotated heads, with [off, off + 2 len(f)) rotated."""
    y = np.array(x, np.float64)
    n = len(f)
    a = np.asarray(pos, np.float64)[:, None] * f[None, :]
    c, s = np.cos(a)[:, None, :] * mscale, np.sin(a)[:, None, :] * mscale * (-1 if grad else 1)
    ia = off + (2 * np.arange(n) if layout == "interleaved" else np.arange(n))
    ib = ia + (1 if layout == "interleaved" else n)
    u, v = x[..., ia].astype(np.float64), x[..., ib].astype(np.float64)
    y[..., ia], y[..., ib] = c * u - s * v, s * u + c * v
    return y


class Paged:
    """A pool with shuffled pages holding the rows of several sequences; every unused row is NaN."""

    def __init__(self, lens, new, page, dtype, device, seed=0, row_stride=ROW, extra_pages=2, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.page, self.dtype = list(lens), list(new), page, dtype
        need = [(l + n + page - 1) // page for l, n in zip(lens, new)]
        total = sum(need) + extra_pages
        order = torch.randperm(total, generator=g).tolist()
        self.table = torch.full((len(lens), max(1, max(need))), 0, dtype=torch.int32)
        host = torch.full((total * page, ROW), float("nan"), dtype=torch.float32)
        self.seq = []                    # every sequence's rows, in the pool's type
        self.slots = []
        for b, (l, n) in enumerate(zip(lens, new)):
            ids = [order.pop() for _ in range(need[b])]
            self.table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
            rows = (torch.randn(l + n, ROW, generator=g) * spread).to(dtype)
            at = torch.tensor([ids[i // page] * page + i % page for i in range(l + n)], dtype=torch.long)
            host[at] = rows.float()
            self.seq.append(rows)
            self.slots.append(at)
        buf = torch.full((total * page, row_stride), float("nan"), dtype=dtype)
        buf[:, :ROW] = host.to(dtype)
        self.rows = buf.to(device)[:, :ROW]
        self.device = device
        self.n_slots = total * page
        self.starts = torch.tensor([sum(self.new[:i]) for i in range(len(self.new) + 1)], dtype=torch.int32, device=device)

    def cache(self, A, mass=None, pos=None):
        return A.KvCache(self.rows, self.page, self.table.to(self.device), torch.tensor(self.lens, dtype=torch.int32, device=self.device),
                         mass=mass, pos=pos)

    def set_row(self, b, i, value):
        """Overwrite row i of sequence b (pool and reference copy)."""
        self.seq[b][i] = value
        self.rows[self.slots[b][i].item()] = self.seq[b][i].to(self.device)


def tree_masks(new, seed=0):
    """Random ancestor masks (each node sees itself and its ancestors), one 64-bit word per token."""
    r = np.random.default_rng(seed)
    out = []
    for n in new:
        m = []
        for j in range(n):
            p = int(r.integers(max(-1, j - 5), j)) if j else -1
            m.append((m[p] if p >= 0 else 0) | 1 << j)
        out += m
    return out


def to_words(masks, device):
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in masks], dtype=torch.int64, device=device)


def chain_masks(new):
    return [(2 << j) - 1 for n in new for j in range(n)]


def scores(pg, b, q, masks, scale):
    """Per token of sequence b: (token, scores [H][rows it sees], those rows [n][576]) in 64 bits; rows it does not see
    are left out, whatever they hold."""
    l, n, t0 = pg.lens[b], pg.new[b], sum(pg.new[:b])
    rows = pg.seq[b].double()
    for j in range(n):
        see = torch.tensor(list(range(l)) + [l + i for i in range(n) if masks[t0 + j] >> i & 1], dtype=torch.long)
        k = rows[see]
        yield t0 + j, see, q[t0 + j].double() @ k.T * scale, k


def tree(pg, q, masks, scale):
    """out [T][H][512], lse [T][H] and the elementwise bound of out's error, all 64 bits.

    The bound: with u the type's unit roundoff, P is rounded to the type once (u sum p|v|; in fp16 also half the
    smallest step, 2^-25 of the largest weight a row can be scaled to, per row seen), out once (u |out|).  A score of
    576 products added in 32 bits is off by at most ds = 576 * 2^-23 * scale * sum|q k|, which moves p by a factor
    within exp(+-2 ds) against the others; the sum over n rows in 32 bits adds n * 2^-23."""
    u = U[pg.dtype]
    T, H = q.shape[:2]
    out, lse = torch.zeros(T, H, LATENT, dtype=torch.float64), torch.full((T, H), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros(T, H, LATENT, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for b in range(len(pg.lens)):
        for t, see, s, k in scores(pg, b, q, masks, scale):
            n = len(see)
            if n == 0:
                continue
            lse[t] = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[t][:, None])
            v = k[:, :LATENT]
            out[t] = p @ v
            av = p @ v.abs()
            ds = 576 * 2.0 ** -23 * scale * (q[t].double().abs() @ k.abs().T).amax(-1)
            tol[t] = av * (u + 2 * ds[:, None] + n * 2.0 ** -23)
            if pg.dtype == torch.float16:
                tol[t] += 2.0 ** -25 * v.abs().sum(0)[None, :]
            tol[t] += u * out[t].abs() + 2.0 ** -24
            ltol[t] = ds + n * 2.0 ** -23 + 4 * 2.0 ** -23 * (1 + lse[t].abs())
    return out, lse, tol, ltol


def mass(pg, q, lse, masks, scale, weight, decay, mass0):
    """The new mass [n_slots] in 64 bits and its bound: each term exp(s - lse) is off by the score's ds (above) and a few
    32-bit roundings of its argument and of the exponential; adding T*H of them in 32 bits adds T*H * 2^-23."""
    out, tol = mass0.double().clone(), torch.zeros(pg.n_slots, dtype=torch.float64)
    for b in range(len(pg.lens)):
        if not pg.new[b]:
            continue
        out[pg.slots[b]] *= decay
        rows = pg.new[b] * q.shape[1]
        for t, see, s, k in scores(pg, b, q, masks, scale):
            if weight[t] == 0:
                continue
            ok = torch.isfinite(lse[t])
            p = torch.where(ok[:, None], torch.exp(s - torch.where(ok, lse[t].double(), torch.zeros(()).double())[:, None]), torch.zeros(()).double())
            ds = 576 * 2.0 ** -23 * scale * (q[t].double().abs() @ k.abs().T).amax(-1, keepdim=True)
            arg = 2.0 ** -22 * (s.abs() + lse[t].double().abs().nan_to_num(posinf=0)[:, None] + 1)
            at = pg.slots[b][see]
            out[at] += float(weight[t]) * p.sum(0)
            tol[at] += float(weight[t]) * (p * (ds + arg + rows * 2.0 ** -23)).sum(0)
        tol[pg.slots[b]] += 4 * 2.0 ** -24 * out[pg.slots[b]].abs()
    return out, tol


def evict(lens, slots, mass, pos, budget, sinks, recent, next_pos):
    """new lengths and the moves [(source slot, destination slot)] of the rule, one row at a time."""
    new, moves = [], []
    for b, l in enumerate(lens):
        if l <= budget:
            new.append(l)
            continue
        new.append(budget)

        def rank(i):
            s = slots[b][i]
            safe = pos[s] < sinks or pos[s] >= next_pos[b] - recent
            m = float(mass[s])
            return (0 if safe else 2 if math.isnan(m) else 1, 0.0 if safe or math.isnan(m) else -m, i)
        keep = set(sorted(range(l), key=rank)[:budget])
        holes = [i for i in range(budget) if i not in keep]
        tail = [i for i in range(budget, l) if i in keep]
        moves += [(int(slots[b][s]), int(slots[b][d])) for s, d in zip(tail, holes)]
    return new, moves
