"""One attention layer's cache side over a decode loop with drafted token trees: the operators of loki_b200.attention in
the order in which a serving loop uses them.

    s = DraftSession(n_seqs=2, heads=128, max_len=8192, budget=4096)
    s.prefill(latent, k_rope, counts)                    # rows of the prompts
    out, lse = s.verify(q, latent, k_rope, parents)      # drafted trees: rotate, append, attend
    s.accept(paths)                                      # keep the accepted nodes, add their weights, evict over budget

The reference drafts and verifies one row after another (src/fused_layer.cu:473-527); here a tree of up to 64 nodes per
sequence is one call, and the cache is cut to `budget` rows by the attention weight that they received.

`python -m loki_b200.draft` runs a small loop on random tensors and prints the cache's lengths.
"""
import torch

from . import attention as A
from .native import ATTN_LATENT, ATTN_MAX_NODES, ATTN_ROPE, ATTN_ROW


def tree_words(parents):
    """64-bit masks of drafted trees: parents[b][j] is the parent of node j of sequence b (-1: the context's last token);
    a node sees its ancestors and itself.  Returns one int per node, in order (two's complement, for an int64 tensor)."""
    words = []
    for p in parents:
        if len(p) > ATTN_MAX_NODES:
            raise ValueError("a tree of %d nodes: at most %d" % (len(p), ATTN_MAX_NODES))
        seen = []
        for j, a in enumerate(p):
            if not -1 <= a < j:
                raise ValueError("node %d: its parent %d must come before it" % (j, a))
            seen.append((seen[a] if a >= 0 else 0) | 1 << j)
        words += [w - (1 << 64) if w >> 63 else w for w in seen]
    return words


class DraftSession:
    """The paged latent cache of n_seqs sequences with everything its decode loop needs.  budget: rows that a sequence keeps
    after each accept() (None: all); sinks first positions and the `recent` last ones are always kept.  rope: a RopeTable
    (default: unstretched, base 10000, max_positions of them, 2 max_len unless given).  Positions grow with every accepted token,
    evicted or not, so max_positions bounds the whole text; a step that would pass it, or the pages, is refused before it starts.
    lens and next_pos are the session's to change: it keeps their values on the host too."""

    def __init__(self, n_seqs, heads, max_len, budget=None, sinks=4, recent=64, decay=1.0, dtype=torch.bfloat16, page=64,
                 scale=192 ** -0.5, rope=None, max_positions=None, layout="interleaved", device=0):
        self.n_seqs, self.heads, self.max_len, self.budget, self.sinks, self.recent = n_seqs, heads, max_len, budget, sinks, recent
        self.decay, self.scale, self.layout = decay, scale, layout
        self.device = torch.device("cuda", device)
        per = (max_len + ATTN_MAX_NODES + page - 1) // page
        new = lambda *shape, dt=torch.int32: torch.zeros(*shape, dtype=dt, device=self.device)
        self.ctx = A.AttnContext(device, n_seqs, n_seqs * ATTN_MAX_NODES)
        self.rope = rope or A.RopeTable(max_positions or 2 * max_len, ATTN_ROPE, device=self.device)
        self.lens, self.next_pos = new(n_seqs), new(n_seqs)
        self.cache = A.KvCache(new(n_seqs * per * page, ATTN_ROW, dt=dtype), page,
                               torch.arange(n_seqs * per, dtype=torch.int32, device=self.device).view(n_seqs, per), self.lens,
                               mass=new(n_seqs * per * page, dt=torch.float32), pos=new(n_seqs * per * page))
        self._room, self._lens, self._next = per * page, [0] * n_seqs, [0] * n_seqs
        self._pending = None

    def slots(self, seq, index):
        """Pool rows of rows `index` of sequences `seq` (tensors of equal shape)."""
        page = self.cache.page_size
        return self.cache.block_table[seq, index // page].long() * page + index % page

    def _tokens(self, counts):
        """starts, and each token's sequence and place in it."""
        counts = torch.as_tensor(counts, dtype=torch.int64)
        if len(counts) != self.n_seqs or bool((counts < 0).any()):
            raise ValueError("counts: one per sequence")
        counts = counts.cpu()
        starts = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        seq = torch.repeat_interleave(torch.arange(self.n_seqs), counts)
        at = torch.arange(int(starts[-1])) - starts[seq]
        return starts.int().to(self.device), seq.to(self.device), at.to(self.device)

    def _fit(self, rows, positions):
        """Refuses rows[b] more rows or positions[b] more positions of sequence b than there is room for."""
        for b, (n, p) in enumerate(zip(rows, positions)):
            if self._lens[b] + n > self._room:
                raise ValueError("sequence %d: %d rows and %d more, its pages hold %d" % (b, self._lens[b], n, self._room))
            if self._next[b] + p > self.rope.max_pos:
                raise ValueError("sequence %d: %d positions and %d more, the rope table has %d" % (b, self._next[b], p, self.rope.max_pos))

    def _grow(self, rows, keep=None):
        """What the device's lens and next_pos become: rows[b] more, then at most `keep`."""
        for b, n in enumerate(rows):
            self._next[b] += n
            self._lens[b] = self._lens[b] + n if keep is None else min(self._lens[b] + n, keep)

    def prefill(self, latent, k_rope, counts):
        """Append the prompts' rows: counts[b] tokens of sequence b, one sequence after another.  Verified trees that were not
        accepted are dropped: the rows take their place."""
        starts, seq, at = self._tokens(counts)
        rows = torch.as_tensor(counts).tolist()
        self._fit(rows, rows)
        self.ctx.append(self.cache, latent, k_rope, starts, (self.next_pos[seq] + at).int(), self.rope, layout=self.layout)
        self._pending = None
        n = starts.diff()
        self.lens += n
        self.next_pos += n
        self._grow(rows)

    def verify(self, q, latent, k_rope, parents):
        """Attention of the drafted trees: q [T][heads][576] (its last 64 values not yet rotated; rotated in place), latent and
        k_rope the nodes' rows, parents[b] the tree of sequence b.  A node's position is its depth below the context.
        Returns out [T][heads][512] and lse [T][heads]; accept() follows."""
        words = tree_words(parents)
        starts, seq, _ = self._tokens([len(p) for p in parents])
        depths, reach = [], []
        for p in parents:
            d = []
            for j, a in enumerate(p):
                d.append(0 if a < 0 else d[a] + 1)
            depths += d
            reach.append(max(d, default=-1) + 1)
        self._fit([len(p) for p in parents], reach)
        if q.dim() != 3 or q.shape[0] != len(words) or q.shape[2] != ATTN_ROW or q.dtype is not self.cache.rows.dtype:
            raise ValueError("q: [%d][heads][%d] of the cache's dtype" % (len(words), ATTN_ROW))
        words = torch.tensor(words, dtype=torch.int64).to(self.device)
        pos = (self.next_pos[seq] + torch.tensor(depths, dtype=torch.int64).to(self.device)).int()
        self.ctx.append(self.cache, latent, k_rope, starts, pos, self.rope, layout=self.layout)      # first: it may refuse its rows
        self._pending = None
        self.ctx.rope(q, pos, self.rope, rot_offset=ATTN_LATENT, layout=self.layout, out=q)
        out, lse = self.ctx.tree(q, self.cache, starts, words, self.scale)
        self._pending = (q, lse, starts, words, [list(p) for p in parents])
        return out, lse

    def accept(self, paths):
        """Keep node paths[b] (the accepted branch, from a root of sequence b's tree down) of every sequence: their queries'
        weights go to the rows they attended to, their rows follow the context, and sequences over budget are cut."""
        if self._pending is None:
            raise ValueError("accept() follows verify()")
        q, lse, starts, words, parents = self._pending
        if len(paths) != self.n_seqs:
            raise ValueError("paths: one per sequence")
        for b, (path, tree) in enumerate(zip(paths, parents)):
            if any(not 0 <= j < len(tree) for j in path) or any(tree[j] != a for j, a in zip(path, [-1, *path])):
                raise ValueError("paths[%d]: each node's parent comes before it, the first has none" % b)
        self._pending = None
        first, w = 0, torch.zeros(sum(len(tree) for tree in parents))
        src_seq, src_at, dst_at = [], [], []
        for b, (path, tree) in enumerate(zip(paths, parents)):
            for k, j in enumerate(path):
                w[first + j] = 1.0
                src_seq.append(b)
                src_at.append(j)
                dst_at.append(k)
            first += len(tree)
        self.ctx.mass(q, lse, self.cache, starts, words, self.scale, weight=w.to(self.device), decay=self.decay)
        seq = torch.tensor(src_seq, dtype=torch.int64, device=self.device)
        base = self.lens[seq].long()
        src = self.slots(seq, base + torch.tensor(src_at, dtype=torch.int64, device=self.device))
        dst = self.slots(seq, base + torch.tensor(dst_at, dtype=torch.int64, device=self.device))
        for t in (self.cache.rows, self.cache.mass, self.cache.pos):
            t[dst] = t[src]                              # read in whole before it is written
        n = torch.tensor([len(p) for p in paths], dtype=torch.int32).to(self.device)
        self.lens += n
        self.next_pos += n
        self._grow([len(p) for p in paths], self.budget)
        if self.budget is not None:
            self.ctx.evict(self.cache, self.budget, self.next_pos, sinks=self.sinks, recent=self.recent, new_lens=self.lens)


def main(steps=6, n_seqs=2, heads=16, nodes=6, prompt=200, budget=192, seed=0):
    import random
    g = torch.Generator(device="cuda").manual_seed(seed)
    pick = random.Random(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)
    s = DraftSession(n_seqs, heads, max_len=prompt + steps * nodes, budget=budget, recent=32)
    s.prefill(randn(n_seqs * prompt, ATTN_LATENT), randn(n_seqs * prompt, ATTN_ROPE), [prompt] * n_seqs)
    for step in range(steps):
        parents = [[pick.randint(-1, j - 1) for j in range(nodes)] for _ in range(n_seqs)]
        T = n_seqs * nodes
        out, _ = s.verify(randn(T, heads, ATTN_ROW), randn(T, ATTN_LATENT), randn(T, ATTN_ROPE), parents)
        paths = []
        for p in parents:                                # the branch that ends in the last node
            j, path = nodes - 1, []
            while j >= 0:
                path.append(j)
                j = p[j]
            paths.append(path[::-1])
        s.accept(paths)
        print("step %d: accepted %s, rows %s, next positions %s, |out| %.3f" %
              (step, [len(p) for p in paths], s.lens.tolist(), s.next_pos.tolist(), out.float().abs().mean()))
    s.ctx.device_error()
    return s


if __name__ == "__main__":
    main()
