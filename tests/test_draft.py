"""The drafted-tree decode loop (loki_b200.draft): tree masks on the CPU, and the whole loop on the GPU against a plain
64-bit one that keeps its rows in lists."""
import numpy as np
import pytest
import torch

from tests import attn_ref as R


def test_tree_words():
    from loki_b200.draft import tree_words
    assert tree_words([[-1, 0, 0, 1], [], [-1, -1]]) == [1, 3, 5, 11, 1, 2]
    chain = tree_words([list(range(-1, 63))])
    assert chain[62] == (1 << 63) - 1 and chain[63] == -1
    with pytest.raises(ValueError):
        tree_words([[-1] * 65])
    with pytest.raises(ValueError):
        tree_words([[0]])


@pytest.mark.gpu
def test_decode_loop_matches_a_plain_one(native):
    """Prompts, then steps of verify and accept with eviction: every step's attention against the rows that the plain loop
    holds, and its masses.  The plain loop takes each step's kept set from the device (two masses may lie closer than the
    sums' rounding) after checking that no row it would have kept has clearly more weight than one that stayed."""
    from loki_b200.draft import DraftSession, tree_words
    g = torch.Generator().manual_seed(4)
    H, budget, sinks, recent, scale = 8, 96, 2, 8, 192 ** -0.5
    s = DraftSession(2, H, max_len=400, budget=budget, sinks=sinks, recent=recent, scale=scale, page=16)
    f = R.freqs(64)
    counts = [150, 60]
    lat, kr = torch.randn(210, 512, generator=g).bfloat16(), torch.randn(210, 64, generator=g).bfloat16()
    s.prefill(lat.cuda(), kr.cuda(), counts)
    next_pos = list(counts)
    for step in range(4):
        parents = [[-1, 0, 0, 1, 3], [-1, 0, 1]] if step % 2 else [[-1, -1], [-1, 0, 0, 0]]
        sizes = [len(p) for p in parents]
        T = sum(sizes)
        q = torch.randn(T, H, 576, generator=g).bfloat16()
        lat, kr = torch.randn(T, 512, generator=g).bfloat16(), torch.randn(T, 64, generator=g).bfloat16()
        lens = s.lens.tolist()
        qd = q.cuda()
        out, lse = s.verify(qd, lat.cuda(), kr.cuda(), parents)
        s.ctx.device_error()
        # positions and rotations
        pos, first = [], 0
        for b, p in enumerate(parents):
            d = []
            for j, a in enumerate(p):
                d.append(0 if a < 0 else d[a] + 1)
            pos += [next_pos[b] + x for x in d]
        rot = R.rope(q.double().numpy(), pos, f, 512, "interleaved")
        assert np.abs(qd.cpu().double().numpy() - rot).max() <= 2.0 ** -8 * np.abs(rot).max()
        pg = R.Paged.__new__(R.Paged)                # the rows that the device holds now, as the reference's cache
        pg.lens, pg.new, pg.dtype, pg.n_slots = lens, sizes, torch.bfloat16, s.cache.rows.shape[0]
        pg.slots = [s.slots(torch.full((l + n,), b, device="cuda"), torch.arange(l + n, device="cuda")).cpu()
                    for b, (l, n) in enumerate(zip(lens, sizes))]
        rows, where = s.cache.rows.cpu(), s.cache.pos.cpu()
        pg.seq = [rows[at] for at in pg.slots]
        for b in range(2):
            new = pg.slots[b][lens[b]:]
            t0 = sum(sizes[:b])
            assert torch.equal(rows[new][:, :512], lat[t0:t0 + sizes[b]]) and where[new].tolist() == pos[t0:t0 + sizes[b]]
        masks = [w % (1 << 64) for w in tree_words(parents)]
        want, wl, tol, ltol = R.tree(pg, qd.cpu(), masks, scale)
        assert ((out.cpu().double() - want).abs() <= tol).all() and ((lse.cpu().double() - wl).abs() <= ltol).all()
        # acceptance: weights of the accepted nodes only, then their rows, then the cut
        paths = [[0, 1, 3], [0, 1, 2]] if step % 2 else [[1], [0, 2]]
        w = torch.zeros(T)
        for b, path in enumerate(paths):
            for j in path:
                w[sum(sizes[:b]) + j] = 1.0
        wm, mt = R.mass(pg, qd.cpu(), lse.cpu(), masks, scale, w, 1.0, s.cache.mass.cpu())
        before = rows.clone()
        s.accept(paths)
        s.ctx.device_error()
        mass, rows, where = s.cache.mass.cpu().double(), s.cache.rows.cpu(), s.cache.pos.cpu()
        for b, path in enumerate(paths):
            next_pos[b] += len(path)
            held = pg.slots[b][:lens[b]].tolist() + [pg.slots[b][lens[b] + j].item() for j in path]
            n = min(len(held), budget)
            assert s.lens.tolist()[b] == n
            got = {tuple(r.tolist()): m for r, m in zip(rows[pg.slots[b][:n]].view(torch.int16), mass[pg.slots[b][:n]].tolist())}
            assert len(got) == n
            old = {tuple(before[at].view(torch.int16).tolist()): (wm[at].item(), mt[at].item(), k < lens[b]) for k, at in enumerate(held)}
            assert set(got) <= set(old)
            for r, m in got.items():
                assert abs(m - old[r][0]) <= old[r][1] + 1e-30
            if len(held) > budget:
                gone = [v for r, v in old.items() if r not in got]
                p = {tuple(r.tolist()): x for r, x in zip(rows[pg.slots[b][:n]].view(torch.int16), where[pg.slots[b][:n]].tolist())}
                free = [got[r] for r, x in p.items() if not (x < sinks or x >= next_pos[b] - recent)]
                assert max(v[0] - v[1] for v in gone) <= min(free) + 1e-6
                assert {x for x in p.values()} >= set(range(sinks)) | set(range(next_pos[b] - recent, next_pos[b]))
        assert s.next_pos.tolist() == next_pos


@pytest.mark.gpu
def test_example_runs(native, capsys):
    from loki_b200 import draft
    s = draft.main(steps=3)
    assert s.lens.tolist() == [192, 192] and "step 2" in capsys.readouterr().out
