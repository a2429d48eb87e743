"""The drafted decode loop's own bookkeeping (loki_b200.draft) without a GPU: the operators are stood in for by calls that
only keep count, on host tensors."""
from types import SimpleNamespace

import pytest
import torch

from loki_b200 import draft


class _Torch:
    """torch with the CPU as its GPU."""

    def __getattr__(self, name):
        return getattr(torch, name)

    @staticmethod
    def device(*_):
        return torch.device("cpu")


class _Ctx:
    def __init__(self, *_):
        self.calls = []

    def __getattr__(self, name):
        def call(*args, **kw):
            self.calls.append(name)
            if name == "evict":
                kw["new_lens"].clamp_(max=args[1])
            if name == "tree":
                return args[0][..., :512].clone(), torch.zeros(args[0].shape[:2])
            return kw.get("out")
        return call


@pytest.fixture()
def session(monkeypatch):
    monkeypatch.setattr(draft, "torch", _Torch())
    monkeypatch.setattr(draft, "A", SimpleNamespace(
        AttnContext=_Ctx, RopeTable=lambda max_pos, *_, **__: SimpleNamespace(max_pos=max_pos),
        KvCache=lambda rows, page, table, lens, mass, pos: SimpleNamespace(rows=rows, page_size=page, block_table=table, lens=lens, mass=mass, pos=pos)))
    return lambda **k: draft.DraftSession(**{**dict(n_seqs=2, heads=1, max_len=64, page=16, dtype=torch.float32), **k})


def _prefill(s, counts):
    s.prefill(torch.zeros(sum(counts), 512), torch.zeros(sum(counts), 64), counts)


def _verify(s, parents):
    n = sum(len(p) for p in parents)
    return s.verify(torch.zeros(n, 1, 576), torch.zeros(n, 512), torch.zeros(n, 64), parents)


def _kept(s, call, match):
    """call() is refused and leaves the session as it is, with nothing queued."""
    was = s.lens.tolist(), s.next_pos.tolist(), len(s.ctx.calls)
    with pytest.raises(ValueError, match=match):
        call()
    assert (s.lens.tolist(), s.next_pos.tolist(), len(s.ctx.calls)) == was


def test_a_long_decode_stops_at_the_tables_end(session):
    """With a budget the cache never fills, and positions grow until the table has no more of them."""
    s = session(budget=32, max_positions=100)
    _prefill(s, [41, 30])
    done = 41
    while done + 3 <= 100:
        _verify(s, [[-1, 0, 1, 0], [-1]])
        s.accept([[0, 1, 2], []])
        done += 3
        assert s.next_pos.tolist() == [done, 30] and s.lens.tolist()[0] == 32
    _kept(s, lambda: _verify(s, [[-1, 0, 1, 0], [-1]]), "position")
    _verify(s, [[-1] * 4, [-1]])                                          # as many nodes, but no deeper than the table
    s.accept([[3], [0]])
    assert s.next_pos.tolist() == [done + 1, 31]
    _kept(s, lambda: _prefill(s, [0, 70]), "position")


def test_rows_beyond_the_pages_are_refused(session):
    """max_len 64 in pages of 16, with room for one tree more: 128 rows a sequence."""
    s = session(budget=None, max_positions=10_000)
    _kept(s, lambda: _prefill(s, [10, 129]), "rows")
    _prefill(s, [10, 126])
    _kept(s, lambda: _verify(s, [[-1], [-1, 0, 1]]), "rows")
    _verify(s, [[-1], [-1, 0]])
    s.accept([[0], [0, 1]])
    assert s.lens.tolist() == [11, 128]
    _kept(s, lambda: _verify(s, [[-1], [-1]]), "rows")
    _verify(s, [[-1], []])
    s.accept([[0], []])
    assert s.lens.tolist() == [12, 128]


def test_a_budget_makes_room(session):
    s = session(budget=100, max_positions=10_000)
    _prefill(s, [128, 1])
    _kept(s, lambda: _verify(s, [[-1], [-1]]), "rows")
    _verify(s, [[], [-1]])
    s.accept([[], [0]])
    assert s.lens.tolist() == [100, 2]
    _verify(s, [list(range(-1, 27)), [-1]])
    s.accept([list(range(28)), [0]])
    assert s.lens.tolist() == [100, 3] and s.next_pos.tolist() == [156, 3]


def test_paths_that_are_no_branches_are_refused(session):
    """A refused accept() changes nothing, and the verified trees can still be accepted."""
    s = session(budget=None)
    _prefill(s, [3, 5])
    with pytest.raises(ValueError, match="verify"):
        s.accept([[], []])
    _verify(s, [[-1, 0, 0, 2], [-1, -1]])
    s.cache.rows[:, 0] = torch.arange(s.cache.rows.shape[0])
    rows, mass = s.cache.rows.clone(), s.cache.mass.clone()
    for paths in ([[0, 2]], [[0, 2], [], []], [[0, 3], []], [[2, 3], []], [[0, 1, 2], []], [[2, 0], []], [[0, 0], []], [[0], [0, 1]], [[4], []], [[-1], []]):
        _kept(s, lambda: s.accept(paths), "paths")
        assert torch.equal(s.cache.rows, rows) and torch.equal(s.cache.mass, mass)
    s.accept([[0, 2, 3], [1]])
    assert s.lens.tolist() == [6, 6] and s.next_pos.tolist() == [6, 6]
    at = s.slots(torch.tensor([0, 0, 0, 1]), torch.tensor([3, 4, 5, 5]))
    assert s.cache.rows[at, 0].tolist() == [rows[i, 0].item() for i in s.slots(torch.tensor([0, 0, 0, 1]), torch.tensor([3, 5, 6, 6]))]
    with pytest.raises(ValueError, match="verify"):
        s.accept([[], []])


def test_a_refused_verify_leaves_its_query_unrotated(session):
    """What does not fit the trees is refused before q is rotated in place."""
    s = session()
    _prefill(s, [3, 5])
    good = dict(q=torch.zeros(3, 1, 576), latent=torch.zeros(3, 512), k_rope=torch.zeros(3, 64), parents=[[-1, 0], [-1]])
    for bad in (dict(q=torch.zeros(2, 1, 576)), dict(q=torch.zeros(3, 1, 512)), dict(q=torch.zeros(3, 1, 576).half()), dict(q=torch.zeros(3, 576))):
        _kept(s, lambda: s.verify(**{**good, **bad}), "q")

    def refuse(*_, **__):
        raise ValueError("latent")
    s.ctx.append = refuse
    _kept(s, lambda: s.verify(**good), "latent")
    del s.ctx.append
    s.verify(**good)
    assert s.ctx.calls[-3:] == ["append", "rope", "tree"]


def test_prompts_drop_the_trees_whose_place_they_take(session):
    s = session()
    _verify(s, [[-1, 0], [-1]])
    _prefill(s, [3, 0])
    with pytest.raises(ValueError, match="verify"):
        s.accept([[0], [0]])
    assert s.lens.tolist() == [3, 0]
