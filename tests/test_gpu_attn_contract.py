"""What the latent-cache attention operators promise around their numbers: captured graphs, streams, workspaces, error
words, refused arguments, and non-finite values where they must and must not show."""
import math

import numpy as np
import pytest
import torch

from tests import attn_ref as R

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5


@pytest.fixture(scope="module")
def A(native):
    from loki_b200 import attention
    return attention


@pytest.fixture()
def ctx(A):
    c = A.AttnContext(0, max_seqs=16, max_tokens=512)
    yield c
    c.close()


def _eviction(lens, page, seed):
    """A filled pool whose rows have random masses and their index as position, and what `expect` needs of it."""
    pg = R.Paged(lens, [0] * len(lens), page, torch.bfloat16, "cuda", seed=seed)
    mass = torch.rand(pg.n_slots, generator=torch.Generator().manual_seed(seed))
    pos = torch.zeros(pg.n_slots, dtype=torch.int32)
    for s in pg.slots:
        pos[s] = torch.arange(len(s), dtype=torch.int32)
    return pg, mass, pos


def _evicted(pg, rows0, mass, pos, budget, nxt):
    """rows, mass and pos after the rule's moves; the new lengths."""
    new, moves = R.evict(pg.lens, pg.slots, mass.numpy(), pos.numpy(), budget, 2, 8, nxt)
    rows, m, p = rows0.clone(), mass.clone(), pos.clone()
    for s, d in moves:
        rows[d], m[d], p[d] = rows0[s], mass[s], pos[s]
    return rows, m, p, new, len(moves)


def test_captured_eviction_after_a_larger_call(A, ctx):
    """A graph that holds an eviction replays rightly after later calls of the context needed larger move lists."""
    pg, mass, pos = _eviction([400], 16, 1)
    md, pd, nxt = mass.cuda(), pos.cuda(), torch.tensor([400], dtype=torch.int32, device="cuda")
    cache, new = pg.cache(A, mass=md, pos=pd), torch.zeros(1, dtype=torch.int32, device="cuda")
    rows0 = pg.rows.clone()
    ctx.evict(cache, 64, nxt, sinks=2, recent=8, new_lens=new)           # makes the lists
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.evict(cache, 64, nxt, sinks=2, recent=8, new_lens=new)
    want_rows, want_m, want_p, want_new, n_moves = _evicted(pg, rows0, mass, pos, 64, [400])
    assert n_moves > 20
    held = []
    for n in (2000, 9000, 30000):                                        # lists of 8, 16 and 32 times the size and more
        big, bm, bp = _eviction([n, n - 7, 5], 64, n)
        bmd, bpd = bm.cuda(), bp.cuda()
        big_nxt = [n, n - 7, 5]
        b0 = big.rows.clone()
        got = ctx.evict(big.cache(A, mass=bmd, pos=bpd), n // 2, torch.tensor(big_nxt, dtype=torch.int32, device="cuda"), sinks=2, recent=8)
        held.append(torch.full((1 << 18,), 0x7fffffff, dtype=torch.int32, device="cuda"))      # memory that was let go is used again
        for t, v in ((pg.rows, rows0), (md, mass), (pd, pos)):
            t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        ctx.device_error()
        assert new.tolist() == want_new
        assert torch.equal(pg.rows.view(torch.int16), want_rows.view(torch.int16)) and torch.equal(md.cpu(), want_m) and torch.equal(pd.cpu(), want_p)
        w_rows, w_m, w_p, w_new, _ = _evicted(big, b0, bm, bp, n // 2, big_nxt)
        assert got.tolist() == w_new and torch.equal(big.rows.view(torch.int16), w_rows.view(torch.int16))
        assert torch.equal(bmd.cpu(), w_m) and torch.equal(bpd.cpu(), w_p)


def _long_eviction(n, budget, bad_page=None):
    """One sequence whose keys do not fit the selection's shared memory, rows coded by their place: what is left of it."""
    page, n_pages = 256, (n + 255) // 256
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    at = ids.long()[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page
    i = torch.arange(n, device="cuda")
    rows = torch.zeros(n_pages * page, R.ROW, dtype=torch.float16, device="cuda")
    rows[at, 0], rows[at, 575] = (i // 1024).half(), (i % 1024).half()
    mass, pos = torch.zeros(n_pages * page, device="cuda"), torch.zeros(n_pages * page, dtype=torch.int32, device="cuda")
    mass[at], pos[at] = (torch.rand(n, generator=g, device="cuda") * 4096).floor(), i.int()          # ties among them
    if bad_page is not None:
        ids[bad_page] = n_pages
    return rows, page, ids[None].contiguous(), mass, pos, at


@pytest.mark.parametrize("bad", [False, True])
def test_eviction_beyond_the_keys_that_fit(A, native, bad):
    """Sequences of more than 8 x 49 152 rows: the same rule, and a bad page id is reported and its rows rank last."""
    n, budget = 400_016, 150_001
    rows, page, table, mass, pos, at = _long_eviction(n, budget, 1500 if bad else None)
    ctx, m0, p0, r0 = A.AttnContext(0, 1, 1), mass.clone(), pos.clone(), rows[:, [0, 575]].clone()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    new = ctx.evict(A.KvCache(rows, page, table, lens, mass=mass, pos=pos), budget, lens.clone(), sinks=4, recent=100)
    torch.cuda.synchronize()
    i = torch.arange(n, device="cuda")
    key = m0[at].double()
    key[(i < 4) | (i >= n - 100)] = math.inf
    key[(i // page == 1500) & bad] = -1.0
    keep = torch.zeros(n, dtype=torch.bool, device="cuda")
    keep[torch.sort(key, descending=True, stable=True).indices[:budget]] = True
    dst, src = at[(i < budget) & ~keep], at[(i >= budget) & keep]
    assert len(dst) == len(src) > 50_000 and new.tolist() == [budget]
    r0[dst], m0[dst], p0[dst] = r0[src], m0[src], p0[src]
    assert torch.equal(rows[:, [0, 575]], r0) and torch.equal(mass, m0) and torch.equal(pos, p0)
    if bad:
        with pytest.raises(native.NativeError, match="page"):
            ctx.device_error()
    ctx.device_error()
    ctx.close()


@pytest.mark.parametrize("n", [100, 9000])
def test_a_seen_nan_reaches_every_output(A, ctx, n):
    """A NaN context row is seen by every token, so every row of out and lse is NaN: also where the cache is shared out in parts
    and another part's scores are so large that the NaN's part has no weight against them."""
    pg = R.Paged([n], [2], 64, torch.bfloat16, "cuda", seed=3)
    q = torch.randn(2, 4, R.ROW, generator=torch.Generator().manual_seed(1)).bfloat16()
    pg.set_row(0, 5, float("nan"))
    pg.set_row(0, n - 10, (6 * q[0, 0].float()).bfloat16())              # a score of about 250 for one (token, head)
    out, lse = ctx.tree(q.cuda(), pg.cache(A), pg.starts, R.to_words([1, 3], "cuda"), SCALE)
    ctx.device_error()
    assert lse.isnan().all() and out.isnan().all()


@pytest.mark.parametrize("H", [1, 20, 24, 128])
def test_mass_of_rows_that_a_nan_token_does_not_see(A, ctx, H):
    """A token that sees a NaN row has lse NaN, and so the rows that it sees have a NaN mass; drafted rows that it does not see
    keep the sum over the tokens that do."""
    pg = R.Paged([130], [3], 64, torch.bfloat16, "cuda", seed=4)
    pg.set_row(0, 131, float("nan"))
    q, masks = torch.randn(3, H, R.ROW, generator=torch.Generator().manual_seed(2)).bfloat16(), [0b001, 0b011, 0b101]
    words = R.to_words(masks, "cuda")
    m0 = torch.rand(pg.n_slots, generator=torch.Generator().manual_seed(3))
    m = m0.cuda()
    cache = pg.cache(A, mass=m)
    _, lse = ctx.tree(q.cuda(), cache, pg.starts, words, SCALE)
    assert lse[1].isnan().all() and not lse[0].isnan().any() and not lse[2].isnan().any()
    ctx.mass(q.cuda(), lse, cache, pg.starts, words, SCALE, decay=0.5)
    at = pg.slots[0]
    want, tol = R.mass(pg, q, lse.cpu(), masks, SCALE, torch.ones(3), 0.5, m0)
    got = m.cpu().double()
    assert got[at[:132]].isnan().all()                                   # the context, and drafted rows 0 and 1, which token 1 sees
    assert abs(got[at[132]] - want[at[132]]) <= tol[at[132]]


@pytest.mark.parametrize("H", [1, 20, 24, 128])
def test_mass_of_an_infinite_row(A, ctx, H):
    """A row whose scores are all -infinity gets no weight, whatever the number of heads."""
    pg = R.Paged([300], [2], 64, torch.bfloat16, "cuda", seed=5)
    q = torch.randn(2, H, R.ROW, generator=torch.Generator().manual_seed(2)).bfloat16()
    q[:, :, 7] = q[:, :, 7].abs() + 0.5
    row = pg.seq[0][40].clone()
    row[7] = -math.inf
    pg.set_row(0, 40, row)
    words = R.to_words([1, 3], "cuda")
    m0 = torch.rand(pg.n_slots, generator=torch.Generator().manual_seed(3))
    m = m0.cuda()
    cache = pg.cache(A, mass=m)
    _, lse = ctx.tree(q.cuda(), cache, pg.starts, words, SCALE)
    assert torch.isfinite(lse).all()
    ctx.mass(q.cuda(), lse, cache, pg.starts, words, SCALE, decay=0.5)
    at = pg.slots[0]
    assert float(m[at[40]]) == 0.5 * float(m0[at[40]])
    assert torch.isfinite(m[at.cuda()]).all()


def test_device_error_waits_for_its_stream_alone(A, ctx, native):
    """device_error(stream) reads and clears the word in the order of that stream; work on another one is not waited for."""
    s = torch.cuda.Stream()
    bad = torch.tensor([16], dtype=torch.int32, device="cuda")
    x, table = torch.zeros(1, 1, 64, device="cuda"), A.RopeTable(16, 64, device="cuda")
    out = torch.empty_like(x)

    def refused():
        ctx.rope(x, bad, table, out=out, stream=s)
        with pytest.raises(native.NativeError):
            ctx.device_error(s)
        ctx.device_error(s)
    torch.cuda.synchronize()
    refused()                                                            # what is loaded on first use is there
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)                                     # half a second on the default stream
    busy = torch.cuda.Event()
    busy.record()
    for _ in range(20):
        refused()
    assert not busy.query()
    torch.cuda.synchronize()


def test_a_failed_call_leaves_no_error_for_the_next(A, native):
    """A context for a device that is not there is refused, and that alone: the next call does not report it again."""
    with pytest.raises(native.NativeError):
        A.AttnContext(99)
    A.RopeTable(16, 64, device="cuda")
    c = A.AttnContext(0, 1, 1)
    c.device_error()
    c.close()


def test_append_behind_the_longest_table(A, ctx, native):
    """Rows that would come after 2^31 - 257 of context, the most that a table can hold, are refused like any beyond the pages."""
    page, pages = 256, 0x7fffff00 // 256
    rows = torch.zeros(2 * page, R.ROW, dtype=torch.bfloat16, device="cuda")
    lens = torch.tensor([page * pages], dtype=torch.int32, device="cuda")
    cache = A.KvCache(rows, page, torch.zeros(1, pages, dtype=torch.int32, device="cuda"), lens)
    T = 600                                                              # from the 257th on the row number passes 2^31
    starts, pos = torch.tensor([0, T], dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    table = A.RopeTable(16, 64, device="cuda")
    ctx.append(cache, torch.ones(T, 512, dtype=torch.bfloat16, device="cuda"), torch.ones(T, 64, dtype=torch.bfloat16, device="cuda"), starts, pos, table)
    with pytest.raises(native.NativeError, match="length"):
        ctx.device_error()
    assert (rows == 0).all()
    cache.lens.fill_(page + 3)                                           # and the same table with rows that it holds
    cache.block_table[0, 1] = 1
    ctx.append(cache, torch.ones(4, 512, dtype=torch.bfloat16, device="cuda"), torch.ones(4, 64, dtype=torch.bfloat16, device="cuda"),
               torch.tensor([0, 4], dtype=torch.int32, device="cuda"), pos[:4], table)
    ctx.device_error()
    assert (rows[page + 3:page + 7] == 1).all() and (rows[:page + 3] == 0).all() and (rows[page + 7:] == 0).all()


def test_rope_of_more_than_2_30_values_a_token_is_refused(A, ctx, native):
    """Heads that a stride of 0 repeats need no memory, and 65 536 of 40 000 values are more than the kernel counts."""
    x = torch.zeros(1, 1, 40000, dtype=torch.bfloat16, device="cuda").expand(1, 65536, 40000)
    out, pos = torch.zeros(1, 1, 40000, dtype=torch.bfloat16, device="cuda").expand(1, 65536, 40000), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(native.NativeError, match="40000"):
        ctx.rope(x, pos, A.RopeTable(16, 64, device="cuda"), out=out)


def _behind(make, value=7):
    """Memory of `make` given back while the current stream still has a write to it in its queue."""
    t = make()
    torch.cuda._sleep(200_000_000)                                       # a tenth of a second
    t.fill_(value)
    del t


def test_results_on_another_stream_have_memory_of_their_own(A, ctx):
    """With stream=, what a call returns is not memory that the current stream still writes to, nor given to it while the call
    runs: rope, a rope table, tree and evict against the same calls on the current stream."""
    pg = R.Paged([200, 90], [3, 1], 64, torch.bfloat16, "cuda", seed=6)
    q, words = torch.randn(4, 8, R.ROW, generator=torch.Generator().manual_seed(1)).bfloat16().cuda(), R.to_words([1, 3, 5, 1], "cuda")
    x, pos, table = q.clone(), torch.arange(4, dtype=torch.int32, device="cuda"), A.RopeTable(300, 64, device="cuda")
    mass, place = torch.rand(pg.n_slots, device="cuda"), torch.arange(pg.n_slots, dtype=torch.int32, device="cuda")
    cache, nxt = pg.cache(A, mass=mass, pos=place), torch.tensor([1 << 20, 1 << 20], dtype=torch.int32, device="cuda")
    state = [t.clone() for t in (pg.rows, mass, place)]

    def calls(stream):
        yield lambda: (ctx.rope(x, pos, table, rot_offset=512, stream=stream),)
        yield lambda: (A.RopeTable(300, 64, device="cuda", stream=stream).table,)
        yield lambda: ctx.tree(q, cache, pg.starts, words, SCALE, stream=stream)
        yield lambda: (ctx.evict(cache, 100, nxt, stream=stream), pg.rows, mass, place)

    def again():
        for t, v in zip((pg.rows, mass, place), state):
            t.copy_(v)
        torch.cuda.synchronize()
    want = []
    for call in calls(None):
        again()
        want.append([t.clone() for t in call()])
    s = torch.cuda.Stream()
    for k, call in enumerate(calls(s)):
        again()
        call()                                                           # the stream's pool has seen such a call
        again()
        shapes = [(t.shape, t.dtype) for t in want[k]]
        for shape, dt in shapes:
            _behind(lambda: torch.empty(shape, dtype=dt, device="cuda"))
        got = call()
        torch.cuda.synchronize()
        for g, w in zip(got, want[k]):
            assert torch.equal(g.view(torch.uint8), w.view(torch.uint8))
    ctx.device_error()


def test_a_dropped_result_is_not_given_away_while_its_call_runs(A, ctx):
    """The result of a call on `stream`, dropped at once, does not become a tensor of the current stream under the call."""
    x, pos, table = torch.randn(8, 16, 64, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda"), A.RopeTable(4, 64, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)
    ctx.rope(x, pos, table, stream=s)                                    # its kernel comes after the sleep
    mine = [torch.full_like(x, 3.0) for _ in range(8)]
    torch.cuda.synchronize()
    assert all((m == 3.0).all() for m in mine)


@pytest.mark.parametrize("H", [1, 3, 20, 128])
def test_mass_of_strided_queries(A, ctx, H):
    """Head-major q, heads and tokens with space between them, every other token of a longer q: the bits of a dense q."""
    lens, new = [300, 70], [5, 2]
    pg = R.Paged(lens, new, 32, torch.bfloat16, "cuda", seed=H)
    T = sum(new)
    q = torch.randn(T, H, R.ROW, generator=torch.Generator().manual_seed(H)).bfloat16().cuda()
    words = R.to_words(R.tree_masks(new, 4), "cuda")
    m = torch.rand(pg.n_slots, device="cuda")
    m0 = m.clone()
    cache = pg.cache(A, mass=m)
    _, lse = ctx.tree(q, cache, pg.starts, words, SCALE)
    ctx.mass(q, lse, cache, pg.starts, words, SCALE, decay=0.5)
    want = m.clone()
    assert not torch.equal(want, m0)
    nan = lambda *s: torch.full(s, float("nan"), dtype=torch.bfloat16, device="cuda")
    forms = {"heads first": nan(H, T, 576).transpose(0, 1), "heads first, spaced": nan(H, T, 584)[:, :, :576].transpose(0, 1),
             "spaced heads": nan(T, H, 640)[:, :, :576], "every other token": nan(2 * T, H, 576)[::2], "part of the heads": nan(T, H + 5, 576)[:, 2:H + 2]}
    for name, qs in forms.items():
        qs.copy_(q)
        m.copy_(m0)
        ctx.mass(qs, lse, cache, pg.starts, words, SCALE, decay=0.5)
        assert torch.equal(m, want), name
    ctx.device_error()


def test_repeated_queries(A, ctx, native):
    """A stride of 0: attention takes it, mass says that it does not."""
    pg = R.Paged([100], [3], 16, torch.bfloat16, "cuda", seed=1)
    m = torch.zeros(pg.n_slots, device="cuda")
    cache = pg.cache(A, mass=m)
    one = torch.randn(1, 1, R.ROW, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    for q in (one.expand(3, 6, R.ROW), one.expand(3, 1, R.ROW).contiguous().expand(3, 6, R.ROW), one.expand(1, 6, R.ROW).contiguous().expand(3, 6, R.ROW)):
        out, lse = ctx.tree(q, cache, pg.starts, None, SCALE)
        o2, l2 = ctx.tree(q.contiguous(), cache, pg.starts, None, SCALE)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
        with pytest.raises(native.NativeError, match="strides"):
            ctx.mass(q, lse, cache, pg.starts, None, SCALE)
    ctx.mass(q.contiguous(), lse, cache, pg.starts, None, SCALE)
    ctx.device_error()


def test_a_captured_step_follows_its_inputs(A, ctx):
    """Rotate, append, attend, add the weights and evict in one graph: replayed on new inputs, lengths and weights it gives the
    bits of the same calls outside a graph."""
    H, page = 8, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    table = A.RopeTable(2000, 64, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    starts, words = i32([0, 3, 5]), R.to_words([1, 3, 5, 1, 3], "cuda")

    def fresh():
        return dict(rows=torch.zeros(32 * page, R.ROW, dtype=torch.bfloat16, device="cuda"), mass=torch.zeros(32 * page, device="cuda"),
                    pos=torch.zeros(32 * page, dtype=torch.int32, device="cuda"), lens=i32([0, 0]), q=torch.zeros(5, H, R.ROW, dtype=torch.bfloat16, device="cuda"),
                    latent=torch.zeros(5, 512, dtype=torch.bfloat16, device="cuda"), k=torch.zeros(5, 64, dtype=torch.bfloat16, device="cuda"),
                    at=i32([0] * 5), w=torch.zeros(5, device="cuda"), next=i32([0, 0]), new=i32([0, 0]),
                    out=torch.zeros(5, H, 512, dtype=torch.bfloat16, device="cuda"), lse=torch.zeros(5, H, device="cuda"))

    def step(s, cache):
        ctx.rope(s["q"], s["at"], table, rot_offset=512, out=s["q"])
        ctx.append(cache, s["latent"], s["k"], starts, s["at"], table)
        ctx.tree(s["q"], cache, starts, words, SCALE, out=s["out"], lse=s["lse"])
        ctx.mass(s["q"], s["lse"], cache, starts, words, SCALE, weight=s["w"], decay=0.9)
        ctx.evict(cache, 100, s["next"], sinks=2, recent=4, new_lens=s["new"])
    block = torch.randperm(32, generator=g, device="cuda").int().view(2, 16).contiguous()
    held, plain = fresh(), fresh()
    caches = [A.KvCache(s["rows"], page, block, s["lens"], mass=s["mass"], pos=s["pos"]) for s in (held, plain)]
    step(held, caches[0])                                                # makes the workspaces
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(held, caches[0])
    for lens in ([140, 3], [0, 250], [101, 100]):
        new = dict(rows=rand(32 * page, R.ROW), mass=torch.rand(32 * page, generator=g, device="cuda"),
                   pos=torch.randint(0, 1500, (32 * page,), generator=g, device="cuda").int(), lens=i32(lens), q=rand(5, H, R.ROW),
                   latent=rand(5, 512), k=rand(5, 64), at=i32([lens[0]] * 3 + [lens[1]] * 2), w=(torch.rand(5, generator=g, device="cuda") * 2 - 0.5),
                   next=i32([l + 1000 for l in lens]))
        for s in (held, plain):
            for name, v in new.items():
                s[name].copy_(v)
        graph.replay()
        step(plain, caches[1])
        torch.cuda.synchronize()
        for name in held:
            assert torch.equal(held[name].view(torch.uint8), plain[name].view(torch.uint8)), (lens, name)
        assert plain["new"].tolist() == [min(l, 100) for l in lens]
    ctx.device_error()
