"""Latent-cache attention operators on the GPU against plain 64-bit forms (tests/attn_ref.py): rotary positions and their
transpose, the append, drafted-tree attention, attention mass, eviction, and what each refuses."""
import math

import numpy as np
import pytest
import torch

from tests import attn_ref as R

pytestmark = pytest.mark.gpu

YARN = dict(base=10000.0, factor=40.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0)


@pytest.fixture(scope="module")
def A(native):
    from loki_b200 import attention
    return attention


@pytest.fixture(scope="module")
def ctx(A):
    c = A.AttnContext(0, max_seqs=64, max_tokens=2048)
    yield c
    c.close()


# ---------------------------------------------------------------- rope
def _rope_tol(x, y, u, off, rot, mscale):
    """Two 32-bit products of a 32-bit table entry (4 roundings of the pair's terms), then one rounding to the type."""
    pair = np.abs(x[..., off:off + rot])
    pair = np.maximum(pair, 1e-30).max(-1, keepdims=True) * 2
    t = np.full(x.shape, 0.0)
    t[..., off:off + rot] = 4 * 2.0 ** -24 * mscale * pair + u * np.abs(y[..., off:off + rot])
    return t + 2.0 ** -25 * (u > 2.0 ** -20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("T,H,off,rot,rest", [(1, 1, 0, 2, 0), (3, 5, 3, 6, 1), (8, 128, 128, 64, 0), (7, 4, 0, 32, 32), (65, 3, 64, 128, 0)])
@pytest.mark.parametrize("grad", [False, True])
def test_rope(A, ctx, dtype, layout, T, H, off, rot, rest, grad):
    ms = 1.37
    g = torch.Generator().manual_seed(T * 1000 + rot)
    x = torch.randn(T, H, off + rot + rest, generator=g).to(dtype)
    pos = torch.randint(0, 100000, (T,), generator=g, dtype=torch.int32)
    table = A.RopeTable(100000, rot, mscale=ms, device="cuda", **YARN)
    y = ctx.rope(x.cuda(), pos.cuda(), table, rot_offset=off, layout=layout, grad=grad)
    xn = x.double().numpy()
    want = R.rope(xn, pos.numpy(), R.freqs(rot, **YARN), off, layout, grad, ms)
    assert (np.abs(y.cpu().double().numpy() - want) <= _rope_tol(xn, want, R.U[dtype] if dtype != torch.float32 else 0, off, rot, ms)).all()
    ctx.device_error()


def test_rope_table_far_positions(A):
    """The entry for position p is cos/sin of the 64-bit angle rounded once."""
    t = A.RopeTable(163840, 64, device="cuda", mscale=1.25, **YARN).table.cpu().double().numpy()
    p = np.array([0, 1, 4095, 4096, 99999, 163839])
    a = p[:, None] * R.freqs(64, **YARN)[None, :]
    assert np.abs(t[p, :, 0] - 1.25 * np.cos(a)).max() <= 1.25 * 2.0 ** -24 + 1e-9
    assert np.abs(t[p, :, 1] - 1.25 * np.sin(a)).max() <= 1.25 * 2.0 ** -24 + 1e-9
    plain = A.RopeTable(50, 8, device="cuda").table.cpu().double().numpy()
    assert np.abs(plain[:, :, 1] - np.sin(np.arange(50)[:, None] * R.freqs(8)[None, :])).max() <= 2.0 ** -24 + 1e-9


def test_rope_in_place_and_strided(A, ctx):
    g = torch.Generator().manual_seed(5)
    table = A.RopeTable(512, 64, device="cuda")
    pos = torch.arange(100, 109, dtype=torch.int32, device="cuda")
    big = torch.randn(6, 9, 200, generator=g).cuda()                     # head-major storage
    x = big[:, :, :192].transpose(0, 1)
    want = ctx.rope(x.contiguous(), pos, table, rot_offset=128)
    assert torch.equal(ctx.rope(x, pos, table, rot_offset=128), want)
    tail = big[:, :, 192:].clone()
    ctx.rope(x, pos, table, rot_offset=128, out=x)
    assert torch.equal(x, want) and torch.equal(big[:, :, 192:], tail)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_gradient_is_the_transpose_and_matches_differences(A, ctx, layout):
    """<rope(x), g> = <x, rope_grad(g)>, and rope_grad(g) is the difference quotient of <rope(x), g> (the map is linear)."""
    gen = torch.Generator().manual_seed(9)
    table = A.RopeTable(5000, 64, mscale=1.2, device="cuda", **YARN)
    pos = torch.randint(0, 5000, (4,), generator=gen, dtype=torch.int32).cuda()
    x, g = torch.randn(4, 3, 96, generator=gen).cuda(), torch.randn(4, 3, 96, generator=gen).cuda()
    y = ctx.rope(x, pos, table, rot_offset=32, layout=layout)
    gx = ctx.rope(g, pos, table, rot_offset=32, layout=layout, grad=True)
    a, b = (y.double() * g.double()).sum(), (x.double() * gx.double()).sum()
    n = x.numel()
    assert abs(float(a - b)) <= 16 * 2.0 ** -24 * 1.2 * n                # 4 roundings a side of O(1) terms, |x|, |g| < 2 rms
    for at in [(0, 0, 3), (1, 2, 40), (3, 1, 95)]:                       # untouched, rotated, rotated
        e = torch.zeros_like(x)
        e[at] = 1.0
        d = ((ctx.rope(x + e, pos, table, rot_offset=32, layout=layout).double() - y.double()) * g.double()).sum()
        assert abs(float(d) - float(gx[at])) <= 32 * 2.0 ** -24 * 1.2 * 8


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("f32_in", [False, True])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("lens,new,page,stride", [([0], [1], 16, 576), ([15, 0, 33], [2, 40, 0], 16, 584), ([250, 7], [13, 64], 256, 640)])
def test_append(A, ctx, dtype, f32_in, layout, lens, new, page, stride):
    pg = R.Paged(lens, new, page, dtype, "cuda", row_stride=stride)
    T = sum(new)
    g = torch.Generator().manual_seed(3)
    it = torch.float32 if f32_in else dtype
    wide = torch.randn(T, 600, generator=g).to(it).cuda()
    latent, kr = wide[:, :512], wide[:, 512:576]                         # row stride 600
    pos = torch.randint(0, 30000, (T,), generator=g, dtype=torch.int32)
    table = A.RopeTable(30000, 64, mscale=1.1, device="cuda", **YARN)
    mass, p = torch.full((pg.n_slots,), 7.0, device="cuda"), torch.full((pg.n_slots,), -1, dtype=torch.int32, device="cuda")
    before = pg.rows.clone()
    ctx.append(pg.cache(A, mass, p), latent, kr, pg.starts, pos.cuda(), table, layout=layout)
    ctx.device_error()
    at = torch.cat([s[l:] for s, l in zip(pg.slots, lens)])
    assert torch.equal(pg.rows[at.cuda(), :512], latent.to(dtype))
    x = kr.cpu().double().numpy()[:, None, :]
    want = R.rope(x, pos.numpy(), R.freqs(64, **YARN), 0, layout, False, 1.1)
    got = pg.rows.cpu()[at][:, 512:].double().numpy()[:, None, :]
    assert (np.abs(got - want) <= _rope_tol(x, want, R.U[dtype], 0, 64, 1.1)).all()
    assert torch.equal(p.cpu()[at], pos) and (mass.cpu()[at] == 0).all()
    rest = torch.ones(pg.n_slots, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(pg.rows.cpu()[rest].view(torch.int16), before.cpu()[rest].view(torch.int16))
    assert (mass.cpu()[rest] == 7).all() and (p.cpu()[rest] == -1).all()


# ---------------------------------------------------------------- tree attention
def _q(pg, H, seed=1, std=1.0):
    return (torch.randn(sum(pg.new), H, R.ROW, generator=torch.Generator().manual_seed(seed)) * std).to(pg.dtype)


def _check_tree(A, ctx, pg, q, masks, scale, words=True):
    out, lse = ctx.tree(q.cuda(), pg.cache(A), pg.starts, R.to_words(masks, "cuda") if words else None, scale)
    ctx.device_error()
    want, wl, tol, ltol = R.tree(pg, q, masks, scale)
    got, gl = out.cpu().double(), lse.cpu().double()
    assert torch.equal(torch.isinf(gl), torch.isinf(wl))
    fin = torch.isfinite(wl)
    assert ((gl - wl).abs()[fin] <= ltol[fin]).all(), float(((gl - wl).abs()[fin] / ltol[fin]).max())
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol.clamp(min=1e-30)).max())
    return out, lse


SCALE = 192 ** -0.5


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H", [1, 3, 20, 64, 128])
@pytest.mark.parametrize("lens,new,page", [([0], [1], 16), ([1], [1], 16), ([77], [1], 32), ([127], [1], 64), ([128], [2], 64), ([129], [5], 128),
                                           ([1000], [8], 256), ([0, 63, 300], [3, 1, 17], 16)])
def test_tree(A, ctx, dtype, H, lens, new, page):
    pg = R.Paged(lens, new, page, dtype, "cuda", seed=H)
    _check_tree(A, ctx, pg, _q(pg, H), R.tree_masks(new, H), SCALE)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tree_widest_and_ragged_batch(A, ctx, dtype):
    lens, new = [0, 5, 64, 191, 700, 33, 0, 256], [64, 1, 63, 2, 7, 0, 1, 33]
    pg = R.Paged(lens, new, 32, dtype, "cuda", seed=2, row_stride=600)
    _check_tree(A, ctx, pg, _q(pg, 12), R.tree_masks(new, 2), SCALE)


def test_tree_long_context_splits(A, ctx):
    pg = R.Paged([9000, 40], [2, 3], 64, torch.bfloat16, "cuda", seed=4)
    _check_tree(A, ctx, pg, _q(pg, 16), R.tree_masks([2, 3], 1), SCALE)


def test_chain_without_words(A, ctx):
    pg = R.Paged([50, 0], [64, 3], 16, torch.bfloat16, "cuda", seed=6)
    _check_tree(A, ctx, pg, _q(pg, 8), R.chain_masks([64, 3]), SCALE, words=False)


def test_rows_that_see_nothing(A, ctx):
    """No context and an empty mask: output 0 and lse -inf, beside rows that see something."""
    pg = R.Paged([0, 0, 10], [3, 1, 2], 16, torch.float16, "cuda", seed=7)
    masks = [0, 0b010, 0b111, 0, 0, 0b11]
    out, lse = _check_tree(A, ctx, pg, _q(pg, 5), masks, SCALE)
    assert (out[0] == 0).all() and (out[3] == 0).all() and torch.isinf(lse[0]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_unseen_rows_never_reach_the_output(A, ctx, dtype, bad):
    """A drafted row of NaN or infinity changes nothing for tokens that do not see it (unused pool rows are NaN anyway)."""
    pg = R.Paged([130], [6], 64, dtype, "cuda", seed=8)
    masks = [0b1, 0b11, 0b100, 0b1001, 0b10100, 0b100100]
    pg.set_row(0, 130 + 1, bad)                     # node 1: seen by itself alone
    q = _q(pg, 9)
    out, lse = ctx.tree(q.cuda(), pg.cache(A), pg.starts, R.to_words(masks, "cuda"), SCALE)
    want, wl, tol, ltol = R.tree(pg, q, masks, SCALE)
    for t in (0, 2, 3, 4, 5):
        assert ((out[t].cpu().double() - want[t]).abs() <= tol[t]).all()
        assert ((lse[t].cpu().double() - wl[t]).abs() <= ltol[t]).all()
    if math.isnan(bad):
        assert out[1].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_growing_maxima_and_large_scores(A, ctx, dtype):
    """Scores that grow along the cache rescale the running sums again and again; a scale that makes one row win all."""
    pg = R.Paged([600], [4], 64, dtype, "cuda", seed=9, spread=0.5)
    q = _q(pg, 6, std=0.5)
    ramp = torch.linspace(0, 6, 604)
    for i in range(604):
        pg.set_row(0, i, (pg.seq[0][i].float() + ramp[i] * q[0, 0].float()).to(dtype))
    masks = R.tree_masks([4], 3)
    _check_tree(A, ctx, pg, q, masks, SCALE)
    _check_tree(A, ctx, pg, q, masks, 4.0 * SCALE)
    for i in range(604):
        pg.set_row(0, i, (pg.seq[0][i].float() - 2 * ramp[i] * q[0, 0].float()).to(dtype))      # falling, all far below 0
    _check_tree(A, ctx, pg, q, masks, SCALE)


def test_tree_strides_streams_and_repeats(A, ctx):
    """Head-major q and out, another stream, and bit-equal repeats."""
    pg = R.Paged([333, 20], [5, 2], 32, torch.bfloat16, "cuda", seed=11)
    q = _q(pg, 20)
    words = R.to_words(R.tree_masks([5, 2], 4), "cuda")
    out, lse = ctx.tree(q.cuda(), pg.cache(A), pg.starts, words, SCALE)
    buf = torch.empty(20, 7, 584, dtype=torch.bfloat16, device="cuda")
    buf[:, :, :576] = q.cuda().transpose(0, 1)
    o2 = torch.empty(20, 7, 520, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _, l2 = ctx.tree(buf[:, :, :576].transpose(0, 1), pg.cache(A), pg.starts, words, SCALE, out=o2[:, :, :512].transpose(0, 1))
    s.synchronize()
    assert torch.equal(o2[:, :, :512].transpose(0, 1), out) and torch.equal(l2, lse)


def test_tree_in_a_graph(A, ctx):
    """A captured call replays on new contents, lengths included."""
    pg = R.Paged([200], [3], 64, torch.bfloat16, "cuda", seed=12)
    q = _q(pg, 8)
    qd, words, cache = q.cuda(), R.to_words(R.tree_masks([3], 1), "cuda"), pg.cache(A)
    out, lse = ctx.tree(qd, cache, pg.starts, words, SCALE)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.tree(qd, cache, pg.starts, words, SCALE, out=out, lse=lse)
    for n in (200, 64, 0):
        cache.lens.fill_(n)
        g.replay()
        torch.cuda.synchronize()
        o2, l2 = ctx.tree(qd, cache, pg.starts, words, SCALE)
        assert torch.equal(out, o2) and torch.equal(lse, l2)


def test_offsets_beyond_32_bits(A, ctx):
    """Pages at the far end of a pool of more than 2^32 bytes (and 2^32 / 2 elements)."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB free")
    page, n_pages = 256, 16000                       # 4.7 GB
    pg = R.Paged([500], [2], page, torch.bfloat16, "cuda", seed=13)
    pool = torch.full((n_pages * page, R.ROW), float("nan"), dtype=torch.bfloat16, device="cuda")
    ids = [n_pages - 1, 9, n_pages - 3]
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    at = torch.tensor([ids[i // page] * page + i % page for i in range(502)], device="cuda")
    pool[at] = pg.seq[0].cuda()
    mass = torch.rand(n_pages * page, device="cuda")
    mass0 = mass.clone()
    cache = A.KvCache(pool, page, table, torch.tensor([500], dtype=torch.int32, device="cuda"), mass=mass,
                      pos=torch.arange(n_pages * page, dtype=torch.int32, device="cuda"))
    q, masks = _q(pg, 7), R.tree_masks([2], 5)
    words = R.to_words(masks, "cuda")
    out, lse = ctx.tree(q.cuda(), cache, pg.starts, words, SCALE)
    want, wl, tol, ltol = R.tree(pg, q, masks, SCALE)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    ctx.mass(q.cuda(), lse, cache, pg.starts, words, SCALE)
    pg2_mass0 = torch.zeros(pg.n_slots)
    pg2_mass0[pg.slots[0]] = mass0[at].cpu()
    wm, mt = R.mass(pg, q, lse.cpu(), masks, SCALE, torch.ones(2), 1.0, pg2_mass0)
    assert ((mass[at].cpu().double() - wm[pg.slots[0]]).abs() <= mt[pg.slots[0]]).all()
    m = mass.cpu().numpy().copy()
    far = torch.full((1,), 1 << 30, dtype=torch.int32, device="cuda")
    ctx.evict(cache, 300, far)
    ctx.device_error()
    _, moves = R.evict([500], [at.tolist()], m, np.arange(n_pages * page), 300, 0, 0, [1 << 30])
    where = {s: i for i, s in enumerate(at.tolist())}
    want = pg.seq[0].clone()
    for s, d in moves:
        want[where[d]] = pg.seq[0][where[s]]
    assert len(moves) > 50 and torch.equal(pool[at].cpu(), want)


# ---------------------------------------------------------------- mass
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H", [1, 20, 128])
@pytest.mark.parametrize("lens,new,page,decay", [([0], [1], 16, 1.0), ([77], [1], 32, 0.5), ([128, 1], [8, 2], 64, 0.95), ([300, 0, 513], [17, 4, 64], 16, 0.0),
                                                 ([255, 40], [3, 0], 256, 1.0)])
def test_mass(A, ctx, dtype, H, lens, new, page, decay):
    pg = R.Paged(lens, new, page, dtype, "cuda", seed=H + 1)
    q, masks = _q(pg, H), R.tree_masks(new, H)
    _, lse, _, _ = R.tree(pg, q, masks, SCALE)
    lse = lse.float()
    w = (torch.rand(sum(new), generator=torch.Generator().manual_seed(5)) < 0.6).float() * 1.5
    m0 = torch.rand(pg.n_slots, generator=torch.Generator().manual_seed(6))
    m = m0.cuda()
    cache = pg.cache(A, mass=m)
    ctx.mass(q.cuda(), lse.cuda(), cache, pg.starts, R.to_words(masks, "cuda"), SCALE, weight=w.cuda(), decay=decay)
    ctx.device_error()
    want, tol = R.mass(pg, q, lse, masks, SCALE, w, decay, m0)
    got = m.cpu().double()
    assert ((got - want).abs() <= tol + 1e-30).all(), float(((got - want).abs() / (tol + 1e-30)).max())


def test_mass_of_tree_sums_to_the_rows(A, ctx):
    """Every (token, head) row gives weight 1 in all; rows beyond the length and unseen NaN drafts add nothing; repeats
    are bit-equal; a row that sees nothing (lse = -inf) adds nothing."""
    pg = R.Paged([400, 0], [5, 2], 64, torch.bfloat16, "cuda", seed=21)
    masks = [0b1, 0b11, 0b101, 0b1001, 0b1, 0, 0b10]
    pg.set_row(0, 404, float("nan"))                 # node 4: seen by nobody
    q = _q(pg, 32).cuda()
    words = R.to_words(masks, "cuda")
    m = torch.zeros(pg.n_slots, device="cuda")
    cache = pg.cache(A, mass=m)
    _, lse = ctx.tree(q, cache, pg.starts, words, SCALE)
    ctx.mass(q, lse, cache, pg.starts, words, SCALE)
    assert torch.isfinite(m).all()
    assert abs(float(m[pg.slots[0].cuda()].double().sum()) - 5 * 32) <= 5 * 32 * 1e-4
    assert abs(float(m[pg.slots[1].cuda()].double().sum()) - 32) <= 32 * 1e-4
    again = torch.zeros_like(m)
    ctx.mass(q, lse, pg.cache(A, mass=again), pg.starts, words, SCALE)
    assert torch.equal(m, again)


def test_mass_weights_and_shared_key_tiles(A, ctx):
    """Few key tiles and many rows, so that several CTA pairs share a tile; weights that are zero, negative or NaN take their
    token out; a sequence whose tokens are all out only decays; calls of other shapes between leave the repeats' bits alone."""
    pg = R.Paged([700, 300, 500, 90], [40, 3, 0, 5], 64, torch.bfloat16, "cuda", seed=31)
    H, new = 40, [40, 3, 0, 5]
    q, masks = _q(pg, H), R.tree_masks(new, 9)
    _, lse, _, _ = R.tree(pg, q, masks, SCALE)
    lse = lse.float()
    w = torch.rand(48, generator=torch.Generator().manual_seed(8)) * 2
    w[torch.arange(1, 40, 4)] = torch.tensor([0.0, -1.0, float("nan"), 0.0, -0.0, float("-inf"), 0.0, 0.0, -3.0, 0.0])
    w[40:43] = 0.0
    m0 = torch.rand(pg.n_slots, generator=torch.Generator().manual_seed(6))
    words, other = R.to_words(masks, "cuda"), R.Paged([1000], [2], 16, torch.bfloat16, "cuda", seed=2)
    qo, mo = _q(other, 16).cuda(), torch.zeros(other.n_slots, device="cuda")
    runs = []
    for _ in range(20):
        m = m0.cuda()
        ctx.mass(q.cuda(), lse.cuda(), pg.cache(A, mass=m), pg.starts, words, SCALE, weight=w.cuda(), decay=0.5)
        ctx.mass(qo, torch.zeros(2, 16, device="cuda"), other.cache(A, mass=mo), other.starts, None, 1e-3)
        runs.append(m)
    ctx.device_error()
    want, tol = R.mass(pg, q, lse, masks, SCALE, torch.where(w > 0, w, torch.zeros(())), 0.5, m0)
    assert ((runs[0].cpu().double() - want).abs() <= tol + 1e-30).all()
    assert all(torch.equal(m, runs[0]) for m in runs)


def test_many_sequences(A):
    """More sequences than a warp has lanes and than a launch has CTA pairs: attention and mass."""
    g = torch.Generator().manual_seed(3)
    n = 230
    lens, new = torch.randint(0, 300, (n,), generator=g).tolist(), torch.randint(0, 4, (n,), generator=g).tolist()
    H, T = 8, sum(new)
    many = A.AttnContext(0, n, T)
    pg = R.Paged(lens, new, 16, torch.bfloat16, "cuda", seed=41)
    q, masks = _q(pg, H), R.tree_masks(new, 5)
    words = R.to_words(masks, "cuda")
    m0 = torch.rand(pg.n_slots, generator=g)
    m = m0.cuda()
    cache = pg.cache(A, mass=m)
    out, lse = many.tree(q.cuda(), cache, pg.starts, words, SCALE)
    w = torch.rand(T, generator=g) * (torch.rand(T, generator=g) < 0.7)
    many.mass(q.cuda(), lse, cache, pg.starts, words, SCALE, weight=w.cuda(), decay=0.25)
    many.device_error()
    want, wl, tol, ltol = R.tree(pg, q, masks, SCALE)
    assert ((out.cpu().double() - want).abs() <= tol).all() and ((lse.cpu().double() - wl).abs() <= ltol).all()
    wm, mt = R.mass(pg, q, lse.cpu(), masks, SCALE, w, 0.25, m0)
    assert ((m.cpu().double() - wm).abs() <= mt + 1e-30).all()
    many.close()


# ---------------------------------------------------------------- eviction
def _evict_case(lens, page, seed, ties=False):
    pg = R.Paged(lens, [0] * len(lens), page, torch.bfloat16, "cuda", seed=seed)
    g = torch.Generator().manual_seed(seed)
    mass = torch.rand(pg.n_slots, generator=g)
    if ties:
        mass = (mass * 4).floor() / 4 * torch.where(torch.rand(pg.n_slots, generator=g) < 0.5, 1.0, -1.0)      # -0 and 0 among them
    pos = torch.full((pg.n_slots,), -7, dtype=torch.int32)
    for s in pg.slots:
        pos[s] = torch.randperm(len(s), generator=g).int()
    return pg, mass, pos


@pytest.mark.parametrize("lens,page,budget,sinks,recent,ties", [
    ([1], 16, 1, 0, 0, False), ([2], 16, 1, 0, 0, False), ([100, 40, 300], 16, 64, 4, 8, False), ([1025, 1024, 5000], 64, 1024, 4, 128, True),
    ([700], 256, 100, 0, 0, True), ([300, 0, 299], 32, 50, 60, 60, False), ([5000], 64, 4999, 0, 0, False), ([5000], 64, 1, 0, 0, True)])
def test_evict(A, ctx, lens, page, budget, sinks, recent, ties):
    pg, mass, pos = _evict_case(lens, page, budget, ties)
    nxt = torch.tensor(lens, dtype=torch.int32)
    md, pd = mass.cuda(), pos.cuda()
    rows0 = pg.rows.clone()
    new = ctx.evict(pg.cache(A, mass=md, pos=pd), budget, nxt.cuda(), sinks=sinks, recent=recent)
    ctx.device_error()
    want, moves = R.evict(lens, pg.slots, mass.numpy(), pos.numpy(), budget, sinks, recent, nxt.tolist())
    assert new.tolist() == want
    rows, m, p = rows0.clone(), mass.clone(), pos.clone()
    for s, d in moves:
        rows[d], m[d], p[d] = rows0[s], mass[s], pos[s]
    assert torch.equal(pg.rows.view(torch.int16), rows.view(torch.int16)) and torch.equal(md.cpu(), m) and torch.equal(pd.cpu(), p)


def test_evict_nan_and_infinite_mass_and_lens_in_place(A, ctx):
    pg, mass, pos = _evict_case([200], 16, 3)
    at = pg.slots[0]
    mass[at[:50]] = float("nan")
    mass[at[150:170]] = float("inf")
    nxt = torch.tensor([200], dtype=torch.int32)
    md, pd = mass.cuda(), pos.cuda()
    cache = pg.cache(A, mass=md, pos=pd)
    new = ctx.evict(cache, 160, nxt.cuda(), sinks=2, recent=2, new_lens=cache.lens)
    want, moves = R.evict([200], pg.slots, mass.numpy(), pos.numpy(), 160, 2, 2, [200])
    assert new is cache.lens and cache.lens.tolist() == want
    m = mass.clone()
    for s, d in moves:
        m[d] = mass[s]
    assert torch.equal(md.cpu().view(torch.int32), m.view(torch.int32))


def test_evicted_cache_attends_as_the_kept_rows(A, ctx):
    """The step that a serving loop takes: append, attend, add the weights, evict, attend again over what is left."""
    pg = R.Paged([512], [1], 64, torch.bfloat16, "cuda", seed=31)
    mass, pos = torch.zeros(pg.n_slots, device="cuda"), torch.zeros(pg.n_slots, dtype=torch.int32, device="cuda")
    pos[pg.slots[0].cuda()] = torch.arange(513, dtype=torch.int32, device="cuda")
    cache = pg.cache(A, mass=mass, pos=pos)
    q = _q(pg, 16)
    words = torch.ones(1, dtype=torch.int64, device="cuda")
    _, lse = ctx.tree(q.cuda(), cache, pg.starts, words, SCALE)
    ctx.mass(q.cuda(), lse, cache, pg.starts, words, SCALE)
    m = mass.cpu()
    new, moves = R.evict([512], pg.slots, m.numpy(), pos.cpu().numpy(), 300, 4, 16, [513])
    last = pg.rows[pg.slots[0][512].item()].clone()
    ctx.evict(cache, 300, torch.tensor([513], dtype=torch.int32, device="cuda"), sinks=4, recent=16, new_lens=cache.lens)
    assert cache.lens.tolist() == new
    pg.rows[pg.slots[0][300].item()] = last                             # the drafted row follows the new length
    out, _ = ctx.tree(q.cuda(), cache, pg.starts, words, SCALE)
    kept = R.Paged([300], [1], 64, torch.bfloat16, "cpu", seed=0)
    kept.seq[0] = pg.rows.cpu()[pg.slots[0][:301]]
    want, _, tol, _ = R.tree(kept, q, [1], SCALE)
    assert ((out.cpu().double() - want).abs() <= tol).all()


# ---------------------------------------------------------------- refusals
def test_refused_arguments(A, ctx, native):
    pg = R.Paged([20], [2], 16, torch.bfloat16, "cuda")
    cache, q = pg.cache(A), _q(pg, 4).cuda()
    words = R.to_words([1, 3], "cuda")
    call = lambda **k: ctx.tree(**{**dict(q=q, cache=cache, starts=pg.starts, tree=words, scale=SCALE), **k})
    with pytest.raises(ValueError):
        call(q=q.half())
    with pytest.raises(ValueError):
        call(q=q[..., :512])
    with pytest.raises(ValueError):
        call(starts=pg.starts.long())
    with pytest.raises(ValueError):
        call(tree=words[:1])
    with pytest.raises(native.NativeError):
        call(scale=0.0)
    with pytest.raises(native.NativeError):
        call(scale=float("nan"))
    with pytest.raises(native.NativeError):
        call(q=_q(pg, 129).cuda())
    odd = torch.zeros(2 * 4 * 580 + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(native.NativeError):
        call(q=odd.as_strided((2, 4, 576), (4 * 580, 580, 1)))                       # stride no multiple of 8
    with pytest.raises(native.NativeError):
        call(q=odd.as_strided((2, 4, 576), (4 * 576, 576, 1), 1))                    # not 16-byte aligned
    small = A.AttnContext(0, max_seqs=1, max_tokens=1)
    with pytest.raises(native.NativeError):
        small.tree(q, cache, pg.starts, words, SCALE)
    with pytest.raises(native.NativeError):
        ctx.mass(q, torch.zeros(2, 4, device="cuda"), cache, pg.starts, words, SCALE)      # no mass array
    m = torch.zeros(pg.n_slots, device="cuda")
    with pytest.raises(native.NativeError):
        ctx.mass(q, torch.zeros(2, 4, device="cuda"), pg.cache(A, mass=m), pg.starts, words, SCALE, decay=1.5)
    with pytest.raises(native.NativeError):
        ctx.evict(pg.cache(A, mass=m), 4, torch.zeros(1, dtype=torch.int32, device="cuda"))      # no pos array
    full = pg.cache(A, mass=m, pos=torch.zeros(pg.n_slots, dtype=torch.int32, device="cuda"))
    with pytest.raises(native.NativeError):
        ctx.evict(full, 0, torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(native.NativeError):
        A.RopeTable(0, 64, device="cuda")
    with pytest.raises(native.NativeError):
        A.RopeTable(16, 63, device="cuda")
    with pytest.raises(native.NativeError):
        A.RopeTable(16, 64, factor=0.5, device="cuda")
    t = A.RopeTable(16, 64, device="cuda")
    with pytest.raises(native.NativeError):
        ctx.rope(torch.zeros(1, 1, 64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), t, rot_offset=8)
    with pytest.raises(ValueError):
        A.KvCache(torch.zeros(24, 576, dtype=torch.bfloat16, device="cuda"), 16, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                  torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(native.NativeError):
        ctx.tree(q, A.KvCache(torch.zeros(48, 576, dtype=torch.bfloat16, device="cuda"), 24, torch.zeros(1, 2, dtype=torch.int32, device="cuda"),
                              torch.zeros(1, dtype=torch.int32, device="cuda")), pg.starts, words, SCALE)


@pytest.mark.parametrize("what", ["page", "len", "start", "nodes", "pos"])
def test_refused_contents_are_reported_and_stay_in_bounds(A, ctx, native, what):
    """Bad device values are clamped or skipped by the kernels' own checks and reported by device_error()."""
    pg = R.Paged([40], [2], 16, torch.bfloat16, "cuda")
    mass, pos = torch.zeros(pg.n_slots, device="cuda"), torch.zeros(pg.n_slots, dtype=torch.int32, device="cuda")
    cache, starts = pg.cache(A, mass, pos), pg.starts
    q, words = _q(pg, 4).cuda(), R.to_words([1, 3], "cuda")
    if what == "page":
        cache.block_table[0, 1] = 1 << 20
    elif what == "len":
        cache.lens.fill_(1 << 20)
    elif what == "start":
        starts = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    elif what == "nodes":
        q, starts = torch.zeros(70, 4, 576, dtype=torch.bfloat16, device="cuda"), torch.tensor([0, 70], dtype=torch.int32, device="cuda")
        words = torch.zeros(70, dtype=torch.int64, device="cuda")
    if what == "pos":
        ctx.rope(torch.zeros(1, 1, 64, device="cuda"), torch.tensor([16], dtype=torch.int32, device="cuda"), A.RopeTable(16, 64, device="cuda"))
        with pytest.raises(native.NativeError):
            ctx.device_error()
        return
    _, lse = ctx.tree(q, cache, starts, words, SCALE)
    with pytest.raises(native.NativeError):
        ctx.device_error()
    ctx.mass(q, torch.zeros_like(lse), cache, starts, words, SCALE)
    with pytest.raises(native.NativeError):
        ctx.device_error()
    ctx.device_error()                               # cleared


def test_no_tokens(A, ctx):
    pg = R.Paged([20], [0], 16, torch.bfloat16, "cuda")
    out, lse = ctx.tree(torch.empty(0, 4, 576, dtype=torch.bfloat16, device="cuda"), pg.cache(A), pg.starts, None, SCALE)
    assert out.shape == (0, 4, 512) and lse.shape == (0, 4)
    x = ctx.rope(torch.empty(0, 2, 64, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), A.RopeTable(4, 64, device="cuda"))
    assert x.shape == (0, 2, 64)


def test_repeated_calls_over_caches_beyond_l2(A):
    """Back-to-back calls that alternate between contexts whose caches come from memory, not L2 (the key half of a tile
    arrives long after the value half of the one before): every call gives the first one's bits."""
    H, T = 128, 1
    sets = []
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n_pages = 480
        rows = torch.randn(n_pages * 64, R.ROW, generator=g, device="cuda").to(torch.bfloat16)
        table = torch.randperm(n_pages, generator=g, device="cuda").int()[None].contiguous()
        cache = A.KvCache(rows, 64, table, torch.tensor([30011 + 100 * seed], dtype=torch.int32, device="cuda"))
        q = torch.randn(T, H, R.ROW, generator=g, device="cuda").to(torch.bfloat16)
        sets.append((A.AttnContext(0, 1, 1), cache, q, torch.tensor([0, T], dtype=torch.int32, device="cuda")))
    first = [c.tree(q, k, s, None, SCALE) for c, k, q, s in sets]
    torch.cuda.synchronize()
    got = [sets[i % 3][0].tree(sets[i % 3][2], sets[i % 3][1], sets[i % 3][3], None, SCALE) for i in range(300)]
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, first[i % 3][0]) and torch.equal(l, first[i % 3][1])
    for c, *_ in sets:
        c.device_error()
        c.close()
