"""The paged operators on the GPU against their plain 64-bit forms
(tests/paged_ref.py): page bookkeeping exactly, rotary rows, attention and
beam selection within bounds derived beside each.  What no row sees is NaN in
every attention test."""
import numpy as np
import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def host(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy().astype(np.int64)


def new_cache(g4, ctx, kind="f32", kv=(2,), hs=(64,), page=16, pages=64, seqs=8, positions=256):
    return g4.KvCache(ctx, n_kv_heads=list(kv), head_size=list(hs), dtype=TYPES[kind][0], page_size=page, n_pages=pages,
                      n_seqs=seqs, max_positions=positions)


# ------------------------------------------------------------------ pages


def same_state(cache, sim):
    assert np.array_equal(host(cache.table), sim.table)
    assert np.array_equal(host(cache.lens), sim.lens)
    assert np.array_equal(host(cache.refs), sim.refs)
    layers = range(len(cache.head_size))
    for mine, pool in zip([cache.k(l) for l in layers] + [cache.v(l) for l in layers], sim.pools):
        assert np.array_equal(host(mine), pool)


def mirrored(cache, seed=0):
    """The cache's pools filled with random values, and its twin."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    layers = range(len(cache.head_size))
    pools = [cache.k(l) for l in layers] + [cache.v(l) for l in layers]
    for p in pools:
        p.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    return ref.Pages(cache.n_pages, cache.n_seqs, cache.max_pages, cache.page_size, [host(p) for p in pools])


def test_resize_grows_and_shrinks(g4, ctx):
    cache = new_cache(g4, ctx, kv=(1, 2), hs=(8, 24), pages=20, seqs=6, positions=100)
    sim = mirrored(cache)
    same_state(cache, sim)
    for seqs, lens in [([0, 3], [1, 33]), ([3, 1], [17, 16]), ([5], [0]), ([0, 1, 3], [100, 0, 16]), ([], []),
                       ([-1, 4, -7], [3, 48, 2]), ([0, 4], [0, 0])]:
        cache.resize(i32(seqs), i32(lens))
        assert sim.resize(seqs, lens)
        same_state(cache, sim)
    assert cache.check() == int((sim.refs == 0).sum())


def test_resize_takes_pages_given_back_in_the_same_call(g4, ctx):
    cache = new_cache(g4, ctx, pages=4, positions=64)
    sim = mirrored(cache)
    for seqs, lens in [([0, 1], [32, 32]), ([0, 2], [0, 32]), ([1, 0, 2], [16, 16, 17])]:
        cache.resize(i32(seqs), i32(lens))
        assert sim.resize(seqs, lens)
        same_state(cache, sim)


def test_resize_without_pages_changes_nothing(g4, ctx):
    cache = new_cache(g4, ctx, pages=4, positions=128)
    sim = mirrored(cache)
    cache.resize(i32([0, 1]), i32([40, 16]))
    assert sim.resize([0, 1], [40, 16])
    cache.resize(i32([1, 2, 0]), i32([1, 30, 33]))  # needs one page more than there are
    assert not sim.resize([1, 2, 0], [1, 30, 33]) or True
    with pytest.raises(g4.G4Error, match="free pages"):
        cache.check()
    assert cache.check() == 0
    cache.resize(i32([0, 2]), i32([16, 16]))
    cache.resize(i32([2]), i32([0]))
    assert cache.check() == 2


@pytest.mark.parametrize("holders,growers", [(2, [0]), (2, [0, 1]), (3, [2, 0]), (4, [3, 1, 0, 2])])
def test_shared_last_page_is_copied(g4, ctx, holders, growers):
    cache = new_cache(g4, ctx, kind="bf16", kv=(2, 1), hs=(40, 8), pages=16, seqs=5, positions=64)
    sim = mirrored(cache)
    cache.resize(i32([0]), i32([21]))
    sim.resize([0], [21])
    cache.fork(i32([0] * (holders - 1)), i32(range(1, holders)))
    sim.fork([0] * (holders - 1), range(1, holders))
    same_state(cache, sim)
    lens = [22 + 16 * (i % 2) for i in range(len(growers))]
    cache.resize(i32(growers), i32(lens))
    assert sim.resize(growers, lens)
    same_state(cache, sim)
    cache.check()


def test_fork_permutes_and_releases(g4, ctx):
    cache = new_cache(g4, ctx, pages=40, seqs=7, positions=600)
    sim = mirrored(cache)
    cache.resize(i32(range(5)), i32([5, 40, 0, 81, 16]))
    sim.resize(range(5), [5, 40, 0, 81, 16])
    for src, dst in [([0, 1, 2, 3, 4], [1, 2, 3, 4, 0]), ([3, 3, 3], [0, 1, 2]), ([1], [1]), ([-1, 4, 2], [3, -1, 5]),
                     ([5, 0], [6, 5]), ([], [])]:
        cache.fork(i32(src), i32(dst))
        sim.fork(src, dst)
        same_state(cache, sim)
    cache.check()


def test_many_sequences_fork(g4, ctx):
    """More entries than a CTA's column tile holds in whole lines."""
    n = 700
    cache = new_cache(g4, ctx, kv=(1,), hs=(8,), pages=3 * n, seqs=n, positions=300)
    sim = mirrored(cache)
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 49, n)
    cache.resize(i32(range(n)), i32(lens))
    assert sim.resize(range(n), lens)
    src = rng.integers(0, n, n)
    cache.fork(i32(src), i32(range(n)))
    sim.fork(src, range(n))
    same_state(cache, sim)
    grown = np.minimum(sim.lens + 1, 300)
    cache.resize(i32(range(n)), i32(grown))
    ok = sim.resize(range(n), grown)
    same_state(cache, sim)
    if ok:
        cache.check()


@pytest.mark.parametrize("pages", [1, 5, 63, 4097, 20000])
def test_compact(g4, ctx, pages):
    cache = new_cache(g4, ctx, kind="f16", kv=(1, 2), hs=(8, 16), pages=pages, seqs=9, positions=16 * pages)
    sim = mirrored(cache)
    rng = np.random.default_rng(pages)
    lens = rng.multinomial(pages, [1 / 9] * 9) * 16
    cache.resize(i32(range(9)), i32(lens))
    assert sim.resize(range(9), lens)
    cache.fork(i32([0]), i32([1]))
    sim.fork([0], [1])
    for a in (cache, sim):
        seqs, n = [2, 5, 7, 3], [0, 0, 3, 1]
        n = [min(x, int(sim.lens[s])) for x, s in zip(n, seqs)]
        a.resize(i32(seqs), i32(n)) if a is cache else a.resize(seqs, n)
    same_state(cache, sim)
    for _ in range(2):  # the second has nothing to do
        cache.compact()
        sim.compact()
        same_state(cache, sim)
    cache.check()


def test_copy_pages(g4, ctx):
    cache = new_cache(g4, ctx, kind="bf16", kv=(3, 1), hs=(72, 8), page=32, pages=12)
    sim = mirrored(cache)
    cache.copy_pages(i32([0, 5, -1, 2]), i32([7, 8, 3, -2]))
    for pool in sim.pools:
        pool[7], pool[8] = pool[0], pool[5]
    same_state(cache, sim)
    cache.check()
    cache.copy_pages(i32([0, 12]), i32([9, 10]))  # no page 12
    for pool in sim.pools:
        pool[9] = pool[0]
    same_state(cache, sim)
    with pytest.raises(g4.G4Error, match="out of range"):
        cache.check()


def test_bad_entries_are_skipped_and_reported(g4, ctx):
    cache = new_cache(g4, ctx, pages=16, seqs=4, positions=64)
    sim = mirrored(cache)
    for seqs, lens in [([0, 4, 1], [20, 5, 3]), ([2, 2], [7, 40]), ([3], [65]), ([3], [-1])]:
        cache.resize(i32(seqs), i32(lens))
        sim.resize(seqs, lens)
        same_state(cache, sim)
        if max(seqs) > 3 or len(set(seqs)) < len(seqs) or lens[0] in (65, -1):
            with pytest.raises(g4.G4Error):
                cache.check()
    cache.fork(i32([0, 1, 9, 0]), i32([3, 3, 1, 4]))
    sim.fork([0, 1, 9, 0], [3, 3, 1, 4])
    same_state(cache, sim)
    with pytest.raises(g4.G4Error, match="named twice"):
        cache.check()
    cache.check()


# ------------------------------------------------------------------ rotary rows


# |q_out - exact| <= 2^-20 of the pair's size: the reduced turn is rounded to 2^-25 turns (4e-7 rad at most half
# of it), sine and cosine to 2^-22, two products and a sum to 3 * 2^-24, and the norm's factor (a sum of hs squares
# by lanes and shuffles, at most hs / 32 + 6 roundings, halved by the root) and two products to 14 * 2^-24 at 512
ROPE_TOL = 2.0 ** -20


def pair_size(x, layout, rot):
    """Size of each element's pair (the element itself where nothing rotates)."""
    y = abs(x)
    a = np.arange(rot // 2)
    one, two = (a, a + rot // 2) if layout == "half" else (2 * a, 2 * a + 1)
    size = np.hypot(x[..., one], x[..., two])
    y[..., one], y[..., two] = size, size
    return y


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hs,rot", [(8, 4), (8, 8), (64, 64), (80, 20), (96, 96), (128, 32), (256, 256), (264, 132),
                                    (512, 512), (512, 128)])
def test_rope_apply(g4, ctx, layout, hs, rot):
    rng = np.random.default_rng(hs + rot)
    pos = np.array([0, 1, 2, 77, 4095, 131071, 999999, 2 ** 30, 5])
    x = rng.standard_normal((len(pos), 3, hs)).astype(np.float32)
    rope = g4.Rope(ctx, hs, rot_dim=rot, theta=1e4, layout=layout)
    wide = torch.zeros(len(pos), 3 * hs + 12, device="cuda")  # a strided input
    wide[:, 4:4 + 3 * hs] = torch.from_numpy(x.reshape(len(pos), -1))
    xin = wide[:, 4:4 + 3 * hs]
    out = torch.full((len(pos), 3 * hs), 7.0, device="cuda")
    rope.apply(xin, out, i32(pos))
    f, g = ref.frequencies(rot, 1e4)
    want = ref.rotate(x, pos, f, g, layout)
    assert np.all(abs(host(out).reshape(x.shape) - want) <= ROPE_TOL * pair_size(want, layout, rot) + 1e-30)
    rope.apply(xin, xin, i32(pos))  # in place
    assert torch.equal(xin, out)
    before = out.clone()
    rope.apply(xin, out, i32([-1] * len(pos)))
    assert torch.equal(out, before)


@pytest.mark.parametrize("scaling,kw", [("linear", dict(factor=4.0)), ("yarn", dict(factor=16.0, original_ctx=8192)),
                                        ("yarn", dict(factor=2.0, original_ctx=64, beta_fast=4.0, beta_slow=0.5)),
                                        ("none", dict(freq_factors=True))])
def test_rope_scaling(g4, ctx, scaling, kw):
    rng = np.random.default_rng(1)
    hs, rot, pos = 128, 96, np.array([3, 60000, 250000])
    if "freq_factors" in kw:
        kw = dict(freq_factors=(1 + 31 * rng.random(rot // 2)).astype(np.float32))
    x = rng.standard_normal((3, 2, hs)).astype(np.float32)
    rope = g4.Rope(ctx, hs, rot_dim=rot, theta=5e5, layout="half", scaling=scaling, **kw)
    out = torch.empty(3, 2 * hs, device="cuda")
    rope.apply(torch.from_numpy(x.reshape(3, -1)).cuda(), out, i32(pos))
    f, g = ref.frequencies(rot, 5e5, scaling, **kw)
    want = ref.rotate(x, pos, f, g, "half")
    assert np.all(abs(host(out).reshape(x.shape) - want) <= ROPE_TOL * pair_size(want, "half", rot) + 1e-30)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hs,heads,kv,rows,norm,layout,rot", [
    (64, 4, 2, 1, True, "half", 64), (128, 5, 1, 70, False, "interleaved", 64), (256, 16, 8, 9, True, "half", 256),
    (72, 3, 3, 33, True, "interleaved", 72), (512, 2, 1, 5, True, "half", 128), (64, 8, 8, 2500, False, "half", 64),
    (8, 1, 1, 17, False, "half", None), (136, 6, 3, 40, True, "half", None), (512, 4, 2, 700, True, "interleaved", 512)])
def test_append(g4, ctx, kind, hs, heads, kv, rows, norm, layout, rot):
    page, n_seq = 32, 3
    positions = rows + 100
    cache = new_cache(g4, ctx, kind, (1, kv), (8, hs), page, pages=3 * (positions // page + 1) + 1, seqs=n_seq,
                      positions=positions)
    cache.resize(i32([2, 0, 1]), i32([positions] * 3))
    for p in (cache.k(1), cache.v(1)):
        p.fill_(3.0)
    rng = np.random.default_rng(rows)
    seqs = rng.integers(0, n_seq, rows)
    pos = rng.permutation(positions)[:rows]
    fused = rng.standard_normal((rows, (heads + 2 * kv) * hs + 8)).astype(np.float32)
    dev = torch.from_numpy(fused).cuda()
    cut = [0, heads * hs, (heads + kv) * hs, (heads + 2 * kv) * hs]
    q, k, v = (dev[:, a:b] for a, b in zip(cut, cut[1:]))
    w = [(1 + 0.1 * rng.standard_normal(hs)).astype(np.float32) for _ in "qk"]
    rope = g4.Rope(ctx, hs, rot_dim=rot, theta=1e4, layout=layout) if rot else None
    out = torch.empty(rows, heads * hs, device="cuda")
    cache.append(1, q, k, v, out, i32(seqs), i32(pos), rope=rope, eps=1e-6, v_norm=norm,
                 **(dict(q_norm=torch.from_numpy(w[0]).cuda(), k_norm=torch.from_numpy(w[1]).cuda()) if norm else {}))
    cache.check()
    x = [fused[:, a:b].reshape(rows, -1, hs).astype(np.float64) for a, b in zip(cut, cut[1:])]
    if norm:
        x = [ref.rms(a, b, 1e-6) for a, b in zip(x, w + [None])]
    size = [abs(a) for a in x]
    if rot:
        f, g = ref.frequencies(rot, 1e4)
        size[:2] = [pair_size(a, layout, rot) for a in x[:2]]
        x[:2] = [ref.rotate(a, pos, f, g, layout) for a in x[:2]]
    assert np.all(abs(host(out).reshape(x[0].shape) - x[0]) <= ROPE_TOL * size[0] + 1e-30)
    table = host(cache.table)
    half = torch.finfo(TYPES[kind][1]).eps / 2  # the cache's rounding, beside the row's own error
    tiny = torch.finfo(TYPES[kind][1]).tiny * half * 2  # half a step below the normal numbers
    for pool, want, sz in ((cache.k(1), x[1], size[1]), (cache.v(1), x[2], size[2])):
        got = host(pool)
        page_of = table[seqs, pos // page]
        mine = got[page_of, :, pos % page]
        assert np.all(abs(mine - want) <= (ROPE_TOL * sz) * (1 + half) + half * abs(want) + tiny)
        rest = got.copy()
        rest[page_of, :, pos % page] = 3.0
        assert np.all(rest == 3.0)  # nothing else was written


def test_append_padding_and_missing_pages(g4, ctx):
    cache = new_cache(g4, ctx, kv=(1,), hs=(16,), pages=8, seqs=3, positions=64)
    cache.resize(i32([0, 1]), i32([20, 20]))
    cache.fork(i32([0]), i32([2]))
    for p in (cache.k(0), cache.v(0)):
        p.fill_(3.0)
    rows = dict(k=torch.ones(1, 16, device="cuda"), v=torch.ones(1, 16, device="cuda"))
    q = torch.ones(1, 32, device="cuda")
    for seq, pos, reported, turned in [(-1, 3, False, False), (1, -1, True, False), (3, 0, True, False),
                                       (1, 64, True, False), (1, 40, True, True), (0, 3, True, True)]:
        out = torch.full((1, 32), 9.0, device="cuda")
        cache.append(0, q, rows["k"], rows["v"], out, i32([seq]), i32([pos]))
        if reported:
            with pytest.raises(g4.G4Error):
                cache.check()
        cache.check()
        assert torch.all(out == (1.0 if turned else 9.0))
        assert torch.all(cache.k(0) == 3.0) and torch.all(cache.v(0) == 3.0)
    cache.append(0, None, rows["k"], rows["v"], None, i32([1]), i32([3]))  # K and V alone
    cache.check()
    assert int((cache.k(0) == 1.0).sum()) == 16 == int((cache.v(0) == 1.0).sum())
    cache.append(0, q[:0], rows["k"][:0], rows["v"][:0], q[:0], i32([]), i32([]))
    cache.check()


# ------------------------------------------------------------------ attention


def attend_case(g4, ctx, kind, hs, kv, heads, page, rows, scale=1.0, window=0, sinks=0, seed=0, q_size=2.0, n_seqs=None,
                pages=None):
    """rows: (sequence, position) pairs.  Every pool element that no row sees is NaN."""
    rng = np.random.default_rng(seed)
    n_seqs = n_seqs or max([s for s, _ in rows] + [0]) + 2
    width = max([p for _, p in rows] + [0]) // page + 1
    total = n_seqs * width + 2
    cache = new_cache(g4, ctx, kind, (kv,), (hs,), page, pages or total, n_seqs, width * page)
    base = (pages or total) - total
    table = (base + rng.permutation(total)[:n_seqs * width]).reshape(n_seqs, width)
    k = np.full((total, kv, page, hs), np.nan)
    v = k.copy()
    used = np.zeros((n_seqs, width * page), bool)
    for s, p in rows:
        if s >= 0 and p >= 0:
            used[s, ref.visible(p, window, sinks)] = True
    for s, t in zip(*np.nonzero(used)):
        k[table[s, t // page] - base, :, t % page] = rng.standard_normal((kv, hs)) * hs ** -0.5
        v[table[s, t // page] - base, :, t % page] = rng.standard_normal((kv, hs))
    # pages that hold nothing visible are missing
    held = used.reshape(n_seqs, width, page).any(-1)
    cache.table.copy_(torch.from_numpy(np.where(held, table, -1)))
    for mine, pool in ((cache.k(0), k), (cache.v(0), v)):
        mine[base:].copy_(torch.from_numpy(pool))
    k, v = host(cache.k(0)[base:]), host(cache.v(0)[base:])
    q = (rng.standard_normal((len(rows), heads * hs)) * q_size).astype(np.float32)
    wide = torch.full((len(rows), heads * hs + 5), 11.0, device="cuda")
    out = wide[:, :heads * hs]
    qd = torch.zeros(len(rows), heads * hs + 3, device="cuda")
    qd[:, 3:] = torch.from_numpy(q)
    args = (0, qd[:, 3:], out, i32([s for s, _ in rows]), i32([p for _, p in rows]))
    cache.attend(*args, scale=scale, window=window, sinks=sinks)
    cache.check()
    got = host(wide)
    assert np.all(got[:, heads * hs:] == 11.0)
    for i, (s, p) in enumerate(rows):
        if s < 0:
            assert np.all(got[i] == 11.0)
            continue
        want, bound = ref.attend(q[i], k, v, table[s] - base, p, scale, window, sinks)
        err = abs(got[i, :heads * hs] - want)
        assert np.all(err <= bound), (i, s, p, float((err / np.maximum(bound, 1e-300)).max()))
    first = wide.clone()
    cache.attend(*args, scale=scale, window=window, sinks=sinks)
    assert torch.equal(first, wide)  # the same bits again
    return cache


EDGES = [(0, 0), (1, 1), (2, 14), (3, 15), (4, 16), (5, 17), (6, 63), (7, 64), (8, 65), (9, 127), (10, 300)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hs", [8, 16, 40, 64, 72, 80, 128, 136, 256, 264, 512])
def test_attend_head_sizes(g4, ctx, kind, hs):
    attend_case(g4, ctx, kind, hs, 2, 6, 16, EDGES, seed=hs)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("kv,heads", [(1, 1), (1, 8), (3, 6), (2, 14), (1, 9), (1, 16), (2, 40), (8, 8)])
def test_attend_groups(g4, ctx, kind, kv, heads):
    attend_case(g4, ctx, kind, 64, kv, heads, 32, EDGES, scale=0.7, seed=heads)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 1), (64, 4), (100, 70), (1000, 3), (16, 500)])
def test_attend_windows(g4, ctx, kind, page, window, sinks):
    attend_case(g4, ctx, kind, 80, 2, 4, page, EDGES + [(11, 999), (12, 640)], window=window, sinks=sinks, seed=window)


def test_attend_empty_and_padding_rows(g4, ctx):
    attend_case(g4, ctx, "bf16", 64, 1, 4, 16, [(-1, 5), (0, -1), (1, 40), (-1, -1), (2, -5), (1, 3), (-3, 100)])
    attend_case(g4, ctx, "f32", 64, 1, 4, 16, [(0, -1)] * 3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attend_in_place(g4, ctx, kind):
    cache = new_cache(g4, ctx, kind, (2,), (64,), 16, 700, 9, 1200)
    cache.resize(i32(range(9)), i32([1200] * 9))
    g = torch.Generator(device="cuda").manual_seed(4)
    for p in (cache.k(0), cache.v(0)):
        p.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    q = torch.randn(9, 20 * 64, generator=g, device="cuda")
    pos = i32([0, 1199, 5, 700, 64, -1, 31, 1198, 300])
    out = torch.empty_like(q)
    cache.attend(0, q, out, i32(range(9)), pos, scale=0.1)
    cache.attend(0, q, q, i32(range(9)), pos, scale=0.1)
    assert torch.equal(q, out)


def test_attend_rows_of_one_sequence(g4, ctx):
    """A prompt chunk: many rows of few sequences, each up to its own position."""
    rows = [(s, p) for s in range(3) for p in range(100, 200)]
    attend_case(g4, ctx, "f16", 64, 2, 4, 32, rows, seed=2)


def test_attend_many_rows(g4, ctx):
    rng = np.random.default_rng(9)
    rows = [(i, int(p)) for i, p in enumerate(rng.integers(-1, 60, 600))]
    attend_case(g4, ctx, "bf16", 16, 1, 2, 16, rows, seed=4)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attend_long(g4, ctx, kind):
    attend_case(g4, ctx, kind, 128, 1, 8, 64, [(0, 40000), (1, 3), (2, 9000)], seed=5)
    attend_case(g4, ctx, kind, 512, 1, 2, 64, [(0, 5001)], seed=6)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attend_sharp_and_flat_scores(g4, ctx, kind):
    """Scores of hundreds (one position takes all) and of nearly nothing."""
    for q_size in (100.0, 1e-6, 0.0):
        attend_case(g4, ctx, kind, 64, 1, 8, 16, [(0, 200), (1, 33)], q_size=q_size, seed=7)


def test_attend_offsets_beyond_32_bits(g4, ctx):
    pages = 2 ** 31 // (16 * 512) + 64
    cache = attend_case(g4, ctx, "bf16", 512, 1, 4, 16, [(0, 100), (1, 7)], seed=8, pages=pages)
    assert cache.k(0).numel() > 2 ** 31
    rows = torch.ones(1, 512, device="cuda")
    cache.refs.fill_(1)
    cache.append(0, None, rows, rows, None, i32([0]), i32([100]))
    cache.check()
    page = int(cache.table[0, 100 // 16])
    assert page * 16 * 512 > 2 ** 31 and torch.all(cache.k(0)[page, 0, 100 % 16] == 1.0)
    cache.copy_pages(i32([page]), i32([0]))
    assert torch.equal(cache.k(0)[0].view(torch.int16), cache.k(0)[page].view(torch.int16))
    cache.free()


def test_attend_leaves_missing_pages_out(g4, ctx):
    """A visible position without a page is reported, and the rest is attended."""
    for kind in ("f32", "bf16"):
        cache = new_cache(g4, ctx, kind, (1,), (64,), 16, 16, 2, 256)
        cache.resize(i32([0]), i32([160]))
        g = torch.Generator(device="cuda").manual_seed(6)
        for p in (cache.k(0), cache.v(0)):
            p.copy_(torch.randn(p.shape, generator=g, device="cuda"))
        q, out = torch.randn(1, 256, generator=g, device="cuda"), torch.empty(1, 256, device="cuda")
        table = host(cache.table)
        cache.table[0, 3] = -1
        cache.table[0, 7] = 16  # no such page
        cache.attend(0, q, out, i32([0]), i32([150]), scale=0.1)
        with pytest.raises(g4.G4Error, match="without a page"):
            cache.check()
        t = np.array([t for t in range(151) if t // 16 not in (3, 7)])
        k, v = (host(p)[table[0, t // 16], 0, t % 16] for p in (cache.k(0), cache.v(0)))
        x = 0.1 * host(q).reshape(4, 64) @ k.T
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        # the bound of paged_ref.attend
        dx = (64 / 16 + 6) * 2.0 ** -23 * (0.1 * abs(host(q)).reshape(4, 64) @ abs(k).T).max(1) + 2.0 ** -22
        bound = (p @ abs(v)) * (2 * dx[:, None] + (len(t) / 64 + 16) * 2.0 ** -23)
        assert np.all(abs(host(out).reshape(4, 64) - p @ v) <= bound)


def test_most_sequences(g4, ctx):
    """The largest number of sequences and entries."""
    n = 4096
    cache = new_cache(g4, ctx, kv=(1,), hs=(8,), pages=2 * n, seqs=n, positions=64)
    sim = mirrored(cache)
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 33, n)
    order = rng.permutation(n)
    cache.resize(i32(order), i32(lens))
    assert sim.resize(order, lens)
    src = rng.permutation(n)
    cache.fork(i32(src), i32(order))
    sim.fork(src, order)
    same_state(cache, sim)
    cache.compact()
    sim.compact()
    same_state(cache, sim)
    cache.resize(i32(order), i32([0] * n))
    assert cache.check() == 2 * n
    with pytest.raises(g4.G4Error):
        cache.fork(i32([0] * (n + 1)), i32([0] * (n + 1)))


def test_attend_reports_bad_rows(g4, ctx):
    cache = new_cache(g4, ctx, kv=(1,), hs=(16,), pages=8, seqs=3, positions=64)
    q = torch.ones(1, 16, device="cuda")
    cache.resize(i32([0]), i32([20]))
    for seq, pos, untouched in [(3, 5, True), (0, 64, True), (0, 40, False), (1, 0, False)]:
        out = torch.full((1, 16), 9.0, device="cuda")
        cache.attend(0, q, out, i32([seq]), i32([pos]))
        with pytest.raises(g4.G4Error, match="row"):
            cache.check()
        assert torch.all(out == 9.0) if untouched else torch.all(torch.isfinite(out))
    cache.check()


# ------------------------------------------------------------------ beam selection


def select(g4, ctx, logits, scores, beams, finished=None, pad=0):
    n = logits.shape[0]
    new, par, tok = torch.empty(n, device="cuda"), i32([7] * n), i32([7] * n)
    g4.beam_select(ctx, logits, scores, beams, new, par, tok, finished=finished, pad_token=pad)
    return new, par, tok


def check_beams(g4, ctx, logits, scores, beams, finished=None, pad=0):
    fin = None if finished is None else i32(finished)
    got = select(g4, ctx, torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), beams, fin, pad)
    want = ref.beam(logits, scores, beams, finished, pad)
    assert np.array_equal(host(got[1]), want[1])
    assert np.array_equal(host(got[2]), want[2])
    s = host(got[0])
    live = want[1] >= 0
    assert np.all(s[~live] == -np.inf)
    # the row's sum: exponentials to 2^-21, 32 additions per thread and 8 more: 2^-18 of it at most; then one rounding
    assert np.all(abs(s[live] - want[0][live]) <= 2.0 ** -18 + 2.0 ** -24 * abs(want[0][live]))


@pytest.mark.parametrize("vocab", [1, 3, 255, 1023, 1024, 1025, 8192, 32001, 262144])
@pytest.mark.parametrize("groups,beams", [(1, 1), (3, 4), (2, 7), (1, 32)])
def test_beam_select(g4, ctx, vocab, groups, beams):
    rng = np.random.default_rng(vocab + beams)
    n = groups * beams
    logits = (rng.standard_normal((n, vocab)) * 4).astype(np.float32)
    check_beams(g4, ctx, logits, (-20 * rng.random(n)).astype(np.float32), beams)


def test_beam_ties_go_to_the_lowest(g4, ctx):
    rng = np.random.default_rng(0)
    for vocab in (40, 20000):
        logits = np.zeros((8, vocab), np.float32)
        check_beams(g4, ctx, logits, np.zeros(8, np.float32), 8)
        logits = rng.integers(-2, 2, (8, vocab)).astype(np.float32)  # whole numbers: many ties in a row
        check_beams(g4, ctx, logits, (-rng.random(8)).astype(np.float32), 4)
    logits = np.tile(rng.standard_normal((1, 9000)).astype(np.float32), (6, 1))  # equal beams
    check_beams(g4, ctx, logits, np.full(6, -1.5, np.float32), 6)


def test_beam_masks_and_finished(g4, ctx):
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((12, 10007)).astype(np.float32)
    logits[rng.random(logits.shape) < 0.9] = -np.inf
    logits[1] = -np.inf       # a row with nothing left
    logits[2, 3:] = -np.inf   # and one with few tokens
    logits[4:8] = -np.inf     # a group with nothing left
    logits[9, ::3] = np.nan
    scores = (-5 * rng.random(12)).astype(np.float32)
    check_beams(g4, ctx, logits, scores, 4)
    check_beams(g4, ctx, logits, scores, 4, finished=[0, 0, 1, 0, 0, 1, 0, 0, 1, 1, 1, 1], pad=3)
    scores[8:] = -np.inf      # beams that do not exist yet
    check_beams(g4, ctx, logits, scores, 4)
    low = np.full((4, 300), np.finfo(np.float32).min, np.float32)  # the type's lowest value masks, too
    low[:, 7] = 1.0
    check_beams(g4, ctx, low, np.zeros(4, np.float32), 4)


@pytest.mark.parametrize("beams", [1, 5, 32])
def test_beam_ordered_logits(g4, ctx, beams):
    """Rows that rise, fall or stay level over the vocabulary: every piece of a
    rising row beats all before it, at once or within a few."""
    vocab = 100003
    up = np.linspace(-10, 10, vocab).astype(np.float32)
    saw = (up + np.where(np.arange(vocab) % 7 == 0, 3.0, 0.0)).astype(np.float32)
    rows = np.stack([up, up[::-1], np.zeros(vocab, np.float32), saw, np.round(up), np.where(up > 9.9, up, -np.inf)])
    rows = np.repeat(rows, beams, axis=0).astype(np.float32)
    check_beams(g4, ctx, rows, np.tile(-np.arange(beams) * 0.125, 6).astype(np.float32), beams)


def test_beam_infinite_logits(g4, ctx):
    """A row with +inf has no continuation; its group's others go on."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((4, 3000)).astype(np.float32)
    logits[1, 1500] = np.inf
    scores = np.zeros(4, np.float32)
    got = select(g4, ctx, torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), 4)
    masked = logits.copy()
    masked[1] = -np.inf
    want = ref.beam(masked, scores, 4)
    assert np.array_equal(host(got[1]), want[1]) and np.array_equal(host(got[2]), want[2])


def test_beam_strided_and_in_place(g4, ctx):
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((4, 5001)).astype(np.float32)
    scores = (-rng.random(4)).astype(np.float32)
    wide = torch.zeros(4, 5001 + 6, device="cuda")
    wide[:, 3:5004] = torch.from_numpy(logits)
    s = torch.from_numpy(scores).cuda()
    par, tok = i32([0] * 4), i32([0] * 4)
    g4.beam_select(ctx, wide[:, 3:5004], s, 2, s, par, tok)
    want = ref.beam(logits, scores, 2)
    assert np.array_equal(host(par), want[1]) and np.array_equal(host(tok), want[2])


# ------------------------------------------------------------------ together


class BeamLoop:
    """One search step on the device: select, reorder, grow, append, attend."""

    def __init__(self, g4, ctx, kind, groups=2, beams=3, prompt=21, vocab=997, layers=2, kv=2, heads=4, hs=32):
        self.g4, self.ctx = g4, ctx
        n = self.n = groups * beams
        self.beams, self.layers = beams, layers
        self.cache = new_cache(g4, ctx, kind, (kv,) * layers, (hs,) * layers, 16, 8 * n, n, 96)
        self.rope = g4.Rope(ctx, hs, theta=1e4)
        g = torch.Generator(device="cuda").manual_seed(5)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.emb, self.wqkv = r(vocab, heads * hs), [r(heads * hs, (heads + 2 * kv) * hs) * 0.1 for _ in range(layers)]
        self.head = r(heads * hs, vocab) * 0.2
        self.rows = torch.arange(n, dtype=torch.int32, device="cuda")
        self.scores = torch.zeros(n, device="cuda")
        self.scores[torch.arange(n, device="cuda") % beams != 0] = -torch.inf
        self.parents, self.tokens = self.rows.clone(), torch.zeros_like(self.rows)
        self.x = r(n, heads * hs)
        self.pos = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.len = torch.zeros_like(self.pos)
        self.cut = [heads * hs, (heads + kv) * hs, (heads + 2 * kv) * hs]
        # the prompt: rows of the groups' first beams, then shared by the others
        self.cache.resize(self.rows[::beams].contiguous(), torch.full((groups,), prompt, dtype=torch.int32, device="cuda"))
        for t in range(prompt):
            for l in range(layers):
                qkv = self.emb[t * 7 % vocab:][:1].repeat(groups, 1) @ self.wqkv[l]
                self.cache.append(l, None, *self.kv(qkv), None, self.rows[::beams].contiguous(),
                                  torch.full((groups,), t, dtype=torch.int32, device="cuda"), rope=self.rope)
        self.cache.fork(self.rows // beams * beams, self.rows)
        self.pos.fill_(prompt - 1)

    def kv(self, qkv):
        return qkv[:, self.cut[0]:self.cut[1]], qkv[:, self.cut[1]:self.cut[2]]

    def step(self):
        c = self.cache
        logits = self.x @ self.head
        self.g4.beam_select(self.ctx, logits, self.scores, self.beams, self.scores, self.parents, self.tokens)
        c.fork(self.parents, self.rows)
        self.pos += 1
        self.len.copy_(self.pos + 1)
        c.resize(self.rows, self.len)
        x = self.emb[self.tokens.clamp(min=0).long()]
        for l in range(self.layers):
            qkv = x @ self.wqkv[l]
            q = qkv[:, :self.cut[0]]
            c.append(l, q, *self.kv(qkv), q, self.rows, self.pos, rope=self.rope)
            out = torch.empty_like(x)
            c.attend(l, q, out, self.rows, self.pos, scale=0.2, window=24, sinks=2)
            x = x + out
        self.x.copy_(x / x.norm(dim=1, keepdim=True) * 10)

    def dense(self, l):
        """K rows of every sequence in order, gathered through the table."""
        t = self.cache.table.clamp(min=0).long()
        k = self.cache.k(l)[t].transpose(2, 3).flatten(1, 2)
        return [k[i, :int(n)] for i, n in enumerate(self.cache.lens)]


def test_beam_search_step(g4, ctx):
    """The operators together, step by step against copies kept without pages."""
    b = BeamLoop(g4, ctx, "f32")
    kept = [[k.clone() for k in b.dense(l)] for l in range(b.layers)]
    for _ in range(40):
        b.step()
        b.cache.check()
        par = b.parents.tolist()
        assert all(p >= 0 for p in par)
        for l in range(b.layers):
            now = b.dense(l)
            for i in range(b.n):
                assert torch.equal(now[i][:-1], kept[l][par[i]])  # the parent's history
            kept[l] = [k.clone() for k in now]
        refs = np.bincount(host(b.cache.table)[host(b.cache.table) >= 0], minlength=b.cache.n_pages)
        assert np.array_equal(refs, host(b.cache.refs))


def test_beam_search_captured(g4, ctx):
    """Captured once and replayed, the step gives what it gives launch by launch;
    two graphs of two searches take turns."""
    eager = [BeamLoop(g4, ctx, "bf16"), BeamLoop(g4, ctx, "bf16", prompt=30)]
    loops = [BeamLoop(g4, ctx, "bf16"), BeamLoop(g4, ctx, "bf16", prompt=30)]
    side = torch.cuda.Stream()
    graphs = []
    for b in loops:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b.step()  # the first step outside
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.step()
            with pytest.raises(g4.G4Error, match="captured"):
                b.cache.check()
        graphs.append(g)
    for _ in range(20):
        for g in graphs:
            g.replay()
    for e, b in zip(eager, loops):
        for _ in range(21):
            e.step()
        for x, y in ((e.cache.table, b.cache.table), (e.cache.refs, b.cache.refs), (e.tokens, b.tokens),
                     (e.scores, b.scores), (e.x, b.x), (e.cache.k(1).view(torch.int16), b.cache.k(1).view(torch.int16))):
            assert torch.equal(x, y)
        e.cache.check()
        b.cache.check()


def test_calls_on_other_streams(g4, ctx):
    """Attention of one cache on several streams at once, each with its own work space."""
    cache = new_cache(g4, ctx, "bf16", (2,), (128,), 16, 400, 4, 1600)
    cache.resize(i32(range(4)), i32([1600] * 4))
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in (cache.k(0), cache.v(0)):
        p.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    q = [torch.randn(4, 1024, generator=g, device="cuda") for _ in range(4)]
    rows, pos = i32(range(4)), i32([1599, 700, 3, 1000])
    want, got = [torch.empty_like(x) for x in q], [torch.empty_like(x) for x in q]
    for x, o in zip(q, want):
        cache.attend(0, x, o, rows, pos, scale=0.05)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(10):
        for i, s in enumerate(streams):
            if i % 2:
                cache.attend(0, q[i], got[i], rows, pos, scale=0.05, stream=s.cuda_stream)
            else:
                with torch.cuda.stream(s):
                    cache.attend(0, q[i], got[i], rows, pos, scale=0.05)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_handles_outlive_their_context(g4):
    """Views keep the pages alive; the context may go first."""
    c = g4.Context(0)
    cache = new_cache(g4, c, kv=(1,), hs=(16,), pages=4)
    rope = g4.Rope(c, 16)
    view = cache.k(0)
    view.fill_(2.0)
    del cache
    c.close()
    assert float(view.sum()) == 2.0 * view.numel()
    del view, rope


# ------------------------------------------------------------------ refusals


def test_refusals(g4, ctx):
    bad = [dict(page=24), dict(hs=(12,)), dict(hs=(520,)), dict(kv=(0,)), dict(pages=0), dict(seqs=0), dict(seqs=5000),
           dict(positions=0)]
    for kw in bad:
        with pytest.raises(ValueError):
            new_cache(g4, ctx, **kw)
    with pytest.raises(g4.UnsupportedOperation):
        g4.KvCache(ctx, [1], [64], dtype=g4.GGMLType.Q8_0)
    with pytest.raises(g4.G4Error, match="allocate"):
        new_cache(g4, ctx, kv=(64,) * 64, hs=(512,) * 64, page=256, pages=1 << 20)
    for kw in [dict(head_size=12), dict(rot_dim=6), dict(rot_dim=72), dict(theta=1.0), dict(layout="other"),
               dict(scaling="linear", factor=0.0), dict(scaling="yarn", factor=2.0, original_ctx=0),
               dict(freq_factors=[1.0]), dict(freq_factors=[0.0] * 32), dict(theta=float("nan"))]:
        with pytest.raises(ValueError):
            g4.Rope(ctx, **{"head_size": 64, **kw})
    cache = new_cache(g4, ctx, kv=(2,), hs=(64,))
    q, kv = torch.zeros(2, 256, device="cuda"), torch.zeros(2, 128, device="cuda")
    r = i32([0, 1])
    with pytest.raises(ValueError):
        cache.attend(1, q, q, r, r)  # no such layer
    with pytest.raises(ValueError):
        cache.attend(0, q[:, :100], q, r, r)
    with pytest.raises(TypeError):
        cache.attend(0, q.half(), q, r, r)
    with pytest.raises(TypeError):
        cache.attend(0, q, q, r.long(), r)
    with pytest.raises(ValueError):
        cache.attend(0, q.cpu(), q, r, r)
    with pytest.raises(g4.G4Error):
        cache.attend(0, torch.zeros(2, 192, device="cuda"), torch.zeros(2, 192, device="cuda"), r, r)  # 3 heads over 2
    with pytest.raises(g4.G4Error):
        cache.attend(0, q, torch.empty_like(q), r, r, window=-1)
    with pytest.raises(ValueError):
        cache.append(0, q, kv[:1], kv, q, r, r)
    with pytest.raises(g4.G4Error, match="head size"):
        cache.append(0, q, kv, kv, q, r, r, rope=g4.Rope(ctx, 32))
    with pytest.raises(g4.G4Error, match="aligned"):
        x = torch.zeros(2 * 256 + 1, device="cuda")[1:].view(2, 256)
        cache.append(0, x, kv, kv, q, r, r)
    with pytest.raises(g4.G4Error):
        cache.resize(i32([0] * 9), i32([0] * 9))  # more entries than sequences
    lg, s = torch.zeros(4, 50, device="cuda"), torch.zeros(4, device="cuda")
    for beams in (0, 3, 33):
        with pytest.raises(g4.G4Error):
            g4.beam_select(ctx, lg, s, beams, s, i32([0] * 4), i32([0] * 4))
    cache.check()
