"""Calls of the paged operators that their documentation allows and that are easy
to get wrong: finite masks, extreme and non-finite values, one-row strides,
arguments on other streams, refused resizes, freed handles."""
import numpy as np
import pytest
import torch

from tests import paged_ref as ref
from tests.test_paged_gpu import (EDGES, ROPE_TOL, attend_case, host, i32, mirrored, new_cache, pair_size, same_state,
                                  select)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ beam selection


def continuations(logits, scores, beams):
    """paged_ref.beam of rows without -inf, with every log probability taken as
    (x - max) - log sum exp(x - max): beside a maximum of -1e20 the logarithm
    would be rounded away."""
    x = np.asarray(logits, np.float64)
    x = x - x.max(1, keepdims=True)
    p = np.asarray(scores, np.float64)[:, None] + (x - np.log(np.exp(x).sum(1, keepdims=True)))
    out = []
    for g in range(0, len(x), beams):
        row, token = np.divmod(np.argsort(-p[g:g + beams].reshape(-1), kind="stable")[:beams], x.shape[1])
        out.append((p[g + row, token], g + row, token))
    return [np.concatenate(a) for a in zip(*out)]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("mask", [-1e6, -3e9, -1e10, -1e11, -1e12, -1e15, -1e20, -1e30, -1e38,
                                  float(np.finfo(np.float32).min)])
def test_beam_finite_masks(g4, ctx, mask, offset):
    """Masks that are very low but finite: pieces of a row without a live token,
    rows without any, a group with fewer live tokens than beams."""
    rng = np.random.default_rng(17)
    beams, vocab = 4, 5003
    logits = np.full((20, vocab), mask, np.float32)
    logits[:4, 2100:2110] = rng.standard_normal((4, 10))
    logits[4:8, [7, 4999]] = rng.standard_normal((4, 2))
    logits[8, 5] = 1.0       # its group's other rows have nothing live
    logits[12:16] = mask     # nor has any row of this group
    logits[16, 3000] = -2.0  # one live token, the other beams do not exist yet
    scores = -1.5 * rng.permutation(20).astype(np.float32) - 0.25
    scores[17:] = -np.inf
    wide = torch.zeros(20, vocab + 5, device="cuda")
    wide[:, offset:offset + vocab] = torch.from_numpy(logits)
    new, par, tok = select(g4, ctx, wide[:, offset:offset + vocab], torch.from_numpy(scores).cuda(), beams)
    want = continuations(logits, scores, beams)
    assert np.array_equal(host(par), want[1]) and np.array_equal(host(tok), want[2])
    # as in test_paged_gpu.py: the row's sum to 2^-18, then one rounding
    assert np.all(abs(host(new) - want[0]) <= 2.0 ** -18 + 2.0 ** -24 * abs(want[0]))


def test_beam_extreme_logits(g4, ctx):
    """The largest finite logits, and both ends of the type in one row."""
    top = float(np.finfo(np.float32).max)
    rng = np.random.default_rng(4)
    logits = np.stack([np.full(3000, top), np.where(rng.random(3000) < 0.5, top, -top),
                       1e38 * rng.random(3000)]).astype(np.float32)
    scores = np.array([-1.0, -2.5, -30.0], np.float32)
    for beams in (1, 3):
        new, par, tok = select(g4, ctx, torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), beams)
        want = continuations(logits, scores, beams)
        assert np.array_equal(host(par), want[1]) and np.array_equal(host(tok), want[2])
        assert np.all(abs(host(new) - want[0]) <= 2.0 ** -18 + 2.0 ** -24 * abs(want[0]))


def test_beam_zeros_of_either_sign(g4, ctx):
    """-0 and +0 are equal: the lower token, the lower beam."""
    for vocab, low, high in ((40, 3, 30), (3000, 100, 101), (3000, 100, 2500), (3000, 2100, 2101)):
        logits = np.full((1, vocab), -1.0, np.float32)
        logits[0, low], logits[0, high] = -0.0, 0.0
        _, _, tok = select(g4, ctx, torch.from_numpy(logits).cuda(), torch.zeros(1, device="cuda"), 1)
        assert tok.tolist() == [low]
    logits = torch.zeros(2, 9, device="cuda")
    new, par, tok = select(g4, ctx, logits, torch.tensor([-0.0, 0.0], device="cuda"), 2, i32([1, 1]), 4)
    assert par.tolist() == [0, 1] and tok.tolist() == [4, 4] and new.tolist() == [0.0, 0.0]


# ------------------------------------------------------------------ pages


def test_resize_to_more_pages_than_32_bits_count(g4, ctx):
    """4096 sequences of 2^20 pages each: 2^31 pages wanted, 2^32, and a few around them."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs a page table of 17 GB")
    n, most = 4096, 1 << 24
    cache = new_cache(g4, ctx, kv=(1,), hs=(8,), pages=40, seqs=n, positions=most)
    cache.resize(i32([5, 0]), i32([17, 33]))
    cache.fork(i32([5, 5]), i32([9, 7]))
    assert cache.check() == 40 - 5
    lens, refs, table = cache.lens.clone(), cache.refs.clone(), cache.table[:16, :8].clone()
    order = torch.arange(n, dtype=torch.int32, device="cuda")
    for many, longest in ((2048, most), (2047, most), (4096, most), (4095, most), (4096, most // 2)):
        cache.resize(order[:many], torch.full((many,), longest, dtype=torch.int32, device="cuda"))
        with pytest.raises(g4.G4Error, match="free pages"):
            cache.check()
        assert torch.equal(cache.lens, lens) and torch.equal(cache.refs, refs)
        assert torch.equal(cache.table[:16, :8], table) and int((cache.table.amax(1) >= 0).sum()) == 4
    cache.resize(i32([9, 1]), i32([18, 40]))  # one copy, three pages
    assert cache.check() == 35 - 4
    del cache


@pytest.mark.parametrize("seqs,lens", [
    ([1, 3, 0, 2], [10, 20, 34, 100]),  # whole pages given back, shared ones among them, then too few
    ([3, 2, 1], [0, 128, 0]),           # a sequence freed, another, and still too few
    ([0, 3, 2, 1], [40, 36, 90, 16]),   # a shared last page that both holders want to grow into
    ([4, 1, 2], [1, 33, 128]),
])
def test_refused_resize_restores_the_pages(g4, ctx, seqs, lens):
    """What a call gives back before it finds too few pages is taken again."""
    cache = new_cache(g4, ctx, kv=(1, 2), hs=(8, 16), pages=8, seqs=5, positions=128)
    sim = mirrored(cache)
    for a in (cache, sim):
        s = (lambda x: i32(x)) if a is cache else (lambda x: x)
        a.resize(s([0, 1]), s([33, 40]))
        a.fork(s([0]), s([3]))
    same_state(cache, sim)
    assert cache.check() == 2
    for _ in range(2):
        cache.resize(i32(seqs), i32(lens))
        assert sim.resize(seqs, lens) is False
        same_state(cache, sim)
        with pytest.raises(g4.G4Error, match="free pages"):
            cache.check()
    cache.resize(i32([1, 3, 2]), i32([0, 35, 50]))  # the same cache goes on
    assert sim.resize([1, 3, 2], [0, 35, 50])
    same_state(cache, sim)
    assert cache.check() == int((sim.refs == 0).sum())


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("power", [122, 119, 100, -99, -95])
def test_attend_query_ranges(g4, ctx, kind, power):
    """Queries of any finite size, the scale bringing the scores back."""
    attend_case(g4, ctx, kind, 64, 1, 8, 16, [(0, 200), (1, 33), (2, 0)], q_size=2.0 ** power, scale=2.0 ** -power,
                seed=11)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_attend_reports_any_entry_that_is_no_page(g4, ctx, kind):
    """A visible position whose table entry is no page, whatever it is."""
    for entry in (-1, -2, -3, -2 ** 31, 16, 2 ** 31 - 1):
        cache = new_cache(g4, ctx, kind, (1,), (64,), 16, 16, 2, 256)
        cache.resize(i32([0]), i32([160]))
        for p in (cache.k(0), cache.v(0)):
            p.fill_(0.5)
        cache.table[0, 3] = entry
        out = torch.empty(1, 128, device="cuda")
        cache.attend(0, torch.ones(1, 128, device="cuda"), out, i32([0]), i32([150]))
        with pytest.raises(g4.G4Error, match="without a page"):
            cache.check()
        assert torch.all(out == 0.5)


@pytest.mark.parametrize("hs", [64, 80, 256, 512])
@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 1), (64, 4), (100, 70), (1000, 3), (16, 500)])
def test_attend_windows_of_an_fp32_cache(g4, ctx, hs, page, window, sinks):
    attend_case(g4, ctx, "f32", hs, 2, 6, page, EDGES + [(11, 999), (12, 640)], window=window, sinks=sinks, seed=hs + window)


@pytest.mark.parametrize("kind,hs", [("f32", 64), ("f32", 128), ("f32", 256), ("f32", 512), ("f16", 128), ("bf16", 256)])
def test_attend_more_rows_than_a_warp_finds(g4, ctx, kind, hs):
    rng = np.random.default_rng(hs)
    for n in (128, 129, 301):
        rows = [(i % 70, int(p)) for i, p in enumerate(rng.permutation(400)[:n] - 2)]
        attend_case(g4, ctx, kind, hs, 1, 3, 32, rows, window=60, sinks=3, seed=n)


# ------------------------------------------------------------------ rows


def test_one_row_of_a_wider_tensor(g4, ctx):
    """The distance between rows does not matter where there is one."""
    hs, heads, kv = 64, 4, 2
    cache = new_cache(g4, ctx, kv=(kv,), hs=(hs,), pages=4, seqs=2, positions=64)
    cache.resize(i32([1]), i32([20]))
    rng = np.random.default_rng(0)
    wide = torch.from_numpy(rng.standard_normal((3, (heads + 2 * kv) * hs + 1)).astype(np.float32)).cuda()
    q, k, v = (wide[:1, a * hs:b * hs] for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    assert q.stride(0) % 4
    rope = g4.Rope(ctx, hs)
    out = torch.empty(heads * hs, 1, device="cuda").t()  # [1, heads * hs], one entry "between rows"
    cache.append(0, q, k, v, out, i32([1]), i32([17]), rope=rope)
    cache.check()
    page = int(cache.table[1, 1])
    f, g = ref.frequencies(hs, 1e4)
    for got, x, turned in ((out, q, True), (cache.k(0)[page, :, 1], k, True), (cache.v(0)[page, :, 1], v, False)):
        x = host(x).reshape(1, -1, hs)
        want = ref.rotate(x, [17], f, g, "half") if turned else x
        assert np.all(abs(host(got).reshape(x.shape) - want) <= ROPE_TOL * pair_size(want, "half", hs))
    again = torch.empty_like(out)
    rope.apply(q, again, i32([17]))
    assert torch.equal(again, out)
    with pytest.raises(g4.G4Error, match="aligned"):  # two rows an odd distance apart
        rope.apply(wide[:2, :hs], torch.empty(2, hs, device="cuda"), i32([1, 2]))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_unrotated_elements_stay(g4, ctx, layout):
    """Elements behind rot_dim, and rows without a rotation, come out as they went
    in, infinities, NaN and signed zeros among them."""
    special = torch.tensor([torch.inf, -torch.inf, torch.nan, -0.0, 3e38, 1e-42], device="cuda")
    x = torch.randn(6, 2 * 96, device="cuda")
    for i in range(6):
        x[i, 40 + 7 * i] = special[i]
        x[i, 96 + 95 - i] = special[5 - i]
    bits = lambda t: t.contiguous().view(torch.int32)  # noqa: E731
    out = torch.empty_like(x)
    g4.Rope(ctx, 96, rot_dim=32, layout=layout).apply(x, out, i32(range(6)))
    assert torch.equal(bits(out.view(6, 2, 96)[..., 32:]), bits(x.view(6, 2, 96)[..., 32:]))
    cache = new_cache(g4, ctx, kv=(2,), hs=(96,), pages=4, seqs=1, positions=64)
    cache.resize(i32([0]), i32([6]))
    cache.append(0, x, x, x, out, i32([0] * 6), i32(range(6)))  # no rotation at all
    cache.check()
    page = int(cache.table[0, 0])
    for got in (out.view(6, 2, 96), cache.k(0)[page, :, :6].transpose(0, 1), cache.v(0)[page, :, :6].transpose(0, 1)):
        assert torch.equal(bits(got), bits(x.view(6, 2, 96)))


@pytest.mark.parametrize("scaling,attn_factor", [("none", 1.75), ("linear", 0.3), ("yarn", 1.2), ("yarn", -2.0)])
def test_rope_attn_factor(g4, ctx, scaling, attn_factor):
    """The factor on cosine and sine instead of the scaling's own."""
    rng = np.random.default_rng(2)
    pos = np.array([0, 9, 70000])
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    kw = {} if scaling == "none" else dict(factor=8.0)
    out = torch.empty(3, 128, device="cuda")
    g4.Rope(ctx, 64, rot_dim=48, scaling=scaling, attn_factor=attn_factor, **kw).apply(
        torch.from_numpy(x.reshape(3, -1)).cuda(), out, i32(pos))
    f, _ = ref.frequencies(48, 1e4, scaling, **kw)
    want = ref.rotate(x, pos, f, attn_factor, "half")
    # one more rounding than ROPE_TOL counts, the factor's, and none of the norm's
    assert np.all(abs(host(out).reshape(x.shape) - want) <= ROPE_TOL * pair_size(want, "half", 48) + 1e-30)


# ------------------------------------------------------------------ handles and streams


def test_half_given_arguments_are_refused(g4, ctx):
    cache = new_cache(g4, ctx, kv=(1,), hs=(16,), pages=4, seqs=2, positions=64)
    cache.resize(i32([0]), i32([20]))
    x, r = torch.ones(1, 16, device="cuda"), i32([0])
    for q, k, v, out in ((x, x, None, x), (x, None, x, x), (x, x, x, None), (None, x, None, None), (x, None, None, None)):
        with pytest.raises(ValueError):
            cache.append(0, q, k, v, out, r, r)
    with pytest.raises(g4.G4Error):
        cache.append(0, None, None, None, None, r, r)
    cache.check()
    assert int((cache.k(0) != 0).sum()) == 0


def test_freed_handles_are_refused(g4, ctx):
    cache = new_cache(g4, ctx, kv=(1,), hs=(16,), pages=4, seqs=2, positions=64)
    cache.resize(i32([0]), i32([20]))
    rope = g4.Rope(ctx, 16)
    x, r = torch.ones(1, 16, device="cuda"), i32([0])
    out = torch.full_like(x, 9.0)
    rope.free()
    with pytest.raises(ValueError, match="freed"):  # and not stored without a rotation
        cache.append(0, x, x, x, out, r, r, rope=rope)
    with pytest.raises(ValueError, match="freed"):
        rope.apply(x, out, r)
    cache.check()
    assert torch.all(out == 9.0) and int((cache.k(0) != 0).sum()) == 0
    cache.free()
    for call in (lambda: cache.append(0, x, x, x, out, r, r), lambda: cache.attend(0, x, out, r, r),
                 lambda: cache.resize(r, r), lambda: cache.fork(r, r), lambda: cache.copy_pages(r, r), cache.compact,
                 cache.check, lambda: cache.table, lambda: cache.k(0)):
        with pytest.raises(ValueError):
            call()


def test_calls_after_the_context_are_refused(g4):
    c = g4.Context(0)
    cache, rope = new_cache(g4, c, kv=(1,), hs=(16,), pages=4), g4.Rope(c, 16)
    x, r = torch.ones(1, 16, device="cuda"), i32([0])
    c.close()
    for call in (lambda: cache.append(0, x, x, x, x, r, r), lambda: cache.attend(0, x, x, r, r),
                 lambda: cache.resize(r, r), lambda: cache.fork(r, r), lambda: cache.copy_pages(r, r), cache.compact,
                 cache.check, lambda: rope.apply(x, x, r), lambda: g4.Rope(c, 16), lambda: new_cache(g4, c),
                 lambda: g4.beam_select(c, x, x[:, 0], 1, x[:, 0], r, r)):
        with pytest.raises(ValueError, match="closed"):
            call()


def test_arguments_freed_before_their_stream_ran(g4, ctx):
    """A call on a named stream keeps its tensors' memory from being handed out
    again until the stream has used it."""
    cache = new_cache(g4, ctx, kv=(1,), hs=(16,), pages=64, seqs=8, positions=64)
    rope = g4.Rope(ctx, 16)
    for p in (cache.k(0), cache.v(0)):
        p.copy_(torch.randn(p.shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda"))
    cache.resize(i32([2]), i32([40]))
    x = torch.randn(4, 16, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    logits, scores = torch.randn(2, 600, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda"), None
    want, turned, scores = torch.empty_like(x), torch.empty_like(x), torch.zeros(2, device="cuda")
    cache.attend(0, x, want, i32([2] * 4), i32([3, 39, 0, 20]))
    rope.apply(x, turned, i32([5, 6, 7, 8]))
    chosen = select(g4, ctx, logits, scores, 2)
    out, out2 = torch.empty_like(x), torch.empty_like(x)
    best = [torch.empty_like(t) for t in chosen]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(300_000_000)  # bounded: about 0.15 s
    at = side.cuda_stream
    cache.resize(i32([0, 1]), i32([20, 33]), stream=at)
    junk = [i32([5, 6]) for _ in range(4)]
    cache.fork(i32([0, 1]), i32([3, 4]), stream=at)
    junk += [i32([7, 7]) for _ in range(4)]
    cache.attend(0, x.clone(), out, i32([2] * 4), i32([3, 39, 0, 20]), stream=at)
    junk += [torch.zeros_like(x), i32([7] * 4), i32([1] * 4)] * 2
    rope.apply(x.clone(), out2, i32([5, 6, 7, 8]), stream=at)
    junk += [torch.zeros_like(x), i32([0] * 4)] * 2
    g4.beam_select(ctx, logits.clone(), scores.clone(), 2, *best, stream=at)
    junk += [torch.zeros_like(logits), torch.ones_like(scores)] * 2
    torch.cuda.synchronize()
    assert cache.lens.tolist() == [20, 33, 40, 20, 33, 0, 0, 0]
    assert torch.equal(out, want) and torch.equal(out2, turned)
    assert all(torch.equal(a, b) for a, b in zip(best, chosen))
    assert ctx.held  # the last call's at least
    assert cache.check() == 64 - 3 - 2 - 3
    assert not ctx.held


def test_arguments_outlive_their_stream(g4, ctx):
    """Tensors used on a batch's stream die after the batch."""
    from tests.test_decode_gpu import SPECS, _models

    _, _, model, _ = _models(g4, ctx, SPECS["q8-gqa8"], seed=21)
    batch = model.new_paged_batch(2, 32, page_size=16)
    seqs, lens = i32([0]), i32([20])
    batch.cache.resize(seqs, lens, stream=batch.stream)
    batch.free()
    model.free()
    del seqs, lens
    more = [i32([k]) for k in range(8)]
    torch.cuda.synchronize()
    assert [int(t) for t in more] == list(range(8))


def test_streams_by_number(g4, ctx):
    """The default stream by its number, and a stream that is being captured."""
    cache = new_cache(g4, ctx, "bf16", (2,), (128,), 16, 400, 4, 1600)
    cache.resize(i32(range(4)), i32([1600] * 4))
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in (cache.k(0), cache.v(0)):
        p.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    q, rows, pos = torch.randn(4, 1024, generator=g, device="cuda"), i32(range(4)), i32([1599, 700, 3, 1000])
    want, out = torch.empty_like(q), torch.zeros_like(q)
    cache.attend(0, q, want, rows, pos, scale=0.05)
    torch.cuda.synchronize()
    cache.attend(0, q, out, rows, pos, scale=0.05, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    logits, scores = torch.randn(4, 5000, generator=g, device="cuda"), torch.zeros(4, device="cuda")
    chosen = select(g4, ctx, logits, scores, 2)
    best = [torch.empty_like(t) for t in chosen]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        at = torch.cuda.current_stream().cuda_stream
        cache.attend(0, q, out, rows, pos, scale=0.05, stream=at)
        g4.beam_select(ctx, logits, scores, 2, *best, stream=at)
    for _ in range(3):
        other = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(8)]  # memory that the graph must not share
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(best, chosen))
        assert all(float(t.sum()) == 7.0 * t.numel() for t in other)
        out.zero_()


def test_no_report_is_lost_to_a_check_on_another_stream(g4, ctx):
    """Attention on one stream records a bad row around the moment when a check on
    another reads and clears the record: one of the checks reports it."""
    cache = new_cache(g4, ctx, kv=(1,), hs=(16,), pages=4, seqs=2, positions=64)
    q, out, seqs, pos = torch.ones(1, 16, device="cuda"), torch.empty(1, 16, device="cuda"), i32([0]), i32([5])
    side, other = torch.cuda.Stream(), torch.cuda.Stream()

    def reports(stream):
        try:
            cache.check(stream=stream.cuda_stream)
        except g4.G4Error:
            return 1
        return 0

    torch.cuda.synchronize()
    for i in range(600):
        with torch.cuda.stream(side):
            torch.cuda._sleep(2500 * (i % 60))
            cache.attend(0, q, out, seqs, pos)  # a visible position without a page
        seen = reports(other)
        side.synchronize()
        assert seen + reports(other) >= 1, i


def test_beam_search_in_occupied_slots_is_refused(g4, ctx):
    """A slot that holds a sequence is not searched over, and keeps it."""
    from tests.test_decode_gpu import SPECS, _models

    m, _, model, _ = _models(g4, ctx, SPECS["q8-gqa8"], seed=21)
    batch = model.new_paged_batch(6, 64, page_size=16)
    prompt = np.concatenate([[2], m.prompt(20, seed=3)]).astype(np.int32)
    want, _ = batch.beam_search(prompt, 3, 4)
    for p, t in enumerate((2, 9, 11)):
        kept, _ = batch.step([t], [p], slots=[1])
    lens = batch.cache.lens.clone()
    with pytest.raises(ValueError, match="slot"):
        batch.beam_search(prompt, 3, 4)
    assert torch.equal(batch.cache.lens, lens)
    again, _ = batch.step([11], [2], slots=[1])  # its last position once more
    assert np.array_equal(again, kept)
    batch.cache.resize(i32([1]), i32([0]), stream=batch.stream)
    got, _ = batch.beam_search(prompt, 3, 4)
    assert np.array_equal(got, want)
    batch.free()
    model.free()
