"""The batched decoder over a paged KV cache (g4_batch_create_paged) against the
CPU oracle: staggered sequences, prompt chunks across page borders, slots
forked from a shared prompt, and beam search against the same search over
oracle states."""
import math

import numpy as np
import pytest
import torch

from oracle import oracle
from tests.conftest import rel_l2
from tests.test_decode_gpu import SPECS, _models

pytestmark = pytest.mark.gpu
TOL = 1e-3  # relative L2 of the logits, as for the contiguous batch


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("name,page", [("q8-swa-shared-noV", 16), ("q8-gqa8", 32)])
def test_paged_batch_vs_oracle(g4, ctx, name, page):
    m, src, model, _ = _models(g4, ctx, SPECS[name], seed=21)
    n_seq, steps, prompt_len = 5, 40, 12
    batch = model.new_paged_batch(n_seq, 48, page_size=page)
    orcs = [oracle.ModelOracle(src) for _ in range(n_seq)]
    prompts = [m.prompt(prompt_len, seed=1000 + i) for i in range(n_seq)]
    pos, tok = [0] * n_seq, [2] * n_seq
    for step in range(steps):
        n = min(n_seq, step // 3 + 1)
        lg, nt = batch.step(tok[:n], pos[:n])
        for i in range(n):
            want = orcs[i].step(tok[i], pos[i])
            assert rel_l2(lg[i], want) < TOL, (name, i, pos[i])
            k = pos[i]
            if k < prompt_len:
                tok[i] = int(prompts[i][k])
            else:
                assert nt[i] == int(np.argmax(want)), (name, i, pos[i])
                tok[i] = int(nt[i])
            pos[i] += 1
    lens = batch.cache.lens.cpu().numpy()
    assert lens.tolist() == pos
    assert batch.cache.check(stream=batch.stream) == batch.n_pages - sum(-(-p // page) for p in pos)
    for o in orcs:
        o.close()
    batch.free()
    model.free()


def test_paged_batch_moe(g4, ctx, monkeypatch):
    """MoE layers beside the paged attention (the fp32 expert kernels, as in the
    contiguous batch's test)."""
    monkeypatch.setenv("G4_MOE_TC", "0")
    m, src, model, _ = _models(g4, ctx, SPECS["moe"], seed=39)
    batch = model.new_paged_batch(2, 32, page_size=16)
    orcs = [oracle.ModelOracle(src) for _ in range(2)]
    prompts = [np.concatenate([[2], m.prompt(11, seed=6000 + i)]) for i in range(2)]
    for p in range(12):
        lg, _ = batch.step([int(t[p]) for t in prompts], [p, p])
        for i in range(2):
            assert rel_l2(lg[i], orcs[i].step(int(prompts[i][p]), p)) < TOL, (i, p)
    for o in orcs:
        o.close()
    batch.free()
    model.free()


def test_paged_prefill_and_forks(g4, ctx):
    """One prompt in chunks that cross page borders, three slots forked from it,
    each going its own way: the shared pages stay, the last one is copied."""
    m, src, model, _ = _models(g4, ctx, SPECS["q8-swa-shared-noV"], seed=21)
    batch = model.new_paged_batch(20, 64, page_size=16, n_pages=12)
    prompt = np.concatenate([[2], m.prompt(36, seed=5)]).astype(np.int32)
    orcs = [oracle.ModelOracle(src) for _ in range(4)]
    want = [o.step(int(t), p) for p, t in enumerate(prompt) for o in orcs[:1]]
    for o in orcs[1:]:
        for p, t in enumerate(prompt):
            o.step(int(t), p)
    for a, b in ((0, 20), (20, 37)):
        lg, _ = batch.step(prompt[a:b], np.arange(a, b), slots=np.zeros(b - a))
        for i, p in enumerate(range(a, b)):
            assert rel_l2(lg[i], want[p]) < TOL, p
    batch.cache.fork(i32([0, 0, 0]), i32([1, 2, 3]), stream=batch.stream)
    assert batch.cache.check(stream=batch.stream) == 12 - 3
    for step in range(6):
        toks = [100 + 7 * s + step for s in range(4)]
        lg, _ = batch.step(toks, [37 + step] * 4)
        for s in range(4):
            assert rel_l2(lg[s], orcs[s].step(toks[s], 37 + step)) < TOL, (step, s)
    # two full pages shared by four, one last page each
    assert batch.cache.check(stream=batch.stream) == 12 - 2 - 4
    assert sorted(batch.cache.refs.cpu().tolist()) == [0] * 6 + [1] * 4 + [4] * 2
    batch.cache.resize(i32([1, 0]), i32([0, 0]), stream=batch.stream)
    batch.cache.compact(stream=batch.stream)
    for s in (2, 3):  # the others go on, their pages moved
        lg, _ = batch.step([9], [43], slots=[s])
        assert rel_l2(lg[0], orcs[s].step(9, 43)) < TOL
    assert batch.cache.refs[:4].min() > 0 and batch.cache.refs[4:].max() == 0
    for o in orcs:
        o.close()
    batch.free()
    model.free()


@pytest.mark.parametrize("dtype", [1, 30])
def test_paged_batch_16_bit_cache(g4, ctx, dtype):
    """K and V rounded to 16 bits (half a step: 2^-11 for f16, 2^-8 for bf16 of
    each element).  A layer's attention output is off by at most that much of its
    values plus the scores' change; over four layers and the residual stream the
    logits stay within 16 half steps."""
    _, src, model, _ = _models(g4, ctx, SPECS["q8-gqa8"], seed=21)
    batch = model.new_paged_batch(2, 40, page_size=16, dtype=dtype)
    orc = oracle.ModelOracle(src)
    tok = 2
    for p in range(30):
        lg, _ = batch.step([tok], [p])
        want = orc.step(tok, p)
        assert rel_l2(lg[0], want) < 16 * (2.0 ** -11 if dtype == 1 else 2.0 ** -8), p
        tok = int(np.argmax(want))
    orc.close()
    batch.free()
    model.free()


def test_paged_batch_without_pages(g4, ctx):
    _, _, model, _ = _models(g4, ctx, SPECS["q8-gqa8"], seed=21)
    batch = model.new_paged_batch(3, 64, page_size=16, n_pages=2)
    batch.step([2, 2], [0, 0])
    with pytest.raises(g4.G4Error, match="NOMEM.*free pages"):
        batch.step([2], [0], slots=[2])
    for p in range(1, 16):
        batch.step([5, 6], [p, p])
    with pytest.raises(g4.G4Error, match="free pages"):
        batch.step([5, 6], [16, 16])
    batch.cache.resize(i32([1]), i32([0]), stream=batch.stream)
    a, _ = batch.step([5], [16])
    # the same history in a contiguous batch
    other = model.new_batch(1, 64)
    other.step([2], [0])
    for p in range(1, 16):
        other.step([5], [p])
    b, _ = other.step([5], [16])
    assert rel_l2(a, b) < TOL
    # a position that other slots share is not overwritten
    batch.cache.fork(i32([0]), i32([2]), stream=batch.stream)
    with pytest.raises(g4.G4Error, match="shared"):
        batch.step([7], [3])
    for kw in (dict(page_size=24), dict(n_pages=0), dict(dtype=8)):
        with pytest.raises(g4.G4Error):
            model.new_paged_batch(2, 64, **kw)
    other.free()
    batch.free()
    model.free()


def oracle_beams(src, prompt, beams, n, eos):
    """The search over oracle states; also the smallest gap between a chosen and
    the best rejected score."""
    def state(tokens):
        o = oracle.ModelOracle(src)
        for p, t in enumerate(tokens):
            lg = o.step(int(t), p)
        o.close()
        return lg

    live = [(0.0, [], False)]
    margin = math.inf
    for _ in range(n):
        cand = []
        for i, (score, toks, done) in enumerate(live):
            if done:
                cand.append((-score, i, 0, toks + [0], True))
                continue
            x = state(list(prompt) + toks).astype(np.float64)
            lse = x.max() + math.log(np.exp(x - x.max()).sum())
            for t in np.argsort(-x, kind="stable")[:beams + 1]:
                cand.append((-(score + x[t] - lse), i, int(t), toks + [int(t)], int(t) == eos))
        cand.sort(key=lambda c: c[:3])
        if len(cand) > beams:
            margin = min(margin, cand[beams][0] - cand[beams - 1][0])
        margin = min([margin] + [b[0] - a[0] for a, b in zip(cand[:beams], cand[1:beams])])
        live = [(-c[0], c[3], c[4]) for c in cand[:beams]]
    return np.array([t for _, t, _ in live]), np.array([s for s, _, _ in live]), margin


@pytest.mark.parametrize("prompt_len,beams,with_eos", [(7, 3, False), (33, 4, True)])
def test_beam_search_vs_oracle(g4, ctx, prompt_len, beams, with_eos):
    m, src, model, _ = _models(g4, ctx, SPECS["q8-gqa8"], seed=21)
    batch = model.new_paged_batch(8, 64, page_size=16)
    prompt = np.concatenate([[2], m.prompt(prompt_len - 1, seed=3)]).astype(np.int32)
    n, eos = 6, None
    if with_eos:  # a token that the search chooses early ends a beam
        eos = int(oracle_beams(src, prompt, beams, 2, None)[0][1, 1])
    tokens, scores, margin = oracle_beams(src, prompt, beams, n, eos)
    assert margin > 1e-4, "ill-conditioned fixture"
    got, got_scores = batch.beam_search(prompt, beams, n, eos=eos)
    assert np.array_equal(got, tokens)
    assert np.allclose(got_scores, scores, atol=1e-3)
    again, _ = batch.beam_search(prompt, beams, n, eos=eos)  # the slots were given back
    assert np.array_equal(again, got)
    assert batch.cache.check(stream=batch.stream) == batch.n_pages
    with pytest.raises(ValueError):
        batch.beam_search(prompt, 9, n)
    with pytest.raises(ValueError):
        batch.beam_search(prompt, beams, 64)
    batch.free()
    model.free()
