"""The paged serving operators, measured: what they compute in plain torch
operations, the calls a user makes of them, and cases over their real range.

  append   query/key norms, rotary positions, and the new K and V rows written
           into the pages of a cache (KvCache.append)
  attend   attention of one new token per row over a paged cache, with an
           optional sliding window and first tokens that stay visible
           (KvCache.attend)
  fork     beams that take over a prompt's pages and grow by one position, the
           shared last page copied (KvCache.fork, KvCache.resize)
  compact  live pages moved to the front of the pool (KvCache.compact)
  beam     the best continuations over beams and vocabulary (beam_select)

With `own` false `run` computes them with elementary torch operations, with
`own` true through the package.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
EPS = 1e-6
_ctx = []


def _package():
    import __graft_entry__

    g4 = __graft_entry__.load_package()
    if not _ctx:
        _ctx.append(g4.Context(0))
    return g4, _ctx[0]


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one token of the dense decoder configuration (8 query heads, one KV head of 256), fp32 cache
        dict(name="append_one", op="append", seqs=1, rows=1, start=200, heads=8, kv=1, hs=256, rot=256, layout="half",
             scaling="none", theta=1e6, norm=True, type="f32", page=16),
        # one step of 64 concurrent sequences of the mixture-of-experts configuration
        dict(name="append_step", op="append", seqs=64, rows=1, start=700, heads=16, kv=8, hs=256, rot=256,
             layout="half", scaling="none", theta=1e6, norm=True, type="bf16", page=32),
        # a long prompt chunk far into a context stretched eightfold, half of each head rotated, interleaved pairs
        dict(name="append_prompt", op="append", seqs=4, rows=2001, start=100000, heads=32, kv=8, hs=128, rot=64,
             layout="interleaved", scaling="yarn", theta=1e4, norm=False, type="f16", page=64),
        # the first answer token of a short question on the dense decoder configuration: latency counts
        dict(name="attend_one", op="attend", seqs=1, lo=201, hi=201, heads=8, kv=1, hs=256, window=0, sinks=0,
             type="f32", page=16),
        # 64 concurrent sequences, sliding-window layers with four first tokens kept
        dict(name="attend_window", op="attend", seqs=64, lo=100, hi=1801, heads=16, kv=8, hs=256, window=512, sinks=4,
             type="bf16", page=32),
        # one sequence at the end of a long document
        dict(name="attend_long", op="attend", seqs=1, lo=131071, hi=131071, heads=32, kv=8, hs=128, window=0, sinks=0,
             type="f16", page=64),
        # a full server: ragged sequences, eight query heads to a KV head
        dict(name="attend_server", op="attend", seqs=96, lo=33, hi=12001, heads=64, kv=8, hs=128, window=0, sinks=0,
             type="bf16", page=16),
        # four beams start from one prompt
        dict(name="fork_small", op="fork", groups=1, beams=4, length=123, layers=2, kv=1, hs=256, type="f32", page=16),
        # a batch of beam searches on a deep model
        dict(name="fork_batch", op="fork", groups=16, beams=4, length=507, layers=8, kv=8, hs=256, type="bf16", page=16),
        # a pool half full after many requests have ended, packed before it shrinks
        dict(name="compact_half", op="compact", pages=4001, live=2001, seqs=50, layers=4, kv=8, hs=128, type="f16",
             page=16),
        # a single search with a constrained vocabulary: masked logits and a finished beam
        dict(name="beam_masked", op="beam", groups=3, beams=5, vocab=32001, masked=0.75, finished=True),
        # 16 searches of 4 beams over the configurations' vocabulary
        dict(name="beam_batch", op="beam", groups=16, beams=4, vocab=262144, masked=0.0, finished=False),
    ]


def _log(rng, a, b):
    return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "fork", "compact", "beam", "beam"])
    kind = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64])
    hs = rng.choice([64, 80, 96, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
    if op == "append":
        rot = rng.choice([hs, hs, hs // 2])
        seqs = _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, rows=rng.choice([1, _log(rng, 1, max(1, 4000 // seqs))]),
                    start=_log(rng, 1, 200000), heads=heads, kv=kv, hs=hs, rot=rot,
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "yarn"]),
                    theta=rng.choice([1e4, 1e6]), norm=rng.random() < 0.5, type=kind, page=page)
    if op == "attend":
        seqs = _log(rng, 1, 128)
        budget = 2_000_000_000 // (seqs * kv * hs * 8)  # fp32 K and V of every sequence at most 2 GB
        hi = _log(rng, 1, max(1, min(100000, budget)))
        windowed = rng.random() < 0.4
        return dict(op=op, seqs=seqs, lo=_log(rng, 1, hi), hi=hi, heads=heads, kv=kv, hs=hs,
                    window=_log(rng, 1, 2000) if windowed else 0, sinks=rng.choice([0, 1, 4, 50]) if windowed else 0,
                    type=kind, page=page)
    if op == "fork":
        return dict(op=op, groups=_log(rng, 1, 16), beams=_log(rng, 2, 8), length=_log(rng, 2, 500),
                    layers=rng.choice([1, 2, 4]), kv=rng.choice([1, 2, 4]), hs=hs, type=kind, page=rng.choice([16, 32]))
    if op == "compact":
        pages = _log(rng, 40, 2000)
        return dict(op=op, pages=pages, live=rng.randint(pages // 4, 3 * pages // 4), seqs=rng.randint(1, 10),
                    layers=rng.choice([1, 2, 4]), kv=rng.choice([1, 2, 4]), hs=hs, type=kind, page=rng.choice([16, 32]))
    return dict(op=op, groups=_log(rng, 1, 16), beams=_log(rng, 1, 8), vocab=_log(rng, 1000, 262144),
                masked=rng.choice([0.0, 0.0, 0.5]), finished=rng.random() < 0.5)


def _lengths(c):
    """Context lengths of a case's sequences: lo to hi in equal steps, in a mixed order."""
    n = c["seqs"]
    at = np.arange(n) * 37 % n if math.gcd(37, n) == 1 else np.arange(n)
    return (c["lo"] + (at * (c["hi"] - c["lo"])) // max(1, n - 1)).astype(np.int64)


def _visible(c):
    """Positions that each sequence's new token sees."""
    n = _lengths(c)
    if not c["window"]:
        return n
    first = np.maximum(0, n - c["window"])
    return n - first + np.minimum(first, c["sinks"])


# ------------------------------------------------------------------ inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _pages(c, seed, first, last):
    """Pages for positions first[i] <= t < last[i] of each sequence, scattered over the pool: (table, refs)."""
    ps = c["page"]
    width = int(max(-(-last // ps)))
    have = (np.arange(width)[None] >= (first // ps)[:, None]) & (np.arange(width)[None] < (-(-last // ps))[:, None])
    total = int(have.sum())
    n_pages = total + 3
    table = np.full(have.shape, -1, np.int64)
    table[have] = np.random.default_rng(seed).permutation(n_pages)[:total]
    refs = np.zeros(n_pages, np.int64)
    refs[table[have]] = 1
    return torch.from_numpy(table.astype(np.int32)).cuda(), torch.from_numpy(refs.astype(np.int32)).cuda()


def _append_inputs(c, seed):
    g = _generator(seed)
    n = c["seqs"] * c["rows"]
    start = c["start"] + np.arange(c["seqs"])  # sequences differ by a position
    table, refs = _pages(c, seed, start, start + c["rows"])
    seqs = torch.arange(c["seqs"], device="cuda", dtype=torch.int32).repeat_interleave(c["rows"])
    pos = torch.from_numpy(np.repeat(start, c["rows"]).astype(np.int32)).cuda()
    pos += torch.arange(c["rows"], device="cuda", dtype=torch.int32).repeat(c["seqs"])
    s = dict(q=_randn(g, n, c["heads"] * c["hs"]), k=_randn(g, n, c["kv"] * c["hs"]), v=_randn(g, n, c["kv"] * c["hs"]),
             seqs=seqs, pos=pos, table=table, refs=refs, start=int(start.max()))
    if c["norm"]:
        s["q_norm"] = (1 + 0.1 * _randn(g, c["hs"])) * c["hs"] ** -0.25
        s["k_norm"] = (1 + 0.1 * _randn(g, c["hs"])) * c["hs"] ** -0.25
    return s


def _attend_inputs(c, seed):
    g = _generator(seed)
    n = _lengths(c)
    table, refs = _pages(c, seed, np.zeros_like(n), n)
    shape = (refs.numel(), c["kv"], c["page"], c["hs"])
    kind = TYPES[c["type"]]
    # scores of a few units of spread, as normed queries and keys give
    return dict(q=_randn(g, c["seqs"], c["heads"] * c["hs"]) * 2.0,
                k=[(_randn(g, *shape) * c["hs"] ** -0.5).to(kind)], v=[_randn(g, *shape).to(kind)],
                seqs=torch.arange(c["seqs"], device="cuda", dtype=torch.int32),
                pos=torch.from_numpy((n - 1).astype(np.int32)).cuda(), table=table, refs=refs)


def _fork_inputs(c, seed):
    """Prompts in sequences [0, groups), beams in the sequences behind them, each beam empty at first."""
    g = _generator(seed)
    n, b, ps = c["groups"], c["beams"], c["page"]
    own_pages = -(-c["length"] // ps)
    n_pages = n * own_pages + 2 * n * b + 1
    width = -(-(c["length"] + 1) // ps)
    table = np.full((n * (b + 1), width), -1, np.int64)
    table[:n, :own_pages] = np.random.default_rng(seed).permutation(n_pages)[:n * own_pages].reshape(n, own_pages)
    refs = np.zeros(n_pages, np.int64)
    refs[table[:n, :own_pages]] = 1
    lens = np.where(np.arange(n * (b + 1)) < n, c["length"], 0)
    shape = (n_pages, c["kv"], ps, c["hs"])
    kind = TYPES[c["type"]]
    beams = torch.arange(n, n * (b + 1), device="cuda", dtype=torch.int32)
    return dict(table=torch.from_numpy(table.astype(np.int32)).cuda(), refs=torch.from_numpy(refs.astype(np.int32)).cuda(),
                lens=torch.from_numpy(lens.astype(np.int32)).cuda(),
                k=[_randn(g, *shape).to(kind) for _ in range(c["layers"])],
                v=[_randn(g, *shape).to(kind) for _ in range(c["layers"])],
                src=torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(b), dst=beams,
                grown=torch.full((n * b,), c["length"] + 1, device="cuda", dtype=torch.int32))


def _compact_inputs(c, seed):
    """Sequences of equal shares of the live pages, which lie anywhere in the pool."""
    g = _generator(seed)
    share = -(-c["live"] // c["seqs"])
    ids = np.random.default_rng(seed).permutation(c["pages"])[:c["live"]]
    table = np.full(c["seqs"] * share, -1, np.int64)
    table[:c["live"]] = ids
    table = table.reshape(c["seqs"], share)
    refs = np.zeros(c["pages"], np.int64)
    refs[ids] = 1
    shape = (c["pages"], c["kv"], c["page"], c["hs"])
    kind = TYPES[c["type"]]
    return dict(table0=torch.from_numpy(table.astype(np.int32)).cuda(), refs0=torch.from_numpy(refs.astype(np.int32)).cuda(),
                lens0=torch.from_numpy(((table >= 0).sum(1) * c["page"]).astype(np.int32)).cuda(),
                k=[_randn(g, *shape).to(kind) for _ in range(c["layers"])],
                v=[_randn(g, *shape).to(kind) for _ in range(c["layers"])])


def _beam_inputs(c, seed):
    g = _generator(seed)
    n = c["groups"] * c["beams"]
    logits = 30.0 * torch.tanh(_randn(g, n, c["vocab"]) * 4.0 / 30.0)  # softcapped, as the decoder's output
    if c["masked"]:
        logits[torch.rand(n, c["vocab"], generator=g, device="cuda") < c["masked"]] = -math.inf
    finished = torch.zeros(n, device="cuda", dtype=torch.int32)
    if c["finished"]:
        finished[torch.rand(n, generator=g, device="cuda") < 0.25] = 1
    return dict(logits=logits, scores=-20.0 * torch.rand(n, generator=g, device="cuda"), finished=finished)


def prepare(case, seed):
    c = case
    op = c["op"]
    s = {"append": _append_inputs, "attend": _attend_inputs, "fork": _fork_inputs, "compact": _compact_inputs,
         "beam": _beam_inputs}[op](c, seed)
    s["case"] = c
    if op == "append":
        shape = (s["refs"].numel(), c["kv"], c["page"], c["hs"])
        s["k_pages"], s["v_pages"] = (torch.zeros(shape, device="cuda", dtype=TYPES[c["type"]]) for _ in "kv")
        s["q_out"] = torch.empty_like(s["q"])
    if op == "attend":
        s["out"] = torch.empty_like(s["q"])
    if op == "compact":
        s["table"], s["refs"], s["lens"] = s["table0"].clone(), s["refs0"].clone(), s["lens0"].clone()
    if op == "beam":
        n = c["groups"] * c["beams"]
        s["new_scores"] = torch.empty(n, device="cuda")
        s["parents"], s["tokens"] = (torch.empty(n, device="cuda", dtype=torch.int32) for _ in "pt")
    if own:
        _handles(s)
    return s


def _handles(s):
    """The cache and the rotary plan that a program keeps, with the case's pages in them."""
    c = s["case"]
    g4, ctx = _package()
    s["g4"], s["ctx"] = g4, ctx
    if c["op"] == "beam":
        return
    layers = c.get("layers", 1)
    width = s["table"].shape[1]
    cache = g4.KvCache(ctx, n_kv_heads=[c["kv"]] * layers, head_size=[c["hs"]] * layers, dtype=GGML[c["type"]],
                       page_size=c["page"], n_pages=s["refs"].numel(), n_seqs=s["table"].shape[0],
                       max_positions=width * c["page"])
    cache.table.copy_(s["table"])
    cache.refs.copy_(s["refs"])
    if "lens" in s:
        cache.lens.copy_(s["lens"])
    if c["op"] == "append":
        cache.k(0).zero_()
        cache.v(0).zero_()
        s["rope"] = g4.Rope(ctx, c["hs"], rot_dim=c["rot"], theta=c["theta"], layout=c["layout"], scaling=c["scaling"],
                            factor=8.0, original_ctx=4096)
    else:
        for l in range(layers):
            cache.k(l).copy_(s["k"][l])
            cache.v(l).copy_(s["v"][l])
        del s["k"], s["v"]
    s["cache"] = cache
    torch.cuda.synchronize()


# ------------------------------------------------------------------ the operators


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _append_own, "attend": _attend_own, "fork": _fork_own, "compact": _compact_own,
                "beam": _beam_own}[op](state)
    return {"append": _append_plain, "attend": _attend_plain, "fork": _fork_plain, "compact": _compact_plain,
            "beam": _beam_plain}[op](state)


def _append_own(s):
    c = s["case"]
    s["cache"].append(0, s["q"], s["k"], s["v"], s["q_out"], s["seqs"], s["pos"], rope=s["rope"],
                      q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), v_norm=c["norm"], eps=EPS)
    return {"q": s["q_out"], "k": s["cache"].k(0), "v": s["cache"].v(0)}


def _attend_own(s):
    c = s["case"]
    s["cache"].attend(0, s["q"], s["out"], s["seqs"], s["pos"], scale=1.0, window=c["window"], sinks=c["sinks"])
    return s["out"]


def _fork_own(s):
    cache = s["cache"]
    cache.fork(s["src"], s["dst"])
    cache.resize(s["dst"], s["grown"])
    layers = range(s["case"]["layers"])
    return {"table": cache.table, "lens": cache.lens, "refs": cache.refs, "k": [cache.k(l) for l in layers],
            "v": [cache.v(l) for l in layers]}


def _compact_own(s):
    cache = s["cache"]
    cache.table.copy_(s["table0"])
    cache.refs.copy_(s["refs0"])
    cache.compact()
    layers = range(s["case"]["layers"])
    return {"table": cache.table, "refs": cache.refs, "k": [cache.k(l) for l in layers],
            "v": [cache.v(l) for l in layers]}


def _beam_own(s):
    s["g4"].beam_select(s["ctx"], s["logits"], s["scores"], s["case"]["beams"], s["new_scores"], s["parents"],
                        s["tokens"], finished=s["finished"], pad_token=0)
    return {"scores": s["new_scores"], "parents": s["parents"], "tokens": s["tokens"]}


def _frequencies(c):
    """Angle per position of each rotated pair, and the factor on cosine and sine, in 64 bits."""
    rot = c["rot"]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    plain = c["theta"] ** (-2.0 * i / rot)
    if c["scaling"] == "none":
        return plain, 1.0
    if c["scaling"] == "linear":
        return plain / 8.0, 1.0
    turns = lambda r: rot * math.log(4096 / (r * 2 * math.pi)) / (2 * math.log(c["theta"]))  # noqa: E731
    low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), rot - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return plain / 8.0 * ramp + plain * (1 - ramp), 0.1 * math.log(8.0) + 1.0


def _rotate(x, c, cos, sin):
    """x [rows, heads, hs] with its first rot elements rotated; cos, sin [rows, 1, rot / 2]."""
    rot = c["rot"]
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if c["layout"] == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([u, w], -1) if c["layout"] == "half" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _rms(x):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)


def _append_plain(s):
    c = s["case"]
    n, hs, ps = s["pos"].numel(), c["hs"], c["page"]
    inv, factor = _frequencies(c)
    angle = (s["pos"].double()[:, None] * inv)[:, None]
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    q, k, v = s["q"].view(n, -1, hs), s["k"].view(n, -1, hs), s["v"].view(n, -1, hs)
    if c["norm"]:
        q, k, v = _rms(q) * s["q_norm"], _rms(k) * s["k_norm"], _rms(v)
    pos = s["pos"].long()
    page = s["table"][s["seqs"].long(), pos // ps].long()
    s["k_pages"][page, :, pos % ps] = _rotate(k, c, cos, sin).to(s["k_pages"].dtype)
    s["v_pages"][page, :, pos % ps] = v.to(s["v_pages"].dtype)
    s["q_out"].copy_(_rotate(q, c, cos, sin).view(n, -1))
    return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}


def _seen(c, pos, t):
    """[rows, positions]: whether the row's token sees position t."""
    p = pos.long()[:, None]
    seen = t <= p
    if c["window"]:
        seen = seen & ((t > p - c["window"]) | (t < c["sinks"]))
    return seen


def _attend_plain(s):
    c = s["case"]
    n, kv, hs = c["seqs"], c["kv"], c["hs"]
    pages = s["table"][s["seqs"].long()].clamp(min=0).long()
    k = s["k"][0][pages].transpose(1, 2).reshape(n, kv, -1, hs).float()
    v = s["v"][0][pages].transpose(1, 2).reshape(n, kv, -1, hs).float()
    seen = _seen(c, s["pos"], torch.arange(k.shape[2], device="cuda"))[:, None, None]
    x = torch.matmul(s["q"].view(n, kv, -1, hs), k.transpose(2, 3)).masked_fill(~seen, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    out = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    s["out"].copy_(out.reshape(n, -1))
    return s["out"]


def _count(ids, n_pages):
    """How often each page stands in ids (-1: none)."""
    ids = ids.reshape(-1).long()
    n = torch.zeros(n_pages + 1, device="cuda", dtype=torch.int32)
    n.index_add_(0, torch.where(ids < 0, n_pages, ids), torch.ones_like(ids, dtype=torch.int32))
    return n[:n_pages]


def _fork_plain(s):
    table, lens, refs, ps = s["table"], s["lens"], s["refs"], s["case"]["page"]
    src, dst = s["src"].long(), s["dst"].long()
    # the beams give back what they hold and share their parents' pages
    rows = table[src]
    refs += _count(rows, refs.numel()) - _count(table[dst], refs.numel())
    table[dst] = rows
    lens[dst] = lens[src]
    # one more position each: a page of its own where the last one is full, a copy of it where others share it
    old, new = lens[dst].long(), s["grown"].long()
    have, want = (old + ps - 1) // ps, (new + ps - 1) // ps
    last = table[dst, (have - 1).clamp(min=0)].long()
    partial = (old % ps != 0) & (new > old)
    same = (last[:, None] == last[None, :]) & partial[:, None] & partial[None, :]
    earlier = torch.tril(same, -1).sum(1)  # sharers that have taken their copy before this one
    copied = partial & (refs[last] - earlier > 1)
    need = want - have + copied
    at = torch.cumsum(need, 0) - need
    free = torch.sort((refs > 0).to(torch.int8), stable=True).indices
    target = torch.where(copied, free[at], last)
    keep = (torch.arange(ps, device="cuda") < (old % ps)[:, None])[:, None, :, None]
    for pool in s["k"] + s["v"]:
        pool[target] = torch.where(keep, pool[last], pool[target])
    refs -= _count(torch.where(copied, last, -1), refs.numel())
    refs += _count(torch.where(copied, target, -1), refs.numel())
    table[dst, (have - 1).clamp(min=0)] = target.int()
    col = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    pick = free[(at + copied)[:, None] + (col - have[:, None]).clamp(min=0)]
    table[dst] = torch.where(fresh, pick.int(), table[dst])
    refs += _count(torch.where(fresh, pick, -1), refs.numel())
    lens[dst] = new.int()
    return {"table": table, "lens": lens, "refs": refs, "k": s["k"], "v": s["v"]}


def _compact_plain(s):
    table, refs = s["table"], s["refs"]
    table.copy_(s["table0"])
    refs.copy_(s["refs0"])
    used = refs > 0
    n = int(used.sum())
    source = torch.nonzero(used[n:])[:, 0] + n
    hole = torch.nonzero(~used[:n])[:, 0]
    for pool in s["k"] + s["v"]:
        pool[hole] = pool[source]
    moved = torch.arange(refs.numel(), device="cuda", dtype=torch.int32)
    moved[source] = hole.int()
    table.copy_(torch.where(table < 0, -1, moved[table.clamp(min=0).long()]))
    refs[hole] = refs[source]
    refs[source] = 0
    return {"table": table, "refs": refs, "k": s["k"], "v": s["v"]}


def _beam_plain(s):
    c = s["case"]
    g, b, width = c["groups"], c["beams"], c["vocab"]
    # candidates of a beam are ordered by their logits alone; across beams the sums are compared in 64 bits
    best, token = torch.topk(s["logits"], min(b, width), dim=1)
    total = torch.logsumexp(s["logits"].double(), 1, keepdim=True)
    score = s["scores"].double()[:, None] + best.double() - total
    done = s["finished"].bool()[:, None]
    first = torch.arange(score.shape[1], device="cuda")[None] == 0
    score = torch.where(done, torch.where(first, s["scores"].double()[:, None], -math.inf), score)
    token = torch.where(done, 0, token)
    value, at = torch.topk(score.view(g, -1), b, dim=1)
    row = torch.arange(g, device="cuda")[:, None] * b + at // score.shape[1]
    s["new_scores"].copy_(value.reshape(-1))
    s["parents"].copy_(row.reshape(-1))
    s["tokens"].copy_(token.view(g, -1).gather(1, at).reshape(-1))
    return {"scores": s["new_scores"], "parents": s["parents"], "tokens": s["tokens"]}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    size = 4 if c.get("type") == "f32" else 2
    if c["op"] == "append":
        n, q, kv = c["seqs"] * c["rows"], c["heads"] * c["hs"], c["kv"] * c["hs"]
        return {"bytes": n * (8 * q + 8 * kv + 2 * size * kv + 12), "flops": n * 6 * (q + kv)}
    if c["op"] == "attend":
        seen = int(_visible(c).sum())
        return {"bytes": 2 * size * seen * c["kv"] * c["hs"] + 8 * c["seqs"] * c["heads"] * c["hs"] + 4 * (seen // c["page"]),
                "flops": 4 * seen * c["heads"] * c["hs"]}
    page = c.get("kv", 0) * c.get("page", 0) * c.get("hs", 0) * size * 2 * c.get("layers", 0)  # K and V, all layers
    if c["op"] == "fork":
        n = c["groups"] * c["beams"]
        filled = c["length"] % c["page"]
        width = -(-(c["length"] + 1) // c["page"])
        return {"bytes": 2 * n * page * filled // c["page"] + 4 * width * (c["groups"] + n), "flops": 0}
    if c["op"] == "compact":
        moved = c["live"] * (c["pages"] - c["live"]) // c["pages"]  # live pages expected behind the first `live`
        return {"bytes": 2 * moved * page + 8 * c["live"] + 4 * c["pages"], "flops": 0}
    n = c["groups"] * c["beams"] * c["vocab"]
    return {"bytes": 4 * n + 20 * c["groups"] * c["beams"], "flops": 3 * n}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    return {"append": _append_exact, "attend": _attend_exact, "beam": _beam_exact}.get(case["op"], lambda c, d: None)(
        case, seed)


def _append_exact(c, seed):
    s = _append_inputs(c, seed)
    n, hs, ps, rot = s["pos"].numel(), c["hs"], c["page"], c["rot"]
    pairs = []
    for i in range(rot // 2):
        f = c["theta"] ** (-2.0 * i / rot)
        if c["scaling"] == "linear":
            f /= 8.0
        elif c["scaling"] == "yarn":
            edge = [rot * math.log(4096 / (r * 2 * math.pi)) / (2 * math.log(c["theta"])) for r in (32.0, 1.0)]
            low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
            part = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
            f = f / 8.0 * part + f * (1.0 - part)
        pairs.append(f)
    factor = 0.1 * math.log(8.0) + 1.0 if c["scaling"] == "yarn" else 1.0
    turn = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda"),
                       s["pos"].double()[:, None] * torch.tensor(pairs, dtype=torch.float64, device="cuda"))[:, None]

    def norm(x, w):
        x = x.double().view(n, -1, hs)
        if not c["norm"]:
            return x
        y = x * torch.rsqrt((x ** 2).sum(-1, keepdim=True) / hs + EPS)
        return y if w is None else y * w.double()

    def rotated(x):
        x = x.clone()
        i = torch.arange(rot // 2, device="cuda")
        one, two = (i, i + rot // 2) if c["layout"] == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., one], x[..., two]) * turn
        x[..., one], x[..., two] = z.real, z.imag
        return x

    out = {"q": rotated(norm(s["q"], s.get("q_norm"))).view(n, -1)}
    place = (s["table"].long()[s["seqs"].long(), s["pos"].long() // ps] * ps + s["pos"].long() % ps)
    for name, x in (("k", rotated(norm(s["k"], s.get("k_norm")))), ("v", norm(s["v"], None))):
        pool = torch.zeros(s["refs"].numel() * ps, c["kv"], hs, dtype=torch.float64, device="cuda")
        pool[place] = x
        out[name] = pool.view(-1, ps, c["kv"], hs).transpose(1, 2).contiguous()
    return out


def _attend_exact(c, seed):
    s = _attend_inputs(c, seed)
    ps, hs, kv, n = c["page"], c["hs"], c["kv"], _lengths(c)
    out = torch.zeros(c["seqs"], kv, c["heads"] // kv, hs, dtype=torch.float64, device="cuda")
    table = s["table"].long()
    for i, length in enumerate(n.tolist()):
        t = torch.arange(length, device="cuda")
        if c["window"]:
            t = t[(t >= length - c["window"]) | (t < c["sinks"])]
        page, slot = table[i, t // ps], t % ps
        k, v = s["k"][0][page, :, slot].double(), s["v"][0][page, :, slot].double()  # [seen, kv, hs]
        x = torch.einsum("hgd,thd->hgt", s["q"][i].double().view(kv, -1, hs), k)
        out[i] = torch.einsum("hgt,thd->hgd", torch.softmax(x, -1), v)
    return out.view(c["seqs"], -1)


def _beam_exact(c, seed):
    s = _beam_inputs(c, seed)
    g, b = c["groups"], c["beams"]
    p = s["logits"].double()
    p = s["scores"].double()[:, None] + torch.log_softmax(p, 1)
    for row in torch.nonzero(s["finished"])[:, 0].tolist():
        p[row] = -math.inf
        p[row, 0] = s["scores"][row].double()
    return {"scores": torch.sort(p.view(g, -1), dim=1, descending=True).values[:, :b].reshape(-1), "parents": None,
            "tokens": None}
