"""Paged serving: a KV cache whose pages sequences share (g4_kv), rotary
positions (g4_rope), attention over the cache and beam search's selection.

The reference keeps one contiguous cache per LlamaState
(model/LlamaState.kt:38-77) and samples one sequence (sampler/Sampler.kt);
these are the operators a server or a beam search needs next to the decoder:

    cache.fork(src, dst)               beams share their parent's pages
    cache.resize(seqs, lens)           one more position each
    cache.append(layer, q, k, v, ...)  norms, rotary positions, K/V rows
    cache.attend(layer, q, out, ...)   softmax(q k) v over the pages
    beam_select(ctx, logits, ...)      the next beams, parents for fork

Tensors are torch CUDA tensors on the context's device; every call is
asynchronous on `stream` (a cudaStream_t as a number; default: torch's current
stream of that device) and may be captured into a CUDA graph.  A named stream is
ordered behind what made the tensors by the caller; they may be dropped as soon
as the call returns.  As everywhere in this package one host thread at a time
uses a context and what was made from it: its calls on a stream share a work
space.  What a call finds wrong in device data is
skipped and reported by KvCache.check().
"""
from __future__ import annotations

import ctypes as C
import struct

import numpy as np

from ._lib import KvConfigStruct, RopeConfigStruct, check, lib
from .floattensor import Context, GGMLType, UnsupportedOperation

_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {"none": 0, "linear": 1, "yarn": 2}


# g4_kv_rows and g4_kv_queries (include/g4.h), packed: a call's arguments are
# built a few hundred nanoseconds faster than as ctypes structures.
_ROWS = struct.Struct("@iiPPPPqqqqPPPPif")
_QUERIES = struct.Struct("@iiPPqqPPfii4x")


def _stream(device: int, stream):
    if stream is not None:
        return int(stream)
    import torch

    return torch._C._cuda_getCurrentRawStream(device)  # torch.cuda.current_stream(device).cuda_stream


def _workspace(ctx: Context, n: int, stream):
    """n bytes for a call's launches.  On torch's current stream one buffer per
    stream is kept (calls on a stream follow one another); a call that is being
    captured, or names its stream, gets its own from torch's allocator, in the
    pool of the graph or stream that uses it."""
    import torch

    if stream is None:
        if torch._C._cuda_getDevice() == ctx.device and not torch._C._cuda_isCurrentStreamCapturing():
            key = torch._C._cuda_getCurrentRawStream(ctx.device)
            kept = ctx.work.get(key)
            if kept is None or kept.numel() < n:
                ctx.work[key] = kept = torch.empty(n, dtype=torch.uint8, device=torch.device("cuda", ctx.device))
            return kept
        return torch.empty(n, dtype=torch.uint8, device=torch.device("cuda", ctx.device))
    with torch.cuda.stream(torch.cuda.ExternalStream(int(stream), device=ctx.device)):
        return torch.empty(n, dtype=torch.uint8, device=torch.device("cuda", ctx.device))


def _release(ctx: Context) -> None:
    """Lets go of what _hold keeps for calls that their streams have passed."""
    import torch

    if not torch._C._cuda_isCurrentStreamCapturing():  # (a capture forbids the query)
        while ctx.held and ctx.held[0][0].query():
            ctx.held.popleft()


def _hold(ctx: Context, stream, *tensors) -> None:
    """Keeps the tensors that a call on a named stream uses until that stream has
    passed the call (seen at the next such call or check), so that torch hands
    their memory to nobody before, even if the caller drops them now.
    Tensor.record_stream would not do: it touches the stream again when the tensor
    dies, which may be after the stream (a freed batch's) has gone.  What a graph
    captures its owner keeps."""
    import torch

    _release(ctx)
    with torch.cuda.stream(torch.cuda.ExternalStream(int(stream), device=ctx.device)):
        if torch._C._cuda_isCurrentStreamCapturing():
            return
        passed = torch.cuda.Event()
        passed.record()
    ctx.held.append((passed, tensors))


def _wrong(device: int, t, name: str, dtype, what: str):
    if t.get_device() != device:
        raise ValueError(f"{name} must be a CUDA tensor on device {device}, got {t.device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    raise ValueError(f"{name} must be {what}, got {tuple(t.shape)} with strides {t.stride()}")


def _vector(device: int, t, name: str, dtype, n: int):
    """Address of a contiguous tensor of n entries."""
    if t.get_device() != device or t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        _wrong(device, t, name, dtype, f"contiguous with {n} entries")
    return t.data_ptr()


def _matrix(device: int, t, name: str, dtype, rows: int, width: int):
    """Address of a [rows, width] tensor with consecutive columns, and the
    entries between its rows."""
    if t.get_device() == device and t.dtype == dtype and t.shape == (rows, width):
        step, one = t.stride()
        if one == 1 or width <= 1:
            return t.data_ptr(), step
    _wrong(device, t, name, dtype, f"[{rows}, {width}] with consecutive columns")


def _int32(**values) -> None:
    """Refuses what a C int does not hold: ctypes would pass its low bits on."""
    for name, v in values.items():
        if not -2 ** 31 <= v < 2 ** 31:
            raise ValueError(f"{name} {v} is beyond 32 bits")


def _open(ctx: Context, what: str) -> None:
    if not ctx.handle:
        raise ValueError(f"{what}: the context is closed")


def _failed(rc: int, ctx: Context, handle, what: str) -> None:
    """Raises what a call's status says; a handle that was freed, or whose context
    is closed, reaches the library as NULL."""
    _open(ctx, what)
    if not handle:
        raise ValueError(f"{what}: it was freed")
    check(rc, ctx.handle, what)


class _Owner:
    """Frees a handle when the last object that uses its memory is gone."""

    def __init__(self, handle, release):
        self.handle, self.release = handle, release

    def free(self) -> None:
        if self.handle:
            self.release(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class _DeviceArray:
    """Device memory of a cache for torch.as_tensor (the tensor keeps its owner alive)."""

    def __init__(self, owner, ptr: int, shape, typestr: str):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape), "typestr": typestr, "version": 2}


class Rope:
    """A rotary plan (g4_rope).  layout "half" pairs element m with m + rot_dim/2,
    "interleaved" 2m with 2m + 1; scaling "none", "linear" or "yarn" for
    contexts `factor` times longer; freq_factors: the model's rope_freqs."""

    def __init__(self, ctx: Context, head_size: int, rot_dim: int | None = None, theta: float = 10000.0,
                 layout: str = "half", scaling: str = "none", factor: float = 1.0, original_ctx: int = 4096,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 0.0, freq_factors=None):
        _open(ctx, "Rope")
        _int32(head_size=head_size, rot_dim=0 if rot_dim is None else rot_dim, original_ctx=original_ctx)
        if layout not in _LAYOUTS or scaling not in _SCALINGS:
            raise ValueError(f"layout {layout!r} (half, interleaved), scaling {scaling!r} (none, linear, yarn)")
        rot_dim = head_size if rot_dim is None else rot_dim
        ff = None if freq_factors is None else np.ascontiguousarray(freq_factors, np.float32)
        if ff is not None and ff.size != rot_dim // 2:
            raise ValueError(f"freq_factors must hold {rot_dim // 2} values, got {ff.size}")
        cfg = RopeConfigStruct(head_size, rot_dim, _LAYOUTS[layout], _SCALINGS[scaling], theta, factor, original_ctx,
                               beta_fast, beta_slow, attn_factor, None if ff is None else ff.ctypes.data)
        h = C.c_void_p()
        rc = lib().g4_rope_create(ctx.handle, C.byref(cfg), C.byref(h))
        if rc == -1:
            raise ValueError(ctx.last_error())
        check(rc, ctx.handle, "g4_rope_create")
        self.ctx, self.head_size, self.handle = ctx, head_size, h
        self._owner = _Owner(h, lib().g4_rope_free)
        self._apply = lib().g4_rope_apply

    def free(self) -> None:
        self.handle = None
        self._owner.free()

    def apply(self, x, out, pos, stream=None) -> None:
        """out = x [rows, heads * head_size] (fp32) rotated at positions pos
        [rows] (int32); out may be x; rows at negative positions stay."""
        import torch

        dev = self.ctx.device
        rows, width = x.shape if x.dim() == 2 else (0, 0)
        if not width or width % self.head_size:
            raise ValueError(f"x must be [rows, heads * {self.head_size}], got {tuple(x.shape)}")
        xp, xs = _matrix(dev, x, "x", torch.float32, rows, width)
        op, os_ = _matrix(dev, out, "out", torch.float32, rows, width)
        pp = _vector(dev, pos, "pos", torch.int32, rows)
        rc = self._apply(self.handle if self.ctx.handle else None, xp, xs, op, os_, width // self.head_size, pp, rows,
                         _stream(dev, stream))
        if rc:
            _failed(rc, self.ctx, self.handle, "g4_rope_apply")
        if stream is not None:
            _hold(self.ctx, stream, x, out, pos)


class KvCache:
    """A paged KV cache (g4_kv): n_pages pages of page_size positions in every
    layer, shared by up to n_seqs sequences of at most max_positions."""

    def __init__(self, ctx: Context, n_kv_heads, head_size, dtype=GGMLType.BF16, page_size: int = 32,
                 n_pages: int = 1024, n_seqs: int = 64, max_positions: int = 4096):
        _open(ctx, "KvCache")
        _int32(page_size=page_size, n_pages=n_pages, n_seqs=n_seqs, max_positions=max_positions)
        heads, sizes = np.array(n_kv_heads, np.int32), np.array(head_size, np.int32)
        if heads.ndim != 1 or heads.shape != sizes.shape or not heads.size:
            raise ValueError("n_kv_heads and head_size must list the same layers")
        cfg = KvConfigStruct(heads.size, heads.ctypes.data, sizes.ctypes.data, int(dtype), page_size, n_pages, n_seqs,
                             max_positions)
        h = C.c_void_p()
        rc = lib().g4_kv_create(ctx.handle, C.byref(cfg), C.byref(h))
        if rc == -2:
            raise UnsupportedOperation(ctx.last_error())
        if rc == -1:
            raise ValueError(ctx.last_error())
        check(rc, ctx.handle, "g4_kv_create")
        self._describe(ctx, h, _Owner(h, lib().g4_kv_free), heads, sizes, dtype, page_size, n_pages, n_seqs,
                       max_positions)

    @staticmethod
    def _of_batch(ctx: Context, batch_handle, *description) -> "KvCache":
        """The cache of a paged batch, which owns it: it and its views end with the batch."""
        cache = KvCache.__new__(KvCache)
        cache._describe(ctx, C.c_void_p(lib().g4_batch_kv(batch_handle)), _Owner(None, None), *description)
        return cache

    def _describe(self, ctx, handle, owner, heads, sizes, dtype, page_size, n_pages, n_seqs, max_positions) -> None:
        self.ctx, self.handle, self._owner = ctx, handle, owner
        self.n_kv_heads, self.head_size = [int(x) for x in heads], [int(x) for x in sizes]
        self.dtype, self.page_size, self.n_pages, self.n_seqs = GGMLType(int(dtype)), page_size, n_pages, n_seqs
        self.max_positions, self.max_pages = max_positions, -(-max_positions // page_size)
        self._work = [lib().g4_kv_attend_workspace(handle, l) for l in range(len(self.head_size))]
        self._views = {}
        self._lib = lib()

    def free(self) -> None:
        """Release the pages (no view of them is used afterwards)."""
        self._views.clear()
        self.handle = None
        self._owner.free()

    # ---- the device state as tensors
    def _view(self, key, ptr, shape, typestr: str):
        t = self._views.get(key)
        if t is None:
            import torch

            at = ptr()
            if not at:
                raise ValueError(f"no {key[0]} {key[1:]} in this cache")
            t = torch.as_tensor(_DeviceArray(self._owner, at, shape, typestr), device=f"cuda:{self.ctx.device}")
            if typestr == "<i2":
                t = t.view(torch.bfloat16)
            self._views[key] = t
        return t

    def _pool(self, name: str, layer: int):
        kind = {GGMLType.F32: "<f4", GGMLType.F16: "<f2", GGMLType.BF16: "<i2"}[self.dtype]
        if not 0 <= layer < len(self.head_size):
            raise ValueError(f"layer {layer} of {len(self.head_size)}")
        return self._view((name, layer), lambda: getattr(lib(), "g4_kv_" + name)(self.handle, layer),
                          (self.n_pages, self.n_kv_heads[layer], self.page_size, self.head_size[layer]), kind)

    def k(self, layer: int):
        """K rows of a layer: [n_pages, n_kv_heads, page_size, head_size]."""
        return self._pool("k", layer)

    def v(self, layer: int):
        """V rows of a layer: [n_pages, n_kv_heads, page_size, head_size]."""
        return self._pool("v", layer)

    @property
    def table(self):
        """Page of each position range of each sequence [n_seqs, max_pages], -1: none."""
        return self._view(("table",), lambda: lib().g4_kv_table(self.handle), (self.n_seqs, self.max_pages), "<i4")

    @property
    def lens(self):
        """Positions each sequence has pages for [n_seqs]."""
        return self._view(("lens",), lambda: lib().g4_kv_lens(self.handle), (self.n_seqs,), "<i4")

    @property
    def refs(self):
        """Sequences that hold each page [n_pages]."""
        return self._view(("refs",), lambda: lib().g4_kv_refs(self.handle), (self.n_pages,), "<i4")

    # ---- pages
    def _pairs(self, fn, a, b, names, stream):
        import torch

        dev, n = self.ctx.device, a.numel()
        ap = _vector(dev, a, names[0], torch.int32, n)
        bp = _vector(dev, b, names[1], torch.int32, n)
        rc = fn(self.handle if self.ctx.handle else None, ap, bp, n, _stream(dev, stream))
        if rc:
            _failed(rc, self.ctx, self.handle, fn.__name__)
        if stream is not None:
            _hold(self.ctx, stream, a, b)

    def resize(self, seqs, lens, stream=None) -> None:
        """Pages for lens[i] positions of sequence seqs[i] (int32 tensors; 0 frees
        it); a shared, partly filled last page is copied when a sequence grows
        into it.  Without enough free pages nothing changes (check())."""
        self._pairs(self._lib.g4_kv_resize, seqs, lens, ("seqs", "lens"), stream)

    def fork(self, src, dst, stream=None) -> None:
        """Sequence dst[i] shares the pages of src[i] as they were before the call
        (its own are given back); negative entries are padding."""
        self._pairs(self._lib.g4_kv_fork, src, dst, ("src", "dst"), stream)

    def copy_pages(self, src, dst, stream=None) -> None:
        """Whole pages src[i] -> dst[i] in every layer."""
        self._pairs(self._lib.g4_kv_copy_pages, src, dst, ("src", "dst"), stream)

    def compact(self, stream=None) -> None:
        """Live pages to the front of the pool; the table follows."""
        rc = self._lib.g4_kv_compact(self.handle if self.ctx.handle else None, _stream(self.ctx.device, stream))
        if rc:
            _failed(rc, self.ctx, self.handle, "g4_kv_compact")

    def check(self, stream=None) -> int:
        """Wait for the stream; raise what the cache's calls recorded, else the
        number of free pages."""
        n = C.c_int()
        rc = self._lib.g4_kv_check(self.handle if self.ctx.handle else None, C.byref(n), _stream(self.ctx.device, stream))
        if self.ctx.held:
            _release(self.ctx)
        if rc:
            _failed(rc, self.ctx, self.handle, "g4_kv_check")
        return n.value

    # ---- rows
    def append(self, layer: int, q, k, v, q_out, seqs, pos, rope: Rope | None = None, q_norm=None, k_norm=None,
               v_norm: bool = False, eps: float = 1e-6, stream=None) -> None:
        """Row i is position pos[i] of sequence seqs[i]: its K and V rows, normed
        and rotated, go into their page, its normed and rotated queries to q_out
        (which may be q; q and q_out None: K and V alone; k and v None: queries
        alone, for a layer that reads another layer's cache).  fp32 rows
        [rows, heads * head_size] with any row stride."""
        import torch

        dev, f32, i32, n = self.ctx.device, torch.float32, torch.int32, pos.numel()
        if not 0 <= layer < len(self.head_size):
            raise ValueError(f"layer {layer} of {len(self.head_size)}")
        if (k is None) is not (v is None) or (q is not None and q_out is None):
            raise ValueError("k and v go together, and q needs q_out")
        hs, width = self.head_size[layer], self.n_kv_heads[layer] * self.head_size[layer]
        heads = qp = qs = op = os_ = kp = ks = vp = vs = 0
        if k is not None:
            kp, ks = _matrix(dev, k, "k", f32, n, width)
            vp, vs = _matrix(dev, v, "v", f32, n, width)
        if q is not None:
            wide = q.shape[-1]
            heads = wide // hs
            if not heads or heads * hs != wide:
                raise ValueError(f"q must be [rows, heads * {hs}], got {tuple(q.shape)}")
            qp, qs = _matrix(dev, q, "q", f32, n, wide)
            op, os_ = _matrix(dev, q_out, "q_out", f32, n, wide)
        rows = _ROWS.pack(n, heads, qp, kp, vp, op, qs, ks, vs, os_, _vector(dev, seqs, "seqs", i32, n),
                          _vector(dev, pos, "pos", i32, n),
                          0 if q_norm is None else _vector(dev, q_norm, "q_norm", f32, hs),
                          0 if k_norm is None else _vector(dev, k_norm, "k_norm", f32, hs), bool(v_norm), eps)
        turns = None
        if rope is not None:
            turns = rope.handle
            if not turns:  # NULL would store the rows without a rotation
                raise ValueError("the rotary plan was freed")
        rc = self._lib.g4_kv_append(self.handle if self.ctx.handle else None, layer, rows, turns, _stream(dev, stream))
        if rc:
            _failed(rc, self.ctx, self.handle, "g4_kv_append")
        if stream is not None:
            _hold(self.ctx, stream, q, k, v, q_out, seqs, pos, q_norm, k_norm)

    def attend(self, layer: int, q, out, seqs, pos, scale: float = 1.0, window: int = 0, sinks: int = 0,
               stream=None) -> None:
        """out[i] = softmax(scale * q[i] . K) V over the positions t <= pos[i] of
        sequence seqs[i]; with a window those above pos[i] - window and the first
        `sinks`.  fp32 rows [rows, heads * head_size] with any row stride; rows
        of negative sequences stay, rows at negative positions get zeros."""
        import torch

        dev, f32, i32, n = self.ctx.device, torch.float32, torch.int32, pos.numel()
        if not 0 <= layer < len(self.head_size):
            raise ValueError(f"layer {layer} of {len(self.head_size)}")
        hs, wide = self.head_size[layer], q.shape[-1]
        heads = wide // hs
        if not heads or heads * hs != wide:
            raise ValueError(f"q must be [rows, heads * {hs}], got {tuple(q.shape)}")
        qp, qs = _matrix(dev, q, "q", f32, n, wide)
        op, os_ = _matrix(dev, out, "out", f32, n, wide)
        rows = _QUERIES.pack(n, heads, qp, op, qs, os_, _vector(dev, seqs, "seqs", i32, n),
                             _vector(dev, pos, "pos", i32, n), scale, window, sinks)
        work = _workspace(self.ctx, self._work[layer], stream)
        rc = self._lib.g4_kv_attend(self.handle if self.ctx.handle else None, layer, rows, work.data_ptr(),
                                    self._work[layer], _stream(dev, stream))
        if rc:
            _failed(rc, self.ctx, self.handle, "g4_kv_attend")
        if stream is not None:
            _hold(self.ctx, stream, q, out, seqs, pos)


def beam_select(ctx: Context, logits, scores, beams: int, new_scores, parents, tokens, finished=None,
                pad_token: int = 0, stream=None) -> None:
    """The `beams` best continuations of every group of `beams` rows of logits
    [rows, vocab] (fp32): new_scores (fp32; may be scores), parents (int32 rows,
    KvCache.fork's src) and tokens (int32), best first; -1 where too few remain.
    finished (int32): rows whose one continuation is pad_token at their score."""
    import torch

    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    dev, f32, i32 = ctx.device, torch.float32, torch.int32
    rows, vocab = logits.shape
    _int32(vocab=vocab, beams=beams, pad_token=pad_token)
    L = lib()
    lp, ls = _matrix(dev, logits, "logits", f32, rows, vocab)
    sp = _vector(dev, scores, "scores", f32, rows)
    fp = None if finished is None else _vector(dev, finished, "finished", i32, rows)
    np_ = _vector(dev, new_scores, "new_scores", f32, rows)
    pp = _vector(dev, parents, "parents", i32, rows)
    tp = _vector(dev, tokens, "tokens", i32, rows)
    work = _workspace(ctx, L.g4_beam_select_workspace(rows, vocab, beams), stream)
    rc = L.g4_beam_select(ctx.handle, lp, ls, vocab, sp, fp, rows, beams, pad_token, np_, pp, tp, work.data_ptr(),
                          work.numel(), _stream(dev, stream))
    if rc:
        _failed(rc, ctx, ctx.handle, "g4_beam_select")
    if stream is not None:
        _hold(ctx, stream, logits, scores, new_scores, parents, tokens, finished)
