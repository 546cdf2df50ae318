"""Refusals of the paged operators' Python layer that need no GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture
def cache(g4):
    """A cache without a library behind it: what is refused here goes no further."""
    c = g4.KvCache.__new__(g4.KvCache)
    c.ctx = type("Ctx", (), {"device": 0, "handle": C.c_void_p(1)})()
    c.handle, c.n_kv_heads, c.head_size, c._work = C.c_void_p(1), [1], [8], [16]
    c.dtype, c._views, c._lib = g4.GGMLType.F32, {}, None
    return c


def test_half_given_arguments(cache):
    x, r = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    for q, k, v, out in ((x, x, None, x), (x, None, x, x), (x, x, x, None), (None, None, x, None), (x, None, None, None)):
        with pytest.raises(ValueError, match="together"):
            cache.append(0, q, k, v, out, r, r)


@pytest.mark.parametrize("name", ["page_size", "n_pages", "n_seqs", "max_positions"])
@pytest.mark.parametrize("excess", [2 ** 32, -2 ** 32, 2 ** 31])
def test_sizes_beyond_32_bits(g4, cache, name, excess):
    """A size is not cut to its low 32 bits (the cache's views would reach past its memory)."""
    good = dict(page_size=16, n_pages=5, n_seqs=2, max_positions=64)
    good[name] += excess
    with pytest.raises(ValueError, match=name):
        g4.KvCache(cache.ctx, [1], [8], **good)


def test_other_numbers_beyond_32_bits(g4, cache):
    x, r = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    for kw in (dict(head_size=2 ** 32 + 64), dict(head_size=64, rot_dim=2 ** 32 + 32),
               dict(head_size=64, scaling="yarn", original_ctx=2 ** 32 + 1)):
        with pytest.raises(ValueError, match="32 bits"):
            g4.Rope(cache.ctx, **kw)
    with pytest.raises(ValueError, match="beams"):
        g4.beam_select(cache.ctx, x, x[:, 0], 2 ** 32 + 2, x[:, 0], r, r)
    with pytest.raises(ValueError, match="pad_token"):
        g4.beam_select(cache.ctx, x, x[:, 0], 2, x[:, 0], r, r, pad_token=2 ** 32)
    model = g4.DecoderModel.__new__(g4.DecoderModel)
    for kw in (dict(n_max=2 ** 32 + 1), dict(max_positions=2 ** 32 + 64), dict(page_size=2 ** 32 + 16),
               dict(n_pages=2 ** 32 + 4)):
        with pytest.raises(ValueError, match="32 bits"):
            model.new_paged_batch(**{**dict(n_max=2, max_positions=64), **kw})
