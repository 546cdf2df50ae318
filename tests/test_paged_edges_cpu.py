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
