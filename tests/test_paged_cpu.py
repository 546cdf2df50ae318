"""Host-side checks of the paged operators, without a GPU: refusals that come
before any device call, the Python layer's checks, and the plain forms the GPU
tests compare with."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import paged_ref as ref


@pytest.fixture
def fake(g4):
    """Zeroed memory in the place of a context: refusals write their message
    there and touch nothing else."""
    return C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


def kv_config(**kw):
    from gemma4_kt_b200._lib import KvConfigStruct

    a = dict(type=30, page_size=16, n_pages=4, n_seqs=2, max_positions=64, heads=[2], sizes=[64])
    a.update(kw)
    heads, sizes = np.array(a["heads"], np.int32), np.array(a["sizes"], np.int32)
    c = KvConfigStruct(heads.size, heads.ctypes.data, sizes.ctypes.data, a["type"], a["page_size"], a["n_pages"],
                       a["n_seqs"], a["max_positions"])
    c.keep = heads, sizes
    return c


@pytest.mark.parametrize("kw,rc", [(dict(type=8), -2), (dict(page_size=48), -1), (dict(page_size=0), -1),
                                   (dict(n_pages=0), -1), (dict(n_pages=(1 << 20) + 1), -1), (dict(n_seqs=4097), -1),
                                   (dict(max_positions=0), -1), (dict(heads=[], sizes=[]), -1), (dict(heads=[0]), -1),
                                   (dict(sizes=[4]), -1), (dict(sizes=[520]), -1), (dict(sizes=[100]), -1)])
def test_cache_configurations_refused(g4, fake, kw, rc):
    h = C.c_void_p(1)
    assert g4.lib().g4_kv_create(fake, C.byref(kv_config(**kw)), C.byref(h)) == rc
    assert not h.value and g4.lib().g4_last_error(fake)


def test_null_handles_refused(g4, fake):
    L = g4.lib()
    h = C.c_void_p()
    assert L.g4_kv_create(None, C.byref(kv_config()), C.byref(h)) == -1
    assert L.g4_kv_create(fake, None, C.byref(h)) == -1 and L.g4_kv_create(fake, C.byref(kv_config()), None) == -1
    assert L.g4_kv_free(None) == -1 and L.g4_rope_free(None) == -1
    assert L.g4_kv_resize(None, None, None, 1, None) == -1 and L.g4_kv_fork(None, None, None, 1, None) == -1
    assert L.g4_kv_compact(None, None) == -1 and L.g4_kv_copy_pages(None, None, None, 1, None) == -1
    assert L.g4_kv_check(None, None, None) == -1
    assert not L.g4_kv_k(None, 0) and not L.g4_kv_v(None, 0) and not L.g4_kv_table(None)
    assert L.g4_kv_append(None, 0, None, None, None) == -1
    assert L.g4_kv_attend(None, 0, None, None, 0, None) == -1 and L.g4_kv_attend_workspace(None, 0) == 0
    assert L.g4_rope_create(None, None, C.byref(h)) == -1 and L.g4_rope_create(fake, None, C.byref(h)) == -1
    assert L.g4_rope_apply(None, None, 0, None, 0, 1, None, 1, None) == -1


def test_rope_configurations_refused(g4, fake):
    from gemma4_kt_b200._lib import RopeConfigStruct

    good = dict(head_size=64, rot_dim=64, layout=0, scaling=0, theta=1e4, factor=1.0, original_ctx=4096, beta_fast=32.0,
                beta_slow=1.0, attn_factor=0.0)
    nan, inf = float("nan"), float("inf")
    for kw in [dict(head_size=0), dict(head_size=60), dict(head_size=1024), dict(rot_dim=0), dict(rot_dim=6),
               dict(rot_dim=68), dict(layout=2), dict(scaling=3), dict(theta=1.0), dict(theta=nan), dict(theta=inf),
               dict(scaling=1, factor=0.0), dict(scaling=1, factor=nan), dict(scaling=2, original_ctx=0),
               dict(scaling=2, beta_fast=0.0), dict(scaling=2, beta_slow=nan), dict(attn_factor=nan)]:
        h = C.c_void_p(1)
        assert g4.lib().g4_rope_create(fake, C.byref(RopeConfigStruct(**{**good, **kw})), C.byref(h)) == -1, kw
        assert not h.value


def test_beam_arguments_refused(g4, fake):
    L = g4.lib()
    p = C.cast(C.create_string_buffer(64), C.c_void_p)
    call = lambda rows=4, vocab=10, stride=10, beams=2, x=p, work=p, size=1 << 20: L.g4_beam_select(  # noqa: E731
        fake, x, stride, vocab, p, None, rows, beams, 0, p, p, p, work, size, None)
    assert call(rows=0) == 0
    for kw in [dict(rows=-2), dict(rows=3), dict(vocab=0), dict(vocab=(1 << 30) + 1, stride=1 << 31), dict(beams=0), dict(beams=33),
               dict(stride=9), dict(x=None), dict(work=None), dict(size=8)]:
        assert call(**kw) == -1, kw
    assert L.g4_beam_select_workspace(0, 10, 2) == 0 and L.g4_beam_select_workspace(4, 10, 33) == 0
    assert L.g4_beam_select_workspace(4, 1025, 2) == 4 * 2 * 8


def test_python_layer_checks_tensors(g4):
    """Tensors of another device, type or shape never reach the library."""
    cache = g4.KvCache.__new__(g4.KvCache)
    cache.ctx = type("Ctx", (), {"device": 0, "handle": None})()
    cache.handle, cache.n_kv_heads, cache.head_size, cache._work = None, [1], [8], [16]
    cache.dtype, cache._views, cache._lib = g4.GGMLType.F32, {}, g4.lib()
    x, r = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: cache.attend(0, x, x, r, r), lambda: cache.append(0, x, x, x, x, r, r),
                 lambda: cache.resize(r, r), lambda: cache.fork(r, r), lambda: cache.copy_pages(r, r),
                 lambda: cache.attend(1, x, x, r, r), lambda: cache.append(-1, x, x, x, x, r, r),
                 lambda: cache.attend(0, x[:, :7], x, r, r), lambda: cache.k(1),
                 lambda: g4.beam_select(cache.ctx, x, x[:, 0], 1, x[:, 0], r, r),
                 lambda: g4.beam_select(cache.ctx, r, x, 1, x, r, r)):
        with pytest.raises(ValueError):
            call()


def test_packed_arguments_match_the_structures():
    """The packed forms of the Python layer have the C structures' layout."""
    from gemma4_kt_b200 import _lib, paged

    assert paged._ROWS.size == C.sizeof(_lib.KvRowsStruct) and paged._QUERIES.size == C.sizeof(_lib.KvQueriesStruct)
    a = (3, 4, 11, 12, 13, 14, 21, 22, 23, 24, 31, 32, 33, 34, 1, 0.5)
    assert bytes(_lib.KvRowsStruct(*a)) == paged._ROWS.pack(*a)
    b = (3, 4, 11, 12, 21, 22, 31, 32, 0.25, 7, 8)
    assert bytes(_lib.KvQueriesStruct(*b)) == paged._QUERIES.pack(*b)


def test_plain_pages():
    """The bookkeeping the GPU tests compare with: no page is lost or held twice."""
    rng = np.random.default_rng(0)
    sim = ref.Pages(40, 6, 8, 16)
    for _ in range(400):
        op = rng.integers(0, 3)
        if op == 0:
            n = rng.integers(1, 7)
            sim.resize(rng.permutation(6)[:n], rng.integers(0, 129, n))
        elif op == 1:
            sim.fork(rng.integers(-1, 6, 6), np.arange(6))
        else:
            sim.compact()
        held = sim.table[sim.table >= 0]
        assert np.array_equal(np.bincount(held, minlength=40), sim.refs)
        assert np.array_equal((sim.table >= 0).sum(1), -(-sim.lens // 16))


def test_plain_attention_windows():
    assert ref.visible(9, 0, 0).tolist() == list(range(10))
    assert ref.visible(9, 3, 2).tolist() == [0, 1, 7, 8, 9]
    assert ref.visible(2, 100, 5).tolist() == [0, 1, 2]
    assert ref.visible(9, 1, 0).tolist() == [9]
