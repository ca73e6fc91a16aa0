"""The paged cache's refusals: every entry point looks its arguments over before it needs a device, so all of this runs
without a GPU (pointers are plain numbers that nothing follows)."""
import ctypes as C

import pytest

from tests import helpers

P = 1 << 20   # an address; never read


@pytest.fixture(scope="module")
def nat():
    helpers.build_library()
    from lazyweights_b200 import _native
    return _native


GOOD = dict(k=P, v=P, type=0, pages=10, heads=4, size=16, dim=128, ps=4 * 16 * 128, hs=16 * 128, ts=128)


def create(nat, **kw):
    a = dict(GOOD, **kw)
    return nat.lib().lw_cache_create(*(a[n] for n in ("k", "v", "type", "pages", "heads", "size", "dim", "ps", "hs", "ts")))


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(type=2), dict(type=-1), dict(pages=0), dict(heads=0), dict(size=0),
                                dict(size=4), dict(size=12), dict(size=1 << 17), dict(dim=0), dict(dim=4), dict(dim=100), dict(dim=136),
                                dict(k=P + 8), dict(v=P + 2), dict(ps=0), dict(ps=-2048), dict(hs=0), dict(ts=120), dict(ts=132),
                                dict(hs=2044), dict(ps=1 << 40)])
def test_pools_that_are_refused(nat, kw):
    assert not create(nat, **kw)
    assert nat.lib().lw_last_status() == nat.LW_ERR_ARG
    assert b"lw_cache_create" in nat.lib().lw_last_error()


@pytest.mark.parametrize("kw", [{}, dict(type=1), dict(size=8), dict(size=24), dict(dim=8, ts=8), dict(pages=1, ps=0), dict(heads=1, hs=3),
                                dict(ts=512, hs=128, ps=512 * 16)])   # heads inside the positions of a page
def test_pools_that_are_taken(nat, kw):
    h = create(nat, **kw)
    assert h and nat.lib().lw_last_status() == 0
    nat.lib().lw_cache_destroy(h)


APPEND = dict(qkv=P, qkv_type=2, row_stride=16 * 128, rows=3, heads=8, cos=P, sin=P, rope_rows=100, rope_half=64, starts=P, lens=P, table=P,
              n=2, cols=5, tstride=5, q=P, qt=8 * 128, qh=128, stream=None)
ATTEND = dict(q=P, qt=8 * 128, qh=128, rows=2, heads=8, lens=P, table=P, cols=5, tstride=5, scale=1.0, window=0, out=P, ot=8 * 128, oh=128,
              space=P, size=1 << 40, stream=None)
PROMPT = dict(q=P, qt=8 * 128, qh=128, rows=7, heads=8, starts=P, lens=P, table=P, n=2, cols=5, tstride=5, scale=1.0, window=0, out=P,
              ot=8 * 128, oh=128, space=P, size=1 << 40, stream=None)

SEQUENCES = [dict(lens=None), dict(table=None), dict(cols=0), dict(tstride=4), dict(rows=0), dict(rows=-1), dict(heads=0), dict(heads=6)]
ROWS = [dict(q=None), dict(q=P + 8), dict(qt=1028), dict(qh=132), dict(qh=64), dict(qt=8), dict(qt=512)]
RESULTS = [dict(out=None), dict(out=P + 2), dict(ot=1020), dict(oh=120), dict(ot=1016), dict(scale=float("nan")), dict(scale=float("inf")),
           dict(window=-1)]


def refused(nat, fn, base, kw):
    h = create(nat)
    try:
        a = dict(base, **kw)
        assert getattr(nat.lib(), fn)(h, *a.values()) == nat.LW_ERR_ARG
        assert fn.encode() in nat.lib().lw_last_error()
        assert getattr(nat.lib(), fn)(None, *dict(base).values()) == nat.LW_ERR_ARG
    finally:
        nat.lib().lw_cache_destroy(h)


@pytest.mark.parametrize("kw", SEQUENCES + ROWS + [dict(n=0), dict(starts=None, rows=1), dict(qkv=None), dict(cos=None), dict(sin=None),
                                                   dict(qkv_type=3), dict(row_stride=2047), dict(qkv=P + 2), dict(rope_rows=0),
                                                   dict(rope_half=0), dict(rope_half=2), dict(rope_half=68), dict(cos=P + 2)])
def test_append_refuses(nat, kw):
    refused(nat, "lw_cache_append", APPEND, kw)


@pytest.mark.parametrize("kw", SEQUENCES + ROWS + RESULTS)
def test_attend_refuses(nat, kw):
    refused(nat, "lw_cache_attend", ATTEND, kw)


@pytest.mark.parametrize("kw", SEQUENCES + ROWS + RESULTS + [dict(n=0), dict(starts=None)])
def test_attend_prompt_refuses(nat, kw):
    refused(nat, "lw_cache_attend_prompt", PROMPT, kw)


def test_a_workspace_too_small_is_refused(nat):
    h = create(nat)
    try:
        for prompt, fn, base in ((0, "lw_cache_attend", ATTEND), (1, "lw_cache_attend_prompt", PROMPT)):
            need = nat.lib().lw_cache_workspace(h, base["heads"], prompt)
            assert need > 0
            for kw in (dict(size=need - 1), dict(space=None), dict(space=P + 8)):
                assert getattr(nat.lib(), fn)(h, *dict(base, **kw).values()) == nat.LW_ERR_ARG
        for bad in ((0, 0), (6, 1), (-4, 0)):
            assert nat.lib().lw_cache_workspace(h, *bad) == nat.LW_ERR_ARG
        assert nat.lib().lw_cache_workspace(None, 8, 0) == nat.LW_ERR_ARG
    finally:
        nat.lib().lw_cache_destroy(h)


def test_without_a_device_good_calls_say_so(nat):
    n = C.c_int(0)
    try:
        rt = C.CDLL("libcudart.so.12")
        if rt.cudaGetDeviceCount(C.byref(n)) == 0 and n.value:
            pytest.skip("there is a device: the pointers above would be followed")
    except OSError:
        import torch
        if torch.cuda.is_available():
            pytest.skip("there is a device: the pointers above would be followed")
    h = create(nat)
    for fn, base in (("lw_cache_append", APPEND), ("lw_cache_attend", ATTEND), ("lw_cache_attend_prompt", PROMPT)):
        assert getattr(nat.lib(), fn)(h, *base.values()) == nat.LW_ERR_NO_DEVICE
    nat.lib().lw_cache_destroy(h)


def test_python_refuses_pools_on_the_host(nat):
    import torch
    import lazyweights_b200 as lw
    with pytest.raises(ValueError):
        lw.PagedCache(torch.zeros(2, 2, 8, 64, dtype=torch.float16), torch.zeros(2, 2, 8, 64, dtype=torch.float16))
    with pytest.raises(ValueError):
        lw.PagedCache(torch.zeros(2, 2, 8, 64), torch.zeros(2, 2, 8, 64))


def test_rows_beyond_32_bits_of_positions_are_refused(nat):
    for fn, base in (("lw_cache_append", APPEND), ("lw_cache_attend_prompt", PROMPT)):
        refused(nat, fn, base, dict(rows=(1 << 30) + 1))


@pytest.mark.parametrize("window", [-1, 2 ** 31, 2 ** 32 + 5, 2 ** 64])
def test_python_windows_that_do_not_fit(window):
    from lazyweights_b200 import paged
    with pytest.raises(ValueError):
        paged._window(window)
    assert paged._window(2 ** 31 - 1) == 2 ** 31 - 1 and paged._window(0) == 0


def test_python_numbers_that_do_not_fit():
    import numpy as np
    from lazyweights_b200.runtime import _int32
    for good in ([1, 2], np.array([[3, -4]]), np.array([5.0, 6.0]), np.zeros(0), np.arange(3, dtype=np.uint8), np.arange(4, dtype=np.int32)[::2]):
        out = _int32(good, "x")
        assert out.dtype == np.int32 and out.flags.c_contiguous and np.array_equal(out, good)
    for bad in ([2 ** 31], [2 ** 32 + 4], np.array([2 ** 32 + 4]), np.array([-2 ** 31 - 1]), [2 ** 70], [1.5], [float("nan")], np.array([2 ** 64 - 1], np.uint64)):
        with pytest.raises(ValueError):
            _int32(bad, "x")
