"""Passes over several sequences with the paged cache against the decoder's own passes, sequence by sequence."""
import numpy as np
import pytest

from oracle import lw_oracle as orc
from tests import helpers

# Two decoders with the same weights that differ in the roundings around attention: queries, probabilities and results in
# fp16 against fp32 in each of two layers, and products of another number of rows, within 1e-3 of each other.  TOL covers those
# where scores are small.  Those of these random weights are not: sum |q k| scale reaches 5000 to 7000, so a query rounded by
# 2^-11 can move a score by 2.5 to 3.4, and where the largest two are closer than that the row's attention changes altogether (the
# float64 model below, with and without the roundings, differs by 0.0001 of the logits at the median position and by up to 0.11 at some).
# So a position's bound is TOL plus twice the most that these roundings - to nearest, up, down, and sixteen times up or down by
# chance, value by value, since which of many close scores wins depends on each - do to the float64 model there.  The sixteen also
# move q, k and v by what products of more than eight rows are off (fp16 activations: up to 3e-4 of a row's largest value, where
# those of one row are within 2e-5), which moves such scores as much.
TOL = 1e-2


def _to_half(x, way):
    """To nearest (0), or up (1) or down (-1), `way` an array of them or one for all."""
    h = x.astype(np.float16)
    step = np.nextafter(h, np.where(np.asarray(way) > 0, np.float16(np.inf), np.float16(-np.inf)))
    return np.where((h.astype(np.float64) - x) * way < 0, step, h).astype(np.float64)


def _model64(W, ids, shape, window, rounded, products=lambda x: x):
    """Logits of all positions in float64; keys and values in fp16 as the caches hold them, queries, probabilities and attention
    through `rounded`."""
    L, H, Hk, Dh = (shape[k] for k in ("n_layers", "n_heads", "n_kv_heads", "head_dim"))
    norms, (cos, sin), n = W["__norms__"], W["__rope__"], len(ids)
    deq = lambda name: orc.dequant(*W[name]).astype(np.float64)
    rms = lambda x, g: x / np.sqrt((x * x).mean(-1, keepdims=True) + shape["eps"]) * g
    c, s = cos[:n, None].astype(np.float64), sin[:n, None].astype(np.float64)

    def rope(x):
        a, b = x[..., :Dh // 2], x[..., Dh // 2:]
        return np.concatenate([a * c - b * s, b * c + a * s], 2)

    i = np.arange(n)
    seen = (i[None] <= i[:, None]) & (i[None] > i[:, None] - (window or n))
    h = W["__embed__"][ids].astype(np.float64)
    for l in range(L):
        qkv = products(rms(h, norms["l%d.ln1" % l]) @ deq("l%d.qkv" % l).T)
        q = rounded(rope(qkv[:, :H * Dh].reshape(n, H, Dh)))
        k = _to_half(rope(qkv[:, H * Dh:(H + Hk) * Dh].reshape(n, Hk, Dh)), 0)
        v = _to_half(qkv[:, (H + Hk) * Dh:].reshape(n, Hk, Dh), 0)
        att = np.zeros((n, H, Dh))
        for j in range(H):
            sc = np.where(seen, q[:, j] @ k[:, j // (H // Hk)].T * Dh ** -0.5, -np.inf)
            e = np.exp(sc - sc.max(1, keepdims=True))
            att[:, j] = rounded(e) @ v[:, j // (H // Hk)] / e.sum(1, keepdims=True)
        h = h + rounded(att).reshape(n, -1) @ deq("l%d.o" % l).T
        xn = rms(h, norms["l%d.ln2" % l])
        g, u = xn @ deq("l%d.gate" % l).T, xn @ deq("l%d.up" % l).T
        h = h + (g / (1 + np.exp(-np.clip(g, -700, 700))) * u) @ deq("l%d.down" % l).T
    return rms(h, norms["lnf"]) @ deq("lm_head").T


def _bounds(W, ids, shape, window=0):
    plain = _model64(W, ids, shape, window, lambda x: x)
    rng = np.random.default_rng(0)
    off = lambda x: x + 3e-4 * np.abs(x).max(1, keepdims=True) * rng.uniform(-1, 1, x.shape)
    runs = [(lambda x: _to_half(x, 0),), (lambda x: _to_half(x, 1),), (lambda x: _to_half(x, -1),)]
    runs += 16 * [(lambda x: _to_half(x, rng.choice((-1, 1), x.shape)), off)]
    effect = [np.abs(_model64(W, ids, shape, window, *run) - plain).max(1) for run in runs]
    return TOL + 2 * np.max(effect, 0) / np.abs(plain).max(1)


def test_without_a_handle():
    helpers.build_library()
    from lazyweights_b200 import _native as nat
    assert nat.lib().rt_pages(None, 10, 16) == nat.LW_ERR_ARG
    assert nat.lib().rt_forward_seqs(None, 1, None, None, None, None, 1, None) == nat.LW_ERR_ARG


def _model(tmp_path, heads, kv_heads, head_dim):
    from lazyweights_b200 import modelgen
    shape = dict(n_layers=2, hidden=512, n_heads=heads, n_kv_heads=kv_heads, head_dim=head_dim, inter=512, vocab=256, eps=1e-5, theta=1e4)
    W = modelgen.write_model(str(tmp_path / "m"), shape, "Q6_K", seed=heads, return_weights=True)
    return str(tmp_path / "m"), W, shape


def _alone(b, ids):
    b.reset()
    return np.stack([b.forward(ids[i:i + 1]) for i in range(len(ids))])


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,head_dim,page,window", [(8, 2, 64, 16, 0), (4, 4, 128, 8, 0), (16, 4, 32, 24, 20), (8, 8, 96, 64, 0)])
def test_several_sequences_as_one_by_one(tmp_path, heads, kv_heads, head_dim, page, window):
    helpers.build_library()
    import lazyweights_b200 as lw
    rng = np.random.default_rng(3)
    lens = [40, 7, 90]
    ids = [rng.integers(0, 256, n).astype(np.int32) for n in lens]
    path, W, shape = _model(tmp_path, heads, kv_heads, head_dim)
    bounds = [_bounds(W, i, shape, window) for i in ids]
    with lw.Bundle(path, max_ctx=256, max_batch=64) as b:
        b.set_window(window)
        alone = [_alone(b, i) for i in ids]
        cols = 128 // page + 1
        pages = rng.permutation(3 * cols).astype(np.int32).reshape(3, cols)
        b.open_pages(3 * cols, page)
        done = [0, 0, 0]
        # prompts of all three, a piece of the third, two sequences one token each, the third alone, all three one by one
        for new in ([30, 5, 20], [0, 0, 60], [1, 1, 0], [0, 0, 4], [1, 1, 1], [1, 0, 1], [7, 0, 4]):
            use = [s for s in range(3) if new[s]]
            got = b.forward_seqs([ids[s][done[s]:done[s] + new[s]] for s in use], [done[s] + new[s] for s in use], pages[use])
            for row, s in zip(got, use):
                done[s] += new[s]
                assert helpers.rel_err(row, alone[s][done[s] - 1]) <= bounds[s][done[s] - 1], (s, done[s])
        assert done == lens
        assert np.array_equal(_alone(b, ids[1])[-1], alone[1][-1])      # the decoder's own cache is as it was
        assert b.kernel_error() == 0


@pytest.mark.gpu
def test_a_common_beginning_is_shared(tmp_path):
    helpers.build_library()
    import lazyweights_b200 as lw
    rng = np.random.default_rng(4)
    head, tails = rng.integers(0, 256, 32).astype(np.int32), [rng.integers(0, 256, n).astype(np.int32) for n in (9, 3)]
    path, W, shape = _model(tmp_path, 8, 2, 64)
    with lw.Bundle(path, max_ctx=128, max_batch=64) as b:
        whole = [np.concatenate([head, t]) for t in tails]
        alone = [_alone(b, i)[-1] for i in whole]
        b.open_pages(5, 16)
        b.forward_seqs([head], [32], [[4, 1]])
        got = b.forward_seqs(tails, [41, 35], [[4, 1, 0], [4, 1, 2]])
        for g, a, i in zip(got, alone, whole):
            assert helpers.rel_err(g, a) <= _bounds(W, i, shape)[-1]


@pytest.mark.gpu
def test_refusals(tmp_path):
    helpers.build_library()
    import lazyweights_b200 as lw
    ids = np.zeros(4, np.int32)
    with lw.Bundle(_model(tmp_path, 8, 2, 64)[0], max_ctx=64, max_batch=8) as b:
        with pytest.raises(lw.LwError):
            b.forward_seqs([ids], [4], [[0]])                  # no pages yet
        for bad in ((0, 16), (4, 12), (4, 0)):
            with pytest.raises(lw.LwError):
                b.open_pages(*bad)
        b.open_pages(3, 16)
        for args in (([ids, ids[:0]], [4, 0], [[0], [1]]), ([ids, ids, ids[:1]], [4, 4, 1], [[0], [1], [2]]), ([ids], [3], [[0]]), ([ids], [65], [[0]]),
                     ([ids], [17], [[0]]), ([ids], [4], [[3]]), ([ids], [4], [[-1]]), ([ids + 256], [4], [[0]]), ([ids - 1], [4], [[0]])):
            with pytest.raises(lw.LwError):
                b.forward_seqs(*args)
        with pytest.raises(ValueError):
            b.forward_seqs([ids], [4, 4], [[0]])
        assert np.isfinite(b.forward_seqs([ids], [4], [[0]])).all() and b.kernel_error() == 0


@pytest.mark.gpu
def test_the_largest_window_is_none(tmp_path):
    helpers.build_library()
    import lazyweights_b200 as lw
    rng = np.random.default_rng(5)
    ids = [rng.integers(0, 256, n).astype(np.int32) for n in (40, 7)]
    with lw.Bundle(_model(tmp_path, 8, 2, 64)[0], max_ctx=128, max_batch=64) as b:
        b.open_pages(8, 16)
        table = [[0, 2, 4, 6], [1, 3, 5, 7]]
        got = []
        for window in (0, 2 ** 31 - 1):
            b.set_window(window)
            got.append((b.forward_seqs(ids, [40, 7], table), b.forward_seqs([i[:1] for i in ids], [41, 8], table)))
        assert all(np.array_equal(x, y) for x, y in zip(*got)) and b.kernel_error() == 0


@pytest.mark.gpu
def test_a_pool_beyond_32_bits_of_positions_is_refused(tmp_path):
    """By its size, before anything is allocated or freed: a product of its bytes could wrap to a small number."""
    helpers.build_library()
    import lazyweights_b200 as lw
    from lazyweights_b200 import _native as nat
    ids = np.arange(5, dtype=np.int32)
    with lw.Bundle(_model(tmp_path, 8, 2, 64)[0], max_ctx=64, max_batch=8) as b:
        b.open_pages(3, 16)
        want = b.forward_seqs([ids], [5], [[1]])
        for pages, size in ((2 ** 31 - 1, 65536), (2 ** 28, 8), (2 ** 15, 65536)):
            with pytest.raises(lw.LwError) as e:
                b.open_pages(pages, size)
            assert e.value.status == nat.LW_ERR_ARG
        assert np.array_equal(b.forward_seqs([ids], [5], [[1]]), want)      # the cache that was there serves on


@pytest.mark.gpu
def test_numbers_that_do_not_fit_are_refused(tmp_path):
    helpers.build_library()
    import lazyweights_b200 as lw
    ids = np.arange(4, dtype=np.int64)
    with lw.Bundle(_model(tmp_path, 8, 2, 64)[0], max_ctx=64, max_batch=8) as b:
        with pytest.raises(ValueError):
            b.open_pages(2 ** 32 + 3, 16)
        b.open_pages(3, 16)
        for args in (([ids + 2 ** 32], [4], [[0]]), ([ids], np.array([2 ** 32 + 4]), [[0]]), ([ids], [4], np.array([[2 ** 32]])), ([ids + 0.5], [4], [[0]])):
            with pytest.raises(ValueError):
                b.forward_seqs(*args)
        want = b.forward_seqs([ids.astype(np.int32)], [4], [[0]])
        assert np.array_equal(b.forward_seqs([ids], np.array([4]), np.array([[0]])), want)


@pytest.mark.gpu
def test_pages_after_a_failed_allocation(tmp_path):
    """open_pages that ran out of memory at any of its buffers (the handle's test switch refuses it on the host) can be called again."""
    helpers.build_library()
    import lazyweights_b200 as lw
    ids = [np.arange(5, dtype=np.int32), np.arange(2, dtype=np.int32)]
    path, table = _model(tmp_path, 8, 2, 64)[0], [[1], [0]]
    with lw.Bundle(path, max_ctx=64, max_batch=8) as b:
        b.open_pages(3, 16)
        want = b.forward_seqs(ids, [5, 2], table)
    for n in (1, 2, 3):
        with lw.Bundle(path, max_ctx=64, max_batch=8) as b:
            try:
                assert lw.lib().lw_debug_set(b"fail_alloc", n) == 0
                with pytest.raises(lw.LwError):
                    b.open_pages(3, 16)
            finally:
                lw.lib().lw_debug_set(b"reset", 0)
            with pytest.raises(lw.LwError):
                b.forward_seqs(ids, [5, 2], table)                  # no pages
            b.open_pages(3, 16)
            assert np.array_equal(b.forward_seqs(ids, [5, 2], table), want), n
