"""Passes over several sequences where attention's scores have ordinary sizes (a few units, not thousands): the roundings around
attention then hardly move the logits, the bound is close to TOL everywhere, and a wrong mask, page or head shows.  Also the passes that
a serving loop is made of: one sequence with one token, and more rows than the products' small-row kernels take."""
import os

import numpy as np
import pytest

from tests import helpers
from tests.test_gpu_sequences import TOL, _alone, _bounds, _model64


def _model(path, heads, kv_heads, head_dim, seed):
    """A Q6_K model whose queries, keys and values are 2^-5 of what the weights' seed gives, through the block scales (in the file and
    in the weights returned)."""
    from lazyweights_b200 import bundle, modelgen
    shape = dict(n_layers=2, hidden=512, n_heads=heads, n_kv_heads=kv_heads, head_dim=head_dim, inter=512, vocab=256, eps=1e-5, theta=1e4)
    W = modelgen.write_model(path, shape, "Q6_K", seed=seed, return_weights=True)
    at = {t["name"]: t for t in bundle.read_manifest(path)[1]}
    with open(os.path.join(path, "weights.bin"), "r+b") as f:
        for l in range(2):
            name = "l%d.qkv" % l
            ty, codes, side = W[name]
            blocks = side.copy().reshape(side.shape[0], -1, 18)
            blocks[:, :, 16:] = (blocks[:, :, 16:].copy().view(np.float16) * np.float16(2.0 ** -5)).view(np.uint8)
            W[name] = ty, codes, blocks.reshape(side.shape)
            assert at[name + ".kqs"]["nbytes"] == blocks.nbytes
            f.seek(at[name + ".kqs"]["offset"])
            f.write(blocks.tobytes())
    return W, shape


CASES = [(8, 2, 64, 16, 0), (4, 4, 128, 8, 0), (16, 4, 32, 24, 20), (8, 8, 96, 64, 33)]


def test_the_bound_bites(tmp_path):
    """A key too many or too few, or the values of a neighbouring position, move the logits by far more than the bound."""
    W, shape = _model(str(tmp_path / "m"), 8, 2, 64, 8)
    ids = np.random.default_rng(3).integers(0, 256, 60).astype(np.int32)
    plain, bound = _model64(W, ids, shape, 0, lambda x: x), _bounds(W, ids, shape)
    assert bound.max() < 3 * TOL
    for other in (_model64(W, ids, shape, 59, lambda x: x)[-1], _model64(W, np.concatenate([ids[:30], ids[29:-1]]), shape, 0, lambda x: x)[-1]):
        assert helpers.rel_err(other, plain[-1]) > 3 * bound[-1]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,head_dim,page,window", CASES)
def test_steps_of_a_serving_loop(tmp_path, heads, kv_heads, head_dim, page, window):
    helpers.build_library()
    import lazyweights_b200 as lw
    rng = np.random.default_rng(3)
    lens = [40, 7, 190]
    ids = [rng.integers(0, 256, n).astype(np.int32) for n in lens]
    W, shape = _model(str(tmp_path / "m"), heads, kv_heads, head_dim, heads)
    bounds = [_bounds(W, i, shape, window) for i in ids]
    with lw.Bundle(str(tmp_path / "m"), max_ctx=256, max_batch=200) as b:
        b.set_window(window)
        alone = [_alone(b, i) for i in ids]
        cols = 256 // page + 1
        pages = rng.permutation(3 * cols).astype(np.int32).reshape(3, cols)
        b.open_pages(3 * cols, page)
        done = [0, 0, 0]
        # one token of one sequence, prompts of 9 to 150 rows in all, prompts and single tokens in one pass, steps of one, two and three
        for new in ([1, 0, 0], [1, 0, 0], [8, 0, 1], [20, 5, 100], [1, 0, 64], [0, 0, 1], [1, 1, 0], [1, 0, 20], [1, 1, 1], [0, 0, 1], [6, 0, 2]):
            use = [s for s in range(3) if new[s]]
            got = b.forward_seqs([ids[s][done[s]:done[s] + new[s]] for s in use], [done[s] + new[s] for s in use], pages[use])
            for row, s in zip(got, use):
                done[s] += new[s]
                assert helpers.rel_err(row, alone[s][done[s] - 1]) <= bounds[s][done[s] - 1], (s, done[s])
        assert done == lens
        assert b.kernel_error() == 0
