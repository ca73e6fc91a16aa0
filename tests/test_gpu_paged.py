"""The paged cache on the GPU against plain 64-bit forms (tests/paged_ref.py, which also derives the bounds)."""
import pytest

from tests import helpers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lw():
    helpers.build_library()
    import lazyweights_b200
    return lazyweights_b200


@pytest.fixture(autouse=True)
def no_error_word(lw):
    yield
    assert lw.lib().lw_kernel_error() == 0


def dtypes():
    import torch
    return {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def problem(lens, news, heads, kv_heads, dim, page, dtype, inner=False, seed=0, gap=0, spread=1.0):
    """Random keys and values at the positions in use, NaN everywhere else in the pools; queries [rows + gap, heads, dim]."""
    import torch
    from tests import paged_ref as ref
    gen = torch.Generator().manual_seed(seed)
    t = dtypes()[dtype]
    pages, table, lens_t, starts = ref.sequences(lens, news, page, gen)
    k, v = (ref.pool(pages, kv_heads, page, dim, t, inner) for _ in range(2))
    for b, n in enumerate(lens):
        for p, f in ((k, spread), (v, 1.0)):
            ref.store(p, table, b, 0, torch.randn(n, kv_heads, dim, generator=gen) * f)
    q = torch.randn(int(starts[-1]) + gap, heads, dim, generator=gen).to(t)
    return dict(k=k, v=v, table=table, lens=lens_t, starts=starts, q=q, news=news)


def on_gpu(t):
    """On the GPU with the same strides (Tensor.cuda keeps those of dense tensors)."""
    return t.cuda()


def check_attention(lw, pr, scale=None, window=0, prompt=True, cache=None):
    import torch
    from tests import paged_ref as ref
    cache = cache or lw.PagedCache(on_gpu(pr["k"]), on_gpu(pr["v"]))
    q, table, lens, starts = (pr[n].cuda() for n in ("q", "table", "lens", "starts"))
    out = torch.full_like(q, 7.0)
    if prompt:
        cache.attend_prompt(q, table, lens, starts, scale=scale, window=window, out=out)
    else:
        cache.attend(q, table, lens, scale=scale, window=window, out=out)
    got = out.cpu().double()
    s = q.shape[2] ** -0.5 if scale is None else scale
    for b, n in enumerate(pr["lens"].tolist()):
        m = pr["news"][b]
        first = int(pr["starts"][b]) if prompt else b
        rows = slice(first, first + m)
        want, bound, _ = ref.attend(pr["q"][rows], ref.load(pr["k"], pr["table"], b, n), ref.load(pr["v"], pr["table"], b, n),
                                    torch.arange(n - m, n), s, window)
        bad = ~((got[rows] - want).abs() <= bound)
        assert not bad.any(), (b, n, m, int(bad.sum()), float((got[rows] - want).abs().max()), torch.nonzero(bad)[:3].tolist())
    if prompt:
        behind = got[int(pr["starts"][-1]):]
        assert (behind == 7.0).all()
    return got


HEADS = [(1, 1, 128), (8, 2, 128), (6, 2, 96), (7, 1, 64), (16, 2, 40), (16, 1, 80), (34, 2, 32), (5, 5, 8), (40, 1, 128)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("page", [8, 16, 24, 64, 256])
def test_one_token(lw, heads, kv_heads, dim, page, dtype):
    lens = [1, 2, 0, 7, 8, 9, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129, 255, 257, 511, 700]
    pr = problem(lens, [1] * len(lens), heads, kv_heads, dim, page, dtype, inner=page == 24, seed=page + heads)
    got = check_attention(lw, pr, prompt=False)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lens", [[1], [64], [4097], [3000, 1], [1, 5000, 2], [10] * 300, [0] * 40 + [2000] + [0] * 400])
def test_one_token_few_and_many(lw, lens, dtype):
    check_attention(lw, problem(lens, [1] * len(lens), 8, 2, 64, 16, dtype, seed=len(lens)), prompt=False)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 300, 10000])
def test_one_token_window(lw, window):
    check_attention(lw, problem([1, 5, 63, 64, 65, 130, 700, 2001], [1] * 8, 6, 3, 128, 16, "fp16", seed=window), prompt=False, window=window)


# (length, new rows): whole prompts, pieces, single rows, nothing; rows around the tiles of 64, 128 and 256
PROMPTS = [(1, 1), (5, 5), (0, 0), (17, 3), (64, 64), (65, 65), (127, 127), (128, 128), (129, 129), (300, 1), (400, 37), (0, 0), (257, 257), (700, 33)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("page", [8, 16, 24, 256])
def test_prompts(lw, heads, kv_heads, dim, page, dtype):
    pr = problem([n for n, _ in PROMPTS], [m for _, m in PROMPTS], heads, kv_heads, dim, page, dtype, inner=page == 16, seed=page + heads, gap=5)
    check_attention(lw, pr)


@pytest.mark.parametrize("lens", [[(1, 1)], [(1500, 1500)], [(4000, 8)], [(2000, 1), (1, 1)], [(3, 1)] * 200, [(0, 0)] * 70 + [(900, 300)] + [(0, 0)] * 300])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 2)])
def test_prompts_few_and_many(lw, lens, heads, kv_heads):
    check_attention(lw, problem([n for n, _ in lens], [m for _, m in lens], heads, kv_heads, 128, 16, "bf16", seed=len(lens), gap=1))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 300])
def test_pairs_whose_second_tile_is_empty(lw, dim, window):
    """Prompts that end inside the first tile of a pair of tiles, so that the second one passes over more position blocks than the
    stages hold, between pairs that need both; several of them per block of the grid."""
    lens = [1055, 1055, 700, 33, 1055, 1090, 1055, 33, 1055, 1055]
    check_attention(lw, problem(lens, lens, 16, 8, dim, 16, "fp16", seed=dim), window=window)


@pytest.mark.parametrize("window", [1, 2, 17, 64, 127, 128, 129, 500, 100000])
def test_prompt_window(lw, window):
    lens = [(1, 1), (70, 70), (300, 200), (128, 128), (900, 40), (1030, 1030)]
    check_attention(lw, problem([n for n, _ in lens], [m for _, m in lens], 4, 2, 128, 32, "fp16", seed=window), window=window)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 128, 2 ** 30])
def test_windows_without_an_end(lw, window):
    """A window that nothing fills is none, up to the largest, also for rows before position 0."""
    import torch
    lens = [(200, 200), (1000, 70), (1, 1), (300, 300)]
    pr = problem([n for n, _ in lens], [m for _, m in lens], 4, 2, 64, 16, "fp16", seed=6)
    pr["starts"] = torch.tensor([0, 200, 270, 271, 591], dtype=torch.int32)      # 20 rows more than the last one has positions
    pr["q"] = torch.randn(591, 4, 64, generator=torch.Generator().manual_seed(1)).half()
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("q", "table", "lens", "starts")]
    got = cache.attend_prompt(*args, window=window)
    assert torch.equal(got, cache.attend_prompt(*args)) and (got[271:291] == 0).all()
    for m in (4, 64):      # tiles of other numbers of tokens
        sub = args[0][:, :1].expand(-1, m, -1).contiguous()
        assert torch.equal(cache.attend_prompt(sub, *args[1:], window=window), cache.attend_prompt(sub, *args[1:]))
    one = [args[0][:4].contiguous(), *args[1:3]]
    assert torch.equal(cache.attend(*one, window=window), cache.attend(*one))
    keep = torch.cat((torch.arange(271), torch.arange(291, 591)))
    check_attention(lw, dict(pr, q=pr["q"][keep], starts=torch.tensor([0, 200, 270, 271, 571], dtype=torch.int32)), window=window)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.25, 2.0])
def test_scales(lw, scale):
    """Equal weights, sharp maxima (scores of a few dozen), a negative scale."""
    for prompt in (True, False):
        lens = [(200, 200), (65, 3)] if prompt else [(200, 1), (65, 1), (1000, 1)]
        check_attention(lw, problem([n for n, _ in lens], [m for _, m in lens], 4, 2, 64, 16, "fp16", seed=3), scale=scale, prompt=prompt)


@pytest.mark.parametrize("order", [1, -1])
def test_maxima_that_move(lw, order):
    """Keys whose length grows or falls along the sequence: the running maximum moves at every step, or never."""
    import torch
    from tests import paged_ref as ref
    for prompt in (True, False):
        pr = problem([1200], [300 if prompt else 1], 4, 2, 128, 16, "bf16", seed=5)
        k = ref.load(pr["k"], pr["table"], 0, 1200)
        ramp = torch.linspace(0.1, 12.0, 1200)
        ref.store(pr["k"], pr["table"], 0, 0, k * (ramp if order > 0 else ramp.flip(0))[:, None, None])
        check_attention(lw, pr, prompt=prompt)


@pytest.mark.parametrize("prompt", [True, False])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("place", [0, 4000, 7999])
def test_many_small_weights(lw, place, dtype, prompt):
    """One position takes almost all of the weight and has values of 0; the 8000 others have e^-17 of its weight each, less than fp16
    can tell from its neighbours 0 and 2^-24, and values of 1: together 0.0003, which is all there is of the result.  Enough
    sequences (on the same pages) that most of them are not split."""
    import math
    import torch
    from tests import paged_ref as ref
    n, new, seqs = 8001, 3 if prompt else 1, 10 if prompt else 64
    pr = problem([n], [new], 32, 32, 64, 16, dtype)
    keys, values = torch.zeros(n, 32, 64), torch.ones(n, 32, 64)
    keys[place, :, 0], values[place] = 17.0, 0.0
    ref.store(pr["k"], pr["table"], 0, 0, keys), ref.store(pr["v"], pr["table"], 0, 0, values)
    q = torch.zeros(seqs * new, 32, 64, dtype=dtypes()[dtype], device="cuda")
    q[:, :, 0] = 1.0
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    table, lens = pr["table"].expand(seqs, -1).contiguous().cuda(), pr["lens"].expand(seqs).contiguous().cuda()
    starts = torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device="cuda")
    out = (cache.attend_prompt(q, table, lens, starts, scale=1.0) if prompt else cache.attend(q, table, lens, scale=1.0)).cpu().double()
    seen = [(pos + (pos < place), float(pos >= place)) for pos in range(n - new, n)]      # positions of value 1, and whether the heavy one is seen
    want = torch.tensor([c * math.exp(-17.0) / (heavy + c * math.exp(-17.0)) for c, heavy in seen] * seqs, dtype=torch.float64)[:, None, None]
    # weights: half a step of the type, or, lifted by 2^7, half of 2^-24 of 2^7 e^-17 = 2^-17.5 (2^-7.5 of it); exponentials 2^-13 of 32-bit scores of
    # at most 17 log2(e) + 15 < 64 (2^-19); sums of n numbers in 32 bits, rounded to nearest or cut; the result's half step
    rel = max(ref.EPS[dtypes()[dtype]], 2.0 ** -7.5) + 2 * (2.0 ** -13 + 2.0 ** -19) + 2 * n * 2.0 ** -23 + ref.EPS[dtypes()[dtype]]
    assert ((out - want).abs() <= rel * want).all(), float(((out - want).abs() / want).max())


@pytest.mark.parametrize("prompt", [True, False])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("score", [2.0 ** 20, 2.9e6, 2.91e6, 2.0 ** 22, 2.0 ** 23 + 2.0 ** 15, 1.2e7, 2.0e7, 4.1e7, 8.0e7, -2.0e7])
def test_scores_of_millions(lw, score, dtype, prompt):
    """Three positions share the largest score, far from all others: the result is the mean of their values, however few digits 32 bits
    leave a score of that size; also where the maximum moves through such sizes on the way, and where the work is split."""
    import torch
    from tests import paged_ref as ref
    t = dtypes()[dtype]
    lens = [300, 700, 6000]
    pr = problem(lens, [40] * 3 if prompt else [1] * 3, 4, 2, 64, 16, dtype, seed=3)
    places = [5, 133, 250]
    pr["q"].zero_()
    pr["q"][:, :, 0] = 4096.0
    for b, n in enumerate(lens):
        # before position 250 ever larger ones, all behind it far smaller; the three the largest
        keys = torch.zeros(n, 2, 64)
        other = score / 4096 * (torch.linspace(0.1, 0.8, n) if score > 0 else torch.linspace(1.8, 1.2, n))
        keys[:, :, 0] = other[:, None]
        keys[places, :, 0] = score / 4096
        ref.store(pr["k"], pr["table"], b, 0, keys)
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[m].cuda() for m in ("q", "table", "lens")]
    out = (cache.attend_prompt(*args, pr["starts"].cuda(), scale=1.0) if prompt else cache.attend(*args, scale=1.0)).cpu().double()
    rows = 40 if prompt else 1
    for b, n in enumerate(lens):
        seen = min(n - rows + 1, n)                                             # every row sees the three
        assert seen > max(places)
        v = ref.load(pr["v"], pr["table"], b, n)[places].repeat_interleave(2, 1)   # [3, heads, dim]
        want, size = v.mean(0), v.abs().mean(0)
        # the three weights are equal, rounded alike (half a step) against an unrounded sum; the result's half step; 32-bit sums
        assert ((out[b * rows:(b + 1) * rows] - want).abs() <= size * (2 * ref.EPS[t] + 2.0 ** -20)).all(), (b, n)


def test_more_rows_than_positions(lw):
    """Rows before position 0 see nothing and give zeros."""
    import torch
    for heads, kv_heads in ((4, 2), (4, 4)):
        pr = problem([5, 130], [5, 130], heads, kv_heads, 64, 16, "fp16")
        cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
        q = torch.randn(12 + 140, heads, 64).half()
        starts = torch.tensor([0, 12, 152], dtype=torch.int32)
        out = torch.full_like(q, 7.0).cuda()
        cache.attend_prompt(q.cuda(), pr["table"].cuda(), pr["lens"].cuda(), starts.cuda(), out=out)
        assert (out[:7] == 0).all() and (out[12:22] == 0).all()
        keep = torch.cat((q[7:12], q[22:]))
        want = torch.empty_like(keep).cuda()
        cache.attend_prompt(keep.cuda(), pr["table"].cuda(), pr["lens"].cuda(), pr["starts"].cuda(), out=want)
        pr["q"] = keep
        check_attention(lw, pr, cache=cache)
        diff = (torch.cat((out[7:12], out[22:])).float() - want.float()).abs().max()   # other tiles, other order of sums
        assert diff <= 4 * 2.0 ** -11 * 4


def test_infinities_and_nan_in_sight_show(lw):
    """A NaN key makes the rows that see it NaN, and no others."""
    import torch
    from tests import paged_ref as ref
    pr = problem([200, 200], [200, 200], 2, 1, 64, 16, "fp16")
    bad = ref.load(pr["k"], pr["table"], 0, 200)
    bad[150] = float("nan")
    ref.store(pr["k"], pr["table"], 0, 0, bad)
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    out = cache.attend_prompt(pr["q"].cuda(), pr["table"].cuda(), pr["lens"].cuda(), pr["starts"].cuda())
    assert torch.isfinite(out[:150]).all() and torch.isnan(out[150:200]).all() and torch.isfinite(out[200:]).all()
    one = cache.attend(pr["q"][:2].contiguous().cuda(), pr["table"].cuda(), pr["lens"].cuda())
    assert torch.isnan(one[0]).all() and torch.isfinite(one[1]).all()


@pytest.mark.parametrize("value", [1.0, float("inf")])
@pytest.mark.parametrize("length,new,low", [(200, 200, 150), (300, 70, 250), (6000, 30, 5980), (6000, 30, 3000), (700, 700, 130), (40000, 5, 39999)])
def test_scores_of_minus_infinity(lw, length, new, low, value):
    """Keys before position `low` whose scores are -inf: rows that see no other are NaN, whether the work on them is split or not,
    and the others are as if those positions were not there; also beside an infinite value that only the last row sees."""
    import torch
    from tests import paged_ref as ref
    pr = problem([length, 100], [new, 100], 4, 2, 64, 16, "fp16", seed=length)
    pr["q"][:, :, 0] = 1.0
    keys, v = (ref.load(pr[n], pr["table"], 0, length) for n in "kv")
    keys[:low, :, 0] = -float("inf")
    v[length - 1, :, 5] = value
    ref.store(pr["k"], pr["table"], 0, 0, keys)
    ref.store(pr["v"], pr["table"], 0, 0, v)
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("q", "table", "lens", "starts")]
    out = cache.attend_prompt(*args).cpu().double()
    first = length - new
    none = max(0, low - first)                 # rows that see positions before `low` alone
    assert torch.isnan(out[:none]).all() and torch.isfinite(out[new:]).all()
    # without those positions: the rest of the sequence, seen from the same places
    clean = torch.where(torch.isfinite(v), v, torch.zeros((), dtype=torch.float64))
    want, bound, _ = ref.attend(pr["q"][none:new], keys[low:], clean[low:], torch.arange(first + none, length) - low, 64 ** -0.5, 0)
    good = ((out[none:new] - want).abs() <= bound)
    if value != 1.0:
        assert not torch.isfinite(out[new - 1, :, 5]).any()
        good[-1, :, 5] = True
    assert good.all()
    for last in (low, length):                 # one token: all scores -inf, or not
        one = cache.attend(args[0][new - 1:new].contiguous(), args[1][:1], torch.full_like(args[2][:1], last)).cpu()
        if last == low:
            assert torch.isnan(one).all()
        else:
            assert ((one.double() - want[-1]).abs() <= bound[-1])[:, :, :5].all()


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("heads,length,new", [(2, 200, 200), (4, 300, 70), (2, 6000, 30)])
def test_values_out_of_sight_do_not_show(lw, heads, length, new, window):
    """Infinite and NaN values: they show in the rows that see their position, in their dimension, and nowhere else; also where
    the rows of one tile see different positions, and where the work on a row is split (the long case)."""
    import torch
    from tests import paged_ref as ref
    pr = problem([length, 100], [new, 100], heads, 1, 64, 16, "fp16", seed=heads)
    v = ref.load(pr["v"], pr["table"], 0, length)
    first = length - new
    places = [(first + new // 2, 3, float("nan")), (length - 1, 5, float("inf")), (first + new // 3, 60, -float("inf")), (max(0, first - 45), 7, float("inf"))]
    for p, d, x in places:
        v[p, 0, d] = x
    ref.store(pr["v"], pr["table"], 0, 0, v)
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    out = cache.attend_prompt(*(pr[n].cuda() for n in ("q", "table", "lens", "starts")), window=window).cpu().double()
    keys = ref.load(pr["k"], pr["table"], 0, length)
    clean = torch.where(torch.isfinite(v), v, torch.zeros((), dtype=torch.float64))
    pos = torch.arange(first, length)
    want, bound, _ = ref.attend(pr["q"][:new], keys, clean, pos, 64 ** -0.5, window)
    shows = torch.zeros(new, 64, dtype=torch.bool)
    for p, d, x in places:
        shows[:, d] |= (pos >= p) & ((pos - window < p) if window else torch.ones(new, dtype=torch.bool))
    shows = shows[:, None].expand(new, heads, 64)
    assert not torch.isfinite(out[:new][shows]).any()
    assert ((out[:new] - want).abs() <= bound)[~shows].all()
    assert torch.isfinite(out[new:]).all()
    one = cache.attend(pr["q"][:2].contiguous().cuda(), pr["table"].cuda(), pr["lens"].cuda(), window=window).cpu()
    assert torch.equal(~torch.isfinite(one[0]), shows[-1]) and torch.isfinite(one[1]).all()


def test_rows_computed_again_do_not_run_out_the_waits(lw):
    """Long contexts whose last value is infinite: the rows that do not see it are computed again, which takes far longer than the
    waits of the block's other warps are given here; they must not give up meanwhile."""
    import torch
    from tests import paged_ref as ref
    length, new, heads = 1500, 300, 32
    pr = problem([length] * 5, [new] * 5, heads, heads, 64, 16, "fp16", seed=9)
    for b in range(5):
        v = ref.load(pr["v"], pr["table"], b, length)
        v[length - 1, :, 5] = float("inf")
        ref.store(pr["v"], pr["table"], b, 0, v)
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("q", "table", "lens", "starts")]
    lib = lw.lib()
    try:
        lib.lw_debug_set(b"wait_limit", 4000)
        out = cache.attend_prompt(*args)
        torch.cuda.synchronize()
        assert lib.lw_kernel_error() == 0
    finally:
        lib.lw_debug_set(b"reset", 0)
    out = out.cpu().double().view(5, new, heads, 64)
    last = new - 256                            # rows of every sequence's second pair of tiles
    for b in range(5):
        k, v = (ref.load(pr[n], pr["table"], b, length)[:-1] for n in "kv")
        want, bound, _ = ref.attend(pr["q"][(b + 1) * new - last:(b + 1) * new - 1], k, v, torch.arange(length - last, length - 1), 64 ** -0.5, 0)
        assert ((out[b, -last:-1] - want).abs() <= bound).all()
        assert torch.isinf(out[b, -1, :, 5]).all() and torch.isfinite(out[b, -1, :, 6:]).all()


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("heads,length,new", [(2, 200, 200), (4, 300, 70), (2, 6000, 30), (1, 6000, 300)])
def test_results_in_the_place_of_the_queries(lw, heads, length, new, window):
    """out = q gives the same bits, also for rows that are computed again beside values that are not finite."""
    import torch
    from tests import paged_ref as ref
    for value in (1.0, float("inf")):
        pr = problem([length, 100], [new, 100], heads, 1, 64, 16, "fp16", seed=heads)
        v = ref.load(pr["v"], pr["table"], 0, length)
        v[length - 1, 0, 5] = v[length - new // 2, 0, 9] = value
        ref.store(pr["v"], pr["table"], 0, 0, v)
        cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
        q, *args = [pr[n].cuda() for n in ("q", "table", "lens", "starts")]
        for call, x, more in ((cache.attend_prompt, q, args), (cache.attend, q[:2].contiguous(), args[:2])):
            want = call(x, *more, window=window)
            same = x.clone()
            call(same, *more, window=window, out=same)
            assert torch.equal(same.view(torch.int16), want.view(torch.int16))


def test_strided_queries_and_results(lw):
    """Queries inside the rows of a fused product, results into a slice of a wider tensor."""
    import torch
    pr = problem([70, 300], [70, 20], 4, 2, 96, 16, "bf16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("table", "lens", "starts")]
    want = cache.attend_prompt(pr["q"].cuda(), *args)
    wide = torch.full((90, 8, 96), 3.0, dtype=torch.bfloat16, device="cuda")
    wide[:, :4] = pr["q"].cuda()
    out = torch.full((90, 12, 104), 5.0, dtype=torch.bfloat16, device="cuda")
    cache.attend_prompt(wide[:, :4], *args, out=out[:, 2:6, :96])
    assert torch.equal(out[:, 2:6, :96], want)
    out[:, 2:6, :96] = 5.0
    assert (out == 5.0).all()
    one = cache.attend(pr["q"][:2].cuda(), *args[:2])
    cache.attend(wide[:2, :4], *args[:2], out=out[:2, 2:6, :96])
    assert torch.equal(out[:2, 2:6, :96], one)


@pytest.mark.parametrize("prompt", [True, False])
def test_heads_outside_the_rows(lw, prompt):
    """Queries and results [heads][rows][dim], passed transposed; pools with the heads outermost."""
    import torch
    pr = problem([300, 41], [70, 41] if prompt else [1, 1], 6, 3, 96, 16, "fp16", seed=8)
    rows = pr["q"].shape[0]
    turned = [pr[n].cuda().transpose(0, 1).contiguous().transpose(0, 1) for n in ("k", "v")]
    cache = lw.PagedCache(*turned)
    q = pr["q"].cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert q.stride(1) == rows * 96 and turned[0].stride(1) > turned[0].stride(0)
    out = torch.full((6, rows, 96), 7.0, dtype=torch.float16, device="cuda").transpose(0, 1)
    args = [pr[n].cuda() for n in ("table", "lens")] + ([pr["starts"].cuda()] if prompt else [])
    (cache.attend_prompt if prompt else cache.attend)(q, *args, out=out)
    plain = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    assert torch.equal(out, (plain.attend_prompt if prompt else plain.attend)(pr["q"].cuda(), *args))
    check_attention(lw, pr, prompt=prompt)


@pytest.mark.parametrize("heads,kv_heads", [(128, 1), (100, 1), (129 * 2 - 2, 2)])
def test_wide_groups(lw, heads, kv_heads):
    """Up to 128 query heads per kv head: one token per tile of rows."""
    for prompt in (True, False):
        check_attention(lw, problem([150, 3], [9, 3] if prompt else [1, 1], heads, kv_heads, 64, 16, "fp16", seed=heads), prompt=prompt)


def test_one_large_page(lw):
    for prompt in (True, False):
        check_attention(lw, problem([1000], [200 if prompt else 1], 4, 2, 64, 4096, "bf16", seed=1), prompt=prompt)


def test_thousands_of_sequences(lw):
    """More sequences than a block has threads, several times over, most of them short or without rows."""
    import torch
    lens = [(i * 7) % 23 for i in range(3000)]
    check_attention(lw, problem(lens, [1] * 3000, 2, 1, 32, 8, "fp16", seed=2), prompt=False)
    news = [min(n, i % 3) for i, n in enumerate(lens)]
    check_attention(lw, problem(lens, news, 2, 1, 32, 8, "fp16", seed=3, gap=2))


def test_rows_before_the_first_sequence(lw):
    import torch
    pr = problem([50, 20], [5, 20], 4, 2, 64, 16, "fp16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    table, lens = pr["table"].cuda(), pr["lens"].cuda()
    want = cache.attend_prompt(pr["q"].cuda(), table, lens, pr["starts"].cuda())
    q = torch.cat((torch.zeros(3, 4, 64, dtype=torch.float16), pr["q"])).cuda()
    out = torch.full_like(q, 7.0)
    cache.attend_prompt(q, table, lens, (pr["starts"] + 3).cuda(), out=out)
    assert (out[:3] == 7).all() and torch.equal(out[3:], want)


@pytest.mark.parametrize("prompt", [True, False])
def test_same_call_same_bits(lw, prompt):
    import torch
    pr = problem([3000, 17], [200, 17] if prompt else [1, 1], 8, 2, 128, 16, "fp16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("q", "table", "lens")] + ([pr["starts"].cuda()] if prompt else [])
    call = cache.attend_prompt if prompt else cache.attend
    first = call(*args)
    for _ in range(5):
        assert torch.equal(call(*args), first)


def test_far_pages(lw):
    """Pages more than 2^31 elements apart."""
    import torch
    from tests import paged_ref as ref
    stride = (1 << 31) + 4096
    raw = [torch.empty(2 * stride + 2 * 16 * 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    pools = [r.as_strided((3, 2, 16, 64), (stride, 16 * 64, 64, 1)) for r in raw]
    gen = torch.Generator().manual_seed(1)
    small = [torch.randn(3, 2, 16, 64, generator=gen).half() for _ in range(2)]
    for p, s in zip(pools, small):
        p.copy_(s)
    pr = dict(k=small[0], v=small[1], table=torch.tensor([[2, 0, 1]], dtype=torch.int32), lens=torch.tensor([45], dtype=torch.int32), news=[45],
              starts=torch.tensor([0, 45], dtype=torch.int32), q=torch.randn(45, 4, 64, generator=gen).half())
    cache = lw.PagedCache(*pools)
    check_attention(lw, pr, cache=cache)
    check_attention(lw, dict(pr, q=pr["q"][:1], news=[1]), cache=cache, prompt=False)
    qkv = torch.randn(1, 8 * 64, generator=gen)
    table = torch.ones(46, 32)
    cache.append(qkv.cuda(), 4, table.cuda(), torch.zeros(46, 32).cuda(), pr["table"].cuda(), pr["lens"].cuda())
    assert torch.equal(pools[0][1, :, 12].cpu(), qkv.view(8, 64)[4:6].half()) and torch.equal(pools[1][1, :, 12].cpu(), qkv.view(8, 64)[6:].half())


# ------------------------------------------------------------------------------------------------------- appending


@pytest.mark.parametrize("rows_type", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(4, 2, 128, 128), (32, 8, 128, 128), (3, 1, 96, 96), (2, 2, 40, 40), (4, 4, 80, 32), (5, 1, 8, 8),
                                                    (64, 8, 64, 64)])
def test_append(lw, heads, kv_heads, dim, rot, dtype, rows_type):
    import torch
    from tests import paged_ref as ref
    t = dtypes()[dtype]
    for case, (lens, news, starts_given, page, off) in enumerate((([40, 1, 0, 300, 17], [40, 1, 0, 20, 3], True, 16, 0),
                                                                  ([5, 0, 64, 65], [1, 1, 1, 1], False, 8, 1), ([1], [1], False, 64, 0),
                                                                  ([70], [70], True, 24, 3))):
        gen = torch.Generator().manual_seed(case)
        pages, table, lens_t, starts = ref.sequences(lens, news, page, gen)
        k, v = (ref.pool(pages, kv_heads, page, dim, t, case == 0, fill=5.0) for _ in range(2))
        rows, width = int(starts[-1]) + 2, (heads + 2 * kv_heads) * dim
        raw = torch.randn(rows * (width + 8) + off, generator=gen).to(dtypes()[rows_type]).cuda()
        qkv = raw[off:].view(rows, width + 8)[:, :width]                     # rows apart, at an odd address where off says so
        angle = torch.rand(400, rot // 2, generator=gen) * 6.3
        cos, sin = angle.cos(), angle.sin()
        gk, gv = on_gpu(k), on_gpu(v)
        q = torch.full((rows, heads, dim), 7.0, dtype=t, device="cuda")
        lw.PagedCache(gk, gv).append(qkv, heads, cos.cuda(), sin.cuda(), table.cuda(), lens_t.cuda(), starts=starts.cuda() if starts_given else None, q=q)
        want_q, err_q = torch.full((rows, heads, dim), 7.0, dtype=torch.float64), torch.zeros(rows, heads, dim, dtype=torch.float64)
        want_k, want_v, err_k = k.double(), v.double(), torch.zeros(k.shape, dtype=torch.float64)
        host = qkv.cpu()
        for b, (n, m) in enumerate(zip(lens, news)):
            if not n:
                continue
            first = int(starts[b]) if starts_given else b
            pos = torch.arange(n - m, n)
            rq, rk, rv, e = ref.rotate(host[first:first + m], heads, kv_heads, dim, cos, sin, pos)
            want_q[first:first + m], err_q[first:first + m] = rq, e[:, :heads]
            at = (table[b, pos // page].long(), slice(None), pos % page)
            want_k[at], want_v[at], err_k[at] = rk, rv, e[:, heads:]
        for got, want, err in ((q, want_q, err_q), (gk, want_k, err_k), (gv, want_v, 0.0)):
            got = got.cpu().double()
            assert ((got - want).abs() <= err * (1 + ref.EPS[t]) + want.abs() * ref.EPS[t] + ref.TINY[t]).all()


def test_append_leaves_what_is_not_its_own(lw):
    """More rows than positions, rows outside all sequences: neither the pools nor q change there."""
    import torch
    k, v = (torch.full((4, 2, 8, 64), 5.0, dtype=torch.float16, device="cuda") for _ in range(2))
    cache = lw.PagedCache(k, v)
    table = torch.tensor([[1, -1], [3, 0]], dtype=torch.int32).cuda()
    q = torch.full((12, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    cos = torch.ones(20, 32, device="cuda")
    cache.append(torch.ones(12, 6 * 64, device="cuda"), 2, cos, cos * 0, table, torch.tensor([3, 10], dtype=torch.int32).cuda(),
                 starts=torch.tensor([1, 6, 8], dtype=torch.int32).cuda(), q=q)
    assert [bool((q[i] == 7).all()) for i in range(12)] == [i in (0, 1, 2, 8, 9, 10, 11) for i in range(12)]
    changed = torch.zeros(4, 8, dtype=torch.bool)
    changed[1, :3] = changed[0, :2] = True
    for p in (k, v):
        assert torch.equal((p == 1).all(3).all(1).cpu(), changed) and ((p == 1) | (p == 5)).all()


# ---------------------------------------------------------------------------------- indexes that are not followed


def test_bad_indexes_are_reported(lw):
    """Pages outside the pool, a length beyond the table, a position beyond the rotation tables: the other sequences' results
    stand, the error word says so."""
    import torch
    pr = problem([40, 40, 40], [2, 2, 2], 4, 2, 64, 16, "fp16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    q, starts = pr["q"].cuda(), pr["starts"].cuda()
    good = cache.attend_prompt(q, pr["table"].cuda(), pr["lens"].cuda(), starts)
    one = cache.attend(q[:3], pr["table"].cuda(), pr["lens"].cuda())
    cols = pr["table"].shape[1]
    for change in ("high", "negative", "length"):
        table, lens = pr["table"].clone(), pr["lens"].clone()
        if change == "length":
            lens[1] = cols * 16 + 5
            table[1] = table[1, 0]
        else:
            table[1, 1] = pr["k"].shape[0] if change == "high" else -1
        got = cache.attend_prompt(q, table.cuda(), lens.cuda(), starts)
        assert lw.lib().lw_kernel_error() == 2
        # another total of work moves the places where the work is split, and with them the order of sums
        close = lambda a, b: (a.float() - b.float()).abs().max() <= 4 * 2.0 ** -11 * 4
        assert close(got[:2], good[:2]) and close(got[4:], good[4:])
        got = cache.attend(q[:3], table.cuda(), lens.cuda())
        assert lw.lib().lw_kernel_error() == 2
        assert close(got[0], one[0]) and close(got[2], one[2])
    k, v = (torch.full((3, 2, 8, 64), 5.0, dtype=torch.float16, device="cuda") for _ in range(2))
    rows, cos = torch.ones(3, 6 * 64, device="cuda"), torch.ones(9, 32, device="cuda")
    for table, lens in (([[0], [3], [1]], [1, 1, 1]), ([[0], [-7], [1]], [1, 1, 1]), ([[0], [2], [1]], [1, 9, 1]), ([[0, 0], [2, 2], [1, 1]], [1, 10, 1])):
        k.fill_(5.0), v.fill_(5.0)
        lw.PagedCache(k, v).append(rows, 2, cos, cos * 0, torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
        assert lw.lib().lw_kernel_error() == 2
        for p in (k, v):
            assert (p[:2, :, 0] == 1).all() and (p[:2, :, 1:] == 5).all() and (p[2] == 5).all()


@pytest.mark.parametrize("prompt", [True, False])
def test_a_lost_copy_ends_the_kernel(lw, prompt):
    """A copy that never arrives (the kernel's own test switch skips it): the wait for it runs out, the kernel ends, the error word
    says so, and the next call is right."""
    import torch
    # long enough for several units in the share of the first block, or warp, which skips one
    pr = problem([20000] * 4, [100 if prompt else 1] * 4, 4, 2, 128, 16, "fp16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("q", "table", "lens")] + ([pr["starts"].cuda()] if prompt else [])
    call = cache.attend_prompt if prompt else cache.attend
    want = call(*args)
    torch.cuda.synchronize()
    lib = lw.lib()
    try:
        for unit in (0, 1):
            lib.lw_debug_set(b"wait_limit", 2000)
            lib.lw_debug_set(b"drop_unit", unit)
            call(*args)
            torch.cuda.synchronize()
            assert lib.lw_kernel_error() == 1
            lib.lw_debug_set(b"reset", 0)
            assert torch.equal(call(*args), want)
    finally:
        lib.lw_debug_set(b"reset", 0)


@pytest.mark.parametrize("window", [0, 50])
def test_a_lost_copy_among_partly_seen_blocks(lw, window):
    """The same where every block of positions is only partly seen, so that values are waited for by the warp that loads them."""
    import torch
    pr = problem([100] * 200, [100] * 200, 4, 2, 128, 16, "fp16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("q", "table", "lens", "starts")]
    want = cache.attend_prompt(*args, window=window)
    torch.cuda.synchronize()
    lib = lw.lib()
    try:
        for unit in (0, 1):
            lib.lw_debug_set(b"wait_limit", 2000)
            lib.lw_debug_set(b"drop_unit", unit)
            cache.attend_prompt(*args, window=window)
            torch.cuda.synchronize()
            assert lib.lw_kernel_error() == 1
            lib.lw_debug_set(b"reset", 0)
            assert torch.equal(cache.attend_prompt(*args, window=window), want)
    finally:
        lib.lw_debug_set(b"reset", 0)


# ------------------------------------------------------------------------------------------- graphs, streams, together


def test_captured_and_replayed(lw):
    """A captured step is replayed with other lengths, pages, rows and contents; two graphs of one cache run side by side."""
    import torch
    before = problem([300, 40, 700], [30, 40, 1], 8, 2, 128, 16, "fp16", seed=1)
    after = problem([20, 811, 0], [20, 51, 0], 8, 2, 128, 16, "fp16", seed=2)
    pages = max(p["k"].shape[0] for p in (before, after))
    cols = max(p["table"].shape[1] for p in (before, after))
    k, v = (torch.zeros(pages, 2, 16, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    table, lens, starts = torch.zeros(3, cols, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    q = torch.zeros(71, 8, 128, dtype=torch.float16, device="cuda")

    def put(pr):
        for dst, src in ((k, pr["k"]), (v, pr["v"]), (lens, pr["lens"]), (starts, pr["starts"]), (q, pr["q"])):
            dst[:src.shape[0]] = src.cuda()
        table[:, :pr["table"].shape[1]] = pr["table"].cuda()

    put(before)
    cache = lw.PagedCache(k, v)
    cache.attend_prompt(q, table, lens, starts), cache.attend(q[:3], table, lens)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((cache.attend_prompt(q, table, lens, starts), cache.attend(q[:3], table, lens)))
        graphs.append(g)
    for pr in (after, before, after):
        put(pr)
        want = cache.attend_prompt(q, table, lens, starts), cache.attend(q[:3], table, lens)
        rows = int(pr["starts"][-1])
        for o in outs:
            o[0].fill_(9.0), o[1].fill_(9.0)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0][:rows], want[0][:rows]) and torch.equal(o[1], want[1])


def test_another_stream(lw):
    import torch
    pr = problem([900, 31], [100, 31], 8, 2, 64, 16, "bf16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    args = [pr[n].cuda() for n in ("q", "table", "lens", "starts")]
    want = cache.attend_prompt(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:                       # two calls of one cache at once
            with torch.cuda.stream(s):
                got.append(cache.attend_prompt(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_python_refusals(lw):
    import torch
    pr = problem([40, 40], [2, 2], 4, 2, 64, 16, "fp16")
    k, v = pr["k"].cuda(), pr["v"].cuda()
    cache = lw.PagedCache(k, v)
    q, table, lens, starts = (pr[n].cuda() for n in ("q", "table", "lens", "starts"))
    cos = torch.ones(64, 32, device="cuda")
    qkv = torch.ones(4, 8 * 64, device="cuda")
    for bad in (dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(table=table.long()), dict(table=table[:1]), dict(lens=lens.cpu()),
                dict(starts=starts[:2]), dict(starts=starts.long()), dict(out=q[:2]), dict(out=q.bfloat16()), dict(table=table.t().contiguous().t())):
        a = dict(dict(q=q, table=table, lens=lens, starts=starts), **bad)
        with pytest.raises(ValueError):
            cache.attend_prompt(**a)
        a.pop("starts")
        if "starts" not in bad:
            with pytest.raises(ValueError):
                cache.attend(**dict(a, q=a["q"][:2] if "q" not in bad else a["q"]) if "out" not in bad else dict(a, q=q[:2], out=q[:1]))
    for bad in (dict(qkv=qkv.double()), dict(qkv=qkv[:, :64]), dict(cos=cos.half()), dict(cos=cos[:, ::2]), dict(sin=cos[:8]), dict(q=q.float()), dict(q=q[:3])):
        with pytest.raises(ValueError):
            cache.append(**dict(dict(qkv=qkv, n_heads=4, cos=cos, sin=cos, table=table, lens=lens, starts=starts), **bad))
    with pytest.raises(lw.LwError):                                              # 3 query heads over 2 kv heads
        cache.append(torch.ones(4, 7 * 64, device="cuda"), 3, cos, cos, table, lens, starts=starts)
    with pytest.raises(lw.LwError):
        cache.attend_prompt(q[:, :3].contiguous(), table, lens, starts)
    with pytest.raises(lw.LwError):
        cache.attend(q[:2], table, lens, scale=float("nan"))
    for pools in ((k, v.bfloat16()), (k, v[:, :1]), (k, v.cpu()), (k.float(), v.float()), (k[..., ::2], v[..., ::2]), (k, v.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            lw.PagedCache(*pools)
    with pytest.raises(lw.LwError):
        lw.PagedCache(k[:, :, :12].contiguous(), v[:, :, :12].contiguous())       # page size


def test_windows_that_do_not_fit_are_refused(lw):
    pr = problem([40, 40], [2, 2], 4, 2, 64, 16, "fp16")
    cache = lw.PagedCache(pr["k"].cuda(), pr["v"].cuda())
    q, table, lens, starts = (pr[n].cuda() for n in ("q", "table", "lens", "starts"))
    for window in (-1, 2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError):
            cache.attend(q[:2], table, lens, window=window)
        with pytest.raises(ValueError):
            cache.attend_prompt(q, table, lens, starts, window=window)


def test_prompt_then_tokens(lw):
    """A whole use: packed prompts are appended and attended to, in two pieces for one of them, then tokens one by one."""
    import torch
    from tests import paged_ref as ref
    heads, kv_heads, dim, page = 8, 2, 128, 16
    gen = torch.Generator().manual_seed(11)
    final = [90, 33]
    pages, table, _, _ = ref.sequences(final, [0, 0], page, gen)
    cache = lw.PagedCache.empty(pages, kv_heads, page, dim)
    angle = torch.arange(128, dtype=torch.float64)[:, None] * (1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim))[None]
    cos, sin = angle.cos().float(), angle.sin().float()
    rows = [torch.randn(n, (heads + 2 * kv_heads) * dim, generator=gen) for n in final]
    steps = [([50, 20], [50, 20]), ([84, 20], [34, 0])] + [([84 + i, 20 + i], [1, 1]) for i in range(1, 7)]
    done = [0, 0]
    for lens, news in steps:
        packed = torch.cat([rows[b][done[b]:done[b] + news[b]] for b in range(2)]).cuda()
        lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
        if news == [1, 1]:
            q = cache.append(packed, heads, cos.cuda(), sin.cuda(), table.cuda(), lens_t)
            out = cache.attend(q, table.cuda(), lens_t)
        else:
            starts = torch.tensor([0, news[0], sum(news)], dtype=torch.int32).cuda()
            q = cache.append(packed, heads, cos.cuda(), sin.cuda(), table.cuda(), lens_t, starts=starts)
            out = cache.attend_prompt(q, table.cuda(), lens_t, starts)
        k, v = cache.k_pages.cpu(), cache.v_pages.cpu()
        first = 0
        for b in range(2):
            pos = torch.arange(lens[b] - news[b], lens[b])
            rq, rk, rv, e = ref.rotate(rows[b][:lens[b]], heads, kv_heads, dim, cos, sin, torch.arange(lens[b]))
            held = ref.load(k, table, b, lens[b])
            assert ((held - rk).abs() <= e[:, heads:] * (1 + ref.EPS[torch.float16]) + rk.abs() * ref.EPS[torch.float16] + ref.TINY[torch.float16]).all()
            want, bound, _ = ref.attend(q[first:first + news[b]].cpu(), held, ref.load(v, table, b, lens[b]), pos, dim ** -0.5, 0)
            assert ((out[first:first + news[b]].cpu().double() - want).abs() <= bound).all()
            first += news[b]
        done = [d + m for d, m in zip(done, news)]
