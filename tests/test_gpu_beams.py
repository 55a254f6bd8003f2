"""Beam search's choice, against fp64 and whole orders of all candidates; the beams' caches brought in line, against copies in numpy."""
import numpy as np
import pytest

import juliavision_b200 as jv
from tests.test_gpu_decode import F16, F32, Cached, ints, near

pytestmark = pytest.mark.gpu


def choice(x, scores, N, ended=None, pad=0):
    """x (B, K, V), scores (B, K): the N best in order, from all candidates sorted."""
    B, K, V = x.shape
    best, parents, tokens = (np.zeros((B, N), t) for t in (np.float64, np.int32, np.int32))
    for b in range(B):
        c = np.full((K, V), -np.inf)
        for k in range(K):
            s = float(scores[b, k])
            if not np.isfinite(s):
                continue
            if ended is not None and ended[b, k]:
                c[k, pad] = s
                continue
            r = x[b, k].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
                top = np.max(r)
                total = top + np.log(np.exp(r - top).sum())
                if np.isfinite(total):
                    c[k] = s + (r - total)
        order = np.lexsort((np.arange(K * V), -c.ravel()))[:N]
        best[b], parents[b], tokens[b] = c.ravel()[order], order // V, order % V
    return best, parents, tokens


def select(ctx, x, scores, N, ended=None, pad=0, device=None):
    B, K, V = x.shape
    d = ctx.toback(x) if device is None else device
    out = [ctx.allocate(t, N, B) for t in (F32, np.int32, np.int32)]
    for o in out:
        ctx.fill_bytes(o, 0xFF)
    ctx.ws.reset()
    jv.beamselect_(ctx, *out, d, ctx.toback(scores.astype(F32)), None if ended is None else ints(ctx, ended), pad)
    ctx.synchronize()
    return [o.to_host() for o in out]


def agree(got, want, tiles=4):
    """Whole numbers equal.  The scores: half a step of fp32, and a log sum whose terms are off by 2^-22 and their fp32 sums by the length of a lane's
    chain (16 additions a tile), 5 steps over lanes and 8 over warps."""
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]), (got, want)
    near(np.where(np.isinf(want[0]) & (got[0] == want[0]), 0, got[0]), np.nan_to_num(want[0], neginf=0),
         np.nan_to_num(2.0 ** -24 * np.abs(want[0]), posinf=0) + 2.0 ** -22 + (16 * tiles + 13) * 2.0 ** -24)


CASES = [  # B, K, V, N
    (1, 1, 1, 1), (1, 1, 32, 32), (2, 3, 5, 15), (1, 5, 51865, 5), (3, 4, 1000, 8), (2, 8, 8193, 16), (1, 32, 777, 32), (7, 2, 70001, 3), (1, 16, 131072, 32),
    (40, 6, 12345, 6), (1, 2, 31, 32), (2, 3, 2, 5)]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [F16, F32])
def test_choice(ctx, case, dtype):
    B, K, V, N = case
    rng = np.random.default_rng(1)
    x = (3 * rng.standard_normal((B, K, V))).astype(dtype)
    scores = (-20 * rng.random((B, K))).astype(F32)
    agree(select(ctx, x, scores, N), choice(x, scores, N))
    ended = rng.random((B, K)) < 0.3
    x[rng.random(x.shape) < 0.2] = -np.inf
    scores[rng.random((B, K)) < 0.2] = -np.inf
    pad = V // 3
    agree(select(ctx, x, scores, N, ended, pad), choice(x, scores, N, ended, pad))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("value", [0.0, -0.0, -7.5, 60000.0])
def test_ties_go_to_the_lowest(ctx, dtype, value):
    """All logits alike, all beams alike; then two heights with the higher one rare; zeros of either sign are one number."""
    x = np.full((2, 4, 9001), value, dtype)
    scores = np.full((2, 4), -3.0, F32)
    agree(select(ctx, x, scores, 20), choice(x, scores, 20), tiles=1)
    x[:, 2, 5000::7] = 0 if value == 0 else value + 1000 if value > 100 else value + 2
    x[:, 1, 100:103] = -value if value == 0 else value
    agree(select(ctx, x, scores, 32), choice(x, scores, 32), tiles=1)


def test_rising_and_falling_rows(ctx):
    """Every element a new largest, or none after the first: the bound of a share moves each tile, or never."""
    V = 60000
    up = (np.arange(V) / 1000).astype(F32)
    x = np.stack((up, up[::-1], np.zeros(V, F32)))[None]
    scores = np.array([[-1.0, -1.0, 40.0]], F32)
    agree(select(ctx, x, scores, 32), choice(x, scores, 32), tiles=8)


def test_what_is_not_finite(ctx):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((2, 6, 3001)).astype(F16)
    scores = -rng.random((2, 6)).astype(F32)
    x[0, 0, 2999], x[0, 1, 7], x[0, 2] = np.nan, np.inf, -np.inf
    scores[0, 3], scores[1, 0], scores[1, 1] = np.nan, np.inf, -np.inf
    for N in (1, 12, 32):
        agree(select(ctx, x, scores, N), choice(x, scores, N))
    x[:] = np.nan
    agree(select(ctx, x, scores, 9), choice(x, scores, 9))
    x[:] = -np.inf
    x[1, 4, 1234] = -1        # one candidate in all
    agree(select(ctx, x, scores, 9), choice(x, scores, 9))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("V", [5, 40, 3000, 60000])
def test_few_tokens_that_may_come(ctx, dtype, V):
    """All but a few logits at -inf: those few, and then the lowest of the others at -inf, whichever of them are among the few."""
    rng = np.random.default_rng(11)
    N = min(20, V)
    x, scores = np.full((6, 2, V), -np.inf, dtype), -rng.random((6, 2)).astype(F32)
    for b, few in enumerate(([], [0], [V - 1, 1], list(range(N - 2)), [0, 2, 3, 4], list(range(max(V - 25, 0), V)))):
        for k in range(2):
            for t in few:
                x[b, k, t] = rng.standard_normal()
    scores[4, 1] = -np.inf
    agree(select(ctx, x, scores, N), choice(x, scores, N))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_strides_and_alignment(ctx, dtype, offset):
    """Rows that start anywhere, beams and searches apart; the two-axis form of a projection's result."""
    rng = np.random.default_rng(3)
    B, K, V, pitch = 2, 3, 2050, 2057
    buf = rng.standard_normal(B * K * pitch + 64).astype(dtype) + 50          # what lies between is larger than any logit
    x = rng.standard_normal((B, K, V)).astype(dtype)
    for b in range(B):
        for k in range(K):
            at = offset + (b * K + k) * pitch
            buf[at:at + V] = x[b, k]
    d = ctx.toback(buf)
    scores = -rng.random((B, K)).astype(F32)
    ptr = d.ptr + offset * np.dtype(dtype).itemsize
    three = jv.DeviceArray(ctx, ptr, dtype, (V, K, B), (1, pitch, K * pitch), owner=d)
    two = jv.DeviceArray(ctx, ptr, dtype, (V, K * B), (1, pitch), owner=d)
    want = choice(x, scores, 7)
    agree(select(ctx, x, scores, 7, device=three), want)
    agree(select(ctx, x, scores, 7, device=two), want)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_that_end_where_a_block_does(ctx, dtype):
    """Rows of an odd pitch start at all places of a vector; those that start on one leave a block without an element."""
    rng = np.random.default_rng(8)
    V = 1024 * (8 if dtype == F16 else 4)
    x, scores = rng.standard_normal((2, 5, V + 1)).astype(dtype), -rng.random((2, 5)).astype(F32)
    d = ctx.toback(x)
    rows = jv.DeviceArray(ctx, d.ptr, dtype, (V, 5, 2), (1, V + 1, 5 * (V + 1)), owner=d)
    for _ in range(3):
        agree(select(ctx, x[..., :V], scores, 9, device=rows), choice(x[..., :V], scores, 9))


def test_recorded_choice(ctx):
    rng = np.random.default_rng(4)
    x, scores = rng.standard_normal((3, 5, 30011)).astype(F16), -rng.random((3, 5)).astype(F32)
    dx, ds = ctx.toback(x), ctx.toback(scores)
    outs = [[ctx.allocate(t, 5, 3) for t in (F32, np.int32, np.int32)] for _ in range(2)]
    graphs = []
    for o in outs:
        ctx.ws.reset()
        jv.beamselect_(ctx, *o, dx, ds)
        ctx.ws.reset()
        graphs.append(ctx.capture(lambda o=o: jv.beamselect_(ctx, *o, dx, ds)))
    for _ in range(3):
        x = rng.standard_normal(x.shape).astype(F16)
        ctx.upload(dx, x)
        for g in graphs:
            g.replay()
        ctx.synchronize()
        for o in outs:
            agree([a.to_host() for a in o], choice(x, scores, 5))


# ---------------------------------------------------------------------------------------------------- the caches
REORDER = [  # searches, beams, E, T, H, lengths, kind, caches
    (1, 1, 64, 16, 1, [5], "int8", 1), (2, 5, 64, 32, 3, [40, 64], "int8", 3), (1, 32, 128, 16, 2, [33], "e4m3", 1), (3, 4, 80, 64, 5, [1, 0, 190], "int8", 2),
    (4, 2, 16, 128, 20, [128, 129, 255, 7], "e4m3", 1), (1, 9, 96, 16, 1, [16], "int8", 2), (2, 17, 48, 32, 2, [95, 96], "int8", 2)]


@pytest.mark.parametrize("case", REORDER, ids=str)
@pytest.mark.parametrize("way", ["random", "rotate", "reverse", "first", "stay"])
@pytest.mark.parametrize("joined", [False, True])
def test_reorder(ctx, case, way, joined):
    B, K, E, T, H, lengths, kind, n = case
    rng = np.random.default_rng(5)
    S, lens = B * K, np.repeat(lengths, K)
    width = max(lengths) // T + 2
    P = S * width + 3
    caches = [Cached(ctx, rng, E, T, H, [P * T], kind, spare=0, joined=joined) for _ in range(n)]
    own = rng.permutation(P)[:S * width].reshape(S, width)
    table = own.copy()
    for s in range(S):
        full = lens[s] // T
        table[s, :full] = own[s // K * K + rng.integers(0, K, full), np.arange(full)]
    parents = {"random": rng.integers(0, K, (B, K)), "rotate": np.tile(np.roll(np.arange(K), 1), (B, 1)), "reverse": np.tile(np.arange(K)[::-1], (B, 1)),
               "first": np.zeros((B, K), int), "stay": np.tile(np.arange(K), (B, 1))}[way]
    source = np.arange(S) // K * K + parents.ravel()
    want_table = np.where(np.arange(width) < (lens // T)[:, None], table[source], own)
    before = [c.host() for c in caches]
    dtable = ints(ctx, table)
    arg = caches[0].cache if n == 1 else [c.cache for c in caches]
    jv.cachereorder_(ctx, arg, dtable, ints(ctx, own), ints(ctx, parents), ints(ctx, lens))
    ctx.synchronize()
    assert np.array_equal(dtable.to_host(), want_table)
    for c, old in zip(caches, before):
        new = c.host()
        for i in range(2):
            data, most = old[i].copy(), old[2 + i].copy()
            for s in range(S):
                full, kept = divmod(lens[s], T)
                if kept:
                    data[own[s, full], :, :kept] = old[i][own[source[s], full], :, :kept]
                    most[own[s, full]] = old[2 + i][own[source[s], full]]
            assert np.array_equal(new[i], data) and np.array_equal(new[2 + i], most)


def test_more_caches_than_a_launch_takes(ctx):
    rng = np.random.default_rng(6)
    made = [Cached(ctx, rng, 16, 16, 1, [64], "int8", spare=0) for _ in range(131)]
    own, parents, lens = np.array([[2, 0], [1, 3]]), [[1, 1]], [21, 21]
    dtable = ints(ctx, [[2, 0], [2, 3]])
    before = [c.host() for c in made]
    jv.cachereorder_(ctx, [c.cache for c in made], dtable, ints(ctx, own), ints(ctx, parents), ints(ctx, lens))
    ctx.synchronize()
    assert np.array_equal(dtable.to_host(), [[2, 0], [2, 3]])
    for c, old in zip(made, before):
        want = old[0].copy()
        want[0, :, :5] = old[0][3, :, :5]
        assert np.array_equal(c.host()[0], want)


@pytest.mark.parametrize("wrong", ["parent", "page", "length", "unequal"])
def test_bad_entries_are_skipped_and_reported(ctx, wrong):
    c = Cached(ctx, np.random.default_rng(7), 64, 16, 2, [96], "int8", spare=0)
    own, parents, lens = np.array([[0, 1], [2, 3], [4, 5]]), np.array([[1, 2, 0]]), np.array([20, 20, 20])
    if wrong == "parent":
        parents = np.array([[3, -1, 1]])
    if wrong == "page":
        own = np.array([[0, 1], [2, 6], [4, -1]])
    if wrong == "length":
        lens = np.array([33, 33, 33])
    if wrong == "unequal":
        lens = np.array([20, 21, 20])
    old = c.host()
    dtable = ints(ctx, own)
    jv.cachereorder_(ctx, c.cache, dtable, ints(ctx, own), ints(ctx, parents), ints(ctx, lens))
    with pytest.raises(jv.B200Error) as e:
        ctx.synchronize()
    assert e.value.code == 4
    ctx.synchronize()
    new = c.host()
    if wrong == "parent":       # beams 0 and 1 stay, 2 follows 1
        want = old[0].copy()
        want[5, :, :4] = old[0][3, :, :4]
        assert np.array_equal(new[0], want) and np.array_equal(dtable.to_host(), [[0, 1], [2, 3], [2, 5]])
    if wrong in ("page", "length"):      # nothing to copy from, or to; or no page that is part full
        assert np.array_equal(new[0], old[0]) and np.array_equal(new[3], old[3])


def test_offsets_past_32_bits(ctx):
    """Searches that lie further than 2^32 bytes apart."""
    rng = np.random.default_rng(9)
    V, K, ldb = 1003, 3, (1 << 31) + 40
    d = ctx.allocate(F16, ldb + K * V)
    x, scores = rng.standard_normal((2, K, V)).astype(F16), -rng.random((2, K)).astype(F32)
    for b in range(2):
        ctx.upload(jv.DeviceArray(ctx, d.ptr + 2 * ldb * b, F16, (V, K), owner=d), x[b])
    agree(select(ctx, x, scores, 5, device=jv.DeviceArray(ctx, d.ptr, F16, (V, K, 2), (1, V, ldb), owner=d)), choice(x, scores, 5))


def test_reorder_past_32_bits(ctx):
    E, T, H, P = 128, 128, 8, 40000                     # 5.2 GB of keys and of values
    c = jv.Cache8(*(ctx.allocate(np.int8, E, T, H, P) for _ in range(2)), *(ctx.allocate(F32, H, P) for _ in range(2)))
    rng = np.random.default_rng(10)
    own = np.array([[39999], [3], [39000]])
    page = lambda a, g: jv.DeviceArray(ctx, a.ptr + g * E * T * H, np.int8, (E, T, H), owner=a)  # noqa: E731
    data = rng.integers(-127, 128, (3, 2, H, T, E)).astype(np.int8)
    for s in range(3):
        for i, a in enumerate((c.k, c.v)):
            ctx.upload(page(a, own[s, 0]), data[s, i])
    jv.cachereorder_(ctx, c, ints(ctx, own), ints(ctx, own), ints(ctx, [[1, 2, 0]]), ints(ctx, [77] * 3))
    ctx.synchronize()
    for s, source in enumerate((1, 2, 0)):
        for i, a in enumerate((c.k, c.v)):
            want = data[s, i].copy()
            want[:, :77] = data[source, i][:, :77]
            assert np.array_equal(page(a, own[s, 0]).to_host(), want)
