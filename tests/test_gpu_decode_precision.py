"""What a decoder's operators keep where fewer bits would go unnoticed beside a rounding to fp16: fp32 results, against fp64."""
import numpy as np
import pytest

import juliavision_b200 as jv
from tests import decode_ref as ref
from tests.test_gpu_decode import F32, Cached, STEP, attend, near

pytestmark = pytest.mark.gpu


def bound(c, q, scale, causal, got):
    """The wanted results and how far off they may be.  Weights in two fp16 halves: 2^-21 of themselves (2^-10 left by the upper half
    where it is cut off, 2^-11 of that by the lower), and fp16's least step, 2^-24, a key, of weights that are 2^6 at least where the row's largest
    product of a weight and its page's scale is.  A score's fp32 sum, off by 2^-20 of the sum of magnitudes at most, moves a weight
    and the row's sum; exponential, sum and quotient 2^-19 together; the result's own rounding."""
    want, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    L, G = q.shape[1], q.shape[2] // c.H
    for b, n in enumerate(c.lens):
        k, v = (ref.tokens(a, t, c.kind, c.table, b, n) for a, t in ((c.k, c.kmax), (c.v, c.vmax)))
        hidden = (np.arange(n) > np.arange(n - L, n)[:, None]) if causal else np.zeros((L, n), bool)
        o, a, reach = ref.attention(q[b].astype(np.float64), k, v, hidden, scale)
        s = np.einsum("lhe,nhe->lhn", q[b].astype(np.float64), np.repeat(k, G, 1)) * scale
        s[np.broadcast_to(hidden[:, None], s.shape)] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        top = np.repeat(c.vmax[c.table[b, np.arange(n) // c.T]], G, 1).T                              # (Hq, n)
        want[b] = o
        tol[b] = a * (2.0 ** -21 + 2 * 2.0 ** -20 * reach + 2.0 ** -19) + n * 2.0 ** -30 * (p * top).max(-1)[..., None] + STEP[F32][0] * np.abs(o)
    near(got, want, tol)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("E, G, L", [(128, 4, 1), (128, 4, 8), (128, 3, 11), (128, 4, 75), (64, 5, 1), (64, 5, 8), (64, 41, 1), (64, 12, 4), (64, 49, 1), (64, 1, 300)])
def test_weights_keep_their_bits(ctx, E, G, L, kind):
    """Few query rows a key head and many, on both sides of where one kernel takes over from the other: rows of nearly equal weights."""
    rng = np.random.default_rng(21)
    c = Cached(ctx, rng, E, 32, 2, [500, 317], kind)
    q = rng.standard_normal((2, L, 2 * G, E)).astype(np.float16)
    scale = 0.6 / E
    got, _, _ = attend(ctx, c, q, None, scale, True, F32)
    bound(c, q, scale, True, got)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("ratio", [20, 28, 36])
@pytest.mark.parametrize("where", ["unseen", "unweighed", "zeros"])
@pytest.mark.parametrize("E, G, L", [(128, 1, 30), (128, 3, 60), (64, 1, 40), (64, 2, 250)])
def test_large_values_reach_only_rows_that_weigh_them(ctx, E, G, L, where, ratio, kind):
    """A page whose largest value is 2^ratio of the others', which a row does not see (the last page, but for the last rows) or gives no weight
    (the first, whose scores are 50 and more below), and pages of zeros beside it: the others' values keep their bits."""
    rng = np.random.default_rng(25)
    n = 16 * 20 + L
    c = Cached(ctx, rng, E, 16, 2, [n], kind)
    q = np.abs(rng.standard_normal((1, L, 2 * G, E))).astype(np.float16)
    scale = 0.5 / E
    page = c.table[0, (n - 1) // 16 if where == "unseen" else 0]
    c.vmax *= np.float32(2.0 ** -20)
    c.vmax[page] *= np.float32(2.0 ** ratio)
    if where == "unweighed":      # sums of E terms of some 0.8 times -kmax
        c.k[page] = -127 if kind == "int8" else 0xfe
        c.kmax[page] = 300.0
    if where == "zeros":
        c.vmax[c.table[0, 1:4]] = 0
        c.k[page] = 0
    for a, host in ((c.cache.k, c.k), (c.cache.kmax, c.kmax), (c.cache.vmax, c.vmax)):
        ctx.upload(a, host)
    got, _, _ = attend(ctx, c, q, None, scale, True, F32)
    bound(c, q, scale, True, got)


# ------------------------------------------------------------------------------------------------- 4-bit products
def product(ctx, rng, N, M, K, group, zeros, scales, size, pad=0, epi="identity"):
    """A product as fp32, the wanted one and the sum of magnitudes."""
    q = rng.integers(0, 16, (K, M)).astype(np.uint8)
    s = scales((K // group, M)).astype(np.float16)
    z = rng.integers(0, 16, (K // group, M)).astype(np.uint8) if zeros else None
    x = (rng.standard_normal((N, K + pad)) * size).astype(np.float16)
    w = jv.pack4(ctx, ctx.toback(q), ctx.toback(s), None if z is None else ctx.toback(z), group)
    d, buf = ctx.toback(x), ctx.allocate(F32, M + 1, N + 1)
    ctx.fill_bytes(buf, 0xFF)
    ctx.ws.reset()
    jv.matmul4_(ctx, jv.DeviceArray(ctx, buf.ptr, F32, (M, N), (1, M + 1), owner=buf), w, jv.DeviceArray(ctx, d.ptr, np.float16, (K, N), (1, K + pad), owner=d),
                epi=epi)
    ctx.synchronize()
    got = buf.to_host()
    assert np.isnan(got[N:]).all() and np.isnan(got[:, M:]).all()
    x, w = x[:, :K].astype(np.float64), ref.weight4(q, s, z, group)
    return got[:N, :M], x @ w, np.abs(x) @ np.abs(w)


def sums(K):
    """fp32 sums of fp16 products, in steps of sixteen at least: each off by 2^-23 of what it adds up, which is the sum of magnitudes at most;
    and a few more where parts meet."""
    return 2.0 ** -23 * (K / 16 + 8)


@pytest.mark.parametrize("N", [96, 97, 300, 513, 600])
@pytest.mark.parametrize("M, K, group, zeros, pad", [(200, 512, 64, False, 0), (333, 480, 32, True, 0), (64, 256, 128, True, 1)])
def test_weights_are_exact_for_any_number_of_tokens(ctx, M, K, group, zeros, pad, N):
    rng = np.random.default_rng(22)
    got, want, reach = product(ctx, rng, N, M, K, group, zeros, lambda n: rng.random(n) * 0.02 + 0.001, 1.0, pad)
    near(got, want, reach * sums(K) + STEP[F32][0] * np.abs(want))


@pytest.mark.parametrize("N", [1, 16, 40, 96, 97, 300, 513])
def test_weights_past_the_range_of_fp16(ctx, N):
    """Scales up to fp16's largest beside ones of 2^-24 and negative ones: (q - z) s is a number for any number of tokens.  In a row with a scale above 4096
    it may be held to 2^-20, off by 2^-21, which is nothing beside what stands at that scale."""
    rng = np.random.default_rng(23)
    M, K, group = 130, 256, 32

    def scales(n):
        s = 2.0 ** rng.uniform(-24, 15.9, n) * rng.choice([-1, 1], n)
        s[:, ::3] = np.minimum(np.abs(s[:, ::3]), 2.0)
        return s

    got, want, reach = product(ctx, rng, N, M, K, group, True, scales, 2.0 ** -6)
    assert np.isfinite(got).all() and np.abs(want).max() > 2.0 ** 13
    near(got, want, reach * sums(K) + STEP[F32][0] * np.abs(want) + 2.0 ** -21 * K * 2.0 ** -6 * 5 * (reach > 256))


def test_many_tokens_through_blocks_of_rows(ctx):
    """More rows than are laid out at a time, the last block of them a part, more tokens than a product takes at a time; every result against a column and
    a row that are summed exactly."""
    rng = np.random.default_rng(24)
    N, M, K, group = 2100, 9000, 4096, 128
    q, s = rng.integers(0, 16, (K, M)).astype(np.uint8), (rng.random((K // group, M)) * 0.02 + 0.001).astype(np.float16)
    x, bias = rng.standard_normal((N, K)).astype(np.float16), rng.standard_normal(M).astype(np.float16)
    w = jv.pack4(ctx, ctx.toback(q), ctx.toback(s), None, group)
    out = ctx.allocate(np.float16, M, N)
    ctx.fill_bytes(out, 0xFF)
    ctx.ws.reset()
    jv.matmul4_(ctx, out, w, ctx.toback(x), ctx.toback(bias), epi="relu")
    got = out.to_host().astype(np.float64)
    assert np.isfinite(got).all()
    rows, tokens = np.r_[0:M:61, M - 1], np.r_[0:N:37, N - 1]
    for m, n in ((rows, slice(None)), (slice(None), tokens)):
        wm, xn = ref.weight4(q[:, m], s[:, m], None, group), x[n].astype(np.float64)
        want, reach = xn @ wm + bias[m].astype(np.float64), np.abs(xn) @ np.abs(wm)
        tol = reach * sums(K) + STEP[np.float16][0] * np.abs(want) + STEP[np.float16][1]
        near(got[n][:, m] if isinstance(n, slice) else got[n], np.maximum(want, 0), tol)


# ---------------------------------------------------------------------------------------------------------- wide tables
@pytest.mark.parametrize("E, G, L", [(128, 2, 1), (128, 4, 8), (64, 3, 100), (128, 1, 700)])
def test_tables_for_longer_sequences(ctx, E, G, L):
    """A table allotted for a hundred times the tokens there are, whose entries past a sequence's length name no page: they are not read."""
    rng = np.random.default_rng(26)
    c = Cached(ctx, rng, E, 16, 2, [900, 701, 0], "int8")
    c.lens[2] = 0
    table = rng.choice([-1, 1 << 30, -(1 << 31)], (3, 6000))
    for b, n in enumerate(c.lens):
        table[b, :-(-n // 16)] = c.table[b, :-(-n // 16)]
    q = rng.standard_normal((3, L, 2 * G, E)).astype(np.float16)
    news = np.array([L, L, 0])
    wide = ctx.toback(table.astype(np.int32))
    c.dtable = wide
    got, want, tol = attend(ctx, c, q, news, 1 / E, True, F32)           # synchronises: an entry that was followed would be reported
    near(got, want, tol)
    new = ctx.toback(rng.standard_normal((3, L, 2, E)).astype(np.float16)).permute((0, 2, 1, 3))
    lens, dnews = (ctx.toback(np.array(v, np.int32)) for v in (c.lens, news))
    jv.cacheappend_(ctx, c.cache, new, new, wide, lens, dnews)
    jv.cacheread_(ctx, ctx.allocate(F32, E, 1000, 2, 3), c.cache, "k", wide, lens)
    ctx.synchronize()


@pytest.mark.parametrize("E, rot, inter", [(1024, 1024, False), (1100, 1024, True), (4096, 1000, False)])
def test_rotary_of_the_widest_heads(ctx, E, rot, inter):
    rng = np.random.default_rng(27)
    x = rng.standard_normal((2, 5, 3, E)).astype(np.float16)
    lens = np.array([100005, 7])
    out = ctx.allocate(np.float16, E, 3, 5, 2).permute((0, 2, 1, 3))
    jv.rotary_(ctx, jv.rotaryplan(ctx, rot, interleaved=inter), out, ctx.toback(x).permute((0, 2, 1, 3)), lens=ctx.toback(lens.astype(np.int32)))
    ctx.synchronize()
    want = ref.rotary(x, (lens - 5)[:, None] + np.arange(5), *jv.rotaryfrequencies(rot), inter)
    # fp32: angles off by 2^-25 turns and the library's sine and cosine by 2^-23 or so, three roundings of at most 2^-24
    slack = 2.0 ** -20 * 2 * np.abs(x.astype(np.float64)).max(-1, keepdims=True)
    near(ctx.contiguous(out.permute((0, 2, 1, 3))).to_host(), want, STEP[np.float16][0] * np.abs(want) + STEP[np.float16][1] + slack)


def test_the_code_of_a_nan_among_values(ctx):
    """A cache that another program filled may hold e4m3's NaN: cacheread says so, attention's keys too; as a value attention takes it as 448, since rows
    that do not see it share its tile."""
    rng = np.random.default_rng(28)
    for L in (2, 90):
        c = Cached(ctx, rng, 64, 16, 1, [200], "e4m3")
        c.v[c.table[0, 3], 0, 5, 7] = 0x7f
        ctx.upload(c.cache.v, c.v)
        out = ctx.allocate(F32, 64, 200, 1, 1)
        jv.cacheread_(ctx, out, c.cache, "v", c.dtable, c.dlens)
        ctx.synchronize()
        assert np.argwhere(np.isnan(out.to_host()[0, 0])).tolist() == [[3 * 16 + 5, 7]]
        c.v[c.table[0, 3], 0, 5, 7] = 0x7e                                       # 448
        q = rng.standard_normal((1, L, 2, 64)).astype(np.float16)
        near(*attend(ctx, c, q, None, 0.01, True))


@pytest.mark.parametrize("N", [1, 40, 300, 513, 600])
def test_infinite_inputs_give_infinite_sums(ctx, N):
    """An infinite input of some tokens against weights that are not zero: infinite of the weight's sign, other tokens as they were."""
    rng = np.random.default_rng(29)
    M, K = 70, 128
    q = rng.integers(0, 7, (K, M)).astype(np.uint8) + rng.integers(0, 2, (K, M)).astype(np.uint8) * 9       # not 8
    q[q == 8] = 9
    s = (rng.random((2, M)) * 0.02 + 0.001).astype(np.float16)
    s[:, ::2] = np.float16(0.0078125)                                  # products that one fp16 number holds
    x = rng.standard_normal((N, K)).astype(np.float16)
    x[N // 2, 5] = np.inf
    w = jv.pack4(ctx, ctx.toback(q), ctx.toback(s), None, 64)
    out = ctx.allocate(F32, M, N)
    jv.matmul4_(ctx, out, w, ctx.toback(x))
    ctx.synchronize()
    got, wd = out.to_host(), ref.weight4(q, s, None, 64)
    assert np.array_equal(got[N // 2], np.where(wd[5] > 0, np.inf, -np.inf))
    rest = np.arange(N) != N // 2
    xd = x[rest].astype(np.float64)
    near(got[rest], xd @ wd, np.abs(xd) @ np.abs(wd) * sums(K) + STEP[F32][0] * np.abs(xd @ wd))


def test_many_tokens_take_a_bounded_workspace(ctx):
    """Rows are laid out some at a time, whatever the shape: 60000 rows' sums alone would be a gigabyte."""
    rng = np.random.default_rng(30)
    N, M, K = 2048, 60000, 64
    q, s = rng.integers(0, 16, (K, M)).astype(np.uint8), (rng.random((1, M)) * 0.02).astype(np.float16)
    x = rng.standard_normal((N, K)).astype(np.float16)
    w = jv.pack4(ctx, ctx.toback(q), ctx.toback(s), None, 64)
    out = ctx.allocate(np.float16, M, N)
    ctx.ws.reset()
    jv.matmul4_(ctx, out, w, ctx.toback(x))
    ctx.synchronize()
    used = ctx.ws.stats()[0]
    ctx.ws.reset()
    assert used <= 257 << 20, used
    got = out.to_host()[::97]
    xd, wd = x[::97].astype(np.float64), ref.weight4(q, s, None, 64)
    near(got, xd @ wd, np.abs(xd) @ np.abs(wd) * sums(K) + STEP[np.float16][0] * np.abs(xd @ wd) + STEP[np.float16][1])


@pytest.mark.parametrize("M, K, N", [(200, 512, 600), (9000, 4096, 520), (8192, 4096, 40), (1000, 512, 300)])
def test_products_are_the_same_twice_and_replayed(ctx, M, K, N):
    """The same bits by calls and by two graphs whose workspaces are one, replayed in turn with calls between them."""
    rng = np.random.default_rng(31)
    q, s = rng.integers(0, 16, (K, M)).astype(np.uint8), (rng.random((K // 64, M)) * 0.02).astype(np.float16)
    w = jv.pack4(ctx, ctx.toback(q), ctx.toback(s), None, 64)
    xs = [ctx.toback(rng.standard_normal((N, K)).astype(np.float16)) for _ in range(2)]
    outs = [ctx.allocate(F32, M, N) for _ in range(2)]
    first = []
    for x, out in zip(xs, outs):
        ctx.ws.reset()
        jv.matmul4_(ctx, out, w, x)
        first.append(out.to_host())
    assert not np.array_equal(*first)
    graphs = []
    for x, out in zip(xs, outs):
        ctx.ws.reset()
        graphs.append(ctx.capture(lambda o=out, x=x: jv.matmul4_(ctx, o, w, x)))
        ctx.fill_bytes(out, 0xFF)
    spare = ctx.allocate(F32, M, N)
    for _ in range(2):
        for g in graphs:
            g.replay()
        ctx.ws.reset()
        jv.matmul4_(ctx, spare, w, xs[0])
    ctx.synchronize()
    assert all(np.array_equal(a, o.to_host()) for a, o in zip(first + first[:1], outs + [spare]))
