"""Attention of packed sequences against fp64 (tests/decode_ref.py), at the lengths, head layouts and masks where it can go wrong.

Tolerances count roundings.  A weight is rounded to fp16 (2^-11 of itself; below 2^-14 of 2^-7 of the heaviest weight a step of 2^-24, so
2^-32 of the heaviest a key), scores are fp32 sums of E products (E 2^-24 of the sum of their sizes, which moves a weight by as much), sums and
exponentials fp32 (2^-21), the result half a step of its type."""
import numpy as np
import pytest

import juliavision_b200 as jv
from tests import decode_ref as ref
from tests.test_gpu_decode import F16, F32, STEP, ints, near

pytestmark = pytest.mark.gpu


class Packed:
    """Sequences side by side: news[b] rows over news[b] + past[b] keys (fewer keys than rows where past is negative), `spare` rows behind."""

    def __init__(self, ctx, rng, E, Hq, H, news, past, spare=2, layout="joined", scale=1.0):
        self.ctx, self.E, self.Hq, self.H = ctx, E, Hq, H
        self.news, self.keys = np.asarray(news), np.asarray(news) + np.asarray(past)
        self.starts, self.kstarts = (np.concatenate(([0], np.cumsum(n))) for n in (self.news, self.keys))
        N, Nk = int(self.starts[-1]) + spare, int(self.kstarts[-1]) + spare
        self.q, self.k, self.v = ((rng.standard_normal((n, h, E)) * scale).astype(F16) for n, h in ((N, Hq), (Nk, H), (Nk, H)))
        self.layout = layout

    def device(self):
        ctx, E = self.ctx, self.E
        if self.layout == "joined":         # keys and values side by side, token-major
            kv = ctx.toback(np.stack((self.k, self.v), 1))
            Nk = len(self.k)
            dk, dv = (jv.DeviceArray(ctx, kv.ptr + i * self.H * E * 2, F16, (E, Nk, self.H), (1, 2 * self.H * E, E), owner=kv) for i in range(2))
            return ctx.toback(self.q).permute((0, 2, 1)), dk, dv
        if self.layout == "heads":          # head-major
            return tuple(ctx.toback(np.ascontiguousarray(a.transpose(1, 0, 2))) for a in (self.q, self.k, self.v))
        out = []                            # rows of an odd pitch, off 16-byte boundaries
        for a in (self.q, self.k, self.v):
            wide = np.zeros(a.shape[:2] + (E + 1,), F16)
            wide[..., 1:] = a
            d = ctx.toback(wide)
            out.append(jv.DeviceArray(ctx, d.ptr + 2, F16, (E, a.shape[0], a.shape[1]), (1, (E + 1) * a.shape[1], E + 1), owner=d))
        return tuple(out)

    def run(self, dtype, causal, scale=None, same=False):
        ctx = self.ctx
        buf = ctx.allocate(dtype, self.E, self.Hq, len(self.q))
        ctx.fill_bytes(buf, 0xFF)
        out = buf.permute((0, 2, 1))
        ctx.ws.reset()
        jv.packedsdpa_(ctx, out, *self.device(), ints(ctx, self.starts), None if same else ints(ctx, self.kstarts), scale=scale, causal=causal)
        ctx.synchronize()
        return buf.to_host()

    def check(self, got, dtype, causal, scale=None):
        E = self.E
        scale = 1.0 / np.sqrt(E) if scale is None else scale
        for b, (n, m) in enumerate(zip(self.news, self.keys)):
            q0, k0 = self.starts[b], self.kstarts[b]
            q, k, v = self.q[q0:q0 + n].astype(np.float64), self.k[k0:k0 + m].astype(np.float64), self.v[k0:k0 + m].astype(np.float64)
            hidden = (np.arange(m) > np.arange(n)[:, None] + (m - n)) if causal else np.zeros((n, m), bool)
            with np.errstate(invalid="ignore"):
                o, a, reach = ref.attention(q, k, v, hidden, scale)
                most = np.max(np.abs(np.where(np.isfinite(v), v, 0)), initial=0)
                mine = got[q0:q0 + n].astype(np.float64)
                same = np.isinf(o) & (mine == o)
                near(np.where(same, 0, mine), np.where(same, 0, o), np.nan_to_num(STEP[dtype][0] * np.abs(o) + STEP[dtype][1] + a * (2.0 ** -11 + 2.0 ** -21 + 4 * E * 2.0 ** -24 * reach),
                                                      posinf=0) + m * 2.0 ** -32 * most)
        assert np.isnan(got[self.starts[-1]:].astype(np.float64)).all()      # rows that belong to nobody


CASES = [  # E, Hq, H, news, past
    (64, 1, 1, [1], [0]), (64, 20, 20, [77], [0]), (128, 4, 1, [1, 0, 2, 127, 128, 129, 130], [0] * 7), (128, 8, 2, [5, 300, 0, 33, 257], [0, 700, 50, 128, 1]),
    (80, 10, 2, [200, 63, 64], [0, 1000, 1]), (72, 7, 1, [100, 37], [0, 3]), (40, 6, 3, [256, 255, 1], [256, 1, 2000]), (128, 71, 1, [9, 40], [0, 0]),
    (96, 5, 5, [1] * 33, [0, 1, 126, 127, 128, 129, 200, 300, 1, 2, 3] * 3), (8, 3, 3, [150], [0]), (33, 4, 2, [70, 5], [0, 9]), (128, 130, 1, [3, 1], [4, 60]),
    (64, 12, 4, [100, 50, 0, 7], [-30, -50, 0, -6]), (128, 2, 1, [700], [0]), (1, 2, 1, [40], [0]), (128, 16, 16, [600, 1], [0, 4000])]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_packed(ctx, case, causal, dtype):
    E, Hq, H, news, past = case
    p = Packed(ctx, np.random.default_rng(1), E, Hq, H, news, past)
    p.check(p.run(dtype, causal), dtype, causal)


@pytest.mark.parametrize("layout", ["heads", "odd"])
@pytest.mark.parametrize("E", [64, 80, 128, 20])
def test_layouts(ctx, layout, E):
    p = Packed(ctx, np.random.default_rng(2), E, 6, 2, [130, 1, 40], [0, 5, 100], layout=layout)
    p.check(p.run(F16, True), F16, True)


@pytest.mark.parametrize("E", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_many_and_long(ctx, E, causal):
    """More pairs of tiles than SMs: the list of the work; and one long among many short, which is cut along its keys."""
    rng = np.random.default_rng(3)
    p = Packed(ctx, rng, E, 8, 4, rng.integers(0, 400, 60), np.zeros(60, int))
    p.check(p.run(F16, causal), F16, causal)
    p = Packed(ctx, rng, E, 4, 2, [3] + [1] * 20 + [50], [20000] + list(rng.integers(0, 100, 20)) + [5000])
    p.check(p.run(F32, causal), F32, causal)


def test_same_places_and_scales(ctx):
    p = Packed(ctx, np.random.default_rng(4), 64, 4, 2, [90, 200], [0, 0])
    for scale in (0.0, 1.0, 3.0):
        p.check(p.run(F32, True, scale, same=True), F32, True, scale)


@pytest.mark.parametrize("E", [64, 96])
def test_far_apart_scores(ctx, E):
    """Maxima that grow along the keys by more than the reference point lets pass."""
    p = Packed(ctx, np.random.default_rng(5), E, 4, 2, [300, 40], [100, 500])
    p.k *= np.linspace(0.1, 12, len(p.k))[:, None, None].astype(F16)
    for causal in (True, False):
        p.check(p.run(F32, causal), F32, causal)


@pytest.mark.parametrize("E", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_hidden_keys_may_hold_anything(ctx, E, causal):
    """Infinities and NaN in keys and values: rows that see them show it, no other row and no other sequence does."""
    rng = np.random.default_rng(6)
    p = Packed(ctx, rng, E, 4, 2, [140, 130, 5], [0, 200, 300])
    for b, at in ((0, 139), (0, 70), (1, 329), (1, 300), (2, 303)):
        p.v[p.kstarts[b] + at, b % 2, 3 + b] = (np.inf, -np.inf, np.nan)[(b + at) % 3]
    p.v[p.kstarts[-1]:] = np.nan
    p.k[p.kstarts[-1]:] = np.nan
    p.k[p.kstarts[1] + 325, 1] = np.nan
    p.v[p.kstarts[1] + 10, 0, 7] = np.inf        # of a block that all rows see
    p.v[p.kstarts[0] + 70, 0, 5], p.v[p.kstarts[0] + 75, 0, 5] = np.inf, -np.inf
    p.check(p.run(F32, causal), F32, causal)


def test_parts_that_meet_hold_anything(ctx):
    """The same where the keys are cut and joined."""
    p = Packed(ctx, np.random.default_rng(7), 128, 2, 1, [20], [30000])
    p.v[30010, 0, 9], p.v[30000, 0, 1], p.v[20, 0, 2] = np.nan, np.inf, -np.inf
    p.check(p.run(F32, True), F32, True)


def test_bad_starts_are_cut_and_reported(ctx):
    for bad in ([0, 50, 20, 60], [0, 30, 60, 1000], [-4, 30, 60, 60], [0, 60, 0, 60]):
        p = Packed(ctx, np.random.default_rng(8), 64, 2, 2, [20, 20, 20], [0, 0, 0], spare=0)
        p.starts = p.kstarts = np.array(bad)
        with pytest.raises(jv.B200Error) as e:
            p.run(F16, True)
        assert e.value.code == 4
        ctx.synchronize()


@pytest.mark.parametrize("E", [64, 128])
def test_calls_one_after_the_other(ctx, E):
    """The same bits from every call, however the loads of its tiles land: no answer depends on which block takes what, or when."""
    rng = np.random.default_rng(10)
    p = Packed(ctx, rng, E, 16, 4, rng.integers(1, 1500, 24), np.zeros(24, int))
    d, ds = p.device(), ints(ctx, p.starts)
    outs = [ctx.allocate(F16, E, 16, len(p.q)) for _ in range(6)]
    for turn in range(5):
        for o in outs:
            ctx.ws.reset()
            jv.packedsdpa_(ctx, o.permute((0, 2, 1)), *d, ds)
        ctx.synchronize()
        first = outs[0].to_host()[:p.starts[-1]]
        assert all(np.array_equal(first, o.to_host()[:p.starts[-1]]) for o in outs[1:])


def test_recorded(ctx):
    """One graph, lengths changed between replays; two graphs share the workspace."""
    rng = np.random.default_rng(9)
    p = Packed(ctx, rng, 128, 8, 2, [400, 700], [0, 3000], spare=0)
    d, ds, dk = p.device(), ints(ctx, p.starts), ints(ctx, p.kstarts)
    outs = [ctx.allocate(F16, 128, 8, len(p.q)) for _ in range(2)]
    views = [o.permute((0, 2, 1)) for o in outs]
    ctx.ws.reset()
    jv.packedsdpa_(ctx, views[0], *d, ds, dk)
    graphs = []
    for o in views:
        ctx.ws.reset()
        graphs.append(ctx.capture(lambda o=o: jv.packedsdpa_(ctx, o, *d, ds, dk)))
    for first in (400, 11, 1090):
        starts, kstarts = np.array([0, first, 1100], np.int32), np.array([0, 2 * first, 4100], np.int32)
        ctx.upload(ds, starts)
        ctx.upload(dk, kstarts)
        for o in outs:
            ctx.fill_bytes(o, 0xFF)
        for g in graphs:
            g.replay()
        ctx.synchronize()
        got = [o.to_host() for o in outs]
        ctx.ws.reset()
        jv.packedsdpa_(ctx, views[0], *d, ds, dk)
        ctx.synchronize()
        assert all(np.array_equal(g, outs[0].to_host()) for g in got)
        p.news, p.keys, p.starts, p.kstarts = np.diff(starts), np.diff(kstarts), starts, kstarts
        p.check(got[0], F16, True)


@pytest.mark.parametrize("E", [64, 128])
def test_more_sequences_than_a_block_lists_at_once(ctx, E):
    """Thousands of sequences, most of them short or empty: their places in memory of the device, pairs beyond those kept in registers."""
    rng = np.random.default_rng(11)
    news = rng.integers(0, 4, 2600)
    news[[5, 1023, 1024, 2599]] = 300, 200, 129, 257
    past = rng.integers(0, 20, 2600)
    past[700] = 9000
    p = Packed(ctx, rng, E, 2, 1, news, past)
    p.check(p.run(F16, True), F16, True)
    p = Packed(ctx, rng, E, 2, 1, [0] * 1500, [3] * 1500, spare=300)
    p.check(p.run(F16, True), F16, True)
    p = Packed(ctx, rng, E, 2, 2, [1] * 1500, rng.integers(0, 300, 1500))          # a token each, as a step of serving is
    p.check(p.run(F32, True), F32, True)


@pytest.mark.parametrize("N", [1, 3, 30000])
def test_no_keys_at_all(ctx, N):
    """Zeros for the rows that are a sequence's, whatever the queries hold."""
    q = ctx.toback(np.full((N, 3, 64), np.nan, F16))
    kv = jv.DeviceArray(ctx, q.ptr, F16, (64, 0, 1), owner=q)
    out = ctx.allocate(F16, 64, 3, N)
    ctx.fill_bytes(out, 0xFF)
    ctx.ws.reset()
    jv.packedsdpa_(ctx, out.permute((0, 2, 1)), q.permute((0, 2, 1)), kv, kv, ints(ctx, [0, N // 2, N - N // 3]), ints(ctx, [0, 0, 0]))
    ctx.synchronize()
    got = out.to_host()
    assert not got[:N - N // 3].any() and np.isnan(got[N - N // 3:]).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("way", ["heads", "odd", "backwards"])
def test_where_results_go(ctx, dtype, way):
    """Head-major, off 16-byte boundaries with something between the rows, and from the last row to the first."""
    E, Hq = 72, 6
    p = Packed(ctx, np.random.default_rng(12), E, Hq, 3, [140, 3, 70, 260], [0, 9, 50, 1])
    N, size = len(p.q), np.dtype(dtype).itemsize
    pitch = E + 3 if way == "odd" else E
    buf = ctx.allocate(dtype, pitch, Hq, N) if way != "heads" else ctx.allocate(dtype, pitch, N, Hq)
    ctx.fill_bytes(buf, 0xFF)
    at, strides = {"heads": (0, (1, E, N * E)), "odd": (1, (1, Hq * pitch, pitch)), "backwards": ((N - 1) * Hq * E, (1, -Hq * E, E))}[way]
    out = jv.DeviceArray(ctx, buf.ptr + at * size, dtype, (E, N, Hq), strides, owner=buf)
    ctx.ws.reset()
    jv.packedsdpa_(ctx, out, *p.device(), ints(ctx, p.starts), ints(ctx, p.kstarts))
    ctx.synchronize()
    got = buf.to_host()
    if way == "heads":
        got = got.transpose(1, 0, 2)
    if way == "odd":
        between = np.delete(got.ravel()[:N * Hq * pitch].reshape(N * Hq, pitch), range(1, E + 1), 1)
        assert np.isnan(between.astype(np.float64)).all()
        got = got[..., 1:E + 1]
    p.check(got[::-1] if way == "backwards" else got, dtype, True)


def test_heads_that_share_memory(ctx):
    """Keys and values broadcast over heads, queries over rows, rows from the last to the first: strides of 0 and below."""
    rng = np.random.default_rng(13)
    E, N, Hq, H = 64, 150, 4, 2
    p = Packed(ctx, rng, E, Hq, H, [90, 60], [0, 0], spare=0)
    p.k[:], p.v[:], p.q[:] = p.k[:, :1], p.v[:, :1], p.q[:1]
    dk, dv, dq = ctx.toback(np.ascontiguousarray(p.k[:, 0])), ctx.toback(np.ascontiguousarray(p.v[::-1, 0])), ctx.toback(p.q[0])
    k = jv.DeviceArray(ctx, dk.ptr, F16, (E, N, H), (1, E, 0), owner=dk)
    v = jv.DeviceArray(ctx, dv.ptr + (N - 1) * E * 2, F16, (E, N, H), (1, -E, 0), owner=dv)
    q = jv.DeviceArray(ctx, dq.ptr, F16, (E, N, Hq), (1, 0, E), owner=dq)
    out = ctx.allocate(F32, E, Hq, N)
    ctx.ws.reset()
    jv.packedsdpa_(ctx, out.permute((0, 2, 1)), q, k, v, ints(ctx, p.starts))
    ctx.synchronize()
    p.check(out.to_host(), F32, True)


def test_two_contexts_at_once(ctx):
    """Calls of two contexts, each with its own stream and workspace, under way at the same time."""
    other = jv.Ctx(0)
    rng = np.random.default_rng(14)
    made = [Packed(c, rng, E, 8, 2, rng.integers(1, 600, 12), [0] * 12) for c, E in ((ctx, 128), (other, 64))]
    held = [(p.device(), ints(p.ctx, p.starts), p.ctx.allocate(F16, p.E, 8, len(p.q))) for p in made]
    for p, (_, _, buf) in zip(made, held):
        p.ctx.fill_bytes(buf, 0xFF)
    for _ in range(8):
        for p, (d, ds, buf) in zip(made, held):
            p.ctx.ws.reset()
            jv.packedsdpa_(p.ctx, buf.permute((0, 2, 1)), *d, ds)
    for p, (_, _, buf) in zip(made, held):
        p.ctx.synchronize()
        p.check(buf.to_host(), F16, True)


@pytest.mark.parametrize("E", [64, 128])
@pytest.mark.parametrize("shape", ["left over", "few", "some long"])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_dealt_out(ctx, E, shape, causal):
    """Pairs that are alike and do not go round the SMs: whole ones first and the rest cut; fewer than SMs; long ones of unequal lengths among
    short ones.  The same bits every time."""
    rng = np.random.default_rng(15)
    news, past, Hq, H = {"left over": ([8] * 160, [1500] * 160, 1, 1), "few": ([130] * 3, [2600] * 3, 4, 2),
                         "some long": ([40, 3, 100, 256] + [20] * 60, [9000, 5000, 12000, 7000] + list(rng.integers(0, 200, 60)), 3, 3)}[shape]
    p = Packed(ctx, rng, E, Hq, H, news, past)
    first = p.run(F16, causal)
    p.check(first, F16, causal)
    for _ in range(3):
        assert np.array_equal(first[:p.starts[-1]], p.run(F16, causal)[:p.starts[-1]])


def test_offsets_past_32_bits(ctx):
    """The last rows of arrays of more than 2^32 bytes, queries and results; keys and values of them through a stride."""
    rng = np.random.default_rng(16)
    E, Hq, n, m = 128, 32, 150, 200
    N, Nk = (1 << 19) + 300, 70000
    p = Packed(ctx, rng, E, Hq, 1, [n], [m - n], spare=0)
    q, out = (ctx.allocate(F16, E, Hq, N) for _ in range(2))
    k = ctx.allocate(F16, 256 * E, Nk)
    last = lambda a, rows: jv.DeviceArray(ctx, a.ptr + 2 * Hq * E * (N - rows), F16, (E, Hq, rows), owner=a)  # noqa: E731
    ctx.upload(last(q, n), p.q)
    ctx.fill_bytes(last(out, n), 0xFF)
    at = lambda i, row: jv.DeviceArray(ctx, k.ptr + 2 * E * (256 * row + i), F16, (E,), owner=k)  # noqa: E731
    for row in range(m):
        for i, a in ((0, p.k), (255, p.v)):
            ctx.upload(at(i, Nk - m + row), np.ascontiguousarray(a[row, 0]))
    dk, dv = (jv.DeviceArray(ctx, k.ptr + 2 * E * i, F16, (E, Nk, 1), (1, 256 * E, E), owner=k) for i in (0, 255))
    ctx.ws.reset()
    jv.packedsdpa_(ctx, out.permute((0, 2, 1)), q.permute((0, 2, 1)), dk, dv, ints(ctx, [N - n, N]), ints(ctx, [Nk - m, Nk]))
    ctx.synchronize()
    p.check(last(out, n).to_host(), F16, True)
