"""Beam search as a decoder runs it: prompts of different lengths side by side (projection, norms and positions, packed attention, cache),
handed to all beams, then step by step (projection, norms and positions, cache, attention over it, logits, choice, caches brought in line),
the first step as it comes, the others as replays of one recording.

Every operator is checked against fp64 on what it really read; the caches, bit for bit, against what the same rows and choices make of them in numpy."""
import math

import numpy as np
import pytest

import juliavision_b200 as jv
from tests import decode_ref as ref
from tests.test_gpu_beams import agree, choice
from tests.test_gpu_decode import F16, F32, STEP, ints, near
from tests.test_gpu_norm_rotary import normed, tolerance

pytestmark = pytest.mark.gpu
D, HQ, H, E, T, V, K, PROMPTS, LAYERS, STEPS, WIDTH = 256, 4, 2, 64, 16, 203, 3, [7, 31], 2, 5, 4
B, WIDE = len(PROMPTS), (HQ + 2 * H) * E


class Layer:
    def __init__(self, ctx, rng, kind):
        self.w, self.o = (ctx.toback((rng.standard_normal((D, m)) / 16).astype(F16)) for m in (WIDE, HQ * E))     # (m, D), HQ E = D
        self.norm = (0.5 + rng.random((2, E))).astype(F16)
        self.dnorm = ctx.toback(self.norm)
        self.cache = c = jv.cache8(ctx, E, T, H, B * K * WIDTH, kind)
        self.kind, self.host = kind, [a.to_host() for a in (c.k, c.kmax, c.v, c.vmax)]

    def append(self, k, v, table, lens, news):
        for i, new in enumerate((k, v)):
            ref.append(self.host[2 * i], self.host[2 * i + 1], self.kind, new, table, lens, news)

    def tokens(self, table, s, n):
        return [ref.tokens(self.host[2 * i], self.host[2 * i + 1], self.kind, table, s, n) for i in range(2)]

    def reorder(self, own, source, lens):
        for i, old in enumerate([a.copy() for a in self.host]):
            for s, (full, kept) in enumerate(zip(lens // T, lens % T)):
                if kept and i % 2:
                    self.host[i][own[s, full]] = old[own[source[s], full]]
                elif kept:
                    self.host[i][own[s, full], :, :kept] = old[own[source[s], full], :, :kept]

    def holds(self):
        c = self.cache
        for have, want in zip((c.k, c.kmax, c.v, c.vmax), self.host):
            assert np.array_equal(have.to_host(), want)


class Buffers:
    """What a layer makes of n tokens: projections, normed and turned queries and keys, attention."""

    def __init__(self, ctx, n):
        self.ctx, self.n = ctx, n
        self.qkv, self.qk, self.att, self.x = (ctx.allocate(F16, m, n) for m in (WIDE, (HQ + H) * E, HQ * E, D))

    def heads(self, a, at, h, L, row=None):
        """h heads from `at` on, of all sequences of L tokens, or of the one from `row` on: (E, L, h, sequences)."""
        d = a.shape[0]
        return jv.DeviceArray(self.ctx, a.ptr + 2 * (at * E + (row or 0) * d), F16, (E, L, h, self.n // L if row is None else 1), (1, d, E, d * L), owner=a)

    def host(self):
        return (a.to_host() for a in (self.qkv, self.qk, self.att))


def flat(a):
    return jv.DeviceArray(a.ctx, a.ptr, a.dtype, a.shape[:3], a.strides[:3], owner=a)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_beam_search(ctx, kind):
    rng = np.random.default_rng(31)
    layers = [Layer(ctx, rng, kind) for _ in range(LAYERS)]
    head = (rng.standard_normal((D, V)) / 8).astype(F16)
    dhead = ctx.toback(head)
    plan, f = jv.rotaryplan(ctx, E), jv.rotaryfrequencies(E)[0]
    S, N = B * K, sum(PROMPTS)
    own = rng.permutation(S * WIDTH).reshape(S, WIDTH)
    down, dtable, table = ints(ctx, own), ints(ctx, own), own.copy()
    caches = [y.cache for y in layers]

    def norms_hold(qkv, qk, layer, at):
        y = qkv.reshape(1, -1, HQ + 2 * H, E)[:, :, :HQ + H]
        each = layer.norm[(np.arange(HQ + H) >= HQ).astype(int)]
        z = normed(y, each, 1e-6)
        want = ref.rotary(z, np.asarray(at)[None], f, 1.0, False)
        near(qk.reshape(y.shape), want, tolerance(want, z, E, 1.0))

    # ------------------------------------------------ the prompts
    starts = np.concatenate(([0], np.cumsum(PROMPTS)))
    places = np.concatenate([np.arange(n) for n in PROMPTS])
    dstarts, dplaces = ints(ctx, starts), ints(ctx, places[None])
    bufs = [Buffers(ctx, N) for _ in layers]
    x = ctx.toback(rng.standard_normal((N, D)).astype(F16))
    for y, b in zip(layers, bufs):
        ctx.ws.reset()
        jv.matmul_(ctx, b.qkv, y.w, x)
        jv.normrotary_(ctx, plan, b.heads(b.qk, 0, HQ + H, N), b.heads(b.qkv, 0, HQ + H, N), y.dnorm, split=HQ, positions=dplaces)
        q, k, v = (flat(b.heads(*a, N)) for a in ((b.qk, 0, HQ), (b.qk, HQ, H), (b.qkv, HQ + H, H)))
        jv.packedsdpa_(ctx, flat(b.heads(b.att, 0, HQ, N)), q, k, v, dstarts)
        for i, n in enumerate(PROMPTS):        # the prompt is its first beam's
            column = jv.DeviceArray(ctx, dtable.ptr + 4 * WIDTH * K * i, np.int32, (WIDTH, 1), owner=dtable)
            jv.cacheappend_(ctx, y.cache, b.heads(b.qk, HQ, H, n, starts[i]), b.heads(b.qkv, HQ + H, H, n, starts[i]), column, ints(ctx, [n]), ints(ctx, [n]))
        jv.matmul_(ctx, b.x, y.o, b.att)
        jv.add_(ctx, b.x, b.x, x)
        x = b.x
    lens = np.repeat(np.array(PROMPTS), K)
    dlens = ints(ctx, lens)
    jv.cachereorder_(ctx, caches, dtable, down, ints(ctx, np.zeros((B, K))), dlens)        # and then all beams'
    ctx.synchronize()
    for y, b in zip(layers, bufs):
        qkv, qk, att = b.host()
        norms_hold(qkv, qk, y, places)
        qk, qkv, att = qk.reshape(N, HQ + H, E), qkv.reshape(N, -1, E), att.reshape(N, HQ, E)
        for i, n in enumerate(PROMPTS):
            r = slice(starts[i], starts[i + 1])
            kv = np.stack((qk[r, HQ:], qkv[r, HQ + H:]))
            y.append(*kv[:, None], table[[i * K]], [n], [n])
            o, a, reach = ref.attention(qk[r, :HQ].astype(np.float64), *kv.astype(np.float64), np.triu(np.ones((n, n), bool), 1), 1 / math.sqrt(E))
            most = np.abs(kv[1].astype(np.float64)).max()
            near(att[r], o, STEP[F16][0] * np.abs(o) + STEP[F16][1] + a * (2.0 ** -11 + 2.0 ** -21 + 4 * E * 2.0 ** -24 * reach) + n * 2.0 ** -32 * most)

    def reordered(source):
        """The beams' caches and table after they went on from `source`."""
        table[:] = np.where(np.arange(WIDTH) < (lens // T)[:, None], table[source], own)
        for y in layers:
            y.reorder(own, source, lens)
            y.holds()
        assert np.array_equal(dtable.to_host(), table)
    reordered(np.arange(S) // K * K)

    # ------------------------------------------------ the steps
    dx = ctx.allocate(F16, D, S)
    bufs = [Buffers(ctx, S) for _ in layers]
    logits, ended = ctx.allocate(F16, V, S), np.zeros((B, K), np.int32)
    scores = np.tile([0.0] + [-np.inf] * (K - 1), (B, 1)).astype(F32)             # all beams are the first one's so far
    dscores, dended, dnews = ctx.toback(scores), ints(ctx, ended), ints(ctx, np.ones(S))
    out = [ctx.allocate(t, K, B) for t in (F32, np.int32, np.int32)]
    table3 = rng.standard_normal((V, D)).astype(F16)                              # the embeddings

    def step():
        x = dx
        ctx.ws.reset()
        for y, b in zip(layers, bufs):
            jv.matmul_(ctx, b.qkv, y.w, x)
            jv.normrotary_(ctx, plan, b.heads(b.qk, 0, HQ + H, 1), b.heads(b.qkv, 0, HQ + H, 1), y.dnorm, split=HQ, lens=dlens, news=dnews)
            jv.cacheappend_(ctx, y.cache, b.heads(b.qk, HQ, H, 1), b.heads(b.qkv, HQ + H, H, 1), dtable, dlens, dnews)
            jv.cachesdpa_(ctx, b.heads(b.att, 0, HQ, 1), b.heads(b.qk, 0, HQ, 1), y.cache, dtable, dlens, dnews)
            jv.matmul_(ctx, b.x, y.o, b.att)
            jv.add_(ctx, b.x, b.x, x)
            x = b.x
        jv.matmul_(ctx, logits, dhead, x)
        jv.beamselect_(ctx, *out, logits, dscores, dended, pad=1)
        jv.cachereorder_(ctx, caches, dtable, down, out[1], dlens)
        ctx.copy(dscores, out[0])

    tokens, graph = np.zeros((B, K), int), None
    for turn in range(STEPS):
        lens = lens + 1
        ctx.upload(dlens, lens.astype(np.int32))
        ctx.upload(dx, (table3[tokens.ravel()] + 0.25 * rng.standard_normal((S, D))).astype(F16))
        ctx.upload(dended, ended)
        if turn == 0:
            step()
        else:
            graph = graph or ctx.capture(step)
            graph.replay()
        ctx.synchronize()
        best, parents, now = (a.to_host() for a in out)
        agree([best, parents, now], choice(logits.to_host().reshape(B, K, V), scores, K, ended, 1))
        source = (np.arange(B)[:, None] * K + parents).ravel()
        for y, b in zip(layers, bufs):
            qkv, qk, att = b.host()
            norms_hold(qkv, qk, y, lens - 1)
            qk, att = qk.reshape(S, 1, HQ + H, E), att.reshape(S, 1, HQ, E)
            y.append(qk[:, :, HQ:], qkv.reshape(S, 1, -1, E)[:, :, HQ + H:], table, lens, np.ones(S, int))
            for s, n in enumerate(lens):
                want, a, r = ref.attention(qk[s, :, :HQ].astype(np.float64), *y.tokens(table, s, n), np.zeros((1, n), bool), 1 / math.sqrt(E))
                near(att[s], want, a * (2.0 ** -11 + 2.0 ** -19 * (r + 1)) + 2.0 ** -11 * np.abs(want) + 2.0 ** -24)
        reordered(source)
        scores, tokens = best, now
        ended = np.take_along_axis(ended, parents, 1)
        if turn == 1:
            ended[0, 1] = 1
