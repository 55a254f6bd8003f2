"""What attention of packed sequences keeps where its results are fp32: weights of more bits than one fp16 number has."""
import numpy as np
import pytest

import juliavision_b200 as jv
from tests import decode_ref as ref
from tests.test_gpu_decode import F32, STEP, ints, near
from tests.test_gpu_packed_attention import Packed

pytestmark = pytest.mark.gpu


def bound(p, got, causal, scale=None):
    """A weight's two halves are off by 2^-22 of it, the exponential unit by 2^-22, its argument (16 at most, where a weight is not 0) by half a step, 2^-21;
    fp16's least step is 2^-24 where the heaviest weight is 2^7 at least: 2^-31 of it a key.  A score's fp32 sum moves a weight and the row's sum, as in
    the other tests.  The second product adds 16 keys at a time in fp32, twice, off by a step 2^-23 of the sum of magnitudes each time; 32 weights
    of a block one after the other in fp32, then the blocks.  The quotient and the result half a step each."""
    E = p.E
    scale = 1.0 / np.sqrt(E) if scale is None else scale
    for b, (n, m) in enumerate(zip(p.news, p.keys)):
        q0, k0 = p.starts[b], p.kstarts[b]
        q, k, v = p.q[q0:q0 + n].astype(np.float64), p.k[k0:k0 + m].astype(np.float64), p.v[k0:k0 + m].astype(np.float64)
        hidden = (np.arange(m) > np.arange(n)[:, None] + (m - n)) if causal else np.zeros((n, m), bool)
        o, a, reach = ref.attention(q, k, v, hidden, scale)
        off = 2.0 ** -20 + 4 * E * 2.0 ** -24 * reach + m / 8 * 2.0 ** -23 + (34 + m / 128) * 2.0 ** -24
        near(got[q0:q0 + n], o, a * off + m * 2.0 ** -31 * np.max(np.abs(v), initial=0) + STEP[F32][0] * np.abs(o) + STEP[F32][1])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("E, Hq, H, news, past", [(64, 4, 2, [300, 1, 140], [0, 200, 70]), (128, 4, 1, [200, 3], [100, 400]), (80, 5, 1, [140], [0]),
                                                  (20, 2, 2, [40, 1], [300, 128]), (128, 16, 16, [200] * 14, [0] * 14), (64, 4, 1, [1] * 40, [129] * 40)])
def test_weights_keep_their_bits(ctx, E, Hq, H, news, past, causal):
    """A row's weights are all alike but the first key's, which is the heaviest where its score is above theirs: what one rounding to fp16 would take off is
    the same for all, up to 2^-11, and so off the result of values above 0."""
    rng = np.random.default_rng(31)
    p = Packed(ctx, rng, E, Hq, H, news, past)
    p.v[:] = np.abs(p.v) + np.float16(0.25)
    for at, end in zip(p.kstarts, p.kstarts[1:]):
        p.k[at + 1:end] = p.k[at:at + 1] * np.float16(0.5)
    bound(p, p.run(F32, causal, 0.5 / E), causal, 0.5 / E)


@pytest.mark.parametrize("E", [64, 128])
def test_parts_keep_their_bits(ctx, E):
    """Keys cut along a long sequence and joined."""
    p = Packed(ctx, np.random.default_rng(32), E, 4, 2, [20, 1], [6000, 3000])
    p.v[:] = np.abs(p.v)
    p.k[1:] = p.k[:1]
    p.k[1:] *= np.float16(0.75)
    bound(p, p.run(F32, True, 0.5 / E), True, 0.5 / E)


@pytest.mark.parametrize("E", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_values_that_are_not_finite(ctx, E, causal):
    """In blocks that every row sees: an infinity is no NaN where the lower half of its weight is 0 or below."""
    rng = np.random.default_rng(33)
    p = Packed(ctx, rng, E, 4, 2, [200, 140], [600, 700])
    for at, h, e, x in ((3, 0, 1, np.inf), (140, 0, 2, -np.inf), (150, 1, 3, np.nan), (299, 0, 1, np.inf), (310, 1, 1, -np.inf), (311, 1, 1, np.inf), (600, 0, 5, np.inf),
                        (801, 1, 0, np.inf), (1200, 0, 7, -np.inf)):
        p.v[at, h, e] = x
    p.check(p.run(F32, causal), F32, causal)
    p.k[:] = p.k[:1]              # equal weights: each a number of fp16
    p.check(p.run(F32, causal), F32, causal)


@pytest.mark.parametrize("E", [64, 128])
def test_calls_and_replays_one_after_the_other(ctx, E):
    """The same bits from every call, however the loads of its tiles land, and from two graphs that share the workspace."""
    rng = np.random.default_rng(34)
    p = Packed(ctx, rng, E, 8, 2, rng.integers(1, 1500, 24), np.zeros(24, int))
    d, ds = p.device(), ints(ctx, p.starts)
    outs = [ctx.allocate(F32, E, 8, len(p.q)) for _ in range(4)]

    def call(o):
        ctx.ws.reset()
        jv.packedsdpa_(ctx, o.permute((0, 2, 1)), *d, ds)
    for o in outs:
        call(o)
    graphs = [ctx.capture(lambda o=o: call(o)) for o in outs[:2]]
    ctx.synchronize()
    first = outs[3].to_host()[:p.starts[-1]]
    for turn in range(4):
        for o in outs:
            ctx.fill_bytes(o, 0xFF)
        for g in graphs:
            g.replay()
        for o in outs[2:]:
            call(o)
        ctx.synchronize()
        assert all(np.array_equal(first, o.to_host()[:p.starts[-1]]) for o in outs)
    bound(p, outs[0].to_host(), True)
