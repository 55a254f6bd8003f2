"""What a decoder's operators keep where fewer bits would go unnoticed beside a rounding to fp16: fp32 results, against fp64."""
import math

import numpy as np
import pytest

from tests import decode_ref as ref
from tests.test_gpu_decode import F32, Cached, STEP, attend, near

pytestmark = pytest.mark.gpu


def bound(c, q, scale, causal, got):
    """The wanted results and how far off they may be.  Weights in two fp16 halves: 2^-21 of themselves (2^-10 left by the upper half
    where it is cut off, 2^-11 of that by the lower), and fp16's least step, 2^-24, a key, of weights that are 2^6 at least where the row's largest
    product of a weight and its page's scale is.  A score's fp32 sum, off by 2^-20 of the sum of magnitudes at most, moves a weight
    and the row's sum; exponential, sum and quotient 2^-19 together; the result's own rounding."""
    want, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    L = q.shape[1]
    for b, n in enumerate(c.lens):
        k, v = (ref.tokens(a, t, c.kind, c.table, b, n) for a, t in ((c.k, c.kmax), (c.v, c.vmax)))
        hidden = (np.arange(n) > np.arange(n - L, n)[:, None]) if causal else np.zeros((L, n), bool)
        o, a, reach = ref.attention(q[b].astype(np.float64), k, v, hidden, scale)
        want[b] = o
        tol[b] = a * (2.0 ** -21 + 2 * 2.0 ** -20 * reach + 2.0 ** -19) + n * 2.0 ** -30 * np.abs(v).max(initial=0) + STEP[F32][0] * np.abs(o)
    near(got, want, tol)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("E, G, L", [(128, 4, 1), (128, 4, 8), (128, 3, 11), (128, 4, 75), (64, 5, 1), (64, 5, 8), (64, 41, 1), (64, 1, 300)])
def test_weights_keep_their_bits(ctx, E, G, L, kind):
    """Few query rows a key head and many, on both sides of where one kernel takes over from the other: rows of nearly equal weights."""
    rng = np.random.default_rng(21)
    c = Cached(ctx, rng, E, 32, 2, [500, 317], kind)
    q = rng.standard_normal((2, L, 2 * G, E)).astype(np.float16)
    scale = 0.6 / E
    got, _, _ = attend(ctx, c, q, None, scale, True, F32)
    bound(c, q, scale, True, got)
