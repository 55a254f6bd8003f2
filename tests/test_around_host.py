"""Refusals of the operators around a decoder's step, without a GPU: norm with rotation, attention of packed sequences, beams' choice,
reordered caches.  The library's own come before it touches a device."""
import numpy as np

import juliavision_b200 as jv
from tests.test_decode_host import F16, F32, I32, FakeCtx, arr, cache, refused


def test_normrotary_refusals():
    plan = jv.rotaryplan(FakeCtx(), 64)
    x, n = arr(F16, (64, 3, 4, 2)), arr(I32, (2,))
    refused(16, jv.normrotary_, plan, arr(F32, (64, 3, 4, 2)), x, lens=n)
    refused(17, jv.normrotary_, plan, arr(F16, (64, 4, 4, 2)), x, lens=n)
    refused(1, jv.normrotary_, plan, x, x)
    refused(1, jv.normrotary_, plan, x, x, positions=arr(I32, (3, 2)), lens=n)
    refused(16, jv.normrotary_, plan, x, x, lens=arr(I32, (3,)))
    refused(18, jv.normrotary_, plan, x, arr(F16, (64, 3, 4, 2), (2, 128, 384, 1536)), lens=n)
    refused(17, jv.normrotary_, plan, arr(F16, (32, 3, 4, 2)), arr(F16, (32, 3, 4, 2)), lens=n)       # 64 of 32 elements
    refused(16, jv.normrotary_, plan, x, x, arr(I32, (64,)), lens=n)
    refused(16, jv.normrotary_, plan, x, x, arr(F16, (64, 2, 1)), lens=n)
    refused(17, jv.normrotary_, plan, x, x, arr(F16, (64, 2)), lens=n)                                # neither one nor four
    refused(17, jv.normrotary_, plan, x, x, arr(F16, (32,)), lens=n)
    refused(17, jv.normrotary_, plan, x, x, arr(F16, (64, 4)), split=2, lens=n)
    refused(18, jv.normrotary_, plan, x, x, arr(F16, (64, 4), (4, 1)), lens=n)
    refused(1, jv.normrotary_, plan, x, x, None, split=2, lens=n)
    for split in (-1, 5):
        refused(1, jv.normrotary_, plan, x, x, arr(F16, (64, 2)), split=split, lens=n)
    for eps in (-1e-6, float("inf"), float("nan")):
        refused(1, jv.normrotary_, plan, x, x, eps=eps, lens=n)
    wide = arr(F16, (4112, 1, 1, 2))
    refused(17, jv.normrotary_, jv.rotaryplan(FakeCtx(), 16), wide, wide, lens=n)


def test_packedsdpa_refusals():
    q, kv, st = arr(F16, (64, 9, 4)), arr(F16, (64, 9, 2)), arr(I32, (4,))
    refused(16, jv.packedsdpa_, q, arr(F32, (64, 9, 4)), kv, kv, st)
    refused(16, jv.packedsdpa_, arr(I32, (64, 9, 4)), q, kv, kv, st)
    refused(16, jv.packedsdpa_, q, arr(F16, (64, 9, 4, 1)), kv, kv, st)
    refused(17, jv.packedsdpa_, q, q, kv, arr(F16, (64, 8, 2)), st)
    refused(17, jv.packedsdpa_, q, q, arr(F16, (32, 9, 2)), arr(F16, (32, 9, 2)), st)
    refused(17, jv.packedsdpa_, q, q, arr(F16, (64, 9, 3)), arr(F16, (64, 9, 3)), st)
    refused(17, jv.packedsdpa_, q, q, arr(F16, (64, 9, 0)), arr(F16, (64, 9, 0)), st)
    refused(17, jv.packedsdpa_, arr(F16, (64, 8, 4)), q, kv, kv, st)
    refused(17, jv.packedsdpa_, q, q, arr(F16, (64, 8, 2)), arr(F16, (64, 8, 2)), st)                 # fewer keys, at the same places
    refused(16, jv.packedsdpa_, q, q, kv, kv, arr(I32, (0,)))
    refused(16, jv.packedsdpa_, q, q, kv, kv, arr(np.int64, (4,)))
    refused(16, jv.packedsdpa_, q, q, kv, kv, arr(I32, (4,), (2,)))
    refused(16, jv.packedsdpa_, q, q, kv, kv, st, arr(I32, (3,)))
    refused(18, jv.packedsdpa_, q, arr(F16, (64, 9, 4), (2, 512, 128)), kv, kv, st)
    refused(18, jv.packedsdpa_, arr(F16, (64, 9, 4), (2, 512, 128)), q, kv, kv, st)
    refused(21, jv.packedsdpa_, arr(F16, (136, 9, 4)), arr(F16, (136, 9, 4)), arr(F16, (136, 9, 2)), arr(F16, (136, 9, 2)), st)
    for scale in (-0.5, float("inf"), float("nan")):
        refused(1, jv.packedsdpa_, q, q, kv, kv, st, scale=scale)
    many = arr(F16, (8, 9, 65536))
    refused(17, jv.packedsdpa_, many, many, many, many, st)


def test_beamselect_refusals():
    best, at, x, scores = arr(F32, (6, 2)), arr(I32, (6, 2)), arr(F16, (50, 3, 2)), arr(F32, (3, 2))
    refused(16, jv.beamselect_, best, at, at, arr(I32, (50, 3, 2)), scores)
    refused(16, jv.beamselect_, best, at, at, arr(F16, (50,)), scores)
    refused(16, jv.beamselect_, best, at, at, x, arr(F32, (6,)))
    refused(16, jv.beamselect_, best, at, at, x, arr(F16, (3, 2)))
    refused(16, jv.beamselect_, arr(F32, (6, 2), (2, 12)), at, at, x, scores)
    refused(16, jv.beamselect_, best, arr(I32, (6, 3)), at, x, scores)
    refused(16, jv.beamselect_, best, at, arr(F32, (6, 2)), x, scores)
    refused(16, jv.beamselect_, best, at, at, x, scores, arr(I32, (2, 3)))
    refused(17, jv.beamselect_, best, at, at, arr(F16, (50, 2, 3)), scores)
    refused(17, jv.beamselect_, best, at, at, arr(F16, (50, 5)), scores)
    refused(17, jv.beamselect_, arr(F32, (6, 1)), at, at, x, scores)
    refused(18, jv.beamselect_, best, at, at, arr(F16, (50, 3, 2), (2, 100, 300)), scores)
    for pad in (-1, 50):
        refused(1, jv.beamselect_, best, at, at, x, scores, arr(I32, (3, 2)), pad)
    refused(17, jv.beamselect_, arr(F32, (33, 1)), arr(I32, (33, 1)), arr(I32, (33, 1)), arr(F16, (50, 3, 1)), arr(F32, (3, 1)))
    refused(17, jv.beamselect_, arr(F32, (4, 1)), arr(I32, (4, 1)), arr(I32, (4, 1)), arr(F16, (50, 33, 1)), arr(F32, (33, 1)))
    refused(17, jv.beamselect_, arr(F32, (7, 1)), arr(I32, (7, 1)), arr(I32, (7, 1)), arr(F16, (2, 3, 1)), arr(F32, (3, 1)))       # 7 of 6


def test_cachereorder_refusals():
    def made(at, E=64, P=5):
        return cache(E=E, P=P, k=arr(np.int8, (E, 16, 2, P), ptr=(2 * at) << 20), v=arr(np.int8, (E, 16, 2, P), ptr=(2 * at + 1) << 20))
    c, t, parents, lens = made(1), arr(I32, (3, 4)), arr(I32, (2, 2)), arr(I32, (4,))
    refused(16, jv.cachereorder_, c, t, t, arr(I32, (4,)), lens)
    refused(1, jv.cachereorder_, [], t, t, parents, lens)                  # without a cache nothing says how long a page is
    refused(16, jv.cachereorder_, c, t, t, arr(np.int64, (2, 2)), lens)
    refused(16, jv.cachereorder_, c, arr(I32, (3, 5)), t, parents, lens)
    refused(16, jv.cachereorder_, c, t, arr(F32, (3, 4)), parents, lens)
    refused(16, jv.cachereorder_, c, arr(I32, (3, 4), (2, 6)), t, parents, lens)
    refused(17, jv.cachereorder_, c, t, arr(I32, (2, 4)), parents, lens)
    refused(16, jv.cachereorder_, c, t, t, parents, arr(I32, (3,)))
    refused(16, jv.cachereorder_, c, t, t, parents, arr(I32, (4,), (2,)))
    refused(17, jv.cachereorder_, [c, made(2, E=128)], t, t, parents, lens)
    refused(17, jv.cachereorder_, [c, made(2, P=7)], t, t, parents, lens)
    refused(1, jv.cachereorder_, cache(), t, t, parents, lens)             # keys and values in one array
    refused(1, jv.cachereorder_, [c, made(2), c], t, t, parents, lens)
    many = arr(I32, (3, 33))
    refused(17, jv.cachereorder_, c, many, many, arr(I32, (33, 1)), arr(I32, (33,)))
