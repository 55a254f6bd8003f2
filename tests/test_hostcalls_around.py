"""The native host side of the entry points around a decoder's step (norm with rotation, attention of packed sequences, beams' choice,
reordered caches) against the Python one: the same arguments for the library, the same refusals.  No GPU: both call recorders."""
import ctypes as C
import itertools
import random

import numpy as np
import pytest

import juliavision_b200 as jv
from juliavision_b200 import _lib
from tests.test_hostcalls_decode import COUNTS, F16, F32, I32, FakeCtx, NoHost, arr, cache, plain, table

NAMES = ("b200_norm_rotary_f16", "b200_attention_packed_f16", "b200_beam_select", "b200_cache_reorder")


class Recorder:
    """Stands for the library.  Arrays behind a pointer (caches of a reordering) are noted by `length` elements."""
    def __init__(self, real):
        self.real, self.calls = real, []
        for n in NAMES:
            setattr(self, n, lambda *a, n=n: self.note(n, a))

    def note(self, n, a):
        a = list(a)
        if n == "b200_cache_reorder":
            at, count = a[1], a[2]
            a[1:3] = [count] + [plain(at[i]) for i in range(count)]
        self.calls.append((n,) + tuple(plain(v) for v in a))
        return 0

    def __getattr__(self, name):
        return getattr(self.real, name)


@pytest.fixture
def both(monkeypatch):
    rec = Recorder(_lib.lib())
    keep = [C.CFUNCTYPE(_lib.SIGNATURES[n][0], *_lib.SIGNATURES[n][1])(getattr(rec, n)) for n in NAMES]
    native = _lib.host()
    native.bindaround(*(C.cast(f, C.c_void_p).value for f in keep))
    monkeypatch.setattr(_lib, "_lib", rec)

    def run(fn, *args, **kw):
        """1 if the native side made the call, and the same one as the Python side; 0 if both left it or refused it alike."""
        seen = []
        for host in (native, NoHost()):
            monkeypatch.setattr(_lib, "_host", host)
            rec.calls.clear()
            try:
                fn(FakeCtx, *args, **kw)
                seen.append(list(rec.calls))
            except Exception as e:
                seen.append((type(e), getattr(e, "code", None)))
        assert seen[0] == seen[1], seen
        return int(isinstance(seen[0], list) and len(seen[0]) == 1)
    yield run
    monkeypatch.undo()
    _lib._host = None
    _lib.host()                       # bound to the library again


def test_normrotary(both):
    random.seed(11)
    taken = 0
    for (E, L, H, B), rot, inter in itertools.product(((64, 1, 8, 3), (80, 5, 2, 1), (20, 0, 2, 2)), (0, 20), (False, True)):
        plan = jv.RotaryPlan(rot, inter, 1.25, arr(np.uint64, (max(rot // 2, 1),)))
        x = arr(F16, (E, L, H, B), (1, 3 * H * E, E, 3 * H * E * L))
        weights = [(None, None), (arr(F32, (E,)), None), (arr(F16, (E, 1)), None), (arr(F16, (E, H)), None), (arr(F32, (E, H), (1, E + 4)), None),
                   (arr(F16, (E, 2)), 1), (arr(F16, (E, 2)), 0), (arr(F16, (E, 2)), H), (arr(F16, (E, 2)), H + 1), (arr(F16, (E, 2)), -1), (None, 1),
                   (arr(F16, (E, 3)), None), (arr(F16, (E + 1,)), None), (arr(I32, (E,)), None), (arr(F16, (E, 2), (2, 2 * E)), 1), (arr(F16, (E,)), 1),
                   (arr(F16, (E, 2)), 1 << 70), (arr(F16, (E, 2)), 1.0), (arr(F16, (E, 2, 1)), 1)]
        for (w, split), lens in itertools.product(weights, COUNTS(B)):
            taken += both(jv.normrotary_, plan, x, x, w, 1e-5, split, lens=lens, news=arr(I32, (B,)))
        for eps in (1, 0.0, np.float64(1e-6), np.float32(0.5)):
            taken += both(jv.normrotary_, plan, arr(F16, (E, L, H, B)), x, weights[1][0], eps, lens=arr(I32, (B,)))
    plan, x = jv.RotaryPlan(64, False, 1.0, arr(np.uint64, (32,))), arr(F16, (64, 2, 3, 1))
    for out in (arr(F16, (64, 2, 3, 2)), arr(F32, (64, 2, 3, 1)), arr(F16, (64, 2, 3))):
        assert not both(jv.normrotary_, plan, out, x, lens=arr(I32, (1,)))
    both(jv.normrotary_, plan, x, x, positions=arr(I32, (2, 1)))
    assert taken > 200


def test_packedsdpa(both):
    random.seed(12)
    taken = 0
    for (E, N, Hq, H, B), extra in itertools.product(((64, 12, 8, 2, 3), (80, 5, 20, 20, 1), (128, 0, 4, 4, 2), (16, 3, 0, 0, 1)), (0, 7)):
        Nk = N + extra
        q, kv = arr(F16, (E, N, Hq), (1, 3 * Hq * E, E)), arr(F16, (E, Nk, H), (1, H * E, E))
        starts = (arr(I32, (B + 1,)), arr(I32, (1, B + 1)), arr(I32, (B + 1,), (2,)), arr(F32, (B + 1,)), arr(I32, (0,)))
        for st, kst, dt in itertools.product(starts, (None, *starts, arr(I32, (B,))), (F16, F32, I32)):
            taken += both(jv.packedsdpa_, arr(dt, (E, N, Hq)), q, kv, kv, st, kst, random.choice((None, 0.5, 1, np.float64(0.1))),
                          random.choice((True, False, 0, None)))
        for bad in (arr(F16, (E, N + 1, Hq)), arr(F16, (E + 8, N, Hq)), arr(F16, (E, N, Hq, 1)), arr(F32, (E, N, Hq)), arr(F16, (E, N, Hq + 1))):
            both(jv.packedsdpa_, q, bad, kv, kv, starts[0], starts[0])
            both(jv.packedsdpa_, bad, q, kv, kv, starts[0], starts[0])
            both(jv.packedsdpa_, q, q, bad, kv, starts[0], starts[0])
            both(jv.packedsdpa_, q, q, kv, bad, starts[0], starts[0])
    assert taken > 40


def test_beamselect(both):
    random.seed(13)
    taken = 0
    for (K, B, V, N), dt, flat, pad in itertools.product(((1, 1, 7, 1), (5, 2, 100, 10), (3, 0, 9, 3), (4, 3, 8, 0)), (F16, F32, I32), (False, True), (0, 3)):
        x = arr(dt, (V, K * B) if flat else (V, K, B), (1, V + pad) if flat else (1, V + pad, K * (V + pad) + 5))
        good = [arr(F32, (N, B)), arr(I32, (N, B)), arr(I32, (N, B)), x, arr(F32, (K, B)), arr(I32, (K, B)), pad]
        taken += both(jv.beamselect_, *good)
        taken += both(jv.beamselect_, *good[:5])
        for at, bads in ((0, (arr(F16, (N, B)), arr(F32, (N, B + 1)), arr(F32, (N,)))), (1, (arr(I32, (N + 1, B)), arr(F32, (N, B)))), (2, (arr(I32, (N, B, 1)),)),
                         (3, (arr(dt, (V, K + 1, B)), arr(dt, (V,)), arr(dt, (V, K, B), (2, 2 * V, 2 * V * K)))), (4, (arr(F32, (K,)), arr(F16, (K, B)))),
                         (5, (arr(I32, (K, B + 1)), arr(F32, (K, B)))), (6, (1 << 70, True, np.int64(2)))):
            for bad in bads:
                both(jv.beamselect_, *(bad if i == at else v for i, v in enumerate(good)))
    assert taken > 20


def test_cachereorder(both):
    random.seed(14)
    taken = 0
    for (K, B, width), count in itertools.product(((1, 1, 3), (4, 2, 1), (3, 2, 5), (2, 0, 2)), (0, 1, 3)):
        caches = [cache(64, 16, 2, 9) for _ in range(count)]
        S = K * B
        for t, own in ((table(width, S), table(width, S)), (table(width, S, 8), table(width, S)), (table(width, S), table(width, S + 1)),
                       (arr(F32, (width, S)), table(width, S)), (arr(I32, (width, S), (2, 16)), table(width, S)), (table(width + 1, S), table(width, S))):
            for lens in COUNTS(S)[:2] + COUNTS(S)[3:]:
                taken += both(jv.cachereorder_, caches, t, own, arr(I32, (K, B)), lens)
            both(jv.cachereorder_, tuple(caches), t, own, arr(I32, (K, B)), arr(I32, (S,)))
            if count == 1:
                both(jv.cachereorder_, caches[0], t, own, arr(I32, (K, B)), arr(I32, (S,)))
        for parents in (arr(I32, (K * B,)), arr(F32, (K, B)), arr(I32, (K, B + 1)), arr(I32, (K, B), (2, 2 * K))):
            both(jv.cachereorder_, caches, table(width, S), table(width, S), parents, arr(I32, (S,)))
        assert not both(jv.cachereorder_, caches + [object()], table(width, S), table(width, S), arr(I32, (K, B)), arr(I32, (S,)))
    taken += both(jv.cachereorder_, [cache(64, 16, 2, 9) for _ in range(150)], table(2, 4), table(2, 4), arr(I32, (2, 2)), arr(I32, (4,)))
    assert taken > 30
