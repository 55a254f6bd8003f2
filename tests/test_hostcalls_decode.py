"""The native host side of a decoder's entry points against the Python one: whatever it takes, it hands the library the very
arguments the Python route would; whatever the Python route refuses, it leaves alone.  No GPU: both call recorders."""
import copy
import ctypes as C
import itertools
import random

import numpy as np
import pytest

import juliavision_b200 as jv
from juliavision_b200 import _lib

NAMES = ("b200_rotary_f16", "b200_cache_append", "b200_cache_read", "b200_cache_attention", "b200_matmul_q4")
F16, F32, I32 = np.float16, np.float32, np.int32


class FakeCtx:
    handle = 4096


class NoHost:
    """The native module answering None to everything: the Python route runs."""
    def __getattr__(self, name):
        return lambda *a: None


def plain(v):
    if isinstance(v, C._Pointer):
        v = v.contents if v else None
    elif hasattr(v, "_obj"):
        v = v._obj
    if isinstance(v, C.Structure):
        return tuple(tuple(x) if isinstance(x, C.Array) else (x or 0) for x in (getattr(v, n) for n, *_ in v._fields_))
    return np.float32(v) if isinstance(v, float) else (v or 0)


class Recorder:
    """Stands for the library: the five entry points note their arguments, the rest is the library's own."""
    def __init__(self, real):
        self.real, self.calls = real, []
        for n in NAMES:
            setattr(self, n, lambda *a, n=n: self.calls.append((n,) + tuple(plain(v) for v in a)) or 0)

    def __getattr__(self, name):
        return getattr(self.real, name)


@pytest.fixture
def both(monkeypatch):
    rec = Recorder(_lib.lib())
    keep = [C.CFUNCTYPE(_lib.SIGNATURES[n][0], *_lib.SIGNATURES[n][1])(getattr(rec, n)) for n in NAMES]
    native = _lib.host()
    native.binddecode(*(C.cast(f, C.c_void_p).value for f in keep))
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


def arr(dt, shape, strides=None, ptr=None):
    return jv.DeviceArray(FakeCtx, ptr or random.randrange(1, 1 << 40) * 16, dt, shape, strides)


def cache(E, T, H, P, kind="int8"):
    dt = np.int8 if kind == "int8" else np.uint8
    return jv.Cache8(arr(dt, (E, T, H, P)), arr(dt, (E, T, H, P), (1, E + 16, T * (E + 16), 2 * H * T * (E + 16))), arr(F32, (H, P)), arr(F32, (H, P)), kind)


def table(width, B, ld=None):
    return arr(I32, (width, B), (1, ld or max(width, 1)))


COUNTS = lambda B: (arr(I32, (B,)), arr(I32, (1, B)), None, arr(F32, (B,)), arr(I32, (B + 1,)), arr(I32, (B,), (2,)))  # noqa: E731


def test_rotary(both):
    random.seed(1)
    taken = 0
    for (E, L, H, B), rot, inter, gain in itertools.product(((64, 1, 8, 3), (80, 5, 2, 1), (20, 0, 2, 2)), (0, 20), (False, True), (1.0, 1, np.float64(1.25))):
        plan = jv.RotaryPlan(rot, inter, gain, arr(np.uint64, (max(rot // 2, 1),)))
        x = arr(F16, (E, L, H, B), (1, 3 * H * E, E, 3 * H * E * L))
        for lens in COUNTS(B):
            taken += both(jv.rotary_, plan, x, x, lens=lens, news=arr(I32, (B,)))
            taken += both(jv.rotary_, plan, arr(F16, (E, L, H, B)), x, lens=arr(I32, (B,)), news=lens)
    plan, x = jv.RotaryPlan(64, False, 1.0, arr(np.uint64, (32,))), arr(F16, (64, 2, 3, 1))
    for out in (arr(F16, (64, 2, 3, 2)), arr(F32, (64, 2, 3, 1)), arr(F16, (64, 2, 3)), arr(I32, (64, 2, 3, 1))):
        assert not both(jv.rotary_, plan, out, x, lens=arr(I32, (1,)))
    assert not both(jv.rotary_, jv.RotaryPlan(64, False, 1.0, None), x, x, lens=arr(I32, (1,)))
    both(jv.rotary_, plan, x, x, positions=arr(I32, (2, 1)))
    assert taken > 60


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_cache(both, kind):
    random.seed(2)
    taken = [0, 0, 0]
    for (E, T, H, P), G, L, B, width in itertools.product(((64, 16, 2, 9), (128, 64, 8, 5)), (1, 4), (1, 7), (1, 3), (0, 1, 6)):
        c = cache(E, T, H, P, kind)
        for t, lens, dt in ((table(width, B), arr(I32, (B,)), F16), (table(width, B, 8), arr(I32, (B, 1)), F32), (table(width, B + 1), arr(I32, (B,)), F16),
                            (arr(F32, (width, B)), arr(I32, (B,)), F16), (arr(I32, (width, B), (2, 16)), arr(I32, (B,)), F16), (table(width, B), None, F16)):
            kv = arr(F16, (E, L, H, B), (1, H * E, E, H * E * L))
            for news in COUNTS(B):
                taken[0] += both(jv.cacheappend_, c, kv, arr(F16, (E, L, H, B)), t, lens, news)
                taken[1] += both(jv.cacheread_, arr(dt, (E, L, H, B)), c, random.choice("kv"), t, lens, news)
                q = arr(F16, (E, L, H * G, B))
                taken[2] += both(jv.cachesdpa_, arr(dt, q.shape), q, c, t, lens, news, random.choice((None, 0.5, -1.0, 1, np.float64(0.1))),
                                 random.choice((True, False, 0, 1, None)))
    c, t, n, q = cache(64, 16, 2, 9, kind), table(4, 1), arr(I32, (1,)), arr(F16, (64, 3, 4, 1))
    for bad in (arr(F16, (64, 3, 3, 1)), arr(F16, (80, 3, 4, 1)), arr(F32, (64, 3, 4, 1)), arr(F16, (64, 3, 4)), arr(F16, (64, 3, 4, 1), (2, 128, 384, 1536))):
        both(jv.cachesdpa_, q, bad, c, t, n)
        both(jv.cachesdpa_, bad, q, c, t, n)
        both(jv.cacheappend_, c, bad, q, t, n)
        both(jv.cacheread_, bad, c, "v", t, n)
    assert not both(jv.cachesdpa_, q, q, object(), t, n)
    assert min(taken) > 50


def test_matmul4(both):
    random.seed(3)
    taken = 0
    for M, K, N, group in itertools.product((1, 64, 1280), (64, 640), (0, 1, 17), (32, 64)):
        W = jv.Weight4(M, K, group, arr(np.uint8, (64,)), arr(np.uint8, (64,)), random.choice((None, arr(np.uint8, (64,)))))
        for dt, pad, bias, epi in ((F16, 0, None, "identity"), (F32, 5, (F16, M), "gelu"), (F16, 0, (F32, M), "relu"), (F16, 0, (F16, M + 1), "none"), (F16, 3, None, "tanh")):
            B, out = arr(F16, (K, N), (1, K + pad)), arr(dt, (M, N), (1, M + pad))
            taken += both(jv.matmul4_, out, W, B, arr(*bias[:1], (bias[1],)) if bias else None, epi)
        both(jv.matmul4_, arr(F16, (M, N + 1)), W, arr(F16, (K, N)))
        both(jv.matmul4_, arr(F16, (M, N)), W, arr(F16, (K + 1, N)))
        both(jv.matmul4_, arr(F16, (M, N)), W, arr(F32, (K, N)))
        both(jv.matmul4_, arr(F16, (M, N)), W, arr(F16, (K, N), (2, 2 * K)))
        both(jv.matmul4_, arr(I32, (M, N)), W, arr(F16, (K, N)))
    assert taken > 60


def test_what_a_copy_of_a_cache_or_weight_holds(both):
    """The structure is read where it is, so that a copy that outlives its original is as good."""
    c = copy.copy(cache(64, 16, 2, 9))
    q = arr(F16, (64, 1, 2, 1))
    assert both(jv.cachesdpa_, q, q, c, table(3, 1), arr(I32, (1,)))
    object.__setattr__(c, "_c", b"short")
    assert not _lib.host().cachesdpa(4096, q, q, c, table(3, 1), arr(I32, (1,)), None, 0.5, True)
