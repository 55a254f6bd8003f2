"""The host side of a decoder's operators, without a GPU: refusals, plans, the rounding of weights, and the look-ups of the
cache on whatever its device arrays may hold."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import juliavision_b200 as jv
from juliavision_b200 import _lib, build
from tests import decode_ref as ref

F16, F32, I32 = np.float16, np.float32, np.int32


class FakeCtx:
    """Zeros where a context would be: a refusal reads none of it."""
    room = C.create_string_buffer(1 << 16)
    handle = C.addressof(room)

    def allocate(self, dtype, *dims):
        return arr(dtype, dims)

    def upload(self, a, host):
        self.last = host.copy()


def arr(dt, shape, strides=None, ptr=1 << 20):
    return jv.DeviceArray(FakeCtx, ptr, dt, shape, strides)


def refused(code, fn, *a, **kw):
    with pytest.raises(jv.B200Error) as e:
        fn(FakeCtx, *a, **kw)
    assert e.value.code == code, e.value


def test_rotary_refusals():
    plan = jv.rotaryplan(FakeCtx(), 64)
    x, n = arr(F16, (64, 3, 4, 2)), arr(I32, (2,))
    refused(16, jv.rotary_, plan, arr(F32, (64, 3, 4, 2)), x, lens=n)
    refused(16, jv.rotary_, plan, x, arr(F16, (64, 3, 4)), lens=n)
    refused(17, jv.rotary_, plan, arr(F16, (64, 4, 4, 2)), x, lens=n)
    refused(1, jv.rotary_, plan, x, x)
    refused(1, jv.rotary_, plan, x, x, positions=arr(I32, (3, 2)), lens=n)
    refused(16, jv.rotary_, plan, x, x, positions=arr(np.int64, (3, 2)))
    refused(16, jv.rotary_, plan, x, x, positions=arr(I32, (2, 3)))
    refused(16, jv.rotary_, plan, x, x, lens=arr(I32, (3,)))
    refused(16, jv.rotary_, plan, x, x, lens=n, news=arr(I32, (2,), (2,)))
    refused(18, jv.rotary_, plan, x, arr(F16, (64, 3, 4, 2), (2, 128, 384, 1536)), lens=n)
    refused(17, jv.rotary_, plan, arr(F16, (32, 3, 4, 2)), arr(F16, (32, 3, 4, 2)), lens=n)       # 64 of 32 elements
    for bad in (dict(rot=3), dict(rot=64, scaling=("log", 2.0)), dict(rot=64, scaling=("linear",)), dict(rot=64, scaling=("ntk", 0)),
                dict(rot=64, scaling=("parts", 2.0, 100, 5.0, 5.0)), dict(rot=64, base=-1.0), dict(rot=64, frequencies=[1.0]),
                dict(rot=2, frequencies=[math.inf])):
        with pytest.raises(jv.B200Error):
            jv.rotaryplan(FakeCtx(), **bad)


def test_rotary_plan():
    """Fixed-point frequencies hold fp64's to 2^-64 turns; the scalings' fastest and slowest pairs are where they should be."""
    ctx = FakeCtx()
    for scaling in (None, ("linear", 4.0), ("ntk", 4.0), ("parts", 32.0, 4096, 1.0, 32.0)):
        f, gain = jv.rotaryfrequencies(128, scaling=scaling)
        jv.rotaryplan(ctx, 128, scaling=scaling)
        # whole units of 2^-64 turns: off by less than one of them
        assert np.all(np.abs(ctx.last.astype(np.float64) * 2.0 ** -64 - f / (2 * math.pi)) <= 2.0 ** -64)
        plain = 10000.0 ** (-np.arange(64) / 64)
        fast, slow = {None: (1, 1), "linear": (4, 4), "ntk": (1, 4), "parts": (1, 32)}[scaling and scaling[0]]
        np.testing.assert_allclose((plain / f)[[0, -1]], (fast, slow), rtol=1e-12)
        assert gain == (0.1 * math.log(32) + 1 if scaling and scaling[0] == "parts" else 1)
    jv.rotaryplan(ctx, 4, frequencies=[2 * math.pi * 3.25, -2 * math.pi * 0.25])
    assert np.allclose(ctx.last.astype(np.float64), [2.0 ** 62, 3 * 2.0 ** 62], rtol=1e-14)


def cache(kind="int8", E=64, T=16, H=2, P=5, **kw):
    dt = np.int8 if kind == "int8" else np.uint8
    return jv.Cache8(kw.get("k", arr(dt, (E, T, H, P))), kw.get("v", arr(dt, (E, T, H, P))), arr(F32, (H, P)), arr(F32, (H, P)), kind)


def test_cache_refusals():
    for bad in (dict(kind="int4"), dict(k=arr(np.uint8, (64, 16, 2, 5))), dict(v=arr(np.int8, (64, 16, 2, 6)))):
        with pytest.raises((jv.B200Error, KeyError)):
            cache(**bad)
    with pytest.raises(jv.B200Error):
        jv.Cache8(arr(np.int8, (64, 16, 2, 5)), arr(np.int8, (64, 16, 2, 5)), arr(F32, (2, 4)), arr(F32, (2, 5)))
    c, n, t = cache(), arr(I32, (3,)), arr(I32, (4, 3))
    kv, q = arr(F16, (64, 1, 2, 3)), arr(F16, (64, 1, 6, 3))
    refused(16, jv.cacheappend_, c, arr(F32, (64, 1, 2, 3)), kv, t, n)
    refused(17, jv.cacheappend_, c, arr(F16, (64, 1, 3, 3)), kv, t, n)
    refused(17, jv.cacheappend_, c, arr(F16, (64, 2, 2, 3)), kv, t, n)
    refused(16, jv.cacheappend_, c, kv, kv, arr(np.int64, (4, 3)), n)
    refused(16, jv.cacheappend_, c, kv, kv, arr(I32, (4, 2)), n)
    refused(16, jv.cacheappend_, c, kv, kv, t, arr(I32, (2,)))
    refused(18, jv.cacheappend_, c, arr(F16, (64, 1, 2, 3), (2, 128, 128, 256)), kv, t, n)
    refused(1, jv.cacheread_, kv, c, "q", t, n)
    refused(16, jv.cacheread_, arr(np.int8, (64, 1, 2, 3)), c, "k", t, n)
    refused(17, jv.cachesdpa_, q, arr(F16, (64, 1, 5, 3)), c, t, n)
    refused(17, jv.cachesdpa_, arr(F16, (64, 2, 6, 3)), q, c, t, n)
    refused(16, jv.cachesdpa_, q, arr(F32, (64, 1, 6, 3)), c, t, n)
    refused(17, jv.cachesdpa_, arr(F16, (80, 1, 6, 3)), arr(F16, (80, 1, 6, 3)), c, t, n)
    call = lambda c: (jv.cacheread_, arr(F16, (c.k.shape[0], 1, c.k.shape[2], 3)), c, "k", t, n)  # noqa: E731
    for E, T in ((72, 16), (8, 16), (144, 16), (64, 8), (64, 48), (64, 256)):
        refused(17, *call(cache(E=E, T=T)))
    refused(18, *call(cache(k=arr(np.int8, (64, 16, 2, 5), ptr=(1 << 20) + 8))))
    refused(18, *call(cache(v=arr(np.int8, (64, 16, 2, 5), (1, 72, 72 * 16, 72 * 32)))))
    refused(17, jv.cacheread_, arr(F16, (64, 1, 2, 3)), c, "k", arr(I32, (0, 3)), n)
    L = _lib.lib()
    s = c._with(t, 3)
    assert L.b200_cache_attention(None, s, 1, 2, 3, _lib.Strided4(), _lib.Strided4(), 0, 1.0, 1, None, None) == 1
    s.kind = 7
    assert L.b200_cache_read(FakeCtx.handle, s, 0, 1, 3, None, None, _lib.Strided4(), 0) == 20


def test_linear4_refusals():
    q, s = arr(np.uint8, (40, 128)), arr(F16, (40, 2))
    refused(16, jv.pack4, arr(np.int8, (40, 128)), s)
    refused(17, jv.pack4, q, s, None, 48)
    refused(17, jv.pack4, arr(np.uint8, (40, 96)), s, None, 64)
    refused(16, jv.pack4, q, arr(F16, (40, 4)))
    refused(16, jv.pack4, q, s, arr(F16, (40, 2)))
    w = jv.Weight4(40, 128, 64, arr(np.uint8, (3 * 2 * 512,)), arr(np.uint8, (192,)), None)
    x, out = arr(F16, (128, 3)), arr(F16, (40, 3))
    refused(16, jv.matmul4_, out, w, arr(F32, (128, 3)))
    refused(17, jv.matmul4_, out, w, arr(F16, (64, 3)))
    refused(17, jv.matmul4_, arr(F16, (41, 3)), w, x)
    refused(18, jv.matmul4_, out, w, arr(F16, (128, 3), (3, 1)))
    refused(19, jv.matmul4_, out, w, x, arr(F16, (41,)))
    refused(1, jv.matmul4_, out, w, x, epi="swish")
    refused(20, jv.matmul4_, arr(np.int8, (40, 3)), w, x)
    n = [C.c_int64() for _ in range(3)]
    at = lambda: [C.byref(v) for v in n]  # noqa: E731
    assert _lib.lib().b200_q4_sizes(40, 160, 32, *at()) == 0 and [v.value for v in n] == [3 * 4 * 512, 5 * 4 * 32, 5 * 4 * 8]
    assert _lib.lib().b200_q4_sizes(40, 160, 64, *at()) == 17 and _lib.lib().b200_q4_sizes(0, 64, 64, *at()) == 17


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantise4(symmetric, group):
    """Every value within half a step of its weight (a whole one where the largest magnitude stands at 8, which there is no code
    for), scales rounded to fp16 once."""
    rng = np.random.default_rng(0)
    W = rng.standard_normal((256, 30)).astype(F16)
    W[:group, 3] = 0
    W[:, 5] = np.abs(W[:, 5]) + F16(1)
    q, s, z = jv.quantise4(W, group, symmetric)
    assert q.dtype == np.uint8 and q.max() <= 15 and s.dtype == F16 and (z is None) == symmetric
    err = np.abs(ref.weight4(q, s, z, group) - W.astype(np.float64))
    step = np.repeat(s.astype(np.float64), group, 0)
    assert np.all(err <= step * (1.01 if symmetric else 0.51 + 16 * 2.0 ** -11))
    assert np.mean(err > 0.51 * step) < 0.05
    for bad in (W[:-1], W[0]):
        with pytest.raises(jv.B200Error):
            jv.quantise4(bad, group)
    W[0, 0] = np.inf
    with pytest.raises(jv.B200Error):
        jv.quantise4(W, group)


def test_the_reference_rounds_to_8_bits_as_torch_does():
    import torch
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.uniform(-448, 448, 4000), 2.0 ** rng.uniform(-12, 8.8, 4000), (ref.E4M3[:126] + ref.E4M3[1:127]) / 2, [0.0, -0.0, 448.0]])
    got = ref.to8(x, "e4m3")
    want = torch.from_numpy(x).to(torch.float32)
    exact = want.double().numpy() == x
    want = want.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert exact[-129:].all() and np.array_equal(got[exact], want[exact]) and np.mean(got == want) > 0.999
    codes = np.arange(256, dtype=np.uint8)
    assert np.array_equal(ref.E4M3, torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)


PROGRAM = r'''
#include <stdio.h>
#include "cache8.cuh"
int main() {
    int status = 0, wrong = 0;
    int32_t table[12] = {0, 4, 5, -1, 2147483647, -2147483647 - 1, 3, 2, 1, 0, 6, 4};
    b200::CacheView c = {};
    c.table = table, c.table_ld = 6, c.P = 5, c.T = 16, c.logT = 4, c.width = 6, c.d_status = &status;
    for (int b = 0; b < 2; ++b)
        for (int i = 0; i < 6; ++i) {
            status = 0;
            const int64_t pg = c.page(b, i);
            const bool bad = table[b * 6 + i] < 0 || table[b * 6 + i] >= 5;
            wrong += pg != (bad ? -1 : table[b * 6 + i]) || status != (bad ? KST_CACHE_PAGE : 0);
        }
    int32_t n[7] = {0, 1, 96, 97, -1, 2147483647, -2147483647 - 1}, cut[7] = {0, 1, 96, 96, 0, 96, 0};
    for (int i = 0; i < 7; ++i) {
        status = 0;
        wrong += c.tokens(i, n) != cut[i] || status != (cut[i] == n[i] ? 0 : KST_CACHE_LENGTH);
        status = 0;
        wrong += c.fresh(i, n, 96) != cut[i] || status != (cut[i] == n[i] ? 0 : KST_CACHE_LENGTH);
        wrong += c.fresh(i, nullptr, 7) != 7;
    }
    printf("%d wrong\n", wrong);
    return wrong != 0;
}
'''


def test_lookups_stay_inside_the_cache(tmp_path):
    """The three look-ups that every kernel goes through, compiled for the host and given numbers that do not fit."""
    src = tmp_path / "lookups.cu"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "lookups")
    subprocess.run([build.NVCC, *build.FLAGS, "-I", build.CSRC, str(src), "-o", exe], check=True, capture_output=True)
    assert subprocess.run([exe], capture_output=True, text=True).stdout == "0 wrong\n"
