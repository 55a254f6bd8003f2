"""Norms of queries and keys with the rotation behind them, against fp64 (tests/decode_ref.py), at the sizes, strides and weights where
they can go wrong.

Tolerances count roundings: half a step of the fp16 result (2^-11 of the value, below 2^-14 2^-25), and fp32's before it: a sum of E squares
in chains of at most max(16, E / 32) and five steps over the lanes, half of whose relative error passes through the root, the root itself (2^-22),
four products, and the angle, sine and cosine as for rotary_."""
import numpy as np
import pytest

import juliavision_b200 as jv
from tests import decode_ref as ref
from tests.test_gpu_decode import F16, F32, STEP, ints, near, tokenmajor

pytestmark = pytest.mark.gpu


def normed(x, weight, eps):
    """x (B, L, H, E), weight (H, E), in fp64."""
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)


def tolerance(want, z, E, gain):
    relative = (max(16, E / 32) + 5) * 2.0 ** -25 + 2.0 ** -22 + 4 * 2.0 ** -24 + 2.0 ** -20
    return STEP[F16][0] * np.abs(want) + STEP[F16][1] + relative * 2 * max(gain, 1.0) * np.abs(z).max(-1, keepdims=True)


CASES = [  # B, L, H, split, E, rot, interleaved, far, weight, eps
    (1, 1, 1, None, 16, 16, False, 0, "all", 1e-6), (3, 1, 40, 32, 64, 64, False, 1500, "split", 1e-6), (2, 37, 5, None, 80, 80, True, 1000, "each", 1e-5),
    (2, 300, 8, 4, 128, 64, False, 100000, "split", 1e-6), (1, 65, 3, 0, 96, 48, True, 1 << 30, "split", 0.0), (4, 7, 2, 2, 20, 10, False, 50, "split", 1e-6),
    (2, 9, 3, None, 64, 0, True, 9, "each", 1e-6), (1, 700, 12, 8, 128, 128, False, 120000, "split", 1e-6), (5, 2, 33, 30, 128, 128, True, (1 << 31) - 10, "split", 1e-6),
    (1, 3, 4, None, 512, 256, False, 40, "none", 1e-6), (2, 2, 3, None, 1056, 1024, False, 40, "all", 1e-6), (3, 11, 1, None, 1, 0, False, 4, "all", 1e-3),
    (2, 5, 7, 3, 256, 256, True, 77, "split", 1e-6), (64, 1, 9, 5, 32, 16, False, 99, "split", 1e-6), (1, 2, 2, None, 4096, 0, False, 3, "each", 1e-6),
    (2, 3, 11, 7, 33, 32, True, 3, "split", 1e-6)]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [F16, F32], ids=["w16", "w32"])
@pytest.mark.parametrize("inplace", [False, True])
def test_norm_rotary(ctx, case, dtype, inplace):
    B, L, H, split, E, rot, inter, far, kind, eps = case
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((B, L, H, E)) * 10.0 ** rng.uniform(-2, 2, (B, L, H, 1))).astype(F16)
    if eps:
        x[0, 0, 0] = 0          # a head of zeros stays one
    news = rng.integers(0, L + 1, B)
    news[0] = L
    lens = news + rng.integers(0, far + 1, B)
    columns = {"all": 1, "split": 2, "each": H, "none": 1}[kind]
    w = (0.5 + rng.random((columns, E))).astype(dtype) if kind != "none" else np.ones((1, E))
    each = w[(np.arange(H) >= split).astype(int)] if kind == "split" else np.broadcast_to(w, (H, E))
    dw = None if kind == "none" else ctx.toback(w)
    if kind == "all" and inplace:
        dw = dw.reshape(E)
    plan = jv.rotaryplan(ctx, rot, interleaved=inter, scaling=("linear", 2.0) if rot else None, gain=1.25)
    d = tokenmajor(ctx, x)
    out = d
    if not inplace:
        buf = ctx.allocate(F16, E, H, L, B)
        ctx.fill_bytes(buf, 0xFF)
        out = buf.permute((0, 2, 1, 3))
    jv.normrotary_(ctx, plan, out, d, dw, eps=eps, split=split, lens=ints(ctx, lens), news=ints(ctx, news))
    ctx.synchronize()
    got = ctx.contiguous(out.permute((0, 2, 1, 3))).to_host()
    z = normed(x, each, eps)
    at = (lens - news)[:, None] + np.arange(L)
    want = ref.rotary(z, at, jv.rotaryfrequencies(rot, scaling=("linear", 2.0) if rot else None)[0], 1.25, inter)
    live = (np.arange(L) < news[:, None])[:, :, None, None] & np.ones(x.shape, bool)
    kept = x.astype(np.float64) if inplace else np.full(x.shape, np.nan)
    near(got, np.where(live, want, kept), np.where(live, tolerance(want, z, E, 1.25), 0))


@pytest.mark.parametrize("strides", ["odd", "even", "planar", "weight"])
def test_strides_and_positions(ctx, strides):
    """Rows, or a weight, off 16-byte boundaries take the element-wise form; positions of their own, broadcast over the batch."""
    B, L, H, E = 2, 13, 3, 32
    rng = np.random.default_rng(2)
    pitch = {"odd": E + 1, "even": E + 8}.get(strides, E)
    host = rng.standard_normal((B, H, L, pitch)).astype(F16)
    d = ctx.toback(host)
    view = jv.DeviceArray(ctx, d.ptr, F16, (E, L, H, B), (1, pitch, L * pitch, H * L * pitch), owner=d)
    wide = E + 1 if strides == "weight" else E
    w = rng.random((H, wide)).astype(F16)
    dw = ctx.toback(w)
    at = rng.integers(-1000, 1000, (1, L))
    out = ctx.allocate(F16, E, L, H, B)
    jv.normrotary_(ctx, jv.rotaryplan(ctx, 16, base=500.0), out, view, jv.DeviceArray(ctx, dw.ptr, F16, (E, H), (1, wide), owner=dw),
                   positions=ints(ctx, at))
    ctx.synchronize()
    z = normed(host[..., :E].transpose(0, 2, 1, 3), w[:, :E], 1e-6)
    want = ref.rotary(z, np.repeat(at, B, 0), jv.rotaryfrequencies(16, 500.0)[0], 1.0, False)
    near(out.to_host().transpose(0, 2, 1, 3), want, tolerance(want, z, E, 1.0))


def test_what_is_not_finite_stays_in_its_head(ctx):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((1, 4, 6, 64)).astype(F16)
    x[0, 1, 2, 5], x[0, 2, 3, 60], x[0, 3, 1, :] = np.inf, np.nan, 65504
    out = ctx.allocate(F16, 64, 4, 6, 1)
    jv.normrotary_(ctx, jv.rotaryplan(ctx, 0), out, tokenmajor(ctx, x), lens=ints(ctx, [4]))
    ctx.synchronize()
    with np.errstate(invalid="ignore"):
        want = normed(x, np.ones((6, 64)), 1e-6)     # a head with an infinity: zeros and a NaN; with a NaN: NaN
    near(out.to_host().transpose(0, 2, 1, 3), want, np.nan_to_num(tolerance(want, np.nan_to_num(want), 64, 1.0)))


def test_as_rotary_behind_a_norm(ctx):
    """Unit weights and heads of one size: what rotary_ gives of heads that are normed already, to the bit where the norm is exact."""
    rng = np.random.default_rng(4)
    x = np.where(rng.random((3, 20, 5, 128)) < 0.5, -1, 1).astype(F16)     # mean squares of 1: the norm divides by 1
    plan = jv.rotaryplan(ctx, 128)
    lens = ints(ctx, [20, 5000, 130000])
    a, b = ctx.allocate(F16, 128, 20, 5, 3), ctx.allocate(F16, 128, 20, 5, 3)
    jv.normrotary_(ctx, plan, a, tokenmajor(ctx, x), eps=0.0, lens=lens)
    jv.rotary_(ctx, plan, b, tokenmajor(ctx, x), lens=lens)
    ctx.synchronize()
    assert np.array_equal(a.to_host(), b.to_host())


def test_recorded(ctx):
    """One graph, lengths raised between replays."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((2, 1, 10, 64)).astype(F16)
    d, w, lens = tokenmajor(ctx, x), ctx.toback((0.5 + rng.random((2, 64))).astype(F16)), ints(ctx, [1, 9])
    plan, out = jv.rotaryplan(ctx, 64), ctx.allocate(F16, 64, 1, 10, 2)
    call = lambda: jv.normrotary_(ctx, plan, out, d, w, split=8, lens=lens)  # noqa: E731
    call()
    g = ctx.capture(call)
    for step in (2, 700):
        ctx.upload(lens, np.array([step, step + 8], np.int32))
        g.replay()
        ctx.synchronize()
        replayed = out.to_host()
        ctx.fill_bytes(out, 0xFF)
        call()
        ctx.synchronize()
        assert np.array_equal(replayed, out.to_host())


def test_offsets_past_32_bits(ctx):
    """Sequences that lie further than 2^32 bytes apart."""
    rng = np.random.default_rng(6)
    E, L, H, apart = 64, 5, 3, (1 << 31) + 64
    d = ctx.allocate(F16, apart + L * H * E)
    x = rng.standard_normal((2, L, H, E)).astype(F16)
    part = lambda b: jv.DeviceArray(ctx, d.ptr + 2 * apart * b, F16, (E, H, L), owner=d)  # noqa: E731
    for b in range(2):
        ctx.upload(part(b), x[b])
    view = jv.DeviceArray(ctx, d.ptr, F16, (E, L, H, 2), (1, H * E, E, apart), owner=d)
    jv.normrotary_(ctx, jv.rotaryplan(ctx, E), view, view, lens=ints(ctx, [L, 99]))
    ctx.synchronize()
    z = normed(x, np.ones((H, E)), 1e-6)
    want = ref.rotary(z, np.array([[0], [94]]) + np.arange(L), jv.rotaryfrequencies(E)[0], 1.0, False)
    near(np.stack([part(b).to_host() for b in range(2)]), want, tolerance(want, z, E, 1.0))
