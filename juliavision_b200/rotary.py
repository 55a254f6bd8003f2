"""Rotary positions for the B200 backend (new surface: the reference has no decoder).

Pair i of a head is turned by position * f_i.  `rotaryplan` makes the frequencies once, in fp64, with the scalings that
stretch a model over a longer context than it was made for; `rotary_` applies them to (E, L, H, B) views, `normrotary_` behind
each head's norm in the same pass.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np

from . import _lib
from ._lib import B200Error, check
from .attention import _s4
from .context import Ctx, DeviceArray, dtcode


@dataclass(frozen=True)
class RotaryPlan:
    """Frequencies of rot / 2 pairs on the device, as fractions of a turn a position in units of 2^-64; which elements make a
    pair; what cosines and sines are multiplied by."""
    rot: int
    interleaved: bool
    gain: float
    freq: DeviceArray


def rotaryfrequencies(rot: int, base: float = 10000.0, scaling: Optional[Tuple] = None) -> Tuple[np.ndarray, float]:
    """Radians a position of each pair, fp64, and the gain.  f_i = base^(-2 i / rot), then by `scaling`:
    None                                  as they are
    ("linear", s)                         f / s: positions s times as close together
    ("ntk", s)                            base * s^(rot / (rot - 2)): the slowest pair s times slower, the fastest as it was
    ("parts", s, original, low, high)     f / s for pairs of fewer than `low` turns over `original` positions, f for more than
                                          `high`, between the two in proportion; the gain is 0.1 ln s + 1
    """
    if rot < 0 or rot % 2:
        raise B200Error(17, f"rotary: {rot} elements are not pairs")
    if not base > 0:
        raise B200Error(1, f"rotary: base {base}")
    kind = None if scaling is None else scaling[0]
    if kind not in (None, "linear", "ntk", "parts") or len(scaling or ()) != {None: 0, "linear": 2, "ntk": 2, "parts": 5}[kind]:
        raise B200Error(1, f"rotary: scaling {scaling}")
    if kind is not None and not scaling[1] > 0:
        raise B200Error(1, f"rotary: scaling by {scaling[1]}")
    if kind == "ntk" and rot > 2:
        base = base * float(scaling[1]) ** (rot / (rot - 2))
    f = np.float64(base) ** (-np.arange(0, rot, 2, dtype=np.float64) / max(rot, 1))
    if kind == "linear":
        f = f / float(scaling[1])
    if kind == "parts":
        s, original, low, high = (float(v) for v in scaling[1:])
        if not high > low:
            raise B200Error(1, f"rotary: scaling {scaling}")
        kept = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
        return f / s * (1 - kept) + f * kept, 0.1 * math.log(s) + 1.0
    return f, 1.0


def rotaryplan(ctx: Ctx, rot: int, base: float = 10000.0, interleaved: bool = False, scaling: Optional[Tuple] = None,
               gain: Optional[float] = None, frequencies: Optional[Sequence[float]] = None) -> RotaryPlan:
    """The plan of the first `rot` (at most 1024) elements of a head.  `frequencies` (rot / 2 radians a position) in the place of base and
    scaling; `gain` in the place of the scaling's own."""
    f, own = rotaryfrequencies(rot, base, scaling)
    if rot > 1024:
        raise B200Error(17, f"rotary: {rot} elements (at most 1024)")
    if frequencies is not None:
        f = np.asarray(frequencies, dtype=np.float64)
        if f.shape != (rot // 2,) or not np.all(np.isfinite(f)):
            raise B200Error(17, f"rotary: {rot // 2} finite frequencies")
    turns = f / (2 * math.pi)
    fixed = np.array([int(math.ldexp(t - math.floor(t), 64)) & (2 ** 64 - 1) for t in turns.tolist()], dtype=np.uint64)
    d = ctx.allocate(np.uint64, max(rot // 2, 1))
    if rot:
        ctx.upload(d, fixed)
    return RotaryPlan(rot, bool(interleaved), own if gain is None else float(gain), d)


def _counts(name: str, a: Optional[DeviceArray], B: int):
    """An int32 number for each sequence."""
    if a is None:
        return None
    if a.dtype != np.int32 or a.size != B or not a.isdense():
        raise B200Error(16, f"{name} must be a dense int32 array of one number a sequence")
    return a.ptr


def _positioned(op: str, out: DeviceArray, x: DeviceArray, positions, lens, news):
    """The checks of the calls that turn heads: (E, L, H, B), and the strides of `positions`."""
    if any(a.ndim != 4 or a.dtype != np.float16 for a in (x, out)):
        raise B200Error(16, f"{op}: x and out must be four-axis fp16 arrays")
    if x.shape != out.shape:
        raise B200Error(17, f"{op}: out is {out.shape}, x {x.shape}")
    E, L, H, B = x.shape
    pl = pb = 0
    if positions is not None:
        if lens is not None or news is not None:
            raise B200Error(1, f"{op}: positions as well as lens or news")
        if positions.dtype != np.int32 or positions.ndim != 2 or any(have not in (1, want) for have, want in zip(positions.shape, (L, B))):
            raise B200Error(16, f"{op}: positions must be an int32 (L, B) array")
        pl, pb = (0 if n == 1 else s for n, s in zip(positions.shape, positions.strides))
    elif lens is None:
        raise B200Error(1, f"{op}: neither positions nor lens")
    return (E, L, H, B), pl, pb


def rotary_(ctx: Ctx, plan: RotaryPlan, out: DeviceArray, x: DeviceArray, positions: Optional[DeviceArray] = None,
            lens: Optional[DeviceArray] = None, news: Optional[DeviceArray] = None) -> DeviceArray:
    """out = x turned by its positions; x and out (E, L, H, B) fp16, E contiguous, any other strides, out x itself or apart from it.
    Token l of sequence b is at positions[l, b] (int32, (L, B), either axis 1 to broadcast) or at lens[b] - news[b] + l, where
    rows from news[b] on (L without `news`) are left as they were.  Heads side by side in one projection take one call."""
    if positions is None:
        rc = _lib.host().rotary(ctx.handle, plan, out, x, lens, news)
        if rc is not None:
            check(rc)
            return out
    (E, L, H, B), pl, pb = _positioned("rotary!", out, x, positions, lens, news)
    xs, os_ = _s4(x), _s4(out)
    check(_lib.lib().b200_rotary_f16(ctx.handle, E, L, H, B, xs, os_, plan.freq.ptr, plan.rot, int(plan.interleaved), plan.gain,
                                     positions.ptr if positions is not None else None, pl, pb, _counts("lens", lens, B),
                                     _counts("news", news, B)))
    return out


def normrotary_(ctx: Ctx, plan: RotaryPlan, out: DeviceArray, x: DeviceArray, weight: Optional[DeviceArray] = None, eps: float = 1e-6,
                split: Optional[int] = None, positions: Optional[DeviceArray] = None, lens: Optional[DeviceArray] = None,
                news: Optional[DeviceArray] = None) -> DeviceArray:
    """Each head divided by the root of its mean square (and of eps), times `weight`, then turned as `rotary_` turns it, in one pass with
    one rounding.  `weight`, fp16 or fp32 with E contiguous: (E,) or (E, 1) for all heads, (E, H) a column a head, or with `split`
    (E, 2): heads before `split` take the first column, the others the second, as queries and keys side by side in one projection do.
    Everything else as for `rotary_`; a plan of 0 elements norms and turns nothing."""
    if positions is None:
        rc = _lib.host().normrotary(ctx.handle, plan, out, x, weight, eps, split, lens, news)
        if rc is not None:
            check(rc)
            return out
    (E, L, H, B), pl, pb = _positioned("normrotary!", out, x, positions, lens, news)
    ptr, code, ld, at = None, 0, 0, -1
    if split is not None and (weight is None or not 0 <= split <= H):
        raise B200Error(1, f"normrotary!: split at {split} of {H} heads, weight {None if weight is None else weight.shape}")
    if weight is not None:
        if weight.dtype not in (np.float16, np.float32) or weight.ndim not in (1, 2):
            raise B200Error(16, "normrotary!: weight must be an fp16 or fp32 (E,) or (E, heads) array")
        columns = 1 if weight.ndim == 1 else weight.shape[1]
        if weight.shape[0] != E or columns != (2 if split is not None else columns if columns == 1 else H):
            raise B200Error(17, f"normrotary!: weight is {weight.shape} for {H} heads of {E}" + ("" if split is None else f" split at {split}"))
        if E > 1 and weight.strides[0] != 1:
            raise B200Error(18, "normrotary!: weight is not contiguous along E")
        ptr, code, ld, at = weight.ptr, dtcode(weight.dtype), 0 if columns == 1 else weight.strides[1], -1 if split is None else int(split)
    xs, os_ = _s4(x), _s4(out)
    check(_lib.lib().b200_norm_rotary_f16(ctx.handle, E, L, H, B, xs, os_, ptr, code, ld, at, float(eps), plan.freq.ptr, plan.rot,
                                          int(plan.interleaved), plan.gain, positions.ptr if positions is not None else None, pl, pb,
                                          _counts("lens", lens, B), _counts("news", news, B)))
    return out
