"""Products with 4-bit weights (new surface beside matmul!, kernels/extern/matmul.jl:78-100): a scale, and perhaps a zero point, for
each group of inputs of an output, w[m, k] = scales[m, g] * (q[m, k] - zeros[m, g]), g = k // group.

`quantise4` rounds an fp16 weight on the host, once, when a model is loaded; `pack4` lays 4-bit values out on the device, from
there or from a checkpoint; `matmul4_` is `matmul_` with such a weight.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Tuple

import numpy as np

from . import _lib
from ._lib import B200Error, check
from .context import Ctx, DeviceArray, dtcode
from .matmul import _colmajor_2d


@dataclass(frozen=True)
class Weight4:
    """A weight (M, K) as the kernels read it (b200_q4 in include/b200dnn.h); `zeros` None stands for 8."""
    M: int
    K: int
    group: int
    data: DeviceArray
    scales: DeviceArray
    zeros: Optional[DeviceArray]

    def __post_init__(self):
        s = _lib.Q4()
        s.data, s.scales, s.zeros = self.data.ptr, self.scales.ptr, self.zeros.ptr if self.zeros is not None else None
        s.M, s.K, s.group = self.M, self.K, self.group
        object.__setattr__(self, "_c", s)


def quantise4(W: np.ndarray, group: int = 64, symmetric: bool = True) -> Tuple[np.ndarray, np.ndarray, Optional[np.ndarray]]:
    """4-bit values, scales and zero points of a weight given in torch order (K, M), as matmul_'s A is uploaded: q (K, M) uint8,
    scales (K / group, M) fp16, zeros (K / group, M) uint8 or None.  Symmetric: codes -8 to 7 and no zero points, every
    value within half a step: the largest at 7, or half a step past the end, whichever leaves the group less error (a relative 2-norm of
    0.088, 0.097 and 0.105 of normal values in groups of 32, 64 and 128).  Otherwise 15 steps from the group's least to its greatest value,
    zero among them.  Weights whose scales fp16 does not hold are refused."""
    if W.ndim != 2 or group not in (32, 64, 128) or W.shape[0] % group:
        raise B200Error(17, f"quantise4: a (K, M) weight of whole groups of {group} (32, 64 or 128)")
    w = W.astype(np.float64).reshape(W.shape[0] // group, group, W.shape[1])
    if not np.all(np.isfinite(w)):
        raise B200Error(1, "quantise4: the weight is not finite")
    lo, hi = np.maximum(-w.min(1), 0), np.maximum(w.max(1), 0)
    if np.max(np.maximum(hi / 7, lo / 8) if symmetric else (hi + lo) / 15, initial=0) >= 65520:      # rounds to infinity
        raise B200Error(1, "quantise4: weights whose scales fp16 does not hold")
    if symmetric:
        each = [np.maximum(hi / (7 + past), lo / (8 + past)).astype(np.float16) for past in (0.5, 0.0)]
        off = []
        for s in each:
            step = np.where(s == 0, 1, s).astype(np.float64)[:, None]
            off.append(np.square(np.clip(np.rint(w / step), -8, 7) * step - w).sum(1))
        s = np.where(off[0] <= off[1], *each)
        z = np.full(s.shape, 8.0)
    else:
        s = ((hi + lo) / 15).astype(np.float16)
        z = np.clip(np.rint(lo / np.where(s == 0, 1, s).astype(np.float64)), 0, 15)
    step = np.where(s == 0, 1, s).astype(np.float64)[:, None]
    q = np.clip(np.rint(w / step) + z[:, None], 0, 15)
    return q.astype(np.uint8).reshape(W.shape), s, None if symmetric else z.astype(np.uint8)


def pack4(ctx: Ctx, q: DeviceArray, scales: DeviceArray, zeros: Optional[DeviceArray] = None, group: int = 64) -> Weight4:
    """The layout of q (M, K) uint8 (0..15), scales (M, K / group) fp16 and zeros (M, K / group) uint8 (0..15) or None, all at any
    strides.  K is a multiple of `group` (32, 64 or 128)."""
    if q.ndim != 2 or q.dtype != np.uint8:
        raise B200Error(16, "pack4: q must be a uint8 (M, K) array")
    M, K = q.shape
    if group not in (32, 64, 128) or M < 1 or K < 1 or K % group:
        raise B200Error(17, f"pack4: {q.shape} in groups of {group} (32, 64 or 128)")
    for name, a, dt in (("scales", scales, np.float16), ("zeros", zeros, np.uint8)):
        if a is not None and (a.dtype != dt or a.shape != (M, K // group)):
            raise B200Error(16, f"pack4: {name} must be a {np.dtype(dt)} {(M, K // group)} array")
    n = [C.c_int64() for _ in range(3)]
    check(_lib.lib().b200_q4_sizes(M, K, group, *(C.byref(v) for v in n)))
    data, s = ctx.allocate(np.uint8, n[0].value), ctx.allocate(np.uint8, n[1].value)
    z = ctx.allocate(np.uint8, n[2].value) if zeros is not None else None
    w = Weight4(M, K, group, data, s, z)
    zs = zeros.strides if zeros is not None else (0, 0)
    check(_lib.lib().b200_q4_pack(ctx.handle, q.ptr, *q.strides, scales.ptr, *scales.strides, zeros.ptr if zeros is not None else None, *zs, w._c))
    return w


def matmul4_(ctx: Ctx, out: DeviceArray, W: Weight4, B: DeviceArray, bias: Optional[DeviceArray] = None,
             epi: str = "identity") -> DeviceArray:
    """out (M, N) = epi(T(bias + W B)): matmul_ with a 4-bit weight, B (K, N) and bias (M) fp16, out fp16 or fp32."""
    rc = _lib.host().matmul4(ctx.handle, out, W, B, bias, _lib.EPI.get(epi))
    if rc is not None:
        check(rc)
        return out
    if B.dtype != np.float16 or B.ndim != 2 or out.ndim != 2:
        raise B200Error(16, "matmul4!: B must be an fp16 (K, N) array, out (M, N)")
    if B.shape[0] != W.K or out.shape != (W.M, B.shape[1]):
        raise B200Error(17, f"matmul4!: W ({W.M}, {W.K}), B {B.shape}, out {out.shape}")
    ldb, ldo = _colmajor_2d(B), _colmajor_2d(out)
    if ldb is None or ldo is None:
        raise B200Error(18, "matmul4!: B and out must have contiguous columns")
    if bias is not None and (bias.dtype != np.float16 or bias.size != W.M or not bias.isdense()):
        raise B200Error(19, "matmul4!: bias must be a dense fp16 (M,) array")
    if epi not in _lib.EPI:
        raise B200Error(1, f"matmul4!: epilogue {epi}")
    check(_lib.lib().b200_matmul_q4(ctx.handle, W._c, B.shape[1], B.ptr, ldb, bias.ptr if bias is not None else None, out.ptr, ldo,
                                    dtcode(out.dtype), _lib.EPI[epi]))
    return out
