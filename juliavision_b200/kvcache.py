"""Keys and values of earlier tokens held in 8 bits, in pages, and attention over them (new surface: the reference has no
decoder; its attention is sdpa, kernels/extern/attention.jl:712-834).

A page holds T tokens of every key head.  Its 8-bit values stand for q * max / 127 (int8) or q * max / 448 (e4m3) with one max
a (page, head).  A sequence's tokens lie in the pages its column of `table` names, in order, so pages can be handed out, shared
between sequences that begin alike, and copied (`ctx.copy` of a page's slice) without touching the others.
"""
from __future__ import annotations

from dataclasses import dataclass
from math import sqrt
from typing import Optional

import numpy as np

from . import _lib
from ._lib import B200Error, check
from .attention import _s4
from .context import Ctx, DeviceArray, dtcode
from .rotary import _counts

KINDS = {"int8": (_lib.I8, np.dtype(np.int8)), "e4m3": (_lib.E4M3, np.dtype(np.uint8))}


@dataclass(frozen=True)
class Cache8:
    """k and v (E, T, H, P) 8-bit arrays (int8, or uint8 that holds e4m3), kmax and vmax (H, P) fp32.  Pages may lie at any strides
    that are multiples of 16 bytes, keys and values in one allocation for instance."""
    k: DeviceArray
    v: DeviceArray
    kmax: DeviceArray
    vmax: DeviceArray
    kind: str = "int8"

    def __post_init__(self):
        if self.kind not in KINDS:
            raise B200Error(20, f"cache: kind {self.kind} (int8 or e4m3)")
        if any(a.ndim != 4 or a.dtype != KINDS[self.kind][1] for a in (self.k, self.v)):
            raise B200Error(16, f"cache: k and v must be four-axis {KINDS[self.kind][1]} arrays")
        E, T, H, P = self.k.shape
        if self.v.shape != self.k.shape:
            raise B200Error(17, f"cache: k is {self.k.shape}, v {self.v.shape}")
        for m in (self.kmax, self.vmax):
            if m.dtype != np.float32 or m.shape != (H, P) or not m.isdense():
                raise B200Error(16, "cache: kmax and vmax must be dense fp32 (heads, pages) arrays")
        s = _lib.Cache8()
        s.k, s.v, s.kmax, s.vmax = self.k.ptr, self.v.ptr, self.kmax.ptr, self.vmax.ptr
        for i in range(4):
            s.kstride[i], s.vstride[i] = self.k.strides[i], self.v.strides[i]
        s.E, s.T, s.H, s.P = E, T, H, P
        s.kind = KINDS[self.kind][0]
        object.__setattr__(self, "_c", s)

    def _with(self, table: DeviceArray, B: int):
        if table.dtype != np.int32 or table.ndim != 2 or table.shape[1] != B or (table.shape[0] != 1 and table.strides[0] != 1):
            raise B200Error(16, "cache: table must be an int32 (pages a sequence, sequences) array, pages contiguous")
        s = _lib.Cache8.from_buffer_copy(self._c)
        s.table, s.width = table.ptr, table.shape[0]
        s.table_ld = table.strides[1] if B > 1 else max(table.shape[0], 1)
        return s


def cache8(ctx: Ctx, E: int, T: int, H: int, P: int, kind: str = "int8") -> Cache8:
    """An empty cache of P pages of T tokens for H heads of E elements, from the pool."""
    if kind not in KINDS:
        raise B200Error(20, f"cache: kind {kind} (int8 or e4m3)")
    k, v = (ctx.allocate(KINDS[kind][1], E, T, H, P) for _ in range(2))
    km, vm = (ctx.allocate(np.float32, H, P) for _ in range(2))
    for a in (k, v, km, vm):
        ctx.fill_bytes(a, 0)
    return Cache8(k, v, km, vm, kind)


def _rows(op: str, a: DeviceArray, E: int, H: int, dtypes=(np.float16,)):
    if a.ndim != 4 or a.dtype not in dtypes:
        raise B200Error(16, f"{op}: a four-axis array of another type is expected")
    if a.shape[0] != E or a.shape[2] != H:
        raise B200Error(17, f"{op}: {a.shape} against heads of {E} elements, {H} of them")
    return _s4(a)


def cacheappend_(ctx: Ctx, cache: Cache8, k: DeviceArray, v: DeviceArray, table: DeviceArray, lens: DeviceArray,
                 news: Optional[DeviceArray] = None) -> Cache8:
    """Write new tokens: k and v (E, L, H, B) fp16, E contiguous; row i of sequence b is its token lens[b] - news[b] + i (lens
    with the new tokens in it), rows from news[b] on (L without `news`) are not tokens.  A page that is written belongs to one
    sequence, and to one place of its table."""
    rc = _lib.host().cacheappend(ctx.handle, cache, k, v, table, lens, news)
    if rc is not None:
        check(rc)
        return cache
    E, T, H, P = cache.k.shape
    ks, vs = _rows("cacheappend!", k, E, H), _rows("cacheappend!", v, E, H)
    if k.shape != v.shape:
        raise B200Error(17, f"cacheappend!: k is {k.shape}, v {v.shape}")
    L, B = k.shape[1], k.shape[3]
    check(_lib.lib().b200_cache_append(ctx.handle, cache._with(table, B), L, B, ks, vs, _counts("lens", lens, B), _counts("news", news, B)))
    return cache


def cacheread_(ctx: Ctx, out: DeviceArray, cache: Cache8, which: str, table: DeviceArray, lens: DeviceArray,
               starts: Optional[DeviceArray] = None) -> DeviceArray:
    """out (E, L, H, B), fp16 or fp32, = the keys ("k") or values ("v") of tokens starts[b] + row (row without `starts`); rows at or
    past lens[b] are left as they were."""
    if which not in ("k", "v"):
        raise B200Error(1, f"cacheread!: {which!r} is neither 'k' nor 'v'")
    rc = _lib.host().cacheread(ctx.handle, out, cache, which == "v", table, lens, starts)
    if rc is not None:
        check(rc)
        return out
    E, T, H, P = cache.k.shape
    os_ = _rows("cacheread!", out, E, H, (np.float16, np.float32))
    L, B = out.shape[1], out.shape[3]
    check(_lib.lib().b200_cache_read(ctx.handle, cache._with(table, B), int(which == "v"), L, B, _counts("starts", starts, B),
                                     _counts("lens", lens, B), os_, dtcode(out.dtype)))
    return out


def cachesdpa_(ctx: Ctx, out: DeviceArray, q: DeviceArray, cache: Cache8, table: DeviceArray, lens: DeviceArray,
               news: Optional[DeviceArray] = None, scale: Optional[float] = None, causal: bool = True) -> DeviceArray:
    """out = softmax(scale * Q K') V over the cache.  q and out (E, L, Hq, B), q fp16, out fp16 or fp32, E contiguous; Hq is a
    multiple of the cache's heads, query head i reads key head i // (Hq // H).  Row i of sequence b is its token
    lens[b] - news[b] + i and sees, when causal, the tokens up to itself, else all lens[b]; a row that sees none comes out as
    zeros, rows from news[b] on (L without `news`) are left as they were.  `out` does not overlap `q`."""
    if scale is None and q.ndim == 4 and q.shape[0] > 0:
        scale = 1.0 / sqrt(q.shape[0])
    rc = _lib.host().cachesdpa(ctx.handle, out, q, cache, table, lens, news, scale, causal)
    if rc is not None:
        check(rc)
        return out
    E, T, H, P = cache.k.shape
    if q.ndim != 4 or q.shape[2] % H:
        raise B200Error(17, f"cachesdpa!: q is {q.shape} over {H} key heads")
    if out.shape != q.shape:
        raise B200Error(17, f"cachesdpa!: out is {out.shape}, q {q.shape}")
    Hq, L, B = q.shape[2], q.shape[1], q.shape[3]
    qs, os_ = _rows("cachesdpa!", q, E, Hq), _rows("cachesdpa!", out, E, Hq, (np.float16, np.float32))
    check(_lib.lib().b200_cache_attention(ctx.handle, cache._with(table, B), L, Hq, B, qs, os_, dtcode(out.dtype),
                                          1.0 / sqrt(E) if scale is None else float(scale), int(bool(causal)), _counts("lens", lens, B),
                                          _counts("news", news, B)))
    return out
