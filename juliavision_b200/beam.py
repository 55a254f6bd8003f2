"""Beam search: the choice of the best continuations, and the beams' caches brought in line with it (new surface: the reference has no
decoder).

A step of a search of K beams: the model's logits, `beamselect_`, `cachereorder_` with the parents it gives, the next token.  Nothing is read
back between, so a step can be recorded; the host follows parents and tokens afterwards, or between replays where it marks beams as ended.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Union

import numpy as np

from . import _lib
from ._lib import B200Error, check
from .context import Ctx, DeviceArray, dtcode
from .kvcache import Cache8


def _dense(op: str, name: str, a: DeviceArray, dtype, shape) -> int:
    if a.dtype != dtype or a.shape != shape or not a.isdense():
        raise B200Error(16, f"{op}: {name} must be a dense {np.dtype(dtype)} {shape} array")
    return a.ptr


def beamselect_(ctx: Ctx, best: DeviceArray, parents: DeviceArray, tokens: DeviceArray, logits: DeviceArray, scores: DeviceArray,
                ended: Optional[DeviceArray] = None, pad: int = 0):
    """The N best of a search's K * V continuations scores[k] + log softmax(logits[:, k])[v], in order, ties to the lowest k V + v: their
    sums, beams and tokens as best (N, B) fp32, parents and tokens (N, B) int32.  logits (V, K, B) or (V, K * B), fp16 or fp32, V contiguous;
    scores (K, B) fp32.  A beam whose number in ended (K, B) int32 is not 0 has one continuation, the token `pad` at its own score.  A
    beam whose score is not finite, or whose logits have no finite log sum (a NaN, +inf, nothing but -inf), offers its tokens at -inf; they come last, lowest
    first.  At most 32 beams and 32 results, which lie apart from what is read."""
    rc = _lib.host().beamselect(ctx.handle, best, parents, tokens, logits, scores, ended, pad)
    if rc is not None:
        check(rc)
        return best, parents, tokens
    if logits.dtype not in (np.float16, np.float32) or logits.ndim not in (2, 3) or scores.ndim != 2 or best.ndim != 2:
        raise B200Error(16, "beamselect!: logits must be an fp16 or fp32 (V, K, B) or (V, K * B) array, scores (K, B), best (N, B)")
    (K, B), V, N = scores.shape, logits.shape[0], best.shape[0]
    if logits.shape[1:] != ((K, B) if logits.ndim == 3 else (K * B,)) or best.shape[1] != B:
        raise B200Error(17, f"beamselect!: logits are {logits.shape} for {B} searches of {K} beams, best {best.shape}")
    if V > 1 and logits.strides[0] != 1:
        raise B200Error(18, "beamselect!: logits are not contiguous along the vocabulary")
    ldk = logits.strides[1]
    ldb = logits.strides[2] if logits.ndim == 3 else K * ldk
    args = [_dense("beamselect!", "scores", scores, np.float32, (K, B)), None if ended is None else _dense("beamselect!", "ended", ended, np.int32, (K, B)),
            int(pad), _dense("beamselect!", "best", best, np.float32, (N, B)), _dense("beamselect!", "parents", parents, np.int32, (N, B)),
            _dense("beamselect!", "tokens", tokens, np.int32, (N, B))]
    check(_lib.lib().b200_beam_select(ctx.handle, V, K, B, N, logits.ptr, dtcode(logits.dtype), ldk, ldb, *args))
    return best, parents, tokens


def cachereorder_(ctx: Ctx, caches: Union[Cache8, Sequence[Cache8]], table: DeviceArray, own: DeviceArray, parents: DeviceArray,
                  lens: DeviceArray) -> DeviceArray:
    """Beam k of search b goes on from the tokens of beam parents[k, b] (parents (K, B) int32, as `beamselect_` gives them).  `caches`: one
    a layer, of the same sizes and strides, which share `table` (pages a sequence, K * B), sequence k + K b being beam k of search b.
    own (pages a sequence, K * B) names the pages that each beam writes, no page twice; a table starts as a copy of it and shares no memory with it.  Whole pages change
    hands in `table`; the page that is not full is copied to the beam's own, and entries behind it become the beam's own again.  lens (K * B): a
    search's beams are equally long.  No array is given twice.  A prompt is handed to all beams by parents of 0 after it has been written as beam 0's."""
    rc = _lib.host().cachereorder(ctx.handle, caches, table, own, parents, lens)
    if rc is not None:
        check(rc)
        return table
    caches = [caches] if isinstance(caches, Cache8) else list(caches)
    if parents.ndim != 2:
        raise B200Error(16, "cachereorder!: parents must be an int32 (K, B) array")
    K, B = parents.shape
    for name, a in (("table", table), ("own", own)):
        if a.dtype != np.int32 or a.ndim != 2 or a.shape[1] != K * B or (a.shape[0] != 1 and a.strides[0] != 1):
            raise B200Error(16, f"cachereorder!: {name} must be an int32 (pages a sequence, {K * B}) array, pages contiguous")
    if own.shape != table.shape:
        raise B200Error(17, f"cachereorder!: table is {table.shape}, own {own.shape}")
    ld = [a.strides[1] if K * B > 1 else max(a.shape[0], 1) for a in (table, own)]
    at = _dense("cachereorder!", "parents", parents, np.int32, (K, B))
    if lens.dtype != np.int32 or lens.size != K * B or not lens.isdense():
        raise B200Error(16, "cachereorder!: lens must be a dense int32 array of one number a beam")
    c = (_lib.Cache8 * len(caches))(*(x._c for x in caches))
    check(_lib.lib().b200_cache_reorder(ctx.handle, C.cast(c, C.POINTER(_lib.Cache8)), len(caches), K, B, table.ptr, ld[0], own.ptr, ld[1],
                                        table.shape[0], at, lens.ptr))
    return table
