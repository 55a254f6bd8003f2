"""Rotary positions, the 8-bit cache and 4-bit products in numpy fp64, from their formulas (torch order: the reverse of the
device arrays').  What holds tokens is (B, L, H, E); a cache is (P, H, T, E) with (P, H) maxima; a table (B, width)."""
import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def e4m3_values():
    """The numbers of the 256 codes; the two NaN codes are NaN."""
    c = np.arange(256)
    s, e, m = np.where(c >> 7, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0)) * s
    v[[0x7f, 0xff]] = np.nan
    return v


E4M3 = e4m3_values()


def number(q, kind):
    return q.astype(np.float64) if kind == "int8" else E4M3[q]


def to8(x, kind):
    """Nearest 8-bit value, ties to even; x within the range."""
    if kind == "int8":
        return np.rint(x).astype(np.int8)
    mag = np.abs(x)
    e = np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -20))), -6)
    e = np.where(mag >= 2.0 ** (e + 1), e + 1, np.where((mag < 2.0 ** e) & (e > -6), e - 1, e))
    steps = np.rint(mag / 2.0 ** (e - 3)).astype(np.int64)          # 8 .. 16 eighths of 2^e, fewer at the lowest exponent
    code = np.where(e == -6, steps, (e.astype(np.int64) + 7) * 8 + (steps - 8))
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def append(cache, top, kind, new, table, lens, news):
    """cache and top in place; new (B, L, H, E) fp16."""
    T = cache.shape[2]
    for b in range(len(lens)):
        at = np.arange(lens[b] - news[b], lens[b])
        rows = np.arange(news[b])[at >= 0]
        at = at[at >= 0]
        for blk in np.unique(at // T):
            pg, mine = table[b, blk], at // T == blk
            t, x = at[mine] % T, new[b, rows[mine]].astype(np.float64)           # (n, H, E)
            held = np.arange(T) < t[0]
            for h in range(cache.shape[1]):
                was = float(top[pg, h]) if held.any() else 0.0
                now = np.max(np.abs(x[:, h]), initial=was) if not np.isnan(was) else np.nan
                if not np.isfinite(now):
                    cache[pg, h, held], cache[pg, h, t], top[pg, h] = 0, 0, np.nan
                    continue
                if held.any() and now != was:
                    cache[pg, h, held] = to8(number(cache[pg, h, held], kind) * was / now, kind)
                cache[pg, h, t] = to8(x[:, h] * TOP[kind] / now, kind) if now else 0
                top[pg, h] = now


def tokens(cache, top, kind, table, b, n):
    """The first n tokens of sequence b: (n, H, E)."""
    T, at = cache.shape[2], np.arange(n)
    pg = table[b, at // T]
    return number(cache[pg, :, at % T], kind) * top[pg].astype(np.float64)[:, :, None] / TOP[kind]


def attention(q, k, v, hidden, scale):
    """One sequence: q (L, Hq, E), k and v (n, H, E), hidden (L, n).  The result, sum p |v|, and the largest sum |q| |k| scale."""
    G = q.shape[1] // k.shape[1]
    o, a, reach = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // G].T * scale
        s[hidden] = -np.inf
        with np.errstate(invalid="ignore"):
            p = np.exp(s - np.where(np.isfinite(s.max(1, initial=-np.inf)), s.max(1, initial=-np.inf), 0)[:, None])
        p[hidden] = 0
        p /= np.where(p.sum(1) == 0, 1, p.sum(1))[:, None]
        vh = v[:, h // G]
        for i in range(len(q)):                    # a hidden key's value, whatever it is, has no part
            seen = ~hidden[i]
            o[i, h], a[i, h] = p[i, seen] @ vh[seen], p[i, seen] @ np.abs(vh[seen])
        reach = max(reach, np.max(np.abs(q[:, h]) @ np.abs(np.nan_to_num(k[:, h // G])).T * abs(scale), initial=0.0))
    return o, a, reach


def rotary(x, at, f, gain, interleaved):
    """x (B, L, H, E), positions at (B, L); a row's positions as exact integers."""
    out = x.astype(np.float64)
    half = len(f)
    angle = at[:, :, None, None].astype(np.float64) * f
    i = np.arange(half)
    u, w = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = out[..., u], out[..., w]
    out[..., u], out[..., w] = gain * (a * np.cos(angle) - b * np.sin(angle)), gain * (b * np.cos(angle) + a * np.sin(angle))
    return out


def weight4(q, scales, zeros, group):
    """(K, M) from (K, M) values, (K / group, M) scales and zero points or None."""
    z = 8.0 if zeros is None else np.repeat(zeros.astype(np.float64), group, 0)
    return (q.astype(np.float64) - z) * np.repeat(scales.astype(np.float64), group, 0)
