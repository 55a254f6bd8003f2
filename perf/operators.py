"""One-token decoding from an 8-bit cache, as cases that can be timed and compared: rotary positions, writing tokens into
a paged cache of 8-bit values with a scale for each block of tokens and head, attention over that cache, and products with
4-bit weights and group scales.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what a program holds before a call,
`run()` is one call.  With `own` false `run()` computes the formulas with elementary tensor operations in fp32 (angles in
fp64); with `own` true it makes the package's calls.  Tensors are in torch order, the reverse of the package's.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # Query and key heads side by side in one projection, one token of eight sequences: the smallest call of a step.
        dict(name="rotary_step_8x40x64", kind="rotary", batch=8, new=1, heads=40, head_dim=64, rot=64, interleaved=False,
             scaling="none", far=1500),
        # The same for two whole prompts, positions past the length that the frequencies were made for.
        dict(name="rotary_prompt_2x8192x40x128", kind="rotary", batch=2, new=8192, heads=40, head_dim=128, rot=128, interleaved=False,
             scaling="parts", far=120000),
        # One token of 64 sequences written into blocks of 16 that are partly full; the blocks it touched read back.
        dict(name="append_step_64x8x128", kind="append", batch=64, new=1, heads=8, head_dim=128, block=16, bits="int8", past=4000),
        # Four ragged prompts written into an empty cache, all of it read back.
        dict(name="append_prompt_4x4096x8x128", kind="append", batch=4, new=4096, heads=8, head_dim=128, block=64, bits="int8", past=0),
        # A decoder's query over an encoder's 1500 tokens held in 8 bits: every key is visible, latency counts.
        dict(name="attend_cross_1x1500_h20", kind="attend", batch=1, new=1, heads=20, kv_heads=20, head_dim=64, block=64, bits="int8",
             length=1500, ragged=False, causal=False),
        # One token of 32 sequences of 1000 to 8192 tokens, four query heads to a key head.
        dict(name="attend_step_32x8192_h32", kind="attend", batch=32, new=1, heads=32, kv_heads=8, head_dim=128, block=64, bits="int8",
             length=8192, ragged=True, causal=True),
        # One token over one very long sequence, 8-bit floating-point values.
        dict(name="attend_step_1x131071_h32", kind="attend", batch=1, new=1, heads=32, kv_heads=8, head_dim=128, block=128, bits="e4m3",
             length=131071, ragged=False, causal=True),
        # Five tokens at once (a draft being checked), five query heads to a key head.
        dict(name="attend_draft_8x5x4096_h20", kind="attend", batch=8, new=5, heads=20, kv_heads=4, head_dim=64, block=32, bits="int8",
             length=4096, ragged=True, causal=True),
        # A piece of a long prompt over what is already in the cache and itself.
        dict(name="attend_prompt_2048x10240_h16", kind="attend", batch=1, new=2048, heads=16, kv_heads=4, head_dim=128, block=64, bits="int8",
             length=10240, ragged=False, causal=True),
        # One token through a 1280-wide projection.
        dict(name="linear4_1x1280x1280", kind="linear4", tokens=1, features=1280, k=1280, group=64, zeros=False, epi="none"),
        # Sixteen tokens of a batch through a large layer.
        dict(name="linear4_16x28672x8192", kind="linear4", tokens=16, features=28672, k=8192, group=128, zeros=False, epi="none"),
        # A ragged batch through a feed-forward layer with its activation; small groups with zero points.
        dict(name="linear4_37x5120x1280", kind="linear4", tokens=37, features=5120, k=1280, group=32, zeros=True, epi="gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "attend", "linear4", "linear4"])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128])
        rot = rng.choice([dim, dim, dim // 2])
        heads, batch = rng.randint(2, 40), _log(rng, 1, 64)
        new = max(1, min(_log(rng, 1, 8192), 2 * 8192 * 40 * 128 // (heads * batch * dim)))
        return dict(kind="rotary", batch=batch, new=new, heads=heads, head_dim=dim, rot=rot, interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "parts"]), far=_log(rng, 10, 1000000))
    if kind == "append":
        heads, dim, block = rng.choice([1, 2, 4, 8, 20]), rng.choice([64, 64, 80, 96, 128]), rng.choice([16, 32, 64, 128])
        batch = _log(rng, 1, 64)
        new = max(1, min(_log(rng, 1, 4096), 4 * 4096 * 8 * 128 // (heads * batch * dim)))
        return dict(kind="append", batch=batch, new=new, heads=heads, head_dim=dim, block=block, bits=rng.choice(["int8", "int8", "e4m3"]),
                    past=_log(rng, 1, 4000))
    if kind == "attend":
        kv, share, dim = rng.choice([1, 2, 4, 8, 20]), rng.choice([1, 1, 2, 4, 5, 7, 8]), rng.choice([64, 64, 80, 96, 128, 128])
        new = rng.choice([1, 1, 1, rng.randint(2, 16), _log(rng, 17, 2048)])
        batch, length = _log(rng, 1, 48), _log(rng, 1, 131071)
        length = max(new, min(length, 150000 * 8 * 128 // (batch * kv * dim)))
        while batch > 1 and batch * kv * share * new * length * dim > 16 * 2048 * 9216 * 128:
            batch = (batch + 1) // 2
        while length > new and batch * kv * share * new * length * dim > 16 * 2048 * 9216 * 128:
            length = max(new, length // 2)
        while new > 1 and batch * kv * share * new * length * dim > 16 * 2048 * 9216 * 128:
            new = (new + 1) // 2
        return dict(kind="attend", batch=batch, new=new, heads=kv * share, kv_heads=kv, head_dim=dim, block=rng.choice([16, 32, 64, 64, 128]),
                    bits=rng.choice(["int8", "int8", "e4m3"]), length=length, ragged=rng.random() < 0.6, causal=rng.random() < 0.8)
    group = rng.choice([32, 64, 64, 128])
    tokens, features, k = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 2, 512)]), _log(rng, 200, 28672), 128 * _log(rng, 4, 64)
    while tokens > 16 and tokens * features * k > 16 * 28672 * 8192:
        tokens //= 2
    return dict(kind="linear4", tokens=tokens, features=features, k=k, group=group, zeros=rng.random() < 0.5,
                epi=rng.choice(["none", "none", "gelu", "relu"]))


# ------------------------------------------------------------------------------------ the inputs
def _randn(gen, shape, scale=1.0, dtype=torch.float16):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _whole(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


MOST = {"int8": 127.0, "e4m3": 448.0}


def _to8(x, most, bits):
    """fp16 values and their block's largest magnitude as 8-bit values (both products are exact; one division rounds)."""
    y = torch.where(most == 0, torch.zeros((), device=x.device), x.float() * MOST[bits] / most)
    return y.round().to(torch.int8) if bits == "int8" else y.to(torch.float8_e4m3fn).view(torch.uint8)


def _number(q, bits):
    return q.float() if bits == "int8" else q.view(torch.float8_e4m3fn).float()


def _cache(gen, pages, heads, block, dim, bits):
    """A cache as earlier tokens left it: (pages, heads, block, dim) 8-bit values, (pages, heads) largest magnitudes."""
    x = _randn(gen, (pages, heads, block, dim)) * (0.5 + torch.rand((1, heads, 1, dim), generator=gen, device="cuda")).half()
    most = x.abs().amax((2, 3)).float()
    return _to8(x, most[:, :, None, None], bits), most


def _inputs(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = np.random.default_rng(seed)
    if c["kind"] == "rotary":
        B, L = c["batch"], c["new"]
        news = [L] + [int(n) for n in host.integers(max(1, L // 2), L + 1, B - 1)]
        lens = [n + int(host.integers(0, c["far"] + 1)) for n in news]
        return dict(x=_randn(gen, (B, L, c["heads"], c["head_dim"])), lens=_whole(lens), news=_whole(news))
    if c["kind"] == "linear4":
        N, M, K, G = c["tokens"], c["features"], c["k"], c["group"]
        s = dict(x=_randn(gen, (N, K)), q=torch.randint(0, 16, (K, M), generator=gen, device="cuda", dtype=torch.uint8),
                 scales=(0.004 + 0.004 * torch.rand((K // G, M), generator=gen, device="cuda")).half(), bias=_randn(gen, (M,), 0.05), zeros=None)
        if c["zeros"]:
            s["zeros"] = torch.randint(5, 11, (K // G, M), generator=gen, device="cuda", dtype=torch.uint8)
        return s
    B, T, E, L = c["batch"], c["block"], c["head_dim"], c["new"]
    if c["kind"] == "append":
        H = c["heads"]
        news = [L] + [int(n) for n in host.integers(max(1, L // 2), L + 1, B - 1)]
        past = [int(host.integers(0, c["past"] + 1)) for _ in range(B)]
    else:
        H = c["kv_heads"]
        news = [L] + ([int(n) for n in host.integers(max(1, L // 2), L + 1, B - 1)] if c["ragged"] else [L] * (B - 1))
        total = [c["length"]] + [int(host.integers(max(L, c["length"] // 8), c["length"] + 1)) if c["ragged"] else c["length"] for _ in range(B - 1)]
        past = [t - n for t, n in zip(total, news)]
    lens = [p + n for p, n in zip(past, news)]
    need = [-(-n // T) for n in lens]
    width, pages = max(need), sum(need)
    order = host.permutation(pages)
    table = np.zeros((B, width), np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(lens=_whole(lens), news=_whole(news), table=torch.from_numpy(table).cuda())
    s["k"], s["kmax"] = _cache(gen, pages, H, T, E, c["bits"])
    s["v"], s["vmax"] = _cache(gen, pages, H, T, E, c["bits"])
    if c["kind"] == "append":
        kv = _randn(gen, (B, L, 2, H, E), 1.1)
        s["new_k"], s["new_v"] = kv[:, :, 0], kv[:, :, 1]
        first = [p // T * T for p in past]           # the first token of the first block that is written
        s["first"] = _whole(first)
        s["rows"] = max(n - f for n, f in zip(lens, first))
    else:
        s["q"] = _randn(gen, (B, L, c["heads"], E))
    return s


def _frequencies(c):
    """Radians a position for each pair of a head, in fp64, and what the cosines and sines are multiplied by."""
    rot, base, name = c["rot"], 10000.0, c["scaling"]
    if name == "ntk":
        base *= 4.0 ** (rot / (rot - 2))
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if name == "linear":
        f = f / 4.0
    if name == "parts":
        turns = 4096 * f / (2 * math.pi)
        kept = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return (f / 32.0 * (1 - kept) + f * kept).cuda(), 0.1 * math.log(32.0) + 1.0
    return f.cuda(), 1.0


# ----------------------------------------------------------------------------------- preparation
_context = None


def _package():
    import juliavision_b200 as jv
    global _context
    if _context is None:
        _context = jv.Ctx(0)
    return jv, _context


_NUMPY = {torch.float16: np.float16, torch.float32: np.float32, torch.int8: np.int8, torch.uint8: np.uint8, torch.int32: np.int32}


def _array(t):
    """A tensor as the device array of the reversed shape and strides."""
    jv, ctx = _package()
    return jv.DeviceArray(ctx, t.data_ptr(), _NUMPY[t.dtype], tuple(reversed(t.shape)), tuple(reversed(t.stride())), owner=t)


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if c["kind"] == "rotary":
        s["freq"], s["gain"] = _frequencies(c)
        s["out"] = torch.zeros_like(s["x"])
    elif c["kind"] == "append":
        s["out"] = [torch.zeros((c["batch"], s["rows"], c["heads"], c["head_dim"]), dtype=torch.float16, device="cuda") for _ in range(2)]
    elif c["kind"] == "attend":
        s["out"] = torch.zeros_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(c["head_dim"])
    else:
        s["out"] = torch.zeros((c["tokens"], c["features"]), dtype=torch.float16, device="cuda")
    if own:      # the handles that a program keeps: views of its arrays, the plan of the positions, the weight as it is laid out
        jv, ctx = _package()
        torch.cuda.synchronize()
        a = s["own"] = {n: _array(t) for n, t in s.items() if isinstance(t, torch.Tensor) and t.dtype in _NUMPY}
        if c["kind"] == "rotary":
            scaling = {"none": None, "linear": ("linear", 4.0), "ntk": ("ntk", 4.0), "parts": ("parts", 32.0, 4096, 1.0, 32.0)}[c["scaling"]]
            a["plan"] = jv.rotaryplan(ctx, c["rot"], base=10000.0, interleaved=c["interleaved"], scaling=scaling)
            for n in ("x", "out"):
                a[n] = a[n].permute((0, 2, 1, 3))              # (E, L, H, B)
        elif c["kind"] == "linear4":
            a["w"] = jv.pack4(ctx, a["q"], a["scales"], a.get("zeros"), c["group"])
            ctx.synchronize()
            del a["q"], s["q"]
        else:
            a["cache"] = jv.Cache8(a["k"], a["v"], a["kmax"], a["vmax"], c["bits"])
            for n in ("q", "new_k", "new_v"):
                if n in a:
                    a[n] = a[n].permute((0, 2, 1, 3))
            outs = s["out"] if c["kind"] == "append" else [s["out"]]
            a["out"] = [_array(t).permute((0, 2, 1, 3)) for t in outs]
    return s


# ------------------------------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    if own:
        return globals()["_own_" + c["kind"]](c, state, state["own"])
    return globals()["_plain_" + c["kind"]](c, state)


def _own_rotary(c, s, a):
    jv, ctx = _package()
    jv.rotary_(ctx, a["plan"], a["out"], a["x"], lens=a["lens"], news=a["news"])
    return s["out"]


def _own_append(c, s, a):
    jv, ctx = _package()
    jv.cacheappend_(ctx, a["cache"], a["new_k"], a["new_v"], a["table"], a["lens"], a["news"])
    jv.cacheread_(ctx, a["out"][0], a["cache"], "k", a["table"], a["lens"], a["first"])
    jv.cacheread_(ctx, a["out"][1], a["cache"], "v", a["table"], a["lens"], a["first"])
    return s["out"]


def _own_attend(c, s, a):
    jv, ctx = _package()
    ctx.ws.reset()
    jv.cachesdpa_(ctx, a["out"][0], a["q"], a["cache"], a["table"], a["lens"], a["news"], scale=s["scale"], causal=c["causal"])
    return s["out"]


def _own_linear4(c, s, a):
    jv, ctx = _package()
    ctx.ws.reset()
    jv.matmul4_(ctx, a["out"], a["w"], a["x"], a["bias"], epi={"none": "identity"}.get(c["epi"], c["epi"]))
    return s["out"]


def _plain_rotary(c, s):
    x, rot = s["x"], c["rot"]
    B, L = x.shape[:2]
    row = torch.arange(L, device="cuda")
    at = (s["lens"] - s["news"])[:, None] + row                                     # (B, L)
    angle = at.double()[:, :, None, None] * s["freq"]                               # (B, L, 1, rot/2), far positions in fp64
    cos, sin = (torch.cos(angle) * s["gain"]).float(), (torch.sin(angle) * s["gain"]).float()
    part = x[..., :rot].float()
    if c["interleaved"]:
        u, w = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((u * cos - w * sin, w * cos + u * sin), -1).flatten(-2)
    else:
        u, w = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat((u * cos - w * sin, w * cos + u * sin), -1)
    y = torch.cat((turned.half(), x[..., rot:]), -1)
    return torch.where((row < s["news"][:, None])[:, :, None, None], y, s["out"])


def _blocks(s, name, first, count):
    """Blocks first[b] ... first[b] + count - 1 of each sequence: their pages (clamped), 8-bit values and largest magnitudes."""
    at = first[:, None] + torch.arange(count, device="cuda")
    page = s["table"].long().gather(1, at.clamp(max=s["table"].shape[1] - 1))
    return page, s[name][page], s[name + "max"][page]


def _plain_append(c, s):
    T, bits, rows = c["block"], c["bits"], s["rows"]
    count = -(-rows // T)
    lens, start, first = s["lens"].long(), (s["lens"] - s["news"]).long(), s["first"].long()
    token = first[:, None] + torch.arange(count * T, device="cuda")                 # (B, count * T)
    fresh = ((token >= start[:, None]) & (token < lens[:, None])).view(-1, count, T)
    old = (token < start[:, None]).view(-1, count, T)
    source = (token - start[:, None]).clamp(0, c["new"] - 1)[:, :, None, None]
    result = []
    for name, out in zip("kv", s["out"]):
        page, q, most = _blocks(s, name, first // T, count)                         # (B, count, H, T, E), (B, count, H)
        new = s["new_" + name].gather(1, source.expand(-1, -1, c["heads"], c["head_dim"]))
        new = new.view(len(lens), count, T, c["heads"], c["head_dim"]).permute(0, 1, 3, 2, 4)
        seen = fresh[:, :, None, :, None]
        kept = torch.where(old.any(-1)[:, :, None], most, torch.zeros_like(most))   # a block's scale stays while its first token does
        top = torch.maximum(kept, torch.where(seen, new, torch.zeros_like(new)).abs().amax((3, 4)).float())
        ratio = _number(q, bits) * most[..., None, None]
        ratio = torch.where(top[..., None, None] == 0, torch.zeros((), device="cuda"), ratio / top[..., None, None])
        ratio = ratio.round().to(torch.int8) if bits == "int8" else ratio.to(torch.float8_e4m3fn).view(torch.uint8)
        q = torch.where(seen, _to8(new, top[..., None, None], bits), torch.where(old[:, :, None, :, None], ratio, q))
        touched = fresh.any(-1)
        s[name][page[touched]] = q[touched]
        s[name + "max"][page[touched]] = top[touched]
        value = (_number(q, bits) * top[..., None, None] / MOST[bits]).half().permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :rows]
        result.append(torch.where((token < lens[:, None])[:, :rows, None, None], value, out))
    return result


def _plain_attend(c, s):
    B, L, H, E = s["q"].shape
    Hk, T, bits = c["kv_heads"], c["block"], c["bits"]
    width = s["table"].shape[1]
    every = torch.zeros(B, dtype=torch.long, device="cuda")
    _, k, kmax = _blocks(s, "k", every, width)
    _, v, vmax = _blocks(s, "v", every, width)
    k = (_number(k, bits) * (kmax[..., None, None] / MOST[bits])).transpose(1, 2).reshape(B, Hk, width * T, E)
    v = (_number(v, bits) * (vmax[..., None, None] / MOST[bits])).transpose(1, 2).reshape(B, Hk, width * T, E)
    q = s["q"].float().permute(0, 2, 1, 3).reshape(B, Hk, H // Hk * L, E)           # (share, L) flattened
    score = torch.matmul(q, k.transpose(2, 3)).view(B, Hk, H // Hk, L, width * T).mul_(s["scale"])
    token, row = torch.arange(width * T, device="cuda"), torch.arange(L, device="cuda")
    last = s["lens"].long()[:, None] - 1
    if c["causal"]:
        last = last + 1 - s["news"].long()[:, None] + row                           # (B, L): a query's own position
    hidden = (token > last[:, :, None])[:, None, None] | (token >= s["lens"][:, None])[:, None, None, None]
    score.masked_fill_(hidden, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, H // Hk * L, width * T), v).view(B, Hk, H // Hk, L, E) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, L, H, E).half()
    return torch.where((row < s["news"][:, None])[:, :, None, None], o, s["out"])


def _plain_linear4(c, s):
    K, M = s["q"].shape
    G = c["group"]
    zero = s["zeros"].float() if s["zeros"] is not None else torch.full((K // G, M), 8.0, device="cuda")
    w = ((s["q"].view(K // G, G, M).float() - zero[:, None]) * s["scales"].float()[:, None]).view(K, M)
    y = torch.matmul(s["x"].float(), w) + s["bias"].float()
    if c["epi"] != "none":     # the activation is applied to the value already rounded
        y = y.half().float()
        y = torch.clamp(y, min=0) if c["epi"] == "relu" else 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    return y.half()


# ------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    if c["kind"] == "linear4":
        N, M, K = c["tokens"], c["features"], c["k"]
        groups = M * (K // c["group"])
        return {"bytes": M * K / 2 + groups * (3 if c["zeros"] else 2) + 2 * (N * K + M + N * M), "flops": 2.0 * N * M * K}
    s = _sizes(c)
    if c["kind"] == "rotary":
        n = s["new"] * c["heads"] * c["head_dim"]
        return {"bytes": 4 * n + 8 * c["batch"], "flops": 3 * n}
    if c["kind"] == "append":
        n = c["heads"] * c["head_dim"]
        # K and V: fp16 tokens in; the 8-bit blocks that are written, and the values read from them
        return {"bytes": 2 * n * (2 * s["new"] + 3 * s["touched"]), "flops": 4 * n * s["touched"]}
    E = c["head_dim"]
    kv = 2 * s["total"] * c["kv_heads"] * (E + 4 / c["block"])
    return {"bytes": kv + 4 * s["new"] * c["heads"] * E, "flops": 4.0 * E * c["heads"] * s["pairs"]}


def _sizes(c):
    """Expected counts of a case whose lengths depend on the seed."""
    B, L = c["batch"], c["new"]
    ragged = c["kind"] != "attend" or c["ragged"]
    new = L + (B - 1) * ((max(1, L // 2) + L) / 2 if ragged else L)
    if c["kind"] == "rotary":
        return dict(new=new)
    if c["kind"] == "append":
        return dict(new=new, touched=new + B * min(c["past"], (c["block"] - 1)) / 2)
    total = c["length"] + (B - 1) * ((max(L, c["length"] // 8) + c["length"]) / 2 if ragged else c["length"])
    mean = new / B
    return dict(new=new, total=total, pairs=new * (total / B - ((mean - 1) / 2 if c["causal"] else 0)))


# ------------------------------------------------------------------------- the definition in fp64
def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    return globals()["_exact_" + c["kind"]](c, s)


def _exact_rotary(c, s):
    x = s["x"].double()
    out = torch.zeros_like(x)
    f, gain = _frequencies(c)
    half = c["rot"] // 2
    a = torch.arange(half, device="cuda")
    first, second = (2 * a, 2 * a + 1) if c["interleaved"] else (a, a + half)
    for b, (n, m) in enumerate(zip(s["lens"].tolist(), s["news"].tolist())):
        turn = torch.polar(torch.full((), gain, dtype=torch.float64, device="cuda"),
                           torch.arange(n - m, n, device="cuda", dtype=torch.float64)[:, None] * f)[:, None]
        z = torch.complex(x[b, :m][..., first], x[b, :m][..., second]) * turn
        out[b, :m] = x[b, :m]
        out[b, :m][..., first] = z.real
        out[b, :m][..., second] = z.imag
    return out


def _exact8(x, bits):
    if bits == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, torch.where(x.abs() < torch.exp2(e), e - 1, e)).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_append(c, s):
    T, bits, top8 = c["block"], c["bits"], MOST[c["bits"]]
    outs = []
    for name in "kv":
        out = torch.zeros((c["batch"], s["rows"], c["heads"], c["head_dim"]), dtype=torch.float64, device="cuda")
        for b, (n, m, f) in enumerate(zip(s["lens"].tolist(), s["news"].tolist(), s["first"].tolist())):
            new = s["new_" + name][b, :m].double()                                  # (m, H, E)
            had = n - m - f                                                         # tokens that the first block held
            page = int(s["table"][b, f // T])
            held, most = _number(s[name][page], bits).double(), s[name + "max"][page].double()
            tokens = torch.cat(((held * most[:, None, None] / top8).transpose(0, 1)[:had], new))
            pad = -len(tokens) % T
            blocks = torch.cat((tokens, tokens.new_zeros((pad,) + tokens.shape[1:]))).view(-1, T, c["heads"], c["head_dim"])
            fresh = blocks.clone()
            fresh[0, :had] = 0
            top = fresh.abs().amax((1, 3), keepdim=True)
            if had:
                top[0] = torch.maximum(top[0], most[None, :, None])
            ratio = torch.where(top == 0, torch.zeros_like(blocks), blocks * top8 / torch.where(top == 0, torch.ones_like(top), top))
            if had:      # what a kept value stands for, without the rounding of its quotient by the 8-bit range
                ratio[0, :had] = (held * most[:, None, None]).transpose(0, 1)[:had] / top[0].clamp(min=1e-300)
            out[b, :n - f] = (_exact8(ratio, bits) * top / top8).flatten(0, 1)[:n - f]
        outs.append(out)
    return outs


def _exact_attend(c, s):
    share, T, top8 = c["heads"] // c["kv_heads"], c["block"], MOST[c["bits"]]
    if sum(a * b for a, b in zip(s["lens"].tolist(), s["news"].tolist())) * c["heads"] * c["head_dim"] > 1e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(s["lens"].tolist(), s["news"].tolist())):
        pages = s["table"][b, :-(-n // T)].long()
        for h in range(c["kv_heads"]):
            kv = []
            for name in "kv":
                x = _number(s[name][pages, h], c["bits"]).double() * s[name + "max"][pages, h].double()[:, None, None] / top8
                kv.append(x.flatten(0, 1)[:n])
            q = s["q"][b, :m, h * share:(h + 1) * share].double()                   # (m, share, E)
            w = torch.einsum("lge,ne->lgn", q, kv[0]) / math.sqrt(c["head_dim"])
            if c["causal"]:
                w.masked_fill_((torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None])[:, None], float("-inf"))
            out[b, :m, h * share:(h + 1) * share] = torch.einsum("lgn,ne->lge", torch.softmax(w, -1), kv[1])
    return out


def _exact_linear4(c, s):
    zero = torch.full_like(s["scales"], 8).double() if s["zeros"] is None else s["zeros"].double()
    each = lambda t: t.double().repeat_interleave(c["group"], 0)  # noqa: E731
    y = s["x"].double() @ ((s["q"].double() - each(zero)) * each(s["scales"])) + s["bias"].double()
    if c["epi"] == "relu":
        y = y.clamp(min=0)
    if c["epi"] == "gelu":
        y = torch.nn.functional.gelu(y)
    return y
