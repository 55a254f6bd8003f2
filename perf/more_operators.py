"""What surrounds a decoder's step, as cases that can be timed and compared: norms of queries and keys with the position
rotation in one pass, attention of packed prompts of different lengths with grouped heads, beam search's choice over beams and
vocabulary, and the reordering of the beams' 8-bit caches.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what a program holds before a call,
`run()` is one call.  With `own` false `run()` computes the formulas with elementary tensor operations in fp32 (angles, and the
sums that candidates are ordered by, in fp64); with `own` true it makes the package's calls.  Tensors are in torch order, the reverse
of the package's.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # One token of eight sequences, 32 query and 8 key heads side by side in one projection: the smallest call of a step.
        dict(name="norm_step_8x40x64", kind="norm", batch=8, new=1, heads=32, kv_heads=8, head_dim=64, rot=64, interleaved=False, far=1500),
        # Two whole prompts, positions far out.
        dict(name="norm_prompt_2x8192x40x128", kind="norm", batch=2, new=8192, heads=32, kv_heads=8, head_dim=128, rot=128, interleaved=False,
             far=120000),
        # Ragged prompts, heads of 96 of which the first 48 elements are turned, neighbours as pairs.
        dict(name="norm_ragged_7x611x24x96", kind="norm", batch=7, new=611, heads=20, kv_heads=4, head_dim=96, rot=48, interleaved=True,
             far=5000),
        # A single short prompt: the smallest call, where latency counts.
        dict(name="prompt_1x77_h20", kind="prompt", batch=1, longest=77, shortest=77, heads=20, kv_heads=20, head_dim=64, past=0, causal=True),
        # 37 prompts of 1 to 2000 tokens side by side, four query heads to a key head.
        dict(name="prompt_37x2000_h32", kind="prompt", batch=37, longest=2000, shortest=1, heads=32, kv_heads=8, head_dim=128, past=0,
             causal=True),
        # One long prompt: the largest.
        dict(name="prompt_1x16384_h32", kind="prompt", batch=1, longest=16384, shortest=16384, heads=32, kv_heads=8, head_dim=128, past=0,
             causal=True),
        # Three pieces of long prompts, each over the keys of the pieces before it and its own; five query heads to a key head of 80.
        dict(name="prompt_3x500_past30000_h20", kind="prompt", batch=3, longest=500, shortest=200, heads=20, kv_heads=4, head_dim=80,
             past=30000, causal=True),
        # An encoder's sequences packed instead of padded: every key of its own sequence is visible.
        dict(name="prompt_16x1500_h20", kind="prompt", batch=16, longest=1500, shortest=300, heads=20, kv_heads=20, head_dim=64, past=0,
             causal=False),
        # Five beams over the vocabulary of a speech decoder: the smallest choice.
        dict(name="beams_1x5x51865", kind="beams", batch=1, beams=5, vocab=51865, keep=5, bits=16, ended=0.0),
        # 64 searches at once, more logits than the L2 cache holds; twice as many candidates kept as beams.
        dict(name="beams_64x8x131072", kind="beams", batch=64, beams=8, vocab=131072, keep=16, bits=16, ended=0.1),
        # The caches of five beams of a speech decoder's 32 layers, half way through a page.
        dict(name="reorder_1x5_32x20x64", kind="reorder", batch=1, beams=5, layers=32, heads=20, head_dim=64, block=64, length=220,
             bits="int8"),
        # 16 searches of four beams each, 16 layers.
        dict(name="reorder_16x4_16x8x128", kind="reorder", batch=16, beams=4, layers=16, heads=8, head_dim=128, block=64, length=700,
             bits="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MOST_PROMPT = 32 * 16384 * 16384 // 2 * 128       # heads x visible pairs x head dim of the largest listed prompt


def draw(rng):
    kind = rng.choice(["norm", "norm", "prompt", "prompt", "prompt", "prompt", "beams", "beams", "reorder"])
    if kind == "norm":
        dim = rng.choice([64, 64, 80, 96, 128, 128])
        rot = rng.choice([dim, dim, dim // 2])
        kv, share, batch = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5]), _log(rng, 1, 64)
        heads = kv * share
        new = max(1, min(_log(rng, 1, 8192), 2 * 8192 * 40 * 128 // ((heads + kv) * batch * dim)))
        return dict(kind="norm", batch=batch, new=new, heads=heads, kv_heads=kv, head_dim=dim, rot=rot, interleaved=rng.random() < 0.4,
                    far=_log(rng, 10, 1000000))
    if kind == "prompt":
        kv, share, dim = rng.choice([1, 2, 4, 8, 20]), rng.choice([1, 1, 2, 4, 5, 7, 8]), rng.choice([40, 64, 64, 72, 80, 96, 128, 128])
        batch, longest = _log(rng, 1, 64), _log(rng, 1, 16384)
        past = _log(rng, 1, 32768) if rng.random() < 0.35 else 0
        causal = rng.random() < 0.8
        while batch > 1 and batch * (longest + past) * kv * dim > 60000 * 8 * 128:
            batch = (batch + 1) // 2
        while longest > 1 and batch * kv * share * longest * (longest / (2 if causal else 1) + past) * dim > MOST_PROMPT:
            longest = (longest + 1) // 2
        shortest = rng.choice([1, longest, max(1, longest // 4)])
        return dict(kind="prompt", batch=batch, longest=longest, shortest=shortest, heads=kv * share, kv_heads=kv, head_dim=dim, past=past,
                    causal=causal)
    if kind == "beams":
        beams, vocab, bits = rng.randint(1, 16), _log(rng, 1000, 131072), rng.choice([16, 16, 32])
        batch = max(1, min(_log(rng, 1, 64), 64 * 8 * 131072 * 16 // (beams * vocab * bits)))
        return dict(kind="beams", batch=batch, beams=beams, vocab=vocab, keep=beams * rng.choice([1, 2]), bits=bits,
                    ended=rng.choice([0.0, 0.2]))
    beams, heads, dim, block = rng.randint(2, 12), rng.choice([1, 4, 8, 20]), rng.choice([64, 80, 128]), rng.choice([16, 32, 64, 128])
    batch, layers, length = _log(rng, 1, 16), rng.randint(1, 32), _log(rng, 1, 1000)
    most = 16 * 4 * 16 * 8 * 128 * 64
    while batch > 1 and batch * beams * layers * heads * dim * block > most:
        batch = (batch + 1) // 2
    while layers > 1 and batch * beams * layers * heads * dim * block > most:
        layers = (layers + 1) // 2
    length = max(1, min(length, 11 * most // (batch * beams * layers * heads * dim)))
    return dict(kind="reorder", batch=batch, beams=beams, layers=layers, heads=heads, head_dim=dim, block=block, length=length,
                bits=rng.choice(["int8", "e4m3"]))


# ------------------------------------------------------------------------------------ the inputs
def _randn(gen, shape, scale=1.0, dtype=torch.float16):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _whole(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _sums(counts):
    return [0] + [int(n) for n in np.cumsum(counts)]


SPARE = 3     # rows behind the last sequence of a packed prompt, which belong to nobody


def _lengths(c):
    """New and earlier tokens of a packed prompt's sequences, the case's own: a seed only changes their order."""
    host = np.random.default_rng(c["batch"] + c["longest"])
    news = [c["longest"]] + [int(n) for n in host.integers(c["shortest"], c["longest"] + 1, c["batch"] - 1)]
    return [(n, int(host.integers(c["past"] // 2, c["past"] + 1))) for n in news]


def _inputs(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = np.random.default_rng(seed)
    B = c["batch"]
    if c["kind"] == "norm":
        L, E, H = c["new"], c["head_dim"], c["heads"] + c["kv_heads"]
        news = [L] + [int(n) for n in host.integers(max(1, L // 2), L + 1, B - 1)]
        lens = [n + int(host.integers(0, c["far"] + 1)) for n in news]
        # the projection's rows hold the values' heads too; heads differ in size, as they do before a norm
        x = _randn(gen, (B, L, H + c["kv_heads"], E)) * (0.2 + 4 * torch.rand((H + c["kv_heads"], 1), generator=gen, device="cuda")).half()
        return dict(x=x, weight=(0.5 + torch.rand((2, E), generator=gen, device="cuda")).half(), lens=_whole(lens), news=_whole(news))
    if c["kind"] == "prompt":
        E, Hq, H = c["head_dim"], c["heads"], c["kv_heads"]
        lengths = [_lengths(c)[i] for i in host.permutation(B)]
        news, past = [n for n, _ in lengths], [p for _, p in lengths]
        N = sum(news) + SPARE
        s = dict(starts=_whole(_sums(news)), kstarts=_whole(_sums([n + p for n, p in zip(news, past)])))
        qkv = _randn(gen, (N, Hq + 2 * H, E))
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
        if c["past"]:     # keys and values of the earlier pieces and this one, from a buffer of their own
            kv = _randn(gen, (N + sum(past), 2, H, E))
            s["k"], s["v"] = kv[:, 0], kv[:, 1]
        s["lengths"] = lengths
        return s
    if c["kind"] == "beams":
        K, V = c["beams"], c["vocab"]
        logits = torch.randn((B, K, V), generator=gen, device="cuda", dtype=torch.float32).mul_(2.5)
        peak = torch.randint(0, V, (B, K, 8), generator=gen, device="cuda")       # a few likely tokens, as a trained model gives
        logits.scatter_add_(2, peak, 6 + 4 * torch.rand((B, K, 8), generator=gen, device="cuda"))
        logits[:, :, torch.randint(0, V, (V // 50,), generator=gen, device="cuda")] = float("-inf")   # tokens that are ruled out
        scores = -30 * torch.rand((B, K), generator=gen, device="cuda")
        if K > 1:
            scores[:, 1:][torch.rand((B, K - 1), generator=gen, device="cuda") < 0.05] = float("-inf")    # beams not begun
        return dict(logits=logits.to(torch.float16 if c["bits"] == 16 else torch.float32), scores=scores,
                    ended=(torch.rand((B, K), generator=gen, device="cuda") < c["ended"]).to(torch.int32))
    K, T, H, E, A = c["beams"], c["block"], c["heads"], c["head_dim"], c["layers"]
    S, width = B * K, -(-c["length"] // T) + 1
    lens = np.repeat(host.integers(max(1, c["length"] // 2), c["length"] + 1, B), K)
    P = S * width
    mine = host.permutation(P).reshape(S, width).astype(np.int32)     # the pages each beam writes
    table = mine.copy()
    for b in range(S):      # pages that are full may be another beam's of the same search
        full = lens[b] // T
        table[b, :full] = mine[b // K * K + host.integers(0, K, full), np.arange(full)]
    stays = host.random((B, K)) < 0.45                                # beams that go on keep their place, the others give way to one of them
    stays[np.arange(B), host.integers(0, K, B)] = True
    parents = np.stack([np.where(row, np.arange(K), host.choice(np.flatnonzero(row), K)) for row in stays])
    kv = [torch.randint(-127, 127, (A, P, H, T, E), generator=gen, device="cuda", dtype=torch.int8) for _ in range(2)]
    if c["bits"] == "e4m3":
        kv = [x.view(torch.uint8).bitwise_and_(0xbf) for x in kv]     # numbers of up to 1.875 in size, no NaN
    most = torch.rand((2, A, P, H), generator=gen, device="cuda")
    return dict(k=kv[0], v=kv[1], kmax=most[0], vmax=most[1], lens=_whole(lens), own=_whole(mine), table=_whole(table), parents=_whole(parents))


EPS = 1e-6


def _frequencies(c):
    """Radians a position of each pair of a head, in fp64."""
    return (10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])).cuda()


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
    if c["kind"] == "norm":
        s["x"] = s["x"][:, :, :c["heads"] + c["kv_heads"]]
        s["freq"] = _frequencies(c)
        s["out"] = torch.zeros(s["x"].shape, dtype=torch.float16, device="cuda")
    elif c["kind"] == "prompt":
        s["out"] = torch.zeros(s["q"].shape, dtype=torch.float16, device="cuda")
        s["scale"] = 1.0 / math.sqrt(c["head_dim"])
    elif c["kind"] == "beams":
        like = dict(size=(c["batch"], c["keep"]), device="cuda")
        s["best"], s["parents"], s["tokens"] = (torch.zeros(dtype=t, **like) for t in (torch.float32, torch.int32, torch.int32))
        s["pad"] = 3
    if own:      # the handles that a program keeps: views of its arrays, the plan of the positions, a cache a layer
        jv, ctx = _package()
        torch.cuda.synchronize()
        a = s["mine"] = {n: _array(t) for n, t in s.items() if isinstance(t, torch.Tensor) and t.dtype in _NUMPY and t.ndim < 5}
        if c["kind"] == "norm":
            a["plan"] = jv.rotaryplan(ctx, c["rot"], base=10000.0, interleaved=c["interleaved"])
            for n in ("x", "out"):
                a[n] = a[n].permute((0, 2, 1, 3))                     # (E, L, H, B)
        elif c["kind"] == "prompt":
            for n in ("q", "k", "v", "out"):
                a[n] = a[n].permute((0, 2, 1))                        # (E, tokens, H)
        elif c["kind"] == "reorder":
            a["caches"] = [jv.Cache8(*(_array(s[n][i]) for n in ("k", "v", "kmax", "vmax")), c["bits"]) for i in range(c["layers"])]
    return s


# ------------------------------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    if own:
        return globals()["_own_" + c["kind"]](c, state, state["mine"])
    return globals()["_plain_" + c["kind"]](c, state)


def _own_norm(c, s, a):
    jv, ctx = _package()
    jv.normrotary_(ctx, a["plan"], a["out"], a["x"], a["weight"], eps=EPS, split=c["heads"], lens=a["lens"], news=a["news"])
    return s["out"]


def _own_prompt(c, s, a):
    jv, ctx = _package()
    ctx.ws.reset()
    jv.packedsdpa_(ctx, a["out"], a["q"], a["k"], a["v"], a["starts"], a["kstarts"], scale=s["scale"], causal=c["causal"])
    return s["out"]


def _own_beams(c, s, a):
    jv, ctx = _package()
    ctx.ws.reset()
    jv.beamselect_(ctx, a["best"], a["parents"], a["tokens"], a["logits"], a["scores"], ended=a["ended"], pad=s["pad"])
    return [s["best"], s["parents"], s["tokens"]]


def _own_reorder(c, s, a):
    jv, ctx = _package()
    jv.cachereorder_(ctx, a["caches"], a["table"], a["own"], a["parents"], a["lens"])
    return [s["table"], s["k"], s["v"], s["kmax"], s["vmax"]]


def _plain_norm(c, s):
    x, rot, H = s["x"], c["rot"], c["heads"]
    B, L = x.shape[:2]
    row = torch.arange(L, device="cuda")
    at = (s["lens"] - s["news"])[:, None] + row                                     # (B, L)
    angle = at.double()[:, :, None, None] * s["freq"]                               # (B, L, 1, rot/2), far positions in fp64
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    z = x.float()
    z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + EPS)
    z[:, :, :H] *= s["weight"][0].float()
    z[:, :, H:] *= s["weight"][1].float()
    part = z[..., :rot]
    if c["interleaved"]:
        u, w = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((u * cos - w * sin, w * cos + u * sin), -1).flatten(-2)
    else:
        u, w = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat((u * cos - w * sin, w * cos + u * sin), -1)
    y = torch.cat((turned, z[..., rot:]), -1).half()
    return torch.where((row < s["news"][:, None])[:, :, None, None], y, s["out"])


def _plain_prompt(c, s):
    out, H, share = s["out"].clone(), c["kv_heads"], c["heads"] // c["kv_heads"]
    q0 = k0 = 0
    for new, past in s["lengths"]:
        n = new + past
        k = s["k"][k0:k0 + n].float().permute(1, 2, 0)                              # (H, E, n)
        v = s["v"][k0:k0 + n].float().transpose(0, 1)                               # (H, n, E)
        rows = max(1, min(new, (1 << 29) // (c["heads"] * n)))                      # of scores at once
        for r in range(0, new, rows):
            m = min(rows, new - r)
            q = s["q"][q0 + r:q0 + r + m].float().view(m, H, share, -1).permute(1, 2, 0, 3).reshape(H, share * m, -1)
            seen = past + r + m if c["causal"] else n                               # keys that some of these rows see
            score = torch.matmul(q, k[:, :, :seen]).mul_(s["scale"])
            if c["causal"]:
                hidden = torch.arange(seen, device="cuda") > past + r + torch.arange(m, device="cuda")[:, None]
                score.view(H, share, m, seen).masked_fill_(hidden, float("-inf"))
            score.sub_(score.amax(-1, keepdim=True)).exp_()
            o = torch.matmul(score, v[:, :seen]) / score.sum(-1, keepdim=True)
            out[q0 + r:q0 + r + m] = o.view(H, share, m, -1).permute(2, 0, 1, 3).reshape(m, c["heads"], -1).half()
        q0, k0 = q0 + new, k0 + n
    return out


def _plain_beams(c, s):
    B, K, V, N = c["batch"], c["beams"], c["vocab"], c["keep"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    candidate = s["scores"].double()[:, :, None] + (x - total)
    over = torch.full((V,), float("-inf"), dtype=torch.float64, device="cuda")
    over[s["pad"]] = 0
    candidate = torch.where(s["ended"][:, :, None] != 0, s["scores"].double()[:, :, None] + over, candidate)
    best, at = torch.sort(candidate.view(B, K * V), dim=-1, descending=True, stable=True)      # ties: the lowest index first
    best, at = best[:, :N], at[:, :N]
    return [best.float(), (at // V).int(), (at % V).int()]


def _plain_reorder(c, s):
    K, T = c["beams"], c["block"]
    lens = s["lens"].long()
    S, width = s["table"].shape
    source = (torch.arange(S, device="cuda") // K * K) + s["parents"].long().view(-1)
    full = lens // T
    page = torch.arange(width, device="cuda")
    s["table"].copy_(torch.where(page < full[:, None], s["table"][source], s["own"]))
    here = s["own"].long().gather(1, full[:, None])[:, 0]                           # the page each beam is writing
    there = here[source]
    kept = torch.arange(T, device="cuda") < (lens % T)[:, None]                     # (S, T)
    some = (lens % T > 0)[:, None]
    for n in "kv":
        x, m = s[n], s[n + "max"]
        x[:, here] = torch.where(kept[:, None, :, None], x[:, there], x[:, here])
        m[:, here] = torch.where(some, m[:, there], m[:, here])
    return [s["table"], s["k"], s["v"], s["kmax"], s["vmax"]]


# ------------------------------------------------------------------------------------------ work
def work(case):
    c, B = case, case["batch"]
    if c["kind"] == "norm":       # lengths depend on the seed: their mean
        L = c["new"]
        tokens = L + (B - 1) * (max(1, L // 2) + L) / 2
        n = tokens * (c["heads"] + c["kv_heads"]) * c["head_dim"]
        return {"bytes": 4 * n + 4 * c["head_dim"] + 8 * B, "flops": 7 * n}
    if c["kind"] == "prompt":
        lengths, E = _lengths(c), c["head_dim"]
        tokens, keys = sum(n for n, _ in lengths), sum(n + p for n, p in lengths)
        pairs = sum(n * (p + (n + 1) / 2 if c["causal"] else p + n) for n, p in lengths)
        return {"bytes": 4 * E * (c["heads"] * tokens + c["kv_heads"] * keys), "flops": 4.0 * E * c["heads"] * pairs}
    if c["kind"] == "beams":
        n = B * c["beams"] * c["vocab"]
        return {"bytes": n * c["bits"] / 8 + B * (8 * c["beams"] + 12 * c["keep"]), "flops": 3 * n}
    K, T = c["beams"], c["block"]
    gone = B * (K - (1 + (K - 1) * 0.45))                                           # beams that give way
    return {"bytes": 2 * gone * c["layers"] * 2 * c["heads"] * (c["head_dim"] * (min(T, c["length"] + 1) - 1) / 2 + 4)
            + 12 * B * K * -(-c["length"] // T), "flops": 0}


# ------------------------------------------------------------------------- the definition in fp64
def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, _inputs(case, seed))


def _exact_norm(c, s):
    H = c["heads"] + c["kv_heads"]
    x = s["x"][:, :, :H].double()
    size = torch.sqrt((x * x).sum(-1, keepdim=True) / c["head_dim"] + EPS)
    weight = torch.cat([s["weight"][i:i + 1].double().expand(n, -1) for i, n in enumerate((c["heads"], c["kv_heads"]))])
    out = torch.zeros_like(x)
    f = _frequencies(c)
    half = c["rot"] // 2
    a = torch.arange(half, device="cuda")
    first, second = (2 * a, 2 * a + 1) if c["interleaved"] else (a, a + half)
    for b, (n, m) in enumerate(zip(s["lens"].tolist(), s["news"].tolist())):
        z = x[b, :m] / size[b, :m] * weight
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.arange(n - m, n, device="cuda", dtype=torch.float64)[:, None] * f)[:, None]
        turned = torch.complex(z[..., first], z[..., second]) * turn
        z[..., first], z[..., second] = turned.real.clone(), turned.imag.clone()
        out[b, :m] = z
    return out


def _exact_prompt(c, s):
    share = c["heads"] // c["kv_heads"]
    if sum(n * (n + p) for n, p in s["lengths"]) * c["heads"] * c["head_dim"] > 1.2e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, kstarts = s["starts"].tolist(), s["kstarts"].tolist()
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        k0, k1 = kstarts[b], kstarts[b + 1]
        row = torch.arange(hi - lo, device="cuda")[:, None] + (k1 - k0 - hi + lo)
        for h in range(c["heads"]):
            k, v = s["k"][k0:k1, h // share].double(), s["v"][k0:k1, h // share].double()
            w = s["q"][lo:hi, h].double() @ k.T / math.sqrt(c["head_dim"])
            if c["causal"]:
                w = torch.where(torch.arange(k1 - k0, device="cuda") <= row, w, float("-inf"))
            out[lo:hi, h] = torch.softmax(w, -1) @ v
    return out


def _exact_beams(c, s):
    V, N = c["vocab"], c["keep"]
    most = min(N + 1, V)
    best, parents, tokens = [], [], []
    for b in range(c["batch"]):
        rows = []
        for k in range(c["beams"]):
            x, score, ended = s["logits"][b, k].double(), float(s["scores"][b, k]), int(s["ended"][b, k])
            if ended:
                rows.append((score, k, 3))
                rows += [(-math.inf, k, t) for t in range(N + 1) if t != 3]
                continue
            value = score + x - torch.logsumexp(x, 0)
            ranked = torch.topk(value, most)
            cut = float(ranked.values[-1])
            some = torch.nonzero(value >= cut)[:, 0][:2 * most] if cut > -math.inf else torch.arange(min(N, V), device="cuda")
            some = torch.cat((some, ranked.indices)).unique()
            rows += zip(value[some].tolist(), [k] * len(some), some.tolist())
        rows.sort(key=lambda r: (-r[0], r[1], r[2]))
        for to, column in zip((best, parents, tokens), zip(*rows[:N])):
            to.append(column)
    return [torch.tensor(best, dtype=torch.float64), torch.tensor(parents, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)]


def _exact_reorder(c, s):
    tops = []
    for name in ("kmax", "vmax"):
        top, was = s[name].double(), s[name].double()
        for b, row in enumerate(s["parents"].tolist()):
            for k, parent in enumerate(row):
                page, n = divmod(int(s["lens"][b * c["beams"]]), c["block"])
                if n:
                    top[:, int(s["own"][b * c["beams"] + k, page])] = was[:, int(s["own"][b * c["beams"] + parent, page])]
        tops.append(top)
    return [None, None, None] + tops       # the rest is whole numbers, moved
