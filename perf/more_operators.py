"""The attention layer of a transformer around its products, as its speed is measured.

``listed()`` holds the fixed cases, ``draw(rng)`` makes further ones of the same
ranges, ``prepare`` / ``run`` / ``work`` / ``exact`` say for a case what a program
holds beforehand, one pass, what the pass cannot do without, and the result in
64 bits.  ``own`` selects what ``run`` computes with: the package's operators, or
their definitions in elementary torch operations.

The operators, on tensors [batch, token, head, Dh]:

- ``rotary``: rotary positions with several axes.  Pair i of a head is turned by
  pos[token, axis(i)] * freq[i]; the pairs are (i, i + P) or (2i, 2i + 1).
- ``qk_norm``: RMS norm of every head of the queries and the keys, times gamma, and
  that rotation, in one pass.
- ``attention``: softmax(scores) v over the keys a query sees.  The scores are
  scale q.k, capped by c tanh(s / c) where there is a cap, plus a bias of the
  distance between key and query: -slope |j - p| or a table's entry at j - p,
  clipped to the table's ends.  A query sees the keys of an interval of its own
  (documents, a prefix, a length) and, where it is causal, none behind itself.

Sizes are those of the SDXL transformer blocks (10 heads of 64, 4096 and 77 tokens,
two guidance halves) and generic ones for grouped heads of 128, long prompts and
single tokens.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _rot(name, B, S, H, Dh, axes, interleaved, t, far=0):
    return {"name": name, "op": "rotary", "B": B, "S": S, "H": H, "Dh": Dh, "axes": axes, "interleaved": interleaved,
            "type": t, "far": far}


def _qk(name, B, S, H, Hkv, Dh, axes, interleaved, t, far=0):
    return {"name": name, "op": "qk_norm", "B": B, "S": S, "H": H, "Hkv": Hkv, "Dh": Dh, "axes": axes,
            "interleaved": interleaved, "type": t, "far": far}


def _att(name, B, Sq, Sk, H, Hkv, Dh, t, mask="none", causal=False, cap=0.0, bias="none", docs=0):
    """mask: none, documents (docs of them, packed), prefix, lengths (keys of a
    cache in use, the queries at their end); bias: none, slope, table."""
    return {"name": name, "op": "attention", "B": B, "Sq": Sq, "Sk": Sk, "H": H, "Hkv": Hkv, "Dh": Dh, "type": t,
            "mask": mask, "causal": causal, "cap": cap, "bias": bias, "docs": docs}


def listed():
    return [
        # the queries of one token on their way into attention, far into a text:
        # the smallest call, where latency is everything
        _rot("rotary_1x1x32x128", 1, 1, 32, 128, 1, False, "fp16", far=100000),
        # image tokens of both guidance halves, rows and columns as axes
        _rot("rotary_2x4096x10x64", 2, 4096, 10, 64, 2, True, "fp16"),
        # one token's queries and keys with grouped heads
        _qk("qk_norm_1x1x32+8x128", 1, 1, 32, 8, 128, 1, False, "bf16", far=100000),
        # odd in tokens and heads, a head size that is no power of two
        _qk("qk_norm_3x325x13+13x80", 3, 325, 13, 13, 80, 2, True, "fp16"),
        # a video's tokens: time, height and width as axes
        _qk("qk_norm_1x8192x32+8x128", 1, 8192, 32, 8, 128, 3, False, "bf16"),
        # one token for each of eight sequences of unlike length, capped scores
        _att("attention_8x1x32768x32/8x128_cap", 8, 1, 32768, 32, 8, 128, "fp16", mask="lengths", causal=True, cap=50.0),
        # a chunk of a prompt over the keys before it, scores falling with distance
        _att("attention_1x64x30001x32x128_slope", 1, 64, 30001, 32, 32, 128, "bf16", causal=True, bias="slope"),
        # prompts through a text encoder with a table of distances
        _att("attention_4x512x64x64_table", 4, 512, 512, 64, 64, 64, "bf16", bias="table"),
        # nine images of unlike size packed into one sequence
        _att("attention_1x8192x10x64_documents", 1, 8192, 8192, 10, 10, 64, "fp16", mask="documents", docs=9),
        # a prompt that sees itself whole, then tokens in order; odd lengths, capped scores
        _att("attention_2x2051x12x80_prefix_cap", 2, 2051, 2051, 12, 12, 80, "fp16", mask="prefix", cap=30.0),
        # a prompt with grouped heads
        _att("attention_1x4096x32/8x128_causal", 1, 4096, 4096, 32, 8, 128, "bf16", causal=True),
        # a long one: only the matrix rate counts
        _att("attention_1x16384x32/8x128_causal", 1, 16384, 16384, 32, 8, 128, "bf16", causal=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm", "attention", "attention", "attention"])
    t = rng.choice(["fp16", "bf16"])
    if op != "attention":
        Dh = rng.choice([40, 64, 64, 72, 80, 96, 128, 128, 256])
        H = _log(rng, 1, 40)
        B = _log(rng, 1, 4)
        S = _log(rng, 1, min(16384, 40_000_000 // (B * H * Dh)))
        axes = rng.choice([1, 2, 3])
        il = rng.random() < 0.5
        far = rng.choice([0, 0, 1000, 1000000])
        if op == "rotary":
            c = _rot("", B, S, H, Dh, axes, il, t, far)
        else:
            c = _qk("", B, S, H, rng.choice([h for h in range(1, H + 1) if H % h == 0]), Dh, axes, il, t, far)
    else:
        Dh = rng.choice([40, 64, 64, 80, 96, 128, 128, 128, 256])
        Hkv, G, B = _log(rng, 1, 16), rng.choice([1, 1, 2, 4, 5, 8]), _log(rng, 1, 8)
        H = Hkv * G
        mask = rng.choice(["none", "none", "documents", "prefix", "lengths"])
        # at most a quarter of the largest listed case's scores
        room = 2_000_000_000 // (B * H)
        if mask == "lengths":
            Sq = _log(rng, 1, 64)
            Sk = _log(rng, Sq, min(65536, room // Sq, 200_000_000 // (B * Hkv * Dh)))
        elif mask == "none" and rng.random() < 0.5:
            Sq = _log(rng, 1, 4096)
            Sk = _log(rng, 1, min(16384, max(1, room // Sq)))
        else:
            Sq = Sk = _log(rng, 16, min(8192, math.isqrt(room)))
        causal = mask == "lengths" or (mask in ("none", "documents") and Sk >= Sq and rng.random() < 0.5)
        c = _att("", B, Sq, Sk, H, Hkv, Dh, t, mask=mask, causal=causal, cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                 bias=rng.choice(["none", "none", "slope", "table"]),
                 docs=_log(rng, 1, min(16, Sq)) if mask == "documents" else 0)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# what a case's masks are: of its sizes alone
# ---------------------------------------------------------------------------
def _documents(case):
    """Where the packed documents start and end."""
    rng = random.Random(case["docs"] * 65537 + case["Sq"])
    return [0] + sorted(rng.sample(range(1, case["Sq"]), case["docs"] - 1)) + [case["Sq"]]


def _prefixes(case):
    rng = random.Random(case["Sq"])
    return [rng.randint(0, case["Sq"] // 2) for _ in range(case["B"])]


def _lengths(case):
    """Keys in use: the first sequence has a full cache, the others down to a quarter."""
    rng = random.Random(case["Sk"] + case["B"])
    lo = max(case["Sq"], case["Sk"] // 4)
    return [case["Sk"]] + [rng.randint(lo, case["Sk"]) for _ in range(case["B"] - 1)]


def _intervals(case):
    """(lo, hi, p): the keys [lo, hi) that query i of batch b sees, and the query's
    place among the keys; int64 [B, Sq] on the CPU."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    i = torch.arange(Sq).repeat(B, 1)
    p = i + Sk - Sq
    lo, hi = torch.zeros_like(i), torch.full_like(i, Sk)
    if case["mask"] == "documents":
        cut = torch.tensor(_documents(case))
        d = torch.searchsorted(cut, i, right=True) - 1
        lo, hi = cut[d], cut[d + 1]
    elif case["mask"] == "prefix":
        hi = torch.maximum(p + 1, torch.tensor(_prefixes(case))[:, None])
    elif case["mask"] == "lengths":
        p = i + (torch.tensor(_lengths(case)) - Sq)[:, None]
    if case["causal"]:
        hi = torch.minimum(hi, p + 1)
    return lo, hi, p


def work(case):
    B, Dh = case["B"], case["Dh"]
    if case["op"] == "attention":
        lo, hi, _ = _intervals(case)
        pairs = int((hi.clamp(0, case["Sk"]) - lo).clamp_min(0).sum()) * case["H"]
        keys = sum(_lengths(case)) if case["mask"] == "lengths" else B * case["Sk"]
        b = 2 * Dh * (2 * B * case["Sq"] * case["H"] + 2 * keys * case["Hkv"])
        return {"bytes": b, "flops": 4.0 * Dh * pairs}
    heads = case["H"] + case.get("Hkv", 0)
    n = B * case["S"]
    return {"bytes": n * heads * Dh * 4 + n * case["axes"] * 4, "flops": n * heads * Dh * (7.0 if "Hkv" in case else 3.0)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _sections(case):
    """Pairs of each axis: the first axis (time) the fewest."""
    P, A = case["Dh"] // 2, case["axes"]
    if A == 1:
        return [P]
    if A == 2:
        return [P // 2, P - P // 2]
    a = P // 8
    return [a, (P - a) // 2, P - a - (P - a) // 2]


def _frequencies(sections):
    """10000^(-i / n) for pair i of an axis of n pairs, as a model keeps them."""
    f = [10000.0 ** (-i / n) for n in sections for i in range(n)]
    return torch.tensor(f, dtype=torch.float64, device=DEV)


def _positions(case):
    """Places of the tokens on each axis: a line, an image's rows and columns, or a
    video's frames, rows and columns, behind `far` others on the first axis."""
    n, A = torch.arange(case["S"]), case["axes"]
    if A == 1:
        p = n[:, None]
    else:
        w = max(1, math.isqrt(case["S"] if A == 2 else max(1, case["S"] // 8)))
        p = torch.stack([n // w, n % w] if A == 2 else [n // (w * w), n // w % w, n % w], 1)
    p = p + torch.tensor([case["far"]] + [0] * (A - 1))
    return p.to(torch.int32).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]
    B, H, Dh = case["B"], case["H"], case["Dh"]
    Hkv = case.get("Hkv", 0)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = {"case": case, "dt": dt}
    if case["op"] != "attention":
        S = case["S"]
        # queries, keys and values side by side, as one projection writes them
        heads = H + 2 * Hkv if Hkv else 3 * H
        spread = torch.exp(0.5 * rnd(heads, Dh))
        x = (rnd(B, S, heads, Dh) * spread).to(dt)
        s["q"] = x[:, :, :H]
        s["q_out"] = torch.empty(B, S, H, Dh, dtype=dt, device=DEV)
        s["pos"], s["sections"] = _positions(case), _sections(case)
        s["freqs"] = _frequencies(s["sections"])
        if Hkv:
            s["k"] = x[:, :, H:H + Hkv]
            s["k_out"] = torch.empty(B, S, Hkv, Dh, dtype=dt, device=DEV)
            s["qg"], s["kg"] = (1.0 + 0.2 * rnd(Dh)).to(dt), (1.0 + 0.2 * rnd(Dh)).to(dt)
        return s
    Sq, Sk = case["Sq"], case["Sk"]
    # normalised queries and keys: scores of a spread of 2 to 3 after the scale
    s["q"] = (1.6 * rnd(B, Sq, H, Dh)).to(dt)
    s["k"] = (1.6 * rnd(B, Sk, Hkv, Dh)).to(dt)
    s["v"] = rnd(B, Sk, Hkv, Dh).to(dt)
    s["out"] = torch.empty(B, Sq, H, Dh, dtype=dt, device=DEV)
    lo, hi, p = _intervals({**case, "causal": False})
    s["range"] = s["q_pos"] = s["slopes"] = s["table"] = None
    if case["mask"] in ("documents", "prefix"):
        s["range"] = torch.stack([lo, hi], 2).to(torch.int32).to(DEV)
    if case["mask"] == "lengths":
        s["q_pos"] = p.to(torch.int32).to(DEV)
    if case["bias"] == "slope":
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV, dtype=torch.float32) / H)
    elif case["bias"] == "table":
        s["table"] = rnd(H, 2 * 128 + 1)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_turn(s, x, gamma):
    """Norm (where there is a gamma) and rotation in fp32, the angles in fp64."""
    c = s["case"]
    v = x.float()
    if gamma is not None:
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * gamma.float()
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=DEV), torch.tensor(s["sections"], device=DEV),
                                   output_size=sum(s["sections"]))
    angle = s["pos"].double()[:, axis] * s["freqs"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if c["interleaved"]:
        a, b = v[..., 0::2], v[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(s["dt"])
    a, b = v.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(s["dt"])


def _plain_attention(s):
    c = s["case"]
    B, Sq, Sk, H, Hkv, Dh = (c[n] for n in ("B", "Sq", "Sk", "H", "Hkv", "Dh"))
    G = H // Hkv
    # [B * Hkv, G * Sq, Dh] and [B * Hkv, Dh, Sk]
    q = s["q"].float().view(B, Sq, Hkv, G, Dh).permute(0, 2, 3, 1, 4).reshape(B * Hkv, G * Sq, Dh)
    kt = s["k"].float().permute(0, 2, 3, 1).reshape(B * Hkv, Dh, Sk)
    v = s["v"].float().transpose(1, 2).reshape(B * Hkv, Sk, Dh)
    j = torch.arange(Sk, device=DEV, dtype=torch.int32)
    p = s["q_pos"] if s["q_pos"] is not None else torch.arange(Sk - Sq, Sk, device=DEV, dtype=torch.int32).expand(B, Sq)
    away = j - p[:, :, None]  # [B, Sq, Sk]
    seen = None
    if s["range"] is not None:
        seen = (j >= s["range"][:, :, :1]) & (j < s["range"][:, :, 1:])
    if c["causal"]:
        seen = away <= 0 if seen is None else seen & (away <= 0)
    parts = []
    step = max(1, (1 << 28) // (G * Sq * Sk))
    for at in range(0, B * Hkv, step):
        n = min(step, B * Hkv - at)
        z = torch.arange(at, at + n, device=DEV)
        x = torch.matmul(q[at:at + n], kt[at:at + n]).view(n, G, Sq, Sk)
        x *= Dh ** -0.5
        if c["cap"]:
            x = c["cap"] * torch.tanh(x / c["cap"])
        h = (z % Hkv)[:, None] * G + torch.arange(G, device=DEV)  # [n, G]
        if s["slopes"] is not None:
            x -= s["slopes"][h][:, :, None, None] * away[z // Hkv][:, None].abs()
        if s["table"] is not None:
            R = s["table"].shape[1] // 2
            x += s["table"][h[:, :, None, None], (away[z // Hkv][:, None].clamp(-R, R) + R)]
        if seen is not None:
            x = torch.where(seen[z // Hkv][:, None], x, -math.inf)
        top = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = e.sum(-1, keepdim=True)
        e /= torch.where(total > 0, total, torch.ones_like(total))
        parts.append(torch.matmul(e.view(n, G * Sq, Sk), v[at:at + n]))
    o = torch.cat(parts) if len(parts) > 1 else parts[0]
    return o.view(B, Hkv, G, Sq, Dh).permute(0, 3, 1, 2, 4).reshape(B, Sq, H, Dh).to(s["dt"])


def _plain(s):
    op = s["case"]["op"]
    if op == "attention":
        return {"o": _plain_attention(s)}
    if op == "rotary":
        return {"q": _plain_turn(s, s["q"], None)}
    return {"q": _plain_turn(s, s["q"], s["qg"]), "k": _plain_turn(s, s["k"], s["kg"])}


def _own(s):
    from dollama_amd import ops

    c = s["case"]
    if c["op"] == "attention":
        return {"o": ops.attention_masked(s["q"], s["k"], s["v"], key_range=s["range"], q_pos=s["q_pos"],
                                          causal=c["causal"], cap=c["cap"], slopes=s["slopes"], rel_bias=s["table"],
                                          out=s["out"])}
    if c["op"] == "rotary":
        return {"q": ops.rotary_axes(s["q"], s["pos"], s["freqs"], s["sections"], interleaved=c["interleaved"],
                                     out=s["q_out"])}
    q, k = ops.qk_norm_rotary(s["q"], s["k"], s["qg"], s["kg"], s["pos"], s["freqs"], s["sections"],
                              interleaved=c["interleaved"], eps=EPS, q_out=s["q_out"], k_out=s["k_out"])
    return {"q": q, "k": k}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the result in 64 bits
# ---------------------------------------------------------------------------
def _turned(s, x, gamma):
    """Every pair as a complex number times e^(i angle)."""
    c = s["case"]
    x = x.to(torch.float64)
    if gamma is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / c["Dh"] + EPS).sqrt() * gamma.to(torch.float64)
    P = c["Dh"] // 2
    order = torch.arange(c["Dh"], device=DEV)
    order = order.view(P, 2).t().reshape(-1) if c["interleaved"] else order  # first parts, then second parts
    x = x[..., order]
    turn = []
    at = 0
    for a, n in enumerate(s["sections"]):
        turn.append(torch.outer(s["pos"][:, a].to(torch.float64), s["freqs"][at:at + n]))
        at += n
    w = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.cat(turn, 1))
    z = torch.complex(x[..., :P].contiguous(), x[..., P:].contiguous()) * w[:, None]
    y = torch.empty_like(x)
    y[..., order] = torch.cat([z.real, z.imag], -1)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return {"q": _turned(s, s["q"], None)}
    if case["op"] == "qk_norm":
        return {"q": _turned(s, s["q"], s["qg"]), "k": _turned(s, s["k"], s["kg"])}
    f64 = torch.float64
    B, Sq, Sk, H, Hkv, Dh = (case[n] for n in ("B", "Sq", "Sk", "H", "Hkv", "Dh"))
    lo, hi, p = (t.to(DEV) for t in _intervals(case))
    o = torch.zeros(B, Sq, H, Dh, dtype=f64, device=DEV)
    j = torch.arange(Sk, device=DEV)
    rows = max(1, min(Sq, (1 << 27) // Sk))
    for b in range(B):
        for h in range(H):
            kt = s["k"][b, :, h // (H // Hkv)].to(f64).t().contiguous()
            v = s["v"][b, :, h // (H // Hkv)].to(f64).contiguous()
            for r in range(0, Sq, rows):
                e = slice(r, min(Sq, r + rows))
                x = s["q"][b, e, h].to(f64) @ kt / math.sqrt(Dh)
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                d = j[None, :] - p[b, e, None]
                if s["slopes"] is not None:
                    x = x - s["slopes"][h].to(f64) * d.abs()
                if s["table"] is not None:
                    R = s["table"].shape[1] // 2
                    x = x + s["table"][h].to(f64)[torch.clip(d, -R, R) + R]
                hidden = (j[None, :] < lo[b, e, None]) | (j[None, :] >= hi[b, e, None])
                x = x.masked_fill(hidden, -math.inf)
                w = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
                o[b, e, h] = w.masked_fill(hidden, 0.0) @ v
    return {"o": o}
