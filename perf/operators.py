"""The 8-bit integer path of the transformer linears, as its speed is measured.

``listed()`` holds the fixed cases, ``draw(rng)`` makes further ones of the same
ranges, ``prepare`` / ``run`` / ``work`` / ``exact`` say for a case what a program
holds beforehand, one pass, what the pass cannot do without, and the result in
64 bits.  ``own`` selects what ``run`` computes with: the package's operators, or
their definitions in elementary torch operations.

The operators, over rows of K values:

- ``quantize`` : q = round(127 x / max|x|), scale = max|x| / 127 per row, and back
- ``rms_norm`` : h = x + residual, y = h / rms(h) * gamma, as 8-bit rows of y
- ``layer_norm``: y = LayerNorm(h) * gamma + beta, as 8-bit rows of y
- ``linear``   : act((xq @ wq.T) * sx * sw + bias) + residual, one scale for each
  row of xq (token) and of wq (output channel)

Rounding is to the nearest integer, halves to the even one.  Sizes are those of
the SDXL transformer blocks (640 / 1280 channels, 4096 / 1024 / 77 tokens, two
guidance halves, the 4x feed-forward) and generic ones for single tokens.
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5


def listed():
    return [
        # one token's feed-forward activations on their way into an 8-bit
        # product: the smallest call, where latency is everything
        {"name": "quantize_1x2560", "op": "quantize", "M": 1, "K": 2560, "f32": False},
        # the hidden rows of a feed-forward layer before its second projection
        {"name": "quantize_2048x5120", "op": "quantize", "M": 2048, "K": 5120, "f32": False},
        # the norm before a layer's projection while one token is served
        {"name": "rms_norm_1x4096", "op": "rms_norm", "M": 1, "K": 4096, "f32": False, "residual": True},
        # the same over all tokens of a guided step, the residual stream in fp32
        {"name": "rms_norm_8192x1280_f32", "op": "rms_norm", "M": 8192, "K": 1280, "f32": True, "residual": True},
        # a transformer block's first norm at the level with the most tokens
        {"name": "layer_norm_8192x640", "op": "layer_norm", "M": 8192, "K": 640, "f32": False, "residual": False},
        # an odd token count and width, whose rows start at no vector boundary
        {"name": "layer_norm_975x1283", "op": "layer_norm", "M": 975, "K": 1283, "f32": False, "residual": True},
        # one token through a square projection: the weight is read once
        {"name": "linear_1x4096x4096", "op": "linear", "M": 1, "N": 4096, "K": 4096, "act": "none", "bias": False,
         "residual": False, "f32": False},
        # a small batch of tokens through a feed-forward projection
        {"name": "linear_13x10240x2560", "op": "linear", "M": 13, "N": 10240, "K": 2560, "act": "silu", "bias": True,
         "residual": False, "f32": False},
        # key / value projection of two prompts of 77 tokens
        {"name": "linear_154x2560x2048", "op": "linear", "M": 154, "N": 2560, "K": 2048, "act": "none", "bias": True,
         "residual": False, "f32": False},
        # odd in every dimension, results added to an fp32 stream
        {"name": "linear_1975x1283x1003_f32", "op": "linear", "M": 1975, "N": 1283, "K": 1003, "act": "none",
         "bias": True, "residual": True, "f32": True},
        # the gated projection of a feed-forward layer, 1024 tokens
        {"name": "linear_2048x10240x1280_geglu", "op": "linear", "M": 2048, "N": 10240, "K": 1280, "act": "geglu",
         "bias": True, "residual": False, "f32": False},
        # a product large enough that only the matrix rate counts
        {"name": "linear_8192x8192x8192", "op": "linear", "M": 8192, "N": 8192, "K": 8192, "act": "none",
         "bias": True, "residual": True, "f32": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "rms_norm", "layer_norm", "linear", "linear", "linear"])
    if op != "linear":
        K = _log(rng, 32, 8192)
        if rng.random() < 0.6:  # widths are multiples of 16 more often than not
            K = -(-K // 16) * 16
        M = _log(rng, 1, min(8192, (1 << 24) // K))
        case = {"op": op, "M": M, "K": K, "f32": rng.random() < 0.3}
        if op != "quantize":
            case["residual"] = rng.random() < 0.6
        return case
    M, N, K = _log(rng, 1, 8192), _log(rng, 16, 12000), _log(rng, 64, 8192)
    if rng.random() < 0.6:
        N, K = -(-N // 16) * 16, -(-K // 16) * 16
    act = rng.choice(["none", "none", "silu", "gelu", "geglu"])
    if act == "geglu":
        N = -(-N // 16) * 16
    return {"op": op, "M": M, "N": N, "K": K, "act": act, "bias": rng.random() < 0.6,
            "residual": rng.random() < 0.5, "f32": act != "geglu" and rng.random() < 0.3}


def work(case):
    M, K = case["M"], case["K"]
    e = 4 if case["f32"] else 2
    if case["op"] == "linear":
        N = case["N"]
        cols = N // 2 if case["act"] == "geglu" else N
        b = M * K + N * K + 4 * (M + N) + M * cols * e
        b += 2 * N if case["bias"] else 0
        b += M * cols * e if case["residual"] else 0
        return {"bytes": b, "flops": 2.0 * M * N * K}
    # x in, the 8-bit values and the fp16 values they stand for out, scales
    b = M * K * (e + 1 + 2) + 4 * M
    if case["op"] != "quantize":
        b += 2 * K * (2 if case["op"] == "layer_norm" else 1)
        b += 2 * M * K * e if case["residual"] else 0  # residual in, new stream out
    return {"bytes": b, "flops": 10.0 * M * K}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(g, M, K):
    """Rows as a transformer's norms and projections meet them: channels of
    unequal spread, a few of them far larger than the rest."""
    spread = torch.exp(0.5 * torch.randn(K, generator=g, device=DEV))
    big = torch.rand(K, generator=g, device=DEV) < 0.004
    return torch.randn(M, K, generator=g, device=DEV) * torch.where(big, 12.0 * spread, spread)


def _int8_rows(v):
    """8-bit rows [M, K] at a row stride of a multiple of 16 bytes, and scales."""
    M, K = v.shape
    s = v.abs().amax(1) / 127.0
    q = torch.zeros(M, -(-K // 16) * 16, dtype=torch.int8, device=DEV)
    q[:, :K] = torch.round(v / s.clamp_min(1e-30)[:, None]).clamp_(-127, 127).to(torch.int8)
    return q[:, :K], s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    M, K = case["M"], case["K"]
    dt = torch.float32 if case["f32"] else torch.float16
    s = {"op": case["op"], "f32": case["f32"], "act": case.get("act")}
    if case["op"] == "linear":
        N = case["N"]
        cols = N // 2 if case["act"] == "geglu" else N
        s["xq"], s["sx"] = _int8_rows(_activations(g, M, K))
        s["wq"], s["sw"] = _int8_rows(torch.randn(N, K, generator=g, device=DEV) * (2.0 / math.sqrt(K)))
        s["bias"] = torch.randn(N, generator=g, device=DEV).half() if case["bias"] else None
        s["res"] = torch.randn(M, cols, generator=g, device=DEV).to(dt) if case["residual"] else None
        s["out"] = torch.empty(M, cols, dtype=dt, device=DEV)
        return s
    s["x"] = _activations(g, M, K).to(dt)
    s["q"] = torch.empty(M, -(-K // 16) * 16, dtype=torch.int8, device=DEV)[:, :K]
    s["scale"] = torch.empty(M, dtype=torch.float32, device=DEV)
    s["y"] = torch.empty(M, K, dtype=torch.float16, device=DEV)
    s["res"] = s["h"] = None
    if case["op"] != "quantize":
        s["gamma"] = (1.0 + 0.3 * torch.randn(K, generator=g, device=DEV)).half()
        if case["op"] == "layer_norm":
            s["beta"] = (0.2 * torch.randn(K, generator=g, device=DEV)).half()
        if case["residual"]:
            s["res"] = torch.randn(M, K, generator=g, device=DEV).to(dt)
            s["h"] = torch.empty(M, K, dtype=dt, device=DEV)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_rows(v):
    """8-bit rows of v (fp32 or fp64 values) as the fp16 values they stand for,
    and the scales; the quotients in 64 bits, since they are rounded to whole
    numbers."""
    v = v.double()
    top = v.abs().amax(1, keepdim=True)
    q = torch.round(v * 127.0 / torch.where(top > 0, top, torch.ones_like(top)))
    scale = (top / 127.0).float()
    return (q * scale.double()).half(), scale[:, 0]


def _plain(s):
    if s["op"] == "linear":
        y = s["xq"].float() @ s["wq"].float().t()
        y = y * s["sx"][:, None] * s["sw"]
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if s["act"] == "silu":
            y = y / (1.0 + torch.exp(-y))
        elif s["act"] == "gelu":
            y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
        elif s["act"] == "geglu":  # columns in groups of 4 values, 4 gates
            v, t = y.view(y.shape[0], -1, 2, 4).unbind(2)
            y = (v * 0.5 * t * (1.0 + torch.erf(t * math.sqrt(0.5)))).reshape(y.shape[0], -1)
        if s["res"] is not None:
            y = y + s["res"].float()
        return {"y": y if s["f32"] else y.half()}
    h = s["x"]
    if s["op"] == "quantize":
        y, scale = _plain_rows(h)
        return {"y": y, "scale": scale}
    if s["res"] is not None:
        h = (h.float() + s["res"].float()).to(h.dtype)
    v = h.double()  # the values are rounded to whole numbers in the end
    if s["op"] == "layer_norm":
        v = v - v.mean(1, keepdim=True)
    n = v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * s["gamma"].double()
    if s["op"] == "layer_norm":
        n = n + s["beta"].double()
    y, scale = _plain_rows(n)
    return {"y": y, "scale": scale} if s["res"] is None else {"y": y, "scale": scale, "h": h}


def _own(s):
    from dollama_amd import ops

    if s["op"] == "linear":
        act = {"none": ops.ACT_NONE, "silu": ops.ACT_SILU, "gelu": ops.ACT_GELU, "geglu": ops.ACT_GEGLU}[s["act"]]
        return {"y": ops.linear_q8(s["xq"], s["sx"], s["wq"], s["sw"], bias=s["bias"], residual=s["res"], act=act,
                                   out=s["out"])}
    if s["op"] == "quantize":
        ops.quantize_rows(s["x"], out=s["q"], scale=s["scale"])
    elif s["op"] == "rms_norm":
        ops.rms_norm_q8(s["x"], s["gamma"], residual=s["res"], eps=EPS, sum_out=s["h"], out=s["q"], scale=s["scale"])
    else:
        ops.layer_norm_q8(s["x"], s["gamma"], s["beta"], residual=s["res"], eps=EPS, sum_out=s["h"], out=s["q"],
                          scale=s["scale"])
    y = ops.dequantize_rows(s["q"], s["scale"], out=s["y"])
    r = {"y": y, "scale": s["scale"]}
    return r if s["res"] is None else {**r, "h": s["h"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the result in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    M, K = case["M"], case["K"]
    if case["op"] == "linear":
        acc = torch.matmul(s["xq"].to(f64), s["wq"].to(f64).t().contiguous())
        acc *= torch.outer(s["sx"].to(f64), s["sw"].to(f64))
        if s["bias"] is not None:
            acc += s["bias"].to(f64)
        ndtr = torch.special.ndtr  # gelu(t) = t Phi(t)
        if case["act"] == "silu":
            acc = acc * torch.sigmoid(acc)
        elif case["act"] == "gelu":
            acc = acc * ndtr(acc)
        elif case["act"] == "geglu":
            col = torch.arange(case["N"] // 2, device=DEV)
            col = col // 4 * 8 + col % 4
            t = acc[:, col + 4]
            acc = acc[:, col] * (t * ndtr(t))
        if s["res"] is not None:
            acc += s["res"].to(f64)
        return {"y": acc}
    out = {}
    v = s["x"].to(f64)
    if s["res"] is not None:
        out["h"] = v + s["res"].to(f64)
        v = out["h"].to(s["x"].dtype).to(f64)  # the stream as it is stored is what the norm reads
    if case["op"] == "rms_norm":
        v = v * s["gamma"].to(f64) / (v.pow(2).sum(1, keepdim=True) / K + EPS).sqrt()
    elif case["op"] == "layer_norm":
        d = v - v.sum(1, keepdim=True) / K
        v = d / (d.pow(2).sum(1, keepdim=True) / K + EPS).sqrt() * s["gamma"].to(f64) + s["beta"].to(f64)
    top = v.abs().max(dim=1, keepdim=True).values
    out["y"] = torch.round(127 * v / top) * (top / 127)
    out["scale"] = top.reshape(M) / 127
    return out
