"""The network-side operators of batchaug_b200, as cases that can be timed: group norm with an
activation, dropout from a counter-based generator, and the two as one call (normalise,
activate, drop), on (B, C, H, W, D) tensors in channels-last or contiguous memory.

``run`` computes them in elementary torch operations while ``own`` is false, and through
``batchaug_b200.ops`` where it is true.  ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# Stream words of the dropout bits (the counter's high word): the high and the low 16 bits of a
# voxel's 32-bit number, and of a channel's.
_VOXEL_HI, _VOXEL_LO = 0x44500000, 0x44510000
_CHANNEL_HI, _CHANNEL_LO = 0x44520000, 0x44530000


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _norm(name, shape, dtype, layout, groups, act, train, affine="f32", p=0.0):
    b, c, h, w, d = shape
    return {"name": name, "op": "norm", "B": b, "C": c, "H": h, "W": w, "D": d, "dtype": dtype,
            "layout": layout, "groups": groups, "act": act, "affine": affine, "p": p,
            "train": train}


def _drop(name, shape, dtype, layout, p, train, channelwise=False, per_element=False):
    b, c, h, w, d = shape
    return {"name": name, "op": "dropout", "B": b, "C": c, "H": h, "W": w, "D": d, "dtype": dtype,
            "layout": layout, "p": p, "channelwise": channelwise, "per_element": per_element,
            "train": train}


def listed():
    return [
        # the z-score of an augmented batch of 4-channel volumes, each channel on its own
        _norm("norm-volumes", (8, 4, 128, 128, 128), "f32", "first", 4, "none", False, "none"),
        # the deepest level of a 3-D U-Net at inference: latency
        _norm("norm-bottleneck", (2, 256, 8, 8, 8), "bf16", "last", 32, "silu", False),
        # a middle level of the same network at inference, rectified
        _norm("norm-middle", (2, 64, 48, 48, 48), "bf16", "last", 16, "relu", False),
        # training steps through one normalisation: a middle level, the full-resolution level
        _norm("norm-train-middle", (2, 64, 64, 64, 64), "bf16", "last", 8, "silu", True),
        _norm("norm-train-full", (2, 32, 128, 128, 128), "bf16", "last", 8, "silu", True),
        # an odd crop and a channel count that 16 bytes do not divide evenly, in single precision
        _norm("norm-train-odd", (3, 20, 45, 37, 29), "f32", "last", 5, "gelu", True),
        # a network kept in the contiguous layout
        _norm("norm-train-first", (2, 32, 64, 64, 64), "f32", "first", 8, "silu", True),
        # normalise, activate, drop: the block of a network trained with dropout
        _norm("block-train", (2, 48, 96, 96, 96), "bf16", "last", 8, "gelu", True, "f32", 0.1),
        # voxel dropout as an augmentation: a rate for each element, some elements left alone
        _drop("dropout-volumes", (16, 4, 128, 128, 128), "bf16", "first", 0.3, False,
              per_element=True),
        # a small feature map: latency
        _drop("dropout-small", (2, 16, 16, 16, 16), "bf16", "last", 0.2, False),
        # an odd volume (no vector width divides it)
        _drop("dropout-odd", (2, 3, 91, 109, 91), "f32", "first", 0.5, False),
        # a feature map, forward and backward
        _drop("dropout-train", (2, 64, 64, 64, 64), "bf16", "last", 0.1, True),
    ]


def _size(rng, lo, hi):
    """A whole number, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm", "dropout", "dropout"])
    train = rng.random() < 0.5
    layout = rng.choice(["last", "last", "first"])
    while True:
        b = rng.choice([1, 2, 2, 3, 4, 8])
        c = rng.choice([1, 2, 3, 4, 8, 12, 16, 20, 24, 32, 33, 48, 64, 96, 128, 256, 320, 512])
        h, w, d = (_size(rng, 4, 144) for _ in range(3))
        if rng.random() < 0.3:  # the usual crops are multiples of 8
            h, w, d = (max(8, v // 8 * 8) for v in (h, w, d))
        # neither below the bottleneck's size by much nor above the full-resolution level's
        if 1 << 14 <= b * c * h * w * d <= 1 << 26:
            break
    dtype = rng.choice(["bf16", "bf16", "f32"])
    p = rng.choice([0.05, 0.1, 0.2, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)])
    if op == "dropout":
        case = _drop("", (b, c, h, w, d), dtype, layout, p, train,
                     channelwise=rng.random() < 0.2, per_element=rng.random() < 0.3)
    else:
        groups = rng.choice([g for g in (1, 2, 4, 5, 8, 11, 16, 32, c) if c % g == 0])
        # a rectifier's gradient jumps at zero, where a rounding decides it: forward only
        act = rng.choice(["none", "silu", "gelu"] + ([] if train else ["relu", "leaky_relu"]))
        case = _norm("", (b, c, h, w, d), dtype, layout, groups, act, train,
                     rng.choice(["f32", "f32", "x", "none"]), rng.choice([0.0, 0.0, p]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# State
# ---------------------------------------------------------------------------

def _laid_out(x, layout):
    return x.contiguous(memory_format=torch.channels_last_3d) if layout == "last" else x


def prepare(case, seed):
    """Features with a mean and a scale of their own in each channel, the gradient that comes
    back to them, weights near one, and the seed of the pass's dropout bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = tuple(case[k] for k in "BCHWD")
    dtype = _DTYPES[case["dtype"]]
    C = shape[1]

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    scale = torch.exp(0.5 * randn(1, C, 1, 1, 1))
    x = _laid_out((randn(*shape) * scale + randn(1, C, 1, 1, 1)).to(dtype), case["layout"])
    state = {"case": case, "x": x.requires_grad_(case["train"]),
             "seed": (seed * 0x9E3779B97F4A7C15 + 0x1234567) & (2**63 - 1)}
    if case["train"]:
        state["dy"] = _laid_out(randn(*shape).to(dtype), case["layout"])
    if case["op"] == "norm":
        state["w"] = state["b"] = None
        if case["affine"] != "none":
            t = dtype if case["affine"] == "x" else torch.float32
            state["w"] = (1.0 + 0.2 * randn(C)).to(t).requires_grad_(case["train"])
            state["b"] = (0.2 * randn(C)).to(t).requires_grad_(case["train"])
        state["p"], state["mask"] = case["p"], None
    elif case["per_element"]:
        B = shape[0]
        state["p"] = torch.rand(B, generator=g, device="cuda") * case["p"]
        state["mask"] = torch.rand(B, generator=g, device="cuda") < 0.75
    else:
        state["p"], state["mask"] = case["p"], None
    return state


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return _plain_norm(state, case) if case["op"] == "norm" else _plain_dropout(state, case)


def _own(state, case):
    from batchaug_b200 import ops

    x = state["x"]
    if case["op"] == "norm":
        w, b = state["w"], state["b"]
        y = ops.group_norm(x, case["groups"], w, b, activation=case["act"], p=state["p"],
                           seed=state["seed"])
        leaves = [x] if w is None else [x, w, b]
    else:
        y = ops.dropout(x, state["p"], state["seed"], mask=state["mask"],
                        channelwise=case["channelwise"])
        leaves = [x]
    if not case["train"]:
        return y
    return [y] + list(torch.autograd.grad(y, leaves, state["dy"]))


# ---------------------------------------------------------------------------
# Plain form
# ---------------------------------------------------------------------------

def _philox(q, elem, stream, seed):
    """Philox4x32-10 of the counters (q, elem, 0, stream | q >> 32) under the key ``seed``: four
    words in [0, 2^32) as int64 tensors of the shape that q and elem broadcast to."""
    low = 0xFFFFFFFF
    c0, c1 = torch.broadcast_tensors(q & low, elem)
    c2, c3 = torch.zeros_like(c0), (q >> 32 | stream).expand_as(c0)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        # the 64-bit products wrap in int64; their halves are read as bits
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return c0, c1, c2, c3


def _halves(words):
    """The eight 16-bit halves of four words, the low half of each first, in a new last axis."""
    return torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], -1)


def _keep(shape, p, seed, channelwise, device):
    """Which values stay: a voxel's (or a channel's) 32-bit number is at least p 2^32."""
    B, C, S = shape[0], shape[1], shape[2] * shape[3] * shape[4]
    elem = torch.arange(B, device=device).view(B, 1, 1)
    n = 1 if channelwise else (S + 7) // 8
    if channelwise:
        q = torch.arange((C + 7) // 8, device=device).view(1, 1, -1)
        streams = _CHANNEL_HI, _CHANNEL_LO
    else:
        q = (torch.arange(C, device=device).view(C, 1) * n
             + torch.arange(n, device=device)).view(1, C, n)
        streams = _VOXEL_HI, _VOXEL_LO
    hi, lo = (_halves(_philox(q, elem, s, seed)) for s in streams)
    number = hi * 65536 + lo
    number = (number.view(B, -1)[:, :C].reshape(B, C, 1) if channelwise
              else number.view(B, C, n * 8)[:, :, :S])
    p = torch.as_tensor(p, dtype=torch.float32, device=device).reshape(-1, 1, 1)
    keep = number >= torch.ceil(p.double() * 2.0**32).to(torch.int64)
    return keep.view(B, C, *((1, 1, 1) if channelwise else shape[2:]))


def _scale(p, device):
    p = torch.as_tensor(p, dtype=torch.float32, device=device).reshape(-1, 1, 1, 1, 1)
    return torch.where(p < 1, 1 / (1 - p), torch.zeros_like(p))


def _plain_dropout(state, case):
    x, p, mask = state["x"].detach(), state["p"], state["mask"]
    keep = _keep(x.shape, p, state["seed"], case["channelwise"], x.device)
    factor = torch.where(keep, _scale(p, x.device), torch.zeros((), device=x.device))
    if mask is not None:
        factor = torch.where(mask.view(-1, 1, 1, 1, 1), factor, torch.ones_like(factor))
    y = (x.float() * factor).to(x.dtype)
    return [y, (state["dy"].float() * factor).to(x.dtype)] if case["train"] else y


def _act(z, act):
    """(act(z), act'(z))"""
    if act == "none":
        return z, torch.ones_like(z)
    if act in ("relu", "leaky_relu"):
        slope = torch.where(z > 0, 1.0, 0.01 if act == "leaky_relu" else 0.0)
        return z * slope, slope
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _plain_norm(state, case):
    x = state["x"].detach()
    B, C, G = x.shape[0], x.shape[1], case["groups"]
    shape, per_c = x.shape, (1, C, 1, 1, 1)
    w = torch.ones(C, device=x.device) if state["w"] is None else state["w"].detach().float()
    b = torch.zeros(C, device=x.device) if state["b"] is None else state["b"].detach().float()

    def grouped_mean(t):
        m = t.reshape(B, G, -1).mean(-1)
        return m.repeat_interleave(C // G, 1).view(B, C, 1, 1, 1)

    v = x.float()
    v = v - grouped_mean(v)
    r = 1 / torch.sqrt(grouped_mean(v * v) + 1e-5)
    xh = v * r
    y, slope = _act(xh * w.view(per_c) + b.view(per_c), case["act"])
    factor = None
    if case["p"] > 0:
        keep = _keep(shape, case["p"], state["seed"], False, x.device)
        factor = torch.where(keep, _scale(case["p"], x.device), torch.zeros((), device=x.device))
        y = y * factor
    y = y.to(x.dtype)
    if not case["train"]:
        return y
    dz = state["dy"].float() * slope
    if factor is not None:
        dz = dz * factor
    g = dz * w.view(per_c)
    dx = (r * (g - grouped_mean(g) - xh * grouped_mean(g * xh))).to(x.dtype)
    if state["w"] is None:
        return [y, dx]
    return [y, dx, (dz * xh).sum((0, 2, 3, 4)).to(state["w"].dtype),
            dz.sum((0, 2, 3, 4)).to(state["b"].dtype)]


# ---------------------------------------------------------------------------
# Work and the definition in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    """A forward pass reads x and writes y; a training pass of a norm also reads x and dy and
    writes dx, one of a dropout reads dy and writes dx."""
    n = case["B"] * case["C"] * case["H"] * case["W"] * case["D"]
    size = 4 if case["dtype"] == "f32" else 2
    train, norm = case["train"], case["op"] == "norm"
    passes = (5 if train else 2) if norm else (4 if train else 2)
    return {"bytes": passes * n * size, "flops": n * ((25 if train else 8) if norm else 2)}


def _mulhilo(a, m):
    """(high, low) 32 bits of a * m, through 16-bit limbs, nothing beyond 2^49."""
    t = (a & 0xFFFF) * m
    u = (a >> 16) * m + (t >> 16)
    return u >> 16, (u & 0xFFFF) << 16 | t & 0xFFFF


def _random_word(block, elem, stream, seed, lane):
    """16 bits, number ``lane`` of eight, of the generator's block for (block, elem, stream)."""
    x = [block % 2**32, elem, torch.zeros_like(block), block // 2**32 + stream]
    key = [seed % 2**32, seed // 2**32]
    for r in range(10):
        if r:
            key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
        h0, l0 = _mulhilo(x[0], 0xD2511F53)
        h1, l1 = _mulhilo(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ key[0], l1, h0 ^ x[3] ^ key[1], l0]
    word = torch.where(lane < 4, torch.where(lane < 2, x[0], x[1]),
                       torch.where(lane < 6, x[2], x[3]))
    return torch.where(lane % 2 == 0, word % 65536, word // 65536)


def _exact_factor(case, state):
    """What each value is multiplied with, one (element, channel) row of voxels at a time."""
    x = state["x"]
    B, C, S = x.shape[0], x.shape[1], x[0, 0].numel()
    rate = torch.as_tensor(state["p"], dtype=torch.float32, device=x.device).double().expand(B)
    factor = torch.ones(B, C, S, dtype=torch.float64, device=x.device)
    voxel = torch.arange(S, device=x.device)
    for e in range(B):
        if state["mask"] is not None and not bool(state["mask"][e]):
            continue
        for c in range(C):
            i = torch.full_like(voxel, c)[:1] if case.get("channelwise") else voxel
            block = i // 8 if case.get("channelwise") else i // 8 + c * ((S + 7) // 8)
            streams = ((_CHANNEL_HI, _CHANNEL_LO) if case.get("channelwise")
                       else (_VOXEL_HI, _VOXEL_LO))
            at = torch.full_like(block, e)
            u = sum(_random_word(block, at, s, state["seed"], i % 8) * k
                    for s, k in zip(streams, (65536, 1)))
            stays = u.double() / 2.0**32 >= rate[e]
            factor[e, c] = torch.where(stays, 1 / (1 - rate[e]), 0.0)
    return factor.view(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    drops = case["op"] == "dropout" or case["p"] > 0
    if drops and case["B"] * case["C"] > 2000:  # its rows take too long one by one
        return None
    x = state["x"].detach().double().contiguous().requires_grad_(case["train"])
    leaves = [x]
    y = x
    if case["op"] == "norm":
        rows = x.view(case["B"], case["groups"], -1)
        var, mean = torch.var_mean(rows, -1, correction=0, keepdim=True)
        y = ((rows - mean) / (var + 1e-5).sqrt()).view(x.shape)
        if state["w"] is not None:
            w, b = (state[k].detach().double().requires_grad_(case["train"]) for k in "wb")
            y = torch.einsum("bchwd,c->bchwd", y, w) + b[:, None, None, None]
            leaves += [w, b]
        act = case["act"]
        if act == "relu":
            y = y.clamp(min=0)
        elif act == "leaky_relu":
            y = torch.maximum(y, 0.01 * y)
        elif act == "silu":
            y = y * torch.sigmoid(y)
        elif act == "gelu":
            y = y * torch.special.ndtr(y)
    if drops:
        y = y * _exact_factor(case, state)
    if not case["train"]:
        return y
    return [y] + list(torch.autograd.grad(y, leaves, state["dy"].double()))
