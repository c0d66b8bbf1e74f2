"""The dropout bits and the group norm in 64 bits, from their definitions, for
the tests of the feature-map operators (numpy and torch on the CPU)."""
from __future__ import annotations

import numpy as np
import torch

HI, LO, CH_HI, CH_LO = 0x44500000, 0x44510000, 0x44520000, 0x44530000


def philox(c0, c1, c2, c3, seed: int):
    """Philox4x32-10 on uint64 arrays of 32-bit counter words; four words."""
    m = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, np.uint64) for v in np.broadcast_arrays(c0, c1, c2, c3)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def halves(q, elem: int, stream: int, seed: int) -> np.ndarray:
    """The eight 16-bit halves of the blocks q of an element, last axis 8."""
    q = np.asarray(q, np.uint64)
    w = philox(q & np.uint64(0xFFFFFFFF), elem & 0xFFFFFFFF, elem >> 32,
               np.uint64(stream) | (q >> np.uint64(32)), seed)
    return np.stack([h for v in w for h in (v & np.uint64(0xFFFF), v >> np.uint64(16))], -1)


def numbers(B, C, S, seed, elem_offset=0, channelwise=False) -> np.ndarray:
    """Every voxel's (or channel's) 32-bit number, (B, C, S) or (B, C, 1)."""
    out = []
    for b in range(B):
        if channelwise:
            q, streams = np.arange((C + 7) // 8), (CH_HI, CH_LO)
        else:
            n = (S + 7) // 8
            q, streams = np.arange(C)[:, None] * n + np.arange(n), (HI, LO)
        hi, lo = (halves(q, elem_offset + b, s, seed) for s in streams)
        r = (hi << np.uint64(16)) | lo
        out.append(r.reshape(-1)[:C].reshape(C, 1) if channelwise
                   else r.reshape(C, -1)[:, :S])
    return np.stack(out)


def factor(shape, p, seed, elem_offset=0, channelwise=False, rescale=True, mask=None):
    """What dropout multiplies each value with, float64 (dropped: 0)."""
    B, C = shape[:2]
    S = int(np.prod(shape[2:]))
    rate = np.broadcast_to(np.asarray(p, np.float32), (B,)).astype(np.float64)
    rate = np.clip(np.where(np.isnan(rate), 0.0, rate), 0.0, 1.0)
    r = numbers(B, C, S, seed, elem_offset, channelwise).astype(np.float64)
    keep = r >= np.ceil(rate * 2.0**32)[:, None, None]
    scale = np.where(rate < 1, 1 / np.where(rate < 1, 1 - rate, 1), 0.0) if rescale else np.ones(B)
    f = np.where(keep, scale[:, None, None], 0.0)
    if mask is not None:
        f = np.where(np.asarray(mask, bool)[:, None, None], f, 1.0)
    return torch.from_numpy(np.broadcast_to(f, (B, C, S)).reshape(shape).copy())


def activation(z: torch.Tensor, act, slope=0.01) -> torch.Tensor:
    if act in (None, "none"):
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "leaky_relu":
        return torch.where(z > 0, z, slope * z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z * 0.5 * torch.erfc(-z / np.sqrt(2.0))


def norm(x, groups, w=None, b=None, eps=1e-5, act=None, slope=0.01, f=None):
    """(out, z) in float64, differentiable; f: dropout's factor."""
    B, C = x.shape[:2]
    r = x.reshape(B, groups, -1)
    m = r.mean(-1, keepdim=True)
    v = ((r - m) ** 2).mean(-1, keepdim=True)
    z = ((r - m) / torch.sqrt(v + eps)).reshape(x.shape)
    per_c = (1, C) + (1,) * (x.dim() - 2)
    if w is not None:
        z = z * w.reshape(per_c)
    if b is not None:
        z = z + b.reshape(per_c)
    y = activation(z, act, slope)
    return (y if f is None else y * f), z
