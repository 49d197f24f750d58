"""The paged K/V cache from its definitions, in 64 bits (numpy): values found by
their address in the page format of include/chonk.h, blocks quantised, attention."""
from __future__ import annotations

import numpy as np

PAGE = 64
TYPES = ("f16", "q8", "q4")


def code_bytes(kv, hd):
    return PAGE * {"f16": 2 * hd, "q8": hd, "q4": hd // 2}[kv]


def part_bytes(kv, hd):
    return code_bytes(kv, hd) + (0 if kv == "f16" else PAGE * hd // 32 * 2)


def addresses(kv, hd, is_v, j):
    """Byte (and, for q4, shift) of every dim of position j in a head's part, and its scale's byte."""
    d = np.arange(hd)
    unit, i, p = (j // 32) * (hd // 32) + d // 32, d % 32, j % 32
    if is_v:
        g, lane, piece, e = (p % 16) // 4, i % 16, i // 16, p % 4 + 4 * (p // 16)
    else:
        g, lane, piece, e = i // 8, p % 16, p // 16, i % 8
    n = 16 * g + lane
    place = (p % 16) // 4 * 8 + p % 4 + 4 * (p // 16)
    scale = code_bytes(kv, hd) + 2 * (unit * 32 + place)
    if kv == "f16":
        return unit * 2048 + piece * 1024 + n * 16 + 2 * e, 0 * d, scale
    if kv == "q8":
        return unit * 1024 + n * 16 + piece * 8 + e, 0 * d, scale
    if is_v:
        return unit * 512 + n * 8 + e, 4 * piece + 0 * d, scale
    return unit * 512 + n * 8 + piece * 4 + e % 4, 4 * (e // 4), scale


def decode(kv, part, hd, is_v, j):
    """Values [hd] of position j in a head's part (uint8 array)."""
    at, shift, scale = addresses(kv, hd, is_v, j)

    def half(a):
        return np.stack([part[a], part[a + 1]], -1).astype(np.uint8).reshape(-1).view(np.float16).astype(np.float64)

    if kv == "f16":
        return half(at)
    c = part[at].astype(np.int64)
    c = c - 128 if kv == "q8" else ((c >> shift) & 15) - 8
    return c * half(scale)


def gather(kv, pages, table, kv_heads, hd, seq, positions):
    """K and V [n, kv_heads, hd] stored at these positions of a sequence."""
    pages = pages.reshape(len(pages), kv_heads, 2, part_bytes(kv, hd))
    out = np.empty((2, len(positions), kv_heads, hd))
    for x, pos in enumerate(positions):
        head = pages[table[seq, pos // PAGE]]
        for h in range(kv_heads):
            for w in (0, 1):
                out[w, x, h] = decode(kv, head[h, w], hd, w == 1, pos % PAGE)
    return out


def owned_bytes(kv, hd, j):
    """Mask over a head's (K, V) bytes of those that hold anything of position j."""
    m = np.zeros((2, part_bytes(kv, hd)), dtype=bool)
    for w in (0, 1):
        at, _, scale = addresses(kv, hd, w == 1, j)
        m[w, at] = True
        if kv == "f16":
            m[w, at + 1] = True
        else:
            m[w, scale] = m[w, scale + 1] = True
    return m


def scales(kv, x):
    """The stored scale of every element's block, as the definition rounds it."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    if kv == "q8":
        d = np.abs(y).max(-1, keepdims=True) / 127
    else:
        d = np.take_along_axis(y, np.abs(y).argmax(-1)[..., None], -1) / -8
    d = np.clip(d, -65504, 65504).astype(np.float16).astype(np.float64)
    return np.broadcast_to(d, y.shape).reshape(x.shape)


def turn(x, weight, eps, cs, interleaved):
    """RMSNorm and rotation of rows [n, heads, hd] by (cos, sin) [n, half, 2]."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    if cs is None:
        return x
    half = cs.shape[1]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def attend(q, k, v, scale):
    """One row: q [heads, hd], k and v [n, kv_heads, hd]. Returns the output and, for
    every head, sum |q k| scale at most and sum p |v| (what errors scale with)."""
    heads, hd = q.shape
    out, mass = np.zeros((heads, hd)), np.zeros((heads, hd))
    reach = np.zeros(heads)
    if len(k) == 0:
        return out, mass, reach
    for h in range(heads):
        kv = h // (heads // k.shape[1])
        s = k[:, kv] @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mass[h] = p @ v[:, kv], p @ np.abs(v[:, kv])
        reach[h] = (np.abs(k[:, kv]) @ np.abs(q[h])).max() * abs(scale)
    return out, mass, reach
