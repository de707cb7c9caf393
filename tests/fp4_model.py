"""The 4-bit KV cache in 64 bits, from its definition: units of bytes from
values, values from units, and attention over them (numpy on the host)."""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
# codes 0..226: 8 multiples of 2^-17, then 3 mantissa bits per power of two from 2^-14
SCALES = np.array([c * 2.0 ** -17 if c < 8 else (8 + c % 8) * 2.0 ** (c // 8 - 18) for c in range(227)])


def nearest_code(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest to x >= 0, the even one on a tie."""
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = np.searchsorted(mid, x, side="left"), np.searchsorted(mid, x, side="right")
    return np.where(lo % 2 == 0, lo, hi)


def quantise(x: np.ndarray):
    """Values [..., D] (64 bits) to codes [..., D] and scale codes [..., D / 16]."""
    x = np.where(np.isnan(x), 0.0, x).reshape(*x.shape[:-1], -1, 16)
    s = nearest_code(np.abs(x).max(-1) / 6, SCALES)
    sv = SCALES[s][..., None]
    y = np.abs(x) / np.where(sv > 0, sv, np.inf)
    y = np.where(np.isinf(x) & (sv > 0), np.inf, y)
    c = nearest_code(y, E2M1) + 8 * (x < 0)
    return c.reshape(*c.shape[:-2], -1).astype(np.uint8), s.astype(np.uint8)


def dequantise(c: np.ndarray, s: np.ndarray) -> np.ndarray:
    """Any scale byte: above 226 too, as the half-precision number it stands for."""
    sv = (s.astype(np.uint16) << 7).view(np.float16).astype(np.float64)
    v = E2M1[c & 7] * np.where(c & 8, -1.0, 1.0)
    return v * np.repeat(sv, 16, -1)


def unit_bytes(c: np.ndarray, s: np.ndarray) -> np.ndarray:
    """[..., 16, D] codes and [..., 16, D / 16] scale codes to units [..., 9 D]."""
    p = (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)
    return np.concatenate([p.reshape(*p.shape[:-2], -1), s.reshape(*s.shape[:-2], -1)], -1)


def unit_codes(u: np.ndarray):
    d = u.shape[-1] // 9
    p = u[..., :8 * d].reshape(*u.shape[:-1], 16, d // 2)
    return np.stack([p & 15, p >> 4], -1).reshape(*p.shape[:-1], d), u[..., 8 * d:].reshape(*u.shape[:-1], 16, d // 16)


def held(layer: np.ndarray) -> np.ndarray:
    """Values of a layer [kv, blocks, heads, tpb / 16, 9 D]: [kv, blocks * tpb, heads, D]."""
    v = dequantise(*unit_codes(layer))  # [kv, blocks, heads, units, 16, D]
    kv, nb, h, u, _, d = v.shape
    return v.transpose(0, 1, 3, 4, 2, 5).reshape(kv, nb * u * 16, h, d)


def write(layer: np.ndarray, rows, slots: np.ndarray) -> None:
    """rows: [k] or [k, v], each [tokens, heads, D] in 64 bits; in place."""
    kv, nb, h, units, nbytes = layer.shape
    d = nbytes // 9
    for side, x in enumerate(rows):
        c, s = quantise(x)
        p = (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < nb * units * 16:
                b, u, t = slot // (16 * units), slot // 16 % units, slot % 16
                layer[side, b, :, u, t * d // 2:(t + 1) * d // 2] = p[i]
                layer[side, b, :, u, 8 * d + t * d // 16:8 * d + (t + 1) * d // 16] = s[i]


def attention(layer, q, tables, lens, cu, scale, causal, tpb):
    """q [tokens, Hq, D] in 64 bits.  Returns out, lse, the sum of weights times |v| (what errors of the
    weights scale with; 2^-21 of the sum of |v| is in it, see attention_bounds) and the largest scale * sum |q| |k|
    of each row (what errors of the scores scale with); rows of no sequence stay NaN."""
    h = layer.shape[2]
    n, hq, d = q.shape
    g = hq // h
    out, weight = np.full((n, hq, d), np.nan), np.zeros((n, hq, d))
    lse, size = np.full((n, hq), np.nan), np.zeros((n, hq))
    for b, length in enumerate(lens.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        length0, length = length, min(max(length, 0), tables.shape[1] * tpb)
        pages = tables[b, :-(-length // tpb)].astype(np.int64)
        good = (pages >= 0) & (pages < layer.shape[1])
        kv = held(layer[:, np.where(good, pages, 0)]) if len(pages) else np.zeros((2, 0, h, d))
        k, v = kv[:, :length]
        there = np.repeat(good, tpb)[:length]
        for i in range(hi - lo):
            end = min(length, length0 - (hi - lo) + i + 1) if causal else length
            seen = there & (np.arange(length) < end)
            for qh in range(hq):
                x = q[lo + i, qh]
                ks, vs = k[seen, qh // g], v[seen, qh // g]
                out[lo + i, qh], lse[lo + i, qh] = 0, -np.inf
                if not len(ks):
                    continue
                s = ks @ x * scale
                m = s.max()
                p = np.exp(s - m)
                out[lo + i, qh] = p @ vs / p.sum()
                weight[lo + i, qh] = p @ np.abs(vs) / p.sum() + 2.0 ** -21 * np.abs(vs).sum(0)
                lse[lo + i, qh] = m + np.log(p.sum())
                size[lo + i, qh] = (np.abs(ks) @ np.abs(x)).max() * abs(scale)
    return out, lse, weight, size


def attention_bounds(weight, size, out, d, dtype):
    """What a kernel with float32 sums and weights rounded to half may be off by: |o|'s own rounding to
    `dtype`; the weights' rounding, half a step of half precision (2^-11) of each |p v|; the scores' error,
    (D / 16 + 8) additions of float32 with 2^-23 each relative to sum |q k|, which moves a weight by as much
    and, through the sum of weights, the result by twice that; the float32 sums over the keys, 2^-14 for up
    to 2^9 partial sums at 2^-23.  Exponentials are good to 2^-20 of a weight beside the argument's rounding,
    which the scores' term covers."""
    half_step = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 0.0}[dtype]
    rel = 2.0 ** -11 + 2.0 ** -14 + 2.0 ** -19 + 2 * (d / 16 + 8) * 2.0 ** -23 * size[..., None]
    e = rel * weight
    return e + half_step * (np.abs(out) + e) + 2.0 ** -24  # the last: half a step of the smallest halves
