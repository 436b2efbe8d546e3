"""Plain restatement in 64 bits of the quantised records and of attention over them."""

from __future__ import annotations

import numpy as np
import torch

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOP = {"bf16": float(torch.finfo(torch.bfloat16).max), "fp16": 65504.0}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def nearest_even(y: np.ndarray, name: str) -> np.ndarray:
    """Codes of the format's values nearest to y (ties to the even code), saturated."""
    if name == "mxint8":
        return np.clip(np.rint(y * 64), -127, 127).astype(np.int64) & 255
    a = np.abs(y)
    d = np.abs(a[..., None] - E2M1)
    best = d.min(-1, keepdims=True)
    code = np.arange(8)
    # of two equally near codes the even one
    pick = np.where(d == best, np.where(code % 2 == 0, 0, 1), 2).argmin(-1)
    return pick + 8 * np.signbit(y)


def quantise(x: np.ndarray, name: str):
    """x [..., D] float64 -> (codes [..., D], scale codes [..., D / 32])."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    limit = 127.5 / 64 if name == "mxint8" else 7.0
    s = np.zeros(b.shape[:-1], np.int64)
    a = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    with np.errstate(all="ignore"):
        for code in range(254, -1, -1):  # the smallest scale that holds the block
            s = np.where(a <= limit * 2.0 ** (code - 127), code, s)
        y = np.where(bad[..., None], 0.0, b) / 2.0 ** (s - 127.0)[..., None]
    codes = np.where(bad[..., None], 0, nearest_even(y, name))
    return codes.reshape(x.shape), np.where(bad, 255, s)


def dequantise(codes: np.ndarray, s: np.ndarray, name: str) -> np.ndarray:
    if name == "mxint8":
        q = np.where(codes >= 128, codes - 256, codes) / 64.0
    else:
        q = np.where(codes >= 8, -1.0, 1.0) * E2M1[codes & 7]
    v = q.reshape(*q.shape[:-1], -1, 32) * 2.0 ** (s[..., None] - 127.0)
    return np.where(s[..., None] == 255, np.nan, v).reshape(codes.shape)


def in_type(v: np.ndarray, dt: str) -> np.ndarray:
    """v (of at most 24 significant bits) as a cache of the type holds it."""
    t = torch.from_numpy(np.clip(v, -TOP[dt], TOP[dt])).float().to(TORCH[dt])
    return t.double().numpy()


def sections(fmt):
    elems = fmt.block_size * fmt.num_heads * fmt.head_dim
    codes = -(-(elems // (2 if fmt.name == "mxfp4" else 1)) // 16) * 16
    return codes, -(-(elems // 32) // 16) * 16


def pack(fmt, k: np.ndarray, v: np.ndarray, out: np.ndarray) -> None:
    """K and V pages [H, bs, D] (float64) -> one layer's bytes of a record."""
    nc, ns = sections(fmt)
    for half, x in enumerate((k, v)):
        q, s = quantise(x, fmt.name)
        pack_codes(fmt, q, s, half, out)


def pack_codes(fmt, q, s, half, out):
    nc, ns = sections(fmt)
    q, s = q.reshape(-1), s.reshape(-1)
    if fmt.name == "mxfp4":
        q = q[0::2] | (q[1::2] << 4)
    out[half * nc:half * nc + q.size] = q
    out[2 * nc + half * ns:2 * nc + half * ns + s.size] = s


def unpack(fmt, layer: np.ndarray, half: int) -> np.ndarray:
    """K or V [H, bs, D] (float64) of one layer's bytes."""
    nc, ns = sections(fmt)
    elems = fmt.block_size * fmt.num_heads * fmt.head_dim
    if fmt.name == "mxfp4":
        b = layer[half * nc:half * nc + elems // 2].astype(np.int64)
        q = np.stack([b & 15, b >> 4], -1).reshape(-1)
    else:
        q = layer[half * nc:half * nc + elems].astype(np.int64)
    s = layer[2 * nc + half * ns:2 * nc + half * ns + elems // 32].astype(np.int64)
    shape = (fmt.num_heads, fmt.block_size, fmt.head_dim)
    return dequantise(q.reshape(shape), s.reshape(*shape[:2], -1), fmt.name)


def rotate(x: np.ndarray, delta: float, inv: np.ndarray, style: str) -> np.ndarray:
    """Rows [..., D] turned by delta; inv: the frequencies of the rotated pairs."""
    r = 2 * inv.size
    c, s = np.cos(delta * inv), np.sin(delta * inv)
    y = x.copy()
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if style == "neox" else \
        (x[..., 0:r:2], x[..., 1:r:2])
    lo, hi = a * c - b * s, b * c + a * s
    if style == "neox":
        y[..., :r // 2], y[..., r // 2:r] = lo, hi
    else:
        y[..., 0:r:2], y[..., 1:r:2] = lo, hi
    return y


def attend(q, k, v, seen, scale):
    """One request's queries [n, Hq, D] over k, v [H, T, D]: (out, lse, sum of p |v|, sum of
    |q| |k| scale at its largest), all float64; seen[i]: tokens that query i sees."""
    n, heads, d = q.shape
    group = heads // k.shape[0]
    out, mag = np.zeros((n, heads, d)), np.zeros((n, heads, d))
    lse, width = np.full((n, heads), -np.inf), np.zeros((n, heads))
    for i in range(n):
        for h in range(heads):
            kk, vv = k[h // group, :seen[i]], v[h // group, :seen[i]]
            if not len(kk):
                continue
            w = kk @ q[i, h] * scale
            top = w.max()
            p = np.exp(w - top)
            lse[i, h] = top + np.log(p.sum())
            p /= p.sum()
            out[i, h], mag[i, h] = p @ vv, p @ np.abs(vv)
            width[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return out, lse, mag, width
