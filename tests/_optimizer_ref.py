"""AdamW restated for the tests: in float32 with every operation rounded on its
own (numpy, the order the kernel documents), and in float64 from the formulas."""
from __future__ import annotations

import math

import numpy as np
import torch

BLOCK = 256
f32 = np.float32


def blocks(x: np.ndarray) -> np.ndarray:
    n = -(-x.size // BLOCK) * BLOCK
    return np.concatenate([x, np.zeros(n - x.size, x.dtype)]).reshape(-1, BLOCK)


def to_8bit(x: np.ndarray, positive: bool = False) -> tuple[np.ndarray, np.ndarray]:
    """(e4m3 codes as uint8, one scale per block) of f32 values."""
    b = blocks(x)
    top = np.abs(b).max(1)
    scale = np.where(top > 0, np.maximum(top * (f32(1) / f32(448)), f32(2.0 ** -126)), f32(0))
    inv = np.where(top > 0, f32(1) / np.where(top > 0, scale, f32(1)), f32(0)).astype(f32)
    q = b * inv[:, None]
    if positive:
        q = np.where(b > 0, np.maximum(q, f32(2.0 ** -9)), q)
    codes = torch.from_numpy(q.reshape(-1)[: x.size].copy()).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).numpy(), scale.astype(f32)


def from_8bit(codes: np.ndarray, scale: np.ndarray, dtype=f32) -> np.ndarray:
    v = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).float().numpy().astype(dtype)
    return v * np.repeat(scale, BLOCK)[: v.size].astype(dtype)


def step_f32(p, m, v, g, step, lr, b1, b2, eps, wd, s=None, bits=32, ms=None, vs=None):
    """New (p, m, v, ms, vs): p the f32 sum; m, v f32 or codes."""
    size = f32(lr / -math.expm1(step * math.log(b1)) if b1 else lr)
    root = f32(1 / math.sqrt(-math.expm1(step * math.log(b2))) if b2 else 1.0)
    if bits == 8:
        m = from_8bit(m, ms)
        v = from_8bit(v, vs)
        v = v * v
    with np.errstate(all="ignore"):
        g = g.astype(f32) * (f32(1) if s is None else f32(s))
        m = m * f32(b1) + g * f32(1 - b1)
        v = v * f32(b2) + (g * f32(1 - b2)) * g
        r = np.sqrt(v)
        p = p * f32(1 - lr * wd) - (m * size) / (r * root + f32(eps))
    assert p.dtype == m.dtype == v.dtype == f32
    if bits == 8:
        m, ms = to_8bit(m)
        v, vs = to_8bit(r, positive=True)
    return p, m, v, ms, vs


def step_f64(p, m, v, g, step, lr, b1, b2, eps, wd):
    """New (p, m, v) in float64, and bounds of what float32 may be off by (half a
    step, u, for each rounding; a constant rounded from 64 bits counts as one)."""
    u = 2.0 ** -24
    p, m, v, g = (np.asarray(x, np.float64) for x in (p, m, v, g))
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    den = np.sqrt(v1 / (1 - b2 ** step)) + eps
    lr1 = lr / (1 - b1 ** step)
    upd = lr1 * m1 / den
    p1 = p * (1 - lr * wd) - upd
    # m: constant, product, sum (3 u) on the magnitudes; v: constant, two products, sum (4 u)
    tm = 3 * u * (np.abs(b1 * m) + np.abs((1 - b1) * g))
    tv = 4 * u * v1
    # update: m's, then constant and product (2), root of v (2 + 1), its constant and product (2),
    # eps and sum (2), division (1); weight: constant, product; difference
    tp = lr1 * tm / den + 10 * u * np.abs(upd) + 2 * u * np.abs(p) + u * np.abs(p1)
    return (p1, m1, v1), (1.01 * tp, 1.01 * tm, 1.01 * tv)
