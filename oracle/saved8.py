"""The training operators with 8-bit saved activations in 64 bits (numpy): what spurfies_amd.ops' checkpoint8, act8, layer_norm and wgrad8 are tested
against.  Written from the definitions in include/spurfies_hip.h; the byte format is computed element by element, without bit tricks."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 32


def pack(x):
    """x [rows, cols] (float64 values of the stored elements) -> codes [rows, 32 * blocks], steps [rows, blocks] (uint8)."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    codes, steps = np.zeros((rows, blocks * BLOCK), np.uint8), np.zeros((rows, blocks), np.uint8)
    for r in range(rows):
        for b in range(blocks):
            v = x[r, b * BLOCK:(b + 1) * BLOCK]
            sign = np.where(v > 0, 0, 128).astype(np.uint8)
            if not np.all(np.isfinite(v)):
                steps[r, b] = 255
                codes[r, b * BLOCK:b * BLOCK + len(v)] = sign
                continue
            top = float(np.abs(v).max())
            s = -126
            if top > 0:
                s = max(-126, math.frexp(top)[1] - 8)
                while np.round(top / 2.0 ** s) > 127:
                    s += 1
                s = min(s, 121)
            steps[r, b] = s + 127
            codes[r, b * BLOCK:b * BLOCK + len(v)] = np.minimum(np.round(np.abs(v) / 2.0 ** s), 127).astype(np.uint8) | sign
    return codes, steps


def restore(codes, steps, cols):
    """float64 values; the sign bit survives as the sign of zero."""
    step = np.where(steps == 255, np.nan, 2.0 ** (steps.astype(np.float64) - 127))
    v = (codes & 127).astype(np.float64) * np.repeat(step, BLOCK, axis=1)
    return np.where(codes > 127, -v, v)[:, :cols]


def erf(x):
    from scipy.special import erf as e

    return e(x)


def act(kind, x, p):
    with np.errstate(over="ignore"):
        if kind == "leaky_relu":
            return np.where(x > 0, x, x * p)
        if kind == "softplus":
            return np.logaddexp(0.0, p * x) / p
        if kind == "silu":
            return x / (1 + np.exp(-x))
        return 0.5 * x * (1 + erf(x / math.sqrt(2)))


def act_slope(kind, x, p):
    """f'(x); leaky_relu: by the sign bit of the restored value."""
    with np.errstate(over="ignore"):
        if kind == "leaky_relu":
            return np.where(np.isnan(x), np.nan, np.where(np.signbit(x), p, 1.0))
        if kind == "softplus":
            return 1 / (1 + np.exp(-p * x))
        s = 1 / (1 + np.exp(-x))
        if kind == "silu":
            return s * (1 + x * (1 - s))
        return 0.5 * (1 + erf(x / math.sqrt(2))) + x * np.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def statistics(x, eps):
    mean = x.mean(axis=1, keepdims=True)
    return mean, 1 / np.sqrt(((x - mean) ** 2).mean(axis=1, keepdims=True) + eps)


def layer_norm(x, w, b, eps):
    mean, rstd = statistics(x, eps)
    return (x - mean) * rstd * w + b


def layer_norm_backward(dy, x, w, mean, rstd):
    """x: as the backward pass reads it (restored, where it was saved in 8 bits); mean, rstd: the forward pass' -> dx, dw, db"""
    n = (x - mean) * rstd
    t = dy * w
    dx = rstd * (t - t.mean(axis=1, keepdims=True) - n * (t * n).mean(axis=1, keepdims=True))
    return dx, (dy * n).sum(axis=0), dy.sum(axis=0)
