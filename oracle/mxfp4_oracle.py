"""MXFP4 Block-ELL in float64 NumPy, from the definition (OCP Microscaling
Formats 1.0): what the GPU operators are tested against, not a fast path.

Blocks of 32 values along the last axis share s = 2^max(floor(log2 a) - 2, -127),
a the block's largest magnitude; codes are e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6),
rounded to nearest, ties to the even code, saturating.
"""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def e2m1(v):
    """Nearest grid value with v's sign; a tie goes to the even code."""
    m = np.minimum(np.abs(v), 6.0)
    hi = np.clip(np.searchsorted(GRID, m, side="left"), 1, 7)
    lo = hi - 1
    d_lo, d_hi = m - GRID[lo], GRID[hi] - m
    code = np.where(d_lo < d_hi, lo, np.where(d_hi < d_lo, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.copysign(GRID[code], v)


def scales(v):
    """s of each block, [..., n / 32]; NaN where the block is not finite."""
    b = np.asarray(v, np.float64).reshape(*v.shape[:-1], -1, BLOCK)
    a = np.abs(b).max(-1)
    ok = np.isfinite(a)
    _, e = np.frexp(np.where(ok & (a > 0), a, 1.0))  # a = f 2^e, f in [1/2, 1)
    E = np.where(a > 0, np.maximum(e - 3, -127), -127)
    return np.where(ok, np.ldexp(1.0, E), np.nan)


def quantize(v):
    """Q(v): the values MXFP4 holds for v."""
    v = np.asarray(v, np.float64)
    s = scales(v)[..., None]
    b = v.reshape(*v.shape[:-1], -1, BLOCK)
    with np.errstate(invalid="ignore"):
        q = e2m1(np.where(np.isnan(s), 0.0, b / s)) * s
    return q.reshape(v.shape)


def quantize_tiles(values, layout):
    """Q of Block-ELL tiles [R, K, B, B], returned [B_in, B_out] (layout 0) or [B_out, B_in] (1) as given."""
    return quantize(values) if layout else np.swapaxes(quantize(np.swapaxes(values, -1, -2)), -1, -2)


def dense(values, cols, C, layout=0):
    """[R*B, C*B] of the live tiles."""
    R, K, B, _ = values.shape
    w = np.zeros((R * B, C * B))
    for r in range(R):
        for k in range(K):
            c = int(cols[r, k])
            if 0 <= c < C:
                t = values[r, k] if layout else values[r, k].T
                w[r * B:(r + 1) * B, c * B:(c + 1) * B] += t
    return w


def tile_grads(grad, cols, B, layout=0):
    """Tiles of a dense weight gradient at the live slots, zeros elsewhere."""
    R, K = cols.shape
    out = np.zeros((R, K, B, B))
    for r in range(R):
        for k in range(K):
            c = int(cols[r, k])
            if 0 <= c < grad.shape[1] // B:
                t = grad[r * B:(r + 1) * B, c * B:(c + 1) * B]
                out[r, k] = t if layout else t.T
    return out


def silu_mul(g, u):
    return g / (1.0 + np.exp(-g)) * u


def swiglu_backward(xq, wg, wu, wd, hq, dy, residual):
    """Straight-through gradients (dx, dWg, dWu, dWd) at the quantised operands (dense)."""
    g, u = xq @ wg.T, xq @ wu.T
    sig = 1.0 / (1.0 + np.exp(-g))
    dh = dy @ wd
    du, dg = dh * g * sig, dh * u * sig * (1.0 + g * (1.0 - sig))
    dx = dg @ wg + du @ wu + (dy if residual else 0.0)
    return dx, dg.T @ xq, du.T @ xq, dy.T @ hq
