"""Oracle: the norms, gate and residual sum between two blocks, in float64 from the definition.

Test infrastructure only (see ``oracle/__init__.py``).
"""

from __future__ import annotations

import numpy as np


def rms(v, eps):
    return 1.0 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)


def residual_norm(x, residual, before, after, gate, scale, eps):
    """(h, y) in float64, and bounds on the errors of fp32 arithmetic in them.

    A sum of squares has positive terms: a chain of at most 16 in a thread, 6 joins in
    a wavefront and 16 of wavefronts err by 38 half steps of it, the mean and eps by 2 more; the
    root halves that, and root and quotient add one each: 22 of the factor.  Two products: 24."""
    half = 2.0 ** -24
    x, residual = np.asarray(x, np.float64), np.asarray(residual, np.float64)
    u, du = x, np.zeros_like(x)
    if after is not None:
        u = x * rms(x, eps) * after
        du = 24 * half * np.abs(u)
    if gate is not None:
        u, du = u * gate, (du + half * np.abs(u)) * np.abs(gate)
    h = residual + scale * u
    dh = np.abs(scale) * (du + half * np.abs(u)) + half * (np.abs(h) + np.abs(scale * u))
    if before is None:
        return h, dh, None, None
    f = rms(h, eps)
    y = h * f * before
    far = np.linalg.norm(dh, axis=-1, keepdims=True) / np.maximum(np.linalg.norm(h, axis=-1, keepdims=True), 1e-300)
    dy = np.abs(f * before) * dh + np.abs(y) * (24 * half + far)
    return h, dh, y, dy * (1 + 1e-3)
