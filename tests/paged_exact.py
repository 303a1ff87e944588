"""Attention over the 8-bit paged cache in float64, and what the errors of the kernels' roundings
are bounded by: for the GPU tests of its forms."""

from __future__ import annotations

import numpy as np
import torch

from test_gpu_paged_kv import HALF, _host


def exact(c, b, q, L, scale, window=0, kept=0, sink=None, causal=True):
    """Sequence b's attention for its last queries q [n, Hq, D]: o, and (all [n, Hq, D] but reach
    [n, Hq, 1])
      size   sum_j w_j |v_j|
      floor  max_j (w_j s_j) sum_j |code_j|, s_j the scale of v_j
      var    sum_j (w_j v_j)^2
      reach  the largest sum_d |q_d k_d| scale."""
    n, Hq, D = q.shape
    H, page = c.k.shape[1], c.k.shape[2]
    block = page // c.vs.shape[2]
    L = max(0, min(L, c.table.shape[1] * page))
    o, size, floor, var = (np.zeros(q.shape) for _ in range(4))
    reach = np.zeros((n, Hq, 1))
    if L == 0:
        return o, size, floor, var, reach
    t = np.arange(L)
    ids = c.table[b][t // page]
    there = (ids >= 0) & (ids < c.k.shape[0])
    ids = np.where(there, ids, 0)
    from oracle import quant as Q

    def rows(codes, scales):
        x = Q.e4m3_to_f32(codes[ids, :, t % page]).astype(np.float64)
        y = scales[ids, :, t % page // block, None].astype(np.float64)
        return np.where(there[:, None, None], x * y, 0.0), np.where(there[:, None], y[..., 0], 0.0)

    (k, _), (v, sv) = rows(c.k, c.ks), rows(c.v, c.vs)
    pos = L - n + np.arange(n)[:, None]
    seen = np.broadcast_to(there, (n, L)).copy()
    if causal:
        seen &= t <= pos
        if window:
            seen &= (t > pos - window) | (t < kept)
    for h in range(Hq):
        g = h // (Hq // H)
        s = np.where(seen, q[:, h].astype(np.float64) @ k[:, g].T * scale, -np.inf)
        m = s.max(1, keepdims=True)
        if sink is not None:
            m = np.maximum(m, sink[h])
        w = np.exp(s - np.where(m > -np.inf, m, 0.0))
        den = w.sum(1, keepdims=True) + (0.0 if sink is None else np.exp(sink[h] - m))
        w /= np.where(den > 0, den, 1.0)
        o[:, h], size[:, h], var[:, h] = w @ v[:, g], w @ np.abs(v[:, g]), w ** 2 @ v[:, g] ** 2
        code = np.abs(v[:, g]) / np.where(sv[:, g] > 0, sv[:, g], 1.0)[:, None]
        floor[:, h] = (w * sv[:, g]).max(1)[:, None] * (seen @ code)
        reach[:, h, 0] = np.where(seen, np.abs(q[:, h].astype(np.float64)) @ np.abs(k[:, g]).T, 0.0).max(1) * scale
    return o, size, floor, var, reach


def check(c, o, q, lens, cu, scale=None, rms=True, parts=1, **kw):
    """A weight is rounded to f16, by 2^-11 of itself at most, or by half of the smallest step,
    2^-25, where the row's largest weight times its value's scale stands at 2^10 or more: 2^-35 of
    that one, in each of the `parts` that a row's keys are taken in with a reference of their own.  Its
    score is an fp32 sum of D products (2^-23 each at most), in normaliser and numerator; exp2, log2
    and the sums over keys and parts take 2^-18.  The roundings of different keys go either way: a
    row's mean square over its D elements is that of evenly spread roundings (a third of the largest
    one's square), with a factor of 2 on its root."""
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    cu = list(range(len(lens) + 1)) if cu is None else cu
    assert o.dtype == q.dtype and o.shape == q.shape
    got, qh, half = _host(o).astype(np.float64), _host(q), HALF[q.dtype]
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    worst = most = 0.0
    for b, L in enumerate(lens):
        if cu[b + 1] == cu[b]:
            continue
        ref, size, floor, var, reach = exact(c, b, qh[cu[b]:cu[b + 1]], L, scale, **kw)
        err = np.abs(got[cu[b]:cu[b + 1]] - ref)
        assert np.isfinite(err).all()
        even = size * (2 * (D + 8) * 2.0 ** -23 * reach + 2.0 ** -18) + parts * 2.0 ** -35 * floor
        bound = even + 2.0 ** -11 * size
        worst = max(worst, float((err / np.maximum(bound + half * (np.abs(ref) + bound) + tiny, 1e-300)).max()))
        if rms:
            spread = (2.0 ** -22 * var + (half * np.abs(ref)) ** 2) / 3.0
            allowed = 2.0 * np.sqrt(spread.mean(-1)) + np.sqrt((even ** 2).mean(-1)) + tiny
            most = max(most, float((np.sqrt((err ** 2).mean(-1)) / np.maximum(allowed, 1e-300)).max()))
    print(f"  worst error / bound {worst:.3f}, mean square {most:.3f}", flush=True)
    assert worst <= 1.0 and most <= 1.0


def ints(v, dev):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device=dev)


def join_tables(c, cu_groups, shared):
    """The full pages among each group's first shared tokens become those of its first sequence."""
    page = c.k.shape[2]
    for g, n in enumerate(shared):
        for b in range(cu_groups[g], cu_groups[g + 1]):
            cols = min(n // page, c.table.shape[1])
            c.table[b, :cols] = c.table[cu_groups[g], :cols]
    c.bt = torch.from_numpy(c.table).to(c.dev)
