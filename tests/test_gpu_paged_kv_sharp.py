"""The attention over the 8-bit paged cache against bounds that a lost key, a weight of too few
bits or one below its type's range does not pass."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as OP
from test_gpu_paged_kv import HALF, Cache, _bytes, _filled, _host, _queries, _widen

pytestmark = pytest.mark.gpu


def _exact(c, b, q, L, scale, window=0, sink=None):
    """Sequence b's causal attention in float64 for its last queries q [n, Hq, D]: o, and what the
    bounds go by (all [n, Hq, D] but reach [n, Hq, 1]):
      size   sum_j w_j |v_j|
      floor  max_j (w_j s_j) sum_j |code_j|, s_j the scale of v_j
      var    sum_j (w_j v_j)^2
      reach  the largest sum_d |q_d k_d| scale."""
    n, Hq, D = q.shape
    H, block = c.k.shape[1], c.k.shape[2] // c.vs.shape[2]
    k, there = OP.rows(c.k, c.ks, c.table[b], L)
    v, _ = OP.rows(c.v, c.vs, c.table[b], L)
    t = np.arange(L)
    page = np.where(there, c.table[b][t // c.k.shape[2]], 0)
    sv = c.vs[page, :, t % c.k.shape[2] // block].astype(np.float64)  # [L, H]
    pos = L - n + np.arange(n)[:, None]
    seen = there & (t <= pos) & ((t > pos - window) if window else True)
    o, size, floor, var = (np.zeros(q.shape) for _ in range(4))
    reach = np.zeros((n, Hq, 1))
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
        code = np.abs(v[:, g]) / np.where(there, sv[:, g], 1.0)[:, None]
        floor[:, h] = (w * np.where(there, sv[:, g], 0.0)).max(1)[:, None] * (seen @ code)
        reach[:, h, 0] = np.where(seen, np.abs(q[:, h].astype(np.float64)) @ np.abs(k[:, g]).T, 0.0).max(1) * scale
    return o, size, floor, var, reach


def _check_sharp(c, q, lens, cu, scale=None, window=0, sink=None, rms=True):
    """A weight is rounded to f16, by 2^-11 of itself at most, or by half of the smallest step,
    2^-25, where the row's largest weight times its value's scale stands at 2^10 or more: 2^-35 of
    that one.  Its score is an fp32 sum of D products (2^-23 each at most), in normaliser and
    numerator; exp2, log2 and the sums over keys take 2^-18.  The roundings of different keys go
    either way: a row's mean square over its D elements is that of evenly spread roundings (a third
    of the largest one's square), with a factor of 2 on its root."""
    dev, D = c.dev, q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    o = c.P.paged_attn(q, c.kv, c.bt, torch.tensor(lens, dtype=torch.int32, device=dev),
                       cu_tokens=torch.tensor(cu, dtype=torch.int32, device=dev), softmax_scale=scale,
                       window=window, sink=None if sink is None else torch.from_numpy(sink).to(dev))
    got, qh, half = _host(o).astype(np.float64), _host(q), HALF[q.dtype]
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    worst = most = 0.0
    for b, L in enumerate(lens):
        if cu[b + 1] == cu[b]:
            continue
        ref, size, floor, var, reach = _exact(c, b, qh[cu[b]:cu[b + 1]], L, scale, window, sink)
        err = np.abs(got[cu[b]:cu[b + 1]] - ref)
        assert np.isfinite(err).all()
        even = size * (2 * (D + 8) * 2.0 ** -23 * reach + 2.0 ** -18) + 2.0 ** -35 * floor
        bound = even + 2.0 ** -11 * size
        worst = max(worst, float((err / np.maximum(bound + half * (np.abs(ref) + bound) + tiny, 1e-300)).max()))
        if rms:
            spread = (2.0 ** -22 * var + (half * np.abs(ref)) ** 2) / 3.0
            allowed = 2.0 * np.sqrt(spread.mean(-1)) + np.sqrt((even ** 2).mean(-1)) + tiny
            most = max(most, float((np.sqrt((err ** 2).mean(-1)) / np.maximum(allowed, 1e-300)).max()))
    print(f"  worst error / bound {worst:.3f}, mean square {most:.3f}", flush=True)
    assert worst <= 1.0 and most <= 1.0
    return o


def _append(c, k, v, start, cu):
    st = torch.tensor(start, dtype=torch.int32, device=c.dev)
    c.P.append_kv(c.kv, k, v, c.bt, st, cu_tokens=torch.tensor(cu, dtype=torch.int32, device=c.dev))
    c.k, c.v = _bytes(c.kv.k).copy(), _bytes(c.kv.v).copy()
    c.ks, c.vs = _host(c.kv.k_scale).copy(), _host(c.kv.v_scale).copy()


@pytest.mark.parametrize("tokens", [0, 16384])
@pytest.mark.parametrize("D,new,dtype", [(64, 1, torch.float16), (128, 1, torch.bfloat16), (256, 1, torch.bfloat16),
                                         (64, 150, torch.bfloat16), (128, 150, torch.float16),
                                         (256, 40, torch.bfloat16)])
@pytest.mark.parametrize("lead,at", [(8.0, 0), (16.0, 0), (20.0, 0), (20.0, 3000)])
def test_small_weights_under_a_dominant_key_without_a_value(gpu, tokens, D, new, dtype, lead, at):
    """One key far above the others (by `lead` in the exponent of e) whose value is zero, as the
    first token's often is: what the others give is all that the row has."""
    L, H, Hq = 4096, 1, 4
    c = Cache(gpu, 1, L, H, D, 64, 16, seed=3)
    g = torch.Generator(device=gpu).manual_seed(D + new)
    k = torch.randn(L, H, D, generator=g, device=gpu)
    k[..., 0] = 0.0
    k[at] = 0.0
    k[at, :, 0] = lead * D ** 0.5 / 8.0
    v = (1.0 + torch.randn(L, H, D, generator=g, device=gpu).abs()) * 512.0
    v[at] = 0.0
    _append(c, k, v, [0], [0, L])
    _widen(c, tokens)
    q = _queries(gpu, new, Hq, D, dtype, 5)
    q[..., 0] = 8.0
    _check_sharp(c, q, [L], [0, new])
