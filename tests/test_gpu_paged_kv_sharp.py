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


CASES = [
    # new, lens, Hq, Hkv, D, page, block, dtype, window, sink
    ([1], [5000], 8, 2, 128, 64, 64, torch.float16, 0, False),
    ([1, 1, 1], [700, 2000, 33], 16, 2, 64, 16, 16, torch.float16, 0, True),
    ([4, 2], [2000, 900], 8, 2, 128, 64, 32, torch.float16, 500, False),
    ([1], [1500], 8, 1, 256, 128, 128, torch.bfloat16, 0, False),
    ([40, 3], [2000, 260], 4, 1, 256, 64, 64, torch.float16, 0, False),
    ([150, 30], [1500, 700], 8, 2, 128, 32, 16, torch.float16, 0, True),
    ([200], [2000], 8, 2, 64, 64, 64, torch.float16, 600, False),
    ([130], [900], 4, 1, 96, 64, 64, torch.bfloat16, 0, False),
]


@pytest.mark.parametrize("tokens", [0, 16384])
@pytest.mark.parametrize("new,lens,Hq,Hkv,D,page,block,dtype,window,sink", CASES)
def test_attention_within_the_roundings_of_its_weights(gpu, tokens, new, lens, Hq, Hkv, D, page, block, dtype,
                                                       window, sink):
    c = _filled(gpu, lens, Hkv, D, page, block, seed=D + Hq)
    _widen(c, tokens)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], Hq, D, dtype, 9)
    s = (np.random.default_rng(2).standard_normal(Hq) * 2).astype(np.float32) if sink else None
    _check_sharp(c, q, lens, cu, window=window, sink=s)


@pytest.mark.parametrize("tokens", [0, 16384])
@pytest.mark.parametrize("new,L,H,D,page,window,dtype", [
    (1, 4500, 8, 128, 64, 0, torch.float16),
    (1, 2300, 4, 64, 16, 1000, torch.float16),
    (1, 2100, 2, 256, 128, 0, torch.bfloat16),
    (20, 1500, 8, 128, 32, 0, torch.float16),    # 32 rows a tile
    (130, 1300, 8, 128, 64, 0, torch.float16),   # chunks
    (150, 1300, 8, 64, 16, 700, torch.float16),
    (40, 700, 4, 256, 64, 0, torch.bfloat16),
])
def test_every_key_counts_once(gpu, tokens, new, L, H, D, page, window, dtype):
    """Values of zero but for one key in each dim of a kv head: the output is that key's weight.
    As many rounds as it takes for every key to have had its dim."""
    c = Cache(gpu, 1, L, H, D, page, 16, seed=4)
    _widen(c, tokens)
    g = torch.Generator(device=gpu).manual_seed(L)
    k = 0.5 * torch.randn(L, H, D, generator=g, device=gpu)
    q = _queries(gpu, new, 2 * H, D, dtype, 11)
    for base in range(0, L, H * D):
        v = torch.zeros(L, H, D, device=gpu)
        t = base + torch.arange(H * D, device=gpu)
        t = t[t < L]
        v[t, (t - base) // D, (t - base) % D] = 1.0 + (t % 7) / 8.0
        _append(c, k, v, [0], [0, L])
        _check_sharp(c, q, [L], [0, new], window=window, rms=False)


@pytest.mark.parametrize("new", [1, 130])
def test_a_sequence_beside_others_of_other_lengths(gpu, new):
    """The seams between workgroups move with the batch; the result stays within its bounds."""
    for others in ([], [40], [3000, 10], [9000], [500] * 30):
        lens = [2500] + others
        c = _filled(gpu, lens, 2, 128, 64, 64, seed=15)
        _widen(c, 16384)
        cu = [0] + np.cumsum([new] + [1] * len(others)).tolist()
        q = _queries(gpu, cu[-1], 8, 128, torch.float16, 12)
        _check_sharp(c, q, lens, cu)
