"""Oracle: rotary positions, the 8-bit paged KV cache and the attention over it, in numpy.

Test infrastructure only (see ``oracle/__init__.py``).  ``rotate`` and
``attention`` compute in float64 from the definition; ``append`` follows the
cache's own arithmetic (fp32, one rounding to e4m3) so that codes and scales
can be compared bit for bit.
"""

from __future__ import annotations

import numpy as np

from . import quant as Q


def pairs(rot: int, offset: int, interleaved: bool):
    """Element indices (a, b) of the pairs."""
    i = np.arange(rot // 2)
    return (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + rot // 2 + i)


def rotate(x, positions, freq, length, offset=0, interleaved=False, inverse=False):
    """x [T, H, D] -> float64; angles positions * freq in float64."""
    y = np.array(x, dtype=np.float64)
    a, b = pairs(2 * len(freq), offset, interleaved)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(freq, np.float64)
    c, s = (length * np.cos(angle))[:, None], (length * np.sin(angle))[:, None]
    if inverse:
        s = -s
    u, w = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


def rotate_f32(x, table_rows, offset=0, interleaved=False):
    """The same in fp32 with the table's own (cos, sin) [T, pairs, 2]: two products, then one
    sum or difference, each rounded."""
    y = np.array(x, dtype=np.float32)
    a, b = pairs(2 * table_rows.shape[1], offset, interleaved)
    c, s = table_rows[:, None, :, 0], table_rows[:, None, :, 1]
    u, w = y[..., a].copy(), y[..., b].copy()
    with np.errstate(invalid="ignore", over="ignore"):
        y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


def block_scale(amax) -> np.float32:
    """The smallest power of two >= 2^-100 with amax <= 448 * scale."""
    e = -100
    if amax > 0:
        m, k = np.frexp(np.float64(amax))  # m in [1/2, 1)
        e = max(int(k) - 9 + (1 if m > 0.875 else 0), -100)
    return np.float32(np.ldexp(1.0, e))


def encode(x):
    """fp32 -> e4m3 bytes; not finite -> the NaN code of its sign."""
    return Q.f32_to_e4m3(np.ascontiguousarray(x, dtype=np.float32))


def append(codes, scales, x, block_table, start, cu):
    """codes uint8 [P, H, page, D], scales fp32 [P, H, nb] updated in place by the fp32 rows
    x [T, H, D] of the sequences cu[b]:cu[b + 1]."""
    P, H, page, _ = codes.shape
    block = page // scales.shape[2]
    for b in range(len(start)):
        at, end, row = int(start[b]), int(start[b]) + int(cu[b + 1] - cu[b]), int(cu[b])
        if at < 0:
            continue
        while at < end:
            upto = min(end, (at // block + 1) * block)
            n = upto - at
            col = at // page
            p = int(block_table[b, col]) if col < block_table.shape[1] else -1
            if 0 <= p < P:
                lo = at % page
                piece, begin = lo // block, lo // block * block
                for h in range(H):
                    v = np.asarray(x[row:row + n, h], np.float32)
                    fine = np.abs(v[np.isfinite(v)])
                    s = block_scale(fine.max() if fine.size else 0.0)
                    old = scales[p, h, piece]
                    if lo > begin:
                        if old >= s:
                            s = old
                        elif old > 0:
                            was = codes[p, h, begin:lo]
                            again = encode(Q.e4m3_to_f32(was) * old / s)
                            codes[p, h, begin:lo] = np.where((was & 0x7F) == 0x7F, was, again)
                    with np.errstate(invalid="ignore", over="ignore"):
                        codes[p, h, lo:lo + n] = encode(v / s)
                    scales[p, h, piece] = s
            at, row = upto, row + n


def rows(codes, scales, table_row, n):
    """float64 values [n, H, D] of a sequence's first n tokens, and which of them are there."""
    P, H, page, D = codes.shape
    block = page // scales.shape[2]
    out, there = np.zeros((n, H, D)), np.zeros(n, bool)
    for t in range(n):
        p = int(table_row[t // page]) if t // page < len(table_row) else -1
        if 0 <= p < P:
            out[t] = Q.e4m3_to_f32(codes[p, :, t % page]).astype(np.float64) * \
                scales[p, :, t % page // block, None].astype(np.float64)
            there[t] = True
    return out, there


def attention(q, k_rows, v_rows, there, first, scale, causal=True, window=0, sink=None, kept=0):
    """One sequence: q [n, Hq, D] at positions first, first + 1, ...; k_rows, v_rows [L, Hkv, D];
    the window does not hide the sequence's `kept` first tokens.
    Returns o [n, Hq, D] float64 and, per element, sum_j w_j |v_j| and the largest
    sum_i |q_i k_i| scale among the keys seen (what rounding errors go by)."""
    n, Hq, D = q.shape
    L, Hkv, _ = k_rows.shape
    o, size, reach = np.zeros((n, Hq, D)), np.zeros((n, Hq, D)), np.zeros((n, Hq, 1))
    q = np.asarray(q, np.float64)
    key = np.arange(L)
    for i in range(n):
        p = first + i
        seen = there.copy()
        if causal:
            seen &= key <= p
            if window:
                seen &= (key > p - window) | (key < kept)
        if not seen.any():
            continue
        for h in range(Hq):
            g = h // (Hq // Hkv)
            kk, vv = k_rows[seen, g], v_rows[seen, g]
            with np.errstate(invalid="ignore"):
                s = kk @ q[i, h] * scale
                m = s.max() if sink is None else max(s.max(), float(sink[h]))
                w = np.exp(s - m)
                den = w.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - m))
                o[i, h] = w @ vv / den
                size[i, h] = w @ np.abs(vv) / den
                reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return o, size, reach


def rotate_axes(x, positions, axes, freq, length=1.0, offset=0, interleaved=False, inverse=False):
    """x [T, H, D] -> float64: pair i turned by its axis' position, positions [A, T], axes [pairs]."""
    y = np.array(x, dtype=np.float64)
    a, b = pairs(2 * len(freq), offset, interleaved)
    angle = np.asarray(positions, np.float64)[np.asarray(axes)].T * np.asarray(freq, np.float64)
    c, s = (length * np.cos(angle))[:, None], (length * np.sin(angle))[:, None]
    if inverse:
        s = -s
    u, w = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y
