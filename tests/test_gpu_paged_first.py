"""Attention over the 8-bit paged cache with a sliding window and first tokens that it does not
hide, against float64."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_exact import check, exact, ints
from test_gpu_paged_kv import Cache, _bytes, _filled, _host, _queries, _widen

pytestmark = pytest.mark.gpu


def _call(c, q, lens, cu, sink=None, **kw):
    return c.P.paged_attn(q, c.kv, c.bt, ints(lens, c.dev), cu_tokens=ints(cu, c.dev),
                          sink=None if sink is None else torch.from_numpy(sink).to(c.dev), **kw)


CASES = [
    # new, lens, Hq, Hkv, D, page, block, dtype, window, first, sink
    ([1], [1], 1, 1, 16, 16, 16, torch.bfloat16, 1, 1, False),
    ([1], [5000], 8, 2, 128, 64, 64, torch.float16, 300, 4, False),
    ([1, 1, 1, 1], [700, 2000, 33, 0], 16, 2, 64, 16, 16, torch.float16, 100, 130, True),
    ([4, 2], [2000, 900], 8, 2, 128, 64, 32, torch.float16, 500, 128, False),
    ([1, 1], [1500, 260], 8, 1, 256, 128, 128, torch.bfloat16, 1, 257, False),
    ([8, 1], [1000, 129], 16, 2, 80, 32, 16, torch.bfloat16, 64, 20, True),   # 32 rows a tile
    ([40, 3], [2000, 260], 4, 1, 256, 64, 64, torch.float16, 70, 33, False),
    ([150, 30], [1500, 700], 8, 2, 128, 32, 16, torch.float16, 200, 5, True),
    ([200], [2000], 8, 2, 64, 64, 64, torch.float16, 600, 64, False),
    ([130], [900], 4, 1, 96, 64, 64, torch.bfloat16, 30, 500, False),
    ([257], [257], 16, 1, 192, 128, 64, torch.bfloat16, 50, 17, False),       # a whole prompt
    ([300, 120], [300, 4000], 4, 1, 128, 16, 16, torch.bfloat16, 90, 70, True),
    ([70, 5], [30, 0], 4, 2, 128, 64, 64, torch.bfloat16, 20, 8, False),      # more queries than keys
    ([200], [1200], 8, 2, 128, 64, 64, torch.bfloat16, 40, 100000, False),    # all of them are first
    ([1], [1200], 8, 2, 128, 64, 64, torch.bfloat16, 40, 1200, False),
]


@pytest.mark.parametrize("tokens", [0, 16384])
@pytest.mark.parametrize("new,lens,Hq,Hkv,D,page,block,dtype,window,first,sink", CASES)
def test_window_and_first_tokens(gpu, tokens, new, lens, Hq, Hkv, D, page, block, dtype, window, first, sink):
    print(f"first new={new} lens={lens} Hq={Hq} Hkv={Hkv} D={D} window={window} first={first}", flush=True)
    c = _filled(gpu, lens, Hkv, D, page, block, seed=D + Hq)
    _widen(c, tokens)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], Hq, D, dtype, 9)
    s = (np.random.default_rng(2).standard_normal(Hq) * 2).astype(np.float32) if sink else None
    o = _call(c, q, lens, cu, s, window=window, first=first)
    check(c, o, q, lens, cu, window=window, kept=first, sink=s)
    if new == [1] * len(new):
        assert torch.equal(_call(c, q, lens, None, s, window=window, first=first), o)


@pytest.mark.parametrize("D,Hq,new", [(64, 4, 1), (128, 4, 1), (256, 4, 1), (128, 8, 5), (64, 4, 150), (128, 4, 150),
                                      (256, 4, 60)])
@pytest.mark.parametrize("tokens", [0, 16384])
def test_every_border_of_the_window_and_the_first_tokens(gpu, D, Hq, new, tokens):
    """First tokens that end on, before and behind the borders of granules and key tiles, windows
    that begin in, next to and behind the tile they end in."""
    L = 700
    c = _filled(gpu, [L], 1, D, 16, 16, seed=D)
    _widen(c, tokens)
    q = _queries(gpu, new, Hq, D, torch.float16, 3)
    for first in (1, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 256):
        for window in (1, 63, 64, 200, L - new - first, L - new - first + 1, L - 1, L, L + 5):
            o = _call(c, q, [L], [0, new], window=window, first=first)
            check(c, o, q, [L], [0, new], window=window, kept=first)


@pytest.mark.parametrize("new", [1, 130])
@pytest.mark.parametrize("window,first", [(100, 70), (500, 4), (3000, 300)])
def test_every_key_counts_once(gpu, new, window, first):
    """Values of zero but for one key in each dim of a kv head: the output is that key's weight."""
    L, H, D = 2200, 8, 64
    c = Cache(gpu, 1, L, H, D, 16, 16, seed=4)
    _widen(c, 16384)
    g = torch.Generator(device=gpu).manual_seed(L)
    k = 0.5 * torch.randn(L, H, D, generator=g, device=gpu)
    q = _queries(gpu, new, 2 * H, D, torch.float16, 11)
    for base in range(0, L, H * D):
        v = torch.zeros(L, H, D, device=gpu)
        t = base + torch.arange(H * D, device=gpu)
        t = t[t < L]
        v[t, (t - base) // D, (t - base) % D] = 1.0 + (t % 7) / 8.0
        c.P.append_kv(c.kv, k, v, c.bt, ints([0], gpu), cu_tokens=ints([0, L], gpu))
        c.k, c.v = _bytes(c.kv.k).copy(), _bytes(c.kv.v).copy()
        c.ks, c.vs = _host(c.kv.k_scale).copy(), _host(c.kv.v_scale).copy()
        check(c, _call(c, q, [L], [0, new], window=window, first=first), q, [L], [0, new], rms=False, window=window,
              kept=first)


@pytest.mark.parametrize("new", [1, 150])
def test_no_first_tokens_is_the_plain_window(gpu, new):
    """And first tokens that the window reaches anyway are the plain result to its last bit, where
    the keys are divided alike."""
    lens = [900, 333]
    c = _filled(gpu, lens, 2, 128, 64, 64, seed=5)
    _widen(c, 16384)
    cu = [0, new, 2 * new]
    q = _queries(gpu, cu[-1], 8, 128, torch.bfloat16, 3)
    assert torch.equal(_call(c, q, lens, cu, window=64, first=0), _call(c, q, lens, cu, window=64))
    check(c, _call(c, q, lens, cu, window=100000, first=9), q, lens, cu)
    # masks that hide nothing of the window: a window as long as the table
    assert torch.equal(_call(c, q, lens, cu, window=16384, first=9), _call(c, q, lens, cu))


@pytest.mark.parametrize("D,new,tokens", [(128, 1, 0), (128, 1, 16384), (64, 6, 0), (256, 40, 16384), (128, 150, 0),
                                          (64, 150, 16384)])
def test_nan_reaches_only_the_rows_that_see_it(gpu, D, new, tokens):
    """Among the first tokens (every row's), behind them and before the window (nobody's), and where
    only some rows' windows reach."""
    L, window, first = 900, 100, 37
    c = _filled(gpu, [L], 2, D, 64, 16, seed=11)
    _widen(c, tokens)
    hidden = L - new - window - 30
    spots = [(36, 0, 3), (37, 0, 5), (hidden, 1, 7), (L - new // 2 - window, 1, D - 6), (L - 1, 0, 9)]
    for t, h, d in spots:
        p, spot = int(c.table[0, t // 64]), t % 64
        c.kv.v.view(torch.uint8)[p, h, spot, d] = 0x7F
        c.v[p, h, spot, d] = 0x7F
    p, spot = int(c.table[0, 38 // 64]), 38  # a key that is hidden as well
    c.kv.k.view(torch.uint8)[p, 1, spot, 5] = 0x7F
    q = _queries(gpu, new, 8, D, torch.bfloat16, 5)
    o = _call(c, q, [L], [0, new], window=window, first=first)
    want = np.zeros((new, 8, D), bool)
    pos = L - new + np.arange(new)
    for t, h, d in spots:
        sees = (t <= pos) & ((t > pos - window) | (t < first))
        want[sees, 4 * h:4 * h + 4, d] = True
    np.testing.assert_array_equal(np.isnan(_host(o)), want)
    c.v[c.v == 0x7F] = 0
    ref, size, floor, _, reach = exact(c, 0, _host(q), L, D ** -0.5, window=window, kept=first)
    # what is not NaN is right: the bound of paged_exact.check, values being of any size
    bound = size * (2 * (D + 8) * 2.0 ** -23 * reach + 2.0 ** -18 + 2.0 ** -11) + 2.0 ** -35 * floor
    assert np.all(np.where(want, 0.0, np.abs(_host(o) - ref)) <= bound + 2.0 ** -8 * (np.abs(ref) + bound))


def test_pages_that_are_none_in_and_behind_the_first_tokens(gpu):
    lens = [900, 500]
    c = _filled(gpu, lens, 2, 128, 16, 16, seed=9)
    c.table[0, 1], c.table[0, 10], c.table[0, 54], c.table[1, :] = -1, 1 << 30, -1, -5
    c.bt = torch.from_numpy(c.table).to(gpu)
    for new in ([1, 1], [20, 3], [150, 2]):
        cu = [0] + np.cumsum(new).tolist()
        q = _queries(gpu, cu[-1], 8, 128, torch.bfloat16, 4)
        o = _call(c, q, lens, cu, window=60, first=50)
        check(c, o, q, lens, cu, window=60, kept=50)
        assert not o[cu[1]:].any()


def test_many_sequences_and_rows_behind_the_last(gpu):
    rng = np.random.default_rng(6)
    lens = rng.integers(0, 400, 150).tolist()
    new = [(1, 3, 0, 40)[i % 4] if i % 30 else 200 for i in range(150)]
    lens = [max(n, h) if i % 5 else h for i, (n, h) in enumerate(zip(new, lens))]
    for D, Hkv, Hq in ((64, 2, 8), (128, 1, 8)):
        c = _filled(gpu, lens, Hkv, D, 16, 16, seed=12)
        cu = [0] + np.cumsum(new).tolist()
        q = _queries(gpu, cu[-1] + 3, Hq, D, torch.float16, 6)
        for tokens in (0, 16384):
            _widen(c, tokens)
            out = torch.full_like(q, 7.0)
            o = _call(c, q, lens, cu, window=80, first=10, out=out)
            assert o.data_ptr() == out.data_ptr() and bool((out[cu[-1]:] == 7.0).all())
            check(c, o, q, lens, cu, window=80, kept=10)


@pytest.mark.parametrize("new", [1, 150])
def test_windows_and_first_tokens_of_any_length(gpu, new):
    lens = [900, 333]
    c = _filled(gpu, lens, 2, 128, 64, 64, seed=6)
    _widen(c, 16384)
    cu = [0, new, 2 * new]
    q = _queries(gpu, cu[-1], 8, 128, torch.bfloat16, 3)
    want = _call(c, q, lens, cu)
    for far in (2 ** 62, 2 ** 63 - 1, 2 ** 64 + 5):
        for kw in (dict(window=far), dict(window=far, first=far), dict(window=far, first=3)):
            assert torch.equal(_call(c, q, lens, cu, **kw), want)
        check(c, _call(c, q, lens, cu, window=3, first=far), q, lens, cu)


@pytest.mark.parametrize("new,tokens", [([1, 4], 0), ([3, 1], 16384), ([130, 1, 0, 300], 0), ([130, 1, 0, 300], 16384)])
def test_strided_queries_and_into_the_queries_themselves(gpu, new, tokens):
    lens = [900 + 7 * i for i in range(len(new))]
    c = _filled(gpu, lens, 2, 128, 64, 32, seed=22)
    _widen(c, tokens)
    cu = [0] + np.cumsum(new).tolist()
    wide = _queries(gpu, cu[-1], 24, 128, torch.bfloat16, 8)
    q = wide[:, 8:16]
    want = _call(c, q, lens, cu, window=200, first=70)
    check(c, want, q.contiguous(), lens, cu, window=200, kept=70)
    held = q.contiguous()
    assert _call(c, held, lens, cu, window=200, first=70, out=held) is held
    assert torch.equal(held, want)


def test_captured_with_other_lengths(gpu):
    c = _filled(gpu, [3000, 17, 900], 2, 128, 64, 64, seed=14)
    _widen(c, 8192)
    q = _queries(gpu, 3, 16, 128, torch.bfloat16, 10)
    lens = ints([3000, 17, 900], gpu)
    run = lambda: c.P.paged_attn(q, c.kv, c.bt, lens, window=200, first=70)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for have in ([3000, 17, 900], [1, 0, 64], [2000, 16, 300], [271, 17, 899]):
        lens.copy_(ints(have, gpu))
        q.mul_(-0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, run())
        check(c, held, q, have, None, window=200, kept=70)
