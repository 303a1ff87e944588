"""Caches whose scales the append would not write: zero, tiny, not a power of two, not finite.  A
stored value is code * scale whatever the scale is; a token is seen by those that may see it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import quant as Q
from test_gpu_paged_kv import Cache, _bytes, _check_attn, _filled, _host, _new, _queries, _widen

pytestmark = pytest.mark.gpu

KERNELS = [(1, 128), (8, 256), (20, 128), (30, 64), (30, 256), (150, 64), (150, 128), (150, 256)]  # queries, head dim
FEW_AND_CHUNKS = pytest.mark.parametrize("new,D", KERNELS)
TOKENS = pytest.mark.parametrize("tokens", [0, 16384])


def _set(c, side, token, value, head=slice(None)):
    """The scale of a token's block (sequence 0)."""
    page, block = c.k.shape[2], c.k.shape[2] // c.ks.shape[2]
    p, piece = int(c.table[0, token // page]), token % page // block
    ours, theirs = ((c.kv.k_scale, c.ks), (c.kv.v_scale, c.vs))[side]
    ours[p, head, piece] = value
    theirs[p, head, piece] = value


@TOKENS
@FEW_AND_CHUNKS
@pytest.mark.parametrize("window", [0, 40])
def test_attention_of_keys_whose_scale_is_zero(gpu, tokens, new, D, window):
    """Scores of zero for those who see them, nothing for the others: the last block, one that the
    rows see in part, one at a window's edge."""
    L = 200
    c = _filled(gpu, [L], 2, D, 64, 16, seed=3)
    for t in (L - 1, L - new // 2 - 1, 100, max(0, L - new - 20)):
        _set(c, 0, t, 0.0, head=t % 2)
    _widen(c, tokens)
    _check_attn(c, _queries(gpu, new, 4, D, torch.bfloat16, 5), [L], [0, new], window=window)


@TOKENS
@FEW_AND_CHUNKS
def test_a_softmax_scale_that_takes_scores_below_the_smallest_float(gpu, tokens, new, D):
    """Keys of zero have the scale 2^-100, and with 1e-25 before it 0 in fp32: equal weights."""
    L = 200
    c = _filled(gpu, [L], 2, D, 64, 16, seed=3)
    for t in range(0, L, 16):
        _set(c, 0, t, 2.0 ** -100)
    _widen(c, tokens)
    _check_attn(c, _queries(gpu, new, 4, D, torch.bfloat16, 5), [L], [0, new], softmax_scale=1e-25)


@TOKENS
@FEW_AND_CHUNKS
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("window", [0, 40])
def test_a_scale_that_is_not_finite_reaches_the_rows_that_see_its_tokens(gpu, tokens, new, D, side, value, window):
    """As NaN, and no other row: those before the block, those whose window is behind it."""
    L = 200
    c = _filled(gpu, [L], 2, D, 64, 16, seed=3)
    c.kv.k.view(torch.uint8)[:, :, :, 0] = 0  # (a code of zero times an infinity is NaN)
    _set(c, side, 180, value, head=0)          # rows from token 176 on
    if window:
        _set(c, side, 100, value, head=1)      # rows up to token 111 + 39
    _widen(c, tokens)
    q = _queries(gpu, new, 4, D, torch.bfloat16, 5)
    lens = torch.tensor([L], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, new], dtype=torch.int32, device=gpu)
    o = _host(c.P.paged_attn(q, c.kv, c.bt, lens, cu_tokens=cu, window=window))
    good = _filled(gpu, [L], 2, D, 64, 16, seed=3)
    good.kv.k.view(torch.uint8)[:, :, :, 0] = 0
    _widen(good, tokens)
    want = _host(good.P.paged_attn(q, good.kv, good.bt, lens, cu_tokens=cu, window=window))
    pos = L - new + np.arange(new)
    bad = np.zeros((new, 4), bool)
    bad[:, :2] = (pos >= 176)[:, None]
    if window:
        bad[:, 2:] = ((pos >= 96) & (pos - window + 1 <= 111))[:, None]
    assert np.isnan(o[bad]).all()
    assert np.isfinite(o[~bad]).all()
    # (the same sums but for where a reference was taken: a rounding of the output and of weights)
    np.testing.assert_allclose(o[~bad], want[~bad], rtol=2.0 ** -6, atol=2.0 ** -8)


@TOKENS
@FEW_AND_CHUNKS
def test_values_whose_scale_is_zero_are_zero(gpu, tokens, new, D):
    """Also alone, where nothing is added to hide them; beside others they take their weight."""
    L = 200
    c = _filled(gpu, [L], 2, D, 64, 16, seed=3)
    for t in range(0, L, 16):
        _set(c, 1, t, 0.0, head=0)  # all of head 0
    _set(c, 1, 40, 0.0, head=1)
    _set(c, 1, L - 1, 0.0, head=1)
    _set(c, 1, 100, 2.0 ** -110, head=1)  # (values below 2^-101: nothing beside the others)
    _widen(c, tokens)
    o = _check_attn(c, _queries(gpu, new, 4, D, torch.bfloat16, 5), [L], [0, new])
    assert bool((o[:, :2] == 0).all())


@pytest.mark.parametrize("dtype,rot", [(torch.bfloat16, 0), (torch.float16, 0), (torch.float32, 0),
                                       (torch.bfloat16, 32), (torch.float32, 32)])
@pytest.mark.parametrize("factor", [1.3, 0.7])
def test_append_beside_a_scale_that_is_no_power_of_two(gpu, dtype, rot, factor):
    """Tokens that fit under it, tokens that it grows for, a NaN and an infinity among them."""
    from sglang_lite_amd import rotary as R

    c = Cache(gpu, 2, 64, 2, 64, 16, 16, seed=8)
    kw = dict(table=R.rotary_table(100, rot, device=gpu)) if rot else {}
    k, v = _new(gpu, 10, 2, 64, dtype, 1, spread=0.0)
    c.append(k, v, [0, 0], [0, 5, 10], **kw)
    for t in (c.kv.k_scale, c.kv.v_scale):
        t.mul_(factor)
    c.ks *= np.float32(factor)
    c.vs *= np.float32(factor)
    k, v = _new(gpu, 8, 2, 64, dtype, 2, spread=0.0)
    k, v = k * 0.25, v * 0.25
    k[2, 0, 50], v[1, 1, 7] = float("nan"), float("inf")
    c.append(k, v, [5, 5], [0, 3, 8], **kw)
    c.check()
    k, v = _new(gpu, 2, 2, 64, dtype, 3, spread=0.0)
    c.append(k * 9, v * 9, [8, 10], None, **kw)
    c.check()


@pytest.mark.parametrize("value", [0.0, float("nan"), float("inf"), -1.0])
def test_append_beside_a_scale_of_zero_or_none(gpu, value):
    """The earlier tokens' values were zero, or NaN, and stay so when the block gets a scale."""
    c = Cache(gpu, 1, 32, 2, 64, 16, 16, seed=8)
    k, v = _new(gpu, 6, 2, 64, torch.bfloat16, 1)
    c.append(k, v, [0], [0, 6])
    c.kv.k_scale.fill_(value)
    c.kv.v_scale.fill_(value)
    p = int(c.table[0, 0])
    k, v = _new(gpu, 4, 2, 64, torch.bfloat16, 2)
    st, cu = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([6], [0, 4]))
    c.P.append_kv(c.kv, k, v, c.bt, st, cu_tokens=cu)
    for codes, scale, x in ((c.kv.k, c.kv.k_scale, k), (c.kv.v, c.kv.v_scale, v)):
        s = _host(scale)[p, :, 0]
        got = Q.e4m3_to_f32(_bytes(codes)[p]) * s[:, None, None]
        assert (s > 0).all() and np.isfinite(s).all()
        assert (got[:, :6] == 0).all() if value == 0 else np.isnan(got[:, :6]).all()
        want = _host(x).transpose(1, 0, 2)
        # e4m3: half a step is 2^-4 of a normal value, 2^-10 of the scale below them
        assert (np.abs(got[:, 6:10] - want) <= np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * s[:, None, None])).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,offset", [(64, 32, 16), (33, 10, 1)])
def test_rotary_leaves_padding_rows_whatever_they_hold(gpu, dtype, interleaved, D, rot, offset):
    """Infinities, NaN, zeros of either sign in a row without a position."""
    from sglang_lite_amd import rotary as R

    table = R.rotary_table(16, rot, scaling={"type": "yarn", "factor": 4.0, "original": 64}, device=gpu)
    x = torch.randn(6, 3, D, device=gpu).to(dtype)
    x[1, :, offset] = float("inf")
    x[1, :, offset + 1] = -0.0
    x[3, 1, offset:offset + rot] = -0.0
    x[3, 2, offset + 2] = float("nan")
    x[4] = float("-inf")
    for at in (torch.tensor([2, -1, 3, -7, -2 ** 31, 5], device=gpu), torch.tensor([2, -1, 3, -7, -3, 5], device=gpu).int()):
        for inverse in (False, True):
            y = R.rotary(x, table, at, interleaved=interleaved, offset=offset, inverse=inverse)
            for r in (1, 3, 4):
                nan = torch.isnan(x[r])
                assert torch.equal(torch.isnan(y[r]), nan)
                assert torch.equal(y[r][~nan], x[r][~nan])
                assert torch.equal(torch.signbit(y[r][~nan]), torch.signbit(x[r][~nan]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_leaves_keys_without_a_position(gpu, dtype, interleaved):
    """As if there were no table: an infinity turns no other element into NaN."""
    from sglang_lite_amd import rotary as R

    table = R.rotary_table(100, 64, device=gpu)
    k, v = _new(gpu, 4, 2, 64, dtype, 4)
    k[1, 0, 3], k[1, 1, 40], k[2, 0, 5] = float("inf"), float("nan"), -0.0
    at = torch.full((4,), -1, dtype=torch.int32, device=gpu)
    one, two = (Cache(gpu, 1, 16, 2, 64, 16, 16, seed=6) for _ in range(2))
    st, cu = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0], [0, 4]))
    one.P.append_kv(one.kv, k, v, one.bt, st, cu_tokens=cu, table=table, positions=at, interleaved=interleaved)
    two.P.append_kv(two.kv, k, v, two.bt, st, cu_tokens=cu)
    for a, b in zip(one.kv, two.kv):
        np.testing.assert_array_equal(_bytes(a), _bytes(b))
