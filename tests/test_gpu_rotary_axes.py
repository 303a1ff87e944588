"""Rotary positions with several axes on the GPU: the rotation of a batch's rows within
its roundings of float64, and keys on their way into the 8-bit paged cache bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as OP

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _host(t):
    return t.detach().to(torch.float32).cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _bytes(t):
    return t.view(torch.uint8).cpu().numpy()


def _bound(x, rot, offset, interleaved, dtype):
    """cos and sin carry half a step of fp32 each, as do the two products and the sum: 4 of |a| + |b|
    with room for their products; below f16's normal range a step is 2^-24."""
    x = np.abs(np.asarray(x, np.float64))
    a, b = OP.pairs(rot, offset, interleaved)
    bound = np.zeros_like(x)
    bound[..., a] = bound[..., b] = 4 * 2.0 ** -24 * (x[..., a] + x[..., b])
    return bound + (2.0 ** -25 if dtype == torch.float16 else 0.0)


CASES = [
    # T, H, D, sections, spread, offset, interleaved, dtype
    (1, 1, 128, (16, 24, 24), False, 0, False, torch.bfloat16),
    (5, 3, 128, (24, 20, 20), True, 0, True, torch.float16),
    (37, 8, 128, (10, 11, 11), False, 64, False, torch.float32),   # sections that end inside a chunk
    (300, 32, 128, (64,), False, 0, False, torch.bfloat16),
    (19, 4, 64, (1, 0, 30, 1), True, 0, False, torch.bfloat16),
    (7, 2, 80, (3, 7), False, 3, False, torch.bfloat16),           # single elements
    (6, 5, 33, (2, 2, 1), True, 1, True, torch.float32),
    (2100, 16, 96, (5, 6, 5), True, 64, True, torch.float32),
]


@pytest.mark.parametrize("T,H,D,sections,spread,offset,interleaved,dtype", CASES)
def test_axes_match_float64(gpu, T, H, D, sections, spread, offset, interleaved, dtype):
    from sglang_lite_amd import rotary as R

    print(f"axes T={T} H={H} D={D} {sections}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(T + D)
    rot, n = 2 * sum(sections), 5000
    table = R.rotary_table(n, rot, device=gpu)
    freq, _ = R.frequencies(rot)
    axes = R.rotary_axes(sections, spread=spread, device=gpu)
    x = torch.randn(T, H, D, generator=g, device=gpu).to(dtype)
    at = torch.randint(0, n, (len(sections), T), generator=g, device=gpu)
    at[:, 0] = n - 1
    for inverse, pos in ((False, at.int()), (True, at)):
        y = R.rotary(x, table, pos, axes=axes, interleaved=interleaved, offset=offset, inverse=inverse)
        assert y.shape == x.shape and y.dtype == dtype
        ref = OP.rotate_axes(_host(x), at.cpu().numpy(), axes.cpu().numpy(), freq.numpy(), 1.0, offset, interleaved,
                             inverse)
        bound = _bound(_host(x), rot, offset, interleaved, dtype)
        err = np.abs(_host(y).astype(np.float64) - ref)
        assert np.all(err <= bound + HALF[dtype] * (np.abs(ref) + bound)), float(err.max())
        rest = np.ones(D, bool)
        rest[offset:offset + rot] = False
        rest = torch.from_numpy(rest).to(gpu)
        assert torch.equal(y[..., rest], x[..., rest])


@pytest.mark.parametrize("spread", [False, True])
def test_one_position_on_every_axis_is_the_plain_rotation(gpu, spread):
    """Text: bit for bit, in place, strided, and where the chunks' paths differ."""
    from sglang_lite_amd import rotary as R

    T, H, D = 70, 4, 128
    table = R.rotary_table(512, 128, device=gpu)
    for sections in ((16, 24, 24), (13, 30, 21)):
        axes = R.rotary_axes(sections, spread=spread, device=gpu)
        fused = torch.randn(T, 3 * H, D, device=gpu).to(torch.bfloat16)
        q = fused[:, H:2 * H]
        at = torch.randint(0, 512, (T,), device=gpu)
        pos = at.expand(3, T)  # (not contiguous: copied)
        want = R.rotary(q, table, at)
        before = fused.clone()
        assert torch.equal(R.rotary(q, table, pos, axes=axes), want)
        assert torch.equal(R.rotary(q, table, pos.int().contiguous(), axes=axes, out=q), want)
        assert torch.equal(q, want) and torch.equal(fused[:, :H], before[:, :H])
        assert torch.equal(fused[:, 2 * H:], before[:, 2 * H:])


def test_padding_far_positions_and_axes_that_are_none(gpu):
    from sglang_lite_amd import rotary as R

    T, H = 9, 2
    for D, vec in ((64, True), (62, False)):  # 16-byte accesses, single elements
        rot = 32
        table = R.rotary_table(100, rot, device=gpu)
        axes = torch.tensor([0, 1] * 8, dtype=torch.uint8, device=gpu)
        x = torch.randn(T, H, D, device=gpu)
        x[2, 0, 0] = float("inf")
        at = torch.randint(0, 100, (2, T), device=gpu, dtype=torch.int64)
        at[1, 2], at[0, 3] = -1, -(2 ** 40)       # padding on either axis
        at[0, 4], at[1, 5] = 100, 2 ** 40         # behind the table: NaN in that axis' pairs alone
        y = R.rotary(x, table, at, axes=axes, interleaved=True)
        assert torch.equal(y[2:4], x[2:4])
        e = torch.arange(rot // 2, device=gpu)
        even = torch.cat([2 * e[0::2], 2 * e[0::2] + 1])
        odd = torch.cat([2 * e[1::2], 2 * e[1::2] + 1])
        assert torch.isnan(y[4][:, even]).all() and torch.isfinite(y[4][:, odd]).all()
        assert torch.isnan(y[5][:, odd]).all() and torch.isfinite(y[5][:, even]).all()
        assert torch.equal(y[..., rot:], x[..., rot:])
        bad = axes.clone()
        bad[3], bad[7] = 2, 255                   # axes that positions do not have
        z = R.rotary(x, table, at.clamp(0, 99), axes=bad, interleaved=True)
        w = R.rotary(x, table, at.clamp(0, 99), axes=axes, interleaved=True)
        lost = torch.tensor([6, 7, 14, 15], device=gpu)
        assert torch.isnan(z[:, :, lost]).all()
        kept = torch.ones(D, dtype=torch.bool, device=gpu)
        kept[lost] = False
        assert torch.equal(z[..., kept], w[..., kept])


def test_inverse_is_the_gradient(gpu):
    """Of L = sum(w * rotary(x)): rotary(w, inverse), against differences."""
    from sglang_lite_amd import rotary as R

    T, H, D = 4, 2, 32
    table = R.rotary_table(256, 32, device=gpu)
    axes = R.rotary_axes((5, 6, 5), spread=True, device=gpu)
    at = torch.randint(0, 256, (3, T), device=gpu)
    x, w = torch.randn(2, T, H, D, device=gpu)
    for inter in (False, True):
        grad = R.rotary(w, table, at, axes=axes, interleaved=inter, inverse=True).double()
        base = R.rotary(x, table, at, axes=axes, interleaved=inter).double()
        for e in (0, 1, 9, 15, 16, 17, 31):
            step = torch.zeros_like(x)
            step[..., e] = 1.0
            more = R.rotary(x + step, table, at, axes=axes, interleaved=inter).double()
            diff = (w.double() * (more - base)).sum(-1)
            # the map is linear: the difference is exact but for fp32 roundings of values below 16
            assert (diff - grad[..., e]).abs().max() <= 32 * 16 * 2.0 ** -23


@pytest.mark.parametrize("B,H,D,page,block,dtype,sections,spread,offset,interleaved", [
    (3, 2, 64, 16, 16, torch.bfloat16, (8, 12, 12), False, 0, False),
    (4, 1, 128, 64, 16, torch.float16, (11, 11, 10), True, 64, True),
    (2, 8, 128, 64, 64, torch.bfloat16, (24, 20, 20), True, 0, False),
    (2, 3, 80, 32, 32, torch.float32, (3, 5), False, 8, False),
    (70, 1, 96, 32, 16, torch.bfloat16, (16, 32), False, 0, False),
])
def test_append_turns_keys_by_axes_bit_for_bit(gpu, B, H, D, page, block, dtype, sections, spread, offset,
                                               interleaved):
    from sglang_lite_amd import paged_kv as P
    from sglang_lite_amd import rotary as R

    print(f"append axes B={B} H={H} D={D} page={page}", flush=True)
    rng = np.random.default_rng(B + D)
    rot, n = 2 * sum(sections), 300
    table = R.rotary_table(n, rot, device=gpu)
    axes = R.rotary_axes(sections, spread=spread, device=gpu)
    cols = -(-200 // page)
    pages = B * cols + 2
    kv = P.PagedKV.empty(pages, H, page, D, block=block, device=gpu)
    for c in (kv.k, kv.v):
        c.view(torch.uint8).fill_(0x7F)
    for s in (kv.k_scale, kv.v_scale):
        s.fill_(float("nan"))
    bt = rng.permutation(pages)[:B * cols].reshape(B, cols).astype(np.int32)
    codes = [_bytes(c).copy() for c in (kv.k, kv.v)]
    scales = [_host(s).copy() for s in (kv.k_scale, kv.v_scale)]
    have = [0] * B
    for step in range(3):
        new = [1] * B if step == 1 else [int(rng.integers(0, 60)) for _ in range(B)]
        cu = [0] + np.cumsum(new).tolist()
        T = sum(new)
        g = torch.Generator(device=gpu).manual_seed(step)
        x = (torch.randn(T, 2, H, D, generator=g, device=gpu) * 3).to(dtype)
        pos = torch.randint(0, n, (len(sections), T), generator=g, device=gpu, dtype=torch.int32)
        if T > 5:
            pos[0, 1], pos[-1, 2], pos[0, 3] = -1, -7, n  # two that are not turned, one that is NaN
        P.append_kv(kv, x[:, 0], x[:, 1], torch.from_numpy(bt).to(gpu),
                    torch.tensor(have, dtype=torch.int32, device=gpu),
                    cu_tokens=None if step == 1 else torch.tensor(cu, dtype=torch.int32, device=gpu), table=table,
                    positions=pos, axes=axes, offset=offset, interleaved=interleaved)
        at, tab = pos.cpu().numpy(), _host(table)
        rows = tab[np.clip(at, 0, n - 1)[axes.cpu().numpy()].T, np.arange(rot // 2)]  # [T, pairs, 2]
        rows[at[axes.cpu().numpy()].T >= n] = np.nan
        rows[(at < 0).any(0)] = (1.0, 0.0)
        k = OP.rotate_f32(_host(x[:, 0]), rows, offset, interleaved)
        OP.append(codes[0], scales[0], k, bt, have, cu)
        OP.append(codes[1], scales[1], _host(x[:, 1]), bt, have, cu)
        have = [h + m for h, m in zip(have, new)]
        np.testing.assert_array_equal(_host(kv.k_scale), scales[0])
        np.testing.assert_array_equal(_host(kv.v_scale), scales[1])
        np.testing.assert_array_equal(_bytes(kv.k), codes[0])
        np.testing.assert_array_equal(_bytes(kv.v), codes[1])


def test_axes_in_a_graph_and_on_another_stream(gpu):
    from sglang_lite_amd import rotary as R

    T, H, D = 40, 8, 128
    table = R.rotary_table(400, 128, device=gpu)
    axes = R.rotary_axes((16, 24, 24), device=gpu)
    x = torch.randn(T, H, D, device=gpu).to(torch.bfloat16)
    pos = torch.randint(0, 400, (3, T), device=gpu, dtype=torch.int32)
    want = R.rotary(x, table, pos, axes=axes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(R.rotary(x, table, pos, axes=axes), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = R.rotary(x, table, pos, axes=axes)
    for i in range(3):
        pos.copy_(torch.randint(0, 400, (3, T), device=gpu, dtype=torch.int32))
        x.mul_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, R.rotary(x, table, pos, axes=axes))


@pytest.mark.parametrize("T,H,D,sections,spread,offset,interleaved,dtype", [
    (16400, 7, 128, (16, 24, 24), False, 0, False, torch.bfloat16),  # two threads a unit: four heads, and three
    (16400, 5, 128, (16, 24, 24), True, 0, False, torch.float32),
    (16400, 9, 128, (10, 11, 11), True, 64, True, torch.float16),    # three: three heads each
    (4100, 32, 128, (24, 20, 20), True, 0, False, torch.bfloat16),   # a token a wavefront
    (4100, 30, 128, (64,), False, 0, True, torch.float32),
    (11000, 14, 96, (13, 11), False, 0, False, torch.float16),
])
def test_many_tokens_of_several_heads_a_thread(gpu, T, H, D, sections, spread, offset, interleaved, dtype):
    """Each token as among few, whose threads have a head each; into a new tensor and in place."""
    from sglang_lite_amd import rotary as R

    print(f"axes T={T} H={H} D={D} {sections}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(T + H)
    rot, n = 2 * sum(sections), 5000
    table = R.rotary_table(n, rot, device=gpu)
    freq, _ = R.frequencies(rot)
    axes = R.rotary_axes(sections, spread=spread, device=gpu)
    x = torch.randn(T, H, D, generator=g, device=gpu).to(dtype)
    at = torch.randint(0, n, (len(sections), T), generator=g, device=gpu)
    at[0, T // 2] = -1
    for pos in (at.int(), at):
        kw = dict(axes=axes, interleaved=interleaved, offset=offset)
        y = R.rotary(x, table, pos, **kw)
        for lo in range(0, T, 400):
            few = R.rotary(x[lo:lo + 400].contiguous(), table, pos[:, lo:lo + 400].contiguous(), **kw)
            assert torch.equal(y[lo:lo + 400], few)
        rows = [0, 1, 2, 63, 64, T // 2 - 1, T // 2 + 1, T - 2, T - 1]
        ref = OP.rotate_axes(_host(x[rows]), at[:, rows].cpu().numpy(), axes.cpu().numpy(), freq.numpy(), 1.0, offset,
                             interleaved)
        bound = _bound(_host(x[rows]), rot, offset, interleaved, dtype)
        err = np.abs(_host(y[rows]).astype(np.float64) - ref)
        assert np.all(err <= bound + HALF[dtype] * (np.abs(ref) + bound)), float(err.max())
        assert torch.equal(y[T // 2], x[T // 2])
        z = x.clone()
        assert R.rotary(z, table, pos, out=z, **kw) is z and torch.equal(z, y)


@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("dtype,sections,spread,interleaved", [
    (torch.bfloat16, (40, 44, 44), True, False),
    (torch.float16, (32, 48, 48), False, True),
    (torch.float32, (43, 43, 42), False, False),
])
def test_append_of_blocks_above_512_threads(gpu, block, dtype, sections, spread, interleaved):
    """Heads of 256: two or four units a thread, whose turns share the wavefront's LDS."""
    from sglang_lite_amd import paged_kv as P
    from sglang_lite_amd import rotary as R

    B, H, D, page, n = 3, 2, 256, 128, 700
    rng = np.random.default_rng(block)
    table = R.rotary_table(n, D, device=gpu)
    axes = R.rotary_axes(sections, spread=spread, device=gpu)
    kv = P.PagedKV.empty(20, H, page, D, block=block, device=gpu)
    for c in (kv.k, kv.v):
        c.view(torch.uint8).fill_(0x7F)
    for s in (kv.k_scale, kv.v_scale):
        s.fill_(float("nan"))
    bt = rng.permutation(20)[:B * 5].reshape(B, 5).astype(np.int32)
    codes = [_bytes(c).copy() for c in (kv.k, kv.v)]
    scales = [_host(s).copy() for s in (kv.k_scale, kv.v_scale)]
    have = [0] * B
    for step, new in enumerate(([300, 1, 130], [60, 127, 128], [1, 64, 33])):
        cu = [0] + np.cumsum(new).tolist()
        T = cu[-1]
        g = torch.Generator(device=gpu).manual_seed(step)
        x = (torch.randn(T, 2, H, D, generator=g, device=gpu) * 3).to(dtype)
        pos = torch.randint(0, n, (len(sections), T), generator=g, device=gpu, dtype=torch.int32)
        pos[0, 1], pos[-1, 2], pos[0, 3] = -1, -7, n
        P.append_kv(kv, x[:, 0], x[:, 1], torch.from_numpy(bt).to(gpu),
                    torch.tensor(have, dtype=torch.int32, device=gpu),
                    cu_tokens=torch.tensor(cu, dtype=torch.int32, device=gpu), table=table, positions=pos, axes=axes,
                    interleaved=interleaved)
        at, tab = pos.cpu().numpy(), _host(table)
        rows = tab[np.clip(at, 0, n - 1)[axes.cpu().numpy()].T, np.arange(D // 2)]
        rows[at[axes.cpu().numpy()].T >= n] = np.nan
        rows[(at < 0).any(0)] = (1.0, 0.0)
        OP.append(codes[0], scales[0], OP.rotate_f32(_host(x[:, 0]), rows, 0, interleaved), bt, have, cu)
        OP.append(codes[1], scales[1], _host(x[:, 1]), bt, have, cu)
        have = [h + m for h, m in zip(have, new)]
        np.testing.assert_array_equal(_host(kv.k_scale), scales[0])
        np.testing.assert_array_equal(_host(kv.v_scale), scales[1])
        np.testing.assert_array_equal(_bytes(kv.k), codes[0])
        np.testing.assert_array_equal(_bytes(kv.v), codes[1])
