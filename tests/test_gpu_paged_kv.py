"""Rotary positions, appending to the 8-bit paged cache and the attention over it,
on the GPU against the oracle: codes and scales bit for bit, rotations and
attention within their roundings of float64."""

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


# ------------------------------------------------------------------- rotary


def _rotary_bound(x, freq, length, offset, interleaved, dtype):
    """|error| of a rotated element: cos and sin carry half a step of fp32 each, as do the two
    products and the sum (3 half steps of |a| + |b|, 4 with room for their products), then the
    rounding of the output; below f16's normal range a step is 2^-24."""
    x = np.abs(np.asarray(x, np.float64))
    a, b = OP.pairs(2 * len(freq), offset, interleaved)
    both = (x[..., a] + x[..., b]) * length
    bound = np.zeros_like(x)
    bound[..., a] = bound[..., b] = 4 * 2.0 ** -24 * both
    return bound + (2.0 ** -25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("T,H,D,rot,offset,interleaved,dtype,scaling", [
    (1, 1, 64, 64, 0, False, torch.bfloat16, None),
    (5, 3, 128, 128, 0, True, torch.float16, {"type": "linear", "factor": 4.0}),
    (37, 8, 128, 64, 64, False, torch.float32, {"type": "ntk", "factor": 8.0}),
    (19, 64, 512, 64, 448, True, torch.bfloat16, {"type": "yarn", "factor": 32.0, "original": 4096}),
    (300, 32, 128, 128, 0, False, torch.bfloat16, None),
    (7, 2, 80, 20, 3, False, torch.bfloat16, None),    # single elements
    (6, 5, 33, 10, 1, True, torch.float32, None),
    (4, 1, 2, 2, 0, True, torch.float16, None),
    (9, 6, 24, 16, 0, False, torch.bfloat16, None),    # an odd number of copied chunks
    (2100, 16, 96, 32, 64, True, torch.float32, None),
])
def test_rotary_matches_float64(gpu, T, H, D, rot, offset, interleaved, dtype, scaling):
    from sglang_lite_amd import rotary as R

    print(f"rotary T={T} H={H} D={D} rot={rot}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(T + D)
    n = 131072
    table = R.rotary_table(n, rot, scaling=scaling, device=gpu)
    freq, length = R.frequencies(rot, scaling=scaling)
    x = torch.randn(T, H, D, generator=g, device=gpu).to(dtype)
    at = torch.randint(0, n, (T,), generator=g, device=gpu)
    at[0] = n - 1
    for inverse, pos in ((False, at.int()), (True, at)):
        y = R.rotary(x, table, pos, interleaved=interleaved, offset=offset, inverse=inverse)
        assert y.shape == x.shape and y.dtype == dtype
        ref = OP.rotate(_host(x), at.cpu().numpy(), freq.numpy(), length, offset, interleaved, inverse)
        bound = _rotary_bound(_host(x), freq, length, offset, interleaved, dtype)
        err = np.abs(_host(y).astype(np.float64) - ref)
        assert np.all(err <= bound + HALF[dtype] * (np.abs(ref) + bound)), float(err.max())
        rest = np.ones(D, bool)
        rest[offset:offset + rot] = False
        assert torch.equal(y[..., torch.from_numpy(rest).to(gpu)], x[..., torch.from_numpy(rest).to(gpu)])


def test_rotary_table_angles_of_far_positions(gpu):
    from sglang_lite_amd import rotary as R

    n = 1 << 20
    table = R.rotary_table(n, 64, scaling={"type": "yarn", "factor": 40.0, "original": 4096}, device=gpu)
    freq, length = R.frequencies(64, scaling={"type": "yarn", "factor": 40.0, "original": 4096})
    p = np.array([0, 1, 4095, 65537, n - 2, n - 1])
    angle = p[:, None] * freq.numpy()
    got = table[torch.from_numpy(p).to(gpu)].cpu().numpy().astype(np.float64)
    # half a step of fp32 at up to `length`, and float64's own angle
    tol = 2.0 ** -24 * length * (1 + 2.0 ** -20)
    assert np.abs(got[..., 0] - length * np.cos(angle)).max() <= tol
    assert np.abs(got[..., 1] - length * np.sin(angle)).max() <= tol


def test_rotary_in_place_strided_and_padding(gpu):
    from sglang_lite_amd import rotary as R

    T, H, D = 33, 4, 128
    table = R.rotary_table(512, 64, device=gpu)
    fused = torch.randn(T, 3 * H, D, device=gpu).to(torch.bfloat16)
    q = fused[:, H:2 * H]
    at = torch.randint(0, 512, (T,), device=gpu, dtype=torch.int32)
    want = R.rotary(q.contiguous(), table, at, offset=32)
    before = fused.clone()
    assert torch.equal(R.rotary(q, table, at, offset=32), want)
    got = R.rotary(q, table, at, offset=32, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, want)
    assert torch.equal(fused[:, :H], before[:, :H]) and torch.equal(fused[:, 2 * H:], before[:, 2 * H:])
    # every third element of a buffer, every other position, one head for all (a broadcast input)
    odd = torch.randn(T, H, 3 * D, device=gpu).to(torch.bfloat16)[..., ::3]
    pos2 = torch.stack([at, at], 1)[:, 0]
    assert torch.equal(R.rotary(odd, table, pos2), R.rotary(odd.contiguous(), table, at))
    one = torch.randn(T, 1, D, device=gpu).to(torch.bfloat16)
    assert torch.equal(R.rotary(one.expand(T, H, D), table, at), R.rotary(one, table, at).expand(T, H, D))
    # rows off a 16-byte boundary take the path of single elements
    off = torch.randn(T * H * D + 1, device=gpu).to(torch.bfloat16)[1:].view(T, H, D)
    assert torch.equal(R.rotary(off, table, at, interleaved=True),
                       R.rotary(off.clone(), table, at, interleaved=True))
    # padding rows stay, positions behind the table give NaN in the rotated part alone
    at[3], at[4], at[5] = -1, 512, 2 ** 31 - 1
    x = torch.randn(T, H, D, device=gpu)
    y = R.rotary(x, table, at)
    assert torch.equal(y[3], x[3])
    assert torch.isnan(y[4:6, :, :64]).all() and torch.equal(y[4:6, :, 64:], x[4:6, :, 64:])


def test_rotary_inverse_is_the_gradient(gpu):
    """Of L = sum(w * rotary(x)): rotary(w, inverse), against the formula and differences."""
    from sglang_lite_amd import rotary as R

    T, H, D = 4, 2, 32
    scaling = {"type": "yarn", "factor": 4.0, "original": 64}
    table = R.rotary_table(256, 32, scaling=scaling, device=gpu)
    at = torch.tensor([0, 3, 200, 255], device=gpu)
    x, w = torch.randn(2, T, H, D, device=gpu)
    for inter in (False, True):
        grad = R.rotary(w, table, at, interleaved=inter, inverse=True).double()
        base = R.rotary(x, table, at, interleaved=inter).double()
        for e in (0, 1, 15, 16, 17, 31):
            step = torch.zeros_like(x)
            step[..., e] = 1.0
            more = R.rotary(x + step, table, at, interleaved=inter).double()
            diff = (w.double() * (more - base)).sum(-1)
            # the map is linear: the difference is exact but for fp32 roundings of values below 16
            assert (diff - grad[..., e]).abs().max() <= 32 * 16 * 2.0 ** -23


# ------------------------------------------------------------------- append


class Cache:
    """A cache, its block table, and the oracle's copy of it."""

    def __init__(self, dev, B, tokens, H, D, page, block, seed, spare=3):
        from sglang_lite_amd import paged_kv as P

        self.P, self.dev = P, dev
        rng = np.random.default_rng(seed)
        cols = -(-tokens // page) + 1
        pages = B * cols + spare
        self.kv = P.PagedKV.empty(pages, H, page, D, block=block, device=dev)
        for c in (self.kv.k, self.kv.v):  # what was never written: NaN codes and scales
            c.view(torch.uint8).fill_(0x7F)
        self.kv.k_scale.fill_(float("nan"))
        self.kv.v_scale.fill_(float("nan"))
        self.table = rng.permutation(pages)[:B * cols].reshape(B, cols).astype(np.int32)
        self.bt = torch.from_numpy(self.table).to(dev)
        self.k, self.v = _bytes(self.kv.k).copy(), _bytes(self.kv.v).copy()
        self.ks, self.vs = _host(self.kv.k_scale).copy(), _host(self.kv.v_scale).copy()

    def append(self, k, v, start, cu, rot=None, table=None, **kw):
        st = torch.tensor(start, dtype=torch.int32, device=self.dev)
        cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=self.dev)
        self.P.append_kv(self.kv, k, v, self.bt, st, cu_tokens=cut, table=table, **kw)
        cu = list(range(len(start) + 1)) if cu is None else cu
        kf, vf = _host(k), _host(v)
        if table is not None:
            at = np.zeros(len(kf), np.int64)
            for b in range(len(start)):
                at[cu[b]:cu[b + 1]] = start[b] + np.arange(cu[b + 1] - cu[b])
            if kw.get("positions") is not None:
                at = kw["positions"].cpu().numpy()
            rows = _host(table)[np.clip(at, 0, len(table) - 1)]
            rows[at >= len(table)] = np.nan
            rows[at < 0] = (1.0, 0.0)
            kf = OP.rotate_f32(kf, rows, kw.get("offset", 0), kw.get("interleaved", False))
        OP.append(self.k, self.ks, kf, self.table, start, cu)
        OP.append(self.v, self.vs, vf, self.table, start, cu)

    def check(self):
        np.testing.assert_array_equal(_host(self.kv.k_scale), self.ks)
        np.testing.assert_array_equal(_host(self.kv.v_scale), self.vs)
        np.testing.assert_array_equal(_bytes(self.kv.k), self.k)
        np.testing.assert_array_equal(_bytes(self.kv.v), self.v)


def _new(dev, T, H, D, dtype, seed, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    size = torch.exp2(spread * torch.randn(T, 1, 1, 1, generator=g, device=dev))
    x = torch.randn(T, 2, H, D, generator=g, device=dev) * size
    x = x.to(dtype)
    return x[:, 0], x[:, 1]  # views of one buffer


APPEND = [
    # B, H, D, page, block, dtype, rot, offset, interleaved
    (3, 2, 64, 16, 16, torch.bfloat16, 64, 0, False),
    (4, 1, 128, 64, 16, torch.float16, 64, 64, True),
    (2, 8, 128, 64, 64, torch.bfloat16, 128, 0, False),
    (3, 3, 80, 32, 32, torch.float32, 16, 8, False),
    (2, 2, 256, 128, 128, torch.bfloat16, 128, 0, True),
    (5, 2, 16, 16, 16, torch.bfloat16, 16, 0, True),
    (70, 1, 96, 32, 16, torch.float16, 0, 0, False),
]


@pytest.mark.parametrize("B,H,D,page,block,dtype,rot,offset,interleaved", APPEND)
def test_append_matches_the_oracle_bit_for_bit(gpu, B, H, D, page, block, dtype, rot, offset, interleaved):
    """Chunks of odd lengths, then single tokens, then chunks again: blocks that begin, continue,
    grow in scale and end inside a chunk."""
    from sglang_lite_amd import rotary as R

    print(f"append B={B} H={H} D={D} page={page} block={block}", flush=True)
    rng = np.random.default_rng(B + D)
    c = Cache(gpu, B, 330, H, D, page, block, seed=D)
    table = R.rotary_table(400, rot, device=gpu) if rot else None
    kw = dict(table=table, interleaved=interleaved, offset=offset) if rot else {}
    have = [0] * B
    for step in range(5):
        if step in (1, 2):
            cu = None
            new = [1] * B
        else:
            new = [int(rng.integers(0, 90)) for _ in range(B)]
            new[0] = (0, 0, 0, 1, 77)[step]
            cu = [0] + np.cumsum(new).tolist()
        T = sum(new)
        k, v = _new(gpu, max(T, 1), H, D, dtype, seed=step)
        c.append(k[:T], v[:T], have, cu, **kw)
        have = [h + n for h, n in zip(have, new)]
        c.check()
    # speculative tokens taken back: the next ones overwrite them
    have = [max(0, h - 5) for h in have]
    k, v = _new(gpu, B, H, D, dtype, seed=99, spread=4.0)
    c.append(k, v, have, None, **kw)
    c.check()


def test_append_values_at_the_scale_borders(gpu):
    """Zeros, the smallest and largest magnitudes, 448 times a power of two and its neighbours,
    NaN and infinities."""
    H, D = 1, 16
    c = Cache(gpu, 1, 512, H, D, 16, 16, seed=1)
    rows = np.zeros((9 * 16, H, D), np.float32)
    specials = [0.0, 448.0, np.nextafter(np.float32(448), np.float32(1e9)), np.nextafter(np.float32(448), np.float32(0)),
                3.4e38, 1e-38, 2.0 ** -100 * 448, 7.0 * 2.0 ** -110, 2.0 ** 120 * 300]
    for i, s in enumerate(specials):
        rows[16 * i + 3] = np.linspace(-s, s, D, dtype=np.float32)
        rows[16 * i + 5, :, 2] = s
    rows[20, 0, 4], rows[21, 0, 5], rows[22, 0, 6] = np.nan, np.inf, -np.inf
    rows[8 * 16, 0, :3] = np.inf, -np.inf, np.nan
    x = torch.from_numpy(rows).to(gpu)
    c.append(x, -x, [0], [0, len(rows)])
    c.check()
    # a growing scale over codes that hold NaN, then a block of nothing finite
    c.append(x[16:19] * 0 + 1.0, x[16:19], [16 * 9], [0, 3])
    c.append(torch.full_like(x[:1], float("nan")), x[1:2], [16 * 9 + 3], [0, 1])
    c.append(x[:1] + 1e6, x[:1] - 1e9, [16 * 9 + 4], [0, 1])
    c.append(torch.full_like(x[:16], float("inf")), torch.full_like(x[:16], float("nan")), [16 * 10], [0, 16])
    c.check()


def test_append_skips_what_has_no_place(gpu):
    """Rows behind the last sequence, tokens behind the table, entries that are no page, a negative
    start, an empty sequence, and a sequence between two others that is skipped."""
    H, D, page, block = 2, 64, 32, 16
    c = Cache(gpu, 5, 64, H, D, page, block, seed=5)
    c.table[1, 1] = -1
    c.table[2, 0] = 10 ** 6
    c.bt = torch.from_numpy(c.table).to(gpu)
    k, v = _new(gpu, 200, H, D, torch.bfloat16, seed=3)
    cols = c.table.shape[1]
    cu = [0, 40, 90, 100, 100, 130]
    start = [page * cols - 20, 10, 0, 7, -4]
    st = torch.tensor(start, dtype=torch.int32, device=gpu)
    c.P.append_kv(c.kv, k, v, c.bt, st, cu_tokens=torch.tensor(cu, dtype=torch.int32, device=gpu))
    # a block that the table does not hold whole is skipped whole: the last 20 tokens fit, and end
    # on the table's last block border
    kf, vf = _host(k), _host(v)
    OP.append(c.k, c.ks, kf, c.table, start, cu)
    OP.append(c.v, c.vs, vf, c.table, start, cu)
    c.check()


def test_append_positions_and_tables_of_their_own(gpu):
    from sglang_lite_amd import rotary as R

    table = R.rotary_table(100, 32, device=gpu)
    c = Cache(gpu, 2, 64, 2, 64, 16, 16, seed=6)
    k, v = _new(gpu, 9, 2, 64, torch.bfloat16, seed=4)
    pos = torch.tensor([5, -1, 99, 100, 3, 3, 2 ** 30, 0, 7], dtype=torch.int32, device=gpu)
    c.append(k, v, [3, 0], [0, 4, 9], table=table, positions=pos, offset=16)
    c.check()


# ---------------------------------------------------------------- attention


def _filled(dev, lens, H, D, page, block, seed, spread=1.0):
    """A cache holding lens[b] random tokens of each sequence."""
    c = Cache(dev, len(lens), max(list(lens) + [1]), H, D, page, block, seed)
    cu = [0] + np.cumsum(lens).tolist()
    if cu[-1]:
        k, v = _new(dev, cu[-1], H, D, torch.float32, seed, spread)
        st = torch.zeros(len(lens), dtype=torch.int32, device=dev)
        c.P.append_kv(c.kv, k, v, c.bt, st, cu_tokens=torch.tensor(cu, dtype=torch.int32, device=dev))
    c.k, c.v = _bytes(c.kv.k).copy(), _bytes(c.kv.v).copy()
    c.ks, c.vs = _host(c.kv.k_scale).copy(), _host(c.kv.v_scale).copy()
    return c


def _attention(c, q, lens, cu, scale, **kw):
    """Oracle over the batch: (o, bound) with NaN where the definition gives NaN."""
    n_rows, Hq, D = q.shape
    o, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(len(lens)):
        r0, r1 = cu[b], cu[b + 1]
        if r1 <= r0:
            continue
        L = min(lens[b], c.table.shape[1] * c.k.shape[2])
        kr, there = OP.rows(c.k, c.ks, c.table[b], L)
        vr, _ = OP.rows(c.v, c.vs, c.table[b], L)
        y, size, reach = OP.attention(q[r0:r1], kr, vr, there, L - (r1 - r0), scale, **kw)
        o[r0:r1] = y
        # a weight: rounded to f16 for the product (2^-11 relative at most, or 2^-25 of the row's
        # reference; 2^-8 is what bf16 would take), its score an fp32 sum
        # of D products (a step of 2^-23 each at most), then in log2 units and through exp2
        # (2^-20 with the sums over keys); normaliser and numerator both carry the score's error
        score = 2 * (D + 8) * 2.0 ** -23 * reach
        bound[r0:r1] = size * (2.0 ** -8 + score + 2.0 ** -18)
    return o, bound


def _check_attn(c, q, lens, cu, out=None, dtype=None, **kw):
    dev = c.dev
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    args = dict(kw)
    if args.get("sink") is not None:
        args["sink"] = torch.from_numpy(args["sink"]).to(dev)
    scale = args.pop("softmax_scale", None)
    kw.pop("softmax_scale", None)
    o = c.P.paged_attn(q, c.kv, c.bt, lt, cu_tokens=cut, softmax_scale=scale, out=out, **args)
    assert o.dtype == q.dtype and o.shape == q.shape
    cu = list(range(len(lens) + 1)) if cu is None else cu
    D = q.shape[2]
    ref, bound = _attention(c, _host(q), lens, cu, D ** -0.5 if scale is None else scale, **kw)
    got = _host(o).astype(np.float64)[:cu[-1]]
    ref, bound = ref[:cu[-1]], bound[:cu[-1]]
    nan = np.isnan(ref)
    np.testing.assert_array_equal(np.isnan(got), nan)
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    tol = np.where(nan, 1.0, bound + HALF[q.dtype] * (np.abs(ref) + bound) + tiny)
    err = np.where(nan, 0.0, np.abs(got - ref))
    worst = float((err / np.maximum(tol, 1e-300)).max()) if err.size else 0.0
    print(f"  worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0
    return o


def _queries(dev, T, Hq, D, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(T, Hq, D, generator=g, device=dev).to(dtype)


DECODE = [
    # lens, Hq, Hkv, D, page, block, dtype, window, sink
    ([1], 1, 1, 16, 16, 16, torch.bfloat16, 0, False),
    ([0, 1, 15, 16, 17, 31, 32, 33], 4, 2, 64, 16, 16, torch.bfloat16, 0, False),
    ([63, 64, 65, 127, 128, 129, 255, 257], 8, 1, 128, 64, 32, torch.float16, 0, True),
    ([500], 32, 8, 128, 64, 64, torch.bfloat16, 0, False),
    ([1000, 3, 0, 700], 8, 8, 96, 32, 16, torch.bfloat16, 0, False),
    ([700, 129, 40], 32, 2, 256, 128, 128, torch.bfloat16, 0, True),
    ([900, 31, 300], 20, 1, 80, 64, 16, torch.float16, 100, True),
    ([2000], 64, 1, 144, 16, 16, torch.bfloat16, 1, False),
    ([5000, 40], 6, 2, 128, 1024, 64, torch.bfloat16, 4999, False),
]


@pytest.mark.parametrize("lens,Hq,Hkv,D,page,block,dtype,window,sink", DECODE)
def test_decode_attention_matches_float64(gpu, lens, Hq, Hkv, D, page, block, dtype, window, sink):
    print(f"decode lens={lens} Hq={Hq} Hkv={Hkv} D={D} page={page}", flush=True)
    c = _filled(gpu, lens, Hkv, D, page, block, seed=D + Hq)
    q = _queries(gpu, len(lens), Hq, D, dtype, 7)
    s = (np.random.default_rng(1).standard_normal(Hq) * 2).astype(np.float32) if sink else None
    _check_attn(c, q, lens, None, window=window, sink=s)


CHUNKS = [
    # new, lens, Hq, Hkv, D, page, block, dtype, causal, window, sink
    ([4, 4, 4], [4, 77, 300], 8, 2, 128, 64, 64, torch.bfloat16, True, 0, False),
    ([1, 0, 33, 2], [50, 9, 33, 400], 4, 4, 64, 16, 16, torch.float16, True, 0, True),
    ([130, 17], [130, 280], 6, 2, 128, 32, 16, torch.bfloat16, True, 0, False),
    ([65, 200], [300, 200], 8, 2, 64, 64, 32, torch.bfloat16, True, 50, True),
    ([40, 3], [100, 260], 4, 1, 256, 64, 64, torch.bfloat16, True, 0, False),
    ([40, 3, 1], [100, 260, 0], 5, 5, 80, 16, 16, torch.float16, False, 0, False),
    ([70, 5], [30, 0], 4, 2, 128, 64, 64, torch.bfloat16, True, 0, False),  # more queries than keys
    ([70, 5], [30, 2], 4, 2, 96, 64, 64, torch.bfloat16, True, 3, True),
    ([257], [700], 16, 1, 192, 128, 64, torch.bfloat16, True, 0, False),
]


@pytest.mark.parametrize("new,lens,Hq,Hkv,D,page,block,dtype,causal,window,sink", CHUNKS)
def test_chunk_attention_matches_float64(gpu, new, lens, Hq, Hkv, D, page, block, dtype, causal, window, sink):
    print(f"chunks new={new} lens={lens} Hq={Hq} Hkv={Hkv} D={D} page={page}", flush=True)
    c = _filled(gpu, lens, Hkv, D, page, block, seed=D + Hq)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], Hq, D, dtype, 8)
    s = (np.random.default_rng(2).standard_normal(Hq) * 2).astype(np.float32) if sink else None
    _check_attn(c, q, lens, cu, causal=causal, window=window, sink=s)


@pytest.mark.parametrize("new,lens,window,D,dtype", [
    ([513], [700], 0, 64, torch.bfloat16),
    ([1, 500, 20], [90, 500, 333], 100, 128, torch.float16),
])
def test_chunks_of_many_row_tiles(gpu, new, lens, window, D, dtype):
    """Enough row tiles to fill the device without sharing any."""
    c = _filled(gpu, lens, 8, D, 32, 32, seed=D)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], 128, D, dtype, 8)
    s = (np.random.default_rng(2).standard_normal(128) * 2).astype(np.float32)
    _check_attn(c, q, lens, cu, window=window, sink=s)


def test_attention_leaves_rows_behind_the_last_sequence(gpu):
    c = _filled(gpu, [40, 70], 2, 64, 16, 16, seed=2)
    q = _queries(gpu, 20, 4, 64, torch.bfloat16, 3)
    out = torch.full_like(q, 7.0)
    o = _check_attn(c, q, [40, 70], [0, 3, 11], out=out)
    assert o.data_ptr() == out.data_ptr() and bool((out[11:] == 7.0).all())


def test_attention_entries_that_are_no_page_and_lengths_past_the_table(gpu):
    lens = [300, 200, 90]
    c = _filled(gpu, lens, 2, 128, 16, 16, seed=9)
    c.table[0, 3] = -1
    c.table[0, 18] = -1     # its last page
    c.table[1, 2] = 1 << 30
    c.table[2, :] = -5      # a sequence without any
    c.bt = torch.from_numpy(c.table).to(gpu)
    for new in ([1, 1, 1], [20, 3, 40]):
        cu = [0] + np.cumsum(new).tolist()
        q = _queries(gpu, cu[-1], 8, 128, torch.bfloat16, 4)
        _check_attn(c, q, lens, cu)
    # more keys than the table can hold: cut to it (all of the table is filled first)
    cap = c.table.shape[1] * 16
    c2 = _filled(gpu, [cap - 16], 1, 64, 16, 16, seed=10)
    k, v = _new(gpu, 16, 1, 64, torch.float32, 5)
    c2.append(k, v, [cap - 16], [0, 16])
    q = _queries(gpu, 1, 4, 64, torch.bfloat16, 4)
    _check_attn(c2, q, [cap + 500], None)


@pytest.mark.parametrize("new,window", [([1], 40), ([6], 0), ([30], 0), ([150], 0), ([150], 60)])
def test_nan_and_infinity_reach_only_the_rows_that_see_them(gpu, new, window):
    """A NaN value or key in the cache is NaN for the queries that see it and nothing for the
    others: behind their own position, before their window, in the same tile or not."""
    L, H, D = 200, 2, 128
    c = _filled(gpu, [L], H, D, 64, 16, seed=11)
    at = lambda t: (int(c.table[0, t // 64]), t % 64)  # noqa: E731
    n = new[0]
    for t, h, d in ((L - 1, 0, 3), (L - n // 2 - 1, 1, 70), (100, 0, 9)):
        p, spot = at(t)
        c.kv.v.view(torch.uint8)[p, h, spot, d] = 0xFF
        c.v[p, h, spot, d] = 0xFF
    if window:
        p, spot = at(L - window - 1)
        c.kv.k.view(torch.uint8)[p, 1, spot, 5] = 0x7F
        c.k[p, 1, spot, 5] = 0x7F
    q = _queries(gpu, n, 8, D, torch.bfloat16, 5)
    _check_attn(c, q, [L], [0, n], window=window)


def _widen(c, tokens):
    """A block table for so many tokens a sequence, the new entries no page: long tables have
    the keys of an item shared between workgroups, short ones do not."""
    B, old = c.table.shape
    t = np.full((B, max(old, -(-tokens // c.k.shape[2]))), -1, dtype=c.table.dtype)
    t[:, :old] = c.table
    c.table, c.bt = t, torch.from_numpy(t).to(c.dev)


@pytest.mark.parametrize("new,lens,Hq,Hkv,D,page,block,dtype,causal,window,sink", CHUNKS + [
    ([1] * len(lens), lens, Hq, Hkv, D, page, block, dtype, True, window, sink)
    for lens, Hq, Hkv, D, page, block, dtype, window, sink in DECODE])
def test_attention_shared_between_workgroups(gpu, new, lens, Hq, Hkv, D, page, block, dtype, causal, window, sink):
    print(f"shared new={new} lens={lens} Hq={Hq} Hkv={Hkv} D={D} page={page}", flush=True)
    c = _filled(gpu, lens, Hkv, D, page, block, seed=D + Hq)
    _widen(c, 16384)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], Hq, D, dtype, 8)
    s = (np.random.default_rng(2).standard_normal(Hq) * 2).astype(np.float32) if sink else None
    _check_attn(c, q, lens, cu, causal=causal, window=window, sink=s)


@pytest.mark.parametrize("D,Hq,Hkv,new", [(128, 8, 2, 16), (128, 8, 2, 17), (64, 4, 1, 16), (64, 4, 1, 17),
                                          (256, 8, 4, 8), (256, 8, 4, 9), (128, 4, 1, 64), (128, 4, 1, 65),
                                          (128, 8, 2, 24), (128, 8, 2, 25), (64, 4, 1, 24), (64, 4, 1, 25),
                                          (256, 8, 4, 16), (256, 8, 4, 17)])
@pytest.mark.parametrize("tokens", [1024, 1040, 2048, 2064, 4200])
def test_attention_on_both_sides_of_its_choices(gpu, D, Hq, Hkv, new, tokens):
    """The most rows that count as few and one token more, one row tile and two; tables that
    hold as much as an item that is not shared, and a page more."""
    lens = [tokens // 4, 70, 333]
    c = _filled(gpu, lens, Hkv, D, 16, 16, seed=D)
    _widen(c, tokens)
    cu = [0, new, 2 * new, 3 * new]
    q = _queries(gpu, cu[-1], Hq, D, torch.bfloat16, 6)
    _check_attn(c, q, lens, cu)


@pytest.mark.parametrize("tokens", [0, 16384])
@pytest.mark.parametrize("new", [1, 3])
def test_attention_of_many_short_sequences(gpu, new, tokens):
    """More sequences than a wavefront has lanes, some without keys or queries."""
    rng = np.random.default_rng(6)
    lens = rng.integers(0, 200, 150).tolist()
    n = [new if i % 7 else 0 for i in range(150)]
    c = _filled(gpu, lens, 2, 64, 16, 16, seed=12)
    _widen(c, tokens)
    cu = [0] + np.cumsum(n).tolist()
    q = _queries(gpu, cu[-1] + 3, 8, 64, torch.float16, 6)
    _check_attn(c, q, lens, cu)


@pytest.mark.parametrize("tokens", [0, 1500, 16384])
@pytest.mark.parametrize("D,Hq,Hkv,dtype", [(128, 8, 2, torch.bfloat16), (64, 40, 2, torch.float16),
                                            (256, 6, 2, torch.bfloat16)])
def test_single_tokens_beside_prompts(gpu, D, Hq, Hkv, dtype, tokens):
    """Chunks and few rows in one batch: no row is missed or taken twice, whichever kernel is its."""
    new = [1, 300, 0, 1, 16, 17, 1, 2, 0, 130, 1, 3]
    lens = [700, 300, 50, 0, 16, 400, 65, 1, 0, 290, 513, 40]
    c = _filled(gpu, lens, Hkv, D, 32, 16, seed=D)
    _widen(c, tokens)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1] + 2, Hq, D, dtype, 4)
    s = (np.random.default_rng(2).standard_normal(Hq) * 2).astype(np.float32)
    out = torch.full_like(q, 7.0)
    _check_attn(c, q, lens, cu, sink=s, window=450, out=out)
    assert bool((out[cu[-1]:] == 7.0).all())


def test_many_single_tokens_beside_prompts(gpu):
    """More sequences than a wavefront has lanes, prompts among the first, the last and between."""
    rng = np.random.default_rng(3)
    new = [400 if b in (0, 70, 139) else int(rng.integers(0, 3)) for b in range(140)]
    lens = [n + int(rng.integers(0, 90)) for n in new]
    assert sum(new) * 16 // 140 > 96  # (rows on average: a batch of chunks)
    c = _filled(gpu, lens, 1, 128, 16, 16, seed=21)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], 16, 128, torch.bfloat16, 4)
    for tokens in (0, 16384):
        _widen(c, tokens)
        _check_attn(c, q, lens, cu)


@pytest.mark.parametrize("new", [2, 150])
def test_windows_past_every_length(gpu, new):
    """A window of 2^31 - 1 and more, with more queries than keys."""
    lens = [new // 2, new + 30]
    c = _filled(gpu, lens, 1, 128, 16, 16, seed=13)
    q = _queries(gpu, 2 * new, 4, 128, torch.bfloat16, 6)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 40):
        _check_attn(c, q, lens, [0, new, 2 * new], window=window)


@pytest.mark.parametrize("D,new,window,tokens", [(64, 150, 60, 0), (256, 150, 60, 0), (256, 5, 0, 4096),
                                                 (64, 4, 0, 4096), (128, 150, 60, 16384), (256, 40, 60, 16384)])
def test_nan_stays_with_its_rows_at_every_width(gpu, D, new, window, tokens):
    L = 200
    c = _filled(gpu, [L], 2, D, 64, 16, seed=11)
    for t, h, d in ((L - 1, 0, 3), (L - new // 2 - 1, 1, D - 6), (100, 0, 9)):
        p, spot = int(c.table[0, t // 64]), t % 64
        c.kv.v.view(torch.uint8)[p, h, spot, d] = 0x7F
        c.v[p, h, spot, d] = 0x7F
    _widen(c, tokens)
    q = _queries(gpu, new, 8, D, torch.bfloat16, 5)
    _check_attn(c, q, [L], [0, new], window=window)


def test_attention_of_large_scores_and_few_survivors(gpu):
    """Scores of hundreds, so that one key takes all and the reference moves often; a query of
    zeros; a scale of its own; a query row that is not finite."""
    c = _filled(gpu, [600, 45], 2, 64, 32, 32, seed=12, spread=3.0)
    q = _queries(gpu, 2, 8, 64, torch.bfloat16, 6) * 20
    q[1, 3] = 0
    _check_attn(c, q, [600, 45], None, softmax_scale=0.5)
    q[0, 2, 5] = float("nan")
    o = c.P.paged_attn(q, c.kv, c.bt, torch.tensor([600, 45], dtype=torch.int32, device=gpu))
    bad = torch.isnan(o).any(-1)
    assert bad[0, 2] and int(bad.sum()) == 1


@pytest.mark.parametrize("new", [1, 50])
def test_strided_and_misaligned_queries(gpu, new):
    c = _filled(gpu, [90], 2, 64, 16, 16, seed=13)
    lens = torch.tensor([90], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, new], dtype=torch.int32, device=gpu)
    base = _queries(gpu, new, 8, 64, torch.bfloat16, 7)
    want = c.P.paged_attn(base, c.kv, c.bt, lens, cu_tokens=cu)
    wide = torch.zeros(new, 20, 64, dtype=torch.bfloat16, device=gpu)
    wide[:, 2:18:2] = base
    off = torch.zeros(base.numel() + 1, dtype=torch.bfloat16, device=gpu)[1:].view_as(base)
    off.copy_(base)
    odd = torch.zeros(new, 8, 128, dtype=torch.bfloat16, device=gpu)[..., ::2]
    odd.copy_(base)
    heads_first = base.transpose(0, 1).contiguous().transpose(0, 1)
    for q in (wide[:, 2:18:2], off, odd, heads_first):
        assert torch.equal(c.P.paged_attn(q, c.kv, c.bt, lens, cu_tokens=cu), want)


def test_cache_offsets_past_32_bits(gpu):
    """Pages beyond 4 GiB of codes: written and read at their own place."""
    from sglang_lite_amd import paged_kv as P

    H, D, page = 8, 128, 64
    pages = (1 << 32) // (H * page * D) + 40
    kv = P.PagedKV.empty(pages, H, page, D, device=gpu)
    lens = [150, 70]
    ids = [[pages - 1, 0, pages - 3], [pages - 7, pages - 2, 5]]
    bt = torch.tensor(ids, dtype=torch.int32, device=gpu)
    k, v = _new(gpu, 220, H, D, torch.bfloat16, 8)
    cu = torch.tensor([0, 150, 220], dtype=torch.int32, device=gpu)
    zero = torch.zeros(2, dtype=torch.int32, device=gpu)
    P.append_kv(kv, k, v, bt, zero, cu_tokens=cu)
    small = P.PagedKV.empty(6, H, page, D, device=gpu)
    near = torch.arange(6, dtype=torch.int32, device=gpu).view(2, 3)
    P.append_kv(small, k, v, near, zero, cu_tokens=cu)
    lt = torch.tensor(lens, dtype=torch.int32, device=gpu)
    q = _queries(gpu, 2, 32, D, torch.bfloat16, 9)
    assert torch.equal(P.paged_attn(q, kv, bt, lt), P.paged_attn(q, small, near, lt))
    q = _queries(gpu, 60, 32, D, torch.bfloat16, 9)
    c2 = torch.tensor([0, 50, 60], dtype=torch.int32, device=gpu)
    assert torch.equal(P.paged_attn(q, kv, bt, lt, cu_tokens=c2), P.paged_attn(q, small, near, lt, cu_tokens=c2))


def test_the_same_call_gives_the_same_bits(gpu):
    """On another stream, and with sequences of other lengths around it that move the seams."""
    c = _filled(gpu, [3000, 17, 900], 2, 128, 64, 64, seed=14)
    q = _queries(gpu, 3, 16, 128, torch.bfloat16, 10)
    lens = torch.tensor([3000, 17, 900], dtype=torch.int32, device=gpu)
    want = c.P.paged_attn(q, c.kv, c.bt, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.P.paged_attn(q, c.kv, c.bt, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


# ------------------------------------------------------------- used together


def _step(P, R, kv, bt, table, q, k, v, start, lens, cu):
    pos = None
    if cu is None:
        pos = start
    else:
        row = torch.arange(q.shape[0], device=q.device, dtype=torch.int32)
        seq = torch.bucketize(row, cu[1:], right=True).clamp_max(start.numel() - 1)
        pos = (start[seq] + row - cu[seq]).int()
    qr = R.rotary(q, table, pos)
    P.append_kv(kv, k, v, bt, start, cu_tokens=cu, table=table)
    return P.paged_attn(qr, kv, bt, lens, cu_tokens=cu)


def test_prefill_then_decode_as_a_server_does(gpu):
    """Two prompts in ragged chunks, then decode steps: every output against float64 attention over
    the cache as it is then, and the cache against the oracle's."""
    from sglang_lite_amd import rotary as R

    B, Hq, H, D, page = 2, 8, 2, 64, 16
    c = Cache(gpu, B, 200, H, D, page, 16, seed=20)
    table = R.rotary_table(256, D, device=gpu)
    freq, length = R.frequencies(D)
    have = [0, 0]
    for i, new in enumerate([[37, 5], [20, 60], [1, 1], [1, 1], [3, 1], [1, 1]]):
        cu = [0] + np.cumsum(new).tolist()
        T = cu[-1]
        q = _queries(gpu, T, Hq, D, torch.bfloat16, 30 + i)
        k, v = _new(gpu, T, H, D, torch.bfloat16, 40 + i)
        pos = torch.cat([torch.arange(h, h + n) for h, n in zip(have, new)]).int().to(gpu)
        qr = R.rotary(q, table, pos)
        c.append(k, v, have, None if new == [1, 1] else cu, table=table)
        c.check()
        have = [h + n for h, n in zip(have, new)]
        _check_attn(c, qr, have, None if new == [1, 1] else cu)


@pytest.mark.parametrize("new", [1, 3])
def test_a_captured_step_replays_with_other_lengths(gpu, new):
    from sglang_lite_amd import paged_kv as P
    from sglang_lite_amd import rotary as R

    B, Hq, H, D, page = 3, 8, 2, 128, 32
    table = R.rotary_table(1024, D, device=gpu)
    bt = torch.arange(B * 20, dtype=torch.int32, device=gpu).view(B, 20)
    T = B * new
    q, k, v = _queries(gpu, T, Hq, D, torch.bfloat16, 1), *_new(gpu, T, H, D, torch.bfloat16, 2)
    cu = None if new == 1 else torch.arange(0, T + 1, new, dtype=torch.int32, device=gpu)
    start = torch.zeros(B, dtype=torch.int32, device=gpu)
    lens = start + new
    one, two = (P.PagedKV.empty(B * 20, H, page, D, block=32, device=gpu) for _ in range(2))
    for x in (*one, *two):
        x.view(torch.uint8).fill_(0x7F)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(P, R, two, bt, table, q, k, v, start, lens, cu)  # loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x in two:
        x.view(torch.uint8).fill_(0x7F)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(P, R, one, bt, table, q, k, v, start, lens, cu)
    have = torch.tensor([0, 40, 300], dtype=torch.int32, device=gpu)
    for kv in (one, two):  # earlier tokens
        kk, vv = _new(gpu, 340, H, D, torch.bfloat16, 5)
        P.append_kv(kv, kk, vv, bt, torch.zeros_like(have),
                    cu_tokens=torch.tensor([0, 0, 40, 340], dtype=torch.int32, device=gpu), table=table)
    for i in range(6):
        q.copy_(_queries(gpu, T, Hq, D, torch.bfloat16, 50 + i))
        kk, vv = _new(gpu, T, H, D, torch.bfloat16, 60 + i)
        k.copy_(kk)
        v.copy_(vv)
        start.copy_(have + i * new)
        lens.copy_(start + new)
        graph.replay()
        want = _step(P, R, two, bt, table, q, k, v, start, lens, cu)
        torch.cuda.synchronize()
        assert torch.equal(held, want), f"replay {i}"
        for x, y in zip(one, two):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), f"replay {i}"


def test_calls_on_two_streams_at_once(gpu):
    c = _filled(gpu, [2000, 700], 2, 128, 64, 64, seed=15)
    lens = torch.tensor([2000, 700], dtype=torch.int32, device=gpu)
    qs = [_queries(gpu, 2, 16, 128, torch.bfloat16, 70 + i) for i in range(8)]
    want = [c.P.paged_attn(q, c.kv, c.bt, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(c.P.paged_attn(q, c.kv, c.bt, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
