"""The norms, gate and residual sum between two blocks on the GPU: within the roundings of
fp32 arithmetic of float64, and the codes bit for bit those of the fp32 result."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import norms as ON
from oracle import quant as OQ

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
FLOOR = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}  # below f16's normal range a step is 2^-24


def _host(t):
    return None if t is None else t.detach().to(F32).cpu().numpy()


def _inputs(dev, T, H, dtype, res, after, gate, wtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=dev)

    x = (randn(T, H) * torch.exp2(2 * randn(T, 1))).to(dtype)
    r = (3 * randn(T, H)).to(res)
    w = (1 + 0.3 * randn(H)).to(wtype)
    v = (1 + 0.3 * randn(H)).to(wtype) if after else None
    m = None if gate is None else torch.tanh(randn(*((H,) if gate == "vector" else (T, H)))).to(wtype)
    return x, r, w, v, m


def _near(got, ref, bound, dtype):
    err = np.abs(_host(got).astype(np.float64) - ref)
    assert np.all(err <= bound + HALF[dtype] * (np.abs(ref) + bound) + FLOOR[dtype]), float(err.max())


@pytest.mark.parametrize("T,H,dtype,res,after,gate,wtype", [
    (1, 1, F32, F32, True, "rows", F32),
    (3, 7, BF16, BF16, False, None, BF16),
    (5, 64, F16, F32, True, "vector", F16),
    (2, 513, BF16, F32, True, "rows", F32),
    (700, 1000, BF16, BF16, True, "rows", BF16),
    (9, 2047, F32, F32, False, "vector", F32),
    (300, 2048, F16, F16, True, None, F32),
    (4, 2049, BF16, BF16, False, "rows", F32),       # two units a thread
    (900, 4096, BF16, BF16, True, "vector", F32),    # more rows than workgroups
    (33, 4100, BF16, F32, True, "rows", BF16),
    (17, 7168, BF16, F32, True, "rows", F32),
    (6, 8192, F32, F32, True, "rows", F32),
    (600, 8200, BF16, BF16, True, "vector", F32),    # weights not kept
    (3, 16384, F32, F32, True, "rows", F32),
    (5, 16383, BF16, F32, False, None, F32),
])
def test_norms_match_float64(gpu, T, H, dtype, res, after, gate, wtype):
    from sglang_lite_amd.norms import residual_norm

    print(f"norm T={T} H={H} {dtype} {res} {after} {gate}", flush=True)
    x, r, w, v, m = _inputs(gpu, T, H, dtype, res, after, gate, wtype, seed=T + H)
    for scale, eps in ((1.0, 1e-6), (-0.37, 1e-2)):
        h, y = residual_norm(x, r, w, after=v, gate=m, scale=scale, eps=eps)
        assert h.dtype == res and y.dtype == dtype and h.shape == y.shape == x.shape
        scale32 = float(np.float32(scale))
        ho, dh, yo, dy = ON.residual_norm(_host(x), _host(r), _host(w), _host(v), _host(m), scale32,
                                          float(np.float32(eps)))
        _near(h, ho, dh, res)
        _near(y, yo, dy, dtype)
        h2, none = residual_norm(x, r, after=v, gate=m, scale=scale, eps=eps)
        assert none is None and torch.equal(h2, h)


@pytest.mark.parametrize("formula", ["torch", "tilelang"])
@pytest.mark.parametrize("T,H,block", [(1, 128, 128), (9, 4096, 128), (700, 2560, 64), (4, 96, 32), (3, 16384, 128),
                                       (40, 7168, 128)])
def test_codes_are_those_of_the_fp32_result(gpu, monkeypatch, formula, T, H, block):
    from sglang_lite_amd import kernel as K
    from sglang_lite_amd.norms import residual_norm

    print(f"norm codes T={T} H={H} block={block}", flush=True)
    monkeypatch.setenv("SGLANG_LITE_AMD_ACT_QUANT", formula)
    x, r, w, v, m = _inputs(gpu, T, H, F32, F32, True, "vector", F32, seed=H)
    if T > 2:
        r[1], x[1] = 0.0, 0.0         # all zeros: the smallest scale
        r[2, 5] = float("nan")        # a row of NaN
    kw = dict(after=v, gate=m, scale=0.7)
    h, y = residual_norm(x, r, w, **kw)
    for fmt, sdt in ((None, F32), ("ue8m0", F32), ("ue8m0", K.E8M0)):
        h2, (q, s) = residual_norm(x, r, w, quant=True, block_size=block, scale_fmt=fmt, scale_dtype=sdt, **kw)
        assert torch.equal(h2.view(torch.int32), h.view(torch.int32))
        assert q.dtype == K.FP8 and s.dtype == sdt and s.shape == (T, H // block)
        mode = K.scale_mode_for(fmt)
        qo, so = OQ.scale_mode_quant(_host(y), mode, block)
        got = s.view(torch.uint8).cpu().numpy() if sdt is K.E8M0 else _host(s)
        rows = np.ones(T, bool)
        if T > 2:
            rows[2] = False
            assert ((q.view(torch.uint8)[2] & 0x7F) == 0x7F).all()
        if sdt is K.E8M0:
            np.testing.assert_array_equal(got[rows], (so.view(np.uint32) >> 23).astype(np.uint8)[rows])
        else:
            np.testing.assert_array_equal(got[rows], so[rows])
        np.testing.assert_array_equal(q.view(torch.uint8).cpu().numpy()[rows], qo[rows])


def test_rows_anywhere_in_memory(gpu):
    """Strided rows, rows off any boundary, leading shapes, broadcast gates: as contiguous copies give."""
    from sglang_lite_amd.norms import residual_norm

    T, H = 30, 1003
    x, r, w, v, m = _inputs(gpu, T, H, BF16, BF16, True, "rows", BF16, seed=1)
    want = residual_norm(x, r, w, after=v, gate=m)

    def placed(t, off, gap):
        big = torch.zeros(T * (H + gap) + off, dtype=t.dtype, device=gpu)
        view = torch.as_strided(big, (T, H), (H + gap, 1), off)
        view.copy_(t)
        return view

    for off, gap in ((0, 0), (1, 1), (3, 5), (8, 13)):
        got = residual_norm(placed(x, off, gap), placed(r, off + 1, gap), w, after=v, gate=placed(m, off, gap + 2))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = residual_norm(x.view(5, 6, H), r.view(5, 6, H), w, after=v, gate=m.view(5, 6, H))
    assert all(torch.equal(a.view(T, H), b) for a, b in zip(got, want))
    one = residual_norm(x[4], r[4], w, after=v, gate=m[4])
    assert all(torch.equal(a, b[4]) for a, b in zip(one, want))
    cols = torch.stack([x, r], -1)  # a last dimension that is not dense
    got = residual_norm(cols[..., 0], cols[..., 1], w, after=v, gate=m)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # gates: of a channel, of a row, of a sequence's rows
    g1 = residual_norm(x, r, w, after=v, gate=m[3])
    assert all(torch.equal(a, b) for a, b in zip(g1, residual_norm(x, r, w, after=v, gate=m[3].expand(T, H))))
    g2 = residual_norm(x, r, w, gate=m[:, :1])
    assert all(torch.equal(a, b) for a, b in zip(g2, residual_norm(x, r, w, gate=m[:, :1].expand(T, H).contiguous())))
    seq = m.view(5, 6, H)[:, :1]
    g3 = residual_norm(x.view(5, 6, H), r.view(5, 6, H), w, gate=seq)
    g4 = residual_norm(x, r, w, gate=seq.expand(5, 6, H).reshape(T, H))
    assert all(torch.equal(a.view(T, H), b) for a, b in zip(g3, g4))
    empty = residual_norm(x[:0], r[:0], w, quant=False)
    assert empty[0].shape == (0, H) and empty[1].shape == (0, H)


def test_in_place(gpu):
    from sglang_lite_amd.norms import residual_norm

    T, H = 600, 4096
    x, r, w, v, m = _inputs(gpu, T, H, BF16, BF16, True, "rows", BF16, seed=2)
    want = residual_norm(x, r, w, after=v, gate=m, scale=0.5)
    wide = torch.zeros(T, 2 * H, dtype=BF16, device=gpu)
    wide[:, :H] = r
    h, y = residual_norm(x, wide[:, :H], w, after=v, gate=m, scale=0.5, inplace=True)
    assert h.data_ptr() == wide.data_ptr() and torch.equal(wide[:, :H], want[0]) and torch.equal(y, want[1])
    assert not wide[:, H:].any()
    # x, or the gate, is the residual
    xx = x.clone()
    want = residual_norm(x, x, w, after=v)
    h, y = residual_norm(xx, xx, w, after=v, inplace=True)
    assert h is xx and torch.equal(h, want[0]) and torch.equal(y, want[1])
    buf = torch.randn(T + 1, H, device=gpu).to(BF16)
    with pytest.raises(ValueError, match="overlaps x"):
        residual_norm(buf[:T], buf[1:], w, inplace=True)
    with pytest.raises(ValueError, match="overlaps the gate"):
        residual_norm(x, buf[1:], w, gate=buf[:T], inplace=True)
    both = torch.randn(T + 1, H, device=gpu)
    for name, given in (("the gate", {"gate": both[0]}), ("before", {"before": both[0]}), ("after", {"after": both[T]})):
        with pytest.raises(ValueError, match=f"overlaps {name}"):
            residual_norm(x, both[:T] if name != "after" else both[1:], **given, inplace=True)
    residual_norm(x, both[1:], both[0], inplace=True)
    with pytest.raises(ValueError, match="inplace"):
        residual_norm(x[:1].expand(T, H), buf[:1].expand(T, H), w, inplace=True)


def test_in_place_beside_its_inputs_in_one_buffer(gpu):
    from sglang_lite_amd.norms import residual_norm

    for T, H in ((600, 4096), (7, 1003), (1, 64)):
        x, r, w, v, m = _inputs(gpu, T, H, BF16, BF16, True, "rows", BF16, seed=T)
        want = residual_norm(x, r, w, after=v, gate=m, scale=0.5)
        wide = torch.zeros(T, 5, H, dtype=BF16, device=gpu)
        wide[:, 0], wide[:, 2], wide[:, 3], wide[T // 2, 1], wide[0, 4] = x, r, m, w, v
        before = wide.clone()
        h, y = residual_norm(wide[:, 0], wide[:, 2], wide[T // 2, 1], after=wide[0, 4], gate=wide[:, 3], scale=0.5,
                             inplace=True)
        assert h.data_ptr() == wide[0, 2].data_ptr() and torch.equal(wide[:, 2], want[0]) and torch.equal(y, want[1])
        before[:, 2] = want[0]
        assert torch.equal(wide, before)


def test_zeros_infinities_and_nan_stay_in_their_rows(gpu):
    from sglang_lite_amd.norms import residual_norm

    T, H = 12, 2000
    x, r, w, v, _ = _inputs(gpu, T, H, F32, F32, True, None, F32, seed=3)
    want = residual_norm(x, r, w, after=v)
    x[1], r[1] = 0.0, 0.0
    x[3, 7] = float("inf")
    r[5, 1999] = float("nan")
    h, y = residual_norm(x, r, w, after=v)
    assert not h[1].any() and not y[1].any()
    assert torch.isnan(h[3, 7]) and torch.isnan(y[3]).all()
    assert torch.isnan(h[5]).sum() == 1 and torch.isnan(y[5]).all()
    keep = [0, 2, 4, 6, 7, 8, 9, 10, 11]
    assert torch.equal(h[keep], want[0][keep]) and torch.equal(y[keep], want[1][keep])


def test_graph_and_stream(gpu):
    from sglang_lite_amd.norms import residual_norm

    T, H = 64, 4096
    x, r, w, v, m = _inputs(gpu, T, H, BF16, F32, True, "vector", F32, seed=4)
    call = lambda: residual_norm(x, r, w, after=v, gate=m, quant=True)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][1], want[1][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, (q, s) = call()
    for i in range(3):
        x.mul_(-1.25)
        r.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        h2, (q2, s2) = call()
        assert torch.equal(h, h2) and torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H,quant", [(8200, 4104, False), (8200, 4100, False), (8320, 4096, True)])
def test_rows_that_pass_the_cache_by(gpu, dtype, T, H, quant):
    """More than 128 MiB of inputs: each row as among few rows, and sampled rows against float64."""
    from sglang_lite_amd.norms import residual_norm

    print(f"norm T={T} H={H} {dtype} quant={quant}", flush=True)
    x, r, w, v, m = _inputs(gpu, T, H, dtype, dtype, True, "vector", F32, seed=T)
    kw = dict(after=v, scale=0.7, quant=quant)
    for gate in (m, torch.tanh(x.float()).to(dtype)):
        h, y = residual_norm(x, r, w, gate=gate, **kw)
        y, s = y if quant else (y, None)
        for lo in range(0, T, 1500):
            part = slice(lo, lo + 1500)
            h2, y2 = residual_norm(x[part], r[part], w, gate=gate if gate.dim() == 1 else gate[part], **kw)
            y2, s2 = y2 if quant else (y2, None)
            assert _same(h[part], h2) and _same(y[part], y2) and (s is None or _same(s[part], s2))
        rows = [0, 1, 511, 512, 767, T // 2, T - 2, T - 1]
        g = _host(gate if gate.dim() == 1 else gate[rows])
        ho, dh, yo, dy = ON.residual_norm(_host(x[rows]), _host(r[rows]), _host(w), _host(v), g,
                                          float(np.float32(0.7)), float(np.float32(1e-6)))
        _near(h[rows], ho, dh, dtype)
        if not quant:
            _near(y[rows], yo, dy, dtype)
        inside = r.clone()
        h2, y2 = residual_norm(x, inside, w, gate=gate, inplace=True, **kw)
        assert h2 is inside and _same(inside, h) and _same(y2[0] if quant else y2, y)


@pytest.mark.parametrize("T,H,block", [(30, 1024, 128), (700, 2560, 64), (5, 8320, 128)])
def test_codes_of_16_bit_rows_are_those_of_their_values(gpu, T, H, block):
    """The arithmetic is fp32 for every type of x and of the residual: the same codes, h rounded once."""
    from sglang_lite_amd import kernel as K
    from sglang_lite_amd.norms import residual_norm

    for dtype, res in ((BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)):
        x, r, w, v, m = _inputs(gpu, T, H, dtype, res, True, "rows", dtype, seed=H)
        for fmt, sdt in ((None, F32), ("ue8m0", K.E8M0)):
            kw = dict(quant=True, block_size=block, scale_fmt=fmt, scale_dtype=sdt, scale=-0.6)
            h, (q, s) = residual_norm(x, r, w, after=v, gate=m, **kw)
            h32, (q32, s32) = residual_norm(x.float(), r.float(), w, after=v, gate=m, **kw)
            assert _same(h, h32.to(res)) and _same(q, q32) and _same(s, s32)
