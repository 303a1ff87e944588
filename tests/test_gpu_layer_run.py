"""The operators of an attention layer as a server runs them together: norms and sum, FP8
projection, rotary positions of several axes, the keys into the cache, attention behind a common
prompt or in a window with first tokens, and the norm behind it; every output against the oracle
on the inputs that it had."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import norms as ON
from oracle import paged as OP
from paged_exact import check, ints
from test_gpu_paged_kv import HALF, _bytes, _host

pytestmark = pytest.mark.gpu

H, HQ, HKV, D, PAGE, BLOCK = 256, 4, 2, 64, 16, 16  # (HQ D = H: the output projection is left out)
SECTIONS = (8, 12, 12)


class Layer:
    """Weights, the cache of a batch that begins with one prompt, and the oracle's copy of it."""

    def __init__(self, dev, B, tokens, prompt, seed=1):
        from sglang_lite_amd import kernel as K
        from sglang_lite_amd import paged_kv as P
        from sglang_lite_amd import rotary as R

        g = torch.Generator(device=dev).manual_seed(seed)

        def randn(*s):
            return torch.randn(*s, generator=g, device=dev)

        self.dev, self.B, self.prompt = dev, B, prompt
        self.w_in, self.s_in = K.per_block_cast_to_fp8(randn((HQ + 2 * HKV) * D, H) / 16, False)
        self.before, self.after = 1 + 0.2 * randn(H), 1 + 0.2 * randn(H)
        self.gate = torch.tanh(randn(H))
        self.table = R.rotary_table(600, D, device=dev)
        self.axes = R.rotary_axes(SECTIONS, spread=True, device=dev)
        cols = -(-tokens // PAGE)
        common = prompt // PAGE
        pages = common + B * (cols - common)
        self.kv = P.PagedKV.empty(pages, HKV, PAGE, D, block=BLOCK, device=dev)
        for x in self.kv:
            x.view(torch.uint8).fill_(0x7F)
        ids = np.random.default_rng(seed).permutation(pages).astype(np.int32)
        own = ids[common:].reshape(B, cols - common)
        self.pages = np.concatenate([np.tile(ids[:common], (B, 1)), own], 1)
        self.bt = torch.from_numpy(self.pages).to(dev)
        self.keep()

    def keep(self):
        self.k, self.v = _bytes(self.kv.k).copy(), _bytes(self.kv.v).copy()
        self.ks, self.vs = _host(self.kv.k_scale).copy(), _host(self.kv.v_scale).copy()

    def step(self, x, residual, start, lens, pos, cu=None, bt=None, **attn):
        """The calls of one step: all of their outputs, in order."""
        from sglang_lite_amd import kernel as K
        from sglang_lite_amd import paged_kv as P
        from sglang_lite_amd import rotary as R
        from sglang_lite_amd.norms import residual_norm

        bt = self.bt if bt is None else bt
        T = x.shape[0]
        h, (codes, s) = residual_norm(x, residual, self.before, quant=True)
        qkv = K.fp8_gemm_as(codes, s, self.w_in, self.s_in, torch.bfloat16).view(T, HQ + 2 * HKV, D)
        q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
        qr = R.rotary(q, self.table, pos, axes=self.axes)
        P.append_kv(self.kv, k, v, bt, start, cu_tokens=cu, table=self.table, positions=pos, axes=self.axes)
        o = P.paged_attn(qr, self.kv, bt, lens, cu_tokens=cu, **attn)
        h2, y = residual_norm(o.view(T, H), h, self.before, after=self.after, gate=self.gate, scale=0.5)
        return h, codes, s, qkv, qr, o, h2, y

    def check(self, got, x, residual, start, lens, pos, cu, rows, **kw):
        h, codes, s, qkv, qr, o, h2, y = got
        before, f32 = _host(self.before), np.float32

        def near(t, ref, bound):
            err = np.abs(_host(t).astype(np.float64) - ref)
            assert np.all(err <= bound + HALF[t.dtype] * (np.abs(ref) + bound)), float(err.max())

        ho, dh, yo, dy = ON.residual_norm(_host(x), _host(residual), before, None, None, 1.0, float(f32(1e-6)))
        near(h, ho, dh)
        # the codes: half a step of e4m3 (2^-4 of the value, 2^-10 below 2^-6) around y / s, which fp32 keeps to
        # 3 half steps beside y's own error
        sc = _host(s).repeat(128, 1).astype(np.float64)
        bound = dy / sc + 3 * 2.0 ** -24 * np.abs(yo / sc)
        err = np.abs(_host(codes).astype(np.float64) - yo / sc)
        assert np.all(err <= bound + np.maximum(2.0 ** -4 * (np.abs(yo / sc) + bound), 2.0 ** -10))
        at, axes = pos.cpu().numpy(), self.axes.cpu().numpy()
        freq = 10000.0 ** (-np.arange(0, D, 2) / D)
        ref = OP.rotate_axes(_host(qkv[:, :HQ]), at, axes, freq)
        a = np.abs(_host(qkv[:, :HQ]).astype(np.float64))
        both = a[..., :D // 2] + a[..., D // 2:]
        near(qr, ref, 4 * 2.0 ** -24 * np.concatenate([both, both], -1))
        rot = _host(self.table)[at[axes].T, np.arange(D // 2)]
        table = self.pages[rows]
        OP.append(self.k, self.ks, OP.rotate_f32(_host(qkv[:, HQ:HQ + HKV]), rot), table, start, cu)
        OP.append(self.v, self.vs, _host(qkv[:, HQ + HKV:]), table, start, cu)
        np.testing.assert_array_equal(_bytes(self.kv.k), self.k)
        np.testing.assert_array_equal(_bytes(self.kv.v), self.v)
        np.testing.assert_array_equal(_host(self.kv.k_scale), self.ks)

        class View:
            k, v, ks, vs = self.k, self.v, self.ks, self.vs

        View.table = table
        check(View, o, qr, lens, cu, parts=2, **kw)
        h2o, dh2, y2o, dy2 = ON.residual_norm(_host(o).reshape(-1, H), _host(h), before, _host(self.after), _host(self.gate), 0.5,
                                              float(f32(1e-6)))
        near(h2, h2o, dh2)
        near(y, y2o, dy2)


def _tokens(layer, T, seed):
    g = torch.Generator(device=layer.dev).manual_seed(seed)
    x = torch.randn(T, H, generator=g, device=layer.dev).to(torch.bfloat16)
    return x, torch.randn(T, H, generator=g, device=layer.dev) * 2


def test_a_prompt_with_pictures_then_answers_behind_it(gpu):
    prompt, B = 200, 5
    L = Layer(gpu, B, 400, prompt)
    rng = np.random.default_rng(0)
    # the prompt, once, in two chunks: text, a picture of 9 x 12 patches, text
    time = np.concatenate([np.arange(60), np.full(108, 60), np.arange(72, 104)])
    height = np.concatenate([np.arange(60), 60 + np.repeat(np.arange(9), 12), np.arange(72, 104)])
    width = np.concatenate([np.arange(60), 60 + np.tile(np.arange(12), 9), np.arange(72, 104)])
    at = np.stack([time, height, width])
    for lo, hi in ((0, 130), (130, prompt)):
        x, r = _tokens(L, hi - lo, lo)
        pos = torch.from_numpy(at[:, lo:hi].astype(np.int32)).to(gpu).contiguous()
        args = (ints([lo], gpu), ints([hi], gpu), pos)
        got = L.step(x, r, *args, cu=ints([0, hi - lo], gpu), bt=L.bt[:1])
        L.check(got, x, r, [lo], [hi], pos, [0, hi - lo], slice(0, 1))
    # what is left of the prompt in a page begun is each sequence's own
    begun = prompt // PAGE
    for b in range(1, B):
        for t in L.kv:
            t.view(torch.uint8)[int(L.pages[b, begun])] = t.view(torch.uint8)[int(L.pages[0, begun])]
    L.keep()
    have = [prompt] * B
    groups, shared = ints([0, B], gpu), ints([prompt], gpu)
    for step in range(4):
        new = [1] * B if step != 2 else [int(n) for n in rng.integers(0, 4, B)]
        cu = [0] + np.cumsum(new).tolist()
        x, r = _tokens(L, cu[-1], 100 + step)
        pos = np.concatenate([np.arange(h, h + n) - 96 for h, n in zip(have, new)]).astype(np.int32)
        pos = torch.from_numpy(np.tile(pos, (3, 1))).to(gpu)
        after = [h + n for h, n in zip(have, new)]
        cut = None if new == [1] * B else ints(cu, gpu)
        got = L.step(x, r, ints(have, gpu), ints(after, gpu), pos, cu=cut, cu_groups=groups, shared=shared)
        L.check(got, x, r, have, after, pos, cu, slice(None))
        have = after


def test_a_captured_step_of_either_form_replays(gpu):
    """With other tokens, lengths and prefixes: as the eager calls on a cache like it."""
    prompt, B = 160, 4
    one, two = (Layer(gpu, B, 320, prompt, seed=3) for _ in range(2))
    x0, r0 = _tokens(one, 2 * prompt, 1)
    for L in (one, two):  # keys and values of the prompt and a little more of each
        for b in range(B):
            n = prompt if b == 0 else prompt // PAGE * PAGE
            pos = torch.arange(n + 40, dtype=torch.int32, device=gpu).expand(3, n + 40).contiguous()
            L.step(x0[:n + 40], r0[:n + 40], ints([0], gpu), ints([n + 40], gpu), pos, cu=ints([0, n + 40], gpu),
                   bt=L.bt[b:b + 1])
    for x, y in zip(one.kv, two.kv):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    x, r = _tokens(one, B, 5)
    start, lens, shared = ints([190] * B, gpu), ints([191] * B, gpu), ints([prompt], gpu)
    pos = torch.full((3, B), 190, dtype=torch.int32, device=gpu)
    groups = ints([0, B], gpu)
    for form in (dict(cu_groups=groups, shared=shared), dict(window=50, first=9)):
        for L in (one, two):  # (loads the kernels, and leaves both caches alike)
            L.step(x, r, start, lens, pos, **form)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = one.step(x, r, start, lens, pos, **form)
        for i in range(4):
            nx, nr = _tokens(one, B, 50 + i)
            x.copy_(nx)
            r.copy_(nr)
            start.copy_(ints([191 + i, 180, 200 + i, 170 + 3 * i], gpu))
            lens.copy_(start + 1)
            pos.copy_(torch.randint(0, 600, (3, B), device=gpu))
            shared.fill_(prompt if i % 2 else 130)
            graph.replay()
            want = two.step(x, r, start, lens, pos, **form)
            torch.cuda.synchronize()
            for a, b in zip((*held, *one.kv), (*want, *two.kv)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), f"replay {i}"
