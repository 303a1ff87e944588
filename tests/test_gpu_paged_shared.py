"""Attention of sequences that begin alike, their common pages read once, against float64
attention of each sequence by itself."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_exact import check, exact, ints, join_tables
from test_gpu_paged_kv import Cache, _bytes, _filled, _host, _queries, _widen

pytestmark = pytest.mark.gpu


def _call(c, q, lens, cu, cu_groups, shared, sink=None, **kw):
    return c.P.paged_attn(q, c.kv, c.bt, ints(lens, c.dev), cu_tokens=ints(cu, c.dev),
                          cu_groups=ints(cu_groups, c.dev), shared=ints(shared, c.dev),
                          sink=None if sink is None else torch.from_numpy(sink).to(c.dev), **kw)


CASES = [
    # new, lens, cu_groups, shared, Hq, Hkv, D, page, block, dtype, causal, sink
    ([1, 1], [300, 400], [0, 2], [256], 1, 1, 16, 16, 16, torch.bfloat16, True, False),
    ([1] * 4, [700, 1500, 641, 2000], [0, 4], [640], 8, 2, 128, 64, 64, torch.float16, True, False),
    ([1] * 5, [700, 300, 650, 129, 500], [1, 4], [257], 16, 2, 64, 16, 16, torch.float16, True, True),
    ([2, 1, 4], [900, 800, 700], [0, 3], [699], 8, 2, 128, 64, 32, torch.float16, True, False),
    ([1, 1, 1], [1500, 1100, 2100], [0, 3], [1024], 8, 1, 256, 128, 128, torch.bfloat16, True, True),
    ([30] * 3, [500, 450, 700], [0, 3], [400], 8, 2, 128, 32, 16, torch.float16, True, False),
    ([40, 3, 1], [400, 460, 380], [0, 3], [384], 5, 5, 80, 16, 16, torch.float16, False, False),
    ([1] * 70, [300 + 3 * i for i in range(70)], [0, 70], [290], 8, 2, 64, 16, 16, torch.bfloat16, True, False),
    ([2] * 40, [600 + i for i in range(40)], [0, 40], [512], 8, 1, 128, 64, 64, torch.float16, True, True),
    ([3] * 12, [400 + i for i in range(12)], [0, 12], [384], 4, 1, 256, 64, 64, torch.bfloat16, True, False),
    ([1] * 9, [400 + i for i in range(9)], [0, 0, 4, 5, 8], [999, 300, 300, 256], 4, 2, 128, 16, 16, torch.bfloat16,
     True, False),                                           # an empty group, one of a single sequence, one outside
    ([70, 1, 0, 60], [600, 500, 100, 520], [0, 4], [400], 8, 2, 128, 64, 64, torch.bfloat16, True, True),
    ([1, 1, 1], [300, 90, 700], [0, 3], [256], 4, 2, 128, 64, 64, torch.bfloat16, True, False),  # one is shorter
    ([1, 1], [2100, 2050], [0, 2], [2049], 4, 2, 64, 1024, 64, torch.bfloat16, True, False),
    ([1, 1], [5, 0], [0, 2], [128], 4, 2, 64, 16, 16, torch.bfloat16, True, False),
]


@pytest.mark.parametrize("tokens", [0, 16384, 1 << 18])  # (wide tables: many rows in two passes)
@pytest.mark.parametrize("new,lens,cu_groups,shared,Hq,Hkv,D,page,block,dtype,causal,sink", CASES)
def test_shared_prefix(gpu, tokens, new, lens, cu_groups, shared, Hq, Hkv, D, page, block, dtype, causal, sink):
    print(f"shared new={new} lens={lens} groups={cu_groups} {shared} Hq={Hq} Hkv={Hkv} D={D} page={page}", flush=True)
    c = _filled(gpu, lens, Hkv, D, page, block, seed=D + Hq)
    join_tables(c, cu_groups, shared)
    _widen(c, tokens)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], Hq, D, dtype, 9)
    s = (np.random.default_rng(2).standard_normal(Hq) * 2).astype(np.float32) if sink else None
    o = _call(c, q, lens, cu, cu_groups, shared, s, causal=causal)
    check(c, o, q, lens, cu, sink=s, causal=causal, parts=2)
    if new == [1] * len(new):
        assert torch.equal(_call(c, q, lens, None, cu_groups, shared, s, causal=causal), o)


def test_what_is_claimed_may_be_more_or_less_than_what_is_there(gpu):
    """More tokens than any sequence has, none, a negative number; groups that reach past the batch or
    begin before it.  (The sums' order is the call's own even where nothing is shared.)"""
    lens = [500, 420, 700, 300]
    c = _filled(gpu, lens, 2, 64, 16, 16, seed=3)
    join_tables(c, [0, 4], [299])
    c.table[1:, :300 // 16] = c.table[0, :300 // 16]
    c.bt = torch.from_numpy(c.table).to(gpu)
    q = _queries(gpu, 4, 8, 64, torch.float16, 4)
    for groups, shared in (([0, 4], [0]), ([0, 4], [-5]), ([0, 4], [127]), ([4, 4], [256]), ([0, 0], [256]),
                           ([2, 3], [256]), ([-3, 1], [256]), ([3, 9], [256]), ([0, 4], [2 ** 31 - 1]), ([0, 4], [299]), ([-1, 7], [299]), ([0, 3], [256]), ([1, 4], [300])):
        o = _call(c, q, lens, None, groups, shared)
        check(c, o, q, lens, None, parts=2)


@pytest.mark.parametrize("B,cu_groups,shared", [(59, [0, 20, 20, 41, 59], [500, 300, 700, 640]),
                                                (62, [1, 60, 62], [500, 700]), (2, [0, 2], [1 << 30]),
                                                (9, [-3, 4, 70], [600, 600]), (5, [2, 5, 5], [-4, 512])])
@pytest.mark.parametrize("each", [1, 2])
def test_groups_found_by_each_workgroup_are_the_planned_ones(gpu, B, cu_groups, shared, each):
    """Few sequences and groups need no plan in front: the same line, so the same bits, as beside empty groups."""
    rng = np.random.default_rng(B)
    new = [int(n) for n in rng.integers(0, each + 1, B)]
    new[-1] = each
    lens = [int(n) for n in rng.integers(700, 1000, B)]
    if B > 50:
        lens[B // 2] = new[B // 2]
    Hq = 16 if B > 50 else 2  # (groups' tiles of 32 rows, or of 16, on both sides)
    c = _filled(gpu, lens, 2, 64, 64, 16, seed=B)
    edges = [min(max(b, 0), B) for b in cu_groups]
    join_tables(c, edges, [max(0, min(n, 700)) for n in shared])
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], Hq, 64, torch.bfloat16, 5)
    more = 5 if B < 60 else 2  # empty groups behind: too many, or too many sequences, to go without a plan
    want = _call(c, q, lens, cu, cu_groups + cu_groups[-1:] * more, shared + [700] * more)
    assert torch.equal(_call(c, q, lens, cu, cu_groups, shared), want)
    check(c, want, q, lens, cu, parts=2)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("lead", [0.0, 12.0])
def test_parts_whose_references_lie_far_apart(gpu, new, lead):
    """The prefix, or what is behind it, has all of the weight, or a value of zero under it."""
    L, H, D, B = 900, 1, 64, 3
    for at, zero in ((3, False), (3, True), (L - 60, False), (L - 60, True)):
        c = Cache(gpu, B, L, H, D, 16, 16, seed=3)
        g = torch.Generator(device=gpu).manual_seed(D + new)
        k, v = (torch.randn(B * L, H, D, generator=g, device=gpu) for _ in range(2))
        k[..., 0] = 0.0
        for b in range(B):
            k[b * L + at] = 0.0
            k[b * L + at, :, 0] = (lead + 8.0) * D ** 0.5 / 8.0
            if zero:
                v[b * L + at] = 0.0
        c.P.append_kv(c.kv, k, v, c.bt, ints([0] * B, gpu), cu_tokens=ints([0, L, 2 * L, 3 * L], gpu))
        c.k, c.v = _bytes(c.kv.k).copy(), _bytes(c.kv.v).copy()
        c.ks, c.vs = _host(c.kv.k_scale).copy(), _host(c.kv.v_scale).copy()
        join_tables(c, [0, B], [640])
        q = _queries(gpu, B * new, 4, D, torch.float16, 5)
        q[..., 0] = 8.0
        cu = [new * b for b in range(B + 1)]
        check(c, _call(c, q, [L] * B, cu, [0, B], [640]), q, [L] * B, cu, parts=2)


@pytest.mark.parametrize("new,B,tokens", [(1, 3, 16384), (1, 40, 16384), (2, 40, 1 << 18), (50, 3, 16384)])
def test_every_key_counts_once(gpu, new, B, tokens):
    """Values of zero but for one key in each dim of a kv head: the output is that key's weight."""
    L, H, D = 1100, 8, 64
    c = Cache(gpu, B, L, H, D, 16, 16, seed=4)
    join_tables(c, [0, B], [770])
    _widen(c, tokens)
    g = torch.Generator(device=gpu).manual_seed(L)
    k = 0.5 * torch.randn(L, H, D, generator=g, device=gpu)
    q = _queries(gpu, B * new, 2 * H, D, torch.float16, 11)
    cu = [new * b for b in range(B + 1)]
    for base in range(0, L, H * D):
        v = torch.zeros(L, H, D, device=gpu)
        t = base + torch.arange(H * D, device=gpu)
        t = t[t < L]
        v[t, (t - base) // D, (t - base) % D] = 1.0 + (t % 7) / 8.0
        for b in range(B):  # (the common pages the same each time)
            c.P.append_kv(c.kv, k, v, c.bt[b:b + 1], ints([0], gpu), cu_tokens=ints([0, L], gpu))
        c.k, c.v = _bytes(c.kv.k).copy(), _bytes(c.kv.v).copy()
        c.ks, c.vs = _host(c.kv.k_scale).copy(), _host(c.kv.v_scale).copy()
        check(c, _call(c, q, [L] * B, cu, [0, B], [770]), q, [L] * B, cu, rms=False, parts=2)


@pytest.mark.parametrize("new,D,tokens", [(1, 128, 0), (6, 64, 0), (20, 128, 0), (20, 128, 1 << 18), (40, 256, 0),
                                          (60, 128, 0)])
def test_nan_reaches_only_the_rows_that_see_it(gpu, new, D, tokens):
    """In a common page: every sequence of the group; behind it: its own."""
    lens = [700, 650, 800]
    c = _filled(gpu, lens, 2, D, 64, 16, seed=11)
    join_tables(c, [0, 2], [600])
    _widen(c, tokens)
    spots = [(0, 5, 0, 3), (0, 639, 1, 9), (1, 640 - 64, 0, 4), (2, 100, 0, 11)]  # sequence, token, head, dim
    for b, t, h, d in spots:
        p, spot = int(c.table[b, t // 64]), t % 64
        c.kv.v.view(torch.uint8)[p, h, spot, d] = 0x7F
        c.v[p, h, spot, d] = 0x7F
    cu = [0, new, 2 * new, 3 * new]
    q = _queries(gpu, 3 * new, 8, D, torch.bfloat16, 5)
    got = np.isnan(_host(_call(c, q, lens, cu, [0, 2], [600])))
    want = np.zeros(got.shape, bool)
    for b in range(3):
        for b2, t, h, d in spots:
            if c.table[b, t // 64] == c.table[b2, t // 64]:
                want[cu[b]:cu[b + 1], 4 * h:4 * h + 4, d] = True
    np.testing.assert_array_equal(got, want)


def test_pages_that_are_none(gpu):
    lens = [900, 800, 700]
    c = _filled(gpu, lens, 2, 128, 16, 16, seed=9)
    c.table[0, 1], c.table[0, 10] = -1, 1 << 30
    join_tables(c, [0, 3], [512])
    c.table[1, 35] = -1
    c.bt = torch.from_numpy(c.table).to(gpu)
    for new in ([1, 1, 1], [20, 3, 9], [100, 20, 120]):
        cu = [0] + np.cumsum(new).tolist()
        q = _queries(gpu, cu[-1], 8, 128, torch.bfloat16, 4)
        check(c, _call(c, q, lens, cu, [0, 3], [512]), q, lens, cu, parts=2)


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 1), (64, 8, 2), (256, 8, 2)])
def test_many_groups_of_many_sizes(gpu, D, Hq, Hkv):
    """More groups and sequences than a wavefront has lanes; groups of few rows and of many, and
    sequences of either in them."""
    rng = np.random.default_rng(8)
    sizes = [int(n) for n in rng.integers(0, 4, 70)] + [30]
    edge = [2] + (2 + np.cumsum(sizes)).tolist()
    B = edge[-1] + 3
    new = [int(n) for n in rng.choice([0, 1, 1, 2, 60], B)]
    shared = [int(n) for n in rng.integers(100, 300, len(sizes))]
    lens = [int(rng.integers(310, 420)) + n for n in new]
    c = _filled(gpu, lens, Hkv, D, 16, 16, seed=12)
    join_tables(c, edge, shared)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1] + 3, Hq, D, torch.float16, 6)
    for tokens in (0, 8192, 1 << 18):
        _widen(c, tokens)
        out = torch.full_like(q, 7.0)
        o = _call(c, q, lens, cu, edge, shared, out=out)
        assert bool((out[cu[-1]:] == 7.0).all())
        check(c, o, q, lens, cu, parts=2)


@pytest.mark.parametrize("new,D,tokens,more", [
    ([0, 1, 1, 0, 1], 128, 0, 0),           # found by each workgroup
    ([0, 0, 2, 1], 64, 16384, 0),
    ([0, 1, 1, 0, 1], 128, 0, 5),           # planned in front
    ([0] * 70 + [1] * 30, 64, 0, 0),
    ([0] * 300 + [1, 2], 256, 0, 0),
    ([0, 40, 40], 128, 1 << 18, 0),         # in two passes
    ([0] * 300 + [60, 1, 0, 60], 64, 1 << 18, 0),
])
def test_sequences_without_queries_in_front_of_a_group(gpu, new, D, tokens, more):
    """Their rows of the block table (no pages, or foreign ones) and lengths are not looked at."""
    B = len(new)
    live = [b for b in range(B) if new[b]]
    lens = [900 if n else 0 for n in new]
    c = _filled(gpu, lens, 2, D, 16, 16, seed=B)
    for b in live[1:]:
        c.table[b, :640 // 16] = c.table[live[0], :640 // 16]
    c.bt = torch.from_numpy(c.table).to(gpu)
    _widen(c, tokens)
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], 16, D, torch.bfloat16, 7)
    for fill, old in ((-1, 0), (int(c.table[live[-1], 50]), 0), (1 << 30, 900), (-1, -3)):
        for b in range(B):
            if new[b] == 0:
                c.table[b] = fill
                lens[b] = old
        c.bt = torch.from_numpy(c.table).to(gpu)
        o = _call(c, q, lens, cu, [0, B] + [B] * more, [650] + [0] * more)
        check(c, o, q, lens, cu, parts=2)


def test_captured_with_other_lengths_and_prefixes(gpu):
    lens0 = [900, 700, 1200, 640]
    c = _filled(gpu, lens0, 2, 128, 64, 64, seed=14)
    join_tables(c, [0, 4], [640])
    _widen(c, 8192)
    q = _queries(gpu, 4, 16, 128, torch.bfloat16, 10)
    lens, groups, shared = ints(lens0, gpu), ints([0, 4], gpu), ints([640], gpu)
    run = lambda: c.P.paged_attn(q, c.kv, c.bt, lens, cu_groups=groups, shared=shared)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for have, g, n in ((lens0, [0, 4], 640), ([800, 650, 1100, 630], [0, 4], 640), ([900, 10, 0, 600], [0, 4], 500),
                       (lens0, [1, 3], 640), (lens0, [0, 4], 0), (lens0, [0, 4], 384)):
        lens.copy_(ints(have, gpu))
        groups.copy_(ints(g, gpu))
        shared.fill_(n)
        q.mul_(-0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, run())
        check(c, held, q, have, None, parts=2)


def test_calls_on_two_streams_at_once(gpu):
    lens = [2000, 1700, 1600]
    c = _filled(gpu, lens, 2, 128, 64, 64, seed=15)
    join_tables(c, [0, 3], [1500])
    qs = [_queries(gpu, 3, 16, 128, torch.bfloat16, 70 + i) for i in range(8)]
    want = [_call(c, q, lens, None, [0, 3], [1500]) for q in qs]
    torch.cuda.synchronize()
    lt, gt, st = ints(lens, gpu), ints([0, 3], gpu), ints([1500], gpu)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(c.P.paged_attn(q, c.kv, c.bt, lt, cu_groups=gt, shared=st))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,Hq,new", [
    (64, 2, [1] * 3), (64, 8, [1] * 6), (64, 8, [6] * 3),       # tiles of 16 rows; groups' of 32; both
    (128, 2, [1] * 3), (112, 8, [1] * 6), (128, 8, [6] * 3),
    (128, 8, [2] * 30), (96, 8, [6] * 10),                      # more than 160 rows of a group
    (256, 2, [1] * 3), (192, 8, [1] * 6), (256, 8, [3] * 20),
])
def test_each_tile_of_one_pass(gpu, D, Hq, new, dtype):
    lens = [500 + 7 * i for i in range(len(new))]
    c = _filled(gpu, lens, 2, D, 32, 32, seed=D + Hq)
    join_tables(c, [0, len(new)], [410])
    cu = [0] + np.cumsum(new).tolist()
    q = _queries(gpu, cu[-1], Hq, D, dtype, 3)
    for tokens in (0, 4096):
        _widen(c, tokens)
        check(c, _call(c, q, lens, cu, [0, len(new)], [410]), q, lens, cu, parts=2)


@pytest.mark.parametrize("new,tokens,more", [([1] * 5, 0, 0), ([2] * 5, 16384, 5), ([60, 1, 0, 40], 1 << 18, 0),
                                             ([200, 150], 1 << 18, 0)])
def test_strided_queries_and_into_the_queries_themselves(gpu, new, tokens, more):
    """By the workgroups themselves, planned in front, in two passes: as into a new tensor."""
    B = len(new)
    lens = [900 + 7 * i for i in range(B)]
    c = _filled(gpu, lens, 2, 128, 64, 32, seed=21)
    join_tables(c, [0, B], [640])
    _widen(c, tokens)
    cu = [0] + np.cumsum(new).tolist()
    wide = _queries(gpu, cu[-1], 48, 128, torch.bfloat16, 8)
    q = wide[:, 16:32]
    groups, shared = [0, B] + [B] * more, [640] + [0] * more
    want = _call(c, q, lens, cu, groups, shared)
    check(c, want, q.contiguous(), lens, cu, parts=2)
    held = q.contiguous()
    assert _call(c, held, lens, cu, groups, shared, out=held) is held
    assert torch.equal(held, want)


def test_exact_of_a_short_row():
    """(the helper's own: a row that sees no key is zero)"""

    class C:
        k = v = np.zeros((1, 1, 16, 16), np.uint8)
        ks = vs = np.ones((1, 1, 1), np.float32)
        table = np.zeros((1, 1), np.int32)

    assert not exact(C, 0, np.ones((2, 1, 16), np.float32), 0, 1.0)[0].any()
