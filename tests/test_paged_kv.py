"""What the rotary positions and the 8-bit paged cache do without a GPU: frequencies, refusals,
the bounds that grids are made from, and the block scale."""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import paged as OP

CSRC = Path(__file__).resolve().parents[1] / "sglang-lite_amd" / "csrc"

WRAPPERS = r"""
#include "sgl_rules.h"
#include "sgl_numeric.h"
using namespace sgl;
extern "C" {
int64_t append_units(int64_t T, int64_t B, int64_t block) { return kv8_append_units(T, B, block); }
int64_t attn_items(int64_t T, int64_t B, int64_t Hkv, int64_t G, int64_t rows) { return kv8_attn_items(T, B, Hkv, G, rows); }
int head_threads(int64_t T, int64_t H, int64_t units, int64_t cus) { return rotary_head_threads(T, H, units, cus); }
float block_scale(float amax) { return kv8_scale(amax); }
void attn_plan(int64_t T, int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t capacity, int64_t cus, int64_t* o) {
  const Kv8AttnPlan p = kv8_attn_plan(T, B, Hkv, G, D, capacity, cus);
  o[0] = p.row_tile;
  o[1] = p.parts;
  o[2] = (int64_t)kv8_attn_workspace(p, Hkv, D);
  const Kv8AttnPlan r = kv8_attn_rest(T, B, Hkv, G, D, capacity, cus);
  o[3] = r.row_tile;
  o[4] = r.items;
  o[5] = p.above;
  o[6] = r.upto;
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv8rules")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text(WRAPPERS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    i64 = ctypes.c_int64
    lib.append_units.restype, lib.append_units.argtypes = i64, [i64] * 3
    lib.attn_items.restype, lib.attn_items.argtypes = i64, [i64] * 5
    lib.head_threads.argtypes = [i64] * 4
    lib.attn_plan.argtypes = [i64] * 7 + [ctypes.c_void_p]
    lib.block_scale.restype, lib.block_scale.argtypes = ctypes.c_float, [ctypes.c_float]
    return lib


@pytest.mark.parametrize("seed", range(40))
def test_grids_cover_every_block_and_row_tile(rules, seed):
    rng = np.random.default_rng(seed)
    B = int(rng.integers(1, 50))
    new = rng.integers(0, (2, 5, 40, 300)[seed % 4], B)
    have = rng.integers(0, 500, B)
    T = int(new.sum()) + int(rng.integers(0, 3))
    for block in (16, 32, 64, 128):
        touched = sum(int((h + n - 1) // block - h // block) + 1 for n, h in zip(new, have) if n)
        assert touched <= rules.append_units(T, B, block) <= max(T, 0)
    for G, rows in ((1, 16), (4, 16), (5, 32), (64, 16), (8, 128), (48, 32)):
        tiles = sum(-(-int(n) * G // rows) for n in new)
        assert tiles * 3 <= rules.attn_items(T, B, 3, G, rows)


def test_attention_plans(rules):
    o = (ctypes.c_int64 * 7)()

    def plan(T, B, Hkv, G, D, capacity, cus=256):
        rules.attn_plan(T, B, Hkv, G, D, capacity, cus, o)
        return o[0], o[1], o[2]

    rng = np.random.default_rng(0)
    for _ in range(2000):
        B, Hkv, G = (int(rng.integers(1, n)) for n in (200, 70, 70))
        T, D = B * int(rng.integers(1, 300)), 16 * int(rng.integers(1, 17))
        rt, parts, ws = plan(T, B, Hkv, G, D, 16 << int(rng.integers(0, 14)), int(rng.integers(8, 400)))
        assert rt in (16, 32, 128, 256) and parts % 8 == 0 and parts >= 0
        assert (rt > 32) == (T * G // B > (96 if D <= 128 else 32))
        assert ws == parts * 2 * Hkv * rt * (D + 2) * 4  # two stretches a workgroup
        # a second launch takes exactly the sequences that the first leaves, all their row tiles
        few = 96 if D <= 128 else 32
        assert o[5] == o[6] == (few if rt > 32 and B >= 8 and T > B else 0)
        assert o[4] == (B * -(-few // o[3]) * Hkv if o[5] else 0)
    # a short table: no sharing, no workspace; few rows up to 2048 tokens where items are many
    assert plan(1, 1, 8, 4, 128, 1024)[1:] == (0, 0) and plan(1, 1, 8, 4, 128, 1040)[1] == 32
    # (the items are a bound, T G / 16 + B row tiles for each of 8 heads: 52 sequences 520, 51 504)
    assert plan(52, 52, 8, 4, 128, 2048)[1] == 0 and plan(51, 51, 8, 4, 128, 2048)[1] == 32 and plan(9, 9, 8, 4, 64, 4096)[1] == 64
    # a chunk's row tiles: two a workgroup are not shared, fewer by how much there is to share
    assert plan(8192, 1, 8, 4, 128, 1 << 17)[1] == 0 and plan(512, 1, 8, 4, 128, 1 << 13)[1] == 32
    assert plan(2048, 1, 8, 4, 128, 4096)[1] == 0 and plan(2048, 1, 8, 4, 128, 8192)[1] == 32


def test_rows_that_overlap():
    from sglang_lite_amd.rotary import _apart

    rng = np.random.default_rng(1)
    for _ in range(3000):
        T, H, D = (int(rng.integers(1, 4)) for _ in range(3))
        s0, s1 = int(rng.integers(0, 14)), int(rng.integers(0, 14))
        at = [t * s0 + h * s1 + d for t in range(T) for h in range(H) for d in range(D)]
        if _apart(T, s0, H, s1, D) or _apart(H, s1, T, s0, D):
            assert len(set(at)) == len(at)


def test_head_threads(rules):
    for T, H in ((1, 1), (16, 32), (1 << 14, 32), (1900, 64), (4000, 7)):
        n = rules.head_threads(T, H, 8, 256)
        assert n in (H, -(-H // 4))
    assert rules.head_threads(1, 32, 8, 256) == 32 and rules.head_threads(1 << 14, 32, 8, 256) == 8


def test_block_scale_is_the_smallest_power_of_two_that_fits(rules):
    rng = np.random.default_rng(0)
    x = np.concatenate([np.float32(2.0) ** rng.integers(-126, 127, 300).astype(np.float32),
                        rng.integers(1, 0x7F800000, 3000).astype(np.uint32).view(np.float32),
                        np.float32(448) * np.float32(2.0) ** np.arange(-120, 119, dtype=np.float32)])
    x = np.concatenate([x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(0)),
                        np.array([0.0, 1e-45, np.finfo(np.float32).max], np.float32)])
    for v in x[np.isfinite(x)]:
        s = rules.block_scale(float(v))
        assert math.frexp(s)[0] == 0.5 and s >= 2.0 ** -100
        assert float(v) <= 448.0 * s
        assert s == 2.0 ** -100 or float(v) > 448.0 * (s / 2)
        assert s == OP.block_scale(v)


def test_frequencies_of_the_scalings():
    from sglang_lite_amd import rotary as R

    plain, one = R.frequencies(64)
    assert one == 1.0 and plain[0] == 1.0 and torch.allclose(plain, 10000.0 ** (-torch.arange(0, 64, 2).double() / 64))
    f, m = R.frequencies(64, scaling={"type": "linear", "factor": 4.0})
    assert torch.equal(f, plain / 4) and m == 1.0
    f, _ = R.frequencies(64, scaling={"type": "ntk", "factor": 8.0})
    assert abs(f[0] - 1.0) < 1e-12 and abs(f[-1] * 8.0 / plain[-1] - 1.0) < 1e-12
    f, m = R.frequencies(64, scaling={"type": "yarn", "factor": 16.0, "original": 4096})
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(f[turns > 40], plain[turns > 40])
    assert torch.allclose(f[turns < 0.8] * 16.0, plain[turns < 0.8])
    assert bool((f[:-1] > f[1:]).all()) and abs(m - (1 + 0.1 * math.log(16.0))) < 1e-15
    assert R.frequencies(64, scaling={"type": "yarn", "factor": 16.0, "original": 4096, "length": 1.0})[1] == 1.0
    for bad in ({"type": "other", "factor": 2.0}, {"type": "linear"}, {"type": "linear", "factor": 0.5}, {}):
        with pytest.raises(ValueError):
            R.frequencies(64, scaling=bad)
    for rot in (0, 7, -2):
        with pytest.raises(ValueError):
            R.frequencies(rot)


def test_rotary_refusals():
    from sglang_lite_amd import rotary as R

    x, pos = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    table = torch.zeros(8, 32, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        R.rotary(x, table, pos)
    with pytest.raises(RuntimeError, match="no CPU path"):
        R.rotary_table(8, 64, device="cpu")
    for args in ((x[0], table, pos), (x, table, pos[:3]), (x, table[..., :1], pos), (x, table.double(), pos),
                 (x, torch.zeros(8, 33, 2), pos)):
        with pytest.raises(ValueError):
            R.rotary(*args)
    for off in (-8, 8):
        with pytest.raises(ValueError):
            R.rotary(x, table, pos, offset=off)
    with pytest.raises(TypeError):
        R.rotary(x.double(), table, pos)
    with pytest.raises(TypeError):
        R.rotary(x, table, pos.float())
    with pytest.raises(ValueError):
        R.rotary_table(0, 64)


def _cache(pages=4, H=2, page=32, D=64, block=16):
    from sglang_lite_amd import paged_kv as P

    return P.PagedKV.empty(pages, H, page, D, block=block, device="cpu")


@pytest.mark.parametrize("kw", [dict(page=24), dict(page=8), dict(page=2048), dict(dim=40), dict(dim=272),
                                dict(dim=0), dict(block=8), dict(block=64), dict(block=24), dict(pages=0),
                                dict(heads=0)])
def test_cache_sizes_that_are_refused(kw):
    from sglang_lite_amd import paged_kv as P

    sizes = dict(pages=4, heads=2, page=32, dim=64) | {k: v for k, v in kw.items() if k != "block"}
    with pytest.raises(ValueError):
        P.PagedKV.empty(**sizes, block=kw.get("block", 16), device="cpu")


def test_append_refusals():
    from sglang_lite_amd import paged_kv as P

    c = _cache()
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    bt, st = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        P.append_kv(c, k, k, bt, st)
    cu, table = torch.zeros(4, dtype=torch.int32), torch.zeros(9, 16, 2)
    bad = [
        (c, k[:, :1], k[:, :1], bt, st), (c, k, k[:2], bt, st), (c, k[..., :32], k[..., :32], bt, st),
        (c, k, k, bt.long(), st), (c, k, k, bt, st.long()), (c, k, k, bt, st[:2]), (c, k, k, bt[0], st),
        (c, k[:2], k[:2], bt, st),                                   # two rows, three sequences
        (c._replace(k=c.k.view(torch.uint8)), k, k, bt, st), (c._replace(v=c.v[:3]), k, k, bt, st),
        (c._replace(k_scale=c.k_scale.double()), k, k, bt, st), (c._replace(v_scale=c.v_scale[:, :1]), k, k, bt, st),
        (c._replace(k=c.k.transpose(0, 1).contiguous().transpose(0, 1)), k, k, bt, st),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            P.append_kv(*args)
    for kw in (dict(cu_tokens=cu[:3]), dict(cu_tokens=cu.long()), dict(positions=st),
               dict(table=torch.zeros(9, 12, 2)), dict(table=table, offset=4), dict(table=table, offset=40),
               dict(table=table, positions=st.long()), dict(table=table, positions=st[:2])):
        with pytest.raises(ValueError):
            P.append_kv(c, k, k, bt, st, **kw)
    for a, b in ((k.double(), k.double()), (k, k.float())):
        with pytest.raises(TypeError):
            P.append_kv(c, a, b, bt, st)


def test_attention_refusals():
    from sglang_lite_amd import paged_kv as P

    c = _cache()
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    bt, n = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        P.paged_attn(q, c, bt, n)
    for args in ((q[:, :3], c, bt, n), (q[..., :32], c, bt, n), (q[0], c, bt, n), (q[:2], c, bt, n),
                 (q, c, bt.long(), n), (q, c, bt, n.long()), (q, c, bt[:2], n)):
        with pytest.raises(ValueError):
            P.paged_attn(*args)
    for kw in (dict(window=-1), dict(window=4, causal=False), dict(sink=torch.zeros(3)),
               dict(sink=torch.zeros(4).double()), dict(cu_tokens=n)):
        with pytest.raises(ValueError):
            P.paged_attn(q, c, bt, n, **kw)
    with pytest.raises(TypeError):
        P.paged_attn(q.float(), c, bt, n)


def test_the_library_refuses_before_any_launch():
    """Through the C ABI with null pointers: sizes, alignment, a missing workspace."""
    from sglang_lite_amd import _lib as L

    one = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(one) + 63) & ~63

    def rotary(**kw):
        a = dict(x=p, dt=0, T=2, H=2, D=64, xt=128, xh=64, table=p, n=8, rot=64, off=0, pos=p, p64=0, il=0,
                 inv=0, out=p, ot=128, oh=64, st=None) | kw
        return list(a.values())

    for kw in (dict(dt=3), dict(T=-1), dict(D=0), dict(rot=63), dict(rot=66), dict(off=-1), dict(off=2), dict(n=0),
               dict(x=None), dict(table=None), dict(pos=None), dict(out=None), dict(x=p + 1), dict(table=p + 4),
               dict(ot=192)):
        with pytest.raises(ValueError, match="rotary"):
            L.call("sgl_rotary", *rotary(**kw))
    L.call("sgl_rotary", *rotary(T=0, x=None))

    def append(**kw):
        a = dict(k=p, kt=128, kh=64, v=p, vt=128, vh=64, dt=0, T=2, B=2, H=2, D=64, cu=None, start=p, bt=p, cols=4,
                 page=32, block=16, pages=8, table=None, n=0, rot=0, off=0, pos=None, il=0, kc=p, vc=p, ks=p, vs=p,
                 st=None) | kw
        return list(a.values())

    for kw in (dict(dt=3), dict(T=3), dict(H=0), dict(D=72), dict(D=512), dict(page=48), dict(block=64), dict(block=4),
               dict(pages=0), dict(cols=0), dict(cols=1 << 27), dict(k=None), dict(start=None), dict(kc=None),
               dict(k=p + 2), dict(kt=127), dict(vh=63), dict(kc=p + 8), dict(table=p, n=4, rot=24),
               dict(table=p, n=4, rot=32, off=36), dict(table=p, n=0, rot=32), dict(table=p + 8, n=4, rot=32),
               dict(table=p, n=4, rot=32, off=4)):
        with pytest.raises(ValueError, match="kv8_append"):
            L.call("sgl_kv8_append", *append(**kw))
    L.call("sgl_kv8_append", *append(T=0, cu=p, k=None))

    def attn(**kw):
        a = dict(q=p, qt=256, qh=64, dt=0, T=2, B=2, H=2, G=2, D=64, cu=None, lens=p, bt=p, cols=4, page=32, block=16,
                 pages=8, kc=p, vc=p, ks=p, vs=p, scale=0.125, causal=1, window=0, sink=None, out=p, ws=None, nws=0,
                 st=None) | kw
        return list(a.values())

    for kw in (dict(dt=2), dict(T=3), dict(G=0), dict(G=40000), dict(D=100), dict(page=20), dict(block=256), dict(window=-1),
               dict(window=3, causal=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(q=None), dict(lens=None), dict(out=None), dict(q=p + 2), dict(qh=60),
               dict(vc=p + 4), dict(out=p + 8)):
        with pytest.raises(ValueError, match="kv8_attn"):
            L.call("sgl_kv8_attn", *attn(**kw))
    with pytest.raises(L.SglError, match="workspace") as e:
        L.call("sgl_kv8_attn", *attn(cols=1000))
    assert e.value.status == L.SGL_ERR_WORKSPACE
    L.call("sgl_kv8_attn", *attn(T=0, cu=p, q=None))
    assert L.load().sgl_kv8_attn_workspace_size(-1, 1, 1, 1, 64, 4096) == 0


def test_oracle_attention_is_a_softmax():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((3, 4, 8)), rng.standard_normal((6, 2, 8)), rng.standard_normal((6, 2, 8))
    o, _, _ = OP.attention(q, k, v, np.ones(6, bool), 3, 0.3)
    kt, vt = (torch.from_numpy(x).repeat_interleave(2, 1).transpose(0, 1) for x in (k, v))
    ref = torch.nn.functional.scaled_dot_product_attention(
        torch.from_numpy(q).transpose(0, 1), kt, vt, scale=0.3,
        attn_mask=torch.arange(6) <= torch.arange(3, 6)[:, None]).transpose(0, 1)
    np.testing.assert_allclose(o, ref.numpy(), rtol=1e-12, atol=1e-12)
