"""What the attention's forms over the 8-bit paged cache (first tokens beside a window, a common
prefix) do without a GPU: refusals, and the rules that divide their work."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

CSRC = Path(__file__).resolve().parents[1] / "sglang-lite_amd" / "csrc"

WRAPPERS = r"""
#include "sgl_rules.h"
using namespace sgl;
extern "C" {
int64_t reach(int64_t T, int64_t B, int64_t cap, int64_t w, int64_t f) { return kv8_attn_reach(T, B, cap, w, f); }
int window_whole(int64_t reach, int64_t items, int64_t cus) { return kv8_window_whole(reach, items, cus); }
int64_t plan_parts(int64_t T, int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t cap, int window) {
  return kv8_attn_plan(T, B, Hkv, G, D, cap, 256, window != 0).parts;
}
void joint(int64_t T, int64_t B, int64_t n, int64_t Hkv, int64_t G, int64_t D, int64_t cap, int64_t* o) {
  const Kv8JointPlan p = kv8_joint_plan(T, B, n, Hkv, G, D, cap, 256);
  o[0] = p.row_tile; o[1] = p.group_rows; o[2] = p.slot_rows; o[3] = p.per_cu; o[4] = p.parts; o[5] = p.items;
  o[6] = p.group_items;
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("forms")
    src, so = d / "r.cpp", d / "r.so"
    src.write_text(WRAPPERS)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o",
                    str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    i64 = ctypes.c_int64
    lib.reach.restype, lib.reach.argtypes = i64, [i64] * 5
    lib.window_whole.argtypes = [i64] * 3
    lib.plan_parts.restype, lib.plan_parts.argtypes = i64, [i64] * 6 + [ctypes.c_int]
    lib.joint.argtypes = [i64] * 7 + [ctypes.c_void_p]
    return lib


def test_window_rules(rules):
    assert rules.reach(1, 1, 20000, 0, 0) == rules.reach(1, 1, 20000, 500, 0) == 20000
    assert rules.reach(1, 1, 20000, 1024, 4) == 1024 + 4 + 1 + 128 and rules.reach(9, 3, 900, 1024, 4) == 900
    assert rules.window_whole(1157, 8, 256) and not rules.window_whole(1633, 8, 256)      # 1 sequence
    assert rules.window_whole(2133, 128, 256) and not rules.window_whole(3133, 128, 256)  # 16
    assert rules.window_whole(4240, 256, 256) and not rules.window_whole(4240, 320, 256)  # 32, 40
    assert rules.window_whole(4240, 512, 256) and not rules.window_whole(8144, 512, 256)  # 64
    # plain calls are divided as before, whatever the window
    assert rules.plan_parts(64, 64, 8, 4, 128, 4240, 0) == 32 and rules.plan_parts(64, 64, 8, 4, 128, 4240, 1) == 0


def test_windows_and_first_tokens_of_any_length(rules):
    """Longer than any table: the table's width, whatever their sum does in 64 bits."""
    for window, first in ((1 << 62, 1 << 62), (2 ** 63 - 1, 1), (1, 2 ** 63 - 1), (2 ** 63 - 1, 2 ** 63 - 1)):
        assert rules.reach(1, 1, 20000, window, first) == 20000
    assert rules.reach(1, 1, 20000, 19000, 900) == 20000 and rules.reach(1, 1, 20000, 9000, 9000) == 18129


def test_joint_plans(rules):
    o = (ctypes.c_int64 * 7)()

    def plan(*a):
        rules.joint(*a, o)
        return list(o)

    rng = np.random.default_rng(0)
    for _ in range(2000):
        B, Hkv, G = (int(rng.integers(1, n)) for n in (200, 20, 40))
        n, D = int(rng.integers(1, B + 1)), 16 * int(rng.integers(1, 17))
        T, cap = B * int(rng.integers(1, 40)), 16 << int(rng.integers(0, 16))
        rt, rg, slot, per_cu, parts, items, group_items = plan(T, B, n, Hkv, G, D, cap)
        few = 96 if D <= 128 else 32
        if T * G // B > few or (T * G // n > few and T * Hkv * G * D * cap > 7e9):
            assert items == 0
            continue
        assert rt in (16, 32) and rg in (16, 32) and rg >= rt and slot == rg and parts % 8 == 0 and parts >= 8
        assert rt == 16 or D <= 128
        assert per_cu in (1, 2) and (per_cu == 1 or D <= 128)
        # a bound on the row tiles of any division of the rows among the sequences, and the groups
        for count, tile, most in ((B, rt, items), (n, rg, group_items)):
            cut = np.sort(rng.integers(0, T + 1, count - 1))
            rows = np.diff(np.concatenate([[0], cut, [T]])) * G
            assert Hkv * int((-(-rows // tile)).sum()) <= most
    assert plan(64, 64, 1, 8, 4, 128, 9192)[5] and not plan(128, 128, 2, 4, 16, 128, 35768)[5]


def test_joint_plans_have_a_kernel(rules):
    """Workgroups a CU that the launch takes for granted: two for heads up to 64, one for groups' tiles of 16 rows
    of wider heads and for heads above 128."""
    o = (ctypes.c_int64 * 7)()
    rng = np.random.default_rng(1)
    seen = set()
    for i in range(20000):
        B, Hkv, G = (int(2 ** rng.uniform(0, n)) for n in (9, 4, 5))
        n, D = int(rng.integers(1, B + 1)), 16 * int(rng.integers(1, 17))
        T, cap = int(rng.integers(1, B * 40)), 16 << int(rng.integers(0, 16))
        rules.joint(T, B, n, Hkv, G, D, cap, o)
        rt, rg, _, per_cu, _, items, _ = o
        if items:
            seen.add((64 if D <= 64 else 128 if D <= 128 else 256, rg, rt, per_cu))
    assert seen == {(64, 16, 16, 2), (64, 32, 16, 2), (64, 32, 32, 2), (128, 16, 16, 1), (128, 32, 16, 1),
                    (128, 32, 16, 2), (128, 32, 32, 1), (128, 32, 32, 2), (256, 16, 16, 1), (256, 32, 16, 1)}


def _args(B=3, heads=2, hq=4, dim=64, page=32):
    from sglang_lite_amd import paged_kv as P

    cache = P.PagedKV.empty(4, heads, page, dim, block=16, device="cpu")
    q = torch.zeros(B, hq, dim, dtype=torch.bfloat16)
    return P, cache, q, torch.zeros(B, 2, dtype=torch.int32), torch.ones(B, dtype=torch.int32)


def test_refusals():
    P, cache, q, bt, lens = _args()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    ok = dict(cu_groups=i32(0, 3), shared=i32(64))
    for kw in (dict(window=8, first=4), ok, dict(cu_groups=i32(0, 1, 3), shared=i32(64, 32), causal=False)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            P.paged_attn(q, cache, bt, lens, **kw)
    for kw in (dict(first=4), dict(window=8, first=-1), dict(window=8, first=2, causal=False), dict(cu_groups=i32(0, 3)),
               dict(shared=i32(64)), dict(ok, window=16), dict(ok, window=16, first=2),
               dict(ok, shared=torch.tensor([64])), dict(ok, cu_groups=torch.tensor([0, 3])),
               dict(ok, cu_groups=i32(0, 1, 3)), dict(cu_groups=i32(0), shared=i32()),
               dict(ok, shared=i32(64)[None]), dict(cu_groups=torch.zeros(4, dtype=torch.int32)[::2], shared=i32(64))):
        with pytest.raises(ValueError):
            P.paged_attn(q, cache, bt, lens, **kw)


def test_entry_points_refuse_before_any_launch():
    from sglang_lite_amd import _lib as L

    lib = L.load()
    head = (None, 512, 64, 0, 3, 3, 2, 4, 64, None, None, None)  # q, strides, dtype, T, B, Hkv, G, D, cu, lens, table

    def first(window, first, causal=1, row_pages=2):
        return lib.sgl_kv8_attn_first(*head, row_pages, 32, 16, 4, None, None, None, None, 1.0, causal, window, first,
                                      None, None, None, 0, None)

    for kw in (dict(window=0, first=4), dict(window=8, first=-1), dict(window=-1, first=0),
               dict(window=8, first=4, causal=0), dict(window=8, first=4, row_pages=0), dict(window=8, first=4)):
        assert first(**kw) == L.SGL_ERR_INVALID_ARG, kw  # (the last one: null pointers)

    def shared(groups, T=3):
        return lib.sgl_kv8_attn_shared(None, 512, 64, 0, T, T, 2, 4, 64, None, None, None, 2, 32, 16, 4, None, None,
                                       None, None, 1.0, 1, None, groups, None, None, None, None, 0, None)

    assert shared(0) == shared(-1) == shared(1 << 25) == shared(1) == L.SGL_ERR_INVALID_ARG
    assert shared(1, T=0) == L.SGL_OK
    size = lib.sgl_kv8_attn_shared_workspace_size
    assert size(64, 64, 8, 4, 128, 9192, 1) > 64 * 32 * 128 * 4 and size(64, 64, 8, 4, 128, 9192, 0) == 0
    assert size(-1, 64, 8, 4, 128, 9192, 1) == 0
    assert lib.sgl_kv8_attn_first_workspace_size(64, 64, 8, 4, 128, 1 << 20, 4096, 4) == 0  # whole items
    assert lib.sgl_kv8_attn_first_workspace_size(1, 1, 8, 4, 128, 1 << 20, 4096, 4) > 0
    assert lib.sgl_kv8_attn_first_workspace_size(1, 1, 8, 4, 128, 1 << 20, -1, 4) == 0
