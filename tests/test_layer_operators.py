"""What the rotary axes and the norms between blocks do without a GPU: the axes of the pairs,
refusals, the plan of the rows."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parents[1] / "sglang-lite_amd" / "csrc"


def test_axes_of_pairs():
    from sglang_lite_amd import rotary as R

    assert R.rotary_axes((2, 1, 1), device="cpu").tolist() == [0, 0, 1, 2]
    assert R.rotary_axes((2, 3, 1), spread=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 1]
    assert R.rotary_axes((24, 20, 20), spread=True, device="cpu").tolist() == [0, 1, 2] * 20 + [0] * 4
    assert R.rotary_axes((0, 2), device="cpu").tolist() == [1, 1]
    assert R.rotary_axes((4,), device="cpu").dtype == torch.uint8
    for bad in ((), (0, 0), (1, -1, 2), (1, 1, 1, 1, 1)):
        with pytest.raises(ValueError):
            R.rotary_axes(bad, device="cpu")


def test_rotary_axes_refusals():
    from sglang_lite_amd import rotary as R

    x, table = torch.zeros(4, 2, 64), torch.zeros(8, 32, 2)
    axes, pos = R.rotary_axes((10, 22), device="cpu"), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        R.rotary(x, table, pos, axes=axes)
    for a, p in ((axes[:-1], pos), (axes.int(), pos), (axes, pos[0]), (axes, pos[:, :3]), (axes, pos[:0]),
                 (axes, torch.zeros(5, 4, dtype=torch.int32)), (axes[None], pos),
                 (torch.zeros(64, dtype=torch.uint8)[::2], pos)):
        with pytest.raises(ValueError):
            R.rotary(x, table, p, axes=a)
    with pytest.raises(TypeError):
        R.rotary(x, table, pos.float(), axes=axes)


def test_append_axes_refusals():
    from sglang_lite_amd import paged_kv as P
    from sglang_lite_amd import rotary as R

    cache = P.PagedKV.empty(4, 2, 32, 64, block=16, device="cpu")
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    bt, st = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    table, axes = torch.zeros(8, 32, 2), R.rotary_axes((12, 20), device="cpu")
    pos = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        P.append_kv(cache, k, k, bt, st, table=table, positions=pos, axes=axes)
    for kw in (dict(table=table, axes=axes), dict(axes=axes, positions=pos),
               dict(table=table, axes=axes, positions=pos[0]), dict(table=table, axes=axes, positions=pos.long()),
               dict(table=table, axes=axes[:8], positions=pos), dict(table=table, positions=pos),
               dict(table=table, axes=axes, positions=torch.zeros(3, 2, dtype=torch.int32).t())):
        with pytest.raises(ValueError):
            P.append_kv(cache, k, k, bt, st, **kw)


def test_norm_refusals():
    from sglang_lite_amd import kernel as K
    from sglang_lite_amd.norms import residual_norm

    x, r, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(4, 256), torch.ones(256)
    with pytest.raises(RuntimeError, match="no CPU path"):
        residual_norm(x, r, w)
    for args, kw in (((x, r[:3], w), {}), ((x, r, w[:100]), {}), ((x, r, w[None]), {}), ((x, r), dict(quant=True)),
                     ((x, r, w), dict(after=w[:1])), ((x, r, w), dict(quant=True, block_size=48)),
                     ((x[:, :100], r[:, :100], w[:100]), dict(quant=True)),
                     ((x, r, w), dict(quant=True, scale_dtype=K.E8M0)),
                     ((torch.zeros(2, 0), torch.zeros(2, 0), torch.zeros(0)), {}),
                     ((torch.zeros(1, 16385), torch.zeros(1, 16385)), {}),
                     ((torch.zeros(()), torch.zeros(()), w), {})):
        with pytest.raises(ValueError):
            residual_norm(*args, **kw)
    for args, kw in (((x.double(), r, w), {}), ((x, r.half(), w), {}), ((x, r, w.double()), {}),
                     ((x, r, w), dict(gate=w.double())), ((x.float(), x, w), {}),
                     ((x, r, w), dict(quant=True, scale_dtype=torch.float16))):
        with pytest.raises(TypeError):
            residual_norm(*args, **kw)


def test_rows_that_meet():
    """What an in-place residual may lie beside: by the bytes of each element."""
    from sglang_lite_amd import norms as N

    buf = torch.zeros(64, dtype=torch.float32)

    def bytes_of(t):
        size = t.element_size()
        return {t.data_ptr() + (i * t.stride(0) + e) * size + k for i in range(t.shape[0]) for e in range(t.shape[1])
                for k in range(size)}

    def refused(check, *a):
        try:
            check(*a, "x")
        except ValueError:
            return True
        return False

    met = 0
    for T, H, hs, h0 in ((1, 4, 4, 7), (3, 4, 4, 8), (3, 4, 9, 0), (4, 3, 10, 12), (1, 5, 11, 20)):
        h = buf.as_strided((T, H), (hs, 1), h0)
        there = bytes_of(h)
        for dtype in (torch.float32, torch.bfloat16):
            flat = buf.view(dtype)
            for xs in (0, 2, 3, hs, 2 * hs):
                for x0 in range(0, flat.numel() - (T - 1) * xs - H + 1):
                    x = flat.as_strided((T, H), (xs, 1), x0)
                    meets = bool(bytes_of(x) & there)
                    same = dtype is torch.float32 and x0 == h0 and (xs == hs or T == 1)
                    if xs * x.element_size() == hs * 4 or xs == 0 or T == 1 or meets:
                        assert refused(N._check_apart, x, h) == (meets and not same), (T, H, hs, h0, dtype, xs, x0)
                    met += meets
            for x0 in range(0, flat.numel() - H + 1):
                w = flat[x0:x0 + H]
                assert refused(N._check_weight, w, h) == bool(bytes_of(w[None]) & there)
    assert met > 100
    wide = torch.zeros(6, 2, 8)
    N._check_apart(wide[:, 1], wide[:, 0], "x")
    N._check_weight(None, wide[:, 0], "before")
    N._check_apart(wide[:0, 0], wide[:0, 0], "x")


def test_entry_points_refuse_before_any_launch():
    from sglang_lite_amd import _lib as L

    lib = L.load()

    def norm(dtype=0, T=4, H=256, res=0, eps=1e-6, quant=0, group=128, mode=0, e8m0=0, before=None):
        return lib.sgl_residual_norm(None, dtype, T, H, H, None, res, H, None, 0, None, 0, 0, 0, 1.0, before, 0, eps,
                                     None, H, None, quant, None, group, mode, e8m0, None)

    assert norm(T=0) == L.SGL_OK
    for kw in (dict(), dict(dtype=3), dict(res=1), dict(T=-1), dict(H=0), dict(H=16385), dict(eps=-1.0),
               dict(eps=float("nan")), dict(quant=1), dict(quant=1, before=1 << 12, group=48),
               dict(quant=1, before=1 << 12, H=200), dict(quant=1, before=1 << 12, mode=4),
               dict(quant=1, before=1 << 12, e8m0=1)):
        assert norm(**kw) == L.SGL_ERR_INVALID_ARG, kw
    rot = (None, 0, 4, 2, 64, 128, 64, None)
    for n_positions, rot_dim, n_axes in ((100, 64, 0), (100, 64, 5), (1 << 31, 64, 2), (100, 65, 2), (100, 64, 2)):
        assert lib.sgl_rotary_axes(*rot, n_positions, rot_dim, 0, None, 0, n_axes, None, 0, 0, None, 128, 64,
                                   None) == L.SGL_ERR_INVALID_ARG


def test_norm_plan(tmp_path):
    src, so = tmp_path / "r.cpp", tmp_path / "r.so"
    src.write_text('#include "sgl_rules.h"\nextern "C" void plan(int64_t T, int64_t u, int64_t cus, int64_t* o) {\n'
                   "  const sgl::NormPlan p = sgl::norm_plan(T, u, cus);\n"
                   "  o[0] = p.threads; o[1] = p.units; o[2] = p.grid;\n}\n"
                   'extern "C" int64_t most() { return sgl::kNormMost; }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o",
                    str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.plan.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_void_p]
    lib.most.restype = ctypes.c_int64
    o = (ctypes.c_int64 * 3)()
    for units in list(range(1, 300)) + list(range(300, lib.most() // 8 + 1, 7)) + [lib.most() // 8]:
        for T in (1, 100, 100000):
            lib.plan(T, units, 256, o)
            threads, per, grid = o
            assert threads % 64 == 0 and 64 <= threads <= 1024 and threads * per >= units
            assert per == (1 if units <= 1024 else 2)
            assert 1 <= grid <= T


def test_rotary_threads_have_all_heads(tmp_path):
    """Four heads a thread at most: the kernel goes over them once."""
    src, so = tmp_path / "h.cpp", tmp_path / "h.so"
    src.write_text('#include "sgl_rules.h"\nextern "C" int threads(int64_t T, int64_t H, int64_t u, int64_t cus) {\n'
                   "  return sgl::rotary_head_threads(T, H, u, cus);\n}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o",
                    str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.threads.argtypes = [ctypes.c_int64] * 4
    for H in list(range(1, 300)) + [4095, 4096, 4097, 65535, 65536]:
        for T in (1, 1000, 100000, 2 ** 31 - 1):
            n = lib.threads(T, H, 8, 256)
            assert n <= H <= 4 * n
