"""An output that lies on its input: only the very same rows are taken."""

from __future__ import annotations

import numpy as np
import pytest
import torch


def _rows(t):
    """The element numbers of a tensor [T, H, D], row by row."""
    T, H, D = t.shape
    s = t.stride()
    at = t.storage_offset() + np.arange(T)[:, None, None] * s[0] + np.arange(H)[:, None] * s[1] + np.arange(D) * s[2]
    return at.reshape(T * H, D)


def test_what_counts_as_overlap():
    """Against the sets of elements: never less is refused than shares memory without being the
    same rows, and with equal strides never more."""
    from sglang_lite_amd.rotary import _apart, check_apart

    rng = np.random.default_rng(0)
    refused = taken = 0
    for _ in range(6000):
        T, H, D = (int(rng.integers(1, 4)) for _ in range(3))
        buf = torch.zeros(400)
        s = [int(v) for v in rng.integers(1, 20, 4)]
        same = rng.random() < 0.7
        if same:
            s[2:] = s[:2]
        if not (_apart(T, s[2], H, s[3], D) or _apart(H, s[3], T, s[2], D)):
            continue
        x = torch.as_strided(buf, (T, H, D), (s[0], s[1], 1), int(rng.integers(0, 60)))
        out = torch.as_strided(buf, (T, H, D), (s[2], s[3], 1), int(rng.integers(0, 60)))
        a, b = _rows(x), _rows(out)
        bad = bool(np.intersect1d(a, b).size) and not np.array_equal(a, b)
        try:
            check_apart(x, out, "t")
            assert not bad
            taken += 1
        except ValueError as e:
            assert "overlaps" in str(e)
            assert bad or not same
            refused += 1
    assert refused > 500 and taken > 500


def test_views_of_a_fused_projection_are_apart():
    from sglang_lite_amd.rotary import check_apart

    fused = torch.zeros(5, 12, 8)
    check_apart(fused[:, :4], fused[:, 8:], "t")
    check_apart(fused[:, 0::2], fused[:, 1::2], "t")
    check_apart(fused[:, :4], fused[:, :4], "t")
    check_apart(fused[:0], fused[:0], "t")
    for x, out in ((fused[:, :4], fused[:, 2:6]), (fused[:4], fused[1:]), (fused[:, 4:8], fused[:, 3:7]),
                   (fused[1:], fused[:4])):
        with pytest.raises(ValueError, match="overlaps"):
            check_apart(x, out, "t")


@pytest.mark.gpu
def test_rotary_and_attention_refuse_what_overlaps(gpu):
    from sglang_lite_amd import paged_kv as P
    from sglang_lite_amd import rotary as R

    T, H, D = 40, 4, 64
    table = R.rotary_table(64, D, device=gpu)
    at = torch.arange(T, device=gpu)
    fused = torch.randn(T, 3 * H, D, device=gpu).to(torch.bfloat16)
    want = R.rotary(fused[:, :H], table, at)
    with pytest.raises(ValueError, match="overlaps"):
        R.rotary(fused[:, :H], table, at, out=fused[:, 2:2 + H])
    with pytest.raises(ValueError, match="overlaps"):
        R.rotary(fused[1:, :H], table, at[1:], out=fused[:-1, :H])
    assert torch.equal(R.rotary(fused[:, :H], table, at, out=fused[:, 2 * H:]), want)
    assert torch.equal(R.rotary(fused[:, :H], table, at, out=fused[:, :H]), want)

    cache = P.PagedKV.empty(4, 2, 32, D, block=16, device=gpu)
    k, v = torch.randn(2, 100, 2, D, device=gpu).to(torch.bfloat16)
    bt = torch.arange(4, dtype=torch.int32, device=gpu).view(1, 4)
    zero, lens = (torch.tensor([n], dtype=torch.int32, device=gpu) for n in (0, 100))
    P.append_kv(cache, k, v, bt, zero, cu_tokens=torch.tensor([0, 100], dtype=torch.int32, device=gpu))
    for n in (1, T):
        cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
        buf = torch.randn(n * H * D + 64, device=gpu).to(torch.bfloat16)
        q = buf[:n * H * D].view(n, H, D)
        want = P.paged_attn(q, cache, bt, lens, cu_tokens=cu)
        with pytest.raises(ValueError, match="overlaps"):
            P.paged_attn(q, cache, bt, lens, cu_tokens=cu, out=buf[64:].view(n, H, D))
        got = P.paged_attn(q, cache, bt, lens, cu_tokens=cu, out=q)
        assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
