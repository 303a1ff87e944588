"""Rotary positions on gfx950.

* ``rotary_table(n_positions, rot_dim, ...)`` -- the rotations of every
  position, made once: fp32 ``[n_positions, rot_dim / 2, 2]`` (cos, sin), from
  angles in 64 bits; plain, or scaled for long contexts.
* ``rotary(x, table, positions, ...)`` -- ``x`` ``[T, H, D]`` with the pairs of
  ``rot_dim`` elements of each head turned by their row's position; ``inverse``
  turns them back, which is also the gradient with respect to ``x``.

``paged_kv.append_kv`` takes the same table and turns the keys on their way
into the cache.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.SGL_BF16, torch.float16: _lib.SGL_F16, torch.float32: _lib.SGL_F32}


def frequencies(rot_dim: int, base: float = 10000.0, scaling: Optional[dict] = None):
    """Radians per position of each pair (fp64 on the CPU), and the factor that
    the rotated elements are multiplied by.

    ``scaling``: None, or a dict with ``type``
      ``"linear"``  ``factor``: every frequency divided by it;
      ``"ntk"``     ``factor``: the base grows so that the slowest pair turns
                    ``factor`` times slower and the fastest as before;
      ``"yarn"``    ``factor``, ``original`` (positions the model was trained
                    on), ``beta_fast`` (32), ``beta_slow`` (1): pairs that turn
                    more than ``beta_fast`` times over ``original`` positions
                    keep their frequency, those below ``beta_slow`` turns have
                    it divided, a linear ramp over the pairs between; ``length``
                    (1 + 0.1 ln factor) multiplies the elements."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even and at least 2, got {rot_dim}")
    if not 1.0 < base < math.inf:
        raise ValueError(f"base must be greater than 1, got {base}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-i / rot_dim), 1.0
    kind, factor = scaling.get("type"), float(scaling.get("factor", 0.0))
    if kind not in ("linear", "ntk", "yarn"):
        raise ValueError(f"scaling type must be linear, ntk or yarn, got {kind!r}")
    if not 1.0 <= factor < math.inf:
        raise ValueError(f"scaling factor must be at least 1, got {factor}")
    if kind == "linear":
        return base ** (-i / rot_dim) / factor, 1.0
    if kind == "ntk":
        if rot_dim == 2:
            return base ** (-i / rot_dim), 1.0
        return (base * factor ** (rot_dim / (rot_dim - 2))) ** (-i / rot_dim), 1.0
    original = float(scaling.get("original", 0.0))
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not 1.0 <= original < math.inf or not 0.0 < slow <= fast < math.inf:
        raise ValueError(f"yarn scaling needs original positions and 0 < beta_slow <= beta_fast, got "
                         f"{scaling.get('original')}, {slow} and {fast}")
    freq = base ** (-i / rot_dim)

    def pair(turns: float) -> float:  # the pair that makes so many turns over `original` positions
        return rot_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo = max(math.floor(pair(fast)), 0)
    hi = min(math.ceil(pair(slow)), rot_dim - 1)
    ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    length = scaling.get("length")
    return freq / factor * ramp + freq * (1 - ramp), \
        0.1 * math.log(factor) + 1.0 if length is None else float(length)


def rotary_table(n_positions: int, rot_dim: int, base: float = 10000.0, *,
                 scaling: Optional[dict] = None, device="cuda") -> torch.Tensor:
    """fp32 ``[n_positions, rot_dim / 2, 2]``: (cos, sin) of each position and pair."""
    if n_positions < 1:
        raise ValueError(f"rotary_table: n_positions must be at least 1, got {n_positions}")
    freq, length = frequencies(rot_dim, base, scaling)
    if torch.device(device).type == "cpu":
        raise RuntimeError("rotary_table: sglang_lite_amd runs only on a ROCm (gfx950) device "
                           "(there is no CPU path)")
    freq = freq.to(device)
    table = torch.empty(n_positions, rot_dim // 2, 2, dtype=torch.float32, device=freq.device)
    _lib.call_on(freq.get_device(), "sgl_rotary_table", freq.data_ptr(), length, n_positions, rot_dim,
                 table.data_ptr())
    return table


def check_table(table: torch.Tensor, offset: int, dim: int, what: str) -> int:
    """rot_dim of a table that fits into heads of ``dim`` elements at ``offset``."""
    shape = table.shape
    if len(shape) != 3 or shape[2] != 2 or table.dtype is not torch.float32 or not table.is_contiguous():
        raise ValueError(f"{what}: table must be a contiguous float32 [positions, pairs, 2], got "
                         f"{table.dtype} {tuple(shape)}")
    rot = 2 * shape[1]
    if offset < 0 or offset + rot > dim:
        raise ValueError(f"{what}: {rot} rotated elements at offset {offset} do not fit into {dim}")
    return rot


def _apart(outer: int, so: int, inner: int, si: int, D: int) -> bool:
    """Whether ``outer`` groups of ``inner`` rows of ``D`` elements, at these strides, lie apart."""
    return (inner <= 1 or si >= D) and (outer <= 1 or so >= (inner - 1) * si + D)


def check_apart(x: torch.Tensor, out: torch.Tensor, what: str) -> None:
    """Refuse an ``out`` whose rows (none on another) share memory with ``x`` ``[T, H, D]`` and are
    not its very rows: one workgroup would overwrite what another is still to read."""
    n, D = out.shape[:2], out.shape[2]
    if 0 in out.shape:
        return
    a, b, size = x.data_ptr(), out.data_ptr(), out.element_size()

    def end(t):  # bytes from its first element to behind its last
        return (sum((m - 1) * s for m, s in zip(t.shape, t.stride())) + 1) * size

    if a + end(x) <= b or b + end(out) <= a:
        return
    d, rest = divmod(b - a, size)
    axes = [(s, m, r) for m, s, r in zip(n, out.stride(), x.stride()) if m > 1]
    if not rest and all(s == r for s, _, r in axes):
        if d == 0:
            return
        # rows (i, j) of x and (i', j') of out meet where d + (i' - i) s0 + (j' - j) s1 is less than D
        near = [d]
        axes.sort(reverse=True)
        for k, (s, m, _) in enumerate(axes):
            reach = sum((m2 - 1) * s2 for s2, m2, _ in axes[k + 1:]) + D - 1
            near = [v - i * s for v in near
                    for i in range(max(1 - m, -((reach - v) // s)), min(m - 1, (v + reach) // s) + 1)]
        if all(abs(v) >= D for v in near):
            return
    raise ValueError(f"{what}: out overlaps the input without being it")


def rotary(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, *,
           interleaved: bool = False, offset: int = 0, inverse: bool = False,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` ``[T, H, D]`` (bf16, f16 or f32; any strides with a dense last
    dimension) with elements ``[offset, offset + rot_dim)`` of every head turned
    by ``positions`` (int32 or int64 ``[T]``): pair ``i`` is elements ``i`` and
    ``i + rot_dim / 2`` of them, or ``2 i`` and ``2 i + 1`` with ``interleaved``.
    A negative position (a padding row) leaves its row as it is, one behind the
    table gives NaN.  ``out`` may be ``x`` itself, or share no memory with its rows."""
    shape = x.shape
    if len(shape) != 3:
        raise ValueError(f"rotary: expected x [T, H, D], got {tuple(shape)}")
    T, H, D = shape
    dt = DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"rotary: x must be bfloat16, float16 or float32, got {x.dtype}")
    rot = check_table(table, offset, D, "rotary")
    if positions.shape != (T,):
        raise ValueError(f"rotary: expected positions [{T}], got {tuple(positions.shape)}")
    wide = positions.dtype is torch.int64
    if not wide and positions.dtype is not torch.int32:
        raise TypeError(f"rotary: positions must be int32 or int64, got {positions.dtype}")
    d = _lib.device_of("rotary", x, table, positions, out)
    xs = x.stride()
    if xs[2] != 1 and D > 1:
        x = x.contiguous()
        xs = x.stride()
    given = out is not None
    if not given:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not x.dtype or (out.stride(2) != 1 and D > 1):
        raise ValueError(f"rotary: out must be {x.dtype} {tuple(shape)} with a dense last "
                         f"dimension, got {out.dtype} {tuple(out.shape)}")
    os = out.stride()
    if not (_apart(T, os[0], H, os[1], D) or _apart(H, os[1], T, os[0], D)):
        raise ValueError("rotary: rows of out overlap")
    if given and out is not x:
        check_apart(x, out, "rotary")
    if not positions.is_contiguous():
        positions = positions.contiguous()
    _lib.call_on(d, "sgl_rotary", x.data_ptr(), dt, T, H, D, xs[0], xs[1], table.data_ptr(),
                 table.shape[0], rot, offset, positions.data_ptr(), wide, interleaved, inverse,
                 out.data_ptr(), os[0], os[1])
    return out


__all__ = ["frequencies", "rotary", "rotary_table"]
