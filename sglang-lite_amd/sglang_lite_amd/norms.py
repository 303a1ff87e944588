"""What stands between two blocks of a layer, on gfx950, in one launch.

``residual_norm(x, residual, before, ...)``: the norm behind the block that made
``x``, its gate and residual scale, the sum with the residual stream, and the
norm before the next block, whose result may come as the e4m3 codes and scales
that ``kernel.fp8_gemm`` reads::

    h, y = residual_norm(x, residual, w)                       # sum and norm
    h, (codes, s) = residual_norm(x, residual, w, quant=True)  # and act_quant
    h, y = residual_norm(x, residual, w, after=v, gate=g, scale=0.5)
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .kernel import E8M0, FP8, scale_mode_for
from .rotary import DTYPES

MAX_DIM = 16384


def _weight(w: torch.Tensor, H: int, name: str) -> int:
    dt = DTYPES.get(w.dtype)
    if dt is None:
        raise TypeError(f"residual_norm: {name} must be bfloat16, float16 or float32, got {w.dtype}")
    if w.shape != (H,) or not w.is_contiguous():
        raise ValueError(f"residual_norm: {name} must be a contiguous [{H}], got {tuple(w.shape)}")
    return dt


def _rows(t: torch.Tensor, H: int):
    """``t`` as rows of ``H`` elements, each dense (a copy where its strides do not allow it), and
    the elements between them."""
    if t.dim() != 2:
        t = t.reshape(-1, H)
    s = t.stride()
    if s[1] != 1 and H > 1:
        t = t.contiguous()
        s = t.stride()
    return t, s[0]


def residual_norm(x: torch.Tensor, residual: torch.Tensor, before: Optional[torch.Tensor] = None, *,
                  after: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  scale: float = 1.0, eps: float = 1e-6, inplace: bool = False, quant: bool = False,
                  block_size: int = 128, scale_fmt: Optional[str] = None,
                  scale_dtype: torch.dtype = torch.float32):
    """``(h, y)`` of ``x`` and ``residual`` ``[..., H]``::

        u = rms(x) * after            (without ``after``: u = x)
        h = residual + scale * gate * u
        y = rms(h) * before           (without ``before``: y is None)

    with ``rms(v) = v / sqrt(mean(v^2) + eps)``.  ``x`` is bf16, f16 or f32,
    ``residual`` of the same type or f32, the weights ``[H]`` and the gate
    (``[H]``, or a shape that broadcasts to x's, which is copied out to it where its rows are not dense or
    not at one stride) any of the three.  ``h`` has residual's type,
    or is ``residual`` itself with ``inplace``; ``y`` has x's.  Everything is
    computed in fp32 and each output rounded once (``y`` is of the unrounded ``h``);
    squares that pass fp32 make zeros and NaN of their row.

    ``quant``: ``y`` is ``(codes, scales)`` as ``act_quant`` gives them of the
    fp32 ``y``: e4m3 ``[..., H]`` and one scale for ``block_size`` elements, by the
    formula of ``scale_fmt`` in ``scale_dtype``."""
    shape = x.shape
    dt = DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"residual_norm: x must be bfloat16, float16 or float32, got {x.dtype}")
    if len(shape) < 1 or residual.shape != shape:
        raise ValueError(f"residual_norm: expected x and residual of one shape [..., H], got {tuple(shape)} and "
                         f"{tuple(residual.shape)}")
    H = shape[-1]
    if not 1 <= H <= MAX_DIM:
        raise ValueError(f"residual_norm: rows of 1 to {MAX_DIM} elements, got {H}")
    rdt = DTYPES.get(residual.dtype)
    if rdt is None or (rdt != dt and rdt != _lib.SGL_F32):
        raise TypeError(f"residual_norm: residual must be {x.dtype} or float32, got {residual.dtype}")
    bdt = adt = gdt = gs = mode = 0
    if before is not None:
        bdt = _weight(before, H, "before")
    if after is not None:
        adt = _weight(after, H, "after")
    if gate is not None:
        gdt = DTYPES.get(gate.dtype)
        if gdt is None:
            raise TypeError(f"residual_norm: gate must be bfloat16, float16 or float32, got {gate.dtype}")
    if quant:
        if before is None:
            raise ValueError("residual_norm: codes are of the norm before the next block, which is missing")
        if block_size not in (32, 64, 128) or H % block_size:
            raise ValueError(f"residual_norm: block_size must be 32, 64 or 128 and divide {H}, got {block_size}")
        if scale_dtype is not torch.float32 and scale_dtype is not E8M0:
            raise TypeError(f"residual_norm: scale_dtype must be float32 or float8_e8m0fnu, got {scale_dtype}")
        mode = scale_mode_for(scale_fmt)
        if scale_dtype is E8M0 and scale_fmt is None:
            raise ValueError("residual_norm: float8_e8m0fnu scales need a scale_fmt (powers of two)")
    d = _lib.device_of("residual_norm", x, residual, before, after, gate)
    gate_rows = False
    if gate is not None:
        if gate.shape == (H,):
            gate = gate if gate.is_contiguous() else gate.contiguous()
        else:
            if gate.shape != shape:
                try:
                    gate = gate.expand(shape)
                except RuntimeError as e:
                    raise ValueError(f"residual_norm: a gate {tuple(gate.shape)} does not broadcast to "
                                     f"{tuple(shape)}") from e
            gate_rows = True
            gate, gs = _rows(gate, H)
    xr, xs = _rows(x, H)
    T = xr.shape[0]
    if inplace:
        try:
            rr = h = residual.view(-1, H)
        except RuntimeError as e:
            raise ValueError("residual_norm: inplace needs a residual whose rows lie at one stride") from e
        rs = hs = rr.stride(0)
        if (H > 1 and rr.stride(1) != 1) or (T > 1 and rs < H):
            raise ValueError("residual_norm: inplace needs dense rows that do not overlap")
        _check_apart(xr, rr, "x")
        if gate_rows:
            _check_apart(gate, rr, "the gate")
        elif gate is not None:
            _check_weight(gate, rr, "the gate")
        _check_weight(before, rr, "before")
        _check_weight(after, rr, "after")
        out = residual
    else:
        rr, rs = _rows(residual, H)
        out = h = torch.empty_like(residual, memory_format=torch.contiguous_format)
        hs = H
    y = scales = None
    if quant:
        y = torch.empty_like(x, dtype=FP8, memory_format=torch.contiguous_format)
        scales = x.new_empty((*shape[:-1], H // block_size), dtype=scale_dtype)
    elif before is not None:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if T:
        _lib.call_on(d, "sgl_residual_norm", xr.data_ptr(), dt, T, H, xs, rr.data_ptr(), rdt, rs,
                     _lib.ptr(after), adt, _lib.ptr(gate), gdt, gate_rows, gs, scale, _lib.ptr(before), bdt, eps,
                     h.data_ptr(), hs, _lib.ptr(y), quant, _lib.ptr(scales), block_size, mode,
                     quant and scale_dtype is E8M0)
    return out, (y, scales) if quant else y


def _meet(x: torch.Tensor, h: torch.Tensor) -> bool:
    """Whether rows ``x`` and ``h`` ``[T, H]``, each dense, share memory; also true of ranges that do where the
    strides differ."""
    if x.numel() == 0 or h.numel() == 0:
        return False
    m, n, size = x.shape[0], h.shape[0], x.element_size()
    xs, hs = x.stride(0) * size, h.stride(0) * h.element_size()  # (bytes from here on)
    wx, wh, far = x.shape[1] * size, h.shape[1] * h.element_size(), x.data_ptr() - h.data_ptr()
    if far + (m - 1) * xs + wx <= 0 or far >= (n - 1) * hs + wh:
        return False
    if m == 1 or xs == 0:
        m, xs = 1, hs
    if n == 1:
        hs = xs
    if xs != hs or xs == 0:
        return True
    # row i of x and row j of h meet where -wx < far + (i - j) xs < wh
    least, most = (-wx - far) // xs + 1, -((far - wh) // xs) - 1
    return max(least, 1 - n) <= min(most, m - 1)


def _check_apart(x: torch.Tensor, h: torch.Tensor, name: str) -> None:
    """Refuse an in-place residual that shares memory with ``x`` and is not its very rows."""
    if x.data_ptr() == h.data_ptr() and x.dtype is h.dtype and (x.shape[0] == 1 or x.stride(0) == h.stride(0)):
        return
    if _meet(x, h):
        raise ValueError(f"residual_norm: the residual written in place overlaps {name} without being it")


def _check_weight(w: Optional[torch.Tensor], h: torch.Tensor, name: str) -> None:
    """Refuse a weight that lies in the rows of an in-place residual: other rows still read it."""
    if w is not None and _meet(w.view(1, -1), h):
        raise ValueError(f"residual_norm: the residual written in place overlaps {name}")


__all__ = ["residual_norm"]
