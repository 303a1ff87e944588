"""An 8-bit paged KV cache of ordinary attention heads, and the attention over it.

The cache (:class:`PagedKV`) keeps keys and values as e4m3 codes ``[pages, Hkv,
page, D]`` with one fp32 scale for each block of tokens and head ``[pages, Hkv,
page / block]``: a stored value is code * scale (finite, not negative; tokens of a scale
that is not are NaN, and the attention takes values of one below 2^-100 as zero).  A
layer's step is

    q = rotary(q, table, positions)
    append_kv(cache, k, v, block_table, start, cu_tokens=cu, table=table)
    o = paged_attn(q, cache, block_table, start + new, cu_tokens=cu)

with the tokens of a batch's sequences one after the other, ``cu_tokens``
(int32 ``[B + 1]``, never falling) saying where each begins; without it every sequence has one
token (decode).  All lengths stay on the device, so a step can be captured into
a HIP graph and replayed with other lengths.
"""

from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from .rotary import DTYPES, check_apart, check_axes, check_table

FP8 = torch.float8_e4m3fn
MAX_DIM = 256


class PagedKV(NamedTuple):
    """The four tensors of a layer's cache: contiguous, on one device."""

    k: torch.Tensor        # float8_e4m3fn [pages, Hkv, page, D]
    v: torch.Tensor        # float8_e4m3fn [pages, Hkv, page, D]
    k_scale: torch.Tensor  # float32 [pages, Hkv, page / block]
    v_scale: torch.Tensor  # float32 [pages, Hkv, page / block]

    @staticmethod
    def empty(pages: int, heads: int, page: int, dim: int, *, block: int = 64,
              device="cuda") -> "PagedKV":
        """Uninitialised: what was never appended is never read."""
        _check_sizes(pages, heads, page, dim, block, "PagedKV.empty")
        k = torch.empty(pages, heads, page, dim, dtype=FP8, device=device)
        s = torch.empty(pages, heads, page // block, dtype=torch.float32, device=device)
        return PagedKV(k, torch.empty_like(k), s, torch.empty_like(s))


def _check_sizes(pages, heads, page, dim, block, what):
    if pages < 1 or heads < 1:
        raise ValueError(f"{what}: needs at least one page and head, got {pages} and {heads}")
    if dim % 16 or not 16 <= dim <= MAX_DIM:
        raise ValueError(f"{what}: head dim must be a multiple of 16 up to {MAX_DIM}, got {dim}")
    if not 16 <= page <= 1024 or page & (page - 1):
        raise ValueError(f"{what}: page must be a power of two from 16 to 1024, got {page}")
    if not 16 <= block <= min(page, 128) or block & (block - 1):
        raise ValueError(f"{what}: block must be a power of two from 16 to 128 and at most the page "
                         f"({page}), got {block}")


def _check_cache(cache: PagedKV, what: str):
    k, v, ks, vs = cache
    shape, scales = k.shape, ks.shape
    if len(shape) != 4 or k.dtype is not FP8 or v.dtype is not FP8 or v.shape != shape:
        raise ValueError(f"{what}: cache codes must be float8_e4m3fn [pages, Hkv, page, D], got "
                         f"{k.dtype} {tuple(shape)} and {v.dtype} {tuple(v.shape)}")
    pages, heads, page, dim = shape
    if len(scales) != 3 or vs.shape != scales or scales[0] != pages or scales[1] != heads or \
            ks.dtype is not torch.float32 or vs.dtype is not torch.float32 or scales[2] < 1 or \
            page % scales[2]:
        raise ValueError(f"{what}: cache scales must be float32 [{pages}, {heads}, page / block], got "
                         f"{ks.dtype} {tuple(scales)} and {vs.dtype} {tuple(vs.shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{what}: the cache's tensors must be contiguous")
    return pages, heads, page, dim, page // scales[2]


def _check_batch(rows: int, block_table: torch.Tensor, lens: torch.Tensor,
                 cu_tokens: Optional[torch.Tensor], name: str, what: str):
    shape = block_table.shape
    if len(shape) != 2 or block_table.dtype is not torch.int32 or not block_table.is_contiguous():
        raise ValueError(f"{what}: block_table must be a contiguous int32 [B, pages], got "
                         f"{block_table.dtype} {tuple(shape)}")
    B = shape[0]
    if lens.dtype is not torch.int32 or lens.shape != (B,) or not lens.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous int32 [{B}], got {lens.dtype} "
                         f"{tuple(lens.shape)}")
    if cu_tokens is None:
        if rows != B:
            raise ValueError(f"{what}: {rows} rows for {B} sequences of one token each; pass cu_tokens")
    elif cu_tokens.dtype is not torch.int32 or cu_tokens.shape != (B + 1,) or \
            not cu_tokens.is_contiguous():
        raise ValueError(f"{what}: cu_tokens must be a contiguous int32 [{B + 1}], got "
                         f"{cu_tokens.dtype} {tuple(cu_tokens.shape)}")
    return shape


def _rows16(x: torch.Tensor, n: int):
    """``x`` and its strides where its rows can be read 16 bytes (``n`` elements) at a
    time, else those of a copy."""
    s = x.stride()
    if s[2] == 1 and s[0] % n == 0 and s[1] % n == 0 and x.data_ptr() % 16 == 0:
        return x, s
    x = x.clone(memory_format=torch.contiguous_format)  # (a fresh buffer, which is aligned)
    return x, x.stride()


@functools.lru_cache(maxsize=1024)
def _workspace(device: int, name: str, *sizes: int) -> int:
    """Bytes for the attention of these sizes: a function of them and of the device's CUs."""
    with torch.cuda.device(device):
        return _lib.size_of(name, *sizes)


def append_kv(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
              start: torch.Tensor, *, cu_tokens: Optional[torch.Tensor] = None,
              table: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
              axes: Optional[torch.Tensor] = None, interleaved: bool = False, offset: int = 0) -> None:
    """Write ``k`` and ``v`` ``[T, Hkv, D]`` (bf16, f16 or f32) into the cache.

    Row ``i`` of sequence ``b`` becomes token ``start[b] + i`` (``start`` int32
    ``[B]``: the tokens it has), in page ``block_table[b, token // page]``.  With
    ``table`` the keys are rotated first, as :func:`rotary.rotary` does, by their
    token's place or by ``positions`` (int32 ``[T]``; with ``axes`` ``[axes, T]``).

    A block of tokens and head has one scale: the smallest power of two that
    brings the largest finite magnitude of its new values down to 448, and not
    below the one it had if it already holds tokens of the sequence, which are
    rounded again where it grew.  A NaN or an infinity is stored as NaN.  Rows
    behind the last sequence, tokens behind the block table, and table entries
    that are no page of the cache are skipped.  Every page that is written to
    must belong to one sequence of the call, at one place of its row; pages that are only read (the full
    pages of a common prefix) may be shared."""
    pages, heads, page, dim, block = _check_cache(cache, "append_kv")
    shape = k.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape:
        raise ValueError(f"append_kv: expected k and v [T, {heads}, {dim}], got {tuple(shape)} and "
                         f"{tuple(v.shape)}")
    dt = DTYPES.get(k.dtype)
    if dt is None or v.dtype is not k.dtype:
        raise TypeError(f"append_kv: k and v must be bfloat16, float16 or float32, got {k.dtype} and "
                        f"{v.dtype}")
    T = shape[0]
    B, columns = _check_batch(T, block_table, start, cu_tokens, "start", "append_kv")
    rot = n_positions = 0
    if table is not None:
        rot = check_table(table, offset, dim, "append_kv")
        n_positions = table.shape[0]
        if rot % 16 or offset % 8:
            raise ValueError(f"append_kv: rotated elements must be a multiple of 16 at an offset that is "
                             f"one of 8, got {rot} at {offset}")
        if axes is not None:
            if positions is None:
                raise ValueError("append_kv: axes without positions")
            n_axes = check_axes(axes, rot, positions, T, "append_kv")
            if n_positions * rot >= 1 << 32:
                raise ValueError(f"append_kv: a table of {n_positions} positions is too large for axes")
            if positions.dtype is not torch.int32 or not positions.is_contiguous():
                raise ValueError(f"append_kv: positions must be contiguous int32, got {positions.dtype}")
        elif positions is not None and (positions.dtype is not torch.int32 or positions.shape != (T,)
                                        or not positions.is_contiguous()):
            raise ValueError(f"append_kv: positions must be a contiguous int32 [{T}], got "
                             f"{positions.dtype} {tuple(positions.shape)}")
    elif positions is not None or axes is not None:
        raise ValueError("append_kv: positions without a rotary table")
    kc, vc, ks, vs = cache
    d = _lib.device_of("append_kv", k, v, block_table, start, cu_tokens, table, positions, axes, kc, vc, ks, vs)
    if T == 0 or B == 0:
        return
    n = 4 if dt == _lib.SGL_F32 else 8
    k, sk = _rows16(k, n)
    v, sv = _rows16(v, n)
    if axes is not None:
        _lib.call_on(d, "sgl_kv8_append_axes", k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], dt, T, B,
                     heads, dim, _lib.ptr(cu_tokens), start.data_ptr(), block_table.data_ptr(), columns, page,
                     block, pages, table.data_ptr(), n_positions, rot, offset, positions.data_ptr(), n_axes,
                     axes.data_ptr(), interleaved, kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr())
        return
    _lib.call_on(d, "sgl_kv8_append", k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], dt, T, B,
                 heads, dim, _lib.ptr(cu_tokens), start.data_ptr(), block_table.data_ptr(), columns,
                 page, block, pages, _lib.ptr(table), n_positions, rot, offset, _lib.ptr(positions),
                 interleaved, kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr())


def paged_attn(q: torch.Tensor, cache: PagedKV, block_table: torch.Tensor, lens: torch.Tensor, *,
               cu_tokens: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
               causal: bool = True, window: int = 0, first: int = 0,
               sink: Optional[torch.Tensor] = None, cu_groups: Optional[torch.Tensor] = None,
               shared: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q`` ``[T, Hq, D]`` (bf16 or f16) over the cache: ``[T, Hq, D]``.

    Sequence ``b`` has ``lens[b]`` keys (int32 ``[B]``), its ``n`` queries being
    the last ``n`` of them; query head ``h`` reads kv head ``h // (Hq / Hkv)``.
    ``causal``: a query sees the keys up to its own position, the last ``window``
    of them if that is not 0 and beside those the sequence's ``first`` tokens; otherwise all.  ``sink`` (float32 ``[Hq]``): a
    logit of each head that takes part in the softmax and has no value.
    ``softmax_scale``: ``D ** -0.5`` by default.  The weights that meet the values
    are rounded by at most 2^-11 of themselves, or 2^-35 of the row's largest (each
    times its value's scale).

    ``cu_groups`` (int32 ``[groups + 1]``, never falling) and ``shared`` (int32 ``[groups]``), without
    a window: sequences ``cu_groups[g]`` to ``cu_groups[g + 1]`` begin alike, the full pages
    among their first ``shared[g]`` tokens being the same in the block table row of each that has queries.  Those
    pages are read once for all of the group's queries, and the result is the same but for the order
    of its sums.  Sequences may stand outside of all groups.  It pays where many rows of few queries each
    share thousands of tokens (60 sequences of two on 8192: 70 us, 176 without), not on short prefixes of
    few sequences, nor for a few chunks of dozens of queries, whose tiles read the prefix once each anyway.

    A row that sees no key is zero;
    rows behind the last sequence are not written (of a new tensor: they hold
    anything).  ``out`` may be ``q`` itself, or share no memory with its rows."""
    pages, heads, page, dim, block = _check_cache(cache, "paged_attn")
    shape = q.shape
    if len(shape) != 3 or shape[2] != dim or shape[1] < 1 or shape[1] % heads:
        raise ValueError(f"paged_attn: expected q [T, Hq, {dim}] with Hq a multiple of {heads}, got "
                         f"{tuple(shape)}")
    dt = DTYPES.get(q.dtype)
    if dt is None or dt == _lib.SGL_F32:
        raise TypeError(f"paged_attn: q must be bfloat16 or float16, got {q.dtype}")
    T, hq, _ = shape
    B, columns = _check_batch(T, block_table, lens, cu_tokens, "lens", "paged_attn")
    if sink is not None and (sink.dtype is not torch.float32 or sink.shape != (hq,)
                             or not sink.is_contiguous()):
        raise ValueError(f"paged_attn: sink must be a contiguous float32 [{hq}], got {sink.dtype} "
                         f"{tuple(sink.shape)}")
    if window < 0 or (window and not causal):
        raise ValueError(f"paged_attn: window ({window}) must not be negative and is for causal attention")
    if first < 0 or (first and not window):
        raise ValueError(f"paged_attn: first ({first}) must not be negative and is for a window")
    groups = 0
    if cu_groups is not None or shared is not None:
        if cu_groups is None or shared is None or window:
            raise ValueError("paged_attn: cu_groups and shared go together, without a window")
        groups = shared.shape[0] if shared.dim() == 1 else 0
        if groups < 1 or shared.dtype is not torch.int32 or cu_groups.dtype is not torch.int32 or \
                cu_groups.shape != (groups + 1,) or not (shared.is_contiguous() and cu_groups.is_contiguous()):
            raise ValueError(f"paged_attn: cu_groups and shared must be contiguous int32 [groups + 1] and "
                             f"[groups], got {cu_groups.dtype} {tuple(cu_groups.shape)} and {shared.dtype} "
                             f"{tuple(shared.shape)}")
    kc, vc, ks, vs = cache
    d = _lib.device_of("paged_attn", q, block_table, lens, cu_tokens, sink, cu_groups, shared, out, kc, vc, ks, vs)
    given = out is not None
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not q.dtype or not out.is_contiguous():
        raise ValueError(f"paged_attn: out must be a contiguous {q.dtype} {tuple(shape)}, got "
                         f"{out.dtype} {tuple(out.shape)}")
    if T == 0 or B == 0:
        return out
    q, sq = _rows16(q, 8)
    if given and out is not q:
        check_apart(q, out, "paged_attn")
    scale = dim ** -0.5 if softmax_scale is None else softmax_scale
    G, tokens = hq // heads, columns * page
    window, first = min(window, tokens), min(first, tokens)  # (64 bits hold them then)
    if groups:
        nws = _workspace(d, "sgl_kv8_attn_shared_workspace_size", T, B, heads, G, dim, tokens, groups)
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device)
        _lib.call_on(d, "sgl_kv8_attn_shared", q.data_ptr(), sq[0], sq[1], dt, T, B, heads, G, dim,
                     _lib.ptr(cu_tokens), lens.data_ptr(), block_table.data_ptr(), columns, page, block, pages,
                     kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), scale, causal, _lib.ptr(sink),
                     groups, cu_groups.data_ptr(), shared.data_ptr(), out.data_ptr(), ws.data_ptr(), nws)
    elif first:
        nws = _workspace(d, "sgl_kv8_attn_first_workspace_size", T, B, heads, G, dim, tokens, window, first)
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
        _lib.call_on(d, "sgl_kv8_attn_first", q.data_ptr(), sq[0], sq[1], dt, T, B, heads, G, dim,
                     _lib.ptr(cu_tokens), lens.data_ptr(), block_table.data_ptr(), columns, page, block, pages,
                     kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), scale, causal, window, first,
                     _lib.ptr(sink), out.data_ptr(), _lib.ptr(ws), nws)
    else:
        nws = _workspace(d, "sgl_kv8_attn_workspace_size", T, B, heads, G, dim, tokens)
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
        _lib.call_on(d, "sgl_kv8_attn", q.data_ptr(), sq[0], sq[1], dt, T, B, heads, G, dim, _lib.ptr(cu_tokens),
                     lens.data_ptr(), block_table.data_ptr(), columns, page, block, pages, kc.data_ptr(),
                     vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), scale, causal, window, _lib.ptr(sink),
                     out.data_ptr(), _lib.ptr(ws), nws)
    return out


__all__ = ["PagedKV", "append_kv", "paged_attn"]
