"""An 8-bit paged KV cache of ordinary attention heads, and the attention over it.

The cache (:class:`PagedKV`) keeps keys and values as e4m3 codes ``[pages, Hkv,
page, D]`` with one fp32 scale for each block of tokens and head ``[pages, Hkv,
page / block]``.  A layer's step is

    q = rotary(q, table, positions)
    append_kv(cache, k, v, block_table, start, cu_tokens=cu, table=table)
    o = paged_attn(q, cache, block_table, start + new, cu_tokens=cu)

with the tokens of a batch's sequences one after the other, ``cu_tokens``
(int32 ``[B + 1]``) saying where each begins; without it every sequence has one
token (decode).  All lengths stay on the device, so a step can be captured into
a HIP graph and replayed with other lengths.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .rotary import DTYPES, check_table

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
    if k.dim() != 4 or k.dtype != FP8 or v.dtype != FP8 or v.shape != k.shape:
        raise ValueError(f"{what}: cache codes must be float8_e4m3fn [pages, Hkv, page, D], got "
                         f"{k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    pages, heads, page, dim = k.shape
    if ks.dim() != 3 or ks.shape != vs.shape or ks.shape[0] != pages or ks.shape[1] != heads or \
            ks.dtype != torch.float32 or vs.dtype != torch.float32 or ks.shape[2] < 1 or \
            page % ks.shape[2]:
        raise ValueError(f"{what}: cache scales must be float32 [{pages}, {heads}, page / block], got "
                         f"{ks.dtype} {tuple(ks.shape)} and {vs.dtype} {tuple(vs.shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{what}: the cache's tensors must be contiguous")
    return pages, heads, page, dim, page // ks.shape[2]


def _check_batch(rows: int, block_table: torch.Tensor, lens: torch.Tensor,
                 cu_tokens: Optional[torch.Tensor], name: str, what: str) -> int:
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or not block_table.is_contiguous():
        raise ValueError(f"{what}: block_table must be a contiguous int32 [B, pages], got "
                         f"{block_table.dtype} {tuple(block_table.shape)}")
    B = block_table.shape[0]
    if lens.dtype != torch.int32 or lens.shape != (B,) or not lens.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous int32 [{B}], got {lens.dtype} "
                         f"{tuple(lens.shape)}")
    if cu_tokens is None:
        if rows != B:
            raise ValueError(f"{what}: {rows} rows for {B} sequences of one token each; pass cu_tokens")
    elif cu_tokens.dtype != torch.int32 or cu_tokens.shape != (B + 1,) or \
            not cu_tokens.is_contiguous():
        raise ValueError(f"{what}: cu_tokens must be a contiguous int32 [{B + 1}], got "
                         f"{cu_tokens.dtype} {tuple(cu_tokens.shape)}")
    return B


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself where its rows can be read 16 bytes at a time, else a copy."""
    n = 16 // x.element_size()
    if x.stride(2) == 1 and x.stride(0) % n == 0 and x.stride(1) % n == 0 and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)  # (a fresh buffer, which is aligned)


def append_kv(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
              start: torch.Tensor, *, cu_tokens: Optional[torch.Tensor] = None,
              table: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
              interleaved: bool = False, offset: int = 0) -> None:
    """Write ``k`` and ``v`` ``[T, Hkv, D]`` (bf16, f16 or f32) into the cache.

    Row ``i`` of sequence ``b`` becomes token ``start[b] + i`` (``start`` int32
    ``[B]``: the tokens it has), in page ``block_table[b, token // page]``.  With
    ``table`` the keys are rotated first, as :func:`rotary.rotary` does, by their
    token's place or by ``positions`` (int32 ``[T]``).

    A block of tokens and head has one scale: the smallest power of two that
    brings the largest finite magnitude of its new values down to 448, and not
    below the one it had if it already holds tokens of the sequence, which are
    rounded again where it grew.  A NaN or an infinity is stored as NaN.  Rows
    behind the last sequence, tokens behind the block table, and table entries
    that are no page of the cache are skipped.  Every page that is written to
    must belong to one sequence of the call; pages that are only read (the full
    pages of a common prefix) may be shared."""
    pages, heads, page, dim, block = _check_cache(cache, "append_kv")
    if k.dim() != 3 or k.shape[1] != heads or k.shape[2] != dim or v.shape != k.shape:
        raise ValueError(f"append_kv: expected k and v [T, {heads}, {dim}], got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    dt = DTYPES.get(k.dtype)
    if dt is None or v.dtype != k.dtype:
        raise TypeError(f"append_kv: k and v must be bfloat16, float16 or float32, got {k.dtype} and "
                        f"{v.dtype}")
    T = k.shape[0]
    B = _check_batch(T, block_table, start, cu_tokens, "start", "append_kv")
    rot = n_positions = 0
    if table is not None:
        rot = check_table(table, offset, dim, "append_kv")
        n_positions = table.shape[0]
        if rot % 16 or offset % 8:
            raise ValueError(f"append_kv: rotated elements must be a multiple of 16 at an offset that is "
                             f"one of 8, got {rot} at {offset}")
        if positions is not None and (positions.dtype != torch.int32 or positions.shape != (T,)
                                      or not positions.is_contiguous()):
            raise ValueError(f"append_kv: positions must be a contiguous int32 [{T}], got "
                             f"{positions.dtype} {tuple(positions.shape)}")
    elif positions is not None:
        raise ValueError("append_kv: positions without a rotary table")
    _lib.require_device(k, v, block_table, start, cu_tokens, table, positions, *cache,
                        what="append_kv")
    _lib.require_same_device(k, v, block_table, start, cu_tokens, table, positions, *cache,
                             what="append_kv")
    if T == 0 or B == 0:
        return
    k, v = _rows16(k), _rows16(v)
    with _lib.on_device(k):
        _lib.call("sgl_kv8_append", k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                  v.stride(1), dt, T, B, heads, dim, _lib.ptr(cu_tokens), start.data_ptr(),
                  block_table.data_ptr(), block_table.shape[1], page, block, pages, _lib.ptr(table),
                  n_positions, rot, offset, _lib.ptr(positions), interleaved, cache.k.data_ptr(),
                  cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                  _lib.stream_of(k))


def paged_attn(q: torch.Tensor, cache: PagedKV, block_table: torch.Tensor, lens: torch.Tensor, *,
               cu_tokens: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
               causal: bool = True, window: int = 0, sink: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q`` ``[T, Hq, D]`` (bf16 or f16) over the cache: ``[T, Hq, D]``.

    Sequence ``b`` has ``lens[b]`` keys (int32 ``[B]``), its ``n`` queries being
    the last ``n`` of them; query head ``h`` reads kv head ``h // (Hq / Hkv)``.
    ``causal``: a query sees the keys up to its own position, the last ``window``
    of them if that is not 0; otherwise all.  ``sink`` (float32 ``[Hq]``): a
    logit of each head that takes part in the softmax and has no value.
    ``softmax_scale``: ``D ** -0.5`` by default.  A row that sees no key is zero;
    rows of ``out`` behind the last sequence are left as they are."""
    pages, heads, page, dim, block = _check_cache(cache, "paged_attn")
    if q.dim() != 3 or q.shape[2] != dim or q.shape[1] < 1 or q.shape[1] % heads:
        raise ValueError(f"paged_attn: expected q [T, Hq, {dim}] with Hq a multiple of {heads}, got "
                         f"{tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"paged_attn: q must be bfloat16 or float16, got {q.dtype}")
    T, hq, _ = q.shape
    B = _check_batch(T, block_table, lens, cu_tokens, "lens", "paged_attn")
    if sink is not None and (sink.dtype != torch.float32 or sink.shape != (hq,)
                             or not sink.is_contiguous()):
        raise ValueError(f"paged_attn: sink must be a contiguous float32 [{hq}], got {sink.dtype} "
                         f"{tuple(sink.shape)}")
    if window < 0 or (window and not causal):
        raise ValueError(f"paged_attn: window ({window}) must not be negative and is for causal attention")
    _lib.require_device(q, block_table, lens, cu_tokens, sink, out, *cache, what="paged_attn")
    _lib.require_same_device(q, block_table, lens, cu_tokens, sink, out, *cache, what="paged_attn")
    if out is None:
        out = torch.empty((T, hq, dim), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"paged_attn: out must be a contiguous {q.dtype} {tuple(q.shape)}, got "
                         f"{out.dtype} {tuple(out.shape)}")
    if T == 0 or B == 0:
        return out
    q = _rows16(q)
    with _lib.on_device(q):
        nws = _lib.size_of("sgl_kv8_attn_workspace_size", T, B, heads, hq // heads, dim)
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device)
        _lib.call("sgl_kv8_attn", q.data_ptr(), q.stride(0), q.stride(1), DTYPES[q.dtype], T, B, heads,
                  hq // heads, dim, _lib.ptr(cu_tokens), lens.data_ptr(), block_table.data_ptr(),
                  block_table.shape[1], page, block, pages, cache.k.data_ptr(), cache.v.data_ptr(),
                  cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                  dim ** -0.5 if softmax_scale is None else float(softmax_scale), causal, int(window),
                  _lib.ptr(sink), out.data_ptr(), ws.data_ptr(), nws, _lib.stream_of(q))
    return out


__all__ = ["PagedKV", "append_kv", "paged_attn"]
