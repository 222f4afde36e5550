"""Operators of generation and serving: rotary positions, a paged key/value
cache, and the attention that reads it.

* ``rotary(x, positions, inv_freq)`` -- rotary positions of one to four axes.
* ``paged_kv_append(k, v, k_cache, v_cache, block_table, kv_lens, ...)`` --
  rotates new keys (and queries) and stores keys and values in their pages.
* ``paged_attention(q, k_cache, v_cache, block_table, kv_lens, ...)`` -- a
  chunk of new tokens per sequence, or one, over the cache that holds them.

A cache is ``[pages, page_size, Hkv, D]`` (permuted views such as a
``[pages, Hkv, page_size, D]`` allocation's are taken as they are); key ``j`` of
sequence ``b`` is row ``j % page_size`` of page ``block_table[b, j // page_size]``.
New tokens of all sequences are packed along their first dimension:
``cu_seqlens [B + 1]`` holds the borders (without it every sequence has one),
``kv_lens [B]`` each sequence's length with its new tokens counted.  Lengths and
tables stay on the device, so a captured CUDA graph serves later steps whose
lengths and pages have changed in place.

One step of a layer::

    q = paged_kv_append(k, v, k_cache, v_cache, block_table, kv_lens,
                        cu_seqlens=cu, q=q, inv_freq=inv_freq)
    o = paged_attention(q, k_cache, v_cache, block_table, kv_lens,
                        cu_seqlens=cu, max_q_len=longest)

Errors are those of ``operators``: ``TypeError``/``ValueError`` for what Python
sees, ``FaError`` for what the C ABI rejects.  What only the device sees -- a page
outside the cache, a length behind its table -- is skipped there and reported by
``device_status()``.
"""

from __future__ import annotations

import math
import struct

import torch

from . import _lib
from .operators import _HALF_TYPES, _on_device, _stream_ptr

_DTYPES = {torch.bfloat16: _lib.FA_BF16, torch.float16: _lib.FA_F16, torch.float32: _lib.FA_F32}
_INTS = (torch.int32, torch.int64)
_FLOATS = (torch.float32, torch.float64)

# The argument structs of include/fa_b200.h: pointers, then 64-bit integers.
_ROTARY = struct.Struct("=4Q24q")
_APPEND = struct.Struct("=11Q35q")
_ATTN = struct.Struct("=7Q22qd")


def _check(name: str, t, dtypes, dims) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in dtypes:
        names = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        raise TypeError(f"{name} must be {names} (got {t.dtype})")
    if t.dim() not in dims:
        want = " or ".join(f"{d}-D" for d in dims)
        raise ValueError(f"{name} must be {want} (got {tuple(t.shape)})")


def _check_rows(name: str, t, dtypes, dims) -> None:
    _check(name, t, dtypes, dims)
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")


def _check_list(name: str, t, size: int) -> None:
    _check(name, t, (torch.int32,), (1,))
    if t.shape[0] != size or (t.stride(0) != 1 and size > 1):
        raise ValueError(f"{name} must be a contiguous [{size}] tensor (got {tuple(t.shape)})")


def _check_devices(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (got device {t.device})")
        if t.device != device:
            raise ValueError(f"{name} must be on {device} like the others (got {t.device})")


def _sections(sections, planes: int):
    """Axis count and the four section ends of the C ABI."""
    if sections is None:
        return 1, (planes, 0, 0, 0)
    ends, total = [], 0
    for s in sections:
        if isinstance(s, bool) or not isinstance(s, int) or s <= 0:
            raise ValueError(f"sections must be positive whole numbers (got {tuple(sections)})")
        total += s
        ends.append(total)
    if not 1 <= len(ends) <= 4 or total != planes:
        raise ValueError(f"sections must be 1 to 4 numbers that add up to {planes}, the number of "
                         f"frequencies (got {tuple(sections)})")
    return len(ends), tuple(ends + [0] * (4 - len(ends)))


def _check_inv_freq(inv_freq) -> int:
    """Number of rotated channels."""
    _check("inv_freq", inv_freq, _FLOATS, (1,))
    if not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous")
    return 2 * inv_freq.shape[0]


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
           sections=None, interleaved: bool = False, inverse: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions on ``x [B, H, S, D]`` or packed tokens ``x [T, H, D]``
    (bf16, fp16 or fp32; any strides of 16-byte multiples, D contiguous).

    The first ``R = 2 * len(inv_freq)`` channels (a multiple of 16, at most D)
    are rotated, plane ``i`` by ``position * inv_freq[i]``: channels ``(i, i +
    R/2)``, or ``(2i, 2i + 1)`` with ``interleaved``.  The others are copied.
    ``positions`` (int32 or int64) is ``[S]`` or ``[B, S]``, ``[T]`` for packed
    tokens; with ``sections``, the number of frequencies of each of up to four
    axes (time, height, width), it has a leading axis dimension.  ``inv_freq``
    is fp32 or fp64; angles are formed in fp64, so far positions stay exact.
    ``inverse`` rotates back, which is also the operator's gradient.  ``out``
    may be ``x``.
    """
    _check_rows("x", x, tuple(_DTYPES), (3, 4))
    R = _check_inv_freq(inv_freq)
    axes, ends = _sections(sections, R // 2)
    if x.dim() == 4:
        B, H, S, D = x.shape
        xs = x.stride()[:3]
        row_dims = (1, 2)
    else:
        S, H, D = x.shape
        B, xs, row_dims = 1, (0, x.stride(1), x.stride(0)), (1,)
    lead = 0 if sections is None else 1
    _check("positions", positions, _INTS, tuple(d + lead for d in row_dims))
    shape, st = tuple(positions.shape), positions.stride()
    if (lead and shape[0] != axes) or shape[-1] != S or \
            (len(shape) - lead == 2 and shape[-2] != B):
        raise ValueError(f"positions {shape} do not match x {tuple(x.shape)}"
                         + (f" and {axes} axes" if lead else ""))
    ps = (st[0] if lead else 0, st[-2] if len(shape) - lead == 2 else 0, st[-1])
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _check_rows("out", out, (x.dtype,), (x.dim(),))
        if out.shape != x.shape:
            raise ValueError("out must have x's shape")
    os = out.stride()[:3] if x.dim() == 4 else (0, out.stride(1), out.stride(0))
    _check_devices(x.device, x=x, positions=positions, inv_freq=inv_freq, out=out)
    if B * H * S == 0:
        return out
    lib = _lib.load()
    args = _ROTARY.pack(x.data_ptr(), out.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
                        _DTYPES[x.dtype], B, H, S, D, R, *xs, *os, axes, *ends, *ps,
                        positions.dtype == torch.int64, inv_freq.dtype == torch.float64,
                        bool(interleaved), bool(inverse))
    with _on_device(x.device):
        rc = lib.fa_rotary(args, _stream_ptr(x.device))
    _lib.check(rc, "fa_rotary")
    return out


def _check_paged(T: int, dtype, D: int, k_cache, v_cache, block_table, kv_lens,
                 cu_seqlens) -> None:
    _check_rows("k_cache", k_cache, (dtype,), (4,))
    _check_rows("v_cache", v_cache, (dtype,), (4,))
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != D:
        raise ValueError(f"caches must both be [pages, page_size, Hkv, {D}] (got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)})")
    _check("block_table", block_table, (torch.int32,), (2,))
    B = block_table.shape[0]
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise ValueError("block_table must be contiguous along its last dimension")
    _check_list("kv_lens", kv_lens, B)
    if cu_seqlens is not None:
        _check_list("cu_seqlens", cu_seqlens, B + 1)
    elif T != B:
        raise ValueError(f"without cu_seqlens every sequence has one new token: {T} tokens, "
                         f"{B} sequences")


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                    v_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_seqlens: torch.Tensor | None = None, q: torch.Tensor | None = None,
                    inv_freq: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, sections=None,
                    interleaved: bool = False,
                    q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores the new tokens' ``k``, ``v [T, Hkv, D]`` (bf16 or fp16) in their
    pages, in place, and returns the queries rotated alike, if any were given.

    ``k_cache``, ``v_cache`` ``[pages, page_size, Hkv, D]`` (page_size a power of
    two, 16 to 1024), ``block_table [B, max_pages]``, ``kv_lens [B]`` and
    ``cu_seqlens [B + 1]`` are int32 and as the module describes.  With
    ``inv_freq`` keys and ``q [T, Hq, D]`` are rotated as by ``rotary``, by the
    token's place in its sequence or by ``positions`` (``[T]``; ``[axes, T]`` with
    ``sections``).  ``q_out`` may be ``q``.

    Rows of no sequence are neither read nor written, in ``q_out`` too.  Tokens
    before their sequence's start (``kv_lens`` below the number of new tokens, as
    in padding sequences of length 0) are not stored.  A place outside the
    table or the cache is skipped, and ``device_status()`` reports it.
    """
    _check_rows("k", k, _HALF_TYPES, (3,))
    _check_rows("v", v, (k.dtype,), (3,))
    if k.shape != v.shape:
        raise ValueError(f"k and v shapes differ: {tuple(k.shape)}, {tuple(v.shape)}")
    T, Hkv, D = k.shape
    _check_paged(T, k.dtype, D, k_cache, v_cache, block_table, kv_lens, cu_seqlens)
    if k_cache.shape[2] != Hkv:
        raise ValueError(f"the caches have {k_cache.shape[2]} heads, k has {Hkv}")
    Hq, qs, qos = 0, (0, 0), (0, 0)
    if q is not None:
        _check_rows("q", q, (k.dtype,), (3,))
        if q.shape[0] != T or q.shape[2] != D:
            raise ValueError(f"q must be [{T}, Hq, {D}] (got {tuple(q.shape)})")
        Hq, qs = q.shape[1], q.stride()[:2]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _check_rows("q_out", q_out, (q.dtype,), (3,))
            if q_out.shape != q.shape:
                raise ValueError("q_out must have q's shape")
        qos = q_out.stride()[:2]
    elif q_out is not None:
        raise ValueError("q_out needs q")
    R, axes, ends, ps = 0, 1, (0, 0, 0, 0), (0, 0)
    if inv_freq is not None:
        R = _check_inv_freq(inv_freq)
        axes, ends = _sections(sections, R // 2)
        if positions is not None:
            lead = 0 if sections is None else 1
            _check("positions", positions, _INTS, (1 + lead,))
            want = (axes, T) if lead else (T,)
            if tuple(positions.shape) != want:
                raise ValueError(f"positions must be {list(want)} (got {tuple(positions.shape)})")
            ps = (positions.stride(0) if lead else 0, positions.stride(-1))
        elif axes > 1:
            raise ValueError("several axes need positions")
    elif positions is not None or sections is not None:
        raise ValueError("positions and sections need inv_freq")
    _check_devices(k.device, k=k, v=v, k_cache=k_cache, v_cache=v_cache,
                   block_table=block_table, kv_lens=kv_lens, cu_seqlens=cu_seqlens, q=q,
                   q_out=q_out, positions=positions, inv_freq=inv_freq)
    if T * Hkv == 0:
        return q_out
    lib = _lib.load()
    args = _APPEND.pack(
        k.data_ptr(), v.data_ptr(), 0 if Hq == 0 else q.data_ptr(),
        0 if Hq == 0 else q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        block_table.data_ptr(), kv_lens.data_ptr(),
        0 if cu_seqlens is None else cu_seqlens.data_ptr(),
        0 if positions is None else positions.data_ptr(),
        0 if inv_freq is None else inv_freq.data_ptr(),
        _DTYPES[k.dtype], T, block_table.shape[0], Hq, Hkv, D, R, k_cache.shape[0],
        k_cache.shape[1], block_table.shape[1], block_table.stride(0), *k.stride()[:2],
        *v.stride()[:2], *qs, *qos, *k_cache.stride()[:3], *v_cache.stride()[:3], axes, *ends,
        *ps, positions is not None and positions.dtype == torch.int64,
        inv_freq is not None and inv_freq.dtype == torch.float64, bool(interleaved))
    with _on_device(k.device):
        rc = lib.fa_paged_append(args, _stream_ptr(k.device))
    _lib.check(rc, "fa_paged_append")
    return q_out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_seqlens: torch.Tensor | None = None, max_q_len: int | None = None,
                    causal: bool = True, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(q K^T * scale) V`` of the new tokens ``q [T, Hq, D]`` (bf16 or
    fp16, D 8 .. 128 in steps of 8) over the paged cache that holds them.

    Caches, table and lengths as in ``paged_kv_append``; query head ``i`` reads
    key head ``i // (Hq // Hkv)``.  With ``causal`` a token sees the keys up to
    its own place in the sequence, else all ``kv_lens[b]``; one that sees none
    gets zeros.  ``scale`` defaults to ``1/sqrt(D)``.  ``max_q_len``, the longest
    sequence's number of new tokens, lets the call choose its kernels (default:
    one without ``cu_seqlens``, else unknown); it never changes what is computed.
    Rows of no sequence are left as they were in ``out``.  Cached values that a
    sequence's tokens see must be finite; rows behind ``kv_lens`` may hold
    anything.
    """
    _check_rows("q", q, _HALF_TYPES, (3,))
    T, Hq, D = q.shape
    _check_paged(T, q.dtype, D, k_cache, v_cache, block_table, kv_lens, cu_seqlens)
    Hkv = k_cache.shape[2]
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads cannot share {Hkv} key heads evenly")
    if max_q_len is None:
        max_q_len = 1 if cu_seqlens is None else T
    elif max_q_len < 0:
        raise ValueError("max_q_len must not be negative")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    else:
        _check_rows("out", out, (q.dtype,), (3,))
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
    _check_devices(q.device, q=q, k_cache=k_cache, v_cache=v_cache, block_table=block_table,
                   kv_lens=kv_lens, cu_seqlens=cu_seqlens, out=out)
    if T * Hq == 0:
        return out
    lib = _lib.load()
    args = _ATTN.pack(
        q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        block_table.data_ptr(), kv_lens.data_ptr(),
        0 if cu_seqlens is None else cu_seqlens.data_ptr(), _DTYPES[q.dtype], T,
        block_table.shape[0], Hq, Hkv, D, k_cache.shape[0], k_cache.shape[1],
        block_table.shape[1], block_table.stride(0), *q.stride()[:2], *out.stride()[:2],
        *k_cache.stride()[:3], *v_cache.stride()[:3], max(1, int(max_q_len)), bool(causal),
        1.0 / math.sqrt(D) if scale is None else float(scale))
    with _on_device(q.device):
        # The workspace is this call's own: on one stream the allocator hands it
        # out again in order, and a captured graph keeps its own.
        size = lib.fa_paged_attn_workspace(args)
        if size < 0:
            _lib.check(-size, "fa_paged_attn")
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        rc = lib.fa_paged_attn(args, ws.data_ptr(), size, _stream_ptr(q.device))
    _lib.check(rc, "fa_paged_attn")
    return out
