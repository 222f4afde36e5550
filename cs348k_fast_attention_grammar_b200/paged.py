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
``cu_seqlens [B + 1]`` holds the borders (without it every sequence has one; those
outside the rows are held to them),
``kv_lens [B]`` each sequence's length with its new tokens counted.  Lengths and
tables stay on the device, so a captured CUDA graph serves later steps whose
lengths and pages have changed in place.

One step of a layer::

    q = paged_kv_append(k, v, k_cache, v_cache, block_table, kv_lens,
                        cu_seqlens=cu, q=q, inv_freq=inv_freq)
    o = paged_attention(q, k_cache, v_cache, block_table, kv_lens,
                        cu_seqlens=cu, max_q_len=longest)

Forward only, like ``operators``: no gradient is recorded.  What a call writes must
not overlap itself or what it reads, but for ``out`` and ``q_out`` as documented.

Errors are those of ``operators``: ``TypeError``/``ValueError`` for what Python
sees, ``FaError`` for what the C ABI rejects.  What only the device sees -- a page
outside the cache, a length beyond its table -- is never written or read outside;
the operators say what they do instead, and ``device_status()`` reports it.
"""

from __future__ import annotations

import torch

from . import _lib

_binding = None


def _native():
    """The binding that checks arguments, allocates outputs and calls the C ABI."""
    global _binding
    if _binding is None:
        _binding = _lib.load_binding()
    return _binding


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
    return (_binding or _native()).rotary(x, positions, inv_freq, sections, interleaved, inverse,
                                          out)


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

    Rows of no sequence have no effect, and ``q_out`` is left as it was there.  Tokens
    before their sequence's start (``kv_lens`` below the number of new tokens, as
    in padding sequences of length 0) are not stored.  A place outside the
    table or the cache is skipped, and ``device_status()`` reports it.
    """
    return (_binding or _native()).paged_kv_append(
        k, v, k_cache, v_cache, block_table, kv_lens, cu_seqlens, q, inv_freq, positions, sections,
        interleaved, q_out)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_seqlens: torch.Tensor | None = None, max_q_len: int | None = None,
                    causal: bool = True, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(q K^T * scale) V`` of the new tokens ``q [T, Hq, D]`` (bf16 or
    fp16, D 8 .. 128 in steps of 8) over the paged cache that holds them.

    Caches, table and lengths as in ``paged_kv_append``; query head ``i`` reads
    key head ``i // (Hq // Hkv)``.  With ``causal`` a token sees the keys up to
    its own place in the sequence, else all ``kv_lens[b]``; one that sees none,
    or none with a score above -infinity, gets zeros.  A score of +infinity or NaN
    makes its token's output NaN.  ``scale`` defaults to ``1/sqrt(D)``.  ``max_q_len``, the longest
    sequence's number of new tokens, lets the call choose its kernels (default:
    one without ``cu_seqlens``, else unknown); it never changes what is computed.
    Rows of no sequence are left as they were in ``out``.  Cached values that a
    sequence's tokens see must be finite; rows behind ``kv_lens`` may hold
    anything.  A page outside the cache reads as keys and values of zero, with
    their share of the weights; where a length goes beyond the table, tokens keep
    their places and see the keys that the table holds (``device_status()``
    reports both).
    """
    return (_binding or _native()).paged_attention(
        q, k_cache, v_cache, block_table, kv_lens, cu_seqlens, max_q_len, causal, scale, out)
