"""Serving: a paged key/value cache, attention over it, and sampling.

What the decoder needs to continue a prompt, most of all to draw many samples
of one prompt: the prompt's keys and values are kept once and read once for the
whole batch. The reference trains only and has no counterpart.

A cache is a pair of tensors ``[pages, kv_heads, page_size, head_dim]`` (any
strides whose last one is 1, e.g. one layer of ``[layers, 2, pages, ...]``).
*Slot* ``s`` is row ``s % page_size`` of page ``s // page_size``. The functions
run on the caller's current stream, allocate with torch's caching allocator and
do not synchronise; lengths, page numbers, slots and positions are read on the
device, so a captured CUDA graph replays with new ones. An index outside its
buffer is not followed and sets bit 4 of ``_native.device_error()``; each
function says what stands in for it. None of the three has a backward.

* :func:`append_kv` -- rotate the new queries and keys, write the new keys and
  values to their slots (``sy_append_kv``);
* :func:`attend_paged` -- attention over the shared prefix and each sequence's
  own pages (``sy_attend``);
* :func:`sample_tokens` -- the next token of every row (``sy_sample``).
"""

from __future__ import annotations

import torch

from . import _sy_torch

__all__ = ["append_kv", "attend_paged", "sample_tokens"]


def append_kv(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    q: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Rotate ``q`` and ``k`` by their positions and write ``k`` and ``v`` into
    the caches, in one launch. Returns the rotated ``q`` (``None`` without it).

    ``k``, ``v`` ``[tokens, kv_heads, head_dim]`` and ``q`` ``[tokens, q_heads,
    head_dim]`` have the caches' dtype (bf16, fp16 or fp32) and may be strided
    views, e.g. the three parts of one projection. ``slots`` (int64
    ``[tokens]``) says where each token goes; a negative slot writes nothing
    (padding; its ``q`` is still rotated), and no two tokens may share one.
    ``positions`` (int32 ``[tokens]``) are rows of ``cos`` and ``sin`` (fp32
    ``[length, r]``, :func:`switchyard.decoder.rope_tables`): columns ``i`` and
    ``i + r`` of a head, ``i < r``, turn against each other, the columns from
    ``2 r`` on are kept. Without the three nothing is rotated. A token whose
    slot or position lies outside writes nothing to the caches; its rotated
    ``q`` is zero if the position does, and as ever if only the slot does.
    """
    return _sy_torch.append_kv(k, v, k_cache, v_cache, slots, q, positions, cos, sin)


def attend_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    kv_lens: torch.Tensor,
    prefix_pages: torch.Tensor | None = None,
    prefix_len: int = 0,
    scale: float | None = None,
    return_lse: bool = False,
):
    """Attention of every sequence's last ``q_len`` tokens over a prefix that
    the batch shares and over the sequence's own keys.

    ``q`` ``[batch, q_len, q_heads, head_dim]`` (bf16 or fp16; rotated);
    query head ``h`` reads key head ``h // (q_heads // kv_heads)``. Sequence
    ``b`` owns the first ``kv_lens[b]`` keys (int32, the ``q_len`` new ones
    among them) of the pages ``page_table[b]`` (int32 ``[batch, width]``;
    entries past its length are not read) and sees, after them in nothing but
    order, the first ``prefix_len`` keys of ``prefix_pages`` (int32). Query
    ``t`` sees the whole prefix and own keys ``j < kv_lens[b] - q_len + t + 1``.
    One token a sequence (``q_len = 1``) is decoding; ``batch = 1`` with
    ``q_len = kv_lens`` reads a prompt.

    Returns ``out`` like ``q``, or ``(out, lse)`` with the fp32 ``[batch,
    q_len, q_heads]`` logarithm of the softmax's denominator. A query that sees
    no key gets 0 and ``-inf``. What a page holds past its sequence's length
    does not matter, NaN included; keys and values that some query of the call
    sees must be finite. A page outside the cache counts as keys and values of
    zero, a length outside ``[0, width * page_size]`` as the nearer end; both
    set the error bit, and the result is not to be used. ``head_dim`` is a multiple of 8 up to 128, ``page_size``
    a multiple of 8. ``scale`` is positive and defaults to ``head_dim ** -0.5``.
    """
    out, lse = _sy_torch.attend_paged(q, k_cache, v_cache, page_table, kv_lens, prefix_pages,
                                      prefix_len, scale, return_lse)
    return (out, lse) if return_lse else out


def sample_tokens(
    logits: torch.Tensor,
    u: torch.Tensor,
    temperature: torch.Tensor | float | None = None,
    top_k: torch.Tensor | int | None = None,
    top_p: torch.Tensor | float | None = None,
    min_p: torch.Tensor | float | None = None,
    return_logprob: bool = False,
):
    """Draw one token a row of ``logits`` ``[rows, vocab]`` (bf16, fp16 or
    fp32) with the given random numbers ``u`` (fp32 ``[rows]`` in [0, 1)).

    The parameters are one number for all rows or a tensor ``[rows]`` (fp32;
    ``top_k`` int32). ``x = logit * (1 / temperature)``; tokens are ranked by
    ``x``, ties by index, and kept if they are among the first ``top_k`` (<= 0:
    all), if the weight of those before them is below ``top_p`` of what
    ``top_k`` left (>= 1: all; the first is always kept) and if their
    probability is at least ``min_p`` times the highest. The token is the first
    in index order at which the kept weights' running total exceeds ``u`` of
    their sum. ``temperature <= 0`` takes the highest logit. Weights are whole
    numbers, ``exp(x - max)`` in units of 2^-40, so the result does not depend
    on any order of summation and repeats bit for bit. NaN counts as ``-inf``;
    a row with no ``x`` above ``-inf`` gives token -1 (so does one whose products
    all overflow, e.g. the type's lowest value at a temperature below 1).

    Returns int64 tokens ``[rows]``, or ``(tokens, logprob)`` with the fp32
    logarithm of the token's share of the kept weight.
    """
    rows = logits.shape[0] if logits.ndim else 0

    def per_row(x, dtype):
        if x is None or isinstance(x, torch.Tensor):
            return x
        return torch.full((rows,), x, dtype=dtype, device=logits.device)

    token, logprob = _sy_torch.sample_tokens(
        logits, u, per_row(temperature, torch.float32), per_row(top_k, torch.int32),
        per_row(top_p, torch.float32), per_row(min_p, torch.float32), return_logprob)
    return (token, logprob) if return_logprob else token
