"""Operators of the attention layers that a striped stack keeps between its Hyena layers.

``qk_norm_rotary`` turns queries and keys by their positions, optionally behind an RMS norm of each head, differentiable;
``rotary_append`` does it for new tokens and stores their keys and values in the pages of a cache;
``paged_decode_attention`` attends from one new token of every sequence to that cache; ``copy_pages`` moves pages where a
sequence is forked or the cache compacted.  ``vortex_b200.cache.PagedKVCache`` keeps the pages and tables,
``vortex_b200.engine.AttentionInferenceEngine`` strings the calls together for a layer.  The reference does the same with
``vortex/ops/embedding/rotary.py:12`` and ``vortex/ops/attn_interface.py:1488`` on a contiguous cache
(``vortex/model/attention.py:352-381``).

Tensors are CUDA tensors of float32, bfloat16 or float16 with unit stride over a head's values; other strides are free.
"""
from __future__ import annotations

import math

import torch

from . import ops


def rotary_inv_freq(dim, base=10000.0, *, scaling=None, factor=1.0, trained_length=None, slow=1.0, fast=32.0, device=None):
    """Frequencies of the ``dim / 2`` pairs of a head, float64 [dim / 2], and the factor that the rotated values take
    (``scale`` of the other functions; 1.0 but for "yarn").

    ``scaling`` stretches a model to contexts ``factor`` times as long:

    * None: ``f_i = base^(-2i/dim)``;
    * "linear": ``f_i / factor``, i.e. positions interpolated (the reference's ``rotary_emb_scaling_factor``);
    * "ntk": ``base`` multiplied by ``factor^(dim / (dim - 2))``: the slowest pair is interpolated, the fastest kept;
    * "yarn": pairs that turn fewer than ``slow`` times over ``trained_length`` tokens are interpolated, those that turn more
      than ``fast`` times kept, the others mixed linearly in the number of turns; values take ``0.1 ln(factor) + 1``
      (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models", 2023)."""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and positive, got {dim}")
    if factor <= 0 or base <= 0:
        raise ValueError("base and factor must be positive")
    even = torch.arange(0, dim, 2, dtype=torch.float64)
    scale = 1.0
    if scaling == "ntk":
        if dim == 2:
            raise ValueError('"ntk" needs more than one pair')
        base = base * factor ** (dim / (dim - 2))
    freq = float(base) ** (-even / dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if not trained_length or fast <= slow:
            raise ValueError('"yarn" needs trained_length and slow < fast')
        kept = ((trained_length * freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        freq = freq / factor * (1 - kept) + freq * kept
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise NotImplementedError(f"unknown scaling {scaling!r}")
    return freq.to(device) if device is not None else freq, scale


def qk_norm_rotary(q, k, positions, inv_freq, q_weight=None, k_weight=None, *, eps=1e-6, interleaved=False, scale=1.0):
    """Queries ``q`` [T, Hq, D] or [B, L, Hq, D] and keys ``k`` [.., Hk, D] (or None) -> new tensors of their shapes (only
    the first without ``k``).

    A head with a weight [D] is divided by its root mean square first, ``u = w x / sqrt(mean x^2 + eps)``.  Then pair i of
    its first ``rot = 2 * len(inv_freq)`` values turns by ``position * inv_freq[i]``: values (2i, 2i + 1) when
    ``interleaved``, else (i, i + rot / 2); rotated values are multiplied by ``scale``, the others kept.  ``positions`` are
    int32 or int64 (any sign, below 2^31), [T], [B, L] or [L] for every batch element; ``inv_freq`` float64 (or float32) on the device, see
    ``rotary_inv_freq``.  Angles are formed and reduced to a turn in 64 bits, the rest in fp32, rounded once.  Differentiable in q, k and the
    weights, once and in reverse mode (a second differentiation raises, as forward mode does); the weights' gradients are
    summed in a fixed order.  D <= 512."""
    qo, ko = ops.qk_norm_rotary(q, k, positions, inv_freq, q_weight, k_weight, eps=eps, interleaved=interleaved, scale=scale)
    return qo if k is None else (qo, ko)


def rotary_append(q, k, v, positions, k_pages, v_pages, block_table, inv_freq=None, q_weight=None, k_weight=None, *,
                  seq_ids=None, eps=1e-6, interleaved=False, scale=1.0):
    """``qk_norm_rotary`` on new tokens, whose keys, and values ``v`` as they are, go to the pages of a cache; returns the
    queries.  One launch; not differentiable (the result is detached, the pools' versions rise).

    ``k_pages``, ``v_pages`` [pages, page_size, Hk, D] (any strides but over D) are written in place.  Token t belongs to row
    ``seq_ids[t]`` (int32 [T]; without it there is one token for every row) of ``block_table`` (int32 [sequences, pages of a
    sequence]) and goes to page ``block_table[row, position // page_size]``, slot ``position % page_size``.  A token of a
    negative position is padding and stored nowhere; one that the table gives no page is not stored either, and
    ``ops.device_status()`` raises.  Two tokens of one call must not share a slot.  ``inv_freq`` None: no rotation."""
    return ops.rotary_append(q, k, v, positions, k_pages, v_pages, block_table, inv_freq, q_weight, k_weight, seq_ids=seq_ids,
                             eps=eps, interleaved=interleaved, scale=scale)


def paged_decode_attention(q, k_pages, v_pages, block_table, seqlens, *, softmax_scale=None, window=0, return_lse=False):
    """One new token of each sequence, ``q`` [B, Hq, D], against its keys and values -> [B, Hq, D] (and the logarithm of the
    softmax's sum, fp32 [B, Hq], with ``return_lse``).

    Key j of sequence b lies at page ``block_table[b, j // page_size]``, slot ``j % page_size``; ``seqlens`` int32 [B] counts
    them, the new token's own (``rotary_append`` it first) among them.  Query heads share key heads in blocks of Hq / Hk.
    Scores are multiplied by ``softmax_scale`` (1 / sqrt(D)); ``window`` > 0 keeps the last so many keys.  A sequence of no
    keys gives zeros and -inf.  ``block_table`` None: contiguous caches [B, keys, Hk, D].  Lengths and table are read on the
    device: the call can be captured and replayed while they change.  Keys that the table gives no page are left out, and
    ``ops.device_status()`` raises (a sequence that is left none gives zeros and -inf as well).  Scores and sums are fp32; where
    16-bit values are multiplied on the tensor cores, probabilities enter as head and remainder of their type, off by 2^-16 of
    themselves at most.  Not differentiable: the result is detached.  D <= 256."""
    out, lse = ops.paged_decode_attention(q, k_pages, v_pages, block_table, seqlens, softmax_scale=softmax_scale, window=window,
                                          want_lse=return_lse)
    return (out, lse) if return_lse else out


def copy_pages(pools, src, dst) -> None:
    """``pool[dst[i]] = pool[src[i]]`` in each of ``pools`` (tensors [pages, ...] of one shape, whose pages are contiguous),
    in one launch for up to 64 pools and 2048 pages.

    ``src`` and ``dst`` are page numbers on the host (lists, or CPU tensors): they become part of the launch, a captured call
    replays the pages it was captured with.  A page may be copied to several; one that is written twice, or both read and
    written, is refused.  The pools must not overlap."""
    src, dst = (x.tolist() if isinstance(x, torch.Tensor) and not x.is_cuda else x for x in (src, dst))
    if isinstance(src, torch.Tensor) or isinstance(dst, torch.Tensor):
        raise TypeError("copy_pages: page numbers are host data")
    ops.copy_pages(pools, src, dst)
