"""Operators for serving many requests at once, over a paged KV cache.

The resident engine (:class:`DecodeEngine`) decodes one stream over a contiguous
cache. These are the attention steps of a batch of requests of any lengths, as one
layer of a model calls them:

* :func:`paged_append` -- q/k RMSNorm, RoPE and the K/V rows into the cache's pages;
* :func:`prompt_attention` -- causal attention of whole prompts, packed one after
  another;
* :func:`paged_attention` -- attention of each request's new tokens over its keys in
  the cache: one token each when decoding, a chunk of a prompt, or a mix of both.

A batch is packed: request ``b``'s new tokens are rows ``cu_q[b] .. cu_q[b+1] - 1``.
Without ``cu_q`` every request brings one token (``[batch, heads, dim]``) or ``n``
(``[batch, n, heads, dim]``). The cache is two pools ``[pages, kv_heads, page_size,
dim]`` (any strides of whole 16 bytes, so another order of the dimensions is a
permuted view), ``block_table[b]`` lists request ``b``'s pages and ``kv_lens[b]``
counts its keys, the new tokens included. BF16 or FP16, heads of 64 or 128, up
to 128 query heads per KV head, pages of a power of two of 16 keys or more; tokens and
requests together, times the query heads, up to 2^30.

A token sees the keys up to its own position; one that sees none gets zeros, one whose
scores are all ``-inf`` NaN. What a page holds past a request's last key reaches no
output, and values that are not finite reach the rows that see them and no others. Rows
of no request (before ``cu_q[0]``, from ``cu_q[-1]`` on) are not written by the
attention; the append gives zeros. Calls run on the current stream, do not synchronise,
and can be captured into a CUDA graph. Host-side misuse raises ``ValueError``; lengths
and page numbers are read on the device, where a wrong one makes its request's new rows
NaN, some or all, and is kept for :func:`serving_status`. These are operators of an
inference framework: results carry no gradients, whatever the inputs do.

There is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import torch

STATUS_NAMES = {
    0: "ok",
    1: "block_table names a page outside the pool",
    2: "kv_lens counts more keys than block_table has pages for, or than 2^30",
    3: "a position past the RoPE tables",
    4: "timeout of a wait inside a kernel",
}

_ops = None


def _extension():
    global _ops
    if _ops is None:
        from . import extension
        _ops = extension()
    return _ops


def prompt_attention(q, k, v, cu_seqlens, *, scale=None, out=None):
    """Causal attention of packed prompts: ``q`` [tokens, heads, dim], ``k`` and ``v``
    [tokens, kv_heads, dim], ``cu_seqlens`` int32 [prompts + 1] on the device. ``scale``
    defaults to ``dim ** -0.5``. Returns [tokens, heads, dim], in ``out`` if given, which may
    be ``q``."""
    return (_ops or _extension()).prompt_attention(q, k, v, cu_seqlens, scale, out)


def paged_attention(q, k_cache, v_cache, block_table, kv_lens, cu_q=None, *, scale=None, out=None):
    """Attention of new tokens over the paged cache (their own K/V rows already in it).
    Returns ``q``'s shape, in ``out`` if given, which may be ``q``."""
    return (_ops or _extension()).paged_attention(q, k_cache, v_cache, block_table, kv_lens, cu_q, scale, out)


def paged_append(qkv, k_cache, v_cache, block_table, kv_lens, cos, sin, cu_q=None, *, q_norm=None, k_norm=None,
                 eps=1e-6, return_k=False):
    """``qkv`` [tokens, heads + 2 kv_heads, dim] (BF16, FP16 or FP32) -> q, normed (where
    ``q_norm`` is given) and turned to its position by ``cos`` / ``sin`` [positions, dim];
    the K rows (likewise) and V rows go to their pages. ``return_k`` also returns the K
    rows packed, as :func:`prompt_attention` takes them."""
    return (_ops or _extension()).paged_append(qkv, k_cache, v_cache, block_table, kv_lens, cos, sin, cu_q, q_norm,
                                               k_norm, eps, return_k)


def serving_status(device=None):
    """(code, name) of the first error that these operators met on ``device`` since the
    last call, replays of graphs included; (0, "ok") if none. Waits for the device."""
    d = torch.device("cuda" if device is None else device)
    code = int(_extension().serving_status(d.index if d.index is not None else torch.cuda.current_device()))
    return code, STATUS_NAMES.get(code, "unknown")
