"""Attention on the two sparse patterns of language models, beside ``rode_sddmm`` and ``rode_spmm``.

On a CSR pattern, attention is an SDDMM (scores at the stored entries), a softmax per row and an SpMM (their product with the
values).  The patterns here need not be stored: a sliding window with first tokens that stay visible, and a prefix that a
batch of requests shares.  Scores, softmax and product run in one pass; the operators launch on torch's current stream and do
not block the host.  No counterpart in the reference.

Types: float32, float16, bfloat16 (all operands of a call alike), sums and softmax in float32.  Head dimension: any multiple of 4
up to 256.  ``k`` and ``v`` may have fewer heads than ``q``: query head h reads key head ``h // (heads // kv_heads)``.  A query
that sees no key gets zeros.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import rode_sddmm_cuda


def _scale(scale: Optional[float], q: torch.Tensor) -> float:
    return float(scale) if scale is not None else max(q.shape[-1], 1) ** -0.5


def rode_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                          q_offsets: Optional[torch.Tensor] = None, k_offsets: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None) -> torch.Tensor:
    """Attention in which a query sees the ``window`` keys up to its own position and the first ``sinks`` keys of its sequence;
    differentiable with respect to q, k and v, once, in reverse mode.

    q [q_rows, heads, dim], k and v [k_rows, kv_heads, dim] hold sequences one behind the other: sequence s is rows
    ``q_offsets[s]`` to ``q_offsets[s + 1]`` of q and ``k_offsets[s]`` to ``k_offsets[s + 1]`` of k and v (int32 on the device, not
    decreasing; k_offsets None: the same as q_offsets; both None: one sequence).  The queries of a sequence are its last
    positions: with n keys and m queries, query i stands at position ``i + n - m``.  ``window`` at least the longest
    sequence: causal attention.  Rows that belong to no sequence get zeros, in the result and in the gradients.

    ``scale`` multiplies the scores, ``dim ** -0.5`` by default.  Operands whose strides the kernels cannot take are copied.
    For the backward pass a call keeps its operands, its result, in 16-bit types one more array of the result's size, and a float per row and head.
    In a graph that is being captured, take gradients by ``torch.autograd.grad``, or with leaves that no eager graph holds: torch ties the
    accumulation into a leaf to the stream of the graph that has seen it first, whatever the operators between."""
    return rode_sddmm_cuda.window_attention(q, k, v, window, sinks, q_offsets, k_offsets, _scale(scale, q))


def rode_window_attention_step(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, window: int,
                               sinks: int = 0, scale: Optional[float] = None) -> torch.Tensor:
    """``rode_window_attention`` for one new token per sequence, against a cache that holds its key and value already.

    q [batch, heads, dim]; k_cache and v_cache [batch, capacity, kv_heads, dim] in any order of the first three dimensions (a
    transposed view of a cache that lies head by head); lengths int32 [batch] on the device: the tokens in each cache, the new
    one among them, taken as at most ``capacity``; a length of 0 gives zeros.  Nothing behind a sequence's length, and nothing
    between its sinks and its window, is read.

    Not differentiable: operands that require gradients are refused, unless gradients are off (``torch.no_grad()``)."""
    return rode_sddmm_cuda.window_attention_step(q, k_cache, v_cache, lengths, window, sinks, _scale(scale, q))


def rode_shared_prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k_cache: torch.Tensor,
                                 v_cache: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token per request, where all requests share a prefix, which is read once for all of them.

    q [batch, heads, dim]; prefix_k and prefix_v [prefix, kv_heads, dim]; k_cache, v_cache and lengths as in
    ``rode_window_attention_step``, for the tokens behind the prefix (a length of 0 is a request that has none yet).  Request b
    sees the whole prefix and the first ``lengths[b]`` rows of its cache.

    Not differentiable: operands that require gradients are refused, unless gradients are off (``torch.no_grad()``)."""
    return rode_sddmm_cuda.shared_prefix_attention(q, prefix_k, prefix_v, k_cache, v_cache, lengths, _scale(scale, q))


def rode_attention_waits_failed(device: Union[torch.device, str, None] = None) -> bool:
    """Whether a kernel of this module on ``device`` (None: the current one) ever gave up a wait between its warps.

    The tensor-core kernels bound such waits to some seconds instead of hanging.  A call has long returned by then, so nothing raises: where this is
    True (an error of this library), the results of at least one call so far are wrong or were not written.  Waits for everything that runs on the
    device (and so cannot be called while a graph is captured); not for every step, but once behind a run whose results count."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"device must be a CUDA device, got {device}")
    return rode_sddmm_cuda.attention_waits_failed(torch.cuda.current_device() if device.index is None else device.index)
