"""torch front end of the serving operators (include/akili_serving.h).

What a transformer layer needs next to the kbt_* projections to answer
prompts and to decode over a paged key/value cache:

* ``rope_table``, ``rope``, ``rope_append`` — rotary positions, the latter
  writing the rotated keys and the values into the cache;
* ``prompt_attention`` — causal attention over packed prompts;
* ``tree_mask``, ``tree_attention`` — attention of new tokens (single ones,
  chunks, drafted trees) over the cache;
* ``cache_accept`` — compaction of the accepted branch after verification.

Tensors are CUDA tensors on the current device with a contiguous last axis;
index tensors are int32 (slots int64).  The other strides are free for the
rotations and ``cache_accept`` (written axes may not be broadcast).  The
attentions load tiles: their q, k, v, pages and outputs start on 16 bytes, with
positive strides that are multiples of 8 elements.  Wrong types, shapes or
devices raise TypeError or ValueError before the launch; the C entry's own
refusals raise ``abi.AkiliError``.

Calls run on ``stream`` (default: the current stream) and do not synchronise;
what they return is allocated on that stream, so a stream whose inputs are ready
needs to wait for nothing else.  The operators have no autograd formulas:
results of inputs that require gradients raise in a backward pass (a cache's
pages carry no history).
"""
from __future__ import annotations

import os

import torch

from . import abi

_MODULE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_serving.so")


class _Native:
    """The compiled front end (csrc/serving_torch.cpp), loaded at the first call."""

    def __getattr__(self, name):
        if not os.path.exists(_MODULE):
            raise FileNotFoundError(
                f"{_MODULE} is not built; run `python -m akili_bench_b200.build` (the CUDA path has no fallback)")
        abi.load()
        from . import _serving
        for n in dir(_serving):
            if not n.startswith("_"):
                setattr(self, n, getattr(_serving, n))
        return self.__dict__[name]


_native = _Native()


def rope_table(max_positions: int, rot_dim: int, base: float = 10000.0, scaling: str | None = None,
               factor: float = 1.0, original_positions: float = 0.0, low: float = 0.0, high: float = 0.0,
               amplitude: float = 0.0, device=None, stream=None) -> torch.Tensor:
    """The table `rope` and `rope_append` read: fp32 [max_positions, rot_dim], cosines then sines.

    scaling (for contexts longer than the trained one): None; "linear"
    (positions divided by `factor`); "base" (NTK-aware: base *
    factor**(rot_dim/(rot_dim-2))); "bands" (frequencies kept where more than
    `high` wavelengths fit `original_positions`, divided by `factor` where
    fewer than `low` do, blended between); "ramp" (YaRN: the same by pair
    index, `high`/`low` turns as the ends of the ramp).  amplitude 0 means 1,
    and 0.1 ln(factor) + 1 for "ramp"."""
    if scaling not in abi.ROPE_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}")
    place = torch.device("cuda" if device is None else device)
    if place.type != "cuda" or place.index not in (None, torch.cuda.current_device()):
        raise ValueError("serving ops take CUDA tensors on the current device")
    return _native.rope_table(max_positions, rot_dim, abi.ROPE_SCALINGS[scaling], base, factor, original_positions, low,
                              high, amplitude, stream)


def rope(q, k, positions, table, interleaved: bool = False, inverse: bool = False, q_out=None, k_out=None,
         stream=None):
    """Rotate the first rot_dim = table.shape[1] values of each head of q [tokens, q_heads, head_dim] and
    k [tokens, k_heads, head_dim] by the angles of their positions (int32 [tokens]).

    Pairs are (i, i + rot_dim/2), or (2i, 2i + 1) when interleaved.  inverse=True rotates back: it is the
    gradient (apply it to dq, dk).  q_out/k_out may be q/k (in place).  A token whose position is outside the
    table is skipped and recorded (``ops.device_status``): its output rows are not written, so that new ones hold
    anything.  Returns (q_out, k_out)."""
    return _native.rope(q, k, positions, table, interleaved, inverse, q_out, k_out, stream)


def rope_append(q, k, v, positions, table, slots, k_pages, v_pages, interleaved: bool = False, q_out=None,
                k_out=None, stream=None):
    """`rope`, with the rotated k and v [tokens, k_heads, head_dim] written to row slots[token] = page *
    page_size + offset (int64; -1: padding, nothing is written) of k_pages/v_pages [num_pages, page_size,
    k_heads, head_dim].  k_out, if given, gets the rotated k as well (`prompt_attention` of the same prompt
    reads it; it may be k).  A token whose position is outside the table is skipped and recorded: nothing is
    written for it, and its rows of a new q_out hold anything.  Returns the rotated q (q_out; may be q)."""
    return _native.rope_append(q, k, v, positions, table, slots, k_pages, v_pages, interleaved, q_out, k_out, stream)


def prompt_attention(q, k, v, cu_q, cu_k=None, softmax_scale: float | None = None, causal: bool = True, out=None,
                     return_lse: bool = False, stream=None):
    """Attention over packed prompts: sequence b has the query rows cu_q[b]:cu_q[b+1] of q [total_q, q_heads,
    head_dim] and the key rows cu_k[b]:cu_k[b+1] (default cu_q) of k, v [total_k, kv_heads, head_dim].

    With n queries and m keys, query i sees the keys j <= i + m - n (causal) or all; one that sees none gives
    0.  Query head h reads key head h // (q_heads // kv_heads).  softmax_scale defaults to head_dim**-0.5;
    0.0 weighs all visible keys alike.  Rows past the last sequence are not written (in a new out and lse they hold
    anything).  Returns out, or (out, lse) with lse fp32 [total_q, q_heads] (natural log, -inf for a row without
    keys)."""
    return _native.prompt_attention(q, k, v, cu_q, cu_k, softmax_scale, causal, out, return_lse, stream)


def tree_mask(parents, cu_q, max_nodes: int, stream=None) -> torch.Tensor:
    """The mask `tree_attention` takes, int32 [total_q, ceil(max_nodes / 32)]: bit j of node i's row is set for
    i itself and its ancestors.  parents int32 [total_q]: the parent's index within its own tree, smaller than
    the node's, or -1 for a root.  max_nodes: at least the largest tree's nodes."""
    return _native.tree_mask(parents, cu_q, (max_nodes + 31) // 32, stream)


def tree_attention(q, k_pages, v_pages, page_table, context_lens, cu_q, mask=None, softmax_scale: float | None = None,
                   out=None, return_lse: bool = False, workspace=None, stream=None):
    """Attention of each sequence's new tokens over its paged cache.

    The new tokens of sequence b are the rows cu_q[b]:cu_q[b+1] of q [total_q, q_heads, head_dim]; their keys
    and values already follow its context_lens[b] sure tokens in the cache (`rope_append`).  Entry j lies in
    row j % page_size of page page_table[b, j // page_size] of k_pages/v_pages [num_pages, page_size, kv_heads,
    head_dim] (any strides, page_size a multiple of 8).  Every new token sees the context and the new tokens
    of its mask row (`tree_mask`); without a mask, itself and those before it (a single token, a chunk).  Rows past
    the last sequence are not written (in a new out and lse they hold anything).
    Returns out, or (out, lse); `workspace` is an optional uint8 tensor of tree_attention_workspace() bytes."""
    return _native.tree_attention(q, k_pages, v_pages, page_table, context_lens, cu_q, mask, softmax_scale, out,
                                  return_lse, workspace, stream)


def tree_attention_workspace(q, k_pages, page_table, context_lens) -> int:
    """Bytes of workspace a `tree_attention` call with these heads and sizes uses."""
    return _native.tree_attention_workspace(q, k_pages, page_table, context_lens)


def cache_accept(k_pages, v_pages, page_table, context_lens, accepted, n_accepted, new_lens=None, stream=None):
    """Move the accepted nodes' cache entries to the end of the sure context, in every layer.

    k_pages/v_pages [layers, num_pages, page_size, kv_heads, head_dim] (or without the layers axis) are changed
    in place: entry context_lens[b] + accepted[b, i] of sequence b moves to context_lens[b] + i for i <
    n_accepted[b].  accepted int32 [batch, any] ascends in each row.  Returns context_lens + n_accepted
    (new_lens, which shares no memory with the index tensors)."""
    return _native.cache_accept(k_pages, v_pages, page_table, context_lens, accepted, n_accepted, new_lens, stream)
