"""torch front end of the serving operators (include/akili_serving.h).

What a transformer layer needs next to the kbt_* projections to answer
prompts and to decode over a paged key/value cache:

* ``rope_table``, ``rope``, ``rope_append`` — rotary positions, the latter
  writing the rotated keys and the values into the cache;
* ``prompt_attention`` — causal attention over packed prompts;
* ``tree_mask``, ``tree_attention`` — attention of new tokens (single ones,
  chunks, drafted trees) over the cache;
* ``cache_accept`` — compaction of the accepted branch after verification.

Tensors are CUDA tensors on the current device, of any strides with a
contiguous last axis; index tensors are int32 (slots int64).  Wrong types,
shapes or devices raise before the launch; the C entry's own refusals raise
``abi.AkiliError``.  Calls run on ``stream`` (default: the current stream)
and do not synchronise.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi

_DTYPES = {torch.float32: abi.DTYPE_F32, torch.float16: abi.DTYPE_F16, torch.bfloat16: abi.DTYPE_BF16}


def _dtype(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


def _call(op: str, arg, stream, *made: torch.Tensor) -> None:
    """Launch akili_<op>; `made` are tensors this call allocated (on the current stream)."""
    if stream is None:
        s = torch.cuda.current_stream().cuda_stream
    else:
        s = stream.cuda_stream
        for t in made:
            t.record_stream(stream)
    rc = getattr(abi.load(), "akili_" + op)(C.byref(arg), s)
    if rc != abi.OK:
        raise abi.AkiliError(op, rc)


def _check_values(first: torch.Tensor, **others: torch.Tensor) -> None:
    """CUDA tensors of one type on the current device with a contiguous last axis."""
    if not first.is_cuda or first.get_device() != torch.cuda.current_device():
        raise ValueError("serving ops take CUDA tensors on the current device")
    if first.stride(-1) != 1 and first.shape[-1] != 1:
        raise ValueError("the last axis must be contiguous")
    for name, t in others.items():
        if t.dtype != first.dtype or t.device != first.device:
            raise ValueError(f"{name} must be {first.dtype} on {first.device}")
        if t.stride(-1) != 1 and t.shape[-1] != 1:
            raise ValueError(f"the last axis of {name} must be contiguous")


def _check_index(name: str, t: torch.Tensor, device, shape: tuple, dtype=torch.int32) -> int:
    """Address of an index tensor of this shape (None matches any size); rows may be strided, the last axis not."""
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}")
    if t.dim() != len(shape) or any(w is not None and w != g for w, g in zip(shape, t.shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if t.numel() and t.stride(-1) != 1 and t.shape[-1] != 1:
        raise ValueError(f"the last axis of {name} must be contiguous")
    return t.data_ptr()


def _check_shape(name: str, t: torch.Tensor, shape: tuple) -> None:
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")


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
    out = torch.empty((max_positions, rot_dim), device=device or "cuda", dtype=torch.float32)
    _check_values(out)
    _call("rope_table", abi.RopeTableArg(max_positions, rot_dim, abi.ROPE_SCALINGS[scaling], 0, base, factor,
                                         original_positions, low, high, amplitude, out.data_ptr()), stream, out)
    return out


def _rope_common(q, k, positions, table):
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("q and k are [tokens, heads, head_dim] with the same tokens and head_dim")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous() or table.device != q.device:
        raise ValueError("table is a contiguous fp32 [max_positions, rot_dim] tensor on the device of q")
    return _check_index("positions", positions, q.device, (q.shape[0],))


def rope(q, k, positions, table, interleaved: bool = False, inverse: bool = False, q_out=None, k_out=None,
         stream=None):
    """Rotate the first rot_dim = table.shape[1] values of each head of q [tokens, q_heads, head_dim] and
    k [tokens, k_heads, head_dim] by the angles of their positions (int32 [tokens]).

    Pairs are (i, i + rot_dim/2), or (2i, 2i + 1) when interleaved.  inverse=True rotates back: it is the
    gradient (apply it to dq, dk).  q_out/k_out may be q/k (in place).  Returns (q_out, k_out)."""
    _check_values(q, k=k)
    pos = _rope_common(q, k, positions, table)
    made = []
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        made.append(q_out)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        made.append(k_out)
    _check_values(q, q_out=q_out, k_out=k_out)
    _check_shape("q_out", q_out, tuple(q.shape))
    _check_shape("k_out", k_out, tuple(k.shape))
    t, hq, d = q.shape
    flags = (abi.ROPE_INTERLEAVED if interleaved else 0) | (abi.ROPE_INVERSE if inverse else 0)
    arg = abi.RopeArg(_dtype(q), flags, t, hq, k.shape[1], d, table.shape[1], table.shape[0], q.data_ptr(),
                      k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), pos, table.data_ptr(), *q.stride()[:2],
                      *k.stride()[:2], *q_out.stride()[:2], *k_out.stride()[:2])
    _call("rope", arg, stream, *made)
    return q_out, k_out


def rope_append(q, k, v, positions, table, slots, k_pages, v_pages, interleaved: bool = False, q_out=None,
                stream=None):
    """`rope`, with the rotated k and v [tokens, k_heads, head_dim] written to row slots[token] = page *
    page_size + offset (int64; -1: padding, nothing is written) of k_pages/v_pages [num_pages, page_size,
    k_heads, head_dim].  Returns the rotated q (q_out; may be q)."""
    if q_out is None:
        q_out, made = torch.empty(q.shape, dtype=q.dtype, device=q.device), True
    else:
        made = False
    _check_values(q, k=k, v=v, k_pages=k_pages, v_pages=v_pages, q_out=q_out)
    pos = _rope_common(q, k, positions, table)
    t, hq, d = q.shape
    hk = k.shape[1]
    _check_shape("v", v, (t, hk, d))
    _check_shape("q_out", q_out, (t, hq, d))
    if k_pages.dim() != 4 or k_pages.shape[2:] != (hk, d) or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages are [num_pages, page_size, k_heads, head_dim]")
    where = _check_index("slots", slots, q.device, (t,), torch.int64)
    arg = abi.RopeArg(_dtype(q), abi.ROPE_INTERLEAVED if interleaved else 0, t, hq, hk, d, table.shape[1],
                      table.shape[0], q.data_ptr(), k.data_ptr(), q_out.data_ptr(), 0, pos, table.data_ptr(),
                      *q.stride()[:2], *k.stride()[:2], *q_out.stride()[:2], 0, 0, v.data_ptr(), where,
                      k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0], k_pages.shape[1], *v.stride()[:2],
                      *k_pages.stride()[:3], *v_pages.stride()[:3])
    _call("rope_append", arg, stream, *((q_out,) if made else ()))
    return q_out


def _attention_out(q, out, return_lse):
    if q.dim() != 3:
        raise ValueError("q is [tokens, q_heads, head_dim]")
    made = []
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        made.append(out)
    lse = None
    if return_lse:
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        made.append(lse)
    return out, lse, made


def prompt_attention(q, k, v, cu_q, cu_k=None, softmax_scale: float | None = None, causal: bool = True, out=None,
                     return_lse: bool = False, stream=None):
    """Attention over packed prompts: sequence b has the query rows cu_q[b]:cu_q[b+1] of q [total_q, q_heads,
    head_dim] and the key rows cu_k[b]:cu_k[b+1] (default cu_q) of k, v [total_k, kv_heads, head_dim].

    With n queries and m keys, query i sees the keys j <= i + m - n (causal) or all; one that sees none gives
    0.  Query head h reads key head h // (q_heads // kv_heads).  softmax_scale defaults to head_dim**-0.5.
    Returns out, or (out, lse) with lse fp32 [total_q, q_heads] (natural log, -inf for a row without keys)."""
    if cu_k is None:
        cu_k = cu_q
    out, lse, made = _attention_out(q, out, return_lse)
    _check_values(q, k=k, v=v, out=out)
    if k.dim() != 3 or k.shape[2] != q.shape[2] or v.shape != k.shape:
        raise ValueError("k and v are [total_k, kv_heads, head_dim]")
    _check_shape("out", out, tuple(q.shape))
    cq = _check_index("cu_q", cu_q, q.device, (None,))
    ck = _check_index("cu_k", cu_k, q.device, tuple(cu_q.shape))
    if cu_q.shape[0] == 0:
        raise ValueError("cu_q has batch + 1 entries")
    t, hq, d = q.shape
    arg = abi.PromptAttentionArg(_dtype(q), hq, k.shape[1], d, cu_q.shape[0] - 1, t, k.shape[0], int(causal),
                                 softmax_scale or 0.0, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                 0 if lse is None else lse.data_ptr(), cq, ck, *q.stride()[:2], *k.stride()[:2],
                                 *v.stride()[:2], *out.stride()[:2])
    _call("prompt_attention", arg, stream, *made)
    return out if lse is None else (out, lse)


def tree_mask(parents, cu_q, max_nodes: int, stream=None) -> torch.Tensor:
    """The mask `tree_attention` takes, int32 [total_q, ceil(max_nodes / 32)]: bit j of node i's row is set for
    i itself and its ancestors.  parents int32 [total_q]: the parent's index within its own tree, smaller than
    the node's, or -1 for a root.  max_nodes: at least the largest tree's nodes."""
    if not parents.is_cuda or parents.get_device() != torch.cuda.current_device():
        raise ValueError("serving ops take CUDA tensors on the current device")
    words = (max_nodes + 31) // 32
    p = _check_index("parents", parents, parents.device, (None,))
    c = _check_index("cu_q", cu_q, parents.device, (None,))
    mask = torch.empty((parents.shape[0], words), dtype=torch.int32, device=parents.device)
    _call("tree_mask", abi.TreeMaskArg(cu_q.shape[0] - 1, parents.shape[0], words, 0, p, c, mask.data_ptr()), stream,
          mask)
    return mask


def tree_attention(q, k_pages, v_pages, page_table, context_lens, cu_q, mask=None, softmax_scale: float | None = None,
                   out=None, return_lse: bool = False, workspace=None, stream=None):
    """Attention of each sequence's new tokens over its paged cache.

    The new tokens of sequence b are the rows cu_q[b]:cu_q[b+1] of q [total_q, q_heads, head_dim]; their keys
    and values already follow its context_lens[b] sure tokens in the cache (`rope_append`).  Entry j lies in
    row j % page_size of page page_table[b, j // page_size] of k_pages/v_pages [num_pages, page_size, kv_heads,
    head_dim] (any strides, page_size a multiple of 8).  Every new token sees the context and the new tokens
    of its mask row (`tree_mask`); without a mask, itself and those before it (a single token, a chunk).
    Returns out, or (out, lse); `workspace` is an optional uint8 tensor of tree_attention_workspace() bytes."""
    out, lse, made = _attention_out(q, out, return_lse)
    _check_values(q, k_pages=k_pages, v_pages=v_pages, out=out)
    t, hq, d = q.shape
    if k_pages.dim() != 4 or k_pages.shape[3] != d or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages are [num_pages, page_size, kv_heads, head_dim]")
    _check_shape("out", out, (t, hq, d))
    batch = context_lens.shape[0]
    table = _check_index("page_table", page_table, q.device, (batch, None))
    lens = _check_index("context_lens", context_lens, q.device, (batch,))
    cq = _check_index("cu_q", cu_q, q.device, (batch + 1,))
    bits = words = mask_stride = 0
    if mask is not None:
        bits, words, mask_stride = _check_index("mask", mask, q.device, (t, None)), mask.shape[1], mask.stride(0)
    ws = ws_bytes = 0
    if workspace is not None:
        if workspace.device != q.device or not workspace.is_contiguous():
            raise ValueError("workspace is a contiguous tensor on the device of q")
        ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    pages, page_size, hk, _ = k_pages.shape
    arg = abi.TreeAttentionArg(_dtype(q), hq, hk, d, batch, t, pages, page_size, page_table.shape[1], words,
                               softmax_scale or 0.0, 0, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                               out.data_ptr(), 0 if lse is None else lse.data_ptr(), table, lens, cq, bits, ws,
                               ws_bytes, *q.stride()[:2], *out.stride()[:2], *k_pages.stride()[:3],
                               *v_pages.stride()[:3], page_table.stride(0), mask_stride)
    _call("tree_attention", arg, stream, *made)
    return out if lse is None else (out, lse)


def tree_attention_workspace(q, k_pages, page_table, context_lens) -> int:
    """Bytes of workspace a `tree_attention` call with these heads and sizes uses."""
    t, hq, d = q.shape
    pages, page_size, hk, _ = k_pages.shape
    arg = abi.TreeAttentionArg(_dtype(q), hq, hk, d, context_lens.shape[0], t, pages, page_size, page_table.shape[1])
    n = C.c_uint64(0)
    rc = abi.load().akili_tree_attention_workspace(C.byref(arg), C.byref(n))
    if rc != abi.OK:
        raise abi.AkiliError("tree_attention_workspace", rc)
    return int(n.value)


def cache_accept(k_pages, v_pages, page_table, context_lens, accepted, n_accepted, new_lens=None, stream=None):
    """Move the accepted nodes' cache entries to the end of the sure context, in every layer.

    k_pages/v_pages [layers, num_pages, page_size, kv_heads, head_dim] (or without the layers axis) are changed
    in place: entry context_lens[b] + accepted[b, i] of sequence b moves to context_lens[b] + i for i <
    n_accepted[b].  accepted int32 [batch, any] ascends in each row.  Returns context_lens + n_accepted
    (new_lens, not context_lens itself)."""
    if k_pages.dim() == 4:
        k_pages, v_pages = k_pages[None], v_pages[None]
    if k_pages.dim() != 5 or v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages are [layers, num_pages, page_size, kv_heads, head_dim]")
    _check_values(k_pages, v_pages=v_pages)
    batch = context_lens.shape[0]
    dev = k_pages.device
    table = _check_index("page_table", page_table, dev, (batch, None))
    lens = _check_index("context_lens", context_lens, dev, (batch,))
    acc = _check_index("accepted", accepted, dev, (batch, None))
    n_acc = _check_index("n_accepted", n_accepted, dev, (batch,))
    made = new_lens is None
    if made:
        new_lens = torch.empty(batch, dtype=torch.int32, device=dev)
    else:
        _check_index("new_lens", new_lens, dev, (batch,))
    layers, pages, page_size, hk, d = k_pages.shape
    arg = abi.CacheAcceptArg(k_pages.element_size(), layers, batch, hk, d, pages, page_size, page_table.shape[1],
                             accepted.shape[1], 0, k_pages.data_ptr(), v_pages.data_ptr(), table, lens, acc, n_acc,
                             new_lens.data_ptr(), *k_pages.stride()[:4], *v_pages.stride()[:4], page_table.stride(0),
                             accepted.stride(0))
    _call("cache_accept", arg, stream, *((new_lens,) if made else ()))
    return new_lens
