"""Attention of drafted tokens over a KV pool, bf16 or quantised.

A draft proposes several continuations of a context at once, as a tree: node i
has a parent among the nodes before it or hangs under the context, and its path
to the context is one candidate continuation. All nodes are scored by one pass
over the pool: node i reads the committed slots and those drafted slots that
`tree_mask[i]` names, its ancestors'. In the strict-past attention of this
package a token reads the tokens before it and not itself, so the mask of a
tree holds the strict ancestors (`tree_mask_from_parents`); any other boolean
mask may be given.

Without a tree_mask the query tokens read the committed slots alone: with one
token per row this is the decode step over a quantised pool (the bf16 pool's
own is strict_causal_attention with one query).

The HIP path is the operator white_matter::tree_attention (wmx_tree_attn): the
query rows of a KV head share one read of its keys and values, products on the
matrix cores with codes converted exactly to bf16, key ranges split over
workgroups and merged in log-sum-exp form.
"""

from __future__ import annotations

from collections.abc import Sequence
from typing import Literal

import torch

from . import _kernels, _native, portable
from .kv_pool import QuantizedPool

_native.load_ops()

_BACKENDS = ("auto", "reference", "hip")


# tree_attention(query, key, value, key_scales, value_scales, kv_lengths,
#     kv_length, tree_mask, key_mask, use_dummy, scale, num_splits) ->
#     (B, n, H, D) bf16, and its argument checks alone, for any device
_tree_attention = torch.ops.white_matter.tree_attention.default
_tree_attention_check = torch.ops.white_matter.tree_attention_check.default


@torch.library.register_fake("white_matter::tree_attention")
def _(query, key, *args):
    batch, heads, nodes, dim = query.shape
    return query.new_empty(batch, nodes, heads, dim, dtype=torch.bfloat16)


def tree_mask_from_parents(
    parents: torch.Tensor | Sequence[int], *, include_self: bool = False, device: torch.device | str | None = None
) -> tuple[torch.Tensor, torch.Tensor]:
    """(tree_mask, depths) of drafted trees given as parents (n,) or (B, n):
    the node that each node hangs under, one before it, or -1 for the context.

    tree_mask (n, n) or (B, n, n) bool: whether node i sees node a, a strict
    ancestor (with include_self also the node itself). depths int64, parents'
    shape: how many nodes lie between a node and the context (a node's position
    is the context's length plus its depth). Built on the host; parents on the
    GPU are copied there first, which a HIP graph capture cannot hold."""
    source = parents if isinstance(parents, torch.Tensor) else torch.as_tensor(parents)
    if device is None:
        device = source.device
    if source.is_cuda:
        _kernels.guard_capture("building a tree mask")
    table = source.cpu()
    if table.ndim not in (1, 2) or (table.numel() and table.dtype not in (torch.int32, torch.int64)):
        raise ValueError("parents must be integer (n,) or (B, n)")
    rows = (table if table.ndim == 2 else table[None]).long()
    nodes = rows.shape[1]
    if bool(((rows < -1) | (rows >= torch.arange(nodes))).any()):
        raise ValueError("a node's parent must be an earlier node, or -1 for the context")
    mask = torch.zeros(rows.shape[0], nodes, nodes, dtype=torch.bool)
    depths = torch.zeros(rows.shape, dtype=torch.int64)
    every = torch.arange(rows.shape[0])
    for i in range(nodes):  # a parent's own row is complete
        p = rows[:, i]
        under = p >= 0
        at = p.clamp_min(0)
        mask[:, i] = mask[every, at] & under[:, None]
        mask[every[under], i, at[under]] = True
        depths[:, i] = torch.where(under, depths[every, at] + 1, 0)
    if include_self:
        mask |= torch.eye(nodes, dtype=torch.bool)
    return mask.view(*table.shape, nodes).to(device), depths.view(table.shape).to(device)


def tree_attention(
    query: torch.Tensor,
    key: torch.Tensor | QuantizedPool,
    value: torch.Tensor | QuantizedPool,
    *,
    kv_lengths: int | torch.Tensor,
    tree_mask: torch.Tensor | None = None,
    use_dummy_token: bool = False,
    key_mask: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    backend: Literal["auto", "reference", "hip"] = "auto",
    num_splits: int = 0,
) -> torch.Tensor:
    """Attention of n drafted tokens per row over a KV pool.

    query (B,H,n,D); key/value (B,Hkv,N,D) bf16 pool views, or QuantizedPools
    of that shape (codes (B,Hkv,N,D), scales (B,Hkv,N): a pool's channel,
    `pool.select(1, channel)`); output (B,n,H,D) in the query's type.

    kv_lengths, an integer or integer (B,), counts the committed real tokens of
    each row, excluding the dummy slot; the drafted tokens' keys and values sit
    in the n slots behind them. Query i sees the dummy (with use_dummy_token),
    the committed slots and, with tree_mask (n,n) or (B,n,n) bool, drafted slot
    a where tree_mask[..., i, a]; of these only those with key_mask (B,N) where
    given. Slots that no query of the row sees may hold anything, NaN included,
    and so may drafted slots for the queries that do not see them. Drafted slots
    past the pool's end are not seen. A query that sees nothing gives zeros.
    Forward only. num_splits sets the key split count of the HIP kernel.
    """
    if backend not in _BACKENDS:
        raise ValueError(f"unsupported tree attention backend: {backend!r}")
    if type(use_dummy_token) is not bool:
        raise ValueError("use_dummy_token must be boolean")
    k, key_scales = key if isinstance(key, QuantizedPool) else (key, None)
    v, value_scales = value if isinstance(value, QuantizedPool) else (value, None)
    lengths, length = (kv_lengths, 0) if isinstance(kv_lengths, torch.Tensor) else (None, kv_lengths)
    if type(length) is not int:
        raise ValueError("kv_lengths must be an integer or integer (B,)")
    dim = query.shape[-1]
    scale = dim**-0.5 if softmax_scale is None else float(softmax_scale)
    # (shapes, types, devices and strides are checked by the operator)
    if backend == "reference" or not query.is_cuda:
        _tree_attention_check(
            query, k, v, key_scales, value_scales, lengths, length, tree_mask, key_mask, use_dummy_token, scale, num_splits
        )
        if backend == "hip":
            raise ValueError("the HIP backend requires GPU tensors")
        return portable.tree_attention_portable(
            query, k, v, key_scales, value_scales, length if lengths is None else lengths, tree_mask, use_dummy_token, key_mask,
            scale,
        )
    padded = _kernels.kernel_head_dim(dim)
    if padded is None:
        raise RuntimeError(f"the gfx950 attention kernels: this path does not support head_dim {dim} (maximum 128)")
    if padded == dim or key_scales is not None:
        out = _tree_attention(
            query, k, v, key_scales, value_scales, lengths, length, tree_mask, key_mask, use_dummy_token, scale, num_splits
        )
    else:
        q, k, v = (_kernels.pad_head_dim(t, padded) for t in (query, k, v))
        out = _tree_attention(
            q, k, v, None, None, lengths, length, tree_mask, key_mask, use_dummy_token, scale, num_splits
        )[..., :dim]
    return out if out.dtype == query.dtype else out.to(query.dtype)
