"""Decoding from drafted tokens: what the nodes of a draft see, their attention over the cache, their verification."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _capi as C
from .kv_cache import KVLayer

_masks = torch.ops.sparse_mlp.draft_masks.default
_attention = torch.ops.sparse_mlp.tree_attention.default
_attention_out = torch.ops.sparse_mlp.tree_attention.out
_verify = torch.ops.sparse_mlp.verify_draft.default


def draft_masks(parents: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """parents int64 [n_seq, nodes] (parent < node, -1 for the root; 64 nodes at most) -> (masks, depth), int64 of the same
    shape: bit j of masks[b, i] is set when node i sees node j (itself and its ancestors); depth counts the ancestors."""
    return _masks(parents)


def tree_attention(q: torch.Tensor, cache: KVLayer, length: torch.Tensor, *, tree: Optional[torch.Tensor] = None,
                   counts: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of drafted tokens q [n_seq, nodes, heads, head_dim] (rotated) over a cache layer that already holds their keys and values.

    length int64 [n_seq]: tokens before the draft, seen by every node; node j stands in slot length[b] + j.  tree: int64 [nodes] or
    [n_seq or 1, nodes], bit j of node i's word set when it sees node j (default: a chain, j <= i).  counts int64 [n_seq]: nodes
    in use (default all).  A node that sees nothing, or is not in use, gets zeros.  heads may be a multiple of the cache's.
    scale: of the scores, head_dim^-1/2 by default.  Waits inside the kernel are bounded: see attention_timed_out."""
    if out is None:
        return _attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, length, tree, counts, scale)
    return _attention_out(q, cache.k, cache.v, cache.k_scale, cache.v_scale, length, tree, counts, scale, out=out)


def attention_timed_out(device: Optional[torch.device] = None) -> bool:
    """True when a wait inside a tree_attention call on the device (default: the current one) gave up since this function last
    said so; rows of that call's result are NaN.  Synchronises the current stream."""
    st = ctypes.c_int()
    with torch.cuda.device(device):
        C.check(C.lib.stx_tree_attention_status(ctypes.byref(st), torch.cuda.current_stream().cuda_stream))
    return st.value != C.OK


def verify_draft(tokens: torch.Tensor, target: torch.Tensor, *, uniform: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None,
                 draft: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens the target accepts, and the token behind them: (path [n_seq, nodes], count [n_seq], next [n_seq]),
    int64; path lists the accepted nodes, the root first, then -1.

    tokens int64 [n_seq, nodes]; node 0 is the root, whose token is settled.  target: the target's probabilities fp32
    [n_seq, nodes, vocabulary] behind each node, with uniform fp32 [n_seq, nodes] in [0, 1); or its tokens int64 [n_seq, nodes]
    (greedy).  parents int64 [n_seq, nodes]: a tree of candidates; None: a chain.  draft fp32 [n_seq, nodes - 1, vocabulary]: for
    a chain whose tokens were drawn, the distribution that node i + 1 was drawn from.  counts: nodes in use.  Either way the
    emitted tokens follow the target's distribution."""
    return _verify(tokens, target, uniform, parents, draft, counts)
