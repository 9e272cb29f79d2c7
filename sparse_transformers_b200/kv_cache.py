"""Key/value cache of a decoder in 16, 32 or 8 bits: written (keys rotated on the way), read back, compacted."""
from __future__ import annotations

from typing import Optional

import torch

from . import _capi as C
from .rope import RotaryPositions

_append = torch.ops.sparse_mlp.kv_append.default
_append_out = torch.ops.sparse_mlp.kv_append.out
_read = torch.ops.sparse_mlp.kv_read.default
_keep = torch.ops.sparse_mlp.kv_keep.default
_DT = {torch.float32: C.F32, torch.float16: C.F16, torch.bfloat16: C.BF16}
_STORE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class KVLayer:
    """One layer of a KVCache: k, v [n_seq, kv_heads, max_len, head_dim] and, for the 8-bit stores, the scales of their rows."""

    def __init__(self, k, v, k_scale, v_scale, dtype):
        self.k, self.v, self.k_scale, self.v_scale, self.dtype = k, v, k_scale, v_scale, dtype

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, *, counts: Optional[torch.Tensor] = None,
               rope: Optional[RotaryPositions] = None, positions: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Writes k, v [n_seq, n_tokens, kv_heads, head_dim] to slots start[b] + t (int64 [n_seq], on the device) for t < counts[b]
        (default: all).  With ``rope`` the keys are rotated on the way, and ``q`` [n_seq, n_tokens, heads, head_dim] as well:
        rotated queries are returned (in ``q_out``, which may be q, or a new tensor; zeros in rows behind counts[b]).
        ``positions`` int64 [n_seq, n_tokens]: of the tokens, default their slots.  Slots outside the cache and rows behind
        counts[b] are left as they were."""
        if rope is not None and rope.head_dim != k.shape[-1]:
            raise RuntimeError(f"kv_append: heads of {k.shape[-1]} values, the rotary plan has {rope.head_dim}")
        plan = (None, False, 1.0) if rope is None else (rope.turns, rope.interleaved, rope.factor)
        args = (self.k, self.v, self.k_scale, self.v_scale, k, v, start, counts, *plan, positions, q)
        return _append(*args) if q_out is None else _append_out(*args, q_out=q_out)

    def read(self, start: Optional[torch.Tensor], n: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [n_seq, kv_heads, n, head_dim] in the model's dtype: what slots start[b] .. start[b] + n - 1 stand for
        (None: from 0); zeros for slots outside the cache."""
        return _read(self.k, self.v, self.k_scale, self.v_scale, _DT[self.dtype], start, n)


class KVCache:
    """Cache of ``layers`` layers for ``n_seq`` sequences of up to ``max_len`` tokens.

    dtype: the model's activations.  store: "same" (rows in dtype), "int8" or "e4m3": codes of 8 bits and one fp32 scale a row
    (a row = one token's key or value of one head), the row's largest magnitude at the end of the codes' range.  Rows that were
    never written read back as zeros.  Memory (k and v): 2 layers n_seq kv_heads max_len (head_dim size + 4 with a scale)."""

    def __init__(self, n_seq: int, kv_heads: int, max_len: int, head_dim: int, *, dtype: torch.dtype = torch.float16, store: str = "same",
                 layers: int = 1, device: torch.device | str = "cuda"):
        if dtype not in _DT:
            raise ValueError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
        if store != "same" and store not in _STORE:
            raise ValueError(f"store must be 'same', 'int8' or 'e4m3', not {store!r}")
        held = _STORE.get(store, dtype)
        shape = (layers, n_seq, kv_heads, max_len, head_dim)
        scale = lambda: torch.zeros(shape[:-1], dtype=torch.float32, device=device) if store != "same" else None
        self._set(torch.zeros(shape, dtype=held, device=device), torch.zeros(shape, dtype=held, device=device), scale(), scale(), dtype)

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None, *, dtype: Optional[torch.dtype] = None) -> "KVCache":
        """A cache over tensors that the caller owns: k, v [layers, n_seq, kv_heads, max_len, head_dim] or without layers, of any
        strides with contiguous heads (the same for k and v); scales likewise, without head_dim.  dtype: the model's
        activations (needed for the 8-bit stores)."""
        dtype = dtype or k.dtype
        if dtype not in _DT:
            raise ValueError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
        if k.dim() not in (4, 5):
            raise ValueError("k must be [n_seq, kv_heads, max_len, head_dim], with or without layers in front")
        if k.dim() == 4:
            k, v, k_scale, v_scale = (None if t is None else t.unsqueeze(0) for t in (k, v, k_scale, v_scale))
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale, dtype)
        return self

    def _set(self, k, v, k_scale, v_scale, dtype):
        self.k, self.v, self.k_scale, self.v_scale, self.dtype = k, v, k_scale, v_scale, dtype
        at = lambda t, i: None if t is None else t[i]
        self._layers = [KVLayer(k[i], v[i], at(k_scale, i), at(v_scale, i), dtype) for i in range(k.shape[0])]

    @property
    def max_len(self) -> int:
        return self.k.shape[3]

    def layer(self, i: int) -> KVLayer:
        return self._layers[i]

    def keep(self, start: torch.Tensor, path: torch.Tensor, counts: torch.Tensor) -> None:
        """In every layer, slot start[b] + i takes the row of slot start[b] + path[b, i] for i < counts[b], as if all rows were
        read first: the accepted nodes of a draft move together behind the sequence."""
        _keep(self.k, self.v, self.k_scale, self.v_scale, _DT[self.dtype], start, path, counts)
