"""Rotary positions: half and interleaved layouts, part of the head, scaled for long contexts.

The reference takes rotary embeddings from transformers (src/models/llama/modelling_llama_skip.py); here the angle of a pair is
formed inside the kernel, in fp64, so there is no table and no largest position.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

# What a scaling must and may say.  original_max_position_embeddings does not matter to linear and ntk, which configurations give it all the same.
_NEEDS = {"none": (), "linear": ("factor",), "ntk": ("factor",),
          "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
          "yarn": ("factor", "original_max_position_embeddings")}
_MAY = {"linear": ("original_max_position_embeddings",), "ntk": ("original_max_position_embeddings",),
        "yarn": ("beta_fast", "beta_slow", "attention_factor")}

_rope = torch.ops.sparse_mlp.rope.default
_rope_out = torch.ops.sparse_mlp.rope.out


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None) -> tuple[list[float], float]:
    """(radians per position of each of the rotary_dim / 2 pairs, factor of the result).

    Unscaled: theta^(-2 i / rotary_dim).  ``scaling`` has a ``rope_type`` and a ``factor``, and as transformers names them:
      linear   every frequency / factor
      ntk      theta * factor^(d / (d - 2)): the slowest pair is slowed by factor, the fastest left alone
      llama3   pairs that turn less than low_freq_factor times within original_max_position_embeddings are slowed by factor,
               those that turn more than high_freq_factor times are left alone, between them a linear blend
      yarn     the same idea, blended linearly over the pair's index between the pairs that turn beta_fast (32) and beta_slow (1)
               times; the result is multiplied by attention_factor (default 0.1 ln(factor) + 1)
    A key that is not known to the rope_type (yarn's mscale, mscale_all_dim and truncate=False among them) is an error: it would
    mean another rotation than this one."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, not {rotary_dim}")
    if not theta > 0:
        raise ValueError(f"theta must be positive, not {theta}")
    scaling = dict(scaling or {})
    kind = scaling.pop("rope_type", scaling.pop("type", "none"))
    scaling.pop("type", None)
    kind = "none" if kind == "default" else kind
    if kind not in _NEEDS:
        raise ValueError(f"unknown rope_type {kind!r} (linear, ntk, llama3, yarn)")
    if kind == "yarn" and scaling.get("truncate") is True:  # the default
        del scaling["truncate"]
    for key in _NEEDS[kind]:
        if scaling.get(key) is None:
            raise ValueError(f"rope_type {kind!r} needs {key}")
    for key in scaling:
        if key not in _NEEDS[kind] + _MAY.get(kind, ()):
            raise ValueError(f"rope_type {kind!r} does not know {key}")
    factor = float(scaling.get("factor", 1.0))
    if not factor > 0:
        raise ValueError(f"factor must be positive, not {factor}")
    if kind == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    w = [theta ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind in ("none", "ntk"):
        return w, 1.0
    if kind == "linear":
        return [x / factor for x in w], 1.0
    orig = float(scaling["original_max_position_embeddings"])
    if not orig > 0:
        raise ValueError(f"original_max_position_embeddings must be positive, not {orig}")
    if kind == "llama3":
        lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not hi > lo:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        keep = [min(1.0, max(0.0, (orig * x / (2 * math.pi) - lo) / (hi - lo))) for x in w]
        return [x * (k + (1.0 - k) / factor) for x, k in zip(w, keep)], 1.0
    if not theta > 1:
        raise ValueError(f"rope_type 'yarn' needs theta above 1, not {theta}")
    index = lambda turns: rotary_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
    lo = max(math.floor(index(float(scaling.get("beta_fast") or 32.0))), 0)
    hi = min(math.ceil(index(float(scaling.get("beta_slow") or 1.0))), rotary_dim - 1)
    slow = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(rotary_dim // 2)]
    given = scaling.get("attention_factor")
    return ([x * (1.0 - s + s / factor) for x, s in zip(w, slow)],
            float(given) if given is not None else (0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0))


class _Rotate(torch.autograd.Function):
    """The rotation is linear: its gradient is the transposed rotation."""

    @staticmethod
    def forward(ctx, x, positions, plan, inverse):
        ctx.save_for_backward(positions)  # often a counter that the caller advances in place: autograd refuses it then
        ctx.plan, ctx.inverse = plan, inverse
        with torch.no_grad():
            return _rope(x, positions, plan.turns, plan.interleaved, plan.factor, inverse)

    @staticmethod
    def backward(ctx, g):
        (positions,) = ctx.saved_tensors
        g = g if g.stride(-1) == 1 else g.contiguous()
        return _Rotate.apply(g, positions, ctx.plan, not ctx.inverse), None, None, None


class RotaryPositions:
    """The rotary plan of a model: which values of a head form pairs and how fast each pair turns.

    head_dim: values of a head; rotary_dim: how many of the first ones are rotated (default all); layout: "half" (pairs
    (i, i + rotary_dim / 2)) or "interleaved" (pairs (2 i, 2 i + 1)); theta, scaling: see rotary_frequencies."""

    def __init__(self, head_dim: int, *, rotary_dim: Optional[int] = None, theta: float = 10000.0, layout: str = "half",
                 scaling: Optional[dict] = None, device: torch.device | str = "cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if not 0 < self.rotary_dim <= self.head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} of a head of {head_dim}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be 'half' or 'interleaved', not {layout!r}")
        self.interleaved = layout == "interleaved"
        self.frequencies, self.factor = rotary_frequencies(self.rotary_dim, theta, scaling)
        self.turns = torch.tensor([w / (2 * math.pi) for w in self.frequencies], dtype=torch.float64, device=device)

    def rotate(self, x: torch.Tensor, positions: torch.Tensor, *, inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [n, heads, head_dim] or [n_seq, n_tokens, heads, head_dim] (any strides with contiguous heads), positions int64
        x.shape[:-2] -> the rotated tensor (``out``, which may be x, or a new one).  ``inverse`` applies the transposed map:
        turned back and multiplied by the same factor.  Differentiable in x without ``out``."""
        if x.shape[-1] != self.head_dim:
            raise RuntimeError(f"rope: heads of {x.shape[-1]} values, the plan has {self.head_dim}")
        if x.requires_grad and torch.is_grad_enabled() and out is None:
            return _Rotate.apply(x, positions, self, inverse)
        if out is None:
            return _rope(x, positions, self.turns, self.interleaved, self.factor, inverse)
        return _rope_out(x, positions, self.turns, self.interleaved, self.factor, inverse, out=out)

    def tables(self, max_len: int) -> tuple[torch.Tensor, torch.Tensor]:
        """cos and sin [max_len, head_dim] in fp32 for stx_attn_decode, which rotates whole heads in the half layout."""
        if self.interleaved or self.rotary_dim != self.head_dim:
            raise ValueError("tables serve the half layout over the whole head")
        a = torch.arange(max_len, dtype=torch.float64, device=self.turns.device)[:, None] * self.turns
        a = 2 * math.pi * (a - a.round())
        a = torch.cat([a, a], dim=-1)
        return (a.cos() * self.factor).float(), (a.sin() * self.factor).float()
