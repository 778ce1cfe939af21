"""Qwen3's attention core with the q/k prologue on the MI355X kernels.

``Qwen3AttentionCore`` is ``Qwen3Attention.forward`` between the fused qkv
projection and ``o_proj`` (qwen_asr_vllm/models/qwen3.py:42-50): per-head
RMSNorm of q and k, rotary embedding at the tokens' positions, then paged
attention with the KV store.  It subclasses :class:`PagedAttention`, so the
model runner binds its cache slices the same way
(engine/model_runner.py:129-131).

* Decode batches (one query per sequence, cache bound) run in ONE launch: the
  paged decode kernel normalises and rotates q and the new key in registers,
  writes the new K/V row and attends (reference: q_norm, k_norm, rotary,
  store_kvcache and attention as separate launches).
* Other batches run the standalone prologue kernel over q and k, then the
  varlen path of :class:`PagedAttention`.  With ``varlen_fuse_prologue``
  set (off by default: faster for large prompt batches alone), prefill batches with
  head_dim 128 and a 16-bit pool or none run the standalone kernel over the
  keys alone, and the varlen launch normalises and rotates the queries
  itself, in registers, at each item's first key tile.

Without a cache (packed sequences, a training pass) the core is differentiable in
q, k, v and the norm weights.

The norm weights and the rotary table mirror the reference modules: weights
``q_norm.weight`` / ``k_norm.weight`` of shape [head_dim]
(layers/layernorm.py:16-17), and the fp32 cos|sin table built on the host by
the reference formula (layers/rotary_embedding.py:18-26).
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import nn

from voiceagent_amd import ops
from voiceagent_amd.layers.attention import PagedAttention


@dataclass(frozen=True)
class RotaryScaling:
    """How a rotary table is stretched for contexts ``factor`` times those it was
    trained on.

    * ``"linear"``: every frequency divided by ``factor``.
    * ``"base"``: the base raised to base * factor^(r / (r - 2)), r the rotated
      elements: the fastest pair keeps its frequency, the slowest is divided by
      ``factor``.
    * ``"yarn"`` (Peng et al., 2023): frequencies that turn at least
      ``beta_fast`` times over ``original_max_position`` stay, those that turn
      ``beta_slow`` times or fewer are divided by ``factor``, with a linear ramp
      between, over the pairs' indices (the paper states one over the turns;
      checkpoints' tables have this one); cosines and sines times
      ``attention_factor`` (0.1 ln factor + 1 if not given)."""

    kind: str
    factor: float
    original_max_position: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None


def _scaled_frequencies(rotary_dim: int, base: float,
                        scaling: RotaryScaling | None) -> tuple[torch.Tensor, float]:
    """(frequencies [r / 2] in float64, factor of the table's entries)."""
    index = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling is not None and scaling.factor < 1.0:
        raise ValueError(f"a rotary scaling's factor must be at least 1, got {scaling.factor}")
    if scaling is not None and scaling.kind == "base":
        if rotary_dim <= 2:
            raise ValueError("scaling by the base needs more than one pair")
        base = base * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-2.0 * index / rotary_dim)
    if scaling is None or scaling.kind == "base":
        return freq, 1.0
    if scaling.kind == "linear":
        return freq / scaling.factor, 1.0
    if scaling.kind != "yarn":
        raise ValueError(f"unknown rotary scaling {scaling.kind!r} (linear, base or yarn)")
    if scaling.original_max_position <= 0:
        raise ValueError("yarn scaling needs original_max_position")

    def pair_of(turns: float) -> float:  # the pair that turns so often over the context
        return (rotary_dim * math.log(scaling.original_max_position / (2 * math.pi * turns))
                / (2 * math.log(base)))

    low = max(math.floor(pair_of(scaling.beta_fast)), 0)
    high = min(math.ceil(pair_of(scaling.beta_slow)), rotary_dim - 1)
    ramp = ((index - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    factor = scaling.attention_factor
    if factor is None:
        factor = 0.1 * math.log(scaling.factor) + 1.0
    return freq * (1.0 - ramp) + freq / scaling.factor * ramp, factor


def rotary_cos_sin_cache(head_dim: int, max_position: int, base: float, *,
                         rotary_dim: int | None = None,
                         scaling: RotaryScaling | None = None) -> torch.Tensor:
    """[max_position, head_dim] fp32 = cos | sin of position x inv_freq
    (RotaryEmbedding.__init__, layers/rotary_embedding.py:18-26).

    ``rotary_dim`` (a part of the head: the table's width) or ``scaling`` given:
    the angles are formed in float64, as those of far positions need (fp32
    angles, the reference's, are off by up to 1e-3 at 32768)."""
    if rotary_dim is not None or scaling is not None:
        width = head_dim if rotary_dim is None else rotary_dim
        if not 0 < width <= head_dim or width % 2:
            raise ValueError(f"rotary_dim {width} must be even and within head_dim {head_dim}")
        freq, factor = _scaled_frequencies(width, float(base), scaling)
        angles = torch.outer(torch.arange(max_position, dtype=torch.float64), freq)
        return (torch.cat((angles.cos(), angles.sin()), dim=-1) * factor).float()
    inv_freq = 1.0 / (base ** (torch.arange(0, head_dim, 2, dtype=torch.float) / head_dim))
    positions = torch.arange(max_position, dtype=torch.float)
    freqs = torch.outer(positions, inv_freq)
    return torch.cat((freqs.cos(), freqs.sin()), dim=-1)


class Qwen3AttentionCore(PagedAttention):
    fuse_prologue = True

    def __init__(self, num_heads: int, head_dim: int, num_kv_heads: int, *, eps: float = 1e-6,
                 max_position: int = 32768, rope_theta: float = 1_000_000.0,
                 rope_scaling: RotaryScaling | None = None):
        super().__init__(num_heads, head_dim, head_dim ** -0.5, num_kv_heads)
        self.eps = eps
        self.q_norm_weight = nn.Parameter(torch.ones(head_dim))
        self.k_norm_weight = nn.Parameter(torch.ones(head_dim))
        self.register_buffer("cos_sin_cache",
                             rotary_cos_sin_cache(head_dim, max_position, rope_theta,
                                                  scaling=rope_scaling),
                             persistent=False)

    def prologue(self, positions: torch.Tensor) -> ops.QKPrologue:
        return ops.QKPrologue(self.q_norm_weight, self.k_norm_weight, self.eps,
                              self.cos_sin_cache, positions)

    def forward(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                v: torch.Tensor) -> torch.Tensor:
        """positions [T] (int64), q [T, Hq, D], k/v [T, Hkv, D]: raw projections."""
        pro = self.prologue(positions)
        if self.fuse_prologue:
            # (a decode step in one launch; prefill batches as varlen_fuse_prologue says)
            return super().forward(q, k, v, prologue=pro)
        # (Over a cache nothing has a gradient, whatever the weights ask for.)
        with torch.set_grad_enabled(torch.is_grad_enabled() and not self.k_cache.numel()):
            qn, kn = ops.qk_norm_rope(q, k, pro)
        return super().forward(qn, kn, v)
