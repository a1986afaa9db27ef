"""Rotary position embeddings with linear position-interpolation scaling.

Reference: megatron/model/positional_embeddings.py:7-51 (complex-multiply RoPE
in fp32; scaling divides positions by rope_scaling_factor). We precompute
cos/sin tables (fp32) once and keep them resident in HBM; the per-layer
application is a fused HIP kernel (ops/csrc/rope.hip) over interleaved pairs.
"""

from __future__ import annotations

import math
import weakref
from typing import Optional

import torch

from ..ops import functional as ops_f


def precompute_freqs(dim: int, end: int, theta: float = 10000.0,
                     scaling_factor: float = 1.0, device=None):
    """cos/sin tables (end, dim/2) fp32."""
    freqs = 1.0 / (
        theta ** (torch.arange(0, dim, 2, device=device)[: dim // 2].float() / dim)
    )
    t = torch.arange(end, device=device).float() / scaling_factor
    angles = torch.outer(t, freqs)  # (end, dim/2)
    return torch.cos(angles), torch.sin(angles)


ROPE_SCALING_TYPES = ("linear", "ntk", "yarn")


def precompute_rotary_tables(dim: int, end: int, theta: float = 10000.0,
                             scaling_type: str = "linear",
                             scaling_factor: float = 1.0,
                             original_max_position: int = 2048, device=None):
    """cos/sin tables (end, dim/2) fp32 for ops.rotary_embedding, with the
    frequencies of a context `scaling_factor` times the trained one.

    Angles are taken in 64 bits, so that far positions keep their phase (in
    32 bits position 100000 would be off by up to 0.004).
      linear: positions are divided by the factor.
      ntk:    the base becomes theta * factor^(dim / (dim - 2)): the slowest
              pair is interpolated by the factor, the fastest one kept.
      yarn:   pairs that turn more than 32 times over the trained
              `original_max_position` are kept, those that turn less than once
              are interpolated, with a linear ramp over the pairs between; cos
              and sin carry the factor 0.1 ln(scaling_factor) + 1."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary dim must be even and positive, not {dim}")
    if scaling_type not in ROPE_SCALING_TYPES:
        raise ValueError(f"scaling_type must be one of {ROPE_SCALING_TYPES}")
    if scaling_factor <= 0 or (scaling_type != "linear" and
                               scaling_factor < 1):
        raise ValueError("scaling_factor must be positive, and 1 or more for "
                         "ntk and yarn")
    if theta <= 1 or end < 1 or original_max_position < 1:
        raise ValueError("theta must exceed 1, lengths must be positive")
    if scaling_type == "ntk" and dim > 2:
        theta = theta * scaling_factor ** (dim / (dim - 2))
    inv = theta ** -(torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    magnitude = 1.0
    if scaling_type == "linear":
        inv = inv / scaling_factor
    elif scaling_type == "yarn" and scaling_factor > 1:
        def pair_of(turns):  # the pair that turns so often
            return (dim * math.log(original_max_position
                                   / (turns * 2 * math.pi))
                    / (2 * math.log(theta)))

        low = max(math.floor(pair_of(32.0)), 0)
        high = min(math.ceil(pair_of(1.0)), dim - 1)
        ramp = (torch.arange(dim // 2, dtype=torch.float64) - low) / max(
            high - low, 0.001)
        ramp = ramp.clamp(0.0, 1.0)
        inv = inv / scaling_factor * ramp + inv * (1 - ramp)
        magnitude = 0.1 * math.log(scaling_factor) + 1.0
    inv = inv.to(device=device)
    angles = torch.outer(
        torch.arange(end, dtype=torch.float64, device=inv.device), inv)
    return (angles.cos() * magnitude).float(), (angles.sin()
                                                * magnitude).float()


class RotaryTables:
    """cos and sin of precompute_rotary_tables, one pair for all layers that
    ask for the same: at 131072 positions of 64 pairs a pair is 64 MB. It is
    gone with the last layer that holds it."""

    _held = weakref.WeakValueDictionary()  # by settings and device

    def __init__(self, settings, device):
        # a layer that trains may come after one that ran in inference mode
        with torch.inference_mode(False):
            self.cos, self.sin = precompute_rotary_tables(
                device=device, **settings)
        if self.cos.is_cuda:  # layers on other streams may be next
            torch.cuda.current_stream(self.cos.device).synchronize()

    @classmethod
    def of(cls, device, **settings):
        key = (str(device), *sorted(settings.items()))
        tables = cls._held.get(key)
        if tables is None:
            tables = cls._held[key] = cls(settings, device)
        return tables


def apply_rotary_emb(query: torch.Tensor, key: torch.Tensor,
                     cos: torch.Tensor, sin: torch.Tensor,
                     position_ids: Optional[torch.Tensor] = None):
    """query (s, b, np, hn), key (s, b, nkv, hn). cos/sin tables indexed by
    absolute position; position_ids (b, s) selects rows for inference with
    KV-cache offsets."""
    if position_ids is None:
        s = query.shape[0]
        c, sn = cos[:s], sin[:s]
        q = ops_f.apply_rope(query, c, sn)
        k = ops_f.apply_rope(key, c, sn)
    else:
        # gather per-position tables: (s, b, hn/2) — inference path, small s
        c = cos[position_ids].transpose(0, 1)  # (s, b, dim/2)
        sn = sin[position_ids].transpose(0, 1)
        q = _apply_rope_positional(query, c, sn)
        k = _apply_rope_positional(key, c, sn)
    return q, k


def _apply_rope_positional(x, cos, sin):
    xf = x.float()
    x1 = xf[..., 0::2]
    x2 = xf[..., 1::2]
    c = cos.unsqueeze(2)  # (s, b, 1, hn/2)
    s = sin.unsqueeze(2)
    o1 = x1 * c - x2 * s
    o2 = x2 * c + x1 * s
    return torch.stack([o1, o2], dim=-1).flatten(-2).to(x.dtype)
