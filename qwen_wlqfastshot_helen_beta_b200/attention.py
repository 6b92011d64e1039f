"""Rotary tables and the paged cache's tensors for the attention operators
(_C.rope_kv_write, _C.kv_read, _C.prompt_attention, _C.paged_attention)."""
from __future__ import annotations

import math
from typing import Dict, Optional

import torch


def rope_frequencies(rot: int, base: float = 10000.0, scaling: Optional[Dict] = None) -> tuple:
    """(float64 [rot / 2] angles per position, factor on cosines and sines).
    `scaling` as in a model's config.json: {"type" or "rope_type": "linear" |
    "dynamic" | "yarn", "factor": f, "original_max_position_embeddings": n}."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    kind = None if scaling is None else scaling.get("rope_type", scaling.get("type"))
    if kind in (None, "default"):
        return base ** (-i / rot), 1.0
    f = float(scaling["factor"])
    if kind == "linear":
        return base ** (-i / rot) / f, 1.0
    if kind == "dynamic":  # the base that stretches the slowest pair by the factor (NTK-aware scaling)
        return (base * f ** (rot / (rot - 2))) ** (-i / rot), 1.0
    if kind == "yarn":
        # YaRN (Peng et al. 2023, section 3): pairs that turn more than beta_fast times over the trained length keep
        # their frequency, those below beta_slow are interpolated, a linear ramp between
        n = int(scaling["original_max_position_embeddings"])
        freq = base ** (-i / rot)
        low, high = (rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))
                     for turns in (float(scaling.get("beta_fast", 32)), float(scaling.get("beta_slow", 1))))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        keep = 1 - ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq / f * (1 - keep) + freq * keep, float(scaling.get("attention_factor", 0.1 * math.log(f) + 1.0))
    raise ValueError(f"rope scaling {kind!r} is not one of linear, dynamic, yarn")


def rope_table(positions: int, rot: int, base: float = 10000.0, scaling: Optional[Dict] = None, device="cuda"):
    """The float32 [positions, rot] table of rope_kv_write: rot / 2 cosines
    then rot / 2 sines per position, computed in 64 bits (an angle's error
    would grow with the position)."""
    freq, factor = rope_frequencies(rot, base, scaling)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return (torch.cat((angle.cos(), angle.sin()), 1) * factor).float()


class PagedKVCache:
    """The k and v pages of one attention layer.  bits 16 holds values of
    `dtype`; bits 8 e4m3 codes and, per row, the exponent of their scale.
    ``cache.tensors`` is (k_cache, v_cache, k_exp, v_exp), the last two None
    with 16 bits."""

    def __init__(self, num_pages: int, num_kv_heads: int, head_size: int, page_size: int = 16, bits: int = 8,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if bits not in (8, 16):
            raise ValueError(f"a cache has 8 or 16 bits per value, not {bits}")
        shape = (int(num_pages), int(num_kv_heads), int(page_size), int(head_size))
        stored = dtype if bits == 16 else torch.float8_e4m3fn
        self.dtype, self.page_size, self.bits = dtype, int(page_size), bits
        self.k, self.v = (torch.zeros(shape, dtype=stored, device=device) for _ in range(2))
        self.k_exp = self.v_exp = None
        if bits == 8:
            self.k_exp, self.v_exp = (torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2))

    @property
    def tensors(self):
        return self.k, self.v, self.k_exp, self.v_exp

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tensors if t is not None)
