"""Rotary tables and the paged cache's tensors for the attention operators
(_C.rope_kv_write, _C.kv_read, _C.prompt_attention, _C.paged_attention)."""
from __future__ import annotations

import math
import warnings
from typing import Dict, Optional

import torch


def rope_frequencies(rot: int, base: float = 10000.0, scaling: Optional[Dict] = None,
                     length: Optional[int] = None) -> tuple:
    """(float64 [rot / 2] angles per position, factor on cosines and sines).
    `scaling` as in a model's config.json: {"type" or "rope_type": "linear" |
    "ntk" | "dynamic" | "yarn", "factor": f, "original_max_position_embeddings":
    n}.  "ntk" stretches the slowest pair by f at every length, "dynamic" by
    what `length` (default: n) needs beyond the n trained positions."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    kind = None if scaling is None else scaling.get("rope_type", scaling.get("type"))
    if kind in (None, "default"):
        return base ** (-i / rot), 1.0

    def given(key, default=None):  # config files have keys with null
        value = scaling.get(key)
        return default if value is None else value

    if given("factor") is None:
        raise ValueError(f"rope scaling {kind!r} needs a factor")
    f = float(scaling["factor"])
    trained = given("original_max_position_embeddings", given("max_position_embeddings"))
    if kind == "linear":
        return base ** (-i / rot) / f, 1.0
    if kind in ("ntk", "dynamic"):  # the base that stretches the slowest pair (NTK-aware scaling)
        stretch = f
        if kind == "dynamic":
            # by f L / n - (f - 1) for sequences of L tokens: 1 up to the trained n
            if trained is not None:
                stretch = max(1.0, f * (length or 0) / int(trained) - (f - 1))
            elif length is not None:
                raise ValueError("dynamic rope scaling needs original_max_position_embeddings")
            else:
                warnings.warn('dynamic rope scaling without any length is a stretch by the factor: say "ntk"', stacklevel=2)
        return (base * stretch ** (rot / (rot - 2))) ** (-i / rot), 1.0
    if kind == "yarn":
        # YaRN (Peng et al. 2023, section 3): pairs that turn more than beta_fast times over the trained length keep
        # their frequency, those below beta_slow are interpolated, a linear ramp between
        if trained is None:
            raise ValueError("yarn rope scaling needs original_max_position_embeddings")
        attention = given("attention_factor")
        other = [key for key in ("mscale", "mscale_all_dim") if attention is None and given(key) is not None]
        other += ["truncate"] if not given("truncate", True) else []
        if other:
            raise ValueError(f"yarn rope scaling with {', '.join(other)} is not supported")
        n = int(trained)
        freq = base ** (-i / rot)
        low, high = (rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))
                     for turns in (float(given("beta_fast", 32)), float(given("beta_slow", 1))))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        keep = 1 - ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq / f * (1 - keep) + freq * keep, 0.1 * math.log(f) + 1.0 if attention is None else float(attention)
    raise ValueError(f"rope scaling {kind!r} is not one of linear, ntk, dynamic, yarn")


def rope_table(positions: int, rot: int, base: float = 10000.0, scaling: Optional[Dict] = None, device="cuda",
               length: Optional[int] = None):
    """The float32 [positions, rot] table of rope_kv_write: rot / 2 cosines
    then rot / 2 sines per position, computed in 64 bits (an angle's error
    would grow with the position).  With dynamic scaling it is the table of
    sequences of `length` tokens (default: positions)."""
    freq, factor = rope_frequencies(rot, base, scaling, positions if length is None else length)
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
