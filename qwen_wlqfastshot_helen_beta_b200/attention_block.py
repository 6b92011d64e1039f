"""The attention block of a decoder layer, every step of it on this package's
kernels: WLQ qkv projection -> rotary positions with the paged cache's write
-> attention -> WLQ o projection, for whole prompts, for chunks of prompts and
for single tokens.

    python -m qwen_wlqfastshot_helen_beta_b200.attention_block --batch 32 --prompt 1024 --gen 16

runs prompts and decoding steps of a random-initialised block with the 7B
model's shapes and prints one JSON line with the time of both.  A decoding step
can be captured in a CUDA graph and replayed: its shapes are fixed and it
reads positions, slots, lengths and the block table from device memory.
"""
from __future__ import annotations

import argparse
import json
from typing import Callable, Optional, Union

import torch

from . import _C
from .attention import PagedKVCache, rope_table
from .synthetic import SyntheticLayer, ceil_div, make_layer


Linear = Union[SyntheticLayer, Callable[[torch.Tensor], torch.Tensor]]


def _linear(layer: Linear, x: torch.Tensor) -> torch.Tensor:
    """One WLQ linear through the batched torch op (h = A x inside or beside it), or the caller's own."""
    if callable(layer):
        return layer(x)
    out = torch.empty((x.shape[0], layer.N), dtype=x.dtype, device=x.device)
    lut, cols, vals, fmt = layer.operands_for(x.dtype)
    torch.ops.wlq_fastShot.gemm(x, layer.q_packed, lut, out, layer.N, layer.K, 4, layer.words_per_row,
                                layer.chunk_offsets, cols, vals, None, layer.lora_B, layer.dora_gamma,
                                layer.lora_scale, layer.group_size, layer.group_offset, fmt, layer.lora_A_act)
    return out


class AttentionBlock:
    """qkv: a WLQ layer with (heads + 2 kv_heads) * head_size rows, o: one
    with hidden_size rows; both prepacked for the activation type of `cache`,
    or functions of the rows, for layers loaded elsewhere (``lambda x:
    method.apply(layer, x)``).  qkv_bias is added to the qkv rows."""

    def __init__(self, qkv: Linear, o: Linear, heads: int, kv_heads: int, head_size: int, cache: PagedKVCache,
                 cos_sin: torch.Tensor, interleaved: bool = False, qkv_bias: Optional[torch.Tensor] = None):
        self.qkv, self.o, self.cache, self.cos_sin, self.interleaved = qkv, o, cache, cos_sin, interleaved
        self.qkv_bias = qkv_bias
        self.heads, self.kv_heads, self.head_size = heads, kv_heads, head_size

    def _project(self, x, positions, slots, want_k):
        qkv = _linear(self.qkv, x)
        if self.qkv_bias is not None:
            qkv = qkv + self.qkv_bias
        h, kv, d = self.heads, self.kv_heads, self.head_size
        q, k, v = (t.view(x.shape[0], -1, d) for t in qkv.split([h * d, kv * d, kv * d], dim=1))
        k_c, v_c, k_exp, v_exp = self.cache.tensors
        # q and (for attention over the prompt itself) k are rotated in place
        _C.rope_kv_write(q, k, v, positions, self.cos_sin, slots, k_c, v_c, q, k if want_k else None, k_exp, v_exp,
                         self.interleaved)
        return q, k, v

    def _finish(self, out):
        return _linear(self.o, out.view(out.shape[0], -1))

    def prompt(self, x: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
               cu_seqlens: torch.Tensor) -> torch.Tensor:
        """Whole prompts [tokens, hidden], packed: attention over their own k and v, which also go to the cache."""
        q, k, v = self._project(x, positions, slots, True)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        _C.prompt_attention(q, k, v, cu_seqlens, out)
        return self._finish(out)

    def extend(self, x: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, block_table: torch.Tensor,
               kv_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None, max_q: int = 1) -> torch.Tensor:
        """New tokens of sequences that are in the cache already: one each, or chunks (cu_q, max_q)."""
        q, _, _ = self._project(x, positions, slots, False)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_c, v_c, k_exp, v_exp = self.cache.tensors
        _C.paged_attention(q, k_c, v_c, block_table, kv_lens, out, cu_q, max_q, k_exp, v_exp)
        return self._finish(out)


def synthetic_block(hidden: int = 3584, heads: int = 28, kv_heads: int = 4, head_size: int = 128, pages: int = 4096,
                    page_size: int = 16, bits: int = 8, dtype: torch.dtype = torch.bfloat16, max_position: int = 32768,
                    group_size: int = 128, seed: int = 0) -> AttentionBlock:
    """A random-initialised block; the defaults are the 7B model's shapes."""
    qkv = make_layer((heads + 2 * kv_heads) * head_size, hidden, group_size=group_size, seed=seed).prepack(dtype)
    o = make_layer(hidden, heads * head_size, group_size=group_size, seed=seed + 1).prepack(dtype)
    return AttentionBlock(qkv, o, heads, kv_heads, head_size,
                          PagedKVCache(pages, kv_heads, head_size, page_size, bits, dtype),
                          rope_table(max_position, head_size, 1e6))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=1024)
    ap.add_argument("--gen", type=int, default=16, help="decoding steps")
    ap.add_argument("--bits", type=int, default=8, choices=(8, 16), help="bits per cached value")
    a = ap.parse_args(argv)
    dev, page = torch.device("cuda"), 16
    per = ceil_div(a.prompt + a.gen + 1, page)
    block = synthetic_block(pages=a.batch * per, page_size=page, bits=a.bits, max_position=max(32768, per * page))
    table = torch.arange(a.batch * per, dtype=torch.int32, device=dev).view(a.batch, per)
    seq = torch.arange(a.batch, device=dev)

    def slots_of(s, pos):
        return table[s, pos // page].long() * page + pos % page

    pos = torch.arange(a.prompt, device=dev).repeat(a.batch)
    slots = slots_of(seq.repeat_interleave(a.prompt), pos)
    cu = (torch.arange(a.batch + 1, device=dev) * a.prompt).to(torch.int32)
    x = torch.randn(a.batch * a.prompt, block.qkv.K, device=dev).bfloat16()
    times = []
    for _ in range(3):
        t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        t0.record()
        block.prompt(x, pos, slots, cu)
        t1.record()
        torch.cuda.synchronize()
        times.append(t0.elapsed_time(t1))

    step_x = torch.randn(a.batch, block.qkv.K, device=dev).bfloat16()
    step_pos = torch.full((a.batch,), a.prompt, device=dev)
    step_slots, lens = slots_of(seq, step_pos), torch.full((a.batch,), a.prompt + 1, dtype=torch.int32, device=dev)
    block.extend(step_x, step_pos, step_slots, table, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.extend(step_x, step_pos, step_slots, table, lens)
    t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    t0.record()
    for _ in range(a.gen):
        graph.replay()
        step_x.copy_(y)
        step_pos += 1
        lens += 1
        step_slots.copy_(slots_of(seq, step_pos))
    t1.record()
    torch.cuda.synchronize()
    print(json.dumps({"metric": "attention block (WLQ qkv, rope + cache write, attention, WLQ o)",
                      "prompt_ms": round(min(times), 4), "step_us": round(1e3 * t0.elapsed_time(t1) / a.gen, 2),
                      "finite": bool(torch.isfinite(y.float()).all()),
                      "config": {"hidden": block.qkv.K, "heads": block.heads, "kv_heads": block.kv_heads,
                                 "batch": a.batch, "prompt": a.prompt, "gen": a.gen, "cache_bits": a.bits,
                                 "dtype": "bf16", "data": "synthetic"}}))


if __name__ == "__main__":
    main()
