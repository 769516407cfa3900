"""Llama engines over the 8-bit paged KV cache (``ops.kv8``): half the cache bytes per token.

Everything but the cache is the base engine's: the same graphs, page pool, drafter and target run on
top.  K and V are rounded to e4m3 as they are appended, with one power-of-two scale per page, side and
head, and every later read (decode, tree verify, causal prefill, copy-on-write, compaction) works on
the codes.  With folded norms the QKV product comes out in fp32 and is rotated and rounded by the
append in one pass, so a key is rounded once.

On CUDA the kernels need head dimension 128 and pages of 8, 16, 32 or 64 slots.
"""

from __future__ import annotations

import torch

from ..ops import kv8
from .engine import LlamaEngine
from .engine_fp8 import Fp8LlamaEngine

KV_CACHES = ("model", "fp8")


def kv8_bytes_per_token(cfg, page_size: int) -> float:
    """Cache bytes per token: one code per element and four scale bytes per page, side and head."""
    return cfg.num_layers * 2 * cfg.num_kv_heads * (cfg.head_dim + 4 / page_size)


class _Kv8Cache:
    """The cache hooks of ``LlamaEngine`` on the 8-bit operators."""

    def _new_cache(self):
        c = self.cfg
        if self.device.type == "cuda" and (c.head_dim != 128 or self.page_size not in (8, 16, 32, 64)):
            raise ValueError("the 8-bit KV cache kernels need head dimension 128 and pages of 8, 16, 32 or 64 slots, "
                             f"not {c.head_dim} and {self.page_size}")
        return kv8.empty_cache(c.num_layers, self.num_pages, c.num_kv_heads, self.page_size, c.head_dim,
                               device=self.device)

    def _reserve_workspace(self, max_positions: int) -> None:
        """The 8-bit operators allocate per call."""

    def _append(self, qkv, li, positions, slots):
        c = self.cfg
        return self.ops.rope_qkv_append8(qkv, self.rope, positions, slots, self.kv[li], c.num_heads, c.num_kv_heads,
                                         out_dtype=self.dtype)

    def _append_normed(self, hb, wqkv, ss, li, positions, slots):
        return self._append(self.ops.lm_head_norm(hb, wqkv, ss, self.cfg.rms_eps), li, positions, slots)

    def _attend(self, q, li, desc, causal_start):
        if causal_start is None:
            return self.ops.attention8(q, self.kv[li], desc, self.scale)
        return self.ops.attention8_causal(q, self.kv[li], desc, causal_start, self.scale)

    def _copy_plan(self, plan: torch.Tensor) -> None:
        self.ops.kv8_copy_pages(self.kv, plan)

    def _copy_plan_counted(self, plan: torch.Tensor, count: torch.Tensor) -> None:
        self.ops.kv8_copy_pages_counted(self.kv, plan, count)

    def _move(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        self.ops.kv8_move_slots(self.kv, src, dst)

    def read_pages(self, pages: torch.Tensor) -> torch.Tensor:
        return self.ops.kv8_read_pages(self.kv, pages.to(self.device), self.dtype)


class Kv8LlamaEngine(_Kv8Cache, LlamaEngine):
    """16-bit weights (fp32 on CPU), 8-bit cache."""


class Kv8Fp8LlamaEngine(_Kv8Cache, Fp8LlamaEngine):
    """Block-scaled fp8 weights, 8-bit cache."""


def make_engine(weights, *, kv_cache: str = "model", **kw) -> LlamaEngine:
    """The engine of 16-bit ``weights`` with the cache in their dtype (``model``) or in 8 bits (``fp8``)."""
    if kv_cache not in KV_CACHES:
        raise ValueError(f"unknown KV cache {kv_cache!r} (choose {' or '.join(KV_CACHES)})")
    return (Kv8LlamaEngine if kv_cache == "fp8" else LlamaEngine)(weights, **kw)
