"""The 8-bit paged KV cache: layout, scales, and what its operators mean.

``data [layers, pages, 2 (k, v), kv_heads, page_size, head_dim]`` holds e4m3 codes and
``scale [layers, pages, 2, kv_heads]`` one fp32 power of two per page, side and head; an element
stands for code * scale.  A scale of 0 marks a page that holds nothing (its codes are zero); the
codes are finite (no NaN code is ever written).

The scale a row needs is 2^e with the smallest e in [``EXP_MIN``, ``EXP_MAX``] for which its largest
magnitude is at most 448 * 2^e.  Rows are written to slots by two operators, appends and moves, with
one rule: the scale of a page becomes the largest its new rows need, or stays if it was larger, and
the page's other slots are rounded again when it grew; writing slot 0 starts the page anew (scale of
the new rows alone, other slots zero).  Where rows name the same slot the later row is kept.
Powers of two make all of it exact but the one rounding to e4m3 (4 significant bits; an element
below scale / 64 keeps fewer).

Pages therefore fill from slot 0, which is how every path of the runtime fills them, and a page that
returns to the pool needs no clearing: its next owner's first token starts it anew.

The same operators exist in ``ops.torch_ops`` (any device, any head dimension; they raise where a
row cannot be stored) and as kernels in ``ops.cuda_ops.CudaOps`` (head dimension 128, pages of 8 to 64
slots; they report through the device error flag and leave that row out).  A row left out writes no slot:
its page does not start anew for it, and where it repeated a slot the earlier row is not stored either.
Indices may be int32 or int64.

Attention holds the rows of q as fp16 after a power of two is taken out of each (elements below 2^-24 of a
row's largest are lost) and rounds the weights of V's codes (softmax weight times the page's v scale) to
fp16: 11 bits down to 2^-21 of the row's largest, fewer below, none under 2^-32 of it.  Statistics, sums
and accumulators are fp32, the output is rounded once.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

E4M3_MAX = 448.0
EXP_MIN, EXP_MAX = -40, 56


@dataclass
class Kv8Cache:
    data: torch.Tensor
    scale: torch.Tensor

    def layer(self, index: int) -> "Kv8Layer":
        return Kv8Layer(self, index)

    def __getitem__(self, index: int) -> Kv8Layer:
        return self.layer(index)


@dataclass
class Kv8Layer:
    """One layer of a cache (a name for it: the kernels take the cache and the index, so no view is made per call)."""

    cache: Kv8Cache
    index: int

    def __post_init__(self) -> None:
        if not 0 <= self.index < self.cache.data.shape[0]:
            raise IndexError(f"layer {self.index} of a cache of {self.cache.data.shape[0]}")

    @property
    def data(self) -> torch.Tensor:
        """[pages, 2, kv_heads, page_size, head_dim]"""
        return self.cache.data[self.index]

    @property
    def scale(self) -> torch.Tensor:
        """[pages, 2, kv_heads]"""
        return self.cache.scale[self.index]

    def values(self) -> torch.Tensor:
        """Every element in fp32."""
        return self.data.float() * self.scale[..., None, None]


def empty_cache(layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int, device=None) -> Kv8Cache:
    """A cache whose pages all hold nothing."""
    shape = (int(layers), int(pages), 2, int(kv_heads))
    data = torch.zeros((*shape, int(page_size), int(head_dim)), dtype=torch.uint8, device=device)
    return Kv8Cache(data.view(torch.float8_e4m3fn), torch.zeros(shape, dtype=torch.float32, device=device))


def pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e for whole e in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def needed_scale(amax: torch.Tensor) -> torch.Tensor:
    """The scale for largest magnitudes ``amax`` (fp32, finite); raises where one is too large."""
    mant, ex = torch.frexp(amax)  # 448 = 0.875 * 2^9
    e = torch.where(mant <= 0.875, ex - 9, ex - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, EXP_MIN)).clamp_min(EXP_MIN)
    if not bool(torch.isfinite(amax).all()) or bool((e > EXP_MAX).any()):
        raise ValueError("the 8-bit KV cache holds finite values up to 448 * 2^56 only")
    return pow2(e)


def encode(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp32 ``x`` as codes of ``scale`` (0 where the scale is 0)."""
    y = torch.where(scale > 0, x / scale, torch.zeros((), device=x.device))
    return y.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def write_rows(data: torch.Tensor, scale: torch.Tensor, rows: torch.Tensor, need: torch.Tensor,
               slots: torch.Tensor) -> None:
    """Write fp32 ``rows [n, layers, 2, kv_heads, hd]`` with needed scales ``need [n, layers, 2, kv_heads]`` at
    ``slots`` of a whole cache's tensors, by the rule above."""
    ps, pages = data.shape[-2], data.shape[1]
    last: dict[int, dict[int, int]] = {}
    for i, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pages * ps:
            raise IndexError(f"slot {slot} is outside the cache of {pages} pages of {ps} slots")
        last.setdefault(slot // ps, {})[slot % ps] = i
    for page, owners in last.items():
        idx = torch.tensor(list(owners.values()), device=data.device)
        offs = torch.tensor(list(owners.keys()), device=data.device)
        old = scale[:, page]
        new = need[idx].amax(0)
        held = data[:, page].float() * old[..., None, None]  # [layers, 2, kv_heads, ps, hd]
        if 0 in owners:
            held = torch.zeros_like(held)
        else:
            new = torch.maximum(new, old)
        held[:, :, :, offs] = rows[idx].permute(1, 2, 3, 0, 4)
        data[:, page] = encode(held, new[..., None, None])
        scale[:, page] = new
