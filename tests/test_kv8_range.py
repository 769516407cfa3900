"""Attention over the 8-bit KV cache at the ends of what its inputs may be: factors outside fp32, light weights, large
scores.  Every case runs through the register pass, the tcgen05 pass with keys split over its slots, and the tcgen05
pass with 256 rows (and the PyTorch form)."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import mod
from test_kv8 import Oracle, check_attention, impl, make_cache, settle

# (device, rows, q heads, kv heads): query rows of a kv head decide the pass once the launch is sized for 2^20 keys
PASSES = [pytest.param("cpu", 3, 4, 1, id="cpu")] + [
    pytest.param("cuda", rows, hq, hkv, id=name, marks=pytest.mark.gpu)
    for name, rows, hq, hkv in (("registers16", 3, 4, 1), ("registers32", 7, 4, 1), ("split-keys", 12, 8, 1),
                                ("rows256", 40, 4, 1))]


def mask_desc(device, rows, length, words, pages):
    """Rows see the marked keys of one page list (bit x of their words for position x)."""
    zero = torch.zeros(rows, dtype=torch.int32, device=device)
    desc = mod("ops.attn_desc").AttnDesc(
        prefix_pages=pages.int().to(device), n_shared_pages=pages.numel(), shared_len=0, mask_base=0, row_full=zero,
        row_len=torch.full_like(zero, length), row_mask=words.to(device), tail_pages=zero[:, None])
    desc._max_keys = 1 << 20
    return desc


def fill(cache, layer, page, side, head, values):
    """One page, side and head set to ``values`` [ps, hd] (fp32)."""
    kv8 = mod("ops.kv8")
    s = kv8.needed_scale(values.abs().max())
    cache.data[layer, page, side, head] = kv8.encode(values, s).to(cache.data.device)
    cache.scale[layer, page, side, head] = s


# --------------------------------------------------------- factors and masks
@pytest.mark.parametrize("device,rows,hq,hkv", PASSES)
@pytest.mark.parametrize("size,scale", [(2.0 ** -120, 128 ** -0.5), (1.0, 1e-37), (1.0, 1e-46), (2.0 ** -120, 1e-30)],
                         ids=["queries", "scale", "zero", "both"])
def test_a_hidden_key_under_a_factor_that_underflows(device, rows, hq, hkv, size, scale):
    """Zero keys (page scale 2^-40) that some rows do not see: every seen key counts the same."""
    ops = impl(device)
    cache = make_cache(device, 1, 9, hkv, 16, 128, seed=rows)
    for page in (2, 5):
        for h in range(hkv):
            fill(cache, 0, page, 0, h, torch.zeros(16, 128))
    g = torch.Generator().manual_seed(rows)
    words = torch.randint(-2 ** 62, 2 ** 62, (rows, 2), generator=g)
    desc = mask_desc(device, rows, 7 * 16 + 3, words, torch.tensor([2, 0, 5, 1, 3, 4, 6, 7]))
    q = (torch.randn(rows, hq, 128, generator=g) * size).bfloat16()
    out = ops.attention8(q.to(device), cache.layer(0), desc, scale)
    settle(ops)
    assert bool(torch.isfinite(out).all())
    check_attention(out, q, Oracle(cache).val[0], desc, scale)


@pytest.mark.parametrize("device,rows,hq,hkv", PASSES)
@pytest.mark.parametrize("size,scale", [(2.0 ** 80, 128 ** -0.5), (1.0, 2.0 ** 100)], ids=["queries", "scale"])
def test_zero_keys_under_a_factor_that_overflows(device, rows, hq, hkv, size, scale):
    """Zero keys beside a hidden one of the largest size: their scores are zero whatever the factor."""
    ops = impl(device)
    cache = make_cache(device, 1, 6, hkv, 16, 128, seed=rows)
    huge = torch.zeros(16, 128)
    huge[5] = 448 * 2.0 ** 56
    for page in range(5):
        for h in range(hkv):
            fill(cache, 0, page, 0, h, huge)
    g = torch.Generator().manual_seed(rows)
    words = torch.randint(0, 2 ** 62, (rows, 1), generator=g)
    for page in range(5):
        words &= ~(1 << (16 * page + 5)) if page < 4 else -1
    words |= 1
    desc = mask_desc(device, rows, 64, words, torch.tensor([3, 0, 4, 1]))
    q = (torch.randn(rows, hq, 128, generator=g).abs() * size).bfloat16()
    out = ops.attention8(q.to(device), cache.layer(0), desc, scale)
    settle(ops)
    check_attention(out, q, Oracle(cache).val[0], desc, scale)
    # The same keys in the rows' private pages.
    full = torch.full((rows,), 5, dtype=torch.int32, device=device)
    desc = mod("ops.attn_desc").AttnDesc(desc.prefix_pages, 0, 0, 0, full, full, desc.row_mask,
                                         (torch.arange(rows, device=device) % 5).int()[:, None])
    out = ops.attention8(q.to(device), cache.layer(0), desc, scale)
    settle(ops)
    check_attention(out, q, Oracle(cache).val[0], desc, scale)
