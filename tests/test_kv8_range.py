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


# -------------------------------------------------------------- light weights
def dense(q, layer, pages, seen, scale):
    """float64 attention of rows that see ``seen`` of the pages' keys: (out, weights, sum of weights times |v|, v)."""
    m, hq, hd = q.shape
    values = layer.values().double()
    hkv = values.shape[2]
    kv = values[pages.long()].permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, hd)[:, :, : seen.shape[1]]
    k, v = (kv[i].repeat_interleave(hq // hkv, 0) for i in (0, 1))
    s = torch.einsum("mhd,hkd->mhk", q.double(), k) * scale
    p = torch.softmax(s.masked_fill(~seen[:, None], -torch.inf), -1)
    return torch.einsum("mhk,hkd->mhd", p, v), p, torch.einsum("mhk,hkd->mhd", p, v.abs()), v


@pytest.mark.parametrize("device,rows,hq,hkv", PASSES)
@pytest.mark.parametrize("depth", [18, 22, 26])
def test_light_keys_beside_heavy_ones_without_value(device, rows, hq, hkv, depth):
    """Every sixteenth key takes all the weight and has no value, the others 2^-depth of it each: the answer is theirs
    alone."""
    ops, kv8 = impl(device), mod("ops.kv8")
    pages = 14
    cache = kv8.empty_cache(1, pages, hkv, 16, 128, device=device)
    g = torch.Generator().manual_seed(depth)
    for page in range(pages):
        for h in range(hkv):
            k, v = torch.zeros(16, 128), torch.randn(16, 128, generator=g)
            k[page % 16, 0] = depth
            v[page % 16] = 0
            fill(cache, 0, page, 0, h, k)
            fill(cache, 0, page, 1, h, v)
    n = pages * 16 - 5
    lens = torch.full((rows,), n, dtype=torch.int32, device=device)
    order = torch.randperm(pages, generator=g).int().to(device)
    desc = mod("ops.attn_desc").single_sequence_desc(order, lens, n)
    desc._max_keys = 1 << 20
    q = torch.zeros(rows, hq, 128, dtype=torch.bfloat16)
    q[..., 0] = 1
    out = ops.attention8(q.to(device), cache.layer(0), desc, math.log(2))  # weights are powers of two
    settle(ops)
    x = torch.arange(n, device=device)
    want, p, mag, v = dense(q.to(device), cache.layer(0), order, x < lens[:, None], math.log(2))
    # Weights of fp16 carry 2^-11, below 2^-14 of fp16's unit an absolute 2^-25 of it, where the largest weight is at
    # least 2^7 units; v scales of the pages differ by a factor of two at most; fp32 sums and the exponential 2^-16.
    light = (p < p.amax(-1, keepdim=True)).sum(-1, keepdim=True) * p.amax(-1, keepdim=True) * 2.0 ** -31 * v.abs().max()
    tol = mag * (2.0 ** -11 + 2.0 ** -16) + want.abs() * 2.0 ** -8 + light
    diff = (out.double().reshape(want.shape) - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())


# (rows, q heads, kv heads, keys): several chunks per slot and CTA, keys split over the slots / 256 rows; and a warp's
# units of the register passes
LONG = [(32, 128, 32, 1500), (40, 128, 32, 1000), (1, 32, 32, 3000), (8, 96, 32, 3000)]


def long_cache(hkv, keys):
    kv8 = mod("ops.kv8")
    g = torch.Generator(device="cuda").manual_seed(keys)
    n = -(-keys // 16)
    cache = kv8.empty_cache(1, n, hkv, 16, 128, device="cuda")
    k, v = (torch.randn(n, hkv, 16, 128, device="cuda", generator=g) for _ in range(2))
    return cache, n, k, v, torch.randperm(n, device="cuda", generator=g).int(), g


def store(cache, pages, k, v):
    kv8 = mod("ops.kv8")
    for side, x in enumerate((k, v)):
        s = kv8.needed_scale(x.abs().amax((-1, -2)))
        cache.data[0, pages.long(), side] = kv8.encode(x, s[..., None, None])
        cache.scale[0, pages.long(), side] = s


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hq,hkv,keys", LONG)
def test_scores_that_rise_along_the_keys(rows, hq, hkv, keys):
    """Half of the rows see scores that rise by 24 binades every 64 keys (the reference moves in every chunk), the other
    half scores that fall as much."""
    ops = impl("cuda")
    cache, n, k, v, pages, g = long_cache(hkv, keys)
    k *= 2.0 ** -4
    k[..., 0] = (torch.arange(n, device="cuda") // 4 * 3).float()[:, None, None]
    store(cache, pages, k, v)
    q = torch.randn(rows, hq, 128, device="cuda", generator=g)
    q[..., 0] = 8 * torch.where(torch.arange(rows * hq, device="cuda").reshape(rows, hq) % 2 == 0, 1.0, -1.0)
    q = q.half()
    lens = torch.full((rows,), keys, dtype=torch.int32, device="cuda")
    scale = math.log(2)
    out = ops.attention8(q, cache.layer(0), mod("ops.attn_desc").single_sequence_desc(pages, lens, keys), scale)
    settle(ops)
    want, p, mag, v = dense(q, cache.layer(0), pages, torch.arange(keys, device="cuda") < lens[:, None], scale)
    # A score is a sum of 128 fp32 products of at most 8 * 3 * keys / 64 binades, each rounded (2^-24 relative, and the
    # sum at most 2^-23 of the largest partial sum per step of 16): 2^-19 of that size with the rounding of u.
    size = 8 * 3 * keys / 64
    tol = mag * (2.0 ** -11 + size * 2.0 ** -19 + 2.0 ** -16) + want.abs() * 2.0 ** -11 + 2.0 ** -24
    tol += keys * 2.0 ** -30 * p.amax(-1, keepdim=True) * v.abs().max()
    diff = (out.double().reshape(want.shape) - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("step", [16, 32])
@pytest.mark.parametrize("rows,hq,hkv,keys", LONG)
def test_scores_beyond_the_steps_of_a_binade(rows, hq, hkv, keys, step):
    """Scores of 1.5 * 2^25 binades, where fp32 goes by fours, and every seventh chunk from the third on has keys that
    lie ``step`` higher: sums of two products 2^22 apart at most, exact in fp32, so that the weights are."""
    ops = impl("cuda")
    cache, n, k, v, pages, g = long_cache(hkv, keys)
    k.zero_()
    k[..., 0] = 1.5 * 2.0 ** 17
    k[8::28, :, ::5, 1] = float(step)
    v = v.clamp(-1.75, 1.75)
    v[:, :, 0, 0] = 1.75  # every page's v scale is 2^-8: u stays a multiple of four
    store(cache, pages, k, v)
    q = torch.zeros(rows, hq, 128, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 2.0 ** 8
    q[..., 1] = 1
    lens = torch.full((rows,), keys, dtype=torch.int32, device="cuda")
    out = ops.attention8(q, cache.layer(0), mod("ops.attn_desc").single_sequence_desc(pages, lens, keys), math.log(2))
    settle(ops)
    want, p, mag, v = dense(q, cache.layer(0), pages, torch.arange(keys, device="cuda") < lens[:, None], math.log(2))
    tol = mag * (2.0 ** -11 + 2.0 ** -16) + want.abs() * 2.0 ** -8 + 2.0 ** -24
    tol += keys * 2.0 ** -32 * p.amax(-1, keepdim=True) * v.abs().max()
    diff = (out.double().reshape(want.shape) - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** 11, 2.0 ** 12, 2.0 ** 13, 2.0 ** 14])
@pytest.mark.parametrize("rows,hq,hkv,keys", LONG)
def test_scores_that_fp32_cannot_resolve(rows, hq, hkv, keys, size):
    """Scores around 2^23 to 2^29 binades, off by whole binades in any 32-bit form: the answer stays an average of the
    values."""
    ops = impl("cuda")
    cache, n, k, v, pages, g = long_cache(hkv, keys)
    store(cache, pages, k * size, v)
    q = (torch.randn(rows, hq, 128, device="cuda", generator=g) * size).bfloat16()
    lens = torch.full((rows,), keys, dtype=torch.int32, device="cuda")
    out = ops.attention8(q, cache.layer(0), mod("ops.attn_desc").single_sequence_desc(pages, lens, keys))
    settle(ops)
    assert bool((out.float().abs() <= cache.layer(0).values()[:, 1].abs().max() * (1 + 2.0 ** -7)).all())
