"""Indices of the 8-bit KV cache operators that name nothing: beyond 32 bits, negative, or mask bits that are not there."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import mod
from test_kv8 import Oracle, assert_pages, check_attention, impl, make_cache, rope, settle
from test_kv8_limits import IMPLS, ints, reported


@pytest.mark.parametrize("device", IMPLS)
def test_negative_pages_are_refused(device):
    """A page before the first one, in a page list, among private pages or to be read back."""
    cache = make_cache(device, 1, 6, 2, 16, 128, seed=0)
    attn_desc = mod("ops.attn_desc")
    q = torch.randn(2, 4, 128, device=device).half()
    lens = ints([40, 30], device)
    zero = torch.zeros(2, 1, dtype=torch.int64, device=device)
    for prefix, shared, tails in (([0, -1, 1], 3, [[0], [0]]), ([0, 1], 2, [[-2], [2]])):
        desc = attn_desc.AttnDesc(ints(prefix, device), shared, 16 * shared, 0, lens, lens, zero, ints(tails, device))
        reported(device, lambda ops: ops.attention8(q, cache.layer(0), desc), 2)
    desc = attn_desc.single_sequence_desc(ints([0, -1], device), lens, 0)
    reported(device, lambda ops: ops.attention8_causal(q, cache.layer(0), desc, 20), 2)
    for what in (cache, cache.layer(0)):
        reported(device, lambda ops: ops.kv8_read_pages(what, ints([1, -1], device), torch.float16), 2)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("rows,hq", [(4, 4), (40, 8)])
@pytest.mark.parametrize("words", [0, 1, 2])
def test_keys_outside_the_mask(device, rows, hq, words):
    """Rows whose own keys end before the mask begins, and keys behind its last word: no bit, no key."""
    ops = impl(device)
    cache = make_cache(device, 1, 14, 1, 16, 128, seed=words)
    g = torch.Generator().manual_seed(rows)
    full = torch.randint(0, 60, (rows,), generator=g).int()
    lens = torch.randint(150, 208, (rows,), generator=g).int()
    mask = torch.full((rows, words), -1, dtype=torch.int64)
    desc = mod("ops.attn_desc").AttnDesc(torch.randperm(14, generator=g).int().to(device), 13, 0, 64, full.to(device),
                                         lens.to(device), mask.to(device),
                                         torch.zeros(rows, 1, dtype=torch.int32, device=device))
    desc._max_keys = 1 << 20
    q = torch.randn(rows, hq, 128, generator=g).half()
    out = ops.attention8(q.to(device), cache.layer(0), desc)
    settle(ops)
    check_attention(out, q, Oracle(cache).val[0], desc, 1 / math.sqrt(128))


def longs(x, device):
    return torch.tensor(x, dtype=torch.int64, device=device)


FAR = [2 ** 32 + 3, -2 ** 32 + 3, 2 ** 40, -1]  # the first two are 3 in their low 32 bits


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("bad", FAR)
def test_append_indices_beyond_32_bits(device, bad):
    cache = make_cache(device, 1, 6, 1, 16, 128, seed=0)
    before = Oracle(cache)
    qkv, table = torch.randn(1, 3 * 128, device=device), rope(8, 128, device)
    for pos, slot in ((0, bad), (bad, 3)):
        reported(device, lambda ops: ops.rope_qkv_append8(qkv, table, longs([pos], device), longs([slot], device),
                                                          cache.layer(0), 1, 1), 2)
        assert_pages(cache, before)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("bad", FAR)
def test_page_indices_beyond_32_bits(device, bad):
    cache = make_cache(device, 2, 6, 2, 16, 128, seed=0)
    before = Oracle(cache)
    for src, dst in ((bad, 5), (5, bad)):
        reported(device, lambda ops: ops.kv8_move_slots(cache, longs([src], device), longs([dst], device)), 2)
    for plan in ((bad, 1, 2), (1, bad, 2), (1, 2, bad)):
        reported(device, lambda ops: ops.kv8_copy_pages(cache, longs([plan], device)), 2)
    assert_pages(cache, before)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("bad", FAR)
def test_read_pages_beyond_32_bits(device, bad):
    cache = make_cache(device, 2, 6, 2, 16, 128, seed=0)
    for what in (cache, cache.layer(1)):
        reported(device, lambda ops: ops.kv8_read_pages(what, longs([2, bad], device), torch.float16), 2)


@pytest.mark.parametrize("device", IMPLS)
def test_indices_of_64_bits(device):
    """The same indices in 64 bits and in 32 give the same cache."""
    ops = impl(device)
    caches = [make_cache(device, 1, 6, 1, 16, 128, seed=0) for _ in range(2)]
    qkv, table = torch.randn(3, 3 * 128, device=device), rope(8, 128, device)
    for cache, make in zip(caches, (ints, longs)):
        ops.rope_qkv_append8(qkv, table, make([5, 6, 7], device), make([14, 15, 16], device), cache.layer(0), 1, 1)
        ops.kv8_move_slots(cache, make([16], device), make([40], device))
        ops.kv8_copy_pages(cache, make([[0, 4, 9]], device))
    settle(ops)
    assert torch.equal(caches[0].scale, caches[1].scale)
    assert torch.equal(caches[0].data.view(torch.uint8), caches[1].data.view(torch.uint8))
    pages = [ops.kv8_read_pages(caches[0], make([4, 1], device), torch.float16) for make in (ints, longs)]
    assert torch.equal(*pages)


@pytest.mark.parametrize("device", IMPLS)
def test_arguments_that_do_not_fit_together(device):
    """Kv heads that are not the cache's, and lists of different lengths."""
    ops = impl(device)
    cache = make_cache(device, 1, 6, 2, 16, 128, seed=0)
    before = Oracle(cache)
    table, layer = rope(8, 128, device), cache.layer(0)
    one, two = ints([1], device), ints([1, 2], device)
    qkv = torch.randn(2, 6 * 128, device=device).half()
    for call in (lambda: ops.rope_qkv_append8(qkv, table, two, two, layer, 4, 1),
                 lambda: ops.rope_qkv_append8(qkv, table, one, two, layer, 2, 2),
                 lambda: ops.rope_qkv_append8(qkv, table, two, one, layer, 2, 2),
                 lambda: ops.kv8_move_slots(cache, two, one),
                 lambda: ops.kv8_move_slots(cache, one, two)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    settle(ops)
    assert_pages(cache, before)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 70])
def test_a_refused_row_that_repeats_a_slot(rows):
    """The later row of a slot counts, also where it cannot be stored: the slot keeps what it held, the rows beside it
    are stored."""
    cache = make_cache("cuda", 1, 8, 1, 16, 128, seed=rows)
    oracle = Oracle(cache)
    qkv = torch.ones(rows, 3 * 128, device="cuda")
    qkv[rows - 1, 300] = math.nan
    slots = list(range(17, 17 + rows - 1)) + [17]
    reported("cuda", lambda ops: ops.rope_qkv_append8(qkv, rope(4, 128, "cuda"), ints([0] * rows, "cuda"),
                                                      ints(slots, "cuda"), cache.layer(0), 1, 1), 5)
    row = (torch.ones(128, dtype=torch.float64), 2.0 ** -8)
    for side in (0, 1):
        for page in range(1, 8):
            oracle.write(0, side, 0, page, {s % 16: row for s in slots[1:-1] if s // 16 == page})
    assert_pages(cache, oracle)
