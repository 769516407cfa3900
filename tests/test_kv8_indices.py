"""Indices of the 8-bit KV cache operators that name nothing: beyond 32 bits, negative, or mask bits that are not there."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import mod
from test_kv8 import Oracle, check_attention, impl, make_cache, settle
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
