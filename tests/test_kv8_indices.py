"""Indices of the 8-bit KV cache operators that name nothing: beyond 32 bits, negative, or mask bits that are not there."""

from __future__ import annotations

import pytest
import torch

from conftest import mod
from test_kv8 import impl, make_cache
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
