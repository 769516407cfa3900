"""The KV-reuse diagnostics on the 8-bit cache."""

from __future__ import annotations

import json

import pytest
import torch

from conftest import mod
from test_kv8_engine import DEVICES, make, presets


@pytest.mark.parametrize("device", DEVICES)
def test_prefix_kv_reads_positions_of_an_8bit_cache(device):
    eng = make(device, presets(device)[0], 1, pages=16, positions=256)
    prompt = torch.randint(0, 1024, (41,), generator=torch.Generator().manual_seed(0)).int().to(eng.device)
    pages = [7, 3, 11]
    slots = torch.tensor([pages[x // 16] * 16 + x % 16 for x in range(41)], dtype=torch.int32, device=eng.device)
    table = torch.tensor(pages, dtype=torch.int32, device=eng.device)
    eng.prefill_sequence(prompt, start_pos=0, slots=slots, pages=table)
    diag = mod("serving.diagnostics")
    kv = diag.prefix_kv(eng, pages, 41)
    eng.ops.check()
    c = eng.cfg
    assert tuple(kv.shape) == (c.num_layers, 2, 41, c.num_kv_heads, c.head_dim) and kv.dtype == eng.dtype
    for layer in (0, c.num_layers - 1):
        values = eng.kv[layer].values().to(eng.dtype)
        for x in (0, 15, 16, 40):
            assert torch.equal(kv[layer, :, x], values[pages[x // 16], :, :, x % 16])
    assert diag.prefix_kv(eng, [], 0).shape[2] == 0
    with pytest.raises(IndexError):
        diag.prefix_kv(eng, pages, 49)


def test_commands_take_the_cache(tmp_path):
    diag = mod("serving.diagnostics")
    base = ["--prompt-token-ids", "3,4,5,6,7,8", "--page-size", "4", "--dtype", "float32", "--device", "cpu",
            "--context-length", "256", "--kv-cache", "fp8"]
    out = tmp_path / "t.json"
    # Both caches hold e4m3 codes of the same rows, under page scales that may differ by the rows that were dropped: a
    # value differs by a step of 2^-3 of its page's largest at most.
    assert diag.main(["target-commit", "--model", "tiny-target", "--d", "2", "--rounds", "2", "--json-out", str(out),
                      *base]) == 0
    assert "max_kv_diff" in json.loads(out.read_text())["rounds"][-1]
    assert diag.main(["drafter-alignment", "--model", "tiny-drafter", "--k", "2", "--d", "2", "--json-out", str(out),
                      *base]) in (0, 1)  # against a recompute without a cache: how near it comes is what it reports
    assert json.loads(out.read_text())["steps"]
    with pytest.raises(SystemExit):
        diag.build_parser().parse_args(["target-commit", "--model", "tiny-target", "--kv-cache", "int4"])
