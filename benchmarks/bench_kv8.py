"""8-bit against 16-bit KV cache on one GPU: attention per layer and whole forwards.

    python benchmarks/bench_kv8.py                       # attention and append, 8B head geometry
    python benchmarks/bench_kv8.py --model llama-8b      # one-row and tree forwards of a model as well
    python benchmarks/bench_kv8.py --max-positions 32768 # launches sized for a longer context, as a server's graphs are

Attention: one captured graph of many calls over several layers (more cache than L2 holds from 16K keys
on), CUDA events around its replay.  Forwards: the engines' own graphs, random-init weights, a cache of
random tokens.
"""

from __future__ import annotations

import argparse
import importlib
import json
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def pkg(name: str):
    return importlib.import_module("0709_b200." + name)


def timed(graph, calls: int, repeats: int = 7) -> float:
    """Median microseconds per call."""
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(3):
        graph.replay()
    out = []
    for _ in range(repeats):
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        out.append(a.elapsed_time(b) * 1e3 / calls)
    return sorted(out)[len(out) // 2]


def captured(fn, calls: int):
    fn()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(calls):
            fn()
    return g


def attention(rows: int, length: int, hq: int, hkv: int, page: int, dtype: torch.dtype, layers: int,
              max_positions: int) -> dict:
    cuda_ops, kv8, attn_desc = pkg("ops.cuda_ops"), pkg("ops.kv8"), pkg("ops.attn_desc")
    dev = torch.device("cuda")
    n = -(-(length + rows) // page)
    kv = torch.randn(layers, n, 2, hkv, page, 128, device=dev).to(dtype)
    scale = kv8.needed_scale(kv.float().abs().amax((-1, -2)))
    cache = kv8.Kv8Cache(kv8.encode(kv.float(), scale[..., None, None]), scale)

    class Holder:  # the 16-bit op finds a layer by its place in its engine's cache
        device = dev

    holder = Holder()
    holder.kv = kv
    ops = cuda_ops.CudaOps(holder)
    pages = torch.randperm(n, device=dev).int()
    lens = torch.full((rows,), length + rows, dtype=torch.int32, device=dev)
    masks = torch.tensor([[(1 << (i + 1)) - 1 if i < 63 else -1] for i in range(rows)], dtype=torch.int64, device=dev)
    desc = attn_desc.single_sequence_desc(pages, lens, length, mask_base=length, masks=masks,
                                          full=torch.full_like(lens, length))
    q = torch.randn(rows, hq, 128, device=dev).to(dtype)
    ops.reserve_attention_workspace(rows, hq, hkv, max(length, max_positions), page)
    if max_positions > length:
        desc._max_keys = max_positions
        desc._splits = ops.attention_splits(rows, hq, hkv, max_positions, page)

    def run16():
        for i in range(layers):
            ops.attention(q, kv[i], desc)

    def run8():
        for i in range(layers):
            ops.attention8(q, cache.layer(i), desc)

    res = {"rows": rows, "length": length, "heads": f"{hq}/{hkv}"}
    for name, fn in (("us_16bit", run16), ("us_8bit", run8)):
        res[name] = round(timed(captured(fn, 4), 4 * layers), 2)
    ops.check()
    return res


def forwards(model: str, length: int, page: int, max_positions: int) -> list[dict]:
    loader, e8 = pkg("models.loader"), pkg("runtime.engine_kv8")
    w = loader.resolve_model(model, dtype="float16", device="cuda", seed=0)
    pages = -(-(length + 64) // page) + 4
    out = []
    for kv_cache in ("model", "fp8"):
        eng = e8.make_engine(w, kv_cache=kv_cache, num_pages=pages, page_size=page,
                             max_positions=max(length + 128, max_positions))
        table = torch.arange(pages, dtype=torch.int32, device="cuda")
        tokens = torch.randint(0, w.config.vocab_size, (length,), device="cuda").int()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        slots = torch.arange(length, dtype=torch.int32, device="cuda")
        for _ in range(2):
            a.record()
            eng.prefill_sequence(tokens, start_pos=0, slots=slots, pages=table)
            b.record()
        torch.cuda.synchronize()
        res = {"kv_cache": kv_cache, "length": length, "prefill_ms": round(a.elapsed_time(b), 2)}
        for rows in (1, 12):
            pos = np.arange(length, length + rows)
            fields = dict(tokens=np.zeros(rows, dtype=np.int64), positions=pos, slots=pos, shared_len=length,
                          n_shared_pages=pages, mask_base=length, row_full=np.full(rows, length),
                          row_len=np.full(rows, length + rows),
                          row_mask=np.array([[(1 << (i + 1)) - 1] for i in range(rows)], dtype=np.int64))
            times = []
            for _ in range(12):
                torch.cuda.synchronize()
                a.record()
                eng.run_rows(16 if rows > 8 else 1, prefix_pages=table, **fields)
                b.record()
                torch.cuda.synchronize()
                times.append(a.elapsed_time(b))
            res[f"forward_{rows}_rows_ms"] = round(sorted(times)[len(times) // 2], 3)
        eng.ops.check()
        out.append(res)
        eng.drop_graphs()
        del eng
        torch.cuda.empty_cache()
    return out


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--model", default=None, help="also time whole forwards of this preset or checkpoint")
    p.add_argument("--lengths", type=int, nargs="+", default=[1024, 4096, 16384, 65536])
    p.add_argument("--rows", type=int, nargs="+", default=[1, 4, 12, 48])
    p.add_argument("--page-size", type=int, default=16)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--max-positions", type=int, default=0,
                   help="longest context that the launches are sized for (default: each length's own)")
    a = p.parse_args(argv)
    for length in a.lengths:
        for rows in a.rows:
            print(json.dumps(attention(rows, length, 32, 8, a.page_size, torch.float16, a.layers,
                                       a.max_positions)), flush=True)
    if a.model:
        for length in a.lengths:
            for r in forwards(a.model, length, a.page_size, a.max_positions):
                print(json.dumps(r), flush=True)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
