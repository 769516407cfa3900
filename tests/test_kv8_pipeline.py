"""The tcgen05 pass of attention over the 8-bit KV cache: the order of its waits, and many chunks per CTA.

The first half is a model of one slot of the pass (the issuer of the products, the softmax warps, the tensor pipe and
the barriers between them) that is walked through every interleaving on the CPU.  A wait names the parity of a phase
only, so it is right only where the phase before the awaited one cannot be the one that is open.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import mod
from test_kv8 import impl, settle

WARPS = 2  # of a slot's four: two are enough to be a chunk apart


# ------------------------------------------------------------------ model
def issuer(n, last):
    """Steps of the products' issuer: ("wait", barrier, phase) and ("do", product, barrier of its commit)."""
    for k in range(n + 1):
        if k < n:
            if k >= 2:
                yield "wait", "pv", k - 2
            yield "do", ("S", k), f"s{k & 1}"
        if k > 0:
            j = k - 1
            yield "wait", f"p{j & 1}", j >> 1
            yield "do", ("PV", j), last if k == n else "pv"


def softmax(n, last, rescales):
    """Steps of a softmax warp; it waits for the product before only in chunks in which its reference moves."""
    for k in range(n):
        yield "wait", f"s{k & 1}", k >> 1
        if k > 0 and (rescales >> k) & 1:
            yield "wait", "pv", k - 1
        yield "arrive", f"p{k & 1}", None
    yield "wait", last, n - 1 if last == "pv" else 0
    yield "leave", None, None


def walk(n, last, rescales=0):
    """The faults that some interleaving reaches: waits that return before their phase ended, and warps that leave the
    loop before every product is done."""
    names = ["pv", "fin", "s0", "s1", "p0", "p1"]
    counts = {"pv": 1, "fin": 1, "s0": 1, "s1": 1, "p0": WARPS, "p1": WARPS}
    progs = [list(issuer(n, last))] + [list(softmax(n, last, rescales))] * WARPS
    faults = set()
    start = ((0,) * len(progs), tuple((0, counts[b]) for b in names), (), 0)  # counters, barriers, queue, products done
    seen, todo = {start}, [start]

    def arrived(bars, name):
        i = names.index(name)
        phase, left = bars[i]
        new = (phase + 1, counts[name]) if left == 1 else (phase, left - 1)
        return bars[:i] + (new,) + bars[i + 1:]

    stuck = True
    while todo:
        pcs, bars, queue, done = todo.pop()
        nxt = []
        if queue:  # the pipe ends its oldest product, and the commit behind it arrives
            (op, bar), rest = queue[0], queue[1:]
            nxt.append((pcs, arrived(bars, bar), rest, done + (op[0] == "PV")))
        for t, prog in enumerate(progs):
            if pcs[t] == len(prog):
                continue
            kind, what, arg = prog[pcs[t]]
            new = pcs[:t] + (pcs[t] + 1,) + pcs[t + 1:]
            if kind == "wait":
                phase = bars[names.index(what)][0]
                if (phase & 1) == (arg & 1):  # the open phase has the awaited parity: not yet
                    continue
                if phase <= arg:
                    faults.add((what, "early"))
                nxt.append((new, bars, queue, done))
            elif kind == "do":
                nxt.append((new, bars, queue + ((what, arg),), done))
            elif kind == "arrive":
                nxt.append((new, arrived(bars, what), queue, done))
            else:
                if done < n:
                    faults.add(("leave", "products open"))
                nxt.append((new, bars, queue, done))
        if not nxt and all(c == len(p) for c, p in zip(pcs, progs)):
            stuck = False
        for s in nxt:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    if stuck:
        faults.add(("end", "never reached"))
    return faults


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
def test_the_last_wait_has_a_barrier_of_its_own(n):
    for rescales in {0, (1 << n) - 1, 0b10, 0b100}:
        assert not walk(n, "fin", rescales)


@pytest.mark.parametrize("n", [2, 3, 4, 5])
def test_a_parity_of_the_products_barrier_does_not_prove_the_last_one(n):
    """What the model finds where the last wait is a phase of the barrier that every product arrives at."""
    assert walk(n, "pv") >= {("pv", "early"), ("leave", "products open")}


# ------------------------------------------------------- many chunks a CTA
def gpu_cache(pages, hkv, ps, seed):
    """Pages of normal values on the GPU."""
    kv8 = mod("ops.kv8")
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = kv8.empty_cache(1, pages, hkv, ps, 128, device="cuda")
    x = torch.randn(1, pages, 2, hkv, ps, 128, device="cuda", generator=g)
    s = kv8.needed_scale(x.abs().amax((-1, -2)))
    cache.data.copy_(kv8.encode(x, s[..., None, None]))
    cache.scale.copy_(s)
    return cache


def check_dense(out, q, layer, pages, seen, scale):
    """``out`` against float64 attention over the pages' keys, of which row r sees ``seen[r]``.

    Weights are rounded to fp16 (2^-11; below 2^-14 of the largest an absolute 2^-25 of it, here with a factor of four
    for pages whose v scales differ), scores come from fp32 sums of 128 products (2^-16 of their magnitudes),
    exponential and sums 2^-17, the output is rounded once.
    """
    m, hq, hd = q.shape
    values = layer.values()
    hkv = values.shape[2]
    g = hq // hkv
    kv = values[pages.long()].permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, hd)[:, :, : seen.shape[1]]
    out = out.reshape(m, hq, hd)
    for h in range(hkv):
        k, v = kv[0, h].double(), kv[1, h].double()
        rows = q[:, h * g:(h + 1) * g].double()
        s = (rows @ k.t()) * scale
        err = ((rows.abs() @ k.abs().t()) * scale).masked_fill(~seen[:, None], 0).amax(-1, keepdim=True)
        some = seen.any(1)[:, None, None]
        p = torch.where(some, torch.softmax(s.masked_fill(~seen[:, None], -torch.inf), -1), torch.zeros_like(s))
        want, mag = p @ v, p @ v.abs()
        top = p.amax(-1, keepdim=True)
        light = ((p < top * 2.0 ** -12) & seen[:, None]).sum(-1, keepdim=True) * top * 2.0 ** -23 * v.abs().max()
        tol = mag * (2.0 ** -11 + 2.0 ** -16 * err + 2.0 ** -17) + light
        tol += want.abs() * torch.finfo(out.dtype).eps / 2 + 2.0 ** -24
        diff = (out[:, h * g:(h + 1) * g].double() - want).abs()
        assert bool((diff <= tol).all()), float((diff / tol).max())


def same_every_time(call, times=8):
    first = call()
    for _ in range(times - 1):
        assert torch.equal(call(), first)
    return first


@pytest.mark.gpu
@pytest.mark.parametrize("ps", [8, 16, 32, 64])
@pytest.mark.parametrize("rows,length", [
    (32, 700), (32, 1500), (32, 3001), (32, 6007),              # 128 rows a head: two slots on alternate chunks
    (40, 64), (40, 65), (40, 130), (40, 300), (40, 1000), (40, 4003)])  # 160 rows a head: both slots on every chunk
def test_tree_of_many_rows(ps, rows, length):
    """One to a dozen chunks per slot and CTA, 32 kv heads so that the device is filled with few splits."""
    ops = impl("cuda")
    n = -(-(length + rows) // ps)
    cache = gpu_cache(n + 2, 32, ps, length)
    g = torch.Generator(device="cuda").manual_seed(rows + ps)
    pages = torch.randperm(n + 2, device="cuda", generator=g)[:n].int()
    words = torch.randint(-2 ** 62, 2 ** 62, (rows, 1), device="cuda", generator=g)
    full = torch.full((rows,), length, device="cuda", dtype=torch.int32)
    full[3] = length // 2
    lens = full + rows
    lens[5] = 0
    desc = mod("ops.attn_desc").AttnDesc(pages, n, length, length, full, lens, words, torch.zeros_like(full)[:, None])
    q = torch.randn(rows, 128, 128, device="cuda", generator=g).to(torch.float16 if ps < 32 else torch.bfloat16)
    out = same_every_time(lambda: ops.attention8(q, cache.layer(0), desc))
    settle(ops)
    x = torch.arange(length + rows, device="cuda")
    marked = ((words >> (x - length).clamp(0, 63)[None]) & 1).bool() & (x >= length)
    check_dense(out, q, cache.layer(0), pages, (x < lens[:, None]) & ((x < full[:, None]) | marked), 1 / math.sqrt(128))


@pytest.mark.gpu
@pytest.mark.parametrize("ps", [8, 16, 32, 64])
@pytest.mark.parametrize("hq,hkv,start,rows", [
    (8, 2, 0, 65), (8, 2, 0, 129), (8, 2, 400, 300),            # output written directly, one to eleven chunks
    (128, 32, 4000, 300),                                       # directly, 64 chunks and more
    (32, 8, 3000, 30), (32, 8, 4000, 100)])                     # keys split, rows of 128 and of 256
def test_causal_chunks(ps, hq, hkv, start, rows):
    ops = impl("cuda")
    n = -(-(start + rows) // ps)
    cache = gpu_cache(n + 2, hkv, ps, rows)
    g = torch.Generator(device="cuda").manual_seed(start + ps)
    pages = torch.randperm(n + 2, device="cuda", generator=g)[:n].int()
    lens = torch.arange(start + 1, start + rows + 1, device="cuda", dtype=torch.int32)
    desc = mod("ops.attn_desc").single_sequence_desc(pages, lens, start)
    q = torch.randn(rows, hq, 128, device="cuda", generator=g).to(torch.bfloat16 if ps < 32 else torch.float16)
    out = same_every_time(lambda: ops.attention8_causal(q, cache.layer(0), desc, start))
    settle(ops)
    x = torch.arange(start + rows, device="cuda")
    check_dense(out, q, cache.layer(0), pages, x < lens[:, None], 1 / math.sqrt(128))
