"""Limits of the 8-bit KV cache operators: refusals, reported errors, long sequences, streams, captured graphs."""

from __future__ import annotations

import dataclasses
import math

import pytest
import torch

from conftest import mod
from test_kv8 import ATTENTIONS, Oracle, assert_pages, check_attention, impl, make_cache, make_desc, rope, settle

IMPLS = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="cuda", marks=pytest.mark.gpu)]


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def reported(device, call, code):
    """The PyTorch form raises; the kernel records ``code`` and the next check raises it."""
    if device == "cpu":
        with pytest.raises((IndexError, ValueError)):
            call(impl(device))
        return
    ops = impl(device)
    call(ops)
    torch.cuda.synchronize()
    with pytest.raises(mod("utils.transfer").KernelError) as e:
        ops.check()
    assert e.value.code == code
    ops.check()


# ---------------------------------------------------------------- reported
@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("bad", [-1, 6 * 16])
def test_append_outside_the_cache(device, bad):
    cache = make_cache(device, 1, 6, 2, 16, 128, seed=0)
    before = Oracle(cache)
    qkv = torch.randn(1, 6 * 128, device=device)
    reported(device, lambda ops: ops.rope_qkv_append8(qkv, rope(4, 128, device), ints([0], device), ints([bad], device),
                                                      cache.layer(0), 2, 2), 2)
    assert_pages(cache, before)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 2.0 ** 66])
@pytest.mark.parametrize("where", ["k", "v"])
def test_append_of_what_cannot_be_stored(device, value, where):
    """The row is left out; the rows beside it are stored (the PyTorch form raises before it writes)."""
    cache = make_cache(device, 1, 6, 1, 16, 128, seed=0)
    oracle = Oracle(cache)
    qkv = torch.ones(2, 3 * 128, device=device)
    qkv[0, 128 + 5 if where == "k" else 256 + 5] = value
    reported(device, lambda ops: ops.rope_qkv_append8(qkv, rope(4, 128, device), ints([0, 0], device),
                                                      ints([16, 17], device), cache.layer(0), 1, 1), 5)
    if device == "cuda":  # slot 16 was not written, so its page does not start anew
        for side in (0, 1):
            oracle.write(0, side, 0, 1, {1: (torch.ones(128, dtype=torch.float64), 2.0 ** -8)})
    assert_pages(cache, oracle)


@pytest.mark.parametrize("device", IMPLS)
def test_append_position_outside_the_table(device):
    cache = make_cache(device, 1, 6, 1, 16, 128, seed=0)
    before = Oracle(cache)
    qkv = torch.randn(1, 3 * 128, device=device)
    reported(device, lambda ops: ops.rope_qkv_append8(qkv, rope(4, 128, device), ints([4], device), ints([3], device),
                                                      cache.layer(0), 1, 1), 2)
    assert_pages(cache, before)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("plan", [[(0, 6, 1)], [(-1, 2, 1)], [(0, 1, 17)], [(0, 1, -1)], [(3, 3, 4)],
                                  [(0, 1, 2), (2, 1, 3)], [(0, 1, 2), (1, 2, 3), (4, 5, 1)]])
def test_copies_that_are_refused(device, plan):
    """A destination that is named twice, or is a source, is refused whatever its order; other copies of the call stand."""
    cache = make_cache(device, 2, 6, 2, 16, 128, seed=0)
    oracle = Oracle(cache)
    if device == "cuda":  # what stands: (1, 2, 3) reads a page that keeps its content, (4, 5, 1) is independent
        for src, dst, n in plan if len(plan) == 3 else []:
            if dst != 1:
                oracle.val[:, dst] = 0
                oracle.val[:, dst, :, :, :n] = oracle.val[:, src, :, :, :n]
                oracle.scale[:, dst] = oracle.scale[:, src]
    reported(device, lambda ops: ops.kv8_copy_pages(cache, ints(plan, device)), 2)
    assert_pages(cache, oracle)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("src,dst", [([-1], [3]), ([3], [96]), ([96], [3])])
def test_moves_outside_the_cache(device, src, dst):
    cache = make_cache(device, 2, 6, 2, 16, 128, seed=0)
    before = Oracle(cache)
    reported(device, lambda ops: ops.kv8_move_slots(cache, ints(src, device), ints(dst, device)), 2)
    assert_pages(cache, before)


@pytest.mark.gpu
def test_bad_pages_are_reported():
    cache = make_cache("cuda", 1, 6, 2, 16, 128, seed=0)
    attn_desc = mod("ops.attn_desc")
    q = torch.randn(2, 4, 128, device="cuda").half()
    many = torch.randn(40, 4, 128, device="cuda").half()
    lens = ints([40, 30], "cuda")
    for pages in ([0, 1, 6], [0, -3, 1], [0, 1]):  # outside the cache, negative, too few
        p = ints(pages, "cuda")
        reported("cuda", lambda ops: ops.attention8(
            q, cache.layer(0), attn_desc.single_sequence_desc(p, lens, 40)), 2)
        long = torch.full((40,), 40, dtype=torch.int32, device="cuda")
        reported("cuda", lambda ops: ops.attention8(
            many, cache.layer(0), attn_desc.single_sequence_desc(p, long, 40)), 2)
    for tails, n in (([[6], [1]], 40), ([[2], [-1]], 40), ([[2], [1]], 70)):  # the last: more keys than private pages
        desc = attn_desc.AttnDesc(ints([0, 1], "cuda"), 2, 32, 32, ints([n, 40], "cuda"), ints([n, 40], "cuda"),
                                  torch.full((2, 1), -1, dtype=torch.int64, device="cuda"), ints(tails, "cuda"))
        reported("cuda", lambda ops: ops.attention8(q, cache.layer(0), desc), 2)
    reported("cuda", lambda ops: ops.attention8_causal(
        q, cache.layer(0), attn_desc.single_sequence_desc(ints([0, 9], "cuda"), lens, 0), 20), 2)
    reported("cuda", lambda ops: ops.kv8_read_pages(cache, ints([1, 6], "cuda"), torch.float16), 2)


# ----------------------------------------------------------------- refused
def test_layers_outside_the_cache():
    cache = mod("ops.kv8").empty_cache(2, 3, 1, 16, 128)
    for index in (-1, 2):
        with pytest.raises(IndexError):
            cache.layer(index)


def test_needed_scale_refuses_what_no_scale_holds():
    kv8 = mod("ops.kv8")
    assert float(kv8.needed_scale(torch.tensor(448.0 * 2.0 ** 56))) == 2.0 ** 56
    for a in (math.inf, math.nan, 449.0 * 2.0 ** 56):
        with pytest.raises(ValueError):
            kv8.needed_scale(torch.tensor(a))


@pytest.mark.gpu
def test_calls_that_are_refused():
    ops, kv8, attn_desc = impl("cuda"), mod("ops.kv8"), mod("ops.attn_desc")
    cache = make_cache("cuda", 1, 6, 2, 16, 128, seed=0)
    layer = cache.layer(0)
    q = torch.randn(2, 4, 128, device="cuda").half()
    lens = ints([3, 5], "cuda")
    desc = attn_desc.single_sequence_desc(ints([0, 1], "cuda"), lens, 5)
    table, one = rope(8, 128, "cuda"), ints([0], "cuda")
    qkv = torch.randn(1, 6 * 128, device="cuda").half()

    def other(data=None, scale=None):
        return kv8.Kv8Cache(cache.data if data is None else data, cache.scale if scale is None else scale).layer(0)

    refused = [
        lambda: ops.attention8(q.float(), layer, desc),
        lambda: ops.attention8(q[..., :64], layer, desc),
        lambda: ops.attention8(q[:, :3], layer, desc),
        lambda: ops.attention8(q.cpu(), layer, desc),
        lambda: ops.attention8(q, layer, desc, -1.0),
        lambda: ops.attention8(q, layer, desc, math.inf),
        lambda: ops.attention8(q[:1], layer, desc),
        lambda: ops.attention8(q, other(data=cache.data[..., :64].contiguous()), desc),
        lambda: ops.attention8(q, other(data=cache.data.float()), desc),
        lambda: ops.attention8(q, other(scale=cache.scale.double()), desc),
        lambda: ops.attention8(q, other(scale=cache.scale[:, :3]), desc),
        lambda: ops.attention8(q, make_cache("cuda", 1, 6, 2, 4, 128, seed=0).layer(0), desc),
        lambda: ops.attention8_causal(q, layer, desc, -1),
        lambda: ops.attention8_causal(q, layer, desc, 31),
        lambda: ops.attention8_causal(q, layer, desc, 2 ** 63 - 1),
        lambda: ops.attention8_causal(q, layer, desc, 2 ** 32),
        lambda: ops.attention8(q, layer, dataclasses.replace(desc, n_shared_pages=2 ** 62)),
        lambda: ops.attention8(q, layer, dataclasses.replace(desc, n_shared_pages=-1)),
        lambda: ops.attention8(q, layer, dataclasses.replace(desc, shared_len=2 ** 32 + 5)),
        lambda: ops.attention8(q, layer, dataclasses.replace(desc, mask_base=2 ** 32)),
        lambda: ops.rope_qkv_append8(qkv, table, one, one, layer, 2, 1),
        lambda: ops.rope_qkv_append8(qkv, table, one, one, layer, 3, 2),
        lambda: ops.rope_qkv_append8(qkv, table, one, one, layer, 2, 2, out_dtype=torch.bfloat16),
        lambda: ops.rope_qkv_append8(qkv, table.half(), one, one, layer, 2, 2),
        lambda: ops.rope_qkv_append8(qkv, table, ints([0, 1], "cuda"), one, layer, 2, 2),
        lambda: ops.kv8_move_slots(cache, ints([1, 2], "cuda"), ints([3], "cuda")),
        lambda: ops.kv8_move_slots(cache, torch.zeros(1025, device="cuda"), torch.zeros(1025, device="cuda")),
        lambda: ops.kv8_copy_pages(cache, ints([[0, 1]], "cuda")),
        lambda: ops.kv8_read_pages(cache, one, torch.float32),
    ]
    for i, call in enumerate(refused):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()
            raise AssertionError(f"call {i} was not refused")
    ops.check()


@pytest.mark.gpu
def test_empty_calls():
    ops, attn_desc = impl("cuda"), mod("ops.attn_desc")
    cache = make_cache("cuda", 2, 6, 2, 16, 128, seed=0)
    before = Oracle(cache)
    none = ints([], "cuda")
    desc = attn_desc.single_sequence_desc(ints([0], "cuda"), none, 0)
    q = torch.empty(0, 4, 128, device="cuda", dtype=torch.half)
    assert ops.attention8(q, cache.layer(0), desc).shape == (0, 512)
    assert ops.attention8_causal(q, cache.layer(0), desc, 0).shape == (0, 512)
    assert ops.rope_qkv_append8(torch.empty(0, 6 * 128, device="cuda").half(), rope(4, 128, "cuda"), none, none,
                                cache.layer(0), 2, 2).shape == (0, 2, 128)
    ops.kv8_move_slots(cache, none, none)
    # A descriptor without any shared key: every row answers zero, or its private keys.
    q = torch.randn(2, 4, 128, device="cuda").half()
    desc = attn_desc.AttnDesc(none, 0, 0, 0, ints([0, 3], "cuda"), ints([0, 3], "cuda"),
                              torch.zeros(2, 1, dtype=torch.int64, device="cuda"), ints([[1], [2]], "cuda"))
    out = ops.attention8(q, cache.layer(0), desc)
    settle(ops)
    assert not out[0].any()
    check_attention(out, q, before.val[0], desc, 1 / math.sqrt(128))
    assert_pages(cache, before)


# ------------------------------------------------------------ long and wide
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind,ps,hq,hkv,length,rows", ATTENTIONS)
def test_attention_sized_for_a_longer_context(dtype, kind, ps, hq, hkv, length, rows):
    """Short contexts in the launch shape of a captured graph that may see 2^20 keys: the pass for long sequences, and
    splits that have no key."""
    ops = impl("cuda")
    pages = 4 + -(-(length + rows + 1) // ps) + (rows * 2 if kind == "routes" else 0)
    desc = make_desc("cuda", kind, ps, length, rows, seed=length + rows, pages=pages)
    desc._max_keys = 1 << 20
    cache = make_cache("cuda", 2, pages, hkv, ps, 128, seed=length)
    q = torch.randn(rows, hq, 128, generator=torch.Generator().manual_seed(rows)).to(dtype)
    out = ops.attention8(q.cuda(), cache.layer(1), desc)
    settle(ops)
    check_attention(out, q, Oracle(cache).val[1], desc, 1 / math.sqrt(128))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,hq,hkv,length,rows", [
    ("tree", 4, 1, 700, 9), ("tree", 8, 1, 1500, 33), ("ragged", 32, 2, 900, 12), ("routes", 8, 2, 1031, 30),
    ("tree", 128, 1, 333, 5), ("ragged", 12, 3, 20000, 5)])
def test_attention_at_more_row_tiles(kind, hq, hkv, length, rows):
    """Several tiles of 16 rows over the same keys, and the other side of the border between the passes."""
    ops = impl("cuda")
    pages = 4 + -(-(length + rows + 1) // 16) + (rows * 2 if kind == "routes" else 0)
    desc = make_desc("cuda", kind, 16, length, rows, seed=length, pages=pages)
    cache = make_cache("cuda", 1, pages, hkv, 16, 128, seed=length)
    q = torch.randn(rows, hq, 128, generator=torch.Generator().manual_seed(rows)).half()
    outs = []
    for keys in (0, 1 << 20):
        desc._max_keys = keys
        outs.append(ops.attention8(q.cuda(), cache.layer(0), desc))
    settle(ops)
    for out in outs:
        check_attention(out, q, Oracle(cache).val[0], desc, 1 / math.sqrt(128))


def torch_attention(q, values, pages, lens, scale):
    """float64 on the GPU, rows that see a prefix of one page list."""
    m, hq, hd = q.shape
    hkv = values.shape[2]
    kv = values[pages.long()].permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, hd)
    out = torch.empty(m, hq, hd, dtype=torch.float64, device=q.device)
    mag = torch.empty_like(out)
    g = hq // hkv
    x = torch.arange(kv.shape[2], device=q.device)
    for h in range(hkv):
        k, v = kv[0, h].double(), kv[1, h].double()
        s = (q[:, h * g:(h + 1) * g].double() @ k.t()) * scale
        p = torch.softmax(s.masked_fill(x[None, None] >= lens[:, None, None], -torch.inf), -1)
        out[:, h * g:(h + 1) * g] = p @ v
        mag[:, h * g:(h + 1) * g] = p @ v.abs()
    return out, mag


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,rows,length", [(32, 32, 1, 80003), (64, 32, 16, 40001), (32, 2, 3, 60000),
                                                (16, 2, 33, 50001), (32, 2, 6, 60000)])
def test_attention_over_long_sequences(hq, hkv, rows, length):
    """Many pages per warp and CTA (rings and page windows wrap), for each of the three passes."""
    ops, kv8, attn_desc = impl("cuda"), mod("ops.kv8"), mod("ops.attn_desc")
    g = torch.Generator(device="cuda").manual_seed(length)
    n = -(-length // 16)
    cache = kv8.empty_cache(1, n, hkv, 16, 128, device="cuda")
    x = torch.randn(1, n, 2, hkv, 16, 128, device="cuda", generator=g)
    x *= torch.exp2(torch.randint(-2, 3, (1, n, 2, hkv, 1, 1), device="cuda", generator=g).float())
    s = kv8.needed_scale(x.abs().amax((-1, -2)))
    cache.data.copy_(kv8.encode(x, s[..., None, None]))
    cache.scale.copy_(s)
    del x
    pages = torch.randperm(n, device="cuda", generator=g).int()
    lens = torch.randint(length // 2, length + 1, (rows,), device="cuda", generator=g).int()
    lens[-1] = length
    q = torch.randn(rows, hq, 128, device="cuda", generator=g).half()
    out = ops.attention8(q, cache.layer(0), attn_desc.single_sequence_desc(pages, lens, length))
    settle(ops)
    want, mag = torch_attention(q, cache.layer(0).values(), pages, lens, 1 / math.sqrt(128))
    # As in check_attention: weights 2^-11 and their sum 2^-11, scores 2^-16 of |q||k| / sqrt(128) < 2^9 (pages up to
    # four times normal size), output 2^-11.
    tol = mag * (2.0 ** -10 + 2.0 ** -7) + want.abs() * 2.0 ** -11
    assert bool(((out.double().reshape(want.shape) - want).abs() <= tol).all())
    assert float((out.double().reshape(want.shape) - want).norm() / want.norm()) < 2.0 ** -10


@pytest.mark.gpu
@pytest.mark.parametrize("moves", [65, 400, 1024])
def test_many_moves(moves):
    ops = impl("cuda")
    cache = make_cache("cuda", 2, 160, 2, 16, 128, seed=moves)
    other = mod("ops.kv8").Kv8Cache(cache.data.cpu(), cache.scale.cpu())
    g = torch.Generator().manual_seed(moves)
    src, dst = (torch.randperm(2560, generator=g)[:moves].int() for _ in range(2))
    mod("ops.torch_ops").kv8_move_slots(other, src, dst)
    ops.kv8_move_slots(cache, src.cuda(), dst.cuda())
    settle(ops)
    assert torch.equal(cache.scale.cpu(), other.scale)
    assert torch.equal(cache.data.cpu().float(), other.data.float())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hq,dtype", [(65, 3, torch.bfloat16), (700, 3, torch.bfloat16), (2100, 32, torch.float16),
                                           (2049, 32, torch.float32)])
def test_append_of_many_rows_in_any_order(rows, hq, dtype):
    """More rows than the latency form takes, shuffled over the pages, some slots named twice; from 64 K (row, head)
    pairs on in the form for long prompts."""
    ops = impl("cuda")
    pages = 60 if rows < 960 else 140
    cache = make_cache("cuda", 1, pages, 2, 16, 128, seed=rows)
    other = mod("ops.kv8").Kv8Cache(cache.data.cpu(), cache.scale.cpu())
    g = torch.Generator().manual_seed(rows)
    slots = torch.randperm(pages * 16, generator=g)[:rows].int()
    slots[3] = slots[rows - 2]
    qkv = torch.randn(rows, (hq + 4) * 128, generator=g).to(dtype)
    pos = torch.zeros(rows, dtype=torch.int32)  # the rotation is the identity: no value is next to a border by rounding
    table = rope(4, 128, "cpu")
    out = torch.float16 if dtype == torch.float32 else dtype
    q = ops.rope_qkv_append8(qkv.cuda(), table.cuda(), pos.cuda(), slots.cuda(), cache.layer(0), hq, 2, out_dtype=out)
    want = mod("ops.torch_ops").rope_qkv_append8(qkv, table, pos, slots, other.layer(0), hq, 2, out_dtype=out)
    settle(ops)
    assert torch.equal(q.cpu(), want)
    assert torch.equal(cache.scale.cpu(), other.scale)
    assert torch.equal(cache.data.cpu().float(), other.data.float())


# ------------------------------------------------- streams, strides, graphs
@pytest.mark.gpu
def test_strided_and_offset_inputs():
    ops, attn_desc = impl("cuda"), mod("ops.attn_desc")
    cache = make_cache("cuda", 1, 6, 2, 16, 128, seed=0)
    oracle = Oracle(cache)
    wide = torch.randn(3, 6 * 128 + 64, device="cuda").half()
    table = rope(8, 128, "cuda")
    pos, slots = ints([1, 2, 3], "cuda"), ints([33, 34, 35], "cuda")
    q = ops.rope_qkv_append8(wide[:, 3:3 + 6 * 128], table, pos, slots, cache.layer(0), 2, 2)  # 6-byte offset
    again = make_cache("cuda", 1, 6, 2, 16, 128, seed=0)
    want = ops.rope_qkv_append8(wide[:, 3:3 + 6 * 128].contiguous(), table, pos, slots, again.layer(0), 2, 2)
    settle(ops)
    assert torch.equal(q, want) and torch.equal(cache.data.view(torch.uint8), again.data.view(torch.uint8))
    qs = torch.randn(2, 8, 256, device="cuda").half()[:, ::2, 64:192]
    desc = attn_desc.single_sequence_desc(ints([0, 4], "cuda"), ints([17, 30], "cuda"), 30)
    out = ops.attention8(qs, cache.layer(0), desc)
    settle(ops)
    check_attention(out, qs, Oracle(again).val[0], desc, 1 / math.sqrt(128))
    assert oracle.ps == 16


@pytest.mark.gpu
def test_two_streams_and_a_captured_graph():
    """Calls in flight on two streams, and a captured call replayed between eager ones, share nothing."""
    ops = impl("cuda")
    cases = []
    for i, (kind, hq, hkv, rows, length) in enumerate((("tree", 8, 2, 13, 3000), ("single", 8, 8, 1, 2500),
                                                       ("routes", 16, 2, 9, 2051))):
        pages = 4 + -(-(length + rows + 1) // 16) + 2 * rows
        desc = make_desc("cuda", kind, 16, length, rows, seed=i, pages=pages)
        cache = make_cache("cuda", 1, pages, hkv, 16, 128, seed=i)
        q = torch.randn(rows, hq, 128, generator=torch.Generator().manual_seed(i)).half().cuda()
        cases.append((q, cache.layer(0), desc))
    want = [ops.attention8(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([ops.attention8(*c) for c in cases])
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for c in cases:
            g = torch.cuda.CUDAGraph()
            g.capture_begin(capture_error_mode="thread_local")
            out = ops.attention8(*c)
            g.capture_end()
            graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (g, _) in zip([*streams, side], graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = [ops.attention8(*c) for c in cases]
        torch.cuda.synchronize()
        assert all(torch.equal(out, b) for (_, out), b in zip(graphs, want))
        assert all(torch.equal(a, b) for a, b in zip(eager, want))
    ops.check()


@pytest.mark.gpu
def test_rows_do_not_touch_each_other():
    """A NaN query spoils its own row only, and a row's result does not depend on the rows behind it."""
    ops, attn_desc = impl("cuda"), mod("ops.attn_desc")
    for rows, hq in ((4, 8), (20, 16), (40, 32)):  # each of the three passes (kv heads 2)
        cache = make_cache("cuda", 1, 40, 2, 16, 128, seed=rows)
        pages = torch.randperm(40, generator=torch.Generator().manual_seed(rows)).int().cuda()
        lens = torch.randint(1, 600, (rows,), generator=torch.Generator().manual_seed(1)).int().cuda()
        q = torch.randn(rows, hq, 128, generator=torch.Generator().manual_seed(2)).half().cuda()
        clean = ops.attention8(q, cache.layer(0), attn_desc.single_sequence_desc(pages, lens, 600))
        q[1, 3, 17] = math.nan
        out = ops.attention8(q, cache.layer(0), attn_desc.single_sequence_desc(pages, lens, 600))
        settle(ops)
        out, clean = out.reshape(rows, hq, 128), clean.reshape(rows, hq, 128)
        assert out[1, 3].isnan().all()
        keep = torch.ones(rows, hq, dtype=torch.bool, device="cuda")
        keep[1, 3] = False
        assert torch.equal(out[keep], clean[keep])


@pytest.mark.gpu
def test_a_whole_step_of_operators():
    """Fork, append, attend, compact, read back, as a step of the runtime strings them together."""
    ops, torch_ops, kv8, attn_desc = impl("cuda"), mod("ops.torch_ops"), mod("ops.kv8"), mod("ops.attn_desc")
    dev = make_cache("cuda", 2, 12, 2, 16, 128, seed=9)
    cpu = kv8.Kv8Cache(dev.data.cpu(), dev.scale.cpu())
    g = torch.Generator().manual_seed(0)
    table = rope(64, 128, "cpu")
    prefix = 37  # two whole pages and five tokens of a third
    outs = []
    for o, cache, to in ((ops, dev, "cuda"), (torch_ops, cpu, "cpu")):
        g.manual_seed(0)
        o.kv8_copy_pages(cache, ints([(2, 5, 5), (2, 6, 5), (2, 7, 5)], to))
        qkv = torch.randn(3, 8 * 128, generator=g).half().to(to)
        slots = ints([5 * 16 + 5, 6 * 16 + 5, 7 * 16 + 5], to)
        q = o.rope_qkv_append8(qkv, table.to(to), ints([0] * 3, to), slots, cache.layer(1), 4, 2)
        desc = attn_desc.AttnDesc(ints([0, 1, 2], to), 2, prefix, prefix, ints([38] * 3, to), ints([38] * 3, to),
                                  torch.full((3, 1), -1, dtype=torch.int64, device=to), ints([[5], [6], [7]], to))
        a = o.attention8(q, cache.layer(1), desc)
        o.kv8_move_slots(cache, ints([6 * 16 + 5], to), ints([2 * 16 + 5], to))
        outs.append((a.cpu(), o.kv8_read_pages(cache, ints([2, 5, 6, 7], to), torch.bfloat16).cpu()))
    settle(ops)
    assert torch.equal(outs[0][1], outs[1][1])
    # Two implementations of one formula in fp32 with 2^-11 weights and 2^-11 outputs.
    assert float((outs[0][0].float() - outs[1][0].float()).norm() / outs[1][0].float().norm()) < 2.0 ** -9
