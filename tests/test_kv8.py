"""Operators of the 8-bit KV cache against plain 64-bit implementations of their definitions.

The CPU half runs ``ops.torch_ops``, the GPU half the kernels of ``ops.cuda_ops``; both are held to the same oracles,
which are written from the definitions (explicit loops over slots and positions) and share no code with either.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import mod

F8 = torch.float8_e4m3fn
IMPLS = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float16, torch.bfloat16]


def impl(device):
    return mod("ops.torch_ops") if device == "cpu" else mod("ops.cuda_ops").CudaOps(device=torch.device("cuda"))


def settle(ops):
    if torch.cuda.is_available():
        torch.cuda.synchronize()
    ops.check()


# ------------------------------------------------------------------ oracle
def o_scale(amax: float) -> float:
    e = -40
    while amax > 448.0 * 2.0 ** e:
        e += 1
    assert e <= 56
    return 2.0 ** e


def o_code(x: torch.Tensor, scale: float) -> torch.Tensor:
    """Nearest e4m3 value of x / scale (float64, ties to even), times scale."""
    y = x.double() / scale
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y.abs().clamp_min(2.0 ** -30))[1] - 1).clamp_min(-6) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * scale


class Oracle:
    """A cache of float64 values [layers][page][side][head] -> [ps, hd] with scales."""

    def __init__(self, cache):
        self.scale = cache.scale.detach().cpu().double().clone()
        self.val = cache.data.detach().cpu().float().double() * self.scale[..., None, None]
        self.ps = self.val.shape[-2]

    def write(self, layer, side, head, page, rows):
        """rows: {offset: (values, needed scale)} of one page."""
        if not rows:
            return
        new = max(s for _, s in rows.values())
        old = float(self.scale[layer, page, side, head])
        v = self.val[layer, page, side, head]
        if 0 in rows:
            v = torch.zeros_like(v)
        else:
            new = max(new, old)
        for off, (x, _) in rows.items():
            v[off] = x
        self.val[layer, page, side, head] = o_code(v, new) if new > 0 else torch.zeros_like(v)
        self.scale[layer, page, side, head] = new


def o_rotate(x, cs):
    half = x.shape[-1] // 2
    c, s = cs[:half], cs[half:]
    return torch.cat((x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s), -1)


def o_attention(q, values, desc, scale):
    """(out, sum of weights times |v|, largest sum of |q k| scale) per row and head, float64, by positions."""
    m, hq, hd = q.shape
    hkv, ps = values.shape[2], values.shape[3]
    out = torch.zeros(m, hq, hd, dtype=torch.float64)
    mag = torch.zeros_like(out)
    err = torch.zeros(m, hq, 1, dtype=torch.float64)
    prefix, tails = desc.prefix_pages.tolist(), desc.tail_pages.tolist()
    for r in range(m):
        where = []
        for x in range(int(desc.row_len[r])):
            if x >= int(desc.row_full[r]):
                b = x - desc.mask_base
                if not 0 <= b < 64 * desc.row_mask.shape[1]:
                    continue
                if not (int(desc.row_mask[r, b // 64]) >> (b % 64)) & 1:
                    continue
            j = x // ps
            page = prefix[j] if j < desc.n_shared_pages or x < desc.shared_len else tails[r][j - desc.n_shared_pages]
            where.append((page, x % ps))
        if not where:
            continue
        pg = torch.tensor([w[0] for w in where])
        off = torch.tensor([w[1] for w in where])
        for h in range(hq):
            k = values[pg, 0, h // (hq // hkv), off]
            v = values[pg, 1, h // (hq // hkv), off]
            prod = k * q[r, h].double().cpu()
            p = torch.softmax(prod.sum(-1) * scale, 0)
            out[r, h] = p @ v
            mag[r, h] = p @ v.abs()
            err[r, h] = float(prod.abs().sum(-1).max()) * scale
    return out, mag, err


# ------------------------------------------------------------------ inputs
def make_cache(device, layers, pages, hkv, ps, hd, seed, empty=()):
    kv8 = mod("ops.kv8")
    g = torch.Generator().manual_seed(seed)
    cache = kv8.empty_cache(layers, pages, hkv, ps, hd, device=device)
    x = torch.randn(layers, pages, 2, hkv, ps, hd, generator=g)
    x *= torch.exp2(torch.randint(-6, 7, (layers, pages, 2, hkv, 1, 1), generator=g).float())
    s = kv8.needed_scale(x.abs().amax((-1, -2)))
    for page in empty:
        s[:, page] = 0
    cache.data.copy_(kv8.encode(x, s[..., None, None]))
    cache.scale.copy_(s)
    return cache


def rope(n, hd, device):
    inv = 500000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cat((ang.cos(), ang.sin()), -1).float().to(device)


def assert_pages(cache, oracle, spread=None):
    """Scales equal, and values equal except where ``spread`` (per element, float64) lets a value next to a rounding
    border fall to the neighbouring code."""
    assert torch.equal(cache.scale.cpu().double(), oracle.scale)
    got = cache.data.cpu().float().double() * oracle.scale[..., None, None]
    if spread is None:
        assert torch.equal(got, oracle.val)
        return
    assert bool(((got - oracle.val).abs() <= spread).all())


# ------------------------------------------------------------------ append
APPENDS = [
    # (page size, q heads, kv heads, slots)
    (16, 4, 2, [5]),
    (16, 8, 8, [16]),                              # starts a page
    (16, 2, 1, [13, 14, 15, 32, 33, 34]),          # over a page boundary
    (8, 6, 2, list(range(3, 40))),                 # five pages in order
    (64, 4, 4, [70, 3, 71, 2, 72, 65, 1]),         # two pages interleaved
    (32, 4, 1, [40, 40, 41, 40, 9]),               # repeated slots: the later row is kept
    (16, 5, 1, [48] * 9 + [7]),                    # padding rows share one slot
]


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("dtype", [*DTYPES, torch.float32])
@pytest.mark.parametrize("ps,hq,hkv,slots", APPENDS)
def test_append(device, dtype, ps, hq, hkv, slots):
    ops = impl(device)
    hd, m = 128, len(slots)
    cache = make_cache(device, 2, 6, hkv, ps, hd, seed=ps + m, empty=(4,))
    oracle = Oracle(cache)
    g = torch.Generator().manual_seed(m)
    qkv = torch.randn(m, (hq + 2 * hkv) * hd, generator=g)
    qkv = (qkv * torch.exp2(torch.randint(-4, 5, (m, 1), generator=g).float())).to(dtype)
    table = rope(4096, hd, device)
    pos = torch.randint(0, 4096, (m,), generator=g)
    out = torch.bfloat16 if dtype == torch.float32 else dtype
    q = ops.rope_qkv_append8(qkv.to(device), table, pos.int().to(device),
                             torch.tensor(slots, dtype=torch.int32, device=device), cache.layer(1), hq, hkv,
                             out_dtype=out)
    settle(ops)
    x = qkv.double().reshape(m, -1, hd)
    cs = table.cpu().double()
    spread = torch.zeros_like(oracle.val)
    for h in range(hkv):
        for side in (0, 1):
            by_page: dict = {}
            for i, s in enumerate(slots):
                v = x[i, hq + side * hkv + h]
                v = o_rotate(v, cs[pos[i]]) if side == 0 else v
                by_page.setdefault(s // ps, {})[s % ps] = (v, o_scale(float(v.abs().max())))
            for page, rows in by_page.items():
                oracle.write(1, side, h, page, rows)
                if side == 0:  # fp32 rotation: two products and a sum, 4 roundings of 2^-24 each
                    s = float(oracle.scale[1, page, 0, h])
                    for off, (v, _) in rows.items():
                        d = float(v.abs().max()) * 2.0 ** -20
                        spread[1, page, 0, h, off] = (o_code(v + d, s) - o_code(v - d, s)).abs()
    assert_pages(cache, oracle, spread)
    want = torch.stack([o_rotate(x[i, :hq], cs[pos[i]]) for i in range(m)])
    assert q.dtype == out and q.shape == want.shape
    tol = torch.finfo(out).eps / 2 * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True) + 2.0 ** -25
    assert bool(((q.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("device", IMPLS)
def test_append_token_by_token_keeps_earlier_rows(device):
    """Rows appended one by one, each larger than the last: the page's scale grows and every earlier row stays within
    the sum of its roundings."""
    ops = impl(device)
    hd, hkv, ps = 128, 2, 16
    kv8 = mod("ops.kv8")
    cache = kv8.empty_cache(1, 3, hkv, ps, hd, device=device)
    oracle = Oracle(cache)
    g = torch.Generator().manual_seed(3)
    table = rope(64, hd, device)
    for step in range(ps + 3):
        qkv = torch.randn(1, (2 + 2 * hkv) * hd, generator=g) * 1.7 ** step
        qkv[:, (2 + hkv) * hd:] = qkv[:, (2 + hkv) * hd:].half().float()
        slot = torch.tensor([16 + step], dtype=torch.int32, device=device)
        ops.rope_qkv_append8(qkv.to(device), table, torch.tensor([0], dtype=torch.int32, device=device), slot,
                             cache.layer(0), 2, hkv)
        for h in range(hkv):
            for side in (0, 1):  # position 0: the rotation is the identity
                v = qkv[0].double().reshape(-1, hd)[2 + side * hkv + h]
                s = 16 + step
                oracle.write(0, side, h, s // ps, {s % ps: (v, o_scale(float(v.abs().max())))})
    settle(ops)
    assert_pages(cache, oracle)


@pytest.mark.parametrize("device", IMPLS)
def test_append_extremes(device):
    """Zeros, the smallest and the largest storable rows."""
    ops = impl(device)
    hd, ps = 128, 16
    cache = mod("ops.kv8").empty_cache(1, 4, 1, ps, hd, device=device)
    oracle = Oracle(cache)
    table = rope(4, hd, device)
    sizes = [0.0, 2.0 ** -60, 2.0 ** -45, 448 * 2.0 ** -40, 448 * 2.0 ** -39 * 1.01, 1.0, 448.0, 449.0, 480.0, 2.0 ** 60]
    for i, a in enumerate(sizes):
        qkv = torch.zeros(1, 3 * hd)
        qkv[0, hd: 3 * hd] = a * torch.linspace(-1, 1, 2 * hd)
        slot = (i % 3) * ps + i // 3
        ops.rope_qkv_append8(qkv.to(device), table, torch.zeros(1, dtype=torch.int32, device=device),
                             torch.tensor([slot], dtype=torch.int32, device=device), cache.layer(0), 1, 1)
        for side in (0, 1):
            v = qkv[0, (1 + side) * hd: (2 + side) * hd].double()
            oracle.write(0, side, 0, slot // ps, {slot % ps: (v, o_scale(float(v.abs().max())))})
    settle(ops)
    assert_pages(cache, oracle)


# ------------------------------------------------------------------- pages
@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("ps", [8, 16, 64])
def test_copy_pages(device, ps):
    ops = impl(device)
    cache = make_cache(device, 3, 10, 2, ps, 128, seed=ps, empty=(7,))
    oracle = Oracle(cache)
    plan = [(0, 4, 1), (0, 5, ps), (1, 6, ps // 2), (7, 2, 3), (3, 8, 0)]
    for src, dst, n in plan:
        oracle.val[:, dst] = 0
        oracle.val[:, dst, :, :, :n] = oracle.val[:, src, :, :, :n]
        oracle.scale[:, dst] = oracle.scale[:, src] if n else 0
    ops.kv8_copy_pages(cache, torch.tensor(plan, dtype=torch.int32, device=device))
    settle(ops)
    assert_pages(cache, oracle)
    ops.kv8_copy_pages(cache, torch.empty(0, 3, dtype=torch.int32, device=device))
    settle(ops)
    assert_pages(cache, oracle)


MOVES = [
    (16, [37, 40, 44], [33, 34, 35]),              # a tree path inside its page
    (16, [20, 47, 50], [15, 16, 17]),              # over a boundary: slot 16 starts a page anew
    (8, [1, 2, 3], [2, 3, 1]),                     # a rotation: sources are read first
    (64, [5, 70, 6], [130, 130, 129]),             # a repeated destination: the later move is kept
    (32, [100], [100]),                            # onto itself
    (8, list(range(0, 48)), list(range(47, -1, -1))),
]


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("ps,src,dst", MOVES)
def test_move_slots(device, ps, src, dst):
    ops = impl(device)
    cache = make_cache(device, 2, 7, 2, ps, 128, seed=len(src), empty=(6,))
    oracle = Oracle(cache)
    before = Oracle(cache)
    for layer in range(2):
        for side in (0, 1):
            for h in range(2):
                by_page: dict = {}
                for a, b in zip(src, dst):
                    by_page.setdefault(b // ps, {})[b % ps] = (before.val[layer, a // ps, side, h, a % ps],
                                                               float(before.scale[layer, a // ps, side, h]))
                for page, rows in by_page.items():
                    oracle.write(layer, side, h, page, rows)
    ops.kv8_move_slots(cache, torch.tensor(src, device=device), torch.tensor(dst, device=device))
    settle(ops)
    assert_pages(cache, oracle)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_read_pages(device, dtype):
    ops = impl(device)
    cache = make_cache(device, 2, 6, 3, 16, 128, seed=1, empty=(2,))
    cache.scale[0, 5] = 2.0 ** 8  # 448 * 2^8 is above fp16's largest number
    oracle = Oracle(cache)
    pages = [5, 0, 2, 5]
    idx = torch.tensor(pages, dtype=torch.int32, device=device)
    lim = torch.finfo(dtype).max
    for got, want in ((ops.kv8_read_pages(cache, idx, dtype), oracle.val[:, pages]),
                      (ops.kv8_read_pages(cache.layer(1), idx, dtype), oracle.val[1, pages])):
        settle(ops)
        assert got.dtype == dtype
        assert torch.equal(got.cpu(), want.clamp(-lim, lim).to(dtype))
    assert ops.kv8_read_pages(cache.layer(0), idx[:0], dtype).shape == (0, 2, 3, 16, 128)


# --------------------------------------------------------------- attention
def make_desc(device, kind, ps, length, rows, seed, pages, depth=5):
    """A descriptor and the number of pages it names (drawn without repetition from ``pages``)."""
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(pages, generator=g).int()
    full = torch.full((rows,), length, dtype=torch.int32)
    mask = torch.full((rows, 1), -1, dtype=torch.int64)
    tails = torch.zeros(rows, 1, dtype=torch.int32)
    n = -(-(length + (rows if kind == "tree" else 1)) // ps)
    shared = n
    base = length
    if kind == "single":
        full += 1
        lens = full.clone()
    elif kind == "ragged":  # rows of one sequence that see less than all of it, the last sees nothing
        lens = torch.randint(0, length + 1, (rows,), generator=g).int()
        lens[-1] = 0
        full = lens.clone()
    elif kind == "tree":
        words = rows // 64 + 1
        lens = full + rows
        mask = torch.zeros(rows, words, dtype=torch.int64)
        for i in range(rows):
            seen = {i}
            a = i
            while a > 0:
                a = int(torch.randint(-1, a, (1,), generator=g))
                if a < 0:
                    break
                seen.add(a)
            for b in seen:
                mask[i, b // 64] |= (1 << (b % 64)) if b % 64 < 63 else -(1 << 63)
        if rows > 2:
            mask[1] = 0
            full[1] = 0  # a row whose mask leaves nothing
    else:  # routes
        shared = length // ps
        t = -(-(length % ps + depth) // ps)
        lens = full + torch.randint(1, depth + 1, (rows,), generator=g).int()
        full = lens.clone()
        tails = perm[n: n + rows * t].reshape(rows, t)
    desc = mod("ops.attn_desc").AttnDesc(
        prefix_pages=perm[:max(n, 1)].contiguous().to(device), n_shared_pages=shared, shared_len=length,
        mask_base=base, row_full=full.to(device), row_len=lens.int().to(device), row_mask=mask.to(device),
        tail_pages=tails.contiguous().to(device))
    return desc


def check_attention(out, q, cache_values, desc, scale):
    want, mag, err = o_attention(q.cpu(), cache_values, desc, scale)
    eps = torch.finfo(out.dtype).eps
    # Weights: rounded to 11 bits at worst (2^-11, and 2^-11 for the sum they are divided by), scores from fp32 sums
    # of 128 products (2^-17 of their magnitudes), exponential and sums 2^-19; then one rounding to the output's type.
    # The tensor-core path of the causal form rounds weights to the output's type (eps / 2 each).
    rel = max(2.0 ** -11, eps / 2) * 2 + 2.0 ** -16 * err + 2.0 ** -18
    tol = mag * rel + want.abs() * eps / 2 + 2.0 ** -24
    diff = (out.cpu().double().reshape(want.shape) - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())


ATTENTIONS = [
    # (kind, page size, q heads, kv heads, length, rows)
    ("single", 16, 4, 1, 0, 1),
    ("single", 16, 8, 2, 1, 1),
    ("single", 16, 8, 8, 37, 1),
    ("single", 8, 32, 8, 1023, 1),
    ("single", 64, 12, 4, 2100, 1),
    ("ragged", 16, 8, 2, 300, 9),
    ("ragged", 32, 6, 2, 65, 40),
    ("tree", 16, 8, 2, 511, 13),
    ("tree", 8, 8, 1, 160, 48),
    ("tree", 16, 4, 4, 33, 70),
    ("tree", 16, 16, 2, 0, 5),
    ("routes", 16, 8, 2, 250, 9),
    ("routes", 16, 8, 2, 256, 3),
    ("routes", 8, 4, 4, 5, 4),
    ("routes", 64, 16, 2, 700, 33),
]


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,ps,hq,hkv,length,rows", ATTENTIONS)
def test_attention(device, dtype, kind, ps, hq, hkv, length, rows):
    ops = impl(device)
    pages = 4 + -(-(length + rows + 1) // ps) + (rows * 2 if kind == "routes" else 0)
    desc = make_desc(device, kind, ps, length, rows, seed=length + rows, pages=pages)
    cache = make_cache(device, 2, pages, hkv, ps, 128, seed=length)
    g = torch.Generator().manual_seed(rows)
    q = torch.randn(rows, hq, 128, generator=g).to(dtype)
    out = ops.attention8(q.to(device), cache.layer(1), desc)
    settle(ops)
    assert out.shape == (rows, hq * 128) and out.dtype == dtype
    check_attention(out, q, Oracle(cache).val[1], desc, 1 / math.sqrt(128))


@pytest.mark.parametrize("device", IMPLS)
def test_attention_scale_and_sharp_scores(device):
    """A softmax scale of the caller's, scores whose softmax is one-hot, V pages 2^12 apart in size."""
    ops = impl(device)
    cache = make_cache(device, 1, 40, 2, 16, 128, seed=0)
    cache.scale[0, 3:9, 1] *= 2.0 ** 12
    cache.scale[0, 20, 1] *= 2.0 ** -12
    desc = make_desc(device, "tree", 16, 400, 7, seed=2, pages=40)
    q = torch.randn(7, 4, 128, generator=torch.Generator().manual_seed(1)).half()
    for scale in (0.7, 1e-4):
        out = ops.attention8(q.to(device), cache.layer(0), desc, scale)
        settle(ops)
        check_attention(out, q, Oracle(cache).val[0], desc, scale)


@pytest.mark.parametrize("device", IMPLS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps,hq,hkv,start,rows", [(16, 4, 2, 0, 1), (16, 8, 2, 0, 45), (8, 8, 8, 77, 30),
                                                  (32, 16, 2, 300, 129), (64, 4, 4, 13, 64),
                                                  (16, 8, 2, 1500, 3), (16, 4, 2, 900, 70)])
def test_attention_causal(device, dtype, ps, hq, hkv, start, rows):
    ops = impl(device)
    pages = 4 + -(-(start + rows) // ps)
    cache = make_cache(device, 1, pages, hkv, ps, 128, seed=start)
    g = torch.Generator().manual_seed(rows)
    order = torch.randperm(pages, generator=g)[: pages - 3].int()
    limit = torch.arange(start + 1, start + rows + 1, dtype=torch.int32)
    desc = mod("ops.attn_desc").single_sequence_desc(order.to(device), limit.to(device), start)
    q = torch.randn(rows, hq, 128, generator=g).to(dtype)
    out = ops.attention8_causal(q.to(device), cache.layer(0), desc, start)
    settle(ops)
    check_attention(out, q, Oracle(cache).val[0], desc, 1 / math.sqrt(128))
