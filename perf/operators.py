"""Operators of the 8-bit paged KV cache: what is measured, in plain torch and through the framework.

The cache holds K and V as e4m3 codes ``data [layers, pages, 2, kv_heads, page_size, 128]`` with one power-of-two
scale per page, side (k, v) and head, ``scale [layers, pages, 2, kv_heads]``: an element stands for code * scale, and
a scale of 0 marks a page that holds nothing.  Every operator below reads or updates such a cache:

- ``append``: rotate a batch's q and k, round k and v to the cache's codes and write them at the rows' slots;
- ``attend``: attention of a few rows over the pages (one token, drafter routes with private tail pages, a masked tree);
- ``prefill``: causal attention of a chunk whose own keys are already in the pages;
- ``fork`` / ``compact``: copy partial pages to private ones / move selected slots together, in every layer.
"""

import importlib
import math

import torch

own = False  # True: run() calls the framework's operators instead of the plain forms

HD = 128            # the head dimension the framework's GPU kernels are built for
E4M3_MAX = 448.0
E_MIN, E_MAX = -40, 56  # exponents a page's scale may take
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ----------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One decoded token of an 8B-shaped model: the smallest append there is.
        {"name": "append one token", "op": "append", "rows": 1, "hq": 32, "hkv": 8, "page": 16, "start": 1029,
         "qkv": "float16", "dtype": "float16"},
        # The nodes of a verify tree, from the fp32 output of the folded-norm QKV product, over a page boundary.
        {"name": "append tree nodes", "op": "append", "rows": 13, "hq": 32, "hkv": 8, "page": 16, "start": 16377,
         "qkv": "float32", "dtype": "float16"},
        # A prompt chunk of odd length.
        {"name": "append prompt chunk", "op": "append", "rows": 5001, "hq": 32, "hkv": 8, "page": 16, "start": 0,
         "qkv": "bfloat16", "dtype": "bfloat16"},
        # A conversation's first words: latency only.
        {"name": "attend first tokens", "op": "attend", "kind": "single", "rows": 1, "hq": 32, "hkv": 8, "page": 16,
         "length": 37, "depth": 0, "dtype": "float16", "empty": False},
        # Nine drafter routes (k = 3, second stage) on one prefix, each with its private tail page.
        {"name": "attend nine routes", "op": "attend", "kind": "routes", "rows": 9, "hq": 32, "hkv": 8, "page": 16,
         "length": 2051, "depth": 6, "dtype": "float16", "empty": False},
        # A deduplicated verify tree of 48 nodes behind a 16k prefix.
        {"name": "attend tree 16k", "op": "attend", "kind": "tree", "rows": 48, "hq": 32, "hkv": 8, "page": 16,
         "length": 16384, "depth": 0, "dtype": "float16", "empty": False},
        # A 13-node tree in 70B head geometry (groups of 8), odd prefix.
        {"name": "attend tree 33k", "op": "attend", "kind": "tree", "rows": 13, "hq": 64, "hkv": 8, "page": 16,
         "length": 33001, "depth": 0, "dtype": "bfloat16", "empty": True},
        # One token behind a long context: the cache's bytes are all that counts.
        {"name": "attend long context", "op": "attend", "kind": "single", "rows": 1, "hq": 32, "hkv": 8, "page": 16,
         "length": 131077, "depth": 0, "dtype": "bfloat16", "empty": False},
        # A short prompt in one chunk.
        {"name": "prefill short prompt", "op": "prefill", "rows": 301, "hq": 32, "hkv": 8, "page": 16, "start": 0,
         "dtype": "float16"},
        # A later chunk of a long prompt.
        {"name": "prefill later chunk", "op": "prefill", "rows": 2048, "hq": 32, "hkv": 8, "page": 16, "start": 6001,
         "dtype": "bfloat16"},
        # Nine routes copy the prefix's partial page in the 16 layers of a 1B-shaped drafter.
        {"name": "fork nine routes", "op": "fork", "count": 9, "hkv": 8, "page": 16, "layers": 16, "pages": 256},
        # The accepted path of a tree moves behind the prefix in the 32 layers of an 8B-shaped target.
        {"name": "compact tree path", "op": "compact", "count": 4, "nodes": 39, "hkv": 8, "page": 16, "layers": 32,
         "pages": 1040, "prefix": 16371},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "prefill", "fork", "compact"))
    hkv = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 4, 8))
    page = rng.choice((8, 16, 16, 32, 64))
    dtype = rng.choice(("float16", "bfloat16"))
    case = {"op": op, "hkv": hkv, "page": page}
    if op == "append":
        rows = _log_int(rng, 1, 5000)
        case.update(rows=rows, hq=hkv * group, start=rng.randrange(0, 20000), dtype=dtype,
                    qkv=rng.choice((dtype, "float32")) if rows <= 64 else dtype)
    elif op == "attend":
        kind = rng.choice(("single", "routes", "tree"))
        rows = 1 if kind == "single" else _log_int(rng, 2, 32 if kind == "routes" else 64)
        case.update(kind=kind, rows=rows, hq=hkv * group, length=_log_int(rng, 1, 131000 if rows == 1 else 16000),
                    depth=rng.randrange(1, 12) if kind == "routes" else 0, dtype=dtype,
                    empty=kind != "single" and rng.random() < 0.3)
    elif op == "prefill":
        rows = _log_int(rng, 2, 1000)
        case.update(rows=rows, hq=hkv * group, start=rng.choice((0, rng.randrange(1, 5000))), dtype=dtype)
    elif op == "fork":
        count = _log_int(rng, 1, 32)
        case.update(count=count, layers=rng.choice((2, 4, 16)), pages=2 * count + rng.randrange(10, 200))
    else:
        nodes = rng.randrange(2, 64)
        prefix = _log_int(rng, 1, 6000)
        case.update(count=rng.randrange(1, min(nodes, 12)), nodes=nodes, layers=rng.choice((2, 4, 16, 32)),
                    prefix=prefix, pages=(prefix + nodes) // page + 2 + rng.randrange(0, 50))
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _exponent(amax):
    """Smallest e in [E_MIN, E_MAX] with amax <= 448 * 2^e (448 = 0.875 * 2^9), exactly."""
    m, ex = torch.frexp(amax)
    e = torch.where(m <= 0.875, ex - 9, ex - 8)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _pow2(e):
    """2^e for whole e, exactly (built from the bits: exp2 may be off by one)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _cache(g, layers, pages, hkv, page):
    """A filled cache: every page's elements are normal, with a size of their own per page, side and head."""
    dev = "cuda"
    size = torch.exp2(torch.randn(layers, pages, 2, hkv, 1, 1, device=dev, generator=g))
    data = torch.empty(layers, pages, 2, hkv, page, HD, device=dev, dtype=torch.float8_e4m3fn)
    scale = torch.empty(layers, pages, 2, hkv, device=dev)
    for layer in range(layers):
        x = torch.randn(pages, 2, hkv, page, HD, device=dev, generator=g) * size[layer]
        s = _pow2(_exponent(x.abs().amax(dim=(3, 4))))
        data[layer] = (x / s[..., None, None]).to(torch.float8_e4m3fn)
        scale[layer] = s
    return data, scale


def _rope_table(positions):
    """cos | sin of every position, angles in 64 bits (theta 500000)."""
    inv = 500000.0 ** (-torch.arange(HD // 2, dtype=torch.float64, device="cuda") * 2.0 / HD)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat((ang.cos(), ang.sin()), dim=-1).float()


def _slots(pages, positions, page):
    return pages[positions // page] * page + positions % page


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, hkv, ps = case["op"], case["hkv"], case["page"]
    st = {"case": case}
    if op == "append":
        rows, hq, start = case["rows"], case["hq"], case["start"]
        first, last = start // ps, (start + rows - 1) // ps
        need = last - first + 1
        data, scale = _cache(g, 1, need + 7, hkv, ps)
        own_pages = torch.randperm(need + 7, device="cuda", generator=g)[:need]  # the sequence's pages, any order
        pos = torch.arange(start, start + rows, device="cuda")
        slots = own_pages[pos // ps - first] * ps + pos % ps
        qkv = torch.randn(rows, (hq + 2 * hkv) * HD, device="cuda", generator=g)
        qkv *= torch.exp2(torch.randn(rows, 1, device="cuda", generator=g))
        st.update(data=data, scale=scale, qkv=qkv.to(DTYPES[case["qkv"]]), table=_rope_table(start + rows),
                  positions=pos.int(), slots=slots.int(), touched=torch.sort(own_pages).values.int())
    elif op == "attend":
        rows, hq, n, kind = case["rows"], case["hq"], case["length"], case["kind"]
        extra = rows if kind == "tree" else (1 if kind == "single" else 0)
        n_pages = (n + extra + ps - 1) // ps
        tail = (n % ps + case["depth"] + ps - 1) // ps if kind == "routes" else 0
        total = n_pages + rows * tail
        data, scale = _cache(g, 1, total + 3, hkv, ps)
        perm = torch.randperm(total + 3, device="cuda", generator=g).int()
        prefix = perm[:n_pages].contiguous()
        q = torch.randn(rows, hq, HD, device="cuda", generator=g).to(DTYPES[case["dtype"]])
        st.update(data=data, scale=scale, q=q, prefix=prefix, shared_len=n, mask_base=n)
        full = torch.full((rows,), n, device="cuda", dtype=torch.int32)
        mask = torch.full((rows, 1), -1, device="cuda", dtype=torch.int64)
        tails = torch.zeros(rows, 1, device="cuda", dtype=torch.int32)
        st["n_shared"] = n_pages
        if kind == "single":
            full += 1
            lens = full.clone()
        elif kind == "tree":  # node i sees itself and its chain of parents, parents drawn among earlier nodes
            lens = full + rows
            up = torch.Generator().manual_seed(seed)
            seen = []
            for i in range(rows):
                parent = int(torch.randint(-1, i, (1,), generator=up)) if i else -1
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
            seen = [v - (1 << 64) if v >= 1 << 63 else v for v in seen]
            mask = torch.tensor(seen, dtype=torch.int64, device="cuda").reshape(rows, 1)
        else:  # routes: whole pages of the prefix are shared, the rest of it and the route's tokens are private
            st["n_shared"] = n // ps
            lens = (full + 1 + torch.arange(rows, device="cuda", dtype=torch.int32) % case["depth"]).int()
            full = lens.clone()
            tails = perm[n_pages: n_pages + rows * tail].reshape(rows, tail).contiguous()
        if case["empty"]:  # a row without a key, as padding rows may be
            full[-1] = 0
            lens[-1] = 0
        st.update(row_full=full, row_len=lens, row_mask=mask, tails=tails)
    elif op == "prefill":
        rows, hq, start = case["rows"], case["hq"], case["start"]
        n_pages = (start + rows + ps - 1) // ps
        data, scale = _cache(g, 1, n_pages + 3, hkv, ps)
        prefix = torch.randperm(n_pages + 3, device="cuda", generator=g)[:n_pages].int()
        q = torch.randn(rows, hq, HD, device="cuda", generator=g).to(DTYPES[case["dtype"]])
        limit = torch.arange(start + 1, start + rows + 1, device="cuda", dtype=torch.int32)
        st.update(data=data, scale=scale, q=q, prefix=prefix, shared_len=start, mask_base=0, n_shared=n_pages,
                  row_full=limit, row_len=limit.clone(), start=start,
                  row_mask=torch.full((rows, 1), -1, device="cuda", dtype=torch.int64),
                  tails=torch.zeros(rows, 1, device="cuda", dtype=torch.int32))
    elif op == "fork":
        data, scale = _cache(g, case["layers"], case["pages"], hkv, ps)
        perm = torch.randperm(case["pages"], device="cuda", generator=g)
        count = case["count"]
        ntok = torch.randint(1, ps + 1, (count,), device="cuda", generator=g)
        dst = perm[:count]
        src = perm[count + torch.randint(0, count, (count,), device="cuda", generator=g)]  # forks share a source
        st.update(data=data, scale=scale, copies=torch.stack((src, dst, ntok), dim=1).int(),
                  touched=torch.sort(dst).values.int())
    else:
        data, scale = _cache(g, case["layers"], case["pages"], hkv, ps)
        prefix, nodes, count = case["prefix"], case["nodes"], case["count"]
        pages = torch.randperm(case["pages"], device="cuda", generator=g)
        path = torch.sort(torch.randperm(nodes - 1, device="cuda", generator=g)[:count] + 1).values  # never node 0 first
        src = _slots(pages, prefix + path, ps)
        dst = _slots(pages, prefix + torch.arange(count, device="cuda"), ps)
        last = (prefix + nodes - 1) // ps
        st.update(data=data, scale=scale, src=src.int(), dst=dst.int(),
                  touched=torch.sort(pages[prefix // ps: last + 1]).values.int())
    return st


# ----------------------------------------------------------------------------------------------- plain forms
def _values(data, scale):
    return data.float() * scale[..., None, None]


def _write(data, scale, rows, slots, touched):
    """Round ``rows`` [n, layers, 2, hkv, hd] to codes at ``slots`` of the pages ``touched`` and update both tensors.

    A page's scale grows to what its new rows need, and what else the page holds is rounded again; a page whose slot 0
    is written starts anew: its scale is that of its new rows, its other slots are zero.
    """
    ps = data.shape[-2]
    at = torch.searchsorted(touched.long(), slots.long() // ps)
    n, layers, _, hkv, _ = rows.shape
    need = _exponent(rows.abs().amax(-1)).float()  # [n, layers, 2, hkv]
    low = torch.full((touched.numel(), layers, 2, hkv), float(E_MIN), device=rows.device)
    e = low.scatter_reduce(0, at[:, None, None, None].expand_as(need), need, "amax")
    anew = torch.zeros(touched.numel(), device=rows.device).scatter_reduce(0, at, (slots % ps == 0).float(), "amax") > 0
    anew = anew[None, :, None, None]
    e = e.transpose(0, 1)  # [layers, pages, 2, hkv]
    old = scale[:, touched.long()]
    s = torch.where(anew, _pow2(e), torch.maximum(old, _pow2(e)))
    held = torch.where(anew[..., None, None], torch.zeros((), device=rows.device),
                       _values(data[:, touched.long()], old))
    held = held.permute(1, 4, 0, 2, 3, 5).contiguous()  # [pages, ps, layers, 2, hkv, hd]
    held[at, slots.long() % ps] = rows
    held = held.permute(2, 0, 3, 4, 1, 5)
    data[:, touched.long()] = (held / s[..., None, None]).to(torch.float8_e4m3fn)
    scale[:, touched.long()] = s


def _rotate(x, cs):
    half = HD // 2
    c, s = cs[:, None, :half], cs[:, None, half:]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def _plain_append(st):
    case = st["case"]
    hq, hkv = case["hq"], case["hkv"]
    x = st["qkv"].float().reshape(case["rows"], hq + 2 * hkv, HD)
    cs = st["table"][st["positions"].long()]
    q = _rotate(x[:, :hq], cs).to(DTYPES[case["dtype"]])
    kv = torch.stack((_rotate(x[:, hq: hq + hkv], cs), x[:, hq + hkv:]), dim=1)  # [rows, 2, hkv, hd]
    _write(st["data"], st["scale"], kv[:, None], st["slots"], st["touched"])
    t = st["touched"].long()
    return {"q": q, "pages": _values(st["data"][0, t], st["scale"][0, t]).to(torch.bfloat16)}


def _plain_attention(st, causal):
    q = st["q"].float()
    rows, hq, _ = q.shape
    hkv, ps = st["data"].shape[3], st["data"].shape[4]
    q = q.reshape(rows, hkv, hq // hkv, HD) / math.sqrt(HD)
    shared = _values(st["data"][0, st["prefix"].long()], st["scale"][0, st["prefix"].long()])
    k, v = (shared[:, i].transpose(0, 1).reshape(hkv, -1, HD) for i in (0, 1))  # [hkv, keys, hd]
    x = torch.arange(k.shape[1], device=q.device)
    full, lens = st["row_full"].long()[:, None], st["row_len"].long()[:, None]
    if causal:
        seen = x[None] < full
    else:
        bit = (x - st["mask_base"]).clamp(0, 63)
        marked = ((st["row_mask"] >> bit[None]) & 1).bool() & (x >= st["mask_base"])
        seen = (x < full) | ((x < lens) & marked)
        seen &= (x // ps < st["n_shared"]) | (x < st["shared_len"])
    scores = torch.einsum("rhgd,hkd->rhgk", q, k).masked_fill(~seen[:, None, None], -math.inf)
    if st["case"].get("kind") == "routes":
        tail = _values(st["data"][0, st["tails"].long()], st["scale"][0, st["tails"].long()])  # [rows, T, 2, hkv, ps, hd]
        tk, tv = (tail[:, :, i].transpose(1, 2).reshape(rows, hkv, -1, HD) for i in (0, 1))
        y = st["n_shared"] * ps + torch.arange(tk.shape[2], device=q.device)
        private = (y < lens) & (y >= st["shared_len"])
        more = torch.einsum("rhgd,rhkd->rhgk", q, tk).masked_fill(~private[:, None, None], -math.inf)
        scores = torch.cat((scores, more), dim=-1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)  # a row without keys answers zero
    out = torch.einsum("rhgk,hkd->rhgd", p[..., : k.shape[1]], v)
    if p.shape[-1] > k.shape[1]:
        out = out + torch.einsum("rhgk,rhkd->rhgd", p[..., k.shape[1]:], tv)
    return {"out": out.reshape(rows, hq * HD).to(st["q"].dtype)}


def _plain_fork(st):
    src, dst, ntok = st["copies"].long().unbind(1)
    ps = st["data"].shape[-2]
    keep = torch.arange(ps, device=src.device)[None, :] < ntok[:, None]
    codes = torch.where(keep[None, :, None, None, :, None], st["data"][:, src].float(), 0.0)
    st["data"][:, dst] = codes.to(torch.float8_e4m3fn)
    st["scale"][:, dst] = st["scale"][:, src]
    t = st["touched"].long()
    return {"pages": _values(st["data"][:, t], st["scale"][:, t]).to(torch.bfloat16)}


def _plain_compact(st):
    data, scale = st["data"], st["scale"]
    ps = data.shape[-2]
    src, dst, touched = st["src"].long(), st["dst"].long(), st["touched"].long()
    at = torch.searchsorted(touched, dst // ps)
    codes = data[:, src // ps, :, :, src % ps].float()  # [n, layers, 2, hkv, hd]
    from_scale = scale[:, src // ps].transpose(0, 1)    # [n, layers, 2, hkv]
    grown = torch.zeros_like(scale[:, touched]).transpose(0, 1).scatter_reduce(
        0, at[:, None, None, None].expand_as(from_scale), from_scale, "amax").transpose(0, 1)
    hit = torch.zeros(touched.numel(), device=src.device).scatter_reduce(0, at, (dst % ps == 0).float(), "amax") > 0
    anew = hit[None, :, None, None]
    old = scale[:, touched]
    s = torch.where(anew, grown, torch.maximum(old, grown))
    held = torch.where(anew[..., None, None], torch.zeros((), device=src.device), _values(data[:, touched], old))
    held = held.permute(1, 4, 0, 2, 3, 5).contiguous()
    held[at, dst % ps] = codes * from_scale[..., None]
    held = held.permute(2, 0, 3, 4, 1, 5)
    data[:, touched] = (held / s[..., None, None]).to(torch.float8_e4m3fn)
    scale[:, touched] = s
    return {"pages": _values(data[:, touched], scale[:, touched]).to(torch.bfloat16)}


# ------------------------------------------------------------------------------------- the framework's calls
def _package(name):
    return importlib.import_module("0709_b200." + name)


def _own(st):
    case = st["case"]
    ops = _package("ops.cuda_ops").shared_ops(st["data"].device)
    cache = _package("ops.kv8").Kv8Cache(st["data"], st["scale"])
    op = case["op"]
    if op == "append":
        layer = cache.layer(0)
        q = ops.rope_qkv_append8(st["qkv"], st["table"], st["positions"], st["slots"], layer, case["hq"], case["hkv"],
                                 out_dtype=DTYPES[case["dtype"]])
        return {"q": q, "pages": ops.kv8_read_pages(layer, st["touched"], torch.bfloat16)}
    if op in ("attend", "prefill"):
        desc = _package("ops.attn_desc").AttnDesc(
            prefix_pages=st["prefix"], n_shared_pages=st["n_shared"], shared_len=st["shared_len"],
            mask_base=st["mask_base"], row_full=st["row_full"], row_len=st["row_len"], row_mask=st["row_mask"],
            tail_pages=st["tails"])
        if op == "prefill":
            return {"out": ops.attention8_causal(st["q"], cache.layer(0), desc, st["start"])}
        return {"out": ops.attention8(st["q"], cache.layer(0), desc)}
    if op == "fork":
        ops.kv8_copy_pages(cache, st["copies"])
    else:
        ops.kv8_move_slots(cache, st["src"], st["dst"])
    return {"pages": ops.kv8_read_pages(cache, st["touched"], torch.bfloat16)}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "append":
        return _plain_append(state)
    if op in ("attend", "prefill"):
        return _plain_attention(state, causal=op == "prefill")
    return _plain_fork(state) if op == "fork" else _plain_compact(state)


# ------------------------------------------------------------------------------------------------------ work
def work(case):
    op, hkv, ps = case["op"], case["hkv"], case["page"]
    page_head = ps * HD + 4  # one page of one head and side: codes and their scale
    if op == "append":
        rows, hq = case["rows"], case["hq"]
        pages = (case["start"] + rows - 1) // ps - case["start"] // ps + 1
        in_b = {"float32": 4}.get(case["qkv"], 2)
        b = rows * (hq + 2 * hkv) * HD * in_b + rows * (HD * 4 + 8) + rows * hq * HD * 2  # qkv, angles, indices; q
        b += rows * 2 * hkv * HD + pages * 2 * hkv * 8                                      # codes; scales read, written
        b += pages * 2 * hkv * (page_head + ps * HD * 2)                                    # the touched pages read back
        return {"bytes": b, "flops": 3 * rows * (hq + hkv) * HD}
    if op == "attend":
        rows, hq, n = case["rows"], case["hq"], case["length"]
        tail = case["depth"] + n % ps if case["kind"] == "routes" else 0
        keys = n + (rows if case["kind"] == "tree" else 1 if case["kind"] == "single" else 0)
        b = (keys + rows * tail) * 2 * hkv * (HD + 4 / ps) + 2 * rows * hq * HD * 2 + keys / ps * 4 + rows * 20
        return {"bytes": b, "flops": 4 * rows * hq * HD * (keys + tail)}
    if op == "prefill":
        rows, hq, start = case["rows"], case["hq"], case["start"]
        b = (start + rows) * 2 * hkv * (HD + 4 / ps) + 2 * rows * hq * HD * 2 + (start + rows) / ps * 4
        return {"bytes": b, "flops": 4 * hq * HD * (rows * start + rows * (rows + 1) / 2)}
    heads = case["layers"] * 2 * hkv
    if op == "fork":
        return {"bytes": case["count"] * heads * (2 * page_head + page_head + ps * HD * 2), "flops": 0}
    pages = (case["prefix"] + case["nodes"] - 1) // ps - case["prefix"] // ps + 1
    return {"bytes": heads * (2 * case["count"] * (HD + 4) + pages * (page_head + ps * HD * 2)), "flops": 0}


# --------------------------------------------------------------------------------------------------- 64 bits
def _exact_pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_code(x, scale):
    """x / scale rounded to the nearest e4m3 number (ties to even), by its definition: 4 significant bits, smallest
    step 2^-9."""
    y = x / scale
    mag = y.abs().clamp_min(2.0 ** -40)
    exponent = torch.frexp(mag)[1].double() - 1  # floor(log2)
    step = _exact_pow2(exponent.clamp_min(-6.0) - 3.0)
    r = torch.round(y / step) * step
    return r.clamp(-E4M3_MAX, E4M3_MAX) * scale


def _exact_scale(amax):
    e = torch.ceil(torch.log2(amax.clamp_min(1e-30) / E4M3_MAX) - 1e-13)
    return _exact_pow2(e.clamp(E_MIN, E_MAX))


def _exact_pages(st, rows_of, touched, ps):
    """The touched pages after writes: rows_of[page] = {offset: ([layers, 2, hkv, hd] values, [layers, 2, hkv] scales)}."""
    out = []
    for page in touched:
        new = rows_of.get(page, {})
        old_s = st["scale"][:, page].double()
        old_v = st["data"][:, page].double() * old_s[..., None, None]
        if not new:
            out.append(old_v)
            continue
        s = torch.stack([sc for _, sc in new.values()]).amax(0)
        if 0 in new:
            page_v = torch.zeros_like(old_v)
        else:
            s = torch.maximum(s, old_s)
            page_v = old_v
        page_v = page_v.clone()
        for off, (val, _) in new.items():
            page_v[:, :, :, off] = val
        out.append(_exact_code(page_v, s[..., None, None]))
    return torch.stack(out)


def exact(case, seed):
    st = prepare(case, seed)
    op, ps = case["op"], case["page"]
    if op == "append":
        hq, hkv, half = case["hq"], case["hkv"], HD // 2
        x = st["qkv"].double().reshape(case["rows"], hq + 2 * hkv, HD)
        cs = st["table"].double()[st["positions"].long()][:, None]
        turned = torch.empty_like(x)
        turned[..., :half] = x[..., :half] * cs[..., :half] - x[..., half:] * cs[..., half:]
        turned[..., half:] = x[..., half:] * cs[..., :half] + x[..., :half] * cs[..., half:]
        kv = torch.stack((turned[:, hq: hq + hkv], x[:, hq + hkv:]), dim=1)[:, None]  # [rows, 1, 2, hkv, hd]
        scales = _exact_scale(kv.abs().amax(-1))
        rows_of = {}
        for i, slot in enumerate(st["slots"].tolist()):
            rows_of.setdefault(slot // ps, {})[slot % ps] = (kv[i], scales[i])
        return {"q": turned[:, :hq], "pages": _exact_pages(st, rows_of, st["touched"].tolist(), ps)[:, 0]}
    if op in ("fork", "compact"):
        touched = st["touched"].tolist()
        if op == "fork":
            made = {}
            for src, dst, n in st["copies"].tolist():
                v = st["data"][:, src].double() * st["scale"][:, src].double()[..., None, None]
                v[:, :, :, n:] = 0.0
                made[dst] = v
            pages = torch.stack([made[p] for p in touched])
        else:
            rows_of = {}
            for a, b in zip(st["src"].tolist(), st["dst"].tolist()):
                s = st["scale"][:, a // ps].double()
                v = st["data"][:, a // ps, :, :, a % ps].double() * s[..., None]
                rows_of.setdefault(b // ps, {})[b % ps] = (v, s)
            pages = _exact_pages(st, rows_of, touched, ps)
        return {"pages": pages.transpose(0, 1)}
    # attention, one kv head at a time
    rows, hq, _ = st["q"].shape
    hkv = case["hkv"]
    group = hq // hkv
    out = torch.zeros(rows, hq, HD, dtype=torch.float64, device="cuda")
    keys = st["prefix"].numel() * ps
    pos = torch.arange(keys, device="cuda").expand(rows, keys)
    page = st["prefix"].long()[pos // ps]
    if op == "attend" and case["kind"] == "routes":  # every row's own walk over its positions
        keys = int(st["row_len"].max())
        pos = torch.arange(keys, device="cuda").expand(rows, keys)
        j = pos // ps
        mine = (j >= st["n_shared"]) & (pos >= st["shared_len"])
        page = torch.where(mine, torch.gather(st["tails"].long(), 1,
                                              (j - st["n_shared"]).clamp(0, st["tails"].shape[1] - 1)),
                           st["prefix"].long()[j.clamp(max=st["prefix"].numel() - 1)])
    see = pos < st["row_full"][:, None]
    if op == "attend":
        bits = torch.gather(st["row_mask"], 1, torch.zeros_like(pos))
        rel = pos - st["mask_base"]
        see = see | ((rel >= 0) & (pos < st["row_len"][:, None]) & (((bits >> rel.clamp(0, 63)) & 1) == 1))
    one_list = not (op == "attend" and case["kind"] == "routes")
    for h in range(hkv):
        def side(i, pg, ps_off):
            return st["data"][0, pg, i, h, ps_off].double() * st["scale"][0, pg, i, h].double()[..., None]
        q = st["q"][:, h * group: (h + 1) * group].double()
        if one_list:
            k, v = side(0, page[0], pos[0] % ps), side(1, page[0], pos[0] % ps)
            w = torch.matmul(q, k.t()) / math.sqrt(HD)
        else:
            k, v = side(0, page, pos % ps), side(1, page, pos % ps)
            w = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(HD)
        w = w.masked_fill(~see[:, None], -math.inf)
        w = torch.where(see.any(1)[:, None, None], torch.softmax(w, dim=-1), torch.zeros((), device="cuda",
                                                                                         dtype=torch.float64))
        out[:, h * group: (h + 1) * group] = torch.matmul(w, v)
    return {"out": out.reshape(rows, hq * HD)}
