"""PyTorch implementations of every kernel's semantics on the paged KV layout.

These run the CPU configuration (fp32 tiny models) and serve as the
per-kernel numerics reference for the CUDA kernels.  KV cache layout for all
paths: ``[layers, pages, 2 (k, v), kv_heads, page_size, head_dim]``.

Reference counterparts of the op semantics: the manual Llama layer around FlashInfer
(src/atlas_0709/flashinfer_full_verify.py:1183-1231), its suffix KV write (:1027-1044),
``topk_logprobs`` (src/atlas_0709/flashinfer_paged/utils.py:11-25) and the tail-page
copy-on-write of the route pool (src/atlas_0709/flashinfer_paged/sglang_runtime.py:708-798).
"""

from __future__ import annotations

import math

import torch

from ..models.llama import GU_BLOCK
from . import kv8
from .attn_desc import AttnDesc


def check() -> None:
    """The CUDA op table's error-flag check; PyTorch ops raise where they fail, so there is nothing to read."""
    return None


def embed(tokens: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    return table[tokens.long()].float()


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out_dtype: torch.dtype) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()).to(out_dtype)


def linear(x: torch.Tensor, w: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    y = x.float() @ w.float().t()
    return y.to(out_dtype or x.dtype)


def linear_residual(x: torch.Tensor, w: torch.Tensor, resid: torch.Tensor) -> torch.Tensor:
    return resid + x.float() @ w.float().t()


def gate_up_silu(x: torch.Tensor, wgu: torch.Tensor) -> torch.Tensor:
    y = x.float() @ wgu.float().t()  # [M, 2F] interleaved in blocks
    m = y.shape[0]
    y = y.reshape(m, -1, 2, GU_BLOCK)
    act = torch.nn.functional.silu(y[:, :, 0]) * y[:, :, 1]
    return act.reshape(m, -1).to(x.dtype)


def _slot_to_page(slots: torch.Tensor, page_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    s = slots.long()
    return s // page_size, s % page_size


def rope_qkv_append(
    qkv: torch.Tensor,
    table: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    kv_layer: torch.Tensor,
    num_heads: int,
    num_kv_heads: int,
) -> torch.Tensor:
    """Rotate q/k, write k and v into the paged cache at ``slots``; return rotated q [M, Hq, hd]."""
    m = qkv.shape[0]
    hd = kv_layer.shape[-1]
    ps = kv_layer.shape[-2]
    q = qkv[:, : num_heads * hd].reshape(m, num_heads, hd)
    k = qkv[:, num_heads * hd: (num_heads + num_kv_heads) * hd].reshape(m, num_kv_heads, hd)
    v = qkv[:, (num_heads + num_kv_heads) * hd:].reshape(m, num_kv_heads, hd)
    half = hd // 2
    cs = table[positions.long()]
    cos, sin = cs[:, None, :half], cs[:, None, half:]

    def rot(x: torch.Tensor) -> torch.Tensor:
        x1, x2 = x[..., :half].float(), x[..., half:].float()
        return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), dim=-1)

    qr = rot(q).to(qkv.dtype)
    kr = rot(k).to(kv_layer.dtype)
    page, off = _slot_to_page(slots, ps)
    kv_layer[page, 0, :, off] = kr
    kv_layer[page, 1, :, off] = v.to(kv_layer.dtype)
    return qr


def _row_positions(desc: AttnDesc, r: int, page_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Visible key positions of row r and their physical slots."""
    n = int(desc.row_len[r])
    pos = torch.arange(n, device=desc.row_len.device)
    full = int(desc.row_full[r])
    vis = pos < full
    if n > full:
        rel = pos - desc.mask_base
        words = desc.row_mask[r]
        inside = (rel >= 0) & (rel < 64 * words.numel())  # no bit, no key
        rel = rel[inside]
        bit = torch.zeros_like(vis)
        bit[inside] = torch.bitwise_and(torch.bitwise_right_shift(words[rel // 64], rel % 64), 1).bool()
        vis = vis | ((pos >= full) & bit)
    pos = pos[vis]
    j = pos // page_size
    shared = (j < desc.n_shared_pages) | (pos < desc.shared_len)
    pages = torch.empty_like(j)
    pages[shared] = desc.prefix_pages.long()[j[shared]]
    if (~shared).any():
        pages[~shared] = desc.tail_pages[r].long()[j[~shared] - desc.n_shared_pages]
    if bool((pages < 0).any()):
        raise IndexError(f"row {r} reads a negative page")
    return pos, pages * page_size + pos % page_size


def attention(q: torch.Tensor, kv_layer: torch.Tensor, desc: AttnDesc, scale: float | None = None) -> torch.Tensor:
    """Paged GQA attention per the descriptor; returns [M, Hq * hd] in q's dtype."""
    m, hq, hd = q.shape
    hkv, ps = kv_layer.shape[2], kv_layer.shape[3]
    group = hq // hkv
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    flat_k = kv_layer[:, 0].permute(0, 2, 1, 3).reshape(-1, hkv, hd)  # [pages*ps, Hkv, hd]
    flat_v = kv_layer[:, 1].permute(0, 2, 1, 3).reshape(-1, hkv, hd)
    out = torch.empty(m, hq, hd, dtype=torch.float32, device=q.device)
    for r in range(m):
        _, slots = _row_positions(desc, r, ps)
        k = flat_k[slots.long()].float().repeat_interleave(group, dim=1)  # [n, Hq, hd]
        v = flat_v[slots.long()].float().repeat_interleave(group, dim=1)
        s = torch.einsum("hd,nhd->hn", q[r].float(), k) * scale
        p = torch.softmax(s, dim=-1)
        out[r] = torch.einsum("hn,nhd->hd", p, v)
    return out.reshape(m, hq * hd).to(q.dtype)


def lm_head(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return x.float() @ w.float().t()


def kv_copy_pages(kv: torch.Tensor, copies: torch.Tensor) -> None:
    """For each (src page, dst page, ntok): copy the first ntok slots in every layer."""
    for src, dst, n in copies.tolist():
        kv[:, dst, :, :, :n] = kv[:, src, :, :, :n]


def kv_move_slots(kv: torch.Tensor, src_slots: torch.Tensor, dst_slots: torch.Tensor) -> None:
    """Move slot contents (all layers, k and v); sources are read before any write."""
    ps = kv.shape[-2]
    sp, so = _slot_to_page(src_slots, ps)
    dp, do = _slot_to_page(dst_slots, ps)
    vals = kv[:, sp, :, :, so].clone()  # [L, n, 2, Hkv, hd]
    kv[:, dp, :, :, do] = vals


# ------------------------------------------------------- 8-bit KV cache
# The rules of the cache (scales, page starts, repeated slots) are those of ``ops.kv8``.
def rope_qkv_append8(
    qkv: torch.Tensor,
    table: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    kv_layer: kv8.Kv8Layer,
    num_heads: int,
    num_kv_heads: int,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """Rotate q/k, write k and v into the 8-bit cache at ``slots``; return rotated q [M, Hq, hd]."""
    m = qkv.shape[0]
    hd = kv_layer.data.shape[-1]
    if num_kv_heads != kv_layer.data.shape[2]:
        raise ValueError(f"{num_kv_heads} kv heads for a cache of {kv_layer.data.shape[2]}")
    if positions.numel() != m or slots.numel() != m:
        raise ValueError(f"{positions.numel()} positions and {slots.numel()} slots for {m} rows")
    x = qkv.float().reshape(m, num_heads + 2 * num_kv_heads, hd)
    if m and not bool(((positions >= 0) & (positions < table.shape[0])).all()):
        raise IndexError(f"position outside the rotary table of {table.shape[0]}")
    cs = table[positions.long()]
    cos, sin = cs[:, None, : hd // 2], cs[:, None, hd // 2:]
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    rot = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    rows = torch.stack((rot[:, num_heads: num_heads + num_kv_heads], x[:, num_heads + num_kv_heads:]), dim=1)[:, None]
    if m:
        kv8.write_rows(kv_layer.data[None], kv_layer.scale[None], rows, kv8.needed_scale(rows.abs().amax(-1)), slots)
    return rot[:, :num_heads].to(out_dtype or qkv.dtype)


def attention8(q: torch.Tensor, kv_layer: kv8.Kv8Layer, desc: AttnDesc, scale: float | None = None) -> torch.Tensor:
    """``attention`` over one layer of the 8-bit cache; a row that sees no key answers zero."""
    return attention(q, kv_layer.values(), desc, scale)


def attention8_causal(q: torch.Tensor, kv_layer: kv8.Kv8Layer, desc: AttnDesc, causal_start: int,
                      scale: float | None = None) -> torch.Tensor:
    """``attention8`` of a chunk at positions ``causal_start ..`` whose own keys are in the cache already."""
    m = q.shape[0]
    limit = torch.arange(causal_start + 1, causal_start + m + 1, dtype=torch.int32, device=q.device)
    return attention8(q, kv_layer, AttnDesc(desc.prefix_pages, int(desc.prefix_pages.numel()), int(causal_start), 0,
                                            limit, limit, desc.row_mask, desc.tail_pages), scale)


def kv8_copy_pages(cache: kv8.Kv8Cache, copies: torch.Tensor) -> None:
    """For each (src page, dst page, ntok): dst gets the first ntok slots and the scale of src in every layer,
    zeros behind them; with ntok 0 it becomes an empty page.  A destination may appear once only, and not as a
    source."""
    plan = copies.tolist()
    pages, ps = cache.data.shape[1], cache.data.shape[-2]
    used = [s for s, _, _ in plan] + [d for _, d, _ in plan]
    for src, dst, n in plan:
        if not (0 <= src < pages and 0 <= dst < pages and 0 <= n <= ps):
            raise IndexError(f"page copy ({src}, {dst}, {n}) is outside the cache of {pages} pages of {ps} slots")
        if used.count(dst) != 1:
            raise IndexError(f"page {dst} is a destination of one copy and named by another")
    data = cache.data.view(torch.uint8)
    for src, dst, n in plan:
        data[:, dst, :, :, :n] = data[:, src, :, :, :n]
        data[:, dst, :, :, n:] = 0
        cache.scale[:, dst] = cache.scale[:, src] if n else 0.0


def kv8_move_slots(cache: kv8.Kv8Cache, src_slots: torch.Tensor, dst_slots: torch.Tensor) -> None:
    """Move slot contents (all layers, k and v); sources are read before any write.  A row needs its source
    page's scale."""
    pages, ps = cache.data.shape[1], cache.data.shape[-2]
    if src_slots.numel() != dst_slots.numel():
        raise ValueError(f"{src_slots.numel()} source slots for {dst_slots.numel()} destinations")
    if src_slots.numel() and not bool(((src_slots >= 0) & (src_slots < pages * ps)).all()):
        raise IndexError(f"source slot outside the cache of {pages} pages of {ps} slots")
    sp, so = _slot_to_page(src_slots, ps)
    need = cache.scale[:, sp].transpose(0, 1)  # [n, layers, 2, kv_heads]
    rows = cache.data.view(torch.uint8)[:, sp, :, :, so].view(torch.float8_e4m3fn).float() * need[..., None]
    kv8.write_rows(cache.data, cache.scale, rows, need, dst_slots)


def kv8_read_pages(cache: kv8.Kv8Cache | kv8.Kv8Layer, pages: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values of ``pages``: [n, 2, kv_heads, page_size, hd] of a layer, [layers, n, ...] of a cache (held to the
    largest finite value of ``dtype``)."""
    idx = pages.long()
    data, scale = cache.data.view(torch.uint8), cache.scale
    if bool((idx < 0).any()):
        raise IndexError("negative page")
    if isinstance(cache, kv8.Kv8Cache):
        data, scale = data[:, idx], scale[:, idx]
    else:
        data, scale = data[idx], scale[idx]
    lim = torch.finfo(dtype).max
    return (data.view(torch.float8_e4m3fn).float() * scale[..., None, None]).clamp(-lim, lim).to(dtype)


def topk_logprobs(logits: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    lp = torch.log_softmax(logits.float(), dim=-1)
    return torch.topk(lp, k=k, dim=-1)
