"""Engines, drafter, target and commands on the 8-bit KV cache."""

from __future__ import annotations

import json

import numpy as np
import pytest
import torch

from conftest import mod
from test_kv8 import Oracle, o_scale

DEVICES = [pytest.param("cpu", id="cpu"), pytest.param("cuda", id="cuda", marks=pytest.mark.gpu)]


def weights(device, preset, seed):
    llama = mod("models.llama")
    dtype = torch.float32 if device == "cpu" else torch.float16
    w = llama.random_weights(llama.get_config(preset), seed=seed, dtype=torch.float32, device=device)
    return llama.weights_to(w, dtype=dtype)


def presets(device):
    return ("tiny-drafter", "tiny-target") if device == "cpu" else ("small-drafter", "small-target")


def make(device, preset, seed, *, pages=256, page_size=16, positions=1024):
    return mod("runtime.engine_kv8").make_engine(weights(device, preset, seed), kv_cache="fp8", num_pages=pages,
                                                 page_size=page_size, max_positions=positions)


class OracleModel:
    """The model in float64 with its keys and values held as the 8-bit cache holds them, one sequence in the pages
    0, 1, .. ; ``step`` appends tokens in one call and returns their logits."""

    def __init__(self, w, pages, ps):
        self.w, self.cfg = w, w.config
        c = self.cfg
        self.cache = Oracle(mod("ops.kv8").empty_cache(c.num_layers, pages, c.num_kv_heads, ps, c.head_dim))
        self.table = mod("models.llama").rope_table(c, pages * ps).double()
        self.len = 0

    def norm(self, x, g):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.cfg.rms_eps) * g.double().cpu()

    def rot(self, x, pos):
        half = x.shape[-1] // 2
        cs = self.table[pos][:, None]
        c, s = cs[..., :half], cs[..., half:]
        return torch.cat((x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s), -1)

    def step(self, tokens):
        c, ps = self.cfg, self.cache.ps
        n, start = len(tokens), self.len
        pos = torch.arange(start, start + n)
        h = self.w.embed.double().cpu()[torch.tensor(tokens)]
        for li, lw in enumerate(self.w.layers):
            qkv = self.norm(h, lw.attn_norm) @ lw.wqkv.double().cpu().t()
            qkv = qkv.reshape(n, c.num_heads + 2 * c.num_kv_heads, c.head_dim)
            q = self.rot(qkv[:, : c.num_heads], pos)
            kv = (self.rot(qkv[:, c.num_heads: c.num_heads + c.num_kv_heads], pos),
                  qkv[:, c.num_heads + c.num_kv_heads:])
            for side in (0, 1):
                for head in range(c.num_kv_heads):
                    for page in range(start // ps, (start + n - 1) // ps + 1):
                        rows = {x % ps: (kv[side][x - start, head], o_scale(float(kv[side][x - start, head].abs().max())))
                                for x in range(max(start, page * ps), min(start + n, (page + 1) * ps))}
                        self.cache.write(li, side, head, page, rows)
            val = self.cache.val[li].permute(1, 2, 0, 3, 4).reshape(2, c.num_kv_heads, -1, c.head_dim)[:, :, : start + n]
            k, v = (val[i].repeat_interleave(c.group, 0) for i in (0, 1))
            s = torch.einsum("nhd,hkd->hnk", q, k) / c.head_dim ** 0.5
            s = s.masked_fill(torch.arange(start + n)[None, None] > pos[None, :, None], -torch.inf)
            a = torch.einsum("hnk,hkd->nhd", torch.softmax(s, -1), v).reshape(n, -1)
            h = h + a @ lw.wo.double().cpu().t()
            gate, up = mod("models.llama").split_gate_up(lw.wgu.double().cpu())
            x = self.norm(h, lw.mlp_norm)
            h = h + (torch.nn.functional.silu(x @ gate.t()) * (x @ up.t())) @ lw.wd.double().cpu().t()
        self.len += n
        return self.norm(h, self.w.final_norm) @ self.w.lm_head.double().cpu().t()


@pytest.mark.parametrize("device", DEVICES)
def test_engine_matches_oracle(device):
    """Prefill, decode steps over a page boundary and a masked batch against the float64 model with the same cache."""
    eng = make(device, presets(device)[1], 2)
    om = OracleModel(eng.w, 8, 16)
    prompt = torch.randint(0, 1024, (29,), generator=torch.Generator().manual_seed(0)).tolist()
    pages = torch.arange(8, dtype=torch.int32, device=eng.device)
    # fp32 on the CPU: a value next to a rounding border may take the neighbouring code, a step of 2^-3 in one of the
    # 64 products of a score.  fp16 on the GPU: activations carry 2^-11 each, so more codes differ by that step; a
    # cache that was off by half a step (2^-4) everywhere would move the logits by less than 2^-4 of their norm.
    tol = 1e-3 if device == "cpu" else 2.0 ** -4

    def close(got, want):
        assert float((got.double().cpu() - want).norm() / want.norm()) < tol

    dev = eng.device
    got = eng.prefill_sequence(torch.tensor(prompt, dtype=torch.int32, device=dev), start_pos=0,
                               slots=torch.arange(29, dtype=torch.int32, device=dev), pages=pages)
    close(got, om.step(prompt)[-1])
    for i, tok in enumerate([7, 900, 33, 512, 5]):
        p = 29 + i
        got = eng.run_rows(1, prefix_pages=pages, tokens=[tok], positions=[p], slots=[p], shared_len=p,
                           n_shared_pages=8, mask_base=p, row_full=[p + 1], row_len=[p + 1])
        close(got[0], om.step([tok])[0])
    chain = [3, 4, 5]  # a chain of three nodes in one masked call
    got = eng.run_rows(4, prefix_pages=pages, tokens=chain, positions=[34, 35, 36], slots=[34, 35, 36], shared_len=34,
                       n_shared_pages=8, mask_base=34, row_full=[34] * 3, row_len=[37] * 3,
                       row_mask=np.array([[1], [3], [7]], dtype=np.int64))
    close(got, om.step(chain))
    eng.ops.check()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("threshold", [None, 1e9], ids=["select", "fallback"])
def test_speculative_generation_runs(device, threshold):
    """Drafter and target on 8-bit caches, every round selecting (tree, forest, copy-on-write, compaction) or every
    round falling back; the physical and logical states are checked after each round."""
    drafter, target, edge, rpc = (mod(x) for x in ("runtime.drafter", "runtime.target", "serving.edge", "serving.rpc"))
    dp, tp = presets(device)
    dr = drafter.DrafterRuntime(make(device, dp, 1))
    tv = target.TargetVerifier(make(device, tp, 2), k=3, d=4, fallback_threshold=threshold)
    gen = edge.PagedDistributedAtlasGenerator(
        config=edge.DistributedAtlasConfig(k=3, d=4, max_new_tokens=24, fixed_forest_depth=1,
                                           validate_state_alignment=True),
        drafter=dr, target_client=rpc.InProcessTargetClient(tv))
    prompt = torch.randint(0, 1024, (75,), generator=torch.Generator().manual_seed(1)).tolist()
    res = gen.generate(prompt)
    assert len(res.generated_token_ids) == 24
    assert {r.decision for r in res.rounds} == {"select" if threshold is None else "fallback_ar"}
    dr.engine.ops.check()
    tv.engine.ops.check()
    assert gen.generate(prompt).generated_token_ids == res.generated_token_ids  # recycled pages carry nothing over


@pytest.mark.parametrize("device", DEVICES)
def test_committed_path_is_compacted(device):
    """After a commit that moves KV, the kept prefix logits agree with a fresh 8-bit prefill of the same tokens."""
    target, types = mod("runtime.target"), mod("types")
    name = presets(device)[1]
    tv = target.TargetVerifier(make(device, name, 2), k=3, d=3, route_selection_policy="first_route")
    prompt = list(range(20, 49))
    tv.prefill(prompt)

    def route(rid, toks):
        return types.VerifyRoutePayload(route_id=rid, token_ids=tuple(toks), draft_logprob=-1.5,
                                        draft_token_logprobs=(-0.5,) * 3)

    res = tv.verify_payloads(prefix_token_ids=prompt, routes=[route(1, [7, 5, 6]), route(0, [7, 8, 9]), route(2, [3, 4, 1])])
    assert res.decision == "select"
    tv.verify_payloads(prefix_token_ids=list(tv.prefix_token_ids),
                       routes=[route(5, [2, 2, 2]), route(6, [2, 3, 3]), route(7, [9, 9, 9])])
    fresh = target.TargetVerifier(make(device, name, 2), k=3, d=3)
    fresh.prefill(list(tv.prefix_token_ids))
    a, b = tv.prefix_logits.float(), fresh.prefix_logits.float()
    # The two caches round the same values under scales that may differ by a power of two (a page's scale also covers
    # rows that were dropped): equal codes but for elements below scale / 64, and border cases as above.
    assert float((a - b).norm() / b.norm()) < 2.0 ** -4


@pytest.mark.gpu
def test_graph_replay_matches_eager():
    eng = make("cuda", "small-target", 4)
    pages = torch.arange(100, dtype=torch.int32, device="cuda")
    g = np.random.default_rng(5)
    rows = 12
    prompt = torch.randint(0, 4096, (300,), generator=torch.Generator().manual_seed(0)).int().cuda()
    eng.prefill_sequence(prompt, start_pos=0, slots=torch.arange(300, dtype=torch.int32, device="cuda"), pages=pages)
    fields = dict(
        tokens=g.integers(0, 4096, rows), positions=np.arange(300, 300 + rows), slots=np.arange(300, 300 + rows),
        shared_len=300, n_shared_pages=100, mask_base=300, row_full=np.full(rows, 300), row_len=np.full(rows, 300 + rows),
        row_mask=np.array([(1 << (i + 1)) - 1 for i in range(rows)])[:, None])
    graph = [eng.run_rows(16, prefix_pages=pages, **fields) for _ in range(2)]
    eng.use_graphs = False
    eager = eng.run_rows(16, prefix_pages=pages, **fields)
    eng.ops.check()
    assert torch.equal(graph[0], graph[1]) and torch.equal(graph[1], eager)


@pytest.mark.gpu
def test_fp8_weights_with_8bit_cache():
    """The block-scaled fp8 engine on the 8-bit cache stays within a half step of e4m3 of the same engine on bf16."""
    fp8, llama, e8 = mod("models.fp8"), mod("models.llama"), mod("runtime.engine_kv8")
    w = fp8.random_weights_fp8(llama.get_config("small-target"), seed=4, dtype=torch.bfloat16, device="cuda")
    toks = torch.arange(100, 160, dtype=torch.int32, device="cuda")
    out = []
    for cls in (mod("runtime.engine_fp8").Fp8LlamaEngine, e8.Kv8Fp8LlamaEngine):
        e = cls(w, num_pages=64, page_size=16, max_positions=256)
        out.append(e.prefill_sequence(toks, start_pos=0, slots=torch.arange(60, dtype=torch.int32, device="cuda"),
                                      pages=torch.arange(4, dtype=torch.int32, device="cuda")))
        e.ops.check()
    assert float((out[0] - out[1]).norm() / out[0].norm()) < 2.0 ** -4


def test_commands_take_the_cache_option(capsys):
    ds, ts = mod("serving.distributed_system"), mod("serving.target_server")
    common = ["--dtype", "float32", "--page-size", "4", "--k", "2", "--d", "2"]
    if torch.cuda.is_available():
        pytest.skip("the commands take the GPU where there is one; tiny models need the CPU")
    assert ds.main(["--drafter-model", "tiny-drafter", "--target-model", "tiny-target", "--prompt-token-ids",
                    "5,6,7,8,9,10,11", "--max-new-tokens", "8", "--warmup-runs", "0", "--drafter-kv-cache", "fp8",
                    "--target-kv-cache", "fp8", *common]) == 0
    assert len(json.loads(capsys.readouterr().out)["generated_token_ids"]) == 8
    args = ts.build_parser().parse_args(["--model", "tiny-target", "--port", "1", "--prefix-len", "64",
                                         "--max-new-tokens-capacity", "32", "--kv-cache", "fp8", *common])
    tv = ts.build_backend(args)
    assert isinstance(tv.engine, mod("runtime.engine_kv8").Kv8LlamaEngine)
    tv.prefill([1, 2, 3])
    with pytest.raises(SystemExit):
        ts.build_parser().parse_args(["--model", "tiny-target", "--port", "1", "--kv-cache", "int4"])


def test_engine_refusals():
    e8 = mod("runtime.engine_kv8")
    w = weights("cpu", "tiny-target", 0)
    with pytest.raises(ValueError, match="KV cache"):
        e8.make_engine(w, kv_cache="int8", num_pages=4, page_size=4, max_positions=16)
    assert type(e8.make_engine(w, num_pages=4, page_size=4, max_positions=16)) is mod("runtime.engine").LlamaEngine
    cfg = w.config
    assert e8.kv8_bytes_per_token(cfg, 16) == cfg.num_layers * 2 * cfg.num_kv_heads * (cfg.head_dim + 0.25)
