"""Block-sparse decode through the engine: LLM(sparse_pages=)."""
import pytest
import torch

from vramancer_b200 import ops
from vramancer_b200.engine.engine import SamplingParams
from vramancer_b200.kv.pool import KVPool, KVPoolSpec
from vramancer_b200.llm import LLM

PROMPTS = [[(7 * i + 3 * j) % 500 for i in range(n)] for j, n in enumerate((130, 75, 16, 1))]


def cpu_llm(model="tiny-qwen3", **kw):
    return LLM(model, device="cpu", dtype=torch.float32, kv_cache_dtype="fp32", max_batch=4, max_model_len=256,
               kv_pages=96, **kw)


def tokens(llm, n=24, prompts=PROMPTS):
    return [r.output_ids for r in llm.generate(prompts, SamplingParams(max_tokens=n))]


@pytest.mark.parametrize("model", ["tiny-qwen3", "tiny-qwen2", "tiny-gpt2", "tiny-moe"])
def test_all_pages_is_dense(model):
    """A budget of all pages gives the dense engine's tokens."""
    dense = tokens(cpu_llm(model))
    assert tokens(cpu_llm(model, sparse_pages=16)) == dense


def count_selections(monkeypatch):
    """A list that grows by one with every call of ops.select_pages."""
    calls, real = [], ops.select_pages
    monkeypatch.setattr(ops, "select_pages", lambda *a, **k: calls.append(1) or real(*a, **k))
    return calls


@pytest.mark.parametrize("model", ["tiny-qwen3", "tiny-qwen2", "tiny-gpt2", "tiny-moe"])
def test_selection_of_all_pages_is_dense(model, monkeypatch):
    """The block table is wider than the budget, the contexts are not: the selection lists
    every page, and the tokens are the dense engine's."""
    wide = dict(device="cpu", dtype=torch.float32, kv_cache_dtype="fp32", max_batch=4, max_model_len=512, kv_pages=96)
    dense = tokens(LLM(model, **wide))
    calls = count_selections(monkeypatch)
    assert tokens(LLM(model, sparse_pages=16, **wide)) == dense
    assert len(calls) >= 20


def test_tensor_parallel():
    """Two ranks, each with its own kv heads' bounds and selections: the tokens of one rank."""
    from vramancer_b200.parallel.tensor_parallel import apply_tensor_parallel
    kw = dict(max_batch=4, max_model_len=256, kv_pages=96)
    one = tokens(cpu_llm("tiny-qwen3", sparse_pages=4), 12)
    assert one != tokens(cpu_llm("tiny-qwen3"), 12)
    tp = apply_tensor_parallel("tiny-qwen3", num_gpus=2, device="cpu", timeout_s=300, sparse_pages=4, **kw)
    try:
        assert tp.generate(PROMPTS, max_tokens=12) == one
    finally:
        tp.shutdown()


def test_model_load_route(monkeypatch):
    """`sparse_pages` of the load request reaches the engine that serves the model."""
    from fastapi.testclient import TestClient

    from vramancer_b200.serving.api import create_app
    monkeypatch.setenv("VRM_API_TOKEN", "t")
    calls = count_selections(monkeypatch)
    with TestClient(create_app()) as c:
        c.headers.update({"Authorization": "Bearer t"})
        for budget in (0, 4):
            r = c.post("/api/models/load", json={"model": "tiny-qwen2", "device": "cpu", "max_model_len": 256,
                                                 "sparse_pages": budget})
            assert r.status_code == 200, r.text
            r = c.post("/v1/completions", json={"prompt": "x" * 120, "max_tokens": 3})
            assert r.status_code == 200 and bool(calls) == (budget > 0), r.text


def reference_step(llm, seq, budget, sinks, recent):
    """Greedy next token of `seq` with every token of it decoded block-sparse: a plain
    forward, one token after the other, over keys and values kept as tensors."""
    cfg, w = llm.cfg, llm.weights
    hq, kh, D = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
    cs = ops.rope_cos_sin(cfg.max_position, cfg.rot_dim, cfg.rope_theta)
    prompt, rest = seq
    state = [[None, None] for _ in range(cfg.num_layers)]
    out = None
    for chunk, sparse in [(prompt, False)] + [([t], True) for t in rest]:
        start = 0 if state[0][0] is None else state[0][0].shape[0]
        r = w["embed"][torch.tensor(chunk)].float()
        T = len(chunk)
        for i in range(cfg.num_layers):
            g = lambda k: w[f"layers.{i}.{k}"]  # noqa: E731,B023
            rms = lambda x, nw: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.norm_eps) * nw  # noqa: E731
            qkv = (rms(r, g("in_norm_w")) @ g("qkv_w").t()).view(T, hq + 2 * kh, D)
            q, k, v = rms(qkv[:, :hq], g("q_norm_w")), rms(qkv[:, hq:hq + kh], g("k_norm_w")), qkv[:, hq + kh:]
            c = cs[start:start + T, None]

            def rot(x):
                a, b = x[..., :D // 2], x[..., D // 2:]
                co, si = c[..., :D // 2], c[..., D // 2:]
                return torch.cat([a * co - b * si, b * co + a * si], -1)
            q, k = rot(q), rot(k)
            K = k if start == 0 else torch.cat([state[i][0], k])
            V = v if start == 0 else torch.cat([state[i][1], v])
            state[i] = [K, V]
            o = torch.zeros(T, hq, D)
            for t in range(T):
                n = start + t + 1
                total = -(-n // 16)
                for h in range(kh):
                    qh = q[t, h * (hq // kh):(h + 1) * (hq // kh)]
                    see = torch.arange(n)
                    if sparse and total > budget:
                        # bounds as the fp32 pool keeps them: rounded to bf16
                        lo = torch.stack([K[16 * p:16 * p + 16, h].amin(0) for p in range(total)]).bfloat16().double()
                        hi = torch.stack([K[16 * p:16 * p + 16, h].amax(0) for p in range(total)]).bfloat16().double()
                        qd = q[t, h * (hq // kh):(h + 1) * (hq // kh)].double()
                        s = (hi * qd.clamp(min=0).sum(0) + lo * qd.clamp(max=0).sum(0)).sum(-1)
                        mid = sorted(range(sinks, total - recent), key=lambda p: (-float(s[p]), p))
                        keep = list(range(sinks)) + mid[:budget - sinks - recent] + list(range(total - recent, total))
                        see = torch.tensor([p * 16 + j for p in sorted(keep) for j in range(16) if p * 16 + j < n])
                    p = torch.softmax(qh @ K[see, h].t() / D ** 0.5, -1)
                    o[t, h * (hq // kh):(h + 1) * (hq // kh)] = p @ V[see, h]
            r = r + o.reshape(T, -1) @ g("o_w").t()
            gu = rms(r, g("post_norm_w")) @ g("gate_up_w").t()
            r = r + (torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]) @ g("down_w").t()
        out = rms(r[-1:], w["final_norm_w"]) @ w["lm_head"].t()
    return int(out.argmax())


def test_decode_reads_the_selected_pages():
    """The engine's tokens are those of a plain block-sparse forward, across pages that fill
    up while decoding."""
    llm = cpu_llm(sparse_pages=4, sparse_sinks=1, sparse_recent=1)
    got = tokens(llm, 12, PROMPTS[:1])[0]
    for k in (1, 4, 8, 12):
        assert reference_step(llm, (PROMPTS[0], got[:k - 1]), 4, 1, 1) == got[k - 1]
    dense = tokens(cpu_llm(), 12, PROMPTS[:1])[0]
    assert dense != got                    # the budget matters for these weights


@pytest.mark.parametrize("spec", [2, 4])
def test_speculative_verify_is_exact(spec):
    """Prompt-lookup drafts are verified with the rows' selected pages: same tokens."""
    plain = tokens(cpu_llm(sparse_pages=4))
    assert tokens(cpu_llm(sparse_pages=4, spec_num_draft=spec)) == plain


def test_prefix_cache_and_batching():
    """Requests that share cached pages, alone or batched, get the same tokens."""
    llm = cpu_llm(sparse_pages=4)
    p = PROMPTS[0]
    alone = [tokens(llm, 8, [x])[0] for x in (p, p[:96] + [5, 6, 7], p)]
    both = tokens(cpu_llm(sparse_pages=4), 8, [p, p[:96] + [5, 6, 7], p])
    assert alone == both


def test_copied_page_takes_its_bounds():
    pool = KVPool(KVPoolSpec(3, 2, 2, 64), "cpu", key_bounds=True)
    pool.cache[1] = 2.0
    pool.key_bounds[1] = 3.0
    pool.copy_page(1, 2)
    assert (pool.cache[2] == 2.0).all() and (pool.key_bounds[2].float() == 3.0).all()
    assert pool.key_bounds.shape == (3, 2, 2, 2, 64)
    assert pool.nbytes() == pool.cache.numel() * 2 + pool.key_bounds.numel() * 2
    plain = KVPool(KVPoolSpec(3, 2, 2, 64), "cpu")
    assert plain.key_bounds is None
    plain.copy_page(0, 1)


def test_refusals():
    for kw in (dict(sparse_pages=2), dict(sparse_pages=4, sparse_recent=0), dict(sparse_pages=4, sparse_sinks=-1),
               dict(sparse_pages=8, kv_offload_pages=4), dict(sparse_pages=8, kv_lender=0)):
        with pytest.raises(ValueError):
            cpu_llm(**kw)
    with pytest.raises(ValueError):
        LLM("tiny-qwen3", device="cpu", dtype=torch.float32, kv_cache_dtype="fp32", max_batch=1, kv_pages=8,
            max_model_len=16 * ops.SELECT_MAX_PAGES + 1, sparse_pages=4)
    with pytest.raises(ValueError):
        KVPool(KVPoolSpec(2, 1, 1, 128, dtype=torch.int8), "cpu", key_bounds=True)


@pytest.mark.parametrize("n", [-1, -128])
def test_negative_budget_is_refused(n, monkeypatch):
    """Not taken for "off": by the engine, and by the commands and the model-load route that
    pass it on."""
    from fastapi.testclient import TestClient

    from vramancer_b200 import cli
    from vramancer_b200.serving.api import create_app
    with pytest.raises(ValueError, match="negative"):
        cpu_llm(sparse_pages=n)
    for command in ("run", "serve"):
        with pytest.raises(ValueError, match="negative"):
            cli.main([command, "tiny-qwen2", "--sparse-pages", str(n)])
    monkeypatch.setenv("VRM_API_TOKEN", "t")
    r = TestClient(create_app()).post("/api/models/load", headers={"Authorization": "Bearer t"},
                                      json={"model": "tiny-qwen2", "device": "cpu", "sparse_pages": n})
    assert r.status_code == 500 and "negative" in r.text


def test_command_line():
    from vramancer_b200.cli import build_parser
    a = build_parser().parse_args(["run", "m", "--sparse-pages", "64"])
    assert a.sparse_pages == 64
    assert build_parser().parse_args(["serve", "m"]).sparse_pages == 0


def test_tensor_parallel_serve_relaunches_with_every_option(monkeypatch):
    """`serve --tp N` starts itself once per GPU: the ranks parse the options that were given."""
    from vramancer_b200 import cli
    given = ["serve", "--model", "tiny-qwen2", "--tp", "2", "--sparse-pages", "64", "--max-model-len", "512",
             "--quantization", "fp8", "--no-cluster", "--profile", "coding", "--num-layers", "1", "--host", "::1",
             "--port", "5031"]
    calls = []
    monkeypatch.delenv("WORLD_SIZE", raising=False)
    monkeypatch.setenv("VRM_N_CTX", "16384")                 # what --profile coding sets
    monkeypatch.setattr(cli.subprocess, "call", lambda cmd: calls.append(cmd) or 0)
    assert cli.main(given) == 0
    cmd, = calls
    at = cmd.index("vramancer_b200")
    assert "--nproc-per-node=2" in cmd[:at]
    parser = cli.build_parser()
    assert vars(parser.parse_args(cmd[at + 1:])) == vars(parser.parse_args(given))


# ------------------------------------------------------------------------- GPU
def gpu_llm(model, kv, graph, **kw):
    return LLM(model, device="cuda", kv_cache_dtype=kv, max_batch=4, max_model_len=512, kv_pages=128,
               use_cuda_graph=graph, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("model,kv", [("tiny-qwen3", "bf16"), ("tiny-qwen2-d128", "bf16"), ("tiny-qwen2-d128", "fp8"),
                                      ("tiny-qwen2-d128", "q4"), ("tiny-gpt2", "bf16")])
def test_graphs_and_eager_agree(model, kv, cuda_errors_clean):
    """CUDA-graph decode (padded batch buckets) and eager decode run the same kernels."""
    prompts = PROMPTS[:3]
    eager = tokens(gpu_llm(model, kv, False, sparse_pages=4), 40, prompts)
    assert tokens(gpu_llm(model, kv, True, sparse_pages=4), 40, prompts) == eager


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "fp8", "q4"])
def test_gpu_logits_against_cpu(kv, cuda_errors_clean):
    """One decode step's logits on the GPU against the CPU path on the same pool: same
    selection, bf16 kernels against fp32 math."""
    from vramancer_b200.engine.runner import PrefillItem
    from vramancer_b200.models.transformer import ForwardBatch
    llm = gpu_llm("tiny-qwen2-d128", kv, False, sparse_pages=4, fold_norms=False)
    ids = PROMPTS[0]
    slots = list(range(len(ids)))
    bt = list(range(10))
    llm.runner.prefill([PrefillItem(ids, 0, slots, bt, len(ids), True)], [0.0], [0], [1.0], [0])
    n = len(ids) + 1
    from vramancer_b200.models.transformer import DecoderModel
    cpu = DecoderModel(llm.cfg, {k: v.cpu() for k, v in llm.weights.items()}, device="cpu")
    cpu.set_sparse(4)
    pool = KVPool(llm.pool.spec, "cpu", kv_scale=llm.pool.kv_scale, key_bounds=True)
    pool.cache.copy_(llm.pool.cache)
    pool.key_bounds.copy_(llm.pool.key_bounds)

    def batch(dev):
        t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        return ForwardBatch(t([9]), t([n - 1]), t([n - 1]), t([bt]), t([n]), True)

    a = llm.model.forward(batch("cuda"), llm.pool).float().cpu()
    b = cpu.forward(batch("cpu"), pool).float()
    assert torch.isfinite(a).all()
    # bf16 activations through two layers: a few units of 2^-8 of the logits' scale
    assert (a - b).abs().max() <= 8 * 2.0 ** -8 * b.abs().max()


@pytest.mark.gpu
def test_gpu_speculative_verify_graph(cuda_errors_clean):
    """Verify steps with selected pages replay their graphs: the same tokens twice."""
    llm = gpu_llm("tiny-qwen3", "bf16", True, sparse_pages=4, spec_num_draft=4, enable_prefix_cache=False)
    first = tokens(llm, 32, PROMPTS[:2])
    assert all(len(x) == 32 for x in first) and llm.runner._verify
    assert tokens(llm, 32, PROMPTS[:2]) == first


def verify_step(llm, ids, bt, n):
    """Logits of `ids`, the last of n tokens of a sequence in the pages `bt`, fed as a verify
    step's rows."""
    from vramancer_b200.models.transformer import ForwardBatch
    m = len(ids)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pos = list(range(n - m, n))
    return llm.model.forward(ForwardBatch(t(ids), t(pos), t([16 * bt[p // 16] + p % 16 for p in pos]), t([bt]), t([n]),
                                          False, cu_q=t([0, m]), max_q_len=m, decode_rows=True), llm.pool)


@pytest.mark.gpu
@pytest.mark.parametrize("model,kv", [("tiny-qwen3", "bf16"), ("tiny-qwen2-d128", "bf16"), ("tiny-qwen2-d128", "fp8"),
                                      ("tiny-qwen2-d128", "q4")])
def test_gpu_selection_of_all_pages_is_dense(model, kv, cuda_errors_clean, monkeypatch):
    """A step over a table wider than the budget: with every page selected the logits are
    those of dense attention on the same pool, with four pages they are others."""
    from vramancer_b200.engine.runner import PrefillItem
    llm = gpu_llm(model, kv, False, sparse_pages=32, enable_prefix_cache=False)
    ids = PROMPTS[0]
    bt = list(range(3, 40))
    slots = [16 * bt[p // 16] + p % 16 for p in range(len(ids))]
    llm.runner.prefill([PrefillItem(ids, 0, slots, bt, len(ids), True)], [0.0], [0], [1.0], [0])
    logits, calls = {}, count_selections(monkeypatch)
    for name, sparse in (("dense", None), ("all", (32, 1, 2)), ("some", (4, 1, 2))):
        llm.model.sparse = sparse
        logits[name] = verify_step(llm, [9, 4, 7], bt, len(ids) + 3).float()
        assert bool(calls) == (sparse is not None)
    # bf16 activations through two layers: a few units of 2^-8 of the logits' scale
    tol = 8 * 2.0 ** -8 * logits["dense"].abs().max()
    assert (logits["all"] - logits["dense"]).abs().max() <= tol
    assert (logits["some"] - logits["dense"]).abs().max() > 2 * tol


@pytest.mark.gpu
@pytest.mark.parametrize("model,kv", [("tiny-qwen3", "bf16"), ("tiny-qwen2-d128", "fp8"), ("tiny-qwen2-d128", "q4")])
def test_gpu_verify_graph_reads_selected_pages(model, kv, cuda_errors_clean):
    """The captured verify step (a batch padded to its bucket, items shorter than the step)
    against the eager one: every token has the eager logits' maximum within rounding, which
    dense attention's logits do not bear out."""
    from vramancer_b200.engine.runner import PrefillItem
    llm = gpu_llm(model, kv, True, sparse_pages=4, enable_prefix_cache=False)
    prompts = [PROMPTS[0], PROMPTS[0][5:] + [3] * 60, PROMPTS[1]]
    tables = [list(range(32 * i, 32 * i + 20)) for i in range(3)]
    pos = lambda i, a, b: [16 * tables[i][p // 16] + p % 16 for p in range(a, b)]  # noqa: E731
    llm.runner.prefill([PrefillItem(p, 0, pos(i, 0, len(p)), tables[i], len(p), True) for i, p in enumerate(prompts)],
                       [0.0] * 3, [0] * 3, [1.0] * 3, [0] * 3)
    before = llm.pool.cache.clone(), llm.pool.key_bounds.clone()
    feeds = [[5, 6, 7, 8, 9], [11], [2, 4, 2]]
    items = [PrefillItem(f, len(p), pos(i, len(p), len(p) + len(f)), tables[i], len(p) + len(f), True)
             for i, (p, f) in enumerate(zip(prompts, feeds))]

    def restore():
        llm.pool.cache.copy_(before[0])
        llm.pool.key_bounds.copy_(before[1])

    for _ in range(2):                                       # captured, then replayed
        got = llm.runner.verify_greedy(items)
        after = llm.pool.cache.clone(), llm.pool.key_bounds.clone()
        restore()
    assert [len(x) for x in got] == [5, 1, 3] and llm.runner._verify
    eager = llm.runner.prefill_logits(items, decode_rows=True).float()
    written = sum((it.slots for it in items), [])
    rest = torch.ones(llm.pool.cache.shape[0], 16, dtype=torch.bool, device="cuda")
    rest.view(-1)[torch.tensor(written, device="cuda")] = False
    moved = (after[0].view(torch.uint8) != before[0].view(torch.uint8)).any(-1).any(1).any(1).any(1)
    assert not (moved & rest).any()                          # padded rows store nothing
    restore()
    dense = llm.runner.prefill_logits(items).float()
    # bf16 activations through two layers: a few units of 2^-8 of the logits' scale
    tol = 8 * 2.0 ** -8 * eager.abs().max()
    tok = torch.tensor(sum(got, []), device="cuda")[:, None]
    assert (eager.gather(1, tok) >= eager.amax(1, keepdim=True) - tol).all()
    assert (dense - eager).abs().max() > 2 * tol
    assert (dense.gather(1, tok) < dense.amax(1, keepdim=True) - tol).any()
