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
