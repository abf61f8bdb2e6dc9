"""Serving operators of block-sparse decode attention over the paged KV pool, with their
plain PyTorch forms.

  append   ops.qk_norm_rope_kv_write   per-head q / k RMSNorm, rotary positions and the KV
           page write of new tokens in one pass, with each written page's key bounds
           (elementwise minimum and maximum of its keys)
  select   ops.select_pages            the pages each query row reads: an upper bound of the
           group's scores from the key bounds, the `budget` best pages of each row
  attend   ops.paged_attention_selected   attention of each query row over its pages

A case is a dict of plain values.  Common keys: "op", head layout "hq" / "kh" / "d", page
format "kv" (bf16, fp8 or q4), "layers" of the pool (the last one is used).  Sequence i of a
ragged case is shorter than the first by a fixed rule, so sizes follow from the case alone;
values and the placement of pages in the pool follow from the seed.
"""
import math

import torch

own = False

PAGE = 16
SINKS, RECENT = 1, 2            # pages at the start and at the end that every row reads


def listed():
    return [
        # one new token of one long conversation (32 / 8 heads, q / k norms): pure latency
        {"name": "append_1", "op": "append", "hq": 32, "kh": 8, "d": 128, "kv": "bf16", "layers": 2, "norm": True,
         "seqs": 1, "new": 1, "start": 32001, "ragged": False},
        # a decode step of a full batch over an fp8 pool, no q / k norms (28 / 4 heads)
        {"name": "append_64_fp8", "op": "append", "hq": 28, "kh": 4, "d": 128, "kv": "fp8", "layers": 1, "norm": False,
         "seqs": 64, "new": 1, "start": 4099, "ragged": True},
        # one prefill step of the engine's default 8192 prompt tokens (32 / 4 heads)
        {"name": "append_8192", "op": "append", "hq": 32, "kh": 4, "d": 128, "kv": "bf16", "layers": 1, "norm": True,
         "seqs": 1, "new": 8192, "start": 0, "ragged": False},
        # ragged prompt chunks that start and end inside pages (40 / 8 heads)
        {"name": "append_ragged", "op": "append", "hq": 40, "kh": 8, "d": 128, "kv": "bf16", "layers": 1, "norm": False,
         "seqs": 5, "new": 777, "start": 1003, "ragged": True},
        # one query over a full 32k context: latency
        {"name": "select_1", "op": "select", "hq": 32, "kh": 8, "d": 128, "kv": "bf16", "layers": 1,
         "seqs": 1, "chunk": 1, "context": 32768, "budget": 128, "ragged": False},
        # the decode batch of the headline workload at long ragged contexts
        {"name": "select_32", "op": "select", "hq": 40, "kh": 8, "d": 128, "kv": "bf16", "layers": 1,
         "seqs": 32, "chunk": 1, "context": 16411, "budget": 64, "ragged": True},
        # speculative verify rows: five query tokens of each of eight sequences
        {"name": "select_verify", "op": "select", "hq": 28, "kh": 4, "d": 128, "kv": "bf16", "layers": 2,
         "seqs": 8, "chunk": 5, "context": 8192, "budget": 48, "ragged": True},
        # the largest: a full batch over fp8 bounds at 32k
        {"name": "select_64_fp8", "op": "select", "hq": 32, "kh": 8, "d": 128, "kv": "fp8", "layers": 1,
         "seqs": 64, "chunk": 1, "context": 32768, "budget": 128, "ragged": False},
        # one query over its 128 pages: latency
        {"name": "attend_1", "op": "attend", "hq": 32, "kh": 8, "d": 128, "kv": "bf16", "layers": 1,
         "seqs": 1, "chunk": 1, "context": 32768, "budget": 128, "ragged": False},
        # the decode batch of the headline workload
        {"name": "attend_32", "op": "attend", "hq": 40, "kh": 8, "d": 128, "kv": "bf16", "layers": 1,
         "seqs": 32, "chunk": 1, "context": 16411, "budget": 128, "ragged": True},
        # the largest: 128 rows over fp8 pages
        {"name": "attend_128_fp8", "op": "attend", "hq": 32, "kh": 8, "d": 128, "kv": "fp8", "layers": 1,
         "seqs": 128, "chunk": 1, "context": 4096, "budget": 128, "ragged": True},
        # verify rows over four-bit pages, 64-dim heads (14 / 2)
        {"name": "attend_verify_q4", "op": "attend", "hq": 14, "kh": 2, "d": 64, "kv": "q4", "layers": 2,
         "seqs": 8, "chunk": 5, "context": 6001, "budget": 48, "ragged": True},
    ]


HEADS = ((32, 8, 128), (40, 8, 128), (28, 4, 128), (32, 4, 128), (14, 2, 64), (32, 8, 64), (12, 12, 64))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, kh, d = rng.choice(HEADS)
    case = {"op": rng.choice(("append", "select", "attend")), "hq": hq, "kh": kh, "d": d,
            "layers": rng.choice((1, 2)), "ragged": rng.random() < 0.7}
    if case["op"] == "append":
        case["kv"] = rng.choice(("bf16", "fp8"))
        case["norm"] = rng.random() < 0.5
        if rng.random() < 0.5:               # a decode step
            case.update(seqs=_log(rng, 1, 128), new=1, start=_log(rng, 17, 8000))
        else:                                # prompt chunks
            case.update(seqs=_log(rng, 1, 8), new=_log(rng, 2, 700), start=_log(rng, 1, 2000))
        return case
    case["kv"] = rng.choice(("bf16", "fp8") if case["op"] == "select" else ("bf16", "fp8", "q4"))
    case["seqs"] = _log(rng, 1, 64)
    case["chunk"] = rng.choice((1, 1, 1, 2, 5, 8)) if case["seqs"] <= 12 else 1
    # at most the largest listed pools: 64 x 8192 tokens of 8 heads x 128 dims
    case["context"] = _log(rng, 100, min(32768, 64 * 8192 // case["seqs"]))
    case["budget"] = _log(rng, 8, 128)
    return case


# ---------------------------------------------------------------- inputs
def _lens(case, full, least):
    """Length of each sequence: `full` for the first, less for the others of a ragged case."""
    n = case["seqs"]
    if not case["ragged"]:
        return [full] * n
    return [max(least, full - (i * 997) % (full // 2 + 1)) for i in range(n)]


def _sizes(case):
    """(cached tokens before the pass, new tokens or query rows, tokens after it) of each sequence."""
    if case["op"] == "append":
        new = _lens(case, case["new"], 1)
        start = [case["start"] + 13 * i for i in range(case["seqs"])]
        return start, new, [a + b for a, b in zip(start, new)]
    ctx = _lens(case, case["context"], case["chunk"])
    new = [case["chunk"]] * case["seqs"]
    return [c - n for c, n in zip(ctx, new)], new, ctx


def _kinds(kv):
    """(pool dtype, key bounds dtype) of a page format."""
    return {"bf16": (torch.bfloat16, torch.bfloat16), "fp8": (torch.float8_e4m3fn, torch.float8_e4m3fn),
            "q4": (torch.uint8, torch.bfloat16)}[kv]


def _row(case):
    """Elements of a stored row: head dims, or the bytes of a four-bit row."""
    return case["d"] * 5 // 8 if case["kv"] == "q4" else case["d"]


def _block_tables(ctx, g):
    pages = [-(-n // PAGE) for n in ctx]
    total, width = sum(pages), max(pages)
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    per = torch.tensor(pages, device="cuda")
    col = torch.arange(width, device="cuda")
    first = torch.cumsum(per, 0) - per
    at = (first[:, None] + col[None, :]).clamp(max=total - 1)
    bt = torch.where(col[None, :] < per[:, None], perm[at], torch.zeros_like(perm[at]))
    return bt.contiguous(), total


def _channels(d, g):
    """Per-dim magnitudes: a few outlier channels, as the keys of trained models have."""
    return 1.0 + 5.0 * (torch.rand(d, generator=g, device="cuda") > 0.95).float()


def _pool(case, pages, g):
    kh, d, n = case["kh"], case["d"], case["layers"]
    dtype, _ = _kinds(case["kv"])
    if case["kv"] == "q4":
        pool = torch.randint(0, 256, (pages, n, 2, kh, PAGE, _row(case)), generator=g, device="cuda", dtype=torch.uint8)
        sm = torch.rand(pages, n, 2, kh, PAGE, d // 32, 2, generator=g, device="cuda")
        sm[..., 0] = 0.1 + 0.2 * sm[..., 0]              # scale
        sm[..., 1] = -3.0 + 1.5 * sm[..., 1]             # minimum
        pool[..., d // 2:] = sm.half().view(torch.uint8).flatten(-2)
        return pool, None
    pool = torch.randn(pages, n, 2, kh, PAGE, d, generator=g, device="cuda", dtype=torch.bfloat16)
    pool[:, :, 0] *= _channels(d, g).bfloat16()
    if case["kv"] == "bf16":
        return pool, None
    scale = 0.02 + 0.03 * torch.rand(n, 2, kh, generator=g, device="cuda")
    return (pool / scale[None, :, :, :, None, None].bfloat16()).clamp(-448, 448).to(dtype), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    before, new, after = _sizes(case)
    hq, kh, d = case["hq"], case["kh"], case["d"]
    T = sum(new)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    bt, pages = _block_tables(after, g)
    s = {"case": case, "hq": hq, "kh": kh, "d": d, "layer": case["layers"] - 1, "bt": bt, "ctx": i32(after),
         "seq": torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))}
    within = torch.arange(T, device="cuda") - torch.repeat_interleave(
        torch.tensor([sum(new[:i]) for i in range(len(new))], device="cuda"), torch.tensor(new, device="cuda"))
    s["pos"] = (torch.tensor(before, device="cuda")[s["seq"]] + within).to(torch.int32)
    _, bdtype = _kinds(case["kv"])
    if case["op"] == "append":
        s["cache"], s["scale"] = _pool(case, pages, g)
        s["bounds"] = torch.zeros(pages, case["layers"], kh, 2, d, device="cuda").to(bdtype)
        s["qkv"] = 2 * torch.randn(T, (hq + 2 * kh) * d, generator=g, device="cuda", dtype=torch.bfloat16)
        s["wq"] = s["wk"] = None
        if case["norm"]:
            s["wq"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).bfloat16()
            s["wk"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).bfloat16()
        page = torch.gather(bt[s["seq"]].long(), 1, (s["pos"].long() // PAGE)[:, None])[:, 0]
        s["slots"] = (page * PAGE + s["pos"].long() % PAGE).to(torch.int32)
        inv = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        ang = torch.outer(torch.arange(max(after), dtype=torch.float64, device="cuda"), inv)
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        return s
    s["budget"] = case["budget"]
    s["q"] = torch.randn(T, hq * d, generator=g, device="cuda", dtype=torch.bfloat16)
    s["cu_q"] = i32([sum(new[:i]) for i in range(len(new) + 1)]) if case["chunk"] > 1 else None
    if case["op"] == "select":
        ch = _channels(d, g)
        mid = torch.randn(pages, case["layers"], kh, d, generator=g, device="cuda") * ch
        half = (0.8 + 0.5 * torch.rand(pages, case["layers"], kh, d, generator=g, device="cuda")) * ch
        b = torch.stack([mid - half, mid + half], 3)
        s["bounds"] = (8 * b if case["kv"] == "fp8" else b).to(bdtype)
        return s
    s["cache"], s["scale"] = _pool(case, pages, g)
    noise = torch.rand(T, kh, bt.shape[1], generator=g, device="cuda", dtype=torch.float64)
    s["pages"] = _choose(noise, s["pos"].long() + 1, case["budget"])
    s["sm_scale"] = 1 / math.sqrt(d)
    return s


# ---------------------------------------------------------------- plain forms
def _choose(score, n, budget):
    """The `budget` pages of each row: the first SINKS and last RECENT pages, then the best
    scores, ties to the lowest page; ascending, -1 behind the last.  score [T, KH, P],
    n [T] tokens a row sees."""
    T, KH, P = score.shape
    page = torch.arange(P, device=score.device)
    total = ((n + PAGE - 1) // PAGE)[:, None, None]
    score = torch.where((page < SINKS) | (page >= total - RECENT), math.inf, score)
    score = torch.where(page < total, score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget]
    order = torch.where(order < total, order, P)
    order = torch.sort(order, dim=-1).values
    out = torch.full((T, KH, budget), -1, dtype=torch.int32, device=score.device)
    out[..., : order.shape[-1]] = torch.where(order < P, order, -1).to(torch.int32)
    return out


def _append_plain(s):
    hq, kh, d, li = s["hq"], s["kh"], s["d"], s["layer"]
    T = s["qkv"].shape[0]
    x = s["qkv"].view(T, hq + 2 * kh, d).float()
    qk, v = x[:, : hq + kh], x[:, hq + kh:]
    if s["wq"] is not None:
        w = torch.cat([s["wq"].float().expand(hq, d), s["wk"].float().expand(kh, d)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    cs = s["cos_sin"][s["pos"].long()][:, None]
    c, sn = cs[..., : d // 2], cs[..., d // 2:]
    a, b = qk[..., : d // 2], qk[..., d // 2:]
    qk = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    kv = torch.stack([qk[:, hq:], v], 1)                                   # [T, 2, KH, D]
    fp8 = s["scale"] is not None
    if fp8:
        kv = (kv / s["scale"][li][None, :, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        kv = kv.to(torch.bfloat16)
    page, off = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    raw = s["cache"].view(torch.uint8) if fp8 else s["cache"]
    raw[page, li, :, :, off] = kv.view(torch.uint8) if fp8 else kv
    last = torch.full((raw.shape[0],), -1, device=page.device).scatter_reduce(0, page, off, "amax")
    rows = raw[page, li, 0]                                                # [T, KH, 16, D]
    rows = (rows.view(torch.float8_e4m3fn) if fp8 else rows).float()
    seen = (torch.arange(PAGE, device=page.device)[None] <= last[page][:, None])[:, None, :, None]
    b = torch.stack([torch.where(seen, rows, math.inf).amin(2), torch.where(seen, rows, -math.inf).amax(2)], 2)
    b = b.to(s["bounds"].dtype)
    (s["bounds"].view(torch.uint8) if fp8 else s["bounds"])[page, li] = b.view(torch.uint8) if fp8 else b
    return {"q": qk[:, :hq].reshape(T, hq * d).to(torch.bfloat16), "cache": s["cache"], "bounds": s["bounds"]}


def _select_plain(s):
    hq, kh, d = s["hq"], s["kh"], s["d"]
    T = s["q"].shape[0]
    q = s["q"].view(T, kh, hq // kh, d).double()            # 64 bits: scores next to the border decide
    up, dn = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)                  # [T, KH, D]
    raw = s["bounds"].view(torch.uint8) if s["bounds"].dtype == torch.float8_e4m3fn else s["bounds"]
    b = raw[s["bt"].long(), s["layer"]].view(s["bounds"].dtype).double()   # [B, P, KH, 2, D]
    b = b.permute(0, 2, 4, 3, 1)[s["seq"]]                                 # [T, KH, D, 2, P]
    score = (dn[..., None] * b[:, :, :, 0]).sum(2) + (up[..., None] * b[:, :, :, 1]).sum(2)
    return _choose(score, s["pos"].long() + 1, s["budget"])


def _values(rows, case):
    """Stored rows as fp32 values."""
    if case["kv"] != "q4":
        return rows.float()
    d = case["d"]
    code = torch.stack([rows[..., : d // 2] & 15, rows[..., : d // 2] >> 4], -1).flatten(-2).float()
    sm = rows[..., d // 2:].contiguous().view(torch.float16).float().unflatten(-1, (d // 32, 2))
    return (code.unflatten(-1, (d // 32, 32)) * sm[..., :1] + sm[..., 1:]).flatten(-2)


def _attend_plain(s):
    hq, kh, d, li = s["hq"], s["kh"], s["d"], s["layer"]
    T, _, S = s["pages"].shape
    sel = s["pages"].long()
    phys = torch.gather(s["bt"].long()[s["seq"]][:, None].expand(T, kh, -1), 2, sel.clamp(min=0))
    head = torch.arange(kh, device=sel.device)[None, :, None]
    fp8 = s["scale"] is not None
    raw = s["cache"].view(torch.uint8) if fp8 else s["cache"]
    kv = [_values(x.view(torch.float8_e4m3fn) if fp8 else x, s["case"]).flatten(2, 3)
          for x in (raw[phys, li, 0, head], raw[phys, li, 1, head])]       # [T, KH, S * 16, D]
    if fp8:
        kv = [x * s["scale"][li, i][None, :, None, None] for i, x in enumerate(kv)]
    key = (sel[..., None] * PAGE + torch.arange(PAGE, device=sel.device)).flatten(2)
    seen = (sel[..., None].expand(T, kh, S, PAGE).flatten(2) >= 0) & (key <= s["pos"][:, None, None])
    q = s["q"].view(T, kh, hq // kh, d).float()
    sc = (q @ kv[0].transpose(-1, -2)) * s["sm_scale"]
    sc = torch.where(seen[:, :, None], sc, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    return ((p @ kv[1]) / p.sum(-1, keepdim=True)).reshape(T, hq * d).to(torch.bfloat16)


def run(s):
    op = s["case"]["op"]
    if own:
        from vramancer_b200 import ops
        if op == "append":
            q = ops.qk_norm_rope_kv_write(s["qkv"], s["wq"], s["wk"], 1e-6, s["pos"], s["cos_sin"], s["cache"],
                                          s["slots"], s["scale"], s["layer"], s["hq"], s["kh"], s["d"],
                                          key_bounds=s["bounds"])
            return {"q": q, "cache": s["cache"], "bounds": s["bounds"]}
        if op == "select":
            return ops.select_pages(s["q"], s["bounds"], s["layer"], s["bt"], s["ctx"], s["hq"], s["budget"],
                                    sinks=SINKS, recent=RECENT, cu_q=s["cu_q"])
        return ops.paged_attention_selected(s["q"], s["cache"], s["layer"], s["bt"], s["ctx"], s["pages"],
                                            s["scale"], s["sm_scale"], s["hq"], cu_q=s["cu_q"])
    return {"append": _append_plain, "select": _select_plain, "attend": _attend_plain}[op](s)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    before, new, after = _sizes(case)
    hq, kh, d, T = case["hq"], case["kh"], case["d"], sum(new)
    el = 1 if case["kv"] == "fp8" else 2
    row = _row(case) * (2 if case["kv"] == "bf16" else 1)
    if case["op"] == "append":
        touched = sum(-(-b // PAGE) - a // PAGE for a, b in zip(before, after))
        old = sum(a % PAGE for a in before)
        return {"bytes": T * ((hq + 2 * kh) + hq) * d * 2 + T * 2 * kh * row + T * (4 * d + 8) + old * kh * row
                + touched * kh * 2 * d * el, "flops": T * (hq + kh) * d * 7}
    pages = [-(-n // PAGE) for n in after]
    if case["op"] == "select":
        scored = [max(0, p - SINKS - RECENT) if p > case["budget"] else 0 for p in pages]
        return {"bytes": sum(scored) * kh * (2 * d * el + 4) + T * hq * d * 2 + T * kh * case["budget"] * 4,
                "flops": sum(n * p for n, p in zip(new, scored)) * kh * 4 * d}
    read = [min(p, case["budget"]) for p in pages]
    union = [min(p, n * r) for p, n, r in zip(pages, new, read)]
    return {"bytes": sum(union) * kh * 2 * PAGE * row + 2 * T * hq * d * 2 + T * kh * case["budget"] * 4,
            "flops": sum(n * r for n, r in zip(new, read)) * PAGE * hq * d * 4}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return None                       # whole numbers
    hq, kh, d, li = s["hq"], s["kh"], s["d"], s["layer"]
    if case["op"] == "attend":
        out = torch.empty(s["q"].shape[0], hq * d, dtype=torch.float64, device="cuda")
        fp8 = s["scale"] is not None
        raw = s["cache"].view(torch.uint8) if fp8 else s["cache"]
        for t in range(out.shape[0]):
            q = s["q"][t].double().view(hq, d)
            n = int(s["pos"][t]) + 1
            for h in range(kh):
                sel = s["pages"][t, h]
                sel = sel[sel >= 0].long()
                tok = (sel[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()
                rows = raw[s["bt"][s["seq"][t]].long()[sel], li, :, h].transpose(0, 1).flatten(1, 2)[:, tok < n]
                if case["kv"] == "q4":
                    byte = rows[..., : d // 2].long()
                    code = torch.empty(*rows.shape[:-1], d, dtype=torch.float64, device="cuda")
                    code[..., 0::2], code[..., 1::2] = (byte % 16).double(), (byte // 16).double()
                    sm = rows[..., d // 2:].contiguous().view(torch.float16).double()
                    kv = code * sm[..., 0::2].repeat_interleave(32, -1) + sm[..., 1::2].repeat_interleave(32, -1)
                elif fp8:
                    kv = rows.view(torch.float8_e4m3fn).double() * s["scale"][li, :, h].double()[:, None, None]
                else:
                    kv = rows.double()
                grp = slice(h * (hq // kh), (h + 1) * (hq // kh))
                p = torch.softmax(q[grp] @ kv[0].t() * s["sm_scale"], -1)
                out[t].view(hq, d)[grp] = p @ kv[1]
        return out
    T = s["qkv"].shape[0]
    x = s["qkv"].double().view(T, -1, d)
    heads = []
    for h in range(hq + kh):
        y = x[:, h]
        if s["wq"] is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * (s["wq"] if h < hq else s["wk"]).double()
        z = torch.complex(y[:, : d // 2], y[:, d // 2:])
        cs = s["cos_sin"][s["pos"].long()].double()
        z = z * torch.complex(cs[:, : d // 2], cs[:, d // 2:])
        heads.append(torch.cat([z.real, z.imag], -1))
    q = torch.stack(heads[:hq], 1).reshape(T, hq * d)
    cache, bounds = s["cache"].double(), s["bounds"].double()
    slots = s["slots"].long()
    for h in range(kh):
        for i, y in enumerate((heads[hq + h], x[:, hq + kh + h])):
            if s["scale"] is not None:
                y = (y / s["scale"][li, i, h].double()).clamp(-448, 448)
            cache[slots // PAGE, li, i, h, slots % PAGE] = y
    ends = torch.tensor(_sizes(case)[2], device="cuda")
    firsts = torch.tensor(_sizes(case)[0], device="cuda") // PAGE
    for b in range(len(ends)):
        n = int(ends[b])
        idx = torch.arange(int(firsts[b]), -(-n // PAGE), device="cuda")
        k = cache[s["bt"][b].long()[idx], li, 0]                                   # [pages, KH, 16, D]
        live = (idx[:, None] * PAGE + torch.arange(PAGE, device="cuda") < n)[:, None, :, None]
        bounds[s["bt"][b].long()[idx], li, :, 0] = k.masked_fill(~live, math.inf).min(2).values
        bounds[s["bt"][b].long()[idx], li, :, 1] = k.masked_fill(~live, -math.inf).max(2).values
    return {"q": q, "cache": cache, "bounds": bounds}
