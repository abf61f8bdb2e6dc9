"""Block-sparse decode attention: append with key bounds, page selection, attention over
selected pages.  Every operator is held against its formula in 64 bits (written here, apart
from the CPU forms of vramancer_b200.ops), on the CPU and on the GPU.

Tolerances.  A value rounded once to a type of unit roundoff u = finfo.eps / 2 is off by at
most u times itself.  fp32 sums of n products add about n * 2^-24 times the sum of their
magnitudes, which the slack terms (2^-18 and above) cover for the lengths used here."""
import math

import pytest
import torch

from vramancer_b200 import ops
from vramancer_b200.kv import q4

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}
POOLS = {"bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn, "q4": torch.uint8}


def make_pool(kind, pages, layers, KH, D, dev, seed=0, scale=1.0):
    """A pool of random rows and its kv_scale (fp8)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, layers, 2, KH, 16, D, generator=g) * scale
    if kind == "q4":
        return q4.quantize(x).to(dev), None
    if kind == "fp8":
        ks = 0.02 + 0.03 * torch.rand(layers, 2, KH, generator=g)
        return (x / ks[None, :, :, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).to(dev), ks.to(dev)
    return x.bfloat16().to(dev), None


def values(cache, kv_scale=None):
    """Pool rows as float64 values [pages, layers, 2, KH, 16, D]."""
    c = cache.cpu()
    if c.dtype == torch.uint8:
        D = c.shape[-1] * 8 // 5
        code = torch.stack([c[..., :D // 2] & 15, c[..., :D // 2] >> 4], -1).flatten(-2).double()
        sm = c[..., D // 2:].contiguous().view(torch.float16).double()
        return code * sm[..., 0::2].repeat_interleave(32, -1) + sm[..., 1::2].repeat_interleave(32, -1)
    v = c.float().double()
    if kv_scale is not None:
        v = v * kv_scale.cpu().double()[None, :, :, :, None, None]
    return v


def tables(lens, width, pages, dev, seed=0):
    """Disjoint random pages for sequences of the given lengths."""
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(pages, generator=g).int()
    bt, at = torch.zeros(len(lens), width, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        p = -(-n // 16)
        bt[i, :p] = perm[at:at + p]
        at += p
    assert at <= pages
    return bt.to(dev)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------------------- append
def append_ref(qkv, wq, wk, eps, pos, cos_sin, Hq, KH, D):
    """(q, k, v) in 64 bits, unrounded: [T, heads, D]."""
    x = qkv.cpu().double().view(qkv.shape[0], Hq + 2 * KH, D).clone()
    for t in range(x.shape[0]):
        for h in range(Hq + KH):
            y = x[t, h]
            if wq is not None:
                y = y / math.sqrt(float(y.square().mean()) + eps) * (wq if h < Hq else wk).cpu().double()
            if cos_sin is not None:
                rot = cos_sin.shape[1]
                cs = cos_sin[int(pos[t])].cpu().double()
                z = torch.complex(y[:rot // 2], y[rot // 2:rot]) * torch.complex(cs[:rot // 2], cs[rot // 2:])
                y = torch.cat([z.real, z.imag, y[rot:]])
            x[t, h] = y
    return x[:, :Hq], x[:, Hq:Hq + KH], x[:, Hq + KH:]


def check_append(dev, kind, Hq, KH, D, starts, news, *, norm, rot, layers=2, layer=1, bounds=True, seed=0,
                 skip=(), qkv_scale=1.0, page_step=1, alias=False):
    g = torch.Generator().manual_seed(seed)
    T, W = sum(news), (Hq + 2 * KH) * D
    ends = [a + b for a, b in zip(starts, news)]
    pages = sum(-(-n // 16) for n in ends) + 3
    cache, ks = make_pool(kind, pages, layers, KH, D, dev, seed + 1)
    bt = tables(ends, max(-(-n // 16) for n in ends), pages, dev, seed + 2)
    buf = (torch.randn(T, W + 24, generator=g) * qkv_scale).bfloat16().to(dev)
    qkv = buf[:, 8:8 + W]                                     # strided rows
    wq = (1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(dev) if norm else None
    wk = (1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(dev) if norm else None
    pos = torch.cat([torch.arange(a, b) for a, b in zip(starts, ends)])
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(news)])
    slots = bt.cpu()[seq, pos // 16] * 16 + pos % 16
    for t in skip:
        slots[t] = -1
    cs = ops.rope_cos_sin(max(ends), rot, 1e4, dev) if rot else None
    kb = ops.key_bounds_for(cache) if bounds else None
    if bounds:                                                # must be left alone where no page is written
        kb.copy_(torch.full(kb.shape, 7.0).to(kb.dtype))
    before, qkv0 = cache.clone(), qkv.clone()
    out = qkv[:, :Hq * D] if alias else None
    q = ops.qk_norm_rope_kv_write(qkv, wq, wk, 1e-6, pos.int().to(dev), cs, cache, slots.int().to(dev), ks, layer,
                                  Hq, KH, D, key_bounds=kb, out=out)
    rq, rk, rv = append_ref(qkv0, wq, wk, 1e-6, pos, cs, Hq, KH, D)
    if alias:
        assert q.data_ptr() == qkv.data_ptr()
        assert torch.equal(qkv[:, Hq * D:], qkv0[:, Hq * D:])
    else:
        assert torch.equal(qkv, qkv0)
    mag = float(rq.abs().max().clamp(min=float(rk.abs().max())))
    tol = U[torch.bfloat16] * rq.abs() + 2.0 ** -18 * mag
    assert ((q.cpu().double().view(T, Hq, D) - rq).abs() <= tol).all()

    # the pool: written rows against the formula, every other byte as it was
    got, raw, raw0 = values(cache, ks)[:, layer], cache.cpu().view(torch.uint8), before.cpu().view(torch.uint8)
    mask = torch.zeros(pages, 16, dtype=torch.bool)
    for t in range(T):
        if slots[t] < 0:
            continue
        p, o = int(slots[t]) // 16, int(slots[t]) % 16
        mask[p, o] = True
        for i, r in ((0, rk[t]), (1, rv[t])):
            e = (got[p, i, :, o] - r).abs()
            if kind == "bf16":
                tol = U[torch.bfloat16] * r.abs() + 2.0 ** -18 * mag
            elif kind == "fp8":
                s = ks[layer, i].cpu().double()[:, None]
                # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below its
                # smallest normal); values past the largest code saturate
                r = r.clamp(-448 * s, 448 * s)
                e = (got[p, i, :, o] - r).abs()
                tol = U[torch.float8_e4m3fn] * r.abs() + s * 2.0 ** -10 + 2.0 ** -18 * mag
            else:
                # half a code step, plus the fp16 rounding of scale (15 steps) and minimum
                gr = r.unflatten(-1, (D // 32, 32))
                span, m = gr.amax(-1) - gr.amin(-1), gr.abs().amax(-1)
                tol = (span / 30 + U[torch.float16] * (span + 2 * m) + 2.0 ** -18 * mag + 2.0 ** -14)
                tol = tol.repeat_interleave(32, -1)
            assert (e <= tol * (1 + 2.0 ** -10)).all(), (kind, t, i, float((e - tol).max()))
    same = raw == raw0
    same[:, layer] |= mask[:, None, None, :, None]
    assert same.all()

    if bounds:
        # the bounds of exactly the stored keys
        stored = values(cache)[:, layer, 0]                                # codes, before kv_scale
        got_b = kb.cpu().float().double()
        for p in range(pages):
            offs = [int(s) % 16 for s in slots if s >= 0 and int(s) // 16 == p]
            if not offs:
                assert (got_b[p] == 7.0).all()
                continue
            rows = stored[p, :, : max(offs) + 1]
            want = torch.stack([rows.amin(1), rows.amax(1)], 1)
            tol = U[torch.bfloat16] * want.abs() + (2.0 ** -18 * mag if kind == "q4" else 0)
            if kind != "q4":
                assert torch.equal(got_b[p, layer], want), p               # stored keys are values of the bounds' type
            assert ((got_b[p, layer] - want).abs() <= tol).all()
            for other in range(layers):
                if other != layer:
                    assert (got_b[p, other] == 7.0).all()


HEADS = [(8, 2, 128), (14, 2, 64), (5, 1, 128), (3, 3, 64)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("Hq,KH,D", HEADS)
@pytest.mark.parametrize("norm,part", [(True, "full"), (False, "full"), (True, "none"), (False, "half")])
def test_append_chunks(dev, kind, Hq, KH, D, norm, part):
    """Ragged chunks: starts and ends inside pages, runs across tile borders, one token."""
    rot = {"full": D, "none": 0, "half": D // 2}[part]
    check_append(dev, kind, Hq, KH, D, [0, 7, 16, 31, 5], [33, 1, 15, 50, 2], norm=norm, rot=rot, seed=Hq + D)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("batch", [1, 2, 17, 40])
def test_append_decode(dev, kind, batch):
    """One token a sequence at every offset of a page, some rows without a slot."""
    check_append(dev, kind, 8, 2, 128, [3 * i + i % 16 for i in range(batch)], [1] * batch, norm=True, rot=128,
                 skip=[1] if batch > 2 else [], seed=batch)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("rot", [2, 34, 126])
def test_append_odd_rotation(dev, rot):
    check_append(dev, "bf16", 4, 2, 128, [3], [21], norm=True, rot=rot, seed=rot)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
def test_append_without_bounds_in_place(dev, kind):
    check_append(dev, kind, 8, 2, 128, [5, 0], [20, 3], norm=True, rot=128, bounds=False, alias=True)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("scale", [1e-6, 1e4])
def test_append_magnitudes(dev, scale):
    """q / k far from 1: the norm's eps counts, fp8 values saturate."""
    for kind in ("bf16", "fp8"):
        check_append(dev, kind, 4, 2, 64, [2], [19], norm=True, rot=64, qkv_scale=scale)
        check_append(dev, kind, 4, 2, 64, [2], [19], norm=False, rot=64, qkv_scale=scale)


@pytest.mark.parametrize("dev", DEVICES)
def test_append_non_finite_keys(dev):
    """Bounds stay finite: an infinite key counts as the largest value, a NaN as both extremes."""
    Hq, KH, D = 2, 1, 64
    qkv = torch.zeros(3, (Hq + 2 * KH) * D).bfloat16()
    qkv[0, Hq * D] = math.inf
    qkv[1, Hq * D + 1] = -math.inf
    qkv[2, Hq * D + 2] = math.nan
    cache = torch.zeros(2, 1, 2, KH, 16, D).bfloat16().to(dev)
    kb = ops.key_bounds_for(cache)
    ops.qk_norm_rope_kv_write(qkv.to(dev), None, None, 0.0, None, None, cache, i32([16, 17, 18], dev), None, 0, Hq,
                              KH, D, key_bounds=kb)
    top = torch.finfo(torch.bfloat16).max
    want = torch.zeros(2, D)
    want[1, 0], want[0, 1], want[0, 2], want[1, 2] = top, -top, -top, top
    assert torch.equal(kb[1, 0, 0].float().cpu(), want)
    assert torch.equal(kb[0].float().cpu(), torch.zeros(1, KH, 2, D))


@pytest.mark.parametrize("dev", DEVICES)
def test_append_rewrites_and_reuses_pages(dev):
    """A page used again starts from its first row; rows behind the last one written (a
    rejected draft) do not count."""
    Hq, KH, D = 2, 1, 64
    cache = torch.zeros(1, 1, 2, KH, 16, D).bfloat16().to(dev)
    kb = ops.key_bounds_for(cache)

    def put(vals, first):
        qkv = torch.zeros(len(vals), (Hq + 2 * KH) * D)
        qkv[:, Hq * D:(Hq + KH) * D] = torch.tensor(vals)[:, None]
        ops.qk_norm_rope_kv_write(qkv.bfloat16().to(dev), None, None, 0.0, None, None, cache,
                                  i32(list(range(first, first + len(vals))), dev), None, 0, Hq, KH, D, key_bounds=kb)
        return float(kb[0, 0, 0, 0, 0]), float(kb[0, 0, 0, 1, 0])

    assert put([1.0, 2.0], 0) == (1, 2)
    assert put([9.0, -9.0], 2) == (-9, 9)
    assert put([3.0], 2) == (1, 3)                # slot 3 is behind
    assert put([5.0], 0) == (5, 5)                # the page starts again
    assert put([4.0] * 15, 1) == (4, 5)


@pytest.mark.parametrize("dev", DEVICES)
def test_append_rising_slots_with_gaps(dev):
    """Tokens of a page in rising slots that leave some out: the rows between count as they
    are in the pool."""
    Hq, KH, D = 2, 1, 64
    cache = torch.zeros(2, 1, 2, KH, 16, D).bfloat16()
    cache[1, 0, 0, 0, :, 0] = torch.arange(16).bfloat16() - 20
    cache = cache.to(dev)
    kb = ops.key_bounds_for(cache)
    qkv = torch.zeros(4, (Hq + 2 * KH) * D)
    qkv[:, Hq * D] = torch.tensor([1.0, 2.0, 3.0, -4.0])
    ops.qk_norm_rope_kv_write(qkv.bfloat16().to(dev), None, None, 0.0, None, None, cache, i32([16, 19, 26, 1], dev),
                              None, 0, Hq, KH, D, key_bounds=kb)
    assert kb[1, 0, 0, :, 0].tolist() == [-19.0, 3.0]          # rows 1..9 but 3: -19 .. -11
    assert kb[0, 0, 0, :, 0].tolist() == [-4.0, 0.0]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -9, 300.0])
def test_bounds_hold_for_every_key(dev, kind, scale):
    """No stored key gives a group a larger sum of scores than its page's bounds do; bounds of
    four-bit keys, which are rounded to bf16, may fall short by half a step of each."""
    Hq, KH, D, n = 8, 2, 64, 71
    g = torch.Generator().manual_seed(int(scale))
    cache, ks = make_pool(kind, 6, 1, KH, D, dev)
    kb = ops.key_bounds_for(cache)
    qkv = (torch.randn(n, (Hq + 2 * KH) * D, generator=g) * scale).bfloat16().to(dev)
    q = ops.qk_norm_rope_kv_write(qkv, None, None, 0.0, None, None, cache, i32(list(range(16, 16 + n)), dev), ks, 0,
                                  Hq, KH, D, key_bounds=kb).cpu().double().view(n, KH, -1, D)
    keys = values(cache)[1:, 0, 0].transpose(0, 1).reshape(KH, -1, D)[:, :n]            # before kv_scale
    b = kb.cpu().float().double()[1:, 0].repeat_interleave(16, 0)[:n].transpose(0, 1)   # [KH, token, 2, D]
    up, dn = q.clamp(min=0).sum(2).transpose(0, 1), q.clamp(max=0).sum(2).transpose(0, 1)
    score = torch.einsum("hqd,hkd->hqk", up, b[:, :, 1]) + torch.einsum("hqd,hkd->hqk", dn, b[:, :, 0])
    exact = torch.einsum("hqd,hkd->hqk", q.sum(2).transpose(0, 1), keys)
    mag = torch.einsum("hqd,hkd->hqk", up, b[:, :, 1].abs()) - torch.einsum("hqd,hkd->hqk", dn, b[:, :, 0].abs())
    slack = U[torch.bfloat16] * (1 + 2.0 ** -7) if kind == "q4" else 0.0                # of the key, by its bound
    assert (exact <= score + (slack + 2.0 ** -45) * mag).all()


# ---------------------------------------------------------------------------- selection
def rows_of(T, ctx, cu):
    if cu is None:
        return {t: (t, ctx[t]) for t in range(T)}
    return {t: (b, ctx[b] - (cu[b + 1] - 1 - t)) for b in range(len(cu) - 1) for t in range(cu[b], cu[b + 1])}


def select_ref(q, kb, layer, bt, rows, Hq, budget, sinks, recent):
    KH, D = kb.shape[2], kb.shape[4]
    G = Hq // KH
    out = {}
    for t, (b, n) in rows.items():
        total = max(0, -(-n // 16))
        for h in range(KH):
            if total <= budget:
                out[t, h] = list(range(total)) + [-1] * (budget - total)
                continue
            qd = q[t, h * G * D:(h + 1) * G * D].cpu().double().view(G, D)
            bd = kb[bt[b, :total].long(), layer, h].cpu().float().double()
            s = (torch.maximum(qd, torch.zeros(1)).sum(0) * bd[:, 1] + torch.minimum(qd, torch.zeros(1)).sum(0) * bd[:, 0]).sum(-1)
            mid = sorted(range(sinks, total - recent), key=lambda p: (-float(s[p]), p))[: budget - sinks - recent]
            out[t, h] = sorted(list(range(sinks)) + mid + list(range(total - recent, total)))
    return out


def check_select(dev, kind, Hq, KH, D, ctx, budget, *, sinks=1, recent=1, chunk=None, seed=0, ints=False, layers=2,
                 layer=1, extra_rows=0):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-n // 16) for n in ctx) + 2
    bt = tables(ctx, max(-(-n // 16) for n in ctx) + 1, pages, dev, seed)
    if ints:                                                  # many exact ties
        mid = torch.randint(-1, 2, (pages, layers, KH, D), generator=g).float()
        kb = torch.stack([mid - 1, mid + 1], 3)
        kb = kb[torch.randint(0, max(2, pages // 8), (pages,), generator=g)]
    else:
        mid, half = (torch.randn(pages, layers, KH, D, generator=g) for _ in range(2))
        kb = torch.stack([mid - half.abs(), mid + half.abs()], 3)
    kb = kb.to(torch.float8_e4m3fn if kind == "fp8" else torch.bfloat16).to(dev)
    cu, T = None, len(ctx)
    if chunk is not None:
        cu = [0]
        for n in chunk:
            cu.append(cu[-1] + n)
        T = cu[-1]
    q = torch.randn(T + extra_rows, Hq * D + 16, generator=g)
    if ints:
        q = torch.randint(-1, 2, q.shape, generator=g).float()
    q = q.bfloat16().to(dev)[:, 8:]
    out = torch.full((T + extra_rows, KH, budget), 77, dtype=torch.int32, device=dev)
    got = ops.select_pages(q, kb, layer, bt, i32(ctx, dev), Hq, budget, sinks=sinks, recent=recent,
                           cu_q=None if cu is None else i32(cu, dev), out=out)
    assert got is out
    want = select_ref(q, kb, layer, bt, rows_of(T, ctx, cu), Hq, budget, sinks, recent)
    got = got.cpu()
    for (t, h), w in want.items():
        assert got[t, h].tolist() == w, (t, h)
    assert (got[T:] == 77).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("Hq,KH,D", HEADS)
@pytest.mark.parametrize("ints", [False, True])
def test_select(dev, kind, Hq, KH, D, ints):
    """No token, one page, the budget exactly, one page more, odd lengths, many pages."""
    check_select(dev, kind, Hq, KH, D, [0, 1, 16, 16 * 9, 16 * 9 + 1, 997, 4000, 333], 9, seed=D + Hq, ints=ints)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("sinks,recent,budget", [(0, 1, 1), (0, 1, 2), (2, 3, 5), (2, 3, 6), (0, 4, 31), (5, 1, 40)])
def test_select_forced_pages(dev, sinks, recent, budget):
    check_select(dev, "bf16", 8, 2, 128, [700, 16 * budget, 16 * budget + 3], budget, sinks=sinks, recent=recent)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_select_rows_of_a_chunk(dev, kind):
    """Verify rows and chunks: each row sees its own length; empty sequences; rows behind the last."""
    check_select(dev, kind, 14, 2, 64, [301, 40, 777, 160], 6, chunk=[5, 0, 33, 1], recent=2, extra_rows=3)


@pytest.mark.parametrize("dev", DEVICES)
def test_select_many_sequences_of_a_chunk(dev):
    check_select(dev, "bf16", 4, 2, 64, [60 + 16 * (i % 5) for i in range(70)], 4, chunk=[1 + i % 3 for i in range(70)])


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [2047, 2048, 8192, 20001])
def test_select_long(pages):
    check_select("cuda", "bf16", 8, 1, 128, [pages * 16 - 5], 128, layers=1, layer=0, seed=pages)
    check_select("cuda", "fp8", 8, 1, 64, [pages * 16 - 5], pages - 3, layers=1, layer=0, seed=pages, ints=True)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("same", [0.0, 1.0, -2.5])
def test_select_all_pages_alike(dev, same):
    """Every score the same (one of them -0): the lowest pages."""
    kb = torch.full((100, 1, 1, 2, 64), same).bfloat16()
    if same == 0.0:
        kb[::2] = -0.0
    bt = torch.arange(100, dtype=torch.int32)[None]
    got = ops.select_pages(torch.ones(1, 64).bfloat16().to(dev), kb.to(dev), 0, bt.to(dev), i32([1600], dev), 1, 20)
    assert got[0, 0].tolist() == list(range(19)) + [99]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float8_e4m3fn])
def test_select_many_equal_scores_at_the_border(dev, dt):
    """Hundreds of pages tie around the border (more than a short list holds), others lie
    above and below: the lowest of the tied."""
    n = 1001
    kb = torch.full((n, 1, 1, 2, 64), 1.0)
    kb[::7] = 2.0
    kb[3::7] = 0.5
    bt = torch.arange(n, dtype=torch.int32)[None]
    got = ops.select_pages(torch.ones(1, 64).bfloat16().to(dev), kb.to(dt).to(dev), 0, bt.to(dev),
                           i32([16 * n], dev), 1, 400, sinks=0, recent=1)
    v = kb[:n - 1, 0, 0, 1, 0].tolist()
    want = sorted(range(n - 1), key=lambda p: (-v[p], p))[:399]
    assert got[0, 0].tolist() == sorted(want) + [n - 1]


@pytest.mark.parametrize("dev", DEVICES)
def test_select_close_scores(dev):
    """Scores that differ in the last place of 64-bit arithmetic's exact sums only: fp32 sums
    would tie or swap them."""
    kb = torch.zeros(64, 1, 1, 2, 64)
    kb[:, 0, 0, 1, 0] = 2.0 ** 20
    kb[:, 0, 0, 1, 1] = torch.arange(64).float() * 2.0 ** -10
    bt = torch.randperm(64, generator=torch.Generator().manual_seed(1)).int()[None]
    got = ops.select_pages(torch.ones(1, 64).bfloat16().to(dev), kb.bfloat16().to(dev), 0, bt.to(dev),
                           i32([1024], dev), 1, 10, sinks=0, recent=1)
    order = sorted(range(63), key=lambda p: -int(bt[0, p]))[:9]
    assert got[0, 0].tolist() == sorted(order) + [63]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("outlier", [8.0, 64.0, 416.0])
@pytest.mark.parametrize("budget", [5, 128])
def test_select_beside_an_outlier_channel(dev, kind, outlier, budget):
    """One channel far above the others, alike in all pages: fp32 scores leave few to many
    pages undecided.  All values are multiples of 1/16, so that 64-bit sums are exact."""
    Hq, KH, D, ctx = 8, 2, 128, [16 * 1500, 16 * 300 - 3, 16 * 2000 + 1]
    g = torch.Generator().manual_seed(int(outlier) + budget)
    pages = sum(-(-n // 16) for n in ctx) + 1
    bt = tables(ctx, 2001, pages, dev, 3)
    step = 4 if kind == "fp8" else 16                         # e4m3 holds quarters up to 4
    mid = torch.randint(-2 * step, 2 * step + 1, (pages, 1, KH, D), generator=g) / step
    half = torch.randint(0, step + 1, (pages, 1, KH, D), generator=g) / step
    kb = torch.stack([mid - half, mid + half], 3)
    kb[..., 77] = outlier
    dt = torch.float8_e4m3fn if kind == "fp8" else torch.bfloat16
    assert torch.equal(kb.to(dt).float(), kb)
    q = torch.randint(-32, 33, (3, Hq, D), generator=g) / 16
    q[:, :, 77] = 4.0
    kb, q = kb.to(dt).to(dev), q.bfloat16().view(3, Hq * D).to(dev)
    got = ops.select_pages(q, kb, 0, bt, i32(ctx, dev), Hq, budget, sinks=1, recent=2).cpu()
    want = select_ref(q, kb, 0, bt, rows_of(3, ctx, None), Hq, budget, 1, 2)
    for (t, h), w in want.items():
        assert got[t, h].tolist() == w, (t, h)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_select_extreme_values(dev, kind):
    """Largest and smallest finite values, subnormals, infinite and NaN queries."""
    dt = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    fi = torch.finfo(dt)
    sub = fi.smallest_normal / 8
    kb = torch.zeros(40, 1, 1, 2, 64)
    kb[:, 0, 0, 1, 0] = torch.tensor([0.0, sub, 2 * sub, -sub, fi.smallest_normal, 1.0, fi.max, -fi.max] * 5)
    q = torch.zeros(4, 64)
    q[0, 0] = 1.0
    q[1, 0] = torch.finfo(torch.bfloat16).max
    q[2, 0] = math.inf
    q[3, 0], q[3, 1] = 1.0, math.nan
    bt = torch.arange(40, dtype=torch.int32).repeat(4, 1)
    args = (0, bt.to(dev), i32([640] * 4, dev), 1, 16)
    got = ops.select_pages(q.bfloat16().to(dev), kb.to(dt).to(dev), *args).cpu()
    mid = list(range(1, 39))
    v = kb.to(dt).double()[:, 0, 0, 1, 0].tolist()
    for t in (0, 1):
        want = sorted(mid, key=lambda p: (-v[p], p))[:14]
        assert got[t, 0].tolist() == [0] + sorted(want) + [39]
    # inf * 0 is NaN and comes first, then +inf; the last row's scores are all NaN
    nan_first = sorted(mid, key=lambda p: (0 if v[p] == 0 else 1 if v[p] > 0 else 2, p))[:14]
    assert got[2, 0].tolist() == [0] + sorted(nan_first) + [39]
    assert got[3, 0].tolist() == list(range(15)) + [39]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("j", [6, 8, 10, 12, 14, 18, 23])
def test_select_beside_cancelling_terms(dev, kind, D, pair, j):
    """One term of every 16 dims is 1 (with `pair` another is -1), the others are 2^-j and
    less, all of one sign: sums that drop low places of the small terms are off alike in all
    pages or not, by up to the selection's error bound.  64-bit sums are exact."""
    Hq, n, budget = 1, 900, 300
    g = torch.Generator().manual_seed(100 * j + D)
    steps = 16 if kind == "fp8" else 128
    kb = torch.randint(steps // 2, steps + 1, (n, 1, 1, 2, D), generator=g).float() / steps
    kb = kb.sort(3).values                                    # minima, maxima
    q = torch.randint(64, 128, (1, D), generator=g).float() / 128 * 2.0 ** -j
    q[0, ::16] = 1.0
    kb[..., ::16] = 1.0
    if pair:
        q[0, 1::16] = -1.0
        kb[..., 1::16] = 1.0
    # half of the pages: small terms in two of three dims only
    kb[::2, :, :, :, 2::3] = torch.where(torch.arange(2, D, 3) % 16 < 2, kb[::2, :, :, :, 2::3], 0.0)
    dt = torch.float8_e4m3fn if kind == "fp8" else torch.bfloat16
    assert torch.equal(kb.to(dt).float(), kb) and torch.equal(q.bfloat16().float(), q)
    bt = torch.randperm(n, generator=g).int()[None]
    kb, q = kb.to(dt).to(dev), q.bfloat16().to(dev)
    got = ops.select_pages(q, kb, 0, bt.to(dev), i32([16 * n - 7], dev), Hq, budget, sinks=1, recent=1).cpu()
    want = select_ref(q, kb, 0, bt, {0: (0, 16 * n - 7)}, Hq, budget, 1, 1)
    assert got[0, 0].tolist() == want[0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("rows,n", [(1, 6001), (3, 2999), (40, 1201)])
def test_select_does_not_depend_on_other_sequences_pages(kind, rows, n, cuda_errors_clean):
    """Pages that are not in a row's table cost it nothing, whatever keys they hold: page 0,
    another sequence's, with the largest bounds.  A row that takes bf16 ones into its error
    bound scores every page in 64 bits, 5 to 15 times as slow at these lengths."""
    dt = torch.float8_e4m3fn if kind == "fp8" else torch.bfloat16
    g = torch.Generator().manual_seed(n)
    mid, half = torch.randn(n + 1, 1, 8, 128, generator=g), torch.rand(n + 1, 1, 8, 128, generator=g)
    kb = torch.stack([mid - half, mid + half], 3).to(dt)
    kb[0] = 0.0
    loud = kb.clone()
    loud[0, :, :, 0], loud[0, :, :, 1] = -torch.finfo(dt).max, torch.finfo(dt).max
    bt = torch.stack([torch.randperm(n, generator=g).int() + 1 for _ in range(rows)]).cuda()
    q = torch.randn(rows, 8 * 128, generator=g).bfloat16().cuda()
    ctx = i32([16 * n - 3 * i for i in range(rows)], "cuda")
    res, us = [], []
    for b in (kb.cuda(), loud.cuda()):
        call = lambda: ops.select_pages(q, b, 0, bt, ctx, 8, 128)  # noqa: E731,B023
        res.append(call())
        times = []
        for _ in range(9):
            a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                call()
            z.record()
            z.synchronize()
            times.append(a.elapsed_time(z) * 200)
        us.append(sorted(times)[4])
    assert torch.equal(*res)
    assert us[1] < 2 * us[0], us


# ---------------------------------------------------------------------------- attention
def attend_ref(q, vals, layer, bt, rows, pages, sm_scale, Hq, kind):
    """{(row, kv head): (output, tolerance)} in 64 bits."""
    KH, D = vals.shape[3], vals.shape[5]
    G = Hq // KH
    out = {}
    for t, (b, n) in rows.items():
        for h in range(KH):
            toks = [(p, o) for p in pages[t, h].tolist() if p >= 0 for o in range(16) if p * 16 + o < n]
            if not toks:
                out[t, h] = (torch.zeros(G, D, dtype=torch.float64), torch.zeros(G, D))
                continue
            at = bt[b].cpu().long()[torch.tensor([p for p, _ in toks])]
            off = torch.tensor([o for _, o in toks])
            k, v = vals[at, layer, 0, h, off], vals[at, layer, 1, h, off]
            qd = q[t, h * G * D:(h + 1) * G * D].cpu().double().view(G, D)
            p = torch.softmax(qd @ k.t() * sm_scale, -1)
            o = p @ v
            a = p @ v.abs()
            # output rounding; the weights' rounding to bf16 / f16; f16 keys and values of
            # four-bit rows (2^-11 of each) move scores by at most 2^-11 sum |q k| each
            tol = U[torch.bfloat16] * o.abs() + 2.0 ** -18 * a
            tol = tol + (2.0 ** -8 if kind == "bf16" else 2.0 ** -11) * a
            if kind == "q4":
                worst = (qd.abs() @ k.abs().t() * abs(sm_scale)).amax(-1, keepdim=True)
                tol = tol + 2.0 ** -11 * a + 2 * 2.0 ** -11 * worst * a
            if kind != "bf16":                               # f16 weights below 2^-14 lose low bits
                tol = tol + 2.0 ** -25 * v.abs().sum(0)
            # fp32 scores: 2^-18 of their magnitudes' sum, twice (numerator and denominator)
            worst = (qd.abs() @ k.abs().t() * abs(sm_scale)).amax(-1, keepdim=True)
            out[t, h] = (o, tol + 2.0 ** -17 * worst * a)
    return out


def choose_pages(rows, KH, T, n_sel, seed, dev, order=False):
    g = torch.Generator().manual_seed(seed)
    pages = torch.full((T, KH, n_sel), -1, dtype=torch.int32)
    for t, (_, n) in rows.items():
        total = max(0, -(-n // 16))
        for h in range(KH):
            k = min(n_sel, total)
            p = torch.randperm(total, generator=g)[:k]
            if k:
                p[0] = total - 1                             # the partly filled page
                p = p.unique()
            pages[t, h, :len(p)] = p.int()[torch.randperm(len(p), generator=g)] if order else p.int()
    return pages.to(dev)


def check_attend(dev, kind, Hq, KH, D, ctx, n_sel, *, chunk=None, layers=2, layer=1, seed=0, extra_rows=0,
                 poison=True, order=False, qs=1.0, sm_scale=None):
    g = torch.Generator().manual_seed(seed)
    n_pages = sum(-(-n // 16) for n in ctx) + 2
    cache, ks = make_pool(kind, n_pages, layers, KH, D, dev, seed)
    bt = tables(ctx, max(1, max(-(-n // 16) for n in ctx)), n_pages, dev, seed)
    cu, T = None, len(ctx)
    if chunk is not None:
        cu = [0]
        for n in chunk:
            cu.append(cu[-1] + n)
        T = cu[-1]
    rows = rows_of(T, ctx, cu)
    pages = choose_pages(rows, KH, T + extra_rows, n_sel, seed, dev, order)
    vals = values(cache, ks)
    if poison and kind != "q4":
        # NaN in every row that no query may read
        keep = torch.zeros(n_pages, KH, 16, dtype=torch.bool)
        for t, (b, n) in rows.items():
            for h in range(KH):
                for p in pages[t, h].tolist():
                    if p >= 0:
                        keep[int(bt[b, p]), h, : max(0, min(16, n - 16 * p))] = True
        c = cache.float()
        m = torch.zeros(c.shape, dtype=torch.bool)
        m[:, layer] = ~keep[:, None, :, :, None]
        cache = c.masked_fill(m.to(dev), math.nan).to(cache.dtype)
    q = (torch.randn(T + extra_rows, Hq * D + 16, generator=g) * qs).bfloat16().to(dev)[:, 8:]
    sm = sm_scale or 1 / math.sqrt(D)
    out = torch.full((T + extra_rows, Hq * D + 8), 7.0).bfloat16().to(dev)
    got = ops.paged_attention_selected(q, cache, layer, bt, i32(ctx, dev), pages, ks, sm, Hq,
                                       cu_q=None if cu is None else i32(cu, dev), out=out)
    assert got is out
    got = got.cpu().double()
    assert (got[T:] == 7.0).all() and (got[:, Hq * D:] == 7.0).all()
    G = Hq // KH
    for (t, h), (o, tol) in attend_ref(q, vals, layer, bt, rows, pages, sm, Hq, kind).items():
        e = (got[t, h * G * D:(h + 1) * G * D].view(G, D) - o).abs()
        assert (e <= tol * (1 + 2.0 ** -10)).all(), (t, h, float((e - tol).max()))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("Hq,KH,D", HEADS + [(8, 1, 128), (7, 1, 64)])
def test_attend(dev, kind, Hq, KH, D):
    check_attend(dev, kind, Hq, KH, D, [0, 1, 15, 16, 17, 100, 333, 1000], 7, seed=D + Hq)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("n_sel", [1, 2, 3, 8, 33, 64])
def test_attend_list_lengths(dev, kind, n_sel):
    """One page to more pages than a warp's batch of list entries, split over a cluster."""
    check_attend(dev, kind, 8, 2, 128, [1025], n_sel, seed=n_sel, order=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
def test_attend_batches(kind):
    """Batches on both sides of every split rule, and lists of several hundred pages."""
    check_attend("cuda", kind, 10, 2, 64, [200 + 7 * i for i in range(40)], 12, layers=1, layer=0)
    check_attend("cuda", kind, 8, 1, 128, [9001], 520, layers=1, layer=0)
    check_attend("cuda", kind, 4, 2, 128, [300] * 100, 5, layers=1, layer=0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
def test_attend_rows_of_a_chunk(dev, kind):
    check_attend(dev, kind, 14, 2, 64, [301, 40, 90, 160], 4, chunk=[5, 0, 20, 1], extra_rows=2)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["fp8", "q4"])
@pytest.mark.parametrize("qs", [2.0 ** -40, 2.0 ** 20])
def test_attend_query_magnitudes(dev, kind, qs):
    """Queries beyond the f16 range (their scale moves into the score's factor)."""
    check_attend(dev, kind, 8, 2, 128, [100, 257], 6, qs=qs, sm_scale=1 / qs / 11)


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_ignores_entries_out_of_reach(dev):
    """-1 anywhere in a list, and pages behind the context, add nothing; a row whose list
    has no page gives zeros."""
    cache, _ = make_pool("bf16", 8, 1, 1, 64, dev)
    bt = torch.arange(8, dtype=torch.int32, device=dev).repeat(3, 1)
    q = torch.randn(3, 128, generator=torch.Generator().manual_seed(0)).bfloat16().to(dev)
    ctx = i32([50, 50, 50], dev)
    a = i32([[[-1, 0, 7, -1, 2, 6]], [[0, 2, -1, -1, -1, -1]], [[-1, 4, -1, 5, -1, -1]]], dev)
    o = ops.paged_attention_selected(q[:1].repeat(3, 1), cache, 0, bt, ctx, a, None, 0.125, 2)
    assert torch.isfinite(o.float()).all() and (o[2] == 0).all()
    assert (o[0].float() - o[1].float()).abs().max() <= 2.0 ** -7 * o[1].float().abs().max()


@pytest.mark.parametrize("dev", DEVICES)
def test_attend_non_finite_scores(dev):
    """As softmax: +inf or only -inf scores give NaN; a -inf score beside finite ones is a zero weight."""
    cache = torch.zeros(2, 1, 2, 1, 16, 64).bfloat16()
    cache[:, 0, 1] = 1.0
    q = torch.zeros(1, 64).bfloat16()
    q[0, 0] = 1.0
    bt, ctx, pages = i32([[0, 1]], dev), i32([32], dev), i32([[[0, 1]]], dev)

    def run(rows, val):
        c = cache.clone()
        c[:, 0, 0, 0, rows, 0] = val
        return ops.paged_attention_selected(q.to(dev), c.to(dev), 0, bt, ctx, pages, None, 1.0, 1).float().cpu()

    assert run(slice(0, 16), -math.inf).isnan().all()
    assert run(slice(3, 4), math.inf).isnan().all()
    assert (run(slice(0, 8), -math.inf) == 1.0).all()


def small_pool(kind, dev, KH=1, D=64, pages=6, scale=1.0, seed=0):
    cache, ks = make_pool(kind, pages, 1, KH, D, dev, seed, scale=scale)
    return cache, ks, torch.arange(pages, dtype=torch.int32, device=dev)[None]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n_sel", [1, 40])
def test_attend_heads_of_unlike_magnitudes(dev, kind, D, n_sel):
    """Heads of one group whose queries lie 2^13 to 2^100 apart: each has its own scores."""
    mags = [1.0, 2.0 ** 13, 2.0 ** 26, 2.0 ** 100, 0.0, 2.0 ** -30, 1.0]
    cache, ks, bt = small_pool(kind, dev, D=D, pages=40, seed=D)
    q = torch.randn(1, 7, D, generator=torch.Generator().manual_seed(D)) * torch.tensor(mags)[:, None]
    q = q.bfloat16().view(1, 7 * D).to(dev)
    pages = torch.arange(n_sel, dtype=torch.int32)[None, None]
    got = ops.paged_attention_selected(q, cache, 0, bt, i32([640], dev), pages.to(dev), ks, 0.2, 7).cpu().double()
    (o, tol), = attend_ref(q, values(cache, ks), 0, bt, {0: (0, 640)}, pages, 0.2, 7, kind).values()
    e = (got.view(7, D) - o).abs()
    assert torch.isfinite(got).all()
    assert (e <= tol * (1 + 2.0 ** -10)).all(), (e - tol).amax(1)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("mag", [2.0 ** 124, 2.0 ** 125, 2.0 ** 126, 2.0 ** 127, 2.0 ** -120])
def test_attend_largest_and_smallest_queries(dev, kind, mag):
    """Finite queries of the last exponents are neither clipped nor taken for infinite.
    Keys of at most 1/16 keep the products finite in 32 bits, and sm_scale is an fp32 value."""
    cache, ks, bt = small_pool(kind, dev, scale=2.0 ** -7)
    if kind == "fp8":
        ks *= 2.0 ** -7
        cache, _, _ = small_pool(kind, dev, scale=1.0)
    assert values(cache, ks).abs().max() <= 1 / 16
    q = torch.zeros(1, 2, 64)
    q[0, 0, 5], q[0, 1, 9] = mag, -1.5 * mag
    q = q.bfloat16().view(1, 128).to(dev)
    pages = torch.arange(6, dtype=torch.int32)[None, None]
    sm = 2.0 ** 7 / mag
    got = ops.paged_attention_selected(q, cache, 0, bt, i32([90], dev), pages.to(dev), ks, sm, 2).cpu().double()
    (o, tol), = attend_ref(q, values(cache, ks), 0, bt, {0: (0, 90)}, pages, sm, 2, kind).values()
    e = (got.view(2, 64) - o).abs()
    assert (e <= tol * (1 + 2.0 ** -10)).all(), (e - tol).amax(1)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n_sel", [1, 40])
def test_attend_non_finite_queries(dev, kind, bad, n_sel):
    """An infinite or NaN query value makes its own head NaN and no other."""
    cache, ks, bt = small_pool(kind, dev, KH=2, pages=40)
    q = torch.randn(1, 6, 64, generator=torch.Generator().manual_seed(7))
    q[0, 1, 33] = bad
    q = q.bfloat16().view(1, 6 * 64).to(dev)
    pages = torch.arange(n_sel, dtype=torch.int32).repeat(1, 2, 1)
    got = ops.paged_attention_selected(q, cache, 0, bt, i32([640], dev), pages.to(dev), ks, 0.125, 6).cpu().double()
    got = got.view(6, 64)
    assert got[1].isnan().all()
    for (t, h), (o, tol) in attend_ref(q, values(cache, ks), 0, bt, {0: (0, 640)}, pages, 0.125, 6, kind).items():
        for i in range(3):
            if 3 * h + i != 1:
                assert ((got[3 * h + i] - o[i]).abs() <= tol[i] * (1 + 2.0 ** -10)).all(), (h, i)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
@pytest.mark.parametrize("below", [12.0, 25.4, 30.0])
@pytest.mark.parametrize("pages", [2, 700])
def test_attend_many_small_weights(dev, kind, below, pages):
    """One token 2^below above all others, which alone have values: their weights add up,
    however small each is."""
    x = torch.zeros(pages, 1, 2, 1, 16, 64)
    x[0, 0, 0, 0, 3, 0] = 1.0                                 # the key that stands out, its value 0
    x[:, 0, 1] = 1.0
    x[0, 0, 1, 0, 3] = 0.0
    dt = POOLS[kind]
    cache, ks = q4.quantize(x) if kind == "q4" else x.to(dt), torch.ones(1, 2, 1) if kind == "fp8" else None
    q = torch.zeros(1, 128)
    q[0, 0], q[0, 64] = 1.0, 0.5
    q = q.bfloat16()
    bt, lst = torch.arange(pages, dtype=torch.int32)[None], torch.arange(pages, dtype=torch.int32)[None, None]
    sm = below * math.log(2)
    got = ops.paged_attention_selected(q.to(dev), cache.to(dev), 0, bt.to(dev), i32([16 * pages], dev), lst.to(dev),
                                       None if ks is None else ks.to(dev), sm, 2).cpu().double().view(2, 64)
    vals = values(cache, ks)[:, 0]
    k, v = vals[:, 0, 0].flatten(0, 1), vals[:, 1, 0].flatten(0, 1)
    s = q.double().view(2, 64) @ k.t() * sm
    w = torch.softmax(s, -1)
    o = w @ v
    # output rounding; each weight's (half a step, in f16 at least 2^-39 of the largest); fp32
    # scores, 2^-18 of their size, above and below the fraction
    half = U[torch.bfloat16] if kind == "bf16" else U[torch.float16]
    small = 0 if kind == "bf16" else 2.0 ** -39 * w.amax(-1, keepdim=True) * 16 * pages
    tol = (U[torch.bfloat16] + half + 2.0 ** -17 * s.abs().amax(-1, keepdim=True) + 2.0 ** -18) * o + small
    if kind == "q4":
        # keys and values become f16: the stored key, 15 * f16(1 / 15) = 1 - 2^-12, lies half a
        # step of f16 from its neighbours.  Scores move by up to 2^-11 of themselves, weights
        # and their sum by that much each; values by 2^-11
        tol = tol + (2 * U[torch.float16] * s.abs().amax(-1, keepdim=True) + U[torch.float16]) * o
    assert ((got - o).abs() <= tol).all(), (float(got[0, 0]), float(o[0, 0]))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n_sel,ctx", [(1, 5), (3, 48), (40, 633), (128, 2049)])
def test_attend_weights_are_not_cut_to_bf16(dev, D, n_sel, ctx):
    """Over bf16 pages only the output is rounded to eight bits: weights keep 16 (2^-16 of
    each), scores and sums are fp32."""
    Hq, KH, n = 8, 2, -(-ctx // 16)
    cache, _ = make_pool("bf16", n, 1, KH, D, dev, seed=D + ctx)
    q = torch.randn(2, Hq * D, generator=torch.Generator().manual_seed(ctx)).bfloat16().to(dev)
    bt = torch.arange(n, dtype=torch.int32, device=dev).repeat(2, 1)
    rows = {0: (0, ctx), 1: (1, max(1, ctx - 9))}
    pages = choose_pages(rows, KH, 2, n_sel, 1, dev)
    sm = 1 / math.sqrt(D)
    got = ops.paged_attention_selected(q, cache, 0, bt, i32([n for _, n in rows.values()], dev), pages, None, sm, Hq)
    got, vals, G = got.cpu().double(), values(cache)[:, 0], Hq // KH
    for t, (b, m) in rows.items():
        for h in range(KH):
            sel = [p for p in pages[t, h].tolist() if p >= 0]
            tok = torch.tensor([16 * p + o for p in sel for o in range(16) if 16 * p + o < m])
            k, v = (vals[:, i, h].flatten(0, 1)[tok] for i in (0, 1))
            qd = q[t, h * G * D:(h + 1) * G * D].cpu().double().view(G, D)
            w = torch.softmax(qd @ k.t() * sm, -1)
            worst = (qd.abs() @ k.abs().t() * sm).amax(-1, keepdim=True)
            o, a = w @ v, w @ v.abs()
            # fp32 scores: 2^-18 of their magnitudes' sum, above and below the fraction; fp32 sums
            tol = U[torch.bfloat16] * o.abs() + (2.0 ** -16 + 2.0 ** -17 * worst + 2.0 ** -18) * a
            e = (got[t, h * G * D:(h + 1) * G * D].view(G, D) - o).abs()
            assert (e <= tol * (1 + 2.0 ** -10)).all(), (t, h, float((e / tol).max()))


# ---------------------------------------------------------------------------- as they are used
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
def test_decode_steps_together(dev, kind):
    """Prompt, then decode steps: append with bounds, select, attend.  The selection is the
    one the stored keys' bounds give, and with a budget of all pages the result is the dense
    kernel's."""
    Hq, KH, D, B = 8, 2, 64, 3
    g = torch.Generator().manual_seed(3)
    ctx = [150, 33, 90]
    steps = 5
    n_pages = sum(-(-(n + steps) // 16) for n in ctx)
    cache, ks = make_pool(kind, n_pages, 1, KH, D, dev)
    kb = ops.key_bounds_for(cache)
    width = max(-(-(n + steps) // 16) for n in ctx)
    bt = tables([n + steps for n in ctx], width, n_pages, dev)
    cs = ops.rope_cos_sin(256, D, 1e4, dev)
    W = (Hq + 2 * KH) * D

    def append(seqs, pos):
        pos, seqs = torch.tensor(pos), torch.tensor(seqs)
        slots = bt.cpu()[seqs, pos // 16] * 16 + pos % 16
        qkv = torch.randn(len(pos), W, generator=g).bfloat16().to(dev)
        return ops.qk_norm_rope_kv_write(qkv, None, None, 0.0, pos.int().to(dev), cs, cache, slots.int().to(dev), ks,
                                         0, Hq, KH, D, key_bounds=kb)

    append([b for b in range(B) for _ in range(ctx[b])], [p for b in range(B) for p in range(ctx[b])])
    for s in range(steps):
        lens = [n + s + 1 for n in ctx]
        q = append(list(range(B)), [n - 1 for n in lens])
        stored = values(cache)[:, 0, 0].amin(2), values(cache)[:, 0, 0].amax(2)
        for b, n in enumerate(lens):
            for p in range(n // 16):                            # full pages
                for i in (0, 1):
                    want = stored[i][int(bt[b, p])]
                    got = kb[int(bt[b, p]), 0, :, i].cpu().float().double()
                    assert ((got - want).abs() <= (U[torch.bfloat16] * want.abs() if kind == "q4" else 0)).all()
        pages = ops.select_pages(q, kb, 0, bt, i32(lens, dev), Hq, 4, sinks=1, recent=1)
        want = select_ref(q, kb, 0, bt, rows_of(B, lens, None), Hq, 4, 1, 1)
        assert all(pages[t, h].tolist() == w for (t, h), w in want.items())
        o = ops.paged_attention_selected(q, cache, 0, bt, i32(lens, dev), pages, ks, 0.125, Hq)
        for (t, h), (r, tol) in attend_ref(q, values(cache, ks), 0, bt, rows_of(B, lens, None), pages.cpu(), 0.125,
                                           Hq, kind).items():
            e = (o.cpu().double()[t].view(KH, -1, D)[h] - r).abs()
            assert (e <= tol * (1 + 2.0 ** -10)).all()
        every = ops.select_pages(q, kb, 0, bt, i32(lens, dev), Hq, width)
        full = ops.paged_attention_selected(q, cache, 0, bt, i32(lens, dev), every, ks, 0.125, Hq)
        dense = ops.paged_attention_decode(q, cache, 0, bt, i32(lens, dev), ks, 0.125, Hq)
        for (t, h), (r, tol) in attend_ref(q, values(cache, ks), 0, bt, rows_of(B, lens, None), every.cpu(), 0.125,
                                           Hq, kind).items():
            e = (full - dense).cpu().double()[t].view(KH, -1, D)[h].abs()
            assert (e <= 2 * tol * (1 + 2.0 ** -10)).all()


def gpu_step(dev="cuda", seed=0, B=5, budget=6):
    """A decode step's inputs on the GPU and the three calls over them."""
    Hq, KH, D = 8, 2, 128
    g = torch.Generator().manual_seed(seed)
    ctx = [400 + 33 * i for i in range(B)]
    n_pages = sum(-(-n // 16) for n in ctx)
    cache, _ = make_pool("bf16", n_pages, 1, KH, D, dev, seed)
    kb = ops.key_bounds_for(cache)
    k = cache[:, 0, 0].float()
    kb[:, 0, :, 0], kb[:, 0, :, 1] = k.amin(2).bfloat16(), k.amax(2).bfloat16()
    bt = tables(ctx, max(-(-n // 16) for n in ctx), n_pages, dev, seed)
    pos = torch.tensor(ctx) - 1
    st = {"qkv": torch.randn(B, (Hq + 2 * KH) * D, generator=g).bfloat16().to(dev), "pos": pos.int().to(dev),
          "slots": (bt.cpu()[torch.arange(B), pos // 16] * 16 + pos % 16).int().to(dev), "ctx": i32(ctx, dev),
          "bt": bt, "cache": cache, "kb": kb, "cs": ops.rope_cos_sin(1024, D, 1e4, dev)}

    def call():
        q = ops.qk_norm_rope_kv_write(st["qkv"], None, None, 0.0, st["pos"], st["cs"], cache, st["slots"], None, 0,
                                      Hq, KH, D, key_bounds=kb)
        pages = ops.select_pages(q, kb, 0, bt, st["ctx"], Hq, budget)
        return q, pages, ops.paged_attention_selected(q, cache, 0, bt, st["ctx"], pages, None, 0.088, Hq)

    return st, call


@pytest.mark.gpu
def test_captured_and_replayed(cuda_errors_clean):
    """Two captured graphs replayed in turn, on new inputs, give what the eager calls give."""
    both = [gpu_step(seed=1), gpu_step(seed=2, B=3)]
    graphs = []
    for st, call in both:
        call()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = call()
        graphs.append((gr, got))
    for turn in range(3):
        for (st, call), (gr, got) in zip(both, graphs):
            st["qkv"].copy_(torch.randn(st["qkv"].shape, generator=torch.Generator().manual_seed(turn)).bfloat16())
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (st, call), (_, got) in zip(both, graphs):
            kept = [x.clone() for x in got]
            for a, b in zip(kept, call()):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [5000, ops.SELECT_MAX_PAGES])
def test_captured_with_wide_tables(width, cuda_errors_clean):
    """A table for very long contexts (more shared memory than a kernel has by default),
    captured, replayed with other lengths, after a call with a narrow table."""
    D, n = 64, 300
    kb, _ = make_pool("bf16", n, 1, 1, D, "cuda")
    kb = torch.stack([kb[:, :, 0, :, 0] - 1, kb[:, :, 0, :, 0] + 1], 3)
    bt = torch.zeros(2, width, dtype=torch.int32, device="cuda")
    bt[:, :n] = torch.arange(n, dtype=torch.int32, device="cuda")
    q = torch.randn(2, D, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    ctx = i32([16 * n, 90], "cuda")
    out = torch.empty(2, 1, 20, dtype=torch.int32, device="cuda")
    call = lambda t: ops.select_pages(q, kb, 0, t, ctx, 1, 20, out=out)  # noqa: E731
    call(bt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(bt)
    for lens in ([16 * n, 90], [1000, 16 * n - 7], [0, 400]):
        ctx.copy_(i32(lens, "cuda"))
        want = call(bt[:, :n].contiguous()).clone()
        out.fill_(-5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_other_streams_and_repeats(cuda_errors_clean):
    """Two streams at once, and the same call again: the same bits."""
    (s1, c1), (s2, c2) = gpu_step(seed=5), gpu_step(seed=6)
    want1, want2 = [x.clone() for x in c1()], [x.clone() for x in c2()]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got1, got2 = [], []
    for _ in range(20):
        with torch.cuda.stream(a):
            got1.append(c1())
        with torch.cuda.stream(b):
            got2.append(c2())
    torch.cuda.synchronize()
    for got, want in ((got1, want1), (got2, want2)):
        for g in got:
            assert all(torch.equal(x, y) for x, y in zip(g, want))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_errors_clean):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements of the pool."""
    KH, D, n = 8, 128, 70000
    cache = torch.empty(n, 1, 2, KH, 16, D, dtype=torch.bfloat16, device="cuda")
    assert cache.numel() > 2 ** 31
    kb = torch.empty(n, 1, KH, 2, D, dtype=torch.bfloat16, device="cuda")
    small, _ = make_pool("bf16", 12, 1, KH, D, "cuda")
    far = torch.arange(n - 12, n, dtype=torch.int32, device="cuda")
    cache[n - 12:] = small
    near = torch.arange(12, dtype=torch.int32, device="cuda")
    qkv = torch.randn(1, 3 * KH * D, device="cuda").bfloat16()
    res = []
    for c, b, bt in ((cache, kb, far), (small, torch.zeros(12, 1, KH, 2, D, device="cuda").bfloat16(), near)):
        b[bt.long(), 0, :, 0] = small[:, 0, 0].amin(2)
        b[bt.long(), 0, :, 1] = small[:, 0, 0].amax(2)
        slot = bt[11:] * 16 + 3
        q = ops.qk_norm_rope_kv_write(qkv, None, None, 0.0, None, None, c, slot, None, 0, KH, KH, D, key_bounds=b)
        p = ops.select_pages(q, b, 0, bt[None], i32([180], "cuda"), KH, 5)
        o = ops.paged_attention_selected(q, c, 0, bt[None], i32([180], "cuda"), p, None, 0.1, KH)
        res.append((q, p, o, c[bt.long()].clone(), b[bt.long()].clone()))
    assert all(torch.equal(x, y) for x, y in zip(*res))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", ["bf16", "fp8", "q4"])
def test_nothing_to_do(dev, kind):
    """No tokens, block tables without columns, lists without entries."""
    KH, D = 2, 64
    cache, ks = make_pool(kind, 3, 1, KH, D, dev)
    kb, before = ops.key_bounds_for(cache), cache.clone()
    none, two = i32([], dev), i32([0, 0], dev)
    q = ops.qk_norm_rope_kv_write(torch.zeros(0, 8 * D).bfloat16().to(dev), None, None, 0.0, None, None, cache, none, ks,
                                  0, 4, KH, D, key_bounds=kb)
    assert q.shape == (0, 4 * D) and torch.equal(cache.view(torch.uint8), before.view(torch.uint8))
    empty = torch.zeros(0, 2, dtype=torch.int32, device=dev)
    p = ops.select_pages(q, kb, 0, empty, none, 4, 3)
    assert p.shape == (0, KH, 3)
    assert ops.paged_attention_selected(q, cache, 0, empty, none, p, ks, 1.0, 4).shape == (0, 4 * D)
    q = torch.ones(2, 4 * D).bfloat16().to(dev)
    flat = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    for ctx in (two, i32([40, 7], dev)):
        p = ops.select_pages(q, kb, 0, flat, ctx, 4, 3)
        assert (p == -1).all() and p.shape == (2, KH, 3)
        o = ops.paged_attention_selected(q, cache, 0, flat, ctx, p, ks, 1.0, 4)
        assert o.shape == (2, 4 * D) and (o == 0).all()
        o = ops.paged_attention_selected(q, cache, 0, torch.zeros(2, 3, dtype=torch.int32, device=dev), ctx,
                                         p[:, :, :0].contiguous(), ks, 1.0, 4)
        assert (o == 0).all()


# ---------------------------------------------------------------------------- refusals
def test_refusals_cpu():
    q = torch.zeros(1, 128).bfloat16()
    kb = torch.zeros(4, 1, 1, 2, 64).bfloat16()
    bt, ctx = i32([[0, 1, 2, 3]], "cpu"), i32([64], "cpu")
    for bad in (dict(budget=1), dict(budget=2, sinks=-1), dict(budget=2, recent=0), dict(budget=3, sinks=2, recent=2)):
        with pytest.raises(ValueError):
            ops.select_pages(q, kb, 0, bt, ctx, 2, **bad)
    with pytest.raises(ValueError):
        ops.select_pages(q, kb, 0, torch.zeros(1, ops.SELECT_MAX_PAGES + 1, dtype=torch.int32), ctx, 2, 3)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_kv_write(q, q[0, :64], None, 0.0, None, None, torch.zeros(1, 1, 2, 1, 16, 32).bfloat16(),
                                  ctx, None, 0, 2, 1, 32)


@pytest.mark.parametrize("dev", DEVICES)
def test_budgets_near_the_32_bit_limit_are_refused(dev):
    """The kernel's indexes run a little past the budget and the sinks: they must not wrap."""
    q = torch.zeros(1, 128).bfloat16().to(dev)
    kb = torch.zeros(4, 1, 1, 2, 64).bfloat16().to(dev)
    bt, ctx = i32([[0, 1, 2, 3]], dev), i32([64], dev)
    for bad in (dict(budget=2 ** 30 + 1), dict(budget=2 ** 31 - 1), dict(budget=2 ** 31 - 1, sinks=2 ** 31 - 100),
                dict(budget=2 ** 31), dict(budget=2 ** 40, sinks=2 ** 40 - 9)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.select_pages(q, kb, 0, bt, ctx, 2, **bad)
    got = ops.select_pages(q, kb, 0, bt, ctx, 2, 100000, sinks=99999)
    assert got[0, 0, :4].tolist() == [0, 1, 2, 3] and (got[0, 0, 4:] == -1).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_lists_near_the_32_bit_limit_are_refused(dev):
    q, cache = torch.zeros(1, 64).bfloat16().to(dev), torch.zeros(2, 1, 2, 1, 16, 64).bfloat16().to(dev)
    bt, ctx = i32([[0, 1]], dev), i32([20], dev)
    for n in (2 ** 30 + 1, 2 ** 31 - 1, 2 ** 31 + 5):
        pages = torch.empty(1, 1, n, dtype=torch.int32, device=dev)          # not touched
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_attention_selected(q, cache, 0, bt, ctx, pages, None, 1.0, 1)
        del pages


@pytest.mark.gpu
def test_block_table_rows_far_apart_are_refused(cuda_errors_clean):
    """The distance of two rows of the table has to fit the kernels' 32 bits."""
    q, kb = torch.zeros(2, 64, device="cuda").bfloat16(), torch.zeros(4, 1, 1, 2, 64, device="cuda").bfloat16()
    cache, ctx = torch.zeros(4, 1, 2, 1, 16, 64, device="cuda").bfloat16(), i32([50, 50], "cuda")
    store = torch.empty(2 ** 31 + 8, dtype=torch.int32, device="cuda")
    far = store.as_strided((2, 4), (2 ** 31, 1))
    far.copy_(i32([[0, 1, 2, 3], [3, 2, 1, 0]], "cuda"))
    pages = i32([[[0, 1]], [[0, 3]]], "cuda")
    with pytest.raises(RuntimeError):
        ops.select_pages(q, kb, 0, far, ctx, 1, 2)
    with pytest.raises(RuntimeError):
        ops.paged_attention_selected(q, cache, 0, far, ctx, pages, None, 1.0, 1)
    one = far[1:]                                             # a single row has no distance
    assert ops.select_pages(q[:1], kb, 0, one, ctx[:1], 1, 2).tolist() == [[[0, 3]]]
    assert (ops.paged_attention_selected(q[:1], cache, 0, one, ctx[:1], pages[:1], None, 1.0, 1) == 0).all()


@pytest.mark.gpu
def test_refusals(cuda_errors_clean):
    dev = "cuda"
    q = torch.zeros(2, 4 * 64, device=dev).bfloat16()
    cache = torch.zeros(4, 2, 2, 2, 16, 64, device=dev).bfloat16()
    kb = ops.key_bounds_for(cache)
    bt, ctx = i32([[0, 1], [2, 3]], dev), i32([20, 20], dev)
    pages = torch.zeros(2, 2, 3, dtype=torch.int32, device=dev)
    sel = dict(q=q, key_bounds=kb, layer=0, block_tables=bt, context_lens=ctx, num_q_heads=4, budget=3)
    att = dict(q=q, cache=cache, layer=0, block_tables=bt, context_lens=ctx, pages=pages, kv_scale=None, sm_scale=1.0,
               num_q_heads=4)
    qkv = torch.zeros(2, 8 * 64, device=dev).bfloat16()
    app = dict(qkv=qkv, wq=None, wk=None, eps=0.0, positions=ctx, cos_sin=torch.zeros(32, 64, device=dev), cache=cache,
               slot_mapping=ctx, kv_scale=None, layer=0, num_q_heads=4, num_kv_heads=2, head_dim=64)
    ops.select_pages(**sel), ops.paged_attention_selected(**att), ops.qk_norm_rope_kv_write(**app)   # as they are: fine
    off = torch.zeros(2 * 4 * 64 + 8, device=dev).bfloat16()
    wrong = [
        (ops.select_pages, sel, dict(budget=1), dict(sinks=-1), dict(recent=0), dict(layer=2), dict(layer=-1),
         dict(num_q_heads=3), dict(num_q_heads=18, q=torch.zeros(2, 18 * 64, device=dev).bfloat16()),
         dict(num_q_heads=8), dict(q=q.float()), dict(q=q.cpu().to(dev).t()), dict(q=off[4:516].view(2, 256)),
         dict(block_tables=bt.long()), dict(block_tables=bt[:1]), dict(context_lens=ctx[:1]),
         dict(context_lens=ctx.long()), dict(cu_q=torch.zeros(3, device=dev)), dict(cu_q=i32([0, 1, 2, 2], dev)),
         dict(key_bounds=kb.float()), dict(key_bounds=kb[:, :, :, :1]), dict(key_bounds=kb.cpu()),
         dict(block_tables=torch.zeros(2, ops.SELECT_MAX_PAGES + 1, dtype=torch.int32, device=dev)),
         dict(out=pages.long()), dict(out=pages[:, :, :2]), dict(out=pages[:1])),
        (ops.paged_attention_selected, att, dict(layer=2), dict(num_q_heads=3), dict(num_q_heads=8),
         dict(q=q.half()), dict(cache=cache.float()), dict(cache=cache[:, :, :, :, :8]), dict(pages=pages.long()),
         dict(pages=pages[:, :1]), dict(pages=pages.cpu()), dict(cache=cache.to(torch.float8_e4m3fn)),
         dict(out=torch.zeros(2, 255, device=dev).bfloat16()), dict(out=q.float()), dict(context_lens=ctx.cpu())),
        (ops.qk_norm_rope_kv_write, app, dict(layer=2), dict(num_q_heads=5), dict(head_dim=32),
         dict(wq=torch.ones(64, device=dev).bfloat16()), dict(slot_mapping=ctx.long()), dict(slot_mapping=ctx[:1]),
         dict(positions=None), dict(positions=ctx.long()), dict(cos_sin=torch.zeros(32, 66, device=dev)),
         dict(cos_sin=torch.zeros(0, 64, device=dev)), dict(cache=cache.float()), dict(key_bounds=kb[:3]),
         dict(key_bounds=kb.to(torch.float8_e4m3fn)), dict(cache=cache.to(torch.float8_e4m3fn)),
         dict(out=qkv[:, 64:320]), dict(out=torch.zeros(1, 256, device=dev).bfloat16()),
         dict(wq=torch.ones(64, device=dev), wk=torch.ones(64, device=dev))),
    ]
    for fn, base, *changes in wrong:
        for ch in changes:
            with pytest.raises(RuntimeError):
                fn(**{**base, **ch})


@pytest.mark.gpu
def test_indexes_out_of_range_are_reported():
    """Pages and positions outside their tables are not read or written: the error word says
    so and the rest of the call is done."""
    assert ops.read_and_clear_errors() == 0
    dev, KH, D = "cuda", 1, 64
    cache, _ = make_pool("bf16", 4, 1, KH, D, dev)
    kb = ops.key_bounds_for(cache)
    q = torch.ones(1, D, device=dev).bfloat16()
    good = ops.paged_attention_selected(q, cache, 0, i32([[0, 1, 2]], dev), i32([48], dev), i32([[[0, 2]]], dev), None, 0.1, 1)
    assert ops.read_and_clear_errors() == 0
    got = ops.paged_attention_selected(q, cache, 0, i32([[0, 4, 2]], dev), i32([48], dev), i32([[[0, 1, 2]]], dev), None, 0.1, 1)
    assert ops.read_and_clear_errors() == 8
    assert (got.float() - good.float()).abs().max() <= 2.0 ** -7 * good.float().abs().max()
    kb[:] = 1.0
    p = ops.select_pages(q, kb, 0, i32([[0, 9, -1, 1, 2, 3]], dev), i32([96], dev), 1, 4, sinks=1, recent=1)
    assert ops.read_and_clear_errors() == 8
    assert p[0, 0].tolist() == [0, 3, 4, 5]                  # unreadable pages come last
    before = cache.clone()
    qkv = torch.ones(2, 3 * D, device=dev).bfloat16()
    cs = ops.rope_cos_sin(8, D, 1e4, dev)
    got = ops.qk_norm_rope_kv_write(qkv, None, None, 0.0, i32([7, 7], dev), cs, cache, i32([64, 2 ** 31 - 1], dev),
                                    None, 0, 1, KH, D, key_bounds=kb)
    assert ops.read_and_clear_errors() == 8
    assert torch.equal(cache, before) and (kb == 1.0).all()
    far = ops.qk_norm_rope_kv_write(qkv, None, None, 0.0, i32([9, -4], dev), cs, cache, i32([-1, -1], dev), None, 0, 1,
                                    KH, D)
    assert ops.read_and_clear_errors() == 8
    assert torch.equal(far[0], got[0])                       # the table's nearest row
