"""Packed prompts and shared prefixes against plain forms in 64 bits.

Tolerances follow from the roundings.  With u = 2^-8 (bf16, 8 bits of
significand) or 2^-11 (fp16, 11 bits) the half-ulp of the output type, an
attention output o = sum p_j v_j carries one rounding of the result (at most
u |o|) and one of each probability (at most u sum p |v|, and far less where
they do not all go one way, which leaves room for the float32 sums).  Where
cached keys are rounded to 11 bits, a score moves by at most
2^-11 sum |q k| scale, and each probability by twice that, relatively.
"""

import math

import pytest
import torch

from oracle import kv_sym

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), what
    err = (got - want).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max()):.3g} of the bound"


# ---- page plan ----------------------------------------------------------------


def plan_reference(lens, ctx, free, page, T, table):
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    cu, pos, slots, rows, taken = [0], [], [], [], 0
    for b, n in enumerate(lens):
        have, need = -(-ctx[b] // page), -(-(ctx[b] + n) // page)
        for e in range(have, need):
            if e < width:
                table[b][e] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(n):
            p = ctx[b] + i
            pg = table[b][p // page] if p // page < width else -1
            pos.append(p)
            rows.append(b)
            slots.append(pg * page + p % page if pg >= 0 else -1)
        cu.append(cu[-1] + n)
    pad = max(0, T - len(pos))
    return (table, cu, (pos + [0] * pad)[:T], (slots + [-1] * pad)[:T], (rows + [-1] * pad)[:T],
            [a + b for a, b in zip(lens, ctx)], [cu[-1], taken])


@pytest.mark.parametrize("B,most,page,room,short", [
    (1, 1, 16, 0, 0), (3, 40, 16, 5, 0), (5, 200, 64, 0, 0), (40, 33, 48, 3, 0), (17, 90, 64, 0, 7), (17, 90, 64, -50, 0),
    (2048, 9, 16, 0, 0), (2049, 9, 16, 2, 0), (5000, 6, 32, 0, 0), (0, 0, 16, 7, 0),
])
def test_plan_pages(dev, B, most, page, room, short):
    from b200flash.paged_prompt import plan_pages

    g = torch.Generator().manual_seed(B + most)
    lens = torch.randint(0, most + 1, (B,), generator=g).tolist()
    ctx = (torch.randint(0, 3 * page, (B,), generator=g) * (torch.rand(B, generator=g) < 0.6)).tolist()
    if B > 2:
        lens[0] = lens[-1] = 0  # requests without tokens at both ends
    need = [-(-(a + b) // page) for a, b in zip(lens, ctx)]
    held = [-(-b // page) for b in ctx]
    width = max(need + [1])
    ids = torch.randperm(sum(need) + 5, generator=g).tolist()
    table = [[-7] * width for _ in range(B)]
    at = 0
    for b in range(B):
        table[b][: held[b]] = ids[at: at + held[b]]
        at += held[b]
    free = ids[at: len(ids) - 5 - short]
    T = max(0, sum(lens) + room)
    want = plan_reference(lens, ctx, free, page, T, table)
    i32 = dict(dtype=torch.int32, device=dev)
    tab = torch.tensor(table, **i32).reshape(B, width)
    p = plan_pages(torch.tensor(lens, **i32), torch.tensor(free, **i32), page, T, tab,
                   context_lens=torch.tensor(ctx, **i32))
    assert tab.tolist() == want[0]
    for name, w in zip(("cu_seqlens", "positions", "slots", "rows", "seq_lens", "counts"), want[1:]):
        assert getattr(p, name).tolist() == w, name


def test_plan_pages_narrow_table_and_no_context(dev):
    from b200flash.paged_prompt import plan_pages

    i32 = dict(dtype=torch.int32, device=dev)
    tab = torch.full((2, 2), -7, **i32)
    p = plan_pages(torch.tensor([40, 16], **i32), torch.tensor([9, 8, 7, 6, 5], **i32), 16, 56, tab)
    assert tab.tolist() == [[9, 8], [6, -7]]  # the third page of request 0 does not fit its row
    assert p.counts.tolist() == [56, 4]
    assert p.slots.tolist() == [9 * 16 + i for i in range(16)] + [8 * 16 + i for i in range(16)] + [-1] * 8 + [
        6 * 16 + i for i in range(16)]


# ---- per-head norm + rotary -----------------------------------------------------


def norm_rope_reference(x, w, pos, inv, eps):
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    r = inv.shape[0]
    a = (pos.double()[:, None] * inv.double())[:, None]
    lo, hi = y[..., :r].clone(), y[..., r: 2 * r].clone()
    y[..., :r] = lo * a.cos() - hi * a.sin()
    y[..., r: 2 * r] = hi * a.cos() + lo * a.sin()
    return y


@pytest.mark.parametrize("T,Hq,Hkv,D,dt,rot", [
    (1, 32, 4, 128, "bf16", None), (3, 5, 1, 64, "f16", None), (37, 8, 8, 128, "f16", None), (130, 6, 2, 256, "bf16", None),
    (64, 32, 4, 128, "bf16", 32), (9, 3, 3, 64, "bf16", 8), (5, 4, 2, 128, "f16", 0),
    (601, 32, 4, 128, "bf16", None), (700, 41, 3, 64, "f16", None), (2049, 9, 1, 256, "bf16", None),
    (1203, 17, 2, 128, "f16", 40),
])
def test_qk_norm_rope(dev, T, Hq, Hkv, D, dt, rot):
    from b200flash.paged_prompt import qk_norm_rope

    g = torch.Generator(device=dev).manual_seed(T)
    wide = torch.randn(T, (Hq + 2 * Hkv) * D + 24, device=dev, generator=g).to(DT[dt])
    qkv = wide[:, 8: 8 + (Hq + 2 * Hkv) * D] if T % 2 else wide[:, : (Hq + 2 * Hkv) * D]  # a strided view
    qn, kn = ((1 + 0.2 * torch.randn(D, device=dev, generator=g)).to(DT[dt]) for _ in range(2))
    pos = torch.randint(0, 1 << 20, (T,), device=dev, generator=g).to(torch.int32)
    inv = None if rot is None else torch.tensor([0.9 ** i for i in range(rot)], dtype=torch.float64, device=dev)
    q, k, v = qk_norm_rope(qkv, Hq, Hkv, pos, qn, kn, eps=1e-5, theta=5e5, inv_freq=inv)
    if inv is None:
        inv = torch.tensor([5e5 ** (-2 * i / D) for i in range(D // 2)], dtype=torch.float64, device=dev)
    x = qkv.reshape(T, Hq + 2 * Hkv, D)
    for got, part, w in ((q, x[:, :Hq], qn), (k, x[:, Hq: Hq + Hkv], kn)):
        want = norm_rope_reference(part, w, pos, inv, 1e-5)
        # one rounding of the result, and float32 arithmetic on the pair it is formed from
        big = norm_rope_reference(part, w, pos * 0, inv[:0], 1e-5).abs().amax(-1, keepdim=True)
        within(got, want, 1.01 * HALF_ULP[DT[dt]] * want.abs() + 2.0 ** -20 * big + 2.0 ** -25)
    assert torch.equal(v, x[:, Hq + Hkv:])


@pytest.mark.parametrize("T", [70, 1300])
@pytest.mark.parametrize("D,dt,bits,page", [(128, "bf16", 8, 64), (64, "bf16", 4, 16), (128, "f16", 2, 48),
                                            (256, "bf16", 8, 16), (128, "f16", 4, 64)])
def test_qk_norm_rope_append(dev, D, dt, bits, page, T):
    """The appended bytes are the quantizer's on the returned k and on v; skipped slots stay untouched."""
    from b200flash.paged_prompt import qk_norm_rope
    from b200flash.quantized_kv_cache import quantize_tensor

    Hq, Hkv = 6, 3
    g = torch.Generator(device=dev).manual_seed(bits)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, device=dev, generator=g).to(DT[dt])
    qkv[4] = 0  # a row of zeros: scale 1
    w = torch.ones(D, device=dev, dtype=DT[dt])
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, device=dev, generator=g)[:T]
    slots[7] = slots[33] = -1
    lead = (pages, Hkv, page)
    cache = [torch.full((*lead, n), 77, dtype=d, device=dev)
             for n, d in ((D * bits // 8, torch.uint8), (D // 64, torch.float32)) * 2]
    q, k, v = qk_norm_rope(qkv, Hq, Hkv, pos, w, w, cache=tuple(cache), slots=slots, bits=bits)
    q2, k2, _ = qk_norm_rope(qkv, Hq, Hkv, pos, w, w)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    for x, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        want_c, want_s = torch.full_like(codes, 77), torch.full_like(scales, 77)
        c, s, _ = quantize_tensor(x.contiguous(), bits, 64)
        for t, slot in enumerate(slots.tolist()):
            if slot >= 0:
                want_c[slot // page, :, slot % page] = c[t]
                want_s[slot // page, :, slot % page] = s[t]
        assert torch.equal(codes, want_c) and torch.equal(scales, want_s)


# ---- prompt attention -------------------------------------------------------------


def attend_reference(q, k, v, causal, scale):
    """(o, sum p |v|, lse) of one sequence in 64 bits."""
    G = q.shape[1] // k.shape[1]
    k, v = (x.double().repeat_interleave(G, 1) for x in (k, v))
    s = torch.einsum("nhd,mhd->hnm", q.double(), k) * scale
    if causal:
        n = s.shape[1]
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), -math.inf)
    p = torch.softmax(s, -1)
    return (torch.einsum("hnm,mhd->nhd", p, v), torch.einsum("hnm,mhd->nhd", p, v.abs()),
            torch.logsumexp(s, -1).transpose(0, 1))


def packed(dev, lens, Hq, Hkv, D, dt, seed=0, pad=0, scale=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(lens) + pad
    q, k, v = (torch.randn(T, h, D, device=dev, generator=g) for h in (Hq, Hkv, Hkv))
    cu = torch.tensor([0] + list(lens), device=dev).cumsum(0).to(torch.int32)
    return (q * scale).to(DT[dt]), k.to(DT[dt]), v.to(DT[dt]), cu


def check_prompt(out, lse, q, k, v, lens, causal, scale=None):
    D = q.shape[2]
    a = 0
    for n in lens:
        s = slice(a, a + n)
        o, o_abs, z = attend_reference(q[s], k[s], v[s], causal, D ** -0.5 if scale is None else scale)
        u = HALF_ULP[q.dtype]
        within(out[s], o, u * (o.abs() + o_abs) + 1e-6, f"rows {a}:{a + n}")
        if lse is not None:
            within(lse[s], z, 1e-5 * z.abs() + 1e-4, "lse")
        a += n
    assert bool((out[a:] == 0).all())
    if lse is not None:
        assert bool((lse[a:] == -math.inf).all())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,Hq,Hkv,D,dt", [
    ([1], 8, 1, 128, "bf16"), ([0, 1, 0, 2, 0], 4, 4, 64, "f16"), ([127, 128, 129], 8, 2, 128, "bf16"),
    ([300, 5, 0, 64], 32, 4, 128, "bf16"), ([513], 3, 1, 128, "f16"), ([100, 31], 6, 2, 80, "bf16"),
    ([260], 5, 5, 8, "bf16"), ([90, 170], 14, 2, 96, "f16"), ([17] * 40, 16, 1, 64, "bf16"), ([257, 40], 24, 1, 120, "f16"),
    ([1100], 2, 2, 128, "bf16"), ([33, 150], 96, 1, 64, "bf16"),
])
def test_prompt_attention(dev, lens, Hq, Hkv, D, dt, causal):
    from b200flash.paged_prompt import prompt_attention

    q, k, v, cu = packed(dev, lens, Hq, Hkv, D, dt, seed=len(lens))
    out, lse = prompt_attention(q, k, v, cu, causal=causal, return_lse=True)
    check_prompt(out, lse, q, k, v, lens, causal)


def test_prompt_attention_padding_views_and_scale(dev):
    """Views of one packed projection, rows past the last sequence, sharp scores, another stream."""
    from b200flash.paged_prompt import prompt_attention

    lens, Hq, Hkv, D = [150, 3, 200], 8, 2, 128
    q, k, v, cu = packed(dev, lens, Hq, Hkv, D, "bf16", seed=5, pad=70, scale=12.0)
    qkv = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    qv, kv, vv = (x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        out, lse = prompt_attention(qv, kv, vv, cu, softmax_scale=0.3, return_lse=True)
    torch.cuda.current_stream(dev).wait_stream(side)
    check_prompt(out, lse, q, k, v, lens, True, 0.3)
    # a layout whose strides do not fit is copied
    odd = torch.empty(q.shape[0], Hq, D + 1, dtype=q.dtype, device=dev)[..., :D]
    odd.copy_(q)
    assert torch.equal(prompt_attention(odd, k, v, cu, softmax_scale=0.3), out)
    assert torch.equal(prompt_attention(q, k, v, cu, softmax_scale=0.3), out)


def test_prompt_attention_growing_scores(dev):
    """Scores that rise along the keys by far more than the exponent range of the running sum allows at once."""
    from b200flash.paged_prompt import prompt_attention

    n, D = 700, 64
    k = torch.zeros(n, 1, D, device=dev)
    k[:, 0, 0] = torch.arange(n, device=dev) / 4
    g = torch.Generator(device=dev).manual_seed(1)
    v = torch.randn(n, 1, D, device=dev, generator=g)
    q = torch.zeros(n, 2, D, device=dev)
    q[:, 0, 0], q[:, 1, 0] = 8.0, -8.0
    q, k, v = (x.to(torch.bfloat16) for x in (q, k, v))
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    out, lse = prompt_attention(q, k, v, cu, softmax_scale=1.0, return_lse=True)
    check_prompt(out, lse, q, k, v, [n], True, 1.0)


def test_prompt_attention_other_sequences_do_not_leak(dev):
    """NaN and infinities of one sequence stay inside it."""
    from b200flash.paged_prompt import prompt_attention

    lens = [70, 90, 200, 45]
    q, k, v, cu = packed(dev, lens, 8, 2, 128, "bf16", seed=3, pad=30)
    clean = prompt_attention(q, k, v, cu)
    for x, bad in ((q, math.nan), (k, math.inf), (v, math.nan)):
        x[160:360] = bad
        x[405:] = bad
    dirty = prompt_attention(q, k, v, cu)
    for a, b in ((0, 160), (360, 405)):
        assert torch.equal(dirty[a:b], clean[a:b])
    assert bool(dirty[160:360].isnan().all()) and bool((dirty[405:] == 0).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_prompt_attention_later_tokens_do_not_leak(dev, bad):
    """A value row that is not finite reaches the rows that see it, and no earlier one."""
    from b200flash.paged_prompt import prompt_attention

    lens = [20, 330]
    q, k, v, cu = packed(dev, lens, 4, 4, 128, "bf16", seed=4)
    clean = prompt_attention(q, k, v, cu)
    at = 20 + 201
    v[at, :, 5] = bad
    k[at + 60] = bad
    dirty = prompt_attention(q, k, v, cu)
    assert torch.equal(dirty[:at], clean[:at])
    assert not bool(dirty[at: at + 60, :, 5].isfinite().any())
    keep = [d for d in range(128) if d != 5]
    assert torch.equal(dirty[at: at + 60, :, keep], clean[at: at + 60, :, keep])
    assert not bool(dirty[at + 60:].isfinite().any())


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 9, 40])
def test_prompt_attention_few_keys(dev, n, causal, dt):
    """Rows of one key are that key's values; short sequences lose no more than two roundings do."""
    from b200flash.paged_prompt import prompt_attention

    lens = [n] * 60
    q, k, v, cu = packed(dev, lens, 16, 4, 128, dt, seed=n)
    out = prompt_attention(q, k, v, cu, causal=causal)
    got, want = [], []
    for b in range(60):
        s = slice(b * n, (b + 1) * n)
        if causal or n == 1:
            assert torch.equal(out[b * n], v[b * n].repeat_interleave(4, 0))
        want.append(attend_reference(q[s], k[s], v[s], causal, 128 ** -0.5)[0])
        got.append(out[s].double())
    got, want = torch.cat(got), torch.cat(want)
    # the output's rounding, and as much again (independent of it) from the rounding of P
    one = (want.to(DT[dt]).double() - want).norm()
    assert float((got - want).norm()) <= 1.45 * float(one)


@pytest.mark.parametrize("scale", [-0.07, 0.0, 1e-12])
def test_prompt_attention_scales(dev, scale):
    from b200flash.paged_prompt import prompt_attention

    lens = [140, 1, 300]
    q, k, v, cu = packed(dev, lens, 8, 2, 128, "bf16", seed=8, pad=3)
    out, lse = prompt_attention(q, k, v, cu, softmax_scale=scale, return_lse=True)
    check_prompt(out, lse, q, k, v, lens, True, scale)


@pytest.mark.parametrize("seed", [0, 1])
def test_prompt_attention_many_sequences(dev, seed):
    """Several hundred sequences, runs of empty ones among them (more than the planner looks at in one go)."""
    from b200flash.paged_prompt import prompt_attention

    g = torch.Generator().manual_seed(seed)
    lens = (torch.randint(0, 30, (400,), generator=g) * (torch.rand(400, generator=g) < 0.5)).tolist()
    lens[100:180] = [0] * 80
    lens[250], lens[399] = 500, 0
    q, k, v, cu = packed(dev, lens, 8, 4, 64, "bf16", seed=seed, pad=300)
    out, lse = prompt_attention(q, k, v, cu, return_lse=True)
    check_prompt(out, lse, q, k, v, lens, True)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_prompt_attention_one_bad_key(dev, dt):
    """NaN in any one key, wherever it lies in a block, makes the rows that see it NaN; an infinite score is softmax's."""
    from b200flash.paged_prompt import prompt_attention

    n = 256
    q, k, v, cu = packed(dev, [n] * 128, 2, 1, 64, dt, seed=2)
    at = torch.arange(128, device=dev) * (n + 1)  # key i of sequence i
    bad = k.clone()
    bad[at] = math.nan
    assert bool(prompt_attention(q, bad, v, cu, causal=False).isnan().all())
    k[at] = 0
    k[at, 0, 0] = math.inf
    out = prompt_attention(q, k, v, cu, causal=False).view(128, n, 2, 64)
    up = (q[:, :, 0] > 0).view(128, n, 2)
    assert bool(out[up].isnan().all())
    for b in (0, 7, 70, 127):
        s = slice(b * n, (b + 1) * n)
        keep = [i for i in range(n) if i != b]
        want, want_abs, _ = attend_reference(q[s], k[s][keep], v[s][keep], False, 0.125)
        down = ~up[b] & (q[s][:, :, 0] < 0)
        within(out[b][down], want[down], HALF_ULP[DT[dt]] * (want.abs() + want_abs)[down] + 1e-6)


# ---- shared prefixes -----------------------------------------------------------------


def paged_rows(dev, n_rows, Hkv, D, bits, page, g, scale=1.0):
    """Random cache rows for sequences of n_rows[i] tokens: (codes, scales, table, values [i] -> [n, Hkv, D])."""
    import numpy as np

    pages = [-(-n // page) for n in n_rows]
    pool = sum(pages) + 2
    x = torch.randn(pool, Hkv, page, D, device=dev, generator=g) * scale
    from b200flash.quantized_kv_cache import quantize_tensor

    codes, scales, _ = quantize_tensor(x.to(torch.bfloat16), bits, 64)
    ids = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
    table = torch.zeros(len(n_rows), max(pages + [1]), dtype=torch.int32, device=dev)
    vals = torch.from_numpy(np.asarray(kv_sym.dequantize_tensor(codes.cpu().numpy(), scales.cpu().numpy(), None, bits,
                                                                tuple(x.shape), 64), np.float64)).to(dev)
    out, at = [], 0
    for i, (n, m) in enumerate(zip(n_rows, pages)):
        table[i, :m] = ids[at: at + m]
        out.append(vals[ids[at: at + m].long()].transpose(1, 2).reshape(-1, Hkv, D)[:n])
        at += m
    return codes.contiguous(), scales.contiguous(), table, out


def run_prefix(dev, off, pre, own, Hq, Hkv, D, bits, page, seed=0, qscale=1.5, kscale=1.0, vscale=1.0, tight=False):
    from b200flash.paged_prompt import shared_prefix_attention

    g = torch.Generator(device=dev).manual_seed(seed)
    B, Ng = len(own), len(pre)
    kc, ks, table, kv = paged_rows(dev, list(pre) + list(own), Hkv, D, bits, page, g, kscale)
    g2 = torch.Generator(device=dev).manual_seed(seed + 1)
    vc, vs, vtable, vv = paged_rows(dev, list(pre) + list(own), Hkv, D, bits, page, g2, vscale)
    # the values live in the pages that the keys' table names
    pool = kc.shape[0]
    vc2, vs2 = vc.clone(), vs.clone()
    used = [-(-n // page) for n in list(pre) + list(own)]
    for i, m in enumerate(used):
        vc2[table[i, :m].long()] = vc[vtable[i, :m].long()]
        vs2[table[i, :m].long()] = vs[vtable[i, :m].long()]
    # what no table names is poison
    named = torch.zeros(pool, dtype=torch.bool, device=dev)
    for i, m in enumerate(used):
        named[table[i, :m].long()] = True
        if m and (list(pre) + list(own))[i] % page:
            last, tail = int(table[i, m - 1]), (list(pre) + list(own))[i] % page
            ks[last, :, tail:] = math.nan
            vs2[last, :, tail:] = math.inf
    ks[~named] = math.nan
    vs2[~named] = math.nan
    q = (qscale * torch.randn(B, Hq, D, device=dev, generator=g)).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)
    kw = dict(max_prefix_len=max(list(pre) + [0]), max_seq_len=max(own)) if tight else {}
    out = shared_prefix_attention(q, kc, ks, vc2, vs2, table[:Ng].contiguous(), torch.tensor(pre, **i32),
                                  torch.tensor(off, **i32), table[Ng:].contiguous(), torch.tensor(own, **i32), bits,
                                  page, Hkv, **kw)
    G = Hq // Hkv
    for b in range(B):
        ks_, vs_ = [kv[Ng + b]], [vv[Ng + b]]
        for gi in range(Ng):
            if off[gi] <= b < off[gi + 1]:
                ks_.insert(0, kv[gi])
                vs_.insert(0, vv[gi])
        k, v = torch.cat(ks_), torch.cat(vs_)
        if not k.shape[0]:
            assert bool((out[b] == 0).all())
            continue
        o, o_abs, _ = attend_reference(q[b][None], k, v, False, D ** -0.5)
        move = 2.0 ** -11 * torch.einsum("hd,mhd->hm", q[b].double().abs(), k.abs().repeat_interleave(G, 1)).amax(-1)
        tol = 2.0 ** -8 * (o[0].abs() + o_abs[0]) + 2 * D ** -0.5 * move[:, None] * o_abs[0] + 1e-6 * vscale
        within(out[b], o[0], tol, f"row {b}")
    return out


@pytest.mark.parametrize("off,pre,own,Hq,Hkv,D,bits,page", [
    ([0, 1], [1], [0], 8, 1, 128, 8, 16),
    ([0, 3], [200], [0, 17, 130], 8, 2, 128, 8, 64),
    ([0, 2, 7], [129, 640], [5, 0, 64, 65, 1, 300, 2], 32, 4, 128, 8, 64),
    ([0, 5], [127], [3, 0, 0, 9, 100], 6, 2, 64, 8, 16),
    ([1, 3, 3, 6], [70, 900, 256], [40, 1, 2, 3, 4, 5, 0, 33], 16, 1, 128, 4, 32),
    ([0, 4], [333], [10, 20, 30, 0], 12, 4, 64, 4, 16),
    ([0, 3], [150], [1, 2, 3], 8, 2, 128, 2, 16),
    ([0, 2], [90], [0, 70], 5, 5, 64, 2, 32),
    ([0, 40], [1500], list(range(40)), 16, 2, 128, 8, 64),
    ([0, 70], [300], [i % 7 for i in range(70)], 8, 1, 128, 8, 128),
    ([0, 2], [0], [0, 50], 8, 2, 128, 8, 64),
    ([0, 3, 40, 41], [5, 3000, 129], [i % 9 for i in range(45)], 16, 4, 128, 8, 64),
    ([], [], [0, 50, 7], 8, 2, 128, 8, 64),
])
@pytest.mark.parametrize("tight", [False, True])
def test_shared_prefix_attention(dev, off, pre, own, Hq, Hkv, D, bits, page, tight):
    run_prefix(dev, off or [0], pre, own, Hq, Hkv, D, bits, page, seed=len(own), tight=tight)


@pytest.mark.parametrize("qscale,kscale,vscale", [(1.0, 1e-4, 1e-7), (1e-5, 3e4, 1.0), (2e5, 1e-5, 1e6), (30.0, 1.0, 1.0)])
def test_shared_prefix_attention_ranges(dev, qscale, kscale, vscale):
    """Queries, keys and values far from 1 (beyond what 16-bit floats of five exponent bits hold)."""
    run_prefix(dev, [0, 3], [400], [0, 30, 100], 8, 2, 128, 8, 64, seed=9, qscale=qscale, kscale=kscale, vscale=vscale)


def test_shared_prefix_attention_many_groups(dev):
    """More groups than a warp looks at in one go, empty ones and empty prefixes among them."""
    off, own = [0], []
    for i in range(75):
        n = (i * 7) % 4
        own += [(i * 13 + j * 5) % 40 for j in range(n)]
        off.append(off[-1] + n)
    run_prefix(dev, off, [(i * 37) % 300 for i in range(75)], own, 8, 2, 64, 8, 16, seed=3)


@pytest.mark.parametrize("n,Hq,Hkv,pre", [(300, 8, 1, [90]), (260, 16, 4, [513]), (1, 16, 1, [2000]), (9, 14, 2, [64])])
def test_shared_prefix_attention_rows(dev, n, Hq, Hkv, pre):
    """Groups of many tiles of rows, and of up to 16 heads to a KV head."""
    run_prefix(dev, [0, n], pre, [i % 3 for i in range(n)], Hq, Hkv, 128, 8, 16, seed=4)


def test_shared_prefix_one_bad_key(dev):
    """NaN in one key of the prefix, wherever it lies in a block."""
    from b200flash.paged_prompt import shared_prefix_attention

    g = torch.Generator(device=dev).manual_seed(7)
    kc, ks, table, _ = paged_rows(dev, [256], 1, 64, 8, 128, g)
    vc, vs, _, _ = paged_rows(dev, [256], 1, 64, 8, 128, g)
    q = torch.randn(2, 4, 64, device=dev, generator=g).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)
    for i in range(128):
        bad = ks.clone()
        bad[table[0, 1], 0, i] = math.nan
        out = shared_prefix_attention(q, kc, bad, vc, vs, table, torch.tensor([256], **i32), torch.tensor([0, 2], **i32),
                                      torch.zeros(2, 1, **i32), torch.zeros(2, **i32), 8, 128, 1)
        assert bool(out.isnan().all()), i


@pytest.mark.parametrize("scale", [-0.07, 0.0])
def test_shared_prefix_scales(dev, scale):
    """A negative scale turns every query about; at 0 every token weighs the same."""
    from b200flash.paged_prompt import shared_prefix_attention

    g = torch.Generator(device=dev).manual_seed(6)
    kc, ks, table, _ = paged_rows(dev, [200, 40, 7], 2, 128, 8, 16, g)
    vc, vs, _, _ = paged_rows(dev, [200, 40, 7], 2, 128, 8, 16, g)
    q = torch.randn(2, 8, 128, device=dev, generator=g).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)

    def run(q, scale):
        return shared_prefix_attention(q, kc, ks, vc, vs, table[:1].contiguous(), torch.tensor([200], **i32),
                                       torch.tensor([0, 2], **i32), table[1:].contiguous(),
                                       torch.tensor([40, 7], **i32), 8, 16, 2, softmax_scale=scale)

    got = run(q, scale)
    want = run(-q, -scale) if scale else run(torch.zeros_like(q), 0.1)
    # the own tokens' kernel rounds its scaled query to 16 bits on either side
    within(got, want, 2.0 ** -7 * want.double().abs() + 2.0 ** -7)


def test_shared_prefix_matches_decode_attention(dev):
    """The same tokens behind a shared prefix and in one table per request."""
    from b200flash.paged_prompt import shared_prefix_attention
    from b200flash.quantized_kv_cache import decode_attention

    B, Hq, Hkv, D, page, npre, nown = 6, 16, 2, 128, 64, 5, 2
    g = torch.Generator(device=dev).manual_seed(2)
    pool = npre + B * nown
    kc, vc = (torch.randint(0, 255, (pool, Hkv, page, D), device=dev, generator=g, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.rand(pool, Hkv, page, D // 64, device=dev, generator=g) * 0.02 for _ in range(2))
    ids = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
    pre, own = ids[:npre][None].contiguous(), ids[npre:].view(B, nown).contiguous()
    lens = torch.tensor([0, 1, 63, 64, 65, 128], dtype=torch.int32, device=dev)
    q = torch.randn(B, Hq, D, device=dev, generator=g).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)
    got = shared_prefix_attention(q, kc, ks, vc, vs, pre, torch.tensor([npre * page], **i32), torch.tensor([0, B], **i32),
                                  own, lens, 8, page, Hkv)
    whole = torch.cat([pre.expand(B, -1), own], 1).contiguous()
    want = decode_attention(q, kc, ks, vc, vs, whole, lens + npre * page, 8, page, Hkv)
    within(got, want, 2.0 ** -7 * want.double().abs() + 2.0 ** -7)


def test_pages_past_32_bits(dev):
    """Pages whose bytes lie past 4 GiB of the pool: the rows appended there, and the attention over them."""
    from b200flash.paged_prompt import qk_norm_rope, shared_prefix_attention

    Hq, Hkv, D, page, small, big = 16, 8, 128, 64, 6, 70_000
    g = torch.Generator(device=dev).manual_seed(8)
    T = 4 * page - 5
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, device=dev, generator=g).to(torch.bfloat16)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    got = []
    for pages in (small, big):
        codes = [torch.empty(pages, Hkv, page, D, dtype=torch.uint8, device=dev) for _ in range(2)]
        scales = [torch.empty(pages, Hkv, page, D // 64, dtype=torch.float32, device=dev) for _ in range(2)]
        ids = pages - 1 - torch.arange(4, **i32)
        slots = ids.long().repeat_interleave(page)[:T] * page + pos % page
        q, _, _ = qk_norm_rope(qkv, Hq, Hkv, pos, w, w, cache=(codes[0], scales[0], codes[1], scales[1]), slots=slots)
        out = shared_prefix_attention(q[-3:], codes[0], scales[0], codes[1], scales[1], ids[None, :3].contiguous(),
                                      torch.tensor([2 * page + 9], **i32), torch.tensor([0, 2], **i32),
                                      ids[3:].expand(3, 1).contiguous(), torch.tensor([40, 0, 7], **i32), 8, page, Hkv)
        rows = [x[ids.long()].transpose(1, 2).flatten(0, 1)[:T].clone() for x in codes + scales]
        got.append([out] + rows)
        del codes, scales
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ---- refusals ------------------------------------------------------------------------


def test_refusals(dev):
    from b200flash import paged_prompt as P

    i32 = dict(dtype=torch.int32, device=dev)
    bf = dict(dtype=torch.bfloat16, device=dev)
    n, free, tab = torch.zeros(2, **i32), torch.zeros(4, **i32), torch.zeros(2, 3, **i32)
    pos, w = torch.zeros(4, **i32), torch.ones(128, **bf)
    qkv = torch.zeros(4, 6 * 128, **bf)
    q, k, cu = torch.zeros(4, 4, 128, **bf), torch.zeros(4, 2, 128, **bf), torch.tensor([0, 4], **i32)
    pages = torch.zeros(3, 2, 16, 128, dtype=torch.uint8, device=dev)
    sc = torch.zeros(3, 2, 16, 2, dtype=torch.float32, device=dev)
    one = torch.zeros(1, **i32)
    bad = [
        lambda: P.plan_pages(n.cpu(), free, 16, 4, tab),
        lambda: P.plan_pages(n.long(), free, 16, 4, tab),
        lambda: P.plan_pages(n, free, 0, 4, tab),
        lambda: P.plan_pages(n, free, 16, -1, tab),
        lambda: P.plan_pages(n, free, 16, 4, tab[:1]),
        lambda: P.plan_pages(n, free, 16, 4, torch.zeros(3, 2, **i32).t()),
        lambda: P.plan_pages(n, free, 16, 4, tab, context_lens=torch.zeros(3, **i32)),
        lambda: P.qk_norm_rope(qkv.float(), 4, 1, pos, w, w),
        lambda: P.qk_norm_rope(qkv, 4, 2, pos, w, w),
        lambda: P.qk_norm_rope(qkv, 4, 1, pos[:3], w, w),
        lambda: P.qk_norm_rope(qkv, 4, 1, pos, w[:64], w),
        lambda: P.qk_norm_rope(qkv, 4, 1, pos, w, w.half()),
        lambda: P.qk_norm_rope(qkv, 4, 1, pos, w, w, inv_freq=torch.ones(7, dtype=torch.float64, device=dev)),
        lambda: P.qk_norm_rope(qkv, 4, 1, pos, w, w, slots=torch.zeros(4, dtype=torch.int64, device=dev)),
        lambda: P.qk_norm_rope(qkv, 4, 1, pos, w, w, cache=(pages, sc, pages, sc),
                               slots=torch.zeros(4, dtype=torch.int64, device=dev)),
        lambda: P.qk_norm_rope(torch.zeros(4, 6 * 96, **bf), 4, 1, pos, torch.ones(96, **bf), torch.ones(96, **bf)),
        lambda: P.prompt_attention(q.cpu(), k, k, cu),
        lambda: P.prompt_attention(q.float(), k.float(), k.float(), cu),
        lambda: P.prompt_attention(q, k, k.half(), cu),
        lambda: P.prompt_attention(q[:, :3], k, k, cu),
        lambda: P.prompt_attention(q, k[:3], k[:3], cu),
        lambda: P.prompt_attention(q, k, k, cu.long()),
        lambda: P.prompt_attention(torch.zeros(4, 4, 136, **bf), torch.zeros(4, 2, 136, **bf),
                                   torch.zeros(4, 2, 136, **bf), cu),
        lambda: P.prompt_attention(torch.zeros(4, 4, 12, **bf), torch.zeros(4, 2, 12, **bf), torch.zeros(4, 2, 12, **bf),
                                   cu),
        lambda: P.shared_prefix_attention(q.half(), pages, sc, pages, sc, tab[:1], one, cu, tab, n, 8, 16, 2),
        lambda: P.shared_prefix_attention(q[:2], pages, sc, pages, sc, tab[:1], one, cu, tab, n, 8, 16, 3),
        lambda: P.shared_prefix_attention(q[:2], pages, sc, pages, sc, tab[:1], one, cu, tab, n, 3, 16, 2),
        lambda: P.shared_prefix_attention(q[:2], pages, sc, pages, sc, tab[:1], one, cu, tab, n, 8, 24, 2),
        lambda: P.shared_prefix_attention(q[:2], pages, sc, pages, sc, tab[:1], n, cu, tab, n, 8, 16, 2),
        lambda: P.shared_prefix_attention(q[:2], pages, sc.double(), pages, sc, tab[:1], one, cu, tab, n, 8, 16, 2),
        lambda: P.shared_prefix_attention(q[:2], pages, sc, pages, sc, tab[:1], one, cu, tab, n, 8, 16, 2, group_size=32),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")


def test_empty_calls(dev):
    from b200flash import paged_prompt as P

    i32 = dict(dtype=torch.int32, device=dev)
    bf = dict(dtype=torch.bfloat16, device=dev)
    w = torch.ones(128, **bf)
    q, k, _ = P.qk_norm_rope(torch.zeros(0, 6 * 128, **bf), 4, 1, torch.zeros(0, **i32), w, w)
    assert q.shape == (0, 4, 128) and k.shape == (0, 1, 128)
    out = P.prompt_attention(q, k, k, torch.zeros(1, **i32))
    assert out.shape == (0, 4, 128)
    out = P.prompt_attention(torch.ones(3, 4, 128, **bf), torch.ones(3, 1, 128, **bf), torch.ones(3, 1, 128, **bf),
                             torch.zeros(1, **i32))
    assert bool((out == 0).all())  # no sequences: every row is padding
