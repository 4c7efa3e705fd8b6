"""Edges of the packed-prompt and shared-prefix operators: tables that lack pages, large scores, rows of very
different magnitudes, infinite scores, captured calls.  Bounds as in test_gpu_paged_prompt.py unless a test says more."""

import math

import pytest
import torch

from test_gpu_paged_prompt import DT, HALF_ULP, attend_reference, packed, paged_rows, within

pytestmark = pytest.mark.gpu


# ---- tables that lack pages ----------------------------------------------------------


@pytest.mark.parametrize("Hq,Hkv,D,bits,page", [
    (8, 2, 128, 8, 64), (8, 2, 128, 8, 16), (16, 1, 128, 8, 16), (8, 2, 64, 8, 64), (8, 2, 128, 4, 16),
    (8, 2, 64, 2, 32), (8, 2, 128, 8, 512),
])
def test_entries_without_a_page_read_page_0(dev, Hq, Hkv, D, bits, page):
    """A table that plan_pages could not fill holds -1; the call stays within the pool and reads page 0 there."""
    from b200flash.paged_prompt import plan_pages, shared_prefix_attention
    from b200flash.quantized_kv_cache import decode_attention

    g = torch.Generator(device=dev).manual_seed(page)
    n = 4
    kc, ks, _, _ = paged_rows(dev, [n * page], Hkv, D, bits, page, g)
    vc, vs, _, _ = paged_rows(dev, [n * page], Hkv, D, bits, page, g)
    i32 = dict(dtype=torch.int32, device=dev)
    table = torch.zeros(2, 3, **i32)
    plan = plan_pages(torch.tensor([page + 3, 2 * page], **i32), torch.tensor([3, 1], **i32), page, 3 * page + 3, table)
    assert table.tolist() == [[3, 1, 0], [-1, -1, 0]] and plan.counts.tolist() == [3 * page + 3, 4]
    q = torch.randn(2, Hq, D, device=dev, generator=g).to(torch.bfloat16)
    prefix, plens = torch.tensor([[2, -1]], **i32), torch.tensor([page + 5], **i32)

    def run(table, prefix):
        return shared_prefix_attention(q, kc, ks, vc, vs, prefix, plens, torch.tensor([0, 2], **i32), table,
                                       plan.seq_lens, bits, page, Hkv)

    assert torch.equal(run(table, prefix), run(table.clamp(min=0), prefix.clamp(min=0)))
    args = (q, kc, ks, vc, vs)
    assert torch.equal(decode_attention(*args, table, plan.seq_lens, bits, page, Hkv),
                       decode_attention(*args, table.clamp(min=0), plan.seq_lens, bits, page, Hkv))


# ---- shared prefixes: large scores ---------------------------------------------------


def exact_rows(dev, rows, D, page, g):
    """One KV head's pages whose key ``t`` holds the whole numbers ``rows[t]`` (codes, scale 1); random values."""
    n = len(rows)
    pages = -(-n // page)
    kc = torch.full((pages, 1, page, D), 127, dtype=torch.uint8, device=dev)
    kc.view(-1, D)[:n] += torch.tensor(rows, device=dev).to(torch.uint8)  # mod 256: signed values
    ks = torch.ones(pages, 1, page, D // 64, device=dev)
    vc, vs, _, _ = paged_rows(dev, [pages * page], 1, D, 8, page, g)
    vc, vs = vc[:pages].contiguous(), vs[:pages].contiguous()
    v = (vc.double() - 127).view(pages, 1, page, -1, 64) * vs.double()[..., None]
    return kc, ks, vc, vs, v.view(pages * page, 1, D)[:n]


@pytest.mark.parametrize("n_own", [0, 60])
@pytest.mark.parametrize("first", [80, 128, 160, 1600, -80, -128, -160, -1600])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_prefix_large_scores(dev, D, first, n_own):
    """Scores of up to 102400 in base 2, of either sign, at several places within a step of a 16-bit float.

    Every product and sum of q and K is a whole number of eighths of at most 24 bits, so a score of M differs from the
    exact one by the rounding of its scaling in base 2 only, 3 * 2^-24 |M|; own tokens are given the roundings of sums of
    codes with 1024 added in float32, 10 * 2^-24 * 1151 sum |q|.  A probability moves by twice ln 2 of that.
    """
    from b200flash.paged_prompt import shared_prefix_attention

    page, n = 64, 300
    g = torch.Generator(device=dev).manual_seed(D + first)
    step = torch.randint(-40, 41, (n + n_own,), device=dev, generator=g).tolist()
    offs = [0, 13, 31, 45, 100]
    rows = [[64, 1, s] + [0] * (D - 3) for s in step]
    kc, ks, vc, vs, v = exact_rows(dev, rows, D, page, g)
    q = torch.zeros(len(offs), 2, D, device=dev)
    q[:, :, 0] = first
    q[:, :, 1] = torch.tensor(offs, device=dev)[:, None]
    q[:, 0, 2], q[:, 1, 2] = 0.125, -0.125
    q = q.to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)
    B = len(offs)
    pages = torch.arange(kc.shape[0], **i32)
    if n_own:  # the prefix's last page and the own tokens' first are different pages
        cut = 256
        own = pages[cut // page:].expand(B, -1).contiguous()
    else:
        cut, own = n, torch.zeros(B, 1, **i32)
    out = shared_prefix_attention(q, kc, ks, vc, vs, pages[None, : -(-cut // page)].contiguous(),
                                  torch.tensor([cut], **i32), torch.tensor([0, B], **i32), own,
                                  torch.full((B,), n + n_own - cut, **i32), 8, page, 1, softmax_scale=math.log(2))
    k = torch.tensor(rows, dtype=torch.float64, device=dev)[:, None]
    for b in range(B):
        o, o_abs, _ = attend_reference(q[b][None], k, v, False, math.log(2))
        most = abs(first) * 64 + 105
        score = 3 * 2.0 ** -24 * most
        if n_own:
            score += 10 * 2.0 ** -24 * 1151 * float(q[b].double().abs().sum(-1).max())
        within(out[b], o[0], 2.0 ** -8 * (o[0].abs() + o_abs[0]) + 2 * math.log(2) * score * o_abs[0] + 1e-6, f"row {b}")


# ---- shared prefixes: rows of very different magnitudes ------------------------------


def cache_of(x, bits, page):
    """Pages (in order) of the rows ``x`` [n, Hkv, D], and the values that they stand for in 64 bits."""
    from b200flash.quantized_kv_cache import quantize_tensor

    n, Hkv, D = x.shape
    pages = max(1, -(-n // page))
    full = torch.zeros(pages * page, Hkv, D, dtype=x.dtype, device=x.device)
    full[:n] = x
    codes, scales, _ = quantize_tensor(full.view(pages, page, Hkv, D).transpose(1, 2).contiguous(), bits, 64)
    c = codes
    if bits < 8:
        c = torch.stack([(codes >> s) & (2 ** bits - 1) for s in range(8 - bits, -1, -bits)], -1).flatten(-2)
    v = (c.double() - (2 ** (bits - 1) - 1)).view(pages, Hkv, page, -1, 64) * scales.double()[..., None]
    return codes, scales, v.reshape(pages, Hkv, page, D).transpose(1, 2).reshape(-1, Hkv, D)[:n]


def run_rows(k, v, own, bits, page, q, softmax_scale, splits=1):
    """Attention of ``q`` over the rows ``k``, ``v`` [n, Hkv, D], as one request's own tokens or as its prefix."""
    from b200flash.paged_prompt import shared_prefix_attention

    dev, n, Hkv = q.device, k.shape[0], k.shape[1]
    kc, ks, kv = cache_of(k, bits, page)
    vc, vs, vv = cache_of(v, bits, page)
    i32 = dict(dtype=torch.int32, device=dev)
    B = q.shape[0]
    table = torch.arange(kc.shape[0], **i32)
    lens = torch.full((B,), n, **i32)
    empty, none = torch.zeros(B, 1, **i32), torch.zeros(B, **i32)
    if own:
        out = shared_prefix_attention(q, kc, ks, vc, vs, empty[:0], none[:0], none[:1], table.expand(B, -1).contiguous(),
                                      lens, bits, page, Hkv, softmax_scale=softmax_scale)
    else:
        out = shared_prefix_attention(q, kc, ks, vc, vs, table[None], lens[:1], torch.tensor([0, B], **i32), empty, none,
                                      bits, page, Hkv, softmax_scale=softmax_scale)
    return out, kv, vv


def check_rows(out, q, kv, vv, softmax_scale, floor):
    """The bound of run_prefix: roundings of P, V and the output, 2^-11 of each product in a score."""
    G = q.shape[1] // kv.shape[1]
    for b in range(q.shape[0]):
        o, o_abs, _ = attend_reference(q[b][None], kv, vv, False, softmax_scale)
        move = 2.0 ** -11 * torch.einsum("hd,mhd->hm", q[b].double().abs(), kv.abs().repeat_interleave(G, 1)).amax(-1)
        within(out[b], o[0], 2.0 ** -8 * (o[0].abs() + o_abs[0]) + 2 * softmax_scale * move[:, None] * o_abs[0] + floor,
               f"row {b}")


FORMS = [  # Hq, Hkv, D, bits, page: every form of the own-token kernel, every width of the prefix kernel
    (8, 2, 128, 8, 64), (8, 2, 128, 8, 16), (16, 1, 128, 8, 16), (8, 2, 64, 8, 64), (8, 2, 128, 4, 16),
    (4, 2, 64, 4, 32), (8, 2, 128, 2, 16), (8, 2, 64, 2, 32), (4, 1, 128, 8, 512),
]


def zeros_among_small_values(dev, form, size, own):
    Hq, Hkv, D, bits, page = form
    g = torch.Generator(device=dev).manual_seed(int(-math.log10(size)) + D)
    n = 300
    k, v = (torch.randn(n, Hkv, D, device=dev, generator=g) for _ in range(2))
    v *= size
    for at in (0, 37, 38, 250, 299):
        k[at] = v[at] = 0  # a group of zeros has scale 1
    k[20, 0, :64] = v[60, :, :64] = v[129, 0, :64] = 0
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    q = torch.randn(3, Hq, D, device=dev, generator=g).to(torch.bfloat16)
    out, kv, vv = run_rows(k, v, own, bits, page, q, D ** -0.5)
    check_rows(out, q, kv, vv, D ** -0.5, 1e-6 * size)
    # small keys: the scores are made up for by the queries
    k2 = (k.float() * size).to(torch.bfloat16)
    q2 = (q.float() / size).to(torch.bfloat16)
    out, kv, vv = run_rows(k2, v, own, bits, page, q2, D ** -0.5)
    check_rows(out, q2, kv, vv, D ** -0.5, 1e-6 * size)


def values_that_jump(dev, form, ratio, own, dtype=torch.bfloat16):
    """Values ``ratio`` times larger or smaller from some token on, to rows that see either side, or both."""
    Hq, Hkv, D, bits, page = form
    g = torch.Generator(device=dev).manual_seed(D + bits)
    n = 300
    for first in (1, 3, 40, 128, 130, 290):
        for scale in (ratio, 1 / ratio):
            k, v = (torch.randn(n, Hkv, D, device=dev, generator=g) for _ in range(2))
            v[first:] *= scale
            k[:, :, 0] = 0
            k[first:, :, 0] = 7.0
            q = torch.randn(3, Hq, D, device=dev, generator=g)
            # scores of the second part: 60 higher, 60 lower, alike
            q[:, :, 0] = torch.tensor([60.0, -60.0, 0.0], device=dev)[:, None] * D ** 0.5 / 7.0
            k, v, q = k.to(dtype), v.to(dtype), q.to(torch.bfloat16)
            out, kv, vv = run_rows(k, v, own, bits, page, q, D ** -0.5)
            check_rows(out, q, kv, vv, D ** -0.5, 1e-6 * min(1.0, scale))


@pytest.mark.parametrize("size", [0.1, 1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("form", FORMS)
def test_own_tokens_of_zeros_among_small_values(dev, form, size):
    zeros_among_small_values(dev, form, size, own=True)


@pytest.mark.parametrize("ratio", [2.0 ** 8, 1e5, 2.0 ** 20])
@pytest.mark.parametrize("form", FORMS)
def test_own_tokens_whose_values_jump(dev, form, ratio):
    values_that_jump(dev, form, ratio, own=True)


@pytest.mark.parametrize("size", [0.1, 1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("form", FORMS)
def test_prefixes_of_zeros_among_small_values(dev, form, size):
    zeros_among_small_values(dev, form, size, own=False)


@pytest.mark.parametrize("ratio", [2.0 ** 8, 1e5, 2.0 ** 20])
@pytest.mark.parametrize("form", FORMS)
def test_prefixes_whose_values_jump(dev, form, ratio):
    values_that_jump(dev, form, ratio, own=False)


@pytest.mark.parametrize("form", [f for f in FORMS if f[3] == 8])
@pytest.mark.parametrize("own", [False, True])
def test_half_precision_rows_whose_values_jump(dev, form, own):
    """Scales of 11 significant bits, as rows appended in fp16 have them."""
    values_that_jump(dev, form, 2.0 ** 10, own, dtype=torch.float16)


# ---- infinite scores, huge values ----------------------------------------------------


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_rows_whose_scores_are_all_minus_infinity(dev, D, causal, dt):
    """The formula gives NaN there, whether or not a block has masked keys; their lse is -inf; other rows are as ever."""
    from b200flash.paged_prompt import prompt_attention

    lens = [256, 300, 128]
    q, k, v, cu = packed(dev, lens, 4, 2, D, dt, seed=D)
    q[:, 0, 0], q[:, 2, 0] = 2.0, 2.0
    q[:, 1, 0], q[:, 3, 0] = 0.0, 0.0
    clean = k.clone()
    k[256:556, :, 0] = -math.inf
    out, lse = prompt_attention(q, k, v, cu, causal=causal, return_lse=True)
    want = prompt_attention(q, clean, v, cu, causal=causal)
    for s in (slice(0, 256), slice(556, 684)):
        assert torch.equal(out[s], want[s])
    assert bool(out[256:556].isnan().all())  # heads 1 and 3: 0 * inf
    assert bool((lse[256:556, 0::2] == -math.inf).all())


def test_prompt_huge_value_behind_a_negligible_score(dev):
    """exp(-300) times the largest bf16 value is 0, wherever the key lies in its block."""
    from b200flash.paged_prompt import prompt_attention

    n = 256
    q, k, v, cu = packed(dev, [n] * 128, 2, 1, 64, "bf16", seed=12)
    at = torch.arange(128, device=dev) * (n + 1)  # key i of sequence i
    q[:, :, 0], k[:, :, 0] = 16.0, 0.0
    k[at, 0, 0] = -150.0  # a score of -300
    v[at] = 3e38
    out = prompt_attention(q, k, v, cu, causal=False, softmax_scale=0.125)
    for b in (0, 5, 6, 7, 62, 70, 126, 127):
        s = slice(b * n, (b + 1) * n)
        keep = [i for i in range(n) if i != b]
        k2, v2 = k[s][keep], v[s][keep]
        o, o_abs, _ = attend_reference(q[s], k2, v2, False, 0.125)
        within(out[s], o, HALF_ULP[torch.bfloat16] * (o.abs() + o_abs) + 1e-6, f"key {b}")


@pytest.mark.parametrize("n_pre,n_own", [(256, 0), (300, 0), (256, 40), (0, 40), (0, 128), (100, 3)])
@pytest.mark.parametrize("D,bits,Hq", [(128, 8, 4), (64, 8, 4), (128, 4, 16)])
def test_shared_prefix_rows_whose_scores_are_all_minus_infinity(dev, D, bits, Hq, n_pre, n_own):
    """NaN, as the formula gives; with one finite score the rest weighs nothing."""
    from b200flash.paged_prompt import shared_prefix_attention

    page = 64
    g = torch.Generator(device=dev).manual_seed(n_pre + n_own)
    npp, npo = -(-n_pre // page), -(-n_own // page)
    kc, ks, _, _ = paged_rows(dev, [(npp + npo + 1) * page], 1, D, bits, page, g)
    vc, vs, _, _ = paged_rows(dev, [(npp + npo + 1) * page], 1, D, bits, page, g)
    kc.fill_({8: 100, 4: 0x33}[bits])  # below the code of 0
    ks.fill_(math.inf)
    q = torch.rand(2, Hq, D, device=dev, generator=g).add(0.5).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)
    pre = torch.arange(npp, **i32)[None] if npp else torch.zeros(1, 1, **i32)
    own = (npp + torch.arange(npo, **i32)).expand(2, npo).contiguous() if npo else torch.zeros(2, 1, **i32)

    def run():
        return shared_prefix_attention(q, kc, ks, vc, vs, pre, torch.tensor([n_pre], **i32), torch.tensor([0, 2], **i32),
                                       own, torch.full((2,), n_own, **i32), bits, page, 1)

    assert bool(run().isnan().all())
    p, s = (npp + (n_own - 1) // page, (n_own - 1) % page) if n_own else ((n_pre - 1) // page, (n_pre - 1) % page)
    ks[p, 0, s] = 0.01
    c = vc[p, 0, s] if bits == 8 else torch.stack([vc[p, 0, s] >> 4, vc[p, 0, s] & 15], -1).flatten()
    want = ((c.double() - (2 ** (bits - 1) - 1)).view(-1, 64) * vs[p, 0, s].double()[:, None]).flatten()
    within(run(), want.expand(2, Hq, D), 2.0 ** -8 * want.abs().expand(2, Hq, D) * 2 + 1e-6)


@pytest.mark.parametrize("Hq,Hkv,D", [(24, 8, 128), (12, 1, 128), (24, 1, 64), (14, 2, 80)])
def test_prompt_groups_that_do_not_divide_a_tile(dev, Hq, Hkv, D):
    """Whatever an earlier call left in shared memory (here NaN queries), the rows of a tile that no head fills stay out."""
    from b200flash.paged_prompt import prompt_attention

    lens = [700, 300, 1]
    q, k, v, cu = packed(dev, lens, Hq, Hkv, D, "bf16", seed=Hq)
    nan = torch.full((8192, 32, 128), math.nan, dtype=torch.bfloat16, device=dev)
    kn = torch.zeros(8192, 4, 128, dtype=torch.bfloat16, device=dev)
    first = prompt_attention(q, k, v, cu, causal=False)
    prompt_attention(nan, kn, kn, torch.tensor([0, 8192], dtype=torch.int32, device=dev))
    assert torch.equal(prompt_attention(q, k, v, cu, causal=False), first)
    for s in (slice(0, 700), slice(700, 1000)):
        o, o_abs, _ = attend_reference(q[s], k[s], v[s], False, D ** -0.5)
        within(first[s], o, HALF_ULP[q.dtype] * (o.abs() + o_abs) + 1e-6)


def test_shared_prefix_many_prefixes_few_requests(dev):
    """Thousands of prefixes, requests behind a few of them: all but their groups are empty."""
    from b200flash.paged_prompt import shared_prefix_attention

    Hq, Hkv, D, page, n = 8, 2, 128, 16, 3000
    g = torch.Generator(device=dev).manual_seed(13)
    at = [5, 5, 700, 2999]  # the prefix of each request
    pre = [(i * 37) % 48 + 1 for i in range(n)]
    kc, ks, table, kv = paged_rows(dev, [48] * 8 + [20] * 4, Hkv, D, 8, page, g)
    vc, vs, _, _ = paged_rows(dev, [48] * 8 + [20] * 4, Hkv, D, 8, page, g)
    i32 = dict(dtype=torch.int32, device=dev)
    q = torch.randn(4, Hq, D, device=dev, generator=g).to(torch.bfloat16)
    prefix = table[torch.arange(n, device=dev) % 8].contiguous()
    off = torch.tensor([sum(p < i for p in at) for i in range(n + 1)], **i32)
    lens = torch.tensor([20, 0, 7, 16], **i32)
    out = shared_prefix_attention(q, kc, ks, vc, vs, prefix, torch.tensor(pre, **i32), off, table[8:].contiguous(), lens, 8,
                                  page, Hkv)
    for b, p in enumerate(at):  # the same request alone
        want = shared_prefix_attention(q[b: b + 1], kc, ks, vc, vs, prefix[p: p + 1], torch.tensor([pre[p]], **i32),
                                       torch.tensor([0, 1], **i32), table[8 + b: 9 + b].contiguous(), lens[b: b + 1], 8, page,
                                       Hkv)
        # other splits: float32 sums in another order, so the two may round to neighbours
        within(out[b], want[0].double(), 2.0 ** -7 * want[0].double().abs() + 1e-4)


def test_shared_prefix_tables_without_columns(dev):
    """No request has tokens of its own yet, or no prefix has any: tables of no pages."""
    from b200flash.paged_prompt import shared_prefix_attention

    g = torch.Generator(device=dev).manual_seed(14)
    kc, ks, table, _ = paged_rows(dev, [90, 40, 7], 2, 128, 8, 16, g)
    vc, vs, _, _ = paged_rows(dev, [90, 40, 7], 2, 128, 8, 16, g)
    q = torch.randn(2, 8, 128, device=dev, generator=g).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)

    def run(prefix, n_pre, own, n_own):
        return shared_prefix_attention(q, kc, ks, vc, vs, prefix, torch.tensor([n_pre], **i32), torch.tensor([0, 2], **i32),
                                       own, torch.tensor(n_own, **i32), 8, 16, 2)

    none = torch.zeros(2, 0, **i32)
    pre, own = table[:1].contiguous(), table[1:].contiguous()
    assert torch.equal(run(pre, 90, none, [0, 0]), run(pre, 90, own, [0, 0]))
    assert torch.equal(run(none[:1], 0, own, [40, 7]), run(pre, 0, own, [40, 7]))
    assert bool((run(none[:1], 0, none, [0, 0]) == 0).all())


# ---- shared prefixes: scales of the softmax against the formula ----------------------


@pytest.mark.parametrize("scale", [-0.07, 0.0, 0.5, 1e-12])
@pytest.mark.parametrize("form", FORMS)
def test_shared_prefix_scales_of_the_softmax(dev, form, scale):
    """Prefix and own tokens under softmax scales of either sign and 0, at the bound of run_prefix."""
    from b200flash.paged_prompt import shared_prefix_attention

    Hq, Hkv, D, bits, page = form
    g = torch.Generator(device=dev).manual_seed(D + bits)
    n_pre, n_own = 200, [40, 0, 7]
    rows = [(torch.randn(n, Hkv, D, device=dev, generator=g).to(torch.bfloat16),
             torch.randn(n, Hkv, D, device=dev, generator=g).to(torch.bfloat16)) for n in [n_pre] + n_own]
    kc, ks, vc, vs, tables, vals, at = [], [], [], [], [], [], 0
    for k, v in rows:
        c, s, kv = cache_of(k, bits, page)
        d, t, vv = cache_of(v, bits, page)
        kc.append(c), ks.append(s), vc.append(d), vs.append(t)
        tables.append(list(range(at, at + c.shape[0])))
        vals.append((kv, vv))
        at += c.shape[0]
    i32 = dict(dtype=torch.int32, device=dev)
    width = max(len(t) for t in tables)
    table = torch.tensor([t + [0] * (width - len(t)) for t in tables], **i32)
    q = torch.randn(3, Hq, D, device=dev, generator=g).to(torch.bfloat16)
    out = shared_prefix_attention(q, torch.cat(kc), torch.cat(ks), torch.cat(vc), torch.cat(vs), table[:1].contiguous(),
                                  torch.tensor([n_pre], **i32), torch.tensor([0, 3], **i32), table[1:].contiguous(),
                                  torch.tensor(n_own, **i32), bits, page, Hkv, softmax_scale=scale)
    for b in range(3):
        k, v = (torch.cat([vals[0][i], vals[1 + b][i]]) for i in (0, 1))
        o, o_abs, _ = attend_reference(q[b][None], k, v, False, scale)
        move = 2.0 ** -11 * torch.einsum("hd,mhd->hm", q[b].double().abs(), k.abs().repeat_interleave(Hq // Hkv, 1)).amax(-1)
        within(out[b], o[0], 2.0 ** -8 * (o[0].abs() + o_abs[0]) + 2 * abs(scale) * move[:, None] * o_abs[0] + 1e-6, f"row {b}")
