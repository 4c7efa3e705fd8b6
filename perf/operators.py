"""Work of the packed-prompt and shared-prefix operators, for measurement.

Four operators serve a batch of prompts over the paged, quantized KV cache:

* ``plan``    block tables, slot map and positions from the requests' lengths;
* ``rope``    RMS norm of each query and key head with the rotary position, optionally appending the
              quantized key and value rows to the pages of the slot map;
* ``prompt``  causal (or full) attention over packed prompts of different lengths, grouped heads;
* ``prefix``  decode attention of requests that share long prefixes held once in the pages, each
              followed by the request's own tokens.

A case names one operator and its sizes.  The lengths of a ragged batch follow from the case
(``lens_seed``), the values of its tensors from the seed given to ``prepare``.
"""

import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # three short chat turns arriving at an idle server
        dict(name="plan_few", op="plan", B=3, tokens=61, max_ctx=200, page=64, lens_seed=1),
        # a full admission wave: every slot of a large server takes a prompt
        dict(name="plan_wave", op="plan", B=509, tokens=200_003, max_ctx=1500, page=64, lens_seed=2),
        # one speculative or chunked step: a handful of tokens through one layer
        dict(name="rope_few", op="rope", tokens=7, Hq=32, Hkv=4, D=128, max_pos=4000, append=False, page=64,
             dtype="bf16"),
        # a packed prompt batch of the default decoder shape, cache rows written in the same pass
        dict(name="rope_append", op="rope", tokens=5003, Hq=32, Hkv=4, D=128, max_pos=5003, append=True, page=64,
             dtype="bf16"),
        # a long packed batch with 8 KV heads
        dict(name="rope_long", op="rope", tokens=32_768, Hq=32, Hkv=8, D=128, max_pos=32_768, append=False, page=64,
             dtype="bf16"),
        # a few short questions: latency counts
        dict(name="prompt_few", op="prompt", B=3, max_len=60, Hq=32, Hkv=4, D=128, causal=True, dtype="bf16",
             lens_seed=3),
        # an ordinary ragged prompt batch of the default decoder shape
        dict(name="prompt_ragged", op="prompt", B=16, max_len=2047, Hq=32, Hkv=4, D=128, causal=True, dtype="bf16",
             lens_seed=4),
        # an encoder-like batch: every token sees its whole sequence, one KV head per query head, 64-wide
        dict(name="prompt_full", op="prompt", B=4, max_len=1500, Hq=16, Hkv=16, D=64, causal=False, dtype="f16",
             lens_seed=5),
        # one long document
        dict(name="prompt_long", op="prompt", B=1, max_len=16_384, Hq=32, Hkv=4, D=128, causal=True, dtype="bf16",
             lens_seed=6),
        # four users behind one short system prompt
        dict(name="prefix_few", op="prefix", B=4, groups=1, prefix=500, max_own=30, Hq=32, Hkv=4, D=128, bits=8,
             page=64, lens_seed=7),
        # a decode batch of the default shape behind one long instruction block
        dict(name="prefix_batch", op="prefix", B=64, groups=1, prefix=8192, max_own=512, Hq=32, Hkv=4, D=128, bits=8,
             page=64, lens_seed=8),
        # two tenants with a book-sized prefix each, 8 KV heads, longer chats
        dict(name="prefix_book", op="prefix", B=128, groups=2, prefix=20_001, max_own=2000, Hq=32, Hkv=8, D=128,
             bits=8, page=64, lens_seed=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "rope", "prompt", "prefix"))
    seed = rng.randrange(1 << 30)
    Hq, Hkv = rng.choice(((32, 4), (32, 8), (16, 16), (8, 1), (24, 8), (16, 2)))
    if op == "plan":
        B = _log(rng, 1, 509)
        return dict(op=op, B=B, tokens=max(B, _log(rng, 8, 200_003)), max_ctx=rng.choice((0, 33, 1500)),
                    page=rng.choice((16, 64, 128)), lens_seed=seed)
    if op == "rope":
        tokens = _log(rng, 1, 32_768)
        return dict(op=op, tokens=tokens, Hq=Hq, Hkv=min(Hkv, 8), D=rng.choice((64, 128)),
                    max_pos=max(tokens, _log(rng, 100, 32_768)), append=rng.random() < 0.3,
                    page=rng.choice((16, 64)), dtype=rng.choice(("bf16", "bf16", "f16")))
    if op == "prompt":
        L = _log(rng, 2, 9000)
        B = min(_log(rng, 1, 40), max(1, 80_000_000 // (L * L)))
        return dict(op=op, B=B, max_len=L, Hq=Hq, Hkv=Hkv, D=rng.choice((64, 80, 128, 128)),
                    causal=rng.random() < 0.8, dtype=rng.choice(("bf16", "bf16", "f16")), lens_seed=seed)
    B, Hkv = _log(rng, 1, 128), min(Hkv, 8)
    return dict(op=op, B=B, groups=rng.randint(1, min(3, B)), prefix=_log(rng, 40, 16_000), max_own=_log(rng, 1, 1200),
                Hq=Hq, Hkv=Hkv, D=rng.choice((64, 128, 128)), bits=rng.choice((8, 8, 4)), page=rng.choice((16, 64)),
                lens_seed=seed)


# ---- sizes that follow from a case ------------------------------------------


def _plan_sizes(c):
    """New tokens of each request (summing to c["tokens"], some zero) and tokens each already holds."""
    r = random.Random(c["lens_seed"])
    w = [0.0 if c["B"] > 4 and r.random() < 0.1 else math.exp(r.gauss(0, 1)) for _ in range(c["B"])]
    if not any(w):
        w[0] = 1.0
    s, got, lens = sum(w), 0, []
    for x in w:
        lens.append(int(c["tokens"] * x / s))
    lens[max(range(c["B"]), key=lambda i: w[i])] += c["tokens"] - sum(lens)
    ctx = [r.randint(0, c["max_ctx"]) if r.random() < 0.7 else 0 for _ in range(c["B"])]
    return lens, ctx


def _prompt_lens(c):
    """Prompt lengths: one of the largest, the others spread below it, one of a single token in larger batches."""
    r = random.Random(c["lens_seed"])
    lens = [c["max_len"]] + [r.randint(max(1, c["max_len"] // 16), c["max_len"]) for _ in range(c["B"] - 1)]
    if c["B"] > 8:
        lens[1] = 1
    r.shuffle(lens)
    return lens


def _prefix_sizes(c):
    """Rows of each group, prefix length of each group, own tokens of each request (some zero)."""
    r = random.Random(c["lens_seed"])
    cuts = sorted(r.sample(range(1, c["B"]), c["groups"] - 1)) if c["groups"] > 1 else []
    off = [0] + cuts + [c["B"]]
    pre = [c["prefix"]] + [max(1, int(c["prefix"] * r.uniform(0.6, 1.0))) for _ in range(c["groups"] - 1)]
    ownl = [r.randint(0, c["max_own"]) for _ in range(c["B"])]
    ownl[r.randrange(c["B"])] = c["max_own"]
    return off, pre, ownl


def work(c):
    if c["op"] == "plan":
        lens, ctx = _plan_sizes(c)
        pages = sum(-(-(a + b) // c["page"]) - -(-b // c["page"]) for a, b in zip(lens, ctx))
        return {"bytes": c["tokens"] * 16 + pages * 8 + c["B"] * 16, "flops": 0}
    if c["op"] == "rope":
        heads = c["Hq"] + c["Hkv"]
        n = c["tokens"] * c["D"]
        b = 4 * n * heads + 4 * c["tokens"]
        if c["append"]:  # V is read too, K and V rows are written as codes and scales
            b += 2 * n * c["Hkv"] + 2 * c["tokens"] * c["Hkv"] * (c["D"] + c["D"] // 64 * 4)
        return {"bytes": b, "flops": 8 * n * heads}
    if c["op"] == "prompt":
        lens = _prompt_lens(c)
        t = sum(lens)
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lens)
        return {"bytes": 4 * t * c["D"] * (c["Hq"] + c["Hkv"]), "flops": 4 * c["D"] * c["Hq"] * pairs}
    off, pre, ownl = _prefix_sizes(c)
    rows = sum(pre) + sum(ownl)
    pairs = sum((b - a) * p for a, b, p in zip(off, off[1:], pre)) + sum(ownl)
    row = c["D"] * c["bits"] // 8 + c["D"] // 64 * 4
    return {"bytes": 2 * rows * c["Hkv"] * row + 4 * c["B"] * c["Hq"] * c["D"], "flops": 4 * c["D"] * c["Hq"] * pairs}


# ---- inputs -----------------------------------------------------------------


def _quantized_rows(shape, D, bits, g):
    """Rows of N(0, 1) values in the cache format: per-64 absmax scales (bf16 values in f32), biased codes."""
    x = torch.randn(*shape, D // 64, 64, device="cuda", generator=g)
    top = {8: 127, 4: 7}[bits]
    s = (x.abs().amax(-1) / top).to(torch.bfloat16).float()
    q = (x / s[..., None]).round_().clamp_(-top, top).add_(top).to(torch.uint8).reshape(*shape, D)
    if bits == 4:
        q = (q[..., 0::2] << 4) | q[..., 1::2]
    return q.contiguous(), s


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    i32 = dict(dtype=torch.int32, device="cuda")
    s = {"case": c}
    if c["op"] == "plan":
        lens, ctx = _plan_sizes(c)
        page = c["page"]
        width = max(-(-(a + b) // page) for a, b in zip(lens, ctx)) + 1
        pool = sum(-(-(a + b) // page) + 1 for a, b in zip(lens, ctx))
        ids = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
        # pages that the requests hold already, then the free list
        held = [-(-b // page) for b in ctx]
        table = torch.full((c["B"], width), -1, **i32)
        cols = torch.arange(width, device="cuda")
        mask = cols[None] < torch.tensor(held, device="cuda")[:, None]
        table[mask] = ids[: sum(held)]
        s.update(lens=torch.tensor(lens, **i32), ctx=torch.tensor(ctx, **i32), free=ids[sum(held):].contiguous(),
                 table=table)
    elif c["op"] == "rope":
        T, dt, D = c["tokens"], _DT[c["dtype"]], c["D"]
        s["qkv"] = torch.randn(T, (c["Hq"] + 2 * c["Hkv"]) * D, device="cuda", generator=g).to(dt)
        s["qn"], s["kn"] = ((1 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(dt) for _ in range(2))
        s["pos"] = torch.randint(0, c["max_pos"], (T,), device="cuda", generator=g).to(torch.int32)
        if c["append"]:
            pages = -(-T // c["page"])
            order = torch.randperm(pages, device="cuda", generator=g)
            t = torch.arange(T, device="cuda")
            s["slots"] = order[t // c["page"]] * c["page"] + t % c["page"]
            lead = (pages, c["Hkv"], c["page"])
            s["cache"] = [torch.zeros(*lead, w, dtype=d, device="cuda")
                          for w, d in ((D, torch.uint8), (D // 64, torch.float32)) * 2]
    elif c["op"] == "prompt":
        lens = _prompt_lens(c)
        T, dt, D = sum(lens), _DT[c["dtype"]], c["D"]
        s["lens"] = lens
        s["cu"] = torch.tensor([0] + lens, **i32).cumsum(0).to(torch.int32)
        s["q"] = (1.5 * torch.randn(T, c["Hq"], D, device="cuda", generator=g)).to(dt)
        s["k"] = torch.randn(T, c["Hkv"], D, device="cuda", generator=g).to(dt)
        s["v"] = torch.randn(T, c["Hkv"], D, device="cuda", generator=g).to(dt)
    else:
        off, pre, ownl = _prefix_sizes(c)
        page, D = c["page"], c["D"]
        npre, nown = [-(-p // page) for p in pre], [-(-n // page) for n in ownl]
        pool = sum(npre) + sum(nown)
        ids = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
        tables, at = [], 0
        for need, n in ((npre, c["groups"]), (nown, c["B"])):
            cols = torch.arange(max(1, max(need)), device="cuda")
            mask = cols[None] < torch.tensor(need, device="cuda")[:, None]
            t = torch.zeros(n, cols.numel(), **i32)
            t[mask] = ids[at: at + sum(need)]
            at += sum(need)
            tables.append(t)
        s["k"], s["ks"] = _quantized_rows((pool, c["Hkv"], page), D, c["bits"], g)
        s["v"], s["vs"] = _quantized_rows((pool, c["Hkv"], page), D, c["bits"], g)
        s["q"] = (1.5 * torch.randn(c["B"], c["Hq"], D, device="cuda", generator=g)).to(torch.bfloat16)
        s.update(ptable=tables[0], table=tables[1], plens=torch.tensor(pre, **i32), lens=torch.tensor(ownl, **i32),
                 off=torch.tensor(off, **i32))
    return s


# ---- the plain forms --------------------------------------------------------


def _plan_plain(s, c):
    page, T = c["page"], c["tokens"]
    lens, ctx, free, table = s["lens"].long(), s["ctx"].long(), s["free"], s["table"]
    zero = lens.new_zeros(1)
    cu = torch.cat([zero, lens.cumsum(0)])
    have, need = (ctx + page - 1) // page, (ctx + lens + page - 1) // page
    first = torch.cat([zero, (need - have).cumsum(0)])
    t = torch.arange(T, device="cuda")
    row = torch.searchsorted(cu[1:], t, right=True)
    pos = ctx[row] + t - cu[row]
    entry = pos // page
    new = first[row] + entry - have[row]
    ids = torch.where(new >= first[row], free[new.clamp(min=0)], table[row, entry]).long()
    e = torch.arange(table.shape[1], device="cuda")[None]
    new = (first[:-1, None] + e - have[:, None]).clamp(0, free.numel() - 1)
    filled = torch.where((e >= have[:, None]) & (e < need[:, None]), free[new], table)
    counts = torch.stack([cu[-1], first[-1]])
    i32 = torch.int32
    return {"table": filled, "cu_seqlens": cu.to(i32), "positions": pos.to(i32), "slots": ids * page + pos % page,
            "rows": row.to(i32), "seq_lens": (ctx + lens).to(i32), "counts": counts.to(i32)}


def _norm_rope_plain(x, w, cos, sin):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _stands_for(codes, scales):
    """The values that 8-bit rows of a cache stand for."""
    v = codes.to(torch.bfloat16).sub_(127)
    return v.view(*scales.shape, 64).mul_(scales[..., None]).view(codes.shape)


def _append_plain(x, codes, scales, slots, page):
    """Quantizes rows [T, Hkv, D] as the cache does (each step rounded to the rows' type) into their slots."""
    dt = x.dtype
    x = x.view(*x.shape[:2], -1, 64).float()
    sc = (x.abs().amax(-1, keepdim=True) / 127).to(dt).float()
    sc = torch.where(sc == 0, torch.ones_like(sc), sc)
    q = (x / sc).to(dt).float().round().clamp(-127, 127) + 127
    codes[slots // page, :, slots % page] = q.to(torch.uint8).flatten(2)
    scales[slots // page, :, slots % page] = sc[..., 0]


def _rope_plain(s, c):
    T, Hq, Hkv, D = c["tokens"], c["Hq"], c["Hkv"], c["D"]
    x = s["qkv"].view(T, Hq + 2 * Hkv, D)
    inv = torch.exp2(torch.arange(D // 2, device="cuda") * (-2.0 / D * math.log2(1e6)))
    ang = (s["pos"].float()[:, None] * inv)[:, None]
    cos, sin = ang.cos(), ang.sin()
    dt = x.dtype
    out = {"q": _norm_rope_plain(x[:, :Hq], s["qn"], cos, sin).to(dt),
           "k": _norm_rope_plain(x[:, Hq:Hq + Hkv], s["kn"], cos, sin).to(dt)}
    if c["append"]:
        kc, ks, vc, vs = s["cache"]
        _append_plain(out["k"], kc, ks, s["slots"], c["page"])
        _append_plain(x[:, Hq + Hkv:], vc, vs, s["slots"], c["page"])
        out.update(kcache=_stands_for(kc, ks), vcache=_stands_for(vc, vs))
    return out


def _softmax_product(scores, mask, v):
    """softmax of scores where ~mask, times v; scores are overwritten."""
    scores.masked_fill_(mask, -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    return (scores @ v) / scores.sum(-1, keepdim=True)


def _prompt_plain(s, c):
    lens, L, B = s["lens"], max(s["lens"]), c["B"]
    G = c["Hq"] // c["Hkv"]
    T = s["q"].shape[0]
    cu = s["cu"].long()
    i = torch.arange(L, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"].float()[at].view(B, L, c["Hkv"], G, c["D"]).permute(0, 2, 3, 1, 4).reshape(B, c["Hkv"], G * L, c["D"])
    k, v = (s[n].float()[at].transpose(1, 2) for n in "kv")
    mask = (i >= (cu[1:] - cu[:-1])[:, None])[:, None, None]
    if c["causal"]:
        mask = mask | (i[None] > i[:, None]).repeat(G, 1)
    o = _softmax_product((q * c["D"] ** -0.5) @ k.transpose(-1, -2), mask, v).view(B, c["Hkv"], G, L, c["D"])
    o = o.permute(0, 3, 1, 2, 4).reshape(B * L, c["Hq"], c["D"])
    t = torch.arange(T, device="cuda")
    row = torch.searchsorted(cu[1:], t, right=True)
    return o[row * L + t - cu[row]].to(s["q"].dtype)


def _pages_plain(codes, scales, table, bits):
    """[n, Hkv, tokens, D] float values of the pages of each row of a table."""
    x = codes[table.long()]
    if bits == 4:
        x = torch.stack([x >> 4, x & 15], -1).flatten(-2)
    sc = scales[table.long()]
    x = (x.float() - {8: 127, 4: 7}[bits]).view(*sc.shape, 64) * sc[..., None]
    x = x.flatten(-2).transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _prefix_plain(s, c):
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    gid = torch.searchsorted(s["off"][1:].long(), torch.arange(B, device="cuda"), right=True)
    q = s["q"].float().view(B, Hkv, -1, D) * D ** -0.5
    pk, pv = (_pages_plain(s[n], s[n + "s"], s["ptable"], c["bits"])[gid] for n in "kv")
    ok, ov = (_pages_plain(s[n], s[n + "s"], s["table"], c["bits"]) for n in "kv")
    at = lambda n, x: (torch.arange(x.shape[2], device="cuda") >= n[:, None])[:, None, None]  # noqa: E731
    mask = torch.cat([at(s["plens"][gid], pk), at(s["lens"], ok)], -1)
    scores = torch.cat([q @ pk.transpose(-1, -2), q @ ok.transpose(-1, -2)], -1)
    scores.masked_fill_(mask, -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    P = pk.shape[2]
    o = (scores[..., :P] @ pv + scores[..., P:] @ ov) / scores.sum(-1, keepdim=True)
    return o.view(B, c["Hq"], D).to(torch.bfloat16)


# ---- one pass ---------------------------------------------------------------


def _package():
    path = os.path.join(_ROOT, "mlx-flash_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    from b200flash import paged_prompt

    return paged_prompt


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"plan": _plan_plain, "rope": _rope_plain, "prompt": _prompt_plain, "prefix": _prefix_plain}[c["op"]](s, c)
    P = _package()
    if c["op"] == "plan":
        p = P.plan_pages(s["lens"], s["free"], c["page"], c["tokens"], s["table"], context_lens=s["ctx"])
        return {"table": s["table"], "cu_seqlens": p.cu_seqlens, "positions": p.positions, "slots": p.slots,
                "rows": p.rows, "seq_lens": p.seq_lens, "counts": p.counts}
    if c["op"] == "rope":
        cache = tuple(s["cache"]) if c["append"] else None
        q, k, _ = P.qk_norm_rope(s["qkv"], c["Hq"], c["Hkv"], s["pos"], s["qn"], s["kn"], eps=1e-6, theta=1e6,
                                 cache=cache, slots=s.get("slots"), bits=8)
        out = {"q": q, "k": k}
        if c["append"]:
            kc, ks, vc, vs = cache
            out.update(kcache=_stands_for(kc, ks), vcache=_stands_for(vc, vs))
        return out
    if c["op"] == "prompt":
        return P.prompt_attention(s["q"], s["k"], s["v"], s["cu"], causal=c["causal"])
    return P.shared_prefix_attention(s["q"], s["k"], s["ks"], s["v"], s["vs"], s["ptable"], s["plens"], s["off"],
                                     s["table"], s["lens"], c["bits"], c["page"], c["Hkv"])


# ---- the definitions in 64 bits ---------------------------------------------


def _attend64(q, k, v, first=None):
    """Attention of q [n, H, D] over k, v [m, Hkv, D]; with first, row i sees keys 0..first + i."""
    n, H, D = q.shape
    m, Hkv = k.shape[:2]
    out = torch.empty_like(q)
    step = max(1, (1 << 26) // max(1, m * (H // Hkv)))
    for h in range(Hkv):
        heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
        for a in range(0, n, step):
            z = torch.einsum("nhd,md->hnm", q[a:a + step, heads], k[:, h]) / math.sqrt(D)
            if first is not None:
                i = torch.arange(a, min(n, a + step), device=q.device)[:, None] + first
                z = z.masked_fill(torch.arange(m, device=q.device)[None] > i, -math.inf)
            out[a:a + step, heads] = torch.einsum("hnm,md->nhd", torch.softmax(z, -1), v[:, h])
    return out


def _values64(codes, scales, bits):
    if bits == 4:
        codes = torch.stack([codes // 16, codes % 16], -1).flatten(-2)
    x = codes.double() - (2 ** (bits - 1) - 1)
    return x * scales.double().repeat_interleave(64, -1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "plan":
        return None
    if c["op"] == "rope":
        D, Hq, Hkv = c["D"], c["Hq"], c["Hkv"]
        x = s["qkv"].double().view(c["tokens"], -1, D)
        i = torch.arange(D // 2, device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           s["pos"].double()[:, None] * torch.pow(torch.tensor(1e6, dtype=torch.float64), -2 * i / D))
        out = {}
        for name, lo, hi, w in (("q", 0, Hq, s["qn"]), ("k", Hq, Hq + Hkv, s["kn"])):
            y = x[:, lo:hi]
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            z = torch.complex(y[..., : D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn[:, None]
            out[name] = torch.cat([z.real, z.imag], -1)
        if c["append"]:  # held in 8 bits: no value in 64 bits
            out.update(kcache=None, vcache=None)
        return out
    if c["op"] == "prompt":
        if c["Hq"] * sum(n * n for n in s["lens"]) > 1 << 34:
            return None
        parts, a = [], 0
        for n in s["lens"]:
            q, k, v = (s[x][a:a + n].double() for x in "qkv")
            parts.append(_attend64(q, k, v, 0 if c["causal"] else None))
            a += n
        return torch.cat(parts)
    off, pre, ownl = _prefix_sizes(c)
    out = torch.empty(c["B"], c["Hq"], c["D"], dtype=torch.float64, device="cuda")

    def rows(name, table, n):
        pages = table[: -(-n // c["page"])].long()
        x = _values64(s[name][pages], s[name + "s"][pages], c["bits"])
        return x.transpose(1, 2).reshape(-1, c["Hkv"], c["D"])[:n]

    for g, p in enumerate(pre):
        shared = [rows(n, s["ptable"][g], p) for n in "kv"]
        for b in range(off[g], off[g + 1]):
            k, v = (torch.cat([x, rows(n, s["table"][b], ownl[b])]) for x, n in zip(shared, "kv"))
            out[b] = _attend64(s["q"][b:b + 1].double(), k, v)[0]
    return out
