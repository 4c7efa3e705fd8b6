"""Packed prompts and requests behind them, against the same tokens stepped one by one through the decoder.

The stepped decoder attends over 8-bit rows from the start, the packed one
over the prompt's own bf16 rows: a row's error is uniform within half a code,
absmax / 254, about 0.7 % of a value's deviation, and every stage of either
path rounds to 8 bits.  Over two layers the logits may differ by 3 % of their
norm.  Seven of eight experts are selected, so a near-tie of the router changes
which of the two smallest gates is left out, no more.
"""

import pytest
import torch

from b200flash.decoder import Qwen3MoeDecoder, Qwen3MoeShape
from b200flash.prompt_serving import SharedPromptBatch

pytestmark = pytest.mark.gpu

SHAPE = Qwen3MoeShape(hidden=512, layers=2, n_heads=8, n_kv_heads=2, head_dim=128, moe_inter=128, n_experts=8, top_k=7,
                      vocab=1000)


def stepped(dev, sequences, seed):
    """Logits after every token of each sequence, one decoder row per sequence."""
    dec = Qwen3MoeDecoder(SHAPE, max_batch=len(sequences), max_context=256, page_size=16, device=dev, seed=seed)
    out = [[] for _ in sequences]
    for i in range(max(len(q) for q in sequences)):
        dec.tokens.copy_(torch.tensor([q[min(i, len(q) - 1)] for q in sequences], dtype=torch.int32))
        dec.positions.fill_(i)
        dec.step()
        for b, q in enumerate(sequences):
            if i < len(q):
                out[b].append(dec.logits[b].float().clone())
    return out


def near(got, want):
    return float((got.float() - want).norm() / want.norm())


def test_shared_prompts_match_stepped_decoding(dev):
    g = torch.Generator().manual_seed(3)
    tok = lambda n: torch.randint(0, SHAPE.vocab, (n,), generator=g).tolist()  # noqa: E731
    prompts = [tok(37), tok(1), tok(130)]
    behind = [0, 0, 2, 2, 2]  # no request behind the second prompt
    own = [tok(18) for _ in behind]
    dec = Qwen3MoeDecoder(SHAPE, max_batch=8, max_context=256, page_size=16, device=dev, seed=11)
    batch = SharedPromptBatch(dec)
    first = batch.add_prompts(prompts[:2])
    logits = torch.cat([first, batch.add_prompts(prompts[2:])])
    want = stepped(dev, prompts, 11)
    for i, p in enumerate(prompts):
        assert near(logits[i], want[i][len(p) - 1]) < 0.03, i
    batch.start(behind, max_own=40)
    want = stepped(dev, [prompts[p] + o for p, o in zip(behind, own)], 11)
    for t in range(18):  # crosses a page of 16
        logits = batch.step(torch.tensor([o[t] for o in own], dtype=torch.int32, device=dev))
        for b, p in enumerate(behind):
            assert near(logits[b], want[b][len(prompts[p]) + t]) < 0.03, (t, b)
    assert bool(torch.isfinite(logits).all())


def test_refusals(dev):
    dec = Qwen3MoeDecoder(SHAPE, max_batch=1, max_context=32, page_size=16, device=dev, seed=1)
    batch = SharedPromptBatch(dec)
    with pytest.raises(ValueError):
        batch.add_prompts([[1, 2], []])
    with pytest.raises(RuntimeError):
        batch.add_prompts([[1] * 16 * (dec.num_pages + 1)])
    batch.add_prompts([[1, 2, 3]])
    with pytest.raises(ValueError):
        batch.start([1])
    batch.start([0], max_own=1)
    with pytest.raises(ValueError):
        batch.step(torch.zeros(2, dtype=torch.int32, device=dev))
    batch.step(torch.zeros(1, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError):
        batch.step(torch.zeros(1, dtype=torch.int32, device=dev))
