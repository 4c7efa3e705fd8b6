"""Pages of SharedPromptBatch: a call that fails keeps none, requests that end give theirs back."""

import pytest
import torch

from b200flash.decoder import Qwen3MoeDecoder
from b200flash.prompt_serving import SharedPromptBatch
from test_gpu_prompt_serving import SHAPE

pytestmark = pytest.mark.gpu


def batch_of(dev):
    return SharedPromptBatch(Qwen3MoeDecoder(SHAPE, max_batch=4, max_context=64, page_size=16, device=dev, seed=5))


def run(dev, fail):
    """Logits of two prompts, then of three requests over 20 steps; with ``fail`` every call fails once before."""
    batch = batch_of(dev)
    forward = batch._forward

    def broken(*args):
        forward(*args)
        raise RuntimeError("out of luck")

    def call(f):
        if fail:
            free, lens = batch._free.tolist(), list(batch.own_lens)
            batch._forward = broken
            with pytest.raises(RuntimeError, match="out of luck"):
                f()
            batch._forward = forward
            assert batch._free.tolist() == free and batch.own_lens == lens
        return f()

    out = [call(lambda: batch.add_prompts([[1, 2, 3] * 7, [9] * 16]))]
    batch.start([0, 0, 1], max_own=40)
    for t in range(20):
        tokens = torch.tensor([t, 500 - t, 7 * t], dtype=torch.int32, device=dev)
        out.append(call(lambda: batch.step(tokens)))
    return out, batch


def test_a_call_that_fails_keeps_no_pages(dev):
    for a, b in zip(run(dev, False)[0], run(dev, True)[0]):
        assert torch.equal(a, b)


def test_requests_that_end_give_their_pages_back(dev):
    out, batch = run(dev, False)
    left = batch._free.shape[0]
    pages = batch.dec.num_pages
    for _ in range(pages):  # more rounds than the pool has pages
        batch.start([0, 0, 1], max_own=40)
        for t in range(20):
            tokens = torch.tensor([t, 500 - t, 7 * t], dtype=torch.int32, device=dev)
            assert torch.equal(batch.step(tokens), out[1 + t])
        assert batch._free.shape[0] == left
    assert len(set(batch._free.tolist())) == left


def test_a_decoder_in_use_is_refused(dev):
    dec = Qwen3MoeDecoder(SHAPE, max_batch=2, max_context=64, page_size=16, device=dev, seed=5)
    dec.step()
    with pytest.raises(ValueError, match="hold tokens"):
        SharedPromptBatch(dec)
    dec.seq_lens.zero_()
    dec.positions.zero_()
    SharedPromptBatch(dec)
    dec.fill_random_context(40)
    with pytest.raises(ValueError, match="hold tokens"):
        SharedPromptBatch(dec)


@pytest.mark.parametrize("bad", [-1, SHAPE.vocab, 1 << 40])
def test_tokens_outside_the_vocabulary_are_refused(dev, bad):
    batch = batch_of(dev)
    with pytest.raises(ValueError, match="tokens must lie"):
        batch.add_prompts([[1, 2], [3, bad]])
    assert batch._free.shape[0] == batch.dec.num_pages
