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
