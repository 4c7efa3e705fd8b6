"""Bounded waits of the packed-prompt and shared-prefix kernels: with copies
held back (b2f_set_producer_stall) and a 20 us limit every wait gives up, the
call reports B2F_ERR_TIMEOUT and the context stays usable: afterwards the same
calls give what they gave before."""

import pytest
import torch

from b200flash import _capi
from b200flash import paged_prompt as P

pytestmark = pytest.mark.gpu

B2F_ERR_TIMEOUT = -5


def calls(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    i32 = dict(dtype=torch.int32, device=dev)
    q, k, v = (torch.randn(700, h, 128, device=dev, generator=g).to(torch.bfloat16) for h in (8, 2, 2))
    cu = torch.tensor([0, 300, 310, 700], **i32)
    qkv = torch.randn(700, 12 * 128, device=dev, generator=g).to(torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16, device=dev)
    pos = torch.arange(700, **i32)
    codes = [torch.randint(0, 255, (12, 2, 64, 128), device=dev, generator=g, dtype=torch.uint8) for _ in range(2)]
    sc = [torch.rand(12, 2, 64, 2, device=dev, generator=g) * 0.02 for _ in range(2)]
    pre = torch.arange(8, **i32)[None]
    table = torch.arange(8, 12, **i32)[:, None].contiguous()
    lens = torch.tensor([0, 1, 40, 64], **i32)
    n = torch.tensor([500], **i32)
    return [
        lambda: P.prompt_attention(q, k, v, cu),
        lambda: P.qk_norm_rope(qkv, 8, 2, pos, w, w)[0],
        lambda: P.shared_prefix_attention(q[:4].contiguous(), codes[0], sc[0], codes[1], sc[1], pre, n,
                                          torch.tensor([0, 4], **i32), table, lens, 8, 64, 2),
    ]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_waits_give_up_and_recover(dev, which):
    f = calls(dev)[which]
    want = f()
    lib = _capi.lib()
    torch.cuda.synchronize()
    _capi.device_status(clear=True)
    assert lib.b2f_set_wait_limit_ns(20_000) == 0
    assert lib.b2f_set_producer_stall(1) == 0
    try:
        f()
        torch.cuda.synchronize()
        assert _capi.device_status(clear=True) == B2F_ERR_TIMEOUT
    finally:
        torch.cuda.synchronize()
        lib.b2f_set_producer_stall(0)
        lib.b2f_set_wait_limit_ns(0)
        _capi.device_status(clear=True)
    assert torch.equal(f(), want)
    assert _capi.device_status(clear=True) == 0


def test_calls_inside_a_graph(dev):
    """The operators are captured and replayed on new inputs in the same buffers."""
    fs = calls(dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        want = [f() for f in fs]
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [f() for f in fs[:2]]
    for x in got:
        x.zero_()
    graph.replay()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    with _capi.dependent_launches(True):
        for f, y in zip(fs, want):
            assert torch.equal(f(), y)
