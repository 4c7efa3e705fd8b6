"""The four packed-prompt operators in CUDA graphs: captured once, replayed on inputs that were written over, with a
rotary base that no call before the capture used, and after calls with many others."""

import pytest
import torch

from b200flash import _capi
from b200flash import paged_prompt as P

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 8, 2, 128, 64


class Buffers:
    """Every input of the four operators, in place; ``fill`` writes another batch into them."""

    def __init__(self, dev):
        i32 = dict(dtype=torch.int32, device=dev)
        bf = dict(dtype=torch.bfloat16, device=dev)
        self.B, self.T, self.pool = 5, 700, 40
        self.new, self.ctx, self.lens = (torch.zeros(self.B, **i32) for _ in range(3))
        self.table, self.free = torch.zeros(self.B, 8, **i32), torch.zeros(30, **i32)
        self.qkv = torch.zeros(self.T, (HQ + 2 * HKV) * D, **bf)
        self.w = torch.ones(D, **bf)
        self.q = torch.zeros(self.B, HQ, D, **bf)
        self.cache = [torch.zeros(self.pool, HKV, PAGE, n, dtype=t, device=dev)
                      for n, t in ((D, torch.uint8), (D // 64, torch.float32)) * 2]
        self.prefix, self.plens, self.off = torch.zeros(2, 9, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32)
        self.own = torch.zeros(self.B, 2, **i32)
        self.dev = dev

    def fill(self, seed):
        g = torch.Generator(device=self.dev).manual_seed(seed)
        r = lambda hi, *n: torch.randint(0, hi, n, device=self.dev, generator=g)  # noqa: E731
        self.new.copy_(r(self.T // self.B + 1, self.B))
        self.ctx.copy_(r(100, self.B))
        ids = torch.randperm(self.pool, device=self.dev, generator=g)
        self.free.copy_(ids[:30])
        self.table.copy_(ids[30:].repeat(4).view(self.B, 8))
        self.qkv.normal_(generator=g)
        self.q.normal_(generator=g)
        for i in (0, 2):
            self.cache[i].copy_(r(255, *self.cache[i].shape))
            self.cache[i + 1].uniform_(0.005, 0.02, generator=g)
        self.prefix.copy_(r(self.pool, 2, 9))
        self.plens.copy_(r(9 * PAGE, 2))
        self.off.copy_(torch.tensor([0, 1 + seed % 3, self.B]))
        self.own.copy_(r(self.pool, self.B, 2))
        self.lens.copy_(r(2 * PAGE + 1, self.B))

    def run(self, theta):
        """The outputs of the four operators; the state they write into (table, cache) is copied first."""
        table, cache = self.table.clone(), [c.clone() for c in self.cache]
        plan = P.plan_pages(self.new, self.free, PAGE, self.T, table, context_lens=self.ctx)
        q, k, v = P.qk_norm_rope(self.qkv, HQ, HKV, plan.positions, self.w, self.w, theta=theta, cache=tuple(cache),
                                 slots=plan.slots)
        o, lse = P.prompt_attention(q, k, v, plan.cu_seqlens, return_lse=True)
        d = P.shared_prefix_attention(self.q, *self.cache, self.prefix, self.plens, self.off, self.own, self.lens, 8,
                                      PAGE, HKV)
        return [table, *cache, *plan, q, k, o, lse, d]


@pytest.mark.parametrize("dependent", [False, True])
def test_graphs_replay_on_new_inputs(dev, dependent):
    theta = 31337.0 + dependent
    b = Buffers(dev)
    b.fill(0)
    b.run(5e5)  # libraries, kernels and workspaces are loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with _capi.dependent_launches(dependent):
        with torch.cuda.graph(graph):
            got = b.run(theta)
    for i in range(80):  # what an evicting cache would not survive
        P.rope_frequencies(D, 7e5 + i, dev)
    junk = [torch.full((64,), -1.0, dtype=torch.float64, device=dev) for _ in range(300)]
    for seed in (1, 2, 3, 4):
        b.fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        first = [x.clone() for x in got]
        with _capi.dependent_launches(dependent):
            want = b.run(theta)
        for i, (x, y) in enumerate(zip(first, want)):
            assert torch.equal(x, y), i
    del junk
    assert _capi.device_status(clear=True) == 0
