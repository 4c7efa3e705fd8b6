"""Requests behind shared prompts, served over a ``Qwen3MoeDecoder``'s weights and pages.

The reference pushes every request's whole prompt through its own cache in
chunks (``continuous_batching.py:556-580``).  Here prompts that several
requests share (a system prompt, a document) are pushed once, all of them in
one packed batch, and the requests decode behind them:

    batch = SharedPromptBatch(decoder)
    batch.add_prompts([[...], [...]])     # packed: any number of prompts of any lengths
    batch.start([0, 0, 0, 1])             # four requests, three behind prompt 0
    logits = batch.step(tokens)           # one token each -> bf16 [4, vocab]

Pages come from one pool: block tables, slots and positions of a step are
formed on the GPU (``plan_pages``), K and V rows are quantized into their
slots by the pass that norms and rotates the heads (``qk_norm_rope``), prompts
attend over themselves (``prompt_attention``), decode rows over their prompt,
read once for all requests behind it, and their own tokens
(``shared_prefix_attention``).
"""

import contextlib
from typing import Sequence

import torch

from ._capi import call, ptr, stream_of
from .moe import moe_block
from .mx_compat import quantized_matmul
from .paged_prompt import plan_pages, prompt_attention, qk_norm_rope, shared_prefix_attention


class SharedPromptBatch:
    """Packed prompts and the requests that decode behind them (one GPU).

    The decoder's whole page pool is the batch's from here on: the decoder's
    own rows hold none (a decoder whose rows do is refused), and neither its
    ``step`` nor another batch runs over it meanwhile.
    """

    def __init__(self, decoder):
        if decoder.world != 1:
            raise ValueError("SharedPromptBatch serves a decoder that holds all of its experts")
        if bool((torch.maximum(decoder.positions, decoder.seq_lens) > 0).any()):
            raise ValueError("the decoder's rows hold tokens in the pages that SharedPromptBatch would write to; zero its "
                             "positions and seq_lens to give them up")
        self.dec = decoder
        self.page = decoder.page
        self.device = decoder.dev
        self._free = torch.arange(decoder.num_pages, dtype=torch.int32, device=self.device)
        self.prompt_lens = []
        self.prefix_table = torch.zeros(0, 1, dtype=torch.int32, device=self.device)
        self.prefix_lens = torch.zeros(0, dtype=torch.int32, device=self.device)
        self.own_lens = []
        self._own_pages = []  # of the started requests, a tensor per step that took some

    # -- pages ------------------------------------------------------------------
    def _pages(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def _take(self, pages: int) -> torch.Tensor:
        if pages > self._free.shape[0]:
            raise RuntimeError(f"{pages} pages wanted, {self._free.shape[0]} free")
        taken, self._free = self._free[:pages], self._free[pages:]
        return taken

    @contextlib.contextmanager
    def _given_back(self):
        """Pages taken inside the block are free again if it raises."""
        before = self._free
        try:
            yield
        except BaseException:
            self._free = before
            raise

    # -- the layers ---------------------------------------------------------------
    def _forward(self, tokens, positions, slots, attend, out_rows):
        """Rows through every layer; ``attend(q, k, v, layer's pages)`` -> attention output; logits of ``out_rows``."""
        dec, s = self.dec, self.dec.s
        T, H = tokens.shape[0], s.hidden
        st = stream_of(self.device)
        e = dec.embed
        h = torch.empty(T, H, dtype=torch.bfloat16, device=self.device)
        xn = torch.empty_like(h)
        one = torch.ones(T, 1, dtype=torch.float32, device=self.device)
        call("b2f_dequantize_affine", ptr(e.wq), ptr(e.scales), ptr(e.biases), 0, T, H, e.bits, e.group_size, ptr(tokens),
             ptr(h), st)
        for ly, kv in zip(dec.layers, dec.kv):
            call("b2f_combine_rmsnorm", ptr(h), 0, 0, T, 0, ptr(ly["in_norm"]), s.rms_eps, H, 0, ptr(xn), st)
            qkv = self._dense(xn, ly["wqkv"])
            q, k, v = qk_norm_rope(qkv, s.n_heads, s.n_kv_heads, positions, ly["q_norm"], ly["k_norm"], eps=s.rms_eps,
                                   theta=s.rope_theta, cache=(kv["kc"], kv["ks"], kv["vc"], kv["vs"]), slots=slots,
                                   bits=s.kv_bits)
            o = self._dense(attend(q, k, v, kv).view(T, -1), ly["wo"])
            call("b2f_combine_rmsnorm", ptr(h), ptr(o), ptr(one), T, 1, ptr(ly["post_norm"]), s.rms_eps, H, ptr(h),
                 ptr(xn), st)
            experts = [(w.wq, w.scales, w.biases) for w in (ly["gate"], ly["up"], ly["down"])]
            h, _, _ = moe_block(xn, ly["wr"], *experts, s.top_k, bias=ly["rbias"], renorm=s.norm_topk,
                                group_size=s.group_size, bits=s.bits, residual=h)
        call("b2f_combine_rmsnorm", ptr(h), 0, 0, T, 0, ptr(dec.final_norm), s.rms_eps, H, 0, ptr(xn), st)
        return self._dense(xn if out_rows is None else xn[out_rows], dec.lm_head)

    @staticmethod
    def _dense(x, w):
        return quantized_matmul(x, w.wq, w.scales, w.biases, True, w.group_size, w.bits)

    # -- prompts ------------------------------------------------------------------
    def add_prompts(self, prompts: Sequence[Sequence[int]]) -> torch.Tensor:
        """Push prompts (token lists, none empty) as one packed batch; returns
        the bf16 ``[len(prompts), vocab]`` logits after each one's last token."""
        if not prompts or any(len(p) == 0 for p in prompts):
            raise ValueError("prompts must be non-empty token lists")
        if not all(0 <= t < self.dec.s.vocab for p in prompts for t in p):
            raise ValueError(f"tokens must lie in 0..{self.dec.s.vocab - 1}: they index the embedding")
        if self.own_lens:
            raise ValueError("prompts are added before the requests start")
        lens = [len(p) for p in prompts]
        T = sum(lens)
        i32 = dict(dtype=torch.int32, device=self.device)
        table = torch.zeros(len(lens), max(self._pages(n) for n in lens), **i32)
        new_lens = torch.tensor(lens, **i32)
        tokens = torch.tensor([t for p in prompts for t in p], **i32)
        with self._given_back():
            plan = plan_pages(new_lens, self._take(sum(self._pages(n) for n in lens)), self.page, T, table)
            logits = self._forward(tokens, plan.positions, plan.slots,
                                   lambda q, k, v, kv: prompt_attention(q, k, v, plan.cu_seqlens),
                                   plan.cu_seqlens[1:].long() - 1)
        self.prompt_lens += lens
        both = torch.zeros(len(self.prompt_lens), max(table.shape[1], self.prefix_table.shape[1]), **i32)
        both[: self.prefix_table.shape[0], : self.prefix_table.shape[1]] = self.prefix_table
        both[self.prefix_table.shape[0]:, : table.shape[1]] = table
        self.prefix_table = both
        self.prefix_lens = torch.cat([self.prefix_lens, new_lens])
        return logits

    # -- requests -----------------------------------------------------------------
    def start(self, prompt_of: Sequence[int], max_own: int = 1024):
        """Start one request per entry, behind the prompt of that index (in
        rising order), each with room for ``max_own`` tokens of its own.
        Requests that were started before end, and give their pages back."""
        n = len(self.prompt_lens)
        if any(p < 0 or p >= n for p in prompt_of) or list(prompt_of) != sorted(prompt_of):
            raise ValueError(f"requests name prompts 0..{n - 1} in rising order")
        i32 = dict(dtype=torch.int32, device=self.device)
        self._free = torch.cat([self._free] + self._own_pages)
        self._own_pages = []
        self.max_own = max_own
        self.own_lens = [0] * len(prompt_of)
        self._lens = torch.zeros(len(prompt_of), **i32)
        self._one = torch.ones(len(prompt_of), **i32)
        self._base = torch.tensor([self.prompt_lens[p] for p in prompt_of], **i32)
        self._groups = torch.tensor([sum(p < g for p in prompt_of) for g in range(n + 1)], **i32)
        self._table = torch.zeros(len(prompt_of), self._pages(max_own), **i32)

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token of each request (int32 ``[B]``, each below ``vocab``) -> bf16 logits ``[B, vocab]``."""
        B = len(self.own_lens)
        if B == 0 or tuple(tokens.shape) != (B,):
            raise ValueError(f"step takes one token for each of the {B} requests")
        if max(self.own_lens) >= self.max_own:
            raise RuntimeError(f"a request has used its {self.max_own} tokens")
        own_lens = [n + 1 for n in self.own_lens]
        s = self.dec.s

        def attend(q, k, v, kv):
            return shared_prefix_attention(q, kv["kc"], kv["ks"], kv["vc"], kv["vs"], self.prefix_table,
                                           self.prefix_lens, self._groups, self._table, plan.seq_lens, s.kv_bits,
                                           self.page, s.n_kv_heads, max_prefix_len=max(self.prompt_lens),
                                           max_seq_len=max(own_lens))

        with self._given_back():
            pages = self._take(sum(n % self.page == 0 for n in self.own_lens))
            plan = plan_pages(self._one, pages, self.page, B, self._table, context_lens=self._lens)
            logits = self._forward(tokens.to(torch.int32), plan.positions + self._base, plan.slots, attend, None)
        # a step that failed leaves nothing behind: its pages, table entries and rows are written again
        if pages.shape[0]:
            self._own_pages.append(pages)
        self._lens, self.own_lens = plan.seq_lens, own_lens
        return logits
