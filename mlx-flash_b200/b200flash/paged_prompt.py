"""Packed prompts over the paged, quantized KV cache, and decode behind shared prefixes.

The reference pushes a prompt through the model in chunks with a causal mask
(``continuous_batching.py:556-580``) and every request attends over its own
cache (``quantized_kv_cache.py:311-358``).  Here a batch of prompts of any
lengths is one packed run of rows:

* :func:`plan_pages`               block tables, slot map and positions from the requests' lengths, on the GPU
* :func:`qk_norm_rope`             per-head RMSNorm + rotary of queries and keys; K and V appended to the pages
* :func:`prompt_attention`         attention of each packed sequence over itself, causal or full
* :func:`shared_prefix_attention`  decode rows that share long prefixes, each prefix read once for its group

All are stream-ordered on the current stream and can be captured in a CUDA
graph.  None waits for the host, but for the first :func:`qk_norm_rope` with a
rotary base, which copies its frequencies from there (not inside a capture).
"""

from typing import NamedTuple, Optional

import torch

from . import _capi
from ._capi import DTYPE_CODES, aligned_contiguous, call, ptr, require_cuda, stream_of
from .quantized_kv_cache import packed_len


class PagePlan(NamedTuple):
    """What :func:`plan_pages` gives for a packed batch (all int32 but ``slots``, int64)."""

    cu_seqlens: torch.Tensor  # [B + 1] packed offset of each request's tokens
    positions: torch.Tensor  # [T] position of each token in its request
    slots: torch.Tensor  # [T] page * page_size + slot of each token, -1 where it has none
    rows: torch.Tensor  # [T] request of each token, -1 past the batch
    seq_lens: torch.Tensor  # [B] tokens of each request with the new ones
    counts: torch.Tensor  # [2] tokens in the batch, pages it takes


def _int32(name, t, n=None):
    """``t`` contiguous, after checking that it is int32 ``[n]`` (None: any length)."""
    if t.dtype is not torch.int32 or t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be int32 [{'*' if n is None else n}], got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _table(name, t, n=None):
    """``t`` contiguous, after checking that it is int32 ``[n, *]``."""
    if t.dtype is not torch.int32 or t.dim() != 2 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be int32 [{'*' if n is None else n}, *], got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def plan_pages(new_lens: torch.Tensor, free_pages: torch.Tensor, page_size: int, total_tokens: int,
               block_table: torch.Tensor, context_lens: Optional[torch.Tensor] = None) -> PagePlan:
    """Plan the pages of a batch in which request ``b`` gets ``new_lens[b]`` tokens.

    ``block_table`` (int32 ``[B, max_pages]``, contiguous) is extended in
    place: request ``b`` keeps the pages of its ``context_lens[b]`` tokens and
    takes the next ``free_pages`` in request order.  ``total_tokens`` is the
    room for tokens (at least the batch's sum; the rest is padding with slot
    -1).  ``counts`` holds the tokens of the batch and the pages it needs --
    more pages than ``free_pages`` has, and the entries that got none are -1.
    """
    dev = require_cuda(new_lens, free_pages, block_table, context_lens)
    if page_size <= 0:
        raise ValueError(f"page_size must be positive, got {page_size}")
    if total_tokens < 0:
        raise ValueError(f"total_tokens must be non-negative, got {total_tokens}")
    n = _int32("new_lens", new_lens)
    B, T = n.shape[0], int(total_tokens)
    if context_lens is not None:
        context_lens = _int32("context_lens", context_lens, B)
    free = _int32("free_pages", free_pages)
    if not block_table.is_contiguous():
        raise ValueError("block_table is extended in place: it must be contiguous")
    _table("block_table", block_table, B)
    # one allocation for the int32 outputs, positions and rows on 16-byte boundaries
    pad = -T % 4
    ints = torch.empty(2 * (T + pad) + 2 * B + 3, dtype=torch.int32, device=dev)
    positions, _, rows, _, cu, lens, counts = ints.split_with_sizes((T, pad, T, pad, B + 1, B, 2))
    out = PagePlan(cu, positions, torch.empty(T, dtype=torch.int64, device=dev), rows, lens, counts)
    ws, ws_bytes = None, 0
    if B > 2048:  # more requests than every CTA scans for itself
        ws_bytes = int(_capi.lib().b2f_page_plan_workspace_bytes(B))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    call("b2f_page_plan", ptr(n), ptr(context_lens), B, ptr(free), free.shape[0], page_size, ptr(block_table),
         max(1, block_table.shape[1]), T, ptr(out.cu_seqlens), ptr(out.positions), ptr(out.slots), ptr(out.rows),
         ptr(out.seq_lens), ptr(out.counts), ptr(ws), ws_bytes, stream_of(dev))
    return out


# Kernels in flight and captured graphs hold the addresses of these: none is ever dropped.
_frequencies = {}


def rope_frequencies(rotary_dim: int, theta: float, device) -> torch.Tensor:
    """``theta ** (-2 i / rotary_dim)`` for ``i < rotary_dim / 2``, float64 on ``device`` (kept per argument).

    A first call inside a capture forms them on the device, in the graph, and
    keeps none: their memory is the graph's.
    """
    key = (rotary_dim, theta, device)
    got = _frequencies.get(key)
    if got is None:
        if torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
            i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
            return torch.pow(theta, i * (-2.0 / rotary_dim))
        got = _frequencies[key] = torch.tensor([theta ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)],
                                               dtype=torch.float64, device=device)
    return got


def qk_norm_rope(qkv: torch.Tensor, n_heads: int, n_kv_heads: int, positions: torch.Tensor, q_norm: torch.Tensor,
                 k_norm: torch.Tensor, eps: float = 1e-6, theta: float = 1e6, inv_freq: Optional[torch.Tensor] = None,
                 cache: Optional[tuple] = None, slots: Optional[torch.Tensor] = None, bits: int = 8):
    """RMSNorm each query and key head of packed rows and turn it by its position.

    ``qkv`` bf16 or fp16 ``[T, (Hq + 2 Hkv) * D]`` (rows ``[q | k | v]``, any
    row stride), ``q_norm`` / ``k_norm`` ``[D]``, ``positions`` int32 ``[T]``.
    ``inv_freq`` (float64, at most ``D / 2`` frequencies, a multiple of 8)
    replaces ``theta ** (-2 i / D)``; fewer than ``D / 2`` rotate the first
    ``2 * len`` values of a head only.  Returns ``(q [T, Hq, D], k [T, Hkv, D],
    v)``, ``v`` a view of ``qkv``.

    With ``cache = (k_codes, k_scales, v_codes, v_scales)`` -- head-major pages
    ``[pages, Hkv, page_size, ...]`` as ``decode_attention`` reads them -- and
    ``slots`` (int64 ``[T]``, -1 skips a row) the rows of k and v are quantized
    into their slots in the same pass.
    """
    dev = require_cuda(qkv, positions, q_norm, k_norm, inv_freq, slots, *(cache or ()))
    Hq, Hkv = int(n_heads), int(n_kv_heads)
    if qkv.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"qkv must be bf16 or fp16, got {qkv.dtype}")
    if Hq <= 0 or Hkv <= 0 or qkv.dim() != 2 or qkv.shape[1] % (Hq + 2 * Hkv):
        raise ValueError(f"qkv {list(qkv.shape)} does not hold {Hq} + 2 * {Hkv} heads a row")
    T, D = qkv.shape[0], qkv.shape[1] // (Hq + 2 * Hkv)
    for w in (q_norm, k_norm):
        if w.dim() != 1 or w.shape[0] != D or w.dtype is not qkv.dtype:
            raise ValueError(f"q_norm and k_norm must be {qkv.dtype} [{D}], got {w.dtype} {list(w.shape)}")
    positions = _int32("positions", positions, T)
    if inv_freq is None:
        inv_freq = rope_frequencies(D, float(theta), dev)
    elif inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or inv_freq.shape[0] * 2 > D or inv_freq.shape[0] % 8:
        raise ValueError(f"inv_freq must be float64 with a multiple of 8 up to {D // 2} values")
    else:
        inv_freq = inv_freq.contiguous()
    if (cache is None) != (slots is None):
        raise ValueError("cache and slots go together")
    x, width = qkv, qkv.shape[1]
    ld, last = x.stride()
    if last != 1 or ld % 8 or ld < width or x.data_ptr() % 16:
        x, ld = aligned_contiguous(x), width
    kc = ks = vc = vs = None
    page_size = 0
    if cache is not None:
        kc, ks, vc, vs = cache
        if slots.dtype != torch.int64 or tuple(slots.shape) != (T,):
            raise ValueError(f"slots must be int64 [{T}]")
        if bits not in (2, 4, 8):
            raise ValueError(f"bits must be 2, 4, or 8, got {bits}")
        page_size = kc.shape[2] if kc.dim() == 4 else 0
        for name, t, dt, w in (("k codes", kc, torch.uint8, packed_len(D, bits, 64)),
                               ("k scales", ks, torch.float32, D // 64),
                               ("v codes", vc, torch.uint8, packed_len(D, bits, 64)),
                               ("v scales", vs, torch.float32, D // 64)):
            if t.dtype != dt or tuple(t.shape) != (kc.shape[0], Hkv, page_size, w) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dt} [pages, {Hkv}, page_size, {w}], got "
                                 f"{t.dtype} {list(t.shape)}")
        slots = slots.contiguous()
    qw, kw = aligned_contiguous(q_norm), aligned_contiguous(k_norm)
    q = torch.empty(T, Hq, D, dtype=qkv.dtype, device=dev)
    k = torch.empty(T, Hkv, D, dtype=qkv.dtype, device=dev)
    call("b2f_qk_norm_rope_rows", ptr(x), ld, DTYPE_CODES[qkv.dtype], T, Hq, Hkv, D, ptr(qw), ptr(kw), float(eps),
         ptr(inv_freq), 2 * inv_freq.shape[0], ptr(positions), ptr(q), ptr(k), ptr(slots), ptr(kc), ptr(ks), ptr(vc),
         ptr(vs), page_size, bits, stream_of(dev))
    return q, k, qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)


def _rows_of_heads(t):
    """A [T, H, D] tensor that the attention kernel takes (copied only where its strides do not fit), its strides."""
    rows, heads, last = t.stride()
    if last != 1 or rows % 8 or heads % 8 or rows <= 0 or heads <= 0 or t.data_ptr() % 16:
        t = aligned_contiguous(t)
        rows, heads, _ = t.stride()
    return t, rows, heads


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, causal: bool = True,
                     softmax_scale: Optional[float] = None, return_lse: bool = False):
    """Attention of packed sequences over themselves.

    ``q`` bf16 or fp16 ``[T, Hq, D]``, ``k`` / ``v`` ``[T, Hkv, D]`` (views of
    packed projections are taken as they are), ``D`` a multiple of 8 up to
    128; sequence ``b`` is rows ``cu_seqlens[b]:cu_seqlens[b + 1]`` (int32,
    rising from 0).  Rows past the last sequence come out 0.  With ``return_lse`` also the
    float32 ``[T, Hq]`` log of each row's softmax sum.
    """
    dev = require_cuda(q, k, v, cu_seqlens)
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must be bf16 or fp16 alike, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"q [T, Hq, D], k and v [T, Hkv, D] expected, got {list(q.shape)}, {list(k.shape)}, "
                         f"{list(v.shape)}")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"num_kv_heads {Hkv} must divide the {Hq} query heads")
    cu = _int32("cu_seqlens", cu_seqlens)
    if cu.shape[0] < 1:
        raise ValueError("cu_seqlens must hold at least one offset")
    if softmax_scale is None:
        softmax_scale = D ** -0.5
    (q, q_row, q_head), (k, k_row, k_head), (v, v_row, v_head) = (_rows_of_heads(t) for t in (q, k, v))
    out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    call("b2f_prompt_attn", ptr(q), q_row, q_head, ptr(k), k_row, k_head, ptr(v), v_row, v_head, DTYPE_CODES[q.dtype],
         ptr(cu), cu.shape[0] - 1, T, Hq, Hkv, D, int(bool(causal)), float(softmax_scale), ptr(out), ptr(lse),
         stream_of(dev))
    return (out, lse) if return_lse else out


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, k_scales: torch.Tensor, v_pages: torch.Tensor,
                            v_scales: torch.Tensor, prefix_table: torch.Tensor, prefix_lens: torch.Tensor,
                            group_offsets: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, bits: int,
                            page_size: int, num_kv_heads: int, softmax_scale: Optional[float] = None,
                            group_size: int = 64, max_prefix_len: Optional[int] = None,
                            max_seq_len: Optional[int] = None) -> torch.Tensor:
    """Decode attention of requests that share prefixes held once in the pages.

    ``q`` bf16 ``[B, Hq, D]``, one token per request; pages as in
    ``decode_attention`` (head-major).  Requests
    ``group_offsets[g]:group_offsets[g + 1]`` (int32 ``[groups + 1]``) attend
    over the ``prefix_lens[g]`` tokens of the pages ``prefix_table[g]``, then
    each over its own ``seq_lens[b]`` tokens of ``block_table[b]``; requests
    outside every group have their own tokens only.  ``max_prefix_len`` and
    ``max_seq_len`` bound the lengths (by default what the tables can hold).
    A table entry below 0 (a page that ``plan_pages`` could not give) reads
    page 0: what such a row gives means nothing, and stays within the pool.
    """
    dev = require_cuda(q, k_pages, k_scales, v_pages, v_scales, prefix_table, prefix_lens, group_offsets, block_table,
                       seq_lens)
    if q.dtype != torch.bfloat16 or q.dim() != 3:
        raise ValueError("q must be bf16 [B, Hq, D]")
    B, Hq, D = q.shape
    Hkv = int(num_kv_heads)
    if Hkv <= 0 or Hq % Hkv:
        raise ValueError(f"num_kv_heads {Hkv} must divide the {Hq} query heads")
    if bits not in (2, 4, 8):
        raise ValueError(f"bits must be 2, 4, or 8, got {bits}")
    if group_size != 64:
        raise ValueError(f"group_size must be 64, got {group_size}")
    if page_size <= 0 or page_size % 16:
        raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    page = Hkv * page_size * D  # values of a page
    for codes, scales in ((k_pages, k_scales), (v_pages, v_scales)):
        if (codes.dtype is not torch.uint8 or scales.dtype is not torch.float32 or not codes.is_contiguous()
                or not scales.is_contiguous() or codes.numel() * 8 != scales.numel() * 64 * bits
                or scales.numel() % (page // 64)):
            raise ValueError(f"K and V must be contiguous pages of {Hkv} x {page_size} rows: uint8 codes and float32 "
                             f"scales, one per 64 values of {bits} bits")
    prefix_table = _table("prefix_table", prefix_table)
    Ng = prefix_table.shape[0]
    prefix_lens = _int32("prefix_lens", prefix_lens, Ng)
    group_offsets = _int32("group_offsets", group_offsets, Ng + 1)
    block_table = _table("block_table", block_table, B)
    seq_lens = _int32("seq_lens", seq_lens, B)
    cap_p, cap_o = prefix_table.shape[1] * page_size, block_table.shape[1] * page_size
    max_p = cap_p if max_prefix_len is None else min(int(max_prefix_len), cap_p)
    max_o = cap_o if max_seq_len is None else min(int(max_seq_len), cap_o)
    if max_p < 0 or max_o < 0:
        raise ValueError("max_prefix_len and max_seq_len must be non-negative")
    if softmax_scale is None:
        softmax_scale = D ** -0.5
    q = aligned_contiguous(q)
    out = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=dev)
    ws_bytes = int(_capi.lib().b2f_shared_prefix_attn_workspace_bytes(B, Hq, Hkv, D, Ng, max_p, max_o))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    call("b2f_shared_prefix_attn", ptr(q), ptr(k_pages), ptr(k_scales), ptr(v_pages), ptr(v_scales),
         ptr(prefix_table), max(1, prefix_table.shape[1]), ptr(prefix_lens), ptr(group_offsets), Ng, ptr(block_table),
         max(1, block_table.shape[1]), ptr(seq_lens), B, Hq, Hkv, D, page_size, bits, group_size, float(softmax_scale),
         max_p, max_o, ptr(ws), ws_bytes, ptr(out), stream_of(dev))
    return out
