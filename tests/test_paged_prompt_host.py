"""Packed prompts and shared prefixes without a GPU: refusals of host tensors
and the index maps of the kernels."""

import numpy as np
import pytest
import torch

from oracle import kv_sym


def test_host_tensors_are_refused():
    from b200flash import paged_prompt as P

    i32 = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 3, dtype=torch.int32)
    x = torch.zeros(4, 6 * 128, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16)
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    c, s = torch.zeros(1, 1, 16, 128, dtype=torch.uint8), torch.zeros(1, 1, 16, 2)
    for f in (lambda: P.plan_pages(i32, i32, 16, 4, t),
              lambda: P.qk_norm_rope(x, 4, 1, torch.zeros(4, dtype=torch.int32), w, w),
              lambda: P.prompt_attention(q, q, q, i32),
              lambda: P.shared_prefix_attention(q, c, s, c, s, t, i32, i32, t, i32, 8, 16, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            f()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rotary_pieces_cover_a_head(D):
    """A lane's two 4-value pieces: every value once, and rotary partners in one lane."""
    for R in range(0, D + 1, 16):
        seen = []
        for sub in range(D // 8):
            turns = sub < R // 8
            a = 4 * sub if turns else R + 8 * (sub - R // 8)
            b = a + R // 2 if turns else a + 4
            seen += list(range(a, a + 4)) + list(range(b, b + 4))
            if turns:
                assert a + 4 <= R // 2 <= b and b + 4 <= R
        assert sorted(seen) == list(range(D))
        # where piece j of the head is found when 8 consecutive values are gathered into a lane
        for j in range(D // 4):
            q8 = R // 8
            lane = j if j < q8 else j - q8 if j < 2 * q8 else q8 + (j - 2 * q8) // 2
            second = False if j < q8 else True if j < 2 * q8 else bool((j - 2 * q8) & 1)
            first = 4 * lane if lane < q8 else R + 8 * (lane - q8)
            at = (first + R // 2 if lane < q8 else first + 4) if second else first
            assert at == 4 * j


@pytest.mark.parametrize("bits", [8, 4, 2])
def test_codes_spread_in_order(bits):
    """The byte order in which a 16-byte chunk of packed codes is spread (a model of the kernel's permutes)."""
    rng = np.random.default_rng(bits)
    D = 1024 // bits
    x = rng.standard_normal((1, D)).astype(np.float32)
    packed, scales, zeros = kv_sym.quantize_tensor(x, bits, 64, "f32")
    words = np.frombuffer(np.asarray(packed, np.uint8).tobytes(), "<u4").astype(np.uint64)[: 4]

    def prmt(a, b, sel):
        src = [(int(a) >> (8 * i)) & 255 for i in range(4)] + [(int(b) >> (8 * i)) & 255 for i in range(4)]
        return sum(src[(sel >> (4 * i)) & 7] << (8 * i) for i in range(4))

    out = []
    for w in words:
        w = int(w)
        if bits == 8:
            out.append(w)
        elif bits == 4:
            hi, lo = (w >> 4) & 0x0F0F0F0F, w & 0x0F0F0F0F
            out += [prmt(hi, lo, 0x5140), prmt(hi, lo, 0x7362)]
        else:
            a, b, c, d = ((w >> s) & 0x03030303 for s in (6, 4, 2, 0))
            p, q, r, t = prmt(a, b, 0x5140), prmt(a, b, 0x7362), prmt(c, d, 0x5140), prmt(c, d, 0x7362)
            out += [prmt(p, r, 0x5410), prmt(p, r, 0x7632), prmt(q, t, 0x5410), prmt(q, t, 0x7632)]
    codes = np.frombuffer(np.array(out, "<u4").tobytes(), np.uint8).astype(np.float32)
    n = codes.size
    want = kv_sym.dequantize_tensor(packed, scales, zeros, bits, x.shape, 64)[0, :n]
    top = 2 ** (bits - 1) - 1
    got = (codes - top) * np.repeat(np.asarray(scales, np.float32)[0], 64)[:n]
    assert np.array_equal(got, want)
