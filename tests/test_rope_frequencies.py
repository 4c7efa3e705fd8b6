"""The rotary frequencies that ``qk_norm_rope`` keeps: kernels in flight and captured graphs hold their addresses, so a
tensor that was handed out stays."""

import torch

from b200flash.paged_prompt import rope_frequencies


def test_frequencies_are_kept():
    cpu = torch.device("cpu")
    first = rope_frequencies(64, 123.5, cpu)
    for i in range(200):
        rope_frequencies(64, 1000.0 + i, cpu)
    assert rope_frequencies(64, 123.5, cpu) is first
    assert first.tolist() == [123.5 ** (-2.0 * i / 64) for i in range(32)]
    assert rope_frequencies(32, 123.5, cpu).shape == (16,)
