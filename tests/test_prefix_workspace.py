"""Workspace of the shared-prefix attention: bounded by the requests, however many prefixes are kept beside them."""

import pytest

from b200flash import _capi


def size(B, groups, Hkv=8):
    return int(_capi.lib().b2f_shared_prefix_attn_workspace_bytes(B, 32, Hkv, 128, groups, 20_000, 1000))


@pytest.mark.parametrize("B", [1, 4, 70])
def test_prefixes_without_requests_take_no_workspace(B):
    assert size(B, 60_000) == size(B, B) < 600 * (1 << 20)


def test_workspace_holds_a_pair_of_tiles_per_group():
    # 32 query heads over 8: 32 requests a tile; groups of 1, 64, 65 and 70 rows have 1 + 1 + 2 + 2 pairs
    B, pairs = 200, 6
    rows = max(148, pairs * 8) * 256
    assert size(B, 4) >= rows * (128 + 2) * 4
