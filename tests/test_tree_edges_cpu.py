"""Host logic of the tree attention at the edges of its sizes: no GPU."""

from __future__ import annotations

import pytest


def workspace_bytes(dtype=0, bits=16, gs=64, B=1, HQ=4, HKV=2, T=3, cap=4096, D=128, bound=None, one_length=1):
    from mlx_motif import _native as N

    return N.lib.motif_sdpa_dual_v_tree_workspace_bytes(dtype, bits, gs, B, HQ, HKV, T, cap, D,
                                                        cap if bound is None else bound, one_length)


@pytest.mark.parametrize("sizes", [
    dict(HQ=1, HKV=2),  # fewer query heads than kv heads: no row, no unit of work
    dict(HQ=3), dict(HQ=0), dict(HKV=0), dict(T=0), dict(T=257), dict(D=0), dict(D=256), dict(B=0), dict(cap=0), dict(gs=0),
    dict(B=1 << 62), dict(HQ=1 << 62, HKV=1 << 61), dict(cap=1 << 62), dict(B=1 << 20), dict(cap=1 << 30),
])
def test_workspace_of_refused_sizes_is_none(sizes):
    assert workspace_bytes(**sizes) == 0


def test_workspace_of_a_length_beyond_the_capacity():
    assert workspace_bytes(bound=1 << 40) == workspace_bytes() > 0
    assert workspace_bytes(bound=-5) == workspace_bytes(bound=0) == workspace_bytes(bound=1)
