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


def test_long_caches_and_many_units_stay_within_32_bits():
    """The kernels place key tiles in 32 bits: 296 parts of 2^24 tiles would pass 2^32 and run as a line (two
    partials a CTA of 64-channel fp32 rows) instead; a line of 2.3·10^9 places is refused before any launch."""
    import ctypes as C

    from mlx_motif import _native as N

    line = 2 * 296 * (2 * 64 + 2) * 4
    one = dict(dtype=2, HQ=1, HKV=1, T=1, D=64)
    assert workspace_bytes(cap=(1 << 30) - 1, **one) == line and workspace_bytes(cap=1 << 29, **one) == line
    assert workspace_bytes(cap=1 << 28, **one) == line // 2  # 296 equal parts
    kv = N.motif_tree_kv()
    for i in range(3):
        kv.data[i] = 1 << 20
    kv.stride[0], kv.stride[1], kv.stride[2] = 256 * 64, 64, 64

    def call(B, HKV):
        return N.lib.motif_sdpa_dual_v_tree(0, 16, 64, 1 << 20, C.byref(kv), None, 0, 0.1, B, HKV, HKV, 1, 1, 64, 1, None, 0,
                                            1 << 20, None, 0, None, None)

    assert call(1000000, 256) == N.ERR_BAD_SHAPE and b"key tiles" in N.lib.motif_last_error()
    assert call(900000, 256) == N.ERR_WORKSPACE  # 2.1·10^9 places
