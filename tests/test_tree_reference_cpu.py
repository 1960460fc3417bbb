"""The torch composition of the tree attention (``MLX_MOTIF_DISABLE_KERNELS=1``): no GPU."""

from __future__ import annotations

import math

import pytest
import torch


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_reference_keeps_hidden_rows_from_a_query(bad):
    """A drafted row that holds NaN or infinities reaches the queries that see it and no other; rows behind the last
    live one reach none. Tolerance: fp32 sums of 40 weights, (40 + 2·16)·2^-24 of A + |o| < 8, against 64 bits."""
    from mlx_motif.kernels import sdpa_dual_v_tree_reference

    g = torch.Generator().manual_seed(0)
    B, HQ, HKV, T, D, cap, n = 2, 4, 2, 4, 16, 48, 40
    q = torch.randn((B, HQ, T, D), generator=g)
    k, v1, v2 = (torch.randn((B, HKV, cap, D), generator=g) for _ in range(3))
    mask = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 1, 0, 1]], dtype=torch.bool)
    clean = [t.clone() for t in (k, v1, v2)]
    for t in (k, v1, v2):
        t[:, :, n:] = bad
    v1[:, :, n - T + 1] = bad  # row 1: seen by rows 1 and 3
    v2[:, :, n - T + 1, 3] = bad
    k[:, :, n - T + 2] = bad  # row 2: seen by itself
    got = sdpa_dual_v_tree_reference(q, k, v1, v2, 0.25, n, mask)
    want = torch.empty((B, HQ, T, 2 * D), dtype=torch.float64)
    for h in range(HQ):
        for t in range(T):
            rows = torch.cat([torch.ones(n - T, dtype=torch.bool), mask[t]])
            kk, a, c = (x[:, h // 2, :n][:, rows].double() for x in clean)
            p = torch.softmax(torch.einsum("bd,bcd->bc", q[:, h, t].double(), kk) * 0.25, -1)
            want[:, h, t] = torch.einsum("bc,bcd->bd", p, torch.cat([a, c], -1))
    tol = 72 * 2.0**-24 * 8
    assert (got[:, :, 0].double() - want[:, :, 0]).abs().max() < tol  # sees neither
    for t in (1, 3):
        assert not torch.isfinite(got[:, :, t, :D]).any() and not torch.isfinite(got[:, :, t, D + 3]).any()
        keep = [c for c in range(D, 2 * D) if c != D + 3]
        assert (got[:, :, t, keep].double() - want[:, :, t, keep]).abs().max() < tol
    if not math.isinf(bad):
        assert torch.isnan(got[:, :, 2]).all()
