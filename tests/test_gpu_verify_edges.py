"""``speculative_verify`` at the edges of its kernels, against the 64-bit rule (``speculative_verify_reference``):
whole numbers, which have to be equal. The drafts are ``test_gpu_tree.py``'s.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_tree import drafts, same, verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [4096, 8200, 16500, 33000, 70000])  # clusters of 1, 2, 4, 8 and 16 CTAs
@pytest.mark.parametrize("T", [1, 2])
def test_walks_in_a_row(cuda, V, T):
    """Few rows, so that little stands between a CTA's start and the first exchange of sums: calls back to back,
    each the same."""
    from mlx_motif.kernels import speculative_verify, speculative_verify_reference

    args = drafts(V + T, 1, T, V, "fp16", tree=False, apart=4.0)
    want = speculative_verify_reference(*args, 0.8)
    dev = [t.cuda() for t in args]
    got = [speculative_verify(*dev, 0.8) for _ in range(100)]
    for r in got:
        same(r, want)
