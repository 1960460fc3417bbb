"""``speculative_verify`` at the edges of its kernels, against the 64-bit rule (``speculative_verify_reference``):
whole numbers, which have to be equal. The drafts are ``test_gpu_tree.py``'s.
"""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

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


LOWEST = {"fp32": torch.finfo(torch.float32).min, "bf16": float(torch.finfo(torch.bfloat16).min), "fp16": -65504.0}


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("temp", [1e-6, 0.3, 0.5, 0.7, 1.0, 1.3, 50.0, 1e6])
@pytest.mark.parametrize("V", [300, 40000])
def test_rows_of_very_large_logits(cuda, dtype, temp, V):
    """A row of the type's lowest value throughout is the uniform law; maxima of ±1e20 (16-bit types: near their
    ends) are one token's or share the law; the residual of such rows."""
    from mlx_motif.kernels import speculative_verify_reference

    B, T = 6, 3
    tok, par, p, q, u = drafts(V, B, T, V, dtype, tree=False)
    low, big = LOWEST[dtype], {"fp32": 1e20, "bf16": 1e20, "fp16": 60000.0}[dtype]
    p[0, 0] = low
    q[1] = low
    p[2], q[2] = low, low
    p[3, 0, 7], p[3, 1, [11, 250]] = big, big
    q[3, 0, 7] = big
    p[4] -= big
    q[4] -= big
    p[5], q[5] = p[5] + big, q[5] + big
    p[5, 0, ::3] = low
    want = speculative_verify_reference(tok, par, p, q, u, temp)
    same(verify(tok, par, p, q, u, temp), want)
    alone = [t[:1, :1].contiguous() for t in (tok, par, p, q, u)]  # the draw alone
    for x in (0.0, 0.25, 0.5, 0.999):
        alone[4].fill_(x)
        r = verify(*alone, temp)
        assert r.next_token.item() == int(x * V), (x, r.next_token.item())


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("V", [5, 300, 4097, 70000])  # within a warp's range, one CTA, several
def test_draws_at_the_ends(cuda, dtype, V):
    """u_0 of 1, or beyond, draws the last token with weight, 0 the first one; with the law's ends masked, after
    rejections too."""
    from mlx_motif.kernels import speculative_verify_reference

    B, T = 4, 3
    tok, _, p, q, u = drafts(V, B, T, V, dtype, tree=False, apart=2.0)
    par = torch.tensor([-1, 0, 0], dtype=torch.int32)
    q = q[:, :1].contiguous()
    g = torch.Generator().manual_seed(V)
    tok[:, 1:] = torch.multinomial(torch.softmax(q[:, 0].double(), -1), 2, replacement=True, generator=g).int()
    p[1, :, -(V // 3) - 1 :] = -float("inf")
    p[2, :, : V // 2] = -float("inf")
    for u0 in (1.0, 1.5, 1.0 - 2.0**-24, 0.0):
        for rest in (0.0, 0.5, 1.0):
            u.fill_(rest)
            u[:, 0] = u0
            want = speculative_verify_reference(tok, par, p, q, u, 0.9)
            same(verify(tok, par, p, q, u, 0.9), want)
            if u0 >= 1.0 and want.accepted[1]:
                assert want.next_token[1] == V - V // 3 - 2


@pytest.mark.parametrize("temp", [0.7, 1.0])
@pytest.mark.parametrize("V", [50, 40000])
def test_drafts_of_tiny_probability(cuda, temp, V):
    """Drafted tokens whose probabilities leave the 32-bit range (2^-126) in one row or both: accepted or not by
    their quotient."""
    from mlx_motif.kernels import speculative_verify_reference

    B, T = 24, 2
    g = torch.Generator().manual_seed(V)
    p, q = torch.randn((B, T, V), generator=g), torch.randn((B, 1, V), generator=g)
    p[:, :, 0], q[:, :, 0] = 20.0, 20.0
    tok = torch.full((B, T), 7, dtype=torch.int32)
    par = torch.tensor([-1, 0], dtype=torch.int32)
    ln2 = 0.6931471805599453
    u = torch.empty((B, T)).fill_(0.3)
    for b in range(B):
        at = -120.0 - b % 12  # log2 of the draft's probability, about; the target's is 0.8 or 3 below it
        q[b, 0, 7] = 20.0 + at * ln2 * temp
        p[b, 0, 7] = 20.0 + (at - (0.8 if b < 12 else 3.0)) * ln2 * temp
    want = speculative_verify_reference(tok, par, p, q, u, temp)
    assert want.accepted.tolist() == [1] * 12 + [0] * 12
    same(verify(tok, par, p, q, u, temp), want)


def test_a_small_call_says_nothing_about_a_large_one(cuda):
    """In a fresh process: a vocabulary whose clusters share SMs, then one whose CTAs take an SM's shared memory."""
    code = """
import torch
from test_gpu_tree import drafts, same, verify
from mlx_motif.kernels import speculative_verify_reference
for V in (32768, 219520, 32768):
    for dtype in ("fp16", "fp32"):
        args = drafts(V, 1, 4, V, dtype, tree=False)
        same(verify(*args, 0.7), speculative_verify_reference(*args, 0.7))
"""
    here = Path(__file__).resolve().parent
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(here), str(here.parent / "mlx-motif_b200"), str(here.parent)]))
    subprocess.run([sys.executable, "-c", code], check=True, env=env, timeout=300)


@pytest.mark.parametrize("B,T,V,tree,dtype", [
    (9, 3, 219520, False, "fp16"),  # nine sequences: clusters of 8, more than shared memory holds
    (1, 4, 256000, False, "bf16"),  # one CTA's sixteenth of the vocabulary does not fit
    (1, 300, 219520, True, "fp16"),  # the rows' records leave no room
    (2, 5, 500001, True, "fp32"),
])
@pytest.mark.parametrize("temp", [0.7, 1.0])
def test_walks_without_kept_exponentials(cuda, B, T, V, tree, dtype, temp):
    """Vocabularies whose exponentials do not fit the cluster's shared memory: every sweep computes them again."""
    from mlx_motif.kernels import speculative_verify_reference

    args = drafts(B + T, B, T, V, dtype, tree, apart=1.5)
    want = speculative_verify_reference(*args, temp)
    same(verify(*args, temp), want)
    hard = args[4].clone().fill_(0.999)  # rejections at every row
    same(verify(*args[:4], hard, temp), speculative_verify_reference(*args[:4], hard, temp))
