"""Tree attention where one CTA runs through several units (a line of key tiles cut over the SMs): per-sequence
lengths and many short units. Each unit's output has to be read from tensor memory before the next unit's first
product replaces it, by the warps with rows and those without. The 64-bit form and the tolerances are
``test_gpu_tree.py``'s.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_tree import DT, attention64, call, check, make, masks, unpack64

pytestmark = pytest.mark.gpu

TYPES = [("fp16", 16, 64), ("bf16", 16, 64), ("fp16", 4, 64), ("bf16", 4, 32), ("fp16", 8, 64), ("bf16", 8, 64)]


def lengths(kind, B, T, cap, rng):
    """Per-sequence lengths. "mixed": units of one tile between units of 16 to 32; "short": one or two tiles."""
    if kind == "mixed":
        return [int(rng.integers(T, 65)) if b % 2 else int(rng.integers(1000, cap + 1)) for b in range(B)]
    return [int(rng.integers(T, min(cap, 110))) for _ in range(B)]


def repeats(q, kv, bits, gs, **kw):
    """One result, the same in ten calls in a row."""
    got = call(q, kv, bits, gs, 0.09, **kw)
    for _ in range(9):
        assert torch.equal(got.nan_to_num(), call(q, kv, bits, gs, 0.09, **kw).nan_to_num())
    return got


@pytest.mark.parametrize("dtype,bits,gs", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,HQ,HKV,T,cap,kind", [
    (32, 24, 8, 5, 2000, "mixed"),  # 15 rows a unit: one warp of a softmax group has rows, some 20 tiles a CTA
    (16, 24, 8, 43, 2000, "mixed"),  # 129 rows: every second unit has a single row
    (160, 16, 8, 9, 112, "short"),  # units of one or two tiles, whole units between two others
])
def test_line_of_units(cuda, B, HQ, HKV, T, cap, kind, D, dtype, bits, gs):
    rng = np.random.default_rng(B + T)
    lens = lengths(kind, B, T, cap, rng)
    q, kv, plain = make(B + D, B, HQ, HKV, T, D, cap, dtype, bits, gs)
    m, m64 = masks("trees", B, T)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = repeats(q, kv, bits, gs, kv_len=n, tree_mask=m)
    want, tol = attention64(q, *plain, 0.09, lens, m64, torch.finfo(DT[dtype]).eps / 2, bits != 16)
    check(got, want, tol, dtype)


@pytest.mark.parametrize("dtype,bits,gs", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_line_of_one_tile_units(cuda, D, dtype, bits, gs):
    """One length on the host, more units than SMs: fourteen segments of one tile in a CTA."""
    B, HQ, HKV, T, cap, n = 256, 16, 8, 3, 64, 41
    q, kv, plain = make(D, B, HQ, HKV, T, D, cap, dtype, bits, gs)
    got = repeats(q, kv, bits, gs, kv_len=n)
    m64 = torch.ones((B, T, T)).tril().bool()
    want, tol = attention64(q, *plain, 0.09, [n] * B, m64, torch.finfo(DT[dtype]).eps / 2, bits != 16)
    check(got, want, tol, dtype)


@pytest.mark.parametrize("dtype,bits,gs", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("B,cap,kind", [(32, 2000, "mixed"), (160, 112, "short")])  # one to three units a CTA, or nine
def test_line_with_broken_drafted_rows(cuda, B, cap, kind, dtype, bits, gs, bad):
    """Every third sequence has one drafted row of NaN or infinities, and all rows behind the last are: the
    records of cleared rows are used again by later units of a CTA, and no other row is touched."""
    HQ, HKV, T, D = 24, 8, 5, 128
    rng = np.random.default_rng(7)
    lens = lengths(kind, B, T, cap, rng)
    q, kv, plain = make(11, B, HQ, HKV, T, D, cap, dtype, bits, gs)
    m, m64 = masks("trees", B, T)
    broken = {b: int(rng.integers(1, T)) for b in range(0, B, 3)}
    for s, t in enumerate(kv):
        for part in ((t,) if bits == 16 else t[1:]):
            for b, n in enumerate(lens):
                part[b, :, n:] = bad
                if b in broken and s:  # V1 and V2: the row's score is finite
                    part[b, :, n - T + broken[b]] = bad
    if bits != 16:
        plain = [unpack64(t, bits, gs) for t in kv]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = repeats(q, kv, bits, gs, kv_len=n, tree_mask=m)
    sees = torch.zeros((B, 1, T, 1), dtype=torch.bool)
    for b, j in broken.items():
        sees[b, 0, :, 0] = m64[b][:, j]
    sees = sees.cuda().expand(got.shape)
    safe = [torch.where(torch.isfinite(p.double()), p.double(), 0.0) for p in plain]
    want, tol = attention64(q, *safe, 0.09, lens, m64, torch.finfo(DT[dtype]).eps / 2, bits != 16)
    assert not torch.isfinite(got[sees]).any()
    check(torch.where(sees, 0.0, got), torch.where(sees, 0.0, want), tol, dtype)


def test_a_timed_out_wait_is_raised_by_the_next_call(cuda, monkeypatch):
    """The failure is made on the host: the library call sets the error word that it was given, as a kernel does
    whose wait ran out. The next call raises, the one after that is served; captured calls carry the word too."""
    import ctypes

    from mlx_motif.kernels import tree

    q, kv, _ = make(0, 1, 4, 2, 3, 64, 64, "fp16")
    want = call(q, kv, 16, 64, 0.1)
    words = []

    class Lib:
        def motif_sdpa_dual_v_tree(self, *args):
            rc = real.motif_sdpa_dual_v_tree(*args)
            words.append(args[-2])
            ctypes.c_int32.from_address(args[-2]).value = 1
            return rc

        def __getattr__(self, name):
            return getattr(real, name)

    real = tree.lib
    with monkeypatch.context() as m:
        m.setattr(tree, "lib", Lib())
        call(q, kv, 16, 64, 0.1)
    with pytest.raises(RuntimeError, match="timed out"):
        call(q, kv, 16, 64, 0.1)
    assert torch.equal(call(q, kv, 16, 64, 0.1), want)
    g = torch.cuda.CUDAGraph()
    with monkeypatch.context() as m, torch.cuda.graph(g):
        m.setattr(tree, "lib", Lib())
        call(q, kv, 16, 64, 0.1)
    assert words[0] == words[1]
    with pytest.raises(RuntimeError, match="timed out"):
        call(q, kv, 16, 64, 0.1)
    g.replay()
    assert torch.equal(call(q, kv, 16, 64, 0.1), want)


def test_first_call_under_capture(cuda):
    """In a fresh process, the device's first call inside a capture."""
    import os
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from test_gpu_tree import call, make
q, kv, _ = make(0, 1, 4, 2, 3, 64, 64, "fp16")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = call(q, kv, 16, 64, 0.1)
g.replay()
assert torch.equal(y, call(q, kv, 16, 64, 0.1))
"""
    here = Path(__file__).resolve().parent
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(here), str(here.parent / "mlx-motif_b200"), str(here.parent)]))
    subprocess.run([sys.executable, "-c", code], check=True, env=env, timeout=300)
