"""Refusals and host logic of the drafted-token operators (tree attention, verification, kept rows): no GPU."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch


def _attn(B=1, HQ=4, HKV=2, T=3, D=64, cap=16, dtype=torch.float16):
    q = torch.zeros((B, HQ, T, D), dtype=dtype)
    kv = [torch.zeros((B, HKV, cap, D), dtype=dtype) for _ in range(3)]
    return q, kv


def test_tree_attention_refusals():
    from mlx_motif.kernels import sdpa_dual_v_tree, sdpa_dual_v_tree_q4

    q, kv = _attn()
    with pytest.raises(AssertionError, match="multiple of 32"):
        sdpa_dual_v_tree(torch.zeros(1, 4, 3, 40), *(torch.zeros(1, 2, 16, 40) for _ in range(3)), 0.1)
    with pytest.raises(AssertionError, match="multiple of H_kv"):
        sdpa_dual_v_tree(q[:, :3], *kv, 0.1)
    with pytest.raises(AssertionError, match="multiple of H_kv"):
        sdpa_dual_v_tree(q, *(t[:, :0] for t in kv), 0.1)
    with pytest.raises(AssertionError, match="must match"):
        sdpa_dual_v_tree(q, kv[0], kv[1][:, :, :8], kv[2], 0.1)
    with pytest.raises(AssertionError, match="1..256 tree rows"):
        sdpa_dual_v_tree(torch.zeros(1, 2, 257, 64), *(torch.zeros(1, 2, 300, 64) for _ in range(3)), 0.1)
    for n in (2, 17, -1):
        with pytest.raises(AssertionError, match="kv_len"):
            sdpa_dual_v_tree(q, *kv, 0.1, kv_len=n)
    with pytest.raises(TypeError, match="device kv_len"):
        sdpa_dual_v_tree(q, *kv, 0.1, kv_len=torch.tensor([3], dtype=torch.int32))  # on the CPU
    with pytest.raises(TypeError, match="bool"):
        sdpa_dual_v_tree(q, *kv, 0.1, tree_mask=torch.zeros(3, 3))
    with pytest.raises(AssertionError, match="tree_mask"):
        sdpa_dual_v_tree(q, *kv, 0.1, tree_mask=torch.ones(3, 4, dtype=torch.bool))
    with pytest.raises(TypeError, match="dtype"):
        sdpa_dual_v_tree(q.double(), *kv, 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        sdpa_dual_v_tree(q, *kv, 0.1)

    def triple(words, groups, dtype=torch.uint32):
        return (torch.zeros((1, 2, 16, words), dtype=torch.int32).view(dtype), *(torch.zeros(1, 2, 16, groups).half()
                                                                                 for _ in range(2)))

    good = triple(8, 1)
    with pytest.raises(AssertionError, match="packed D"):
        sdpa_dual_v_tree_q4(q, triple(4, 1), good, good, 0.1)
    with pytest.raises(AssertionError, match="bits"):
        sdpa_dual_v_tree_q4(q, good, good, good, 0.1, bits=3)
    with pytest.raises(AssertionError, match="group_size"):
        sdpa_dual_v_tree_q4(q, good, good, good, 0.1, group_size=48)
    with pytest.raises(AssertionError, match="scales"):
        sdpa_dual_v_tree_q4(q, good, good, triple(8, 2), 0.1)
    with pytest.raises(TypeError, match="uint32"):
        sdpa_dual_v_tree_q4(q, triple(8, 1, torch.float32), good, good, 0.1)


def test_tree_attention_abi_refusals():
    from mlx_motif import _native as N

    kv = N.motif_tree_kv()
    for i in range(3):
        kv.data[i] = 1 << 20
        kv.scales[i] = kv.biases[i] = 1 << 20
    kv.stride[0], kv.stride[1], kv.stride[2] = 2 * 64 * 128, 64 * 128, 128
    big = 1 << 30

    def call(dtype=0, bits=16, gs=64, q=1 << 20, kvp=C.byref(kv), B=1, HQ=4, HKV=2, T=3, cap=64, D=128, n=10, ws=1 << 20,
             wsb=big, y=1 << 20, n_step=0, mask=None, mask_b=0):
        return N.lib.motif_sdpa_dual_v_tree(dtype, bits, gs, q, kvp, mask, mask_b, 0.1, B, HQ, HKV, T, cap, D, n, None,
                                            n_step, y, ws, wsb, None, None)

    assert call(q=None) == N.ERR_NULL and call(y=None) == N.ERR_NULL and call(kvp=None) == N.ERR_NULL
    assert call(dtype=7) == N.ERR_DTYPE and call(bits=5) == N.ERR_DTYPE
    assert call(D=96) == N.ERR_BAD_CONTRACT and call(HQ=5) == N.ERR_BAD_CONTRACT and call(T=0) == N.ERR_BAD_CONTRACT
    assert call(T=257, n=300, cap=300) == N.ERR_BAD_CONTRACT
    assert call(n=2) == N.ERR_BAD_SHAPE and call(n=65) == N.ERR_BAD_SHAPE and call(B=0) == N.ERR_BAD_SHAPE
    assert call(cap=1 << 40) == N.ERR_BAD_SHAPE and call(mask=1, mask_b=4) == N.ERR_BAD_SHAPE
    assert call(q=(1 << 20) + 8) == N.ERR_BAD_CONTRACT and b"16-byte" in N.lib.motif_last_error()
    assert call(bits=4, gs=48) == N.ERR_BAD_CONTRACT and call(bits=4, gs=4) == N.ERR_BAD_CONTRACT
    long = dict(dtype=2, cap=4096, n=4096)  # parts that meet in the workspace
    assert call(wsb=64, **long) == N.ERR_WORKSPACE and call(ws=None, **long) == N.ERR_WORKSPACE
    kv.stride[2] = 130
    assert call() == N.ERR_BAD_CONTRACT and b"strides" in N.lib.motif_last_error()
    kv.stride[2] = 128
    kv.data[1] = None
    assert call() == N.ERR_NULL


def test_verify_refusals():
    from mlx_motif.kernels import speculative_verify

    B, T, V = 2, 3, 10
    tok, par = torch.zeros((B, T), dtype=torch.int32), torch.zeros((B, T), dtype=torch.int32)
    p, q, u = torch.zeros(B, T, V), torch.zeros(B, T, V), torch.zeros(B, T)
    with pytest.raises(AssertionError, match="tokens"):
        speculative_verify(tok[:, :2], par, p, q, u, 1.0)
    with pytest.raises(AssertionError, match="parents"):
        speculative_verify(tok, par[:1], p, q, u, 1.0)
    with pytest.raises(AssertionError, match="p_logits"):
        speculative_verify(tok, par, p[0], q, u, 1.0)
    with pytest.raises(AssertionError, match="q_logits"):
        speculative_verify(tok, par, p, q[:, :, :9], u, 1.0)
    with pytest.raises(AssertionError, match="q_logits"):
        speculative_verify(tok, par, p, torch.zeros(B, 4, V), u, 1.0)
    with pytest.raises(AssertionError, match="needed"):
        speculative_verify(tok, par, p, None, u, 1.0)
    with pytest.raises(AssertionError, match="uniforms"):
        speculative_verify(tok, par, p, q, u[:, :2], 1.0)
    for bad in (-0.5, float("nan"), float("inf"), 1e-9, 1e9):
        with pytest.raises(AssertionError, match="temperature"):
            speculative_verify(tok, par, p, q, u, bad)
    with pytest.raises(TypeError, match="int32"):
        speculative_verify(tok.long(), par, p, q, u, 1.0)
    with pytest.raises(TypeError, match="float32"):
        speculative_verify(tok, par, p, q, u.double(), 1.0)
    with pytest.raises(TypeError, match="one type"):
        speculative_verify(tok, par, p, q.half(), u, 1.0)
    with pytest.raises(TypeError, match="dtype"):
        speculative_verify(tok, par, p.double(), q.double(), u, 1.0)
    with pytest.raises(ValueError, match="CUDA"):
        speculative_verify(tok, par, p, q, u, 1.0)


def test_verify_abi_refusals():
    from mlx_motif import _native as N

    def call(dtype=0, p=1, q=1, u=1, R=2, B=1, T=2, V=8, temp=0.7, par_b=0, ws=1 << 20, wsb=1 << 40, out=1):
        return N.lib.motif_speculative_verify(dtype, p, 16, 8, q, 16, 8, R, 1, 1, par_b, u, B, T, V, temp, out, 1, 1, ws,
                                              wsb, None)

    assert call(p=None) == N.ERR_NULL and call(q=None) == N.ERR_NULL and call(u=None) == N.ERR_NULL
    assert call(out=None) == N.ERR_NULL
    assert call(V=1 << 30) == N.ERR_BAD_SHAPE and call(temp=1e-7) == N.ERR_BAD_CONTRACT
    assert call(temp=-1.0) == N.ERR_BAD_CONTRACT and call(temp=float("nan")) == N.ERR_BAD_CONTRACT
    assert call(R=3) == N.ERR_BAD_SHAPE and call(T=0) == N.ERR_BAD_SHAPE and call(T=1025) == N.ERR_BAD_SHAPE
    assert call(V=0) == N.ERR_BAD_SHAPE and call(par_b=1) == N.ERR_BAD_SHAPE
    assert call(ws=None) == N.ERR_WORKSPACE and call(wsb=0) == N.ERR_WORKSPACE
    assert call(dtype=9) == N.ERR_DTYPE


def test_verify_reference_follows_the_targets_law():
    """The 64-bit rule itself: over many draws the first emitted token of a two-child tree is distributed as
    the target's law, whatever the draft (tolerance: 5 standard deviations of a frequency, 5·sqrt(1/4n))."""
    from mlx_motif.kernels import speculative_verify_reference

    g = torch.Generator().manual_seed(0)
    V, n = 5, 4000
    p = torch.randn((1, 3, V), generator=g)
    q = torch.randn((1, 1, V), generator=g)
    law_q = torch.softmax(q[0, 0].double(), -1)
    counts = torch.zeros(V)
    par = torch.tensor([-1, 0, 0], dtype=torch.int32)
    for _ in range(n):
        kids = torch.multinomial(law_q, 2, replacement=True, generator=g).int()
        tok = torch.cat([torch.zeros(1, dtype=torch.int32), kids])[None]
        r = speculative_verify_reference(tok, par, p, q, torch.rand((1, 3), generator=g), 1.0)
        first = int(tok[0, r.path[0, 1]]) if int(r.accepted[0]) else int(r.next_token[0])
        counts[first] += 1
    want = torch.softmax(p[0, 0].double(), -1)
    assert (counts / n - want).abs().max() < 5 * (0.25 / n) ** 0.5


def test_tree_mask_from_parents():
    from mlx_motif.kernels import tree_mask_from_parents

    rng = np.random.default_rng(0)
    for T in (1, 2, 7, 64):
        par = [-1] + [int(rng.integers(0, i)) for i in range(1, T)]
        want = np.zeros((T, T), dtype=bool)
        for i in range(T):
            j = i
            while j >= 0:
                want[i, j] = True
                j = par[j]
        got = tree_mask_from_parents(torch.tensor(par, dtype=torch.int32))
        assert got.dtype == torch.bool and (got.numpy() == want).all()
    chain = tree_mask_from_parents(torch.arange(-1, 255, dtype=torch.int32))  # as deep as it is long
    assert (chain == torch.ones(256, 256).tril().bool()).all()


def test_keep_rows_refusals():
    from mlx_motif.cache import KVCache, MotifGroupedKVCache, MotifGroupedQuantizedKVCache, keep_rows, kv_slots

    from mlx_motif import _native as N

    with pytest.raises(ValueError, match="no caches"):
        kv_slots([])
    with pytest.raises(ValueError, match="empty"):
        kv_slots([MotifGroupedKVCache()])
    with pytest.raises(ValueError, match="empty"):
        kv_slots([KVCache()])
    with pytest.raises(ValueError, match="empty"):
        kv_slots([MotifGroupedQuantizedKVCache()])

    def on_host(cls, names):
        c = cls()
        for name in names:
            setattr(c, name, torch.zeros(1, 2, 256, 64, dtype=torch.float16))
        return c

    four, stock = on_host(MotifGroupedKVCache, ("k1", "k2", "v1", "v2")), on_host(KVCache, ("keys", "values"))
    with pytest.raises(ValueError, match="twice"):  # its rows would be moved twice
        kv_slots([four, on_host(MotifGroupedKVCache, ("k1", "k2", "v1", "v2")), four])
    four.v2 = four.k2
    with pytest.raises(ValueError, match="twice"):
        kv_slots([four])
    with pytest.raises(ValueError, match="stock"):
        kv_slots([on_host(MotifGroupedKVCache, ("k1", "k2", "v1", "v2")), stock])

    structs = (N.motif_kv4_slots * 2)()
    for s in structs:
        for i in range(4):
            s.data[i] = s.scales[i] = s.biases[i] = 1 << 20
        s.bits, s.group_size, s.batch, s.heads, s.capacity, s.head_dim = 16, 64, 1, 2, 64, 128

    def call(n=2, path=1, T=4, path_b=4, base=0, limit=64, base_step=0, base_dev=None, dtype=0):
        return N.lib.motif_kv4_keep_rows(dtype, structs, n, path, path_b, 1, T, base, base_dev, base_step, limit, None)

    assert call(path=None) == N.ERR_NULL and call(n=0) == N.ERR_BAD_SHAPE and call(dtype=5) == N.ERR_DTYPE
    assert call(base=61) == N.ERR_BAD_SHAPE and call(base=-1) == N.ERR_BAD_SHAPE and call(T=0) == N.ERR_BAD_SHAPE
    assert call(limit=65) == N.ERR_BAD_SHAPE and call(path_b=3) == N.ERR_BAD_SHAPE
    assert call(base_dev=1, base_step=2) == N.ERR_BAD_SHAPE
    structs[1].heads = 3
    assert call() == N.ERR_BAD_SHAPE and b"differs" in N.lib.motif_last_error()
    structs[1].heads = 2
    structs[1].data[3] = None
    assert call() == N.ERR_NULL
    structs[1].data[3] = (1 << 20) + 1
    assert call() == N.ERR_BAD_CONTRACT and b"misaligned" in N.lib.motif_last_error()
