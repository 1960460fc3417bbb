"""The drafted-token operators on the GPU against plain 64-bit forms: tree attention over fp16 / bf16 / fp32
and packed caches, verification from given uniforms, the moved rows of the cache, and a run of the three.

Tolerances of the attention, per output element, with h = eps/2 of the type (half a rounding step),
A = Σ_c p_c·|v_c| and X = max_c scale·Σ_d |q_d·k_cd| of the query row, all in 64 bits:

* the result's own rounding: h·|o|;
* 16-bit types round every weight p_c once, the same rounded weights being summed: o moves by
  |Σ δ_c·p_c·(v_c − o)| ≤ h·(A + |o|), |δ_c| ≤ h;
* packed caches round the rebuilt K and V once to the type: the scores move by at most h·X, so the weights
  by a factor e^(±2hX) against their sum, o by (e^(2hX) − 1)·(A + |o|), and V's rounding adds h·A;
* fp32 sums: a score of D terms errs by at most (D + 8)·2^-24·X (products exact in fp32 for 16-bit inputs, so
  this holds for every type), exp2 by 2^-22 relative, sums over n weights by n·2^-24 relative, each of them
  entering twice (sum and normaliser): 2·((D + 8)·2^-24·X + 2^-21 + n·2^-24)·(A + |o|). Rebasing the maximum
  and joining parts rounds each part a few times more: 64·2^-24·A covers it.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def random_tree(T, rng, width=4):
    return [-1] + [0 if i <= width else int(rng.integers(max(0, i - 8), i)) for i in range(1, T)]


def ancestors(parents):
    m = np.zeros((len(parents), len(parents)), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return torch.from_numpy(m)


def unpack64(triple, bits, gs):
    w, s, b = triple
    w = w.view(torch.int32).long()
    q = torch.stack([(w >> (bits * j)) & (2**bits - 1) for j in range(32 // bits)], -1).flatten(-2)
    return q.double() * s.double().repeat_interleave(gs, -1) + b.double().repeat_interleave(gs, -1)


def attention64(q, k, v1, v2, scale, lens, mask, h, packed, chunk=64):
    """(o, tolerance) in 64 bits, a head at a time; k, v1, v2 are 64-bit or the caller's rows."""
    B, HQ, T, D = q.shape
    gqa = HQ // k.shape[1]
    out = torch.zeros((B, HQ, T, 2 * D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = lens[b]
        first = n - T
        see = torch.zeros((T, n), dtype=torch.bool, device=q.device)
        see[:, : max(first, 0)] = True
        lo = max(first, 0)
        m = mask[b].to(q.device)
        see[:, lo:n] = m[:, lo - first : n - first]
        for x in range(HQ):
            kk, a, c = (t[b, x // gqa, :n].double() for t in (k, v1, v2))
            if n == 0:
                continue
            vis = see.any(0)  # a row nobody sees may hold anything
            kk, a, c = (torch.where(vis[:, None], t, 0.0) for t in (kk, a, c))
            vv = torch.cat([a, c], -1)
            qq = q[b, x].double()
            # a hidden row must not reach a query: the product over visible rows only, row by row where rows differ
            s = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            den = p.sum(-1, keepdim=True)
            p = p / torch.where(den == 0, 1.0, den)
            o = torch.empty((T, 2 * D), dtype=torch.float64, device=q.device)
            A = torch.empty_like(o)
            for t in range(T):
                if bool(torch.isfinite(vv).all()):
                    o, A = p @ vv, p @ vv.abs()
                    break
                rows = see[t]
                o[t], A[t] = p[t, rows] @ vv[rows], p[t, rows] @ vv[rows].abs()
            X = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~see, 0.0).amax(-1, keepdim=True)
            e = 2 * ((D + 8) * 2.0**-24 * X + 2.0**-21 + n * 2.0**-24)
            t_ = h * o.abs() + e * (A + o.abs()) + 64 * 2.0**-24 * A
            if h > 1e-6:
                t_ = t_ + h * (A + o.abs())
                if packed:
                    t_ = t_ + torch.expm1(2 * h * X) * (A + o.abs()) + h * A
            out[b, x], tol[b, x] = o, t_ + 1e-30
    return out, tol


def check(got, want, tol, dtype, what=""):
    tiny = {"fp16": 2.0**-25, "bf16": 0.0, "fp32": 0.0}[dtype]  # half the smallest fp16 step
    err = (got.double() - want).abs()
    bad = ~(err <= tol + tiny) & ~(torch.isnan(want) & torch.isnan(got))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).nan_to_num().max()):.2f} x its tolerance"


def make(seed, B, HQ, HKV, T, D, cap, dtype, bits=16, gs=64):
    from mlx_motif.quantization import quantize

    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(s, generator=g, device="cuda")

    q = randn(B, HQ, T, D).to(DT[dtype])
    rows = [(randn(B, HKV, cap, D) * s).to(DT[dtype]) for s in (1.0, 0.5, 0.5)]
    if bits == 16:
        return q, rows, rows
    packed = [quantize(r, gs, bits) for r in rows]
    return q, packed, [unpack64(t, bits, gs) for t in packed]


def masks(kind, B, T, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "causal":
        return None, torch.ones((B, T, T)).tril().bool()
    if kind == "tree":
        m = ancestors(random_tree(T, rng))
        return m.cuda(), m.expand(B, T, T)
    if kind == "trees":
        m = torch.stack([ancestors(random_tree(T, rng)) for _ in range(B)])
        return m.cuda(), m
    m = torch.from_numpy(rng.random((B, T, T)) < 0.3)  # no tree: any pattern
    m[:, 0] = False  # a row without a drafted row
    return m.cuda(), m


def call(q, kv, bits, gs, scale, **kw):
    from mlx_motif.kernels import sdpa_dual_v_tree, sdpa_dual_v_tree_q4

    if bits == 16:
        return sdpa_dual_v_tree(q, *kv, scale, **kw)
    return sdpa_dual_v_tree_q4(q, *kv, scale, group_size=gs, bits=bits, **kw)


CASES = [
    # B, HQ, HKV, T, D, cap, n, mask
    (1, 3, 1, 1, 128, 1, 1, "causal"),  # one row, one key
    (1, 4, 4, 1, 64, 64, 64, "causal"),
    (1, 2, 2, 2, 128, 256, 2, "tree"),  # the tree is all there is
    (1, 2, 1, 5, 64, 256, 5, "any"),  # and its row 0 sees nothing
    (1, 6, 2, 5, 128, 256, 169, "causal"),
    (2, 8, 4, 7, 64, 100, 63, "trees"),  # lengths around the tiles' edges, odd capacities
    (2, 4, 2, 3, 128, 77, 65, "tree"),
    (1, 2, 2, 9, 128, 128, 127, "any"),
    (1, 4, 2, 4, 128, 192, 129, "trees"),
    (1, 8, 1, 17, 64, 128, 128, "tree"),
    (1, 3, 1, 43, 128, 520, 517, "trees"),  # 129 packed rows
    (1, 8, 1, 64, 128, 1024, 1000, "tree"),  # 512 packed rows
    (1, 2, 1, 256, 64, 300, 300, "any"),  # the largest tree, over more than two tiles
    (3, 24, 8, 6, 128, 2304, 2200, "trees"),
    (4, 24, 8, 43, 128, 1024, 1000, "trees"),  # several units per SM, each second one with a single row
    (5, 6, 2, 22, 64, 4096, 4001, "tree"),
]


@pytest.mark.parametrize("B,HQ,HKV,T,D,cap,n,mask", CASES)
@pytest.mark.parametrize("dtype,bits,gs", [("fp16", 16, 64), ("bf16", 16, 64), ("fp32", 16, 64), ("fp16", 4, 64),
                                           ("fp16", 4, 32), ("bf16", 4, 64), ("fp16", 8, 64), ("bf16", 8, 32),
                                           ("fp32", 4, 64)])
def test_tree_attention(cuda, B, HQ, HKV, T, D, cap, n, mask, dtype, bits, gs):
    q, kv, plain = make(n, B, HQ, HKV, T, D, cap, dtype, bits, gs)
    m, m64 = masks(mask, B, T)
    scale = D**-0.5
    got = call(q, kv, bits, gs, scale, kv_len=n, tree_mask=m)
    assert got.shape == (B, HQ, T, 2 * D) and got.dtype == q.dtype
    want, tol = attention64(q, *plain, scale, [n] * B, m64, torch.finfo(DT[dtype]).eps / 2, bits != 16)
    check(got, want, tol, dtype)
    assert torch.equal(got, call(q, kv, bits, gs, scale, kv_len=n, tree_mask=m))  # a fixed order of sums


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("bits,gs,D", [(4, 8, 128), (4, 16, 128), (4, 128, 128), (4, 8, 64), (8, 8, 128), (8, 16, 64),
                                       (8, 128, 128)])
def test_tree_attention_group_sizes(cuda, dtype, bits, gs, D):
    """Groups within a chunk of eight channels up to a whole row, in tiles that several parts share."""
    B, HQ, HKV, T, cap, n = 2, 6, 2, 11, 1024, 901
    g = torch.Generator(device="cuda").manual_seed(gs)
    q = torch.randn((B, HQ, T, D), generator=g, device="cuda").to(DT[dtype])
    packed = []
    for _ in range(3):
        words = torch.randint(-(2**31), 2**31, (B, HKV, cap, D * bits // 32), generator=g, device="cuda").int().view(torch.uint32)
        scales = (torch.rand((B, HKV, cap, D // gs), generator=g, device="cuda") * 2.0 / 2**bits + 0.01).to(DT[dtype])
        biases = (torch.randn((B, HKV, cap, D // gs), generator=g, device="cuda") * 0.5 - 1.0).to(DT[dtype])
        packed.append((words, scales, biases))
    m, m64 = masks("trees", B, T)
    got = call(q, packed, bits, gs, 0.05, kv_len=n, tree_mask=m)
    want, tol = attention64(q, *(unpack64(t, bits, gs) for t in packed), 0.05, [n] * B, m64, torch.finfo(DT[dtype]).eps / 2, True)
    check(got, want, tol, dtype)


@pytest.mark.parametrize("dtype,bits", [("fp16", 16), ("bf16", 4), ("fp16", 8), ("fp32", 16)])
@pytest.mark.parametrize("cap", [640, 16384])
def test_tree_attention_one_device_length(cuda, dtype, bits, cap):
    """One length on the device, the launch shaped for the capacity: parts without a tile, an empty cache."""
    B, HQ, HKV, T, D = 1, 6, 2, 9, 128
    q, kv, plain = make(2, B, HQ, HKV, T, D, cap, dtype, bits)
    m, m64 = masks("trees", B, T)
    n_dev = torch.zeros(1, dtype=torch.int32, device="cuda")
    for n in (0, 3, 9, 64, 65, 200, 640):
        n_dev.fill_(n)
        got = call(q, kv, bits, 64, 0.1, kv_len=n_dev, tree_mask=m)
        want, tol = attention64(q, *plain, 0.1, [n], m64, torch.finfo(DT[dtype]).eps / 2, bits != 16)
        check(got, want, tol, dtype, str(n))


@pytest.mark.parametrize("dtype,bits", [("fp16", 16), ("fp32", 16), ("bf16", 4)])
def test_tree_attention_device_lengths(cuda, dtype, bits):
    """One length per sequence read on the device: empty, shorter than the tree, beyond the capacity."""
    B, HQ, HKV, T, D, cap = 7, 6, 2, 5, 128, 1100
    lens = [0, 1, 4, 5, 700, 1100, 5000]
    q, kv, plain = make(1, B, HQ, HKV, T, D, cap, dtype, bits)
    m, m64 = masks("trees", B, T)
    n_dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = call(q, kv, bits, 64, 0.1, kv_len=n_dev, tree_mask=m)
    want, tol = attention64(q, *plain, 0.1, [min(x, cap) for x in lens], m64, torch.finfo(DT[dtype]).eps / 2, bits != 16)
    check(got, want, tol, dtype)
    assert (got[0] == 0).all()
    one = call(q, kv, bits, 64, 0.1, kv_len=n_dev[4:5], tree_mask=m)
    want, tol = attention64(q, *plain, 0.1, [700] * B, m64, torch.finfo(DT[dtype]).eps / 2, bits != 16)
    check(one, want, tol, dtype)


@pytest.mark.parametrize("dtype,bits", [("fp16", 16), ("bf16", 16), ("fp32", 16), ("fp16", 4)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n", [190, 700, 9000])  # a unit in one CTA, in a cluster, in parts joined by a second launch
def test_tree_attention_hidden_rows_may_hold_anything(cuda, dtype, bits, bad, n):
    """Rows behind the last live one, and drafted rows as seen by queries they are hidden from, do not reach
    a result; queries that see such a row get what the formula gives."""
    B, HQ, HKV, T, D, cap = 1, 4, 2, 6, 128, 9216
    q, kv, plain = make(3, B, HQ, HKV, T, D, cap, dtype, bits)
    par = [-1, 0, 0, 1, 1, 2]
    m = ancestors(par)
    rows = [n - T + 2, n - T + 4]  # drafted rows 2 and 4; row 5 descends from row 2
    for i, t in enumerate(kv):
        if bits == 16:
            t[:, :, n:] = bad
            t[:, :, rows[0]] = bad if i else t[:, :, rows[0]]  # V1, V2 of row 2
            t[:, :, rows[1]] = bad  # K, V1, V2 of row 4
        else:
            for part in t[1:]:
                part[:, :, n:] = bad
                part[:, :, rows[1]] = bad
    if bits != 16:
        plain = [unpack64(t, bits, 64) for t in kv]
    got = call(q, kv, bits, 64, 0.09, kv_len=n, tree_mask=m.cuda())
    touched = [4] if bits != 16 else [2, 4, 5]
    clean = [t for t in range(T) if t not in touched]
    assert torch.isfinite(got[:, :, clean]).all()
    safe = [torch.where(torch.isfinite(p.double()), p.double(), 0.0) for p in plain]
    want, tol = attention64(q, *safe, 0.09, [n], m[None], torch.finfo(DT[dtype]).eps / 2, bits != 16)
    check(got[:, :, clean], want[:, :, clean], tol[:, :, clean], dtype)
    assert torch.isnan(got[:, :, 4]).all() or not math.isnan(bad)
    if bits == 16:  # rows 2 and 5 see a finite key with non-finite values
        assert not torch.isfinite(got[:, :, [2, 5]]).any()


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_tree_attention_visible_nonfinite_row_by_channel(cuda, dtype):
    """A visible row with one infinite channel: the other channels keep their values."""
    B, HQ, HKV, T, D, cap, n = 1, 2, 1, 3, 64, 128, 100
    q, kv, _ = make(4, B, HQ, HKV, T, D, cap, dtype)
    want, tol = attention64(q, *kv, 0.1, [n], torch.ones((1, T, T)).tril().bool(), torch.finfo(DT[dtype]).eps / 2, False)
    kv[1][:, :, n - 2, 5] = float("inf")  # drafted row 1, channel 5 of V1
    got = call(q, kv, 16, 64, 0.1, kv_len=n)
    assert torch.isfinite(got[:, :, 0]).all() and torch.isposinf(got[:, :, 1:, 5]).all()
    keep = [c for c in range(2 * D) if c != 5]
    check(got[..., keep], want[..., keep], tol[..., keep], dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_tree_attention_strided_operands(cuda, dtype):
    """Heads of an interleaved cache read in place (the stock cache's k1 = keys[:, 0::2]), a transposed q,
    a cache slice that starts off a 16-byte boundary, and a sliced mask."""
    B, HQ, HKV, T, D, cap, n = 2, 4, 2, 6, 64, 320, 301
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn((B, T, HQ, D), generator=g, device="cuda").to(DT[dtype]).transpose(1, 2)
    big = [torch.randn((B, 2 * HKV, cap, D), generator=g, device="cuda").to(DT[dtype]) for _ in range(3)]
    kv = [t[:, 0::2] for t in big]
    m = torch.ones((2 * T, 2 * T), dtype=torch.bool, device="cuda").tril()[:T, :T]
    h = torch.finfo(DT[dtype]).eps / 2
    want, tol = attention64(q, *kv, 0.125, [n] * B, m.cpu().expand(B, T, T), h, False)
    check(call(q, kv, 16, 64, 0.125, kv_len=n, tree_mask=m), want, tol, dtype)
    odd = []
    for t in kv:
        flat = torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")[3:].view(B, HKV, cap, D)
        odd.append(flat.copy_(t))
    check(call(q, odd, 16, 64, 0.125, kv_len=n), want, tol, dtype)
    wide = [torch.randn((B, HKV, cap, 2 * D), device="cuda").to(DT[dtype]) for _ in range(3)]  # rows 2D apart
    for w, t in zip(wide, kv):
        w[..., :D] = t
    check(call(q, [w[..., :D] for w in wide], 16, 64, 0.125, kv_len=n), want, tol, dtype)
    want, tol = attention64(q, *kv, 0.125, [n - 1] * B, m.cpu().expand(B, T, T), h, False)
    short = [t[:, :, : n - 1] for t in kv]  # capacity n - 1 inside a longer buffer
    check(call(q, short, 16, 64, 0.125), want, tol, dtype)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_tree_attention_scales(cuda, scale):
    for dtype in ("fp16", "fp32"):
        q, kv, plain = make(6, 1, 2, 1, 4, 128, 128, dtype)
        want, tol = attention64(q, *plain, scale, [100], torch.ones((1, 4, 4)).tril().bool(), torch.finfo(DT[dtype]).eps / 2, False)
        check(call(q, kv, 16, 64, scale, kv_len=100), want, tol, dtype)


def test_tree_attention_single_rows_equal_the_decode_operator(cuda):
    """T = 1 is sdpa_dual_v; a causal tree of T rows is T decode steps (each within its own tolerance)."""
    from mlx_motif.kernels import sdpa_dual_v

    q, kv, plain = make(7, 1, 24, 8, 4, 128, 512, "fp16")
    want, tol = attention64(q, *plain, 0.088, [400], torch.ones((1, 4, 4)).tril().bool(), 2.0**-11, False)
    got = call(q, kv, 16, 64, 0.088, kv_len=400)
    check(got, want, tol, "fp16")
    for t in range(4):
        one = sdpa_dual_v(q[:, :, t : t + 1], *kv, 0.088, kv_len=397 + t)
        check(one, want[:, :, t : t + 1], tol[:, :, t : t + 1], "fp16")
        check(call(q[:, :, t : t + 1], kv, 16, 64, 0.088, kv_len=397 + t), want[:, :, t : t + 1], tol[:, :, t : t + 1], "fp16")


@pytest.mark.parametrize("dtype,bits", [("fp16", 16), ("fp16", 4), ("fp32", 16)])
def test_tree_attention_in_graphs_and_streams(cuda, dtype, bits):
    """Captured calls replay at other lengths and values, two graphs and two streams at once."""
    B, HQ, HKV, T, D, cap = 2, 6, 2, 5, 128, 1024
    sets = []
    for seed in (8, 9):
        q, kv, plain = make(seed, B, HQ, HKV, T, D, cap, dtype, bits)
        n = torch.tensor([600, 90], dtype=torch.int32, device="cuda")
        call(q, kv, bits, 64, 0.1, kv_len=n)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call(q, kv, bits, 64, 0.1, kv_len=n)
        sets.append((q, kv, plain, n, g, y))
    streams = [torch.cuda.Stream() for _ in sets]
    for lens in ([600, 90], [5, 1024], [1000, 333]):
        for s in sets:
            s[3].copy_(torch.tensor(lens, dtype=torch.int32))
            s[0].mul_(-1)
        torch.cuda.synchronize()
        for _ in range(3):
            for s, st in zip(sets, streams):
                with torch.cuda.stream(st):
                    s[4].replay()
        torch.cuda.synchronize()
        for q, kv, plain, n, g, y in sets:
            want, tol = attention64(q, *plain, 0.1, lens, torch.ones((B, T, T)).tril().bool(),
                                    torch.finfo(DT[dtype]).eps / 2, bits != 16)
            check(y, want, tol, dtype)


# ---------------------------------------------------------------- verification


def drafts(seed, B, T, V, dtype, tree=True, spread=3.0, apart=0.6):
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    par = [random_tree(T, rng) if tree else list(range(-1, T - 1)) for _ in range(B)]
    R = max(1, 1 + max(max(p) for p in par))
    base = torch.randn((B, T, V), generator=g) * spread
    p = (base + torch.randn((B, T, V), generator=g) * apart).to(DT[dtype])
    q = base[:, :R].to(DT[dtype]).contiguous()
    tok = torch.zeros((B, T), dtype=torch.int32)
    for b in range(B):
        for i in range(1, T):
            tok[b, i] = int(torch.multinomial(torch.softmax(q[b, par[b][i]].double(), -1), 1, generator=g))
    u = torch.rand((B, T), generator=g)
    return tok, torch.tensor(par, dtype=torch.int32), p, q, u


def same(got, want):
    for name in ("accepted", "path", "next_token"):
        a, b = getattr(got, name).cpu(), getattr(want, name).cpu()
        assert a.dtype == torch.int32 and torch.equal(a, b), f"{name}: {a.tolist()} != {b.tolist()}"


def verify(tok, par, p, q, u, temp):
    from mlx_motif.kernels import speculative_verify

    return speculative_verify(tok.cuda(), par.cuda(), p.cuda(), None if q is None else q.cuda(),
                              None if u is None else u.cuda(), temp)


@pytest.mark.parametrize("B,T,V,tree", [(1, 1, 1, False), (1, 2, 1, False), (2, 1, 500, False), (3, 5, 7, False),
                                        (1, 5, 219520, False), (5, 9, 501, True), (2, 33, 1000, True),
                                        (1, 64, 4097, True), (4, 6, 32001, True), (1, 300, 64, True)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("temp", [0.0, 0.7, 1.0])
def test_verify_equals_the_rule(cuda, B, T, V, tree, dtype, temp):
    """Whole numbers: equal to the 64-bit rule. (A flip needs a uniform within about 2^-24 of a border: the
    inputs are fixed, so a pass is a pass.)"""
    from mlx_motif.kernels import speculative_verify_reference

    args = drafts(T + V, B, T, V, dtype, tree)
    same(verify(*args, temp), speculative_verify_reference(*args, temp))


def test_verify_rejects_all_and_accepts_all(cuda):
    """The residual after many rejected children, a draft equal to its target, and uniforms at the ends."""
    from mlx_motif.kernels import speculative_verify_reference

    V, T = 50, 9
    for seed in range(20):
        tok, _, p, q, u = drafts(seed, 3, T, V, "fp32", tree=False, apart=4.0)
        par = torch.tensor([-1] + [0] * (T - 1), dtype=torch.int32)  # all children of the root
        q = q[:, :1].contiguous()
        g = torch.Generator().manual_seed(seed)
        tok[:, 1:] = torch.multinomial(torch.softmax(q[:, 0], -1), T - 1, replacement=True, generator=g).int()
        same(verify(tok, par, p, q, u, 1.0), speculative_verify_reference(tok, par, p, q, u, 1.0))
        hard = torch.full_like(u, 1 - 2.0**-24)
        same(verify(tok, par, p, q, hard, 1.0), speculative_verify_reference(tok, par, p, q, hard, 1.0))
        zero = torch.zeros_like(u)
        same(verify(tok, par, p, q, zero, 1.0), speculative_verify_reference(tok, par, p, q, zero, 1.0))
    tok, par, p, _, u = drafts(1, 2, 6, 300, "fp16", tree=False)
    q = p[:, :5].contiguous()
    for i in range(1, 6):
        tok[:, i] = q[:, i - 1].float().argmax(-1).int()
    r = verify(tok, par, p, q, torch.full_like(u, 1 - 2.0**-24), 0.7)
    assert r.accepted.tolist() == [5, 5] and r.path.tolist() == [list(range(6))] * 2


def test_verify_follows_the_targets_law(cuda):
    """30000 sequences of a two-level tree in one call: the first emitted token has the target's law
    (5 standard deviations of a frequency)."""
    B, V = 30000, 6
    g = torch.Generator(device="cuda").manual_seed(2)
    p = torch.randn((1, 4, V), generator=g, device="cuda").expand(B, 4, V)  # one row for all: strides of 0
    q = torch.randn((1, 1, V), generator=g, device="cuda").expand(B, 1, V)
    kids = torch.multinomial(torch.softmax(q[0, 0], -1), B * 3, replacement=True, generator=g).view(B, 3).int()
    tok = torch.cat([torch.zeros((B, 1), dtype=torch.int32, device="cuda"), kids], 1)
    par = torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
    r = verify(tok, par, p, q, torch.rand((B, 4), generator=g, device="cuda"), 1.0)
    first = torch.where(r.accepted > 0, tok.gather(1, r.path[:, 1:2].long().clamp_min(0))[:, 0], r.next_token)
    freq = torch.bincount(first.long(), minlength=V).double() / B
    want = torch.softmax(p[0, 0].double(), -1)
    assert (freq - want).abs().max() < 5 * (0.25 / B) ** 0.5


def test_verify_odd_rows(cuda):
    """Padding tokens, masked (-inf) and NaN and +inf logits, rows without a finite logit, a row without a
    draft row, parents shared by the batch, strided logits."""
    from mlx_motif.kernels import speculative_verify_reference

    tok, par, p, q, u = drafts(3, 6, 8, 130, "fp32")
    p[0, 0, 5:] = -math.inf
    q[1, 0, :100] = -math.inf
    p[2, 0, ::2] = math.nan
    p[3, 0] = -math.inf  # no law
    p[4, 0, 17] = math.inf
    q[4, 0, 17] = math.inf
    tok[5, 1:] = torch.tensor([-1, 130, 2**31 - 1, -(2**31), -1, -1, -1], dtype=torch.int32)
    for temp in (0.0, 0.9):
        want = speculative_verify_reference(tok, par, p, q, u, temp)
        same(verify(tok, par, p, q, u, temp), want)
        assert want.next_token[3] == 0 and want.accepted[3] == 0 and want.accepted[5] == 0
        same(verify(tok, par[0], p, q, u, temp), speculative_verify_reference(tok, par[0], p, q, u, temp))
        short = q[:, :1].contiguous()  # rows 1.. have no draft row
        same(verify(tok, par, p, short, u, temp), speculative_verify_reference(tok, par, p, short, u, temp))
        wide = torch.randn((6, 9, 300))
        wide[:, :8, :130] = p
        got = verify(tok, par, wide.cuda()[:, :8, :130], q.cuda().transpose(1, 2).contiguous().transpose(1, 2), u, temp)
        same(got, want)


def test_verify_greedy_ties_take_the_first(cuda):
    p = torch.zeros((1, 2, 5000))
    p[0, 0, [70, 4000]] = 2.0
    p[0, 1, :] = -0.0
    p[0, 1, 9] = 0.0
    for dtype in DT.values():
        r = verify(torch.tensor([[0, 70]], dtype=torch.int32), torch.tensor([-1, 0], dtype=torch.int32), p.to(dtype), None,
                   None, 0.0)
        assert (r.accepted.item(), r.next_token.item(), r.path.tolist()) == (1, 0, [[0, 1]])
        r = verify(torch.tensor([[0, 4000]], dtype=torch.int32), torch.tensor([-1, 0], dtype=torch.int32), p.to(dtype), None,
                   None, 0.0)
        assert (r.accepted.item(), r.next_token.item()) == (0, 70)


def test_verify_in_a_graph_and_on_two_streams(cuda):
    from mlx_motif.kernels import speculative_verify, speculative_verify_reference

    sets = []
    for seed in (5, 6):
        a = [t.cuda() for t in drafts(seed, 3, 7, 9001, "fp16")]
        speculative_verify(*a, 0.8)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = speculative_verify(*a, 0.8)
        sets.append((a, g, r, torch.cuda.Stream()))
    for round_ in range(3):
        for i, (a, *_) in enumerate(sets):
            for t, x in zip(a, drafts(10 * round_ + i, 3, 7, 9001, "fp16")):
                if t.shape == x.shape:
                    t.copy_(x)
        torch.cuda.synchronize()
        for _ in range(3):
            for a, g, r, s in sets:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for a, g, r, s in sets:
            same(r, speculative_verify_reference(*(t.cpu() for t in a), 0.8))


# ---------------------------------------------------------------- the accepted rows


def filled(kind, B, H, n, D, dtype, seed):
    from mlx_motif.cache import KVCache, MotifGroupedKVCache, MotifGroupedQuantizedKVCache, MotifVanillaKVCache

    g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(h):
        return torch.randn((B, h, n, D), generator=g, device="cuda").to(DT[dtype])

    if kind == "stock":
        c = KVCache()
        c.update_and_fetch(rows(2 * H), rows(2 * H))
        return c
    if kind == "vanilla":
        c = MotifVanillaKVCache()
        c.update_and_fetch(rows(2 * H), rows(2 * H))
        return c
    c = MotifGroupedKVCache() if kind == "rows" else MotifGroupedQuantizedKVCache(group_size=kind[1], bits=kind[0])
    c.update_and_fetch_4(*(rows(H) for _ in range(4)))
    return c


def bytes_of(cache):
    return [t.view(torch.uint8).cpu().clone() for t in cache._buffers()]


def moved(bufs, path, accepted, base):
    """The plain form, on bytes."""
    out = [t.clone() for t in bufs]
    for o, t in zip(out, bufs):
        for b in range(t.shape[0]):
            for j in range(1, accepted[b] + 1):
                o[b, :, base[b] + j] = t[b, :, base[b] + path[b][j]]
    return out


@pytest.mark.parametrize("kind,dtype", [("rows", "fp16"), ("rows", "bf16"), ("rows", "fp32"), ((4, 64), "fp16"),
                                        ((4, 32), "bf16"), ((8, 64), "fp16"), ("stock", "fp16"), ("vanilla", "fp16")])
@pytest.mark.parametrize("B,H,D,n,T", [(1, 8, 128, 200, 26), (2, 2, 64, 256, 9), (1, 1, 64, 64, 64), (3, 2, 128, 5, 2),
                                       (1, 2, 64, 3, 1)])
def test_keep_rows(cuda, kind, dtype, B, H, D, n, T):
    """Every kept count, overlapping moves (a chain's rows stay, a row can be both source and place), bytes."""
    from mlx_motif.cache import keep_rows, kv_slots

    rng = np.random.default_rng(n + T)
    for acc in sorted({0, 1, min(3, T - 1), T // 2, T - 1}):
        caches = [filled(kind, B, H, n, D, dtype, s) for s in range(3)]
        before = [bytes_of(c) for c in caches]
        path = np.full((B, T), -1, np.int32)
        accepted = [max(0, min(T - 1, acc - b)) for b in range(B)]
        for b in range(B):
            path[b, 0] = 0
            path[b, 1 : accepted[b] + 1] = np.sort(rng.permutation(np.arange(1, T))[: accepted[b]])
        p_dev, a_dev = torch.from_numpy(path).cuda(), torch.tensor(accepted, dtype=torch.int32, device="cuda")
        keep_rows(kv_slots(caches), p_dev, a_dev, n - T)
        for c, was in zip(caches, before):
            assert c.offset == n
            for got, want in zip(bytes_of(c), moved(was, path, accepted, [n - T] * B)):
                assert torch.equal(got, want)
        one = filled(kind, B, H, n, D, dtype, 0)
        one.keep_rows(p_dev, a_dev)  # its last T rows
        assert all(torch.equal(x, y) for x, y in zip(bytes_of(one), bytes_of(caches[0])))


@pytest.mark.parametrize("kind", ["rows", (4, 64), "stock"])
def test_keep_rows_refuses_views_of_replaced_buffers(cuda, kind):
    """A cache that grew has other buffers than its view: the call is refused and moves nothing."""
    from mlx_motif.cache import keep_rows, kv_slots

    caches = [filled(kind, 1, 2, 256, 64, "fp16", s) for s in range(3)]  # full: the next row makes it grow
    slots = kv_slots(caches)
    path, accepted = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0, 2, -1]], [1]))
    keep_rows(slots, path, accepted, 253)
    new = torch.zeros(1, 4 if kind == "stock" else 2, 1, 64, dtype=torch.float16, device="cuda")
    caches[1].update_and_fetch(new, new) if kind == "stock" else caches[1].update_and_fetch_4(new, new, new, new)
    before = [bytes_of(c) for c in caches]
    with pytest.raises(ValueError, match="kv_slots again"):
        keep_rows(slots, path, accepted, 253)
    for c, was in zip(caches, before):
        assert all(torch.equal(x, y) for x, y in zip(bytes_of(c), was))


def test_keep_rows_many_layers_device_bases_and_stray_paths(cuda):
    """More caches than one launch takes; one base per sequence, on the device, bases outside the cache; path
    entries that are no place of the tree; counts outside it."""
    from mlx_motif.cache import keep_rows, kv_slots

    T = 6
    caches = [filled("rows", 5, 1, 256, 64, "fp16", s) for s in range(70)]
    before = [bytes_of(c) for c in caches]
    base = torch.tensor([0, 100, 250, 253, -3], dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 2, 4, -1, -1, -1], [0, 3, 99, 5, 2, -7], [0, 5, -1, -1, -1, -1], [0, 2, 4, 5, -1, -1],
                         [0, 2, 3, -1, -1, -1]], dtype=torch.int32, device="cuda")
    accepted = torch.tensor([2, 100, 1, 3, 2], dtype=torch.int32, device="cuda")
    keep_rows(kv_slots(caches), path, accepted, base)
    # sequence 1: entries 99 and those not above their place move nothing; 3: rows 257, 258 are beyond the capacity
    want_path = [[0, 2, 4], [0, 3, 2, 5], [0, 5], [0, 2], [0]]
    want_acc = [2, 3, 1, 1, 0]
    for c, was in zip(caches, before):
        for got, want in zip(bytes_of(c), moved(was, want_path, want_acc, [0, 100, 250, 253, 0])):
            assert torch.equal(got, want)
    stock = [filled("stock", 1, 2, 256, 64, "fp16", 1)]
    was = bytes_of(stock[0])
    far = torch.tensor([300], dtype=torch.int32, device="cuda")  # inside the views' doubled capacity, outside the cache
    keep_rows(kv_slots(stock), path[:1], accepted[:1], far)
    assert all(torch.equal(a, b) for a, b in zip(bytes_of(stock[0]), was))
    with pytest.raises(AssertionError, match="outside capacity"):
        keep_rows(kv_slots(stock), path[:1], accepted[:1], 251)
    with pytest.raises(AssertionError, match="path"):
        keep_rows(kv_slots(stock), path[:2], accepted[:1], 0)
    with pytest.raises(TypeError, match="int32"):
        keep_rows(kv_slots(stock), path[:1].long(), accepted[:1], 0)
    with pytest.raises(AssertionError, match="differs"):
        keep_rows(kv_slots([filled("rows", 1, 1, 256, 64, "fp16", 0), filled("rows", 1, 2, 256, 64, "fp16", 0)]), path[:1],
                  accepted[:1], 0)


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("kind", ["rows", (4, 64)])
def test_a_cycle_of_tree_speculation(cuda, kind):
    """Append a tree, attend, verify, keep the accepted path, and attend with the next token: the same as a
    cache to which only the accepted rows were ever appended."""
    from mlx_motif.cache import MotifGroupedKVCache, MotifGroupedQuantizedKVCache, keep_rows, kv_slots
    from mlx_motif.kernels import sdpa_dual_v_tree, sdpa_dual_v_tree_q4, speculative_verify, tree_mask_from_parents

    H, HQ, D, T, V, n0 = 2, 6, 128, 12, 700, 130
    layers = 3
    g = torch.Generator(device="cuda").manual_seed(0)

    def new():
        return MotifGroupedKVCache() if kind == "rows" else MotifGroupedQuantizedKVCache(group_size=64, bits=4)

    def rows(S):
        return [torch.randn((1, H, S, D), generator=g, device="cuda").half() for _ in range(4)]

    def put(c, r):
        return c.update_and_fetch_4(*r) if kind == "rows" else c.update_and_fetch_4_quantized(*r)

    def attend(c, q, mask=None):
        f = sdpa_dual_v_tree if kind == "rows" else sdpa_dual_v_tree_q4
        return f(q, c.k1, c.v1, c.v2, D**-0.5, kv_len=c.offset, tree_mask=mask)

    caches, plain = [new() for _ in range(layers)], [new() for _ in range(layers)]
    for c, o in zip(caches, plain):
        r = rows(n0)
        put(c, r)
        put(o, r)
    for cycle in range(4):
        tok, par, p, q, u = (t.cuda() for t in drafts(cycle, 1, T, V, "fp16"))
        mask = tree_mask_from_parents(par)
        drafted = [rows(T) for _ in range(layers)]
        Q = torch.randn((1, HQ, T, D), generator=g, device="cuda").half()
        outs = []
        for c, r in zip(caches, drafted):
            put(c, r)
            outs.append(attend(c, Q, mask))
        res = speculative_verify(tok, par, p, q, u, 0.8)
        base = caches[0].offset - T
        keep_rows(kv_slots(caches), res.path, res.accepted, base)
        k = int(res.accepted[0])
        idx = res.path[0, : k + 1].long()
        for c, o, r, y in zip(caches, plain, drafted, outs):
            assert c.trim(T - 1 - k) == T - 1 - k
            put(o, [x[:, :, idx] for x in r])
            assert c.offset == o.offset
            for a, b in zip(c.state, o.state):
                for x, z in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
                    assert torch.equal(x, z)
            # the accepted rows' outputs are those of the chain they form (same values, other order of sums)
            chain = attend(o, Q[:, :, idx])
            err = (chain.float() - y[:, :, idx].float()).abs().max()
            assert float(err) <= 2 * 2.0**-11 * 2 * 2.5, float(err)  # both round p and o: 2h(A + |o|), A <= 2.5 here


def test_operators_refuse_cpu_tensors_and_mixed_devices(cuda):
    from mlx_motif.kernels import sdpa_dual_v_tree, speculative_verify

    q, kv, _ = make(0, 1, 2, 1, 3, 64, 64, "fp16")
    with pytest.raises(ValueError, match="device"):
        sdpa_dual_v_tree(q, kv[0].cpu(), kv[1], kv[2], 0.1)
    with pytest.raises(ValueError, match="device"):
        sdpa_dual_v_tree(q, *kv, 0.1, tree_mask=torch.ones((3, 3), dtype=torch.bool))
    with pytest.raises(TypeError, match="kv_len"):
        sdpa_dual_v_tree(q, *kv, 0.1, kv_len=torch.tensor([1.0, 2.0], device="cuda"))
    tok, par, p, lq, u = drafts(0, 1, 3, 50, "fp16")
    with pytest.raises(ValueError, match="device"):
        speculative_verify(tok, par.cuda(), p.cuda(), lq.cuda(), u.cuda(), 1.0)
