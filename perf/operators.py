"""Workloads of the drafted-token operators: attention for a tree of drafted tokens over a KV cache, the
verification of the drafted tokens, and the move of the accepted rows to the front of the tree's cache rows.

``run`` computes an operator in elementary torch operations (``own = False``) or through this package's entry
points (``own = True``) on what ``prepare`` made.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_PKG = str(Path(__file__).resolve().parent.parent / "mlx-motif_b200")


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import mlx_motif.cache
    import mlx_motif.kernels

    return mlx_motif


# --------------------------------------------------------------------------------------------- cases


def _attn(name, B, HQ, HKV, T, D, cap, n, dtype, bits=16, gs=64, mask="tree", lens="host"):
    """n: live cache rows, the T drafted ones included; lens "device": each sequence has its own length, drawn
    from [n/4, n], in an int32 tensor on the GPU."""
    return dict(name=name, op="attn", B=B, HQ=HQ, HKV=HKV, T=T, D=D, cap=cap, n=n, dtype=dtype, bits=bits, gs=gs,
                mask=mask, lens=lens)


def _verify(name, B, T, V, dtype, temperature, tree):
    """T rows: the last committed token and T - 1 drafted ones. tree: "chain" or "tree"."""
    return dict(name=name, op="verify", B=B, T=T, V=V, dtype=dtype, temperature=temperature, tree=tree)


def _keep(name, layers, B, H, D, cap, base, T, accepted, dtype, bits=16, gs=64):
    return dict(name=name, op="keep", layers=layers, B=B, H=H, D=D, cap=cap, base=base, T=T, accepted=accepted,
                dtype=dtype, bits=bits, gs=gs)


def listed():
    return [
        # a chain of four drafted tokens after a 164-token prompt, the 12.7B-class model's origin heads: latency
        _attn("attn_chain5_p164", 1, 24, 8, 5, 128, 256, 169, "fp16", mask="chain"),
        # a tree over the 2.6B-class model's 3204-token prompt (its q1 stripes on k1)
        _attn("attn_tree26_bf16", 1, 8, 2, 26, 128, 3328, 3230, "bf16"),
        # a wide tree over the 16000-token prompt, fp16 cache
        _attn("attn_tree64_16k", 1, 24, 8, 64, 128, 16384, 16064, "fp16"),
        # a small tree over the same prompt in the packed q4 cache
        _attn("attn_q4_tree17_16k", 1, 24, 8, 17, 128, 16384, 16017, "fp16", bits=4),
        # eight requests of different lengths served together, each with its own tree
        _attn("attn_batch8_tree31", 8, 24, 8, 31, 128, 8192, 8192, "fp16", lens="device"),
        # full precision, 64-wide heads, odd sizes
        _attn("attn_fp32_d64", 2, 8, 4, 7, 64, 1280, 1031, "fp32"),
        # the speculative decoder's cycle: four drafted tokens, the 219520-token vocabulary
        _verify("verify_chain5", 1, 5, 219520, "fp16", 0.7, "chain"),
        # a wide tree against the same vocabulary
        _verify("verify_tree64", 1, 64, 219520, "fp16", 0.7, "tree"),
        # sixteen requests with small trees, a smaller and odd vocabulary
        _verify("verify_batch16_tree9", 16, 9, 32001, "bf16", 1.0, "tree"),
        # greedy verification of a longer chain, fp32 logits
        _verify("verify_greedy17", 1, 17, 219520, "fp32", 0.0, "chain"),
        # after the verification: three accepted rows of a 26-row tree, 48 layers, fp16 cache
        _keep("keep_fp16_48l", 48, 1, 8, 128, 1024, 820, 26, 3, "fp16"),
        # the packed q4 cache, eight accepted rows of 64
        _keep("keep_q4_48l", 48, 1, 8, 128, 1024, 900, 64, 8, "fp16", bits=4),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        t = top.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for k in t:
            t[k] = max(t[k], w[k])
    while True:
        op = rng.choice(["attn", "attn", "attn", "verify", "verify", "keep"])
        if op == "attn":
            dtype, bits = rng.choice([("fp16", 16), ("fp16", 16), ("bf16", 16), ("fp32", 16), ("fp16", 4), ("bf16", 4),
                                      ("fp16", 8)])
            T, D = _log_int(rng, 1, 64), rng.choice([64, 128, 128, 128])
            HKV, gqa = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
            B = _log_int(rng, 1, 8)
            n = _log_int(rng, T, 2048 if dtype == "fp32" else 16384)
            cap = -(-(n + rng.randrange(512)) // 256) * 256
            c = _attn("", B, HKV * gqa, HKV, T, D, cap, n, dtype, bits, rng.choice([32, 64]),
                      rng.choice(["tree", "chain"]), rng.choice(["host", "device"]))
        elif op == "verify":
            c = _verify("", _log_int(rng, 1, 16), _log_int(rng, 1, 64), _log_int(rng, 500, 219520),
                        rng.choice(["fp16", "bf16", "fp32"]), rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]),
                        rng.choice(["tree", "chain"]))
        else:
            acc = rng.randrange(0, 12)
            T = 2 * acc + 1 + rng.randrange(0, 40)
            base = _log_int(rng, 1, 1500)
            c = _keep("", rng.choice([1, 2, 12, 32, 48]), rng.choice([1, 1, 2, 4]), rng.choice([1, 2, 4, 8]),
                      rng.choice([64, 128]), -(-(base + T) // 256) * 256, base, T, acc, rng.choice(["fp16", "bf16"]),
                      rng.choice([16, 4, 8]))
        c.pop("name")
        # no more than the largest listed case of the operator (a cache's buffers included)
        size = _cache_bytes(c) if op == "keep" else work(c)["bytes"]
        limit = 48 * 4 * 8 * 1024 * 256 if op == "keep" else top[op]["bytes"]
        if size <= limit and work(c)["flops"] <= max(top[op]["flops"], 1):
            return c


def _row_bytes(c):
    """Bytes of one cache row of one slot and head."""
    e = DT[c["dtype"]].itemsize
    return c["D"] * e if c["bits"] == 16 else c["D"] * c["bits"] // 8 + 2 * e * (c["D"] // c["gs"])


def _cache_bytes(c):
    return c["layers"] * 4 * c["B"] * c["H"] * c["cap"] * _row_bytes(c)


def work(case):
    c = case
    e = DT[c["dtype"]].itemsize
    if c["op"] == "attn":
        rows = c["B"] * c["n"] if c["lens"] == "host" else sum(_lengths(c))
        out = c["B"] * c["HQ"] * c["T"] * c["D"] * e
        return {"bytes": rows * c["HKV"] * 3 * _row_bytes(c) + 3 * out + c["B"] * c["T"] ** 2,
                "flops": 2 * rows * c["HQ"] * c["T"] * 3 * c["D"]}
    if c["op"] == "verify":
        # each logit read once: the target's T rows and (T > 0) the draft's rows of the nodes that have children
        rows = c["T"] + (_draft_rows(c) if c["temperature"] > 0 else 0)
        return {"bytes": c["B"] * rows * c["V"] * e, "flops": c["B"] * rows * c["V"] * (4 if c["temperature"] > 0 else 1)}
    return {"bytes": 2 * c["layers"] * 4 * c["B"] * c["H"] * c["accepted"] * _row_bytes(c), "flops": 0}


# --------------------------------------------------------------------------------------------- inputs


def _tree(T, kind, rng):
    """parents of T rows, row 0 the root (-1), every parent before its children: a chain, or a tree whose root has
    up to four children and whose other rows hang on one of the eight rows before them."""
    if kind == "chain":
        return [i - 1 for i in range(T)]
    return [-1] + [0 if i <= 4 else int(rng.integers(max(0, i - 8), i)) for i in range(1, T)]


def _shape_rng(c):
    """Shapes (tree, lengths) belong to the case, not to the seed of its values."""
    return np.random.default_rng([c["B"], c["T"]])


def _trees(c):
    rng = _shape_rng(c)
    return [_tree(c["T"], c.get("tree", c.get("mask")), rng) for _ in range(c["B"])]


def _draft_rows(c):
    return max(1, 1 + max(max(p) for p in _trees(c)))


def _lengths(c):
    rng = _shape_rng(c)
    lo = max(c["T"], c["n"] // 4)
    return [int(x) for x in rng.integers(lo, c["n"] + 1, c["B"])]


def _masks(c):
    """mask[b, i, j]: row i descends from row j or is it."""
    m = np.zeros((c["B"], c["T"], c["T"]), dtype=bool)
    for b, parents in enumerate(_trees(c)):
        for i, p in enumerate(parents):
            if p >= 0:
                m[b, i] = m[b, p]
            m[b, i, i] = True
    return m


def _pack(x, bits, gs, dtype):
    """(..., D) -> (words uint32, scales, biases): affine codes by group, little-endian in 32-bit words."""
    g = x.reshape(*x.shape[:-1], -1, gs).float()
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / (2**bits - 1)).clamp_min(1e-4).to(dtype).float()
    b = lo.to(dtype).float()
    q = ((g - b) / s).round().clamp(0, 2**bits - 1).to(torch.int32).reshape(*x.shape[:-1], -1, 32 // bits)
    w = torch.zeros(q.shape[:-1], dtype=torch.int32, device=x.device)
    for j in range(32 // bits):
        w |= q[..., j] << (bits * j)
    return w.view(torch.uint32), s[..., 0].to(dtype), b[..., 0].to(dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DT[c["dtype"]]

    def randn(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    if c["op"] == "attn":
        q = randn(c["B"], c["HQ"], c["T"], c["D"])
        kv = [randn(c["B"], c["HKV"], c["cap"], c["D"], std=s) for s in (1.0, 0.5, 0.5)]
        if c["bits"] != 16:
            kv = [_pack(x, c["bits"], c["gs"], dt) for x in kv]
        mask = None if c["mask"] == "chain" else torch.from_numpy(_masks(c)).cuda()
        n = c["n"] if c["lens"] == "host" else torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
        return dict(case=c, q=q, kv=kv, mask=mask, n=n, scale=c["D"] ** -0.5)

    if c["op"] == "verify":
        B, T, V = c["B"], c["T"], c["V"]
        parents = torch.tensor(_trees(c), dtype=torch.int32, device="cuda")
        R = _draft_rows(c)
        # a draft that resembles its target: common logits of spread 3, each with its own deviation
        p, q = (torch.empty((B, r, V), dtype=dt, device="cuda") for r in (T, R))
        up = parents.long().clamp_min(0)
        tokens = torch.zeros((B, T), dtype=torch.int32, device="cuda")
        for b in range(B):
            base = torch.randn((T, V), generator=g, device="cuda") * 3
            p[b] = (base + torch.randn((T, V), generator=g, device="cuda") * 0.6).to(dt)
            q[b] = base[:R].to(dt)
            # every drafted token is drawn from its parent's draft row (temperature 0: mostly its largest)
            w = torch.softmax(q[b].double() / max(c["temperature"], 0.1), dim=-1)
            tokens[b] = torch.multinomial(w[up[b]].float(), 1, generator=g)[:, 0].int()
        u = torch.rand((B, T), generator=g, device="cuda")
        # the tree's width is the drafting program's own knowledge
        width = max(max((t.count(i) for i in range(T)), default=0) for t in _trees(c))
        return dict(case=c, tokens=tokens, parents=parents, mask=torch.from_numpy(_masks(c)).cuda(), p=p, q=q, u=u,
                    temperature=c["temperature"], width=width)

    L, B, H, cap, D = (c[k] for k in ("layers", "B", "H", "cap", "D"))
    if c["bits"] == 16:
        bufs = [torch.empty((L, 4, B, H, cap, D), dtype=dt, device="cuda")]
        for li in range(L):
            bufs[0][li] = randn(4, B, H, cap, D)
    else:
        bufs = [torch.randint(-(2**31), 2**31, (L, 4, B, H, cap, D * c["bits"] // 32), generator=g, device="cuda",
                              dtype=torch.int64).int()]
        bufs += [randn(L, 4, B, H, cap, D // c["gs"]) for _ in range(2)]
    rng = np.random.default_rng(seed)
    path = np.full((B, c["T"]), -1, dtype=np.int32)
    path[:, 0] = 0
    for b in range(B):
        # rows behind the accepted ones' places, so that a pass finds its sources unchanged by the pass before it
        rows = np.sort(rng.permutation(np.arange(c["accepted"] + 1, c["T"]))[: c["accepted"]])
        path[b, 1:c["accepted"] + 1] = rows
    state = dict(case=c, bufs=bufs, path=torch.from_numpy(path).cuda(), base=c["base"],
                 accepted=torch.full((B,), c["accepted"], dtype=torch.int32, device="cuda"))
    if own:  # the program's caches, and its handle on all their layers
        m = _package()
        caches = []
        for li in range(L):
            if c["bits"] == 16:
                k = m.cache.MotifGroupedKVCache()
                k.k1, k.k2, k.v1, k.v2 = bufs[0][li]
            else:
                k = m.cache.MotifGroupedQuantizedKVCache(group_size=c["gs"], bits=c["bits"])
                k.k1, k.k2, k.v1, k.v2 = (tuple((x.view(torch.uint32) if i == 0 else x)[li, s] for i, x in enumerate(bufs))
                                          for s in range(4))
            k.offset = c["base"] + c["T"]
            caches.append(k)
        state["slots"] = m.cache.kv_slots(caches)
    return state


# --------------------------------------------------------------------------------------------- one pass


def run(state):
    return {"attn": _run_attn, "verify": _run_verify, "keep": _run_keep}[state["case"]["op"]](state)


def _unpack(t, bits, gs):
    w, s, b = t
    shifts = torch.arange(0, 32, bits, dtype=torch.int32, device=w.device)
    q = (w.view(torch.int32).unsqueeze(-1) >> shifts) & (2**bits - 1)
    x = q.reshape(*w.shape[:-1], -1, gs).float() * s.float().unsqueeze(-1) + b.float().unsqueeze(-1)
    return x.reshape(*w.shape[:-1], -1)


def _run_attn(st):
    c, q, kv, mask, n, scale = (st[k] for k in ("case", "q", "kv", "mask", "n", "scale"))
    if own:
        k = _package().kernels
        if c["bits"] == 16:
            return k.sdpa_dual_v_tree(q, *kv, scale, kv_len=n, tree_mask=mask)
        return k.sdpa_dual_v_tree_q4(q, *kv, scale, group_size=c["gs"], bits=c["bits"], kv_len=n, tree_mask=mask)
    B, HQ, T, D = q.shape
    N = n if isinstance(n, int) else c["cap"]
    if c["bits"] == 16:
        k, v1, v2 = (x[:, :, :N].float() for x in kv)
    else:
        k, v1, v2 = (_unpack(tuple(y[:, :, :N] for y in x), c["bits"], c["gs"]) for x in kv)
    qf = q.float().reshape(B, c["HKV"], -1, D)
    s = (qf @ k.transpose(-1, -2) * scale).view(B, HQ, T, N)
    if mask is None:
        mask = torch.ones((T, T), dtype=torch.bool, device=q.device).tril()
    first = (n if isinstance(n, int) else n.long()[:, None, None]) - T
    col = torch.arange(N, device=q.device) - first  # (N) or (B, 1, N): the drafted rows count from 0
    col = col.expand(B, T, N)
    seen = torch.gather(mask.expand(B, T, T), 2, col.clamp(0, T - 1)) & (col < T) | (col < 0)
    s = s.masked_fill(~seen[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    den = p.sum(-1, keepdim=True)
    p = (p / torch.where(den == 0, 1.0, den)).view(B, c["HKV"], -1, N)
    return torch.cat([p @ v1, p @ v2], dim=-1).view(B, HQ, T, 2 * D).to(q.dtype)


def _run_verify(st):
    tokens, parents, p, q, u, temp = (st[k] for k in ("tokens", "parents", "p", "q", "u", "temperature"))
    if own:
        r = _package().kernels.speculative_verify(tokens, parents, p, q if temp > 0 else None, u, temp)
        return {"accepted": r.accepted, "path": r.path, "next_token": r.next_token}
    B, T, V = p.shape
    tok, up = tokens.long(), parents.long().clamp_min(0)
    at, row = torch.arange(B, device=p.device)[:, None], torch.arange(T, device=p.device)
    # how many elder siblings a row has; the root is nobody's child
    sibling = (parents[:, :, None] == parents[:, None, :]) & (row[:, None] > row)
    rank = torch.where(row > 0, sibling.sum(-1), -1)
    if temp > 0:
        P, Q = (torch.softmax(x.double() / temp, dim=-1) for x in (p, q))
        Q = torch.cat([Q, Q.new_zeros((B, T - Q.shape[1], V))], dim=1)
        px, qx = P[at, up, tok], Q[at, up, tok]
        a, S = torch.zeros_like(px), torch.ones_like(px)  # a row's residual: (P - a Q)+ / S
        ok = torch.zeros_like(rank, dtype=torch.bool)
        for r in range(st["width"]):  # every row's r-th child at once
            now = rank == r
            left = (px - a[at, up] * qx).clamp_min(0)
            ok |= now & (u.double() * qx * S[at, up] < left)
            asked = (now[:, :, None] & (up[:, :, None] == row)).any(1)  # rows that have an r-th child
            a = torch.where(asked, a + S, a)
            S = torch.where(asked, (P - a[..., None] * Q).clamp_min(0).sum(-1), S)
    else:
        best = p.float().argmax(-1)
        ok = (row > 0) & (tok == best[at, up])
    taken = ok & ~(sibling & ok[:, None, :]).any(-1) | (row == 0)
    on_path = ~(st["mask"] & ~taken[:, None, :]).any(-1)
    accepted = on_path.sum(-1) - 1
    path = torch.where(on_path, row, T).sort(-1).values
    last = path.gather(1, accepted[:, None])
    path = torch.where(path == T, -1, path)
    if temp > 0:
        wide = P[at, last][:, 0]
        rest = (wide - a[at, last] * Q[at, last][:, 0]).clamp_min(0)
        C = torch.where(rest.sum(-1, keepdim=True) > 0, rest, wide).cumsum(-1)
        nxt = torch.searchsorted(C, u[:, :1].double() * C[:, -1:], right=True)
        nxt = torch.minimum(nxt, (C == C[:, -1:]).float().argmax(-1, keepdim=True))
    else:
        nxt = best[at, last]
    return {"accepted": accepted.int(), "path": path.int(), "next_token": nxt[:, 0].int()}


def _run_keep(st):
    c, bufs, path, accepted, base = (st[k] for k in ("case", "bufs", "path", "accepted", "base"))
    if own:
        _package().cache.keep_rows(st["slots"], path, accepted, base)
        return bufs
    at, j = torch.arange(c["B"], device=path.device)[:, None], torch.arange(c["T"], device=path.device)
    src = base + torch.where((j > 0) & (j <= accepted[:, None]), path.long(), j)
    for x in bufs:  # codes, scales, biases: every layer and slot at once
        x[:, :, at, :, base + j] = x[:, :, at, :, src]
    return bufs


# --------------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence and row by row; the moved cache rows are copies, not
    computed numbers (None)."""
    c = case
    if c["op"] == "keep":
        return None
    st = prepare(case, seed)
    if c["op"] == "attn":
        out = torch.empty((c["B"], c["HQ"], c["T"], 2 * c["D"]), dtype=torch.float64, device="cuda")
        lens = [c["n"]] * c["B"] if c["lens"] == "host" else _lengths(c)
        seen = np.tril(np.ones((c["B"], c["T"], c["T"]), dtype=bool)) if c["mask"] == "chain" else _masks(c)
        gqa = c["HQ"] // c["HKV"]
        for b, n in enumerate(lens):
            hide = torch.zeros((c["T"], n), dtype=torch.bool)
            hide[:, n - c["T"]:] = ~torch.from_numpy(seen[b])
            hide = hide.cuda()
            for h in range(c["HKV"]):
                k, v1, v2 = (_rows64(t, b, h, n, c) for t in st["kv"])
                for x in range(h * gqa, (h + 1) * gqa):
                    s = torch.einsum("td,nd->tn", st["q"][b, x].double(), k) * st["scale"]
                    w = torch.softmax(s.masked_fill(hide, -math.inf), dim=1)
                    out[b, x, :, :c["D"]] = torch.einsum("tn,nd->td", w, v1)
                    out[b, x, :, c["D"]:] = torch.einsum("tn,nd->td", w, v2)
        return out
    B, T = c["B"], c["T"]
    accepted, nxt = np.zeros(B, np.int32), np.zeros(B, np.int32)
    path = np.full((B, T), -1, np.int32)
    for b in range(B):
        parents, toks, us = (st[k][b].cpu().numpy() for k in ("parents", "tokens", "u"))
        cur, kept = 0, [0]
        rest = wide = _law(st["p"][b, 0], c["temperature"])
        for i in range(1, T):
            if parents[i] != cur:
                continue
            if c["temperature"] > 0:
                draft = _law(st["q"][b, cur], c["temperature"])
                good = float(us[i]) * draft[toks[i]] < rest[toks[i]]
            else:
                good = toks[i] == wide.argmax()
            if good:
                cur = i
                kept.append(i)
                rest = wide = _law(st["p"][b, cur], c["temperature"])
            elif c["temperature"] > 0:
                rest = np.maximum(rest - draft, 0.0)
                rest = rest / rest.sum() if rest.sum() > 0 else rest
        accepted[b] = len(kept) - 1
        path[b, :len(kept)] = kept
        if c["temperature"] > 0:
            w = rest if rest.sum() > 0 else wide
            C = np.cumsum(w)
            nxt[b] = min(np.searchsorted(C, float(us[0]) * C[-1], side="right"), np.flatnonzero(w)[-1])
        else:
            nxt[b] = wide.argmax()
    return {"accepted": torch.from_numpy(accepted), "path": torch.from_numpy(path), "next_token": torch.from_numpy(nxt)}


def _law(row, temperature):
    x = row.cpu().double().numpy()
    if temperature == 0:
        return x
    w = np.exp((x - x.max()) / temperature)
    return w / w.sum()


def _rows64(t, b, h, n, c):
    """Rows [0, n) of one slot's head in 64 bits."""
    if c["bits"] == 16:
        return t[b, h, :n].double()
    w, s, z = (x[b, h, :n] for x in t)
    w = w.view(torch.int32).long() & 0xFFFFFFFF
    per = 32 // c["bits"]
    out = torch.empty((n, c["D"]), dtype=torch.float64, device=w.device)
    for ch in range(c["D"]):
        code = (w[:, ch // per] >> (c["bits"] * (ch % per))) & (2 ** c["bits"] - 1)
        out[:, ch] = code.double() * s[:, ch // c["gs"]].double() + z[:, ch // c["gs"]].double()
    return out
