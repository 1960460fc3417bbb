"""Verification of drafted tokens against the target's probabilities: ``speculative_verify``.

The acceptance rule of the reference's speculative loop (``MotifSpeculativeDecoding.swift``: min(1, p/q), the
residual max(0, p − q), a bonus token from the last row) for trees and batches, with the random numbers given:
the same inputs give the same tokens. ``SpeculativeDecoder`` keeps ``motif_speculative_accept``, which draws
its own numbers for one chain.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from ._common import _DISABLE, check, contiguous, dtype_code, lib, on_device, ptr, stream, workspace


class VerifyResult(NamedTuple):
    accepted: torch.Tensor  # (B,) int32: drafted tokens accepted
    path: torch.Tensor  # (B, T) int32: row 0, the accepted rows in order, then -1
    next_token: torch.Tensor  # (B,) int32


def speculative_verify_reference(tokens, parents, p_logits, q_logits, uniforms, temperature) -> VerifyResult:
    """The rule in 64 bits on the host, sequence by sequence."""
    B, T = tokens.shape
    V = p_logits.shape[-1]
    par = parents.cpu().expand(B, T).tolist()
    tok = tokens.cpu().tolist()
    u = None if uniforms is None else uniforms.double().cpu()
    accepted, nxt = [], []
    path = torch.full((B, T), -1, dtype=torch.int32)
    R = 0 if q_logits is None else q_logits.shape[1]

    def law(row):
        x = row.double().cpu()
        x = torch.where(x.isnan(), -math.inf, x)
        m = x.max()
        if m == -math.inf:
            return torch.zeros(V, dtype=torch.float64)
        w = torch.where(x == m, 1.0, torch.exp((x - m) / temperature))
        return w / w.sum()

    def greedy(row):
        x = row.float().cpu()
        x = torch.where(x.isnan(), -math.inf, x)
        return int(x.argmax()) if x.max() > -math.inf else -1

    for b in range(B):
        cur, kept = 0, [0]
        P = law(p_logits[b, 0]) if temperature > 0 else greedy(p_logits[b, 0])
        a, S, Q = 0.0, 1.0, None
        for i in range(1, T):
            x = tok[b][i]
            if par[b][i] != cur or not 0 <= x < V:
                continue
            if temperature > 0:
                if cur >= R:
                    continue
                Q = law(q_logits[b, cur]) if Q is None else Q
                ok = float(u[b, i]) * float(Q[x]) * S < float(P[x]) - a * float(Q[x])
                if not ok:
                    a += S
                    S = float((P - a * Q).clamp_min(0).sum())
            else:
                ok = x == P
            if ok:
                cur = i
                kept.append(i)
                P = law(p_logits[b, i]) if temperature > 0 else greedy(p_logits[b, i])
                a, S, Q = 0.0, 1.0, None
        accepted.append(len(kept) - 1)
        path[b, : len(kept)] = torch.tensor(kept, dtype=torch.int32)
        if temperature > 0:
            w = (P - a * Q).clamp_min(0) if a > 0 and S > 0 else P
            run = w.cumsum(0)
            live = (w > 0).nonzero()
            at = int(torch.searchsorted(run, float(u[b, 0]) * run[-1], right=True))
            nxt.append(min(at, int(live[-1])) if len(live) else 0)
        else:
            nxt.append(max(P, 0))
    dev = p_logits.device
    return VerifyResult(torch.tensor(accepted, dtype=torch.int32, device=dev), path.to(dev),
                        torch.tensor(nxt, dtype=torch.int32, device=dev))


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*shape) -> int:
    return lib.motif_speculative_verify_workspace_bytes(*shape)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Logits whose vocabulary axis is contiguous (batch and row strides are passed on)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def speculative_verify(tokens: torch.Tensor, parents: torch.Tensor, p_logits: torch.Tensor,
                       q_logits: torch.Tensor | None, uniforms: torch.Tensor | None,
                       temperature: float) -> VerifyResult:
    """Walk each sequence's tree of drafted tokens with the target's laws.

    Row 0 is the last committed token; row i ≥ 1 is drafted token ``tokens[b, i]``, a child of row
    ``parents[…, i]`` < i. tokens (B, T) int32; parents (T,) or (B, T) int32; p_logits (B, T, V), the target's
    row after each tree row; q_logits (B, R, V), R ≤ T, the draft's row r, from which row r's children were
    drawn independently (what rows without children hold does not matter); uniforms (B, T) fp32 in [0, 1):
    [b, i] tests row i, [b, 0] draws the next token (from 1 on the last one with weight). Children are tested in
    ascending order: accepted with probability min(1, w(x) / q(x)), w = p, after each rejection
    w = max(0, w − q) renormalised; the next token is drawn from the last w. At ``temperature`` 0 (q_logits and
    uniforms may be None) a child is accepted if it is the target's argmax. Returns (accepted, path, next_token)
    on the device: no synchronisation.

    A token outside [0, V) is never accepted (padding of a smaller tree). NaN logits count as −inf. ``temperature``
    is 0 or in [1e-6, 1e6].
    """
    if _DISABLE:
        return speculative_verify_reference(tokens, parents, p_logits, q_logits, uniforms, temperature)
    temperature = float(temperature)
    assert p_logits.dim() == 3, f"p_logits {tuple(p_logits.shape)} must be (B, T, V)"
    B, T, V = p_logits.shape
    assert T >= 1 and V >= 1, f"p_logits {tuple(p_logits.shape)} must have a row and a token"
    assert tokens.shape == (B, T), f"tokens {tuple(tokens.shape)} must be ({B}, {T})"
    assert parents.shape == (B, T) or parents.shape == (T,), f"parents {tuple(parents.shape)} must be ({T},) or ({B}, {T})"
    assert temperature == 0 or 1e-6 <= temperature <= 1e6, f"temperature {temperature} must be 0 or in [1e-6, 1e6]"
    dev = p_logits.device
    if tokens.dtype != torch.int32 or parents.dtype != torch.int32:
        raise TypeError(f"tokens and parents must be int32, got {tokens.dtype} and {parents.dtype}")
    code = dtype_code(p_logits)
    sampled = temperature > 0
    R = 0
    if sampled:
        assert q_logits is not None and uniforms is not None, "q_logits and uniforms are needed at a temperature > 0"
        assert q_logits.dim() == 3 and q_logits.shape[0] == B and q_logits.shape[2] == V and 1 <= q_logits.shape[1] <= T, \
            f"q_logits {tuple(q_logits.shape)} must be ({B}, 1..{T}, {V})"
        assert uniforms.shape == (B, T), f"uniforms {tuple(uniforms.shape)} must be ({B}, {T})"
        if q_logits.dtype != p_logits.dtype:
            raise TypeError(f"q_logits {q_logits.dtype} and p_logits {p_logits.dtype} must have one type")
        if uniforms.dtype != torch.float32:
            raise TypeError(f"uniforms must be float32, got {uniforms.dtype}")
        R = q_logits.shape[1]
    for t in (tokens, parents, q_logits, uniforms) if sampled else (tokens, parents):
        if t.device != dev:
            raise ValueError(f"tensors on {t.device} and {dev}: all operands must be on one CUDA device")
    out = VerifyResult(tokens.new_empty(B), tokens.new_empty((B, T)), tokens.new_empty(B))
    if B == 0:
        return out
    with on_device(dev):
        p = _rows(p_logits)
        q = _rows(q_logits) if sampled else None
        tok, par = contiguous(tokens), contiguous(parents)
        u = contiguous(uniforms) if sampled else None
        ws_bytes = _workspace_bytes(B, T, R, V)
        ws = workspace(ws_bytes, dev)
        accepted, path, next_token = out
        pb, pr, _ = p.stride()
        qb, qr, _ = q.stride() if sampled else (0, 0, 0)
        check(lib.motif_speculative_verify(code, p.data_ptr(), pb, pr, ptr(q), qb, qr, R, tok.data_ptr(), par.data_ptr(),
                                           T if parents.dim() == 2 else 0, ptr(u), B, T, V, temperature,
                                           accepted.data_ptr(), path.data_ptr(), next_token.data_ptr(),
                                           ws.data_ptr(), ws_bytes, stream(dev)), "speculative_verify")
    return out
