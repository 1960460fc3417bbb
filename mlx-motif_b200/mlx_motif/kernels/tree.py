"""Attention for a tree of drafted tokens over a KV cache: ``sdpa_dual_v_tree`` and ``sdpa_dual_v_tree_q4``.

``sdpa_dual_v`` / ``sdpa_dual_v_q4`` (``kernels/attention.py``) for the T query rows of a verify forward: the
drafted rows are the cache's last T live rows, every row sees the context before them and, among them, the
rows its mask names (its ancestors and itself; causal without a mask). The reference verifies chains only, as
causal prompt blocks; same shapes, runtime ``kv_len`` and assertion style as the decode operators otherwise.
"""

from __future__ import annotations

import ctypes
import functools
import math
import struct

import torch

from .._native import motif_tree_kv
from ._common import _DISABLE, check, contiguous, dtype_code, lib, on_device, ptr, stream, workspace

MAX_TREE_ROWS = 256


def tree_mask_from_parents(parents: torch.Tensor) -> torch.Tensor:
    """(T,) or (B, T) parent rows (``parents[..., 0]`` ignored, every other parent before its child) ->
    the boolean (…, T, T) mask of each row's ancestors and itself, on ``parents``' device."""
    T = parents.shape[-1]
    eye = torch.eye(T, dtype=torch.bool, device=parents.device)
    up = parents.long().clone()
    up[..., 0] = -1
    link = (up[..., :, None] == torch.arange(T, device=parents.device)).float()  # link[i, j]: j is i's parent
    mask = (eye.float() + link).expand(*parents.shape, T)
    for _ in range(max(1, math.ceil(math.log2(max(T, 2))))):  # paths of up to 1, 2, 4, … steps
        mask = (mask @ mask).clamp_max(1.0)
    return mask > 0


def sdpa_dual_v_tree_reference(q, k, v1, v2, scale, kv_len=None, tree_mask=None):
    """Torch composition (fp32 math, result in q.dtype)."""
    B, HQ, T, D = q.shape
    cap = k.shape[2]
    n = _lengths(kv_len, cap, B, q.device)
    pos = torch.arange(cap, device=q.device)
    j = pos - (n[:, None] - T)  # (B, cap): tree row of a cache row
    if tree_mask is None:
        tree_mask = torch.ones((T, T), dtype=torch.bool, device=q.device).tril()
    m = tree_mask.bool().expand(B, T, T)
    seen = torch.gather(m, 2, j.clamp(0, T - 1)[:, None, :].expand(B, T, cap))
    seen = (seen | (j < 0)[:, None, :]) & (pos < n[:, None])[:, None, :]
    gqa = HQ // k.shape[1]
    k, v1, v2 = (t.float().repeat_interleave(gqa, dim=1) for t in (k, v1, v2))
    s = torch.matmul(q.float(), k.transpose(-1, -2)) * scale
    s = s.masked_fill(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    den = p.sum(-1, keepdim=True)
    p = p / torch.where(den == 0, 1.0, den)
    out = []
    for v in (v1, v2):
        finite = torch.isfinite(v)
        o = torch.matmul(p, torch.where(finite, v, 0.0))
        # a row that a query does not see may hold anything: infinities and NaN go to those that see it, row by row
        for c in (~finite).any(-1).any(0).any(0).nonzero()[:, 0].tolist():
            rest = torch.where(finite[:, :, c], 0.0, v[:, :, c])[:, :, None]
            o = o + torch.where(seen[:, None, :, c, None], p[..., c, None] * rest, 0.0)
        out.append(o)
    return torch.cat(out, dim=-1).to(q.dtype)


def _lengths(kv_len, cap: int, B: int, device) -> torch.Tensor:
    if isinstance(kv_len, torch.Tensor):
        return kv_len.to(torch.int64).clamp(0, cap).expand(B)
    return torch.full((B,), cap if kv_len is None else int(kv_len), dtype=torch.int64, device=device)


def sdpa_dual_v_tree_q4_reference(q, k_q, v1_q, v2_q, scale, group_size: int = 64, bits: int = 4, kv_len=None,
                                  tree_mask=None):
    """Dequantize K, V1, V2, then the tree reference."""
    from .attention import _dequantize_triple

    k, v1, v2 = (_dequantize_triple(t, group_size, bits, q.dtype) for t in (k_q, v1_q, v2_q))
    return sdpa_dual_v_tree_reference(q, k, v1, v2, scale, kv_len, tree_mask)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous on a 16-byte boundary (a copy where it is not)."""
    t = contiguous(t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _row_strides(t: torch.Tensor):
    """(batch, head, row) element strides of a (B, H, cap, D) view whose rows the kernels can read in place,
    else None. A dimension of one entry has the stride it would have in a contiguous tensor."""
    B, H, cap, D = t.shape
    unit = 16 // t.element_size()
    sb, sh, sr, sd = t.stride()
    sr = sr if cap > 1 else D
    sh = sh if H > 1 else cap * sr
    sb = sb if B > 1 else H * sh
    if sd != 1 or sr < D or sr % unit or sh % unit or sb % unit or min(sh, sb) <= 0 or t.data_ptr() % 16:
        return None
    return sb, sh, sr


def _check_q(q, shape_kv, name: str):
    B, HQ, T, D = q.shape
    HKV, cap = shape_kv[1], shape_kv[2]
    assert D % 32 == 0, f"D={D} must be a multiple of 32"
    assert HKV >= 1 and HQ >= 1 and HQ % HKV == 0, f"H_q={HQ} must be a multiple of H_kv={HKV}"
    assert 1 <= T <= MAX_TREE_ROWS, f"{name} takes 1..{MAX_TREE_ROWS} tree rows, got {T}"
    return B, HQ, T, D, HKV, cap


def _check_len(kv_len, B: int, T: int, cap: int, device):
    """(host length, device pointer, stride)."""
    if kv_len is None:
        kv_len = cap
    if isinstance(kv_len, torch.Tensor):
        if kv_len.dtype != torch.int32 or not kv_len.is_cuda or kv_len.numel() not in (1, B) or not kv_len.is_contiguous():
            raise TypeError(f"a device kv_len must be a contiguous int32 CUDA tensor of 1 or {B} elements")
        _check_device(kv_len, device)
        return 0, kv_len.data_ptr(), int(kv_len.numel() > 1)
    n = int(kv_len)
    assert T <= n <= cap, f"kv_len={n} must be in [{T}, {cap}]"
    return n, None, 0


def _check_mask(mask, B: int, T: int, device):
    """(mask kept alive, batch stride)."""
    if mask is None:
        return None, 0
    if mask.dtype != torch.bool:
        raise TypeError(f"tree_mask must be a bool tensor, got {mask.dtype}")
    assert mask.shape == (T, T) or mask.shape == (B, T, T), f"tree_mask {tuple(mask.shape)} must be ({T}, {T}) or ({B}, {T}, {T})"
    _check_device(mask, device)
    return contiguous(mask), T * T if mask.dim() == 3 else 0


def _check_device(t: torch.Tensor, device) -> None:
    if t.device != device:
        raise ValueError(f"tensors on {t.device} and {device}: all operands must be on one CUDA device")


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index, *shape) -> int:
    return lib.motif_sdpa_dual_v_tree_workspace_bytes(*shape)


_err_words: dict = {}  # device index -> (pinned int32 word, its value through ctypes)


def _err_word(dev) -> int | None:
    """Address of the device's error word, in pinned host memory: a kernel sets it when a pipeline wait runs out, and
    the next call raises without a synchronisation. A first call under capture, where host memory cannot be
    pinned, goes without."""
    known = _err_words.get(dev.index)
    if known is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        word = torch.zeros(1, dtype=torch.int32, pin_memory=True)
        known = _err_words[dev.index] = word, ctypes.c_int32.from_address(word.data_ptr())
    word, value = known
    if value.value:
        value.value = 0
        raise RuntimeError("sdpa_dual_v_tree: a pipeline wait of an earlier call timed out; its rows are NaN")
    return word.data_ptr()


def _launch(q, parts, strides, bits, group_size, scale, HKV, cap, kv_len, tree_mask, name):
    """parts: data, scales, biases of k, v1, v2 in turn (scales and biases None for plain rows)."""
    B, HQ, T, D = q.shape
    dev = q.device
    code = dtype_code(q)
    for t in parts:
        if t is not None and t.device != dev:
            _check_device(t, dev)
    n, n_dev, n_step = _check_len(kv_len, B, T, cap, dev)
    mask, mask_b = _check_mask(tree_mask, B, T, dev)
    y = q.new_empty((B, HQ, T, 2 * D))
    if B == 0 or cap == 0:
        return y.zero_()
    with on_device(dev):
        qc = _aligned(q)
        # motif_tree_kv: data[3], scales[3], biases[3], stride[3]
        at = [0 if t is None else t.data_ptr() for t in parts]
        kv = motif_tree_kv.from_buffer_copy(_KV.pack(*at[0::3], *at[1::3], *at[2::3], *strides))
        ws_bytes = _workspace_bytes(dev.index, code, bits, group_size, B, HQ, HKV, T, cap, D, cap if n_dev else n, 1 - n_step)
        ws = workspace(ws_bytes, dev) if ws_bytes else None
        err = _err_word(dev)
        check(lib.motif_sdpa_dual_v_tree(code, bits, group_size, qc.data_ptr(), kv, ptr(mask), mask_b, float(scale), B, HQ,
                                         HKV, T, cap, D, n, n_dev, n_step, y.data_ptr(), ptr(ws), ws_bytes, err,
                                         stream(dev)), name)
    return y


_KV = struct.Struct("12q")


def sdpa_dual_v_tree(q: torch.Tensor, k: torch.Tensor, v1: torch.Tensor, v2: torch.Tensor, scale: float, kv_len=None,
                     tree_mask: torch.Tensor | None = None) -> torch.Tensor:
    """Shared-QK, dual-V SDPA of the T rows of a drafted tree with native GQA broadcast.

    q (B, H_q, T, D); k, v1, v2 (B, H_kv, KV_cap, D), read in place where their rows are 16-byte aligned
    (head and batch strides as they are). The tree's rows are cache rows [kv_len − T, kv_len), already
    appended; ``kv_len`` (default KV_cap) is an int, or an int32 CUDA tensor of one length or one per
    sequence (read on the device). ``tree_mask`` (T, T) or (B, T, T) bool: row t sees tree row j where
    tree_mask[t, j]; None is causal. Every row sees the rows before the tree. Returns (B, H_q, T, 2·D) =
    cat([SDPA(q,k,v1), SDPA(q,k,v2)], axis=-1), zeros for a row that sees nothing. A kernel whose pipeline stalls
    for half a second gives NaN rows; the next call on the device then raises RuntimeError.
    """
    if _DISABLE:
        return sdpa_dual_v_tree_reference(q, k, v1, v2, scale, kv_len, tree_mask)
    B, HQ, T, D, HKV, cap = _check_q(q, k.shape, "sdpa_dual_v_tree")
    assert k.shape == v1.shape == v2.shape == (B, HKV, cap, D), "k, v1, v2 must match (B, H_kv, KV_cap, D)"
    if not k.dtype == v1.dtype == v2.dtype == q.dtype:
        k, v1, v2 = (t.to(q.dtype) for t in (k, v1, v2))
    if k.is_contiguous() and v1.is_contiguous() and v2.is_contiguous() and \
            (k.data_ptr() | v1.data_ptr() | v2.data_ptr()) % 16 == 0:
        strides = (HKV * cap * D, cap * D, D)
    else:
        strides = _row_strides(k)
        if strides is None or _row_strides(v1) != strides or _row_strides(v2) != strides:
            k, v1, v2 = (_aligned(t) for t in (k, v1, v2))
            strides = (HKV * cap * D, cap * D, D)
    return _launch(q, (k, None, None, v1, None, None, v2, None, None), strides, 16, 64, scale, HKV, cap, kv_len, tree_mask,
                   "sdpa_dual_v_tree")


def sdpa_dual_v_tree_q4(q: torch.Tensor, k_q: tuple, v1_q: tuple, v2_q: tuple, scale: float, group_size: int = 64,
                        bits: int = 4, kv_len=None, tree_mask: torch.Tensor | None = None) -> torch.Tensor:
    """``sdpa_dual_v_tree`` over a packed cache: k_q, v1_q, v2_q are ``(data uint32, scales, biases)``
    triples of (B, H_kv, KV_cap, D) tensors in the MLX affine layout (bits 4 or 8)."""
    if _DISABLE:
        return sdpa_dual_v_tree_q4_reference(q, k_q, v1_q, v2_q, scale, group_size, bits, kv_len, tree_mask)
    assert bits in (4, 8), f"bits={bits} must be 4 or 8"
    B, HQ, T, D, HKV, cap = _check_q(q, k_q[0].shape, "sdpa_dual_v_tree_q4")
    n_uint = k_q[0].shape[3]
    assert n_uint * (32 // bits) == D, f"k_data last axis = {n_uint} ⇒ packed D = {n_uint * (32 // bits)}, expected {D}"
    assert group_size >= 8 and group_size % 8 == 0 and D % group_size == 0, \
        f"group_size={group_size} must be a multiple of 8 that divides D={D}"
    parts = []
    for data, scales, biases in (k_q, v1_q, v2_q):
        assert data.shape == (B, HKV, cap, n_uint), "k, v1, v2 data must match (B, H_kv, KV_cap, D·bits/32)"
        assert scales.shape == biases.shape == (B, HKV, cap, D // group_size), \
            "scales and biases must match (B, H_kv, KV_cap, D/group_size)"
        if data.dtype not in (torch.uint32, torch.int32):
            raise TypeError(f"packed data must be uint32, got {data.dtype}")
        parts += [_aligned(t) for t in (data, scales.to(q.dtype), biases.to(q.dtype))]
    return _launch(q, parts, (0, 0, 0), bits, int(group_size), scale, HKV, cap, kv_len, tree_mask, "sdpa_dual_v_tree_q4")
