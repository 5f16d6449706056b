"""Paged key / value cache operators of the serving path (csrc/llm/paged_append.cu, csrc/llm/paged_attention.cu).

A cache layer is a pair of tensors ``k_pages``, ``v_pages`` of shape ``[n_pages, kv_heads, page, head_dim]`` (fp16 or bf16,
any page and head strides, ``head_dim`` contiguous) and an int32 ``block_table [n_seq, max_pages]``: position ``p`` of
sequence ``s`` is row ``p % page`` of page ``block_table[s, p // page]``.  Entries of pages that no position uses are
never read.  Indices live on the device, so they are checked there: a sequence, position, length or page out of range is
reported by ``_native.check_status()`` and its access skipped (its key counts as masked).  Sequence ``-1`` marks a padded token: it
appends nothing, and its output rows are zero.

On CPU tensors (fp32 included) the same functions run in plain PyTorch.  The reference has no cached attention
(example-cli/src/model/transformer.rs:221-270 declares a cache that nothing uses).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _native


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 block_table: torch.Tensor, pos: torch.Tensor, seq: Optional[torch.Tensor], inv_freq: torch.Tensor, *,
                 interleaved: bool = False, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates ``q [n, H, D]`` and ``k [n, Hkv, D]``, appends ``k`` and ``v`` to the cache, returns the rotated ``q``.

    ``pos``, ``seq``: int32 ``[n]``, the position and sequence of each token (``seq=None``: token ``t`` is sequence ``t``);
    no position of a sequence may come twice in one call (which of the two stays is undefined).
    ``inv_freq``: fp32 ``[R / 2]``, radians per position of each rotated pair, ``R <= D``; values from ``R`` on pass through.
    Pairs are ``(2i, 2i+1)`` (``interleaved``) or ``(i, i + R/2)``.  ``q_norm`` / ``k_norm [D]``: RMSNorm weights applied
    to every head before the rotation.  ``q_out`` may be ``q`` itself, ``k_out`` (the rotated keys, also in the
    cache) ``k`` itself; other overlaps of inputs and outputs are not allowed.  Inference only: inputs that ask for gradients are refused.
    """
    if k_pages.device.type == "cpu":
        _no_gradients("paged_append", q, k, v, k_pages, v_pages, inv_freq, q_norm, k_norm, q_out, k_out)
        return _append_cpu(q, k, v, k_pages, v_pages, block_table, pos, seq, inv_freq, interleaved, q_norm, k_norm, eps, q_out, k_out)
    return _native.load(required=True).paged_append(q, k, v, k_pages, v_pages, block_table, pos, seq, inv_freq, interleaved, q_norm,
                                                    k_norm, eps, q_out, k_out)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    kv_len: torch.Tensor, seq: Optional[torch.Tensor] = None, *, scale: Optional[float] = None, window: int = 0,
                    softcap: float = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(f(scale q K^T)) V`` of every token over its sequence's cached positions ``[0, kv_len)``.

    ``q [n, H, D]`` (``H`` a multiple of the cache's heads, ``D`` a multiple of 8 up to 256), ``kv_len``, ``seq``: int32 ``[n]``.
    ``window > 0`` keeps the last ``window`` of these positions, ``softcap > 0`` applies
    ``f(x) = softcap tanh(x / softcap)`` (1e-6 to 1e30); ``scale`` defaults to ``1 / sqrt(D)``.  A token that sees no position gets zeros.
    What the cache holds beyond the visible positions (NaN included) does not matter.  Inference only: inputs that ask for gradients are refused.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if k_pages.device.type == "cpu":
        _no_gradients("paged_attention", q, k_pages, v_pages, out)
        return _attention_cpu(q, k_pages, v_pages, block_table, kv_len, seq, scale, window, softcap, out)
    return _native.load(required=True).paged_attention(q, k_pages, v_pages, block_table, kv_len, seq, scale, window, softcap, out)


def _no_gradients(op, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{op} has no backward pass: call it under torch.no_grad()")


def _check_cpu(op, k_pages, v_pages, block_table, n, **indices):
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != k_pages.device:
        raise RuntimeError(f"{op}: k_pages and v_pages must be [n_pages, kv_heads, page, head_dim] alike in size, dtype and device")
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise RuntimeError(f"{op}: block_table must be int32 [n_seq, max_pages]")
    for name, t in indices.items():
        if t is not None and (t.dtype != torch.int32 or t.shape != (n,)):
            raise RuntimeError(f"{op}: {name} must be an int32 tensor of {n} elements")


def _page_of(op, block_table, s, p, page, n_pages):
    """The pages of positions ``p`` of sequence ``s``; bad indices raise here (the kernels record them)."""
    from ..error import IndexOutOfBounds
    if not 0 <= s < block_table.shape[0] or (p.numel() and (int(p.min()) < 0 or int(p.max()) // page >= block_table.shape[1])):
        raise IndexOutOfBounds(f"{op}: sequence {s} or one of its positions is outside the block table")
    pages = block_table[s, p // page].long()
    if pages.numel() and (int(pages.min()) < 0 or int(pages.max()) >= n_pages):
        raise IndexOutOfBounds(f"{op}: the block table of sequence {s} names a page that does not exist")
    return pages


def _append_cpu(q, k, v, k_pages, v_pages, block_table, pos, seq, inv_freq, interleaved, q_norm, k_norm, eps, q_out, k_out):
    op, n, rot = "paged_append", q.shape[0], 2 * inv_freq.numel()
    _check_cpu(op, k_pages, v_pages, block_table, n, pos=pos, seq=seq)
    hkv, page, D = k_pages.shape[1:]
    if q.dim() != 3 or q.shape[2] != D or k.shape != (n, hkv, D) or v.shape != k.shape:
        raise RuntimeError(f"{op}: q must be [n_tok, heads, head_dim], k and v [n_tok, kv heads, head_dim]")
    if rot > D:
        raise RuntimeError(f"{op}: inv_freq must have at most head_dim / 2 elements")
    seq = torch.arange(n, dtype=torch.int32) if seq is None else seq
    ang = pos.double()[:, None, None] * inv_freq.double()
    cs, sn = ang.cos().float(), ang.sin().float()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))

    def turn(x, w):
        y = x.float()
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.float() if w is not None else y.clone()
        a, b = y[..., first].clone(), y[..., second].clone()
        y[..., first], y[..., second] = a * cs - b * sn, a * sn + b * cs
        y[seq == -1] = 0.0
        return y.to(x.dtype)
    qr, kr = turn(q, q_norm), turn(k, k_norm)
    for t in range(n):
        if int(seq[t]) != -1:
            p = int(pos[t])
            pg = int(_page_of(op, block_table, int(seq[t]), pos[t: t + 1].long(), page, k_pages.shape[0])[0])
            k_pages[pg, :, p % page], v_pages[pg, :, p % page] = kr[t], v[t]
    if k_out is not None:
        k_out.copy_(kr)
    return qr if q_out is None else q_out.copy_(qr)


def _attention_cpu(q, k_pages, v_pages, block_table, kv_len, seq, scale, window, softcap, out):
    op, n = "paged_attention", q.shape[0]
    _check_cpu(op, k_pages, v_pages, block_table, n, kv_len=kv_len, seq=seq)
    hkv, page, D = k_pages.shape[1:]
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % hkv:
        raise RuntimeError(f"{op}: q must be [n_tok, heads, head_dim] with a multiple of {hkv} heads")
    if not abs(scale) <= 1e30 or not (softcap == 0 or 1e-6 <= softcap <= 1e30) or window < 0:
        raise RuntimeError(f"{op}: scale must be finite, softcap 0 (none) or from 1e-6 to 1e30, window not negative")
    res = torch.zeros(n, q.shape[1], D, dtype=q.dtype)
    for t in range(n):
        s, length = t if seq is None else int(seq[t]), int(kv_len[t])
        if s == -1 or length == 0:
            continue
        if length < 0:
            from ..error import IndexOutOfBounds
            raise IndexOutOfBounds(f"{op}: negative length")
        at = torch.arange(max(0, length - window) if window else 0, length)
        pages = _page_of(op, block_table, s, at, page, k_pages.shape[0])
        kk = k_pages[pages, :, at % page].float().transpose(0, 1)                # [Hkv, L, D]
        vv = v_pages[pages, :, at % page].float().transpose(0, 1)
        x = (q[t].float().view(hkv, -1, D) @ kk.transpose(1, 2)) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        res[t] = (torch.softmax(x, -1) @ vv).view(-1, D).to(q.dtype)
    return res if out is None else out.copy_(res)
