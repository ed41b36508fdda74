"""64-bit answers of the row operators and of the row selection (test infrastructure only).

Written from the formulas, row by row; nothing here is shared with the product package.

* ``norm_rope``       the norm and the rotation of rows
* ``e4m3_rows``       codes and scales of rows quantized with one scale each
* ``index_rows``      a sequence's rows of a paged index cache, native or fp8
* ``select_ids``      the ids ``sparse_topk_indices`` returns
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import torch

E4M3_MAX = 448.0


def norm_rope(x: torch.Tensor, *, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
              angles: Optional[torch.Tensor] = None, offset: int = 0,
              interleaved: bool = True) -> torch.Tensor:
    """``x`` [..., D] in 64 bits; ``angles`` [..., R] (cosines, sines) broadcasts against it."""
    y = x.double().clone()
    if weight is not None:
        n = weight.numel()
        y[..., :n] *= weight.double() / torch.sqrt((y[..., :n] ** 2).mean(-1, keepdim=True) + eps)
    if angles is not None:
        r = angles.shape[-1]
        c, s = angles.double()[..., :r // 2], angles.double()[..., r // 2:]
        first = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
        second = first + 1 if interleaved else first + r // 2
        a, b = y[..., offset + first].clone(), y[..., offset + second].clone()
        y[..., offset + first] = a * c - b * s
        y[..., offset + second] = b * c + a * s
    return y


def e4m3_rows(y: torch.Tensor):
    """Codes (as e4m3 numbers, 64 bits) and scales of ``y`` [n, d], one scale a row."""
    scale = (y.abs().amax(-1, keepdim=True) / E4M3_MAX).float()
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = (y / scale.double()).clamp(-E4M3_MAX, E4M3_MAX)
    return codes.float().to(torch.float8_e4m3fn).double(), scale


def index_pages(rows: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp8 index pages [blocks, bs, 1, d + 4] from codes [blocks, bs, d] and scales [blocks, bs]."""
    blocks, bs, d = rows.shape
    codes = rows.float().to(torch.float8_e4m3fn).view(torch.uint8).reshape(blocks, bs * d)
    tail = scales.float().contiguous().view(torch.uint8).reshape(blocks, bs * 4)
    return torch.cat([codes, tail], dim=1).view(blocks, bs, 1, d + 4)


def index_rows(pool: torch.Tensor, d: int) -> torch.Tensor:
    """All rows [blocks * bs, d] of an index cache in 64 bits."""
    if pool.dtype != torch.uint8:
        return pool.reshape(-1, d).double()
    blocks, bs = pool.shape[:2]
    flat = pool.reshape(blocks, -1)
    codes = flat[:, :bs * d].contiguous().view(torch.float8_e4m3fn).float().double()
    scale = flat[:, bs * d:].contiguous().view(torch.float32).double()
    return (codes.view(blocks, bs, d) * scale.view(blocks, bs, 1)).view(-1, d)


def select_row(q: torch.Tensor, w: torch.Tensor, rows: torch.Tensor, ids: Sequence[int],
               k: int) -> List[int]:
    """The ids of the ``k`` best of ``rows`` [n, d], which are index rows ``ids``, ascending."""
    if len(ids) <= k:
        return sorted(ids)
    score = torch.zeros(len(ids), dtype=torch.float64)
    for h in range(q.shape[0]):
        dot = (rows * q[h]).sum(1)
        score = score + w[h] * torch.where(dot < 0, torch.zeros_like(dot), dot)
    vals = score.tolist()
    low = float("-inf")
    key = [low if v != v else v for v in vals]
    order = sorted(range(len(ids)), key=lambda i: (-key[i], ids[i]))
    return sorted(ids[i] for i in order[:k])


def select_ids(q_index, weights, index_k, index_block_table, seqused_kv, topk, cmp_ratio=1,
               cu_seqlens_q=None, layout_q="TND", max_seqlen_kv=None) -> torch.Tensor:
    """What ``sparse_topk_indices`` returns, from CPU tensors, row by row in 64 bits."""
    h, d = q_index.shape[-2:]
    blocks, bs = index_k.shape[:2]
    q, w = q_index.reshape(-1, h, d).double(), weights.reshape(-1, h).double()
    pool = index_rows(index_k, d)
    out = torch.full((q.shape[0], topk), -1, dtype=torch.int32)
    width = index_block_table.shape[1] * bs
    if max_seqlen_kv is not None:
        width = min(width, max(max_seqlen_kv // cmp_ratio, 1))
    nb = (q_index.shape[0] if layout_q == "BSND" else cu_seqlens_q.numel() - 1)
    for b in range(nb):
        if layout_q == "BSND":
            s_max = q_index.shape[1]
            first = b * s_max
            rows = s_max if cu_seqlens_q is None else int(cu_seqlens_q[b + 1] - cu_seqlens_q[b])
        else:
            first, rows = int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1] - cu_seqlens_q[b])
        page = [int(p) for p in index_block_table[b]]
        for s in range(rows):
            thr = (int(seqused_kv[b]) - rows + s + 1) // cmp_ratio
            ids = [j for j in range(max(min(thr, width), 0)) if 0 <= page[j // bs] < blocks]
            at = torch.tensor([page[j // bs] * bs + j % bs for j in ids], dtype=torch.long)
            got = select_row(q[first + s], w[first + s], pool[at] if ids else pool[:0], ids, topk)
            out[first + s, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out.view(*q_index.shape[:-2], 1, topk)
