"""``sparse_topk_indices``: the rows that sparse attention should read, by a cheap score.

The attention takes ``cmp_sparse_indices``, the compressed rows each query row attends. This
chooses them: a few narrow index heads score every causal row of a paged index cache, and the
ids of the best ``topk`` come back in the form the attention takes. No reference counterpart
(the ids are an input there, api.py:137).
"""

from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib
from .rows import _DTYPES, _FP8_TYPES, INDEX_DIMS, _plain, device_int32, launch_on, no_grad_inputs


@functools.lru_cache(maxsize=256)
def _workspace_bytes(sizes: tuple) -> int:
    """Workspace of a call with these sizes (the int32 fields of ``SasSelectArgs``)."""
    need = _lib.load().sas_topk_select_workspace(_lib.pack_select_args(*[0] * 9, *sizes))
    if need < 0:
        raise RuntimeError(_lib.last_error())
    return need


def sparse_topk_indices(q_index: torch.Tensor, *, weights: torch.Tensor, index_k: torch.Tensor,
                        index_block_table: torch.Tensor, seqused_kv: torch.Tensor, topk: int,
                        cu_seqlens_q: Optional[torch.Tensor] = None,
                        cmp_ratio: Optional[int] = None, layout_q: str = "TND",
                        max_seqlen_kv: Optional[int] = None) -> torch.Tensor:
    """Ids of the ``topk`` best index rows of each query row: a ``cmp_sparse_indices``.

    Query row ``t`` at causal position ``p`` (its sequence's last row is at ``seqused_kv - 1``, as in
    ``sparse_attn_sharedkv``) scores the index rows ``j < (p + 1) // cmp_ratio``:

        ``s(t, j) = scale_j * sum_h weights[t, h] * max(0, q_index[t, h] . index_k[j])``

    ``q_index``: ``[T, H, D]`` (TND, with ``cu_seqlens_q``) or ``[B, S, H, D]`` (BSND; with
    ``cu_seqlens_q`` only the first rows of each sequence are in use), bf16 / fp16, ``H`` up to 128,
    ``D`` 64 or 128. ``weights``: ``q_index.shape[:-1]``. ``index_k``: ``[blocks, block_size, 1, D]``
    of q's type, or fp8 index pages ``[blocks, block_size, 1, D + 4]`` uint8 (``append_kv_rope``
    writes both). ``index_block_table``: ``[>= B, table_len]``; a row on a page outside the pool is
    never chosen. ``cmp_ratio``: raw rows per index row, as in ``sparse_attn_sharedkv`` (default 4,
    api.py:287). ``max_seqlen_kv``: no sequence is longer (saves workspace where the table is
    wide; index rows from ``max_seqlen_kv // cmp_ratio`` on are not looked at).

    Returns int32 ``[T, 1, topk]`` / ``[B, S, 1, topk]``: ascending ids, ``-1`` behind the last
    (the whole row for a query row with nothing to attend, or of no sequence). The choice
    is that of scores in 64 bits, the lowest ids among equal ones, so it does not change with the
    batch or the split of the work; NaN scores rank lowest. Runs on the current stream of
    ``q_index``'s device, never waits for it, and may be captured in a HIP graph.
    """
    assert layout_q in ("TND", "BSND"), f"unsupported layout_q={layout_q!r}"
    no_grad_inputs("sparse_topk_indices", q_index, weights, index_k)
    dtype = q_index.dtype
    if dtype not in _DTYPES:
        raise ValueError(f"unsupported torch dtype {dtype}")
    if layout_q == "TND":
        assert cu_seqlens_q is not None, "cu_seqlens_q is required for TND"
        if q_index.dim() != 3:
            raise ValueError(f"TND q_index must be [T, H, D], got {tuple(q_index.shape)}")
        nb, rows_per_seq, total = cu_seqlens_q.numel() - 1, 0, q_index.shape[0]
        if nb < 0:
            raise ValueError("cu_seqlens_q must have batch + 1 entries")
    else:
        if q_index.dim() != 4:
            raise ValueError(f"BSND q_index must be [B, S, H, D], got {tuple(q_index.shape)}")
        nb, rows_per_seq = q_index.shape[:2]
        total = nb * rows_per_seq
        if cu_seqlens_q is not None and cu_seqlens_q.numel() != nb + 1:
            raise ValueError(f"cu_seqlens_q must have {nb + 1} entries")
    h, d = q_index.shape[-2:]
    k = int(topk)
    ratio = int(cmp_ratio) if cmp_ratio is not None else 4  # api.py:287
    if not 1 <= h <= _lib.SELECT_MAX_HEADS or d not in INDEX_DIMS:
        raise ValueError(f"index heads: 1 to {_lib.SELECT_MAX_HEADS} of {INDEX_DIMS} dims "
                         f"(got {h} of {d})")
    if k < 1:
        raise ValueError("topk must be >= 1")
    if ratio < 1:
        raise ValueError("cmp_ratio must be >= 1")
    if weights.shape != q_index.shape[:-1]:
        raise ValueError(f"weights must be {tuple(q_index.shape[:-1])} (got {tuple(weights.shape)})")
    if not weights.is_floating_point():
        raise ValueError("weights must be floating point")
    fp8 = index_k.dtype in _FP8_TYPES
    if index_k.dim() != 4 or index_k.shape[2] != 1 or index_k.shape[3] != (d + 4 if fp8 else d):
        raise ValueError(f"index_k must be [blocks, block_size, 1, {d}], or {d + 4} bytes a row in "
                         f"fp8 (got {tuple(index_k.shape)})")
    if not fp8 and index_k.dtype != dtype:
        raise ValueError("index_k must have q_index's dtype, or be fp8 pages")
    blocks, block_size = index_k.shape[:2]
    if blocks < 1 or block_size < 1:
        raise ValueError("index_k has no rows")
    if blocks * block_size >= 1 << 31:
        raise ValueError("index_k has 2^31 rows or more")
    if fp8 and block_size * (d + 4) % 16:
        raise ValueError(f"fp8 index pages must be a multiple of 16 bytes (block_size {block_size})")
    if index_block_table.dim() != 2 or index_block_table.shape[0] < nb or \
            index_block_table.shape[1] < 1:
        raise ValueError(f"index_block_table must be [>= {nb}, table_len] "
                         f"(got {tuple(index_block_table.shape)})")
    if seqused_kv.numel() < nb:
        raise ValueError(f"seqused_kv has {seqused_kv.numel()} entries for {nb} sequences")
    max_keys = index_block_table.shape[1] * block_size
    if max_seqlen_kv is not None:
        if max_seqlen_kv < 0:
            raise ValueError("max_seqlen_kv must be >= 0")
        max_keys = min(max_keys, max(int(max_seqlen_kv) // ratio, 1))
    if max_keys > _lib.SELECT_MAX_KEYS:
        raise ValueError(f"more than {_lib.SELECT_MAX_KEYS} index rows a sequence: pass max_seqlen_kv")
    if total >= 1 << 31 or total * k >= 1 << 40:
        raise ValueError("too many query rows in one call")

    dev = q_index.device
    if not q_index.is_cuda:
        raise RuntimeError("sparse_topk_indices runs on a ROCm GPU; q_index is on " + str(dev))
    if index_k.device != dev or weights.device != dev:
        raise ValueError("all tensors must be on q_index's device")
    i32 = torch.int32
    q, keys = _plain(q_index), _plain(index_k)
    w = weights if weights.dtype == torch.float32 else weights.float()
    if not w.is_contiguous():
        w = w.contiguous()
    table, lens = device_int32(index_block_table, dev), device_int32(seqused_kv, dev)
    cu = None if cu_seqlens_q is None else device_int32(cu_seqlens_q, dev)
    out = torch.empty((*q_index.shape[:-2], 1, k), dtype=i32, device=dev)
    if total == 0:
        return out
    if nb == 0:
        return out.fill_(-1)
    sizes = (nb, total, rows_per_seq, h, d, k, ratio, blocks, block_size, table.shape[1], max_keys,
             _DTYPES[dtype], _lib.ROW_FP8_INDEX if fp8 else _lib.ROW_NATIVE)
    need = _workspace_bytes(sizes)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    packed = _lib.pack_select_args(q.data_ptr(), w.data_ptr(), keys.data_ptr(), table.data_ptr(),
                                   0 if cu is None else cu.data_ptr(), lens.data_ptr(),
                                   out.data_ptr(), ws.data_ptr(), need, *sizes)
    launch_on(q_index.get_device(), _lib.load().sas_topk_select, packed)
    return out
