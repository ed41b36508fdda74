"""Norm and rotation of query heads, and of new rows on their way into a paged cache.

The attention calls take queries whose rotary dims are rotated already and caches whose rows
somebody wrote. These two make them, each in one pass over the data, in the HIP library:

* ``norm_rope_heads``  the heads of a batch of tokens (``sas_norm_rope``)
* ``append_kv_rope``   new rows into a bf16 / fp16 cache, a cache of 656-byte fp8 rows
                       (``kv_fp8``) or fp8 index pages (``sas_kv_append_rope``)

A row ``x`` of ``D`` dims becomes ``x[d] * w[d] / sqrt(mean(x[:N]**2) + eps)`` for ``d < N``
(``N = norm_weight.numel()``, the other dims as they are), then the dims
``[rope_offset, rope_offset + R)`` are rotated by the angles of the row's position. All of it is
in fp32 and rounded once, to the output's type. Inputs that require a gradient are refused: the
library has no backward pass.

fp8 index pages (``[blocks, block_size, 1, D + 4]`` uint8) hold, for a page of ``block_size``
rows, their ``block_size * D`` e4m3 codes and behind those their fp32 scales, one per row
(``amax / 448``, 1 for a zero row).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_FP8_TYPES = (torch.uint8, torch.float8_e4m3fn)
INDEX_DIMS = (64, 128)


def no_grad_inputs(who: str, *tensors) -> None:
    """Refuse inputs whose gradient the caller would silently not get."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{who} has no backward pass: call it under torch.no_grad()")


def launch_on(dev: torch.device, entry, args) -> None:
    """Enqueue a library call on the current stream of ``dev``."""
    if torch.cuda.current_device() == dev.index:
        rc = entry(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = entry(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    if rc != _lib.SAS_OK:
        raise RuntimeError(_lib.last_error())


def _device_int32(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != dev:
        t = t.to(device=dev, dtype=torch.int32)
    return t.reshape(-1).contiguous()


def _common(who: str, x: torch.Tensor, tokens: int, positions: Optional[torch.Tensor],
            cos_sin: Optional[torch.Tensor], norm_weight: Optional[torch.Tensor], norm_eps: float,
            rope_offset: Optional[int], interleaved: bool) -> Tuple[_lib.SasRowArgs, list]:
    """The arguments both calls share, checked, and the tensors behind their pointers."""
    no_grad_inputs(who, x, cos_sin, norm_weight)
    d, dev = x.shape[-1], x.device
    if x.dtype not in _DTYPES:
        raise ValueError(f"{who}: rows must be bf16 or fp16 (got {x.dtype})")
    if d % 8 or not 8 <= d <= _lib.ROW_MAX_DIM:
        raise ValueError(f"{who}: the row width must be a multiple of 8 up to {_lib.ROW_MAX_DIM} "
                         f"(got {d})")
    a = _lib.SasRowArgs()
    keep = []
    a.tokens, a.dim, a.dtype, a.eps = tokens, d, _DTYPES[x.dtype], norm_eps
    a.interleaved = int(bool(interleaved))
    if norm_weight is not None:
        n = norm_weight.numel()
        if norm_weight.dim() != 1 or n % 8 or not 8 <= n <= d:
            raise ValueError(f"{who}: norm_weight must have a multiple of 8 entries up to the row "
                             f"width {d} (got {tuple(norm_weight.shape)})")
        if norm_weight.dtype not in (torch.float32, x.dtype):
            raise ValueError(f"{who}: norm_weight must be fp32 or the rows' type")
        if norm_weight.device != dev:
            raise ValueError(f"{who}: all tensors must be on the rows' device")
        norm_weight = _aligned(norm_weight.contiguous())
        a.norm_weight, a.norm_dim = norm_weight.data_ptr(), n
        a.norm_weight_fp32 = int(norm_weight.dtype == torch.float32)
        keep.append(norm_weight)
    if (cos_sin is None) != (positions is None):
        raise ValueError(f"{who}: positions and cos_sin belong together")
    if cos_sin is not None:
        if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or cos_sin.shape[0] < 1:
            raise ValueError(f"{who}: cos_sin must be fp32 [positions, rotated dims]")
        r = cos_sin.shape[1]
        off = d - r if rope_offset is None else int(rope_offset)
        if r % (8 if interleaved else 16) or r < 8 or off % 8 or off < 0 or off + r > d:
            raise ValueError(
                f"{who}: cannot rotate dims [{off}, {off + r}) of {d}: the offset must be a multiple "
                "of 8 and their number of 8 (interleaved pairs) or 16 (halves)")
        if positions.numel() != tokens:
            raise ValueError(f"{who}: positions must have one entry for each of {tokens} rows "
                             f"(got {positions.numel()})")
        if cos_sin.device != dev:
            raise ValueError(f"{who}: all tensors must be on the rows' device")
        cos_sin = _aligned(cos_sin.contiguous())
        positions = _device_int32(positions, dev) if dev.type == "cuda" else positions
        a.positions, a.cos_sin = positions.data_ptr(), cos_sin.data_ptr()
        a.max_position, a.rope_dim, a.rope_offset = cos_sin.shape[0], r, off
        keep += [positions, cos_sin]
    elif rope_offset is not None:
        raise ValueError(f"{who}: rope_offset without cos_sin")
    return a, keep


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` or a copy of it that starts on 16 bytes."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def norm_rope_heads(q: torch.Tensor, *, positions: Optional[torch.Tensor] = None,
                    cos_sin: Optional[torch.Tensor] = None,
                    norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                    rope_offset: Optional[int] = None, interleaved: bool = True,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RMS norm and rotation of every head of ``q`` ``[..., H, D]`` (bf16 / fp16).

    ``norm_weight``: ``[N]`` (fp32 or q's type); the first ``N`` dims of each head are
    normalised. ``positions``: one entry per token (``q.shape[:-2]`` flattened); ``cos_sin``:
    ``[max_position, R]`` fp32, ``R / 2`` cosines and then ``R / 2`` sines of each position;
    dims ``[rope_offset, rope_offset + R)`` are rotated (default: the last ``R``), in pairs
    ``(2i, 2i + 1)`` when ``interleaved``, else ``(i, i + R / 2)``. A position outside the table
    gives NaN in the rotated dims. Either part may be left out. ``out``: where the result
    goes (``q`` itself is allowed: dims that nothing changes are then not touched).
    """
    who = "norm_rope_heads"
    if q.dim() < 2:
        raise ValueError(f"{who}: q must be [..., heads, head dim] (got {tuple(q.shape)})")
    h, d = q.shape[-2], q.shape[-1]
    if h < 1:
        raise ValueError(f"{who}: q has no heads")
    tokens = q.numel() // (h * d) if d else 0
    a, keep = _common(who, q, tokens, positions, cos_sin, norm_weight, norm_eps, rope_offset,
                      interleaved)
    if tokens * h >= 1 << 31:
        raise ValueError(f"{who}: 2^31 heads or more in one call")
    if out is not None:
        no_grad_inputs(who, out)
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"{who}: out must have q's shape, type and device")
    if q.device.type != "cuda":
        raise RuntimeError(f"{who} runs on a ROCm GPU; q is on {q.device}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    x, y = _token_view(q, h, d), _token_view(out, h, d)
    if y is None:
        raise ValueError(f"{who}: out must have heads of contiguous dims aligned to 16 bytes, its "
                         "tokens one stride apart")
    if x is None:
        x = q.reshape(tokens, h, d).contiguous()
        x = _aligned(x)
    elif x.data_ptr() != y.data_ptr() or x.stride() != y.stride():
        _no_overlap(who, x, y)
    if tokens == 0:
        return out
    a.heads = h
    if x.data_ptr() == y.data_ptr() and not a.norm_dim:
        # in place: only the rotated dims are read and written
        if not a.rope_dim:
            return out
        x = y = x[..., a.rope_offset:a.rope_offset + a.rope_dim]
        a.dim, a.rope_offset = a.rope_dim, 0
    a.x, a.out = x.data_ptr(), y.data_ptr()
    a.x_token_stride, a.x_head_stride = x.stride(0), x.stride(1)
    a.out_token_stride, a.out_head_stride = y.stride(0), y.stride(1)
    launch_on(q.device, _lib.load().sas_norm_rope, a)
    del keep
    return out


def _token_view(t: torch.Tensor, h: int, d: int) -> Optional[torch.Tensor]:
    """``t`` as ``[tokens, h, d]`` without a copy, as the kernel can read it, or None."""
    try:
        v = t if t.dim() == 3 else t.view(-1, h, d)
    except RuntimeError:
        return None
    if d > 1 and v.stride(2) != 1 or v.data_ptr() % 16:
        return None
    if v.shape[0] > 1 and v.stride(0) % 8 or h > 1 and v.stride(1) % 8:
        return None
    return v


def _no_overlap(who: str, x: torch.Tensor, y: torch.Tensor) -> None:
    """Refuse an ``out`` that shares memory with ``q`` other than by being it."""
    if x.numel() == 0 or x.untyped_storage().data_ptr() != y.untyped_storage().data_ptr():
        return
    spans = []
    for t in (x, y):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        spans.append((t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()))
    if spans[0][0] < spans[1][1] and spans[1][0] < spans[0][1]:
        raise ValueError(f"{who}: out overlaps q without being q")


def append_kv_rope(cache: torch.Tensor, kv: torch.Tensor, slot_mapping: torch.Tensor, *,
                   positions: Optional[torch.Tensor] = None,
                   cos_sin: Optional[torch.Tensor] = None,
                   norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                   rope_offset: Optional[int] = None, interleaved: bool = True) -> None:
    """Normalise and rotate ``kv`` rows on their way into ``cache`` (in place, asynchronous).

    ``kv``: ``[n, D]`` or ``[n, 1, D]`` bf16 / fp16. ``slot_mapping``: ``[n]`` int, flat row index
    ``block * block_size + offset``; negative entries and entries past the pool are skipped, two
    rows with one slot leave unspecified contents there. The norm and the rotation are those of
    ``norm_rope_heads``; either may be left out.

    ``cache`` ``[blocks, block_size, 1, width]``, contiguous, decides the format: kv's type with
    ``width = D``; uint8 / float8_e4m3fn with 656 bytes a row for ``D = 576`` bf16 rows (the
    format of ``append_kv_fp8``, quantized from the fp32 result); uint8 / float8_e4m3fn with
    ``width = D + 4`` for fp8 index pages, ``D`` 64 or 128. Runs on the current stream of the
    cache's device.
    """
    who = "append_kv_rope"
    if kv.dim() not in (2, 3) or (kv.dim() == 3 and kv.shape[1] != 1):
        raise ValueError(f"{who}: kv must be [n, D] or [n, 1, D] (got {tuple(kv.shape)})")
    n, d = kv.shape[0], kv.shape[-1]
    a, keep = _common(who, kv, n, positions, cos_sin, norm_weight, norm_eps, rope_offset,
                      interleaved)
    if cache.dim() != 4 or cache.shape[2] != 1:
        raise ValueError(f"{who}: cache must be [blocks, block_size, 1, width] "
                         f"(got {tuple(cache.shape)})")
    if not cache.is_contiguous():
        raise ValueError(f"{who}: cache must be contiguous (it is written in place)")
    blocks, block_size, _, width = cache.shape
    if cache.dtype in _FP8_TYPES:
        if width == _lib.FP8_ROW_BYTES and d == 576 and kv.dtype == torch.bfloat16:
            a.row_format = _lib.ROW_FP8_DS_MLA
        elif width == d + 4 and d in INDEX_DIMS:
            a.row_format = _lib.ROW_FP8_INDEX
            if block_size * width % 16:
                raise ValueError(f"{who}: fp8 index pages must be a multiple of 16 bytes "
                                 f"(block_size {block_size})")
        else:
            raise ValueError(f"{who}: an fp8 cache has rows of {_lib.FP8_ROW_BYTES} bytes for 576 "
                             f"bf16 dims, or of D + 4 for D in {INDEX_DIMS} (got width {width} for "
                             f"{d} dims of {kv.dtype})")
    elif cache.dtype != kv.dtype or width != d:
        raise ValueError(f"{who}: a native cache has kv's type and width (got {cache.dtype} of "
                         f"{width} for {kv.dtype} of {d})")
    if slot_mapping.numel() != n:
        raise ValueError(f"{who}: slot_mapping must have one entry per kv row")
    if slot_mapping.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{who}: slot_mapping must be int32 or int64")
    if blocks * block_size >= 1 << 31:
        raise ValueError(f"{who}: 2^31 cache rows or more")
    if cache.device.type != "cuda" or kv.device != cache.device:
        raise RuntimeError(f"{who} runs on a ROCm GPU; cache and kv must share it")
    if cache.data_ptr() % 16:
        raise ValueError(f"{who}: cache must be aligned to 16 bytes")
    if n == 0 or cache.numel() == 0:
        return
    rows = kv.reshape(n, d) if kv.dim() == 3 else kv
    if (rows.stride(1) != 1 or (n > 1 and rows.stride(0) % 8) or rows.data_ptr() % 16):
        rows = _aligned(rows.contiguous())
    if slot_mapping.dtype == torch.int64:
        # (a slot past int32 is past the pool; narrowing alone could bring it back inside)
        slot_mapping = slot_mapping.clamp(-1, (1 << 31) - 1)
    slots = _device_int32(slot_mapping, cache.device)
    keep += [rows, slots]
    a.heads, a.x, a.out, a.slots = 1, rows.data_ptr(), cache.data_ptr(), slots.data_ptr()
    a.x_token_stride = rows.stride(0)
    a.cache_rows, a.block_size = blocks * block_size, block_size
    launch_on(cache.device, _lib.load().sas_kv_append_rope, a)
    del keep
