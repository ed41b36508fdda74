"""Norm and rotation of query heads, and of new rows on their way into a paged cache.

The attention calls take queries whose rotary dims are rotated already and caches whose rows
somebody wrote. These two make them, each in one pass over the data, in the HIP library:

* ``norm_rope_heads``  the heads of a batch of tokens (``sas_norm_rope``)
* ``append_kv_rope``   new rows into a bf16 / fp16 cache, a cache of 656-byte fp8 rows
                       (``kv_fp8``) or fp8 index pages (``sas_kv_append_rope``)

A row ``x`` of ``D`` dims becomes ``x[d] * w[d] / sqrt(mean(x[:N]**2) + eps)`` for ``d < N``
(``N = norm_weight.numel()``, the other dims as they are), then the dims
``[rope_offset, rope_offset + R)`` are rotated by the angles of the row's position. All of it is
in fp32 (in 64 bits for rows that end in fp8) and rounded once, to the output's type. Inputs that require a gradient are refused: the
library has no backward pass.

fp8 index pages (``[blocks, block_size, 1, D + 4]`` uint8) hold, for a page of ``block_size``
rows, their ``block_size * D`` e4m3 codes and behind those their fp32 scales, one per row
(``amax / 448``, 1 for a zero row).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_FP8_TYPES = (torch.uint8, torch.float8_e4m3fn)
INDEX_DIMS = (64, 128)


def no_grad_inputs(who: str, *tensors) -> None:
    """Refuse inputs whose gradient the caller would silently not get."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{who} has no backward pass: call it under torch.no_grad()")


def launch_on(index: int, entry, packed: bytes) -> None:
    """Enqueue a library call on the current stream of GPU ``index``."""
    # (the raw handle: torch.cuda.current_stream makes an object first, 1.5 us of a 10 us call)
    if torch.cuda.current_device() == index:
        rc = entry(packed, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(packed, torch._C._cuda_getCurrentRawStream(index))
    if rc != _lib.SAS_OK:
        raise RuntimeError(_lib.last_error())


def device_int32(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """``t`` as contiguous int32 on ``dev``: itself where it is that already."""
    if t.dtype != torch.int32 or t.device != dev:
        t = t.to(device=dev, dtype=torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _common(who, x, d, tokens, positions, cos_sin, norm_weight, norm_eps, rope_offset, interleaved):
    """The arguments both calls share, checked.

    Returns the tensors behind the pointers (kept alive until the launch) and the values of
    ``SasRowArgs`` that follow from them: (positions, cos_sin, norm_weight pointers), (norm_dim,
    rope_dim, rope_offset, interleaved, max_position, dtype, norm_weight_fp32), eps.
    """
    no_grad_inputs(who, x, cos_sin, norm_weight)
    dtype, dev = x.dtype, x.device
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{who}: rows must be bf16 or fp16 (got {dtype})")
    if d % 8 or not 8 <= d <= _lib.ROW_MAX_DIM:
        raise ValueError(f"{who}: the row width must be a multiple of 8 up to {_lib.ROW_MAX_DIM} "
                         f"(got {d})")
    p_pos = p_cos = p_w = n = r = off = table = w_fp32 = 0
    if norm_weight is not None:
        n = norm_weight.numel()
        if norm_weight.dim() != 1 or n % 8 or not 8 <= n <= d:
            raise ValueError(f"{who}: norm_weight must have a multiple of 8 entries up to the row "
                             f"width {d} (got {tuple(norm_weight.shape)})")
        w_fp32 = int(norm_weight.dtype == torch.float32)
        if not w_fp32 and norm_weight.dtype != dtype:
            raise ValueError(f"{who}: norm_weight must be fp32 or the rows' type")
        if norm_weight.device != dev:
            raise ValueError(f"{who}: all tensors must be on the rows' device")
        norm_weight = _plain(norm_weight)
        p_w = norm_weight.data_ptr()
    if (cos_sin is None) != (positions is None):
        raise ValueError(f"{who}: positions and cos_sin belong together")
    if cos_sin is not None:
        if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or cos_sin.shape[0] < 1:
            raise ValueError(f"{who}: cos_sin must be fp32 [positions, rotated dims]")
        table, r = cos_sin.shape
        off = d - r if rope_offset is None else int(rope_offset)
        if r % (8 if interleaved else 16) or r < 8 or off % 8 or off < 0 or off + r > d:
            raise ValueError(
                f"{who}: cannot rotate dims [{off}, {off + r}) of {d}: the offset must be a multiple "
                "of 8 and their number of 8 (interleaved pairs) or 16 (halves)")
        if table >= 1 << 31:
            raise ValueError(f"{who}: 2^31 positions or more")
        if positions.numel() != tokens:
            raise ValueError(f"{who}: positions must have one entry for each of {tokens} rows "
                             f"(got {positions.numel()})")
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{who}: positions must be int32 or int64")
        if cos_sin.device != dev:
            raise ValueError(f"{who}: all tensors must be on the rows' device")
        if x.is_cuda:
            if positions.dtype == torch.int64:
                positions = _narrow(positions)
            positions = device_int32(positions, dev)
        cos_sin = _plain(cos_sin)
        p_pos, p_cos = positions.data_ptr(), cos_sin.data_ptr()
    elif rope_offset is not None:
        raise ValueError(f"{who}: rope_offset without cos_sin")
    return ((positions, cos_sin, norm_weight), (p_pos, p_cos, p_w),
            (n, r, off, 1 if interleaved else 0, table, code, w_fp32), norm_eps)


def _plain(t: torch.Tensor) -> torch.Tensor:
    """``t`` or a contiguous copy of it that starts on 16 bytes."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _narrow(t: torch.Tensor) -> torch.Tensor:
    """int64 places inside int32: one past it stays out of range instead of coming back inside."""
    return t.clamp(-1, (1 << 31) - 1)


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
    shape = q.shape
    if len(shape) < 2:
        raise ValueError(f"{who}: q must be [..., heads, head dim] (got {tuple(shape)})")
    h, d = shape[-2], shape[-1]
    if h < 1:
        raise ValueError(f"{who}: q has no heads")
    tokens = q.numel() // (h * d) if d else 0
    keep, pointers, (n, r, off, *rest), eps = _common(
        who, q, d, tokens, positions, cos_sin, norm_weight, norm_eps, rope_offset, interleaved)
    if tokens * h >= 1 << 31:
        raise ValueError(f"{who}: 2^31 heads or more in one call")
    if out is not None:
        no_grad_inputs(who, out)
        if out.shape != shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"{who}: out must have q's shape, type and device")
    if not q.is_cuda:
        raise RuntimeError(f"{who} runs on a ROCm GPU; q is on {q.device}")
    x = _token_view(q, h, d)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
        y = (out.data_ptr(), h * d, d)
        if x is None:
            q = _plain(q)
            x = (q.data_ptr(), h * d, d)
    else:
        y = _token_view(out, h, d)
        if y is None:
            raise ValueError(f"{who}: out must have heads of contiguous dims aligned to 16 bytes, "
                             "its tokens one stride apart")
        if _overlaps_itself(tokens, h, d, y):
            raise ValueError(f"{who}: out overlaps itself")
        if x is None:
            _no_overlap(who, q, out)
            q = _plain(q)
            x = (q.data_ptr(), h * d, d)
        elif x != y:
            _no_overlap(who, q, out)
    if tokens == 0:
        return out
    skip = 0
    if x == y and not n:
        # in place: only the rotated dims are read and written
        if not r:
            return out
        skip, d, off = 2 * off, r, 0
    packed = _lib.pack_row_args(x[0] + skip, y[0] + skip, *pointers, 0, x[1], x[2], y[1], y[2], 0,
                                tokens, h, d, n, r, off, *rest, 0, 0, eps, 0)
    launch_on(q.get_device(), _lib.load().sas_norm_rope, packed)
    del keep
    return out


def _token_view(t: torch.Tensor, h: int, d: int) -> Optional[Tuple[int, int, int]]:
    """(address, token stride, head stride) of ``t`` as ``[tokens, h, d]`` as the kernel can read
    it, or None."""
    at = t.data_ptr()
    if at % 16:
        return None
    if t.is_contiguous():
        return at, h * d, d
    if t.dim() != 3:
        try:
            t = t.view(-1, h, d)
        except RuntimeError:
            return None
    tokens, heads, dims = t.stride()
    if dims != 1 or (t.shape[0] > 1 and tokens % 8) or (h > 1 and heads % 8):
        return None
    return at, tokens - tokens % 8, heads - heads % 8  # (strides of one are not used)


def _overlaps_itself(tokens: int, h: int, d: int, view: Tuple[int, int, int]) -> bool:
    _, by_token, by_head = view
    spans = sorted((s, n) for s, n in ((by_token, tokens), (by_head, h)) if n > 1)
    reach = d
    for s, n in spans:
        if s < reach:
            return True
        reach += (n - 1) * s
    return False


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
    format of ``append_kv_fp8``, and its bytes where nothing changes the latent dims); uint8 / float8_e4m3fn with
    ``width = D + 4`` for fp8 index pages, ``D`` 64 or 128. Runs on the current stream of the
    cache's device.
    """
    who = "append_kv_rope"
    shape = kv.shape
    if len(shape) not in (2, 3) or (len(shape) == 3 and shape[1] != 1):
        raise ValueError(f"{who}: kv must be [n, D] or [n, 1, D] (got {tuple(shape)})")
    n_rows, d = shape[0], shape[-1]
    keep, pointers, (n, r, off, *rest), eps = _common(
        who, kv, d, n_rows, positions, cos_sin, norm_weight, norm_eps, rope_offset, interleaved)
    if cache.dim() != 4 or cache.shape[2] != 1:
        raise ValueError(f"{who}: cache must be [blocks, block_size, 1, width] "
                         f"(got {tuple(cache.shape)})")
    if not cache.is_contiguous():
        raise ValueError(f"{who}: cache must be contiguous (it is written in place)")
    blocks, block_size, _, width = cache.shape
    dtype = cache.dtype
    row_format = _lib.ROW_NATIVE
    if dtype in _FP8_TYPES:
        if width == _lib.FP8_ROW_BYTES and d == 576 and kv.dtype == torch.bfloat16:
            row_format = _lib.ROW_FP8_DS_MLA
        elif width == d + 4 and d in INDEX_DIMS:
            row_format = _lib.ROW_FP8_INDEX
            if block_size * width % 16:
                raise ValueError(f"{who}: fp8 index pages must be a multiple of 16 bytes "
                                 f"(block_size {block_size})")
        else:
            raise ValueError(f"{who}: an fp8 cache has rows of {_lib.FP8_ROW_BYTES} bytes for 576 "
                             f"bf16 dims, or of D + 4 for D in {INDEX_DIMS} (got width {width} for "
                             f"{d} dims of {kv.dtype})")
    elif dtype != kv.dtype or width != d:
        raise ValueError(f"{who}: a native cache has kv's type and width (got {dtype} of "
                         f"{width} for {kv.dtype} of {d})")
    if slot_mapping.numel() != n_rows:
        raise ValueError(f"{who}: slot_mapping must have one entry per kv row")
    if slot_mapping.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{who}: slot_mapping must be int32 or int64")
    cache_rows = blocks * block_size
    if cache_rows >= 1 << 31:
        raise ValueError(f"{who}: 2^31 cache rows or more")
    dev = cache.device
    if not cache.is_cuda or kv.device != dev:
        raise RuntimeError(f"{who} runs on a ROCm GPU; cache and kv must share it")
    at = cache.data_ptr()
    if at % 16:
        raise ValueError(f"{who}: cache must be aligned to 16 bytes")
    if n_rows == 0 or cache_rows == 0:
        return
    stride, first = kv.stride(0), kv.data_ptr()
    if first < at + cache_rows * width * cache.element_size() and \
            at < first + 2 * ((n_rows - 1) * stride + d):
        raise ValueError(f"{who}: kv overlaps the cache")
    if kv.stride(-1) != 1 or stride % 8 or kv.data_ptr() % 16:
        kv = _plain(kv)
        stride = d
    if slot_mapping.dtype == torch.int64:
        slot_mapping = _narrow(slot_mapping)
    slots = device_int32(slot_mapping, dev)
    packed = _lib.pack_row_args(kv.data_ptr(), at, *pointers, slots.data_ptr(), stride, 0, 0, 0,
                                cache_rows, n_rows, 1, d, n, r, off, *rest, row_format, block_size,
                                eps, 0)
    launch_on(cache.get_device(), _lib.load().sas_kv_append_rope, packed)
    del keep
