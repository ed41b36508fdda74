"""A sparse-attention layer's step out of the package's own calls, as a serving program makes them:
rotated queries, rows appended to the caches, the rows chosen, the attention over them.

Checked end to end against the same step in 64 bits: from the raw projections the queries, rows
and index keys are normalised and rotated, the ids chosen and the attention computed without the
package. The index keys of both are the ones the cache holds (a bf16 or fp8 key is what the choice
is made of), so the ids have to be equal; the outputs are held to the attention's own tolerance
against golden, atol = rtol = 2e-2.
"""

import math

import pytest
import torch

from oracle import row_ops
from sparse_attn_sharedkv_amd import (append_kv_rope, norm_rope_heads, sparse_attn_sharedkv,
                                      sparse_flash_mla, sparse_topk_indices)

pytestmark = pytest.mark.gpu
requires_gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a ROCm GPU")

BF = torch.bfloat16
HEADS, D, ROPE, IH, ID, BS = 16, 576, 64, 8, 128, 16


def _table(positions):
    inv = 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=torch.float64) / ROPE)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _attend(q, rows, ids, scale):
    """One query row over ``rows[ids]`` in 64 bits, no sink."""
    kv = rows[ids]
    p = torch.softmax(q @ kv.T * scale, dim=-1)
    return p @ kv[:, :512]


@requires_gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 5])
def test_step(rows, fp8):
    g = torch.Generator().manual_seed(rows + 10 * fp8)
    lens = [200, 33, 150]
    b, k, t = len(lens), 48, rows * len(lens)
    blocks = sum(-(-n // BS) for n in lens)
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    table = torch.full((b, max(-(-n // BS) for n in lens)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lens):
        c = -(-n // BS)
        table[i, :c] = perm[at:at + c]
        at += c
    cos_sin = _table(256)
    w_kv, w_ik = 1 + 0.1 * torch.randn(512, generator=g), 1 + 0.1 * torch.randn(ID, generator=g)
    latent = [torch.randn((n, D), generator=g).to(BF) for n in lens]
    index = [torch.randn((n, ID), generator=g).to(BF) for n in lens]
    q = (torch.randn((t, HEADS, D), generator=g) * 0.5).to(BF)
    qi = torch.randn((t, IH, ID), generator=g).to(BF)
    w = torch.randn((t, IH), generator=g)
    slot = torch.cat([(table[i, torch.arange(n) // BS] * BS + torch.arange(n) % BS) for i, n in enumerate(lens)])
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32)
    qpos = torch.cat([torch.arange(n - rows, n) for n in lens]).to(torch.int32)
    scale = 1 / math.sqrt(D)

    cs = cos_sin.cuda()
    cache = torch.zeros((blocks, BS, 1, 656 if fp8 else D), dtype=torch.uint8 if fp8 else BF, device="cuda")
    keys = torch.zeros((blocks, BS, 1, ID + 4 if fp8 else ID), dtype=cache.dtype, device="cuda")
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    cu = torch.arange(0, t + 1, rows, dtype=torch.int32).cuda()
    sinks = torch.full((HEADS,), float("-inf")).cuda()
    append_kv_rope(cache, torch.cat(latent).cuda(), slot.cuda(), positions=pos.cuda(), cos_sin=cs,
                   norm_weight=w_kv.cuda())
    append_kv_rope(keys, torch.cat(index).cuda(), slot.cuda(), positions=pos.cuda(), cos_sin=cs,
                   norm_weight=w_ik.cuda(), rope_offset=0, interleaved=False)
    qr = norm_rope_heads(q.cuda(), positions=qpos.cuda(), cos_sin=cs)
    qir = norm_rope_heads(qi.cuda(), positions=qpos.cuda(), cos_sin=cs, rope_offset=0, interleaved=False)
    ids = sparse_topk_indices(qir, weights=w.cuda(), index_k=keys, index_block_table=table.cuda(),
                              seqused_kv=lens_d, topk=k, cu_seqlens_q=cu, cmp_ratio=1)
    args = dict(ori_kv=cache, ori_block_table=table.cuda(), cmp_kv=cache, cmp_block_table=table.cuda(),
                cmp_sparse_indices=ids, cu_seqlens_q=cu, seqused_kv=lens_d, sinks=sinks,
                softmax_scale=scale, cmp_ratio=1, ori_win_left=-1, topk_cmp=k, head_dim_v=512)
    out = sparse_attn_sharedkv(qr, **args, schedule="device")
    assert torch.equal(out, sparse_flash_mla(qr, **args)) or torch.allclose(
        out.float(), sparse_flash_mla(qr, **args).float(), atol=1e-2)

    want_ids = row_ops.select_ids(qir.cpu(), w, keys.cpu(), table, torch.tensor(lens), k, 1, cu.cpu())
    assert torch.equal(ids.cpu(), want_ids)
    tok, at = 0, 0
    for i, n in enumerate(lens):
        kv = row_ops.norm_rope(latent[i], weight=w_kv, angles=cos_sin[:n], offset=512)
        if fp8:  # what 656-byte rows hold of it
            codes, sc = row_ops.e4m3_rows(kv[:, :512].reshape(-1, 128))
            kv = torch.cat([(codes * sc.double()).view(n, 512), kv[:, 512:]], dim=1)
        for s in range(rows):
            qq = row_ops.norm_rope(q[tok], angles=cos_sin[n - rows + s][None], offset=512)
            sel = want_ids[tok, 0]
            ref = _attend(qq, kv, sel[sel >= 0].long(), scale)
            err = (out[tok].double().cpu() - ref).abs() - 2e-2 * ref.abs()
            assert err.max() <= 2e-2, f"row {tok}: {err.max()}"
            tok += 1


@requires_gpu
def test_step_in_a_graph():
    # a decode step captured once: positions, lengths and slots change between replays
    g = torch.Generator().manual_seed(3)
    b, k, pages, cs = 4, 64, 16, _table(256).cuda()
    table = torch.randperm(b * pages, generator=g).to(torch.int32).view(b, pages).cuda()
    cache = (torch.randn((b * pages, BS, 1, D), generator=g) * 0.5).to(BF).cuda()
    keys = torch.randn((b * pages, BS, 1, ID), generator=g).to(BF).cuda()
    new, newi = torch.zeros((b, D), dtype=BF).cuda(), torch.zeros((b, ID), dtype=BF).cuda()
    q, qi = torch.zeros((b, 1, HEADS, D), dtype=BF).cuda(), torch.zeros((b, 1, IH, ID), dtype=BF).cuda()
    w = torch.randn((b, 1, IH), generator=g).cuda()
    lens, slots = torch.full((b,), 100, dtype=torch.int32).cuda(), torch.zeros(b, dtype=torch.int32).cuda()
    pos = torch.zeros(b, dtype=torch.int32).cuda()
    sinks = torch.full((HEADS,), float("-inf")).cuda()

    def step():
        append_kv_rope(cache, new, slots, positions=pos, cos_sin=cs)
        append_kv_rope(keys, newi, slots, positions=pos, cos_sin=cs, rope_offset=0)
        qr = norm_rope_heads(q, positions=pos, cos_sin=cs)
        qir = norm_rope_heads(qi, positions=pos, cos_sin=cs, rope_offset=0)
        ids = sparse_topk_indices(qir, weights=w, index_k=keys, index_block_table=table, seqused_kv=lens,
                                  topk=k, cmp_ratio=1, layout_q="BSND")
        return ids, sparse_attn_sharedkv(
            qr, ori_kv=cache, ori_block_table=table, cmp_kv=cache, cmp_block_table=table,
            cmp_sparse_indices=ids, seqused_kv=lens, sinks=sinks, softmax_scale=1 / 24, cmp_ratio=1,
            ori_win_left=-1, topk_cmp=k, head_dim_v=512, layout_q="BSND", schedule="device")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, out = step()
    for n in ([101, 130, 60, 255], [102, 131, 61, 256], [7, 64, 65, 200], [103, 132, 62, 90]):
        for t in (new, newi, q, qi):
            t.copy_(torch.randn(t.shape, generator=g).to(BF))
        at = torch.tensor(n) - 1
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        pos.copy_(at.to(torch.int32))
        slots.copy_((table.cpu()[torch.arange(b), at // BS] * BS + at % BS).to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got_ids, got = ids.clone(), out.clone()
        want_ids, want = step()
        assert torch.equal(got_ids, want_ids) and torch.equal(got, want), n
