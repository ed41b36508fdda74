"""``norm_rope_heads`` and ``append_kv_rope`` on a GPU against 64-bit answers.

Tolerances. The kernel works in fp32 and rounds once. With u = 2^-24: the sum of at most 1024
squares is 16 fused steps and 6 exchanges deep (22 u), its mean, root and quotient 4 u more, so
the factor is off by at most 15 u (the root halves the sum's part), the two products by 2 u, and
a rotation's two products and its sum by 3 u of |a| + |b|: below 20 u = 2^-19.6 of |a| + |b| in
all; 2^-19 is allowed. The rounding to the output's type adds half a step: eps / 2 of the value,
and 2^-25 where fp16 runs out of exponents. e4m3 codes are within half a step of the value
(2^-4 of it, 2^-10 of the scale near zero), and the fp32 scale within 2^-19.
"""

import pytest
import torch

from oracle import row_ops
from sparse_attn_sharedkv_amd import append_kv_fp8, append_kv_rope, norm_rope_heads

pytestmark = pytest.mark.gpu
requires_gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a ROCm GPU")

BF, H = torch.bfloat16, torch.float16
FP32 = 2.0 ** -19


def _angles(positions, r, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand((positions, r // 2), generator=g, dtype=torch.float64) * 6.283
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _reach(x, weight, eps, r, offset, interleaved):
    """|a| + |b| of every element's pair (the element itself where nothing rotates)."""
    y = row_ops.norm_rope(x, weight=weight, eps=eps).abs()
    if r:
        first = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
        second = first + 1 if interleaved else first + r // 2
        both = y[..., offset + first] + y[..., offset + second]
        y[..., offset + first] = both
        y[..., offset + second] = both
    return y


def _check(got, want, reach, dtype, what):
    off = (got.double().cpu() - want).abs()
    slack = FP32 * reach
    tol = torch.finfo(dtype).eps / 2 * (want.abs() + slack) + slack + (2.0 ** -25 if dtype == H else 0)
    worst = (off - tol).max().item()
    assert worst <= 0, f"{what}: {worst} over the bound"


def _data(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


CASES = [  # tokens, heads, d, norm dims, rotated dims, offset, interleaved
    (1, 1, 8, 8, 8, 0, True), (1, 1, 64, 0, 64, 0, False), (5, 3, 64, 64, 16, 48, False),
    (7, 5, 72, 40, 8, 32, True), (3, 2, 128, 128, 128, 0, False), (4, 16, 128, 64, 64, 64, True),
    (9, 1, 192, 192, 32, 8, False), (2, 7, 256, 256, 0, 0, True), (6, 4, 512, 512, 64, 448, True),
    (6, 4, 512, 0, 0, 0, True), (5, 3, 576, 512, 64, 512, True), (5, 3, 576, 576, 64, 512, False),
    (2, 2, 576, 576, 576, 0, False), (3, 1, 1024, 1024, 1024, 0, False), (3, 2, 1000, 40, 48, 952, False),
    (130, 8, 136, 136, 64, 16, True),
]


@requires_gpu
@pytest.mark.parametrize("dtype", [BF, H])
@pytest.mark.parametrize("case", CASES)
def test_norm_rope_heads(case, dtype):
    t, h, d, n, r, off, inter = case
    x = _data((t, h, d), dtype, seed=d + t)
    w = _data((n,), torch.float32, 1).add(1) if n else None
    if w is not None and d % 16 == 0:
        w = w.to(dtype)
    table = _angles(40, r) if r else None
    pos = torch.randint(0, 40, (t,), dtype=torch.int32) if r else None
    want = row_ops.norm_rope(x, weight=w, eps=1e-5, angles=table[pos.long()][:, None] if r else None,
                             offset=off, interleaved=inter)
    reach = _reach(x, w, 1e-5, r, off, inter)
    kw = dict(positions=pos.cuda() if r else None, cos_sin=table.cuda() if r else None,
              norm_weight=w.cuda() if n else None, norm_eps=1e-5, rope_offset=off if r else None,
              interleaved=inter)
    q = x.cuda()
    got = norm_rope_heads(q, **kw)
    assert torch.equal(q.cpu(), x), "the input changed"
    _check(got, want, reach, dtype, "out of place")
    again = norm_rope_heads(q, out=q, **kw)
    assert again is q and torch.equal(q, got), "in place"


@requires_gpu
def test_strided_queries_and_outputs():
    # heads inside a wider projection, tokens of every second row, a transposed batch
    wide = _data((6, 4 * 192 + 64), BF, 3).cuda()
    table, pos = _angles(9, 32).cuda(), torch.arange(6, dtype=torch.int32).cuda()
    w = torch.ones(128).cuda()
    q = wide[:, 64:].view(6, 4, 192)[:, :, :128]
    want = norm_rope_heads(q.contiguous(), positions=pos, cos_sin=table, norm_weight=w)
    assert torch.equal(norm_rope_heads(q, positions=pos, cos_sin=table, norm_weight=w), want)
    out = torch.zeros(12, 5, 128, dtype=BF, device="cuda")
    got = norm_rope_heads(q, positions=pos, cos_sin=table, norm_weight=w, out=out[::2, :4])
    assert torch.equal(got, want) and not out[1::2].any() and not out[:, 4].any()
    t = q.transpose(0, 1).contiguous().transpose(0, 1)       # [tokens, heads] in head order
    assert torch.equal(norm_rope_heads(t, positions=pos, cos_sin=table, norm_weight=w), want)
    odd = torch.zeros(6 * 4 * 128 + 1, dtype=BF, device="cuda")[1:].view(6, 4, 128)
    odd.copy_(q)                                             # not on 16 bytes: copied first
    assert torch.equal(norm_rope_heads(odd, positions=pos, cos_sin=table, norm_weight=w), want)
    with pytest.raises(ValueError, match="aligned"):
        norm_rope_heads(q, positions=pos, cos_sin=table, out=odd)
    with pytest.raises(ValueError, match="overlaps"):
        norm_rope_heads(wide[:5, :512].view(5, 4, 128), positions=pos[:5], cos_sin=table,
                        out=wide[1:, :512].view(5, 4, 128))
    for out in (torch.zeros(1, 4, 128, dtype=BF, device="cuda").expand(6, 4, 128),
                torch.zeros(6, 1, 128, dtype=BF, device="cuda").expand(6, 4, 128),
                torch.zeros(8 * 64 * 8, dtype=BF, device="cuda").as_strided((6, 4, 128), (512, 64, 1))):
        with pytest.raises(ValueError, match="itself"):
            norm_rope_heads(q, positions=pos, cos_sin=table, out=out)
    same = norm_rope_heads(q[:1].expand(6, 4, 128), positions=pos, cos_sin=table, norm_weight=w)
    assert torch.equal(same[0], want[0]) and not torch.equal(same[1], want[1])
    four = norm_rope_heads(q.reshape(2, 3, 4, 128), positions=pos.view(2, 3).long(), cos_sin=table,
                           norm_weight=w)
    assert torch.equal(four.view(6, 4, 128), want)
    assert norm_rope_heads(q[:0], positions=pos[:0], cos_sin=table).shape == (0, 4, 128)


@requires_gpu
@pytest.mark.parametrize("inter", [True, False])
def test_positions_outside_the_table(inter):
    x = _data((4, 2, 64), BF, 5).cuda()
    pos = torch.tensor([0, -1, 8, 7], dtype=torch.int32).cuda()
    got = norm_rope_heads(x, positions=pos, cos_sin=_angles(8, 32).cuda(), interleaved=inter)
    assert torch.equal(got[..., :32], x[..., :32])
    assert got[1:3, :, 32:].isnan().all() and not got[[0, 3]].isnan().any()


@requires_gpu
def test_rows_of_extremes():
    # zeros (eps decides), values near the types' limits, infinities and NaN in other rows
    x = torch.zeros(6, 1, 64, dtype=BF)
    x[1] = 1e-20
    x[2, 0, 3] = 3e38
    x[3, 0, 5] = float("inf")
    x[4, 0, 5] = float("nan")
    x[5] = 2.0
    got = norm_rope_heads(x.cuda(), norm_weight=torch.ones(64).cuda()).cpu()
    assert not got[0].any() and got[1].abs().max() < 1e-16
    assert got[4].isnan().all() and torch.equal(got[5], torch.ones(1, 64, dtype=BF))
    assert not got[[0, 1, 5]].isnan().any()


def _slots(n, rows, seed):
    g = torch.Generator().manual_seed(seed)
    s = torch.randperm(rows, generator=g)[:n].to(torch.int32)
    if n > 4:
        s[1], s[n - 2] = -1, rows       # skipped: padding, past the pool
    return s


@requires_gpu
@pytest.mark.parametrize("dtype", [BF, H])
@pytest.mark.parametrize("n,d,norm,r,off,inter", [
    (1, 576, 512, 64, 512, True), (37, 576, 0, 64, 512, False), (33, 512, 512, 64, 448, True),
    (20, 128, 128, 32, 0, False), (50, 64, 64, 64, 0, True), (6, 576, 576, 0, 0, True),
    (3, 8, 0, 0, 0, True), (300, 1024, 1024, 128, 0, False)])
def test_append_native(n, d, norm, r, off, inter, dtype):
    x = _data((n, d), dtype, n + d)
    w = (_data((norm,), torch.float32, 2) + 1) if norm else None
    table = _angles(50, r) if r else None
    pos = torch.randint(0, 50, (n,), dtype=torch.int32) if r else None
    old = _data((23, 16, 1, d), dtype, 9)
    cache, slots = old.cuda(), _slots(n, 23 * 16, n)
    append_kv_rope(cache, x.cuda(), slots.cuda(), positions=pos.cuda() if r else None,
                   cos_sin=table.cuda() if r else None, norm_weight=w.cuda() if norm else None,
                   rope_offset=off if r else None, interleaved=inter)
    want = row_ops.norm_rope(x, weight=w, angles=table[pos.long()] if r else None, offset=off,
                             interleaved=inter)
    reach = _reach(x, w, 1e-6, r, off, inter)
    got, kept = cache.cpu().view(-1, d), (slots >= 0) & (slots < 23 * 16)
    _check(got[slots[kept].long()], want[kept], reach[kept], dtype, "rows")
    rest = torch.ones(23 * 16, dtype=torch.bool)
    rest[slots[kept].long()] = False
    assert torch.equal(got[rest], old.view(-1, d)[rest]), "other rows changed"


def _check_codes(codes, scale, want, reach, what):
    """Codes [n, d] and scales [n, 1] against the values they stand for."""
    amax = want.abs().amax(1, keepdim=True)
    ideal = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    slack = FP32 * reach
    assert ((scale.double() - ideal).abs() <= slack.amax(1, keepdim=True) / 448 + 2.0 ** -23 * ideal).all(), what
    off = (codes.double() * scale.double() - want).abs()
    half = torch.maximum(want.abs() * 2.0 ** -4, 2.0 ** -10 * scale.double())
    assert (off <= half * (1 + 2.0 ** -18) + 2 * slack).all(), what


@requires_gpu
@pytest.mark.parametrize("n,norm,inter", [(1, 512, True), (67, 512, False), (40, 0, True), (9, 576, True)])
def test_append_fp8_rows(n, norm, inter):
    x = _data((n, 576), BF, n, scale=3.0)
    x[n // 2, 128:256] = 0                     # a block of zeros: scale 1
    w = (_data((norm,), torch.float32, 2) + 1).to(BF) if norm else None
    table, pos = _angles(50, 64), torch.randint(0, 50, (n,), dtype=torch.int32)
    cache, slots = torch.full((5, 16, 1, 656), 7, dtype=torch.uint8).cuda(), _slots(n, 80, n)
    append_kv_rope(cache, x.cuda(), slots.cuda(), positions=pos.cuda(), cos_sin=table.cuda(),
                   norm_weight=w.cuda() if norm else None, interleaved=inter)
    want = row_ops.norm_rope(x, weight=w, angles=table[pos.long()], offset=512, interleaved=inter)
    reach = _reach(x, w, 1e-6, 64, 512, inter)
    kept = (slots >= 0) & (slots < 80)
    rows = cache.cpu().view(-1, 656)[slots[kept].long()]
    codes = rows[:, :512].contiguous().view(torch.float8_e4m3fn).float().view(-1, 128)
    scale = rows[:, 512:528].contiguous().view(torch.float32).view(-1, 1)
    _check_codes(codes, scale, want[kept][:, :512].reshape(-1, 128), reach[kept][:, :512].reshape(-1, 128),
                 "latent")
    _check(rows[:, 528:].contiguous().view(BF), want[kept][:, 512:], reach[kept][:, 512:], BF, "rope")
    assert (cache.cpu().view(-1, 656)[[i for i in range(80) if i not in slots[kept].tolist()]] == 7).all()


@requires_gpu
def test_append_fp8_without_parts_is_the_plain_writer():
    x, slots = _data((51, 576), BF, 4).cuda(), _slots(51, 128, 3).cuda()
    one = torch.zeros(8, 16, 1, 656, dtype=torch.uint8, device="cuda")
    two = torch.zeros_like(one)
    append_kv_fp8(one, x, slots)
    append_kv_rope(two, x, slots)
    assert torch.equal(one, two)
    append_kv_rope(two.view(torch.float8_e4m3fn), x.view(51, 1, 576), slots.long())
    assert torch.equal(one, two)


@requires_gpu
@pytest.mark.parametrize("dtype", [BF, H])
@pytest.mark.parametrize("d,bs", [(64, 4), (128, 16), (128, 64), (64, 100)])
def test_append_index_pages(d, bs, dtype):
    n = 70
    x = _data((n, d), dtype, d + bs)
    x[5] = 0
    w = _data((d,), torch.float32, 2) + 1
    table, pos = _angles(50, 32), torch.randint(0, 50, (n,), dtype=torch.int32)
    blocks = 400 // bs
    cache, slots = torch.full((blocks, bs, 1, d + 4), 9, dtype=torch.uint8).cuda(), _slots(n, blocks * bs, d)
    append_kv_rope(cache, x.cuda(), slots.cuda(), positions=pos.cuda(), cos_sin=table.cuda(),
                   norm_weight=w.cuda(), rope_offset=0, interleaved=False)
    want = row_ops.norm_rope(x, weight=w, angles=table[pos.long()], offset=0, interleaved=False)
    reach = _reach(x, w, 1e-6, 32, 0, False)
    kept = (slots >= 0) & (slots < blocks * bs)
    at = slots[kept].long()
    flat = cache.cpu().view(blocks, -1)
    codes = flat[:, :bs * d].contiguous().view(torch.float8_e4m3fn).float().view(-1, d)
    scale = flat[:, bs * d:].contiguous().view(torch.float32).view(-1, 1)
    _check_codes(codes[at], scale[at], want[kept], reach[kept], "index rows")
    rest = torch.ones(blocks * bs, dtype=torch.bool)
    rest[at] = False
    assert (flat[:, :bs * d].reshape(-1, d)[rest] == 9).all()
    assert (flat[:, bs * d:].reshape(-1, 4)[rest] == 9).all()


@requires_gpu
def test_append_odd_inputs():
    table, pos = _angles(9, 32).cuda(), torch.arange(6, dtype=torch.int32).cuda()
    wide = _data((6, 300), BF, 3).cuda()
    x = wide[:, 40:168]                                  # 16-byte rows of stride 300: copied
    want = torch.zeros(2, 8, 1, 128, dtype=BF, device="cuda")
    got = want.clone()
    slots = torch.arange(6).cuda()
    append_kv_rope(want, x.contiguous(), slots, positions=pos, cos_sin=table)
    append_kv_rope(got, x, slots, positions=pos, cos_sin=table)
    assert torch.equal(got, want)
    wide = _data((6, 304), BF, 3).cuda()                 # read where they are
    append_kv_rope(want, wide[:, 40:168].contiguous(), slots, positions=pos, cos_sin=table)
    append_kv_rope(got, wide[:, 40:168], slots, positions=pos, cos_sin=table)
    assert torch.equal(got, want)
    before = got.clone()
    append_kv_rope(got, x[:0], slots[:0])
    append_kv_rope(got, x, torch.tensor([1 << 32, (1 << 32) + 1, -1, 16, 1 << 40, -(1 << 40)]).cuda())
    assert torch.equal(got, before)
    with pytest.raises(ValueError, match="overlaps"):
        append_kv_rope(got, got.view(16, 128)[2:8], slots)
    nan = x.clone()
    nan[2, 7] = float("nan")
    pages = torch.zeros(2, 8, 1, 132, dtype=torch.uint8, device="cuda")
    append_kv_rope(pages, nan.contiguous(), slots, positions=pos, cos_sin=table)
    scale = pages.view(2, -1)[:, 1024:].contiguous().view(torch.float32).view(-1)
    assert scale[2].isnan() and not scale[[0, 1, 3, 4, 5]].isnan().any()


@requires_gpu
def test_other_stream_and_graph():
    x = _data((33, 8, 576), BF, 1).cuda()
    table, pos = _angles(64, 64).cuda(), torch.arange(33, dtype=torch.int32).cuda()
    want = norm_rope_heads(x, positions=pos, cos_sin=table)
    cache0 = torch.zeros(4, 16, 1, 576, dtype=BF, device="cuda")
    slots = torch.arange(33, dtype=torch.int32).cuda()
    append_kv_rope(cache0, x[:, 0], slots, positions=pos, cos_sin=table)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(norm_rope_heads(x, positions=pos, cos_sin=table), want)
    torch.cuda.current_stream().wait_stream(s)
    static, cache = x.clone(), torch.zeros_like(cache0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = norm_rope_heads(static, positions=pos, cos_sin=table)
        append_kv_rope(cache, static[:, 0], slots, positions=pos, cos_sin=table)
    for k in range(3):
        static.copy_(x * (k + 1))
        cache.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = norm_rope_heads(static, positions=pos, cos_sin=table)
        append_kv_rope(cache0, static[:, 0], slots, positions=pos, cos_sin=table)
        assert torch.equal(out, eager) and torch.equal(cache, cache0)
