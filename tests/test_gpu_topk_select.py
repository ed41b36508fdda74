"""``sparse_topk_indices`` on a GPU: the ids of 64-bit scores, exactly.

The ids have to be those of the oracle, which scores row by row in 64 bits; there is no
tolerance. Random inputs leave gaps between scores far above what 64-bit sums in different orders
differ by (about 1e-15 of a score); inputs with ties hold small whole numbers, whose scores are
exact in any order.
"""

import pytest
import torch

from oracle import row_ops
from sparse_attn_sharedkv_amd import sparse_topk_indices

pytestmark = pytest.mark.gpu
requires_gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a ROCm GPU")

BF, H = torch.bfloat16, torch.float16


def _case(*, rows, lens, heads=4, d=128, k=16, bs=16, ratio=1, dtype=BF, fp8=False, layout="TND", seed=0,
          whole=False, extra_blocks=3, wide=0):
    """CPU arguments of one call; unused slots of the pool hold NaN."""
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    n_of = [max(n // ratio, 0) for n in lens]
    per = [-(-n // bs) for n in n_of]
    blocks = sum(per) + extra_blocks
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    table = torch.full((b, max(per + [1]) + wide), -1, dtype=torch.int32)

    def values(*shape):
        if whole:
            return torch.randint(-2, 3, shape, generator=g).float()
        return torch.randn(shape, generator=g)

    x = values(blocks * bs, d)
    if fp8:
        codes, scale = row_ops.e4m3_rows(x.double())
        if whole:
            codes, scale = x.double(), torch.ones(blocks * bs, 1)
    used, at = torch.zeros(blocks * bs, dtype=torch.bool), 0
    for i, n in enumerate(per):
        table[i, :n] = perm[at:at + n]
        for j in range(n_of[i]):
            used[int(table[i, j // bs]) * bs + j % bs] = True
        at += n
    if fp8:
        scale[~used] = float("nan")
        pool = row_ops.index_pages(codes.view(blocks, bs, d), scale.view(blocks, bs))
    else:
        x[~used] = float("nan")
        pool = x.to(dtype).view(blocks, bs, 1, d)
    t = sum(rows)
    q, w = values(t, heads, d).to(dtype), values(t, heads)
    args = dict(q_index=q, weights=w, index_k=pool, index_block_table=table, topk=k, cmp_ratio=ratio,
                seqused_kv=torch.tensor(lens, dtype=torch.int32), layout_q=layout)
    if layout == "TND":
        args["cu_seqlens_q"] = torch.tensor([0] + rows, dtype=torch.int32).cumsum(0).to(torch.int32)
    else:
        s = rows[0]
        args.update(q_index=q.view(b, s, heads, d), weights=w.view(b, s, heads))
    return args


def _cuda(args):
    return {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in args.items()}


def _check(args, what=""):
    want = row_ops.select_ids(**args)
    got = sparse_topk_indices(**_cuda(args)).cpu()
    assert got.dtype == torch.int32 and got.shape == want.shape
    bad = (got != want).view(-1, args["topk"]).any(1).nonzero().view(-1).tolist()
    assert not bad, f"{what}: rows {bad[:5]} of {got.view(-1, args['topk']).shape[0]} differ"
    return got


@requires_gpu
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (H, False), (BF, True), (H, True)])
@pytest.mark.parametrize("heads,d", [(1, 128), (3, 64), (16, 128), (33, 64), (64, 128), (100, 128), (128, 64)])
def test_decode(heads, d, dtype, fp8):
    # one row a sequence, lengths of zero and one, at the top-k, around tile and page ends
    lens = [0, 1, 16, 17, 31, 32, 33, 95, 129, 300]
    _check(_case(rows=[1] * len(lens), lens=lens, heads=heads, d=d, dtype=dtype, fp8=fp8, seed=heads + d),
           f"{heads} heads of {d}")


@requires_gpu
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (H, False), (BF, True), (H, True)])
@pytest.mark.parametrize("heads,d", [(2, 128), (24, 64), (64, 128), (96, 128), (128, 64)])
def test_ragged_rows(heads, d, dtype, fp8):
    # chunks of many rows with single rows and a sequence without rows between them
    rows, lens = [1, 37, 0, 1, 1, 64, 9], [200, 37, 90, 150, 64, 131, 77]
    _check(_case(rows=rows, lens=lens, heads=heads, d=d, dtype=dtype, fp8=fp8, seed=heads + d, k=24),
           f"{heads} heads of {d}")


@requires_gpu
@pytest.mark.parametrize("rows,layout", [(1, "BSND"), (2, "BSND"), (3, "TND"), (5, "BSND"), (8, "TND")])
@pytest.mark.parametrize("bs,ratio,k", [(1, 1, 5), (16, 4, 16), (24, 3, 1), (64, 1, 50), (128, 2, 33)])
def test_layouts_pages_and_ratios(rows, layout, bs, ratio, k):
    lens = [260, 3, 131, rows, 400]
    _check(_case(rows=[rows] * 5, lens=[max(n, rows) for n in lens], layout=layout, bs=bs, ratio=ratio, k=k,
                 heads=6, seed=bs + k), f"{rows} rows, pages of {bs}")


@requires_gpu
@pytest.mark.parametrize("n,k", [(4096, 512), (4097, 2048), (9000, 1), (20011, 2048), (32768, 7), (40003, 2048)])
@pytest.mark.parametrize("fp8", [False, True])
def test_long_rows(n, k, fp8):
    # every size of the selection kernel (rows in LDS, rows in memory), with few heads
    _check(_case(rows=[1, 1], lens=[n, n // 3], heads=5, d=64, k=k, bs=64, fp8=fp8, seed=n))


@requires_gpu
@pytest.mark.parametrize("heads", [1, 4, 64])
@pytest.mark.parametrize("rows", [1, 6])
def test_ties_take_the_lowest_ids(heads, rows):
    # whole numbers: many equal scores, with one head half of them 0
    _check(_case(rows=[rows] * 3, lens=[700, 90, 1500], heads=heads, d=64, k=100, whole=True, seed=heads),
           "whole numbers")
    _check(_case(rows=[rows] * 3, lens=[700, 90, 1500], heads=heads, d=64, k=100, whole=True, fp8=True,
                 seed=heads), "whole numbers, fp8")


@requires_gpu
@pytest.mark.parametrize("n", [300, 6000])
def test_equal_keys(n):
    # all keys alike, all zero, zero weights: the first k rows (more of them than fit the list)
    args = _case(rows=[1, 5], lens=[n, n // 2], heads=4, d=64, k=40, bs=64, whole=True)
    first = torch.arange(40, dtype=torch.int32)
    for keys in (1.0, 0.0):
        args["index_k"] = torch.full_like(args["index_k"], keys)
        assert (_check(args) == first).all()
    args["index_k"] = torch.randn_like(args["index_k"])
    args["weights"] = torch.zeros_like(args["weights"])
    assert (_check(args) == first).all()
    args["weights"] = torch.full_like(args["weights"], -1.0)
    args["index_k"] = torch.ones_like(args["index_k"]) * torch.randint(
        0, 2, args["index_k"].shape[:3] + (1,))
    _check(args, "two scores")


@requires_gpu
def test_scores_closer_than_fp32():
    # keys that differ by one step of one element: their fp32 scores are mostly equal or swapped
    args = _case(rows=[1, 4], lens=[3000, 2000], heads=8, d=128, k=700, bs=64, dtype=H)
    base = torch.randn(1, 1, 1, 128) * 8
    base[..., 5] = 2.0 ** -8
    keys = base.expand(args["index_k"].shape).to(H).clone()
    step = torch.randint(0, 1024, keys.shape[:3])
    keys[..., 5] = (2.0 ** -8 * (1 + step / 1024)).to(H)
    args["index_k"] = keys
    args["q_index"] = args["q_index"].abs() * torch.sign(base.view(128)).to(H)
    _check(args)


@requires_gpu
def test_wide_spread_of_scores():
    # magnitudes over many decades, both signs; an outlier that stretches the range
    args = _case(rows=[1, 1, 1], lens=[5000, 3000, 2000], heads=4, d=64, k=300, bs=64)
    scale = 10.0 ** torch.randint(-12, 13, args["index_k"].shape[:3] + (1,)).float()
    args["index_k"] = (args["index_k"].float() * scale).to(BF)
    _check(args, "decades")
    args = _case(rows=[1, 1], lens=[5000, 3000], heads=4, d=64, k=300, bs=64, seed=2)
    flat = args["index_k"].view(-1, 64)
    flat[int(args["index_block_table"][0, 3]) * 64 + 5] = 1e30
    _check(args, "outlier")


@requires_gpu
def test_missing_pages():
    # pages outside the pool in the middle of a sequence: never read, never chosen
    args = _case(rows=[1, 1, 7], lens=[500, 90, 400], heads=4, d=64, k=60, bs=16)
    table = args["index_block_table"]
    table[0, 3], table[0, 10], table[1, 0], table[1, 2] = -1, 1 << 20, -(1 << 31), 1 << 30
    table[2, :5] = -1
    _check(args)
    table[0] = -1
    got = _check(args)
    assert (got[0] == -1).all()


@requires_gpu
@pytest.mark.parametrize("rows", [1, 6])
def test_not_a_number(rows):
    # NaN and infinite keys, queries and weights: NaN scores rank lowest, the row is scored in 64 bits
    args = _case(rows=[rows] * 3, lens=[150, 130, 140], heads=4, d=64, k=30, bs=16)
    flat, table = args["index_k"].view(-1, 64), args["index_block_table"]
    flat[int(table[0, 1]) * 16 + 3, 7] = float("nan")
    flat[int(table[0, 4]) * 16 + 5, 9] = float("inf")
    flat[int(table[1, 2]) * 16 + 1] = 3e38
    q, w = args["q_index"], args["weights"]
    q[2 * rows:, 1, 3] = float("nan")
    w[rows:2 * rows, 2] = float("inf")
    _check(args)


@requires_gpu
def test_rows_of_no_sequence():
    args = _case(rows=[2, 30], lens=[200, 180], heads=4, d=64, k=20)
    t = args["q_index"].shape[0]
    args["q_index"] = torch.cat([args["q_index"][:9], args["q_index"], args["q_index"][:5]])
    args["weights"] = torch.cat([args["weights"][:9], args["weights"], args["weights"][:5]])
    args["cu_seqlens_q"] = args["cu_seqlens_q"] + 9
    got = _check(args)
    assert (got[:9] == -1).all() and (got[9 + t:] == -1).all()
    # BSND with fewer rows in use than the layout holds
    for s in (2, 6):
        args = _case(rows=[s] * 3, lens=[120, 90, 200], heads=4, d=64, k=20, layout="BSND")
        args["cu_seqlens_q"] = torch.tensor([0, 1, s + 1, s + 1], dtype=torch.int32)
        _check(args, f"BSND of {s}")
    # lengths below the row count: the first rows have nothing to attend
    args = _case(rows=[6, 3], lens=[60, 50], heads=4, d=64, k=20)
    args["seqused_kv"] = torch.tensor([2, -5], dtype=torch.int32)
    got = _check(args)
    assert (got[:4] == -1).all() and (got[6:] == -1).all()
    empty = _cuda(_case(rows=[1], lens=[60], heads=4, d=64, k=20))
    empty.update(q_index=empty["q_index"][:0], weights=empty["weights"][:0])
    assert sparse_topk_indices(**empty).shape == (0, 1, 20)
    none = _cuda(_case(rows=[1], lens=[60], heads=4, d=64, k=20))
    none["cu_seqlens_q"] = none["cu_seqlens_q"][:1]
    assert (sparse_topk_indices(**none) == -1).all()


@requires_gpu
def test_wide_tables_and_max_seqlen():
    # a table far wider than the sequences; the rows then take several passes of the workspace
    args = _case(rows=[1100, 1100], lens=[1200, 1150], heads=2, d=64, k=64, bs=64, wide=2030)
    assert args["index_block_table"].shape[1] * 64 * 2200 * 4 > 1 << 30
    got = _check(args)
    args["max_seqlen_kv"] = 1200
    assert torch.equal(_check(args), got)
    args["max_seqlen_kv"] = 500
    assert _check(args).max() < 500


@requires_gpu
def test_strided_and_other_types():
    args = _cuda(_case(rows=[1, 9], lens=[300, 200], heads=4, d=64, k=20))
    want = sparse_topk_indices(**args)
    q, w = args["q_index"], args["weights"]
    wide = torch.zeros(10, 4, 80, dtype=BF, device="cuda")
    wide[..., 8:72] = q
    table = args["index_block_table"].long()
    got = sparse_topk_indices(**dict(
        args, q_index=wide[..., 8:72], index_block_table=torch.cat([table, table])[:, :],
        weights=w.t().contiguous().t(), seqused_kv=args["seqused_kv"].long(),
        cu_seqlens_q=args["cu_seqlens_q"].long(), index_k=torch.cat([args["index_k"]] * 2, 2)[:, :, :1]))
    assert torch.equal(got, want)
    half = w.to(BF)
    assert torch.equal(sparse_topk_indices(**dict(args, weights=half)),
                       sparse_topk_indices(**dict(args, weights=half.float())))


@requires_gpu
def test_choice_does_not_depend_on_the_batch():
    # a row alone, in a batch (another split of the keys) and among many rows (the other kernel)
    args = _case(rows=[1] * 24, lens=[2500 + 7 * i for i in range(24)], heads=32, d=128, k=256, bs=64)
    got = sparse_topk_indices(**_cuda(args))
    for i in (0, 11, 23):
        one = dict(args, q_index=args["q_index"][i:i + 1], weights=args["weights"][i:i + 1],
                   index_block_table=args["index_block_table"][i:i + 1],
                   seqused_kv=args["seqused_kv"][i:i + 1], cu_seqlens_q=torch.tensor([0, 1]))
        assert torch.equal(sparse_topk_indices(**_cuda(one))[0], got[i])
        many = dict(one, q_index=one["q_index"].expand(8, -1, -1), weights=one["weights"].expand(8, -1),
                    cu_seqlens_q=torch.tensor([0, 8]))
        assert torch.equal(sparse_topk_indices(**_cuda(many))[7], got[i])


@requires_gpu
@pytest.mark.parametrize("rows", [1, 6])
def test_graph_with_other_lengths(rows):
    args = _cuda(_case(rows=[rows] * 4, lens=[900, 700, 800, 650], heads=16, d=128, k=128, bs=64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = sparse_topk_indices(**args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_topk_indices(**args)
    for lens in ([900, 700, 800, 650], [6, 300, 129, 128], [640, 640, 640, 640], [900, 700, 800, 650]):
        args["seqused_kv"].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sparse_topk_indices(**args)), lens
    assert torch.equal(out, want)


@requires_gpu
@pytest.mark.parametrize("n,k", [(40003, 8000), (40003, 30000), (270001, 600), (9001, 8990), (2049, 2048)])
def test_wide_selections_and_the_longest_rows(n, k):
    # more ids, or longer rows, than the registers' path takes: the same steps from memory
    _check(_case(rows=[1, 1], lens=[n, n - 7], heads=3, d=64, k=k, bs=128, seed=n + k))


@requires_gpu
@pytest.mark.parametrize("n", [700, 6000, 20000, 50000])
def test_uneven_scores(n):
    # a periodic row (what a sample of it sees is not what it is) and rows with a few scores far
    # above the rest, so that most of a histogram's range is empty
    args = _case(rows=[1, 1], lens=[n, n - 100], heads=4, d=64, k=n // 9, bs=64, seed=n)
    flat, table = args["index_k"].view(-1, 64), args["index_block_table"]
    j = torch.arange(n - 100)
    rows0 = (table[0, j // 64] * 64 + j % 64).long()
    rows1 = (table[1, j // 64] * 64 + j % 64).long()
    flat[rows0[j % 32 < 4]] *= 1e-3
    flat[rows1[[3, n // 2, n - 200]]] *= 1e5
    _check(args)


@requires_gpu
def test_a_nan_key_in_a_long_row():
    args = _case(rows=[1, 5], lens=[9000, 8500], heads=2, d=64, k=512, bs=64)
    flat, table = args["index_k"].view(-1, 64), args["index_block_table"]
    flat[int(table[0, 9]) * 64 + 5, 3] = float("nan")
    flat[int(table[1, 20]) * 64 + 7, 1] = float("-inf")
    _check(args)


@requires_gpu
def test_many_rows_take_the_single_wave_path():
    # from 512 rows of short sequences on a wave owns a row
    _check(_case(rows=[300, 1, 400], lens=[420, 1900, 401], heads=3, d=64, k=50, bs=16, ratio=1), "many rows")
    _check(_case(rows=[600], lens=[600], heads=2, d=64, k=40, bs=16, whole=True), "ties in many rows")


@requires_gpu
def test_sequences_without_rows_or_pages():
    args = _case(rows=[0, 0, 3, 0], lens=[50, 0, 60, 10], heads=4, d=64, k=20)
    _check(args)
    args["index_block_table"] = torch.full_like(args["index_block_table"], -1)
    assert (_check(args) == -1).all()


@requires_gpu
@pytest.mark.parametrize("heads", [4, 40])
@pytest.mark.parametrize("keys,weights", [(2.0 ** -66, 1.0), (1.0, 2.0 ** -125), (2.0 ** -40, 2.0 ** -90), (2.0 ** 60, 2.0 ** 40)])
def test_small_and_large_magnitudes(heads, keys, weights):
    # squares, products or scores outside fp32's range: the choice is still that of 64 bits
    args = _case(rows=[1, 5], lens=[400, 300], heads=heads, d=64, k=50, bs=16, seed=heads)
    args["index_k"] = (args["index_k"].float() * keys).to(BF)
    args["weights"] = args["weights"] * weights
    _check(args)


@requires_gpu
@pytest.mark.parametrize("dtype,scale", [(H, 2.0 ** -18), (H, 2.0 ** -22), (BF, 2.0 ** -130)])
def test_subnormal_keys(dtype, scale):
    # keys below their type's normal range, alone and among ordinary ones
    args = _case(rows=[1, 5], lens=[400, 300], heads=8, d=128, k=50, bs=16, dtype=dtype, seed=7)
    plain = args["index_k"].clone()
    args["index_k"] = (plain.float() * scale).to(dtype)
    _check(args, "all")
    some = torch.rand(plain.shape[:3] + (1,)) < 0.5
    args["index_k"] = torch.where(some, args["index_k"], plain)
    args["weights"] = -args["weights"].abs()  # (scores at most 0: the small keys' are the largest)
    _check(args, "some")


@requires_gpu
@pytest.mark.parametrize("rows", [[1, 3, 4, 5, 1, 2, 0, 40, 3], [200] + [1] * 20, [1] * 20 + [9] * 8, [3] * 12, [6, 0, 0, 0]])
def test_mixed_steps(rows):
    # short and long row counts in one call: each sequence has the kernel of its own count
    lens = [n + 37 * (i % 5) + 20 for i, n in enumerate(rows)]
    _check(_case(rows=rows, lens=lens, heads=20, d=128, k=18, bs=16, seed=len(rows)), str(rows))
    if max(rows) <= 9:  # the same in a padded batch
        s = max(rows) + 2
        args = _case(rows=[s] * len(rows), lens=[n + s for n in lens], heads=5, d=64, k=18, layout="BSND")
        args["cu_seqlens_q"] = torch.tensor([0] + rows, dtype=torch.int32).cumsum(0).to(torch.int32)
        _check(args, f"padded {rows}")
