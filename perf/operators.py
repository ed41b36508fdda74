"""The operators around sparse attention: choosing the rows, rotating the queries, writing the caches.

A decode step or a prefill chunk of a sparse-attention layer makes three kinds of call before the
attention itself, and the cases here are those calls:

* ``topk``    ``sparse_topk_indices``: scores every causal row of the index cache with a few cheap
              heads and returns the ids of the best ``topk`` of each query row;
* ``append``  ``append_kv_rope``: normalises and rotates new rows on their way into a paged cache
              (bf16 / fp16 rows, 656-byte fp8 rows, fp8 index pages);
* ``rope``    ``norm_rope_heads``: the norm and the rotation of the query heads.

Where ``own`` is false ``run`` computes them in elementary torch operations. Index scores are
formed in 64 bits there, because an id is chosen or not by values next to a border; rows are in 32.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
EXACT_FLOPS = 3e11      # a 64-bit answer by sequences over this takes too long
SCORE_BYTES = 24 << 30  # what the plain scores and keys of a drawn case may take

_TOPK = dict(kind="topk", batch=1, q_lo=1, q_hi=1, heads=64, d=128, ratio=1, topk=2048,
             ctx_lo=1024, ctx_hi=1024, block=64, layout="BSND", dtype="bf16", keys="native")
_APPEND = dict(kind="append", n=128, pool=65536, block=64, d=576, rope=64, offset=512, norm=512,
               dtype="bf16", rows="native", interleaved=True, skipped=False)
_ROPE = dict(kind="rope", tokens=64, heads=64, d=576, rope=64, offset=512, norm=0, dtype="bf16",
             interleaved=True)


def listed():
    return [
        # the smallest selection: two short sequences with few index heads
        dict(_TOPK, name="topk_b2_h16_ctx1024", batch=2, heads=16, topk=256),
        # a decode batch over a compressed index cache
        dict(_TOPK, name="topk_b32_h64_ctx16384_r4", batch=32, ratio=4, topk=512, ctx_lo=16384,
             ctx_hi=16384),
        # a full decode batch at a long context
        dict(_TOPK, name="topk_b64_h64_ctx32768", batch=64, ctx_lo=32768, ctx_hi=32768),
        # two speculative rows a sequence, an odd batch, contexts shorter than the top-k among them
        dict(_TOPK, name="topk_b13_s2_h32_fp16", batch=13, q_lo=2, q_hi=2, heads=32, ctx_lo=700,
             ctx_hi=20000, dtype="fp16"),
        # long contexts over an fp8 index cache, ragged
        dict(_TOPK, name="topk_fp8_b128_h64_long", batch=128, ctx_lo=32768, ctx_hi=131072,
             layout="TND", keys="fp8"),
        # a mixed step: decode rows and prefill chunks of odd lengths
        dict(_TOPK, name="topk_mixed_b23_h64_fp16", batch=23, q_lo=1, q_hi=157, ratio=4, topk=512,
             ctx_lo=300, ctx_hi=6000, layout="TND", dtype="fp16"),
        # the 8K prefill: the best 512 of each row's compressed rows
        dict(_TOPK, name="topk_prefill_t8192_r4", q_lo=8192, q_hi=8192, ratio=4, topk=512,
             ctx_lo=8192, ctx_hi=8192, block=128, layout="TND"),
        # a decode step's new rows into an fp8 cache
        dict(_APPEND, name="append_fp8_n128", rows="fp8"),
        # a prefill's rows into a bf16 cache, padding among them
        dict(_APPEND, name="append_bf16_n16381", n=16381, skipped=True),
        # a prefill's index keys into fp8 pages: the whole key normalised, its first dims rotated
        dict(_APPEND, name="append_index_fp8_n8192", n=8192, d=128, offset=0, norm=128,
             rows="fp8_index", interleaved=False),
        # the queries of a decode batch: only their last dims are rotated
        dict(_ROPE, name="rope_b64_h128_d576", heads=128),
        # the queries of an 8K prefill: every head normalised and rotated
        dict(_ROPE, name="norm_rope_t8192_h64_d512", tokens=8192, d=512, offset=448, norm=512),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["topk", "topk", "topk", "append", "rope"])
    if kind == "append":
        rows = rng.choice(["native", "native", "fp8", "fp8_index"])
        n = _log_int(rng, 1, 16384)
        c = dict(_APPEND, rows=rows, n=n, pool=n + rng.randrange(1, 32768),
                 block=rng.choice([16, 64, 128]), interleaved=rng.choice([True, False]),
                 skipped=rng.choice([True, False]))
        if rows == "native":
            d = rng.choice([128, 512, 576])
            r = rng.choice([32, 64])
            c.update(d=d, rope=r, offset=rng.choice([0, d - r]), dtype=rng.choice(["bf16", "fp16"]),
                     norm=rng.choice([0, d, d - 64]))
        elif rows == "fp8":
            c.update(norm=rng.choice([0, 512]))
        else:
            d = rng.choice([64, 128])
            c.update(d=d, rope=32, offset=rng.choice([0, d - 32]), norm=rng.choice([0, d]))
        return c
    if kind == "rope":
        d = rng.choice([64, 128, 512, 576])
        r = min(rng.choice([32, 64, 128]), d)
        heads = rng.choice([1, 7, 16, 32, 64, 128])
        most = max(8192 * 64 * 512 // (heads * d), 1)
        return dict(_ROPE, tokens=_log_int(rng, 1, min(most, 16384)), heads=heads, d=d, rope=r,
                    offset=rng.choice([0, d - r]), norm=rng.choice([0, d]),
                    dtype=rng.choice(["bf16", "fp16"]), interleaved=rng.choice([True, False]))
    c = dict(_TOPK, heads=rng.choice([4, 16, 32, 64, 64, 128]), d=rng.choice([64, 128, 128]),
             dtype=rng.choice(["bf16", "bf16", "fp16"]), keys=rng.choice(["native", "native", "fp8"]),
             block=rng.choice([16, 64, 64, 128]), layout=rng.choice(["BSND", "TND"]),
             ratio=rng.choice([1, 1, 4]),
             topk=rng.choice([256, 512, 1024, 2048, 2048, rng.randrange(1, 2049)]))
    form = rng.choice(["decode", "decode", "mixed", "prefill"])
    c["ctx_hi"] = _log_int(rng, 100, 131072)
    c["ctx_lo"] = rng.choice([c["ctx_hi"], rng.randrange(c["ctx_hi"] // 4, c["ctx_hi"] + 1)])
    if form == "decode":
        s = rng.choice([1, 1, 1, 2, 3])
        c.update(batch=_log_int(rng, 1, 128), q_lo=s, q_hi=s)
    elif form == "mixed":
        c.update(layout="TND", batch=rng.randrange(3, 40), q_lo=1, q_hi=rng.randrange(20, 161))
        c["ctx_hi"] = min(c["ctx_hi"], 8192)
    else:
        t = _log_int(rng, 100, 8192)
        c.update(layout="TND", batch=rng.choice([1, 1, 2, 3]), ratio=4)
        c.update(q_hi=max(t // c["batch"], 1), q_lo=max(t // c["batch"] // 2, 2))
        c["q_lo"] = min(c["q_lo"], c["q_hi"])
        c["ctx_hi"] = c["q_hi"] + rng.choice([0, 0, rng.randrange(0, 4097)])
    c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])

    def over():
        n = _width(c)
        plain = 8 * c["batch"] * n * (c["q_hi"] * c["heads"] + c["d"])
        return plain > SCORE_BYTES or 2 * c["batch"] * c["q_hi"] * n * c["heads"] * c["d"] > 2e11

    while over() and c["batch"] > 1:
        c["batch"] = (c["batch"] + 1) // 2
    while over():
        c["ctx_hi"] = max(c["ctx_hi"] * 2 // 3, 1)
        c["q_hi"] = min(c["q_hi"], c["ctx_hi"])
        c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])
        c["q_lo"] = min(c["q_lo"], c["q_hi"])
    # (a row with no more rows than the top-k takes them all, whatever their scores)
    c["topk"] = min(c["topk"], max(c["ctx_lo"] // c["ratio"] * 3 // 4, 1))
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _width(case):
    """Rows that a sequence's block table can name."""
    longest = max(case["ctx_hi"], case["q_hi"])
    return max(-(-(longest // case["ratio"]) // case["block"]), 1) * case["block"]


def _lengths(case, seed):
    """Query rows and context lengths by sequence (never shorter than the rows). The row counts
    are the case's own, in an order of the seed's, so every seed has as many tokens."""
    b, lo, hi = case["batch"], case["q_lo"], case["q_hi"]
    g = torch.Generator().manual_seed(seed * 8 + 1)
    if case["layout"] == "BSND" or lo == hi:
        rows = torch.full((b,), hi)
    else:
        mix = torch.Generator().manual_seed(lo + 1000 * hi + b)
        rows = torch.randint(lo, hi + 1, (b,), generator=mix)
        if lo == 1:  # a mixed step: most sequences decode one row
            rows = torch.where(torch.rand(b, generator=mix) < 0.7, torch.ones_like(rows), rows)
        rows = rows[torch.randperm(b, generator=g)]
    kv = torch.randint(case["ctx_lo"], case["ctx_hi"] + 1, (b,), generator=g)
    return rows.tolist(), torch.maximum(kv, rows).tolist()


def _to_e4m3(x):
    """fp8 codes of ``x`` [n, d] fp32 with one scale a row: (e4m3 [n, d], fp32 [n, 1])."""
    scale = x.abs().amax(dim=1, keepdim=True) / E4M3_MAX
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _topk_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, lens = _lengths(case, seed)
    t, h, d, bs, dt = sum(rows), case["heads"], case["d"], case["block"], _dtype(case)
    per = [max(-(-(n // case["ratio"]) // bs), 1) for n in lens]
    perm = torch.randperm(sum(per), generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), _width(case) // bs), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = perm[at:at + n]
        at += n
    blocks = sum(per)
    if case["keys"] == "fp8":
        # a page: the codes of its rows, then a scale for each row
        pool = torch.empty((blocks, bs * (d + 4)), dtype=torch.uint8, device="cuda")
        step = max((1 << 20) // bs, 1)
        for b0 in range(0, blocks, step):
            n = min(step, blocks - b0)
            codes, scale = _to_e4m3(torch.randn((n * bs, d), generator=g, device="cuda"))
            pool[b0:b0 + n, :bs * d] = codes.view(torch.uint8).view(n, bs * d)
            pool[b0:b0 + n, bs * d:] = scale.view(torch.uint8).view(n, bs * 4)
        pool = pool.view(blocks, bs, 1, d + 4)
    else:
        pool = torch.randn((blocks, bs, 1, d), generator=g, device="cuda", dtype=dt)
    q = torch.randn((t, h, d), generator=g, device="cuda", dtype=dt)
    w = torch.randn((t, h), generator=g, device="cuda") / math.sqrt(h * d)
    args = dict(index_k=pool, index_block_table=table, topk=case["topk"], cmp_ratio=case["ratio"],
                seqused_kv=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                layout_q=case["layout"])
    if case["layout"] == "TND":
        cu = torch.tensor([0] + rows, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        args.update(q_index=q, weights=w, cu_seqlens_q=cu)
    else:
        args.update(q_index=q.view(-1, rows[0], h, d), weights=w.view(-1, rows[0], h))
    return args, rows, lens


def _angles(rope, positions):
    """[positions, rope] fp32: the cosines of the angles, then their sines."""
    inv = 10000.0 ** (-torch.arange(0, rope, 2, device="cuda", dtype=torch.float64) / rope)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _append_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, d, bs, dt = case["n"], case["d"], case["block"], _dtype(case)
    blocks = -(-case["pool"] // bs)
    kv = torch.randn((n, d), generator=g, device="cuda", dtype=dt)
    slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:n].to(torch.int32)
    if case["skipped"]:
        slots[torch.rand(n, generator=g, device="cuda") < 0.05] = -1
    if case["rows"] == "native":
        cache = torch.randn((blocks, bs, 1, d), generator=g, device="cuda", dtype=dt)
    else:
        width = 656 if case["rows"] == "fp8" else d + 4
        cache = torch.zeros((blocks, bs, 1, width), dtype=torch.uint8, device="cuda")
    pos = torch.randint(0, 65536, (n,), generator=g, device="cuda").to(torch.int32)
    w = 1 + 0.1 * torch.randn(case["norm"], generator=g, device="cuda") if case["norm"] else None
    return dict(cache=cache, kv=kv, slot_mapping=slots, positions=pos,
                cos_sin=_angles(case["rope"], 65536), norm_weight=None if w is None else w.to(dt),
                rope_offset=case["offset"], interleaved=case["interleaved"], norm_eps=1e-6)


def _rope_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn((case["tokens"], case["heads"], case["d"]), generator=g, device="cuda",
                    dtype=_dtype(case))
    pos = torch.randint(0, 131072, (case["tokens"],), generator=g, device="cuda").to(torch.int32)
    w = 1 + 0.1 * torch.randn(case["norm"], generator=g, device="cuda") if case["norm"] else None
    return dict(q=q, positions=pos, cos_sin=_angles(case["rope"], 131072), norm_weight=w,
                rope_offset=case["offset"], interleaved=case["interleaved"], norm_eps=1e-6)


def prepare(case, seed):
    if case["kind"] == "topk":
        return dict(case=case, args=_topk_inputs(case, seed)[0])
    make = _append_inputs if case["kind"] == "append" else _rope_inputs
    return dict(case=case, args=make(case, seed))


# ---------------------------------------------------------------------------
# The calls, and the same in elementary operations
# ---------------------------------------------------------------------------

def _pages(args, case):
    """A sequence's index rows in order, [batch, width, d] in 64 bits (any row where no page is)."""
    pool, bs, d = args["index_k"], case["block"], case["d"]
    page = args["index_block_table"].clamp(min=0).long()
    if case["keys"] == "fp8":
        flat = pool.view(pool.shape[0], -1)
        codes = flat[:, :bs * d].view(torch.float8_e4m3fn)[page.reshape(-1)].float()
        scale = flat[:, bs * d:].view(torch.float32)[page.reshape(-1)]
        rows = codes.view(-1, bs, d).double() * scale.view(-1, bs, 1).double()
        return rows.view(page.shape[0], -1, d)
    return pool[page].view(page.shape[0], -1, d).double()


def _plain_topk(args, case):
    h, d, k = case["heads"], case["d"], case["topk"]
    q = args["q_index"].reshape(-1, h, d)
    w = args["weights"].reshape(-1, h)
    t, lens, b, s = q.shape[0], args["seqused_kv"].long(), case["batch"], case["q_hi"]
    if case["layout"] == "TND":
        cu = args["cu_seqlens_q"].long()
    else:
        cu = torch.arange(b + 1, device="cuda") * s
    row = torch.arange(t, device="cuda")
    of = torch.searchsorted(cu, row, right=True) - 1
    at = of * s + row - cu[of]                       # the row's place among [batch, s] padded rows
    qp = torch.zeros((b * s, h, d), dtype=torch.float64, device="cuda").index_copy_(0, at, q.double())
    wp = torch.zeros((b * s, h, 1), dtype=torch.float64, device="cuda")
    wp.index_copy_(0, at, w.double().unsqueeze(2))
    keys = _pages(args, case).transpose(1, 2).contiguous()
    x = torch.bmm(qp.view(b, s * h, d), keys).view(b * s, h, -1)
    score = x.relu_().mul_(wp).sum(dim=1)[at]        # [t, width]
    end = lens[of] - (cu[of + 1] - cu[of]) + (row - cu[of]) + 1
    thr = torch.div(end, case["ratio"], rounding_mode="floor")
    col = torch.arange(score.shape[1], device="cuda")
    score.masked_fill_(col >= thr[:, None], -math.inf)
    best = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k]
    best = best.masked_fill(best >= thr[:, None], score.shape[1])
    best = torch.sort(best, dim=1).values
    best = best.masked_fill(best >= score.shape[1], -1).to(torch.int32)
    out = torch.full((t, k), -1, dtype=torch.int32, device="cuda")
    out[:, :best.shape[1]] = best
    return out.view(*args["q_index"].shape[:-2], 1, k)


def _norm_rope(x, args, case, table):
    """The norm over the first dims and the rotation, on ``x`` [..., d] in its own (wide) type."""
    r, o, n = case["rope"], case["offset"], case["norm"]
    if n:
        inv = torch.rsqrt(x[..., :n].square().mean(dim=-1, keepdim=True) + args["norm_eps"])
        x = torch.cat([x[..., :n] * inv * args["norm_weight"].to(x.dtype), x[..., n:]], dim=-1)
    cos, sin = table[..., :r // 2], table[..., r // 2:]
    y = x[..., o:o + r]
    if case["interleaved"]:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([x[..., :o], y, x[..., o + r:]], dim=-1)


def _plain_append(args, case):
    cache, slots = args["cache"], args["slot_mapping"].long()
    table = args["cos_sin"][args["positions"].long()]
    y = _norm_rope(args["kv"].float(), args, case, table)
    if case["skipped"]:
        kept = slots >= 0
        y, slots = y[kept], slots[kept]
    if case["rows"] == "native":
        cache.view(-1, case["d"])[slots] = y.to(cache.dtype)
    elif case["rows"] == "fp8":
        flat = cache.view(-1, 656)
        codes, scale = _to_e4m3(y[:, :512].reshape(-1, 128))
        flat[slots] = torch.cat([codes.view(torch.uint8).view(-1, 512),
                                 scale.view(-1, 4).view(torch.uint8),
                                 y[:, 512:].to(torch.bfloat16).view(torch.uint8)], dim=1)
    else:
        codes, scale = _to_e4m3(y)
        page, at = slots // case["block"], slots % case["block"]
        c, s = _index_pages(cache, case)
        c.view(torch.uint8)[page, at] = codes.view(torch.uint8)
        s[page, at] = scale.view(-1)


def _index_pages(cache, case):
    """An fp8 index cache's codes [blocks, block, d] and scales [blocks, block]."""
    flat, bs, d = cache.view(cache.shape[0], -1), case["block"], case["d"]
    codes = flat[:, :bs * d].view(torch.float8_e4m3fn).unflatten(1, (bs, d))
    return codes, flat[:, bs * d:].view(torch.float32)


def _parts(cache, case):
    """What a cache holds, as numbers: its rows, or its codes, scales and unquantized dims."""
    if case["rows"] == "native":
        return cache
    if case["rows"] == "fp8":
        return (cache[..., :512].view(torch.float8_e4m3fn), cache[..., 512:528].view(torch.float32),
                cache[..., 528:].view(torch.bfloat16))
    return _index_pages(cache, case)


def run(state):
    case, args = state["case"], state["args"]
    if case["kind"] == "topk":
        if own:
            from sparse_attn_sharedkv_amd import sparse_topk_indices
            return sparse_topk_indices(**args)
        return _plain_topk(args, case)
    if case["kind"] == "append":
        if own:
            from sparse_attn_sharedkv_amd import append_kv_rope
            append_kv_rope(**args)
        else:
            _plain_append(args, case)
        return _parts(args["cache"], case)
    if own:
        from sparse_attn_sharedkv_amd import norm_rope_heads
        return norm_rope_heads(**args)
    table = args["cos_sin"][args["positions"].long()].unsqueeze(1)
    return _norm_rope(args["q"].float(), args, case, table).to(args["q"].dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and the 64-bit answer
# ---------------------------------------------------------------------------

def work(case):
    """Every input read once and every output written once; a score's products count as flops."""
    if case["kind"] == "append":
        out = {"native": 2 * case["d"], "fp8": 656, "fp8_index": case["d"] + 4}[case["rows"]]
        return dict(bytes=case["n"] * (2 * case["d"] + 8 + 4 * case["rope"] + out), flops=0)
    if case["kind"] == "rope":
        row = 4 * case["heads"] * case["d"] + 4 * case["rope"] + 4
        return dict(bytes=case["tokens"] * row, flops=0)
    rows, lens = _lengths(case, 1)  # (the counts of one seed: others differ by little)
    h, d, k, ratio = case["heads"], case["d"], case["topk"], case["ratio"]
    key = d + 4 if case["keys"] == "fp8" else 2 * d
    nbytes = flops = 0
    for r, n in zip(rows, lens):
        thr = [(n - r + s + 1) // ratio for s in range(r)]
        pairs = sum(x for x in thr if x > k)  # a row with no more than k rows takes them all
        flops += 2 * pairs * h * d
        nbytes += (thr[-1] * key if thr[-1] > k else 0) + r * 4 * k
        nbytes += sum(h * (2 * d + 4) for x in thr if x > k)
    return dict(bytes=nbytes, flops=flops)


def _exact_topk(case, seed):
    args, rows, lens = _topk_inputs(case, seed)
    h, d, k = case["heads"], case["d"], case["topk"]
    q, w = args["q_index"].reshape(-1, h, d).double(), args["weights"].reshape(-1, h).double()
    keys = _pages(args, case)
    out = torch.full((q.shape[0], k), -1, dtype=torch.int32, device="cuda")
    tok = 0
    for b, (r, n) in enumerate(zip(rows, lens)):
        for s0 in range(0, r, 64):
            m = min(64, r - s0)
            thr = (torch.arange(n - r + s0, n - r + s0 + m, device="cuda") + 1) // case["ratio"]
            top = max(int(thr.max()), 1)
            x = torch.zeros((m, top), dtype=torch.float64, device="cuda")
            for i in range(h):
                x += w[tok:tok + m, i, None] * (q[tok:tok + m, i] @ keys[b, :top].T).clamp(min=0)
            x[torch.arange(top, device="cuda") >= thr[:, None]] = -math.inf
            order = x.sort(dim=1, descending=True, stable=True)
            ids = torch.where(order.values > -math.inf, order.indices, 1 << 30)[:, :k].sort(dim=1)
            ids = torch.where(ids.values < 1 << 30, ids.values, -1)
            out[tok:tok + m, :ids.shape[1]] = ids.to(torch.int32)
            tok += m
    return out.view(*args["q_index"].shape[:-2], 1, k)


def exact(case, seed):
    if case["kind"] == "topk":
        return None if work(case)["flops"] > EXACT_FLOPS else _exact_topk(case, seed)
    args = _append_inputs(case, seed) if case["kind"] == "append" else _rope_inputs(case, seed)
    x = (args["kv"] if case["kind"] == "append" else args["q"]).double()
    r, o, n = case["rope"], case["offset"], case["norm"]
    if n:
        x[..., :n] /= (x[..., :n].pow(2).sum(-1, keepdim=True) / n + args["norm_eps"]).sqrt()
        x[..., :n] *= args["norm_weight"].double()
    turn = torch.complex(*args["cos_sin"][args["positions"].long()].double().split(r // 2, dim=1))
    y = x[..., o:o + r]
    pairs = y.unflatten(-1, (r // 2, 2)) if case["interleaved"] else y.unflatten(-1, (2, r // 2)).mT
    z = torch.view_as_complex(pairs.contiguous())
    z = torch.view_as_real(z * (turn if case["kind"] == "append" else turn[:, None]))
    x[..., o:o + r] = (z if case["interleaved"] else z.mT).flatten(-2)
    if case["kind"] == "rope":
        return x
    keep = args["slot_mapping"] >= 0
    slots, x = args["slot_mapping"][keep].long(), x[keep]
    total = args["cache"].shape[0] * case["block"]
    if case["rows"] == "native":
        whole = args["cache"].double().view(total, -1)
        whole[slots] = x
        return whole.view(args["cache"].shape)
    part = 128 if case["rows"] == "fp8" else case["d"]
    lat = x[:, :512].unflatten(1, (-1, part)) if case["rows"] == "fp8" else x[:, None]
    scale = lat.abs().amax(-1) / E4M3_MAX
    step = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = (lat / step[..., None]).float().to(torch.float8_e4m3fn).double().flatten(1)
    codes = torch.zeros((total, codes.shape[1]), dtype=torch.float64, device="cuda").index_copy_(
        0, slots, codes)
    step = torch.zeros((total, step.shape[1]), dtype=torch.float64, device="cuda").index_copy_(
        0, slots, step)
    if case["rows"] == "fp8":
        rope = torch.zeros((total, 64), dtype=torch.float64, device="cuda").index_copy_(
            0, slots, x[:, 512:])
        return codes, step, rope
    return codes, step
