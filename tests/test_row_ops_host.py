"""Refusals of the row operators and of the row selection, on CPU tensors: nothing is launched.

Every condition the kernels rely on is checked on the host, in the Python entry points and again
in the C ones. A well-formed call on CPU tensors raises RuntimeError: there is no CPU path.
"""

import ctypes
import re

import pytest
import torch

from sparse_attn_sharedkv_amd import _lib, append_kv_rope, norm_rope_heads, sparse_topk_indices

BF, H, F = torch.bfloat16, torch.float16, torch.float32


def _rope(**over):
    kw = dict(q=torch.zeros(3, 4, 128, dtype=BF), positions=torch.zeros(3, dtype=torch.int32),
              cos_sin=torch.zeros(16, 64), norm_weight=torch.ones(128))
    kw.update(over)
    return kw


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(3, 4, 128)), dict(q=torch.zeros(128, dtype=BF)),
    dict(q=torch.zeros(3, 0, 128, dtype=BF)),
    dict(q=torch.zeros(3, 4, 124, dtype=BF), norm_weight=None),
    dict(q=torch.zeros(3, 4, 1032, dtype=BF), norm_weight=None),
    dict(norm_weight=torch.ones(124)), dict(norm_weight=torch.ones(136)),
    dict(norm_weight=torch.ones(1, 128)), dict(norm_weight=torch.ones(128, dtype=H)),
    dict(norm_weight=torch.ones(0)),
    dict(cos_sin=None), dict(positions=None), dict(cos_sin=torch.zeros(16, 64, dtype=BF)),
    dict(cos_sin=torch.zeros(64)), dict(cos_sin=torch.zeros(0, 64)),
    dict(cos_sin=torch.zeros(16, 136)), dict(cos_sin=torch.zeros(16, 60)),
    dict(cos_sin=torch.zeros(16, 24), interleaved=False),
    dict(rope_offset=68), dict(rope_offset=-8), dict(rope_offset=72),
    dict(positions=torch.zeros(4, dtype=torch.int32)),
    dict(positions=None, cos_sin=None, rope_offset=0),
    dict(out=torch.zeros(3, 4, 128, dtype=H)), dict(out=torch.zeros(3, 4, 64, dtype=BF)),
])
def test_norm_rope_refusals(bad):
    with pytest.raises(ValueError, match="norm_rope_heads"):
        norm_rope_heads(**_rope(**bad))


def _append(**over):
    kw = dict(cache=torch.zeros(4, 16, 1, 576, dtype=BF), kv=torch.zeros(5, 576, dtype=BF),
              slot_mapping=torch.zeros(5, dtype=torch.int32),
              positions=torch.zeros(5, dtype=torch.int32), cos_sin=torch.zeros(16, 64),
              norm_weight=torch.ones(512))
    kw.update(over)
    return kw


def _u8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


@pytest.mark.parametrize("bad", [
    dict(kv=torch.zeros(5, 2, 576, dtype=BF)), dict(kv=torch.zeros(576, dtype=BF)),
    dict(cache=torch.zeros(64, 576, dtype=BF)), dict(cache=torch.zeros(4, 16, 2, 576, dtype=BF)),
    dict(cache=torch.zeros(4, 16, 1, 576, dtype=H)), dict(cache=torch.zeros(4, 16, 1, 512, dtype=BF)),
    dict(cache=torch.zeros(16, 4, 1, 576, dtype=BF).transpose(0, 1)),
    dict(cache=_u8(4, 16, 1, 580)), dict(cache=_u8(4, 16, 1, 576)),
    dict(cache=_u8(4, 16, 1, 656), kv=torch.zeros(5, 576, dtype=H)),
    dict(cache=_u8(4, 16, 1, 656), kv=torch.zeros(5, 512, dtype=BF)),
    dict(cache=_u8(4, 6, 1, 132), kv=torch.zeros(5, 128, dtype=BF), norm_weight=None),
    dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), dict(slot_mapping=torch.zeros(5)),
    dict(positions=torch.zeros(4, dtype=torch.int32)), dict(norm_weight=torch.ones(584)),
])
def test_append_refusals(bad):
    with pytest.raises(ValueError, match="append_kv_rope"):
        append_kv_rope(**_append(**bad))


def _topk(**over):
    kw = dict(q_index=torch.zeros(3, 4, 128, dtype=BF), weights=torch.zeros(3, 4),
              index_k=torch.zeros(4, 16, 1, 128, dtype=BF),
              index_block_table=torch.zeros(2, 4, dtype=torch.int32),
              seqused_kv=torch.ones(2, dtype=torch.int32), topk=8, cmp_ratio=1,
              cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32))
    kw.update(over)
    return kw


@pytest.mark.parametrize("bad", [
    dict(q_index=torch.zeros(3, 4, 128)), dict(q_index=torch.zeros(1, 3, 4, 128, dtype=BF)),
    dict(layout_q="BSND"), dict(q_index=torch.zeros(3, 129, 128, dtype=BF), weights=torch.zeros(3, 129)),
    dict(q_index=torch.zeros(3, 4, 96, dtype=BF)), dict(topk=0), dict(cmp_ratio=0),
    dict(weights=torch.zeros(3, 5)), dict(weights=torch.zeros(3, 4, dtype=torch.int32)),
    dict(index_k=torch.zeros(4, 16, 1, 128, dtype=H)), dict(index_k=torch.zeros(4, 16, 1, 64, dtype=BF)),
    dict(index_k=_u8(4, 16, 1, 128)), dict(index_k=_u8(4, 6, 1, 132)),
    dict(index_k=torch.zeros(4, 16, 128, dtype=BF)), dict(index_k=torch.zeros(0, 16, 1, 128, dtype=BF)),
    dict(index_block_table=torch.zeros(1, 4, dtype=torch.int32)),
    dict(index_block_table=torch.zeros(8, dtype=torch.int32)),
    dict(index_block_table=torch.zeros(2, 0, dtype=torch.int32)),
    dict(seqused_kv=torch.ones(1, dtype=torch.int32)), dict(max_seqlen_kv=-1),
    dict(index_block_table=torch.zeros(2, (1 << 20) + 1, dtype=torch.int32)),
    dict(cu_seqlens_q=torch.zeros(0, dtype=torch.int32)),
])
def test_topk_refusals(bad):
    with pytest.raises(ValueError):
        sparse_topk_indices(**_topk(**bad))


def test_topk_layout_assertions():
    with pytest.raises(AssertionError):
        sparse_topk_indices(**_topk(layout_q="BNSD"))
    with pytest.raises(AssertionError):
        sparse_topk_indices(**_topk(cu_seqlens_q=None))


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        norm_rope_heads(**_rope())
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        append_kv_rope(**_append())
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        sparse_topk_indices(**_topk())


def test_gradients_are_refused():
    for call, kw, name in ((norm_rope_heads, _rope(), "q"), (append_kv_rope, _append(), "kv"),
                           (norm_rope_heads, _rope(), "norm_weight"),
                           (sparse_topk_indices, _topk(), "weights"),
                           (sparse_topk_indices, _topk(), "q_index")):
        kw[name] = kw[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            call(**kw)
        with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm GPU"):
            call(**kw)


def _row_args(**over):
    a = _lib.SasRowArgs()
    a.x = a.out = a.positions = a.cos_sin = a.norm_weight = a.slots = 4096
    a.tokens, a.heads, a.dim, a.norm_dim, a.rope_dim, a.rope_offset = 2, 1, 128, 128, 64, 64
    a.interleaved, a.max_position, a.block_size, a.cache_rows = 1, 16, 16, 64
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(heads=0), dict(dim=0), dict(dim=1032), dict(dim=12), dict(dtype=2),
    dict(norm_dim=136), dict(norm_dim=4), dict(norm_dim=-8), dict(rope_dim=60),
    dict(rope_dim=24, interleaved=0), dict(rope_offset=72), dict(rope_offset=-8), dict(rope_offset=4),
    dict(x=None), dict(out=None), dict(norm_weight=None), dict(positions=None), dict(cos_sin=None),
    dict(max_position=0), dict(x=4104), dict(out=4104), dict(cos_sin=4100), dict(norm_weight=4100),
    dict(x_token_stride=4), dict(x_head_stride=4), dict(tokens=1 << 30, heads=2),
])
def test_row_entries_refuse(bad):
    lib = _lib.load()
    for entry, name in ((lib.sas_norm_rope, "sas_norm_rope"), (lib.sas_kv_append_rope, "sas_kv_append_rope")):
        assert entry(ctypes.byref(_row_args(**bad)), None) == -1
        assert name in _lib.last_error()
        assert entry(None, None) == -1


def test_row_entries_refuse_their_own():
    lib = _lib.load()
    for bad in (dict(out_token_stride=4), dict(out_head_stride=4)):
        assert lib.sas_norm_rope(ctypes.byref(_row_args(**bad)), None) == -1
    for bad in (dict(heads=2), dict(cache_rows=-1), dict(row_format=3), dict(slots=None),
                dict(row_format=1), dict(row_format=2, dim=256), dict(row_format=2, block_size=0),
                dict(row_format=2, cache_rows=65), dict(row_format=2, block_size=6, cache_rows=66)):
        assert lib.sas_kv_append_rope(ctypes.byref(_row_args(**bad)), None) == -1
    assert lib.sas_norm_rope(ctypes.byref(_row_args(tokens=0)), None) == 0   # nothing to do
    assert lib.sas_kv_append_rope(ctypes.byref(_row_args(tokens=0)), None) == 0


def _select_args(**over):
    a = _lib.SasSelectArgs()
    a.q = a.weights = a.keys = a.block_table = a.seqused_kv = a.out = a.workspace = 4096
    a.workspace_bytes = 1 << 40
    a.batch, a.tokens, a.rows_per_seq, a.heads, a.dim, a.topk, a.cmp_ratio = 2, 2, 1, 4, 128, 8, 1
    a.block_num, a.block_size, a.table_len, a.max_keys = 4, 16, 4, 64
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad, rc", [
    (dict(batch=-1), -1), (dict(tokens=-1), -1), (dict(heads=0), -1), (dict(heads=129), -1),
    (dict(dim=96), -2), (dict(topk=0), -1), (dict(cmp_ratio=0), -1), (dict(dtype=2), -1),
    (dict(key_format=1), -1), (dict(block_num=0), -1), (dict(block_size=0), -1),
    (dict(table_len=0), -1), (dict(block_num=1 << 28), -2), (dict(max_keys=65), -1),
    (dict(max_keys=0), -1), (dict(key_format=2, block_size=6, max_keys=8), -1),
    (dict(rows_per_seq=3), -1), (dict(rows_per_seq=0), -1), (dict(q=None), -1), (dict(out=None), -1),
    (dict(workspace=None), -1), (dict(q=4100), -1), (dict(workspace=4104), -1),
    (dict(workspace_bytes=16), -3),
])
def test_select_entry_refuses(bad, rc):
    assert _lib.load().sas_topk_select(ctypes.byref(_select_args(**bad)), None) == rc
    assert "sas_topk_select" in _lib.last_error()


def test_select_workspace():
    lib = _lib.load()
    need = lib.sas_topk_select_workspace(ctypes.byref(_select_args()))
    assert 2 * 64 * 4 < need < 1 << 16          # two rows of 64 scores and the norms
    wide = _select_args(tokens=1 << 16, batch=1 << 16, max_keys=1 << 17, table_len=1 << 13)
    assert lib.sas_topk_select_workspace(ctypes.byref(wide)) < 600 << 20  # passes, not all rows
    assert lib.sas_topk_select_workspace(ctypes.byref(_select_args(dim=7))) == -1
    assert lib.sas_topk_select(ctypes.byref(_select_args(tokens=0, batch=0)), None) == 0
    assert re.search(r"SAS_SELECT_MAX_KEYS \(1 << 24\)", open(
        __file__.replace("tests/test_row_ops_host.py", "include/sas_mi355x.h")).read())
    assert _lib.SELECT_MAX_KEYS == 1 << 24
