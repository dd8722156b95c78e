"""The attention and eviction entry points without a GPU: what the C boundary refuses, and the oracle they are held to."""
from __future__ import annotations

import ctypes as C
import math
import time

import pytest
import torch

from oracle import attention as oat
from triattention_amd import _lib


def _layout(**kw):
    base = dict(num_layers=2, num_kv_heads=4, head_dim=128, block_size=16, kv_dtype=0, stride_block=16 * 4 * 128,
                stride_token=4 * 128, stride_head=128, k_layers=8, v_layers=8)
    base.update(kw)
    return _lib.KvLayout(**base)


def _batch(**kw):
    base = dict(num_seqs=3, max_seq_len=100, max_budget=50, block_table_pitch=7, block_table=8, seq_lens=8, budgets=8)
    base.update(kw)
    return _lib.Batch(**base)


def _attend(**kw):
    base = dict(layer=0, num_q_heads=8, num_rows=3, max_rows=1, q_dtype=0, num_blocks=40, q=16, q_stride_row=8 * 128,
                q_stride_head=128, out=16, out_stride_row=8 * 128, out_stride_head=128, scale=0.1, k_scale=1.0, v_scale=1.0)
    base.update(kw)
    return _lib.AttendParams(**base)


def _blocks(**kw):
    base = dict(bounds=16, top_blocks=8, sink_blocks=1, recent_blocks=2, group_reduce=1, blocks=8)
    base.update(kw)
    return _lib.BlockParams(**base)


def _evict(**kw):
    base = dict(num_blocks=40, window_size=4, protect_prefill=0, layer_reduce=0, shared=0, weights=16,
                weights_stride_layer=40 * 16 * 4)
    base.update(kw)
    return _lib.EvictParams(**base)


def test_attention_plans_are_made_without_a_device():
    lib = _lib.load()
    assert lib.tri_attend_workspace_bytes(C.byref(_layout()), C.byref(_batch()), C.byref(_attend())) > 0
    assert lib.tri_attend_blocks_workspace_bytes(C.byref(_layout()), C.byref(_batch()), C.byref(_attend()), C.byref(_blocks())) > 0
    assert lib.tri_evict_workspace_bytes(C.byref(_layout()), C.byref(_batch()), C.byref(_evict())) >= 3 * 4 * 100 * 4
    # weights need the scores of every row besides
    plain = lib.tri_attend_workspace_bytes(C.byref(_layout()), C.byref(_batch()), C.byref(_attend()))
    more = lib.tri_attend_workspace_bytes(C.byref(_layout()), C.byref(_batch()), C.byref(_attend(weights=16)))
    assert more >= plain + 3 * 8 * 100 * 4


@pytest.mark.parametrize("layout,batch,params,code,word", [
    (dict(head_dim=96), {}, {}, _lib.TRI_ERR_UNSUPPORTED, b"head_dim"),
    (dict(v_layers=None), {}, {}, _lib.TRI_ERR_INVALID_ARGUMENT, b"v_layers"),
    (dict(stride_token=1 << 25), {}, {}, _lib.TRI_ERR_UNSUPPORTED, b"stride_token"),
    (dict(kv_dtype=1), {}, {}, _lib.TRI_ERR_UNSUPPORTED, b"queries of type"),
    ({}, dict(num_seqs=0), {}, _lib.TRI_ERR_INVALID_ARGUMENT, b"num_seqs"),
    ({}, dict(seq_lens=None), {}, _lib.TRI_ERR_INVALID_ARGUMENT, b"seq_lens"),
    ({}, {}, dict(layer=2), _lib.TRI_ERR_INVALID_ARGUMENT, b"layer"),
    ({}, {}, dict(layer=-1), _lib.TRI_ERR_INVALID_ARGUMENT, b"layer"),
    ({}, {}, dict(num_q_heads=6), _lib.TRI_ERR_INVALID_ARGUMENT, b"multiple"),
    ({}, {}, dict(q_dtype=2), _lib.TRI_ERR_UNSUPPORTED, b"q_dtype"),
    ({}, {}, dict(num_blocks=0), _lib.TRI_ERR_INVALID_ARGUMENT, b"num_blocks"),
    ({}, {}, dict(max_rows=0, row_starts=8), _lib.TRI_ERR_UNSUPPORTED, b"max_rows"),
    ({}, {}, dict(max_rows=65, row_starts=8), _lib.TRI_ERR_UNSUPPORTED, b"max_rows"),
    ({}, {}, dict(num_rows=4), _lib.TRI_ERR_INVALID_ARGUMENT, b"row_starts"),
    ({}, {}, dict(max_rows=2), _lib.TRI_ERR_INVALID_ARGUMENT, b"row_starts"),
    ({}, {}, dict(parents=8), _lib.TRI_ERR_INVALID_ARGUMENT, b"parents"),
    ({}, {}, dict(q_stride_row=8 * 128 + 4), _lib.TRI_ERR_INVALID_ARGUMENT, b"strides"),
    ({}, {}, dict(out_stride_head=64), _lib.TRI_ERR_INVALID_ARGUMENT, b"out_stride_head"),
    ({}, {}, dict(out_stride_row=64), _lib.TRI_ERR_INVALID_ARGUMENT, b"out_stride_row"),
    ({}, {}, dict(scale=math.nan), _lib.TRI_ERR_INVALID_ARGUMENT, b"finite"),
    ({}, {}, dict(scale=0.0), _lib.TRI_ERR_INVALID_ARGUMENT, b"positive"),
    ({}, {}, dict(scale=-1.0), _lib.TRI_ERR_INVALID_ARGUMENT, b"positive"),
    ({}, {}, dict(v_scale=math.inf), _lib.TRI_ERR_INVALID_ARGUMENT, b"finite"),
    ({}, {}, dict(weight_mode=2), _lib.TRI_ERR_INVALID_ARGUMENT, b"weight_mode"),
    ({}, {}, dict(q=None), _lib.TRI_ERR_INVALID_ARGUMENT, b"NULL"),
    ({}, {}, dict(out=8), _lib.TRI_ERR_INVALID_ARGUMENT, b"aligned"),
])
def test_attention_refuses(layout, batch, params, code, word):
    lib = _lib.load()
    args = C.byref(_layout(**layout)), C.byref(_batch(**batch)), C.byref(_attend(**params))
    assert lib.tri_attend_paged(*args, 256, 1 << 40, None) == code
    assert word in lib.tri_last_error()
    if "q" not in params and "out" not in params:
        assert lib.tri_attend_workspace_bytes(*args) == 0


def test_plans_of_many_sequences_stay_small_and_are_made_quickly():
    """A long sequence among many short ones is cut, the partial results stay within 512 MiB, and no number of sequences makes the host search long."""
    lib = _lib.load()
    for num, rows in ((600, 1), (600, 64), (4096, 1)):
        lens = [100 + i % 7 for i in range(num - 1)] + [120000]
        host = (C.c_int32 * num)(*lens)
        batch = _batch(num_seqs=num, max_seq_len=max(lens), block_table_pitch=7500, seq_lens_host=C.cast(host, C.c_void_p))
        p = _attend(num_rows=num * rows, max_rows=rows, row_starts=8)
        args = C.byref(_layout()), C.byref(batch), C.byref(p)
        nbytes = lib.tri_attend_workspace_bytes(*args)
        assert 0 < nbytes <= (512 << 20) + 1024, (num, rows, nbytes)
        start = time.perf_counter()
        for _ in range(100):
            lib.tri_attend_workspace_bytes(*args)
        assert time.perf_counter() - start < 1.0


def test_tables_too_narrow_for_the_longest_sequence_are_refused():
    lib = _lib.load()
    kv, batch = C.byref(_layout()), C.byref(_batch(block_table_pitch=6))
    for code in (lib.tri_attend_paged(kv, batch, C.byref(_attend()), 256, 1 << 40, None),
                 lib.tri_attend_blocks(kv, batch, C.byref(_attend()), C.byref(_blocks()), 256, 1 << 40, None),
                 lib.tri_block_bounds(kv, batch, 40, 0, 16, 40 * 4 * 256, None),
                 lib.tri_select_by_weight(kv, batch, C.byref(_evict()), None, 8, 256, 1 << 40, None),
                 lib.tri_evict_step(kv, batch, C.byref(_evict()), 8, 256, 1 << 40, None)):
        assert code == _lib.TRI_ERR_INVALID_ARGUMENT and b"block_table_pitch" in lib.tri_last_error()


def test_attention_refuses_a_missing_small_or_unaligned_workspace():
    lib = _lib.load()
    args = C.byref(_layout()), C.byref(_batch(max_seq_len=100000)), C.byref(_attend())
    need = lib.tri_attend_workspace_bytes(*args)
    assert need > 256
    for at, size in ((None, need), (256, need - 1), (128, need)):
        assert lib.tri_attend_paged(*args, at, size, None) == _lib.TRI_ERR_WORKSPACE


@pytest.mark.parametrize("params,block,code,word", [
    (dict(row_starts=8), {}, _lib.TRI_ERR_UNSUPPORTED, b"one row"),
    (dict(weights=16), {}, _lib.TRI_ERR_UNSUPPORTED, b"no weights"),
    ({}, dict(top_blocks=0), _lib.TRI_ERR_INVALID_ARGUMENT, b"of 0"),
    ({}, dict(sink_blocks=-1), _lib.TRI_ERR_INVALID_ARGUMENT, b"sink"),
    ({}, dict(sink_blocks=5, recent_blocks=4), _lib.TRI_ERR_INVALID_ARGUMENT, b"recent"),
    ({}, dict(group_reduce=2), _lib.TRI_ERR_INVALID_ARGUMENT, b"group_reduce"),
    ({}, dict(bounds=None), _lib.TRI_ERR_INVALID_ARGUMENT, b"bounds"),
    ({}, dict(bounds=8), _lib.TRI_ERR_INVALID_ARGUMENT, b"bounds"),
    ({}, dict(blocks=None), _lib.TRI_ERR_INVALID_ARGUMENT, b"blocks"),
])
def test_attention_over_blocks_refuses(params, block, code, word):
    lib = _lib.load()
    assert lib.tri_attend_blocks(C.byref(_layout()), C.byref(_batch()), C.byref(_attend(**params)), C.byref(_blocks(**block)), 256,
                                 1 << 40, None) == code
    assert word in lib.tri_last_error()


@pytest.mark.parametrize("args,word", [((0, 1, 16, 40 * 4 * 256), b"num_blocks"), ((40, -1, 16, 40 * 4 * 256), b"new_tokens"),
                                       ((40, 1, None, 40 * 4 * 256), b"bounds"), ((40, 1, 8, 40 * 4 * 256), b"bounds"),
                                       ((40, 1, 16, 40 * 4 * 256 - 8), b"less than a layer")])
def test_block_bounds_refuse(args, word):
    lib = _lib.load()
    assert lib.tri_block_bounds(C.byref(_layout()), C.byref(_batch()), *args, None) == _lib.TRI_ERR_INVALID_ARGUMENT
    assert word in lib.tri_last_error()


@pytest.mark.parametrize("batch,params,word", [
    (dict(budgets=None), {}, b"budgets"), (dict(max_budget=0), {}, b"max_budget"), ({}, dict(num_blocks=0), b"num_blocks"),
    ({}, dict(window_size=-1), b"window_size"), ({}, dict(layer_reduce=3), b"layer_reduce"), ({}, dict(protect_prefill=1), b"prefill_lens"),
    ({}, dict(weights_stride_layer=40 * 16 * 4 - 1), b"less than a layer"), ({}, dict(weights=None), b"weights"),
])
def test_eviction_refuses(batch, params, word):
    lib = _lib.load()
    args = C.byref(_layout()), C.byref(_batch(**batch)), C.byref(_evict(**params))
    assert lib.tri_select_by_weight(*args, None, 8, 256, 1 << 40, None) == _lib.TRI_ERR_INVALID_ARGUMENT
    assert word in lib.tri_last_error()
    assert lib.tri_evict_step(*args, 8, 256, 1 << 40, None) == _lib.TRI_ERR_INVALID_ARGUMENT


def test_eviction_refuses_without_a_table_or_a_list():
    lib = _lib.load()
    args = C.byref(_layout()), C.byref(_batch(block_table=None)), C.byref(_evict())
    assert lib.tri_evict_step(*args, 8, 256, 1 << 40, None) == _lib.TRI_ERR_INVALID_ARGUMENT
    args = C.byref(_layout()), C.byref(_batch()), C.byref(_evict())
    assert lib.tri_select_by_weight(*args, None, None, 256, 1 << 40, None) == _lib.TRI_ERR_INVALID_ARGUMENT
    assert lib.tri_select_by_weight(*args, None, 8, 256, 16, None) == _lib.TRI_ERR_WORKSPACE


# ------------------------------------------------------------------ the oracle itself
def test_oracle_attention_is_a_softmax_over_what_a_row_sees():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(3, 4, 8, generator=g)
    k, v = torch.randn(9, 2, 8, generator=g).double(), torch.randn(9, 2, 8, generator=g).double()
    v[7] = math.nan                      # new token 1: seen by itself and by no other row below
    out, lse, weights, _, _ = oat.attend(q, k, v, torch.ones(9, dtype=torch.bool), [-1, 5, 0], 0.3)
    seen = {0: [0, 1, 2, 3, 4, 5, 6], 1: [0, 1, 2, 3, 4, 5, 7], 2: [0, 1, 2, 3, 4, 5, 6, 8]}
    for i, tokens in seen.items():
        for h in range(4):
            s = torch.tensor([float(q[i, h].double() @ k[t, h // 2]) * 0.3 for t in tokens], dtype=torch.float64)
            p = s.exp() / s.exp().sum()
            assert abs(float(lse[i, h]) - math.log(float(s.exp().sum()))) < 1e-12
            want = sum(p[x] * v[t, h // 2] for x, t in enumerate(tokens))
            if i == 1:
                assert bool(out[i, h].isnan().all())
            else:
                assert float((out[i, h] - want).abs().max()) < 1e-12
    # every row gives a weight of one per query head
    assert abs(float(weights.sum()) - 3 * 4) < 1e-12
    none = oat.attend(q[:1], k[:1], v[:1], torch.zeros(1, dtype=torch.bool), [-1], 0.3)
    assert float(none[0].abs().max()) == 0 and bool((none[1] == -math.inf).all())


def test_oracle_block_choice_and_keep_rows_break_ties_low():
    q = torch.tensor([[1.0, -2.0]])
    bounds = torch.tensor([[0.0, 0.0], [1.0, 1.0]]).expand(5, 1, 2, 2).clone()
    assert oat.choose_blocks(q, bounds, 2, 0, 0, True) == [[0, 1]]
    assert oat.choose_blocks(q, bounds, 2, 0, 1, True) == [[0, 4]]
    bounds[3, 0, 0, 1] = -1.0            # q . k may reach 1 * 1 + -2 * -1
    assert oat.choose_blocks(q, bounds, 1, 0, 0, True) == [[3]]
    w = torch.tensor([[[1.0], [5.0], [5.0], [0.0]], [[3.0], [1.0], [1.0], [0.0]]])      # [L, T, H]
    assert oat.keep_rows(oat.weight_scores(w, "mean", False, 1, 0), 2) == [[1, 3]]
    assert oat.keep_rows(oat.weight_scores(w, None, False, 0, 0), 2) == [[1, 2], [0, 1]]
    assert oat.keep_rows(oat.weight_scores(w, "max", True, 0, 1), 2) == [[0, 1]]
