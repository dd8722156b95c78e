"""Attention over the paged cache, block-sparse decoding and eviction by weight on an MI355X: the calls at the edge of what the
entry points allow, against the definitions in 64 bits (oracle/attention.py).  Cases and tolerances are those of
test_gpu_attention.py.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch

from oracle import attention as oat
from test_gpu_attention import BF16, DEV, EPS, FP8, FP16, Case, _check_rows, _check_weights, _weights
from triattention_amd import ops

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- more rows than max_rows
def _expected_of_first_rows(case, kept):
    """What oracle.attend gives for the first kept[b] rows of every sequence: they see no later new token, so the sequence might
    end behind the last of them.  The slots of the new tokens behind it receive nothing."""
    want = []
    for b, m in enumerate(kept):
        k, v, there = case.sequence(b)
        t = case.lens[b] - case.rows[b] + m
        part = slice(case.starts[b], case.starts[b] + m)
        o, z, w, mean_abs, reach = oat.attend(case.q[part], k[:t], v[:t], there[:t], case.parents[part], case.scale)
        want.append((o, z, torch.cat([w, torch.zeros(case.rows[b] - m, case.h, dtype=torch.float64)]), mean_abs, reach))
    return want


def _check_first_rows(case, kept, out, lse, want):
    at = torch.tensor([case.starts[b] + i for b, m in enumerate(kept) for i in range(m)], dtype=torch.long)
    view = copy.copy(case)
    view.starts = [sum(kept[:b]) for b in range(len(kept) + 1)]
    _check_rows(view, out.cpu()[at], lse.cpu()[at], want)
    return at


@pytest.mark.parametrize("heads,rows,most,types", [
    ((4, 2), [16, 3, 9, 0], 8, dict()), ((4, 2), [6, 1, 5, 2], 1, dict(dtype=FP16)), ((16, 16), [5, 2, 9, 3], 4, dict(dtype=FP8, row_scales=True)),
    ((8, 1), [12, 4, 3, 0], 4, dict()), ((40, 2), [7, 9, 2, 1], 1, dict(dtype=FP8, query=FP16, row_scales=True)),
    ((32, 2), [20, 8, 9, 40], 8, dict()), ((16, 1), [100, 64, 65, 2], 64, dict(dtype=FP16)), ((2, 2), [130, 70, 90, 3], 2, dict()),
    ((8, 2), [130, 70, 90, 3], 33, dict(dtype=FP8)),
])
@pytest.mark.parametrize("mode", ["add", "set"])
def test_rows_beyond_max_rows_are_left_out_and_the_others_are_what_they_are(heads, rows, most, types, mode):
    """The new tokens are the last of the sequence whether their rows are computed or not: kept rows see none behind them, the slots
    of all new tokens are written."""
    lens = [300, 90, 200, 60]
    case = Case(lens, q_heads=heads[0], kv_heads=heads[1], dim=64, rows=rows, seed=most + rows[0], **types)
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    out = torch.full_like(case.q, 7.0).to(DEV)
    print(f"rows beyond {most}: heads={heads} rows={rows} {types} {mode}", flush=True)
    _, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=most,
                              weights=weights, weight_mode=mode, out=out, want_lse=True)
    kept = [min(n, most) for n in rows]
    want = _expected_of_first_rows(case, kept)
    at = _check_first_rows(case, kept, out, lse, want)
    left = torch.ones(len(out), dtype=torch.bool)
    left[at] = False
    assert bool((out.cpu()[left] == 7.0).all())
    _check_weights(case, weights, before, want, mode)


def test_odd_numbers_of_tokens_whose_rows_are_left_out_reach_nobody():
    """NaN keys, values and value scales of new tokens behind max_rows, of some more than 64 behind the first."""
    for heads in ((4, 2), (32, 2)):
        case = Case([300, 90], q_heads=heads[0], kv_heads=heads[1], rows=[130, 12], seed=4, dtype=FP8, row_scales=True)
        for b, i in ((0, 5), (0, 63), (0, 64), (0, 70), (0, 129), (1, 11)):
            t = case.lens[b] - case.rows[b] + i
            at = case.tables[b][t // case.block], t % case.block
            case.cache[1][0].view(torch.uint8)[at][:] = 0x7f
            case.cache[0][0].view(torch.uint8)[at][:] = 0x7f
            case.scales[1][0][at] = math.nan
        kv, batch = case.device()
        print(f"odd numbers behind max_rows {heads}", flush=True)
        out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=4, want_lse=True)
        _check_first_rows(case, [4, 4], out, lse, _expected_of_first_rows(case, [4, 4]))


@pytest.mark.parametrize("heads", [(4, 2), (40, 2)])
def test_rows_that_q_does_not_have_are_left_out(heads):
    """row_starts that name more rows than q has: the last sequence's first rows are there."""
    case = Case([90, 200], q_heads=heads[0], kv_heads=heads[1], rows=[3, 9], seed=6)
    kv, batch = case.device()
    print(f"rows q does not have {heads}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q[:8].to(DEV), row_starts=case.dev_starts, parents=case.dev_parents[:8], max_rows=9, want_lse=True)
    _check_first_rows(case, [3, 5], out, lse, _expected_of_first_rows(case, [3, 5]))


def test_without_max_rows_every_row_is_computed():
    case = Case([90, 200], rows=[3, 9], seed=6)
    kv, batch = case.device()
    print("no max_rows", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, want_lse=True)
    _check_rows(case, out, lse, case.expected())


# ------------------------------------------------------------------------ out in place of q
@pytest.mark.parametrize("heads,dim,rows", [((8, 2), 64, [1, 1]), ((8, 1), 128, [4, 3]), ((32, 1), 128, [1, 1]), ((33, 1), 64, [1, 1]),
                                            ((32, 2), 128, [9, 4]), ((9, 1), 256, [9, 2])])
@pytest.mark.parametrize("layout", ["same", "beside", "shifted_rows"])
def test_out_may_be_q(heads, dim, rows, layout):
    """The same memory, or parts of one tensor with q and out in turn: what a call with memory of its own gives.  A copy of q
    is what the weights of many rows then go by."""
    case = Case([3000, 41], q_heads=heads[0], kv_heads=heads[1], dim=dim, rows=rows, seed=dim + heads[0])
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    args = dict(row_starts=case.dev_starts, parents=case.dev_parents, max_rows=max(rows), want_lse=True)
    want, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, **args)
    n = len(case.q)
    if layout == "same":
        q = out = case.q.to(DEV)
    elif layout == "beside":                  # the rows of q and out in turn
        room = torch.empty(n, 2, heads[0], dim, dtype=BF16, device=DEV)
        q, out = room[:, 0], room[:, 1]
    else:                                     # heads before rows, q's rows ahead of out's in every head
        room = torch.empty(heads[0], 2 * n, dim, dtype=BF16, device=DEV)
        q, out = room[:, :n].transpose(0, 1), room[:, n:].transpose(0, 1)
    q.copy_(case.q)
    again = before.to(DEV)
    print(f"out in q's memory heads={heads} dim={dim} rows={rows} {layout}", flush=True)
    got, lse2 = ops.attend_paged(kv, batch, q, weights=again, out=out, **args)
    assert torch.equal(got, want) and torch.equal(lse, lse2)
    assert torch.equal(again, weights)
    _check_weights(case, again, before, case.expected(), "add")


def test_out_in_q_s_memory_captured():
    """The copy of q is of the call: every replay takes what then stands there."""
    case = Case([700, 41], q_heads=32, kv_heads=2, rows=[9, 4], seed=2)
    kv, batch = case.device()
    args = dict(row_starts=case.dev_starts, parents=case.dev_parents, max_rows=9, want_lse=True)
    buf = case.q.to(DEV)
    weights = torch.zeros(1, case.pool, 16, 2, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attend_paged(kv, batch, buf, weights=weights, out=buf, **args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, lse = ops.attend_paged(kv, batch, buf, weights=weights, weight_mode="set", out=buf, **args)
    for rep in range(3):
        q = torch.randn(case.q.shape, device=DEV).to(BF16)
        expect = torch.zeros_like(weights)
        want, want_lse = ops.attend_paged(kv, batch, q, weights=expect, weight_mode="set", **args)
        buf.copy_(q)
        weights.zero_()
        print(f"replay {rep}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf, want) and torch.equal(lse, want_lse) and torch.equal(weights, expect)


# --------------------------------------------------------------------------------- no rows
@pytest.mark.parametrize("heads,most", [((8, 2), 1), ((8, 2), 16), ((16, 1), 64)])
@pytest.mark.parametrize("mode", ["add", "set"])
def test_a_call_of_no_rows(heads, most, mode):
    """Nothing to attend: no error; "set" writes a weight of nothing for every token, "add" adds it."""
    case = Case([5000, 41, 0], q_heads=heads[0], kv_heads=heads[1], dim=64, rows=[0, 0, 0], seed=3)
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"no rows {heads} {most} {mode}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, max_rows=most, weights=weights, weight_mode=mode,
                                want_lse=True)
    assert out.shape == (0, heads[0], 64) and lse.shape == (0, heads[0])
    expect = before.clone()
    if mode == "set":
        for b, t in enumerate(case.lens):
            for i in range(t):
                expect[0, case.tables[b][i // 16], i % 16] = 0
    assert torch.equal(weights.cpu(), expect)
    out, none = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, max_rows=most)
    assert len(out) == 0 and none is None


# ------------------------------------------------------------- infinities and NaN in the cache
@pytest.mark.parametrize("heads,lens", [((4, 1), [9000]), ((8, 2), [300]), ((40, 2), [9000])])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_odd_values_are_seen_however_little_they_weigh(heads, lens, odd):
    """A value that is no number, of a token whose weight is less than fp32 holds: not hidden, whichever workgroup or wave had it."""
    case = Case(lens, q_heads=heads[0], kv_heads=heads[1], dim=64, seed=9)
    t = lens[0]
    g = heads[0] // heads[1]
    case.q[:] = case.q[:, :1].abs() + 0.5                # (the same query for all heads)
    for h in range(heads[1]):
        case.cache[0][0][case.tables[0][0], 3, h] = case.q[0, h * g] * 40
    at = t - 30
    case.cache[1][0][case.tables[0][at // 16], at % 16, 0, 5] = odd
    kv, batch = case.device()
    print(f"odd value of no weight {heads} {odd}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), want_lse=True)
    out = out.cpu().float()
    assert bool((~torch.isfinite(out[0, :g, 5])).all())
    out[0, :g, 5] = 0
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("query", [BF16, FP16])
@pytest.mark.parametrize("heads,rows", [((4, 2), 1), ((40, 2), 1)])
def test_infinite_value_scales(heads, rows, query):
    """The only scale of a sequence, the first one and one among others."""
    case = Case([1, 200, 200, 16], q_heads=heads[0], kv_heads=heads[1], dim=64, seed=8, dtype=FP8, query=query, row_scales=True)
    for b, i in ((0, 0), (1, 0), (2, 77)):
        case.scales[1][0][case.tables[b][i // 16], i % 16, 0] = math.inf
    case.scales[1][0][torch.tensor(case.tables[3])] = 0.0
    kv, batch = case.device()
    print(f"infinite scales {heads} {query}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), want_lse=True)
    _check_rows(case, out, lse, case.expected())


# -------------------------------------------------------------------------- chosen blocks
def test_first_and_last_blocks_are_read_whatever_others_score():
    """More blocks with a NaN or infinite key than are chosen: those asked for by place are among them all the same."""
    case = Case([16 * 40], seed=1)
    for j in range(2, 38):
        case.cache[0][0][case.tables[0][j], 3, 0, 5] = math.nan
        case.cache[0][0][case.tables[0][j], 3, 1] = math.inf * torch.sign(case.q[0, 4].float())
    case.q[0, 4:] = case.q[0, 4]
    kv, batch = case.device()
    bounds = ops.update_block_bounds(kv, batch, ops.block_bounds(kv))
    print("blocks by place", flush=True)
    _, _, blocks = ops.attend_blocks(kv, batch, case.q.to(DEV), bounds, top_blocks=7, sink_blocks=1, recent_blocks=2)
    want = oat.choose_blocks(case.q[0], oat.bounds_of(case.cache[0][0], case.tables[0], 640, BF16), 7, 1, 2, True)
    assert want == [[0, 2, 3, 4, 5, 38, 39]] * 2
    assert blocks[0].tolist() == want


@pytest.mark.parametrize("types", [dict(), dict(dtype=FP16), dict(dtype=FP8), dict(dtype=FP8, row_scales=True)], ids=["bf16", "fp16", "fp8", "fp8_scaled"])
@pytest.mark.parametrize("block", [1, 16])
def test_keys_lie_within_their_block_s_bounds(types, block):
    """Exactly, but for scaled fp8 keys: there the bounds are rounded to bf16, by at most half a step (2^-8 of the bound)."""
    case = Case([333], block=block, seed=block, garbage=None, **types)
    kv, batch = case.device()
    print(f"bounds {types} {block}", flush=True)
    bounds = ops.update_block_bounds(kv, batch, ops.block_bounds(kv)).cpu()
    k, _ = oat.rows_of(case.cache[0][0], case.tables[0], 333, case.scales[0][0])
    b = bounds[0, torch.tensor([case.tables[0][i // block] for i in range(333)])].double()
    # (the scaled key itself is a product in fp32)
    slack = (2.0 ** -8 + 2.0 ** -23) if types.get("row_scales") else 0.0
    assert bool((k >= b[:, :, 0] - slack * b[:, :, 0].abs()).all()) and bool((k <= b[:, :, 1] + slack * b[:, :, 1].abs()).all())


# ------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("reduce,shared", [("mean", False), ("max", False), (None, False), ("mean", True), ("max", True)])
def test_negative_nan_weights_are_kept_first_too(reduce, shared):
    """A NaN counts as more than any number whatever its sign bit."""
    case = Case([200], q_heads=8, kv_heads=4, layers=2, seed=3, garbage=None)
    kv, batch = case.device(budgets=[20])
    before = _weights(case)
    odd = [4, 50, 51, 100]
    for t in odd:
        before[:, case.tables[0][t // 16], t % 16, 1] = torch.tensor(-0x400000, dtype=torch.int32).view(torch.float32)
    assert int(before[0, case.tables[0][0], 4, 1:2].contiguous().view(torch.int32)[0]) == -0x400000
    weights = before.to(DEV)
    print(f"negative NaN {reduce} {shared}", flush=True)
    keep, scores = ops.select_by_weight(kv, batch, weights, ops.EvictConfig(window_size=8, layer_reduce=reduce, shared=shared), want_scores=True)
    keep, scores = keep.cpu(), scores.cpu()
    for r in range(len(keep)):
        if shared or r % 4 == 1:
            assert set(odd) <= set(keep[r].tolist()), r
            assert bool(torch.isnan(scores[r, odd]).all())
        assert set(range(192, 200)) <= set(keep[r].tolist()), r


def test_eviction_of_long_rows_keeps_what_the_definition_keeps_in_every_head():
    """Rows longer than a tile of the weights' move, every head's list against the definition."""
    case = Case([9000], q_heads=4, kv_heads=4, dim=64, layers=2, seed=2, garbage=None)
    kv, batch = case.device(budgets=[5000])
    before = _weights(case)
    before[1, case.tables[0][7], 3, 2] = math.inf
    weights = before.to(DEV)
    print("evict long", flush=True)
    keep = ops.evict_step(kv, batch, weights, ops.EvictConfig(window_size=0)).cpu()
    slots = torch.tensor([case.tables[0][i // 16] * 16 + i % 16 for i in range(9000)])
    flat = before.view(2, -1, 4)[:, slots]
    mean = (flat.double().sum(0) / 2).float()
    for h in range(4):
        want = torch.sort(mean[:, h], descending=True, stable=True).indices[:5000].sort().values
        assert torch.equal(keep[h].long(), want), h
        assert torch.equal(weights.cpu().view(2, -1, 4)[:, slots[:5000], h], flat[:, want, h])
    assert 7 * 16 + 3 in keep[2].tolist()


# ------------------------------------------------------------- what weights are rounded to
ROUNDING = [dict(), dict(dtype=FP16), dict(dtype=FP8), dict(dtype=FP8, row_scales=True), dict(dtype=FP8, query=FP16),
            dict(dtype=FP8, query=FP16, row_scales=True)]


@pytest.mark.parametrize("types", ROUNDING, ids=["bf16", "fp16", "fp8", "fp8_scaled", "fp8_fp16q", "fp8_fp16q_scaled"])
@pytest.mark.parametrize("dim,heads,rows", [(64, (4, 2), 1), (128, (8, 2), 4), (256, (16, 1), 1), (64, (32, 16), 2), (128, (20, 1), 1), (64, (32, 2), 4),
                                            (256, (8, 2), 9), (64, (32, 2), 7), (128, (40, 1), 3), (128, (32, 1), 8), (256, (32, 1), 5)])
def test_weights_are_rounded_as_stated(types, dim, heads, rows):
    """Two numbers of the queries' type: half a step of half a step.  One of them beyond 64 rows, and of fp8 beyond 16.  Tokens of like
    weights and values of either sign, whose sums leave the rounding errors bare."""
    case = Case([70, 1, 33, 150], q_heads=heads[0], kv_heads=heads[1], dim=dim, rows=[rows, 1, rows, rows], seed=dim + rows, q_scale=0.2, **types)
    if heads == (32, 16):                     # (enough of them that a wave has a head to itself)
        case = Case([9000 - 7 * i for i in range(4)], q_heads=32, kv_heads=16, dim=dim, rows=[rows] * 4, seed=dim + rows, q_scale=0.2, **types)
    kv, batch = case.device()
    print(f"rounding {types} dim={dim} heads={heads} rows={rows}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=rows, want_lse=True)
    step = EPS[case.query]
    two = rows * heads[0] // heads[1] <= (16 if types.get("dtype") == FP8 else 64)
    _check_rows(case, out, lse, case.expected(), weight_eps=step * step if two else step)


# ----------------------------------------------------------- scratch of a long sequence among short ones
@pytest.mark.parametrize("types", [dict(), dict(dtype=FP8, row_scales=True)], ids=["bf16", "fp8"])
@pytest.mark.parametrize("mode", ["add", "set"])
def test_weights_of_a_long_sequence_among_many_short_ones(types, mode):
    """Scores of all of them would take more than the cache: the weights come from the keys, of single rows too."""
    lens = [20000] + [1 + 7 * i % 90 for i in range(899)]
    heads = (64, 2)
    case = Case(lens, q_heads=heads[0], kv_heads=heads[1], dim=64, seed=4, garbage=None, **types)
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    print(f"long among short {types} {mode}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, weight_mode=mode, want_lse=True)
    assert torch.cuda.max_memory_allocated() - held < 1 << 30
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, mode)


# -------------------------------------------------------------- sizes beyond 32 bits
def test_sizes_beyond_32_bits_are_not_cut():
    """A window of more tokens than there can be guards all; counts that no call can have are refused."""
    case = Case([100, 40], seed=1, garbage=None)
    kv, batch = case.device(budgets=[30, 20])
    weights = _weights(case).to(DEV)
    bounds = ops.block_bounds(kv)
    q = case.q.to(DEV)
    print("beyond 32 bits", flush=True)
    for window in (100, (1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 40):
        keep, _ = ops.select_by_weight(kv, batch, weights, ops.EvictConfig(window_size=window))
        assert keep[0].tolist() == list(range(30)) and keep[2].tolist() == list(range(20)) + [-1] * 10
    every = ops.update_block_bounds(kv, batch, bounds.clone())
    for new in (100, 1 << 31, (1 << 32) + 1):
        assert torch.equal(ops.update_block_bounds(kv, batch, bounds.clone(), new_tokens=new), every)
    for args in (dict(top_blocks=(1 << 32) + 4), dict(top_blocks=4, sink_blocks=1 << 32), dict(top_blocks=4, recent_blocks=(1 << 32) + 1),
                 dict(top_blocks=4, sink_blocks=-1, recent_blocks=3)):
        with pytest.raises(ValueError):
            ops.attend_blocks(kv, batch, q, bounds, **args)
    for most in ((1 << 32) + 1, 0, -1, 65):
        with pytest.raises(ValueError):
            ops.attend_paged(kv, batch, q, row_starts=case.dev_starts, max_rows=most)
    with pytest.raises(ValueError):
        ops.select_by_weight(kv, batch, weights, ops.EvictConfig(window_size=-1))
