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
from test_gpu_attention import BF16, DEV, FP8, FP16, Case, _check_rows, _check_weights, _weights
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
