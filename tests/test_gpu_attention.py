"""Attention over the paged cache, block-sparse decoding and eviction by weight on an MI355X, against the
definitions in 64 bits (oracle/attention.py).

Tolerances, from the arithmetic the header states (eps: half a step of a type, 2^-8 bf16, 2^-11 fp16, 2^-24 fp32):
 * a score is an fp32 sum of D exact products: off by at most D * 2^-24 * scale * sum |q_d k_d|; with row scales one
   product more (2^-24 of the score, inside the same bound);
 * lse: that, T additions of positive terms in fp32 (T * 2^-24), and a few steps of the exponential and the logarithm;
 * a weight p: e^(2 * score error) and the exponential's steps, relative;
 * out: every weight is rounded once to 16 bits for the product (eps of the weighted mean of |v|; weights below
   the smallest normal fp16 number by 2^-25 absolutely), fp32 accumulation of T terms, one rounding at the end (eps of out).
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as oat
from triattention_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
EPS = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}


class Case:
    """A cache of some sequences with everything the calls need, on the CPU and on the device."""

    def __init__(self, lens, q_heads=8, kv_heads=2, dim=128, block=16, dtype=BF16, query=None, row_scales=False, rows=None,
                 parents=None, layers=1, seed=0, pool=None, garbage=math.nan, kv_axis_apart=True, q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.block, self.hq, self.h, self.d, self.layers = list(lens), block, q_heads, kv_heads, dim, layers
        self.query = query or (dtype if dtype != FP8 else BF16)
        counts = [-(-t // block) for t in lens]
        self.pool = pool or sum(counts) + 3
        order = torch.randperm(self.pool, generator=g).tolist()
        self.tables, at = [], 0
        for n in counts:
            self.tables.append(order[at:at + n])
            at += n
        self.pitch = max(max(counts), 1) + 1
        self.cache, self.scales = ([], []), ([], [])
        for side in (0, 1):
            for _ in range(layers):
                x = torch.randn(self.pool, block, kv_heads, dim, generator=g)
                if side == 0:
                    x = x + 0.5 * torch.randn(1, 1, kv_heads, dim, generator=g)
                sc = None
                if dtype == FP8:
                    if row_scales:
                        sc = (x.abs().amax(-1) / 448 * (0.5 + torch.rand(self.pool, block, kv_heads, generator=g)))
                        x = x / sc.unsqueeze(-1)
                    x = x.clamp(-448, 448)
                x = x.to(dtype)
                # nothing that no sequence owns may matter
                if garbage is not None:
                    used = torch.zeros(self.pool, block, dtype=torch.bool)
                    for table, t in zip(self.tables, self.lens):
                        for i in range(t):
                            used[table[i // block], i % block] = True
                    if dtype == FP8:
                        x.view(torch.uint8)[~used] = 0x7f
                    else:
                        x[~used] = garbage
                self.cache[side].append(x)
                self.scales[side].append(sc)
        self.rows = rows if rows is not None else [1] * len(self.lens)
        starts = [sum(self.rows[:i]) for i in range(len(self.rows) + 1)]
        self.starts = starts
        if parents == "chain":
            self.parents = [i - 1 for n in self.rows for i in range(n)]
        else:
            self.parents = [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for n in self.rows for i in range(n)]
        self.q = (q_scale * torch.randn(starts[-1], q_heads, dim, generator=g)).to(self.query)
        self.scale = dim ** -0.5

    def device(self, budgets=None, prefill=None, host_lens=None):
        put = lambda lists: [x.to(DEV) for x in lists]           # noqa: E731
        self.k, self.v = put(self.cache[0]), put(self.cache[1])
        scaled = self.scales[0][0] is not None
        self.ks = [x.reshape(-1).contiguous().to(DEV) for x in self.scales[0]] if scaled else None
        self.vs = [x.reshape(-1).contiguous().to(DEV) for x in self.scales[1]] if scaled else None
        kv = ops.PagedKV(self.k, self.v, "half", self.ks, self.vs)
        table = torch.full((len(self.lens), self.pitch), -7, dtype=torch.int32)
        for i, t in enumerate(self.tables):
            table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        batch = ops.StepBatch(torch.device(DEV), host_lens or self.lens, block_tables=table.to(DEV), budgets=budgets, prefill_lens=prefill)
        if host_lens:
            batch.seq_lens.copy_(torch.tensor(self.lens, dtype=torch.int32))
        self.dev_starts = torch.tensor(self.starts, dtype=torch.int32, device=DEV)
        self.dev_parents = torch.tensor(self.parents or [0], dtype=torch.int32, device=DEV)[:len(self.parents)]
        return kv, batch

    def sequence(self, b, layer=0):
        k, there = oat.rows_of(self.cache[0][layer], self.tables[b], self.lens[b], self.scales[0][layer])
        v, _ = oat.rows_of(self.cache[1][layer], self.tables[b], self.lens[b], self.scales[1][layer])
        return k, v, there

    def expected(self, layer=0):
        """Per sequence: what oracle.attend returns for its rows."""
        got = []
        for b in range(len(self.lens)):
            k, v, there = self.sequence(b, layer)
            part = slice(self.starts[b], self.starts[b + 1])
            got.append(oat.attend(self.q[part], k, v, there, self.parents[part], self.scale))
        return got


def _score_error(case, reach):
    return case.d * 2.0 ** -24 * case.scale * reach


def _check_rows(case, out, lse, want, scale_v=1.0, weight_eps=None, more=0.0):
    """out and lse of every row of every sequence within the bounds above."""
    out, lse = out.cpu(), lse.cpu()
    eps = EPS[case.query]
    weight_eps = weight_eps or (EPS[BF16] if case.cache[0][0].dtype == FP8 else eps)
    for b, (o, z, _, mean_abs, reach) in enumerate(want):
        part = slice(case.starts[b], case.starts[b + 1])
        if part.start == part.stop:
            continue
        t = case.lens[b]
        err = _score_error(case, reach)
        got_z = lse[part].double()
        assert torch.equal(torch.isneginf(got_z), torch.isneginf(z)), (b, got_z, z)
        seen = ~torch.isneginf(z)
        tol = err + (t + 16) * 2.0 ** -24 + 2.0 ** -22 * z.abs()
        assert bool(((got_z - z).abs() <= tol)[seen].all()), (b, float(((got_z - z).abs() - tol)[seen].max()))
        got = out[part].double()
        assert bool((got[~seen] == 0).all())
        finite = torch.isfinite(o)
        assert torch.equal(torch.isnan(got), torch.isnan(o)), b
        assert torch.equal(got[~finite & ~torch.isnan(o)], o[~finite & ~torch.isnan(o)])
        vmax = max(1e-30, float(mean_abs[torch.isfinite(mean_abs)].abs().max()) if mean_abs.numel() else 0)
        bound = ((weight_eps + 2 * err.unsqueeze(-1) + (t + 64) * 2.0 ** -24) * mean_abs + eps * o.abs()
                 + t * 2.0 ** -25 * vmax * 8) * abs(scale_v) + 1e-30 + more
        if eps == EPS[FP16]:
            bound = bound + 2.0 ** -25           # (an output below the smallest normal number)
        off = (got - o * scale_v).abs()
        assert bool((off[finite] <= bound[finite]).all()), (b, float((off - bound)[finite].max()))


def _check_weights(case, weights, before, want, mode, layer=0):
    """Every slot of the cache's weights: those of a sequence changed as defined, all others as they were."""
    got = weights[layer].cpu()
    expect = before[layer].double().clone()
    tol = torch.zeros_like(expect)
    for b, (_, _, w, _, reach) in enumerate(want):
        t, n = case.lens[b], case.rows[b]
        err = float(_score_error(case, reach).max()) if reach.numel() else 0.0
        for i in range(t):
            p = case.tables[b][i // case.block]
            if not 0 <= p < case.pool:
                continue
            had = 0.0 if mode == "set" or i >= t - n else before[layer][p, i % case.block].double()
            expect[p, i % case.block] = had + w[i]
            tol[p, i % case.block] = w[i] * (2 * err + (t + 64) * 2.0 ** -24 + 2.0 ** -21) + (had + w[i]) * (n * case.hq + 2) * 2.0 ** -24
    assert bool(((got.double() - expect).abs() <= tol).all()), float(((got.double() - expect).abs() - tol).max())


def _weights(case, seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(case.layers, case.pool, case.block, case.h, generator=g) * 4


# ---------------------------------------------------------------- a decoding step with weights
TYPES = [dict(), dict(dtype=FP16), dict(dtype=FP8), dict(dtype=FP8, query=FP16, row_scales=True), dict(dtype=FP8, row_scales=True)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("types", TYPES, ids=["bf16", "fp16", "fp8", "fp8_fp16q_scaled", "fp8_scaled"])
@pytest.mark.parametrize("mode", ["add", "set"])
def test_decoding_step_with_weights(dim, types, mode):
    case = Case([1, 15, 16, 17, 33, 0, 129, 260], dim=dim, seed=dim, **types)
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"decode dim={dim} {types} {mode}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, weight_mode=mode, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, mode)


@pytest.mark.parametrize("heads", [(1, 1), (5, 5), (12, 3), (28, 4), (16, 1), (17, 1), (40, 2), (130, 2)])
def test_decoding_step_head_layouts(heads):
    """One to sixty-five query heads per KV head: from one row to more than a wave's tiles."""
    case = Case([70, 200, 5], q_heads=heads[0], kv_heads=heads[1], dim=64, seed=heads[0])
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"decode heads={heads}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, "add")


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,rows", [((8, 2), 1), ((40, 2), 1), ((8, 2), 9), ((16, 4), 40)])
@pytest.mark.parametrize("scales", ["none", "rows", "growing", "apart", "zero"])
def test_fp8_rows_with_fp16_queries_round_as_fp16(dim, heads, rows, scales):
    """Weights are rounded to fp16 (half a step, 2^-11), whatever scales the rows bring along: growing ones, which O has to follow, ones far
    apart and ones that are 0.  fp16 has 2^-25 absolutely for small weights: of the largest scale, times at most 448, a token."""
    case = Case([70, 333, 1], q_heads=heads[0], kv_heads=heads[1], dim=dim, rows=[min(rows, 70), rows, 1], seed=dim + rows, dtype=FP8, query=FP16,
                row_scales=scales != "none")
    more = 0.0
    if scales in ("growing", "apart", "zero"):
        s = case.scales[1][0]
        for table, t in zip(case.tables, case.lens):
            for i in range(t):
                at = (table[i // 16], i % 16)
                if scales == "growing":
                    s[at] *= 2.0 ** (i / 16 - 10)
                elif scales == "apart":
                    s[at] *= 2.0 ** ((i * 37 % 14) - 7)
                elif i < 40:
                    s[at] = 0.0
        tops = [max(float(s[p].amax()) for p in table) for table in case.tables]
        more = max(t * 2.0 ** -25 * 448 * top for t, top in zip(case.lens, tops))
    kv, batch = case.device()
    print(f"fp8 with fp16 queries dim={dim} heads={heads} rows={rows} {scales}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=rows, want_lse=True)
    _check_rows(case, out, lse, case.expected(), weight_eps=EPS[FP16], more=more)


@pytest.mark.parametrize("block", [1, 3, 8, 16, 24, 48, 128, 300])
@pytest.mark.parametrize("types", [dict(), dict(dtype=FP8, row_scales=True)], ids=["bf16", "fp8"])
def test_block_sizes(block, types):
    case = Case([150, 37, 299], block=block, rows=[1, 3, 9], seed=block, **types)
    kv, batch = case.device()
    print(f"block={block} {types}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=9, want_lse=True)
    _check_rows(case, out, lse, case.expected())


def test_long_and_split_sequences():
    """Enough tokens for many splits, few sequences for many; the joined parts are those of one pass."""
    for lens, heads in (([5000], (4, 1)), ([2100, 1, 900], (8, 2))):
        case = Case(lens, q_heads=heads[0], kv_heads=heads[1], dim=64, seed=len(lens), q_scale=3.0)
        kv, batch = case.device()
        before = _weights(case)
        weights = before.to(DEV)
        print(f"long {lens}", flush=True)
        out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, want_lse=True)
        want = case.expected()
        _check_rows(case, out, lse, want)
        _check_weights(case, weights, before, want, "add")


@pytest.mark.parametrize("dim,rows,types", [
    (64, 1, dict()), (64, 3, dict(dtype=FP8, row_scales=True)), (128, 1, dict(dtype=FP16)), (128, 4, dict()),
    (128, 2, dict(dtype=FP8, query=FP16, row_scales=True)), (256, 1, dict(dtype=FP8)), (256, 2, dict()),
])
def test_many_tokens_and_heads(dim, rows, types):
    """So many that a wave has a KV head to itself: empty sequences, short ones and those of several splits, some pages bad."""
    lens = [9000, 1, 0, 700, 33, 12500, 4, 2048, 9985, 31]
    case = Case(lens, q_heads=32, kv_heads=16, dim=dim, rows=[min(rows, t) for t in lens], seed=dim + rows, **types)
    case.tables[0][100], case.tables[0][101], case.tables[3][-1] = -1, case.pool, 1 << 30
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"many dim={dim} rows={rows} {types}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=rows,
                                weights=weights, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, "add")


def test_blocks_of_many_heads():
    """Lists of blocks long enough that a wave has a KV head, and so a list, to itself: all blocks chosen is all of the cache."""
    case = Case([600 - 7 * i for i in range(56)], q_heads=32, kv_heads=32, dim=64, block=32, seed=5)
    kv, batch = case.device()
    bounds = ops.update_block_bounds(kv, batch, ops.block_bounds(kv))
    print("blocks of many heads", flush=True)
    q = case.q.to(DEV)
    out, lse, blocks = ops.attend_blocks(kv, batch, q, bounds, top_blocks=19, want_lse=True)
    _check_rows(case, out, lse, case.expected())
    assert blocks[0].tolist() == [list(range(19))] * 32
    # ten of them: the same blocks in a call of its own for each sequence, which shares the heads' tokens among waves
    out, lse, blocks = ops.attend_blocks(kv, batch, q, bounds, top_blocks=10, want_lse=True)
    for b in (0, 20, 55):
        one = ops.StepBatch(torch.device(DEV), [case.lens[b]], block_tables=torch.tensor([case.tables[b]], dtype=torch.int32, device=DEV))
        alone, lse1, blocks1 = ops.attend_blocks(kv, one, q[b:b + 1], bounds, top_blocks=10, want_lse=True)
        assert torch.equal(blocks1[0], blocks[b])
        assert float((lse1[0] - lse[b]).abs().max()) < 1e-4
        assert float((alone[0].float() - out[b].float()).abs().max()) <= 2.0 ** -6 * float(alone.float().abs().max())


# ----------------------------------------------------------------------------------- trees
@pytest.mark.parametrize("dim,heads,rows,types", [
    (128, (8, 2), [4, 1, 0, 7], dict()), (128, (8, 2), [16, 3, 20, 5], dict()), (128, (8, 1), [16, 9, 1, 0], dict()),
    (128, (16, 2), [40, 64, 5, 1], dict()), (64, (8, 1), [64, 33, 2, 64], dict(dtype=FP16)),
    (256, (8, 2), [30, 2, 61, 8], dict()), (128, (8, 2), [33, 2, 9, 64], dict(dtype=FP8, row_scales=True)),
    (64, (16, 1), [64, 1, 17, 30], dict(dtype=FP8, query=FP16)), (256, (4, 2), [3, 30, 0, 1], dict(dtype=FP8, row_scales=True)),
    (64, (2, 2), [2, 8, 16, 17], dict()),
])
def test_trees(dim, heads, rows, types):
    lens = [90, 64, 31, 400]
    case = Case(lens, q_heads=heads[0], kv_heads=heads[1], dim=dim, rows=rows, seed=dim + rows[0], **types)
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"tree dim={dim} heads={heads} rows={rows} {types}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=max(rows),
                                weights=weights, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, "add")


@pytest.mark.parametrize("dim,heads,rows,block,types", [
    (128, (32, 2), [5, 0, 64, 9], 24, dict()), (64, (24, 8), [40, 64, 0, 1], 3, dict(dtype=FP16)),
    (256, (9, 1), [8, 3, 30, 0], 16, dict(dtype=FP8, row_scales=True)), (128, (33, 1), [1, 1, 1, 1], 64, dict(dtype=FP8, query=FP16)),
    (256, (6, 3), [64, 2, 50, 7], 20, dict(dtype=FP16)),
])
@pytest.mark.parametrize("mode", ["add", "set"])
def test_weights_of_many_rows(dim, heads, rows, block, types, mode):
    """More rows of a KV head than leave their scores behind: short sequences, fewer tokens than rows, none, bad pages, blocks of
    any size."""
    lens = [290, 50, 71, 3]
    case = Case(lens, q_heads=heads[0], kv_heads=heads[1], dim=dim, rows=rows, block=block, seed=dim + rows[0], **types)
    case.tables[0][1], case.tables[1][-1] = case.pool, -3
    kv, batch = case.device(host_lens=[300] * 4) if block == 20 else case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"weights of many rows dim={dim} heads={heads} rows={rows} block={block} {types} {mode}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=max(rows),
                                weights=weights, weight_mode=mode, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, mode)


def test_trees_without_parents_are_chains_and_may_fill_the_cache():
    """parents=None: each row follows the one before it.  Sequences that hold nothing but their new tokens."""
    case = Case([12, 64, 3, 200], rows=[12, 64, 3, 33], parents="chain", seed=5)
    kv, batch = case.device()
    print("chains", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, max_rows=64, want_lse=True)
    _check_rows(case, out, lse, case.expected())


@pytest.mark.parametrize("heads", [(4, 2), (32, 2)])
@pytest.mark.parametrize("types", [dict(), dict(dtype=FP16), dict(dtype=FP8, row_scales=True)], ids=["bf16", "fp16", "fp8"])
def test_odd_numbers_reach_only_the_rows_that_see_them(heads, types):
    """An infinity and a NaN among the keys and values of drafted tokens: rows of other branches are as if the token were not
    there; rows that see it get what the definition gives."""
    case = Case([50, 140], q_heads=heads[0], kv_heads=heads[1], rows=[6, 9], seed=11, **types)
    case.parents = [-1, 0, 0, 1, 2, -1] + [-1, -1, 0, 1, 2, 3, 4, 1, 7]
    fp8 = types.get("dtype") == FP8

    def spoil(side, b, i, d, value):
        t = case.lens[b] - case.rows[b] + i
        row = case.cache[side][0][case.tables[b][t // case.block], t % case.block, 0]
        if fp8:
            row.view(torch.uint8)[d] = 0x7f            # (e4m3 has no infinity)
        else:
            row[d] = value

    spoil(1, 0, 1, 3, math.inf)
    spoil(1, 0, 2, 7, math.nan)
    spoil(1, 1, 3, 0, -math.inf)
    spoil(0, 1, 6, 5, math.nan)
    kv, batch = case.device()
    print(f"odd numbers heads={heads} {types}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=9, want_lse=True)
    out, lse = out.cpu(), lse.cpu()
    g = heads[0] // heads[1]
    clean = 0
    for b, (o, z, *_) in enumerate(case.expected()):
        part = slice(case.starts[b], case.starts[b + 1])
        assert torch.equal(torch.isnan(lse[part]), torch.isnan(z))
        assert torch.equal(torch.isnan(out[part].double()), torch.isnan(o))
        odd = torch.isinf(o)
        assert torch.equal(out[part].double()[odd], o[odd])
        fine = torch.isfinite(o)
        assert float((out[part].double() - o)[fine].abs().max()) < 0.1
        clean += int(fine[:, :g].all(-1).sum())
    assert clean > 0


@pytest.mark.parametrize("heads,block", [((4, 2), 16), ((24, 2), 16), ((4, 2), 24), ((80, 2), 8), ((32, 16), 16)])
@pytest.mark.parametrize("query", [BF16, FP16])
def test_scales_that_are_no_numbers(heads, block, query):
    """NaN in the scales of slots that no sequence owns (behind the ends, in bad pages' place, in blocks not used): nothing of it
    is seen.  In a drafted token's: the rows that see it get NaN, others what they had."""
    case = Case([50, 140, 33], q_heads=heads[0], kv_heads=heads[1], rows=[6, 9, 1], block=block, seed=41, dtype=FP8, query=query, row_scales=True)
    case.parents = [-1, 0, 0, 1, 2, -1] + [-1, -1, 0, 1, 2, 3, 4, 1, 7] + [-1]
    used = torch.zeros(case.pool, block, dtype=torch.bool)
    for table, t in zip(case.tables, case.lens):
        for i in range(t):
            used[table[i // block], i % block] = True
    for side in (0, 1):
        case.scales[side][0][~used] = math.nan

    def run():
        kv, batch = case.device()
        out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=9, want_lse=True)
        return out, lse

    print(f"scales that are no numbers {heads} {block} {query}", flush=True)
    _check_rows(case, *run(), case.expected())
    t = 140 - 9 + 3                                     # the second sequence's fourth draft: seen by itself, 5 and nobody else
    case.scales[1][0][case.tables[1][t // block], t % block, 0] = math.nan
    out, lse = run()
    _check_rows(case, out, lse, case.expected())
    g = heads[0] // heads[1]
    odd = torch.isnan(out[6:15, :g].cpu()).all(-1).all(-1)
    assert odd.tolist() == [False, False, False, True, False, True, False, False, False]


@pytest.mark.parametrize("heads", [(4, 2), (20, 1)])
def test_bad_pages_hold_no_tokens(heads):
    """Table entries outside the pool, first, last and in the middle: their tokens are seen by nobody and keep no weight."""
    case = Case([100, 47, 16], q_heads=heads[0], kv_heads=heads[1], seed=8)
    case.tables[0][2], case.tables[0][0] = -1, case.pool
    case.tables[1][2] = 1 << 30
    case.tables[2][0] = -(1 << 31)
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"bad pages heads={heads}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, "add")


def test_rows_behind_the_last_sequence_stay_and_parents_out_of_range_are_roots():
    case = Case([40, 90], rows=[3, 5], seed=2)
    kv, batch = case.device()
    q = torch.cat([case.q, torch.full((4, case.hq, case.d), math.nan, dtype=BF16)]).to(DEV)
    parents = torch.cat([case.dev_parents, torch.tensor([900, -5, 7, 1], dtype=torch.int32, device=DEV)])
    out = torch.full_like(q, 7.0)
    for i in (1, 5):                                  # self and later tokens are no parents
        parents[i] = i - case.starts[1 if i >= 3 else 0] + (i == 5)
        case.parents[i] = -1
    print("rows behind", flush=True)
    got, lse = ops.attend_paged(kv, batch, q, row_starts=case.dev_starts, parents=parents, max_rows=5, out=out, want_lse=True)
    assert got is out and bool((out[8:] == 7.0).all())
    _check_rows(case, out[:8], lse[:8], case.expected())


@pytest.mark.parametrize("dim,types", [(128, dict()), (64, dict(dtype=FP8, row_scales=True))])
def test_strides_scales_and_layers(dim, types):
    """q and out as parts of wider tensors, heads before rows; the second of three layers; k_scale and v_scale."""
    case = Case([33, 170, 9], dim=dim, layers=3, seed=6, **types)
    kv, batch = case.device()
    wide = torch.full((case.hq, 3, dim + 32), 9.0, dtype=case.query, device=DEV)
    q = wide[:, :, 8:8 + dim].transpose(0, 1)
    q.copy_(case.q)
    room = torch.full((3, 2 * case.hq, dim), 5.0, dtype=case.query, device=DEV)
    out = room[:, case.hq:, :]
    before = _weights(case)
    weights = before.to(DEV)
    print(f"strides dim={dim} {types}", flush=True)
    _, lse = ops.attend_paged(kv, batch, q, layer=1, scale=0.11 / 0.5, k_scale=0.5, v_scale=3.0, out=out, weights=weights, want_lse=True)
    case.scale = 0.11
    want = case.expected(layer=1)
    _check_rows(case, out, lse, [(o, *rest) for o, *rest in want], scale_v=3.0)
    _check_weights(case, weights, before, want, "add", layer=1)
    assert bool((room[:, :case.hq] == 5.0).all())
    assert torch.equal(weights[[0, 2]].cpu(), before[[0, 2]])


def test_dense_cache_without_a_table():
    g = torch.Generator().manual_seed(9)
    k = torch.randn(2, 77, 2, 64, generator=g).to(BF16)
    v = torch.randn(2, 77, 2, 64, generator=g).to(BF16)
    kv = ops.PagedKV([k.to(DEV)], [v.to(DEV)])
    batch = ops.StepBatch(torch.device(DEV), [77, 40])
    q = torch.randn(2, 8, 64, generator=g).to(BF16)
    print("dense", flush=True)
    out, lse = ops.attend_paged(kv, batch, q.to(DEV), want_lse=True)
    for b, t in enumerate((77, 40)):
        o, z, *_ = oat.attend(q[b:b + 1], k[b, :t].double(), v[b, :t].double(), torch.ones(t, dtype=torch.bool), [-1], 64 ** -0.5)
        assert float((lse[b].cpu().double() - z[0]).abs().max()) < 1e-4
        assert float((out[b].cpu().double() - o[0]).abs().max()) < 2.0 ** -7 * float(v.abs().max())


def test_offsets_beyond_32_bits():
    """Pages at the far end of a pool of more than 2^32 bytes a side."""
    pages = (1 << 32) // (16 * 2 * 128 * 2) + 40
    k = torch.empty(pages, 16, 2, 128, dtype=BF16, device=DEV)
    v = torch.empty(pages, 16, 2, 128, dtype=BF16, device=DEV)
    case = Case([300, 64], seed=4)
    far = {p: pages - 1 - p for p in range(case.pool)}
    for p in range(case.pool):
        k[far[p]], v[far[p]] = case.cache[0][0][p].to(DEV), case.cache[1][0][p].to(DEV)
    kv = ops.PagedKV([k], [v])
    table = torch.zeros(2, case.pitch, dtype=torch.int32)
    for i, t in enumerate(case.tables):
        table[i, :len(t)] = torch.tensor([far[p] for p in t], dtype=torch.int32)
    batch = ops.StepBatch(torch.device(DEV), case.lens, block_tables=table.to(DEV))
    weights = torch.zeros(1, pages, 16, 2, device=DEV)
    print("far pages", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    assert abs(float(weights.double().sum()) - 2 * case.hq) < 1e-3
    bounds = torch.zeros(1, pages, 2, 2, 128, dtype=BF16, device=DEV)
    ops.update_block_bounds(kv, batch, bounds)
    out2, _, blocks = ops.attend_blocks(kv, batch, case.q.to(DEV), bounds, top_blocks=19)
    assert blocks[0, 0].tolist() == list(range(19)) and torch.equal(out2, out)


# ---------------------------------------------------------------------------- chosen blocks
@pytest.mark.parametrize("types", TYPES, ids=["bf16", "fp16", "fp8", "fp8_fp16q_scaled", "fp8_scaled"])
@pytest.mark.parametrize("dim,heads,block", [(128, (8, 2), 16), (64, (28, 4), 32), (256, (4, 4), 16), (64, (6, 1), 8), (128, (9, 1), 1),
                                             (64, (32, 2), 20)])
def test_blocks_are_chosen_and_read_as_defined(dim, heads, block, types):
    group = "max" if heads[0] % 2 == 0 else "mean"
    case = Case([0, 1, 45, 16 * block + 3, 200, 90], q_heads=heads[0], kv_heads=heads[1], dim=dim, block=block, seed=dim + block, **types)
    kv, batch = case.device()
    bounds = ops.block_bounds(kv)
    untouched = bounds.clone()
    print(f"blocks dim={dim} heads={heads} block={block} {types}", flush=True)
    ops.update_block_bounds(kv, batch, bounds)
    want_bounds = untouched.cpu().clone()
    for b, t in enumerate(case.lens):
        if t:
            want_bounds[0, torch.tensor(case.tables[b])] = oat.bounds_of(case.cache[0][0], case.tables[b], t, bounds.dtype, case.scales[0][0])
    assert torch.equal(bounds.cpu().view(torch.int16), want_bounds.view(torch.int16))
    top, sinks, recent = 5, 1, 2
    out, lse, blocks = ops.attend_blocks(kv, batch, case.q.to(DEV), bounds, top_blocks=top, sink_blocks=sinks, recent_blocks=recent,
                                         group_reduce=group, want_lse=True)
    blocks = blocks.cpu()
    g = heads[0] // heads[1]
    want = []
    for b, t in enumerate(case.lens):
        o, z = torch.zeros(1, case.hq, dim, dtype=torch.float64), torch.full((1, case.hq), -math.inf, dtype=torch.float64)
        mean_abs, reach = torch.zeros_like(o), torch.zeros_like(z)
        if t:
            chosen = oat.choose_blocks(case.q[b], want_bounds[0, torch.tensor(case.tables[b])], top, sinks, recent, group == "max")
            k, v, _ = case.sequence(b)
            for h in range(case.h):
                assert blocks[b, h].tolist() == chosen[h] + [-1] * (top - len(chosen[h])), (b, h)
                at = torch.tensor([i for j in chosen[h] for i in range(j * block, min(t, (j + 1) * block))])
                part = slice(h * g, (h + 1) * g)
                o[:, part], z[:, part], _, mean_abs[:, part], reach[:, part] = oat.attend(
                    case.q[b:b + 1, part], k[at, h:h + 1], v[at, h:h + 1], torch.ones(len(at), dtype=torch.bool), [-1], case.scale)
        else:
            assert bool((blocks[b] == -1).all())
        want.append((o, z, None, mean_abs, reach))
    _check_rows(case, out, lse, want)


def test_bounds_follow_new_tokens_and_odd_keys_are_always_read():
    case = Case([40, 33, 16, 130], layers=2, seed=3)
    kv, batch = case.device()
    bounds = ops.block_bounds(kv).fill_(5.0)
    print("bounds of new tokens", flush=True)
    ops.update_block_bounds(kv, batch, bounds, new_tokens=18)
    got = bounds.cpu()
    for layer in range(2):
        fresh = {case.tables[b][j] for b, t in enumerate(case.lens) for j in range(max(t - 18, 0) // 16, -(-t // 16))}
        for b, t in enumerate(case.lens):
            full = oat.bounds_of(case.cache[0][layer], case.tables[b], t, BF16)
            for j, p in enumerate(case.tables[b]):
                want = full[j] if p in fresh else torch.full_like(full[j], 5.0)
                assert torch.equal(got[layer, p], want), (layer, b, j)
    # more new tokens than a sequence has: all of them
    fresh = ops.update_block_bounds(kv, batch, torch.full_like(bounds, 5.0))
    for most in (131, (1 << 31) - 1):
        assert torch.equal(ops.update_block_bounds(kv, batch, torch.full_like(bounds, 5.0), new_tokens=most), fresh)
    # a NaN key: its block counts as the best one
    t = 70
    case.cache[0][0][case.tables[3][t // 16], t % 16, 1, 3] = math.nan
    kv, batch = case.device()
    ops.update_block_bounds(kv, batch, bounds)
    _, _, blocks = ops.attend_blocks(kv, batch, case.q.to(DEV), bounds, top_blocks=2, sink_blocks=0, recent_blocks=1)
    assert blocks[3, 1].tolist() == [t // 16, 8]


def test_equal_blocks_go_to_the_lowest():
    case = Case([16 * 40], seed=1)
    for p in case.tables[0]:
        case.cache[0][0][p] = case.cache[0][0][case.tables[0][0]]
    kv, batch = case.device()
    bounds = ops.update_block_bounds(kv, batch, ops.block_bounds(kv))
    print("ties", flush=True)
    _, _, blocks = ops.attend_blocks(kv, batch, case.q.to(DEV), bounds, top_blocks=7, sink_blocks=0, recent_blocks=2)
    assert blocks[0].tolist() == [[0, 1, 2, 3, 4, 38, 39]] * 2


# --------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("types", [dict(), dict(dtype=FP16, dim=64), dict(dtype=FP8, row_scales=True), dict(dtype=FP8, dim=256)],
                         ids=["bf16", "fp16_d64", "fp8_scaled", "fp8_d256"])
@pytest.mark.parametrize("reduce,shared,prefill", [("mean", False, 0), ("max", False, 9), (None, False, 0), ("mean", True, 9), (None, True, 0)])
@pytest.mark.parametrize("heads", [(8, 4), (6, 3)])
def test_eviction_moves_what_the_weights_keep(types, reduce, shared, prefill, heads):
    lens, budgets, window = [70, 33, 20, 1, 300, 40], [40, 33, 7, 1, 64, 12], 5
    case = Case(lens, q_heads=heads[0], kv_heads=heads[1], layers=3, seed=heads[1], garbage=None, **types)
    kv, batch = case.device(budgets=budgets, prefill=[prefill] * len(lens))
    before = _weights(case)
    before[:, :, 3] = before[:, :, 4]                    # ties
    before = (before * 8).round() / 8
    weights = before.to(DEV)
    ev = ops.EvictConfig(window_size=window, protect_prefill=prefill > 0, layer_reduce=reduce, shared=shared)
    print(f"evict {types} {reduce} shared={shared} heads={heads}", flush=True)
    keep, scores = ops.select_by_weight(kv, batch, weights, ev, want_scores=True)
    again = ops.evict_step(kv, batch, weights, ev)
    assert torch.equal(keep, again)
    keep, scores = keep.cpu(), scores.cpu()
    n_rows = (case.layers if reduce is None else 1) * (1 if shared else case.h)
    k_want, v_want, w_want = [c.clone() for c in case.cache[0]], [c.clone() for c in case.cache[1]], before.clone()
    ks_want = [s.clone() for s in case.scales[0]] if case.scales[0][0] is not None else None
    vs_want = [s.clone() for s in case.scales[1]] if ks_want else None
    raw = lambda c: c.view(torch.uint8) if c.dtype == FP8 else c.view(torch.int16)           # noqa: E731
    for b, t in enumerate(lens):
        slots = [(case.tables[b][i // 16], i % 16) for i in range(t)]
        w = torch.stack([before[:, p, o] for p, o in slots], 1)                          # [L, T, H]
        want = oat.weight_scores(w, reduce, shared, window, prefill)
        rows = slice(b * n_rows, (b + 1) * n_rows)
        assert torch.equal(scores[rows, :t], want) and bool((scores[rows, t:] == -math.inf).all())
        kept = oat.keep_rows(want, budgets[b])
        for r, row in enumerate(kept):
            assert keep[b * n_rows + r].tolist() == row + [-1] * (max(budgets) - budgets[b]), (b, r)
        for layer in range(case.layers):
            for h in range(case.h):
                row = kept[(layer * (1 if shared else case.h) if reduce is None else 0) + (0 if shared else h)]
                for j, i in enumerate(row):
                    (p, o), (sp, so) = slots[j], slots[i]
                    raw(k_want[layer])[p, o, h] = raw(case.cache[0][layer])[sp, so, h]
                    raw(v_want[layer])[p, o, h] = raw(case.cache[1][layer])[sp, so, h]
                    w_want[layer, p, o, h] = before[layer, sp, so, h]
                    if ks_want:
                        ks_want[layer][p, o, h] = case.scales[0][layer][sp, so, h]
                        vs_want[layer][p, o, h] = case.scales[1][layer][sp, so, h]
    assert torch.equal(weights.cpu(), w_want)
    for layer in range(case.layers):
        assert torch.equal(raw(case.k[layer].cpu()), raw(k_want[layer])) and torch.equal(raw(case.v[layer].cpu()), raw(v_want[layer]))
        if ks_want:
            assert torch.equal(case.ks[layer].cpu(), ks_want[layer].reshape(-1)) and torch.equal(case.vs[layer].cpu(), vs_want[layer].reshape(-1))


def test_eviction_of_long_rows_and_odd_weights():
    """Rows longer than a tile of the weights' move; infinite weights keep their tokens."""
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
        assert torch.equal(keep[h].long(), want) and 7 * 16 + 3 in want if h == 2 else True
        assert torch.equal(weights.cpu().view(2, -1, 4)[:, slots[:5000], h], flat[:, keep[h].long(), h])
        assert torch.equal(weights.cpu().view(2, -1, 4)[:, slots[5000:], h], flat[:, 5000:, h])


# -------------------------------------------------------------------- as a program uses them
def _decode_program(kv, batch, q, weights, bounds):
    """One step of each kind on one cache: attention with weights, bounds of the new token, chosen blocks."""
    out, lse = ops.attend_paged(kv, batch, q, weights=weights, want_lse=True)
    ops.update_block_bounds(kv, batch, bounds, new_tokens=1)
    sparse, _, blocks = ops.attend_blocks(kv, batch, q, bounds, top_blocks=4)
    return out, lse, sparse, blocks


def test_a_request_through_prompt_decoding_eviction_and_drafts():
    """All of it in the order of a program: the last tokens of a prompt weigh it, decoding steps add, the cache is evicted by
    what they added, goes on with chosen blocks and a tree of drafts; every call against the definition on the cache as
    it then is."""
    g = torch.Generator().manual_seed(77)
    case = Case([120, 75], q_heads=8, kv_heads=2, dim=64, seed=21, garbage=None, pool=40, rows=[8, 8], parents="chain")
    for t in case.tables:
        t.extend([p for p in range(40) if all(p not in x for x in case.tables)][:3])
    case.pitch = max(len(t) for t in case.tables)
    kv, _ = case.device()
    weights = torch.full((1, 40, 16, 2), math.nan, device=DEV)
    bounds = ops.block_bounds(kv)

    def batch_of(**kw):
        return ops.StepBatch(torch.device(DEV), case.lens, block_tables=case.tables, **kw)

    def sync_cpu():
        case.cache = ([case.k[0].cpu()], [case.v[0].cpu()])

    print("program: prompt", flush=True)
    out, lse = ops.attend_paged(kv, batch_of(), case.q.to(DEV), row_starts=case.dev_starts, max_rows=8, weights=weights, weight_mode="set",
                                want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    before = torch.zeros(1, 40, 16, 2)
    held = weights.cpu().nan_to_num(nan=0.0)
    _check_weights(case, held, before, want, "set")
    case.rows, case.starts, case.parents = [1, 1], [0, 1, 2], [-1, -1]
    for step in range(3):
        case.lens = [t + 1 for t in case.lens]
        for b, t in enumerate(case.lens):
            at = case.tables[b][(t - 1) // 16], (t - 1) % 16
            case.k[0][at] = torch.randn(2, 64, generator=g).to(BF16).to(DEV)
            case.v[0][at] = torch.randn(2, 64, generator=g).to(BF16).to(DEV)
        sync_cpu()
        case.q = torch.randn(2, 8, 64, generator=g).to(BF16)
        before = weights.cpu().clone()
        print(f"program: step {step}", flush=True)
        out, lse = ops.attend_paged(kv, batch_of(), case.q.to(DEV), weights=weights, want_lse=True)
        want = case.expected()
        _check_rows(case, out, lse, want)
        live = weights.cpu().nan_to_num(nan=0.0)
        _check_weights(case, live, before.nan_to_num(nan=0.0), want, "add")
    print("program: eviction", flush=True)
    w_before, k_before = weights.cpu().clone(), case.k[0].cpu().clone()
    keep = ops.evict_step(kv, batch_of(budgets=[64, 50]), weights, ops.EvictConfig(window_size=8)).cpu()
    for b, n in enumerate((64, 50)):
        slots = [(p // 16, p % 16) for p in range(case.lens[b])]
        w = torch.stack([w_before[:, case.tables[b][i], o] for i, o in slots], 1)
        kept = oat.keep_rows(oat.weight_scores(w, "mean", False, 8, 0), n)
        for h in range(2):
            assert keep[b * 2 + h, :n].tolist() == kept[h]
            for j, i in enumerate(kept[h]):
                src, dst = (case.tables[b][i // 16], i % 16, h), (case.tables[b][j // 16], j % 16, h)
                assert torch.equal(case.k[0][dst].cpu(), k_before[src]) and float(weights[0][dst]) == float(w_before[0][src])
    case.lens = [64, 50]
    sync_cpu()
    print("program: chosen blocks", flush=True)
    ops.update_block_bounds(kv, batch_of(), bounds)
    out, lse, blocks = ops.attend_blocks(kv, batch_of(), case.q.to(DEV), bounds, top_blocks=4, want_lse=True)
    want = case.expected()
    assert blocks[:, 0].tolist() == [[0, 1, 2, 3], [0, 1, 2, 3]]           # four blocks are all there are
    _check_rows(case, out, lse, want)
    print("program: drafts", flush=True)
    case.rows, case.starts, case.parents = [5, 4], [0, 5, 9], [-1, 0, 0, 1, 2, -1, -1, 0, 1]
    case.lens = [69, 54]
    case.q = torch.randn(9, 8, 64, generator=g).to(BF16)
    case.dev_starts = torch.tensor(case.starts, dtype=torch.int32, device=DEV)
    case.dev_parents = torch.tensor(case.parents, dtype=torch.int32, device=DEV)
    out, lse = ops.attend_paged(kv, batch_of(), case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=5, want_lse=True)
    _check_rows(case, out, lse, case.expected())


def test_captured_steps_replay_with_new_lengths_and_share_nothing():
    """Two programs captured on one stream each, replayed in turn with eager work between: lengths, queries and weights change
    in place, every replay equals the eager call on the same values."""
    cases = [Case([200, 37], seed=1), Case([64, 333], seed=2, rows=[1, 1])]
    graphs = []
    for i, case in enumerate(cases):
        kv, batch = case.device()
        q, weights, bounds = case.q.to(DEV), _weights(case).to(DEV), ops.block_bounds(kv)
        ops.update_block_bounds(kv, batch, bounds)
        _decode_program(kv, batch, q, weights.clone(), bounds)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _decode_program(kv, batch, q, weights.clone(), bounds)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _decode_program(kv, batch, q, weights, bounds)
        graphs.append((graph, got, kv, batch, q, weights, bounds))
    for rep in range(4):
        for i, (graph, got, kv, batch, q, weights, bounds) in enumerate(graphs):
            case = cases[i]
            lens = [max(0, t - rep * (3 + 40 * i)) for t in case.lens]
            batch.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            q.copy_(torch.randn(q.shape, device=DEV))
            weights.copy_(_weights(case, seed=rep).to(DEV))
            saved_w, saved_b = weights.clone(), bounds.clone()
            print(f"replay {rep} of graph {i} lens {lens}", flush=True)
            graph.replay()
            torch.cuda.synchronize()
            kept = [x.clone() for x in got]
            w_after, b_after = weights.clone(), bounds.clone()
            weights.copy_(saved_w)
            bounds.copy_(saved_b)
            eager = _decode_program(kv, batch, q, weights, bounds)
            torch.cuda.synchronize()
            for x, y in zip(kept, eager):
                assert torch.equal(x, y), (rep, i)
            assert torch.equal(w_after, weights) and torch.equal(b_after, bounds)


@pytest.mark.parametrize("types", [dict(), dict(dtype=FP8, row_scales=True)], ids=["bf16", "fp8"])
def test_captured_eviction_replays_with_new_weights_and_lengths(types):
    """evict_step in a graph: every replay, on other weights and lengths, is the eager call on the same cache."""
    case = Case([300, 90, 45], layers=2, seed=9, garbage=None, **types)
    kv, batch = case.device(budgets=[64, 40, 45])
    ev = ops.EvictConfig(window_size=16)
    state = [*case.k, *case.v, *(case.ks or []), *(case.vs or [])]
    fresh = [x.clone() for x in state]
    weights = _weights(case).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.evict_step(kv, batch, weights, ev)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = ops.evict_step(kv, batch, weights, ev)
    raw = lambda x: x.view(torch.uint8) if x.dtype == FP8 else x           # noqa: E731
    for rep, lens in enumerate(([300, 90, 45], [70, 90, 44], [1, 50, 0], [299, 40, 45])):
        print(f"eviction replay {rep} {lens}", flush=True)
        new = _weights(case, seed=20 + rep).to(DEV)
        batch.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))

        def restore():
            for x, y in zip(state, fresh):
                raw(x).copy_(raw(y))
            weights.copy_(new)

        restore()
        graph.replay()
        torch.cuda.synchronize()
        got = [raw(x).clone() for x in state] + [weights.clone(), keep.clone()]
        restore()
        eager = ops.evict_step(kv, batch, weights, ev)
        for x, y in zip(got, [raw(x) for x in state] + [weights, eager]):
            assert torch.equal(x, y), rep


def test_another_stream_and_two_calls_at_once():
    """Calls on two streams at the same time give what they give one after the other."""
    case = Case([700, 300, 41], seed=12)
    kv, batch = case.device()
    q = [torch.randn(case.q.shape, device=DEV).to(BF16) for _ in range(2)]
    want = [ops.attend_paged(kv, batch, x, want_lse=True) for x in q]
    bounds = ops.update_block_bounds(kv, batch, ops.block_bounds(kv))
    want_blocks = [ops.attend_blocks(kv, batch, x, bounds, top_blocks=6) for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    print("two streams", flush=True)
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.attend_paged(kv, batch, q[i], want_lse=True), ops.attend_blocks(kv, batch, q[i], bounds, top_blocks=6)))
    torch.cuda.synchronize()
    for i in range(2):
        for (out, lse), (sparse, _, blocks) in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
            assert torch.equal(sparse, want_blocks[i][0]) and torch.equal(blocks, want_blocks[i][2])


def test_lengths_on_the_device_below_and_above_the_host_s():
    """The grid goes by the batch's max_seq_len: shorter lengths written into the device array are read, longer ones count as it."""
    case = Case([20, 90, 0], seed=14)
    kv, batch = case.device(host_lens=[90, 90, 90])
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), want_lse=True)
    _check_rows(case, out, lse, case.expected())
    print("lengths", flush=True)
    batch.seq_lens.copy_(torch.tensor([20, 1 << 30, -5], dtype=torch.int32))
    again, lse2 = ops.attend_paged(kv, batch, case.q.to(DEV), want_lse=True)
    assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("heads", [(4, 2), (40, 2)])
def test_fewer_tokens_than_rows(heads):
    """Lengths on the device below the number of rows: the rows are those of the newest tokens, the first of them have none."""
    case = Case([3, 1, 40, 0], q_heads=heads[0], kv_heads=heads[1], rows=[7, 4, 9, 5], parents="chain", seed=15)
    kv, batch = case.device(host_lens=[48] * 4)
    before = _weights(case)
    weights = before.to(DEV)
    print(f"fewer tokens than rows {heads}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), row_starts=case.dev_starts, parents=case.dev_parents, max_rows=9,
                                weights=weights, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, "add")


@pytest.mark.parametrize("heads", [(6, 3), (16, 4)])
def test_a_long_sequence_among_many_short_ones(heads):
    case = Case([1 + 5 * i % 37 for i in range(150)] + [5003], q_heads=heads[0], kv_heads=heads[1], dim=256, seed=heads[1])
    kv, batch = case.device()
    before = _weights(case)
    weights = before.to(DEV)
    print(f"one long {heads}", flush=True)
    out, lse = ops.attend_paged(kv, batch, case.q.to(DEV), weights=weights, want_lse=True)
    want = case.expected()
    _check_rows(case, out, lse, want)
    _check_weights(case, weights, before, want, "add")


def test_weights_that_are_no_numbers_are_kept_first():
    """NaN weights, more than the budget in one head: the lists stay ascending positions, the rows they name are moved."""
    case = Case([200, 90], seed=3, garbage=None)
    kv, batch = case.device(budgets=[60, 30])
    before = _weights(case)
    odd = [(case.tables[0][t // 16], t % 16) for t in range(0, 200, 2)]
    for p, o in odd:
        before[0, p, o, 1] = math.nan
    before[0, case.tables[1][2], 5, 0] = math.nan
    weights = before.to(DEV)
    print("NaN weights", flush=True)
    keep = ops.evict_step(kv, batch, weights, ops.EvictConfig(window_size=8)).cpu()
    for b, h, t, n in ((0, 0, 200, 60), (0, 1, 200, 60), (1, 0, 90, 30), (1, 1, 90, 30)):
        row = keep[b * 2 + h, :n]
        assert bool((row[1:] > row[:-1]).all()) and int(row[0]) >= 0 and int(row[-1]) < t
        for j, i in enumerate(row.tolist()):
            src, dst = (case.tables[b][i // 16], i % 16, h), (case.tables[b][j // 16], j % 16, h)
            assert torch.equal(case.k[0][dst].cpu(), case.cache[0][0][src])
            assert torch.equal(weights[0][dst].cpu().view(torch.int32), before[0][src].view(torch.int32))
    assert all(i % 2 == 0 for i in keep[1, :60].tolist())
    assert 2 * 16 + 5 in keep[2, :30].tolist()


def test_refusals_of_the_python_layer():
    case = Case([30, 20], layers=2, seed=1)
    kv, batch = case.device(budgets=[10, 10])
    q = case.q.to(DEV)
    weights = torch.zeros(2, case.pool, 16, 2, device=DEV)
    bounds = ops.block_bounds(kv)
    ev = ops.EvictConfig()

    def refused(kind, call, *args, **kw):
        with pytest.raises(kind):
            call(*args, **kw)

    refused(ValueError, ops.attend_paged, kv, batch, q.cpu())
    refused(ValueError, ops.attend_paged, kv, batch, q[0])
    refused(ValueError, ops.attend_paged, kv, batch, q.float())
    refused(ValueError, ops.attend_paged, kv, batch, q[..., :64])
    refused(ValueError, ops.attend_paged, kv, batch, q.to(FP16))
    refused(ValueError, ops.attend_paged, kv, batch, q[:1])
    refused(ValueError, ops.attend_paged, kv, batch, q.transpose(1, 2).contiguous().transpose(1, 2))
    refused(IndexError, ops.attend_paged, kv, batch, q, layer=2)
    refused(ValueError, ops.attend_paged, kv, batch, q, weight_mode="sum")
    refused(ValueError, ops.attend_paged, kv, batch, q, weights=weights[:1])
    refused(ValueError, ops.attend_paged, kv, batch, q, weights=weights.double())
    refused(ValueError, ops.attend_paged, kv, batch, q, weights=weights.transpose(1, 2).contiguous().transpose(1, 2))
    refused(ValueError, ops.attend_paged, kv, batch, q, out=q[:1].clone())
    refused(ValueError, ops.attend_paged, kv, batch, q, scale=0.0)
    refused(ValueError, ops.attend_paged, kv, batch, q, max_rows=2)
    refused(ValueError, ops.attend_paged, kv, batch, q, row_starts=case.dev_starts.long())
    refused(ValueError, ops.attend_paged, kv, batch, q, row_starts=case.dev_starts[:2])
    refused(ValueError, ops.attend_paged, kv, batch, q, row_starts=case.dev_starts, parents=case.dev_parents[:1])
    refused(ValueError, ops.attend_paged, kv, batch, q, row_starts=case.dev_starts, max_rows=65)
    refused(ValueError, ops.attend_paged, ops.PagedKV(case.k), batch, q)
    short = ops.StepBatch(torch.device(DEV), [30, 20], block_tables=torch.zeros(2, 1, dtype=torch.int32, device=DEV))
    refused(IndexError, ops.attend_paged, kv, short, q)
    refused(ValueError, ops.attend_paged, kv, ops.StepBatch(torch.device(DEV), [30, 20]), q)
    refused(ValueError, ops.update_block_bounds, kv, batch, bounds[:1])
    refused(ValueError, ops.update_block_bounds, kv, batch, bounds.to(FP16))
    refused(ValueError, ops.update_block_bounds, kv, batch, bounds, new_tokens=0)
    refused(ValueError, ops.attend_blocks, kv, batch, q, bounds, top_blocks=0)
    refused(ValueError, ops.attend_blocks, kv, batch, q, bounds, top_blocks=2, sink_blocks=2)
    refused(ValueError, ops.attend_blocks, kv, batch, q, bounds, top_blocks=2, group_reduce="sum")
    refused(ValueError, ops.select_by_weight, kv, batch, weights[:1], ev)
    refused(ValueError, ops.select_by_weight, kv, batch, weights, ops.EvictConfig(layer_reduce="sum"))
    refused(ValueError, ops.select_by_weight, kv, batch, weights, ops.EvictConfig(protect_prefill=True))
    refused(ValueError, ops.select_by_weight, kv, batch, weights, ev, keep=torch.zeros(3, dtype=torch.int32, device=DEV))
    refused(ValueError, ops.select_by_weight, kv, case.device()[1], weights, ev)
    refused(ValueError, ops.evict_step, ops.PagedKV(case.k), batch, weights, ev)
    half = Case([30], dtype=FP8, row_scales=True, seed=1)
    half.device()
    refused(ValueError, ops.attend_paged, ops.PagedKV(half.k, half.v, "half", half.ks), half.device()[1], half.q.to(DEV))
    # a call that was refused has launched nothing
    torch.cuda.synchronize()
    assert float(weights.abs().max()) == 0.0
