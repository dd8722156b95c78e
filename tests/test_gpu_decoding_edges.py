"""Writing and reading the paged cache, verification of drafts and the move of accepted rows on an MI355X: the calls at the edge of what
the entry points allow, against the definitions in 64 bits (oracle/decoding.py) or, where the header states each step of the
arithmetic, against those steps bit for bit.  Cases and tolerances are those of test_gpu_decoding.py.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import decoding as odec
from test_gpu_decoding import BF16, DEV, FP8, FP16, FP32, Drafts, Step, _bits, _check_written
from triattention_amd import ops

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------- codes
def _codes(x: torch.Tensor, unit) -> torch.Tensor:
    """e4m3 codes as the header states them: the 32-bit quotient, rounded to nearest, beyond 448 the largest."""
    return (x.float() / unit).clamp(-448, 448).to(FP8).view(torch.uint8)


def _still(s: Step):
    """Positions of zero: keys go into the cache as they come."""
    s.positions = torch.zeros_like(s.positions)
    return s


def _slots(s: Step, cache):
    where = odec.places(s.lens, s.starts, s.num_rows, s.tables, s.block, s.pool)
    return torch.stack([cache.cpu().view(s.pool, s.block, s.h, -1)[page, off] for _, page, off in where])


@pytest.mark.parametrize("query", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_codes_of_rows_are_those_of_their_quotients(query, dim):
    """Rows whose largest number is an odd multiple of a power of two and that hold 3/64 of it, 21 of their scales: a tie of two codes, but
    for the rounding of the scale.  Behind them rows of ordinary numbers, 2^19 in all."""
    rows = 2 ** 18 // (8 * dim)
    s = _still(Step([rows + 9], rows=[rows], q_heads=8, kv_heads=8, dim=dim, dtype=FP8, query=query, row_scales=True, seed=dim))
    for i in range(128):
        s.qkv[i // 8, 8 + i % 8, 5], s.qkv[i // 8, 16 + i % 8, 9] = 64.0 + i / 2, -64.0 - i / 2
        s.qkv[i // 8, 8 + i % 8, 6], s.qkv[i // 8, 16 + i % 8, 60] = 3 * (64 + i / 2) / 64, 3 * (64 + i / 2) / 64
    kv, batch = s.device()
    s.write(kv, batch)
    for cache, scales, x in ((s.dk[0], s.dks[0], s.k), (s.dv[0], s.dvs[0], s.v)):
        unit = (x.float().abs().amax(-1) / 448).clamp(min=2.0 ** -126)
        assert torch.equal(_bits(_slots(s, scales).squeeze(-1)), _bits(unit))
        got, want = _slots(s, cache.view(torch.uint8)), _codes(x, unit.unsqueeze(-1))
        assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("unit", [130 / 19, 156 / 21, 148 / 31 * 2.0 ** -7, 0.02, 1.9 * 2.0 ** -120, 3e38, 2.0 ** -100, 1.3 * 2.0 ** 90])
def test_codes_of_a_tensors_scale_are_those_of_the_quotients(unit):
    """One scale for all: all bf16 numbers whose codes are not 0 or the largest, and some that are."""
    unit = float(torch.tensor(unit, dtype=FP32))
    s = _still(Step([2100], rows=[2048], q_heads=2, kv_heads=2, dim=64, dtype=FP8, seed=3))
    numbers = torch.arange(0, 0x7f80, dtype=torch.int32).to(torch.int16).view(BF16)
    ratio = numbers.double() / unit
    numbers = numbers[(ratio > 2.0 ** -13) & (ratio < 2000)]
    assert numbers.numel() > 1000
    both = torch.cat([numbers, -numbers])
    x = both.repeat(-(-2048 * 2 * 64 // both.numel()))[:2048 * 2 * 64].view(2048, 2, 64)
    s.qkv[:, 2:4], s.qkv[:, 4:6] = x, x.flip(-1)
    kv, batch = s.device()
    s.write(kv, batch, k_scale=unit, v_scale=unit)
    for cache, rows in ((s.dk[0], s.k), (s.dv[0], s.v)):
        got, want = _slots(s, cache.view(torch.uint8)), _codes(rows, unit)
        # (a rotation by nothing makes + 0 of - 0 + 0)
        zero = want & 0x7f == 0
        assert torch.equal(got[~zero], want[~zero]) and bool((got[zero] & 0x7f == 0).all()), int((got != want)[~zero].sum())


@pytest.mark.parametrize("row_scales", [True, False])
def test_values_of_nothing_keep_their_sign_as_codes(row_scales):
    s = _still(Step([20], rows=[8], q_heads=2, kv_heads=2, dim=64, dtype=FP8, row_scales=row_scales, seed=4))
    s.qkv[:, 4:, 0::3], s.qkv[:, 4:, 1::3] = -0.0, 0.0
    s.qkv[0, 4:] = -0.0
    s.qkv[1, 4:, 2::3] = -2.0 ** -30
    kv, batch = s.device()
    s.write(kv, batch, **({} if row_scales else dict(v_scale=0.3)))
    unit = (s.v.float().abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -126) if row_scales else torch.tensor(0.3)
    assert torch.equal(_slots(s, s.dv[0].view(torch.uint8)), _codes(s.v, unit))


# ------------------------------------------------------------------------------------ angles
@pytest.mark.parametrize("far", [1 << 12, 1 << 20, (1 << 31) - 1, 1 << 44])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dim,scale", [(64, 1.0), (128, 1.3), (256, 1.0)])
def test_unit_pairs_are_turned_into_cosines_and_sines_rounded_once(far, half, dim, scale):
    """Pairs (1, 0) and (0, 1): 2^20 and more cosines and sines of the 64-bit angle, in 32 bits and then in fp16.  The kernel's are off by 2^-40 of a
    number of ordinary size before that: 2^20 numbers lie that near the middle between two of 32 bits, where that is one of fp16 too, 2^-9 times."""
    rows, f = 4096 * 128 // dim, dim // 2
    s = Step([rows], rows=[rows], q_heads=2, kv_heads=2, dim=dim, dtype=FP16, half=half, far=far, seed=dim)
    s.qkv[:, :4] = 0.0
    first = torch.zeros(dim, dtype=torch.bool)
    first[:f] = True
    if not half:
        first = torch.arange(dim) % 2 == 0
    s.qkv[:, 0::2, first] = 1.0
    s.qkv[:, 1:4:2, ~first] = 1.0
    kv, batch = s.device()
    out = s.write(kv, batch, rotary_scale=scale).cpu()
    keys = _slots(s, s.dk[0])
    angle = s.positions[0].double()[:, None] * s.inv_freq.double()
    c, n = (torch.tensor(scale, dtype=FP32).double() * x for x in (torch.cos(angle), torch.sin(angle)))
    c, n = c.float().to(FP16), n.float().to(FP16)
    for got in (out, keys):
        for head, (one, two) in enumerate(((c, n), (-n, c))):
            # (by value: the sign of a zero is that of a sum)
            assert torch.equal(got[:, head, first], one), int((got[:, head, first] != one).sum())
            assert torch.equal(got[:, head, ~first], two), int((got[:, head, ~first] != two).sum())


@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("wide", [True, False])
def test_one_axis_of_positions_for_all(rows, wide):
    """Plain text on three axes: one axis expanded, a slice of a longer one, is what three copies of it are."""
    s = Step([40, 7], rows=[rows, rows if rows < 7 else 7], axes=3, norm=BF16, seed=41, wide=wide, far=100000)
    s.positions = s.positions[:1].expand(3, -1).contiguous()
    kv, batch = s.device()
    want = s.write(kv, batch)
    _check_written(s, want)
    k, v = s.dk[0].clone(), s.dv[0].clone()
    line = torch.cat([s.dpos[0], s.dpos[0] + 1])
    s.dpos = line[:s.num_rows].expand(3, -1)
    assert rows == 1 or s.dpos.stride(0) == 0
    s.dk[0].view(torch.int16).zero_(), s.dv[0].view(torch.int16).zero_()
    got = s.write(kv, batch)
    where = odec.places(s.lens, s.starts, s.num_rows, s.tables, s.block, s.pool)
    assert torch.equal(_bits(got), _bits(want))
    for new, old in ((s.dk[0], k), (s.dv[0], v)):
        for _, page, off in where:
            assert torch.equal(_bits(new[page, off]), _bits(old[page, off]))


# -------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("norm", [BF16, FP32])
@pytest.mark.parametrize("dtype,row_scales", [(BF16, False), (FP8, True), (FP8, False)])
def test_rows_whose_squares_are_infinite_are_nothing(half, norm, dtype, row_scales):
    """Squares beyond 32 bits are infinite, and numbers over their root 0, the largest bf16 numbers too (times a norm's 1.9 they pass 32 bits); an
    infinity over it is none, and its pair with it.  A row whose squares 32 bits hold stays what it is."""
    s = Step([20], rows=[6], dtype=dtype, row_scales=row_scales, half=half, norm=norm, seed=31)
    s.norms = [torch.full_like(w, 1.875) for w in s.norms]
    most = float(torch.finfo(BF16).max)
    s.qkv[0, :10, 7] = most                       # a pair's first, then its second, then both, then all
    s.qkv[1, :10, 64 + 7] = -most
    s.qkv[2, :10, 0::2] = most
    s.qkv[3, :10] = most
    s.qkv[4, :10, 9] = math.inf
    s.qkv[5, :10] = s.qkv[5, :10] * 2.0 ** 50
    kv, batch = s.device()
    out = s.write(kv, batch).cpu().double()
    where = odec.places(s.lens, s.starts, s.num_rows, s.tables, s.block, s.pool)
    (wq, off_q), _ = s.expected()
    k = torch.stack([s.dk[0].cpu()[page, off].float().double() for _, page, off in where])
    pair = [9, 9 + 64] if half else [8, 9]
    for got in (out, k):
        assert bool((got[:4] == 0).all())
        assert bool(torch.isnan(got[4][:, pair]).all())
        rest = torch.ones(128, dtype=torch.bool)
        rest[pair] = False
        assert bool((got[4][:, rest] == 0).all()) and bool((got[5] != 0).any())
    assert bool(((out[5] - wq[5]).abs() <= off_q[5] * (1 + 2 ** -8) + 2.0 ** -8 * wq[5].abs() + 2.0 ** -133).all())
    if row_scales:
        scales = _slots(s, s.dks[0]).squeeze(-1)
        assert bool((scales[:5] == 2.0 ** -126).all()) and bool((scales[5] > 2.0 ** -126).all())


# --------------------------------------------------------------------------------- verification
@pytest.mark.parametrize("least", [-895, -899, -901, -906, -910, -950])
@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_verify_pieces_of_weights_that_are_nothing_together_are_something(least, kind):
    """Tokens of 2^least of the largest, 2048 and more of them one behind the other: beyond 2^-900 each is one that a random number of 0 or 1 names, below
    it they are nothing, whatever they are together."""
    vocab, a, b = 3 * 2048 + 100, 4096 - 7, 2048 + 5
    for low in (range(0, 2048), range(4096, vocab)):
        for u in (0.0, 0.5, 1.0):
            d = Drafts([2], vocab, tree=kind == "tree", draft=kind == "draft", seed=1)
            d.target[0] = -math.inf
            d.target[0, low.start:low.stop] = least * math.log(2)
            d.target[0, a], d.target[0, b] = 0.0, -1.0
            d.uniforms[0, 1] = u
            if kind == "draft":        # the draft is sure of a, which is rejected
                d.draft[1] = 0.0
                d.draft[1, a], d.tokens[1], d.uniforms[1, 0] = 1.0, a, 0.999
            there = ([b] if kind == "draft" else [b, a]) + (list(low) if least > -900 else [])
            want = min(there) if u == 0 else max(there) if u == 1 else b if kind == "draft" else a
            if kind == "tree":
                d.tokens[1] = -1       # (no child holds the drawn token)
            rows, counts, following = d.run(max_rows=2)
            assert (rows.tolist(), counts.tolist(), following.tolist()) == ([[0, -1]], [1], [want]), (low, u)


@pytest.mark.parametrize("temperature", [math.inf, 1e38, 1e36, 1e31, 1e30, 1e28, 1e27, 1.0])
@pytest.mark.parametrize("kind", ["tree", "draft"])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_verify_infinities_beside_numbers_that_weigh_something(temperature, kind, dtype):
    """An infinity is the largest finite number: at a temperature high enough the others of its piece and of other pieces weigh as much, or what
    their distance leaves them."""
    d = Drafts([3, 2, 4, 2], 4500, dtype=dtype, tree=kind == "tree", draft=kind == "draft", temperatures=[temperature] * 4, seed=17)
    for r, places in enumerate([[3000], [7, 8, 4400], [0], [2047, 2048], [], [4499], [100], list(range(0, 4500, 9)), [1, 3001], [5], [9]]):
        if dtype is FP32:              # numbers next to the largest, 2^104 of one another
            d.target[r, 20:24] = torch.tensor([0x7f7fffff, 0x7f7ffffe, 0x7f7ffff0, 0x7f7f0000], dtype=torch.int32).view(FP32)
            d.target[r, 3000:3004] = d.target[r, 20:24].clone()
        d.target[r, 50:60], d.target[r, 60:62] = -math.inf, math.nan
        d.target[r, places] = math.inf
    if kind == "draft":
        g = torch.Generator().manual_seed(18)
        d.draft = torch.softmax(0.5 * torch.randn(d.draft.shape, generator=g), -1)
        for r in range(d.draft.shape[0]):
            d.tokens[r] = odec.draw(d.draft[r].double(), float(torch.rand(1, generator=g)))
    else:
        for b, m in enumerate(d.rows):
            for r in range(d.starts[b] + 1, d.starts[b] + m):
                up = d.starts[b] + d.parents[r]
                d.tokens[r] = odec.draw(odec.distribution(d.target[up], temperature, False), float(d.uniforms[up, 1]))
    lengths = d.check(d.run(max_rows=4), 4)
    assert kind == "draft" or max(lengths) > 1


@pytest.mark.parametrize("seqs", [64, 65, 130, 4097, 5000])
@pytest.mark.parametrize("kind", ["tree", "chain", "draft"])
def test_verify_finds_the_sequence_of_a_row(seqs, kind):
    """Uneven and empty sequences with temperatures of their own, greedy ones among them, rows behind the last one and rows beyond
    max_rows: on both sides of 64 sequences, where a row's sequence is found another way, and of 64 x 64."""
    g = torch.Generator().manual_seed(seqs)
    many = seqs > 1000
    rows = torch.randint(0, 3 if many else 6, (seqs,), generator=g).tolist()
    rows[0], rows[1], rows[-1] = 7, 0, 2
    temperatures = [(0.0, 0.4, 1.0, 2.5)[int(torch.randint(0, 4, (1,), generator=g))] for _ in rows]
    d = Drafts(rows, 37, tree=kind == "tree", draft=kind == "draft", temperatures=temperatures, seed=seqs, pad=5)
    for width in ((4,) if many else (3, 4, 7)):
        lengths = d.check(d.run(max_rows=width), width)
        assert max(lengths) > 1 and min(lengths) == 0


@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_verify_many_sequences_of_several_pieces(kind):
    g = torch.Generator().manual_seed(9)
    rows = torch.randint(0, 4, (70,), generator=g).tolist()
    temperatures = [(0.0, 0.3, 1.0, math.inf)[i % 4] for i in range(70)]
    d = Drafts(rows, 4100, tree=kind == "tree", draft=kind == "draft", temperatures=temperatures, seed=10, pad=1)
    d.check(d.run(max_rows=2), 2)


def test_verify_probabilities_of_many_sequences():
    g = torch.Generator().manual_seed(11)
    rows = torch.randint(0, 5, (200,), generator=g).tolist()
    for draft in (False, True):
        d = Drafts(rows, 50, tree=not draft, draft=draft, probs=True, seed=12, pad=2)
        d.check(d.run(max_rows=3), 3)


@pytest.mark.parametrize("dtype,bits", [(FP32, 0x7f800001), (FP32, -0x800001 + 2), (BF16, 0x7f81), (BF16, -127), (FP16, 0x7c01), (FP16, -1023)])
@pytest.mark.parametrize("kind", ["tree", "draft"])
@pytest.mark.parametrize("greedy", [False, True])
def test_verify_signalling_nan_count_as_nothing(dtype, bits, kind, greedy):
    """NaN of either sign whose highest bit of the mantissa is not set, in every piece, and one row of nothing else."""
    d = Drafts([4, 3, 6], 4500, dtype=dtype, tree=kind == "tree", draft=kind == "draft", temperatures=[0.0 if greedy else 0.8] * 3, seed=51)
    raw = d.target.view({4: torch.int32, 2: torch.int16}[d.target.element_size()])
    raw[:, 0::7] = bits
    raw[:, 2047:2050] = bits
    raw[5] = bits
    assert bool(torch.isnan(d.target[5]).all())
    d.check(d.run(max_rows=6), 6)


# --------------------------------------------------------------------------- one step after another
@pytest.mark.parametrize("dtype,row_scales", [(BF16, False), (FP8, True)])
def test_the_next_steps_lengths_stay_on_the_device(dtype, row_scales):
    """A batch made for the longest lengths, its lengths rewritten from what acceptance returns: what batches made anew for every step give, in
    the cache and read back from it."""
    g = torch.Generator().manual_seed(61)
    now, longest, steps = [30, 5, 17], [64, 64, 64], 4
    tables = torch.randperm(3 * 4 + 2, generator=g)[:12].view(3, 4).tolist()
    inv = torch.tensor([1e4 ** (-i / 64) for i in range(64)], dtype=FP32, device=DEV)
    caches = []
    for _ in range(2):
        k, v = (torch.zeros(14, 16, 2, 128, dtype=dtype, device=DEV) for _ in range(2))
        scales = [torch.ones(14 * 16 * 2, device=DEV) for _ in range(2)] if row_scales else [None, None]
        caches.append((k, v, scales, ops.PagedKV([k], [v], "half", *([x] if x is not None else None for x in scales))))
    kept = ops.StepBatch(torch.device(DEV), longest, block_tables=tables)
    lens = torch.tensor(now, dtype=torch.int32, device=DEV)
    for step in range(steps):
        rows = torch.randint(1, 6, (3,), generator=g).tolist()
        starts = torch.tensor([0, rows[0], rows[0] + rows[1], sum(rows)], dtype=torch.int32, device=DEV)
        torch.add(lens, torch.tensor(rows, dtype=torch.int32, device=DEV), out=kept.seq_lens)
        anew = ops.StepBatch(torch.device(DEV), [t + n for t, n in zip(now, rows)], block_tables=tables)
        qkv = torch.randn(sum(rows), 8, 128, generator=g).to(BF16).to(DEV)
        pos = torch.arange(sum(rows), device=DEV)
        counts = [1 + int(torch.randint(0, n, (1,), generator=g)) for n in rows]
        path = torch.full((3, 6), -1, dtype=torch.int32)
        for b, (n, c) in enumerate(zip(rows, counts)):
            path[b, :c] = torch.tensor([0] + sorted((torch.randperm(n - 1, generator=g)[:c - 1] + 1).tolist()))
        outs, new = [], []
        for (_, _, _, kv), batch in zip(caches, (kept, anew)):
            outs.append(ops.write_paged(kv, batch, qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], pos, inv, row_starts=starts))
            new.append(ops.accept_drafts(kv, batch, starts, path.to(DEV), torch.tensor(counts, dtype=torch.int32, device=DEV)))
        assert torch.equal(_bits(outs[0]), _bits(outs[1])) and torch.equal(new[0], new[1])
        lens, now = new[0], [t + c for t, c in zip(now, counts)]
        assert lens.tolist() == now
    for a, b in zip(caches[0][:2], caches[1][:2]):
        assert torch.equal(_bits(a), _bits(b))
    kept.seq_lens.copy_(lens)
    starts = torch.tensor([0, now[0], now[0] + now[1], sum(now)], dtype=torch.int32, device=DEV)
    anew = ops.StepBatch(torch.device(DEV), now, block_tables=tables)
    for x, y in zip(ops.read_paged(caches[0][3], kept, starts, sum(now)), ops.read_paged(caches[1][3], anew, starts, sum(now))):
        assert torch.equal(_bits(x), _bits(y))
