"""Writing and reading the paged cache, verification of drafts and the move of accepted rows on an MI355X, against the definitions in 64 bits
(oracle/decoding.py).

Tolerances, from the arithmetic the header states (eps: half a step of a type, 2^-8 bf16, 2^-11 fp16, 2^-24 fp32, 2^-4 e4m3):
 * the norm's sum of D squares in fp32: (D + 2) * 2^-24 of it, half of that of its root, and a few steps for root and products;
 * cos and sin: 2^-23 absolutely (the angle's 64-bit remainder, the series and its roundings), so a rotated number is off
   by that and a few steps of 2^-24, of the sum of both products' magnitudes: together (D / 2 + 20) * 2^-24 * (|n1| + |n2|) * rotary_scale;
 * one rounding at the end: eps of the value (below a type's smallest normal number half its last step absolutely: fp16 2^-25, e4m3 2^-10);
 * a row's scale: what its largest number is off by / 448, and two steps; codes: the quotient's error, and one rounding.
Whole numbers (accepted rows, counts, tokens) are equal.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import decoding as odec
from triattention_amd import ops, rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
EPS = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}
# Below a type's smallest normal number (2^-126, fp16 2^-14) its steps are 2^-133, 2^-24 and 2^-149: half a step of the rounding, and for a
# product in 32 bits before it half of 2^-149 twice.
TINY = {BF16: 2.0 ** -134 + 2.0 ** -149, FP16: 2.0 ** -25, FP32: 2.0 ** -149}


def _bits(x: torch.Tensor) -> torch.Tensor:
    return x.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()])


class Step:
    """A cache of some sequences and the rows of their last tokens, on the CPU and on the device."""

    def __init__(self, lens, rows=None, q_heads=8, kv_heads=2, dim=128, block=16, dtype=BF16, query=None, row_scales=False, half=True, axes=1,
                 far=0, norm=None, layers=1, seed=0, pad_rows=0, wide=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.block, self.hq, self.h, self.d, self.layers, self.half = list(lens), block, q_heads, kv_heads, dim, layers, half
        self.query = query or (dtype if dtype not in (FP8, torch.uint8) else BF16)
        self.dtype, self.fp8 = dtype, dtype in (FP8, torch.uint8)
        self.rows = rows if rows is not None else [1] * len(self.lens)
        self.starts = [sum(self.rows[:i]) for i in range(len(self.rows) + 1)]
        self.num_rows = self.starts[-1] + pad_rows
        counts = [-(-t // block) for t in lens]
        self.pool = sum(counts) + 3
        order = torch.randperm(self.pool, generator=g).tolist()
        self.tables, at = [], 0
        for n in counts:
            self.tables.append(order[at:at + n])
            at += n
        self.cache = [[torch.randint(0, 127 if self.fp8 else 0x3000, (self.pool, block, kv_heads, dim), generator=g,
                                     dtype=torch.uint8 if self.fp8 else torch.int16).view(FP8 if self.fp8 else dtype)
                       for _ in range(layers)] for _ in range(2)]
        self.scales = ([[torch.rand(self.pool, block, kv_heads, generator=g) + 0.5 for _ in range(layers)] for _ in range(2)]
                       if row_scales else None)
        self.weights = torch.rand(layers, self.pool, block, kv_heads, generator=g)
        n = self.num_rows
        self.qkv = (1.5 * torch.randn(n, q_heads + 2 * kv_heads, dim, generator=g)).to(self.query)
        self.q, self.k, self.v = self.qkv[:, :q_heads], self.qkv[:, q_heads:q_heads + kv_heads], self.qkv[:, q_heads + kv_heads:]
        self.norms = [None, None]
        if norm is not None:
            self.norms = [(1 + 0.4 * torch.randn(dim, generator=g)).to(norm) for _ in range(2)]
        self.inv_freq = rope.default_inv_freq(dim, 1e6)
        self.positions = torch.randint(-far if far else 0, far or 5000, (axes, n), generator=g, dtype=torch.int64)
        self.freq_axes = torch.randint(0, axes, (dim // 2,), generator=g, dtype=torch.int32) if axes > 1 else None
        self.wide = wide

    def put(self, x):
        return None if x is None else x.to(DEV)

    def device(self, lens=None):
        raw = (lambda x: x.view(torch.uint8).to(DEV) if self.dtype == torch.uint8 else x.to(DEV))      # noqa: E731
        self.dk, self.dv = ([raw(x) for x in side] for side in self.cache)
        self.dks, self.dvs = ([[x.reshape(-1).to(DEV) for x in side] for side in self.scales] if self.scales else (None, None))
        kv = ops.PagedKV(self.dk, self.dv, "half" if self.half else "interleaved", self.dks, self.dvs)
        table = torch.full((len(self.lens), max([len(t) for t in self.tables] + [1]) + 1), -7, dtype=torch.int32)
        for i, t in enumerate(self.tables):
            table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        batch = ops.StepBatch(torch.device(DEV), lens or self.lens, block_tables=table.to(DEV))
        if lens:
            batch.seq_lens.copy_(torch.tensor(self.lens, dtype=torch.int32))
        self.dstarts = torch.tensor(self.starts, dtype=torch.int32, device=DEV)
        pos = self.positions.to(torch.int64 if self.wide else torch.int32)
        self.dpos = (pos if pos.shape[0] > 1 else pos[0]).to(DEV)
        self.dqkv = self.qkv.to(DEV)
        self.dq, self.dk_new, self.dv_new = (self.dqkv[:, :self.hq], self.dqkv[:, self.hq:self.hq + self.h], self.dqkv[:, self.hq + self.h:])
        return kv, batch

    def write(self, kv, batch, q=None, k=None, v=None, **kw):
        args = dict(row_starts=self.dstarts, freq_axes=self.put(self.freq_axes), q_norm=self.put(self.norms[0]), k_norm=self.put(self.norms[1]))
        args.update(kw)
        return ops.write_paged(kv, batch, self.dq if q is None else q, self.dk_new if k is None else k, self.dv_new if v is None else v, self.dpos,
                               self.inv_freq.to(DEV), **args)

    def expected(self, eps=1e-6, scale=1.0):
        """Rotated queries and keys in 64 bits and what they may be off by before they are rounded."""
        axes = None if self.freq_axes is None else self.freq_axes.tolist()
        got = []
        for x, w in zip((self.q, self.k), self.norms):
            n = odec.normed(x, w, eps)
            y = odec.rotated(n, self.positions, self.inv_freq, axes, self.half, scale)
            f = self.d // 2
            both = (n[..., :f].abs() + n[..., f:].abs()).repeat(1, 1, 2) if self.half else \
                (n[..., 0::2].abs() + n[..., 1::2].abs()).repeat_interleave(2, -1)
            got.append((y, (self.d / 2 + 20) * 2.0 ** -24 * both * abs(scale)))
        return got


def _near(got, want, off, dtype, what):
    """Within the error before the rounding, and one rounding."""
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), what
    fine = torch.isfinite(want)
    excess = ((got - want).abs() - (off * (1 + 2 ** -8) + EPS[dtype] * want.abs() + TINY[dtype]))[fine]
    assert excess.numel() == 0 or float(excess.max()) <= 0, (what, float(excess.max()))


def _check_written(s: Step, out, out_before=None, k_scale=1.0, v_scale=1.0, eps=1e-6, scale=1.0, layer=0):
    """The queries, and the whole cache: the rows' slots, and everything else as it was."""
    (wq, off_q), (wk, off_k) = s.expected(eps, scale)
    where = odec.places(s.lens, s.starts, s.num_rows, s.tables, s.block, s.pool)
    mine = torch.tensor([w is not None for w in where], dtype=torch.bool)
    _near(out.cpu()[mine], wq[mine], off_q[mine], s.query, "queries")
    if out_before is not None:
        assert torch.equal(_bits(out.cpu()[~mine]), _bits(out_before.cpu()[~mine]))
    rows = [i for i, w in enumerate(where) if w is not None and w[1] >= 0]
    page, off = torch.tensor([where[i][1] for i in rows], dtype=torch.long), torch.tensor([where[i][2] for i in rows], dtype=torch.long)
    rows = torch.tensor(rows, dtype=torch.long)
    touched = torch.zeros(s.pool, s.block, dtype=torch.bool)
    touched[page, off] = True
    sides = ((s.dk, s.dks, wk, off_k, k_scale), (s.dv, s.dvs, s.v.double(), torch.zeros(s.v.shape, dtype=torch.float64), v_scale))
    for side, (cache, scales, want, err, tensor_scale) in enumerate(sides):
        for l in range(s.layers):
            got = cache[l].cpu()
            before = s.cache[side][l].view(got.dtype)
            kept = ~touched if l == layer else torch.ones_like(touched)
            assert torch.equal(_bits(got[kept]), _bits(before[kept])), (side, l)
            if s.scales:
                sc = scales[l].cpu().view(s.pool, s.block, s.h)
                assert torch.equal(_bits(sc[kept]), _bits(s.scales[side][l][kept]))
        got = cache[layer].cpu()
        raw = got.view(torch.uint8)[page, off].view(FP8) if s.fp8 else got[page, off]
        w, e = want[rows], err[rows]
        if not s.fp8:
            if side == 1:
                assert torch.equal(_bits(raw), _bits(s.v[rows]))
            else:
                _near(raw, w, e, s.query, "keys")
            continue
        if s.scales:
            sc = scales[layer].cpu().view(s.pool, s.block, s.h)[page, off].double()
            want_scale = odec.row_scale(w)
            most = torch.where(torch.isfinite(w), e, torch.zeros_like(e)).amax(-1)       # (the scale goes by the finite numbers)
            assert bool(((sc - want_scale).abs() <= most / 448 * (1 + 2 ** -8) + want_scale * 2.0 ** -23).all())
            unit = sc.unsqueeze(-1)
        else:
            unit = torch.tensor(tensor_scale, dtype=torch.float32).double()
        codes = raw.float().double()
        fine = torch.isfinite(w)
        assert torch.equal(torch.isnan(codes), ~fine)
        quotient = (w / unit).clamp(-448, 448)
        tol = e / unit * (1 + 2 ** -8) + quotient.abs() * (2.0 ** -4 + 2.0 ** -22) + 2.0 ** -10
        assert bool(((codes - quotient).abs() <= tol)[fine].all())


# ------------------------------------------------------------------------------------- writing
@pytest.mark.parametrize("dim,q_heads,kv_heads", [(128, 8, 2), (64, 8, 8), (256, 6, 3), (128, 32, 8), (64, 3, 1), (128, 5, 5), (256, 2, 1), (128, 28, 4)])
@pytest.mark.parametrize("dtype,query,row_scales", [(BF16, None, False), (FP16, None, False), (FP8, BF16, True), (FP8, FP16, False),
                                                    (torch.uint8, BF16, False)])
def test_write(dim, q_heads, kv_heads, dtype, query, row_scales):
    s = Step([40, 3, 17, 1, 33], rows=[5, 3, 1, 0, 33], q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=dtype, query=query,
             row_scales=row_scales, norm=FP32, seed=dim + q_heads, layers=2, pad_rows=2)
    kv, batch = s.device()
    before = torch.full((s.num_rows, q_heads, dim), 7.0, dtype=s.query, device=DEV)
    scaled = s.fp8 and not row_scales
    more = dict(k_scale=0.03, v_scale=0.02) if scaled else {}
    out = s.write(kv, batch, layer=1, out=before.clone(), **more)
    _check_written(s, out, before, layer=1, **more)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("norm", [None, BF16, FP32])
@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_write_styles(half, norm, axes, dim):
    s = Step([50, 7], rows=[9, 7], dim=dim, half=half, norm=norm, axes=axes, seed=4, wide=axes == 1)
    out = s.write(*s.device())
    _check_written(s, out)


@pytest.mark.parametrize("far", [1 << 20, (1 << 31) - 1, 1 << 40])
@pytest.mark.parametrize("half", [True, False])
def test_write_far_positions(far, half):
    # (2^-24 of a turn of the fastest frequency at 2^40 is beyond the position's own 53 bits of a product: 2^40 * 1 has none lost)
    s = Step([64, 64], rows=[20, 31], far=far, half=half, seed=5, dtype=FP16)
    out = s.write(*s.device())
    _check_written(s, out)


@pytest.mark.parametrize("block", [1, 8, 16, 24, 64])
def test_write_blocks_and_one_row_a_sequence(block):
    s = Step([block, block + 1, 2 * block, 3 * block - 1, 1], block=block, seed=6, norm=BF16)
    kv, batch = s.device()
    out = s.write(kv, batch, row_starts=None)
    _check_written(s, out)


def test_write_only_one_norm_and_scaled_rotation():
    for which in (0, 1):
        s = Step([20], rows=[6], norm=BF16, seed=7)
        s.norms[which] = None
        out = s.write(*s.device(), eps=1e-2, rotary_scale=1.7)
        _check_written(s, out, eps=1e-2, scale=1.7)


def test_write_in_place_and_from_other_strides():
    s = Step([30, 9], rows=[12, 9], norm=BF16, seed=8)
    kv, batch = s.device()
    q = s.dq
    out = s.write(kv, batch, out=q)
    assert out.data_ptr() == q.data_ptr()
    _check_written(s, out)
    # heads first, rows padded, and a row that serves every row of V
    s = Step([30, 9], rows=[12, 9], norm=BF16, seed=8)
    s.v = s.v[:1].expand(21, -1, -1)
    kv, batch = s.device()
    heads_first = torch.empty(s.hq, 21, s.d + 8, dtype=BF16, device=DEV)[:, :, :s.d].transpose(0, 1)
    heads_first.copy_(s.dq)
    k = torch.empty(21, s.h, 2 * s.d, dtype=BF16, device=DEV)[:, :, :s.d]
    k.copy_(s.dk_new)
    into = torch.empty(s.hq, 21, s.d, dtype=BF16, device=DEV).transpose(0, 1)
    out = s.write(kv, batch, q=heads_first, k=k, v=s.dv_new[:1].expand(21, -1, -1), out=into)
    _check_written(s, out)


def test_write_into_one_tensor_of_keys_and_values():
    """[blocks, 2, ...]: K and V of a block side by side, the pool's strides are not its sizes'."""
    s = Step([40, 21], rows=[11, 4], seed=9, norm=FP32)
    kv, batch = s.device()
    both = torch.stack([s.dk[0], s.dv[0]], 1).contiguous()
    kv = ops.PagedKV.from_kv_caches([both], kv_axis=1)
    out = s.write(kv, batch)
    s.dk, s.dv = [both[:, 0].contiguous()], [both[:, 1].contiguous()]
    _check_written(s, out)


@pytest.mark.parametrize("seqs", [63, 64, 65, 300, 5000])
def test_write_finds_the_sequence_of_a_row(seqs):
    g = torch.Generator().manual_seed(seqs)
    rows = torch.randint(0, 3, (seqs,), generator=g).tolist()
    s = Step([r + i % 3 for i, r in enumerate(rows)], rows=rows, q_heads=2, kv_heads=2, dim=64, block=4, seed=seqs, pad_rows=3)
    kv, batch = s.device(lens=[max(x, 1) for x in s.lens])
    before = torch.zeros(s.num_rows, 2, 64, dtype=BF16, device=DEV)
    out = s.write(kv, batch, out=before.clone())
    _check_written(s, out, before)


def test_rows_before_the_first_sequence():
    """row_starts need not begin at 0: rows before it belong to no sequence, in every call."""
    s = Step([20, 33], rows=[4, 6], norm=FP32, seed=23, pad_rows=5)
    s.starts = [3, 7, 13]
    kv, batch = s.device()
    before = torch.full((s.num_rows, s.hq, s.d), 7.0, dtype=BF16, device=DEV)
    out = s.write(kv, batch, out=before.clone())
    _check_written(s, out, before)
    got = tuple(torch.full((s.num_rows, s.h, s.d), 9.0, dtype=BF16, device=DEV) for _ in range(2))
    ops.read_paged(kv, batch, s.dstarts, s.num_rows, out=got)
    mine = torch.zeros(s.num_rows, dtype=torch.bool)
    mine[3:13] = True
    assert torch.equal(_bits(got[1].cpu()[mine]), _bits(s.v[mine])) and bool((got[1].cpu()[~mine] == 9).all()) and bool((got[0].cpu()[~mine] == 9).all())
    for draft in (False, True):
        d = Drafts([4, 6], 3000, draft=draft, seed=24, pad=5)
        d.starts, d.target, d.uniforms, d.tokens = [3, 7, 13], d.target.roll(3, 0), d.uniforms.roll(3, 0), d.tokens.roll(3, 0)
        d.draft = None if d.draft is None else d.draft.roll(3, 0)
        d.check(d.run(max_rows=8), 8)


def test_write_more_rows_than_tokens_and_pages_outside():
    s = Step([5, 40, 0], rows=[9, 20, 2], seed=10)
    kv, batch = s.device(lens=[5, 40, 1])
    for i, bad in enumerate((-1, s.pool, 1 << 30)):
        s.tables[1][i] = bad
        batch.block_table[1, i] = bad
    out = s.write(kv, batch)
    _check_written(s, out)


@pytest.mark.parametrize("row_scales", [True, False])
def test_write_numbers_that_are_none(row_scales):
    s = Step([30], rows=[8], dtype=FP8, row_scales=row_scales, seed=11)
    s.qkv[0, :, 3] = math.inf                     # rotation makes NaN of an infinity
    s.qkv[1, :, 5] = math.nan
    s.qkv[2] = 0.0
    s.qkv[3] = 1e-30
    s.qkv[4, 8:] = 3e38
    s.qkv[5, :, 0] = -math.inf
    s.positions[0, 5] = 0                         # an angle of zero: inf * 0
    s.qkv[6, :, 100] = 1e30
    s.qkv[7] = s.qkv[7] * 1e-3
    kv, batch = s.device()
    out = s.write(kv, batch, **({} if row_scales else dict(k_scale=0.01, v_scale=0.01)))
    _check_written(s, out, **({} if row_scales else dict(k_scale=0.01, v_scale=0.01)))
    got = (s.dvs[0].view(s.pool, 16, 2) if row_scales else None)
    if row_scales:
        page, off = s.tables[0][(30 - 8 + 2) // 16], (30 - 8 + 2) % 16
        assert bool((got[page, off].cpu() == 2.0 ** -126).all())


def test_write_values_keep_their_bits():
    s = Step([20], rows=[4], seed=12)
    s.qkv[0, 10:, :4] = torch.tensor([0x7f81, 0x7fc1, -128, -1], dtype=torch.int16).view(BF16)
    s.qkv[1, 10:, :2] = torch.tensor([math.inf, -0.0]).to(BF16)
    out = s.write(*s.device())
    _check_written(s, out)


def test_write_behind_2_31_elements():
    """Slots whose place passes 32 bits, in a pool of 4.3 GB a side."""
    h, d, block = 8, 128, 16
    blocks = (1 << 31) // (block * h * d) + 64
    k = torch.zeros(blocks, block, h, d, dtype=BF16, device=DEV)
    v = torch.zeros(blocks, block, h, d, dtype=BF16, device=DEV)
    s = Step([20, 35], rows=[20, 7], q_heads=8, kv_heads=h, dim=d, seed=13)
    old = s.tables
    s.tables = [[blocks - 1, blocks - 3], [blocks - 2, 5, blocks - 60]]
    assert [len(t) for t in old] == [len(t) for t in s.tables]
    s.device()
    kv = ops.PagedKV([k], [v])
    batch = ops.StepBatch(torch.device(DEV), s.lens, block_tables=s.tables)
    s.write(kv, batch)
    (_, _), (wk, off_k) = s.expected()
    for row, (b, page, off) in enumerate(odec.places(s.lens, s.starts, s.num_rows, s.tables, block, blocks)):
        _near(k[page, off].cpu(), wk[row], off_k[row], BF16, row)
        assert torch.equal(_bits(v[page, off].cpu()), _bits(s.v[row]))
    total = int((k != 0).any(-1).any(-1).sum())
    assert total == s.num_rows
    rk, rv = ops.read_paged(kv, batch, s.dstarts, s.num_rows)
    where = odec.places(s.lens, s.starts, s.num_rows, s.tables, block, blocks)
    assert torch.equal(_bits(rk), _bits(torch.stack([k[p, o] for _, p, o in where])))
    assert torch.equal(_bits(rv.cpu()), _bits(s.v[:s.num_rows]))


@pytest.mark.parametrize("rows", [2047, 2049, 9000, 17000])
def test_write_many_rows(rows):
    """Row counts on both sides of where waves share rows and rows are read past the caches, a sample of rows checked."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    hq, h, d, block = 24, 4, 128, 16
    blocks = -(-rows // block)
    k, v = (torch.zeros(blocks, block, h, d, dtype=BF16, device=DEV) for _ in range(2))
    kv = ops.PagedKV([k], [v])
    batch = ops.StepBatch(torch.device(DEV), [rows], block_tables=[list(range(blocks))])
    qkv = torch.randn(rows, hq + 2 * h, d, generator=g, device=DEV).to(BF16)
    q, kn, vn = qkv[:, :hq], qkv[:, hq:hq + h], qkv[:, hq + h:]
    norm = (1 + 0.3 * torch.randn(d, generator=g, device=DEV))
    pos = torch.arange(rows, dtype=torch.int32, device=DEV)
    inv = rope.default_inv_freq(d, 1e6)
    out = ops.write_paged(kv, batch, q, kn, vn, pos, inv.to(DEV), row_starts=torch.tensor([0, rows], dtype=torch.int32, device=DEV), q_norm=norm, k_norm=norm)
    assert torch.equal(_bits(v.view(-1, h, d)[:rows]), _bits(vn))
    pick = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:64]
    at = pick.to(DEV)
    for x, got in ((q[at], out[at]), (kn[at], k.view(-1, h, d)[at])):
        n = odec.normed(x.cpu(), norm.cpu(), 1e-6)
        want = odec.rotated(n, pick[None], inv, None, True)
        both = (n[..., :d // 2].abs() + n[..., d // 2:].abs()).repeat(1, 1, 2)
        _near(got, want, (d / 2 + 20) * 2.0 ** -24 * both, BF16, "sample")


@pytest.mark.parametrize("rows", [8000, 15000])
@pytest.mark.parametrize("dtype,row_scales", [(BF16, False), (FP16, False), (FP8, True), (FP8, False)])
@pytest.mark.parametrize("half,norm", [(True, True), (False, False)])
def test_write_of_many_rows_is_that_of_few(rows, dtype, row_scales, half, norm):
    """74 and 138 MB of rows, read and stored past the caches: the bits of three calls of a third, with the queries in place and beside."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    hq, h, d, block, n = 28, 4, 128, 16, rows // 3
    lens = [n, n, rows - 2 * n]
    query = FP16 if dtype is FP16 else BF16
    tables, at = [], 0
    for x in lens:
        tables.append(list(range(at, at + -(-x // block))))
        at += -(-x // block)
    starts = [0, n, 2 * n, rows]
    qkv = torch.randn(rows, hq + 2 * h, d, generator=g, device=DEV).to(query)
    w = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(query) if norm else None
    pos = torch.arange(rows, device=DEV) + 1000
    inv = rope.default_inv_freq(d, 1e6).to(DEV)
    style = "half" if half else "interleaved"

    def cache():
        k, v = (torch.zeros(at, block, h, d, dtype=torch.uint8 if dtype is FP8 else dtype, device=DEV) for _ in range(2))
        if dtype is FP8:
            k, v = k.view(FP8), v.view(FP8)
        scales = [torch.zeros(at * block * h, device=DEV) for _ in range(2)] if row_scales else None
        return k, v, scales, ops.PagedKV([k], [v], style, [scales[0]] if scales else None, [scales[1]] if scales else None)

    def write(kv, of, a, b, out=None):
        batch = ops.StepBatch(torch.device(DEV), [lens[i] for i in of], block_tables=[tables[i] for i in of])
        dstarts = torch.tensor([starts[i] - a for i in of] + [b - a], dtype=torch.int32, device=DEV)
        x = rest[a:b]
        return ops.write_paged(kv, batch, x[:, :hq], x[:, hq:hq + h], x[:, hq + h:], pos[a:b], inv, row_starts=dstarts, q_norm=w, k_norm=w, out=out)

    rest = qkv
    k1, v1, s1, kv1 = cache()
    parts = torch.cat([write(kv1, [i], starts[i], starts[i + 1]) for i in range(3)])
    for in_place in (False, True):
        rest = qkv.clone()
        k2, v2, s2, kv2 = cache()
        whole = write(kv2, [0, 1, 2], 0, rows, rest[:, :hq] if in_place else None)
        for a, b in [(parts, whole), (k1, k2), (v1, v2)] + (list(zip(s1, s2)) if s1 else []):
            assert torch.equal(_bits(a), _bits(b))


def test_a_step_on_another_stream_than_the_default_one():
    """Behind work of that stream which its inputs come from, without a wait of the host."""
    s = Step([50, 21], rows=[9, 4], dtype=FP8, row_scales=True, norm=BF16, seed=33)
    kv, batch = s.device()
    want = s.write(kv, batch).clone()
    rk, rv = ops.read_paged(kv, batch, s.dstarts, s.num_rows)
    accepted = torch.tensor([[0, 3, 8], [0, 2, -1]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([3, 2], dtype=torch.int32, device=DEV)
    lens = ops.accept_drafts(kv, batch, s.dstarts, accepted, counts)
    after = [x.clone() for x in (s.dk[0], s.dv[0])]
    kv, batch = s.device()
    q = s.dq.clone()
    s.dq.zero_()
    accepted_too = torch.zeros_like(accepted)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        s.dq.copy_(q)
        accepted_too.copy_(accepted)
        out = s.write(kv, batch)
        k2, v2 = ops.read_paged(kv, batch, s.dstarts, s.num_rows)
        lens2 = ops.accept_drafts(kv, batch, s.dstarts, accepted_too, counts)
    torch.cuda.synchronize()
    for a, b in ((want, out), (rk, k2), (rv, v2), (lens, lens2), (after[0], s.dk[0]), (after[1], s.dv[0])):
        assert torch.equal(_bits(a), _bits(b))


def test_without_a_block_table():
    """A dense cache: a sequence is one block of it.  Written, read, and its accepted rows moved."""
    s = Step([40, 33, 12], rows=[40, 5, 12], block=64, layers=2, norm=FP32, seed=22)
    s.tables = [[0], [1], [2]]
    kv, _ = s.device()
    batch = ops.StepBatch(torch.device(DEV), s.lens)
    out = s.write(kv, batch, layer=1)
    _check_written(s, out, layer=1)
    k, v = ops.read_paged(kv, batch, s.dstarts, s.num_rows, layer=1)
    assert torch.equal(_bits(v.cpu()), _bits(s.v))
    for l in range(2):
        for side, cache in ((0, s.dk), (1, s.dv)):
            s.cache[side][l] = cache[l].cpu()
    paths = [[0, 3, 39, -1], [1, 2, 4, -1], [0, 1, 2, 11]]
    counts = [3, 3, 4]
    lens = ops.accept_drafts(kv, batch, s.dstarts, torch.tensor(paths, dtype=torch.int32, device=DEV), torch.tensor(counts, dtype=torch.int32, device=DEV))
    _check_accepted(s, paths, counts, lens.cpu(), None, 4)
    with pytest.raises(ValueError):
        s.write(kv, ops.StepBatch(torch.device(DEV), [65, 33, 12]))


def test_write_refuses_tensors():
    s = Step([20], rows=[4], norm=BF16)
    kv, batch = s.device()
    good = dict(q=s.dq, k=s.dk_new, v=s.dv_new)
    for name, bad in (("q", s.dq.float()), ("q", s.dq[:, :, :64]), ("k", s.dk_new[:3]), ("v", s.dv_new[:, :1]), ("k", s.dk_new.to(FP16)),
                      ("v", s.dv_new.cpu()), ("q", s.dq[0])):
        with pytest.raises(ValueError):
            s.write(kv, batch, **{**good, name: bad})
    for kw in (dict(q_norm=torch.ones(128, device=DEV)), dict(k_norm=torch.ones(64, dtype=BF16, device=DEV)), dict(row_starts=s.dstarts.long()),
               dict(row_starts=s.dstarts[:1]), dict(out=torch.empty(4, 8, 64, dtype=BF16, device=DEV)),
               dict(freq_axes=torch.zeros(63, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            s.write(kv, batch, **kw)
    with pytest.raises(IndexError):
        s.write(kv, batch, layer=1)
    good_pos = s.dpos
    for bad in (s.dpos.float(), s.dpos[:3], s.dpos.expand(2, -1), s.dpos.cpu()):
        s.dpos = bad
        with pytest.raises(ValueError):
            s.write(kv, batch)
    s.dpos = good_pos
    with pytest.raises(Exception, match="k_scale"):
        s.write(kv, batch, k_scale=0.5)
    with pytest.raises(ValueError):
        s.write(ops.PagedKV(s.dk), batch)


def test_write_replayed():
    s = Step([40, 25], rows=[3, 2], norm=BF16, dtype=FP8, row_scales=True, seed=14)
    kv, batch = s.device(lens=[40, 40])
    out = torch.empty(5, s.hq, s.d, dtype=BF16, device=DEV)
    side = torch.cuda.Stream()
    inv, axes, qn, kn = s.inv_freq.to(DEV), None, s.put(s.norms[0]), s.put(s.norms[1])
    call = lambda: ops.write_paged(kv, batch, s.dq, s.dk_new, s.dv_new, s.dpos, inv, row_starts=s.dstarts, q_norm=qn, k_norm=kn, out=out)   # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens, rows, seed in (([40, 25], [3, 2], 1), ([12, 31], [0, 5], 2), ([9, 16], [4, 1], 3)):
        g = torch.Generator().manual_seed(seed)
        s.lens, s.rows, s.starts = lens, rows, [0, rows[0], sum(rows)]
        s.qkv.copy_(torch.randn(s.qkv.shape, generator=g).to(BF16))
        s.positions = torch.randint(0, 100000, (1, 5), generator=g)
        for side_no in (0, 1):
            (s.dk, s.dv)[side_no][0].copy_(s.cache[side_no][0])
            (s.dks, s.dvs)[side_no][0].copy_(s.scales[side_no][0].view(-1))
        s.dqkv.copy_(s.qkv)
        s.dpos.copy_(s.positions[0])
        s.dstarts.copy_(torch.tensor(s.starts, dtype=torch.int32))
        batch.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _check_written(s, out)


# -------------------------------------------------------------------------------------- reading
@pytest.mark.parametrize("dim,kv_heads", [(128, 8), (64, 1), (64, 8), (256, 3), (128, 1), (64, 5), (256, 16)])
@pytest.mark.parametrize("dtype,row_scales", [(BF16, False), (FP16, False), (FP8, True), (FP8, False), (torch.uint8, False)])
@pytest.mark.parametrize("out", [BF16, FP16, FP32])
def test_read(dim, kv_heads, dtype, row_scales, out):
    s = Step([40, 1, 0, 33, 7], rows=[40, 3, 1, 20, 0], q_heads=kv_heads, kv_heads=kv_heads, dim=dim, dtype=dtype, row_scales=row_scales, seed=dim,
             layers=2)
    kv, batch = s.device(lens=[40, 1, 1, 33, 7])
    s.tables[3][1] = s.pool + 2
    batch.block_table[3, 1] = s.pool + 2
    n = s.num_rows + 3
    got = tuple(torch.full((n, kv_heads, dim), 9.0, dtype=out, device=DEV) for _ in range(2))
    back = ops.read_paged(kv, batch, s.dstarts, n, layer=1, k_scale=0.5, v_scale=1.7, out=got)
    assert back[0] is got[0] and back[1] is got[1]
    where = odec.places(s.lens, s.starts, n, s.tables, s.block, s.pool)
    for side, scale in ((0, 0.5), (1, torch.tensor(1.7).item())):
        x = got[side].cpu()
        for row, place in enumerate(where):
            if place is None:
                assert bool((x[row] == 9).all())
            elif place[1] < 0:
                assert bool((x[row] == 0).all())
            else:
                want = s.cache[side][1].view(torch.uint8)[place[1], place[2]].view(FP8).float().double() if s.fp8 else \
                    s.cache[side][1][place[1], place[2]].double()
                if row_scales:
                    want = want * s.scales[side][1][place[1], place[2]].double().unsqueeze(-1)
                # two products of 32 bits, one rounding
                want = want * scale
                if out == FP16:
                    big = want.abs() > 65519.9
                    assert bool(torch.isinf(x[row])[want.abs() > 65520.1].all())
                    want, held = torch.where(big, 0.0, want), torch.where(big, 0.0, x[row].double())
                else:
                    held = x[row].double()
                _near(held, want, want.abs() * 2.0 ** -22, out, (side, row))


def test_read_is_what_was_written():
    for dtype in (BF16, FP16):
        s = Step([100, 61], rows=[100, 17], dtype=dtype, q_heads=4, kv_heads=4, norm=FP32, seed=15)
        kv, batch = s.device()
        s.write(kv, batch)
        k, v = ops.read_paged(kv, batch, s.dstarts, s.num_rows)
        assert k.dtype == dtype and torch.equal(_bits(v.cpu()), _bits(s.v))
        (_, _), (wk, off) = s.expected()
        _near(k, wk, off, dtype, "keys")
    s = Step([100], rows=[100], dtype=FP8, row_scales=True, seed=16)
    kv, batch = s.device()
    s.write(kv, batch)
    _, v = ops.read_paged(kv, batch, s.dstarts, 100, dtype=FP32)
    want = s.v.double()
    unit = odec.row_scale(want).unsqueeze(-1)
    assert bool(((v.cpu().double() - want).abs() <= want.abs() * (2.0 ** -4 + 2.0 ** -21) + unit * 2.0 ** -10).all())
    assert ops.read_paged(kv, batch, s.dstarts, 100)[0].dtype == BF16


@pytest.mark.parametrize("rows", [8191, 8192, 16385, 40000])
def test_read_many_rows(rows):
    for h, d in ((8, 64), (1, 64), (2, 128)):
        k = torch.randn(-(-rows // 16), 16, h, d, device=DEV).to(FP16)
        v = torch.randn(-(-rows // 16), 16, h, d, device=DEV).to(FP16)
        kv = ops.PagedKV([k], [v])
        batch = ops.StepBatch(torch.device(DEV), [rows], block_tables=[list(range(k.shape[0]))])
        starts = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
        rk, rv = ops.read_paged(kv, batch, starts, rows)
        assert torch.equal(_bits(rk), _bits(k.view(-1, h, d)[:rows])) and torch.equal(_bits(rv), _bits(v.view(-1, h, d)[:rows]))
        rk, rv = ops.read_paged(kv, batch, starts, rows, dtype=FP32)
        assert torch.equal(rk, k.view(-1, h, d)[:rows].float()) and torch.equal(rv, v.view(-1, h, d)[:rows].float())


def test_read_refuses():
    s = Step([20], rows=[4])
    kv, batch = s.device()
    with pytest.raises(TypeError):
        ops.read_paged(kv, batch, s.dstarts, 4, dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.read_paged(kv, batch, s.dstarts, -1)
    with pytest.raises(ValueError):
        ops.read_paged(kv, batch, s.dstarts.cpu(), 4)
    with pytest.raises(ValueError):
        ops.read_paged(kv, batch, s.dstarts, 4, out=(torch.empty(4, 2, 128, device=DEV), torch.empty(3, 2, 128, device=DEV)))
    with pytest.raises(IndexError):
        ops.read_paged(kv, batch, s.dstarts, 4, layer=-1)


# ---------------------------------------------------------------------------------- verification
class Drafts:
    """Rows of some sequences with logits, drafted tokens and random numbers, on the CPU."""

    def __init__(self, rows, vocab, dtype=FP32, tree=False, draft=False, temperatures=None, probs=False, seed=0, spread=3.0, pad=0, gap=0, agree=0.6):
        g = torch.Generator().manual_seed(seed)
        self.rows, self.vocab, self.probs = list(rows), vocab, probs
        self.starts = [sum(rows[:i]) for i in range(len(rows) + 1)]
        n = self.starts[-1] + pad
        self.parents = [max(-1, i - 1 - int(torch.randint(0, 3, (1,), generator=g))) if tree and i > 1 else i - 1 for m in rows for i in range(m)]
        self.parents += [0] * pad
        self.tree = tree
        logits = spread * torch.randn(n, vocab + gap, generator=g)
        logits = (torch.softmax(logits, -1) if probs else logits).to(dtype)
        self.target = logits[:, :vocab]
        self.temperatures = temperatures
        self.draft = torch.softmax(self.target.float() * 0.7 + 0.8 * torch.randn(n, vocab, generator=g), -1) if draft else None
        self.uniforms = torch.rand(n, 2, generator=g)
        self.tokens = torch.randint(0, vocab, (n,), generator=g, dtype=torch.int32)
        for b, m in enumerate(rows):
            for i in range(1, m):
                r = self.starts[b] + i
                if draft:
                    self.tokens[r] = odec.draw(self.draft[r].double(), float(torch.rand(1, generator=g)))
                elif float(torch.rand(1, generator=g)) < agree and self.parents[r] >= 0:
                    up = self.starts[b] + self.parents[r]
                    t = 1.0 if temperatures is None else temperatures[b]
                    self.tokens[r] = odec.largest(self.target[up]) if not t > 0 else \
                        odec.draw(odec.distribution(self.target[up], t, probs), float(self.uniforms[up, 1]))

    def run(self, max_rows=None, target=None, draft=None):
        put = lambda x: None if x is None else x.to(DEV)        # noqa: E731
        t = None if self.temperatures is None else torch.tensor(self.temperatures, device=DEV)
        return ops.verify_drafts(put(self.target) if target is None else target, put(self.tokens),
                                 torch.tensor(self.starts, dtype=torch.int32, device=DEV), put(self.uniforms), max_rows=max_rows,
                                 parents=torch.tensor(self.parents, dtype=torch.int32, device=DEV) if self.tree else None,
                                 draft_probs=put(self.draft) if draft is None else draft, temperatures=t, probs=self.probs)

    def check(self, got, max_rows=None):
        rows, counts, following = (x.cpu() for x in got)
        width = max_rows or min(max(self.target.shape[0], 1), 64)
        assert rows.shape == (len(self.rows), width)
        lengths = []
        for b, m in enumerate(self.rows):
            m, at = min(m, width), self.starts[b]
            part = slice(at, at + m)
            path, tok = odec.verify_sequence(self.target[part], self.tokens[part], self.uniforms[part], self.parents[part] if self.tree else None,
                                             1.0 if self.temperatures is None else self.temperatures[b],
                                             None if self.draft is None else self.draft[part], self.probs)
            assert rows[b].tolist() == path + [-1] * (width - len(path)), (b, path, rows[b].tolist())
            assert (int(counts[b]), int(following[b])) == (len(path), tok), (b, path, tok)
            lengths.append(len(path))
        return lengths


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 511, 513, 2047, 2048, 2049, 5003])
@pytest.mark.parametrize("kind", ["tree", "chain", "draft"])
def test_verify_vocabularies(vocab, kind):
    d = Drafts([6, 1, 0, 9, 3, 12], vocab, tree=kind == "tree", draft=kind == "draft", temperatures=[0.7, 1.0, 0.5, 0.0, 2.0, 1.0], seed=vocab)
    lengths = d.check(d.run())
    assert kind == "draft" or vocab < 3 or max(lengths) > 1       # (these drafts have little to do with the target)


@pytest.mark.parametrize("vocab", [300, 2048, 5003, 20001])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_verify_drafts_near_the_target(vocab, dtype):
    """Drafts of a distribution close to the row's before them: several accepted, ends by rejection and by running out."""
    d = Drafts([6, 1, 8, 9, 3, 12, 4, 5], vocab, dtype=dtype, draft=True, temperatures=[0.7, 1.0, 0.5, 0.0, 2.0, 1.0, 0.3, 1.0], seed=vocab)
    g = torch.Generator().manual_seed(vocab + 1)
    for b, m in enumerate(d.rows):
        for r in range(d.starts[b] + 1, d.starts[b] + m):
            t = max(d.temperatures[b], 0.3)
            d.draft[r] = torch.softmax((d.target[r - 1].float() + 0.3 * torch.randn(vocab, generator=g)) / t, -1)
            d.tokens[r] = odec.draw(d.draft[r].double(), float(torch.rand(1, generator=g)))
    lengths = d.check(d.run())
    assert max(lengths) > 3 and any(1 <= n < m for n, m in zip(lengths, d.rows))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("kind", ["tree", "chain", "draft"])
@pytest.mark.parametrize("gap", [0, 5])
def test_verify_types_and_strides(dtype, kind, gap):
    d = Drafts([5, 20, 8, 1], 3001, dtype=dtype, tree=kind == "tree", draft=kind == "draft", seed=3, gap=gap, pad=2)
    wide = torch.zeros(d.target.shape[0], 3001 + gap, dtype=dtype, device=DEV)[:, :3001]
    wide.copy_(d.target)
    q = None
    if d.draft is not None:
        q = torch.zeros(d.target.shape[0], 3001 + 2 * gap, device=DEV)[:, :3001]
        q.copy_(d.draft)
    d.check(d.run(target=wide, draft=q))


@pytest.mark.parametrize("vocab", [131072, 131073, 300007])
@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_verify_large_vocabularies(vocab, kind):
    d = Drafts([4, 3, 6], vocab, dtype=BF16, tree=kind == "tree", draft=kind == "draft", temperatures=[1.0, 0.0, 0.8], seed=5, spread=4.0)
    d.check(d.run())


@pytest.mark.parametrize("draft", [False, True])
def test_verify_probabilities(draft):
    d = Drafts([5, 9, 1, 7], 4100, probs=True, draft=draft, seed=6)
    d.target[3] *= 3.0                                  # (their sum need not be one)
    d.target[6, 100] = math.nan
    d.target[7, 200] = -0.5
    d.target[8, 300] = math.inf
    d.check(d.run())


@pytest.mark.parametrize("kind", ["tree", "chain", "draft"])
def test_verify_sixty_four_rows_and_no_more(kind):
    d = Drafts([64, 70, 2], 600, tree=kind == "tree", draft=kind == "draft", seed=7, agree=0.95)
    lengths = d.check(d.run())
    assert kind == "draft" or max(lengths) > 5
    d.check(d.run(max_rows=64), 64)
    d.check(d.run(max_rows=5), 5)
    d.check(d.run(max_rows=1), 1)


@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_verify_masks_and_odd_numbers(kind):
    """Rows with -inf, NaN, infinities, lowest values of the type, nothing at all; temperatures of every kind."""
    temps = [1.0, 1.0, 1.0, 0.0, 1.0, 1e-30, math.inf, math.nan, -1.0, 1e-3, 0.0, 1.0, 5e-324 * 0 + 1e-38]
    d = Drafts([3] * len(temps), 4500, tree=kind == "tree", draft=kind == "draft", temperatures=temps, seed=8)
    x = d.target
    x[0:3, 10:] = -math.inf                            # a few tokens left
    x[3:6] = -math.inf                                 # nothing left
    x[6:9, ::2] = math.nan
    x[9:12] = -math.inf                                # greedy, nothing left
    x[12, 4000] = x[12, 77] = math.inf                 # two tokens share everything
    x[13, 2000:] = torch.finfo(torch.float32).min
    x[30:33, 4096:] = math.inf                         # greedy, the first of many
    x[33] = torch.finfo(torch.float32).min             # all alike
    d.check(d.run())


def test_verify_infinities_among_the_largest_numbers():
    """+inf counts as the largest finite number, in one piece of a row and across pieces, greedy and drawn."""
    most = torch.finfo(torch.float32).max
    d = Drafts([1] * 8, 9000, temperatures=[0.0, 0.0, 0.0, 0.0, 1.0, 1.0, 1.0, 1.0], seed=21)
    for b in (0, 4):
        d.target[b, [17, 30]] = torch.tensor([most, math.inf])
        d.target[b + 1, [17, 5000]] = torch.tensor([most, math.inf])
        d.target[b + 2, [17, 5000]] = torch.tensor([math.inf, most])
        d.target[b + 3, [4500, 4501, 8999]] = torch.tensor([math.nan, math.inf, math.inf])
    for u in (0.0, 0.49, 0.51, 0.99):
        d.uniforms[:] = u
        got = d.run()
        d.check(got)
        assert got[2].cpu().tolist() == [17, 17, 17, 4501] + ([17, 17, 17, 4501] if u < 0.5 else [30, 5000, 5000, 8999])


def test_verify_uniforms_at_their_ends():
    for kind in ("tree", "draft"):
        values = [0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, math.nan, 2.0 ** -149, 5.0]
        d = Drafts([2] * len(values), 2500, tree=kind == "tree", draft=kind == "draft", seed=9)
        d.target[:, :3] = -math.inf
        d.target[:, 2400:] = -math.inf
        for b, u in enumerate(values):
            d.uniforms[2 * b:2 * b + 2] = u
        d.check(d.run())


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_verify_boundaries_are_exact(dtype):
    """Equal logits, a power of two of them: u = k / V is the boundary in front of token k, which u does not exceed."""
    v = 4096
    rows = 256
    d = Drafts([1] * rows, v, dtype=dtype, seed=10)
    d.target[:] = 3.25
    ks = torch.randint(0, v, (rows,), generator=torch.Generator().manual_seed(2))
    d.uniforms[:, 1] = ks.float() / v
    _, counts, following = d.run()
    assert torch.equal(following.cpu().long(), ks) and bool((counts == 1).all())
    d.uniforms[:, 1] = torch.nextafter(ks.float().clamp(min=1) / v, torch.zeros(1))
    assert torch.equal(d.run()[2].cpu().long(), ks.clamp(min=1) - 1)


def test_verify_ties_tokens_outside_and_siblings():
    # greedy: the first of equal logits, wherever the others are
    d = Drafts([2, 2, 2], 7000, temperatures=[0.0] * 3, seed=11)
    d.target[:] = 0.0
    d.target[0, [5, 2050, 6999]] = 2.0
    d.target[2, [2047, 2048]] = 2.0
    d.target[4, 6999] = 2.0
    d.tokens[1], d.tokens[3], d.tokens[5] = 5, 2048, 6999
    assert d.check(d.run()) == [2, 1, 2]
    # a token outside the vocabulary is never accepted, with and without draft probabilities
    for draft in (False, True):
        d = Drafts([3, 3], 100, draft=draft, seed=12)
        d.tokens[1], d.tokens[4] = -1, 100
        d.check(d.run())
    # siblings with the same token: the first; a parent that is no row of the tree is never reached
    d = Drafts([6, 6], 50, tree=True, temperatures=[0.0, 0.0], seed=13)
    best = [odec.largest(d.target[i]) for i in range(12)]
    d.parents = [-1, 0, 0, 1, 2, 2] + [-1, -1, 7, 3, 9, 0]
    d.tokens = torch.tensor([0, best[0], best[0], best[1], best[2], best[2]] + [0, best[6], best[7], best[9], 1, best[6]], dtype=torch.int32)
    got = d.run()
    d.check(got)
    assert got[0].cpu()[0, :3].tolist() == [0, 1, 3] and int(got[1][1]) == 2


def test_verify_a_draft_that_is_the_target_is_accepted():
    """q = p: every row is accepted, whatever the random numbers below one; and a certain draft leaves what it is not."""
    d = Drafts([12, 12], 5000, draft=True, probs=True, seed=14)
    d.target = d.draft.roll(-1, 0)
    d.uniforms[:, 0] = 0.999
    for b in range(2):
        for i in range(1, 12):
            r = 12 * b + i
            d.draft[r] = d.target[r - 1] / d.target[r - 1].double().sum().float()
            d.tokens[r] = int(torch.randint(0, 5000, (1,), generator=torch.Generator().manual_seed(r)))
    assert d.check(d.run()) == [12, 12]
    d.draft.zero_()
    d.draft[torch.arange(24), d.tokens.long()] = 1.0
    d.uniforms[:, 0] = 0.5
    assert d.check(d.run()) == [1, 1]


def test_verify_keeps_the_targets_distribution():
    """All drafts of a vocabulary of six by a grid of both random numbers, weighted with the draft's probabilities: the token behind the first row
    has the target's distribution, up to the grid."""
    steps, v = 64, 6
    g = torch.Generator().manual_seed(15)
    logits, q = torch.randn(v, generator=g) * 1.3, torch.softmax(torch.randn(v, generator=g), -1)
    grid = (torch.arange(steps) + 0.5) / steps
    seqs = v * steps * steps
    tok = torch.arange(v).repeat_interleave(steps * steps)
    u0, u1 = grid.repeat_interleave(steps).repeat(v), grid.repeat(v * steps)
    tokens = torch.stack([torch.zeros_like(tok), tok], 1).view(-1).int()
    uniforms = torch.zeros(seqs, 2, 2)
    uniforms[:, 1, 0], uniforms[:, 0, 1] = u0, u1
    rows, counts, following = ops.verify_drafts(logits.expand(2 * seqs, -1).contiguous().to(DEV), tokens.to(DEV),
                                                torch.arange(0, 2 * seqs + 1, 2, dtype=torch.int32, device=DEV), uniforms.view(-1, 2).to(DEV), max_rows=2,
                                                draft_probs=q.expand(2 * seqs, -1).contiguous().to(DEV))
    got = torch.zeros(v, dtype=torch.float64)
    first = torch.where(counts.cpu() == 2, tok, following.cpu().long())
    got.index_add_(0, first, q.double()[tok] / steps / steps)
    assert float((got - torch.softmax(logits.double(), -1)).abs().max()) < 2.0 / steps


@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_verify_replayed(kind):
    d = Drafts([5, 3, 7], 9000, dtype=BF16, tree=kind == "tree", draft=kind == "draft", temperatures=[1.0, 0.0, 0.6], seed=16)
    target, tokens, uniforms = d.target.to(DEV), d.tokens.to(DEV), d.uniforms.to(DEV)
    starts = torch.tensor(d.starts, dtype=torch.int32, device=DEV)
    parents = torch.tensor(d.parents, dtype=torch.int32, device=DEV) if d.tree else None
    draft, temps = None if d.draft is None else d.draft.to(DEV), torch.tensor(d.temperatures, device=DEV)
    call = lambda: ops.verify_drafts(target, tokens, starts, uniforms, max_rows=8, parents=parents, draft_probs=draft, temperatures=temps)   # noqa: E731
    call()
    graphs, outs = [], []
    for _ in range(2):                                     # two graphs of the same call, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for again in range(4):
        e = Drafts([5, 3, 7], 9000, dtype=BF16, tree=d.tree, draft=d.draft is not None, temperatures=[0.0, 0.9, 1.3], seed=20 + again)
        for held, new in ((target, e.target), (tokens, e.tokens), (uniforms, e.uniforms), (temps, torch.tensor(e.temperatures))):
            held.copy_(new)
        if d.tree:
            parents.copy_(torch.tensor(e.parents, dtype=torch.int32))
        if draft is not None:
            draft.copy_(e.draft)
        graphs[again % 2].replay()
        e.check(call(), 8)
        e.check(outs[again % 2], 8)


def test_verify_on_two_streams_at_once():
    cases = [Drafts([6, 4, 8], 20000 + i, dtype=BF16, draft=i % 2 == 1, tree=i % 2 == 0, seed=30 + i) for i in range(4)]
    cases[0].run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], []
    for d, stream in zip(cases, streams):
        with torch.cuda.stream(stream):
            got.append([d.run() for _ in range(3)])
    torch.cuda.synchronize()
    for d, answers in zip(cases, got):
        for a in answers:
            d.check(a)


def test_verify_of_no_rows():
    starts = torch.zeros(4, dtype=torch.int32, device=DEV)
    for draft in (None, torch.zeros(0, 100, device=DEV)):
        rows, counts, following = ops.verify_drafts(torch.zeros(0, 100, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), starts,
                                                    torch.zeros(0, 2, device=DEV), max_rows=3, draft_probs=draft)
        assert bool((rows == -1).all()) and bool((counts == 0).all()) and bool((following == -1).all())


def test_verify_refuses_tensors():
    d = Drafts([3], 50)
    ok = dict(target=d.target.to(DEV), tokens=d.tokens.to(DEV), row_starts=torch.tensor([0, 3], dtype=torch.int32, device=DEV), uniforms=d.uniforms.to(DEV))
    ops.verify_drafts(**ok)
    for kw in (dict(target=ok["target"].double()), dict(target=ok["target"][:, ::2]), dict(target=ok["target"][0]), dict(tokens=ok["tokens"].long()),
               dict(tokens=ok["tokens"][:2]), dict(uniforms=ok["uniforms"][:, :1]), dict(uniforms=ok["uniforms"].double()),
               dict(row_starts=ok["row_starts"][:1]), dict(row_starts=ok["row_starts"].long()), dict(max_rows=0), dict(max_rows=65),
               dict(draft_probs=torch.zeros(3, 49, device=DEV)), dict(draft_probs=torch.zeros(3, 50, dtype=BF16, device=DEV)),
               dict(temperatures=torch.ones(2, device=DEV)), dict(probs=True, target=ok["target"].to(BF16)), dict(parents=torch.zeros(3, device=DEV)),
               dict(tokens=ok["tokens"].cpu())):
        with pytest.raises(ValueError):
            ops.verify_drafts(**{**ok, **kw})
    with pytest.raises(Exception, match="temperatures"):
        ops.verify_drafts(**ok, probs=True, temperatures=torch.ones(1, device=DEV))
    with pytest.raises(Exception, match="chains"):
        ops.verify_drafts(**ok, draft_probs=torch.zeros(3, 50, device=DEV), parents=torch.zeros(3, dtype=torch.int32, device=DEV))


# ------------------------------------------------------------------------------------ acceptance
def _check_accepted(s: Step, paths, counts, lens, weights, width):
    want = [[x.clone() for x in side] for side in s.cache]
    scales = [[x.clone() for x in side] for side in s.scales] if s.scales else None
    w = s.weights.clone()
    for b, t in enumerate(s.lens):
        n = s.rows[b]
        moves = odec.accepted_moves(paths[b], min(counts[b], width), n)
        assert int(lens[b]) == max(t - n + len(moves), 0)
        slot = lambda i: (s.tables[b][(t - n + i) // s.block], (t - n + i) % s.block)      # noqa: E731
        for r, j in moves:
            if t - n + j < 0:
                continue
            (fp, fo), (tp, to) = slot(r), slot(j)
            if not (0 <= fp < s.pool and 0 <= tp < s.pool):
                continue
            for l in range(s.layers):
                for side in (0, 1):
                    x = _bits(want[side][l]) if s.fp8 else want[side][l]
                    x = want[side][l].view(torch.uint8) if s.fp8 else want[side][l]
                    x[tp, to] = x[fp, fo]
                    if scales:
                        scales[side][l][tp, to] = scales[side][l][fp, fo]
                w[l, tp, to] = w[l, fp, fo]
    for l in range(s.layers):
        for side, cache in ((0, s.dk), (1, s.dv)):
            assert torch.equal(_bits(cache[l].cpu()), _bits(want[side][l].view(cache[l].dtype))), (l, side)
            if scales:
                assert torch.equal((s.dks, s.dvs)[side][l].cpu().view(s.pool, s.block, s.h), scales[side][l])
    if weights is not None:
        assert torch.equal(weights.cpu(), w)


@pytest.mark.parametrize("dtype,row_scales", [(BF16, False), (FP16, False), (FP8, True), (torch.uint8, False)])
@pytest.mark.parametrize("dim,kv_heads,block", [(128, 8, 16), (64, 3, 8), (256, 9, 24), (64, 1, 1), (128, 2, 64)])
@pytest.mark.parametrize("with_weights", [False, True])
def test_accept(dtype, row_scales, dim, kv_heads, block, with_weights):
    s = Step([70, 9, 130, 20, 64, 3], rows=[16, 9, 64, 4, 64, 5], q_heads=kv_heads, kv_heads=kv_heads, dim=dim, block=block, dtype=dtype,
             row_scales=row_scales, layers=3, seed=dim + block)
    kv, batch = s.device()
    g = torch.Generator().manual_seed(17)
    width = 64
    paths, counts = [], []
    for n, c in zip(s.rows, (5, 9, 64, 1, 30, 3)):
        p = sorted(torch.randperm(n, generator=g)[:c].tolist())
        paths.append(p + [-1] * (width - len(p)))
        counts.append(c)
    weights = s.weights.to(DEV) if with_weights else None
    lens = ops.accept_drafts(kv, batch, s.dstarts, torch.tensor(paths, dtype=torch.int32, device=DEV), torch.tensor(counts, dtype=torch.int32, device=DEV),
                             weights=weights)
    _check_accepted(s, paths, counts, lens.cpu(), weights, width)


def test_accept_lists_that_are_no_paths():
    s = Step([40, 40, 40, 40, 40, 5, 40], rows=[8, 8, 8, 8, 0, 9, 8], layers=2, seed=18)
    kv, batch = s.device()
    s.tables[6][2] = s.pool + 1
    batch.block_table[6, 2] = s.pool + 1
    paths = [[0, 3, 3, 5], [0, 3, 8, 7], [0, -1, 2, 3], [5, 4, -1, -1], [0, 1, 2, 3], [0, 5, 7, 8], [0, 2, 5, 7]]
    counts = [4, 4, 4, -3, 2, 4, 1 << 20]
    lens = ops.accept_drafts(kv, batch, s.dstarts, torch.tensor(paths, dtype=torch.int32, device=DEV), torch.tensor(counts, dtype=torch.int32, device=DEV))
    _check_accepted(s, paths, counts, lens.cpu(), None, 4)


def test_accept_replayed_behind_verification():
    """Both captured together, replayed with other logits: the moves follow the new answers."""
    s = Step([60, 45], rows=[7, 5], layers=2, seed=19)
    kv, batch = s.device()
    d = Drafts(s.rows, 500, tree=True, temperatures=[0.0, 1.0], seed=40, agree=0.9)
    held = [d.target.to(DEV), d.tokens.to(DEV), d.uniforms.to(DEV), torch.tensor(d.parents, dtype=torch.int32, device=DEV)]
    temps = torch.tensor(d.temperatures, device=DEV)

    def call():
        rows, counts, following = ops.verify_drafts(held[0], held[1], s.dstarts, held[2], max_rows=7, parents=held[3], temperatures=temps)
        return rows, counts, following, ops.accept_drafts(kv, batch, s.dstarts, rows, counts)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for again in range(4):
        e = Drafts(s.rows, 500, tree=True, temperatures=[0.0, 1.0], seed=41 + again, agree=0.9)
        for x, new in zip(held, (e.target, e.tokens, e.uniforms, torch.tensor(e.parents, dtype=torch.int32))):
            x.copy_(new)
        for side, cache in ((0, s.dk), (1, s.dv)):
            for l in range(2):
                cache[l].copy_(s.cache[side][l])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        e.check(got[:3], 7)
        _check_accepted(s, got[0].cpu().tolist(), got[1].cpu().tolist(), got[3].cpu(), None, 7)


def test_accept_refuses_tensors():
    s = Step([20], rows=[4])
    kv, batch = s.device()
    rows, counts = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    ops.accept_drafts(kv, batch, s.dstarts, rows, counts)
    for kw in (dict(rows=rows[0]), dict(rows=rows.long()), dict(rows=torch.zeros(2, 4, dtype=torch.int32, device=DEV)), dict(counts=counts.long()),
               dict(rows=torch.zeros(1, 65, dtype=torch.int32, device=DEV)), dict(row_starts=s.dstarts[:1]), dict(weights=torch.zeros(1, 3, device=DEV))):
        args = {**dict(row_starts=s.dstarts, rows=rows, counts=counts), **kw}
        with pytest.raises(ValueError):
            ops.accept_drafts(kv, batch, args.pop("row_starts"), args.pop("rows"), args.pop("counts"), **args)


# ------------------------------------------------------------------------------- all of it together
class TinyModel:
    """Embeddings, projections and an output of fixed random numbers: two layers of attention over the cache, no residual."""

    def __init__(self, vocab=61, hq=8, h=2, d=64, layers=2, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.vocab, self.hq, self.h, self.d, self.layers = vocab, hq, h, d, layers
        w = hq * d
        rnd = lambda *shape: (torch.randn(*shape, generator=g) / shape[0] ** 0.5).to(DEV)       # noqa: E731
        self.embed = torch.randn(vocab, w, generator=g).to(DEV)
        self.proj = [rnd(w, (hq + 2 * h) * d) for _ in range(layers)]
        self.head = rnd(w, vocab) * 6
        self.norm = [(1 + 0.2 * torch.randn(d, generator=g)).to(DEV) for _ in range(2)]
        self.inv_freq = rope.default_inv_freq(d, 1e4).to(DEV)

    def forward(self, kv, batch, tokens, positions, starts, parents, max_rows, weights):
        """Logits [rows, vocab] of the rows, whose keys and values are then cached in every layer."""
        x = self.embed[tokens.long()]
        for l in range(self.layers):
            qkv = (x @ self.proj[l]).to(FP16).view(len(x), self.hq + 2 * self.h, self.d)
            q, k, v = qkv[:, :self.hq], qkv[:, self.hq:self.hq + self.h], qkv[:, self.hq + self.h:]
            q = ops.write_paged(kv, batch, q, k, v, positions, self.inv_freq, layer=l, row_starts=starts, q_norm=self.norm[0], k_norm=self.norm[1])
            out, _ = ops.attend_paged(kv, batch, q, layer=l, row_starts=starts, parents=parents, max_rows=max_rows, weights=weights)
            x = x + out.float().view(len(x), -1)
        return x @ self.head


@pytest.mark.parametrize("dtype", [FP16, FP8])
def test_drafted_decoding_gives_the_tokens_of_single_steps(dtype):
    """Write, attend, verify, accept over trees of drafts, some right and some wrong, against one token at a time: the same tokens, and the same rows in
    the cache.  Attention rounds differently where a row is one of many: that the logits it leads to differ by less than half of what the
    largest leads by is asserted of every token."""
    m = TinyModel(seed=3)
    block, pool, steps, first = 16, 64, 24, [11, 30]
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, m.vocab, (n,), generator=g).tolist() for n in first]
    tables = [list(range(0, 20)), list(range(20, 40))]

    def fresh():
        kind = dict(dtype=FP16) if dtype == FP16 else dict(dtype=FP8)
        k, v = ([torch.zeros(pool, block, m.h, m.d, device=DEV, **kind) for _ in range(m.layers)] for _ in range(2))
        ks, vs = (([torch.ones(pool * block * m.h, device=DEV) for _ in range(m.layers)] for _ in range(2)) if dtype == FP8 else (None, None))
        return ops.PagedKV(k, v, "half", ks, vs), k, v, torch.zeros(m.layers, pool, block, m.h, device=DEV)

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)           # noqa: E731

    def prompt(kv, weights):
        """The prompt's rows, all but the last token's, then the state: tokens cached, and the token to come next."""
        n = [len(p) - 1 for p in prompts]
        batch = ops.StepBatch(torch.device(DEV), n, block_tables=tables)
        m.forward(kv, batch, i32([t for p in prompts for t in p[:-1]]), i32([i for c in n for i in range(c)]), i32([0, n[0], sum(n)]), None, 64, weights)
        return n, [p[-1] for p in prompts]

    # one token at a time
    kv, k1, v1, w1 = fresh()
    lens, last = prompt(kv, w1)
    single = [[t] for t in last]
    lead, alone = [], []
    for _ in range(steps):
        batch = ops.StepBatch(torch.device(DEV), [t + 1 for t in lens], block_tables=tables)
        logits = m.forward(kv, batch, i32(last), i32(lens), None, None, None, w1)
        top = logits.topk(2, -1)
        lead.append((top.values[:, 0] - top.values[:, 1]).tolist())
        alone.append(logits)
        last, lens = top.indices[:, 0].tolist(), [t + 1 for t in lens]
        for b in range(2):
            single[b].append(last[b])
    # trees of five drafts: the right continuation on one branch, wrong tokens on the others
    kv, k2, v2, w2 = fresh()
    lens, last = prompt(kv, w2)
    made = [[t] for t in last]
    accepted = []
    while min(len(x) for x in made) <= steps:
        rows, parents, tokens, positions, starts = [], [], [], [], [0]
        for b in range(2):
            known = single[b][len(made[b]):] + [0] * 6
            wrong = [(t + 1) % m.vocab for t in known]
            tree = [(-1, last[b], 0), (0, wrong[0], 1), (0, known[0], 1), (1, known[1], 2), (2, known[1], 2), (4, wrong[2] if len(made[b]) % 2 else known[2], 3)]
            if b == 1:
                tree = tree[:4] if len(made[b]) % 3 == 0 else tree
            for p, t, depth in tree:
                parents.append(p)
                tokens.append(t)
                positions.append(lens[b] + depth)
            rows.append(len(tree))
            starts.append(starts[-1] + len(tree))
        batch = ops.StepBatch(torch.device(DEV), [t + n for t, n in zip(lens, rows)], block_tables=tables)
        logits = m.forward(kv, batch, i32(tokens), i32(positions), i32(starts), i32(parents), 6, w2)
        path, counts, following = ops.verify_drafts(logits, i32(tokens), i32(starts), torch.zeros(len(tokens), 2, device=DEV), max_rows=6,
                                                    parents=i32(parents), temperatures=torch.zeros(2, device=DEV))
        new = ops.accept_drafts(kv, batch, i32(starts), path, counts, weights=w2)
        for b in range(2):
            c = int(counts[b])
            for i, r in enumerate(path[b, :c].tolist()):
                at = len(made[b]) - 1 + i
                if at < steps:
                    assert float((logits[starts[b] + r] - alone[at][b]).abs().max()) < lead[at][b] / 2, (at, b)
            accepted.append(c)
            made[b] += [tokens[starts[b] + r] for r in path[b, 1:c].tolist()] + [int(following[b])]
            assert int(new[b]) == lens[b] + c
            lens[b], last[b] = int(new[b]), int(following[b])
    assert max(accepted) >= 4 and min(accepted) >= 1
    for b in range(2):
        n = min(len(made[b]), steps + 1)
        assert made[b][:n] == single[b][:n]
    # the first layer's rows go by token and position alone: the same bits either way
    for side1, side2 in ((k1, k2), (v1, v2)):
        for b in range(2):
            cached = first[b] - 1 + steps
            page = [tables[b][t // block] for t in range(cached)]
            off = [t % block for t in range(cached)]
            a, c = (x[0].view(torch.uint8) if dtype == FP8 else x[0] for x in (side1, side2))
            assert torch.equal(_bits(a[page, off]), _bits(c[page, off]))
