"""The entry points around attention without a GPU: what the C boundary refuses, plans, the axes of frequencies, and the oracle they are
held to."""
from __future__ import annotations

import ctypes as C
import math
import re
import subprocess

import pytest
import torch

from oracle import decoding as odec
from test_attention import _batch, _layout
from triattention_amd import _lib, build, ops, rope

INVALID, UNSUPPORTED = _lib.TRI_ERR_INVALID_ARGUMENT, _lib.TRI_ERR_UNSUPPORTED


def _write(**kw):
    base = dict(layer=0, num_q_heads=8, num_rows=3, num_blocks=40, dtype=0, num_axes=1, q=16, k=16, v=16, out=16, q_stride_row=8 * 128,
                q_stride_head=128, k_stride_row=4 * 128, k_stride_head=128, v_stride_row=4 * 128, v_stride_head=128, out_stride_row=8 * 128,
                out_stride_head=128, positions=16, inv_freq=16, eps=1e-6, rotary_scale=1.0, k_scale=1.0, v_scale=1.0)
    base.update(kw)
    return _lib.WriteParams(**base)


def _read(**kw):
    base = dict(layer=0, num_rows=3, num_blocks=40, out_dtype=0, row_starts=8, k_out=16, v_out=16, k_scale=1.0, v_scale=1.0)
    base.update(kw)
    return _lib.ReadParams(**base)


def _verify(**kw):
    base = dict(num_seqs=3, num_rows=10, max_rows=5, vocab=1000, target_dtype=0, target=16, target_stride=1000, tokens=8, row_starts=8,
                uniforms=8, rows=8, counts=8, next=8)
    base.update(kw)
    return _lib.VerifyParams(**base)


def _accept(**kw):
    base = dict(num_blocks=40, max_rows=5, row_starts=8, rows=8, counts=8, new_lens=32)
    base.update(kw)
    return _lib.AcceptParams(**base)


FP8 = dict(kv_dtype=2, k_scale_layers=8)


@pytest.mark.parametrize("layout,batch,params,code,word", [
    (dict(head_dim=96), {}, {}, UNSUPPORTED, b"head_dim"),
    (dict(v_layers=None), {}, {}, INVALID, b"v_layers"),
    (dict(kv_dtype=1), {}, {}, UNSUPPORTED, b"rows of type"),
    (dict(stride_head=1 << 27), {}, {}, UNSUPPORTED, b"stride_head"),
    (dict(stride_token=1 << 25), {}, {}, UNSUPPORTED, b"stride_token"),
    ({}, dict(num_seqs=0), {}, INVALID, b"num_seqs"),
    ({}, dict(seq_lens=None), {}, INVALID, b"seq_lens"),
    ({}, dict(block_table_pitch=6), {}, INVALID, b"block_table_pitch"),
    ({}, dict(block_table=None), {}, INVALID, b"block"),
    ({}, {}, dict(layer=2), INVALID, b"layer"),
    ({}, {}, dict(layer=-1), INVALID, b"layer"),
    ({}, {}, dict(num_q_heads=6), INVALID, b"multiple"),
    ({}, {}, dict(num_q_heads=0), INVALID, b"multiple"),
    ({}, {}, dict(dtype=2), UNSUPPORTED, b"dtype"),
    ({}, {}, dict(num_blocks=0), INVALID, b"num_blocks"),
    ({}, {}, dict(num_rows=-1), INVALID, b"num_rows"),
    ({}, {}, dict(num_rows=4), INVALID, b"row_starts"),
    ({}, {}, dict(num_rows=1 << 26, row_starts=8), UNSUPPORTED, b"in one call"),
    ({}, {}, dict(q=None), INVALID, b"q is NULL"),
    ({}, {}, dict(k=None), INVALID, b"k is NULL"),
    ({}, {}, dict(v=None), INVALID, b"v is NULL"),
    ({}, {}, dict(out=None), INVALID, b"out is NULL"),
    ({}, {}, dict(q=8), INVALID, b"aligned"),
    ({}, {}, dict(k_stride_row=4 * 128 + 4), INVALID, b"strides"),
    ({}, {}, dict(v_stride_head=1 << 27), UNSUPPORTED, b"heads of v"),
    ({}, {}, dict(q_stride_head=-128), UNSUPPORTED, b"heads of q"),
    ({}, {}, dict(out_stride_head=64), INVALID, b"out"),
    ({}, {}, dict(out_stride_row=64), INVALID, b"out"),
    ({}, {}, dict(positions=None), INVALID, b"positions"),
    ({}, {}, dict(inv_freq=None), INVALID, b"inv_freq"),
    ({}, {}, dict(num_axes=0), INVALID, b"axes"),
    ({}, {}, dict(num_axes=3, position_stride=2), INVALID, b"axes"),
    ({}, {}, dict(eps=-1e-6), INVALID, b"eps"),
    ({}, {}, dict(eps=math.nan), INVALID, b"eps"),
    ({}, {}, dict(rotary_scale=math.inf), INVALID, b"rotary_scale"),
    ({}, {}, dict(k_scale=0.5), INVALID, b"k_scale"),
    (dict(FP8, v_scale_layers=8), {}, dict(v_scale=2.0), INVALID, b"v_scale"),
    (FP8, {}, dict(k_scale=0.0), INVALID, b"k_scale"),
    (FP8, {}, dict(k_scale=-1.0), INVALID, b"k_scale"),
    (FP8, {}, dict(v_scale=math.nan), INVALID, b"v_scale"),
    (FP8, {}, dict(v_scale=1e-39), INVALID, b"reciprocals"),
])
def test_writing_refuses(layout, batch, params, code, word):
    lib = _lib.load()
    assert lib.tri_write_paged(C.byref(_layout(**layout)), C.byref(_batch(**batch)), C.byref(_write(**params)), None) == code
    assert word in lib.tri_last_error()


@pytest.mark.parametrize("layout,batch,params,code,word", [
    (dict(v_layers=None), {}, {}, INVALID, b"v_layers"),
    ({}, dict(block_table_pitch=6), {}, INVALID, b"block_table_pitch"),
    ({}, {}, dict(layer=2), INVALID, b"layer"),
    ({}, {}, dict(num_blocks=0), INVALID, b"num_blocks"),
    ({}, {}, dict(row_starts=None), INVALID, b"row_starts"),
    ({}, {}, dict(out_dtype=3), INVALID, b"out_dtype"),
    ({}, {}, dict(num_rows=-1), INVALID, b"num_rows"),
    ({}, {}, dict(num_rows=1 << 26), UNSUPPORTED, b"in one call"),
    ({}, {}, dict(k_out=None), INVALID, b"k_out"),
    ({}, {}, dict(v_out=8), INVALID, b"aligned"),
    ({}, {}, dict(k_scale=math.inf), INVALID, b"finite"),
])
def test_reading_refuses(layout, batch, params, code, word):
    lib = _lib.load()
    assert lib.tri_read_paged(C.byref(_layout(**layout)), C.byref(_batch(**batch)), C.byref(_read(**params)), None) == code
    assert word in lib.tri_last_error()


@pytest.mark.parametrize("params,code,word", [
    (dict(num_seqs=0), INVALID, b"sequences"),
    (dict(num_rows=-1), INVALID, b"rows"),
    (dict(max_rows=0), UNSUPPORTED, b"max_rows"),
    (dict(max_rows=65), UNSUPPORTED, b"max_rows"),
    (dict(vocab=0), INVALID, b"vocab"),
    (dict(vocab=(1 << 31) - 1, target_stride=(1 << 31) - 1), UNSUPPORTED, b"vocab"),
    (dict(target_dtype=3), INVALID, b"target_dtype"),
    (dict(target_probs=1), UNSUPPORTED, b"fp32 probabilities"),
    (dict(target_probs=1, target_dtype=2, temperatures=8), INVALID, b"temperatures"),
    (dict(draft_probs=8, draft_stride=1000, parents=8), UNSUPPORTED, b"chains"),
    (dict(target_stride=999), INVALID, b"stride"),
    (dict(draft_probs=8, draft_stride=999), INVALID, b"stride"),
    (dict(num_rows=1 << 20, vocab=1 << 25, target_stride=1 << 25), UNSUPPORTED, b"in one call"),
    (dict(num_rows=1 << 20, vocab=1 << 17, target_stride=1 << 17), UNSUPPORTED, b"in one call"),
])
def test_verification_refuses(params, code, word):
    lib = _lib.load()
    p = _verify(**params)
    assert lib.tri_verify_workspace_bytes(C.byref(p)) == 0
    assert lib.tri_verify_drafts(C.byref(p), 256, 1 << 40, None) == code
    assert word in lib.tri_last_error()


@pytest.mark.parametrize("params", [
    dict(num_seqs=1 << 24, max_rows=1),                                     # 2^24 sequences of four waves would fit, of eight not
    dict(num_seqs=(1 << 23) + 1, max_rows=1, draft_probs=8, draft_stride=1000),
    dict(num_seqs=1 << 21, max_rows=64),
])
def test_verification_refuses_launches_beyond_the_largest(params):
    """Whole workgroups count: a sequence of one row or piece takes one."""
    lib = _lib.load()
    p = _verify(**params)
    assert lib.tri_verify_drafts(C.byref(p), 256, 1 << 40, None) == UNSUPPORTED
    assert b"in one call" in lib.tri_last_error()


@pytest.mark.parametrize("params,word", [
    (dict(rows=None), b"rows"), (dict(counts=None), b"counts"), (dict(next=None), b"next"), (dict(row_starts=None), b"row_starts"),
    (dict(target=None), b"target"), (dict(tokens=None), b"tokens"), (dict(uniforms=None), b"uniforms"),
    (dict(target=17), b"aligned"), (dict(target_dtype=2, target=18), b"aligned"), (dict(draft_probs=2, draft_stride=1000), b"aligned"),
])
def test_verification_refuses_pointers(params, word):
    lib = _lib.load()
    p = _verify(**params)
    assert lib.tri_verify_drafts(C.byref(p), 256, 1 << 40, None) == INVALID
    assert word in lib.tri_last_error()


def test_verification_needs_its_workspace():
    lib = _lib.load()
    for p in (_verify(), _verify(draft_probs=8, draft_stride=1000), _verify(num_rows=0)):
        need = lib.tri_verify_workspace_bytes(C.byref(p))
        assert need >= 256
        for at, size in ((None, need), (256, need - 1), (128, need)):
            assert lib.tri_verify_drafts(C.byref(p), at, size, None) == _lib.TRI_ERR_WORKSPACE
    # sixteen bytes for 2048 logits of a row
    big = _verify(num_rows=384, vocab=131072, target_stride=131072)
    assert 384 * 64 * 16 <= lib.tri_verify_workspace_bytes(C.byref(big)) <= 384 * 64 * 16 + 2048


@pytest.mark.parametrize("layout,batch,params,code,word", [
    (dict(v_layers=None), {}, {}, INVALID, b"v_layers"),
    ({}, dict(block_table_pitch=6), {}, INVALID, b"block_table_pitch"),
    ({}, {}, dict(num_blocks=0), INVALID, b"num_blocks"),
    ({}, {}, dict(max_rows=0), UNSUPPORTED, b"max_rows"),
    ({}, {}, dict(max_rows=65), UNSUPPORTED, b"max_rows"),
    ({}, {}, dict(row_starts=None), INVALID, b"row_starts"),
    ({}, {}, dict(rows=None), INVALID, b"rows"),
    ({}, {}, dict(counts=None), INVALID, b"counts"),
    ({}, dict(seq_lens=24), dict(new_lens=24), INVALID, b"new_lens"),
    (dict(num_layers=4096), dict(num_seqs=2048), {}, UNSUPPORTED, b"in one call"),
    ({}, {}, dict(weights=16, weights_stride_layer=40 * 16 * 4 - 1), INVALID, b"less than a layer"),
])
def test_acceptance_refuses(layout, batch, params, code, word):
    lib = _lib.load()
    assert lib.tri_accept_drafts(C.byref(_layout(**layout)), C.byref(_batch(**batch)), C.byref(_accept(**params)), None) == code
    assert word in lib.tri_last_error()


def test_calls_of_no_rows_do_nothing():
    lib = _lib.load()
    kv, batch = C.byref(_layout()), C.byref(_batch())
    assert lib.tri_write_paged(kv, batch, C.byref(_write(num_rows=0, row_starts=8, q=None, k=None, v=None, out=None, positions=None)), None) == 0
    assert lib.tri_read_paged(kv, batch, C.byref(_read(num_rows=0, k_out=None, v_out=None)), None) == 0


def test_missing_parameters_are_refused():
    lib = _lib.load()
    kv, batch = C.byref(_layout()), C.byref(_batch())
    assert lib.tri_write_paged(kv, batch, None, None) == INVALID
    assert lib.tri_read_paged(kv, batch, None, None) == INVALID
    assert lib.tri_accept_drafts(kv, batch, None, None) == INVALID
    assert lib.tri_verify_drafts(None, 256, 1 << 20, None) == INVALID
    assert lib.tri_verify_workspace_bytes(None) == 0
    assert lib.tri_write_paged(None, batch, C.byref(_write()), None) == INVALID
    assert lib.tri_write_paged(kv, None, C.byref(_write()), None) == INVALID


@pytest.mark.parametrize("kind", [_lib.WriteParams, _lib.ReadParams, _lib.VerifyParams, _lib.AcceptParams])
def test_packed_parameters_are_the_structures_bytes(kind):
    fields = [1000003 * (i + 1) if t is not C.c_float else 0.5 + i for i, (_, t) in enumerate(kind._fields_)]
    packed = _lib.packer(kind)(*fields)
    whole = kind.from_buffer_copy(packed)
    assert len(packed) == C.sizeof(kind)
    assert [getattr(whole, name) for name, _ in kind._fields_] == fields


def test_verification_of_host_tensors_is_refused():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.verify_drafts(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), torch.zeros(2, 2))


# --------------------------------------------------------------------------------------- axes
def test_section_axes():
    assert rope.section_axes([2, 3, 1]).tolist() == [0, 0, 1, 1, 1, 2]
    assert rope.section_axes([2, 0, 1]).tolist() == [0, 0, 2]
    assert rope.section_axes([3, 2, 2], interleaved=True).tolist() == [0, 1, 2, 0, 1, 2, 0]
    assert rope.section_axes([24, 20, 20], interleaved=True).tolist() == [f % 3 if f < 60 else 0 for f in range(64)]
    assert rope.section_axes([1, 3], interleaved=True).tolist() == [0, 1, 1, 1]
    assert rope.section_axes([16, 24, 24]).dtype == torch.int32
    for bad in ([], [0, 0], [-1, 3]):
        with pytest.raises(ValueError):
            rope.section_axes(bad)


# ------------------------------------------------------------------------------ the oracle itself
def test_oracle_rotation_turns_pairs_and_keeps_their_length():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 2, 8, generator=g).double()
    pos = torch.tensor([[0, 1, 7, 100000, 3]])
    inv = torch.tensor([1.0, 0.1, 0.01, 0.001])
    for half in (True, False):
        y = odec.rotated(x, pos, inv, None, half)
        assert torch.equal(y[0], x[0])
        pair = (lambda z, k: (z[..., k], z[..., k + 4])) if half else (lambda z, k: (z[..., 2 * k], z[..., 2 * k + 1]))
        for k in range(4):
            (a, b), (c, d) = pair(x, k), pair(y, k)
            assert float((torch.hypot(a, b) - torch.hypot(c, d)).abs().max()) < 1e-12
        # one step of a position is one angle: q . k goes by the difference of positions alone
        q, k = odec.rotated(x, pos + 5, inv, None, half), odec.rotated(x.flip(-1), pos + 2, inv, None, half)
        q2, k2 = odec.rotated(x, pos + 3, inv, None, half), odec.rotated(x.flip(-1), pos, inv, None, half)
        assert float(((q * k).sum(-1) - (q2 * k2).sum(-1)).abs().max()) < 1e-9
    several = odec.rotated(x, torch.stack([pos[0], pos[0] * 0]), inv, [0, 1, 0, 7], True)
    assert torch.equal(several[..., 1], x[..., 1]) and torch.equal(several[..., 5], x[..., 5])
    assert torch.equal(several[..., 3], odec.rotated(x, pos, inv, None, True)[..., 3])


def test_oracle_draws_and_verification():
    w = torch.tensor([0.0, 0.25, 0.0, 0.5, 0.25, 0.0], dtype=torch.float64)
    assert [odec.draw(w, u) for u in (0.0, 0.2499, 0.25, 0.7499, 0.75, 0.9999, 1.0, -1.0, math.nan)] == [1, 1, 3, 3, 4, 4, 4, 1, 1]
    assert odec.draw(torch.zeros(3, dtype=torch.float64), 0.5) == -1
    logits = torch.tensor([[0.0, 3.0, 3.0], [1.0, 0.0, -math.inf], [math.nan, -math.inf, 5.0]])
    u = torch.zeros(3, 2)
    assert odec.verify_sequence(logits, [9, 1, 0], u, None, 0.0) == ([0, 1, 2], 2)
    assert odec.verify_sequence(logits, [9, 2, 0], u, None, 0.0) == ([0], 1)
    # a tree: both children of row 0, the first that holds the token
    assert odec.verify_sequence(logits, [9, 0, 1], u, [-1, 0, 0], 0.0) == ([0, 2], 2)
    assert odec.verify_sequence(logits, [9, 1, 1], u, [-1, 0, 0], 0.0) == ([0, 1], 0)
    # a draft of certainty: accepted iff u < p, and what is left has none of it
    certain = torch.tensor([[0.0, 0.0, 0.0], [0.0, 1.0, 0.0]])
    p = odec.distribution(torch.tensor([0.0, 1.0, 0.5]), 1.0, False)
    for first in (0.0, 0.4, 0.6, 0.99):
        for second in (0.1, 0.9):
            path, tok = odec.verify_sequence(torch.tensor([[0.0, 1.0, 0.5], [5.0, 0.0, 0.0]]), [0, 1], torch.tensor([[0.0, second], [first, 0.0]]), None,
                                             1.0, certain)
            if first < float(p[1]):
                assert path == [0, 1] and tok == 0
            else:
                assert path == [0] and tok == (0 if second < float(p[0] / (p[0] + p[2])) else 2)


def test_oracle_verification_keeps_the_targets_distribution():
    """Summed over what the draft proposes and both random numbers, the token behind a row has the target's distribution."""
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(2, 4, generator=g) * 1.5
    q = torch.softmax(torch.randn(4, generator=g), -1)
    p = odec.distribution(logits[0], 1.0, False)
    steps, got = 40, torch.zeros(4, dtype=torch.float64)
    for x in range(4):
        for i in range(steps):
            for j in range(steps):
                u = torch.tensor([[0.0, (j + 0.5) / steps], [(i + 0.5) / steps, 0.0]])
                path, tok = odec.verify_sequence(logits, [0, x], u, None, 1.0, torch.stack([q, q]))
                got[x if len(path) == 2 else tok] += float(q[x]) / steps / steps
    assert float((got - p).abs().max()) < 2.0 / steps


def test_oracle_moves_end_where_a_list_is_no_path():
    assert odec.accepted_moves([0, 2, 5, -1], 3, 6) == [(0, 0), (2, 1), (5, 2)]
    assert odec.accepted_moves([0, 2, 2], 3, 6) == [(0, 0), (2, 1)]
    assert odec.accepted_moves([0, 2, 6], 3, 6) == [(0, 0), (2, 1)]
    assert odec.accepted_moves([-1, 2], 2, 6) == []
    assert odec.accepted_moves([0, 1, 2], 9, 2) == [(0, 0), (1, 1)]


@pytest.mark.parametrize("stride,word", [(0, b"eps"), (3, b"eps"), (1, b"axes"), (2, b"axes"), (-1, b"axes"), (-3, b"axes")])
def test_axes_of_positions_are_apart_or_the_same(stride, word):
    """(what is refused behind them says that they are not)"""
    params = _write(num_axes=3, position_stride=stride, eps=-1.0)
    assert _lib.load().tri_write_paged(C.byref(_layout()), C.byref(_batch()), C.byref(params), None) == INVALID
    assert word in _lib.load().tri_last_error()


# ------------------------------------------------------------------------------------- waits
def test_stores_of_every_wave_have_arrived_before_its_workgroup_is_counted(tmp_path):
    """The last workgroup of a sequence reads what every wave of the others stored.  A barrier does not wait for stores on their way, and the
    counting thread's write-back waits for its own wave's alone: in the compiled kernels each wave waits for its stores right before
    the barrier behind which the write-back stands."""
    try:
        compiler = build.hipcc()
    except RuntimeError as exc:
        pytest.skip(str(exc))
    out = tmp_path / "verify.s"
    subprocess.run([compiler, *build.HIPCC_FLAGS, f"-I{build.INCLUDE}", f"-I{build.CSRC}", "--cuda-device-only", "-S", str(build.CSRC / "tri_verify.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    kernels, lines = {}, None
    for line in out.read_text().splitlines():
        if m := re.match(r"(_Z\w*verify_(?:walk|chain)_kernel\w*):", line):
            lines = kernels.setdefault(m[1], [])
        elif ".end_amdhsa_kernel" in line or line.startswith("\t.section"):
            lines = None
        elif lines is not None and (words := line.split(";")[0].split()):
            lines.append(words)
    assert len(kernels) == 8
    for name, lines in kernels.items():
        counts = [i for i, words in enumerate(lines) if words[0] == "buffer_wbl2"]
        assert counts, name
        for at in counts:
            barrier = max(i for i in range(at) if lines[i][0] == "s_barrier")
            # back from the barrier, with no way in from elsewhere and no store between
            for words in reversed(lines[:barrier]):
                assert not words[0].endswith(":") and "store" not in words[0] and "atomic" not in words[0], (name, words)
                if words[0] == "s_waitcnt" and "vmcnt(0)" in words[1:]:
                    break
