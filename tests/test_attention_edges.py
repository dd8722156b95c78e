"""The attention and eviction entry points without a GPU: plans and refusals of calls at the edge of what they allow."""
from __future__ import annotations

import ctypes as C

from test_attention import _attend, _batch, _blocks, _evict, _layout
from triattention_amd import _lib


def test_scratch_for_a_copy_of_q_where_out_lies_in_its_memory():
    """Only where weights of many rows are wanted, by the elements that q and out span; without addresses as if they overlapped."""
    lib = _lib.load()
    rows, heads = 60, 64

    def need(**kw):
        p = _attend(num_q_heads=heads, num_rows=rows, max_rows=20, row_starts=8, q_stride_row=heads * 128, out_stride_row=heads * 128, **kw)
        got = lib.tri_attend_workspace_bytes(C.byref(_layout()), C.byref(_batch()), C.byref(p))
        assert got > 0
        return got

    size = rows * heads * 128 * 2
    base = need(q=1 << 20, out=(1 << 20) + size, weights=16)
    for q, out in ((1 << 20, 1 << 20), ((1 << 20) + size - 16, 1 << 20), (1 << 20, (1 << 20) + size - 16), (None, None)):
        assert need(q=q, out=out, weights=16) == base + size
    assert need(q=(1 << 20) + size, out=1 << 20, weights=16) == base
    assert need(q=16, out=16) == need(q=1 << 20, out=(1 << 20) + size)


def test_without_a_table_a_sequence_is_one_block():
    lib = _lib.load()
    kv, batch = C.byref(_layout()), C.byref(_batch(block_table=None, max_seq_len=17))
    fits = C.byref(_batch(block_table=None, max_seq_len=16))
    for code in (lib.tri_attend_paged(kv, batch, C.byref(_attend()), 256, 1 << 40, None),
                 lib.tri_attend_blocks(kv, batch, C.byref(_attend()), C.byref(_blocks()), 256, 1 << 40, None),
                 lib.tri_block_bounds(kv, batch, 40, 0, 16, 40 * 4 * 256, None),
                 lib.tri_select_by_weight(kv, batch, C.byref(_evict()), None, 8, 256, 1 << 40, None)):
        assert code == _lib.TRI_ERR_INVALID_ARGUMENT and b"block" in lib.tri_last_error()
    assert lib.tri_attend_workspace_bytes(kv, fits, C.byref(_attend())) > 0


def test_scratch_of_scores_is_bounded_by_the_cache():
    """A long sequence among many short ones: no more than 2 GiB, or K and V of the batch in one layer, for scores; batches of one length
    keep theirs."""
    lib = _lib.load()

    def need(lens, q_heads, dtype, weights, host=True):
        arr = (C.c_int32 * len(lens))(*lens)
        batch = _batch(num_seqs=len(lens), max_seq_len=max(lens), block_table_pitch=max(lens), seq_lens_host=C.cast(arr, C.c_void_p) if host else None)
        p = _attend(num_q_heads=q_heads, num_rows=len(lens), q_stride_row=q_heads * 128, out_stride_row=q_heads * 128, weights=weights)
        got = lib.tri_attend_workspace_bytes(C.byref(_layout(kv_dtype=dtype, k_scale_layers=8, v_scale_layers=8)), C.byref(batch), C.byref(p))
        assert got > 0
        return got

    for q_heads, dtype in ((4, 0), (32, 0), (128, 0), (32, 2)):
        size = 1 if dtype == 2 else 2
        for lens in ([60000] + [100 + 2 * i for i in range(399)], [100000] * 3 + [7] * 1000, [200000] + [50000] * 30):
            cache = sum(lens) * 4 * 128 * 2 * size
            parts = need(lens, q_heads, dtype, None)
            assert need(lens, q_heads, dtype, 16) <= parts + max(2 << 30, cache) + len(lens) * q_heads * 132 * 4 + 4096, (q_heads, dtype, lens[0])
        same = [131072] * 40
        for host in (True, False):
            assert need(same, q_heads, dtype, 16, host) >= 40 * 131072 * q_heads * 4
