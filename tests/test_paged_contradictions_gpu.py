"""Starts, lengths and pages on the device that contradict each other or the tensors: what is reported, and what is left as it was."""
import ctypes as C

import numpy as np
import pytest

from paged_batches import Batch, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seqs,rows,heads,kv_heads,length", [(60, 1920, 64, 64, 600000), (200, 6400, 32, 32, 131072), (4096, 4096, 32, 8, 16384)])
def test_starts_that_fall_and_would_be_more_work_than_can_be_counted(ctx, n_seqs, rows, heads, kv_heads, length):
    """Every other sequence claims all rows: 2^32 steps and more.  Reported, and the next call is as ever.  (A plan of a warp that the merge works out itself, one
    that it reads, one of a whole block.)"""
    import runit_mac_b200 as R
    tiles, steps = -(-rows * (heads // kv_heads) // 16), (length + 31) // 32
    assert (n_seqs // 2) * tiles * kv_heads * steps >= 1 << 32
    page, dim = 64, 64
    ld = -(-length // page)
    pool = ctx.buffer_from(np.zeros(kv_heads * page * dim, np.uint16))
    table, lens = ctx.buffer_from(np.zeros((n_seqs, ld), np.int32)), ctx.buffer_from(np.full(n_seqs, length, np.int32))
    starts = ctx.buffer_from(np.array([i % 2 * rows for i in range(n_seqs + 1)], np.int32))
    cfg = R.PagedCfg(heads=heads, kv_heads=kv_heads, dim=dim, page=page, n_pages=1, type=R.TYPE_F16, window=0, scale=0.125, cap=0.0, slopes=None, k_pages=pool.ptr, v_pages=pool.ptr)
    batch = R.PagedBatch(n_seqs=n_seqs, rows=rows, table_ld=ld, shared_len=0, table=table.ptr, q_start=starts.ptr, kv_len=lens.ptr)
    n = R.paged_attention_scratch_bytes(ctx, cfg, batch)
    q, out = ctx.buffer_from(np.zeros(rows * heads * dim, np.uint16)), ctx.buffer_from(np.full(rows * heads * dim, 0x3C00, np.uint16))
    R.paged_attention(ctx, C.byref(cfg), C.byref(batch), q, heads * dim, out, heads * dim, ctx.new_buffer(n), n)
    with pytest.raises(R.KernelError) as e:
        ctx.flush()
    assert e.value.status == 2 and "paged cache" in str(e.value)
    b = Batch(6, [(1, 90), (2, 200), (1, 70)], 4, 2, 64, 16, "bf16")
    check(b, b.attend(ctx), "afterwards")
