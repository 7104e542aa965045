"""Starts, lengths and pages on the device that contradict each other or the tensors: what is reported, and what is left as it was."""
import ctypes as C
import time

import numpy as np
import pytest

from paged_batches import Batch, check, from_bits, to_bits

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


def _append(ctx, b, proj):
    """Pages and queries that an append without rotation leaves, and whether it was reported."""
    import runit_mac_b200 as R
    keep, cfg, batch = b.upload(ctx)
    q = ctx.buffer_from(to_bits(np.full((b.rows, b.heads * b.dim), -3.0), b.kind))
    R.paged_append(ctx, C.byref(cfg), C.byref(batch), ctx.buffer_from(proj), R.TYPE_F32, proj.shape[1], None, 0, q, b.heads * b.dim)
    told = False
    try:
        ctx.flush()
    except R.KernelError as e:
        assert e.status == 2 and "paged cache" in str(e)
        told = True
    k, v = (from_bits(keep[n].download(np.uint16, b.k.size), b.kind).reshape(b.k.shape) for n in ("k", "v"))
    return k, v, from_bits(q.download(np.uint16, b.rows * b.heads * b.dim), b.kind).reshape(b.rows, b.heads, b.dim), told


@pytest.mark.parametrize("beyond", [0, 1, 2, 3, 40, 2 ** 30])
def test_an_append_behind_the_table_leaves_the_positions_in_front(ctx, beyond):
    """Three rows of a sequence whose length exceeds its pages: those with a place go there, the others nowhere; no other position changes."""
    b = Batch(3, [(2, 20), (3, 64), (1, 9)], 2, 1, 64, 16, "f16", poison=5.0, table_extra=0)
    proj = b.rng.normal(0, 1, (6, 256)).astype(np.float32)
    b.kv_len[1] = 64 + beyond
    k, v, q, told = _append(ctx, b, proj)
    assert told == (beyond > 0)
    x = from_bits(to_bits(proj, "f16"), "f16").reshape(6, 4, 64)
    want_k, want_v, want_q = b.k.copy(), b.v.copy(), np.full((6, 2, 64), -3.0)
    for s, r, p in ((0, 0, 18), (0, 1, 19), (1, 2, 61 + beyond), (1, 3, 62 + beyond), (1, 4, 63 + beyond), (2, 5, 8)):
        if p < 64:
            want_q[r] = x[r, :2]
            want_k[b.table[s, p // 16], :, p % 16], want_v[b.table[s, p // 16], :, p % 16] = x[r, 2:3], x[r, 3:]
    for got, want in ((k, want_k), (v, want_v), (q, want_q)):
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("entries", ["none", "others"])
def test_an_append_at_shared_positions_goes_to_the_pages_of_the_first_sequence(ctx, entries):
    """Sequences that end inside the shared positions, or whose rows begin there; what their own table rows hold for those positions is not looked at, be it no
    page or one of another sequence."""
    b = Batch(5, [(2, 40), (3, 33), (2, 20), (1, 60)], 2, 1, 64, 16, "bf16", shared=32, poison=5.0)
    b.table[1:, :2] = -7 if entries == "none" else b.table[[0, 0, 0], [2, 2, 2]][:, None]
    proj = b.rng.normal(0, 1, (8, 256)).astype(np.float32)
    k, v, q, told = _append(ctx, b, proj)
    assert not told
    x = from_bits(to_bits(proj, "bf16"), "bf16").reshape(8, 4, 64)
    want_k, want_v = b.k.copy(), b.v.copy()
    for s, r, p in ((0, 0, 38), (0, 1, 39), (0, 2, 30), (0, 3, 31), (1, 4, 32), (0, 5, 18), (0, 6, 19), (3, 7, 59)):
        want_k[b.table[s, p // 16], :, p % 16], want_v[b.table[s, p // 16], :, p % 16] = x[r, 2:3], x[r, 3:]
    np.testing.assert_array_equal(k, want_k)
    np.testing.assert_array_equal(v, want_v)
    np.testing.assert_array_equal(q, x[:, :2])


@pytest.mark.parametrize("what", ["pages", "lengths"])
@pytest.mark.parametrize("op", ["append", "single rows", "a prompt"])
def test_many_contradictions_take_no_longer_than_one(ctx, op, what):
    """Every page (or length) bad, call after call: each flush reports it, and no call takes a hundred times what a good one does."""
    import runit_mac_b200 as R
    n_seqs, rows, heads, length = {"append": (4, 1000, 8, 4000), "single rows": (16, 1, 8, 8000), "a prompt": (2, 300, 8, 6000)}[op]
    page, dim, ld = 16, 64, 500
    pool, table = ctx.buffer_from(np.zeros(heads * page * dim, np.uint16)), ctx.buffer_from(np.zeros((n_seqs, ld), np.int32))
    starts, lens = ctx.buffer_from(np.arange(n_seqs + 1, dtype=np.int32) * rows), ctx.buffer_from(np.full(n_seqs, length, np.int32))
    cfg = R.PagedCfg(heads=heads, kv_heads=heads, dim=dim, page=page, n_pages=1, type=R.TYPE_F16, window=0, scale=0.125, cap=0.0, slopes=None, k_pages=pool.ptr, v_pages=pool.ptr)
    batch = R.PagedBatch(n_seqs=n_seqs, rows=n_seqs * rows, table_ld=ld, shared_len=0, table=table.ptr, q_start=starts.ptr, kv_len=lens.ptr)
    n, width = R.paged_attention_scratch_bytes(ctx, cfg, batch), heads * dim
    proj, q, out, scratch = ctx.buffer_from(np.zeros((n_seqs * rows, 3 * width), np.uint16)), ctx.buffer_from(np.zeros((n_seqs * rows, width), np.uint16)), ctx.new_buffer(n_seqs * rows * width * 2), ctx.new_buffer(n)

    def timed(bad):
        took = []
        for _ in range(4):
            t = time.perf_counter()
            if op == "append":
                R.paged_append(ctx, C.byref(cfg), C.byref(batch), proj, R.TYPE_F16, 3 * width, None, 0, q, width)
            else:
                R.paged_attention(ctx, C.byref(cfg), C.byref(batch), q, width, out, width, scratch, n)
            if bad:
                with pytest.raises(R.KernelError) as e:
                    ctx.flush()
                assert e.value.status == 2
            else:
                ctx.flush()
            took.append(time.perf_counter() - t)
        return min(took)

    good = timed(False)
    if what == "pages":
        table.upload(np.full((n_seqs, ld), -7, np.int32))
    else:
        lens.upload(np.full(n_seqs, ld * page + 1, np.int32))
    assert timed(True) <= 20 * good + 2e-3
    table.upload(np.zeros((n_seqs, ld), np.int32))
    lens.upload(np.full(n_seqs, length, np.int32))
    timed(False)
