"""Values that are no numbers among many rows that share keys: rows that see them carry them at no cost, rows that do not are as without them."""
import ctypes as C
import time

import numpy as np
import pytest

from paged_batches import Batch, from_bits, to_bits

pytestmark = pytest.mark.gpu


def _timed(ctx, b, calls=4):
    """The output, and the shortest time of a call, in seconds."""
    import runit_mac_b200 as R
    keep, cfg, batch = b.upload(ctx)
    ld, n = b.heads * b.dim, R.paged_attention_scratch_bytes(ctx, cfg, batch)
    q, out, scratch = ctx.buffer_from(to_bits(b.q, b.kind)), ctx.new_buffer(b.rows * ld * 2), ctx.new_buffer(n)
    took = []
    for _ in range(calls):
        t = time.perf_counter()
        R.paged_attention(ctx, C.byref(cfg), C.byref(batch), q, ld, out, ld, scratch, n)
        ctx.flush()
        took.append(time.perf_counter() - t)
    return from_bits(out.download(np.uint16, b.rows * ld), b.kind).reshape(b.rows, b.heads, b.dim), min(took)


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("seqs,heads,shared,window,at", [([(512, 8192)], 8, 0, 0, 100), ([(300, 6000), (260, 4000)], 8, 0, 0, 2000), ([(40, 4096 + 40 + i) for i in range(20)], 8, 4096, 0, 3000),
                                                         ([(512, 8192)], 8, 0, 900, 7600), ([(1024, 3000)], 64, 0, 0, 1500)])
@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128)])
def test_a_value_that_all_rows_see_costs_nothing(ctx, value, seqs, heads, shared, window, at, kind, dim):
    """The same bits in all other dimensions, and about the same time (a row done again takes several times a whole call)."""
    b = Batch(3, seqs, heads, heads, dim, 64, kind, shared=shared, window=window)
    want, clean = _timed(ctx, b)
    assert np.isfinite(want).all()
    b.v[b.table[0, at // 64], 2, at % 64, 7] = value
    got, took = _timed(ctx, b)
    for s, (nq, n) in enumerate(seqs):
        rows = slice(int(b.q_start[s]), int(b.q_start[s + 1]))
        here = s == 0 or at < shared
        sees = np.array([here and at <= p and (not window or p - at < window) for p in range(n - nq, n)])
        assert sees.all() or not here
        x = got[rows]
        assert (np.isfinite(x[:, 2, 7]) != sees).all()
        x = x.copy()
        if here:
            x[:, 2, 7] = want[rows][:, 2, 7]
        np.testing.assert_array_equal(x, want[rows])
    assert took <= 3 * clean + 1e-3, (took, clean)


@pytest.mark.parametrize("seqs,shared,window,spots", [([(200, 3001)], 0, 0, [3000, 2990, 2801]), ([(200, 3001)], 0, 777, [2900, 2050, 2100]), ([(150, 1237), (130, 950)], 0, 0, [1236, 949]),
                                                      ([(1, 200 + i) if i % 2 else (1, 1100 + i) for i in range(200)], 1024, 0, [230, 900]),
                                                      ([(1, 1100 + 9 * i) for i in range(200)], 1024, 1000, [330, 900])])
@pytest.mark.parametrize("cap,slopes", [(0.0, None), (8.0, [0.01 * (i + 1) for i in range(16)])])
def test_rows_on_either_side_of_a_value(ctx, seqs, shared, window, spots, cap, slopes):
    """Every row against the definition: the ones that do not see a place by the bound of any row, over numbers of positions that are no multiples of anything."""
    b = Batch(8, seqs, 16, 4, 64, 16, "f16", shared=shared, window=window, cap=cap, slopes=slopes)
    ref, bound = b.reference()
    for i, p in enumerate(spots):
        for s in range(len(seqs) if p >= shared else 1):
            if p < seqs[s][1]:
                b.v[b.table[s, p // 16], 1, p % 16, 3] = np.inf if i % 2 else np.nan
    got = b.attend(ctx)[:b.n_rows].astype(np.float64)
    for s, (nq, n) in enumerate(seqs):
        for i in range(nq):
            r, p = int(b.q_start[s]) + i, n - nq + i
            seen = any(j <= p and (not window or p - j < window) for j in spots)
            x, off = got[r].copy(), bound[r] + 2.0 ** -25
            if seen:
                assert not np.isfinite(x[4:8, 3]).any()
                x[4:8, 3] = ref[r, 4:8, 3]
            assert (np.abs(x - ref[r]) <= off).all(), (s, i)
