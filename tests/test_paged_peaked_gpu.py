"""Attention whose rows have one key far ahead of thousands of others: what the others leave together is far above each one's share."""
import numpy as np
import pytest

from paged_batches import Batch, check, rounded

pytestmark = pytest.mark.gpu


def _peaked(n_seqs, rows, length, heads, kv_heads, dim, kind, lead, shared=0, at=0):
    """n_seqs sequences over the same pages.  The key at position `at` is `lead` (in units of the exponent) ahead of the others, whose scores differ by some 0.1,
    and has values of 0, as a position has that takes up attention which is wanted nowhere; the others' values are 1 on average."""
    b = Batch(n_seqs + length, [(rows, length)], heads, kv_heads, dim, 16, kind, poison=0.0, shared=shared)
    rng, used = b.rng, -(-length // 16)
    u = np.where(rng.random(dim) < 0.5, -1.0, 1.0)
    b.k[b.table[0, :used]] = rounded(rng.normal(0, 0.1, (used, kv_heads, 16, dim)), kind)
    b.v[b.table[0, :used]] = rounded(rng.normal(1, 0.5, (used, kv_heads, 16, dim)), kind)
    page = b.table[0, at // 16]
    b.k[page, :, at % 16], b.v[page, :, at % 16] = rounded(lead / dim ** 0.5 * u, kind), 0.0
    b.seqs = [(rows, length)] * n_seqs
    b.table = np.repeat(b.table, n_seqs, 0)
    b.q_start, b.kv_len = (np.arange(n_seqs + 1) * rows).astype(np.int32), np.full(n_seqs, length, np.int32)
    b.n_rows = b.rows = n_seqs * rows
    b.q = np.broadcast_to(u.astype(np.float32), (b.rows, heads, dim)).copy()
    return b


PEAKED = {
    "single rows": dict(n_seqs=150, rows=1, length=2000, heads=4, kv_heads=4, dim=64),
    "drafts, 128": dict(n_seqs=80, rows=3, length=1500, heads=8, kv_heads=4, dim=128),
    "a prompt": dict(n_seqs=1, rows=200, length=3000, heads=8, kv_heads=8, dim=64),
    "prompts, 128": dict(n_seqs=3, rows=150, length=2000, heads=8, kv_heads=4, dim=128),
    "shared by many rows": dict(n_seqs=300, rows=1, length=1100, heads=16, kv_heads=4, dim=64, shared=1024),
    "ahead of one's own": dict(n_seqs=300, rows=1, length=1100, heads=16, kv_heads=4, dim=64, shared=1024, at=1030),
    "shared by few rows": dict(n_seqs=20, rows=1, length=4200, heads=8, kv_heads=2, dim=128, shared=4096),
}


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lead", [12.0, 15.0, 17.0])
@pytest.mark.parametrize("name", PEAKED)
def test_a_key_far_ahead_of_the_others(ctx, name, lead, kind):
    """The bound is that of every batch: a weight is off by half a step of the cache's type relative to its own size, also those e^-17 below the largest."""
    b = _peaked(kind=kind, lead=lead, **PEAKED[name])
    check(b, b.attend(ctx), name)


@pytest.mark.parametrize("rows,n_seqs,shared", [(1, 40, 0), (200, 1, 0), (1, 300, 512)])
@pytest.mark.parametrize("late", [3.0, 5.0, 5.5])
def test_values_near_the_end_of_the_range(ctx, rows, n_seqs, shared, late):
    """A key somewhat ahead of those in front of it, with values of which e^late do not fit f32: its weight is 1 of the sum, whatever it is before that is divided by."""
    b = _peaked(n_seqs, rows, 700, 16, 4, 64, "bf16", late, shared=shared, at=150)
    b.v[b.table[0, :-(-700 // 16)]] = 0.0
    b.v[b.table[0, 150 // 16], :, 150 % 16] = rounded(np.full((4, 64), 2.9e38 / np.exp(late) * 2.5), "bf16")
    check(b, b.attend(ctx))
