"""The paged operators where the tensors are far larger than what a call looks at: pools and rows beyond 2^32 elements, tables for many times the lengths; and the
same tokens however they are split over steps."""
import ctypes as C

import numpy as np
import pytest

from paged_batches import Batch, check, from_bits, rounded, to_bits
from test_logprobs_gpu import _check
from test_paged_chain_gpu import VOCAB, Server, _pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [dict(seqs=[(1, 200), (3, 77)]), dict(seqs=[(150, 300)]), dict(seqs=[(1, 129 + i) for i in range(60)], shared=128)])
def test_pools_beyond_32_bits(ctx, case):
    """Pages from both ends of pools of 2^32 elements and more: append (its rows read back there), then attention.  (Only the pages in use are ever touched.)"""
    import torch
    import runit_mac_b200 as R
    heads, kvh, dim, page, far = 8, 2, 128, 64, 2 ** 32 // (2 * 64 * 128)
    b = Batch(4, heads=heads, kv_heads=kvh, dim=dim, page=page, kind="bf16", poison=0.0, **case)
    where = np.where(np.arange(b.n_pages) % 2 == 0, np.arange(b.n_pages), far + np.arange(b.n_pages))
    n_pages = far + b.n_pages
    pools = {n: torch.empty((n_pages, kvh, page, dim), dtype=torch.int16, device="cuda") for n in ("k", "v")}
    index = torch.from_numpy(where).cuda()
    for n, x in (("k", b.k), ("v", b.v)):
        pools[n][index] = torch.from_numpy(to_bits(x, "bf16").view(np.int16)).cuda()
    torch.cuda.synchronize()
    keep, cfg, batch = b.upload(ctx)
    table = ctx.buffer_from(np.where((b.table >= 0) & (b.table < b.n_pages), where[b.table], -7).astype(np.int32))
    cfg.n_pages, cfg.k_pages, cfg.v_pages, batch.table = n_pages, pools["k"].data_ptr(), pools["v"].data_ptr(), table.ptr
    row, width = (heads + 2 * kvh) * dim, heads * dim
    proj = b.rng.normal(0, 1, (b.rows, row)).astype(np.float32)
    q = ctx.new_buffer(b.rows * width * 2)
    R.paged_append(ctx, C.byref(cfg), C.byref(batch), ctx.buffer_from(proj), R.TYPE_F32, row, None, 0, q, width)
    ctx.flush()
    x = rounded(proj, "bf16").reshape(b.rows, -1, dim)
    for s, (nq, n) in enumerate(b.seqs):
        for i in range(nq):
            p = n - nq + i
            pg = b.table[0 if p < b.shared else s, p // page]
            b.k[pg, :, p % page], b.v[pg, :, p % page] = x[b.q_start[s] + i, heads:heads + kvh], x[b.q_start[s] + i, heads + kvh:]
    for n, want in (("k", b.k), ("v", b.v)):
        np.testing.assert_array_equal(from_bits(pools[n][index].cpu().numpy().view(np.uint16), "bf16"), want)
    check(b, b.attend(ctx, keep=(keep, cfg, batch)))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_of_logits_beyond_32_bits(ctx, kind):
    """Three rows 2^31 elements apart (of which only their first ones are ever touched)."""
    import torch
    import runit_mac_b200 as R
    n, ld, k = 5003, 2 ** 31 + 5, 7
    x = rounded(np.random.default_rng(2).normal(0, 3, (3, n)), kind)
    wide = torch.empty(2 * ld + n, dtype=torch.float32 if kind == "f32" else torch.int16, device="cuda")
    for r in range(3):
        wide[r * ld:r * ld + n] = torch.from_numpy(x[r] if kind == "f32" else to_bits(x[r], kind).view(np.int16)).cuda()
    torch.cuda.synchronize()
    tokens = np.array([3, n - 1, 700], np.int32)
    lp, h, ids, top = ctx.new_buffer(12), ctx.new_buffer(12), ctx.new_buffer(12 * k), ctx.new_buffer(12 * k)
    R.token_logprobs(ctx, wide, R.TYPE_F32 if kind == "f32" else R.TYPE_BF16, ld, n, 3, ctx.buffer_from(tokens), lp, h, k, ids, top)
    ctx.flush()
    _check(x, tokens, k, (lp.download(np.float32, 3), h.download(np.float32, 3), ids.download(np.int32, 3 * k).reshape(3, k), top.download(np.float32, 3 * k).reshape(3, k)))


WIDE = {
    "single rows": dict(seqs=[(1, 1 + 31 * i) for i in range(20)], heads=8, kv_heads=2, dim=64, page=16, kind="f16"),
    "prompts": dict(seqs=[(300, 310), (40, 700), (0, 0), (256, 256)], heads=8, kv_heads=2, dim=128, page=64, kind="bf16"),
    "prompts behind shared positions": dict(seqs=[(60, 200), (90, 128 + 90), (33, 400)], heads=8, kv_heads=2, dim=64, page=32, kind="f16", shared=128),
    "a prompt beside single rows": dict(seqs=[(1, 150 + i) for i in range(40)] + [(128, 500)], heads=4, kv_heads=4, dim=64, page=16, kind="bf16"),
    "a window": dict(seqs=[(300, 900)], heads=4, kv_heads=1, dim=128, page=128, kind="f16", window=200),
}


@pytest.mark.parametrize("name", WIDE)
def test_tables_for_many_times_the_lengths(ctx, name):
    """A table for 131072 positions, as a step has it that is recorded once: most of the parts that the kernel for many rows cuts them into are empty."""
    b = Batch(sum(map(ord, name)), table_extra=131072 // WIDE[name]["page"], **WIDE[name])
    check(b, b.attend(ctx), name)


def test_the_same_tokens_over_other_steps(ctx):
    """Log probabilities of a recorded serving step over two splits of the same tokens.  What may differ is the order of sums, and through it roundings to bf16 on the
    way (queries, keys, weights, outputs, norms of 2 layers: 12 at 2^-9 each on average, of logits of some 3: 2^-9 sqrt(12) 3 = 0.02 for one of them); the largest of some
    hundred lies within four times that if all the roundings differed."""
    def serve(split):
        s = Server(ctx, 3, 40, _pages(3, 4, 2))
        rng = np.random.default_rng(31)
        ids = rng.integers(0, VOCAB, (3, 60))
        n, out = np.zeros(3, np.int64), {}
        ctx.graph_begin()
        s.step()
        graph = ctx.graph_end()
        for take in split:
            starts = np.concatenate([[0], np.cumsum(take)])
            n = n + take
            s.place(starts, n, np.concatenate([ids[k, n[k] - take[k]:n[k]] for k in range(3)]), np.concatenate([ids[k, n[k] - take[k] + 1:n[k] + 1] for k in range(3)]))
            graph.launch()
            ctx.flush()
            lp = s.get("lp")[:, 0]
            for k in range(3):
                for i in range(take[k]):
                    out[k, int(n[k]) - take[k] + i] = lp[starts[k] + i]
        graph.destroy()
        return out

    whole, single = serve([(20, 4, 12), (1, 20, 1), (11, 8, 19)]), serve([(1, 1, 1)] * 32)
    assert set(whole) == set(single)
    assert max(abs(whole[p] - single[p]) for p in whole) <= 0.08
