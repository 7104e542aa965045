"""Calls of three launches (shared positions beside own ones, then the merge), of which the later ones begin before the earlier ones have ended: behind producers,
recorded, on other streams, two at once, and over lengths that change from step to step without anybody's waiting."""
import ctypes as C

import numpy as np
import pytest

from paged_batches import Batch, check, from_bits, to_bits
from test_paged_gpu import _frequencies

pytestmark = pytest.mark.gpu

THREE = {
    "split kernel first": dict(seqs=[(1, 512 + 1 + 11 * i % 60) for i in range(300)], heads=16, kv_heads=4, dim=64, page=16, kind="f16", shared=512),
    "split kernel first, 128": dict(seqs=[(1, 768 + 1 + 13 * i % 90) for i in range(120)], heads=32, kv_heads=4, dim=128, page=64, kind="bf16", shared=768),
    "many rows of both": dict(seqs=[(30 + i, 256 + 30 + i + 7 * i) for i in range(8)], heads=8, kv_heads=2, dim=128, page=32, kind="f16", shared=256, extra_rows=5),
}


def _counted(ctx, b):
    before = ctx.launches
    got = b.attend(ctx)
    assert ctx.launches - before == 3
    return got


@pytest.mark.parametrize("name", THREE)
def test_however_the_launches_are_issued(ctx, name):
    import torch
    import runit_mac_b200 as R
    b = Batch(sum(map(ord, name)), **THREE[name])
    want = _counted(ctx, b)
    check(b, want, name)
    side = torch.cuda.Stream()
    other = R.Context(0, stream=side.cuda_stream)
    try:
        for pdl in (0, 1, 2):
            other.set_tuning("pdl", pdl)
            for _ in range(3):
                np.testing.assert_array_equal(want, _counted(other, b))
    finally:
        other.close()


def test_two_such_calls_at_once(ctx):
    import runit_mac_b200 as R
    other = R.Context(0)
    try:
        runs = []
        for c, name in ((ctx, "split kernel first"), (other, "many rows of both"), (other, "split kernel first, 128"), (ctx, "many rows of both")):
            b = Batch(len(runs), **THREE[name])
            want = _counted(c, b)
            keep, cfg, batch = b.upload(c)
            ld, n = b.heads * b.dim, R.paged_attention_scratch_bytes(c, cfg, batch)
            outs = [c.buffer_from(np.zeros(b.rows * ld, np.uint16)) for _ in range(10)]
            runs.append((c, b, want, keep, cfg, batch, ld, n, c.buffer_from(to_bits(b.q, b.kind)), outs, c.new_buffer(n)))
        for i in range(10):
            for c, b, want, keep, cfg, batch, ld, n, q, outs, scratch in runs:
                R.paged_attention(c, C.byref(cfg), C.byref(batch), q, ld, outs[i], ld, scratch, n)
        ctx.flush()
        other.flush()
        for c, b, want, keep, cfg, batch, ld, n, q, outs, scratch in runs:
            for o in outs:
                np.testing.assert_array_equal(from_bits(o.download(np.uint16, b.rows * ld), b.kind).reshape(want.shape)[:b.n_rows], want[:b.n_rows])
    finally:
        other.close()


@pytest.mark.parametrize("name", THREE)
@pytest.mark.parametrize("recorded", [False, True])
def test_steps_over_changing_lengths_without_a_wait(ctx, name, recorded):
    """Two layers of append and attention, one scratch, step after step in one stream: starts, lengths and projections of each step are copied into place on
    the stream, so that every launch finds what the one before it has just written.  The same bits as with launches one behind the other and a wait after each."""
    import torch
    import runit_mac_b200 as R
    case = THREE[name]
    b = Batch(5, poison=0.0, **case)
    rng = np.random.default_rng(17)
    row, width, steps, n_seqs = (b.heads + 2 * b.kv_heads) * b.dim, b.heads * b.dim, 12, len(b.seqs)
    most = np.array([n for _, n in b.seqs])
    lens = np.stack([rng.integers(b.shared + 1, most + 1) if s % 3 else most for s in range(steps)]).astype(np.int32)
    takes = np.stack([np.minimum([q if s % 2 else int(rng.integers(0, q + 1)) for q, _ in b.seqs], lens[s] - b.shared) for s in range(steps)])
    starts = np.concatenate([np.zeros((steps, 1), np.int64), np.cumsum(takes, 1)], 1).astype(np.int32)
    proj = torch.from_numpy(rng.normal(0, 1, (steps, 2, b.rows, row)).astype(np.float32)).cuda()
    lens_d, starts_d = torch.from_numpy(lens).cuda(), torch.from_numpy(starts).cuda()
    torch.cuda.synchronize()

    def serve(pdl, wait, record):
        side = torch.cuda.Stream()
        c = R.Context(0, stream=side.cuda_stream)
        try:
            c.set_tuning("pdl", pdl)
            layers = [b.upload(c) for _ in range(2)]
            for keep, cfg, batch in layers[1:]:                       # one batch, two layers' pages
                batch.table, batch.q_start, batch.kv_len = (layers[0][0][k].ptr for k in ("table", "q_start", "kv_len"))
            now_lens, now_starts, now_proj = torch.zeros(n_seqs, dtype=torch.int32, device="cuda"), torch.zeros(n_seqs + 1, dtype=torch.int32, device="cuda"), torch.zeros_like(proj[0])
            for _, _, batch in layers:
                batch.q_start, batch.kv_len = now_starts.data_ptr(), now_lens.data_ptr()
            n = R.paged_attention_scratch_bytes(c, layers[0][1], layers[0][2])
            scratch, freq = c.new_buffer(n), c.buffer_from(_frequencies(b.dim))
            q, out = (torch.zeros((2, b.rows, width), dtype=torch.int16, device="cuda") for _ in range(2))
            got = torch.zeros((steps, 2, b.rows, width), dtype=torch.int16, device="cuda")
            torch.cuda.synchronize()

            def step():
                for i, (keep, cfg, batch) in enumerate(layers):
                    R.paged_append(c, C.byref(cfg), C.byref(batch), now_proj[i], R.TYPE_F32, row, freq, b.dim, q[i], width)
                    R.paged_attention(c, C.byref(cfg), C.byref(batch), q[i], width, out[i], width, scratch, n)

            graph, before = None, c.launches
            if record:
                c.graph_begin()
                step()
                graph = c.graph_end()
                torch.cuda.synchronize()
            with torch.cuda.stream(side):
                for s in range(steps):
                    now_lens.copy_(lens_d[s])
                    now_starts.copy_(starts_d[s])
                    now_proj.copy_(proj[s])
                    graph.launch() if graph else step()
                    got[s].copy_(out)
                    if wait:
                        c.flush()
            c.flush()
            assert graph or c.launches - before == 8 * steps
            pages = [keep[k].download(np.uint16, b.k.size) for keep, _, _ in layers for k in ("k", "v")]
            result = got.cpu().numpy().view(np.uint16)
            if graph:
                graph.destroy()
            return result, pages
        finally:
            c.close()

    want, want_pages = serve(0, True, False)
    for _ in range(3):
        got, pages = serve(1, False, recorded)
        for s in range(steps):
            live = int(starts[s, -1])
            np.testing.assert_array_equal(got[s, :, :live], want[s, :, :live], err_msg="step %d" % s)
        for x, y in zip(pages, want_pages):
            np.testing.assert_array_equal(x, y)
