"""The operators over a paged cache as they are used: one behind the other with the framework's own products, in recorded lists, on other streams, side by
side, and with more sequences than fit a warp's plan."""
import ctypes as C

import numpy as np
import pytest

from paged_batches import EPS, Batch, check, from_bits, rounded, to_bits

pytestmark = pytest.mark.gpu


def _mixed(seed, n, most, shared=0, rows=lambda i: i % 2):
    rng = np.random.default_rng(seed)
    return [(rows(i), shared + rows(i) + int(rng.integers(0, most))) for i in range(n)]


MANY = {
    "half of them empty": dict(seqs=_mixed(1, 600, 150), heads=4, kv_heads=2, dim=64, page=16, kind="f16"),
    "nearly all empty": dict(seqs=_mixed(2, 1000, 90, rows=lambda i: int(i % 333 == 5)), heads=8, kv_heads=1, dim=128, page=32, kind="bf16", extra_rows=2),
    "one behind a warp's plan": dict(seqs=_mixed(3, 257, 60, rows=lambda i: 1), heads=2, kv_heads=2, dim=64, page=16, kind="bf16"),
    "with shared positions": dict(seqs=_mixed(4, 300, 40, 160, rows=lambda i: i % 3), heads=4, kv_heads=2, dim=64, page=16, kind="f16", shared=160),
    "shared by few rows": dict(seqs=_mixed(5, 400, 40, 96, rows=lambda i: int(i % 50 == 1)), heads=4, kv_heads=4, dim=64, page=16, kind="f16", shared=96, window=90),
    "prompts": dict(seqs=_mixed(6, 50, 100, rows=lambda i: 37 * i % 60), heads=8, kv_heads=2, dim=64, page=16, kind="bf16"),
    "prompts behind shared positions": dict(seqs=_mixed(7, 5, 50, 256, rows=lambda i: 13 + 40 * i), heads=4, kv_heads=1, dim=128, page=64, kind="f16", shared=256, extra_rows=1),
    "nobody has a row": dict(seqs=[(0, 40)] * 3, heads=4, kv_heads=2, dim=64, page=16, kind="f16", extra_rows=3),
    "nobody has a row behind shared positions": dict(seqs=[(0, 80)] * 3, heads=4, kv_heads=2, dim=64, page=16, kind="f16", shared=64, extra_rows=40),
}


@pytest.mark.parametrize("name", MANY)
def test_many_sequences(ctx, name):
    b = Batch(sum(map(ord, name)), **MANY[name])
    got = b.attend(ctx)
    assert (got[b.n_rows:] == rounded(-3.0, b.kind)).all()
    check(b, got, name)


BEHIND = {
    "single rows": dict(seqs=[(1, 512 + 1 + 11 * i % 60) for i in range(300)], heads=16, kv_heads=4, dim=64, page=16, kind="f16", shared=512),
    "drafts, cap, bias": dict(seqs=[(3, 512 + 3 + 7 * i % 50) for i in range(60)], heads=32, kv_heads=4, dim=128, page=64, kind="bf16", shared=512, cap=20.0, slopes=[0.1 / (i + 1) for i in range(32)]),
    "a window that reaches back": dict(seqs=[(1, 1024 + 9 * i % 500) for i in range(90)], heads=32, kv_heads=2, dim=64, page=32, kind="f16", shared=1024, window=700, extra_rows=2),
    "some end inside": dict(seqs=[(1, 1 + 37 * i % 511) if i % 3 == 0 else (i % 4, 512 + 5 * i % 90) for i in range(160)], heads=32, kv_heads=2, dim=128, page=128, kind="f16", shared=512),
}


@pytest.mark.parametrize("name", BEHIND)
def test_many_rows_behind_shared_positions(ctx, name):
    """Enough of both that the kernel for many rows takes the shared ones: three launches."""
    b = Batch(sum(map(ord, name)), **BEHIND[name])
    before = ctx.launches
    got = b.attend(ctx)
    assert ctx.launches - before == 3
    assert (got[b.n_rows:] == rounded(-3.0, b.kind)).all()
    check(b, got, name)


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_values_behind_shared_positions_that_a_row_does_not_see(ctx, value):
    """Rows that end inside the shared positions do not see what comes after them there; the others carry it."""
    b = Batch(3, [(1, 100 + i) if i % 2 else (1, 1024 + 1 + i % 30) for i in range(100)], 32, 2, 64, 16, "f16", shared=1024)
    clean, bound = b.reference()
    b.v[b.table[0, 300 // 16], 0, 300 % 16, 5] = value
    b.k[b.table[0, 400 // 16], 1, 400 % 16, 3] = np.nan
    before = ctx.launches
    got = b.attend(ctx)
    assert ctx.launches - before == 3
    for r, (_, n) in enumerate(b.seqs):
        for h in range(32):
            x, ref, off = got[r, h].astype(np.float64), clean[r, h], bound[r, h]
            if h // 16 == 1 and n > 400:
                assert np.isnan(x).all()
                continue
            if h // 16 == 0 and n > 300:
                assert not np.isfinite(x[5])
                x, ref, off = np.delete(x, 5), np.delete(ref, 5), np.delete(off, 5)
            assert (np.abs(x - ref) <= off + 2.0 ** -25).all(), (r, h)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("cap,scale", [(10.0, None), (10.0, -0.125), (1e-4, None), (1e7, None), (50.0, 3.0)])
def test_capped_scores_of_every_size(ctx, kind, rows, cap, scale):
    """Keys that are small at first, then large, then small again, so that scores over the cap reach from 0.01 to 30 within one row; caps far below and far above them."""
    b = Batch(rows, [(rows, 900)], 4, 2, 64, 32, kind, cap=cap, scale=scale)
    for p in range(900):
        b.k[b.table[0, p // 32], :, p % 32] *= 0.125 if p < 400 else 6.0 if 520 <= p < 530 else 1.0
    b.k = rounded(b.k, kind)
    check(b, b.attend(ctx))


@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("scale,slopes", [(0.0, None), (-0.2, None), (0.0, [0.3, -0.2, 0.0, 1.5])])
def test_scales_that_are_not_positive(ctx, rows, scale, slopes):
    """All scores alike (the mean of the values), the least product first, and a bias that alone decides."""
    b = Batch(rows, [(rows, 300), (1, 33)], 4, 2, 128, 16, "f16", scale=scale, slopes=slopes)
    check(b, b.attend(ctx))


def test_attention_does_not_write_over_its_queries(ctx):
    import runit_mac_b200 as R
    b = Batch(2, [(1, 20)], 4, 2, 64, 16, "f16")
    keep, cfg, batch = b.upload(ctx)
    n = R.paged_attention_scratch_bytes(ctx, cfg, batch)
    q, scratch, before = ctx.new_buffer(4096), ctx.new_buffer(n), ctx.launches
    with pytest.raises(R.KernelError) as e:
        R.paged_attention(ctx, C.byref(cfg), C.byref(batch), q, 256, q, 256, scratch, n)
    assert e.value.status == 2 and ctx.launches == before


def test_append_over_the_projected_queries(ctx):
    """Queries of the cache's type may go back to where they were: the same as to rows of their own."""
    import runit_mac_b200 as R
    b = Batch(3, [(40, 50), (1, 20)], 6, 2, 64, 16, "bf16", poison=1.0)
    row, freq = (6 + 4) * 64, 1e4 ** (-2.0 * np.arange(32) / 64)
    fb = ctx.buffer_from(np.stack([freq.astype(np.float32), (freq - freq.astype(np.float32)).astype(np.float32)]))
    proj = to_bits(np.random.default_rng(2).normal(0, 1, (b.rows, row)), "bf16")
    keep, cfg, batch = b.upload(ctx)
    p, q = ctx.buffer_from(proj), ctx.new_buffer(b.rows * 6 * 64 * 2)
    R.paged_append(ctx, C.byref(cfg), C.byref(batch), p, R.TYPE_BF16, row, fb, 64, q, 6 * 64)
    R.paged_append(ctx, C.byref(cfg), C.byref(batch), p, R.TYPE_BF16, row, fb, 64, p, row)
    ctx.flush()
    np.testing.assert_array_equal(p.download(np.uint16, b.rows * row).reshape(b.rows, row)[:, :6 * 64], q.download(np.uint16, b.rows * 6 * 64).reshape(b.rows, 6 * 64))


SOME = [dict(seqs=[(1, 700), (3, 40), (0, 0), (1, 5)], heads=14, kv_heads=2, dim=64, page=16, kind="f16"),
        dict(seqs=[(1, 320 + 9 * i) for i in range(30)], heads=8, kv_heads=2, dim=128, page=64, kind="bf16", shared=320),
        dict(seqs=[(150, 400), (130, 130)], heads=4, kv_heads=2, dim=128, page=32, kind="f16", cap=15.0)]


@pytest.mark.parametrize("case", range(len(SOME)))
def test_without_dependent_launches_and_on_another_stream(ctx, case):
    """The launches' order does not rest on how they are issued: the same bits one behind the other, and on a stream that the caller brings."""
    import torch
    import runit_mac_b200 as R
    b = Batch(21, **SOME[case])
    want = b.attend(ctx)
    check(b, want)
    side = torch.cuda.Stream()
    other = R.Context(0, stream=side.cuda_stream)
    try:
        other.set_tuning("pdl", 0)
        np.testing.assert_array_equal(want, b.attend(other))
        other.set_tuning("pdl", 2)
        np.testing.assert_array_equal(want, b.attend(other))
    finally:
        other.close()


def test_two_calls_at_once(ctx):
    """Two contexts, each with its stream and scratch, many calls in flight: what each gives alone."""
    import runit_mac_b200 as R
    other = R.Context(0)
    try:
        runs = []
        for c, b in ((ctx, Batch(1, **SOME[0])), (other, Batch(2, **SOME[1])), (other, Batch(3, **SOME[2]))):
            want = b.attend(c)
            keep, cfg, batch = b.upload(c)
            ld, n = b.heads * b.dim, R.paged_attention_scratch_bytes(c, cfg, batch)
            q, outs, scratch = c.buffer_from(to_bits(b.q, b.kind)), [c.new_buffer(b.rows * ld * 2) for _ in range(12)], c.new_buffer(n)
            runs.append((c, b, want, keep, cfg, batch, ld, n, q, outs, scratch))
        for i in range(12):
            for c, b, want, keep, cfg, batch, ld, n, q, outs, scratch in runs:
                R.paged_attention(c, C.byref(cfg), C.byref(batch), q, ld, outs[i], ld, scratch, n)
        ctx.flush()
        other.flush()
        for c, b, want, keep, cfg, batch, ld, n, q, outs, scratch in runs:
            for o in outs:
                np.testing.assert_array_equal(from_bits(o.download(np.uint16, b.rows * ld), b.kind).reshape(want.shape), want)
    finally:
        other.close()


def test_starts_that_do_not_rise_are_reported_by_the_append(ctx):
    """A row whose sequence ends before it belongs to nobody: nothing is written for it, and the pages' other rows stay."""
    import runit_mac_b200 as R
    for starts in ([0, 9, 2, 5], [0, 3, 9, 4], [0, 9, 9, 5], [3, 3, 6, 9]):
        b = Batch(3, [(3, 32), (3, 48), (3, 16)], 2, 1, 64, 16, "f16", poison=5.0, table_extra=0)
        b.q_start = np.array(starts, np.int32)
        keep, cfg, batch = b.upload(ctx)
        proj = ctx.buffer_from(np.random.default_rng(1).normal(0, 1, (9, 256)).astype(np.float32))
        R.paged_append(ctx, C.byref(cfg), C.byref(batch), proj, R.TYPE_F32, 256, None, 0, None, 0)
        with pytest.raises(R.KernelError) as e:
            ctx.flush()
        assert e.value.status == 2
        # pages that no sequence has are untouched
        k = from_bits(keep["k"].download(np.uint16, b.k.size), "f16").reshape(b.k.shape)
        free = sorted(set(range(b.n_pages)) - set(b.table[b.table >= 0].tolist()))
        np.testing.assert_array_equal(k[free], b.k[free])


# ── a serving step ──

WIDTH, HEADS, KV, DIM, PAGE, VOCAB, LAYERS = 256, 8, 2, 64, 16, 1500, 2
ROW, OUT = (HEADS + 2 * KV) * DIM, HEADS * DIM


class Server:
    """A small transformer's layers over the framework's operators: norm, one product for queries, keys and values, append, attention, product into the stream;
    norm, head, log probabilities.  All sizes are fixed; lengths, rows and tokens are device memory."""

    def __init__(self, ctx, n_seqs, rows, pages, shared=0):
        import runit_mac_b200 as R
        self.R, self.ctx, self.rows = R, ctx, rows
        rng = np.random.default_rng(77)
        bf = lambda a: to_bits(a, "bf16")
        self.embed = rng.normal(0, 1, (VOCAB, WIDTH)).astype(np.float32)
        self.w_qkv = [rounded(rng.normal(0, 1.5 / WIDTH ** 0.5, (ROW, WIDTH)), "bf16") for _ in range(LAYERS)]
        self.w_out = [rounded(rng.normal(0, 1 / OUT ** 0.5, (WIDTH, OUT)), "bf16") for _ in range(LAYERS)]
        self.w_head = rounded(rng.normal(0, 3 / WIDTH ** 0.5, (VOCAB, WIDTH)), "bf16")
        self.d = {"qkv": [ctx.buffer_from(bf(w)) for w in self.w_qkv], "out": [ctx.buffer_from(bf(w)) for w in self.w_out], "head": ctx.buffer_from(bf(self.w_head)),
                  "gain": ctx.buffer_from(np.ones(1, np.float32))}
        f = 1e4 ** (-2.0 * np.arange(DIM // 2) / DIM)
        self.freq = np.stack([f.astype(np.float32), (f - f.astype(np.float32)).astype(np.float32)])
        self.d["freq"] = ctx.buffer_from(self.freq)
        self.d["table"], self.d["q_start"], self.d["kv_len"] = ctx.buffer_from(pages), ctx.new_buffer(4 * (n_seqs + 1)), ctx.new_buffer(4 * n_seqs)
        n_pages = int(pages.max()) + 1
        shape = n_pages * KV * PAGE * DIM
        self.d["k"], self.d["v"] = ([ctx.buffer_from(np.zeros(shape, np.uint16)) for _ in range(LAYERS)] for _ in range(2))
        self.cfg = [R.PagedCfg(heads=HEADS, kv_heads=KV, dim=DIM, page=PAGE, n_pages=n_pages, type=R.TYPE_BF16, window=0, scale=DIM ** -0.5, cap=0.0, slopes=None,
                               k_pages=self.d["k"][i].ptr, v_pages=self.d["v"][i].ptr) for i in range(LAYERS)]
        self.batch = R.PagedBatch(n_seqs=n_seqs, rows=rows, table_ld=pages.shape[1], shared_len=shared, table=self.d["table"].ptr, q_start=self.d["q_start"].ptr,
                                  kv_len=self.d["kv_len"].ptr)
        new = ctx.new_buffer
        self.n = R.paged_attention_scratch_bytes(ctx, self.cfg[0], self.batch)
        self.b = {"x": new(rows * WIDTH * 4), "y": new(rows * WIDTH * 2), "proj": new(rows * ROW * 4), "q": new(rows * OUT * 2), "o": new(rows * OUT * 2),
                  "logits": new(rows * VOCAB * 4), "tokens": new(rows * 4), "lp": new(rows * 4), "h": new(rows * 4), "ids": new(rows * 5 * 4), "top": new(rows * 5 * 4),
                  "scratch": new(self.n)}
        self.b["o"].upload(np.zeros(rows * OUT, np.uint16))          # rows of nobody go through the products all the same
        self.b["q"].upload(np.zeros(rows * OUT, np.uint16))

    def place(self, starts, lens, ids, tokens):
        self.d["q_start"].upload(np.asarray(starts, np.int32))
        self.d["kv_len"].upload(np.asarray(lens, np.int32))
        self.x0 = np.zeros((self.rows, WIDTH), np.float32)
        self.x0[:len(ids)] = self.embed[ids]
        self.b["tokens"].upload(np.asarray(list(tokens) + [-1] * (self.rows - len(tokens)), np.int32))
        self.b["x"].upload(self.x0)

    def layer(self, i):
        R, c, b, d, T = self.R, self.ctx, self.b, self.d, self.rows
        R.norm_gain_rows(c, b["x"], d["gain"], 1e-5, b["y"], 0, T, WIDTH)
        R.gemm_bf16_rows(c, d["qkv"][i], b["y"], b["proj"], ROW, T, ROW, WIDTH, 0, 0, None, None)
        R.paged_append(c, C.byref(self.cfg[i]), C.byref(self.batch), b["proj"], R.TYPE_F32, ROW, d["freq"], DIM, b["q"], OUT)
        R.paged_attention(c, C.byref(self.cfg[i]), C.byref(self.batch), b["q"], OUT, b["o"], OUT, b["scratch"], self.n)
        R.gemm_bf16_rows(c, d["out"][i], b["o"], b["x"], WIDTH, T, WIDTH, OUT, 0, 1, None, None)

    def answer(self):
        R, c, b, d, T = self.R, self.ctx, self.b, self.d, self.rows
        R.norm_gain_rows(c, b["x"], d["gain"], 1e-5, b["y"], 0, T, WIDTH)
        R.gemm_bf16_rows(c, d["head"], b["y"], b["logits"], VOCAB, T, VOCAB, WIDTH, 0, 0, None, None)
        R.token_logprobs(c, b["logits"], R.TYPE_F32, VOCAB, VOCAB, T, b["tokens"], b["lp"], b["h"], 5, b["ids"], b["top"])

    def step(self):
        for i in range(LAYERS):
            self.layer(i)
        self.answer()

    def get(self, name, kind="f32"):
        w = {"x": WIDTH, "y": WIDTH, "proj": ROW, "q": OUT, "o": OUT, "logits": VOCAB, "lp": 1, "h": 1, "ids": 5, "top": 5}[name]
        t = {"f32": np.float32, "i32": np.int32, "bf16": np.uint16}[kind]
        a = self.b[name].download(t, self.rows * w)
        return (from_bits(a, "bf16") if kind == "bf16" else a).reshape(self.rows, w)


def _pages(n_seqs, each, seed):
    return np.random.default_rng(seed).permutation(n_seqs * each).reshape(n_seqs, each).astype(np.int32)


def test_a_serving_step_stage_by_stage(ctx):
    """Ragged prompts, then a token each: every stage against its definition in 64 bits over what the stage before it has left on the device."""
    starts, lens = [0, 7, 7, 40, 41], [7, 0, 33, 1]
    s = Server(ctx, 4, 44, _pages(4, 4, 1))
    rng = np.random.default_rng(5)
    n = np.array(lens)
    for turn in range(3):
        live = starts[-1]
        ids, tokens = rng.integers(0, VOCAB, live), rng.integers(0, VOCAB, live)
        s.place(starts, n, ids, tokens)
        for i in range(LAYERS):
            before = s.get("x").astype(np.float64)
            s.layer(i)
            ctx.flush()
            y, proj, q, o, x = s.get("y", "bf16").astype(np.float64), s.get("proj").astype(np.float64), s.get("q", "bf16"), s.get("o", "bf16").astype(np.float64), s.get("x")
            norm = before / np.sqrt((before ** 2).mean(1, keepdims=True) + 1e-5)
            assert (np.abs(y - norm) <= np.abs(norm) * (2.0 ** -8 + 2.0 ** -18) + 1e-30).all()
            w = s.w_qkv[i].astype(np.float64)
            assert (np.abs(proj - y @ w.T) <= WIDTH * 2.0 ** -24 * (np.abs(y) @ np.abs(w).T) + 1e-30).all()
            # the rotation, by each row's position
            pos = np.zeros(s.rows, np.int64)
            for k in range(4):
                pos[starts[k]:starts[k + 1]] = np.arange(n[k] - (starts[k + 1] - starts[k]), n[k])
            a = pos[:, None] * s.freq.astype(np.float64).sum(0)
            p = proj.reshape(s.rows, -1, DIM)
            lo, hi = p[:, :HEADS + KV, :32], p[:, :HEADS + KV, 32:]
            co, si = np.cos(a)[:, None], np.sin(a)[:, None]
            turned, size = np.concatenate([lo * co - hi * si, lo * si + hi * co], 2), np.tile(np.abs(lo) + np.abs(hi), 2)
            off = np.abs(q.reshape(s.rows, HEADS, DIM) - turned[:, :HEADS]) - (EPS["bf16"] / 2 * np.abs(turned[:, :HEADS]) + 2.0 ** -21 * size[:, :HEADS])
            assert (off[:live] <= 0).all()
            # attention over the pages as they are, keys of this step among them
            b = Batch(0, [(starts[k + 1] - starts[k], int(n[k])) for k in range(4)], HEADS, KV, DIM, PAGE, "bf16", extra_rows=s.rows - live, poison=0.0)
            shape = (s.cfg[i].n_pages, KV, PAGE, DIM)
            b.k, b.v = (from_bits(s.d[t][i].download(np.uint16, int(np.prod(shape))), "bf16").reshape(shape) for t in ("k", "v"))
            b.table, b.q = _pages(4, 4, 1), q.reshape(s.rows, HEADS, DIM)
            check(b, o.reshape(s.rows, HEADS, DIM).astype(np.float32), "turn %d layer %d" % (turn, i))
            for k in range(4):
                for r in range(starts[k], starts[k + 1]):
                    pg = b.table[k, pos[r] // PAGE]
                    np.testing.assert_array_equal(b.v[pg, :, pos[r] % PAGE], rounded(p[r, HEADS + KV:], "bf16"))
            w = s.w_out[i].astype(np.float64)
            want = before + o @ w.T
            assert (np.abs(x - want) <= OUT * 2.0 ** -24 * (np.abs(o) @ np.abs(w).T) + 2.0 ** -24 * np.abs(want) + 2.0 ** -24 * np.abs(before) + 1e-30).all()
        s.answer()
        ctx.flush()
        z = s.get("logits").astype(np.float64)[:live]
        lp = z - z.max(1, keepdims=True)
        lp = lp - np.log(np.exp(lp).sum(1, keepdims=True))
        got = s.get("lp")[:, 0]
        assert (got[live:] == 0).all()
        want = lp[np.arange(live), tokens]
        assert (np.abs(got[:live] - want) <= 2.0 ** -15 + np.abs(want) * 2.0 ** -22).all()
        order = np.argsort(-s.get("logits")[:live], 1, kind="stable")[:, :5]
        np.testing.assert_array_equal(s.get("ids", "i32")[:live], order)
        # from here on one token for each of those that have begun
        starts = [0, 1, 1, 2, 3]
        n = n + np.array([1, 0, 1, 1])


def test_a_recorded_serving_step(ctx):
    """One recording serves every step: prompts of any split, then single tokens.  The same bits as the calls themselves, and what stands in the cache afterwards
    does not depend on how the tokens were split over steps by more than their products' order of summation."""
    def serve(run, s, split):
        rng = np.random.default_rng(12)
        ids = rng.integers(0, VOCAB, (3, 60))
        n, out = np.zeros(3, np.int64), {}
        for take in split:
            starts = np.concatenate([[0], np.cumsum(take)])
            n = n + take
            rows = np.concatenate([ids[k, n[k] - take[k]:n[k]] for k in range(3)])
            nxt = np.concatenate([ids[k, n[k] - take[k] + 1:n[k] + 1] for k in range(3)])
            s.place(starts, n, rows, nxt)
            run(s)
            ctx.flush()
            lp = s.get("lp")[:, 0]
            for k in range(3):
                for i in range(take[k]):
                    out[k, int(n[k]) - take[k] + i] = lp[starts[k] + i]
        return out

    split = [(20, 1, 12), (1, 1, 1), (0, 14, 1), (1, 0, 1), (10, 6, 3)]
    made = [Server(ctx, 3, 36, _pages(3, 4, 2)) for _ in range(2)]
    plain = serve(Server.step, made[0], split)
    ctx.graph_begin()
    made[1].step()
    graph = ctx.graph_end()
    recorded = serve(lambda s: graph.launch(), made[1], split)
    assert plain == recorded and len(plain) == sum(map(sum, split))
    graph.destroy()
    # one token at a time: another order of the same sums.  Rounded to bf16 on the way (queries, keys, weights, outputs, norms: 2^-9 of each on average, 2 layers, logits
    # of some 3), the log probabilities of two such runs agree to some 2^-9 x sqrt(12) x 3 = 0.02; a wrong position or page moves them by 1 and more.
    single = serve(Server.step, Server(ctx, 3, 36, _pages(3, 4, 2)), [(1, 1, 1)] * 22 + [(1, 0, 0)] * 10)
    both = [p for p in plain if p in single]
    assert len(both) >= 60
    assert max(abs(plain[p] - single[p]) for p in both) <= 0.2
