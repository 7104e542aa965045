"""The paged cache on the device: rows appended with their rotation, and the attention that reads them, against the definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from paged_batches import EPS, Batch, check, from_bits, rounded, to_bits

pytestmark = pytest.mark.gpu


# ── append ──

def _append(ctx, b, proj, kind, rot, freq, pad=0, with_q=True, q_fill=-3.0):
    import runit_mac_b200 as R
    keep, cfg, batch = b.upload(ctx)
    width, row = b.heads * b.dim, (b.heads + 2 * b.kv_heads) * b.dim
    x = np.full((b.rows, row + pad), 77.0, np.float32)
    x[:, :row] = proj
    pb = ctx.buffer_from(x if kind == "f32" else to_bits(x, kind))
    qb = ctx.buffer_from(to_bits(np.full((b.rows, width + pad), q_fill), b.kind)) if with_q else None
    fb = ctx.buffer_from(freq) if rot else None
    t = {"f32": R.TYPE_F32, "f16": R.TYPE_F16, "bf16": R.TYPE_BF16}[kind]
    R.paged_append(ctx, C.byref(cfg), C.byref(batch), pb, t, row + pad, fb, rot, qb, width + pad)
    ctx.flush()
    q = None
    if with_q:
        q = from_bits(qb.download(np.uint16, b.rows * (width + pad)), b.kind).reshape(b.rows, width + pad)
        assert (q[:, width:] == rounded(q_fill, b.kind)).all()
        q = q[:, :width].reshape(b.rows, b.heads, b.dim)
    return q, *(from_bits(keep[n].download(np.uint16, b.k.size), b.kind).reshape(b.k.shape) for n in ("k", "v"))


def _frequencies(rot, base=1e6):
    f = base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    hi = f.astype(np.float32)
    return np.stack([hi, (f - hi).astype(np.float32)])


APPEND = [
    # rows and lengths, heads, key heads, dim, page, type of the projection, of the cache, rotated, stride beyond the row
    ([(1, 1)], 1, 1, 64, 16, "f32", "f16", 64, 0),
    ([(1, 131072)], 28, 4, 128, 16, "f32", "f16", 128, 0),
    ([(1, 1000003)], 4, 1, 128, 256, "f32", "bf16", 128, 0),
    ([(3, 17), (0, 5), (1, 16), (20, 33)], 14, 2, 64, 16, "bf16", "bf16", 64, 8),
    ([(65, 130), (64, 64)], 16, 16, 128, 64, "f16", "f16", 64, 16),
    ([(5, 40)], 6, 3, 64, 32, "f32", "bf16", 24, 4),
    ([(5, 40)], 6, 3, 64, 32, "f32", "bf16", 32, 3),
    ([(2, 9), (2, 300)], 8, 1, 128, 128, "bf16", "bf16", 2, 1),
    ([(7, 70)], 12, 12, 64, 64, "f16", "f16", 0, 0),
    ([(1, 5 + i) for i in range(300)], 4, 2, 64, 16, "f32", "f16", 64, 0),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(ctx, case):
    """Bound: cos and sin within 2^-22 of the true ones (angle to 2^-24 of a turn's share after the correction, functions to two units), products and
    their sum in f32, one rounding to the type."""
    seqs, heads, kvh, dim, page, kind, cache, rot, pad = APPEND[case]
    long = max(n for _, n in seqs)
    b = Batch(case + 1, seqs, heads, kvh, dim, page, cache, extra_rows=2, spare_pages=2, poison=5.0) if long < 5000 else _far(case + 1, seqs, heads, kvh, dim, page, cache)
    rng = np.random.default_rng(case)
    proj = rounded(rng.normal(0, 2, (b.rows, (heads + 2 * kvh) * dim)), kind)
    freq = _frequencies(rot)
    q, k, v = _append(ctx, b, proj, kind, rot, freq, pad)
    want_k, want_v, want_q = b.k.astype(np.float64), b.v.astype(np.float64), np.full((b.rows, heads, dim), -3.0)
    scale_k, scale_q = np.zeros_like(want_k), np.zeros_like(want_q)
    h = rot // 2
    x = proj.reshape(b.rows, heads + 2 * kvh, dim).astype(np.float64)
    for s, (nq, n) in enumerate(seqs):
        for i in range(nq):
            r, p = int(b.q_start[s]) + i, n - nq + i
            a = p * (freq[0].astype(np.float64) + freq[1].astype(np.float64))
            y, size = x[r].copy(), np.abs(x[r])
            lo, hi = x[r, :heads + kvh, :h], x[r, :heads + kvh, h:2 * h]
            y[:heads + kvh, :h], y[:heads + kvh, h:2 * h] = lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a)
            size[:heads + kvh, :h] = size[:heads + kvh, h:2 * h] = np.abs(lo) + np.abs(hi)
            want_q[r], scale_q[r] = y[:heads], size[:heads]
            pg = b.table[s, p // page]
            want_k[pg, :, p % page], scale_k[pg, :, p % page] = y[heads:heads + kvh], size[heads:heads + kvh]
            want_v[pg, :, p % page] = y[heads + kvh:]
    half = EPS[cache] / 2
    with np.errstate(over="ignore"):
        assert (np.abs(q - want_q) <= half * np.abs(want_q) + 2.0 ** -21 * scale_q + 2.0 ** -25).all()
        assert (np.abs(k - want_k) <= half * np.abs(want_k) + 2.0 ** -21 * scale_k + 2.0 ** -25).all()
    np.testing.assert_array_equal(v, rounded(want_v, cache))
    # no rotation: copies, to the bit
    if rot == 0:
        np.testing.assert_array_equal(q, rounded(want_q, cache))
    # keys and values alone: the same
    _, k2, v2 = _append(ctx, b, proj, kind, rot, freq, pad, with_q=False)
    np.testing.assert_array_equal(k, k2)
    np.testing.assert_array_equal(v, v2)


def _far(seed, seqs, heads, kvh, dim, page, kind):
    """One row far out: only the page of that position is real."""
    (nq, n), = seqs
    b = Batch(seed, [(nq, (n - 1) % page + 1)], heads, kvh, dim, page, kind, extra_rows=2, poison=5.0, table_extra=0)
    table = np.full((1, -(-n // page)), -7, np.int32)
    table[0, (n - 1) // page] = b.table[0, 0]
    b.table, b.table_ld, b.seqs, b.kv_len = table, table.shape[1], seqs, np.array([n], np.int32)
    return b


def test_append_reports_what_the_cache_does_not_hold(ctx):
    """A page outside the pool, a length beyond the table, a length shorter than the rows: reported, nothing written there, the rest done."""
    import runit_mac_b200 as R
    for what in ("page", "negative page", "length", "short", "starts"):
        b = Batch(3, [(1, 20), (2, 30), (1, 9)], 4, 2, 64, 16, "f16", poison=5.0)
        rng = np.random.default_rng(5)
        proj = rng.normal(0, 1, (b.rows, 8 * 64)).astype(np.float32)
        _, good_k, _ = _append(ctx, b, proj, "f32", 0, None)
        place = b.table[1, 1], slice(12, 14)                        # rows 1 and 2: positions 28 and 29 of sequence 1
        if what == "page":
            b.table[1, 1] = b.n_pages
        elif what == "negative page":
            b.table[1, 1] = -1
        elif what == "length":
            b.kv_len[1] = b.table_ld * 16 + 1
        elif what == "short":
            b.kv_len[1] = 1
        else:
            b.q_start[2] = 900
        with pytest.raises(R.KernelError) as e:
            _append(ctx, b, proj, "f32", 0, None)
        assert e.value.status == 2 and "paged cache" in str(e.value)
        ctx.flush()                                                  # told once
        if what in ("page", "negative page"):
            keep, cfg, batch = b.upload(ctx)
            R.paged_append(ctx, C.byref(cfg), C.byref(batch), ctx.buffer_from(proj), R.TYPE_F32, 512, None, 0, None, 0)
            with pytest.raises(R.KernelError):
                ctx.flush()
            k = from_bits(keep["k"].download(np.uint16, b.k.size), "f16").reshape(b.k.shape)
            want = good_k.copy()
            want[place[0], :, place[1]] = b.k[place[0], :, place[1]]
            np.testing.assert_array_equal(k, want)


# ── attention ──

def _alibi(heads):
    return [2.0 ** (-8 * (i + 1) / heads) for i in range(heads)]


ATTENTION = {
    "one key": dict(seqs=[(1, 1)], heads=1, kv_heads=1, dim=64, page=16, kind="f16"),
    "small model": dict(seqs=[(1, 777)], heads=14, kv_heads=2, dim=64, page=16, kind="bf16"),
    "lengths around a page": dict(seqs=[(1, n) for n in (1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65)], heads=8, kv_heads=4, dim=128, page=16, kind="f16"),
    "lengths around a tile": dict(seqs=[(1, n) for n in (127, 128, 129, 255, 256, 257, 500, 3)], heads=7, kv_heads=1, dim=128, page=64, kind="bf16"),
    "empty sequences": dict(seqs=[(0, 0), (1, 40), (0, 17), (0, 0), (1, 5), (0, 3)], heads=4, kv_heads=4, dim=64, page=32, kind="f16", extra_rows=5),
    "a row before the sequence": dict(seqs=[(1, 50)], heads=4, kv_heads=1, dim=64, page=16, kind="f16", extra_rows=1),
    "many query heads per key head": dict(seqs=[(1, 70), (1, 200)], heads=24, kv_heads=1, dim=64, page=16, kind="bf16"),
    "more heads than a tile": dict(seqs=[(1, 70), (2, 41)], heads=160, kv_heads=1, dim=64, page=16, kind="f16"),
    "odd group": dict(seqs=[(1, 130), (1, 61), (3, 90)], heads=15, kv_heads=3, dim=128, page=16, kind="f16"),
    "drafts": dict(seqs=[(4, 300), (1, 4), (4, 4), (3, 77)], heads=28, kv_heads=4, dim=128, page=32, kind="bf16"),
    "window 1": dict(seqs=[(1, 90), (3, 64), (2, 2)], heads=8, kv_heads=2, dim=64, page=16, kind="f16", window=1),
    "window 17": dict(seqs=[(1, 90), (30, 64), (2, 2), (1, 17), (1, 18)], heads=8, kv_heads=2, dim=64, page=16, kind="f16", window=17),
    "window 100, bias": dict(seqs=[(1, 333), (9, 128), (150, 300)], heads=8, kv_heads=2, dim=128, page=64, kind="bf16", window=100, slopes=_alibi(8)),
    "cap": dict(seqs=[(1, 200), (5, 60)], heads=12, kv_heads=12, dim=64, page=128, kind="f16", cap=30.0),
    "small cap": dict(seqs=[(1, 200), (70, 160)], heads=4, kv_heads=2, dim=128, page=32, kind="bf16", cap=0.75),
    "large scores": dict(seqs=[(1, 300), (40, 170)], heads=4, kv_heads=2, dim=64, page=32, kind="f16", scale=4.0),
    "prompt": dict(seqs=[(200, 200)], heads=4, kv_heads=2, dim=64, page=16, kind="f16"),
    "prompts behind a cache": dict(seqs=[(129, 400), (1, 1), (128, 128), (127, 300), (1, 500)], heads=2, kv_heads=1, dim=128, page=64, kind="bf16"),
    "prompt, pages of 256": dict(seqs=[(300, 310)], heads=2, kv_heads=2, dim=128, page=256, kind="f16"),
    "prompt, odd group, bias": dict(seqs=[(90, 111), (33, 33)], heads=7, kv_heads=1, dim=64, page=16, kind="bf16", slopes=_alibi(7), cap=20.0),
    "shared, few rows": dict(seqs=[(1, 70), (1, 100), (1, 65)], heads=4, kv_heads=2, dim=64, page=16, kind="f16", shared=64),
    "shared, many rows": dict(seqs=[(1, 512 + 1 + 7 * i % 60) for i in range(40)], heads=14, kv_heads=2, dim=64, page=32, kind="bf16", shared=512),
    "shared, many rows, 128": dict(seqs=[(1, 320 + 1 + 11 * i % 90) for i in range(37)], heads=28, kv_heads=4, dim=128, page=64, kind="f16", shared=320, extra_rows=3),
    "shared, drafts, bias, cap": dict(seqs=[(3, 160 + 3 + 5 * i % 40) for i in range(30)], heads=8, kv_heads=2, dim=128, page=16, kind="bf16", shared=160, slopes=_alibi(8), cap=25.0),
    "shared, window reaches back": dict(seqs=[(1, 260 + 9 * i % 70) for i in range(33)], heads=8, kv_heads=2, dim=64, page=16, kind="f16", shared=256, window=50),
    "shared, some end inside": dict(seqs=[(1, 10), (1, 200), (2, 128), (1, 127), (20, 120), (1, 129), (0, 0), (1, 300)], heads=16, kv_heads=2, dim=64, page=16, kind="f16", shared=128),
    "shared, long": dict(seqs=[(1, 4096 + 1 + 13 * i % 200) for i in range(16)], heads=16, kv_heads=1, dim=128, page=128, kind="bf16", shared=4096),
    "shared, whole lengths": dict(seqs=[(1, 256)] * 20, heads=8, kv_heads=1, dim=64, page=16, kind="f16", shared=256),
    "many sequences": dict(seqs=[(1, 1 + 37 * i % 210) for i in range(200)], heads=8, kv_heads=2, dim=64, page=16, kind="bf16"),
    "long": dict(seqs=[(1, 20000)], heads=4, kv_heads=2, dim=64, page=64, kind="f16"),
}


@pytest.mark.parametrize("name", ATTENTION)
def test_attention(ctx, name):
    b = Batch(sum(map(ord, name)), **ATTENTION[name])
    got = b.attend(ctx)
    assert (got[b.n_rows:] == rounded(-3.0, b.kind)).all()           # nobody's rows
    check(b, got, name)


@pytest.mark.parametrize("name", ["small model", "drafts", "prompts behind a cache", "shared, many rows, 128"])
def test_attention_of_strided_rows(ctx, name):
    b = Batch(11, **ATTENTION[name])
    wide = b.attend(ctx, pad=24)
    np.testing.assert_array_equal(wide, b.attend(ctx))
    np.testing.assert_array_equal(wide, b.attend(ctx))               # the same bits each time


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("seqs,shared,window", [([(4, 61), (2, 9)], 0, 0), ([(140, 300)], 0, 0), ([(1, 96 + 2 + i) for i in range(40)], 96, 0), ([(40, 100)], 0, 20), ([(1, 150)], 0, 33)])
@pytest.mark.parametrize("kind,dim", [("f16", 64), ("bf16", 128)])
def test_values_that_a_row_does_not_see(ctx, value, seqs, shared, window, kind, dim):
    """A key and a value that are no numbers, at the last position and at one in the middle of each sequence: rows that see the position carry it, the
    others stay as the formula has them."""
    b = Batch(9, seqs, 8, 2, dim, 16, kind, shared=shared, window=window)
    clean, bound = b.reference()
    spots = []
    for s, (nq, n) in enumerate(seqs):
        for p in {n - 1, max(n - nq - 1, shared), max(n // 2, shared)}:
            if p < n:
                pg = b.table[s, p // 16]
                b.v[pg, 0, p % 16, 5] = value
                b.k[pg, 1, p % 16, 3] = np.nan                       # a score that is no number: the whole row, where it is seen
                spots.append((s, p))
    got = b.attend(ctx)[:b.n_rows]
    g = b.heads // b.kv_heads
    for s, (nq, n) in enumerate(seqs):
        for i in range(nq):
            r, p = int(b.q_start[s]) + i, n - nq + i
            seen = any(t == s and at <= p and (not window or p - at < window) for t, at in spots)
            for h in range(b.heads):
                x = got[r, h].astype(np.float64)
                if seen and h // g == 1:
                    assert np.isnan(x).all(), (r, h)
                    continue
                if seen:
                    assert not np.isfinite(x[5]), (r, h)
                    x = np.delete(x, 5)
                    ref, off = np.delete(clean[r, h], 5), np.delete(bound[r, h], 5)
                else:
                    ref, off = clean[r, h], bound[r, h]
                assert (np.abs(x - ref) <= off + 2.0 ** -25).all(), (r, h)


def test_a_row_that_sees_nothing_is_zero(ctx):
    """Lengths shorter than the rows are reported; rows in front of position 0 come out as zeros, the others as they should."""
    import runit_mac_b200 as R
    b = Batch(4, [(1, 30), (5, 5), (1, 12)], 4, 2, 64, 16, "f16")
    good = b.attend(ctx)
    b.kv_len[1] = 3
    keep, cfg, batch = b.upload(ctx)
    q, out = ctx.buffer_from(to_bits(b.q, "f16")), ctx.buffer_from(to_bits(np.full_like(b.q, 8.0), "f16"))
    n = R.paged_attention_scratch_bytes(ctx, cfg, batch)
    R.paged_attention(ctx, C.byref(cfg), C.byref(batch), q, 256, out, 256, ctx.new_buffer(n), n)
    with pytest.raises(R.KernelError) as e:
        ctx.flush()
    assert e.value.status == 2
    got = from_bits(out.download(np.uint16, b.q.size), "f16").reshape(b.q.shape)
    assert (got[1:3] == 0).all() and np.isfinite(got).all()
    np.testing.assert_array_equal(got[[0, 6]], good[[0, 6]])


@pytest.mark.parametrize("what", ["page", "negative page", "length", "starts", "shared page"])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_reports_what_the_cache_does_not_hold(ctx, what, rows):
    import runit_mac_b200 as R
    b = Batch(6, [(rows, 90), (rows, 200), (1, 70)], 4, 2, 64, 16, "bf16", shared=64, poison=1.0)
    if what == "page":
        b.table[1, 5] = b.n_pages
    elif what == "negative page":
        b.table[1, 7] = -2
    elif what == "length":
        b.kv_len[1] = b.table_ld * 16 + 5
    elif what == "starts":
        b.q_start[1:3] = [5000, 2]
    else:
        b.table[0, 2] = 1 << 30
    with pytest.raises(R.KernelError) as e:
        b.attend(ctx)
    assert e.value.status == 2 and "paged cache" in str(e.value)
    ctx.flush()
    c = Batch(6, [(rows, 90), (rows, 200), (1, 70)], 4, 2, 64, 16, "bf16", shared=64)
    check(c, c.attend(ctx), "afterwards")


@pytest.mark.parametrize("shared", [0, 64])
def test_a_recorded_step_serves_other_lengths(ctx, shared):
    """One recording of append and attention; lengths, pages and rows change in device memory between its replays.  Two recordings that share their
    scratch give the same when they are replayed in turn."""
    import runit_mac_b200 as R
    heads, kvh, dim, page = 8, 2, 64, 16
    base = Batch(1, [(1, 250)] * 6, heads, kvh, dim, page, "f16", shared=shared, poison=1.0)
    keep, cfg, batch = base.upload(ctx)
    row = (heads + 2 * kvh) * dim
    proj, q, out = ctx.new_buffer(6 * row * 4), ctx.new_buffer(6 * heads * dim * 2), ctx.new_buffer(6 * heads * dim * 2)
    n = R.paged_attention_scratch_bytes(ctx, cfg, batch)
    scratch, freq = ctx.new_buffer(n), ctx.buffer_from(_frequencies(dim))

    def step():
        R.paged_append(ctx, C.byref(cfg), C.byref(batch), proj, R.TYPE_F32, row, freq, dim, q, heads * dim)
        R.paged_attention(ctx, C.byref(cfg), C.byref(batch), q, heads * dim, out, heads * dim, scratch, n)

    graphs = []
    for _ in range(2):
        ctx.graph_begin()
        step()
        graphs.append(ctx.graph_end())
    rng = np.random.default_rng(8)
    for turn in range(4):
        lens = rng.integers(max(shared, 1) + 1, 250, 6).astype(np.int32)
        starts = np.array([0, 1, 2, 2, 3, 5, 6] if turn % 2 else range(7), np.int32)
        keep["kv_len"].upload(lens)
        keep["q_start"].upload(starts)
        proj.upload(rng.normal(0, 1, (6, row)).astype(np.float32))
        results = []
        for run in (graphs[0].launch, graphs[1].launch, step):
            run()
            ctx.flush()
            results.append(out.download(np.uint16, 6 * heads * dim))
        np.testing.assert_array_equal(results[0], results[1])
        np.testing.assert_array_equal(results[0], results[2])
        # the definition, on what the append has left in the pages
        b = Batch(1, [(1, 250)] * 6, heads, kvh, dim, page, "f16", shared=shared, poison=1.0)
        b.k, b.v = (from_bits(keep[x].download(np.uint16, b.k.size), "f16").reshape(b.k.shape) for x in ("k", "v"))
        b.kv_len, b.q_start = lens, starts
        b.seqs = [(int(starts[i + 1] - starts[i]), int(lens[i])) for i in range(6)]
        b.q = from_bits(q.download(np.uint16, 6 * heads * dim), "f16").reshape(6, heads, dim)
        check(b, from_bits(results[0], "f16").reshape(6, heads, dim), "turn %d" % turn)
    for g in graphs:
        g.destroy()


def test_refusals(ctx):
    """A bad description or tensor launches nothing and says why."""
    import runit_mac_b200 as R
    b = Batch(2, [(1, 20)], 4, 2, 64, 16, "f16")
    keep, cfg, batch = b.upload(ctx)
    q, out, proj, freq = ctx.new_buffer(4096), ctx.new_buffer(4096), ctx.new_buffer(8192), ctx.buffer_from(_frequencies(64))
    n = R.paged_attention_scratch_bytes(ctx, cfg, batch)
    scratch = ctx.new_buffer(n)
    before = ctx.launches

    def refused(f, status=2, **change):
        saved = {k: (t, getattr(t, k)) for k in change for t in (cfg, batch) if hasattr(t, k)}
        for k, (t, _) in saved.items():
            setattr(t, k, change[k])
        with pytest.raises(R.KernelError) as e:
            f()
        assert e.value.status == status, (change, str(e.value))
        for k, (t, v) in saved.items():
            setattr(t, k, v)

    def attention(q=q, ldq=256, out=out, ldo=256, scratch=scratch, n=n):
        R.paged_attention(ctx, C.byref(cfg), C.byref(batch), q, ldq, out, ldo, scratch, n)

    def append(proj=proj, kind=R.TYPE_F32, ld=512, freq=freq, rot=64, q=q, ldq=256):
        R.paged_append(ctx, C.byref(cfg), C.byref(batch), proj, kind, ld, freq, rot, q, ldq)

    for f in (attention, append):
        for change in (dict(heads=0), dict(heads=5), dict(kv_heads=0), dict(dim=96), dict(page=24), dict(page=8), dict(page=512), dict(n_pages=0), dict(n_pages=1 << 31),
                       dict(type=0), dict(type=3), dict(scale=float("nan")), dict(cap=-1.0), dict(cap=float("inf")), dict(n_seqs=0), dict(n_seqs=4097), dict(rows=0),
                       dict(rows=1 << 30), dict(table_ld=0), dict(table_ld=1 << 28), dict(shared_len=8), dict(shared_len=16 * 64), dict(k_pages=None), dict(v_pages=None),
                       dict(k_pages=keep["k"].ptr + 64), dict(table=None), dict(table=keep["table"].ptr + 2), dict(q_start=None), dict(kv_len=None)):
            refused(f, **change)
    for a in (dict(q=None), dict(out=None), dict(q=q.ptr + 8), dict(out=out.ptr + 2), dict(ldq=255), dict(ldo=248), dict(ldq=0), dict(scratch=None), dict(scratch=scratch.ptr + 128)):
        refused(lambda: attention(**a))
    refused(lambda: attention(n=n - 1), status=3)
    for a in (dict(proj=None), dict(proj=proj.ptr + 2), dict(kind=R.TYPE_BF16), dict(kind=7), dict(ld=511), dict(freq=None), dict(rot=63), dict(rot=66), dict(ldq=255), dict(q=q.ptr + 1)):
        refused(lambda: append(**a))
    with pytest.raises(R.KernelError):
        R.paged_attention(ctx, None, C.byref(batch), q, 256, out, 256, scratch, n)
    with pytest.raises(R.KernelError):
        R.paged_append(ctx, C.byref(cfg), None, proj, R.TYPE_F32, 512, freq, 64, q, 256)
    assert ctx.launches == before
    attention()
    append()
    ctx.flush()
