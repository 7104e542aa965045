"""Log probabilities, entropy and alternatives of rows of logits against the definitions in 64 bits."""
import numpy as np
import pytest

from paged_batches import from_bits, rounded, to_bits

pytestmark = pytest.mark.gpu


def _run(ctx, x, kind, tokens, k, pad=0, entropy=True, at=0):
    import runit_mac_b200 as R
    rows, n = x.shape
    wide = np.full((rows, n + pad), 1e4, np.float32)
    wide[:, :n] = x
    bits = wide.reshape(-1) if kind == "f32" else to_bits(wide, kind).reshape(-1)
    buf = ctx.buffer_from(np.concatenate([np.zeros(at, bits.dtype), bits]))
    t = {"f32": R.TYPE_F32, "f16": R.TYPE_F16, "bf16": R.TYPE_BF16}[kind]
    tb = None if tokens is None else ctx.buffer_from(np.asarray(tokens, np.int32))
    lb = None if tokens is None else ctx.new_buffer(rows * 4)
    eb = ctx.new_buffer(rows * 4) if entropy else None
    ib, vb = (ctx.new_buffer(rows * k * 4), ctx.new_buffer(rows * k * 4)) if k else (None, None)
    R.token_logprobs(ctx, buf.ptr + at * bits.itemsize, t, n + pad, n, rows, tb, lb, eb, k, ib, vb)
    ctx.flush()
    return (None if lb is None else lb.download(np.float32, rows), eb.download(np.float32, rows) if entropy else None,
            ib.download(np.int32, rows * k).reshape(rows, k) if k else None, vb.download(np.float32, rows * k).reshape(rows, k) if k else None)


def _check(x, tokens, k, got):
    """Bound: d = x - m is off by 2^-24 |d|, an exponential by 2^-22 plus what its argument is off by (2^-23 |d|), their f32 sum by 2^-16 of it in the
    worst case (chains of at most 256 terms a thread): log Z by 2^-15, a log probability by that and the rounding of its own magnitude."""
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        d = x - m
        e = np.exp(d)
        z = e.sum(1, keepdims=True)
        lp = d - np.log(z)
        h = (np.log(z) - (e * np.where(e > 0, d, 0)).sum(1, keepdims=True) / z)[:, 0]
    logprob, entropy, ids, top = got
    for r in range(len(x)):
        if logprob is not None:
            t = int(tokens[r])
            want = lp[r, t] if 0 <= t < x.shape[1] else 0.0
            assert logprob[r] == want or abs(logprob[r] - want) <= 2.0 ** -15 + abs(want) * 2.0 ** -22, (r, logprob[r], want)
        if entropy is not None:
            mass = (e[r] * -np.where(e[r] > 0, d[r], 0)).sum() / z[r, 0]
            assert abs(entropy[r] - h[r]) <= min(1.0, 4 * np.log(z[r, 0]) + 4 * mass) * 2.0 ** -14 + h[r] * 2.0 ** -16 + 2.0 ** -23, (r, entropy[r], h[r])
        if k:
            want = np.argsort(-x[r], kind="stable")[:k]
            np.testing.assert_array_equal(ids[r], want)
            w = lp[r, want]
            some = np.isfinite(w)
            np.testing.assert_array_equal(top[r][~some], w[~some])
            assert (np.abs(top[r][some] - w[some]) <= 2.0 ** -15 + np.abs(w[some]) * 2.0 ** -22).all(), r


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,k,pad,at", [(1, 1, 1, 0, 0), (3, 2, 2, 1, 0), (2, 31, 31, 0, 0), (5, 33, 32, 3, 1), (4, 255, 7, 0, 3), (1, 1000, 20, 0, 0), (2, 4097, 5, 5, 2),
                                             (7, 32000, 1, 0, 0), (300, 999, 3, 1, 0), (1, 50304, 32, 0, 0), (8, 151936, 20, 0, 0), (3, 152065, 32, 7, 1), (700, 2048, 0, 0, 0),
                                             (160, 20000, 9, 0, 0)])
def test_rows(ctx, kind, rows, n, k, pad, at):
    rng = np.random.default_rng(rows * 7 + n)
    x = rng.normal(0, 3, (rows, n))
    x[0] *= 4
    x = rounded(x, kind)
    tokens = rng.integers(0, n, rows)
    _check(x, tokens, k, _run(ctx, x, kind, tokens, k, pad, at=at))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 5000, 60000])
def test_order_of_equal_logits(ctx, kind, n):
    """Ties go to the lowest index: few distinct values, zeros of either sign, a row of one value, ascending and descending rows."""
    rng = np.random.default_rng(n)
    x = np.stack([rng.integers(-2, 3, n).astype(np.float32), np.zeros(n, np.float32), np.where(rng.random(n) < 0.5, -0.0, 0.0).astype(np.float32),
                  np.linspace(-9, 9, n).astype(np.float32), np.linspace(9, -9, n).astype(np.float32), np.full(n, -1e30, np.float32)])
    x = rounded(x, kind)
    tokens = rng.integers(0, n, len(x))
    _check(x, tokens, 32, _run(ctx, x, kind, tokens, 32))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [64, 30000])
def test_masked_entries(ctx, kind, n):
    """-Inf entries (and the type's lowest value) have no mass; a row with one finite entry is certain of it; a row without any has neither mass nor entropy."""
    rng = np.random.default_rng(n + 1)
    low = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}[kind]
    x = rounded(rng.normal(0, 2, (6, n)), kind)
    x[0, rng.random(n) < 0.7] = -np.inf
    x[1] = -np.inf
    x[1, n // 3] = 4.0
    x[2] = -np.inf
    x[3, rng.random(n) < 0.7] = low
    x[4] = low
    x[5, :-1] = -np.inf
    tokens = [int(np.argmax(x[0])), n // 3, 5, 0, 9, 0]
    logprob, entropy, ids, top = _run(ctx, x, kind, tokens, 8)
    rest = [0, 1, 3, 4, 5]
    _check(x[rest], [tokens[r] for r in rest], 8, (logprob[rest], entropy[rest], ids[rest], top[rest]))
    assert logprob[1] == 0 and entropy[1] == 0 and logprob[5] == -np.inf
    assert logprob[2] == -np.inf and entropy[2] == 0 and (top[2] == -np.inf).all() and (ids[2] == np.arange(8)).all()


def test_tokens_outside_and_parts_of_the_results(ctx):
    rng = np.random.default_rng(3)
    x = rng.normal(0, 2, (5, 777)).astype(np.float32)
    tokens = [-1, 777, 3, 2 ** 31 - 1, -2 ** 31]
    full = _run(ctx, x, "f32", tokens, 4)
    _check(x, tokens, 4, full)
    assert (full[0][[0, 1, 3, 4]] == 0).all()
    none = _run(ctx, x, "f32", None, 4)
    assert none[0] is None
    for a, b in zip(full[1:], none[1:]):
        np.testing.assert_array_equal(a, b)
    only = _run(ctx, x, "f32", tokens, 0, entropy=False)
    np.testing.assert_array_equal(only[0], full[0])


@pytest.mark.parametrize("n", [50, 40000])
def test_nan(ctx, n):
    """A NaN is the first of the alternatives and makes its row's values NaN; other rows keep theirs."""
    rng = np.random.default_rng(4)
    x = rng.normal(0, 2, (3, n)).astype(np.float32)
    clean = _run(ctx, x, "f32", [1, 1, 1], 3)
    x[1, n // 2] = np.nan
    x[1, 7] = np.nan
    logprob, entropy, ids, top = _run(ctx, x, "f32", [1, 1, 1], 3)
    assert np.isnan(logprob[1]) and np.isnan(entropy[1]) and np.isnan(top[1]).all() and list(ids[1][:2]) == [7, n // 2]
    for a, b in zip(clean, (logprob, entropy, ids, top)):
        np.testing.assert_array_equal(a[[0, 2]], b[[0, 2]])


def test_certain_rows_keep_their_digits(ctx):
    """One entry ahead of the rest by 12 to 60: log probability and entropy are tiny, and right to a few units of f32 all the same."""
    n = 3000
    x = np.zeros((4, n), np.float32)
    for r, lead in enumerate((12.0, 20.0, 30.0, 60.0)):
        x[r, 17 * r] = lead
    tokens = [17 * r for r in range(4)]
    logprob, entropy, _, _ = _run(ctx, x, "f32", tokens, 0)
    for r, lead in enumerate((12.0, 20.0, 30.0, 60.0)):
        rest = (n - 1) * np.exp(-lead)
        want_h = np.log1p(rest) + rest * lead / (1 + rest)
        # Z = 1 + rest in f32: rest survives to 2^-24 absolute, so does log Z
        assert abs(logprob[r] + np.log1p(rest)) <= 2.0 ** -23 + rest * 2.0 ** -20
        assert abs(entropy[r] - want_h) <= 2.0 ** -23 + want_h * 2.0 ** -18


def test_refusals(ctx):
    import runit_mac_b200 as R
    x, t, f, i = ctx.new_buffer(4096), ctx.new_buffer(64), ctx.new_buffer(4096), ctx.new_buffer(4096)
    ok = dict(logits=x, type=R.TYPE_F32, ld=100, n=100, rows=4, tokens=t, logprob=f, entropy=None, k=3, top_ids=i, top_logprobs=i)
    before = ctx.launches
    for change in (dict(logits=None), dict(type=3), dict(type=-1), dict(ld=99), dict(n=0), dict(rows=0), dict(tokens=None), dict(logprob=None), dict(k=33), dict(k=101, n=100),
                   dict(k=3, n=2), dict(top_ids=None), dict(top_logprobs=None), dict(k=0), dict(logits=x.ptr + 2), dict(tokens=t.ptr + 1), dict(entropy=f.ptr + 2),
                   dict(tokens=None, logprob=None, k=0, top_ids=None, top_logprobs=None)):
        with pytest.raises(R.KernelError) as e:
            R.token_logprobs(ctx, *{**ok, **change}.values())
        assert e.value.status == 2
    assert ctx.launches == before
