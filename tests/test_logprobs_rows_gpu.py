"""Log probabilities of more rows than blocks, of rows that hold +Inf, and of rows whose alternatives all lie in one lane's entries."""
import numpy as np
import pytest

from paged_batches import rounded
from test_logprobs_gpu import _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(700, 300, 3), (1300, 5000, 4), (2400, 77, 32), (593, 30001, 1)])
def test_more_rows_than_blocks(ctx, kind, rows, n, k):
    rng = np.random.default_rng(rows + n)
    x = rounded(rng.normal(0, 3, (rows, n)), kind)
    tokens = rng.integers(0, n, rows)
    _check(x, tokens, k, _run(ctx, x, kind, tokens, k))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [70, 40000])
def test_infinite_logits(ctx, kind, n):
    """+Inf minus itself is no number: the row's values are NaN, its alternatives in order all the same; the rows beside it keep theirs."""
    rng = np.random.default_rng(n)
    x = rounded(rng.normal(0, 2, (4, n)), kind)
    clean = _run(ctx, x, kind, [1] * 4, 6)
    x[1, n // 2] = np.inf
    x[2, [3, n - 1]] = np.inf
    logprob, entropy, ids, top = _run(ctx, x, kind, [1] * 4, 6)
    for r in (1, 2):
        assert np.isnan(logprob[r]) and np.isnan(entropy[r]) and np.isnan(top[r]).all()
        np.testing.assert_array_equal(ids[r], np.argsort(-x[r], kind="stable")[:6])
    for a, b in zip(clean, (logprob, entropy, ids, top)):
        np.testing.assert_array_equal(a[[0, 3]], b[[0, 3]])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 60000), (200, 60000)])
@pytest.mark.parametrize("k", [1, 7, 32])
def test_alternatives_next_to_each_other(ctx, kind, rows, n, k):
    """The largest entries side by side, at the distance of the lanes' vectors, in the first and in the last places: whoever keeps one largest entry a lane has to look again."""
    rng = np.random.default_rng(k)
    x = rng.normal(0, 1, (rows, n))
    per = 4 if kind == "f32" else 8
    for r in range(rows):
        way = r % 4
        at = (np.arange(40) + 17 * r if way == 0 else np.arange(40) * 32 * per + r if way == 1 else np.arange(40) if way == 2 else n - 1 - np.arange(40)) % n
        x[r, at] = 9 + rng.permutation(40) / 8
    x = rounded(x, kind)
    tokens = rng.integers(0, n, rows)
    _check(x, tokens, k, _run(ctx, x, kind, tokens, k))
