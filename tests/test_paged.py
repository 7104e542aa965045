"""The paged operators' host side without a GPU: descriptions that are refused, sizes of the scratch, and the tests' own reference."""
import ctypes as C

import numpy as np
import pytest

from paged_batches import Batch, from_bits, rounded, to_bits


def _described(**change):
    from runit_mac_b200 import _lib, dispatch as R
    cfg = R.PagedCfg(heads=28, kv_heads=4, dim=128, page=64, n_pages=1000, type=R.TYPE_F16, window=0, scale=0.1, cap=0.0)
    batch = R.PagedBatch(n_seqs=8, rows=8, table_ld=100, shared_len=0)
    for k, v in change.items():
        setattr(cfg if hasattr(cfg, k) else batch, k, v)
    return _lib.load().runit_paged_attention_scratch_bytes(C.byref(cfg), C.byref(batch))


@pytest.mark.parametrize("change", [dict(heads=0), dict(heads=30), dict(heads=1028), dict(kv_heads=0), dict(dim=32), dict(dim=256), dict(page=0), dict(page=48), dict(page=8),
                                    dict(page=512), dict(n_pages=0), dict(n_pages=0xFFFFFFFF), dict(n_pages=1 << 24), dict(type=0), dict(type=3), dict(scale=float("inf")),
                                    dict(cap=float("nan")), dict(cap=-2.0), dict(n_seqs=0), dict(n_seqs=5000), dict(rows=0), dict(rows=1 << 28), dict(table_ld=0),
                                    dict(table_ld=1 << 26), dict(shared_len=63), dict(shared_len=6464), dict(n_seqs=4096, table_ld=1 << 20)])
def test_descriptions_that_are_refused(change):
    assert _described(**change) == 0


@pytest.mark.parametrize("cap,scale,fits", [(1e-40, 0.1, False), (1e-38, -3.0, True)])       # 3 / 1e-38 = 3e38 is below f32's largest, 3.4e38; 0.1 / 1e-40 = 1e39 is not
def test_a_cap_that_the_scale_cannot_be_divided_by(cap, scale, fits):
    assert (_described(cap=cap, scale=scale) > 0) == fits and _described(cap=1e-30, scale=scale) > 0


def test_scratch_goes_with_the_sizes_alone():
    base = _described()
    assert base > 0 and _described() == base
    assert _described(shared_len=6400) >= base
    assert _described(rows=4096, n_seqs=4096) < 1 << 31


def test_null_arguments_without_a_device():
    from runit_mac_b200 import _lib
    lib = _lib.load()
    assert lib.runit_paged_attention_scratch_bytes(None, None) == 0
    assert lib.runit_paged_attention(None, None, None, None, 0, None, 0, None, 0) == 2
    assert lib.runit_paged_append(None, None, None, None, 0, 0, None, 0, None, 0) == 2
    assert lib.runit_token_logprobs(None, None, 0, 0, 0, 0, None, None, None, 0, None, None) == 2


def test_the_reference_of_the_tests():
    """Rounding as the types have it, and the batch's own definition against a direct one on a single sequence."""
    x = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -2.0 ** -130, np.inf, np.nan, 3.0e38], np.float32)
    y = rounded(x, "bf16")
    assert y[1] == 1.0 and y[2] == 1 + 2.0 ** -6 and np.isinf(y[4]) and np.isnan(y[5])
    np.testing.assert_array_equal(from_bits(to_bits(x[:4], "f16"), "f16"), x[:4].astype(np.float16).astype(np.float32))
    b = Batch(1, [(3, 40), (1, 21)], 4, 2, 64, 16, "f16", shared=16, window=9, cap=5.0, slopes=[0.5, 0.25, 0.1, 0.0])
    out, bound = b.reference()
    assert np.isfinite(out).all() and (bound > 0).all()
    k, v = b.seq_kv(1)
    q = b.q[3, 2].astype(np.float64)
    t = 5 * np.tanh(k[1] @ q / 8 / 5) - 0.1 * (20 - np.arange(21))
    w = np.where(20 - np.arange(21) < 9, np.exp(t), 0)
    np.testing.assert_allclose(out[3, 2], (w / w.sum()) @ v[1], rtol=1e-6)
