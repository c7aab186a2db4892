"""The products with packed weights at the ends of their ranges, against float64 restatements: numbers that are not
finite and whom they may reach, the largest and the least inputs, and what the forms keep of weights of many bits.

Tolerances are those of test_linear_gpu (an output's rounding, K 2^-24 T for float32 sums of K terms, T the sum over
absolute values, and what a form's operands lose), with the operands' part named by each test."""
import numpy as np
import pytest

from seedpack_amd import linear
from seedpack_amd.gpuquant import GPUQuant
from seedpack_amd.requant import QFUN
from tests.test_linear_gpu import (BF16, F16, _named, adapters, close, gated_backward64, inputs, project64, random_blocks,  # noqa: F401
                                   rng, slack, store, up, weights, wide)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("m,k,rank", [(40, 512, 5), (150, 512, 5), (300, 512, 16), (300, 2048, 20)])
def test_adapter_that_is_not_finite(m, k, rank, bad, kind):
    """one number of one adapter's second matrix: its own rows have what the definition says in that column; rows of
    other adapters and of none, in the same tile, are bit for bit as without it"""
    g = rng(40, m, k, kind is F16)
    n, pool = 140, 3
    w, w64 = weights(g, linear.F16 if kind is F16 else linear.BF16, n, k)
    x, x64 = inputs(g, m, k, kind)
    ad, a, b, s = adapters(g, pool, rank, n, k, kind)
    which = g.integers(-1, pool, m).astype(np.int32)
    clean = linear.project(up(x), w, ad, up(which)).to_host()
    worse = b.copy()
    worse[1, 9, 2] = bad
    got = linear.project(up(x), w, linear.Adapters(ad.a, up(store(worse, kind)), ad.scale), up(which)).to_host()
    mine = which == 1
    assert mine.any() and not mine.all()
    assert np.array_equal(got[~mine], clean[~mine])
    rest = np.arange(n) != 9
    y, total = project64(x64[mine], w64, a, b, s, which[mine])
    close(np.ascontiguousarray(got[mine][:, rest]), y[:, rest], slack(total[:, rest], k + rank), kind)
    want = bad * np.sign(x64[mine] @ a[1][2])
    assert np.array_equal(wide(got[mine][:, 9]), want, equal_nan=True)


@pytest.mark.parametrize("m", [1, 3, 20, 64, 100, 150])
@pytest.mark.parametrize("t", [linear.F16, linear.BF16, 2, 8, 12, 13, 14, 3, 16, 20, 23])
def test_project_largest_inputs(t, m):
    """BF16 inputs so large that the sums come near the largest float32 and codes times inputs pass it: finite as
    the definition is"""
    g = rng(41, t, m)
    n, k = 37, 512
    w, w64 = weights(g, t, n, k)
    x = g.normal(0, 1, (m, k))
    x *= 2.0 ** np.floor(np.log2(2.0 ** 127 / (np.abs(x) @ np.abs(w64.T)).max(1, keepdims=True)))
    x = store(np.clip(x, -3e38, 3e38), BF16)
    y, total = project64(wide(x), w64)
    assert total.max() < 3.4e38 and np.isfinite(wide(x)).all()
    close(linear.project(up(x), w).to_host(), y, slack(total, k), BF16)


@pytest.mark.parametrize("m", [1, 20, 64])
@pytest.mark.parametrize("t", [2, 8, 12, 13, 14])
def test_gated_largest_inputs(t, m):
    """the same gate beside an up projection of zeros: zeros, not an infinity times zero"""
    g = rng(42, t, m)
    n, k = 37, 512
    gate, w64 = weights(g, t, n, k)
    zero = linear.Weight(t, up(np.zeros(gate.data.nbytes, np.uint8)), n, k)
    x = g.normal(0, 1, (m, k))
    x *= 2.0 ** np.floor(np.log2(2.0 ** 127 / (np.abs(x) @ np.abs(w64.T)).max(1, keepdims=True)))
    assert (wide(linear.gated(up(store(np.clip(x, -3e38, 3e38), BF16)), gate, zero).to_host()) == 0).all()


@pytest.mark.parametrize("m", [1, 3, 40, 64])
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("t", [linear.F16, linear.BF16, 8, 12, 14, 10, 19])
def test_few_rows_with_numbers_that_are_not_finite(t, kind, m):
    """all of a row infinite or NaN, or one number in its first or last places: every output of the row as defined"""
    g = rng(43, t, m, kind is F16)
    n, k = 70, 1280
    w, w64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    clean = linear.project(up(x), w).to_host()
    for at, v in ((0, np.nan), (k - 1, np.nan), (slice(0, None), np.nan), (0, np.inf), (k - 1, -np.inf), (777, np.inf)):
        bad = x64.copy()
        bad[m // 2, at] = v
        got = linear.project(up(store(bad, kind)), w).to_host()
        keep = np.arange(m) != m // 2
        assert np.array_equal(got[keep], clean[keep])
        row = wide(got[m // 2])
        if np.isnan(v):
            assert np.isnan(row).all()
        else:
            with np.errstate(invalid="ignore"):
                assert np.array_equal(row, v * w64[:, at], equal_nan=True)
