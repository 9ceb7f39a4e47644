"""Orthogonalised updates at the ends of what their values can be; bars as in
the tests of ordinary ones."""
import numpy as np
import pytest

from oracle import few_bits

from test_orthogonalize_gpu import DTYPES, HALF_STEP, _bars, _check, _dev, _gradient

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(40, 30), (200, 300), (300, 200)])
def test_norms_past_float32(gpu, shape, dtype):
    """Finite values whose norm has no float32, or few of its bits: by powers of
    two the bits of ordinary ones, and by the default eps where that is nothing
    beside the norm."""
    g = _gradient(shape, dtype, size=1.0)
    g = few_bits.round_to(g / np.abs(g).max(), dtype)
    want = gpu.orthogonalize(_dev(gpu, g, dtype), eps=0.0).to_numpy()
    assert np.isfinite(want).all() and np.abs(want).max() > 0
    for scale in (2.0 ** 127, 2.0 ** 124, 2.0 ** -100, 2.0 ** -110):
        got = gpu.orthogonalize(_dev(gpu, g * np.float32(scale), dtype), eps=0.0).to_numpy()
        np.testing.assert_array_equal(got, want, err_msg=str(scale))
    np.testing.assert_array_equal(gpu.orthogonalize(_dev(gpu, g * np.float32(2.0 ** 127), dtype)).to_numpy(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps", [1, 2, 5])
@pytest.mark.parametrize("shape", [(1, 1), (16, 40), (128, 100), (300, 200), (260, 700)])
def test_one_direction(gpu, shape, steps, dtype):
    """Matrices of rank one, of one entry and of equal entries, whose Gram
    matrix and polynomial are as large as they get (2.8 of the 4.0 that the
    planes hold)."""
    rng = np.random.default_rng(shape[1])
    one = np.zeros(shape)
    one[-1, shape[1] // 2] = -3.0
    for g in (np.outer(rng.standard_normal(shape[0]), rng.standard_normal(shape[1])), np.ones(shape), one):
        g = few_bits.round_to(g, dtype)
        _check(gpu.orthogonalize(_dev(gpu, g, dtype), steps=steps).to_numpy(), *_bars(g, dtype, steps=steps),
               HALF_STEP[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(64, 120), (200, 300), (300, 200)])
@pytest.mark.parametrize("below", [2.0 ** -10, 2.0 ** -20, 2.0 ** -27])
def test_rows_far_below_the_largest(gpu, shape, below, dtype):
    g = _gradient(shape, dtype, size=1.0)
    g[::3] *= below
    g = few_bits.round_to(g, dtype)
    _check(gpu.orthogonalize(_dev(gpu, g, dtype)).to_numpy(), *_bars(g, dtype), HALF_STEP[dtype])
