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
