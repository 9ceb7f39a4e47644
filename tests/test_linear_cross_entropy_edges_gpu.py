"""Cross entropy of a linear layer and its gradient where operands are read in
place out of larger tensors, and at values that are not ordinary; float64
beside them."""
import numpy as np
import pytest

from oracle import few_bits
from oracle import training as O

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


def _dev(gpu, a, dtype="float32"):
    t = gpu.from_numpy(np.ascontiguousarray(a, np.float32))
    return t if dtype == "float32" else gpu.cast(t, dtype)


def _columns(gpu, a, dtype, ld, off):
    """a as the columns from `off` on of rows of `ld` values that are not
    numbers: the last one's storage ends with it where off + columns = ld."""
    wide = np.full((a.shape[0], ld), np.nan, np.float32)
    wide[:, off:off + a.shape[1]] = a
    return gpu.slice(_dev(gpu, wide, dtype), 1, off, off + a.shape[1])


# rows of 16-byte chunks, so that 16-bit operands are read where they are: few
# features and more than a tile's columns, views that end with their rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,K,V,ld,off", [
    (64, 64, 128, 128, 64), (8, 64, 1024, 512, 448), (128, 72, 256, 136, 64), (256, 264, 512, 1024, 760),
    (300, 768, 1000, 2304, 768), (33, 520, 257, 1024, 504), (1, 8, 5, 16, 8)])
def test_columns_of_wider_rows(gpu, R, K, V, ld, off, dtype):
    rng = np.random.default_rng(R + K + V)
    w = few_bits.round_to(rng.standard_normal((V, K)) * 3 / np.sqrt(K), dtype)
    x = few_bits.round_to(rng.standard_normal((R, K)), dtype)
    t = rng.integers(-1, V, R).astype(np.int32)
    g = rng.random(R).astype(np.float32)

    def all_of(a, b):
        ti = gpu.from_numpy(t)
        out = gpu.linear_cross_entropy(a, b, ti)
        return [v.to_numpy() for v in (*out, *gpu.linear_cross_entropy_backward(_dev(gpu, g), a, b, ti, *out))]

    plain = _dev(gpu, x, dtype), _dev(gpu, w, dtype)
    want = all_of(*plain)
    assert all(np.isfinite(v).all() for v in want)
    views = _columns(gpu, x, dtype, ld, off), _columns(gpu, w, dtype, ld, off)
    for a, b in ((views[0], plain[1]), (plain[0], views[1]), views):
        for got, v in zip(all_of(a, b), want):
            np.testing.assert_array_equal(got, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 40, 700])
def test_an_infinite_logit_is_not_a_certain_word(gpu, dtype, V):
    """One word of +inf: rows that see it have no loss and no sum, be it their
    target, another word or the only one; rows that see it as -inf do without
    it."""
    word, K = V // 2, 16
    rng = np.random.default_rng(V)
    x = few_bits.round_to(rng.standard_normal((6, K)), dtype)
    w = few_bits.round_to(rng.standard_normal((V, K)), dtype)
    x[:, 0], w[word, 0] = [1, 2, 1, 0.5, -1, -2], np.inf
    t = np.array([word, 0, -100, V - 1, 0, -100], np.int32)
    loss, lse = (a.to_numpy() for a in gpu.linear_cross_entropy(_dev(gpu, x, dtype), _dev(gpu, w, dtype),
                                                                gpu.from_numpy(t)))
    assert np.isnan(lse[:4]).all() and np.isnan(loss[[0, 1, 3]]).all() and loss[2] == 0 and loss[5] == 0
    if dtype != "float32" and word != 0:
        want = O.linear_cross_entropy(x[4:], np.delete(w, word, 0), [0, -100])
        np.testing.assert_allclose(lse[4:], want[1], rtol=1e-5, atol=1e-4)
        np.testing.assert_allclose(loss[4:], want[0], rtol=1e-4, atol=1e-4)


def test_products_past_float32_are_not_certain_words(gpu):
    """bfloat16 operands whose one product overflows, as the target."""
    x, w = np.zeros((2, 8), np.float32), np.eye(5, 8, dtype=np.float32)
    x[0, 3], w[3, 3], x[1, 1] = 2.0 ** 100, 2.0 ** 100, 4.0
    loss, lse = (a.to_numpy() for a in gpu.linear_cross_entropy(_dev(gpu, x, "bfloat16"), _dev(gpu, w, "bfloat16"),
                                                                gpu.from_numpy(np.array([3, 1], np.int32))))
    assert np.isnan(loss[0]) and np.isnan(lse[0])
    np.testing.assert_allclose([loss[1], lse[1]], [np.log(4 + np.exp(4)) - 4, np.log(4 + np.exp(4))], rtol=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,bad", [(20, 5), (33, 32), (300, 131), (5000, 4999)])
def test_rows_without_weight_and_without_a_loss(gpu, R, bad, dtype):
    """A row with a word as its target whose loss is not a number, left out by a
    weight of 0: dx is zero there, and all else is as without the row."""
    K, V = 24, 90
    rng = np.random.default_rng(R)
    x = few_bits.round_to(rng.standard_normal((R, K)), dtype)
    w = few_bits.round_to(rng.standard_normal((V, K)), dtype)
    t = rng.integers(0, V, R).astype(np.int32)
    g, h = rng.random(R).astype(np.float32) / R, rng.standard_normal(R).astype(np.float32) / R
    g[bad] = h[bad] = 0
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
    good = [a.to_numpy() for a in gpu.linear_cross_entropy(*dev)]
    for of_lse in (None, _dev(gpu, h)):
        want = [a.to_numpy() for a in gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *map(gpu.from_numpy, good),
                                                                        grad_lse=of_lse)]
        assert (want[0][bad] == 0).all()
        for value in ((np.nan, np.nan), (np.nan, np.inf), (np.inf, np.inf), (np.inf, 3.0)):
            loss, lse = (a.copy() for a in good)
            loss[bad], lse[bad] = value
            got = gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, _dev(gpu, loss), _dev(gpu, lse), grad_lse=of_lse)
            for a, b in zip(got, want):
                np.testing.assert_array_equal(a.to_numpy(), b)


@pytest.mark.parametrize("dtype", ["bfloat16"])
def test_a_row_that_overflows_is_left_out_by_its_weight(gpu, dtype):
    """The same from the forward pass: finite values whose products overflow."""
    rng = np.random.default_rng(1)
    x = few_bits.round_to(rng.standard_normal((9, 16)), dtype)
    w = few_bits.round_to(rng.standard_normal((50, 16)), dtype)
    t, g = rng.integers(0, 50, 9).astype(np.int32), rng.random(9).astype(np.float32)
    g[4] = 0

    def run(x):
        dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
        out = gpu.linear_cross_entropy(*dev)
        return [a.to_numpy() for a in (*out, *gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *out))]

    want = run(x)
    x[4] = few_bits.round_to(np.sign(x[4]) * 3e38, dtype)
    loss, lse, dx, dw = run(x)
    assert not np.isfinite(loss[4])
    rest = np.arange(9) != 4
    for a, b in ((loss[rest], want[0][rest]), (lse[rest], want[1][rest]), (dx[rest], want[2][rest]), (dw, want[3])):
        np.testing.assert_allclose(a, b, rtol=1e-5, atol=1e-5 * np.abs(b).max())
    assert (dx[4] == 0).all()
