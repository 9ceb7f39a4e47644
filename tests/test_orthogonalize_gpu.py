"""Orthogonalised updates and the optimiser's step on the device, against
float64.

Bars.  What the device rounds is known: the factors of every product, to one
float16 plane (bfloat16, and float16 before the last three steps) or two
(float32, float16's last three steps, float16 of a short side and all small
matrices), and the sums to float32.  The
oracle makes the same roundings on the same matrix, and what they do to it,
d = oracle with roundings - oracle without, measures the conditioning of this
matrix; the device's roundings fall elsewhere (sums differ in their last
places) but are as many and as large.  The bar is twice |d| in the Frobenius
norm and four times its largest value anywhere, plus the sums in float32
(2^-22 sqrt(side) for each of the 15 products, of entries below 1.3) and the
result's own rounding."""
import numpy as np
import pytest

from oracle import few_bits
from oracle import training as O

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SHAPES = [(1, 1), (1, 5), (7, 3), (33, 65), (64, 128), (128, 64), (130, 257), (200, 40), (3, 70, 70),
          (32, 257, 300), (32, 300, 257), (64, 257, 260), (64, 260, 257), (2, 3, 16, 24), (10, 128), (1, 512), (512, 20), (128, 128), (100, 160), (129, 33)]


def _dev(gpu, a, dtype="float32"):
    t = gpu.from_numpy(np.ascontiguousarray(a, np.float32))
    return t if dtype == "float32" else gpu.cast(t, dtype)


def _gradient(shape, dtype, seed=0, size=1e-3):
    """A few strong directions and noise."""
    rng = np.random.default_rng(seed + sum(shape))
    m, n = shape[-2:]
    r = max(1, min(m, n) // 8)
    strong = rng.standard_normal((*shape[:-2], m, r)) @ rng.standard_normal((*shape[:-2], r, n)) / np.sqrt(r)
    return few_bits.round_to(size * (strong + 0.3 * rng.standard_normal(shape)), dtype)


def _bars(g, dtype, **kw):
    """(result, bar of the Frobenius norm, bar of a value) of each matrix."""
    want = O.orthogonalize(g, **kw)
    steps, (m, n) = kw.get("steps", 5), g.shape[-2:]
    small = min(m, n) <= 128 and -(-m // 32) * -(-n // 32) <= 16
    halves = {"float32": [2] * steps, "bfloat16": [2 if small else 1] * steps,
              "float16": [2 if i + 3 >= steps or min(m, n) <= 256 else 1 for i in range(steps)]}[dtype]
    d = O.orthogonalize(g, halves=halves, **kw) - want
    side = np.sqrt(min(g.shape[-2:]))
    sums = 15 * 2.0 ** -22 * side
    norm = 2 * np.sqrt((d * d).sum((-2, -1))) + sums * np.sqrt((want * want).sum((-2, -1)) / side)
    value = 4 * np.abs(d).max((-2, -1)) + sums * np.abs(want).max((-2, -1))
    return want, norm, value


def _check(got, want, norm, value, u, scale=1.0):
    e = np.abs(got.astype(np.float64) - want)
    round_off = u * np.abs(want)
    assert (np.sqrt((e * e).sum((-2, -1))) <= scale * norm + np.sqrt((round_off ** 2).sum((-2, -1)))).all()
    assert (e <= scale * value[..., None, None] + round_off + 2.0 ** -25 * (u == 2.0 ** -11)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_vs_oracle(gpu, shape, dtype):
    g = _gradient(shape, dtype)
    out = gpu.orthogonalize(_dev(gpu, g, dtype))
    assert out.shape == list(shape) and out.dtype == dtype
    _check(out.to_numpy(), *_bars(g, dtype), HALF_STEP[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (5, 9), (64, 128), (96, 40), (257, 130)])
def test_muon_step_vs_oracle(gpu, shape, dtype):
    rng = np.random.default_rng(sum(shape))
    n = 3
    w = few_bits.round_to(rng.standard_normal((n, *shape)) * 0.02, dtype)
    g = _gradient((n, *shape), dtype)
    m = (4 * _gradient((n, *shape), "float32", 5)).astype(np.float32)
    for nesterov in (True, False):
        dw, dm, dg = [_dev(gpu, a, dtype) for a in w], [_dev(gpu, a) for a in m], [_dev(gpu, a, dtype) for a in g]
        gpu.muon_step_(dw, dm, dg, lr=0.05, beta=0.9, weight_decay=0.1, nesterov=nesterov)
        rate = 0.05 * np.sqrt(max(1.0, shape[0] / shape[1]))
        for i in range(n):
            want, mom = O.muon_step(w[i], m[i], g[i], 0.05, 0.9, 0.1, nesterov)
            np.testing.assert_allclose(dm[i].to_numpy(), mom, rtol=2.0 ** -22, atol=2.0 ** -22 * np.abs(m[i]).max())
            u = g[i] + 0.9 * mom if nesterov else mom
            _, norm, value = _bars(u, dtype)
            # U itself is float32's
            _check(dw[i].to_numpy(), want, rate * norm, rate * value + 2.0 ** -23 * np.abs(want).max(), HALF_STEP[dtype])
