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


# products whose last tiles, or all of them, are cut along k and joined: of 128
# and of 256 wide, of X and of the Gram matrix itself, ragged, from either side
@pytest.mark.parametrize("shape,dtype,steps", [
    ((90, 257, 1500), "bfloat16", 5), ((90, 900, 257), "float32", 5), ((27, 1500, 300), "float32", 5),
    ((27, 300, 3000), "float16", 5), ((2300, 2300), "float32", 1), ((5700, 2850), "float32", 1)])
def test_cut_products_vs_oracle(gpu, shape, dtype, steps):
    g = _gradient(shape, dtype)
    out = gpu.orthogonalize(_dev(gpu, g, dtype), steps=steps)
    out, again = out.to_numpy(), gpu.orthogonalize(_dev(gpu, g, dtype), steps=steps).to_numpy()
    np.testing.assert_array_equal(out, again)
    some = [0, len(g) // 2, len(g) - 1] if g.ndim == 3 else ...
    _check(out[some], *_bars(g[some], dtype, steps=steps), HALF_STEP[dtype])


def test_eager_entry(gpu):
    from applegpu_runtime import eager as E
    E.init()
    g = _gradient((3, 40, 70), "float32")
    np.testing.assert_array_equal(E.orthogonalize(E.from_numpy(g.astype(np.float32)), steps=3).numpy(),
                                  gpu.orthogonalize(_dev(gpu, g), steps=3).to_numpy())


def test_cut_products_of_a_smaller_last_group(gpu):
    """More matrices than a launch takes by their addresses: the last ones, fewer,
    are cut elsewhere than the first."""
    rng = np.random.default_rng(3)
    n, shape = 40, (700, 2000)
    g = [_gradient(shape, "float32", seed=i) for i in range(2)]
    w, mom = [_dev(gpu, np.zeros(shape)) for _ in range(n)], [_dev(gpu, np.zeros(shape)) for _ in range(n)]
    gpu.muon_step_(w, mom, [_dev(gpu, g[i % 2]) for i in range(n)], lr=1.0, beta=0.0)
    bars = [_bars(a, "float32") for a in g]
    for i in (0, 1, 31, 32, 39):
        _check(-w[i].to_numpy(), *bars[i % 2], HALF_STEP["float32"])


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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps", [1, 2, 3, 7])
def test_steps(gpu, dtype, steps):
    for shape in ((40, 30), (200, 300)):
        g = _gradient(shape, dtype, seed=steps)
        out = gpu.orthogonalize(_dev(gpu, g, dtype), steps=steps)
        _check(out.to_numpy(), *_bars(g, dtype, steps=steps), HALF_STEP[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_singular_values_come_near_one(gpu, dtype):
    g = _gradient((150, 400), dtype)
    s = np.linalg.svd(gpu.orthogonalize(_dev(gpu, g, dtype)).to_numpy().astype(np.float64), compute_uv=False)
    assert s.max() < 1.3 and np.median(s) > 0.6


def test_views_and_sizes_of_values(gpu):
    """A transposed or cut view is as its copy; the size of the values matters
    by eps alone."""
    for shape in ((50, 90), (300, 200)):
        g = _gradient(shape, "float32")
        want = gpu.orthogonalize(_dev(gpu, g)).to_numpy()
        t = gpu.transpose(_dev(gpu, np.ascontiguousarray(g.T)))
        np.testing.assert_array_equal(gpu.orthogonalize(t).to_numpy(), want)
        wide = np.zeros((shape[0] + 3, shape[1] + 5), np.float32)
        wide[2:-1, 3:-2] = g
        cut = gpu.slice(gpu.slice(_dev(gpu, wide), 0, 2, 2 + shape[0]), 1, 3, 3 + shape[1])
        np.testing.assert_array_equal(gpu.orthogonalize(cut).to_numpy(), want)
        for scale in (2.0 ** -60, 2.0 ** 40, 2.0 ** 90):
            got = gpu.orthogonalize(_dev(gpu, g * np.float32(scale)), eps=0.0).to_numpy()
            same = gpu.orthogonalize(_dev(gpu, g), eps=0.0).to_numpy()
            np.testing.assert_allclose(got, same, rtol=0, atol=2e-6 * np.abs(same).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(4, 30, 50), (3, 200, 300)])
def test_zeros_and_what_is_not_finite_stay_in_their_matrix(gpu, dtype, shape):
    g = _gradient(shape, dtype)
    want = gpu.orthogonalize(_dev(gpu, g, dtype)).to_numpy()
    bad = g.copy()
    bad[0] = 0
    bad[1, 3, 5] = np.nan
    for eps in (1e-7, 0.0):
        got = gpu.orthogonalize(_dev(gpu, bad, dtype), eps=eps).to_numpy()
        assert (got[0] == 0).all() and np.isnan(got[1]).all() and np.isfinite(got[2:]).all()
    np.testing.assert_array_equal(gpu.orthogonalize(_dev(gpu, bad, dtype)).to_numpy()[2:], want[2:])


def test_nothing_to_do(gpu):
    assert gpu.orthogonalize(gpu.zeros([0, 5, 7])).shape == [0, 5, 7]
    assert gpu.orthogonalize(gpu.zeros([3, 0])).shape == [3, 0]
    gpu.muon_step_([], [], [])


@pytest.mark.parametrize("shape", [(20, 30), (130, 200)])
def test_many_matrices_in_groups(gpu, shape):
    """More matrices than a launch takes by their addresses: as one by one."""
    n = 37
    rng = np.random.default_rng(1)
    w = rng.standard_normal((n, *shape)).astype(np.float32)
    g = _gradient((n, *shape), "float32")
    together = [[_dev(gpu, a) for a in v] for v in (w, np.zeros_like(w), g)]
    gpu.muon_step_(*together, lr=0.1)
    for i in (0, 31, 32, 36):
        alone = [_dev(gpu, v[i]) for v in (w, np.zeros_like(w), g)]
        gpu.muon_step_(*alone, lr=0.1)
        np.testing.assert_array_equal(together[0][i].to_numpy(), alone[0].to_numpy())
        np.testing.assert_array_equal(together[1][i].to_numpy(), alone[1].to_numpy())


def test_odd_places_of_views(gpu):
    """Weights, momenta and gradients that start at any element."""
    for dtype in DTYPES:
        for shape in ((24, 40), (160, 200)):
            size = shape[0] * shape[1]
            rng = np.random.default_rng(2)
            flat = rng.standard_normal(3 * size + 9).astype(np.float32) * 1e-2
            flat = few_bits.round_to(flat, dtype)
            m = rng.standard_normal(size + 3).astype(np.float32) * 1e-2
            d, dm = _dev(gpu, flat, dtype), _dev(gpu, m)
            view = lambda t, at: gpu.reshape(gpu.slice(t, 0, at, at + size), list(shape))
            w, g, mom = view(d, 1), view(d, size + 4), view(dm, 3)
            gpu.muon_step_(w, mom, g, lr=0.1)
            cut = [flat[1:1 + size].reshape(shape), m[3:].reshape(shape), flat[size + 4:2 * size + 4].reshape(shape)]
            same = [_dev(gpu, cut[0], dtype), _dev(gpu, cut[1]), _dev(gpu, cut[2], dtype)]
            gpu.muon_step_(*same, lr=0.1)
            got = d.to_numpy()
            np.testing.assert_array_equal(got[1:1 + size], same[0].to_numpy().reshape(-1))
            np.testing.assert_array_equal(np.delete(got, np.arange(1, 1 + size)),
                                          np.delete(flat, np.arange(1, 1 + size)))   # nothing beside it
            np.testing.assert_array_equal(dm.to_numpy()[3:], same[1].to_numpy().reshape(-1))
            np.testing.assert_array_equal(dm.to_numpy()[:3], m[:3])


def test_what_was_asked_before_the_step_sees_the_weights_before(gpu):
    rng = np.random.default_rng(3)
    w, m, g = (rng.standard_normal((16, 24)).astype(np.float32) for _ in range(3))
    dw, dm, dg = (_dev(gpu, a) for a in (w, m, g))
    x = _dev(gpu, rng.standard_normal((4, 24)))
    y = gpu.relu(gpu.matmul(x, gpu.transpose(dw)) + gpu.full([4, 16], 1.0))
    mm = gpu.transpose(dm) + gpu.transpose(dm)
    gpu.muon_step_(dw, dm, dg, lr=0.5)
    after = dw.to_numpy()
    assert not np.array_equal(after, w)
    np.testing.assert_allclose(y.to_numpy(), np.maximum(x.to_numpy() @ w.T + 1, 0), rtol=1e-3, atol=1e-4)
    np.testing.assert_array_equal(mm.to_numpy(), 2 * m.T)


def test_refusals(gpu):
    z = lambda *s, dtype="float32": gpu.zeros(list(s), dtype)
    with pytest.raises(ValueError, match="at least 2D"):
        gpu.orthogonalize(z(5))
    with pytest.raises(ValueError, match="orthogonalize"):
        gpu.orthogonalize(gpu.cast(z(5, 5), "int32"))
    for steps in (0, -1, 101):
        with pytest.raises(ValueError, match="steps"):
            gpu.orthogonalize(z(5, 5), steps=steps)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            gpu.orthogonalize(z(5, 5), eps=eps)
    a, b, c = z(4, 6), z(4, 6), z(4, 6)
    for t in (a, b, c):
        t.eval()
    with pytest.raises(ValueError, match="weights, 2 momenta"):
        gpu.muon_step_([a], [b, c], [c])
    with pytest.raises(ValueError, match="one shape"):
        gpu.muon_step_(a, z(6, 4), c)
    with pytest.raises(ValueError, match="one shape"):
        gpu.muon_step_([a, z(5, 5)], [b, z(5, 5)], [c, z(5, 5)])
    with pytest.raises(ValueError, match="one shape"):
        gpu.muon_step_(z(4), z(4), z(4))
    with pytest.raises(ValueError, match="must be float32"):
        gpu.muon_step_(z(4, 6, dtype="float16"), z(4, 6, dtype="float16"), z(4, 6, dtype="float16"))
    with pytest.raises(ValueError, match="Dtype mismatch"):
        gpu.muon_step_(z(4, 6, dtype="float16"), b, c)
    with pytest.raises(ValueError, match="contiguous"):
        gpu.muon_step_(gpu.transpose(z(6, 4)), b, c)
    with pytest.raises(ValueError, match="share storage"):
        gpu.muon_step_([a, a], [b, c], [z(4, 6), z(4, 6)])
    with pytest.raises(ValueError, match="share storage"):
        gpu.muon_step_(a, b, b)
    with pytest.raises(ValueError, match="share storage"):
        gpu.muon_step_(a, b, a)
    whole = z(8, 6)
    whole.eval()
    with pytest.raises(ValueError, match="share storage"):
        gpu.muon_step_(gpu.slice(whole, 0, 0, 4), b, gpu.slice(whole, 0, 3, 7))
    for kw in (dict(lr=float("nan")), dict(beta=float("inf")), dict(weight_decay=float("nan"))):
        with pytest.raises(ValueError, match="finite"):
            gpu.muon_step_(a, b, c, **kw)
    with pytest.raises(ValueError, match="expected GpuTensor"):
        gpu.muon_step_(a, b, np.zeros((4, 6), np.float32))
    assert (a.to_numpy() == 0).all()
    gpu.muon_step_([a, z(4, 6)], [b, z(4, 6)], [c, c])   # one gradient for two weights is a read
