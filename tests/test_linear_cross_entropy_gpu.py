"""Cross entropy of a linear layer over a vocabulary and its gradient on the
device, against float64.

Bars.  A logit is a sum of K exact products (16-bit operands) in float32: at
most one rounding for each 16 products and 16 more inside and behind, each half
a step of a partial sum, so off by (K / 16 + 16) 2^-24 S with S = sum |x| |w|.
float32 operands are two float16 planes: what their halves (2^-22 each) and the
left out product of the low halves (2^-22) lose is 3 2^-22 S, and what is below
float16's smallest step 2^-38 of the operand's largest value times the other's
sum; three products are summed.  The sum of exponentials adds 2^-20 (1 + |d|)
relative at most for an exponent d, of which those above -20 count.  d = p - 1 is rounded
once to the operands' 16 bits (planes: 2^-22) before its products, and the
results once to theirs; float16 holds d down to 2^-38 of the largest weight."""
import numpy as np
import pytest

from oracle import few_bits
from oracle import training as O

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SIZES = [(1, 1, 1), (1, 8, 2), (3, 7, 5), (5, 64, 100), (33, 65, 130), (64, 72, 257), (130, 200, 515),
         (257, 96, 1000), (31, 1280, 300), (600, 40, 17000)]


def _dev(gpu, a, dtype="float32"):
    t = gpu.from_numpy(np.ascontiguousarray(a, np.float32))
    return t if dtype == "float32" else gpu.cast(t, dtype)


def _case(R, K, V, dtype, seed=0):
    rng = np.random.default_rng(seed + R + K + V)
    w = few_bits.round_to(rng.standard_normal((V, K)) * 3 / np.sqrt(K), dtype)
    t = rng.integers(0, V, R)
    # from a word like any other to one that is nearly certain
    x = few_bits.round_to(rng.standard_normal((R, K)) + 3 * rng.random((R, 1)) * w[t], dtype)
    t[rng.random(R) < 0.1] = -100
    return x, w, t.astype(np.int32)


def _logit_bar(x, w, dtype):
    ax, aw = np.abs(x).astype(np.float64), np.abs(w).astype(np.float64)
    S, K = ax @ aw.T, x.shape[1]
    if dtype != "float32":
        return (K / 16 + 16) * 2.0 ** -24 * S
    small = 2.0 ** -38 * (ax.max() * aw.sum(1)[None, :] + aw.max() * ax.sum(1)[:, None])
    return (3 * K / 16 + 16) * 2.0 ** -24 * S + 3 * 2.0 ** -22 * S + small


def _check_forward(gpu, x, w, t, dtype, got=None):
    got = got or gpu.linear_cross_entropy(_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t))
    loss, lse = (a.to_numpy() for a in got)
    want = O.linear_cross_entropy(x, w, t)
    assert loss.dtype == lse.dtype == np.float32
    z = _logit_bar(x, w, dtype).max(1)
    # a loss is off by the logits' bars and its exponentials', relative to it
    # where it is small (1 - p = loss then) and at most absolutely
    rel = 2 * z + 24 * 2.0 ** -20
    assert (np.abs(loss - want[0]) <= rel * np.minimum(1.0, 2 * want[0]) * np.exp(2 * z) + 2.0 ** -23 * want[0] + 1e-37).all()
    assert (np.abs(lse - want[1]) <= z + 21 * 2.0 ** -20 + 2.0 ** -23 * np.abs(want[1])).all()
    assert (loss[(t < 0) | (t >= w.shape[0])] == 0).all()
    return got


def _check_backward(gpu, x, w, t, dtype, g, h, got=None):
    R, K, V = x.shape[0], x.shape[1], w.shape[0]
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
    if got is None:
        loss, lse = gpu.linear_cross_entropy(*dev)
        got = gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, loss, lse,
                                                grad_lse=None if h is None else _dev(gpu, h))
    dx, dw = (a.to_numpy().astype(np.float64) for a in got)
    want = O.linear_cross_entropy_backward(x, w, t, g, h)
    d = np.abs(O.logit_gradients(x, w, t, g, h))
    # |d| is off by p's error: the logit's and the sum's bars and the
    # exponential's, and by its rounding
    z = _logit_bar(x, w, dtype)
    lse = O.linear_cross_entropy(x, w, t)[1]
    most = (np.abs(g) + (0 if h is None else np.abs(h)))
    hold = 2.0 ** -22 if dtype == "float32" else HALF_STEP[dtype]
    p_err = z + z.max(1, keepdims=True) + 46 * 2.0 ** -20 + 2.0 ** -23 * np.abs(lse)[:, None]
    d_err = d * (p_err + hold) + 2.0 ** -38 * most.max()
    if h is not None:   # g (p - 1) + h p of a target can cancel
        p = np.abs(O.logit_gradients(x, w, t, np.zeros_like(g), np.abs(h)))
        d_err += 2 * p * p_err
    ax, aw = np.abs(x).astype(np.float64), np.abs(w).astype(np.float64)
    u = HALF_STEP[dtype]
    for name, a, b, err, n in (("dx", dx, want[0], d_err @ aw, V), ("dw", dw, want[1], d_err.T @ ax, R)):
        whole = (d @ aw) if name == "dx" else (d.T @ ax)
        sums = (3 * n / 16 + 32) * 2.0 ** -24 + (3 * 2.0 ** -22 if dtype == "float32" else 0)
        tiny = 2.0 ** -25 if dtype == "float16" else 1e-38   # below the result's smallest step
        bar = err + whole * sums + u * np.abs(b) + tiny
        bad = np.abs(a - b) > bar
        assert not bad.any(), (name, np.argwhere(bad)[:3], np.abs(a - b)[bad][:3], bar[bad][:3])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,K,V", SIZES)
def test_loss_vs_oracle(gpu, R, K, V, dtype):
    _check_forward(gpu, *_case(R, K, V, dtype), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,K,V", SIZES)
def test_gradient_vs_oracle(gpu, R, K, V, dtype):
    x, w, t = _case(R, K, V, dtype)
    rng = np.random.default_rng(R)
    g = rng.random(R).astype(np.float32) / R
    h = (rng.standard_normal(R) * 0.01 / R).astype(np.float32)
    _check_backward(gpu, x, w, t, dtype, g, None)
    _check_backward(gpu, x, w, t, dtype, g, h)


# ── layouts, types and shapes ───────────────────────────────────────────────
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_lead_dims(gpu, dtype):
    """Rows further apart than they are long, rows that start at odd places, a
    transposed weight, 3-D x, int64 targets: as the contiguous ones."""
    x, w, t = _case(12, 40, 90, dtype)
    want = [a.to_numpy() for a in gpu.linear_cross_entropy(_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t))]
    g = np.random.default_rng(2).random(12).astype(np.float32)
    wide = np.zeros((12, 49), np.float32)
    wide[:, 3:43] = x
    wide_w = np.zeros((90, 41), np.float32)
    wide_w[:, 1:] = w
    xv = gpu.slice(_dev(gpu, wide, dtype), 1, 3, 43)
    views = [xv, _dev(gpu, x, dtype)], [gpu.slice(_dev(gpu, wide_w, dtype), 1, 1, 41),
                                        gpu.transpose(_dev(gpu, np.ascontiguousarray(w.T), dtype))]
    grads = None
    for a in views[0]:
        for b in views[1]:
            got = gpu.linear_cross_entropy(a, b, gpu.from_numpy(t.astype(np.int64)))
            for u, v in zip(got, want):
                np.testing.assert_array_equal(u.to_numpy(), v)
            gr = [u.to_numpy() for u in gpu.linear_cross_entropy_backward(_dev(gpu, g), a, b, gpu.from_numpy(t), *got)]
            for u, v in zip(gr, grads or gr):
                np.testing.assert_array_equal(u, v)
            grads = grads or gr
    x3 = gpu.reshape(_dev(gpu, x, dtype), [3, 4, 40])
    loss, lse = gpu.linear_cross_entropy(x3, _dev(gpu, w, dtype), gpu.from_numpy(t.reshape(3, 4)))
    assert loss.shape == lse.shape == [3, 4]
    np.testing.assert_array_equal(loss.to_numpy().reshape(-1), want[0])
    dx, dw = gpu.linear_cross_entropy_backward(_dev(gpu, g.reshape(3, 4)), x3, _dev(gpu, w, dtype),
                                               gpu.from_numpy(t.reshape(3, 4)), loss, lse)
    assert dx.shape == [3, 4, 40] and dw.shape == [90, 40]
    np.testing.assert_array_equal(dx.to_numpy().reshape(12, 40), grads[0])
    one = gpu.linear_cross_entropy(_dev(gpu, x[0], dtype), _dev(gpu, w, dtype), gpu.from_numpy(t[:1]))
    np.testing.assert_allclose(one[0].to_numpy(), want[0][:1], rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_weights_far_apart(gpu, dtype):
    """Columns out of rows of 2^21 values and more, which no tile's loads reach
    across: as the contiguous ones."""
    x, w, t = _case(3, 8, 4, dtype)
    wide = gpu.zeros([4, (1 << 21) + 8], dtype)
    part = gpu.slice(wide, 1, 16, 24)
    gpu.blit_copy(_dev(gpu, w, dtype), part)
    g = np.full(3, 0.5, np.float32)
    dev = [_dev(gpu, x, dtype), part, gpu.from_numpy(t)]
    got = _check_forward(gpu, x, w, t, dtype, gpu.linear_cross_entropy(*dev))
    _check_backward(gpu, x, w, t, dtype, g, None, gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *got))


# d lies in groups of 64 words (32 for float32's planes): ends within, at and
# just past a group and a tile of words, and of rows
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", [(32, 63), (33, 65), (63, 255), (64, 256), (65, 257), (129, 511), (256, 1025), (300, 32)])
def test_gradient_at_the_edges_of_words_and_rows(gpu, R, V, dtype):
    x, w, t = _case(R, 40, V, dtype, seed=9)
    g = np.random.default_rng(V).random(R).astype(np.float32) / R
    _check_backward(gpu, x, w, t, dtype, g, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [80, 83, 86, 120])
def test_all_but_certain_rows_of_large_weight(gpu, gap, dtype):
    """1 - p of every target is about exp(-gap), down to nothing: gradients of
    that size, finite whatever the weights.  Off by lse's rounding (gap 2^-24),
    the exponent's (1.5 gap 2^-24) and exp2's below float32's normal range."""
    x, w = np.full((3, 1), gap, np.float32), np.array([[1.0], [0.0]], np.float32)
    t, g = np.zeros(3, np.int32), np.full(3, 1000, np.float32)
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
    got = gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *gpu.linear_cross_entropy(*dev))
    for a, b in zip(got, O.linear_cross_entropy_backward(x, w, t, g, None)):
        bar = (2 * HALF_STEP[dtype] + 4 * gap * 2.0 ** -24) * np.abs(b) + 3 * 1000 * gap * 2.0 ** -126
        assert (np.abs(a.to_numpy() - b) <= bar + (2.0 ** -25 if dtype == "float16" else 0)).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_even_weights_are_not_rounded(gpu, dtype):
    """Rows of one weight g have d = g (p - 1) of their targets alike, whose
    rounding, the same in every row, no sum would take back: dw of a word that
    is the target of some is off by its own rounding and by what p and the
    other words' parts are rounded by, also for a g between two 16-bit values."""
    R, K, V = 96, 64, 4096
    u, rng = HALF_STEP[dtype], np.random.default_rng(5)
    x = few_bits.round_to(rng.standard_normal((R, K)), dtype)
    w = few_bits.round_to(rng.standard_normal((V, K)) * 2.0 ** -12, dtype)   # p is near 1 / V everywhere
    t = (np.arange(R) % 24 * 7).astype(np.int32)
    g = np.full(R, 1 + 0.9 * u, np.float32)
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
    dw = gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *gpu.linear_cross_entropy(*dev))[1].to_numpy()
    want = O.linear_cross_entropy_backward(x, w, t, g, None)[1]
    d = O.logit_gradients(x, w, t, g, None)
    hit = d < 0
    # targets' d lie within 2^-18 of the largest, which is held as it is: less
    # than half a step of 16 bits below it, so they are held as the largest
    assert 1 - d[hit].max() / d[hit].min() < 2.0 ** -18
    err = (np.abs(d) * np.where(hit, 2.0 ** -18, 1.01 * u)).T @ np.abs(x).astype(np.float64)
    assert (np.abs(dw - want) <= u * np.abs(want) * (1 + u) + err + 2.0 ** -20 * (np.abs(d).T @ np.abs(x))).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("R,words", [(1, 1), (3, 1), (5, 5), (20, 7), (31, 31), (32, 2)])
def test_few_rows_lose_nothing(gpu, R, words, dtype):
    """dw of up to 32 rows is off by its own rounding and by what the parts of
    words that are no targets are rounded by; the targets' parts, the largest,
    are given back."""
    K, V = 72, 4096
    u, rng = HALF_STEP[dtype], np.random.default_rng(R + words)
    x = few_bits.round_to(rng.standard_normal((R, K)), dtype)
    w = few_bits.round_to(rng.standard_normal((V, K)) * 2.0 ** -12, dtype)
    t = (rng.permutation(R) % words * 13).astype(np.int32)
    t[rng.random(R) < 0.05] = -1
    g = (rng.random(R) + 0.5).astype(np.float32)
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
    dw = gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *gpu.linear_cross_entropy(*dev))[1].to_numpy()
    want = O.linear_cross_entropy_backward(x, w, t, g, None)[1]
    d = O.logit_gradients(x, w, t, g, None)
    err = (np.abs(d) * np.where(d < 0, 2.0 ** -20, 1.01 * u)).T @ np.abs(x).astype(np.float64)
    # float16 values below 2^-14 are 2^-24 apart, not 2^-10 of themselves: words
    # that are no targets have |dw| of g p |x| = 1e-6 here, rounded by up to 2^-25
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0
    assert (np.abs(dw - want) <= u * np.abs(want) * (1 + u) + err + 2.0 ** -20 * (np.abs(d).T @ np.abs(x)) + tiny).all()


# few words and many rows: dw in parts
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,K,V", [(5000, 70, 30), (3001, 129, 200)])
def test_gradient_of_few_words(gpu, R, K, V, dtype):
    x, w, t = _case(R, K, V, dtype, seed=4)
    g = np.random.default_rng(V).random(R).astype(np.float32) / R
    got = _check_backward(gpu, x, w, t, dtype, g, None)
    again = _check_backward(gpu, x, w, t, dtype, g, None)
    for a, b in zip(got, again):
        np.testing.assert_array_equal(a.to_numpy(), b.to_numpy())


def test_most_rows(gpu):
    x, w, t = _case(1 << 20, 8, 5, "float16", seed=6)
    _check_backward(gpu, x, w, t, "float16", np.full(1 << 20, 2.0 ** -10, np.float32), None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_words(gpu, dtype):
    x, w, t = _case(2, 8, (1 << 21) + 3, dtype, seed=7)
    _check_forward(gpu, x, w, t, dtype)
    _check_backward(gpu, x, w, t, dtype, np.full(2, 0.5, np.float32), None)


def test_no_rows(gpu):
    for dtype in DTYPES:
        x, w = gpu.zeros([0, 8], dtype), gpu.zeros([5, 8], dtype)
        t = gpu.from_numpy(np.zeros(0, np.int32))
        loss, lse = gpu.linear_cross_entropy(x, w, t)
        assert loss.shape == lse.shape == [0]
        dx, dw = gpu.linear_cross_entropy_backward(gpu.zeros([0]), x, w, t, loss, lse)
        assert dx.shape == [0, 8] and (dw.to_numpy() == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_targets_that_are_no_words(gpu, dtype):
    """No target at all: the losses are 0 and lse is there; the gradient of the
    loss is zero, that of lse is p's."""
    x, w, t = _case(9, 24, 50, dtype)
    for bad in (-100, -1, 50, 2 ** 31 - 1):
        t[:] = bad
        _check_forward(gpu, x, w, t, dtype)
        g, h = np.ones(9, np.float32), np.full(9, 0.1, np.float32)
        dx, dw = _check_backward(gpu, x, w, t, dtype, g, None)
        assert (dx.to_numpy() == 0).all() and (dw.to_numpy() == 0).all()
        _check_backward(gpu, x, w, t, dtype, g, h)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_what_is_not_finite_stays_in_its_row(gpu, dtype):
    x, w, t = _case(70, 64, 300, dtype)
    want = [a.to_numpy() for a in gpu.linear_cross_entropy(_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t))]
    bad = x.copy()
    bad[3, 5], bad[40, 0] = np.nan, np.inf
    t[40] = 7
    loss, lse = gpu.linear_cross_entropy(_dev(gpu, bad, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t))
    rest = np.setdiff1d(np.arange(70), [3, 40])
    for a, b in zip((loss, lse), want):
        got = a.to_numpy()
        assert np.isnan(got[[3, 40]][(t[[3, 40]] >= 0) | (a is lse)]).all()
        np.testing.assert_array_equal(got[rest], b[rest])
    # rows without weight: their gradient is zero whatever they hold
    t[[3, 40]] = -100
    g = np.full(70, 0.01, np.float32)
    dx, _ = gpu.linear_cross_entropy_backward(_dev(gpu, g), _dev(gpu, bad, dtype), _dev(gpu, w, dtype),
                                              gpu.from_numpy(t), loss, lse)
    dx = dx.to_numpy()
    assert (dx[[3, 40]] == 0).all() and np.isfinite(dx).all()


def test_words_ruled_out(gpu):
    """A weight row that gives -inf has no part in the sum; as a target its
    loss is infinite."""
    for dtype in ("float16", "bfloat16"):
        x, w, t = _case(6, 16, 40, dtype)
        x = np.abs(x) + 0.25
        x = few_bits.round_to(x, dtype)
        w[7] = -np.inf
        t[:] = [0, 1, 7, 2, -100, 3]
        loss, lse = (a.to_numpy() for a in gpu.linear_cross_entropy(_dev(gpu, x, dtype), _dev(gpu, w, dtype),
                                                                    gpu.from_numpy(t)))
        keep = np.delete(np.arange(40), 7)
        want = O.linear_cross_entropy(x, w[keep], np.where(t > 7, t - 1, t))
        rows = [0, 1, 3, 4, 5]
        np.testing.assert_allclose(loss[rows], want[0][rows], rtol=1e-4, atol=1e-4)
        np.testing.assert_allclose(lse, want[1], rtol=1e-5, atol=1e-4)
        assert np.isposinf(loss[2])


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e25])
def test_float32_of_any_size(gpu, size):
    """Operands far from 1 whose products are ordinary keep their 22 bits."""
    x, w, t = _case(40, 48, 70, "float32")
    x, w = (x * np.float32(size)).astype(np.float32), (w / np.float32(size)).astype(np.float32)
    _check_forward(gpu, x, w, t, "float32")
    g = np.random.default_rng(3).random(40).astype(np.float32)
    dev = [_dev(gpu, x), _dev(gpu, w), gpu.from_numpy(t)]
    loss, lse = gpu.linear_cross_entropy(*dev)
    dx, dw = (a.to_numpy() for a in gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, loss, lse))
    want = O.linear_cross_entropy_backward(x, w, t, g)
    for a, b in zip((dx, dw), want):
        assert np.linalg.norm(a - b) <= 1e-5 * np.linalg.norm(b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_any_size(gpu, dtype):
    """Weights of the rows far from 1, and unlike: what fp16 holds goes by the
    largest."""
    x, w, t = _case(33, 40, 200, dtype)
    for scale in (1e-20, 1e-6, 1e3):
        g = np.random.default_rng(4).random(33).astype(np.float32) * np.float32(scale)
        dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
        loss, lse = gpu.linear_cross_entropy(*dev)
        dx, dw = (a.to_numpy().astype(np.float64) for a in gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, loss, lse))
        want = O.linear_cross_entropy_backward(x, w, t, g)
        small = 6e-8 if dtype == "float16" else 0.0   # below float16's smallest step
        for a, b in zip((dx, dw), want):
            bar = 6 * HALF_STEP[dtype] if dtype != "float32" else 1e-5
            assert np.linalg.norm(a - b) <= bar * np.linalg.norm(b) + small * np.sqrt(b.size)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nearly_certain_words_keep_their_digits(gpu, dtype):
    """Losses down to 1e-30 and the gradients that go with them."""
    V, K = 40, 32
    w = np.eye(V, K, dtype=np.float32)
    x = np.zeros((4, K), np.float32)
    t = np.array([3, 5, 7, 9], np.int32)
    for r, size in enumerate((8.0, 20.0, 40.0, 64.0)):
        x[r, t[r]] = size
    loss, lse = gpu.linear_cross_entropy(_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t))
    want = O.linear_cross_entropy(x, w, t)
    # an exponent is off by 2^-24 of its size, once for the sum and once for its reference
    np.testing.assert_allclose(loss.to_numpy(), want[0], rtol=64 * 2.0 ** -22)
    for r in range(4):   # one row alone: what fp16 holds goes by the largest
        sel = slice(r, r + 1)
        dev = [_dev(gpu, x[sel], dtype), _dev(gpu, w, dtype), gpu.from_numpy(t[sel])]
        loss1, lse1 = gpu.linear_cross_entropy(*dev)
        g = np.ones(1, np.float32)
        dx, _ = gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, loss1, lse1)
        d = O.logit_gradients(x[sel], w, t[sel], g)[0]
        got = dx.to_numpy()[0]
        if dtype != "float16":
            np.testing.assert_allclose(got[t[r]], d[t[r]], rtol=2.0 ** -7 if dtype == "bfloat16" else 1e-4)
        else:   # d times 2^13 in float16, the result in float16
            np.testing.assert_allclose(got[t[r]], d[t[r]], rtol=2.0 ** -10, atol=6e-8)


# ── sizes past one piece ────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype,R,V", [("bfloat16", 33000, 17000), ("float16", 33001, 17003), ("float32", 17000, 17000)])
def test_vocabulary_in_pieces(gpu, dtype, R, V):
    """More logits than are held at once: sums over the vocabulary in pieces,
    against float64 some rows at a time."""
    import torch
    K = 16
    rng = np.random.default_rng(R)
    w = few_bits.round_to(rng.standard_normal((V, K)), dtype)
    t = rng.integers(0, V, R)
    x = few_bits.round_to(rng.standard_normal((R, K)) + w[t], dtype)
    t[::17] = -100
    g = rng.random(R).astype(np.float32)
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t.astype(np.int32))]
    loss, lse = gpu.linear_cross_entropy(*dev)
    dx, dw = (a.to_numpy().astype(np.float64) for a in gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, loss, lse))
    tw = torch.tensor(w, dtype=torch.float64)
    want_l, want_x, want_w = [], [], torch.zeros_like(tw)
    for lo in range(0, R, 2048):
        xi = torch.tensor(x[lo:lo + 2048], dtype=torch.float64)
        ti, gi = torch.tensor(t[lo:lo + 2048]), torch.tensor(g[lo:lo + 2048]).double()
        z = xi @ tw.t()
        s = torch.logsumexp(z, 1)
        d = torch.exp(z - s[:, None])
        there = ti >= 0
        row = torch.arange(len(ti))[there]
        want_l.append(torch.where(there, s - z.gather(1, ti.clamp(min=0)[:, None])[:, 0], 0.0))
        d[row, ti[there]] -= 1.0
        d *= torch.where(there, gi, 0.0)[:, None]
        want_x.append(d @ tw)
        want_w += d.t().contiguous() @ xi
    for a, b, bar in ((loss.to_numpy(), torch.cat(want_l), 1e-5), (dx, torch.cat(want_x), 4 * HALF_STEP[dtype] + 1e-5),
                      (dw, want_w, 4 * HALF_STEP[dtype] + 1e-5)):
        b = b.cpu().numpy()
        assert np.linalg.norm(a - b) <= bar * np.linalg.norm(b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_vs_differences(gpu, dtype):
    """The gradient's direction against the loss's own differences along it."""
    x, w, t = _case(20, 32, 60, dtype)
    g = np.random.default_rng(5).random(20).astype(np.float32)
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
    out = gpu.linear_cross_entropy(*dev)
    dx, dw = (a.to_numpy().astype(np.float64) for a in gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *out))

    def value(a, b):
        return (g * O.linear_cross_entropy(a, b, t)[0]).sum()

    for a, d, f in ((x, dx, lambda v: value(v, w)), (w, dw, lambda v: value(x, v))):
        h = 1e-6 / np.abs(d).max()
        slope = (f(a + h * d) - f(a - h * d)) / (2 * h)
        assert abs(slope - (d * d).sum()) <= (8 * HALF_STEP[dtype] + 1e-5) * (d * d).sum()


def test_same_bits_every_time(gpu):
    for dtype in DTYPES:
        x, w, t = _case(300, 64, 2000, dtype)
        g = np.ones(300, np.float32)
        first = None
        for _ in range(3):
            dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
            out = gpu.linear_cross_entropy(*dev)
            got = [a.to_numpy() for a in (*out, *gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *out))]
            for a, b in zip(got, first or got):
                np.testing.assert_array_equal(a, b)
            first = first or got


def test_refusals(gpu):
    x, w = gpu.zeros([4, 8]), gpu.zeros([5, 8])
    t = gpu.from_numpy(np.zeros(4, np.int32))
    with pytest.raises(ValueError, match="Dtype mismatch"):
        gpu.linear_cross_entropy(x, gpu.zeros([5, 8], "float16"), t)
    with pytest.raises(ValueError, match="does not match weight"):
        gpu.linear_cross_entropy(x, gpu.zeros([5, 9]), t)
    with pytest.raises(ValueError, match="does not match weight"):
        gpu.linear_cross_entropy(x, gpu.zeros([8]), t)
    with pytest.raises(ValueError, match="int32 or int64"):
        gpu.linear_cross_entropy(x, w, gpu.zeros([4]))
    with pytest.raises(ValueError, match="do not match x"):
        gpu.linear_cross_entropy(x, w, gpu.from_numpy(np.zeros(3, np.int32)))
    with pytest.raises(ValueError, match="do not match x"):
        gpu.linear_cross_entropy(x, w, gpu.from_numpy(np.zeros((2, 2), np.int32)))
    with pytest.raises(ValueError, match="0 words"):
        gpu.linear_cross_entropy(x, gpu.zeros([0, 8]), t)
    with pytest.raises(ValueError, match="linear_cross_entropy"):
        gpu.linear_cross_entropy(gpu.cast(x, "int32"), gpu.cast(w, "int32"), t)
    loss, lse = gpu.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="grad_loss must be float32"):
        gpu.linear_cross_entropy_backward(gpu.zeros([4], "float16"), x, w, t, loss, lse)
    with pytest.raises(ValueError, match="lse must be float32"):
        gpu.linear_cross_entropy_backward(gpu.zeros([4]), x, w, t, loss, gpu.zeros([3]))
    with pytest.raises(ValueError, match="grad_lse must be float32"):
        gpu.linear_cross_entropy_backward(gpu.zeros([4]), x, w, t, loss, lse, grad_lse=gpu.zeros([2]))
    rows = (1 << 20) + 1
    many = gpu.zeros([rows])
    with pytest.raises(ValueError, match="rows at once"):
        gpu.linear_cross_entropy_backward(many, gpu.zeros([rows, 1]), gpu.zeros([2, 1]),
                                          gpu.from_numpy(np.zeros(rows, np.int32)), many, many)
