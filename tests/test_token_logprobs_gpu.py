"""Log probabilities of given tokens, entropies, alternatives and gradients on
the device, against float64.

Bars.  Each exponential is off by at most 2^-22 (1 + |d|) relative for an
exponent d (the float32 difference, its product with log2 e, the exponential),
so a log sum by 2^-22 (1 + mean |d|) and its own rounding, and the entropy, a
mean of d, by as much times its size; with mean |d| <= H + log V that gives
2^-20 (1 + H + |value|) + 2^-23 |max| for each of the three outputs.  Indices:
none.  Gradients: p is off by 2^-21 (2 + |log p| + |lse|) relative, and the
result is rounded once."""
import numpy as np
import pytest

from oracle import few_bits as O

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _dev(gpu, a, dtype="float32"):
    t = gpu.from_numpy(np.ascontiguousarray(a, np.float32))
    return t if dtype == "float32" else gpu.cast(t, dtype)


def _rows(rng, R, V, dtype, std=3.0):
    z = rng.standard_normal((R, V)).astype(np.float32) * std
    if V > 8:
        z[:, rng.integers(1, V, V // 8)] = -np.inf      # words ruled out
    tokens = rng.integers(0, V, R)
    tokens[rng.random(R) < 0.1] = -100
    return O.round_to(z, dtype), tokens.astype(np.int32)


def _close(got, want, H, top):
    bar = 2.0 ** -20 * (1 + np.where(np.isfinite(H), np.abs(H), 0) + np.abs(want)) + 2.0 ** -23 * np.abs(top)
    inf = np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf])
    assert (np.abs(got[~inf] - want[~inf]) <= np.broadcast_to(bar, want.shape)[~inf]).all()


def _check(gpu, z, tokens, top_k, dtype):
    got = [t.to_numpy() for t in gpu.token_logprobs(_dev(gpu, z, dtype), gpu.from_numpy(tokens), top_k=top_k)]
    want = O.token_logprobs(z, tokens, top_k)
    top = np.where(np.isfinite(z), z, 0).max(1)
    for g, w in zip(got[:3], want[:3]):
        assert g.dtype == np.float32 and g.shape == w.shape
        _close(g.astype(np.float64), w, want[1], top)
    if top_k:
        np.testing.assert_array_equal(got[4], want[4])
        _close(got[3].astype(np.float64), want[3], want[1][:, None], top[:, None])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("R,V,top_k", [(1, 1, 1), (3, 2, 2), (2, 63, 5), (5, 64, 32), (4, 255, 1), (2, 1000, 20),
                                       (3, 4097, 7), (1, 20011, 32), (9, 50257, 20), (300, 300, 3), (70, 8191, 0)])
def test_vs_oracle(gpu, dtype, R, V, top_k):
    z, tokens = _rows(np.random.default_rng(R + V), R, V, dtype)
    _check(gpu, z, tokens, top_k, dtype)


@pytest.mark.parametrize("V", [50257, 130000, 400001])
def test_long_rows(gpu, V):
    """Vocabularies past what a block holds in registers."""
    rng = np.random.default_rng(V)
    z, tokens = _rows(rng, 3, V, "bfloat16")
    _check(gpu, z, tokens, 20, "bfloat16")
    z, tokens = _rows(rng, 2, V, "float32")
    _check(gpu, z, tokens, 5, "float32")


def test_many_rows(gpu):
    """More rows than one grid dimension takes."""
    rng = np.random.default_rng(0)
    z, tokens = _rows(rng, 70000, 12, "float32")
    got = gpu.token_logprobs(gpu.from_numpy(z), gpu.from_numpy(tokens), top_k=2)
    at = np.r_[0:50, 65500:65600, 69950:70000]
    want = O.token_logprobs(z[at], tokens[at], 2)
    for g, w in zip(got[:3], want[:3]):
        _close(g.to_numpy()[at].astype(np.float64), w, want[1], 20.0)
    np.testing.assert_array_equal(got[4].to_numpy()[at], want[4])
    ones = gpu.from_numpy(np.ones(70000, np.float32))
    d = gpu.token_logprobs_backward(ones, None, gpu.from_numpy(z), gpu.from_numpy(tokens), got[1], got[2]).to_numpy()
    assert np.abs(d[at] - O.token_logprobs_backward(np.ones(len(at)), None, z[at], tokens[at])).max() <= 2.0 ** -18


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_orders_that_gather_the_largest(gpu, dtype):
    """Rising, falling and equal rows, ties across the row, and the largest
    all in one place: equal values by index, whatever the layout."""
    V = 6000
    rng = np.random.default_rng(1)
    up = np.linspace(-4, 4, V)
    z = np.stack([up, up[::-1], np.zeros(V), np.where(np.arange(V) % 2 == 0, 0.0, -0.0), np.repeat(up[::100], 100),
                  np.where((np.arange(V) > 3000) & (np.arange(V) < 3040), 5 + up, up - 5),
                  np.where(np.arange(V) % 64 == 7, 5.0, 0.0), rng.integers(0, 3, V).astype(float),
                  np.where(np.arange(V) == V - 1, 9.0, -np.inf), np.where(np.arange(V) < 10, np.arange(V), -np.inf)])
    z = O.round_to(z.astype(np.float32), dtype)
    tokens = np.array([0, 1, 5999, 3, 4, 3020, 7, 8, V - 1, 3], np.int32)
    for k in (1, 5, 32):
        _check(gpu, z, tokens, k, dtype)


def test_rows_without_a_word_and_with_nan(gpu):
    z = np.array([[-np.inf] * 70, [0.5] * 70, [0.5] * 70, [0.5] * 70], np.float32)
    z[1, 33], z[2, 2], z[3, 1] = np.nan, np.inf, -np.inf
    tokens = np.array([4, 5, -1, 1], np.int32)
    lp, H, lse, tl, ti = (t.to_numpy() for t in gpu.token_logprobs(gpu.from_numpy(z), gpu.from_numpy(tokens), top_k=3))
    assert lp[0] == lse[0] == -np.inf and H[0] == 0 and (tl[0] == -np.inf).all()
    assert np.isnan([lp[1], H[1], lse[1], H[2], lse[2]]).all() and lp[2] == 0
    assert lp[3] == -np.inf and np.isfinite(H[3])
    np.testing.assert_array_equal(ti, [[0, 1, 2], [33, 0, 1], [2, 0, 1], [0, 2, 3]])
    g = gpu.from_numpy(np.ones(4, np.float32))
    d = gpu.token_logprobs_backward(g, g, gpu.from_numpy(z), gpu.from_numpy(tokens), gpu.from_numpy(H),
                                    gpu.from_numpy(lse)).to_numpy()
    assert (d[0] == 0).all() and np.isnan(d[1]).all() and np.isfinite(d[3]).all()


def test_nearly_certain_rows_keep_their_digits(gpu):
    """One word with all but 1e-6 of the probability: the log probability and
    entropy are small numbers, relative to which the error is small."""
    z = np.zeros((2, 1000), np.float32)
    z[0, 3], z[1, 999] = 20.0, 24.0
    tokens = np.array([3, 999], np.int32)
    lp, H, _ = (t.to_numpy().astype(np.float64) for t in gpu.token_logprobs(gpu.from_numpy(z), gpu.from_numpy(tokens)))
    want = O.token_logprobs(z, tokens)
    assert (np.abs(lp - want[0]) <= 2.0 ** -17 * np.abs(want[0])).all()
    assert (np.abs(H - want[1]) <= 2.0 ** -17 * np.abs(want[1])).all()


def test_shapes_views_and_index_types(gpu):
    rng = np.random.default_rng(2)
    z, _ = _rows(rng, 12, 257, "float16")
    tokens = rng.integers(-1, 258, 12)
    want = O.token_logprobs(z, tokens, 2)
    big = np.zeros((12, 300), np.float16)
    big[:, 5:262] = z
    for zt in (gpu.from_numpy(z.astype(np.float16)), gpu.slice(gpu.from_numpy(big), 1, 5, 262),
               gpu.transpose(gpu.from_numpy(np.ascontiguousarray(z.T.astype(np.float16))))):
        for idx in (np.int32, np.int64):
            got = gpu.token_logprobs(zt, gpu.from_numpy(tokens.astype(idx)), top_k=2)
            _close(got[0].to_numpy().astype(np.float64), want[0], want[1], 15.0)
            np.testing.assert_array_equal(got[4].to_numpy(), want[4])
    got = gpu.token_logprobs(gpu.reshape(gpu.from_numpy(z.astype(np.float16)), [3, 4, 257]),
                             gpu.from_numpy(tokens.astype(np.int32).reshape(3, 4)), top_k=2)
    assert [t.shape for t in got] == [[3, 4]] * 3 + [[3, 4, 2]] * 2
    np.testing.assert_array_equal(got[4].to_numpy().reshape(12, 2), want[4])
    one = gpu.token_logprobs(gpu.from_numpy(z[0]), gpu.from_numpy(tokens[:1].astype(np.int32)))
    assert one[0].shape == [1]
    _close(one[2].to_numpy().astype(np.float64), want[2][:1], want[1][:1], 15.0)
    # an entry of int64 that only its low half would put inside the row
    far = gpu.from_numpy(np.array([2 ** 32 + 3], np.int64))
    assert gpu.token_logprobs(gpu.from_numpy(z[:1]), far)[0].to_numpy()[0] == 0


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (5, 257), (2, 4096), (4, 50257), (600, 33)])
@pytest.mark.parametrize("entropy", [True, False])
def test_gradients_vs_formula(gpu, dtype, R, V, entropy):
    rng = np.random.default_rng(R * V)
    z, tokens = _rows(rng, R, V, dtype)
    g, gh = rng.standard_normal((2, R)).astype(np.float32)
    gh = gh if entropy else None
    zt, t = _dev(gpu, z, dtype), gpu.from_numpy(tokens)
    _, H, lse = gpu.token_logprobs(zt, t)
    d = gpu.token_logprobs_backward(gpu.from_numpy(g), gpu.from_numpy(gh) if entropy else None, zt, t, H, lse)
    assert d.dtype == dtype and d.shape == [R, V]
    want = O.token_logprobs_backward(g, gh, z, tokens)
    _, Hw, lw, _, _ = O.token_logprobs(z, tokens)
    logp = z.astype(np.float64) - lw[:, None]
    p = np.exp(logp)
    logp = np.where(p > 0, logp, 0)
    rate = 2.0 ** -21 * (2 + np.abs(logp) + np.abs(lw)[:, None] + Hw[:, None])
    size = np.abs(g)[:, None] + (np.abs(gh)[:, None] * (1 + np.abs(logp + Hw[:, None])) if entropy else 0)
    bar = rate * p * size + 2.0 ** -22 * np.abs(g)[:, None] * (want != 0) + HALF_STEP[dtype] * np.abs(want)
    bar = bar + {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -133, "float32": 1e-37}[dtype]
    got = d.to_numpy().astype(np.float64)
    assert (np.abs(got - want) <= bar).all(), np.abs(got - want).max()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V,off", [(2, 0), (40, 0), (1000, 0), (1000, 1), (1000, 1024), (50257, 0), (50257, -64),
                                   (130001, 0)])
@pytest.mark.parametrize("view", [False, True])
def test_gradients_of_nearly_certain_rows_keep_their_digits(gpu, dtype, V, off, view):
    """One word with all but e^-8 .. e^-80 of the probability, and 3/4 and
    about; T = sum exp(z_i - z_j) of the others to 2^-21 (2 + |z_i - z_j|)
    relative gives 1 - p = T / (1 + T) and log p = -log1p(T) as well, whatever
    is added to the row; the entropy is given to 2^-17."""
    rng = np.random.default_rng(V)
    R = 12
    z = O.round_to(rng.standard_normal((R, V)).astype(np.float32), dtype)
    at = rng.integers(0, V, R)
    at[:3] = 0, V - 1, V // 2
    lift = np.array([8, 12, 16, 20, 24, 32, 80, 0.5, 1, 1.5, 2, 4], np.float32)
    z[np.arange(R), at] = lift + np.log(np.float32(V)) + 1
    z = O.round_to(z + off, dtype).astype(np.float64)
    tokens = np.where(np.arange(R) % 4 == 3, (at + 1) % V, at).astype(np.int32)
    tokens[5] = -100
    zj = z[np.arange(R), at][:, None]
    e = np.exp(z - zj)
    e[np.arange(R), at] = 0
    T = e.sum(1, keepdims=True)
    e[np.arange(R), at] = 1
    p, logp = e / (1 + T), (z - zj) - np.log1p(T)
    H = -(p * logp).sum(1, keepdims=True)
    g, gh = rng.standard_normal((2, R)).astype(np.float32)
    lse = (zj + np.log1p(T)).astype(np.float32)
    one = np.arange(V) == tokens[:, None]
    rest = np.where(one & (np.arange(V) == at[:, None]), T / (1 + T), one - p) * (tokens >= 0)[:, None]
    want = g[:, None] * rest - gh[:, None] * p * (logp + H)
    zt = _dev(gpu, z, dtype)
    if view:    # rows that begin anywhere
        zt = gpu.slice(_dev(gpu, np.pad(z, ((0, 0), (3, 6))), dtype), 1, 3, 3 + V)
    d = gpu.token_logprobs_backward(gpu.from_numpy(g), gpu.from_numpy(gh), zt, gpu.from_numpy(tokens),
                                    gpu.from_numpy(H[:, 0].astype(np.float32)), gpu.from_numpy(lse[:, 0]))
    got = d.to_numpy().astype(np.float64)
    rate = 2.0 ** -21 * (2 + np.where(p > 0, zj - z, 0) + np.abs(lse))
    size = np.abs(g)[:, None] * (1 + 2 * one) * p + np.abs(gh)[:, None] * p * (1 + np.abs(logp) + H)
    bar = rate * size
    # the certain element, and the token among the others
    sure = (np.arange(V) == at[:, None]) & (p > 0.75)
    far = np.where(p > 0, zj - z, 0).max(1, keepdims=True)
    tight = 2.0 ** -21 * (2 + far) * (np.abs(g)[:, None] * np.where(one, T, p) + np.abs(gh)[:, None] * p * (np.abs(logp) + H)) \
        + 2.0 ** -17 * np.abs(gh)[:, None] * p * H
    bar = np.where(sure, tight, bar + 2.0 ** -22 * np.abs(g)[:, None] * one)
    # (a p below float32's normal range may be taken as 0: an error of at most 2^-126 in it, times the gradients' factor,
    # and of V of them in T)
    bar = bar + 2.0 ** -126 * (np.abs(g)[:, None] + np.abs(gh)[:, None] * (1 + np.abs(logp) + H)) * np.where(sure, V, 1)
    bar = bar + HALF_STEP[dtype] * np.abs(want) + {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -133, "float32": 2.0 ** -149}[dtype]
    assert (np.abs(got - want) <= bar).all(), (np.abs(got - want) / bar).max()


def test_gradients_vs_differences(gpu):
    """Differences of the device's own outputs along a direction: the step is
    1/64, so a third derivative of at most 8 |direction|^3 adds 2^-12, and the
    outputs' errors (2^-20 each) 2^-14."""
    rng = np.random.default_rng(3)
    z = (rng.standard_normal((4, 40)) * 1.5).astype(np.float32)
    tokens = gpu.from_numpy(np.array([3, 0, 39, 7], np.int32))
    u = rng.standard_normal((4, 40))
    u /= np.linalg.norm(u, axis=1, keepdims=True)
    g = gpu.from_numpy(np.ones(4, np.float32))
    f = lambda a: [t.to_numpy().astype(np.float64) for t in gpu.token_logprobs(gpu.from_numpy(a), tokens)[:2]]  # noqa: E731
    h = 2.0 ** -6
    hi, lo = (f((z + s * h * u).astype(np.float32)) for s in (1, -1))
    zt = gpu.from_numpy(z)
    _, H, lse = gpu.token_logprobs(zt, tokens)
    none = gpu.from_numpy(np.zeros(4, np.float32))
    for i, pair in enumerate(((g, None), (none, g))):
        d = gpu.token_logprobs_backward(pair[0], pair[1], zt, tokens, H, lse).to_numpy().astype(np.float64)
        assert np.abs((hi[i] - lo[i]) / (2 * h) - (d * u).sum(1)).max() <= 2.0 ** -11


def test_captured_and_replayed(gpu):
    rng = np.random.default_rng(0)
    z, t = gpu.zeros([3, 50257], "float16"), gpu.zeros([3], "int32")
    z2, t2 = gpu.zeros([200, 777]), gpu.zeros([200], "int32")
    graphs = [gpu.capture(lambda: gpu.token_logprobs(z, t, top_k=5)), gpu.capture(lambda: gpu.token_logprobs(z2, t2, top_k=3))]
    for _ in range(4):
        for g, a, b in zip(graphs, (z, z2), (t, t2)):
            x, tokens = _rows(rng, *a.shape, "float16")
            a.write(x.astype(a.dtype))
            b.write(tokens)
            g.replay()
            eager = gpu.token_logprobs(_dev(gpu, x, a.dtype), gpu.from_numpy(tokens), top_k=g.outputs[3].shape[1])
            for p, q in zip(g.outputs, eager):
                np.testing.assert_array_equal(p.to_numpy(), q.to_numpy())
    for g in graphs:
        g.destroy()


def test_empty_and_refusals(gpu):
    z, t = gpu.zeros([2, 30]), gpu.zeros([2], "int32")
    out = gpu.token_logprobs(gpu.zeros([0, 30]), gpu.zeros([0], "int32"), top_k=2)
    assert [x.to_numpy().shape for x in out] == [(0,)] * 3 + [(0, 2)] * 2
    for bad in [dict(k=31), dict(k=33), dict(k=-1), dict(t=gpu.zeros([3], "int32")), dict(t=gpu.zeros([2])),
                dict(t=gpu.zeros([2, 1], "int32")), dict(z=gpu.zeros([2, 0])), dict(z=gpu.zeros([2, 30], "int32"))]:
        with pytest.raises(ValueError, match="token_logprobs"):
            gpu.token_logprobs(bad.get("z", z), bad.get("t", t), top_k=bad.get("k", 0))
    _, H, lse = gpu.token_logprobs(z, t)
    g = gpu.zeros([2])
    for bad in [dict(g=gpu.zeros([3])), dict(g=gpu.zeros([2], "float16")), dict(h=gpu.zeros([1])),
                dict(H=gpu.zeros([2], "int32")), dict(lse=gpu.zeros([4])), dict(t=gpu.zeros([3], "int32"))]:
        with pytest.raises(ValueError, match="token_logprobs_backward"):
            gpu.token_logprobs_backward(bad.get("g", g), bad.get("h"), z, bad.get("t", t), bad.get("H", H),
                                        bad.get("lse", lse))
