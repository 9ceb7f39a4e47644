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


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
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


# ── float32 operands whose rows are far apart ───────────────────────────────
# Rows hold 22 bits of each value and no less than 2^-24 of the row's largest;
# where rows are further apart than that allows, 24 bits.  Sums of K products:
# one rounding each at most.
def _far_logit_bar(x, w):
    ax, aw = np.abs(x).astype(np.float64), np.abs(w).astype(np.float64)
    held = 2.0 ** -24 * (ax.max(1)[:, None] * aw.sum(1)[None, :] + ax.sum(1)[:, None] * aw.max(1)[None, :])
    return (x.shape[1] + 16) * 2.0 ** -24 * (ax @ aw.T) + 3 * 2.0 ** -22 * (ax @ aw.T) + held


def _far_check(gpu, x, w, t, g, seen):
    """Loss and gradient of the rows with weight, by the words in `seen` (the
    others are ruled out: p is 0)."""
    dev = [_dev(gpu, x), _dev(gpu, w), gpu.from_numpy(t)]
    out = gpu.linear_cross_entropy(*dev)
    dx, dw = (a.to_numpy().astype(np.float64) for a in gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *out))
    loss, lse = (a.to_numpy() for a in out)
    rows = np.flatnonzero(g)
    place = np.full(len(w), -100)
    place[seen] = np.arange(len(seen))
    xs, ws, ts = x[rows], w[seen], place[t[rows]]
    want = O.linear_cross_entropy(xs, ws, ts)
    z = _far_logit_bar(xs, ws)
    top = z.max(1)
    bar = 2 * top + 24 * 2.0 ** -20
    assert (np.abs(loss[rows] - want[0]) <= bar * np.minimum(1.0, 2 * want[0]) * np.exp(2 * top) + 2.0 ** -23 * want[0]).all()
    assert (np.abs(lse[rows] - want[1]) <= top + 21 * 2.0 ** -20 + 2.0 ** -23 * np.abs(want[1])).all()
    rdx, rdw = O.linear_cross_entropy_backward(xs, ws, ts, g[rows])
    d = np.abs(O.logit_gradients(xs, ws, ts, g[rows]))
    d_err = d * (z + top[:, None] + 46 * 2.0 ** -20 + 2.0 ** -23 * np.abs(want[1])[:, None]) + 2.0 ** -37 * g.max()
    ax, aw = np.abs(xs).astype(np.float64), np.abs(ws).astype(np.float64)
    sums = (len(seen) + len(rows) + 48) * 2.0 ** -24 + 3 * 2.0 ** -22
    # a value of an operand is off by at most 2^-24 of its row's largest
    bx = d_err @ aw + sums * (d @ aw) + 2.0 ** -24 * (d @ aw.max(1))[:, None]
    bw = d_err.T @ ax + sums * (d.T @ ax) + 2.0 ** -24 * (d.T @ ax.max(1))[:, None]
    assert (np.abs(dx[rows] - rdx) <= bx).all()
    assert (np.abs(dw[seen] - rdw) <= bw).all()
    rest = np.setdiff1d(np.arange(len(w)), seen)
    assert (dw[rest] == 0).all() and (dx[g == 0] == 0).all()


FAR = [(1, 8, 5), (5, 33, 70), (40, 48, 300), (64, 100, 257), (200, 64, 1000), (330, 40, 600), (513, 129, 130), (3000, 20, 40)]


@pytest.mark.parametrize("R,K,V", FAR)
@pytest.mark.parametrize("far", [2.0 ** 13, 2.0 ** 20, 2.0 ** 27, 2.0 ** 40, 2.0 ** 100])
def test_one_row_far_above_the_others(gpu, R, K, V, far):
    """What a padding row holds takes nothing from the other rows."""
    rng = np.random.default_rng(R + K)
    x, w = rng.standard_normal((R + 1, K)).astype(np.float32), rng.standard_normal((V, K)).astype(np.float32)
    t, g = rng.integers(0, V, R + 1).astype(np.int32), (rng.random(R + 1) / R + 0.01).astype(np.float32)
    x[R // 2] *= np.float32(far)
    t[R // 2], g[R // 2] = -100, 0
    _far_check(gpu, x, w, t, g, np.arange(V))


@pytest.mark.parametrize("R,K,V", FAR)
@pytest.mark.parametrize("far", [2.0 ** 13, 2.0 ** 20, 2.0 ** 27, 2.0 ** 40, 2.0 ** 100])
def test_one_word_far_below_the_others(gpu, R, K, V, far):
    """A word that large values rule out in every row."""
    rng = np.random.default_rng(R + K + 1)
    x, w = rng.standard_normal((R, K)).astype(np.float32), rng.standard_normal((V + 1, K)).astype(np.float32)
    t, g = rng.integers(0, V, R).astype(np.int32), (rng.random(R) / R + 0.01).astype(np.float32)
    x[:, 0] = np.abs(x[:, 0]) + 0.5
    w[V] = 0
    w[V, 0] = -far
    _far_check(gpu, x, w, t, g, np.arange(V))


@pytest.mark.parametrize("R,K,V", FAR)
def test_rows_far_below_the_others(gpu, R, K, V):
    """Rows and words of 2^-30 of the others keep their bits."""
    rng = np.random.default_rng(R + K + 2)
    x, w = rng.standard_normal((R, K)).astype(np.float32), rng.standard_normal((V, K)).astype(np.float32)
    t, g = rng.integers(0, V, R).astype(np.int32), (rng.random(R) / R + 0.01).astype(np.float32)
    x[::3] *= np.float32(2.0 ** -30)
    w[1::5] *= np.float32(2.0 ** -30)
    _far_check(gpu, x, w, t, g, np.arange(V))


@pytest.mark.parametrize("R", [3, 200, 400])
def test_words_ruled_out_in_float32(gpu, R):
    """A float32 weight row that gives -inf has no part in the sum either."""
    rng = np.random.default_rng(R)
    x, w = np.abs(rng.standard_normal((R, 16))).astype(np.float32) + 0.25, rng.standard_normal((40, 16)).astype(np.float32)
    w[7] = -np.inf
    t = np.where(np.arange(R) % 3 == 0, 7, np.where(np.arange(R) % 3 == 1, 8, -100)).astype(np.int32)
    loss, lse = (a.to_numpy() for a in gpu.linear_cross_entropy(_dev(gpu, x), _dev(gpu, w), gpu.from_numpy(t)))
    want = O.linear_cross_entropy(x, np.delete(w, 7, 0), np.where(t == 8, 7, -100))
    np.testing.assert_allclose(lse, want[1], rtol=1e-6, atol=1e-5)
    np.testing.assert_allclose(loss[t != 7], want[0][t != 7], rtol=1e-5, atol=1e-5)
    assert np.isposinf(loss[t == 7]).all()


@pytest.mark.parametrize("R,K,V", [(17000, 16, 17000), (2100, 72, 9000)])
def test_many_rows_far_apart(gpu, R, K, V):
    """Whole rounds of large tiles, and the vocabulary in pieces, with products of
    the float32 values: a row of 2^40 times the others without weight, a third of
    them of 2^-30, against float64 some rows at a time."""
    import torch
    rng = np.random.default_rng(R)
    x, w = rng.standard_normal((R, K)).astype(np.float32), rng.standard_normal((V, K)).astype(np.float32)
    t, g = rng.integers(0, V, R).astype(np.int32), rng.random(R).astype(np.float32)
    x[::3] *= np.float32(2.0 ** -30)
    x[R // 2] *= np.float32(2.0 ** 40)
    t[R // 2] = -100
    dev = [_dev(gpu, x), _dev(gpu, w), gpu.from_numpy(t)]
    out = gpu.linear_cross_entropy(*dev)
    dx, dw = (a.to_numpy().astype(np.float64) for a in gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *out))
    tw = torch.tensor(w, dtype=torch.float64)
    loss, want_x, want_w = [], [], torch.zeros_like(tw)
    for lo in range(0, R, 2048):
        xi, ti = torch.tensor(x[lo:lo + 2048], dtype=torch.float64), torch.tensor(t[lo:lo + 2048]).long()
        z = xi @ tw.t()
        s = torch.logsumexp(z, 1)
        there = ti >= 0
        loss.append(torch.where(there, s - z.gather(1, ti.clamp(min=0)[:, None])[:, 0], 0.0))
        d = torch.exp(z - s[:, None])
        row = torch.arange(len(ti))[there]
        d[row, ti[there]] -= 1.0
        d *= torch.where(there, torch.tensor(g[lo:lo + 2048]).double(), 0.0)[:, None]
        want_x.append(d @ tw)
        want_w += d.t().contiguous() @ xi
    np.testing.assert_allclose(out[0].to_numpy(), torch.cat(loss).numpy(), rtol=1e-5, atol=1e-5)
    want_x = torch.cat(want_x).numpy()
    # row by row: p's error, 46 2^-20 at most, and the sums'
    bad = np.linalg.norm(dx - want_x, axis=1) > 1e-4 * np.linalg.norm(want_x, axis=1)
    assert not bad.any()
    assert np.linalg.norm(dw - want_w.numpy()) <= 1e-4 * np.linalg.norm(want_w.numpy())


@pytest.mark.parametrize("R,K,V", [(5, 33, 70), (40, 48, 300), (330, 40, 600)])
@pytest.mark.parametrize("size", [2.0 ** -124, 2.0 ** -115, 2.0 ** -100, 2.0 ** -80, 2.0 ** 80, 2.0 ** 100, 2.0 ** 115, 2.0 ** 124])
def test_float32_of_the_ends(gpu, R, K, V, size):
    """Operands near the ends of float32 whose products are ordinary."""
    rng = np.random.default_rng(R + K + 3)
    x = rng.uniform(0.5, 1.0, (R, K)).astype(np.float32) * rng.choice([-1, 1], (R, K)).astype(np.float32)
    w = rng.uniform(0.5, 1.0, (V, K)).astype(np.float32) * rng.choice([-1, 1], (V, K)).astype(np.float32)
    x, w = x * np.float32(size), w / np.float32(size)
    t, g = rng.integers(0, V, R).astype(np.int32), (rng.random(R) / R + 0.01).astype(np.float32)
    dev = [_dev(gpu, x), _dev(gpu, w), gpu.from_numpy(t)]
    out = gpu.linear_cross_entropy(*dev)
    loss, lse = (a.to_numpy() for a in out)
    want = O.linear_cross_entropy(x, w, t)
    z = _far_logit_bar(x, w).max(1)
    bar = 2 * z + 24 * 2.0 ** -20
    assert (np.abs(loss - want[0]) <= bar * np.minimum(1.0, 2 * want[0]) * np.exp(2 * z) + 2.0 ** -23 * want[0]).all()
    assert (np.abs(lse - want[1]) <= z + 21 * 2.0 ** -20 + 2.0 ** -23 * np.abs(want[1])).all()
    d = np.abs(O.logit_gradients(x, w, t, g))
    d_err = d * (2 * z[:, None] + 46 * 2.0 ** -20 + 2.0 ** -23 * np.abs(want[1])[:, None]) + 2.0 ** -37 * g.max()
    ax, aw = np.abs(x).astype(np.float64), np.abs(w).astype(np.float64)
    sums = (R + V + 48) * 2.0 ** -24 + 3 * 2.0 ** -22 + 2.0 ** -24
    got = gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *out)
    for a, b, e, s in zip(got, O.linear_cross_entropy_backward(x, w, t, g), (d_err @ aw, d_err.T @ ax), (d @ aw, d.T @ ax)):
        # (results may lie below float32's normal range)
        assert (np.abs(a.to_numpy() - b) <= e + sums * s + 2.0 ** -149 * 1024).all()


# ── logits that are large and finite ────────────────────────────────────────
def _large(R, V, size, dtype, twice, seed):
    """Operands whose logits are exact: up to `size` in most rows and a sixteenth
    of it apart, ordinary in one.  The largest word is there twice or once."""
    if dtype == "float16" and size > 2.0 ** 31:
        size = 2.0 ** 29
    root = 2.0 ** (np.floor(np.log2(size)) // 2)
    rng = np.random.default_rng(seed)
    x, w = np.zeros((R, 8)), np.zeros((V, 8))
    x[:, 0] = root
    w[:, 0] = root * rng.choice([-0.75, -0.5, -0.25, 0.0, 0.25, 0.5], V)
    words = rng.permutation(V)
    top, low = words[:2], words[2]
    w[top if twice else top[:1], 0] = root
    if not twice:
        w[low, 0] = -root              # the one that is the largest of the row that looks the other way
    x[R // 3, 0] = -root
    x[R // 2, :2] = 0, 1.0             # a row of ordinary logits
    w[:, 1] = rng.integers(-3, 4, V)
    t = np.where(np.arange(R) % 3 == 0, top[0], rng.integers(0, V, R)).astype(np.int32)
    return x.astype(np.float32), w.astype(np.float32), t, rng


SIZES = [2.0 ** 15, 2.0 ** 21, 2.0 ** 24, 2.0 ** 31, 2.0 ** 60, 1e38]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("R,V", [(2, 3), (5, 900), (70, 300), (700, 130)])
def test_large_logits(gpu, R, V, size, dtype):
    """Losses and sums to their own rounding and that of the exponentials, 2^-20
    (1 + |d|) for exponents of up to 6 (the logits are exact); where two words
    share the largest, each has a loss of log 2."""
    x, w, t, _ = _large(R, V, size, dtype, True, R + V)
    loss, lse = (a.to_numpy() for a in gpu.linear_cross_entropy(_dev(gpu, x, dtype), _dev(gpu, w, dtype),
                                                                gpu.from_numpy(t)))
    want = O.linear_cross_entropy(x, w, t)
    np.testing.assert_allclose(lse, want[1], rtol=2.0 ** -20, atol=7 * 2.0 ** -20)
    np.testing.assert_allclose(loss, want[0], rtol=2.0 ** -20, atol=7 * 2.0 ** -20)
    top = [r for r in range(0, R, 3) if x[r, 0] > 0]
    np.testing.assert_allclose(loss[top], np.log(2), rtol=2.0 ** -19)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("R,V", [(2, 3), (5, 900), (70, 300), (700, 130)])
def test_gradient_of_large_logits(gpu, R, V, size, dtype):
    """One word is the largest by far: p is 0 or 1 but in the row of ordinary
    logits, whose p is off by its exponent's and the sum's 7 2^-20 each; d and the
    results are rounded once each."""
    x, w, t, rng = _large(R, V, size, dtype, False, R + V)
    g = (rng.random(R) + 0.5).astype(np.float32)
    dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
    dx, dw = (a.to_numpy().astype(np.float64) for a in
              gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *gpu.linear_cross_entropy(*dev)))
    d = O.logit_gradients(x, w, t, g)
    half = {"float32": 2.0 ** -22, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[dtype]
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0
    for got, want, of in ((dx, d @ w, np.abs(d) @ np.abs(w)), (dw, d.T @ x, np.abs(d).T @ np.abs(x))):
        fits = np.abs(want) < {"float16": 65504.0}.get(dtype, 3.3e38)   # (a sum past the type is infinite)
        assert (np.abs(got - want) <= of * (2 * half + 2.0 ** -16) + tiny)[fits].all()


def test_eager_entries(gpu):
    """The eager module's entries give the bits of the package's."""
    from applegpu_runtime import eager as E
    E.init()
    rng = np.random.default_rng(8)
    x, w = rng.standard_normal((9, 24)).astype(np.float32), rng.standard_normal((50, 24)).astype(np.float32)
    t, g = rng.integers(-1, 50, 9).astype(np.int32), rng.random(9).astype(np.float32)
    want = gpu.linear_cross_entropy(*map(gpu.from_numpy, (x, w, t)))
    got = E.linear_cross_entropy(*map(E.from_numpy, (x, w, t)))
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.numpy(), b.to_numpy())
    for h in (None, rng.standard_normal(9).astype(np.float32)):
        a = E.linear_cross_entropy_backward(*map(E.from_numpy, (g, x, w, t)), *got, None if h is None else E.from_numpy(h))
        b = gpu.linear_cross_entropy_backward(*map(gpu.from_numpy, (g, x, w, t)), *want,
                                              grad_lse=None if h is None else gpu.from_numpy(h))
        for u, v in zip(a, b):
            np.testing.assert_array_equal(u.numpy(), v.to_numpy())
    with pytest.raises(RuntimeError, match="differ in number"):
        E.muon_step_([E.from_numpy(x)], [], [])
    with pytest.raises(RuntimeError, match="must be float32 with one value a row"):
        E.linear_cross_entropy_backward(*map(E.from_numpy, (g[:8], x, w, t)), *got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_threads(gpu, dtype):
    """Calls of several threads at once, with workspaces: the bits of one."""
    from concurrent.futures import ThreadPoolExecutor
    rng = np.random.default_rng(9)
    x, w = rng.standard_normal((300, 64)).astype(np.float32), rng.standard_normal((2000, 64)).astype(np.float32)
    t, g = rng.integers(-1, 2000, 300).astype(np.int32), rng.random(300).astype(np.float32)

    def run(_):
        dev = [_dev(gpu, x, dtype), _dev(gpu, w, dtype), gpu.from_numpy(t)]
        out = gpu.linear_cross_entropy(*dev)
        return [a.to_numpy() for a in (*out, *gpu.linear_cross_entropy_backward(_dev(gpu, g), *dev, *out),
                                       gpu.orthogonalize(dev[1]))]

    want = run(0)
    with ThreadPoolExecutor(4) as pool:
        for got in pool.map(run, range(12)):
            for a, b in zip(got, want):
                np.testing.assert_array_equal(a, b)
