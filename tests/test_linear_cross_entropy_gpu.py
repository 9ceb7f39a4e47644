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
