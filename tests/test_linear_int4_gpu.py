"""Linear layers with 4-bit weights on the device, against float64.

Bars.  Codes, scales and dequantised values: none.  Products: codes are taken
as code + 16 in the matrix units and 24 of them is subtracted again, so that a
group of at most 128 terms loses at most 16 roundings of sums of 24 |x| s; the
groups, waves and the bias are added in float32, at most K / 32 + 32 of them:
2^-24 (16 * 24 + K / 32 + 32) sum |x| s.  float32 activations are split into
three 8-bit parts (2^-24 relative).  16-bit weights of many rows (more than 256
in the narrow matrices here, fewer in wide ones) may be rounded to the type
once: half a step of sum |x| |w|.  gelu has a
slope of at most 1.13.  The output is rounded once."""
import numpy as np
import pytest

from oracle import few_bits as O

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _dev(gpu, a, dtype="float32"):
    t = gpu.from_numpy(np.ascontiguousarray(a, np.float32))
    return t if dtype == "float32" else gpu.cast(t, dtype)


def _weights(rng, N, K, dtype):
    """Rows of unlike size, a row of zeros among them."""
    w = rng.standard_normal((N, K)).astype(np.float32) * np.exp(rng.standard_normal((N, 1))).astype(np.float32) * 0.05
    w[N // 2] = 0
    return O.round_to(w, dtype)


def _pack(codes):
    """O.pack_int4 without its loops."""
    N, K = codes.shape
    T, S = -(-N // 16), -(-K // 128)
    u = np.full((T * 16, S * 128), 8, np.uint8)
    u[:N, :K] = codes + 8
    u = u.reshape(T, 16, S, 4, 4, 4, 2).transpose(0, 2, 3, 1, 4, 6, 5).reshape(T, S, 64, 16, 2)
    return u[..., 0] | u[..., 1] << 4


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (16, 128, 128), (17, 33, 32), (40, 200, 64), (130, 259, 128),
                                       (33, 1280, 128)])
def test_quantize_bit_exact(gpu, dtype, N, K, group):
    rng = np.random.default_rng(N + K)
    w = _weights(rng, N, K, dtype)
    codes, scales = O.quantize_int4(w, group, dtype)
    for t in (_dev(gpu, w, dtype), gpu.transpose(_dev(gpu, w.T, dtype))):   # also read through strides
        packed, s = gpu.quantize_int4(t, group)
        assert packed.dtype == "uint8" and s.dtype == dtype
        np.testing.assert_array_equal(s.to_numpy().astype(np.float32), scales)
        np.testing.assert_array_equal(packed.to_numpy(), _pack(codes))
        if N * K < 20000:
            np.testing.assert_array_equal(packed.to_numpy(), O.pack_int4(codes))
        back = gpu.dequantize_int4(packed, s, K, group)
        assert back.dtype == dtype
        want = O.round_to(O.values_int4(codes, scales, group).astype(np.float32), dtype)
        np.testing.assert_array_equal(back.to_numpy().astype(np.float32), want)


def test_quantize_infinities(gpu):
    w = np.ones((20, 70), np.float32)
    w[3, 40], w[5, 2] = np.inf, np.nan
    packed, s = gpu.quantize_int4(gpu.from_numpy(w), 32)
    back = gpu.dequantize_int4(packed, s, 70, 32).to_numpy()
    bad = np.zeros((20, 70), bool)
    bad[3, 32:64] = bad[5, :32] = True
    np.testing.assert_array_equal(np.isnan(back), bad)
    assert np.abs(back[~bad] - 1).max() <= 2.0 ** -22
    x = np.ones((2, 70), np.float32)
    y = gpu.linear_int4(gpu.from_numpy(x), packed, s, group=32).to_numpy()
    np.testing.assert_array_equal(np.isnan(y).all(0), np.isin(np.arange(20), (3, 5)))
    assert not np.isnan(np.delete(y, (3, 5), 1)).any()


def _check(gpu, rng, dtype, M, N, K, group, act=None, bias=True, lead=None):
    w = _weights(rng, N, K, dtype)
    codes, scales = O.quantize_int4(w, group, dtype)
    x = O.round_to(rng.standard_normal((M, K)).astype(np.float32), dtype)
    b = O.round_to(rng.standard_normal(N).astype(np.float32), dtype) if bias else None
    packed, s = gpu.from_numpy(_pack(codes)), _dev(gpu, scales, dtype)
    xt = _dev(gpu, x.reshape(lead + [K]) if lead else x, dtype)
    y = gpu.linear_int4(xt, packed, s, _dev(gpu, b, dtype) if bias else None, act, group=group)
    assert y.shape == (lead or [M]) + [N] and y.dtype == dtype
    got = y.to_numpy().reshape(M, N).astype(np.float64)
    wv = O.values_int4(codes, scales, group)
    want = O.linear(x, wv, b, act)
    step = np.repeat(scales.T.astype(np.float64), group, 1)[:, :K]
    ax = np.abs(x).astype(np.float64)
    bar = 2.0 ** -24 * (16 * 24 + K / 32 + 32) * (ax @ step.T) + 2.0 ** -22 * (np.abs(b) if bias else 0)
    if dtype != "float32" and M > 256:
        bar += HALF_STEP[dtype] * (ax @ np.abs(wv).T)
    bar = 1.13 * bar + (HALF_STEP[dtype] + 2.0 ** -20) * np.abs(want) + (2.0 ** -25 if dtype == "float16" else 0)
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bar
    assert over.max() <= 0, (np.abs(got - want).max(), over.max(), np.unravel_index(over.argmax(), over.shape))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 130, 256, 257, 400])
@pytest.mark.parametrize("N,K,group", [(48, 256, 128), (33, 321, 32), (17, 64, 64)])
def test_rows_and_odd_sizes(gpu, dtype, M, N, K, group):
    _check(gpu, np.random.default_rng(M * N), dtype, M, N, K, group)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 5, 7), (1, 16, 31), (5, 15, 129), (1, 1000, 4100), (8, 3840, 1280),
                                   (1, 50257, 64), (4, 100, 8192)])
def test_sizes(gpu, dtype, M, N, K):
    for group in (32, 64, 128):
        _check(gpu, np.random.default_rng(N + K), dtype, M, N, K, group, bias=group != 64)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_exact"])
@pytest.mark.parametrize("M", [1, 20, 100, 300])
def test_epilogues(gpu, dtype, act, M):
    _check(gpu, np.random.default_rng(7), dtype, M, 70, 300, 64, act, bias=act != "relu")


@pytest.mark.parametrize("dtype,M,N,K", [("float16", 1, 70, 300), ("bfloat16", 40, 70, 300), ("float16", 600, 999, 64),
                                         ("float32", 3, 70, 300), ("float32", 300, 70, 300), ("bfloat16", 2100, 999, 64)])
def test_relu_of_nan_and_infinities_is_the_frameworks(gpu, dtype, M, N, K):
    """The same, whatever kernels the number of rows takes: relu(NaN) = 0."""
    rng = np.random.default_rng(2)
    packed, s = gpu.quantize_int4(_dev(gpu, _weights(rng, N, K, dtype), dtype), 64)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0, 5], x[M - 1, 0] = np.nan, np.inf
    x = _dev(gpu, x, dtype)
    y = gpu.linear_int4(x, packed, s, None, "relu", group=64).to_numpy().astype(np.float32)
    want = gpu.relu(gpu.linear_int4(x, packed, s, group=64)).to_numpy().astype(np.float32)
    np.testing.assert_array_equal(y, want)
    assert (y[0] == 0).all() and not np.isnan(y).any()


def test_leading_dims_and_views(gpu):
    rng = np.random.default_rng(11)
    _check(gpu, rng, "float16", 6, 40, 96, 32, lead=[2, 3])
    _check(gpu, rng, "float16", 1, 40, 96, 32, lead=[])
    # rows that are a slice at an offset 16 bytes do not divide, and a transposed view
    w = _weights(rng, 40, 96, "float16")
    packed, s = gpu.quantize_int4(_dev(gpu, w, "float16"), 32)
    wv = gpu.dequantize_int4(packed, s, 96, 32).to_numpy().astype(np.float64)
    big = rng.standard_normal((5, 103)).astype(np.float16)
    for off in (0, 3, 7):
        y = gpu.linear_int4(gpu.slice(gpu.from_numpy(big), 1, off, off + 96), packed, s, group=32).to_numpy()
        want = big[:, off:off + 96].astype(np.float64) @ wv.T
        assert np.abs(y - want).max() <= 2.0 ** -11 * np.abs(want).max() + 1e-4
    t = gpu.linear_int4(gpu.transpose(gpu.from_numpy(np.ascontiguousarray(big[:, :96].T))), packed, s, group=32)
    np.testing.assert_array_equal(t.to_numpy(), gpu.linear_int4(gpu.from_numpy(big[:, :96].copy()), packed, s,
                                                                group=32).to_numpy())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("M", [1, 16, 80, 280])
def test_magnitudes_and_infinities_in_rows(gpu, dtype, M):
    """Rows of unlike size; an infinity or NaN in one row stays in that row."""
    rng = np.random.default_rng(M)
    N, K, group = 50, 160, 32
    w = _weights(rng, N, K, dtype)
    w[N // 2] = w[0]
    codes, scales = O.quantize_int4(w, group, dtype)
    x = rng.standard_normal((M, K)) * np.exp(rng.uniform(-8, 8, (M, 1)))
    x = O.round_to(x.astype(np.float32), dtype)
    wv = O.values_int4(codes, scales, group)
    want = O.linear(x, wv)
    if M > 1:
        x[1, 3], x[M - 1, 5] = np.inf, np.nan
    y = gpu.linear_int4(_dev(gpu, x, dtype), gpu.from_numpy(_pack(codes)), _dev(gpu, scales, dtype), group=group)
    y = y.to_numpy().astype(np.float64)
    good = np.ones(M, bool)
    if M > 1:
        good[[1, M - 1]] = False
        assert not np.isfinite(y[~good]).any()
    ax = np.abs(np.where(np.isfinite(x), x, 0)).astype(np.float64)
    step = np.repeat(scales.T.astype(np.float64), group, 1)[:, :K]
    bar = 2.0 ** -24 * (16 * 24 + K / 32 + 32) * (ax @ step.T) + (HALF_STEP[dtype] + 2.0 ** -20) * np.abs(want)
    bar = bar + (HALF_STEP[dtype] * (ax @ np.abs(wv).T) if M > 256 else 0) + (2.0 ** -25 if dtype == "float16" else 0)
    # The largest rows pass float16's range: 65520 is halfway to the step after the largest value, so an exact
    # value further from it than the bar above has to be an infinity of its sign, or has to be finite.
    top = 65520.0 if dtype == "float16" else np.inf
    inf = np.isinf(y)
    assert (np.sign(y) == np.sign(want))[good & inf.any(1)][inf[good & inf.any(1)]].all()
    assert (np.abs(want) + bar >= top)[inf & good[:, None]].all()
    assert inf[(np.abs(want) - bar > top) & good[:, None]].all()
    assert (np.abs(y - want) <= bar)[good[:, None] & ~inf].all()


def test_captured_and_replayed(gpu):
    rng = np.random.default_rng(0)
    w = _weights(rng, 96, 256, "float16")
    packed, s = gpu.quantize_int4(_dev(gpu, w, "float16"), 64)
    gpu.eval_many([packed, s])
    graphs = []
    for M in (4, 100, 300):
        x = gpu.zeros([M, 256], "float16")
        graphs.append((x, gpu.capture(lambda x=x: gpu.linear_int4(x, packed, s, group=64))))
    for _ in range(4):
        for x, g in graphs:
            a = rng.standard_normal(x.shape).astype(np.float16)
            x.write(a)
            g.replay()
            np.testing.assert_array_equal(g.outputs.to_numpy(),
                                          gpu.linear_int4(gpu.from_numpy(a), packed, s, group=64).to_numpy())
    for _, g in graphs:
        g.destroy()


# ── many 16-bit rows ────────────────────────────────────────────────────────
# Sizes that take row tiles of 64, 96, 128 and 160 (256 compute units), last
# columns and rows that fill no tile, K that fills no stage of 64, and rows that
# are padded to whole vectors first; then sizes for which the weights become
# values in memory (a long K with few tiles, and very many rows).
MANY = [(520, 999, 200, 32), (1100, 2001, 72, 64), (1540, 2001, 136, 128), (1900, 2200, 64, 32), (257, 8200, 131, 64),
        (40, 21000, 64, 128), (700, 1024, 4130, 128), (4200, 200, 72, 32)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,N,K,group", MANY)
def test_many_rows(gpu, dtype, M, N, K, group):
    """The weights are rounded to the type (half a step of sum |x| |w|, or 2^-25
    of sum |x| where float16 values are subnormal), the exact products added in float32, at most K + 2 of them, the bias and the
    residual among them, and the output is rounded once."""
    rng = np.random.default_rng(M + N)
    w = _weights(rng, N, K, dtype)
    codes, scales = O.quantize_int4(w, group, dtype)
    x = O.round_to(rng.standard_normal((M, K)).astype(np.float32), dtype)
    b = O.round_to(rng.standard_normal(N).astype(np.float32), dtype)
    r = O.round_to(rng.standard_normal((M, N)).astype(np.float32), dtype)
    wv = O.values_int4(codes, scales, group)
    want = O.linear(x, wv, b)
    size = np.abs(x).astype(np.float64) @ np.abs(wv).T
    tiny = 2.0 ** -25 * np.abs(x).astype(np.float64).sum(1, keepdims=True) if dtype == "float16" else 0
    bar = (HALF_STEP[dtype] + 2.0 ** -24 * (K + 2)) * 1.01 * size + tiny + 2.0 ** -24 * (K + 2) * (np.abs(b) + np.abs(r))
    bar = bar + HALF_STEP[dtype] * 1.01 * (np.abs(want) + bar) + (2.0 ** -24 if dtype == "float16" else 0)
    packed, s, xt, bt = gpu.from_numpy(_pack(codes)), _dev(gpu, scales, dtype), _dev(gpu, x, dtype), _dev(gpu, b, dtype)
    got = gpu.linear_int4(xt, packed, s, bt, group=group).to_numpy().astype(np.float64)
    assert (np.abs(got - want) <= bar).all(), (np.abs(got - want) - bar).max()
    for act in ("relu", "gelu"):
        got = gpu.linear_int4(xt, packed, s, bt, act, group=group).to_numpy().astype(np.float64)
        assert (np.abs(got - O.linear(x, wv, b, act)) <= 1.13 * bar + 2.0 ** -20).all()
    y = gpu.linear_int4(xt, packed, s, bt, group=group) + _dev(gpu, r, dtype)
    both = want + r
    # (the sum may be rounded before the residual is added)
    bar = bar + HALF_STEP[dtype] * 1.01 * (np.abs(both) + np.abs(want) + bar)
    assert (np.abs(y.to_numpy().astype(np.float64) - both) <= bar).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,N,K,group", MANY)
def test_many_rows_pick_single_weights(gpu, dtype, M, N, K, group):
    """Rows with a single 1 give the dequantised weights themselves, to the bit:
    every code meets its own column and scale."""
    rng = np.random.default_rng(M)
    w = _weights(rng, N, K, dtype)
    packed, s = gpu.quantize_int4(_dev(gpu, w, dtype), group)
    back = gpu.dequantize_int4(packed, s, K, group).to_numpy().astype(np.float32)
    at = np.arange(M) % K
    x = np.zeros((M, K), np.float32)
    x[np.arange(M), at] = 1
    got = gpu.linear_int4(_dev(gpu, x, dtype), packed, s, group=group).to_numpy().astype(np.float32)
    np.testing.assert_array_equal(got, back[:, at].T)


def test_many_rows_keep_infinities_to_themselves(gpu):
    rng = np.random.default_rng(9)
    M, N, K = 1100, 2001, 200
    packed, s = gpu.quantize_int4(_dev(gpu, _weights(rng, N, K, "float16"), "float16"), 64)
    x = rng.standard_normal((M, K)).astype(np.float16)
    good = gpu.linear_int4(gpu.from_numpy(x), packed, s, group=64).to_numpy()
    rows = [0, 95, 96, 640, M - 1]
    x[rows, [0, 199, 63, 64, 130]] = [np.inf, np.nan, -np.inf, np.nan, np.inf]
    got = gpu.linear_int4(gpu.from_numpy(x), packed, s, group=64).to_numpy()
    keep = np.ones(M, bool)
    keep[rows] = False
    np.testing.assert_array_equal(got[keep], good[keep])
    assert not np.isfinite(got[rows][:, np.arange(N) != N // 2]).all(1).any()


def test_many_rows_of_views_captured_and_replayed(gpu):
    """Scales and rows that begin inside other tensors, also at odd halves of a
    word; replays with eager work between them."""
    rng = np.random.default_rng(4)
    M, N, K, group = 600, 2001, 160, 32
    w = _weights(rng, N, K, "float16")
    packed, s = gpu.quantize_int4(_dev(gpu, w, "float16"), group)
    want_of = lambda a: gpu.linear_int4(gpu.from_numpy(a), packed, s, group=group).to_numpy()
    flat = gpu.from_numpy(np.concatenate([np.full(1, 7, np.float16), s.to_numpy().ravel()]))
    inside = gpu.reshape(gpu.slice(flat, 0, 1, 1 + s.shape[0] * N), [s.shape[0], N])
    x = gpu.zeros([M + 1, K], "float16")
    y = gpu.zeros([M, K + 8], "float16")
    for t in (x, y, inside):
        t.eval()
    graph = gpu.capture(lambda: (gpu.linear_int4(gpu.slice(x, 0, 1, M + 1), packed, inside, group=group),
                                 gpu.linear_int4(gpu.slice(y, 1, 0, K), packed, s, group=group)))
    for _ in range(4):
        a, b = rng.standard_normal((M + 1, K)).astype(np.float16), rng.standard_normal((M, K + 8)).astype(np.float16)
        x.write(a)
        y.write(b)
        graph.replay()
        for got, rows in zip(graph.outputs, (a[1:], b[:, :K])):
            np.testing.assert_array_equal(got.to_numpy(), want_of(np.ascontiguousarray(rows)))
    graph.destroy()


@pytest.mark.parametrize("dtype,M,N,K", [("float32", 300, 96, 250), ("float16", 4200, 200, 72), ("bfloat16", 600, 999, 67)])
def test_two_graphs_with_workspaces_replayed_in_turn(gpu, dtype, M, N, K):
    rng = np.random.default_rng(5)
    made = []
    for seed in (0, 1):
        packed, s = gpu.quantize_int4(_dev(gpu, _weights(rng, N, K, dtype), dtype), 32)
        x = gpu.zeros([M, K], dtype)
        for t in (packed, s, x):
            t.eval()
        made.append((x, packed, s, gpu.capture(lambda x=x, p=packed, s=s: gpu.linear_int4(x, p, s, None, "gelu", group=32))))
    for _ in range(3):
        new = []
        for x, _, _, _ in made:
            new.append(_dev(gpu, rng.standard_normal((M, K)), dtype))
            gpu.blit_copy(new[-1], x)
        for x, _, _, g in made:
            g.replay()
        for (x, packed, s, g), a in zip(made, new):
            want = gpu.linear_int4(a, packed, s, None, "gelu", group=32).to_numpy()
            np.testing.assert_array_equal(g.outputs.to_numpy(), want)
    for *_, g in made:
        g.destroy()


def test_empty_rows(gpu):
    packed, s = gpu.quantize_int4(gpu.from_numpy(np.ones((16, 128), np.float32)))
    assert gpu.linear_int4(gpu.zeros([0, 128]), packed, s).to_numpy().shape == (0, 16)


def test_refusals(gpu):
    w = gpu.zeros([40, 200], "float16")
    packed, s = gpu.quantize_int4(w, 64)
    x = gpu.zeros([2, 200], "float16")
    for bad in (0, 16, 48, 256):
        with pytest.raises(ValueError, match="quantize_int4"):
            gpu.quantize_int4(w, bad)
    with pytest.raises(ValueError, match="quantize_int4"):
        gpu.quantize_int4(gpu.zeros([4], "float16"))
    with pytest.raises(ValueError):
        gpu.quantize_int4(gpu.zeros([4, 32], "int32"))
    with pytest.raises(ValueError):
        gpu.quantize_int4(gpu.zeros([4, 0], "float16"))
    call = lambda x=x, p=packed, s=s, b=None, act=None, g=64: gpu.linear_int4(x, p, s, b, act, group=g)  # noqa: E731
    for bad in [dict(g=32), dict(g=128), dict(g=7), dict(x=gpu.zeros([2, 300], "float16")),
                dict(x=gpu.zeros([2, 257], "float16")), dict(x=gpu.zeros([2, 200])), dict(x=gpu.zeros([2, 0], "float16")),
                dict(p=gpu.zeros([3, 2, 64, 16], "int8")), dict(p=gpu.zeros([2, 2, 64, 16], "uint8")),
                dict(p=gpu.zeros([40, 100], "uint8")), dict(s=gpu.zeros([4, 64], "float16")), dict(s=gpu.zeros([4, 40])),
                dict(b=gpu.zeros([39], "float16")), dict(b=gpu.zeros([40])), dict(act="tanh")]:
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError, match="dequantize_int4"):
        gpu.dequantize_int4(packed, s, 300, 64)


# ── norms and residuals of a graph ──────────────────────────────────────────
def _norm(x, g, b):
    m = x.mean(-1, keepdims=True)
    return (x - m) / np.sqrt(((x - m) ** 2).mean(-1, keepdims=True) + 1e-5) * g + b


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("M,N,K", [(1, 48, 128), (8, 5200, 1280), (16, 33, 896), (7, 40, 2048), (3, 17, 40), (2, 20, 33),
                                   (16, 20, 1000), (17, 48, 128), (90, 48, 128), (300, 48, 130)])
@pytest.mark.parametrize("group", [32, 128])
def test_layer_norm_and_residual_around(gpu, dtype, M, N, K, group):
    """r + act(layer_norm(x) W^T + b): the norm's output is rounded once more
    (half a step of each normalised value against |W|)."""
    rng = np.random.default_rng(M + K)
    w = _weights(rng, N, K, dtype)
    codes, scales = O.quantize_int4(w, group, dtype)
    wv = O.values_int4(codes, scales, group)
    x, r, g, b, bias = (O.round_to(rng.standard_normal(s).astype(np.float32) + o, dtype)
                        for s, o in (((M, K), 0.5), ((M, N), 0), ((K,), 1), ((K,), 0), ((N,), 0)))
    d = [_dev(gpu, a, dtype) for a in (x, r, g, b, bias)]
    packed, s = gpu.from_numpy(_pack(codes)), _dev(gpu, scales, dtype)
    before = gpu.graph_stats()["launches_saved"]
    y = d[1] + gpu.linear_int4(gpu.layer_norm(d[0], d[2], d[3]), packed, s, d[4], "gelu", group=group)
    got = y.to_numpy().astype(np.float64)
    saved = gpu.graph_stats()["launches_saved"] - before
    assert saved == 1 + (dtype != "float32" and M <= 16 and K % 8 == 0 and M * K <= 14336)
    n = _norm(x.astype(np.float64), g, b)
    lin = O.linear(n, wv, bias)
    want = r + O.linear(n, wv, bias, "gelu")
    half = HALF_STEP[dtype]
    step = np.repeat(scales.T.astype(np.float64), group, 1)[:, :K]
    bar = 2.0 ** -24 * (16 * 24 + K / 32 + 32) * (np.abs(n) @ step.T) + (half + 2.0 ** -20) * (np.abs(n) @ np.abs(wv).T)
    bar = bar + (half * (np.abs(n) @ np.abs(wv).T) if M > 256 else 0)
    bar = 1.13 * bar + (half + 2.0 ** -20) * (np.abs(lin) + np.abs(want)) + 2.0 ** -20
    assert (np.abs(got - want) <= bar).all(), (np.abs(got - want) / bar).max()


def test_what_else_reads_a_norm_or_a_product_keeps_it(gpu):
    rng = np.random.default_rng(1)
    w = _weights(rng, 32, 64, "float16")
    packed, s = gpu.quantize_int4(_dev(gpu, w, "float16"), 32)
    x, g, b = (_dev(gpu, rng.standard_normal(sh).astype(np.float32), "float16") for sh in ((4, 64), (64,), (64,)))
    n = gpu.layer_norm(x, g, b)
    y = gpu.linear_int4(n, packed, s, group=32)
    z = y + y                                   # the product twice
    v = gpu.linear_int4(gpu.layer_norm(x, g, b), packed, s, group=32) + gpu.slice(_dev(gpu, np.ones((1, 32)), "float16"), 0, 0, 1)
    np.testing.assert_allclose(v.to_numpy(), y.to_numpy() + np.float16(1), rtol=2e-3, atol=2e-3)
    np.testing.assert_array_equal(z.to_numpy(), y.to_numpy() + y.to_numpy())
    again = gpu.linear_int4(gpu.from_numpy(n.to_numpy()), packed, s, group=32).to_numpy()
    np.testing.assert_array_equal(y.to_numpy(), again)
    p, q = gpu.linear_int4(x, packed, s, group=32), gpu.linear_int4(x, packed, s, group=32)
    t = p + q                                   # two products: one is the other's residual
    np.testing.assert_allclose(t.to_numpy().astype(np.float64), 2 * gpu.linear_int4(x, packed, s, group=32).to_numpy(),
                               rtol=2e-3, atol=2e-3)
    # a view of a larger buffer as the norm's input, at an offset 16 bytes do not divide
    big = _dev(gpu, rng.standard_normal((4, 67)).astype(np.float32), "float16")
    part = gpu.slice(big, 1, 3, 67)
    a = gpu.linear_int4(gpu.layer_norm(part, g, b), packed, s, group=32).to_numpy()
    c = gpu.linear_int4(gpu.layer_norm(gpu.from_numpy(part.to_numpy()), g, b), packed, s, group=32).to_numpy()
    np.testing.assert_allclose(a, c, rtol=2e-3, atol=2e-3)


# ── infinities and values next to the type's largest ────────────────────────
def _huge_rows(rng, M, K, dtype):
    """Rows with one or two values that are infinite or next to the largest of
    the type, ordinary ones between them."""
    x = rng.standard_normal((M, K)).astype(np.float32)
    huge = {"float16": [6e4, 65504.0], "bfloat16": [2e37, 3.3e38], "float32": [2e37, np.finfo(np.float32).max]}[dtype]
    for m in range(0, M, 2 if M > 1 else 1):
        v = ([np.inf, -np.inf] + huge + [-huge[0], -huge[1]])[(m // 2 + K) % 6]
        x[m, rng.integers(0, K)] = v
        if m % 5 == 3:
            x[m, rng.integers(0, K)] = np.inf
    return O.round_to(x, dtype)


@pytest.mark.parametrize("dtype,M,N,K,group", [
    (t, *size) for t in ("float16", "bfloat16", "float32")
    for size in ((1, 70, 33, 32), (1, 70, 64, 64), (1, 70, 300, 128), (2, 70, 300, 64), (16, 5200, 256, 32),
                 (17, 70, 300, 64), (40, 70, 136, 32), (130, 70, 300, 128))] + [
    ("float16", 300, 70, 300, 64), ("bfloat16", 300, 70, 300, 64), ("float16", 600, 999, 64, 32),
    ("bfloat16", 600, 999, 64, 64), ("float16", 4200, 60, 72, 32), ("bfloat16", 2100, 999, 64, 128)])
def test_infinities_and_largest_values_are_the_products(gpu, dtype, M, N, K, group):
    """sum x code scale, whatever kernels the number of rows takes: an infinity
    gives infinities of the weights' signs (NaN where a weight is 0), and a
    large x what it is worth.  Sums of such rows are added value by value: K
    roundings, and those of the waves and the bias."""
    rng = np.random.default_rng(M + N + K)
    w = O.round_to(rng.standard_normal((N, K)).astype(np.float32) * 0.02, dtype)
    codes, scales = O.quantize_int4(w, group, dtype)
    wv = O.values_int4(codes, scales, group)
    x = _huge_rows(rng, M, K, dtype)
    packed, s, xt = gpu.from_numpy(_pack(codes)), _dev(gpu, scales, dtype), _dev(gpu, x, dtype)
    rows = np.r_[0:min(M, 60), max(0, M - 8):M]
    with np.errstate(invalid="ignore"):
        want = np.stack([(x[m].astype(np.float64) * wv).sum(1) for m in rows])
    ax = np.abs(np.where(np.isfinite(x), x, 0)).astype(np.float64)[rows]
    step = np.repeat(scales.T.astype(np.float64), group, 1)[:, :K]
    bar = 2.0 ** -24 * (16 * 24 + K + 34) * (ax @ step.T)
    if dtype != "float32":
        bar = bar + HALF_STEP[dtype] * 1.01 * (ax @ np.abs(wv).T) + (2.0 ** -25 * ax.sum(1, keepdims=True) if dtype == "float16" else 0)
    finite = np.isfinite(want)
    bar = bar + HALF_STEP[dtype] * 1.01 * (np.abs(np.where(finite, want, 0)) + bar) + 2.0 ** -25
    assert finite.any() or M == 1
    for act in (None, "relu"):
        got = gpu.linear_int4(xt, packed, s, None, act, group=group).to_numpy().astype(np.float64)[rows]
        exact = want if act is None else np.where(want > 0, want, 0)   # (relu(NaN) = 0 here)
        keep = np.isfinite(exact)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(exact))
        np.testing.assert_array_equal(got[np.isinf(exact)], exact[np.isinf(exact)])
        assert (np.abs(got[keep] - exact[keep]) <= bar[keep]).all()


def test_normalised_rows_of_large_gain(gpu):
    """The same where the rows come out of the layer_norm in the launch."""
    rng = np.random.default_rng(3)
    M, N, K, group = 4, 48, 128, 64
    w = O.round_to(rng.standard_normal((N, K)).astype(np.float32) * 0.02, "bfloat16")
    codes, scales = O.quantize_int4(w, group, "bfloat16")
    wv = O.values_int4(codes, scales, group)
    x = O.round_to(rng.standard_normal((M, K)).astype(np.float32), "bfloat16")
    g, b = np.full(K, O.round_to(np.float32(4e37), "bfloat16")), np.zeros(K, np.float32)
    y = gpu.linear_int4(gpu.layer_norm(*(_dev(gpu, a, "bfloat16") for a in (x, g, b))), gpu.from_numpy(_pack(codes)),
                        _dev(gpu, scales, "bfloat16"), group=group).to_numpy().astype(np.float64)
    n = _norm(x.astype(np.float64), g.astype(np.float64), b)
    want = n @ wv.T
    bar = (2.0 ** -8 + 2.0 ** -18) * (np.abs(n) @ np.abs(wv).T) + 2.0 ** -8 * np.abs(want)
    assert (np.abs(y - want) <= bar).all()


# ── many float32 rows ───────────────────────────────────────────────────────
@pytest.mark.parametrize("M", [16, 200, 300, 1000])
def test_float32_rows_keep_their_bits_whatever_their_number(gpu, M):
    """Rows of a single value v: v code scale, whose sums of v (code + 24) and
    -24 v (at most 31 |v| and 24 |v|, three parts each) and their difference
    round by at most 2^-24 (31 * 3 + 24 * 3 + 7) |v| before the scale, and the
    scale's product and the waves' sums by 3 steps of the result."""
    rng = np.random.default_rng(M)
    N, K, group = 300, 512, 64
    w = rng.standard_normal((N, K)).astype(np.float32)
    codes, scales = O.quantize_int4(w, group)
    x = np.zeros((M, K), np.float32)
    at = rng.integers(0, K, M)
    v = rng.standard_normal(M).astype(np.float32)
    x[np.arange(M), at] = v
    got = gpu.linear_int4(gpu.from_numpy(x), gpu.from_numpy(_pack(codes)), gpu.from_numpy(scales), group=group).to_numpy()
    want = v[:, None].astype(np.float64) * O.values_int4(codes, scales, group)[:, at].T
    bar = 2.0 ** -24 * (172 * np.abs(v)[:, None] * scales[at // group] + 3 * np.abs(want))
    assert (np.abs(got - want) <= bar).all(), (np.abs(got - want) / bar).max()


@pytest.mark.parametrize("M,N,K,group", [(300, 70, 300, 64), (1000, 999, 64, 32), (4200, 60, 72, 128)])
def test_float32_infinities_of_many_rows(gpu, M, N, K, group):
    test_infinities_and_largest_values_are_the_products(gpu, "float32", M, N, K, group)


def test_float32_rows_of_more_than_one_grid(gpu):
    rng = np.random.default_rng(0)
    M, N, K = 65535 * 64 + 70, 16, 8
    packed, s = gpu.quantize_int4(gpu.from_numpy(_weights(rng, N, K, "float32")), 32)
    x = rng.standard_normal((M, K)).astype(np.float32)
    r = np.arange(M * N, dtype=np.float32).reshape(M, N) % 7
    got = (gpu.from_numpy(r) + gpu.linear_int4(gpu.from_numpy(x), packed, s, None, "relu", group=32)).to_numpy()
    for lo in (0, 65535 * 64 - 70, M - 70):
        part = gpu.linear_int4(gpu.from_numpy(x[lo:lo + 70]), packed, s, None, "relu", group=32).to_numpy()
        want = r[lo:lo + 70] + part.astype(np.float64)
        assert (np.abs(got[lo:lo + 70] - want) <= 2.0 ** -23 * np.abs(want)).all()
