"""A key/value cache in 8 bits on the device: append, read and attention,
against the float32-exact and float64 oracle.

Bars.  Codes, scales and values: none (the same float32 operations).
Attention: with P_j the exact weights, an error of d in each score moves the
output by at most 2 d max|v|, d being (D + 16) 2^-24 scale sum_d |q_d k_d|
(float32 sums over D, q kept to 2^-22, the float32 exponent); weights kept to
w relative (2^-11 where the output has 16 bits, 2^-22 where it has 32) move it
by w max|v|, n of them summed in float32 by (n + 16) 2^-24 max|v|; the output
is rounded once."""
import numpy as np
import pytest

from oracle import few_bits as O

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _dev(gpu, a, dtype="float32"):
    t = gpu.from_numpy(np.ascontiguousarray(a, np.float32))
    return t if dtype == "float32" else gpu.cast(t, dtype)


def _cache(rng, B, H, Tmax, D, block):
    codes = rng.integers(-127, 128, (B, H, Tmax, D)).astype(np.int8)
    scales = (np.abs(rng.standard_normal((B, H, -(-Tmax // block)))) * 0.01 + 1e-3).astype(np.float32)
    return codes, scales


def _upload(gpu, *arrays):
    return [gpu.from_numpy(a) for a in arrays]


# ── append and read ─────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("block,Tmax,T,pos", [
    (16, 64, 1, [0, 5, 15, 16, 63, 64]),       # a block's first and last row, the last row, past the end
    (16, 50, 1, [49, 50, -1, 2, 2**31 - 1, -2**31]),
    (32, 100, 7, [0, 31, 60, 97, -3, 99]),     # across blocks, past either end
    (64, 129, 129, [0, 1, 64, -60, 128, 3]),
    (128, 300, 140, [0, 100, 127, 128, 200, 299]),
    (16, 1, 1, [0, 0, 1, 0, -1, 0]),
])
def test_append_bit_exact(gpu, dtype, D, block, Tmax, T, pos):
    rng = np.random.default_rng(D + block + T)
    B, H = len(pos), 3
    kc, ks = _cache(rng, B, H, Tmax, D, block)
    vc, vs = _cache(rng, B, H, Tmax, D, block)
    rows = [O.round_to((rng.standard_normal((B, H, T, D)) * s).astype(np.float32), dtype) for s in (0.5, 2.0)]
    dev = _upload(gpu, kc, ks, vc, vs)
    p = gpu.from_numpy(np.array(pos, np.int32))
    gpu.kv_write_int8(*dev, _dev(gpu, rows[0], dtype), _dev(gpu, rows[1], dtype), p, block=block)
    for codes, scales, x in ((kc, ks, rows[0]), (vc, vs, rows[1])):
        O.append_int8(codes, scales, x, pos, block)
    for t, want in zip(dev, (kc, ks, vc, vs)):
        np.testing.assert_array_equal(t.to_numpy(), want)
    start = np.array([max(-2, min(int(q), Tmax)) - 1 for q in pos], np.int32)
    got = gpu.kv_read_int8(*dev, gpu.from_numpy(start), T + 3, block=block, dtype=dtype)
    for t, codes, scales in ((got[0], kc, ks), (got[1], vc, vs)):
        v = O.round_to(O.values_int8(codes, scales, block), dtype)
        at = start[:, None].astype(np.int64) + np.arange(T + 3)
        want = np.where(((at >= 0) & (at < Tmax))[:, None, :, None],
                        np.stack([v[b][:, np.clip(at[b], 0, Tmax - 1)] for b in range(B)]), 0)
        np.testing.assert_array_equal(t.to_numpy(), want.astype(np.float32))


def test_append_token_by_token_from_views(gpu):
    """Rows that are views of a fused projection, at offsets 16 bytes do and do
    not divide, into a cache that is a slice of a larger one: 40 appends, a
    rollback, and the rest of the larger cache left as it was."""
    rng = np.random.default_rng(3)
    B, H, Tmax, D, block = 2, 3, 48, 64, 16
    big = [_cache(rng, B, H + 2, Tmax, D, block) for _ in range(2)]
    dev = [gpu.from_numpy(a) for pair in big for a in pair]
    part = [gpu.slice(t, 1, 1, 1 + H) for t in dev]
    want = [a[:, 1:1 + H] for pair in big for a in pair]
    order = list(range(40)) + [21, 22, 23, 16]
    for n, p in enumerate(order):
        qkv = O.round_to(rng.standard_normal((B, 1, 3 * H * D + 1)).astype(np.float32), "float16") * (1 + n % 5)
        off = n % 2
        t = gpu.slice(gpu.from_numpy(qkv.astype(np.float16)), 2, off, off + 3 * H * D)
        r = [gpu.transpose_dims(gpu.reshape(gpu.slice(t, 2, j * H * D, (j + 1) * H * D), [B, 1, H, D]), 1, 2)
             for j in (1, 2)]
        pos = np.array([p, p + 3], np.int32)
        gpu.kv_write_int8(*part, r[0], r[1], gpu.from_numpy(pos), block=block)
        for j in (1, 2):
            x = qkv.astype(np.float16).astype(np.float32)   # what the device was given
            x = x[:, :, off + j * H * D:off + (j + 1) * H * D].reshape(B, 1, H, D).transpose(0, 2, 1, 3)
            O.append_int8(want[2 * j - 2], want[2 * j - 1], x, pos, block)
    for t, a in zip(dev, [a for pair in big for a in pair]):
        np.testing.assert_array_equal(t.to_numpy(), a)


def test_infinities_zeros_and_tiny_values(gpu):
    B, H, D, block = 1, 4, 32, 16
    codes, scales = np.zeros((B, H, 32, D), np.int8), np.zeros((B, H, 2), np.float32)
    rows = np.zeros((B, H, 20, D), np.float32)
    rows[0, 0, 3, 1], rows[0, 1, 17, 2] = np.inf, np.nan
    rows[0, 2] = np.float32(1e-44)          # a scale below float32's smallest
    dev = _upload(gpu, codes, scales, codes.copy(), scales.copy())
    r = gpu.from_numpy(rows)
    zero = gpu.from_numpy(np.zeros(1, np.int32))
    gpu.kv_write_int8(*dev, r, r, zero, block=block)
    O.append_int8(codes, scales, rows, [0], block)
    np.testing.assert_array_equal(dev[0].to_numpy(), codes)
    np.testing.assert_array_equal(dev[1].to_numpy(), scales)
    got = gpu.kv_read_int8(*dev, zero, 20, block=block)[0].to_numpy()
    np.testing.assert_array_equal(got, O.values_int8(codes, scales, block)[:, :, :20])
    # a row appended to such a block leaves it so, and one at its start ends it
    one = gpu.from_numpy(np.ones((B, H, 1, D), np.float32))
    gpu.kv_write_int8(*dev, one, one, gpu.from_numpy(np.array([4], np.int32)), block=block)
    assert np.isinf(dev[1].to_numpy()[0, 0, 0])
    gpu.kv_write_int8(*dev, one, one, zero, block=block)
    assert (dev[1].to_numpy()[0, :, 0] == np.float32(1) / np.float32(127)).all()


# ── attention ───────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_append_halves_and_every_size_bit_exact(gpu, dtype):
    """Values that lie at or next to the middle of two codes, of every size
    down to the smallest, and scales that are subnormal themselves."""
    rng = np.random.default_rng(8)
    B, H, T, D, block = 1, 64, 32, 64, 16
    lo, hi = {"float32": (-149, 127), "float16": (-24, 15), "bfloat16": (-133, 127)}[dtype]
    size = np.ldexp(1.0, np.linspace(lo, hi, H).round().astype(int))[None, :, None, None]
    x = (rng.integers(-126, 127, (B, H, T, D)) + 0.5) / 127.0
    x = x * (1 + rng.choice([0, 1, -1], x.shape) * 2.0 ** -23)
    x[:, :, ::block, 0] = 1.0
    x = O.round_to((x * size).astype(np.float32), dtype)
    codes, scales = np.zeros((B, H, T, D), np.int8), np.zeros((B, H, T // block), np.float32)
    dev = _upload(gpu, codes, scales, codes.copy(), scales.copy())
    r = _dev(gpu, x, dtype)
    np.testing.assert_array_equal(r.to_numpy().astype(np.float32), x)
    gpu.kv_write_int8(*dev, r, r, gpu.from_numpy(np.zeros(1, np.int32)), block=block)
    O.append_int8(codes, scales, x, [0], block)
    for t, want in zip(dev, (codes, scales, codes, scales)):
        np.testing.assert_array_equal(t.to_numpy(), want)


def _bar(q, k, v, scale, dtype, n):
    vmax = np.abs(v).max()
    d = (q.shape[-1] + 16) * 2.0 ** -24 * scale * np.abs(q).max() * np.abs(k).sum(-1).max()
    w = 2.0 ** -11 if dtype != "float32" else 2.0 ** -22
    return vmax * (2 * d + w + (n + 16) * 2.0 ** -24), HALF_STEP[dtype]


def _check(got, want, bar):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bar[1] * np.abs(want)
    assert off.max() <= bar[0], (off.max(), bar)


def _attend(gpu, rng, dtype, D, block, Tmax, Tq, G, lens, scale=None, H=2):
    B = len(lens)
    kc, ks = _cache(rng, B, H, Tmax, D, block)
    vc, vs = _cache(rng, B, H, Tmax, D, block)
    q = O.round_to(rng.standard_normal((B, H * G, Tq, D)).astype(np.float32), dtype)
    k, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
    want = O.decode_attention(q, k, v, lens, scale)
    # what no query sees: codes of any kind, blocks whose scale is not a number
    for b, n in enumerate(lens):
        n = min(max(int(n), 0), Tmax)
        for codes, scales in ((kc, ks), (vc, vs)):
            codes[b, :, n:] = rng.integers(-128, 128, codes[b, :, n:].shape)
            scales[b, :, -(-n // block):] = rng.choice([np.nan, np.inf, -np.inf, 1e30])
    dev = _upload(gpu, kc, ks, vc, vs)
    out = gpu.decode_attention_int8(_dev(gpu, q, dtype), *dev, gpu.from_numpy(np.array(lens, np.int32)), block=block,
                                    scale=scale)
    bar = _bar(q, k, v, scale or D ** -0.5, dtype, Tmax)
    _check(out.to_numpy(), want, bar)
    return dev, q, want, bar


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("block,Tmax,Tq,G,lens", [
    (16, 1, 1, 1, [1, 0, 5]),
    (16, 40, 1, 1, [40, 17, 1]),
    (32, 130, 1, 4, [130, 33, 32]),
    (64, 513, 1, 2, [513, 64, 65]),
    (128, 1000, 1, 1, [1000, 999, 1]),
    (16, 700, 3, 1, [700, 2, 1]),       # queries that see nothing
    (16, 333, 17, 1, [333, 17, 5]),
    (64, 200, 40, 3, [200, 41, 0]),
])
def test_attention_vs_oracle(gpu, dtype, D, block, Tmax, Tq, G, lens):
    _attend(gpu, np.random.default_rng(Tmax + D), dtype, D, block, Tmax, Tq, G, lens)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("B,H,G,Tmax", [(1, 1, 1, 9001), (1, 3, 5, 4100), (9, 20, 1, 129), (2, 2, 16, 2000),
                                         (1, 1, 33, 3000), (40, 8, 1, 300)])
def test_attention_grids(gpu, dtype, B, H, G, Tmax):
    """Few long rows, many short ones, more query heads a cache head than a
    tile has: every way that the work is split."""
    rng = np.random.default_rng(B + G)
    lens = [Tmax] + [int(x) for x in rng.integers(0, Tmax + 1, B - 1)]
    _attend(gpu, rng, dtype, 64, 32, Tmax, 1, G, lens, H=H)


@pytest.mark.parametrize("scale", [0.02, 3.0])
def test_attention_scale_and_peaked_rows(gpu, scale):
    """A softmax scale of the caller's, up to rows with all weight on one key."""
    _attend(gpu, np.random.default_rng(8), "float16", 64, 16, 500, 2, 2, [500, 77], scale=scale)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_attention_magnitudes(gpu, dtype):
    """Queries and scales far from 1, in one row: large and tiny heads."""
    rng = np.random.default_rng(4)
    B, H, Tmax, D, block = 1, 4, 90, 64, 16
    kc, ks = _cache(rng, B, H, Tmax, D, block)
    vc, vs = _cache(rng, B, H, Tmax, D, block)
    big = np.array([1.0, 1e4, 1e-4, 1.0], np.float32)[None, :, None]
    ks, vs = ks / big, vs * np.array([1e-6, 1.0, 1.0, 50.0], np.float32)[None, :, None]
    vs[:, :, 2] *= 1e-3          # neighbouring blocks of unlike scale
    q = O.round_to((rng.standard_normal((B, H, 1, D)) * big[..., None]).astype(np.float32), dtype)
    out = gpu.decode_attention_int8(_dev(gpu, q, dtype), *_upload(gpu, kc, ks, vc, vs),
                                    gpu.from_numpy(np.array([Tmax], np.int32)), block=block).to_numpy()
    k, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
    want = O.decode_attention(q, k, v, [Tmax])
    for h in range(H):
        bar, half = _bar(q[:, h], k[:, h], v[:, h], D ** -0.5, dtype, Tmax)
        if dtype == "float16":
            half_abs = 2.0 ** -25     # float16's smallest step, for the tiny head
            bar = bar + half_abs
        _check(out[:, h], want[:, h], (bar, half))


def test_attention_marks_what_it_sees(gpu):
    """A NaN block that a query sees reaches that query and head only."""
    rng = np.random.default_rng(6)
    kc, ks = _cache(rng, 2, 3, 64, 64, 16)
    vc, vs = _cache(rng, 2, 3, 64, 64, 16)
    ks[0, 1, 2], vs[1, 2, 1] = np.nan, np.inf
    vc[1, 2, 16:32, :] = 0
    q = rng.standard_normal((2, 3, 1, 64)).astype(np.float32)
    out = gpu.decode_attention_int8(gpu.from_numpy(q), *_upload(gpu, kc, ks, vc, vs),
                                    gpu.from_numpy(np.array([33, 20], np.int32)), block=16).to_numpy()
    nan = np.isnan(out).all((2, 3))
    np.testing.assert_array_equal(nan, [[False, True, False], [False, False, True]])
    assert np.isfinite(out[~nan]).all()


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("G", [1, 3])
def test_append_and_attend_in_one_call(gpu, dtype, G):
    """k_new, v_new: the same cache and output as an append and an attention,
    with lengths that name no row."""
    rng = np.random.default_rng(2)
    lens = np.array([1, 16, 17, 33, 48, 49, 0, 200], np.int32)
    B, H, Tmax, D, block = len(lens), 2, 48, 64, 16
    kc, ks = _cache(rng, B, H, Tmax, D, block)
    vc, vs = _cache(rng, B, H, Tmax, D, block)
    q, k_new, v_new = (O.round_to((rng.standard_normal((B, h, 1, D)) * 2).astype(np.float32), dtype)
                       for h in (H * G, H, H))
    one, two = _upload(gpu, kc, ks, vc, vs), _upload(gpu, kc, ks, vc, vs)
    L = gpu.from_numpy(lens)
    a = gpu.decode_attention_int8(_dev(gpu, q, dtype), *one, L, block=block, k_new=_dev(gpu, k_new, dtype),
                                  v_new=_dev(gpu, v_new, dtype)).to_numpy()
    gpu.kv_write_int8(*two, _dev(gpu, k_new, dtype), _dev(gpu, v_new, dtype), gpu.from_numpy(lens - 1), block=block)
    b = gpu.decode_attention_int8(_dev(gpu, q, dtype), *two, L, block=block).to_numpy()
    for x, y in zip(one, two):
        np.testing.assert_array_equal(x.to_numpy(), y.to_numpy())
    for codes, scales, x in ((kc, ks, k_new), (vc, vs, v_new)):
        O.append_int8(codes, scales, x, lens - 1, block)
    for x, y in zip(one, (kc, ks, vc, vs)):
        np.testing.assert_array_equal(x.to_numpy(), y)
    k, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
    bar = _bar(q, k, v, D ** -0.5, dtype, Tmax)
    want = O.decode_attention(q, k, v, lens)
    _check(a, want, bar)
    _check(b, want, bar)


def test_captured_steps_replayed(gpu):
    """One append-and-attend step captured and replayed over advancing
    positions, a second graph between the replays, every replay checked."""
    rng = np.random.default_rng(12)
    B, H, Tmax, D, block = 2, 2, 40, 64, 16
    kc, ks = np.zeros((B, H, Tmax, D), np.int8), np.zeros((B, H, 3), np.float32)
    vc, vs = kc.copy(), ks.copy()
    dev = _upload(gpu, kc, ks, vc, vs)
    q, kn, vn = (gpu.zeros([B, H, 1, D], "float16") for _ in range(3))
    lens = gpu.from_numpy(np.ones(B, np.int32))
    graph = gpu.capture(lambda: gpu.decode_attention_int8(q, *dev, lens, block=block, k_new=kn, v_new=vn))
    long = _upload(gpu, *(x for _ in range(2) for x in _cache(rng, 1, 1, 5000, D, block)))
    ql = gpu.from_numpy(rng.standard_normal((1, 1, 1, D)).astype(np.float32))
    L = gpu.from_numpy(np.array([5000], np.int32))
    other = gpu.capture(lambda: gpu.decode_attention_int8(ql, *long, L, block=block))
    other.replay()
    first = other.outputs.to_numpy()
    for t in range(20):
        x = [rng.standard_normal((B, H, 1, D)).astype(np.float16) for _ in range(3)]
        for a, b in zip((q, kn, vn), x):
            a.write(b)
        n = np.array([t + 1, t + 19], np.int32)
        lens.write(n)
        graph.replay()
        other.replay()
        for codes, scales, r in ((kc, ks, x[1]), (vc, vs, x[2])):
            O.append_int8(codes, scales, r.astype(np.float32), n - 1, block)
        for a, b in zip(dev, (kc, ks, vc, vs)):
            np.testing.assert_array_equal(a.to_numpy(), b)
        k, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
        qq = x[0].astype(np.float32)
        _check(graph.outputs.to_numpy(), O.decode_attention(qq, k, v, n), _bar(qq, k, v, D ** -0.5, "float16", Tmax))
        np.testing.assert_array_equal(other.outputs.to_numpy(), first)
    graph.destroy()
    other.destroy()


def test_same_call_same_bits(gpu):
    rng = np.random.default_rng(1)
    dev = _upload(gpu, *(x for _ in range(2) for x in _cache(rng, 3, 2, 3000, 128, 64)))
    q = gpu.cast(gpu.from_numpy(rng.standard_normal((3, 8, 1, 128)).astype(np.float32)), "bfloat16")
    L = gpu.from_numpy(np.array([3000, 1234, 2], np.int32))
    runs = [gpu.decode_attention_int8(q, *dev, L, block=64).to_numpy() for _ in range(5)]
    for r in runs[1:]:
        np.testing.assert_array_equal(r, runs[0])


def test_unaligned_and_transposed_queries(gpu):
    rng = np.random.default_rng(9)
    B, H, Tq, D, block, Tmax = 2, 3, 2, 64, 16, 70
    kc, ks = _cache(rng, B, H, Tmax, D, block)
    vc, vs = _cache(rng, B, H, Tmax, D, block)
    dev = _upload(gpu, kc, ks, vc, vs)
    k, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
    flat = rng.standard_normal((B, Tq, H * D + 3)).astype(np.float16)
    for off in (0, 1, 3):
        t = gpu.slice(gpu.from_numpy(flat), 2, off, off + H * D)
        q = gpu.transpose_dims(gpu.reshape(t, [B, Tq, H, D]), 1, 2)
        ref = flat[:, :, off:off + H * D].reshape(B, Tq, H, D).transpose(0, 2, 1, 3).astype(np.float32)
        out = gpu.decode_attention_int8(q, *dev, gpu.from_numpy(np.array([70, 9], np.int32)), block=block).to_numpy()
        _check(out, O.decode_attention(ref, k, v, [70, 9]), _bar(ref, k, v, D ** -0.5, "float16", Tmax))


def test_cache_past_two_to_the_31(gpu):
    """One head's codes past 2^31 bytes: rows written, read and attended to
    near the far end."""
    D, block = 64, 128
    Tmax = (1 << 25) + 1000
    kc, vc = (gpu.zeros([1, 1, Tmax, D], "int8") for _ in range(2))
    ks, vs = (gpu.zeros([1, 1, -(-Tmax // block)]) for _ in range(2))
    rng = np.random.default_rng(0)
    rows = rng.standard_normal((2, 1, 1, 200, D)).astype(np.float32)
    pos = np.array([Tmax - 300], np.int32)
    gpu.kv_write_int8(kc, ks, vc, vs, gpu.from_numpy(rows[0]), gpu.from_numpy(rows[1]), gpu.from_numpy(pos), block=block)
    got = gpu.kv_read_int8(kc, ks, vc, vs, gpu.from_numpy(pos), 200, block=block)
    for t, x in zip(got, rows):
        assert np.abs(t.to_numpy() - x).max() <= 0.5001 * np.abs(x).max() / 127 + 1e-6
    k, v = got[0].to_numpy(), got[1].to_numpy()
    # one key takes all weight: the rows of zeros before it score 0
    q = (k[:, :, 57:58] * 40).astype(np.float32)
    out = gpu.decode_attention_int8(gpu.from_numpy(q), kc, ks, vc, vs,
                                    gpu.from_numpy(np.array([Tmax - 100], np.int32)), block=block).to_numpy()
    s = np.concatenate([(k[0, 0] @ q[0, 0, 0].astype(np.float64)) / 8, [0.0]])
    e = np.exp(s - s.max())
    e[-1] *= Tmax - 300
    want = (e[:-1] @ v[0, 0].astype(np.float64)) / e.sum()
    d = (D + 16) * 2.0 ** -24 / 8 * np.abs(q).max() * np.abs(k).sum(-1).max()
    assert np.abs(out[0, 0, 0] - want).max() <= np.abs(v).max() * (2 * d + 2.0 ** -20)


# ── blocks that are not finite ──────────────────────────────────────────────
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_appended_infinities_reach_every_query_that_sees_them(gpu, dtype, D, bad):
    """A block given an infinity or NaN as a key or as a value makes the
    queries that see it NaN, in every head, and no others."""
    rng = np.random.default_rng(D)
    B, H, T, block = 3, 64, 40, 16
    for which in (0, 1):
        dev = _upload(gpu, *(a for _ in range(2) for a in (np.zeros((B, H, T, D), np.int8), np.zeros((B, H, 3), np.float32))))
        x = [rng.standard_normal((B, H, 33, D)).astype(np.float32) for _ in range(2)]
        x[which][:, :, 20, 3] = bad
        gpu.kv_write_int8(*dev, *(_dev(gpu, a, dtype) for a in x), gpu.from_numpy(np.zeros(B, np.int32)), block=block)
        q = _dev(gpu, rng.standard_normal((B, H, 2, D)).astype(np.float32), dtype)
        out = gpu.decode_attention_int8(q, *dev, gpu.from_numpy(np.array([33, 17, 16], np.int32)), block=block).to_numpy()
        np.testing.assert_array_equal(np.isnan(out.astype(np.float32)).all(-1), [[[True, True]] * H, [[False, True]] * H, [[False, False]] * H])
        np.testing.assert_array_equal(np.isnan(out.astype(np.float32)).any(-1), np.isnan(out.astype(np.float32)).all(-1))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("which", [0, 1])
def test_an_infinity_appended_in_the_launch(gpu, dtype, which):
    rng = np.random.default_rng(5)
    B, H, T, D, block = 2, 64, 40, 64, 16
    kc, ks = _cache(rng, B, H, T, D, block)
    vc, vs = _cache(rng, B, H, T, D, block)
    new = [rng.standard_normal((B, H, 1, D)).astype(np.float32) for _ in range(2)]
    new[which][1, :, 0, 7] = np.inf
    out = gpu.decode_attention_int8(_dev(gpu, rng.standard_normal((B, H, 1, D)).astype(np.float32), dtype),
                                    *_upload(gpu, kc, ks, vc, vs), gpu.from_numpy(np.array([36, 36], np.int32)),
                                    block=block, k_new=_dev(gpu, new[0], dtype), v_new=_dev(gpu, new[1], dtype)).to_numpy()
    assert np.isfinite(out[0].astype(np.float32)).all() and np.isnan(out[1].astype(np.float32)).all()


# ── blocks of unlike scale ──────────────────────────────────────────────────
RATIOS = [(t, k) for t, ks in (("float16", (0, 12, 24)), ("bfloat16", (0, 24, 40, 100)), ("float32", (0, 12, 24, 60, 100)))
          for k in ks]


@pytest.mark.parametrize("dtype,k", RATIOS)
@pytest.mark.parametrize("T,block,at", [(32, 16, 0), (32, 16, 1), (300, 32, 3), (300, 16, 18), (3000, 64, 0), (3000, 128, 20)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_a_scale_without_weight_moves_nothing(gpu, dtype, k, T, block, at, D):
    """All weight on the rows of one block, equal keys of which the output is
    the plain mean; the values of the others, 2^k as large, have weights below
    2^-200.  n equal weights kept to w, and n + 16 roundings of the sums."""
    rng = np.random.default_rng(T + k)
    H, nb = 3, -(-T // block)
    q = O.round_to(rng.choice([-1.0, 1.0], (1, H, 1, D)).astype(np.float32) * 2, dtype)
    kc = np.zeros((1, H, T, D), np.int8)
    rows = slice(at * block, min((at + 1) * block, T))
    kc[:, :, rows] = (np.sign(q) * 100).astype(np.int8)
    ks = np.full((1, H, nb), 240 * np.log(2) * D ** 0.5 / (200 * D), np.float32)    # a score of 240 ln 2
    vc = rng.integers(-127, 128, (1, H, T, D)).astype(np.int8)
    vs = np.full((1, H, nb), 1e-5 * 2.0 ** k, np.float32)
    vs[:, :, at] = 1e-5
    out = gpu.decode_attention_int8(_dev(gpu, q, dtype), *_upload(gpu, kc, ks, vc, vs),
                                    gpu.from_numpy(np.array([T], np.int32)), block=block).to_numpy().astype(np.float64)
    v = O.values_int8(vc, vs, block)[:, :, rows].astype(np.float64)
    want, n = v.mean(2, keepdims=True), v.shape[2]
    w = 2.0 ** -11 if dtype != "float32" else 2.0 ** -22
    bar = (w + (n + 16) * 2.0 ** -24) * np.abs(v).mean(2, keepdims=True) + HALF_STEP[dtype] * np.abs(want)
    assert (np.abs(out - want) <= bar + 2.0 ** -25 * (dtype == "float16")).all(), np.abs(out - want).max()


@pytest.mark.parametrize("dtype,k", RATIOS)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_a_scale_that_a_query_does_not_see_moves_nothing_of_it(gpu, dtype, k, D):
    """Three queries of a chunk, the last two of which see one and two rows of
    a block 2^k as large: each is as exact as the rows it sees."""
    rng = np.random.default_rng(k)
    H, T, block = 3, 32, 16
    kc, ks = _cache(rng, 1, H, T, D, block)
    vc, _ = _cache(rng, 1, H, T, D, block)
    vs = np.full((1, H, 2), 1e-5, np.float32)
    vs[:, :, 1] *= np.float32(2.0 ** k)
    q = O.round_to(rng.standard_normal((1, H, 3, D)).astype(np.float32), dtype)
    out = gpu.decode_attention_int8(_dev(gpu, q, dtype), *_upload(gpu, kc, ks, vc, vs),
                                    gpu.from_numpy(np.array([18], np.int32)), block=block).to_numpy()
    kv, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
    want = O.decode_attention(q, kv, v, [18])
    for i in range(3):
        bar = _bar(q, kv, v[:, :, :16 + i], D ** -0.5, dtype, T)
        _check(out[:, :, i], want[:, :, i], (bar[0] + 2.0 ** -25 * (dtype == "float16"), bar[1]))


@pytest.mark.parametrize("dtype,k", [("float16", 20), ("bfloat16", 60), ("float32", 60), ("float32", 100)])
@pytest.mark.parametrize("T,block", [(48, 16), (3000, 64)])
def test_a_small_weight_on_large_values_counts(gpu, dtype, k, T, block):
    """Rows whose weights are 2^-k of the others' and whose values are 2^k of
    theirs: sum P_j |v_j| of both parts, each kept to its own error."""
    rng = np.random.default_rng(k)
    H, D, nb = 2, 64, -(-T // block)
    q = O.round_to(rng.choice([-1.0, 1.0], (1, H, 1, D)).astype(np.float32) * 2, dtype)
    kc = np.zeros((1, H, T, D), np.int8)
    kc[:, :, block:2 * block] = (np.sign(q) * 100).astype(np.int8)
    ks = np.full((1, H, nb), k * np.log(2) * D ** 0.5 / (200 * D), np.float32)
    vc = rng.integers(-127, 128, (1, H, T, D)).astype(np.int8)
    vs = np.full((1, H, nb), 1e-5 * 2.0 ** k, np.float32)
    vs[:, :, 1] = 1e-5
    out = gpu.decode_attention_int8(_dev(gpu, q, dtype), *_upload(gpu, kc, ks, vc, vs),
                                    gpu.from_numpy(np.array([T], np.int32)), block=block).to_numpy().astype(np.float64)
    kv, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
    want, size = O.decode_attention(q, kv, v, [T]), O.decode_attention(q, kv, np.abs(v), [T])
    d = (D + 16) * 2.0 ** -24 * k * np.log(2)
    w = 2.0 ** -11 if dtype != "float32" else 2.0 ** -22
    bar = (2 * d + w + (T + 16) * 2.0 ** -24) * size + HALF_STEP[dtype] * np.abs(want)
    assert (np.abs(out - want) <= bar + 2.0 ** -25 * (dtype == "float16")).all(), (np.abs(out - want) / bar).max()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("T,B,size", [(100, 1, 2e38), (600, 8, 2e38), (3000, 1, 2e38), (3000, 40, 1e35), (100, 1, 1e-36),
                                      (3000, 1, 1e-36), (100, 1, 2e-41)])
def test_values_next_to_the_largest_and_smallest(gpu, dtype, T, B, size):
    """A mean of values is as large as they are, however many they are."""
    rng = np.random.default_rng(T)
    H, D, block = 2, 64, 16
    kc, ks = _cache(rng, B, H, T, D, block)
    vc, vs = _cache(rng, B, H, T, D, block)
    vc[..., ::2] = np.abs(vc[..., ::2])     # half of the columns do not cancel
    vs[:] = np.float32(size / 127)
    q = O.round_to(rng.standard_normal((B, H, 1, D)).astype(np.float32), dtype)
    out = gpu.decode_attention_int8(_dev(gpu, q, dtype), *_upload(gpu, kc, ks, vc, vs),
                                    gpu.from_numpy(np.full(B, T, np.int32)), block=block).to_numpy()
    kv, v = O.values_int8(kc, ks, block), O.values_int8(vc, vs, block)
    bar = _bar(q, kv, v, D ** -0.5, dtype, T)
    _check(out, O.decode_attention(q, kv, v, [T] * B),
           (bar[0] + 2.0 ** (-133 if dtype == "bfloat16" else -148), bar[1]))


@pytest.mark.parametrize("dtype,D", [("float16", 64), ("float32", 64), ("bfloat16", 32), ("float32", 32)])
def test_many_heads_over_long_rows(gpu, dtype, D):
    """160 contexts past 2048 rows, whole in blocks of 16 or 8 waves, the last
    of them appended in the launch too."""
    rng = np.random.default_rng(D)
    B, H, Tmax, block = 8, 20, 2200, 32
    lens = [Tmax, 2049, 1, 0, 2100, 513, 2176, 2177]
    dev, q, want, bar = _attend(gpu, rng, dtype, D, block, Tmax, 1, 1, lens, H=H)
    new = [O.round_to(rng.standard_normal((B, H, 1, D)).astype(np.float32), dtype) for _ in range(2)]
    held = [t.to_numpy() for t in dev]
    for codes, scales, x in ((held[0], held[1], new[0]), (held[2], held[3], new[1])):
        O.append_int8(codes, scales, x, np.array(lens) - 1, block)
    out = gpu.decode_attention_int8(_dev(gpu, q, dtype), *dev, gpu.from_numpy(np.array(lens, np.int32)), block=block,
                                    k_new=_dev(gpu, new[0], dtype), v_new=_dev(gpu, new[1], dtype)).to_numpy()
    for t, a in zip(dev, held):
        np.testing.assert_array_equal(t.to_numpy(), a)
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = (O.values_int8(held[i][b:b + 1, :, :n], held[i + 1][b:b + 1, :, :-(-n // block)], block) for i in (0, 2))
        _check(out[b:b + 1], O.decode_attention(q[b:b + 1], k, v, [n]), _bar(q[b:b + 1], k, v, D ** -0.5, dtype, Tmax))


# ── what was asked for before a write ───────────────────────────────────────
def _small(gpu, rng):
    return _upload(gpu, *(x for _ in range(2) for x in _cache(rng, 1, 2, 40, 64, 16)))


def test_reads_asked_for_before_a_write_see_what_was_there(gpu):
    rng = np.random.default_rng(3)
    dev = _small(gpu, rng)
    part = [gpu.slice(t, 1, 0, 1) for t in dev]
    rows = [gpu.from_numpy(rng.standard_normal((1, 2, 8, 64)).astype(np.float32)) for _ in range(2)]
    q, lens = gpu.from_numpy(rng.standard_normal((1, 2, 1, 64)).astype(np.float32)), gpu.from_numpy(np.array([40], np.int32))
    zero, ten = (gpu.from_numpy(np.array([n], np.int32)) for n in (0, 10))
    was = [t.to_numpy() for t in gpu.kv_read_int8(*dev, zero, 40)] + [gpu.decode_attention_int8(q, *dev, lens).to_numpy()]
    read, view, seen = (gpu.kv_read_int8(*dev, zero, 40), gpu.kv_read_int8(*part, zero, 40),
                        gpu.decode_attention_int8(q, *dev, lens) + q)
    gpu.kv_write_int8(*dev, *rows, ten)
    for a, b in zip(read, was):
        np.testing.assert_array_equal(a.to_numpy(), b)
    for a, b in zip(view, was):
        np.testing.assert_array_equal(a.to_numpy(), b[:, :1])
    np.testing.assert_array_equal(seen.to_numpy(), was[2] + q.to_numpy())
    assert (gpu.kv_read_int8(*dev, zero, 40)[0].to_numpy() != was[0]).any()
    # rows that are made of a read of the cache they are written to
    want = [t.to_numpy() for t in gpu.kv_read_int8(*dev, ten, 8)]
    gpu.kv_write_int8(*dev, *(t + t for t in gpu.kv_read_int8(*dev, ten, 8)), zero)
    for a, b in zip(gpu.kv_read_int8(*dev, zero, 8), want):
        assert np.abs(a.to_numpy() - 2 * b).max() <= np.abs(2 * b).max() / 254 * 1.001


def test_appends_and_reads_keep_the_order_they_were_asked_for(gpu):
    rng = np.random.default_rng(4)
    q, *new = (rng.standard_normal((1, 2, 1, 64)).astype(np.float32) * s for s in (1, 1, 1, 9, 9))
    q, *new = (gpu.from_numpy(a) for a in (q, *new))
    lens = [gpu.from_numpy(np.array([n], np.int32)) for n in (20, 21)]
    zero = gpu.from_numpy(np.zeros(1, np.int32))
    one, two = _small(gpu, np.random.default_rng(5)), _small(gpu, np.random.default_rng(5))

    def steps(dev, now):
        out = list(gpu.kv_read_int8(*dev, zero, 40))
        now(out)
        for i in (0, 1):
            out.append(gpu.decode_attention_int8(q, *dev, lens[i], k_new=new[2 * i], v_new=new[2 * i + 1]))
            now(out)
            out += gpu.kv_read_int8(*dev, zero, 40)
            now(out)
        return out

    want = [t.to_numpy() for t in steps(one, lambda out: gpu.eval_many(out))]
    got = steps(two, lambda out: None)
    for a, b in zip(reversed(got), reversed(want)):     # the last first
        np.testing.assert_array_equal(a.to_numpy(), b)
    for a, b in zip(one, two):
        np.testing.assert_array_equal(a.to_numpy(), b.to_numpy())


# ── refusals ────────────────────────────────────────────────────────────────
def test_refusals(gpu):
    def cache(B=2, H=2, T=32, D=64, n=2):
        return [gpu.zeros([B, H, T, D], "int8"), gpu.zeros([B, H, n]), gpu.zeros([B, H, T, D], "int8"),
                gpu.zeros([B, H, n])]

    c, rows, pos = cache(), gpu.zeros([2, 2, 1, 64], "float16"), gpu.from_numpy(np.zeros(2, np.int32))
    write = lambda c=c, k=rows, v=rows, p=pos, b=16: gpu.kv_write_int8(*c, k, v, p, block=b)  # noqa: E731
    for bad in [dict(b=8), dict(b=24), dict(b=256), dict(b=32), dict(p=gpu.zeros([3], "int32")),
                dict(p=gpu.zeros([2], "int64")), dict(k=gpu.zeros([2, 2, 1, 64])), dict(k=gpu.zeros([2, 2, 2, 64], "float16")),
                dict(k=gpu.zeros([2, 1, 1, 64], "float16")), dict(k=gpu.zeros([2, 2, 1, 64], "int8")),
                dict(k=gpu.zeros([2, 2, 33, 64], "float16"), v=gpu.zeros([2, 2, 33, 64], "float16")),
                dict(c=[c[0], c[1], c[0], c[3]]), dict(c=[c[0], c[1], c[2], c[1]]), dict(c=[c[0], c[1], c[2], c[0]]),
                dict(c=[rows, c[1], c[2], c[3]]), dict(c=cache(D=48)), dict(c=[c[0], c[1]] + cache(T=31)[2:])]:
        with pytest.raises(ValueError, match="kv_write_int8"):
            write(**bad)
    with pytest.raises(ValueError, match="kv_read_int8"):
        gpu.kv_read_int8(*c, pos, -1)
    with pytest.raises(ValueError, match="kv_read_int8"):
        gpu.kv_read_int8(*c, pos, 4, dtype="int32")
    q = gpu.zeros([2, 4, 1, 64], "float16")
    lens = gpu.from_numpy(np.ones(2, np.int32))
    call = lambda q=q, c=c, lens=lens, **kw: gpu.decode_attention_int8(q, *c, lens, **kw)  # noqa: E731
    for bad in [dict(q=gpu.zeros([2, 3, 1, 64], "float16")), dict(q=gpu.zeros([2, 2, 33, 64], "float16")),
                dict(q=gpu.zeros([2, 2, 1, 32], "float16")), dict(q=gpu.zeros([2, 2, 64], "float16")),
                dict(q=gpu.zeros([1, 2, 1, 64], "float16")), dict(q=gpu.zeros([2, 2, 1, 64], "int32")),
                dict(scale=0.0), dict(scale=float("nan")), dict(lens=gpu.zeros([2], "int64")),
                dict(lens=gpu.zeros([3], "int32")), dict(q=gpu.zeros([2, 2, 2, 64], "float16"), k_new=rows, v_new=rows),
                dict(k_new=gpu.zeros([2, 2, 2, 64], "float16"), v_new=rows), dict(k_new=gpu.zeros([2, 2, 1, 64]), v_new=rows),
                dict(block=32)]:
        with pytest.raises(ValueError, match="decode_attention_int8"):
            call(**bad)
    with pytest.raises(ValueError):
        call(k_new=rows)
    # codes whose rows are not at 16-byte boundaries
    odd = gpu.slice(gpu.zeros([2, 2, 32, 72], "int8"), 3, 8, 72)
    odd.eval()
    with pytest.raises(ValueError, match="16-byte"):
        gpu.kv_write_int8(odd, c[1], c[2], c[3], rows, rows, pos)
