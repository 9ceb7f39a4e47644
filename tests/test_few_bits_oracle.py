"""The oracle of the 8-bit cache, the 4-bit weights and the token log
probabilities against closed forms, brute force and PyTorch (no GPU)."""
import numpy as np
import pytest
import torch

from oracle import few_bits as B

RNG = np.random.default_rng(5)


def test_append_rounds_a_fresh_block_once():
    rows = RNG.standard_normal((2, 3, 32, 32)).astype(np.float32)
    codes, scales = np.zeros((2, 3, 40, 32), np.int8), np.full((2, 3, 3), 9.0, np.float32)
    B.append_int8(codes, scales, rows, [0, 0], 16)
    v = B.values_int8(codes, scales, 16)[:, :, :32]
    step = np.abs(rows).reshape(2, 3, 2, -1).max(-1) / 127
    np.testing.assert_allclose(scales[:, :, :2], step, rtol=1e-6)
    assert (np.abs(v - rows).reshape(2, 3, 2, -1) <= 0.5001 * step[..., None]).all()
    assert (scales[:, :, 2] == 9).all() and (codes[:, :, 32:] == 0).all()   # nothing behind the last row


def test_append_row_by_row_grows_and_keeps_what_came_before():
    rows = (RNG.standard_normal((1, 1, 16, 32)) * np.linspace(0.1, 3, 16)[:, None]).astype(np.float32)
    codes, scales = RNG.integers(-127, 128, (1, 1, 16, 32)).astype(np.int8), np.ones((1, 1, 1), np.float32)
    for t in range(16):
        behind = codes[:, :, t + 1:].copy()
        B.append_int8(codes, scales, rows[:, :, t:t + 1], [t], 16)
        np.testing.assert_array_equal(codes[:, :, t + 1:], behind)
    # every growth adds half a step of a scale that ends at the largest
    v = B.values_int8(codes, scales, 16)
    top = np.abs(rows).max() / 127
    assert abs(float(scales[0, 0, 0]) - top) < 1e-6
    assert np.abs(v - rows).max() <= 16 * 0.5 * top


def test_append_drops_rows_outside_and_marks_infinities():
    codes, scales = np.zeros((2, 1, 20, 32), np.int8), np.zeros((2, 1, 2), np.float32)
    rows = np.ones((2, 1, 6, 32), np.float32)
    B.append_int8(codes, scales, rows, [-2, 17], 16)
    assert (codes[0, 0, :4] == 127).all() and (codes[0, 0, 4:] == 0).all()
    assert (codes[1, 0, 17:20] == 127).all() and (codes[1, 0, :17] == 0).all()
    rows[0, 0, 3, 5] = np.inf
    B.append_int8(codes, scales, rows, [0, 20], 16)
    assert np.isnan(B.values_int8(codes, scales, 16)[0, 0, :16]).all()
    assert (B.values_int8(codes, scales, 16)[0, 0, 16:] == 0).all()


def test_attention_is_torch_sdpa():
    q = RNG.standard_normal((2, 6, 3, 32))
    k, v = RNG.standard_normal((2, 2, 2, 9, 32))
    out = B.decode_attention(q, k, v, [9, 2])
    t = [torch.tensor(x) for x in (q, np.repeat(k, 3, 1), np.repeat(v, 3, 1))]
    for b, n in enumerate((9, 2)):
        seen = torch.arange(9)[None] <= n - 3 + torch.arange(3)[:, None]
        want = torch.nn.functional.scaled_dot_product_attention(
            t[0][b], t[1][b], t[2][b], attn_mask=seen).numpy()
        first = max(0, 3 - n)
        np.testing.assert_allclose(out[b, :, first:], want[:, first:], atol=1e-12)
        assert (out[b, :, :first] == 0).all()


@pytest.mark.parametrize("N,K,group", [(16, 128, 128), (5, 33, 32), (17, 200, 64)])
def test_int4_packing_by_bits(N, K, group):
    w = RNG.standard_normal((N, K)).astype(np.float32)
    codes, scales = B.quantize_int4(w, group)
    assert np.abs(B.values_int4(codes, scales, group) - w).max() <= 0.5001 * scales.max()
    words = np.ascontiguousarray(B.pack_int4(codes)).view("<u4")   # [tiles, steps, 64, 4]
    back = np.zeros((words.shape[0] * 16, words.shape[1] * 128), np.int32)
    for t, s, l, i in np.ndindex(*words.shape):
        for j in range(8):
            e = 2 * j if j < 4 else 2 * (j - 4) + 1
            back[t * 16 + l % 16, s * 128 + 32 * (l // 16) + 8 * i + e] = int(words[t, s, l, i] >> 4 * j & 15) - 8
    np.testing.assert_array_equal(back[:N, :K], codes)
    assert (back[N:] == 0).all() and (back[:, K:] == 0).all()


def test_logprobs_and_their_gradient_against_torch():
    z = RNG.standard_normal((7, 50)) * 3
    z[2, 5:20] = -np.inf
    tokens = np.array([3, 49, 2, 0, -100, 50, 7])
    lp, H, lse, tl, ti = B.token_logprobs(z, tokens, 4)
    t = torch.tensor(z, requires_grad=True)
    logp = torch.log_softmax(t, 1)
    there = (tokens >= 0) & (tokens < 50)
    want = torch.where(torch.tensor(there), logp[torch.arange(7), torch.tensor(tokens).clamp(0, 49)], 0.0)
    want_H = torch.special.entr(logp.exp()).sum(1)
    np.testing.assert_allclose(lp, want.detach().numpy(), atol=1e-12)
    np.testing.assert_allclose(H, want_H.detach().numpy(), atol=1e-12)
    np.testing.assert_allclose(lse, torch.logsumexp(t, 1).detach().numpy(), atol=1e-12)
    np.testing.assert_array_equal(ti, torch.topk(t, 4, 1).indices.numpy())
    np.testing.assert_allclose(tl, np.take_along_axis(logp.detach().numpy(), ti, 1), atol=1e-12)
    g, gh = RNG.standard_normal((2, 7))
    got = B.token_logprobs_backward(g, gh, z, tokens)
    # against differences of the function itself
    f = lambda x: sum((g * B.token_logprobs(x, tokens)[0] + gh * B.token_logprobs(x, tokens)[1]))  # noqa: E731
    for r, j in [(0, 3), (0, 4), (1, 0), (2, 2), (2, 30), (4, 1), (5, 9), (6, 7)]:
        a, b = z.copy(), z.copy()
        a[r, j] += 1e-5
        b[r, j] -= 1e-5
        assert abs((f(a) - f(b)) / 2e-5 - got[r, j]) < 1e-8
    assert (got[2, 5:20] == 0).all()


def test_logprobs_edges():
    z = np.array([[-np.inf, -np.inf, -np.inf], [1.0, np.nan, 2.0], [0.0, -0.0, 0.0], [np.inf, 0.0, 0.0]])
    lp, H, lse, tl, ti = B.token_logprobs(z, [1, 0, 2, -1], 3)
    assert lp[0] == -np.inf and H[0] == 0 and lse[0] == -np.inf and (tl[0] == -np.inf).all()
    assert np.isnan(lp[1]) and np.isnan(H[1]) and np.isnan(lse[1])
    np.testing.assert_array_equal(ti, [[0, 1, 2], [1, 2, 0], [0, 1, 2], [0, 1, 2]])
    assert lp[3] == 0 and np.isnan(lse[3])
