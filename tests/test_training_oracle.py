"""The oracle of the training operators against closed forms, differences and
PyTorch (no GPU)."""
import numpy as np
import pytest
import torch

from oracle import training as O

RNG = np.random.default_rng(7)


def _ce(R, K, V):
    x, w = RNG.standard_normal((R, K)), RNG.standard_normal((V, K))
    t = RNG.integers(0, V, R)
    t[::3] = -100
    return x, w, t


@pytest.mark.parametrize("R,K,V", [(1, 3, 1), (5, 4, 7), (9, 16, 40)])
def test_cross_entropy_and_gradient_vs_torch(R, K, V):
    x, w, t = _ce(R, K, V)
    g, h = RNG.standard_normal(R), RNG.standard_normal(R)
    tx, tw = (torch.tensor(a, requires_grad=True) for a in (x, w))
    z = tx @ tw.t()
    loss = torch.nn.functional.cross_entropy(z, torch.tensor(t), reduction="none", ignore_index=-100)
    lse = torch.logsumexp(z, 1)
    ((loss * torch.tensor(g)).sum() + (lse * torch.tensor(h)).sum()).backward()
    got = O.linear_cross_entropy(x, w, t)
    np.testing.assert_allclose(got[0], loss.detach().numpy(), rtol=1e-12, atol=1e-12)
    np.testing.assert_allclose(got[1], lse.detach().numpy(), rtol=1e-12)
    dx, dw = O.linear_cross_entropy_backward(x, w, t, g, h)
    np.testing.assert_allclose(dx, tx.grad.numpy(), rtol=1e-10, atol=1e-12)
    np.testing.assert_allclose(dw, tw.grad.numpy(), rtol=1e-10, atol=1e-12)


def test_gradient_vs_differences():
    x, w, t = _ce(4, 5, 6)
    g, h = RNG.standard_normal(4), RNG.standard_normal(4)
    dx, dw = O.linear_cross_entropy_backward(x, w, t, g, h)

    def value(x, w):
        loss, lse = O.linear_cross_entropy(x, w, t)
        return (g * loss + h * lse).sum()

    for a, grad, f in ((x, dx, lambda a: value(a, w)), (w, dw, lambda a: value(x, a))):
        for at in np.ndindex(a.shape):
            step = np.zeros_like(a)
            step[at] = 1e-6
            assert abs((f(a + step) - f(a - step)) / 2e-6 - grad[at]) < 1e-7


def test_nearly_certain_word_keeps_its_digits():
    x, w = np.array([[40.0, 1.0]]), np.array([[1.0, 0.0], [0.0, 1.0]])
    loss, _ = O.linear_cross_entropy(x, w, [0])
    np.testing.assert_allclose(loss, np.exp(-39.0), rtol=1e-12)


@pytest.mark.parametrize("shape", [(1, 1), (5, 9), (9, 5), (3, 8, 8)])
def test_orthogonalize_acts_on_singular_values(shape):
    g = RNG.standard_normal(shape)
    u, s, vt = np.linalg.svd(g, full_matrices=False)
    s = s / np.sqrt((s * s).sum(-1, keepdims=True))
    for _ in range(5):
        s = O.COEFFS[0] * s + O.COEFFS[1] * s ** 3 + O.COEFFS[2] * s ** 5
    np.testing.assert_allclose(O.orthogonalize(g, eps=0.0), (u * s[..., None, :]) @ vt, atol=1e-9)


def test_orthogonalize_of_zeros_and_roundings():
    assert (O.orthogonalize(np.zeros((4, 6))) == 0).all()
    g = RNG.standard_normal((40, 60))
    want = O.orthogonalize(g)
    err = [np.linalg.norm(O.orthogonalize(g, halves=n) - want) / np.linalg.norm(want) for n in (1, 2)]
    assert 1e-6 < err[0] < 5e-3 and err[1] < 5e-6


def test_muon_step_vs_torch():
    w, m, g = (RNG.standard_normal((6, 4)) for _ in range(3))
    tw, tm, tg = (torch.tensor(a) for a in (w, m, g))
    tm = tm * 0.9 + tg
    for nesterov, u in ((True, tg + 0.9 * tm), (False, tm)):
        want = tw * (1 - 0.1 * 0.5) - 0.1 * np.sqrt(1.5) * torch.tensor(O.orthogonalize(u.numpy()))
        got = O.muon_step(w, m, g, 0.1, 0.9, 0.5, nesterov)
        np.testing.assert_allclose(got[0], want.numpy(), atol=1e-12)
        np.testing.assert_allclose(got[1], tm.numpy(), atol=1e-12)
