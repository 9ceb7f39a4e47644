"""numpy restatement of the operators of a training step (test infrastructure
only), from their definitions in float64: the cross entropy of a linear layer
with its gradient, orthogonalised updates and the step that applies them.  The
reference has none of them; what pins these functions is
tests/test_training_oracle.py: closed forms, differences and PyTorch CPU.
"""
from __future__ import annotations

import numpy as np

F32, F64 = np.float32, np.float64
COEFFS = (3.4445, -4.7750, 2.0315)


def linear_cross_entropy(x, w, targets):
    """(loss, lse) of the logits x w^T; a target that is no word has loss 0."""
    z = np.asarray(x, F64) @ np.asarray(w, F64).T
    R, V = z.shape
    t = np.asarray(targets, np.int64)
    there = (t >= 0) & (t < V)
    zt = z[np.arange(R), np.clip(t, 0, V - 1)]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        top = z.max(1)
        lse = top + np.log(np.exp(z - top[:, None]).sum(1))
        # loss = log(1 + sum of the others' exp(z - zt))
        others = z.copy()
        others[np.arange(R)[there], t[there]] = -np.inf
        m = others.max(1, initial=-np.inf)
        ref = np.where(np.isfinite(m), m, 0.0)
        rest = np.exp(others - ref[:, None]).sum(1)
        loss = np.where(zt >= m, np.log1p(rest * np.exp(ref - zt)), (m - zt) + np.log(rest + np.exp(zt - ref)))
    return np.where(there, loss, 0.0), lse


def logit_gradients(x, w, targets, g_loss, g_lse=None):
    """d = g_loss (p - [v = t]) + g_lse p of every logit [R, V]."""
    z = np.asarray(x, F64) @ np.asarray(w, F64).T
    R, V = z.shape
    loss, lse = linear_cross_entropy(x, w, targets)
    t = np.asarray(targets, np.int64)
    there = (t >= 0) & (t < V)
    g = np.where(there, np.asarray(g_loss, F64), 0.0)
    h = np.zeros(R) if g_lse is None else np.asarray(g_lse, F64)
    p = np.exp(z - lse[:, None])
    d = p * (g + h)[:, None]
    at = np.arange(R)[there]
    d[at, t[there]] = g[there] * np.expm1(-loss[there]) + h[there] * p[at, t[there]]
    return np.where(((g != 0) | (h != 0))[:, None], d, 0.0)


def linear_cross_entropy_backward(x, w, targets, g_loss, g_lse=None):
    d = logit_gradients(x, w, targets, g_loss, g_lse)
    return d @ np.asarray(w, F64), d.T @ np.asarray(x, F64)


# ── orthogonalised updates ──────────────────────────────────────────────────
def planes(a, n, unit=2.0 ** 14):
    """Values held times `unit` as n float16 planes (high, then what it left)."""
    out, rest = np.zeros_like(a), np.asarray(a, F64) * unit
    for _ in range(n):
        h = rest.astype(np.float16).astype(F64)
        out, rest = out + h, rest - h
    return out / unit


def orthogonalize(g, steps=5, eps=1e-7, halves=0):
    """[..., m, n] by Newton-Schulz products in float64.  With halves = 1 or 2
    (or one for each step) the factors of every product are rounded as the
    device holds them (that many float16 planes), for a measure of what these
    roundings alone do; with 2, products are summed in float32 too."""
    a, b, c = COEFFS
    g = np.asarray(g, F64)

    per_step = list(halves) if isinstance(halves, (list, tuple)) else [halves] * steps

    def hold(x):
        return planes(x, n) if n else x

    def mul(x, y):
        if n == 2:   # high x high + high x low + low x high, float32 sums
            (xh, yh) = (planes(x, 1), planes(y, 1))
            (xl, yl) = (x - xh, y - yh)
            x32 = np.concatenate([xh, xh, xl], -1).astype(F32)
            y32 = np.concatenate([yh, yl, yh], -2).astype(F32)
            return (x32 @ y32).astype(F64)
        return x @ y

    norm = np.sqrt((g * g).sum((-2, -1), keepdims=True)) + eps
    x = g / np.where(norm > 0, norm, 1.0)
    tall = g.shape[-2] > g.shape[-1]
    for n in per_step:
        xr = hold(x)
        xt = np.swapaxes(xr, -1, -2)
        A = hold(mul(xt, xr) if tall else mul(xr, xt))
        B = hold(b * A + c * mul(A, A))
        x = a * x + (mul(xr, B) if tall else mul(B, xr))
        if n:
            x = x.astype(F32).astype(F64)
    return x


def muon_step(w, mom, grad, lr, beta, decay, nesterov=True, steps=5, eps=1e-7, halves=0):
    """(weight, momentum) after one step."""
    mom = beta * np.asarray(mom, F64) + np.asarray(grad, F64)
    u = np.asarray(grad, F64) + beta * mom if nesterov else mom
    rate = lr * np.sqrt(max(1.0, w.shape[-2] / w.shape[-1]))
    return (1.0 - lr * decay) * np.asarray(w, F64) - rate * orthogonalize(u, steps, eps, halves), mom
