"""numpy restatement of the operators in few bits and of token log
probabilities (test infrastructure only), from their definitions.  The
reference has none of them; what pins these functions is
tests/test_few_bits_oracle.py: closed forms, brute force and PyTorch CPU.

Codes and scales follow float32 arithmetic exactly (a maximum, one division,
one rounding half to even), everything that is summed float64.
"""
from __future__ import annotations

import numpy as np

F32, F64 = np.float32, np.float64


def round_to(a, dtype: str):
    """float32 values rounded to a device dtype, as float32."""
    a = np.asarray(a, F32)
    if dtype == "float16":
        with np.errstate(over="ignore"):
            return a.astype(np.float16).astype(F32)
    if dtype == "bfloat16":
        u = a.view(np.uint32).astype(np.uint64)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(F32)
        return np.where(np.isnan(a), a, r)
    return a


# ── cache in 8 bits ─────────────────────────────────────────────────────────
def append_int8(codes, scales, rows, pos, block):
    """rows [B, H, T, D] become rows pos[b].. of codes [B, H, Tmax, D] with
    scales [B, H, ceil(Tmax / block)], in place, block by block."""
    B, H, T, _ = rows.shape
    Tmax = codes.shape[2]
    for b in range(B):
        p = int(pos[b])
        a, end = max(p, 0), min(p + T, Tmax)
        while a < end:
            n = a // block
            lo, z = n * block, min((n + 1) * block, end)
            for h in range(H):
                x = rows[b, h, a - p:z - p].astype(F32)
                mags = np.abs(x)
                s = F32(np.nan) if np.isnan(mags).any() else F32(mags.max()) / F32(127)
                old = F32(scales[b, h, n]) if lo < a else F32(0)
                if not (np.isnan(old) or s < old or s == old):   # grows (NaN above all)
                    ok = np.isfinite(s) and s > 0
                    rate = old / s if ok else F32(0)
                    codes[b, h, lo:a] = np.rint(codes[b, h, lo:a].astype(F32) * rate).astype(np.int8)
                    old = s
                s = old
                ok = np.isfinite(s) and s > 0
                c = np.rint(x / s) if ok else np.zeros_like(x)
                codes[b, h, a:z] = np.clip(c, -127, 127).astype(np.int8)
                scales[b, h, n] = s
            a = z


def values_int8(codes, scales, block):
    """float32 values of codes [B, H, Tmax, D]."""
    with np.errstate(invalid="ignore"):
        return codes.astype(F32) * np.repeat(scales, block, axis=2)[:, :, :codes.shape[2], None].astype(F32)


def decode_attention(q, k, v, lens, scale=None):
    """q [B, Hq, Tq, D] over values k, v [B, H, Tmax, D] in float64: query row
    i of sequence b sees rows j <= lens[b] - Tq + i; zeros where it sees none."""
    B, Hq, Tq, D = q.shape
    H, Tmax = k.shape[1], k.shape[2]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out = np.zeros((B, Hq, Tq, D), F64)
    for b in range(B):
        n = int(min(max(int(lens[b]), 0), Tmax))
        for h in range(Hq):
            kk, vv = k[b, h * H // Hq].astype(F64), v[b, h * H // Hq].astype(F64)
            for i in range(Tq):
                m = n - Tq + i + 1
                if m <= 0:
                    continue
                s = kk[:m] @ q[b, h, i].astype(F64) * scale
                e = np.exp(s - s.max())
                out[b, h, i] = e @ vv[:m] / e.sum()
    return out


# ── 4-bit weights ───────────────────────────────────────────────────────────
def quantize_int4(w, group, dtype="float32"):
    """(codes [N, K], scales [ceil(K / group), N]) of W [N, K], the scales
    rounded to dtype."""
    N, K = w.shape
    G = -(-K // group)
    codes, scales = np.zeros((N, K), np.int8), np.zeros((G, N), F32)
    for g in range(G):
        x = w[:, g * group:(g + 1) * group].astype(F32)
        s = round_to(np.abs(x).max(1) / F32(7), dtype)
        scales[g] = s
        ok = np.isfinite(s) & (s > 0)
        r = np.zeros_like(x)
        r[ok] = np.rint(x[ok] / s[ok, None])
        codes[:, g * group:(g + 1) * group] = np.clip(r, -7, 7).astype(np.int8)
    return codes, scales


def pack_int4(codes):
    """The packed bytes [ceil(N / 16), ceil(K / 128), 64, 16] of codes [N, K]."""
    N, K = codes.shape
    out = np.full((-(-N // 16), -(-K // 128), 64, 16), 0x88, np.uint8)
    for k in range(K):
        e = k % 8
        nib = e // 2 + 4 * (e % 2)
        byte = k % 32 // 8 * 4 + nib // 2
        for n in range(N):
            at = (n // 16, k // 128, n % 16 + 16 * (k % 128 // 32), byte)
            u = int(codes[n, k]) + 8
            out[at] = (int(out[at]) & ~(15 << 4 * (nib % 2))) | u << 4 * (nib % 2)
    return out


def values_int4(codes, scales, group):
    """float64 values [N, K] (exact: a code times a scale)."""
    return codes.astype(F64) * np.repeat(scales.T.astype(F64), group, axis=1)[:, :codes.shape[1]]


def linear(x, w, bias=None, act=None):
    y = x.astype(F64) @ w.T
    if bias is not None:
        y = y + bias.astype(F64)
    if act == "relu":
        return np.maximum(y, 0)
    if act == "gelu":
        u = np.clip(0.7978845608 * (y + 0.044715 * y ** 3), -10, 10)
        return 0.5 * y * (1 + np.tanh(u))
    if act == "gelu_exact":
        from scipy.special import erf
        return 0.5 * y * (1 + erf(y / np.sqrt(2.0)))
    return y


# ── log probabilities ───────────────────────────────────────────────────────
def token_logprobs(z, tokens, top_k=0):
    """(logprobs, entropy, lse, top_logprobs, top_ids) of rows z [R, V]."""
    z = np.asarray(z, F64)
    R, V = z.shape
    lp, H, lse = np.zeros(R), np.zeros(R), np.zeros(R)
    tl, ti = np.zeros((R, top_k)), np.zeros((R, top_k), np.int32)
    for r in range(R):
        row, t = z[r], int(tokens[r])
        m = np.nan if np.isnan(row).any() else row.max()
        if m == -np.inf:
            lse[r], lp[r] = m, m if 0 <= t < V else 0.0
            logp = np.full(V, -np.inf)
        elif not np.isfinite(m):
            lse[r] = H[r] = np.nan
            lp[r] = np.nan if 0 <= t < V else 0.0
            logp = np.full(V, np.nan)
        else:
            e = np.exp(row - m)
            lse[r] = m + np.log(e.sum())
            logp = row - m - np.log(e.sum())
            H[r] = -(np.exp(logp) * np.where(e > 0, logp, 0.0)).sum()
            lp[r] = logp[t] if 0 <= t < V else 0.0
        # larger first, equal ones by index, NaN above all
        order = np.lexsort((np.arange(V), -np.where(np.isnan(row), np.inf, row), ~np.isnan(row)))[:top_k]
        ti[r], tl[r] = order, logp[order]
    return lp, H, lse, tl, ti


def token_logprobs_backward(g_lp, g_h, z, tokens):
    """Gradient of sum(g_lp logprobs + g_h entropy) with respect to z, float64."""
    z = np.asarray(z, F64)
    _, H, lse, _, _ = token_logprobs(z, tokens)
    out = np.zeros_like(z)
    for r in range(z.shape[0]):
        t = int(tokens[r])
        if lse[r] == -np.inf:
            continue
        logp = z[r] - lse[r]
        p = np.exp(logp)
        if 0 <= t < z.shape[1]:
            out[r] -= g_lp[r] * p
            out[r, t] += g_lp[r]
        if g_h is not None:
            out[r] -= g_h[r] * np.where(p > 0, p * (np.where(p > 0, logp, 0) + H[r]), 0.0)
    return out
