"""The operators of a language model's training step at its two ends, as cases
that can be timed and compared: the softmax cross entropy of a linear layer
over a vocabulary, whose logits are never kept, and its gradient; and the
orthogonalised update of a weight matrix (Newton-Schulz products), alone and
as an optimiser's step with momentum in place.

`listed()` gives the fixed cases, `draw(rng)` one more of the same ranges;
`prepare`, `run`, `work` and `exact` take a case.  With `own` false, `run`
computes each operator's plain form in elementary torch operations; with `own`
true it calls the framework's operator.  Inputs are made on the GPU from the
seed.

  loss       z = x w^T, lse = log sum exp z, loss = lse - z[target]; a target
             that is no word (-100) has loss 0
  gradient   d = grad_loss (softmax z - onehot) + grad_lse softmax z;
             dx = d w, dw = d^T x
  update     X = G / (|G| + eps), the shorter side first; five times
             A = X X^T, B = b A + c A A, X = a X + B X
  step       M = beta M + G, U = G + beta M, W = (1 - lr decay) W
             - lr sqrt(max(1, rows / columns)) update(U)
"""
from __future__ import annotations

import math

import torch

own = False

VOCAB = 50257
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
COEFFS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.01


# ── the cases ───────────────────────────────────────────────────────────────
def listed():
    return [
        # the loss of one word of GPT-2 large: the read of the whole table
        dict(name="ce_token_f16", kind="loss", R=1, K=1280, V=VOCAB, dtype="float16"),
        # a prompt scored in fp32
        dict(name="ce_prompt_f32", kind="loss", R=255, K=768, V=VOCAB, dtype="float32"),
        # a small model of odd sizes, whose rows no 16-byte load fits
        dict(name="ce_odd_f16", kind="loss", R=1111, K=515, V=10007, dtype="float16"),
        # the words of a training batch (8 texts of 1024, one word less)
        dict(name="ce_text_bf16", kind="loss", R=8191, K=768, V=VOCAB, dtype="bfloat16"),
        # the gradient of a short answer's words, for fine tuning
        dict(name="ce_grad_answer_f16", kind="loss_grad", R=61, K=1280, V=VOCAB, dtype="float16"),
        # the gradient of one text in fp32
        dict(name="ce_grad_f32", kind="loss_grad", R=1023, K=768, V=VOCAB, dtype="float32"),
        # that of a training batch
        dict(name="ce_grad_text_bf16", kind="loss_grad", R=8191, K=768, V=VOCAB, dtype="bfloat16"),
        # the hidden layer of the small MLP: only the latency of a call counts
        dict(name="ortho_small_f32", kind="ortho", L=1, m=128, n=64, dtype="float32"),
        # the attention projections of GPT-2's twelve layers at once
        dict(name="ortho_layers_bf16", kind="ortho", L=12, m=768, n=768, dtype="bfloat16"),
        # a widening layer of GPT-2 large, four layers at once
        dict(name="ortho_wide_f16", kind="ortho", L=4, m=5120, n=1280, dtype="float16"),
        # the hidden layers of the wide MLP, in fp32
        dict(name="muon_mlp_f32", kind="muon", L=2, m=4096, n=4096, dtype="float32"),
        # the joined query, key and value weights of GPT-2's twelve layers
        dict(name="muon_qkv_bf16", kind="muon", L=12, m=768, n=2304, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["loss", "loss_grad", "loss_grad", "ortho", "muon"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if kind in ("loss", "loss_grad"):
        K, V = _log(rng, 64, 1280), _log(rng, 100, VOCAB)
        if rng.random() < 0.5:
            K = -(-K // 64) * 64
        # no more work than the listed cases have, and logits that fit the plain form
        most = 8191 * 768 * VOCAB // (K * V) // (1 if dtype != "float32" else 3)
        return dict(kind=kind, R=_log(rng, 1, max(1, min(16384, most))), K=K, V=V, dtype=dtype)
    m, n = _log(rng, 8, 4096), _log(rng, 8, 4096)
    short, long = min(m, n), max(m, n)
    most = 2 * 4096 ** 3 // (short * short * long)
    return dict(kind=kind, L=_log(rng, 1, max(1, min(16, most))), m=m, n=n, dtype=dtype)


# ── inputs, from the seed alone ─────────────────────────────────────────────
def _rand(seed):
    g = torch.Generator("cuda")
    g.manual_seed(int(seed))

    def randn(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    return g, randn


def _gradients(c, randn):
    """Gradients of L matrices as training gives them: a few directions hold
    most of each, the sizes differ from matrix to matrix."""
    L, m, n = c["L"], c["m"], c["n"]
    r = max(1, min(m, n) // 8)
    size = torch.exp(randn(L, 1, 1)) * 1e-3
    strong = torch.matmul(randn(L, m, r), randn(L, r, n)) / math.sqrt(r)
    return size * (strong + 0.3 * randn(L, m, n))


def _inputs(c, seed):
    g, randn = _rand(seed)
    dt = getattr(torch, c["dtype"])
    if c["kind"] == "ortho":
        return dict(g=_gradients(c, randn).to(dt))
    if c["kind"] == "muon":
        L, m, n = c["L"], c["m"], c["n"]
        return dict(w=randn(L, m, n, std=0.02).to(dt), m=4.0 * _gradients(c, randn), g=_gradients(c, randn).to(dt))
    R, K, V = c["R"], c["K"], c["V"]
    w = randn(V, K, std=4.0 / math.sqrt(K)).to(dt)
    t = torch.randint(0, V, (R,), generator=g, device="cuda")
    u = torch.rand((R,), generator=g, device="cuda")
    # from a word that is as likely as any other to one that is nearly certain
    x = (randn(R, K) + 1.5 * u[:, None] * w[t].float()).to(dt)
    pad = torch.rand((R,), generator=g, device="cuda") > 0.95
    t = torch.where(pad, -100, t).to(torch.int32)
    if R == 1:
        t.clamp_(min=0)
    if c["kind"] == "loss":
        return dict(x=x, w=w, t=t)
    loss, lse = _f64_loss(x, w, t)
    weight = torch.rand((R,), generator=g, device="cuda") / R
    return dict(x=x, w=w, t=t, loss=loss.float(), lse=lse.float(), g_loss=weight, g_lse=2e-3 * weight * lse.float())


# ── what a user's program has in hand ───────────────────────────────────────
def prepare(case, seed):
    s = _inputs(case, seed)
    if own:   # a program of the framework holds its data as the framework's tensors
        one_each = case["kind"] == "muon"   # and a model's weights one by one
        s = {k: [_upload(x) for x in v] if one_each else _upload(v) for k, v in s.items()}
    return dict(s, case=dict(case))


# ── one pass, plain ─────────────────────────────────────────────────────────
def _loss(s):
    z = s["x"].float() @ s["w"].float().t()
    t = s["t"].long()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    there = (t >= 0) & (t < z.shape[1])
    at = t.clamp(0, z.shape[1] - 1)[:, None]
    lse = top[:, 0] + torch.log(e.sum(1))
    zt = z.gather(1, at)[:, 0]
    # the rest of the sum without the target's own part: a nearly certain
    # word's loss keeps its digits
    rest = e.scatter(1, at, 0.0).sum(1)
    loss = torch.where(zt == top[:, 0], torch.log1p(rest), lse - zt)
    return [torch.where(there, loss, 0.0), lse]


def _loss_grad(s):
    x, w, t = s["x"].float(), s["w"].float(), s["t"].long()[:, None]
    V = w.shape[0]
    p = torch.exp(x @ w.t() - s["lse"][:, None])
    there = (t >= 0) & (t < V)
    g, h = s["g_loss"][:, None] * there, s["g_lse"][:, None]
    d = p * (g + h)
    at = t.clamp(0, V - 1)
    # p - 1 of the target from its loss, which keeps the digits of 1 - p
    word = g * torch.expm1(-s["loss"][:, None]) + h * p.gather(1, at)
    d.scatter_(1, at, torch.where(there, word, d.gather(1, at)))
    return [(d @ w).to(s["x"].dtype), (d.t() @ x).to(s["w"].dtype)]


def _orthogonal(g):
    """[L, m, n] float32 to its orthogonalised form."""
    a, b, c = COEFFS
    x = g.mT.contiguous() if g.shape[1] > g.shape[2] else g
    x = x / (torch.sqrt((x.double() ** 2).sum((1, 2), keepdim=True)).float() + EPS)
    for _ in range(STEPS):
        A = torch.matmul(x, x.mT)
        x = a * x + torch.matmul(b * A + c * torch.matmul(A, A), x)
    return x.mT if g.shape[1] > g.shape[2] else x


def _muon(s):
    w, m, g = s["w"], s["m"], s["g"].float()
    m.mul_(BETA).add_(g)
    o = _orthogonal(g + BETA * m)
    rate = LR * math.sqrt(max(1.0, w.shape[1] / w.shape[2]))
    w.copy_((1.0 - LR * DECAY) * w.float() - rate * o)
    return [list(w), list(m)]   # matrix by matrix


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["kind"] == "loss":
        return _loss(s)
    if c["kind"] == "loss_grad":
        return _loss_grad(s)
    return _orthogonal(s["g"].float()).to(s["g"].dtype) if c["kind"] == "ortho" else _muon(s)


# ── one pass, by the framework ──────────────────────────────────────────────
def _package():
    import os
    import sys
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "applegpu-runtime_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import applegpu_runtime as gpu
    return gpu


class _Buffer:
    """A device buffer as torch takes one; keeps its owner alive."""

    def __init__(self, ptr, shape, typestr, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "strides": None, "typestr": typestr, "data": (ptr, False),
                                         "version": 3}


_TYPESTR = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2", "int32": "<i4"}


def _view(gpu, t, shape, dtype):
    """A GpuTensor's values as a torch tensor, in place; evaluates it first."""
    ptr = gpu.lib.applegpu_eager_data_ptr(t.id)
    if not ptr:
        raise RuntimeError(gpu.ffi_error())
    x = torch.as_tensor(_Buffer(ptr, tuple(shape), _TYPESTR[dtype], t), device="cuda")
    return x.view(torch.bfloat16) if dtype == "bfloat16" else x


def _upload(t):
    """A GpuTensor with the values of a tensor on torch's GPU."""
    gpu = _package()
    dtype = str(t.dtype).replace("torch.", "")
    out = gpu.zeros(list(t.shape), dtype)
    gpu.synchronize()
    _view(gpu, out, t.shape, dtype).copy_(t)
    torch.cuda.synchronize()
    return out


def _own(s, c):
    gpu = _package()
    dtype = c["dtype"]
    if c["kind"] == "loss":
        got = gpu.linear_cross_entropy(s["x"], s["w"], s["t"])
        return [_view(gpu, t, (c["R"],), "float32") for t in got]
    if c["kind"] == "loss_grad":
        dx, dw = gpu.linear_cross_entropy_backward(s["g_loss"], s["x"], s["w"], s["t"], s["loss"], s["lse"],
                                                   grad_lse=s["g_lse"])
        return [_view(gpu, dx, (c["R"], c["K"]), dtype), _view(gpu, dw, (c["V"], c["K"]), dtype)]
    shape = (c["m"], c["n"])
    if c["kind"] == "ortho":
        return _view(gpu, gpu.orthogonalize(s["g"], steps=STEPS, eps=EPS), (c["L"],) + shape, dtype)
    gpu.muon_step_(s["w"], s["m"], s["g"], lr=LR, beta=BETA, weight_decay=DECAY, steps=STEPS, eps=EPS)
    return [[_view(gpu, t, shape, dtype) for t in s["w"]], [_view(gpu, t, shape, "float32") for t in s["m"]]]


# ── what a pass cannot do without ───────────────────────────────────────────
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["kind"] in ("loss", "loss_grad"):
        R, K, V = c["R"], c["K"], c["V"]
        if c["kind"] == "loss":
            return dict(bytes=e * K * (R + V) + 12 * R, flops=2 * R * K * V)
        # the logits are formed again, then two products
        return dict(bytes=2 * e * K * (R + V) + 20 * R, flops=6 * R * K * V)
    L, short, long = c["L"], min(c["m"], c["n"]), max(c["m"], c["n"])
    # X X^T and A A are symmetric: half of each is enough
    flops = L * STEPS * (3 * short * short * long + short ** 3)
    n = L * short * long
    return dict(bytes=n * (2 * e if c["kind"] == "ortho" else 3 * e + 8), flops=flops)


# ── the same outputs in 64 bits, from the definitions ───────────────────────
def _f64_loss(x, w, t):
    """Loss and log sum of exponentials, some rows at a time."""
    V, w = w.shape[0], w.double()
    losses, sums = [], []
    for lo in range(0, x.shape[0], 2048):
        z, ti = x[lo:lo + 2048].double() @ w.t(), t[lo:lo + 2048].long()
        there = (ti >= 0) & (ti < V)
        pick = torch.nn.functional.one_hot(ti.clamp(0, V - 1), V).bool()
        zt = z[pick]
        # loss = log(1 + sum of the others' exp(z - zt))
        others = torch.logsumexp(z.masked_fill(pick, float("-inf")), 1)
        losses.append(torch.where(there, torch.nn.functional.softplus(others - zt, threshold=700.0), 0.0))
        sums.append(torch.logaddexp(others, zt))
    return torch.cat(losses), torch.cat(sums)


def _f64_orthogonal(g):
    """One matrix after the other, by the singular values' polynomial applied
    as products of the Gram matrix of the shorter side."""
    a, b, c = COEFFS
    out = []
    for x in g.double():
        tall = x.shape[0] > x.shape[1]
        x = x / (torch.linalg.vector_norm(x) + EPS)
        for _ in range(STEPS):
            gram = x.t().contiguous() @ x if tall else x @ x.t().contiguous()
            poly = a * torch.eye(gram.shape[0], dtype=x.dtype, device=x.device) + b * gram + c * (gram @ gram)
            x = x @ poly if tall else poly @ x
        out.append(x)
    return torch.stack(out)


def exact(case, seed):
    c, i = case, _inputs(case, seed)
    if c["kind"] == "loss":
        return list(_f64_loss(i["x"], i["w"], i["t"]))
    if c["kind"] == "loss_grad":
        # by the loss and the sum as given
        w, V = i["w"].double(), c["V"]
        dx, dw = [], torch.zeros_like(w)
        for lo in range(0, c["R"], 2048):
            x, t, loss, lse, g, h = (i[k][lo:lo + 2048].double() for k in ("x", "t", "loss", "lse", "g_loss", "g_lse"))
            there = (t >= 0) & (t < V)
            d = torch.exp(x @ w.t() - lse[:, None])
            row, at = torch.arange(len(t), device=t.device)[there], t[there].long()
            pt = d[row, at]
            d *= (torch.where(there, g, 0.0) + h)[:, None]
            d[row, at] = -g[there] * (1.0 - torch.exp(-loss[there])) + h[there] * pt
            dx.append(d @ w)
            dw += d.t().contiguous() @ x
        return [torch.cat(dx), dw]
    if c["kind"] == "ortho":
        return _f64_orthogonal(i["g"])
    m = BETA * i["m"].double() + i["g"].double()
    o = _f64_orthogonal(i["g"].double() + BETA * m)
    w = i["w"].double() * (1.0 - LR * DECAY) - LR * math.sqrt(max(1.0, c["m"] / c["n"])) * o
    return [list(w), list(m)]
