"""The operators of serving and scoring a GPT-2 in few bits, as cases that can
be timed and compared: attention over a key/value cache held in 8 bits with a
scale for each block of tokens and head, the append to that cache, linear
layers with 4-bit weights and group scales, and the log probabilities of given
tokens with their entropy, top alternatives and gradient.

`listed()` gives the fixed cases, `draw(rng)` one more of the same ranges;
`prepare`, `run`, `work` and `exact` take a case.  With `own` false, `run`
computes each operator's plain form in elementary torch operations; with `own`
true it calls the framework's operator.  Inputs are made on the GPU from the
seed.

Layouts that both forms share:
  cache      codes int8 [B, H, Tmax, D]; scales float32 [B, H, ceil(Tmax / block)],
             value = code * scale of the row's block
  4 bits     packed uint8 [ceil(N / 16), ceil(K / 128), 64, 16], tiles of 16 rows by
             128 columns of W [N, K]: byte run l of a tile holds the 32 codes of row
             l % 16 from column 32 (l / 16) on, eight codes to each 4 bytes, as
             code + 8: nibble j of the four bytes (lowest first) is code 2 j for
             j < 4 and code 2 (j - 4) + 1 for the others; scales [ceil(K / group), N]
"""
from __future__ import annotations

import math

import torch

own = False

VOCAB = 50257
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


# ── the cases ───────────────────────────────────────────────────────────────
def listed():
    return [
        # one token of one sequence with a short context: only the latency of
        # a call counts
        dict(name="cache_token_f16", kind="attention", B=1, H=12, G=1, D=64, Tq=1, context=100, Tmax=128, block=16,
             dtype="float16"),
        # one token of a batch at long contexts of unlike lengths, four query
        # heads to each key/value head: the read of the whole cache
        dict(name="cache_token_long_bf16", kind="attention", B=4, H=8, G=4, D=128, Tq=1, context=32700, Tmax=32768,
             block=32, dtype="bfloat16"),
        # a chunk of a prompt against what the cache holds already, in fp32
        dict(name="cache_chunk_f32", kind="attention", B=2, H=12, G=1, D=64, Tq=37, context=999, Tmax=1000, block=64,
             dtype="float32"),
        # the keys and values of one token of each of 8 sequences, at
        # positions of their own, appended and read back
        dict(name="cache_append_bf16", kind="cache", B=8, H=20, D=64, T=1, context=600, block=16, dtype="bfloat16"),
        # those of a batch of prompts, of a length that no block divides
        dict(name="cache_prompt_f16", kind="cache", B=8, H=20, D=64, T=509, context=0, block=16, dtype="float16"),
        # a decode step's widening layer for one sequence
        dict(name="int4_token_f16", kind="linear", M=1, K=1280, N=5120, group=128, act="gelu", dtype="float16"),
        # a large layer for a batch of 16 sequences: the read of the weights
        dict(name="int4_batch_bf16", kind="linear", M=16, K=8192, N=8192, group=64, act="", dtype="bfloat16"),
        # the same weights' layer over the rows of a batch of prompts
        dict(name="int4_prompt_f16", kind="linear", M=1111, K=1280, N=3840, group=128, act="", dtype="float16"),
        # a decode step's picks with five alternatives each, for 8 sequences
        dict(name="logprobs_token_f16", kind="logprobs", R=8, V=VOCAB, top_k=5, dtype="float16"),
        # the scoring of a whole text with 20 alternatives for each word
        dict(name="logprobs_text_f32", kind="logprobs", R=2047, V=VOCAB, top_k=20, dtype="float32"),
        # the gradient of those log probabilities and entropies for a short
        # answer, and for the words of a training batch
        dict(name="logprobs_grad_f32", kind="logprobs_grad", R=33, V=VOCAB, dtype="float32"),
        dict(name="logprobs_grad_bf16", kind="logprobs_grad", R=2047, V=VOCAB, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "cache", "linear", "linear", "logprobs", "logprobs_grad"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if kind == "attention":
        B, H, G = _log(rng, 1, 16), rng.randint(1, 20), rng.choice([1, 1, 2, 4])
        D, block = rng.choice([32, 64, 64, 128]), rng.choice([16, 32, 64, 128])
        Tq = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        # no more rows than the listed cases read, and scores that fit the plain form
        most = min(32768, 4 * 8 * 32768 * 128 // (B * H * D), (1 << 27) // (B * H * G * Tq))
        context = _log(rng, min(most, max(16, Tq)), most)
        return dict(kind=kind, B=B, H=H, G=G, D=D, Tq=min(Tq, context), context=context,
                    Tmax=context + rng.randint(0, 100), block=block, dtype=dtype)
    if kind == "cache":
        B, H, D = _log(rng, 1, 16), rng.randint(1, 20), rng.choice([32, 64, 64, 128])
        return dict(kind=kind, B=B, H=H, D=D, T=_log(rng, 1, min(1024, 8 * 20 * 64 * 509 // (B * H * D))),
                    context=rng.choice([0, _log(rng, 1, 1024)]), block=rng.choice([16, 32, 64, 128]), dtype=dtype)
    if kind == "linear":
        K, N = _log(rng, 64, 8192), _log(rng, 64, 8192)
        return dict(kind=kind, M=_log(rng, 1, max(16, min(1111, 1111 * 1280 * 3840 // (K * N)))), K=K, N=N,
                    group=rng.choice([32, 64, 128]), act=rng.choice(["", "relu", "gelu"]), dtype=dtype)
    V = _log(rng, 100, VOCAB)
    R = _log(rng, 1, min(4096, 2047 * VOCAB // V))
    if kind == "logprobs":
        return dict(kind=kind, R=R, V=V, top_k=rng.choice([0, 1, rng.randint(2, 20)]), dtype=dtype)
    return dict(kind=kind, R=R, V=V, dtype=dtype)


# ── inputs, from the seed alone ─────────────────────────────────────────────
def _rand(seed):
    g = torch.Generator("cuda")
    g.manual_seed(int(seed))

    def randn(*shape, std=1.0, dtype="float32"):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(getattr(torch, dtype))

    return g, randn


def _cache(c, randn, g, Tmax):
    """Codes and scales of B * H heads: rows of a size that differs from head
    to head and from block to block, as keys and values have them."""
    B, H, D, block = c["B"], c["H"], c["D"], c["block"]
    nb = -(-Tmax // block)
    codes = (torch.randn((B, H, Tmax, D), generator=g, device="cuda") * 40).round_().clamp_(-127, 127).to(torch.int8)
    return codes, torch.exp(randn(B, H, nb, std=0.3)) * randn(B, H, 1).abs().add_(0.3) * 0.02


def _write_span(c):
    """Rows of the blocks that an append of T rows touches at most."""
    return ((c["T"] + c["block"] - 2) // c["block"] + 1) * c["block"]


def _logits(c, randn, g):
    """Logits of a vocabulary: a few words likely, some of them ruled out."""
    R, V = c["R"], c["V"]
    z = randn(R, V, std=2.0)
    z += 3.0 * torch.rand((R, 1), generator=g, device="cuda") * randn(1, V)
    z[:, torch.randint(0, V, (V // 100 + 1,), generator=g, device="cuda")] = float("-inf")
    z[:, 0] = 1.0   # no row without a word
    z = z.to(getattr(torch, c["dtype"]))
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda")
    # most of the words asked for are likely ones; a padded place has none
    likely = z.float().add_(randn(R, V, std=0.1)).argmax(1)
    u = torch.rand((R,), generator=g, device="cuda")
    tokens = torch.where(u < 0.7, likely, tokens)
    tokens = torch.where(torch.isinf(z.gather(1, tokens[:, None])[:, 0]), 0, tokens)
    return z, torch.where(u > 0.95, -100, tokens).to(torch.int32)


def _inputs(c, seed):
    g, randn = _rand(seed)
    kind = c["kind"]
    if kind == "attention":
        kc, ks = _cache(c, randn, g, c["Tmax"])
        vc, vs = _cache(c, randn, g, c["Tmax"])
        lens = torch.randint(0, c["context"] + 1, (c["B"],), generator=g, device="cuda")
        lens = torch.maximum(lens, lens.new_tensor(c["context"] // 2))
        lens[0] = c["context"]
        return dict(q=randn(c["B"], c["H"] * c["G"], c["Tq"], c["D"], dtype=c["dtype"]), kc=kc, ks=ks, vc=vc, vs=vs,
                    lens=lens.to(torch.int32))
    if kind == "cache":
        B, H, D, T, block = (c[k] for k in ("B", "H", "D", "T", "block"))
        Tmax = -(-c["context"] // block) * block + _write_span(c) + block
        kc, ks = _cache(c, randn, g, Tmax)
        vc, vs = _cache(c, randn, g, Tmax)
        pos = torch.randint(0, c["context"] + 1, (B,), generator=g, device="cuda")
        pos[0] = c["context"]
        return dict(kc=kc, ks=ks, vc=vc, vs=vs, k=randn(B, H, T, D, dtype=c["dtype"]),
                    v=randn(B, H, T, D, dtype=c["dtype"]), pos=pos.to(torch.int32),
                    start=(pos // block * block).to(torch.int32))
    if kind == "linear":
        M, K, N, group = c["M"], c["K"], c["N"], c["group"]
        tiles, steps, groups = -(-N // 16), -(-K // 128), -(-K // group)
        codes = torch.full((tiles * 16, steps * 128), 8, dtype=torch.int32, device="cuda")
        codes[:N, :K] = torch.randint(1, 16, (N, K), generator=g, device="cuda", dtype=torch.int32)
        # [tile, row, step, run, 4-byte word, code, even or odd] to the order of
        # the runs; the even codes of a word come before the odd ones
        codes = codes.view(tiles, 16, steps, 4, 4, 4, 2).permute(0, 2, 3, 1, 4, 6, 5).reshape(tiles, steps, 64, 16, 2)
        packed = (codes[..., 0] | codes[..., 1] << 4).to(torch.uint8)
        scales = (torch.rand((groups, N), generator=g, device="cuda") + 0.5) * (0.2 / math.sqrt(K))
        return dict(x=randn(M, K, dtype=c["dtype"]), packed=packed, scales=scales.to(getattr(torch, c["dtype"])),
                    bias=randn(N, std=0.1, dtype=c["dtype"]))
    z, tokens = _logits(c, randn, g)
    if kind == "logprobs":
        return dict(z=z, tokens=tokens)
    _, H, lse = _f64_logprobs(z, tokens)[:3]
    return dict(z=z, tokens=tokens, H=H.float(), lse=lse.float(), g_lp=randn(c["R"]), g_H=randn(c["R"], std=0.1))


# ── what a user's program has in hand ───────────────────────────────────────
def prepare(case, seed):
    s = dict(_inputs(case, seed), case=dict(case))
    if own:   # a program of the framework holds its data as the framework's tensors
        s = {k: _upload(v) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    return s


# ── one pass, plain ─────────────────────────────────────────────────────────
def _values(codes, scales, block):
    """A cache's rows as the float32 values they stand for."""
    return codes.float() * scales.repeat_interleave(block, 2)[:, :, :codes.shape[2], None]


def _attention(s, c):
    """softmax(q k^T / sqrt(D)) v over the rows j <= len - Tq + i of query i;
    a query that sees no row gets zeros."""
    B, H, G, D, Tq, Tmax = (c[k] for k in ("B", "H", "G", "D", "Tq", "Tmax"))
    k, v = _values(s["kc"], s["ks"], c["block"]), _values(s["vc"], s["vs"], c["block"])
    scores = torch.matmul(s["q"].float().view(B, H, G * Tq, D), k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    j, i = torch.arange(Tmax, device="cuda"), torch.arange(Tq, device="cuda")
    seen = j <= s["lens"].view(B, 1, 1) - Tq + i[:, None]                      # [B, Tq, Tmax]
    scores = scores.view(B, H, G, Tq, Tmax).masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top)).view(B, H, G * Tq, Tmax)
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(B, H * G, Tq, D).to(s["q"].dtype)


def _append(codes, scales, rows, pos, start, c):
    """The rows become rows pos.. of the cache, in place.  A block's scale is
    its largest value / 127; one that held rows before `pos` keeps them, its
    scale grows where the new rows need it, and their codes with it.  Returns
    the touched blocks' rows."""
    B, H, D, T, block = (c[k] for k in ("B", "H", "D", "T", "block"))
    W = _write_span(c)
    at = start.long()[:, None] + torch.arange(W, device="cuda")                # [B, W]
    p = pos.long()[:, None]
    new, kept = (at >= p) & (at < p + T), at < p
    x = rows.float().gather(2, (at - p).clamp_(0, T - 1)[:, None, :, None].expand(B, H, W, D))
    x = torch.where(new[:, None, :, None], x, 0.0)
    blocks = (at[:, ::block] // block)[:, None].expand(B, H, W // block)
    was = scales.gather(2, blocks)
    held = kept[:, None, ::block]
    s = torch.maximum(torch.where(held, was, 0.0), x.abs().view(B, H, W // block, block * D).amax(-1) / 127.0)
    s = torch.where(new.view(B, 1, W // block, block).any(-1), s, was)
    scales.scatter_(2, blocks, s)
    wide = s.repeat_interleave(block, 2)[..., None]
    rate = (was / s).repeat_interleave(block, 2)[..., None]
    where = at[:, None, :, None].expand(B, H, W, D)
    old = codes.gather(2, where).float()
    grown = kept[:, None, :, None] & (rate < 1.0)
    code = torch.where(new[:, None, :, None], torch.round(x / wide).clamp_(-127, 127),
                       torch.where(grown, torch.round(old * rate), old))
    codes.scatter_(2, where, code.to(torch.int8))
    return (code * wide).to(rows.dtype)


def _linear(s, c):
    M, K, N = c["M"], c["K"], c["N"]
    byte = s["packed"]
    tiles, steps = byte.shape[:2]
    nib = torch.stack((byte & 15, byte >> 4), -1).view(tiles, steps, 4, 16, 4, 2, 4)
    nib = nib.permute(0, 3, 1, 2, 4, 6, 5).reshape(tiles * 16, steps * 128)[:N, :K]
    w = (nib.float() - 8.0) * s["scales"].float().t().repeat_interleave(c["group"], 1)[:, :K]
    y = s["x"].float() @ w.t() + s["bias"].float()
    if c["act"] == "relu":
        y = y.clamp_min(0.0)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y * y * y)))
    return y.to(s["x"].dtype)


def _logprobs(s, c):
    z, t = s["z"].float(), s["tokens"].long()
    R, V = z.shape
    top = z.amax(1, keepdim=True)
    d = z - top
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    H = log_total - torch.where(e > 0, e * d, 0.0).sum(1) / total
    lse = top[:, 0] + log_total
    there = (t >= 0) & (t < V)
    lp = torch.where(there, d.gather(1, t.clamp(0, V - 1)[:, None])[:, 0] - log_total, 0.0)
    if not c["top_k"]:
        return [lp, H, lse]
    # the largest values in order, equal ones by index: a whole number that
    # grows with the value, then with the distance from the end
    bits = (z + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) << 32) + (V - 1 - torch.arange(V, device="cuda"))
    ids = V - 1 - (key.topk(c["top_k"], 1).values & 0xFFFFFFFF)
    return [lp, H, lse, z.gather(1, ids) - lse[:, None], ids.to(torch.int32)]


def _logprobs_grad(s):
    z, t = s["z"].float(), s["tokens"].long()[:, None]
    R, V = z.shape
    logp = z - s["lse"][:, None]
    p = torch.exp(logp)
    there = ((t >= 0) & (t < V)).float()
    g = -p * (s["g_lp"][:, None] * there) - s["g_H"][:, None] * torch.where(p > 0, p * (logp + s["H"][:, None]), 0.0)
    g.scatter_add_(1, t.clamp(0, V - 1), s["g_lp"][:, None] * there)
    return g.to(s["z"].dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["kind"] == "attention":
        return _attention(s, c)
    if c["kind"] == "cache":
        return [_append(s["kc"], s["ks"], s["k"], s["pos"], s["start"], c),
                _append(s["vc"], s["vs"], s["v"], s["pos"], s["start"], c)]
    if c["kind"] == "linear":
        return _linear(s, c)
    return _logprobs(s, c) if c["kind"] == "logprobs" else _logprobs_grad(s)


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

    def __init__(self, ptr, shape, strides, typestr, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "strides": strides, "typestr": typestr, "data": (ptr, False),
                                         "version": 3}


_TYPESTR = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2", "int32": "<i4", "int8": "|i1", "uint8": "|u1"}


def _view(gpu, t, shape, dtype, strides=None):
    """A GpuTensor's values as a torch tensor, in place (strides in elements);
    evaluates it first."""
    code = _TYPESTR[dtype]
    if strides is not None:
        strides = tuple(int(code[-1]) * n for n in strides)
    ptr = gpu.lib.applegpu_eager_data_ptr(t.id)
    if not ptr:
        raise RuntimeError(gpu.ffi_error())
    x = torch.as_tensor(_Buffer(ptr, tuple(shape), strides, code, t), device="cuda")
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
    kind = c["kind"]
    if kind == "attention":
        B, Hq, Tq, D = c["B"], c["H"] * c["G"], c["Tq"], c["D"]
        o = gpu.decode_attention_int8(s["q"], s["kc"], s["ks"], s["vc"], s["vs"], s["lens"], block=c["block"])
        # stored token by token: [B, Tq, heads, D]
        return _view(gpu, o, (B, Hq, Tq, D), c["dtype"], (Tq * Hq * D, D, Hq * D, 1))
    if kind == "cache":
        gpu.kv_write_int8(s["kc"], s["ks"], s["vc"], s["vs"], s["k"], s["v"], s["pos"], block=c["block"])
        W = _write_span(c)
        got = gpu.kv_read_int8(s["kc"], s["ks"], s["vc"], s["vs"], s["start"], W, block=c["block"], dtype=c["dtype"])
        return [_view(gpu, t, (c["B"], c["H"], W, c["D"]), c["dtype"]) for t in got]
    if kind == "linear":
        y = gpu.linear_int4(s["x"], s["packed"], s["scales"], s["bias"], c["act"] or None, group=c["group"])
        return _view(gpu, y, (c["M"], c["N"]), c["dtype"])
    if kind == "logprobs":
        got = gpu.token_logprobs(s["z"], s["tokens"], top_k=c["top_k"])
        out = [_view(gpu, t, (c["R"],), "float32") for t in got[:3]]
        if c["top_k"]:
            out += [_view(gpu, got[3], (c["R"], c["top_k"]), "float32"),
                    _view(gpu, got[4], (c["R"], c["top_k"]), "int32")]
        return out
    g = gpu.token_logprobs_backward(s["g_lp"], s["g_H"], s["z"], s["tokens"], s["H"], s["lse"])
    return _view(gpu, g, (c["R"], c["V"]), c["dtype"])


# ── what a pass cannot do without ───────────────────────────────────────────
def work(case):
    c, kind, e = case, case["kind"], SIZE[case["dtype"]]
    if kind == "attention":
        # lengths lie between half the context and all of it, one at the top
        rows = c["B"] * c["H"] * (0.75 * (c["B"] - 1) + 1) / c["B"] * c["context"]
        queries = c["B"] * c["H"] * c["G"] * c["Tq"] * c["D"]
        return dict(bytes=2 * rows * (c["D"] + 4 / c["block"]) + 2 * e * queries,
                    flops=4 * rows * c["G"] * c["Tq"] * c["D"])
    if kind == "cache":
        n = 2 * c["B"] * c["H"] * c["D"]
        kept = 0 if c["context"] == 0 else (c["block"] - 1) / 2
        # rows and kept codes read, codes written; read back as values
        return dict(bytes=n * (c["T"] * (e + 1) + 2 * kept + _write_span(c) * (1 + e)), flops=6 * n * c["T"])
    if kind == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        return dict(bytes=N * K / 2 + e * (-(-K // c["group"]) * N + M * K + N + M * N), flops=2 * M * K * N)
    n = c["R"] * c["V"]
    return dict(bytes=e * n + c["R"] * (16 + 8 * c["top_k"]), flops=6 * n) if kind == "logprobs" else \
        dict(bytes=2 * e * n + 20 * c["R"], flops=8 * n)


# ── the same outputs in 64 bits, from the definitions ───────────────────────
def _f64_logprobs(z, tokens):
    z = z.double()
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    H = torch.special.entr(logp.exp()).sum(1)
    V = z.shape[1]
    t = tokens.long()
    lp = logp[torch.arange(len(t), device=z.device), t.clamp(0, V - 1)]
    return torch.where((t < 0) | (t >= V), torch.zeros_like(lp), lp), H, lse, logp


def _f64_append(codes, scales, rows, pos, start, c):
    """Block by block, row by row as the append is defined: a scale and the
    codes that go by it are float32's, the values they stand for exact."""
    B, H, D, T, block = (c[k] for k in ("B", "H", "D", "T", "block"))
    W = _write_span(c)
    out = torch.empty((B, H, W, D), dtype=torch.float64, device="cuda")
    for b, (p, T0) in enumerate(zip(pos.tolist(), start.tolist())):
        for lo in range(T0, T0 + W, block):
            hi, n = lo + block, lo // block
            a, z = max(lo, p), min(hi, p + T)
            code, s = codes[b, :, lo:hi].double(), scales[b, :, n]
            if a < z:
                x = rows[b, :, a - p:z - p].float()
                most = x.abs().amax((1, 2)) / 127.0
                grown = torch.maximum(s, most) if lo < p else most
                if lo < p:
                    rate = (s / grown)[:, None, None]
                    code[:, :a - lo] = torch.round(code[:, :a - lo].float() * rate).double()
                code[:, a - lo:z - lo] = torch.round(x / grown[:, None, None]).double()
                s = grown
            out[b, :, lo - T0:hi - T0] = code * s.double()[:, None, None]
    return out


def exact(case, seed):
    c, kind = case, case["kind"]
    i = _inputs(c, seed)
    if kind == "attention":
        B, H, G, D, Tq, block = (c[k] for k in ("B", "H", "G", "D", "Tq", "block"))
        out = torch.zeros((B, H, G, Tq, D), dtype=torch.float64, device="cuda")
        for b, n in enumerate(i["lens"].tolist()):
            row = torch.arange(n, device="cuda") // block
            k, v = (i[x][b, :, :n].double() * i[y][b].double()[:, row, None] for x, y in (("kc", "ks"), ("vc", "vs")))
            q = i["q"][b].double().view(H, G * Tq, D)
            scores = (q @ k.transpose(1, 2).contiguous() / math.sqrt(D)).view(H, G, Tq, n)
            last = n - Tq + torch.arange(Tq, device="cuda")
            hidden = torch.arange(n, device="cuda")[None] > last[:, None]
            w = torch.softmax(scores.masked_fill(hidden, float("-inf")), -1).nan_to_num_(0.0)
            out[b] = (w.view(H, G * Tq, n) @ v).view(H, G, Tq, D)
        return out.view(B, H * G, Tq, D)
    if kind == "cache":
        return [_f64_append(i["kc"], i["ks"], i["k"], i["pos"], i["start"], c),
                _f64_append(i["vc"], i["vs"], i["v"], i["pos"], i["start"], c)]
    if kind == "linear":
        K, N = c["K"], c["N"]
        k, n = torch.arange(K, device="cuda"), torch.arange(N, device="cuda")[:, None]
        e = k % 8
        nibble = e // 2 + 4 * (e % 2)
        run, byte = n % 16 + 16 * (k % 128 // 32), k % 32 // 8 * 4 + nibble // 2
        code = (i["packed"][n // 16, k // 128, run, byte].long() >> (nibble % 2 * 4) & 15) - 8
        y = i["x"].double() @ (code.double() * i["scales"].double()[k // c["group"]].t()).t() + i["bias"].double()
        if c["act"] == "relu":
            return torch.relu(y)
        return torch.nn.functional.gelu(y, approximate="tanh") if c["act"] == "gelu" else y
    if kind == "logprobs":
        lp, H, lse, logp = _f64_logprobs(i["z"], i["tokens"])
        if not c["top_k"]:
            return [lp, H, lse]
        ids = torch.sort(i["z"].float(), dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
        return [lp, H, lse, logp.gather(1, ids), None]
    # dz = g_lp (1[j = t] - p) - g_H p (log p + H), with H and the sum as given
    z, t = i["z"].double(), i["tokens"].long()
    logp = z - i["lse"].double()[:, None]
    p = logp.exp()
    there = ((t >= 0) & (t < c["V"])).double()
    g_lp = i["g_lp"].double() * there
    inner = torch.where(p > 0, p * (logp + i["H"].double()[:, None]), torch.zeros_like(p))
    one = torch.nn.functional.one_hot(t.clamp(0, c["V"] - 1), c["V"]).double()
    return g_lp[:, None] * (one - p) - i["g_H"].double()[:, None] * inner
