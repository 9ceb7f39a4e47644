"""The operators in few bits as they are used: GPT-2 generation with 4-bit
weights, an 8-bit cache and the log probabilities of its picks, and the
scoring of texts, against a float64 forward of the same quantised weights and
cache.

Bars.  The model runs in float16: a layer rounds about 10 values after one
another (norms, projections, attention, residuals), each to half a step
2^-11 of values of the residual's size, so L layers leave about
10 L 2^-11 of the logits' size; twice that is asked for."""
import numpy as np
import pytest

from oracle import few_bits as O

pytestmark = pytest.mark.gpu

CFG = dict(n_layer=2, n_head=2, n_embd=128, vocab_size=211, n_positions=96)
GROUP = 32
BAR = 2 * 10 * CFG["n_layer"] * 2.0 ** -11


def _f16(a):
    return np.asarray(a, np.float32).astype(np.float16).astype(np.float64)


@pytest.fixture(scope="module")
def weights():
    from applegpu_runtime.models import gpt2 as G
    rng = np.random.default_rng(11)
    w = G.random_weights(CFG, seed=5, std=0.15)
    for k in w:
        if k.endswith(".bias"):
            w[k] = (rng.standard_normal(w[k].shape) * 0.1).astype(np.float32)
    return w


def _values(weights, bits):
    """The weights that the device's model stands for, float64."""
    out = {}
    for k, v in weights.items():
        h = _f16(v)
        if bits == 4 and k.endswith((".c_attn.weight", ".c_proj.weight", ".c_fc.weight")):
            c, s = O.quantize_int4(h.T.astype(np.float32), GROUP, "float16")
            h = O.values_int4(c, s, GROUP).T
        out[k] = h
    return out


def _norm(x, w, p):
    m = x.mean(-1, keepdims=True)
    return (x - m) / np.sqrt(((x - m) ** 2).mean(-1, keepdims=True) + 1e-5) * w[p + ".weight"] + w[p + ".bias"]


class Reference:
    """Float64 GPT-2 of one sequence with a cache in `bits` bits."""

    def __init__(self, w, bits, max_len, block=16):
        H, d, L = CFG["n_head"], CFG["n_embd"], CFG["n_layer"]
        self.w, self.bits, self.block = w, bits, block
        self.codes = np.zeros((2, L, 1, H, max_len, d // H), np.int8)
        self.scales = np.zeros((2, L, 1, H, -(-max_len // block)), np.float32)
        self.rows = np.zeros((2, L, 1, H, max_len, d // H))
        self.n = 0

    def logits(self, ids):
        """Of the last len(ids) positions; a prompt attends to its own rows
        before they are rounded, a later token to the cache."""
        w, H, d = self.w, CFG["n_head"], CFG["n_embd"]
        T = len(ids)
        x = w["transformer.wte.weight"][ids] + w["transformer.wpe.weight"][self.n:self.n + T]
        for i in range(CFG["n_layer"]):
            p = f"transformer.h.{i}"
            qkv = _norm(x, w, p + ".ln_1") @ w[p + ".attn.c_attn.weight"] + w[p + ".attn.c_attn.bias"]
            q, k, v = (t.reshape(T, H, d // H).transpose(1, 0, 2)[None] for t in np.split(qkv, 3, -1))
            for j, t in enumerate((k, v)):
                self.rows[j, i, :, :, self.n:self.n + T] = t
                if self.bits == 8:
                    O.append_int8(self.codes[j, i], self.scales[j, i], _f16(t).astype(np.float32), [self.n], self.block)
            if self.bits == 8 and self.n:
                kk, vv = (O.values_int8(self.codes[j, i], self.scales[j, i], self.block) for j in (0, 1))
            else:
                kk, vv = self.rows[0, i], self.rows[1, i]
            a = O.decode_attention(q, kk, vv, [self.n + T])[0].transpose(1, 0, 2).reshape(T, d)
            x = x + a @ w[p + ".attn.c_proj.weight"] + w[p + ".attn.c_proj.bias"]
            f = O.linear(_norm(x, w, p + ".ln_2"), w[p + ".mlp.c_fc.weight"].T, w[p + ".mlp.c_fc.bias"], "gelu")
            x = x + f @ w[p + ".mlp.c_proj.weight"] + w[p + ".mlp.c_proj.bias"]
        self.n += T
        return _norm(x, w, "transformer.ln_f") @ w["transformer.wte.weight"].T


@pytest.mark.parametrize("weight_bits,cache_bits,T", [(16, 8, 7), (4, 16, 33), (4, 8, 1), (4, 8, 19)])
@pytest.mark.parametrize("capture", [True, False])
def test_generation(gpu, weights, weight_bits, cache_bits, T, capture):
    """Prompts, then tokens one at a time, teacher-forced into the reference;
    what is said about each pick is of the logits that it was picked from."""
    from applegpu_runtime.models import gpt2 as G
    B, steps, k = 2, 40, 3
    prompt = np.random.default_rng(T).integers(0, CFG["vocab_size"], (B, T))
    model = G.load_model(weights, CFG, "float16", weight_bits=weight_bits, group=GROUP)
    gen = G.Generation(model, prompt, steps, capture=capture, cache_bits=cache_bits, logprobs=k)
    toks, logits = gen.run(keep_logits=True)
    lp, H, tl, ti = gen.pick_logprobs()
    assert toks.shape == lp.shape == H.shape == (B, steps + 1) and tl.shape == ti.shape == (B, steps + 1, k)
    w = _values(weights, weight_bits)
    for b in range(B):
        ref = Reference(w, cache_bits, T + steps)
        want = [ref.logits(prompt[b])[-1]] + [ref.logits([t])[-1] for t in toks[b, :-1]]
        size = np.abs(want).max()
        for s in range(steps + 1):
            z = logits[s, b].astype(np.float64)
            assert np.abs(z - want[s]).max() <= BAR * size, (b, s, np.abs(z - want[s]).max() / size)
            one = O.token_logprobs(z[None], toks[b, s:s + 1], k)
            assert toks[b, s] == z.argmax() == ti[b, s, 0]
            np.testing.assert_array_equal(ti[b, s], one[4][0])
            np.testing.assert_allclose(lp[b, s], one[0][0], atol=1e-5)
            np.testing.assert_allclose(H[b, s], one[1][0], atol=1e-5)
            np.testing.assert_allclose(tl[b, s], one[3][0], atol=1e-5)
    again, _ = gen.run(keep_logits=True)      # a cache that is full of an earlier run
    np.testing.assert_array_equal(again, toks)
    gen.destroy()


def test_capture_and_eager_agree(gpu, weights):
    from applegpu_runtime.models import gpt2 as G
    model = G.load_model(weights, CFG, "bfloat16", weight_bits=4, group=GROUP)
    prompt = np.random.default_rng(0).integers(0, CFG["vocab_size"], (3, 21))
    got = []
    for capture in (True, False):
        cache = G.KVCache(CFG, 3, 60, "bfloat16", bits=8, block=32)
        assert cache.nbytes() < 0.6 * G.KVCache(CFG, 3, 60, "bfloat16").nbytes()
        got.append(G.generate_greedy(model, prompt, 30, cache=cache, capture=capture, keep_logits=True))
    np.testing.assert_array_equal(got[0][0], got[1][0])
    np.testing.assert_array_equal(got[0][1], got[1][1])


@pytest.mark.parametrize("weight_bits", [16, 4])
def test_score(gpu, weights, weight_bits):
    """Log probabilities of whole texts, one of them padded, against the
    reference's, and against those of the padded text alone."""
    from applegpu_runtime.models import gpt2 as G
    model = G.load_model(weights, CFG, "float16", weight_bits=weight_bits, group=GROUP)
    ids = np.random.default_rng(3).integers(0, CFG["vocab_size"], (3, 50))
    ids[1, 20:] = -1
    lp, H, lse, tl, ti = (t.to_numpy() for t in G.gpt2_score(model, ids, top_k=4))
    assert lp.shape == (3, 50) and ti.shape == (3, 50, 4)
    w = _values(weights, weight_bits)
    for b, n in enumerate((50, 20, 50)):
        z = Reference(w, 16, 50).logits(ids[b, :n])
        want = O.token_logprobs(z, np.r_[ids[b, 1:n], -1], 4)
        bar = 2 * BAR * np.abs(z).max()    # of a difference of two logits
        assert np.abs(lp[b, :n] - want[0]).max() <= bar
        assert np.abs(H[b, :n] - want[1]).max() <= bar * np.log(CFG["vocab_size"])
        assert np.abs(tl[b, :n] - want[3]).max() <= bar
        assert (lp[b, n - 1:] == 0).all()
    alone = G.gpt2_score(model, ids[1:2, :20], top_k=4)
    assert np.abs(alone[0].to_numpy() - lp[1:2, :20]).max() <= 2 * BAR * np.abs(z).max()


def test_refusals(gpu, weights):
    from applegpu_runtime.models import gpt2 as G
    for bad in [dict(weight_bits=3), dict(dtype="float32", weight_bits=4), dict(weight_bits=4, kmajor=False),
                dict(weight_bits=4, group=48)]:
        with pytest.raises(ValueError):
            G.load_model(weights, CFG, **dict(dict(dtype="float16"), **bad))
    with pytest.raises(ValueError):
        G.KVCache(CFG, 1, 20, bits=4)
    model = G.load_model(weights, CFG, "float16")
    with pytest.raises(ValueError):
        G.gpt2_score(model, [1, 2, 3])
    with pytest.raises(ValueError):
        G.gpt2_score(model, np.zeros((1, 97), int))
    gen = G.Generation(model, [[1, 2]], 1, capture=False)
    with pytest.raises(ValueError):
        gen.pick_logprobs()
