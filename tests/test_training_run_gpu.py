"""The training operators as they are used together: a small language model
(table, hidden matrix, tied head) trained by its cross entropy and orthogonalised
updates, against the same in float64; captured and replayed; in GPT-2's loss,
the MLP's step and on the torch device.

Bars.  A float32 run rounds a handful of float32 values a step (products of 22
bits or more) and its updates are Lipschitz in them with a constant of a few
hundred at most (five steps multiply a small singular value by up to 3.4 each):
2^-22 x 500 = 1.2e-4 a step of the update's size."""
import numpy as np
import pytest

from oracle import training as O

pytestmark = pytest.mark.gpu

V, D, T = 97, 40, 60


def _model(seed):
    rng = np.random.default_rng(seed)
    table = (rng.standard_normal((V, D)) * 0.3).astype(np.float32)
    hidden = (rng.standard_normal((D, D)) / np.sqrt(D)).astype(np.float32)
    ids = rng.integers(0, V, T + 1).astype(np.int32)
    target = ids[1:].copy()
    target[5] = -100
    return table, hidden, ids[:-1], target


def _device_step(gpu, table, hidden, mom, ids, target, lr=0.05):
    """e = table[ids]; x = e hidden^T; loss of x against the tied table."""
    e = gpu.embedding(table, ids)
    x = gpu.matmul(e, gpu.transpose(hidden))
    loss, lse = gpu.linear_cross_entropy(x, table, target)
    g = gpu.full([T], 1.0 / T, "float32")
    dx, dtable = gpu.linear_cross_entropy_backward(g, x, table, target, loss, lse)
    dhidden = gpu.matmul(gpu.transpose(dx), e)
    de = gpu.matmul(dx, hidden)
    dtable = dtable + gpu.embedding_backward(de, ids, V)
    gpu.eval_many([loss, dhidden, dtable])
    gpu.muon_step_(hidden, mom[0], dhidden, lr=lr, beta=0.9)
    gpu.muon_step_(table, mom[1], dtable, lr=lr, beta=0.9)
    return loss


def _oracle_step(table, hidden, mom, ids, target, lr=0.05):
    e = table[ids]
    x = e @ hidden.T
    loss, _ = O.linear_cross_entropy(x, table, target)
    dx, dtable = O.linear_cross_entropy_backward(x, table, target, np.full(T, np.float32(1.0 / T)))
    dhidden, de = dx.T @ e, dx @ hidden
    np.add.at(dtable, ids, de)
    hidden, mom[0] = O.muon_step(hidden, mom[0], dhidden, lr, 0.9, 0.0)
    table, mom[1] = O.muon_step(table, mom[1], dtable, lr, 0.9, 0.0)
    return loss, table, hidden


def test_steps_of_a_tied_model(gpu):
    table, hidden, ids, target = _model(0)
    dev = [gpu.from_numpy(a) for a in (table, hidden)]
    mom = [gpu.from_numpy(np.zeros_like(a)) for a in (hidden, table)]
    di, dt = gpu.from_numpy(ids), gpu.from_numpy(target)
    t, h, om = table.astype(np.float64), hidden.astype(np.float64), [0.0, 0.0]
    for step in range(3):
        loss = _device_step(gpu, *dev, mom, di, dt)
        want, t, h = _oracle_step(t, h, om, ids, target)
        bar = 1.2e-4 * (step + 1)
        np.testing.assert_allclose(loss.to_numpy(), want, rtol=bar, atol=bar)
        for a, b in zip(dev, (t, h)):
            assert np.abs(a.to_numpy() - b).max() <= 4 * bar * 0.05 * np.sqrt(V / D) + 1e-6


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_captured_step_replays(gpu, dtype):
    """The whole step as a graph, replayed with other work between, against
    eager steps of a second model; two graphs at once keep to their own
    workspaces."""
    table, hidden, ids, target = _model(1)

    def build():
        cast = lambda a: gpu.from_numpy(a) if dtype == "float32" else gpu.cast(gpu.from_numpy(a), dtype)
        dev = [cast(a) for a in (table, hidden)]
        for a in dev:
            a.eval()
        return dev, [gpu.from_numpy(np.zeros_like(a)) for a in (hidden, table)], gpu.from_numpy(ids), gpu.from_numpy(target)

    def step(s):
        (tb, hd), mom, i, t = s
        x = gpu.matmul(gpu.embedding(tb, i), gpu.transpose(hd))
        loss, lse = gpu.linear_cross_entropy(x, tb, t)
        dx, dt = gpu.linear_cross_entropy_backward(gpu.full([T], 1.0 / T, "float32"), x, tb, t, loss, lse)
        gpu.eval_many([loss, dx, dt])
        gpu.muon_step_(tb, mom[1], dt, lr=0.05)
        return [loss, dx, gpu.orthogonalize(dx)]

    states = [build() for _ in range(3)]
    graphs = [gpu.capture(lambda s=s: step(s)) for s in states[:2]]
    for rep in range(4):
        for g in graphs:
            g.replay()
        junk = gpu.linear_cross_entropy(gpu.zeros([300, 64]), gpu.zeros([500, 64]),
                                        gpu.from_numpy(np.zeros(300, np.int32)))[0].to_numpy()
        np.testing.assert_allclose(junk, np.log(500), rtol=1e-5)
        want = [a.to_numpy() for a in step(states[2])]
        for g, s in zip(graphs, states):
            for a, b in zip(g.outputs, want):
                np.testing.assert_array_equal(a.to_numpy(), b, err_msg=f"replay {rep}")
            np.testing.assert_array_equal(s[0][0].to_numpy(), states[2][0][0].to_numpy())
    for g in graphs:
        g.destroy()


CFG = dict(n_layer=2, n_head=2, n_embd=128, vocab_size=211, n_positions=96)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_gpt2_loss(gpu, dtype):
    """The loss without logits is the score's log probabilities, and its
    gradient what the logits' gradient gives."""
    from applegpu_runtime.models import gpt2 as G
    model = G.load_model(G.random_weights(CFG, seed=5, std=0.15), CFG, dtype)
    rng = np.random.default_rng(0)
    ids = rng.integers(0, CFG["vocab_size"], (3, 30)).astype(np.int32)
    ids[1, 20:] = -1
    loss = G.gpt2_loss(model, ids).to_numpy()
    lp, _, _ = (a.to_numpy() for a in G.gpt2_score(model, ids))
    # the score's logits are rounded to the model's type, and where float32
    # takes its products from bf16 halves, to 2^-16 of their terms
    bar = 2.0 ** -9 if dtype == "float16" else 2.0 ** -13
    np.testing.assert_allclose(loss, -lp, atol=bar * 16, rtol=bar)
    assert (loss[:, -1] == 0).all() and (loss[1, 19:] == 0).all() and (loss[0, :-1] > 0).all()
    l2, dx, dw = G.gpt2_loss(model, ids, grads=True)
    np.testing.assert_array_equal(l2.to_numpy(), loss)
    assert dx.shape == [3, 30, 128] and dw.shape == [211, 128]
    x, nxt = G._text_hidden(model, ids)
    w = model["weights"]
    x = gpu.layer_norm(x, w["transformer.ln_f.weight"], w["transformer.ln_f.bias"])
    n = int((nxt >= 0).sum())
    want = O.linear_cross_entropy_backward(x.to_numpy(), w["transformer.wte.weight"].to_numpy(), nxt.reshape(-1),
                                           np.full(90, 1.0 / n))
    for a, b in zip((dx.to_numpy().reshape(90, 128), dw.to_numpy()), want):
        assert np.linalg.norm(a - b) <= (1e-5 if dtype == "float32" else 2.0 ** -9) * np.linalg.norm(b)
    with pytest.raises(ValueError, match="ids must be"):
        G.gpt2_loss(model, [1, 2])


def test_mlp_with_orthogonalised_updates(gpu):
    from applegpu_runtime import eager as E
    from applegpu_runtime.models.mlp import EagerMLP
    rng = np.random.default_rng(3)
    sizes = [12, 20, 20, 20, 3]
    params = [((rng.standard_normal((o, i)) * 0.4).astype(np.float32), rng.standard_normal(o).astype(np.float32) * 0.1)
              for i, o in zip(sizes, sizes[1:])]
    x, y = rng.standard_normal((16, 12)).astype(np.float32), rng.standard_normal((16, 3)).astype(np.float32)
    mlp = EagerMLP(params, optimizer="muon", muon_lr=0.03, muon_beta=0.9)
    ps = [(w.astype(np.float64), b.astype(np.float64)) for w, b in params]
    moms = [np.zeros_like(w) for w, _ in ps]
    for step in range(2):
        loss = mlp.train_step(E.from_numpy(x), E.from_numpy(y), lr=0.05).numpy()
        acts = [x.astype(np.float64)]
        for i, (w, b) in enumerate(ps):
            z = acts[-1] @ w.T + b
            acts.append(np.maximum(z, 0) if i < len(ps) - 1 else z)
        diff = acts[-1] - y
        assert abs(float(loss[0]) - (diff ** 2).mean()) <= 1e-3 * (diff ** 2).mean()
        g = 2 * diff / diff.size
        new = []
        for i in range(len(ps) - 1, -1, -1):
            w, b = ps[i]
            dw, db = g.T @ acts[i], g.sum(0)
            g = (g @ w) * (acts[i] > 0)
            if i < len(ps) - 1:
                w2, moms[i] = O.muon_step(w, moms[i], dw, 0.03, 0.9, 0.0)
            else:
                w2 = w - 0.05 * dw
            new.append((w2, b - 0.05 * db))
        ps = new[::-1]
    for (w, b), (rw, rb) in zip(mlp.numpy_params(), ps):
        # gradients come from products of bf16 halves (2^-16), and a small
        # direction's share of them is multiplied by up to 500
        assert np.abs(w - rw).max() <= 0.03 * 500 * 2.0 ** -16 * 2 and np.abs(b - rb).max() <= 1e-4
    with pytest.raises(ValueError, match="optimizer"):
        EagerMLP(params, optimizer="adam")


@pytest.fixture(scope="module")
def torch_dev(gpu):
    import torch
    from applegpu_runtime.cpp_backend import load_cpp_backend
    load_cpp_backend()
    return torch


def test_torch_device(torch_dev):
    """Loss, gradients and the optimiser's step on the torch device against
    torch on the CPU."""
    torch = torch_dev
    from applegpu_runtime.training import Muon, linear_cross_entropy
    torch.manual_seed(0)
    x, w = torch.randn(4, 15, 32), torch.randn(70, 32) * 0.5
    t = torch.randint(0, 70, (4, 15))
    t[0, 3] = -100
    xc, wc = x.clone().double().requires_grad_(), w.clone().double().requires_grad_()
    z = xc @ wc.t()
    want = torch.nn.functional.cross_entropy(z.reshape(-1, 70), t.reshape(-1), reduction="none").reshape(4, 15)
    (want.sum() / 59 + 1e-3 * torch.logsumexp(z, -1).sum()).backward()
    xd, wd = (a.to("applegpu").requires_grad_() for a in (x, w))
    loss, lse = linear_cross_entropy(xd, wd, t.to("applegpu"))
    np.testing.assert_allclose(loss.detach().cpu().numpy(), want.detach().numpy(), rtol=1e-5, atol=1e-5)
    (loss.sum() * (1.0 / 59) + lse.sum() * 1e-3).backward()
    for a, b in ((xd.grad, xc.grad), (wd.grad, wc.grad)):
        assert torch.linalg.vector_norm(a.cpu().double() - b) <= 1e-5 * torch.linalg.vector_norm(b)
    params = [torch.nn.Parameter((torch.randn(24, 32) * 0.1).to("applegpu")) for _ in range(2)]
    other = torch.nn.Parameter((torch.randn(32, 24) * 0.1).to("applegpu"))
    start = [p.detach().cpu().double().numpy() for p in (*params, other)]
    opt = Muon([*params, other], lr=0.05, beta=0.9, weight_decay=0.1)
    moms = [0.0] * 3
    for _ in range(2):
        for i, p in enumerate((*params, other)):
            p.grad = (torch.randn(*p.shape) * 1e-3).to("applegpu")
            g = p.grad.cpu().double().numpy()
            start[i], moms[i] = O.muon_step(start[i], moms[i], g, 0.05, 0.9, 0.1)
        opt.step()
    for p, b in zip((*params, other), start):
        np.testing.assert_allclose(p.detach().cpu().numpy(), b, atol=1e-4 * 0.05 * 2)
    with pytest.raises(ValueError, match="matrices"):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="applegpu device"):
        linear_cross_entropy(x, w, t)


def test_torch_step_is_seen_by_autograd(torch_dev):
    """A product whose saved weights the optimiser has stepped since refuses its
    backward pass, as behind any other write in place."""
    torch = torch_dev
    from applegpu_runtime.training import Muon
    w = torch.nn.Parameter((torch.randn(8, 8) * 0.1).to("applegpu"))
    x = torch.randn(4, 8).to("applegpu").requires_grad_()
    y = (x @ w).sum()
    w.grad = torch.randn(8, 8).to("applegpu")
    before = w._version
    Muon([w]).step()
    assert w._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_torch_without_rows(torch_dev):
    """No rows: no losses, and gradients of zeros."""
    torch = torch_dev
    from applegpu_runtime.training import linear_cross_entropy
    w = torch.randn(5, 8).to("applegpu").requires_grad_()
    x = torch.randn(2, 8).to("applegpu")[:0].requires_grad_()
    loss, lse = linear_cross_entropy(x, w, torch.zeros(2, dtype=torch.int64).to("applegpu")[:0])
    assert loss.shape == lse.shape == (0,)
    loss.sum().backward()
    assert x.grad.shape == (0, 8) and not w.grad.cpu().any()
