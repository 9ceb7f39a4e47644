"""The loss, its gradient and the updates in captured graphs, at sizes whose
launches share a workspace: every replay against the same calls made eagerly,
bit for bit, with new inputs and other work between the replays."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


def _dev(gpu, a, dtype="float32"):
    t = gpu.from_numpy(np.ascontiguousarray(a, np.float32))
    return t if dtype == "float32" else gpu.cast(t, dtype)


def _junk(gpu):
    """Work that takes workspaces of its own and fills them."""
    rng = np.random.default_rng(1)
    a = gpu.orthogonalize(_dev(gpu, rng.standard_normal((2, 300, 500))))
    b, _ = gpu.linear_cross_entropy(_dev(gpu, rng.standard_normal((200, 64))), _dev(gpu, rng.standard_normal((900, 64))),
                                    gpu.from_numpy(rng.integers(0, 900, 200).astype(np.int32)))
    return float(np.abs(a.to_numpy()).max()) + float(b.to_numpy().sum())


# in one block; a chain of launches; symmetric products cut and joined
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,m,k", [(2, 40, 60), (3, 200, 300), (2, 300, 200), (2, 1500, 260), (1, 64, 4096)])
def test_steps_replay(gpu, n, m, k, dtype):
    rng = np.random.default_rng(m)
    w = rng.standard_normal((n, m, k)) * 0.02

    def build():
        made = [[_dev(gpu, a, dtype) for a in w], [_dev(gpu, np.zeros((m, k))) for _ in w],
                [_dev(gpu, np.zeros((m, k)), dtype) for _ in w]]
        for t in sum(made, []):
            t.eval()
        return made

    def step(s):
        gpu.muon_step_(*s, lr=0.05, weight_decay=0.1)
        return [gpu.orthogonalize(s[0][0], steps=2)]

    states = [build() for _ in range(3)]
    graphs = [gpu.capture(lambda s=s: step(s)) for s in states[:2]]
    for rep in range(4):
        for i in range(n):
            g = _dev(gpu, rng.standard_normal((m, k)) * 1e-3, dtype)
            for s in states:
                gpu.blit_copy(g, s[2][i])
        for g in graphs:
            g.replay()
        assert np.isfinite(_junk(gpu))
        want = step(states[2])[0].to_numpy()
        for g, s in zip(graphs, states):
            np.testing.assert_array_equal(g.outputs[0].to_numpy(), want, err_msg=f"replay {rep}")
            for a, b in zip(s[0] + s[1], states[2][0] + states[2][1]):
                np.testing.assert_array_equal(a.to_numpy(), b.to_numpy(), err_msg=f"replay {rep}")
    for g in graphs:
        g.destroy()


# few rows; parts of dx and of dw; the vocabulary in pieces
@pytest.mark.parametrize("R,K,V,dtype", [(5, 72, 300, "float16"), (300, 64, 2000, "float32"), (300, 64, 2000, "bfloat16"),
                                         (5000, 70, 30, "float32"), (5000, 70, 30, "bfloat16"),
                                         (33000, 16, 17000, "bfloat16"), (17000, 16, 17000, "float32")])
def test_loss_and_gradient_replay(gpu, R, K, V, dtype):
    """float32 rows change from replay to replay between those that share a
    power of two and those too far apart for one."""
    rng = np.random.default_rng(R)
    ins = [_dev(gpu, np.zeros((R, K)), dtype), _dev(gpu, rng.standard_normal((V, K)), dtype),
           gpu.from_numpy(np.zeros(R, np.int32)), gpu.from_numpy(np.full(R, 1 / R, np.float32))]
    for t in ins:
        t.eval()

    def run():
        x, w, t, g = ins
        loss, lse = gpu.linear_cross_entropy(x, w, t)
        return [loss, lse, *gpu.linear_cross_entropy_backward(g, x, w, t, loss, lse)]

    graphs = [gpu.capture(run) for _ in range(2)]
    for rep in range(4):
        x = rng.standard_normal((R, K))
        if rep % 2:
            x[R // 2] *= 2.0 ** 30 if dtype == "float32" else 1.0
        gpu.blit_copy(_dev(gpu, x, dtype), ins[0])
        t = rng.integers(-1, V, R).astype(np.int32)
        t[R // 2] = -100
        ins[2].write(t)
        for g in graphs:
            g.replay()
        assert np.isfinite(_junk(gpu))
        want = [a.to_numpy() for a in run()]
        assert all(np.isfinite(a).all() for a in want)
        for g in graphs:
            for a, b in zip(g.outputs, want):
                np.testing.assert_array_equal(a.to_numpy(), b, err_msg=f"replay {rep}")
    for g in graphs:
        g.destroy()


@pytest.mark.parametrize("shape", [(16, 24), (150, 200)])
def test_what_was_asked_before_a_capture(gpu, shape):
    """A result recorded before a capture whose step writes what it reads would
    only be there after a replay: the step is refused until it is evaluated.
    What is recorded within the capture sees the weights before its step."""
    rng = np.random.default_rng(4)
    w, m, g = (rng.standard_normal(shape).astype(np.float32) for _ in range(3))
    dw, dm, dg = (_dev(gpu, a) for a in (w, m, g))
    other = _dev(gpu, w) + _dev(gpu, w)          # reads nothing that is written
    for i, asked in enumerate((lambda: gpu.transpose(dw) + gpu.transpose(dw), lambda: gpu.relu(dm * dm))):
        y = asked()
        with pytest.raises(ValueError, match="before the graph capture"):
            gpu.capture(lambda: gpu.muon_step_(dw, dm, dg, lr=0.5))
        np.testing.assert_array_equal(y.to_numpy(), 2 * w.T if i == 0 else np.maximum(m * m, 0))
    np.testing.assert_array_equal(dw.to_numpy(), w)

    def step():
        y = dw + dw
        gpu.muon_step_(dw, dm, dg, lr=0.5)
        return [y, dw + dw]

    graph = gpu.capture(step)
    np.testing.assert_array_equal(other.to_numpy(), 2 * w)
    before = w
    for _ in range(3):
        graph.replay()
        np.testing.assert_array_equal(graph.outputs[0].to_numpy(), 2 * before)
        before = dw.to_numpy()
        np.testing.assert_array_equal(graph.outputs[1].to_numpy(), 2 * before)
    graph.destroy()
