"""The loss and the optimiser on the torch device: 16-bit types, layouts, small
shapes, and a run that goes on from a checkpoint.

Bars.  A logit of K exact products in float32 sums is off by (K / 16 + 16)
2^-24 of their magnitudes, a loss by twice that and its exponentials' 2^-15.
Gradients are off by their own rounding and by that of the logits' gradient,
half a step of the type each, and by p's error, which is the logits'."""
import numpy as np
import pytest

from oracle import few_bits
from oracle import training as O

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
HALF_STEP = {"float32": 2.0 ** -22, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # float32: two planes


@pytest.fixture(scope="module")
def torch_dev(gpu):
    import torch
    from applegpu_runtime.cpp_backend import load_cpp_backend
    load_cpp_backend()
    return torch


def _to(torch, a, dtype):
    return torch.tensor(a, dtype=getattr(torch, dtype)).to("applegpu")


def _case(R, K, V, dtype, seed=0):
    rng = np.random.default_rng(seed + R)
    x = few_bits.round_to(rng.standard_normal((R, K)), dtype)
    w = few_bits.round_to(rng.standard_normal((V, K)) * 0.5, dtype)
    t = rng.integers(0, V, R)
    t[::7] = -100
    return x, w, t


def _check_grads(x, w, t, dtype, g, h, got):
    want = O.linear_cross_entropy_backward(x, w, t, g, h)
    # in the norm: d's and the result's rounding, and p's error
    z = ((x.shape[1] / 16 + 16) * 2.0 ** -24 + 3 * 2.0 ** -22) * (np.abs(x) @ np.abs(w).T).max()
    bar = 3 * HALF_STEP[dtype] + 2 * z + 46 * 2.0 ** -20
    for a, b in zip(got, want):
        a = a.cpu().double().numpy()
        assert a.shape == b.shape
        assert np.linalg.norm(a - b) <= bar * np.linalg.norm(b) + 2.0 ** -25 * np.sqrt(b.size) * (dtype == "float16")


@pytest.mark.parametrize("ints", ["int32", "int64"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_and_gradients(torch_dev, dtype, ints):
    torch = torch_dev
    from applegpu_runtime.training import linear_cross_entropy
    x, w, t = _case(60, 40, 97, dtype)
    xd, wd = (_to(torch, a, dtype).requires_grad_() for a in (x, w))
    loss, lse = linear_cross_entropy(xd, wd, _to(torch, t, ints))
    want = O.linear_cross_entropy(x, w, t)
    for a, b in zip((loss, lse), want):
        assert a.dtype == torch.float32 and tuple(a.shape) == (60,)
        np.testing.assert_allclose(a.detach().cpu().numpy(), b, rtol=1e-4, atol=1e-4)
    g, h = np.full(60, np.float32(1 / 51)), np.full(60, np.float32(1e-3))
    (loss.sum() * (1 / 51) + lse.sum() * 1e-3).backward()
    assert xd.grad.dtype == wd.grad.dtype == getattr(torch, dtype)
    _check_grads(x, w, t, dtype, g, h, (xd.grad, wd.grad))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(torch_dev, dtype):
    """x and the weight as transposed and as cut views, targets with strides:
    the same bits as of the contiguous ones."""
    torch = torch_dev
    from applegpu_runtime.training import linear_cross_entropy
    x, w, t = _case(32, 64, 80, dtype)
    g = np.random.default_rng(1).random(32).astype(np.float32)

    def run(make_x, make_w, make_t):
        bx, bw, ti = make_x(), make_w(), make_t()
        xv, wv = bx[1](bx[0].requires_grad_()), bw[1](bw[0].requires_grad_())
        loss, lse = linear_cross_entropy(xv, wv, ti)
        (loss * torch.tensor(g).to("applegpu")).sum().backward()
        return [loss.detach().cpu(), lse.detach().cpu(), bx[1](bx[0].grad).cpu(), bw[1](bw[0].grad).cpu()]

    def plain(a):
        return lambda: (_to(torch, a, dtype), lambda v: v)

    def turned(a):
        return lambda: (_to(torch, np.ascontiguousarray(a.T), dtype), lambda v: v.t())

    def cut(a):
        wide = np.zeros((a.shape[0], 2 * a.shape[1]), np.float32)
        wide[:, a.shape[1]:] = a
        return lambda: (_to(torch, wide, dtype), lambda v: v[:, a.shape[1]:])

    ti = lambda: _to(torch, t, "int64")
    far = lambda: _to(torch, np.stack([t, t], 1), "int64")[:, 1]
    want = run(plain(x), plain(w), ti)
    for mx, mw, mt in ((turned, plain, ti), (plain, turned, far), (cut, cut, ti)):
        for a, b in zip(run(mx(x), mw(w), mt), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_without_a_row_dimension(torch_dev, dtype):
    """x [K] and a target []: losses and gradients of their shapes."""
    torch = torch_dev
    from applegpu_runtime.training import linear_cross_entropy
    x, w, t = _case(2, 24, 30, dtype)
    xd, wd = (_to(torch, a, dtype).requires_grad_() for a in (x[1], w))
    loss, lse = linear_cross_entropy(xd, wd, torch.tensor(int(t[1])).to("applegpu"))
    assert loss.shape == lse.shape == ()
    want = O.linear_cross_entropy(x[1:], w, t[1:])
    np.testing.assert_allclose([loss.item(), lse.item()], [want[0][0], want[1][0]], rtol=1e-4)
    (loss + lse * 0.5).backward()
    assert xd.grad.shape == (24,)
    _check_grads(x[1:], w, t[1:], dtype, np.ones(1), np.full(1, 0.5), (xd.grad[None], wd.grad))


@pytest.mark.parametrize("lead", [(0,), (0, 3), (2, 0)])
def test_tensors_of_no_rows(torch_dev, lead):
    """Tensors of no elements, with storages of none."""
    torch = torch_dev
    from applegpu_runtime.training import linear_cross_entropy
    w = torch.randn(5, 8).to("applegpu").requires_grad_()
    x = torch.empty(*lead, 8, device="applegpu").requires_grad_()
    loss, lse = linear_cross_entropy(x, w, torch.empty(*lead, dtype=torch.int64, device="applegpu"))
    assert tuple(loss.shape) == tuple(lse.shape) == lead
    loss.sum().backward()
    assert tuple(x.grad.shape) == (*lead, 8) and not w.grad.cpu().any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_of_every_type(torch_dev, dtype):
    """Muon's step on matrices of one block and of many, against the update's
    definition: off by the roundings that the oracle's own planes make, by the
    weights' rounding and float32's."""
    torch = torch_dev
    from applegpu_runtime.training import Muon
    for m, n in ((24, 40), (150, 260), (260, 150)):
        rng = np.random.default_rng(m)
        w = few_bits.round_to(rng.standard_normal((m, n)) * 0.1, dtype)
        p = torch.nn.Parameter(_to(torch, w, dtype))
        opt = Muon([p], lr=0.05, beta=0.9, weight_decay=0.1)
        g = few_bits.round_to(rng.standard_normal((m, n)) * 1e-3, dtype)
        p.grad = _to(torch, g, dtype)
        opt.step()
        one = dtype == "bfloat16" and min(m, n) > 128
        want, mom = O.muon_step(w, 0.0, g, 0.05, 0.9, 0.1)
        near, _ = O.muon_step(w, 0.0, g, 0.05, 0.9, 0.1, halves=1 if one else 2)
        u = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[dtype]
        got = p.detach().cpu().double().numpy()
        sums = 15 * 2.0 ** -22 * np.sqrt(min(m, n)) * 0.05 * np.sqrt(max(1.0, m / n)) * 1.3
        assert (np.abs(got - want) <= u * np.abs(want) + 4 * np.abs(near - want).max() + sums + 2.0 ** -25).all()
        assert opt.state[p]["momentum"].dtype == torch.float32
        np.testing.assert_allclose(opt.state[p]["momentum"].cpu().numpy(), mom, rtol=2.0 ** -22)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_run_goes_on_from_a_checkpoint(torch_dev, dtype, tmp_path):
    """Two steps, a checkpoint, two more steps by a new optimiser: the bits of
    four steps at a stretch."""
    torch = torch_dev
    from applegpu_runtime.training import Muon
    rng = np.random.default_rng(2)
    start = [few_bits.round_to(rng.standard_normal(s) * 0.1, dtype) for s in ((24, 40), (24, 40), (150, 260))]
    grads = [[few_bits.round_to(rng.standard_normal(a.shape) * 1e-3, dtype) for a in start] for _ in range(4)]

    def made(arrays):
        params = [torch.nn.Parameter(_to(torch, a, dtype)) for a in arrays]
        return params, Muon(params, lr=0.05, beta=0.9)

    def steps(params, opt, some):
        for gs in some:
            for p, g in zip(params, gs):
                p.grad = _to(torch, g, dtype)
            opt.step()

    params, opt = made(start)
    steps(params, opt, grads[:2])
    torch.save({"opt": {"state": {i: {"momentum": s["momentum"].cpu()} for i, s in opt.state_dict()["state"].items()},
                        "param_groups": opt.state_dict()["param_groups"]},
                "params": [p.detach().cpu() for p in params]}, tmp_path / "c.pt")
    saved = torch.load(tmp_path / "c.pt", weights_only=True)
    again = [torch.nn.Parameter(p.to("applegpu")) for p in saved["params"]]
    others = [torch.nn.Parameter(p.to("applegpu")) for p in saved["params"]]
    from_file, from_device = Muon(again), Muon(others)
    from_file.load_state_dict(saved["opt"])
    from_device.load_state_dict(opt.state_dict())
    steps(params, opt, grads[2:])
    steps(again, from_file, grads[2:])
    steps(others, from_device, grads[2:])
    for p, a, b in zip(params, again, others):
        assert torch.equal(p.detach().cpu(), a.detach().cpu()) and torch.equal(p.detach().cpu(), b.detach().cpu())
        want = opt.state[p]["momentum"].cpu()
        assert torch.equal(want, from_file.state[a]["momentum"].cpu())
        assert torch.equal(want, from_device.state[b]["momentum"].cpu())


def test_shapes_follow_x(torch_dev):
    """A row with a row dimension keeps it, whatever its target's shape."""
    torch = torch_dev
    from applegpu_runtime.training import linear_cross_entropy
    w = torch.randn(7, 8).to("applegpu")
    one = torch.tensor(3).to("applegpu")
    for x, t, shape in ((torch.randn(1, 8), one, (1,)), (torch.randn(8), one.reshape(1), (1,)), (torch.randn(8), one, ())):
        loss, lse = linear_cross_entropy(x.to("applegpu"), w, t)
        assert tuple(loss.shape) == tuple(lse.shape) == shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_is_left_behind(torch_dev, gpu, dtype):
    """Losses, gradients and steps hand back all that they make, refused calls
    too."""
    torch = torch_dev
    from applegpu_runtime.training import Muon, linear_cross_entropy
    x, w, t = _case(12, 24, 30, dtype)
    xd, ti = _to(torch, x, dtype).requires_grad_(), _to(torch, t, "int64")
    p = torch.nn.Parameter(_to(torch, w, dtype))
    opt = Muon([p], lr=0.01)

    def step():
        opt.zero_grad()
        xd.grad = None
        linear_cross_entropy(xd, p, ti)[0].sum().backward()
        opt.step()
        with pytest.raises(ValueError, match="does not match weight"):
            linear_cross_entropy(xd, p[:, :5], ti)

    for _ in range(3):
        step()
    count = gpu.tensor_count()
    for _ in range(20):
        step()
    assert gpu.tensor_count() == count
