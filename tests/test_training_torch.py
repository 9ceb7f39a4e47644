"""The optimiser's state on its way through a checkpoint (no GPU: its steps
are tested on the device)."""
import copy
import io

import pytest
import torch

from applegpu_runtime.training import Muon

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _stepped(dtype):
    """An optimiser with momenta as its steps leave them: float32, with bits
    that no 16-bit type holds."""
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(4, 6).to(dtype)) for _ in range(3)]
    opt = Muon([{"params": params[:2]}, {"params": params[2:], "lr": 0.5}], lr=0.1)
    for p in params[1:]:   # (the first has had no gradient yet)
        opt.state[p]["momentum"] = torch.randn(4, 6)
    return params, opt


def _same(opt, params, want, others):
    assert [g["lr"] for g in opt.param_groups] == [0.1, 0.5]
    assert "momentum" not in opt.state.get(params[0], {})
    for p, q in zip(params[1:], others[1:]):
        m = opt.state[p]["momentum"]
        assert m.dtype == torch.float32 and m.device == p.device
        assert torch.equal(m, want.state[q]["momentum"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_state_keeps_float32_momenta(dtype):
    others, opt = _stepped(dtype)
    params = [torch.nn.Parameter(torch.zeros(4, 6, dtype=dtype)) for _ in range(3)]
    new = Muon([{"params": params[:2]}, {"params": params[2:]}])
    new.load_state_dict(opt.state_dict())
    _same(new, params, opt, others)
    # the loaded momenta are the optimiser's own
    new.state[params[1]]["momentum"].zero_()
    assert opt.state[others[1]]["momentum"].abs().sum() > 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_state_through_a_file_and_again(dtype):
    others, opt = _stepped(dtype)
    f = io.BytesIO()
    torch.save(opt.state_dict(), f)
    f.seek(0)
    saved = torch.load(f, weights_only=True)
    params = [torch.nn.Parameter(torch.zeros(4, 6, dtype=dtype)) for _ in range(3)]
    new = Muon([{"params": params[:2]}, {"params": params[2:]}])
    kept = copy.deepcopy(saved)
    new.load_state_dict(saved)
    _same(new, params, opt, others)
    for i in kept["state"]:   # what was loaded stays as it was
        assert torch.equal(saved["state"][i]["momentum"], kept["state"][i]["momentum"])
    third = Muon([{"params": params[:2]}, {"params": params[2:]}])
    third.load_state_dict(new.state_dict())
    _same(third, params, opt, others)


def test_loading_refuses_what_does_not_fit():
    _, opt = _stepped(torch.bfloat16)
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4, 6))]).load_state_dict(opt.state_dict())
