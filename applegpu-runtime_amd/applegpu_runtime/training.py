"""Training a language model on the `applegpu` torch device: the cross entropy
of a linear layer over a vocabulary, whose logits are never in memory, and the
optimiser with orthogonalised updates.

    load_cpp_backend()
    loss, lse = linear_cross_entropy(hidden, wte.weight, tokens)   # one value a row
    loss.mean().backward()
    Muon(hidden_matrices, lr=0.02).step()

Both run the library's kernels (linear_cross_entropy, its backward and
muon_step of the C ABI); tensors on other devices raise.
"""
from __future__ import annotations

import ctypes

import torch

from ._native import lib, eager_error, ffi_error

_WIRE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 10, torch.int32: 5, torch.int64: 6}


class _Ids:
    """Runtime ids of torch tensors (views of their storages), freed at the end."""

    def __enter__(self):
        self._made = []
        return self

    def __exit__(self, *exc):
        for i in self._made:
            lib.applegpu_eager_free(i)

    def of(self, t: torch.Tensor) -> int:
        if t.device.type not in ("applegpu", "privateuseone"):
            raise ValueError(f"expected a tensor on the applegpu device, got {t.device}")
        if t.dtype not in _WIRE:
            raise ValueError(f"dtype {t.dtype} is not supported here")
        base = lib.applegpu_eager_find_by_data_ptr(ctypes.c_void_p(t.untyped_storage().data_ptr()))
        if not base:
            raise RuntimeError("applegpu tensor whose storage the runtime does not know")
        nd = max(t.dim(), 1)
        shape = (ctypes.c_uint64 * nd)(*([int(s) for s in t.shape] or [1]))
        strides = (ctypes.c_uint64 * nd)(*([int(s) for s in t.stride()] or [1]))
        vid = ctypes.c_uint64(0)
        p = lib.applegpu_eager_view_typed(base, shape, strides, nd, t.storage_offset() * t.element_size(),
                                          _WIRE[t.dtype], ctypes.byref(vid))
        if not p and not vid.value:
            raise RuntimeError(eager_error())
        self._made.append(vid.value)
        return vid.value


def _op(name: bytes, tensors):
    with _Ids() as ids:
        ins = (ctypes.c_uint64 * len(tensors))(*[ids.of(t) for t in tensors])
        out = (ctypes.c_uint64 * 2)()
        if lib.applegpu_eager_op(name, ins, len(tensors), None, 0, None, 0, out, 2) < 0:
            raise ValueError(eager_error())
    return tuple(torch.ops.applegpu.wrap_eager(int(i)) for i in out)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target):
        loss, lse = _op(b"linear_cross_entropy", [x, weight, target])
        ctx.save_for_backward(x, weight, target, loss, lse)
        return loss, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, g_lse):
        x, weight, target, loss, lse = ctx.saved_tensors
        dx, dw = _op(b"linear_cross_entropy_backward", [g_loss, x, weight, target, loss, lse, g_lse])
        return dx, dw, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor):
    """(loss, lse), float32 [...], of the logits x @ weight.T for x [..., K],
    weight [V, K] and int32 or int64 targets [...]; a target outside [0, V)
    (ignore_index -100) has loss 0.  Differentiable in x and weight for up to
    2^20 rows."""
    loss, lse = _LinearCrossEntropy.apply(x, weight, target)
    # (the library's tensors have one dimension at least)
    return (loss, lse) if x.dim() > 1 or target.dim() else (loss.reshape(()), lse.reshape(()))


class Muon(torch.optim.Optimizer):
    """momentum = beta momentum + grad, U = grad + beta momentum (or the
    momentum, without nesterov), weight = (1 - lr weight_decay) weight - lr
    sqrt(max(1, rows / columns)) orthogonalize(U), for matrices; those of one
    shape and type are stepped together."""

    def __init__(self, params, lr=0.02, beta=0.95, weight_decay=0.0, nesterov=True, steps=5, eps=1e-7):
        super().__init__(params, dict(lr=lr, beta=beta, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                                      eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon steps matrices, got a parameter of shape {tuple(p.shape)}")

    def load_state_dict(self, state_dict):
        """As of any optimiser; the momenta stay float32, as they were saved
        (the base class casts state to its parameter's type)."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(ids, [p for group in self.param_groups for p in group["params"]]):
            if "momentum" in saved.get(i, {}):
                self.state[p]["momentum"] = saved[i]["momentum"].to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is not None:
                    alike.setdefault((tuple(p.shape), p.dtype), []).append(p)
            for params in alike.values():
                for p in params:
                    if "momentum" not in self.state[p]:
                        self.state[p]["momentum"] = torch.empty(p.shape, dtype=torch.float32, device=p.device).zero_()
                with _Ids() as ids:
                    arrays = [(ctypes.c_uint64 * len(params))(*[ids.of(t) for t in ts])
                              for ts in (params, [self.state[p]["momentum"] for p in params], [p.grad for p in params])]
                    if lib.applegpu_muon_step(*arrays, len(params), group["lr"], group["beta"], group["weight_decay"],
                                              int(group["nesterov"]), group["steps"], group["eps"]) != 0:
                        raise ValueError(ffi_error())
                # autograd learns of writes from the tensors' versions
                torch.autograd.graph.increment_version([*params, *(self.state[p]["momentum"] for p in params)])
        return loss
