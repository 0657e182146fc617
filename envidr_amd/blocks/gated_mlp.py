"""The gated feed-forward block (envidr_gated_mlp_*, csrc/gated_mlp.hip):  y = (act(x Wg^T) * (x Wu^T)) Wd^T  and its gradients."""
from __future__ import annotations

import functools

import torch

from .. import _lib
from . import _bind
from .dropout import CounterDropout

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}      # gelu: the tanh form


def _rows(t: torch.Tensor) -> torch.Tensor:
    """a matrix whose rows the kernels can walk: adjacent elements, any row pitch that keeps rows apart"""
    pitch, step = t.stride()
    if step == 1 and t.shape[1] <= pitch <= 1 << 21:
        return t
    # contiguous() makes the elements adjacent (reshape alone would not: a matrix whose strides merge, t[:, ::2], is a view as one row too), but
    # leaves a matrix of one row its pitch, whatever that is; the two views put it right
    return t.contiguous().reshape(-1).view(t.shape)


def _sizes(x, wg, wd):
    return x.shape[0], x.shape[1], wg.shape[0], wd.shape[0]


@functools.lru_cache(maxsize=256)
def _workspace_bytes(M, D, F, O, code, backward):
    _bind.sizes("gated_mlp", M=M, D=D, F=F, O=O)
    return max(_bind.lib().envidr_gated_mlp_workspace_bytes(M, D, F, O, code, backward), 16)


def _forward(x, wg, wu, wd, code, act):
    lib = _bind.lib()
    M, D, F, O = _sizes(x, wg, wd)
    n = _workspace_bytes(M, D, F, O, code, 0)
    y = x.new_empty((M, O))
    with _bind.on_device(x) as stream:
        ws = x.new_empty(n, dtype=torch.uint8)
        _bind.check(lib.envidr_gated_mlp_forward(x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0), wd.data_ptr(), wd.stride(0),
                                                 M, D, F, O, code, act, y.data_ptr(), O, ws.data_ptr(), n, stream), "envidr_gated_mlp_forward")
    return y


class _GatedMlp(torch.autograd.Function):
    """Keeps x and the weights: the backward pass forms the hidden layer again."""

    @staticmethod
    def forward(ctx, x, wg, wu, wd, code, act):
        ctx.save_for_backward(x, wg, wu, wd)
        ctx.code, ctx.act = code, act
        return _forward(x, wg, wu, wd, code, act)

    @staticmethod
    @_bind.differentiable_once
    def backward(ctx, dy):
        x, wg, wu, wd = ctx.saved_tensors
        lib = _bind.lib()
        M, D, F, O = _sizes(x, wg, wd)
        dy = _rows(dy)
        n = _workspace_bytes(M, D, F, O, ctx.code, 1)
        grads = [x.new_empty(shape) if want else None for want, shape in zip(ctx.needs_input_grad, ((M, D), (F, D), (F, D), (O, F)))]
        at = [None if g is None else g.data_ptr() for g in grads]
        with _bind.on_device(x) as stream:
            ws = x.new_empty(n, dtype=torch.uint8)
            _bind.check(lib.envidr_gated_mlp_backward(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0),
                                                      wd.data_ptr(), wd.stride(0), M, D, F, O, ctx.code, ctx.act, at[0], D, at[1], at[2], at[3],
                                                      ws.data_ptr(), n, stream), "envidr_gated_mlp_backward")
        return (*grads, None, None)


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """(act(x Wg^T) * (x Wu^T)) Wd^T:  x [..., D], w_gate and w_up [F, D], w_down [O, F] (as nn.Linear keeps them) -> [..., O].

    One dtype (float32, bfloat16 or float16) and one device for all; any strides; activation "silu", "gelu" (tanh form), "relu" or
    "sigmoid".  Differentiable once, w.r.t. every tensor.  Products accumulate in 32 bits; in the 16-bit dtypes the hidden layer is rounded
    to the dtype once, between the products (forward of up to 32 rows: not at all).  float32 carries 24-bit operands through the bf16 matrix cores
    (beyond 64 rows: an infinity in them gives NaN, and of numbers below 2^-108 what is above 2^-126 counts).  torch.autocast casts nothing here: inside
    such a region the caller gives x and the weights one dtype.  A forward-mode tangent is refused."""
    code = _bind.same_kind("gated_mlp", x, w_gate=w_gate, w_up=w_up, w_down=w_down)
    if activation not in ACTIVATIONS:
        raise _lib.EnvidrError(f"gated_mlp: activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.dim() != 2 or w_down.shape[1] != w_gate.shape[0] or x.shape[-1] != w_gate.shape[1]:
        raise _lib.EnvidrError(f"gated_mlp: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}, w_down {tuple(w_down.shape)}: "
                               "x [..., D], w_gate and w_up [F, D], w_down [O, F] are wanted")
    if 0 in w_gate.shape or 0 in w_down.shape:
        raise _lib.EnvidrError("gated_mlp: a width is zero")
    rows = _rows(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    if _bind.differentiated(x, w_gate, w_up, w_down):
        y = _GatedMlp.apply(rows, _rows(w_gate), _rows(w_up), _rows(w_down), code, ACTIVATIONS[activation])
    else:
        y = _forward(rows, _rows(w_gate), _rows(w_up), _rows(w_down), code, ACTIVATIONS[activation])
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[-1])


class GatedMLP(torch.nn.Module):
    """A gated feed-forward block of width d_in -> d_hidden -> d_out (d_in when not given), without biases.  residual: adds x to the result; p: dropout
    on the result in training, its masks from `seed` (`CounterDropout`'s)."""

    def __init__(self, d_in: int, d_hidden: int, d_out: int | None = None, activation: str = "silu", residual: bool = False, p: float = 0.0, seed: int | None = None):
        super().__init__()
        d_out = d_in if d_out is None else d_out
        if residual and d_out != d_in:
            raise _lib.EnvidrError(f"GatedMLP: a residual needs d_out = d_in, not {d_out} and {d_in}")
        if activation not in ACTIVATIONS:
            raise _lib.EnvidrError(f"GatedMLP: activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
        self.activation, self.residual = activation, residual
        self.w_gate = torch.nn.Parameter(torch.empty(d_hidden, d_in))
        self.w_up = torch.nn.Parameter(torch.empty(d_hidden, d_in))
        self.w_down = torch.nn.Parameter(torch.empty(d_out, d_hidden))
        for w in (self.w_gate, self.w_up, self.w_down):
            torch.nn.init.xavier_uniform_(w)
        self.drop = CounterDropout(p, seed)

    def forward(self, x: torch.Tensor, rng: torch.Tensor | None = None) -> torch.Tensor:
        """rng: the dropout's call (`self.drop.draw()`), for a pass that is run twice"""
        y = gated_mlp(x, self.w_gate, self.w_up, self.w_down, self.activation)
        return self.drop(y, residual=x if self.residual else None, rng=rng)
