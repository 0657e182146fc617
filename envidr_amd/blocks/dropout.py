"""Counter-based dropout (envidr_dropout, csrc/dropout.hip): the mask is a function of the generator's two numbers and the element's index, so it
is never stored; the backward pass computes it again."""
from __future__ import annotations

import torch

from .. import _lib
from . import _bind


def _launch(x, residual, rng, p, code):
    y = torch.empty_like(x)
    lib = _bind.lib()
    with _bind.on_device(x) as stream:
        _bind.check(lib.envidr_dropout(x.data_ptr(), None if residual is None else residual.data_ptr(), rng.data_ptr(), x.numel(), p, code,
                                       y.data_ptr(), stream), "envidr_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rng, p, code):
        ctx.save_for_backward(rng)
        ctx.p, ctx.code = p, code
        return _launch(x, residual, rng, p, code)

    @staticmethod
    @_bind.differentiable_once
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        dx = _launch(dy.contiguous(), None, rng, ctx.p, ctx.code) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """residual + keep * x / (1 - p), keep drawn from the counter-based generator `rng` (int64 [2] on x's device: key, call number).

    The same rng gives the same mask, whatever the dtype and the strides of x; a program that wants another mask for each call gives each its
    own call number (`CounterDropout` does).  rng must keep its values until the backward pass has run.  p counts in steps of 2^-16; p = 1
    drops everything."""
    code = _bind.same_kind("dropout", x, residual=residual)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise _lib.EnvidrError(f"dropout: p={p} is not a probability")
    if rng.dtype != torch.int64 or rng.shape != (2,) or rng.device != x.device or not rng.is_contiguous():
        raise _lib.EnvidrError("dropout: rng is two adjacent int64 numbers (key, call number) on the device of x")
    if residual is not None:
        if residual.shape != x.shape:
            raise _lib.EnvidrError(f"dropout: residual {tuple(residual.shape)} is not x {tuple(x.shape)}")
        residual = residual.contiguous()
    x = x.contiguous()
    if _bind.differentiated(x, residual):
        return _Dropout.apply(x, residual, rng, p, code)
    return _launch(x, residual, rng, p, code)


class CounterDropout(torch.nn.Module):
    """`dropout` with a generator of its own: in training every forward call takes the next call number (on the device, so a captured step draws
    a new mask at every replay); in evaluation x (+ residual) passes through.  One instance belongs to one stream at a time.

    seed: the generator's key.  Modules of one key that are called in step drop the same elements (so do a module and its copy); without a seed the key
    is drawn from torch's default CPU generator, another for each module and the same again after `torch.manual_seed`.

    A pass that is run twice (activation checkpoints) has to draw twice alike: take the call's generator first, rng = module.draw(), and hand it to
    the forward call that is checkpointed, checkpoint(module, x, rng=rng).  A training call without one inside a backward pass is refused: its mask
    would not be the one of the pass that it repeats."""

    def __init__(self, p: float = 0.1, seed: int | None = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise _lib.EnvidrError(f"CounterDropout: p={p} is not a probability")
        self.p = float(p)
        if seed is None:
            seed = int(torch.empty((), dtype=torch.int64, device="cpu").random_())
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))

    def draw(self) -> torch.Tensor:
        """the generator's next call: a copy of its own, for `forward` and for `dropout`"""
        if not self.rng.is_cuda:
            raise _lib.EnvidrError(f"CounterDropout: the generator is on {self.rng.device}: move the module to the GPU")
        used = torch.empty_like(self.rng)
        with _bind.on_device(self.rng) as stream:
            _bind.check(_bind.lib().envidr_dropout_step(self.rng.data_ptr(), used.data_ptr(), stream), "envidr_dropout_step")
        return used

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, rng: torch.Tensor | None = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else x + residual
        _bind.same_kind("CounterDropout", x, residual=residual)
        if rng is None:
            if self.rng.device != x.device:
                raise _lib.EnvidrError(f"CounterDropout: the generator is on {self.rng.device}, x on {x.device}: move the module")
            # (the number of the backward pass that this thread is in: what torch's own checkpoints go by)
            if torch._C._current_graph_task_id() != -1:
                raise _lib.EnvidrError("CounterDropout: called inside a backward pass, where a recomputed call would draw another mask: give it the "
                                       "first call's generator (rng = module.draw(), module(x, rng=rng))")
            rng = self.draw()
        return dropout(x, self.p, rng, residual=residual)

    def extra_repr(self) -> str:
        return f"p={self.p}"
