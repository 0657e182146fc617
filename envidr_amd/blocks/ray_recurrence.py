"""A gated linear recurrence along the samples of packed rays (envidr_ray_recurrence_*, csrc/ray_recurrence.hip)."""
from __future__ import annotations

import functools

import torch

from .. import _lib
from . import _bind


@functools.lru_cache(maxsize=256)
def _sizes(T, N, C):
    """bytes of the workspace, floats of what the forward pass leaves for the backward one"""
    _bind.sizes("ray_recurrence", N=N, C=C)
    lib = _bind.lib()
    return max(lib.envidr_ray_recurrence_workspace_bytes(T, N, C), 16), lib.envidr_ray_recurrence_saved_floats(T, N, C)


def _forward(gate, value, rays, state, code, blend, keep):
    lib = _bind.lib()
    T, C = gate.shape
    N = rays.shape[0]
    n, n_saved = _sizes(T, N, C)
    h = torch.empty_like(gate)
    last = gate.new_empty((N, C), dtype=torch.float32)
    saved = gate.new_empty(n_saved, dtype=torch.float32) if keep else None
    with _bind.on_device(gate) as stream:
        ws = gate.new_empty(n, dtype=torch.uint8)
        _bind.check(lib.envidr_ray_recurrence_forward(gate.data_ptr(), value.data_ptr(), rays.data_ptr(), None if state is None else state.data_ptr(), T, N, C, code, blend,
                                                      h.data_ptr(), last.data_ptr(), saved.data_ptr() if keep else None, ws.data_ptr(), n, stream),
                    "envidr_ray_recurrence_forward")
    return h, last, saved


class _RayRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, value, state, rays, code, blend):
        h, last, saved = _forward(gate, value, rays, state, code, blend, True)
        ctx.save_for_backward(gate, value, state, rays, saved)
        ctx.code, ctx.blend = code, blend
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @_bind.differentiable_once
    def backward(ctx, dh, dlast):
        gate, value, state, rays, saved = ctx.saved_tensors
        lib = _bind.lib()
        T, C = gate.shape
        N = rays.shape[0]
        n = _sizes(T, N, C)[0]
        dh = torch.zeros_like(gate) if dh is None else dh.contiguous()
        if dlast is not None:
            dlast = dlast.contiguous()
        dgate, dvalue = torch.empty_like(gate), torch.empty_like(gate)
        dstate = gate.new_empty((N, C), dtype=torch.float32) if ctx.needs_input_grad[2] else None
        with _bind.on_device(gate) as stream:
            ws = gate.new_empty(n, dtype=torch.uint8)
            _bind.check(lib.envidr_ray_recurrence_backward(dh.data_ptr(), None if dlast is None else dlast.data_ptr(), gate.data_ptr(), value.data_ptr(), rays.data_ptr(),
                                                           None if state is None else state.data_ptr(), saved.data_ptr(), T, N, C, ctx.code, ctx.blend,
                                                           dgate.data_ptr(), dvalue.data_ptr(), None if dstate is None else dstate.data_ptr(), ws.data_ptr(), n, stream),
                        "envidr_ray_recurrence_backward")
        return dgate, dvalue, dstate, None, None, None


def ray_recurrence(gate: torch.Tensor, value: torch.Tensor, rays: torch.Tensor, state: torch.Tensor | None = None, blend: bool = True):
    """h_t = a_t h_{t-1} + (1 - a_t) value_t, a_t = sigmoid(gate_t), along the samples of each ray -> (h [T, C], last [N, C]).

    gate, value [T, C] (float32, bfloat16 or float16), rays int32 [N, 3] = (id, offset, count) as `march_rays_train` returns them: rows offset ..
    offset + count - 1 are one ray's samples in order; rays may come in any order but share no rows and
    no ids.  state float32 [N, C]: h before the
    first sample, by id (zeros when not given); last float32 [N, C]: h after the last one, to go on from.  blend=False: h_t = a_t h_{t-1} + value_t.
    Rows that belong to no ray, and their gradients, are zero.  States are carried in 32 bits.  Differentiable once w.r.t. gate, value and state."""
    code = _bind.same_kind("ray_recurrence", gate, value=value)
    if gate.dim() != 2 or value.shape != gate.shape or gate.shape[1] == 0:
        raise _lib.EnvidrError(f"ray_recurrence: gate {tuple(gate.shape)} and value {tuple(value.shape)} are [T, C] both, C >= 1")
    if rays.dim() != 2 or rays.shape[1] != 3 or rays.dtype != torch.int32 or rays.device != gate.device:
        raise _lib.EnvidrError(f"ray_recurrence: rays is int32 [N, 3] on {gate.device}, not {rays.dtype} {tuple(rays.shape)} on {rays.device}")
    if state is not None and (state.dtype != torch.float32 or state.shape != (rays.shape[0], gate.shape[1]) or state.device != gate.device):
        raise _lib.EnvidrError(f"ray_recurrence: state is float32 [{rays.shape[0]}, {gate.shape[1]}] on {gate.device}, not {state.dtype} {tuple(state.shape)} on {state.device}")
    gate, value, rays = gate.contiguous(), value.contiguous(), rays.contiguous()
    state = None if state is None else state.contiguous()
    if _bind.differentiated(gate, value, state):
        return _RayRecurrence.apply(gate, value, state, rays, code, int(blend))
    h, last, _ = _forward(gate, value, rays, state, code, int(blend), False)
    return h, last


def rays_of_lengths(lengths: torch.Tensor) -> torch.Tensor:
    """`rays` int32 [N, 3] of N sequences packed one behind the other, from their lengths [N] (none negative, below 2^31 rows in all:
    not checked, the lengths stay on their device)"""
    count = lengths.reshape(-1).to(torch.int64)
    first = torch.cumsum(count, 0) - count
    return torch.stack([torch.arange(count.shape[0], device=count.device), first, count], 1).to(torch.int32)
