"""ctypes signatures of include/envidr_blocks.h and the checks its wrappers share."""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from .. import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_P, _U, _U64, _I64, _I, _D = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int64, ctypes.c_int, ctypes.c_double

# entry point -> (result, arguments); include/envidr_blocks.h in its order
SIGNATURES = {
    "envidr_blocks_abi_version": (_I, []),
    "envidr_gated_mlp_workspace_bytes": (_U64, [_U, _U, _U, _U, _I, _I]),
    "envidr_gated_mlp_forward": (_I, [_P, _I64, _P, _I64, _P, _I64, _P, _I64, _U, _U, _U, _U, _I, _I, _P, _I64, _P, _U64, _P]),
    "envidr_gated_mlp_backward": (_I, [_P, _I64, _P, _I64, _P, _I64, _P, _I64, _P, _I64, _U, _U, _U, _U, _I, _I, _P, _I64, _P, _P, _P, _P, _U64, _P]),
    "envidr_ray_recurrence_saved_floats": (_U64, [_U64, _U, _U]),
    "envidr_ray_recurrence_workspace_bytes": (_U64, [_U64, _U, _U]),
    "envidr_ray_recurrence_forward": (_I, [_P, _P, _P, _P, _U64, _U, _U, _I, _I, _P, _P, _P, _P, _U64, _P]),
    "envidr_ray_recurrence_backward": (_I, [_P, _P, _P, _P, _P, _P, _P, _U64, _U, _U, _I, _I, _P, _P, _P, _P, _U64, _P]),
    "envidr_dropout": (_I, [_P, _P, _P, _U64, _D, _I, _P, _P]),
    "envidr_dropout_step": (_I, [_P, _P, _P]),
}

_bound = None


def lib() -> ctypes.CDLL:
    """the library with this header's entry points bound; raises if it lacks one"""
    global _bound
    if _bound is None:
        loaded = _lib.load()
        for name, (result, arguments) in SIGNATURES.items():
            fn = getattr(loaded, name, None)
            if fn is None:
                raise _lib.EnvidrError(f"libenvidr_amd.so does not export {name}")
            fn.restype, fn.argtypes = result, arguments
        _bound = loaded
    return _bound


def check(rc: int, name: str) -> None:
    if rc:
        raise _lib.EnvidrError(f"{name} failed ({rc}): {lib().envidr_last_error().decode()}")


def same_kind(name: str, first: torch.Tensor, **others: torch.Tensor | None) -> int:
    """the dtype code of `first`; raises unless it is a GPU tensor of a supported dtype and the others share its dtype and device"""
    if not first.is_cuda:
        raise _lib.EnvidrError(f"{name}: needs GPU tensors (got a {first.device} tensor); envidr_amd has no CPU path")
    dtype, device = first.dtype, first.device
    if dtype not in DTYPES:
        raise _lib.EnvidrError(f"{name}: {dtype} is not one of {', '.join(str(d) for d in DTYPES)}")
    for what, t in others.items():
        if t is not None and (t.dtype != dtype or t.device != device):
            raise _lib.EnvidrError(f"{name}: {what} is {t.dtype} on {t.device}, the first tensor {dtype} on {device}")
    return DTYPES[dtype]


def differentiated(*tensors: torch.Tensor | None) -> bool:
    """must a call on these go through its autograd function: for their gradients, or, where forward-mode derivatives are being taken (a tensor
    that carries a tangent requires no gradient), for torch's refusal there"""
    if forward_ad._current_level >= 0:
        return True
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def differentiable_once(backward):
    """for the `backward` of an autograd function: under create_graph its gradients, differentiated again, raise.  (torch's own decorator asks the
    incoming gradient only: where that is a constant, as for normals by autograd.grad(sdf, positions, ones, create_graph=True), it hands out constants,
    and a loss on them would silently lose its gradient.)"""
    @functools.wraps(backward)
    def run(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        out = out if isinstance(out, tuple) else (out,)
        error = torch._C._functions.DelayedError(b"the block operators are differentiable once: their gradients have none", len(out))
        return error(*(None if t is None else t.detach().requires_grad_(True) for t in out))
    return run


def sizes(name: str, **n: int) -> None:
    """raises unless the sizes pass through a C uint32"""
    for what, value in n.items():
        if value >> 32:
            raise _lib.EnvidrError(f"{name}: {what}={value} is too large")


class on_device:
    """The tensor's device as the current one for the launches inside (a no-op when it is already), and its current stream."""

    __slots__ = ("index", "before")

    def __init__(self, t: torch.Tensor):
        self.index = t.get_device()

    def __enter__(self) -> int:
        # (the current device and stream as numbers: a torch.cuda.current_stream() is an object that takes as long as a small launch)
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc) -> None:
        if self.before != self.index:
            torch.cuda.set_device(self.before)
