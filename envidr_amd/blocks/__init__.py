"""Block operators: the pieces of a learnt block over packed ray samples, beside the dense layers (`envidr_amd.fused`), the encoders and the
compositors (`envidr_amd.raymarching`).

- `gated_mlp(x, w_gate, w_up, w_down)`: the gated feed-forward block (act(x Wg^T) * (x Wu^T)) Wd^T, `GatedMLP` its module;
- `ray_recurrence(gate, value, rays)`: a gated linear recurrence along the samples of each ray of `march_rays_train`, `rays_of_lengths` for
  sequences that come from elsewhere;
- `dropout(x, p, rng)`: counter-based dropout with an optional residual sum, `CounterDropout` its module.

fp32, bfloat16 and float16; differentiable once; the C entry points are declared in include/envidr_blocks.h.
"""
from ._bind import DTYPES
from .dropout import CounterDropout, dropout
from .gated_mlp import ACTIVATIONS, GatedMLP, gated_mlp
from .ray_recurrence import ray_recurrence, rays_of_lengths

__all__ = ["gated_mlp", "GatedMLP", "ray_recurrence", "rays_of_lengths", "dropout", "CounterDropout", "ACTIVATIONS", "DTYPES"]
