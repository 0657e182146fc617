"""The block operators have no forward-mode derivative: a tensor that carries a tangent is refused, never stripped of it."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def _calls():
    from envidr_amd.blocks import CounterDropout, GatedMLP, dropout, gated_mlp, ray_recurrence
    z = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    x, wg, wu, wd = z(20, 8), z(16, 8), z(16, 8), z(8, 16)
    rays, state = torch.tensor([[0, 0, 20]], dtype=torch.int32, device="cuda"), z(1, 8)
    rng = torch.tensor([1, 2], dtype=torch.int64, device="cuda")
    drop, block = CounterDropout(0.5, seed=1).cuda().train(), GatedMLP(8, 16).cuda()
    for p in block.parameters():
        p.requires_grad_(False)
    return {"gated_mlp": (gated_mlp, (x, wg, wu, wd)), "ray_recurrence": (lambda g, v, s: ray_recurrence(g, v, rays, state=s)[0], (x, z(20, 8), state)),
            "dropout": (lambda a, r: dropout(a, 0.5, rng, residual=r), (x, z(20, 8))), "CounterDropout": (drop, (x,)), "GatedMLP": (block, (x,))}


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
@pytest.mark.parametrize("name", ["gated_mlp", "ray_recurrence", "dropout", "CounterDropout", "GatedMLP"])
def test_a_tangent_is_refused(name, grad):
    call, tensors = _calls()[name]
    want = call(*tensors) if name != "CounterDropout" else None
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        if want is not None:
            assert torch.equal(call(*tensors), want)            # (no tangent among them: the call goes through)
        for i in range(len(tensors)):
            duals = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
            with pytest.raises(NotImplementedError, match="forward mode"):
                call(*duals)
    if want is not None:
        assert torch.equal(call(*tensors), want)
