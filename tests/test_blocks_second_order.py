"""The block operators are differentiable once: what create_graph hands out raises when it is differentiated, also where the incoming gradient is a
constant (normals by autograd.grad with ones, then a loss on them)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("constant", [True, False], ids=["constant", "variable"])
@pytest.mark.parametrize("name", ["gated_mlp", "ray_recurrence", "dropout", "dropout with a residual"])
def test_a_loss_on_gradients_raises(name, constant):
    from envidr_amd.blocks import dropout, gated_mlp, ray_recurrence
    z = lambda *s: torch.randn(*s, device="cuda", requires_grad=True)  # noqa: E731
    x, other, rest = z(20, 8), z(20, 8), z(5)
    w = z(16, 8), z(16, 8), z(8, 16)
    rays, rng = torch.tensor([[0, 0, 20]], dtype=torch.int32, device="cuda"), torch.tensor([1, 2], dtype=torch.int64, device="cuda")
    call, leaves = {"gated_mlp": (lambda: gated_mlp(x, *w), [x, *w]), "ray_recurrence": (lambda: ray_recurrence(x, other, rays)[0], [x, other]),
                    "dropout": (lambda: dropout(x, 0.5, rng), [x]), "dropout with a residual": (lambda: dropout(x, 0.5, rng, residual=other), [x, other])}[name]
    dy = torch.ones(20, 8, device="cuda", requires_grad=not constant)
    plain = torch.autograd.grad(call(), leaves, dy)
    assert not any(t.requires_grad for t in plain if t is not dy)     # (a residual's gradient is dy itself)
    grads = torch.autograd.grad(call(), leaves, dy, create_graph=True)
    for p, g in zip(plain, grads):
        assert torch.equal(p, g) and g.requires_grad
        with pytest.raises(RuntimeError, match="differentiable once"):
            (g.square().sum() + rest.sum()).backward()
    for t in leaves:
        t.grad = None
    (call() * dy).sum().backward(create_graph=True)               # (handed out and not differentiated: as ever)
    assert all(torch.equal(p, t.grad) for p, t in zip(plain, leaves))
