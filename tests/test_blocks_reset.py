"""The recurrence where gates let go of large states: the bounds here hold an error to what the definition joins, a |h| + (1 - a) |v|, so that
nothing is left of a state that a closed gate replaced; and infinities, which stay what the definition makes of them."""
import numpy as np
import pytest
import torch

from tests.block_cases import HALF_STEP, TINY, U, within

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
pytestmark = pytest.mark.gpu


def _definition(gate, value, state, dh, dt):
    """one ray of all rows: h, last, dgate in 64 bits and their bounds.  A step's own error: the weights a and 1 - a (in fp32 a few u; in the 16-bit
    types the exponent's rounding, 1.3 |gate| u, comes on top), a product and a sum: (12 + 1.3 |gate|) u of a |h| + (1 - a) |v|."""
    e = (12 + (0 if dt == torch.float32 else 1.3) * np.abs(gate)) * U
    a, an = 1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate))
    h, hb, prev, prevb = (np.zeros_like(gate) for _ in range(4))
    c, cb, mag = state.copy(), np.zeros_like(state), np.abs(state)
    for t in range(len(gate)):
        prev[t], prevb[t] = c, cb
        mag = a[t] * mag + an[t] * np.abs(value[t])
        c, cb = a[t] * c + an[t] * value[t], a[t] * cb + e[t] * mag
        h[t], hb[t] = c, cb
    dgate, dgb = np.zeros_like(gate), np.zeros_like(gate)
    E, Eb, Em = np.zeros_like(state), np.zeros_like(state), np.zeros_like(state)
    for t in range(len(gate) - 1, -1, -1):
        G, Gm = dh[t] + E, np.abs(dh[t]) + Em
        Gb = Eb + e[t] * Gm
        src, w = prev[t] - value[t], a[t] * an[t]
        srcb = prevb[t] + 2 * U * (np.abs(prev[t]) + np.abs(value[t]))
        dgate[t], dgb[t] = G * src * w, w * (Gb * (np.abs(src) + srcb) + np.abs(G) * srcb) + 3 * e[t] * w * Gm * (np.abs(src) + srcb)
        E, Eb, Em = a[t] * G, a[t] * Gb + e[t] * a[t] * Gm, a[t] * Gm
    r, tiny = HALF_STEP[dt], TINY[dt]
    stored = lambda v, b: (v, b + r * (np.abs(v) + b) + tiny)  # noqa: E731
    return {"h": stored(h, hb), "last": (c, cb + U * (np.abs(c) + cb)), "dgate": stored(dgate, dgb)}


@pytest.mark.parametrize("T", [40, 2000], ids=["one piece", "cut"])
@pytest.mark.parametrize("C", [5, 64])
@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_a_closed_gate_forgets_a_large_state(dt, C, T):
    from envidr_amd.blocks import ray_recurrence
    rng = np.random.RandomState(T + C)
    gate = np.where(rng.rand(T, C) < 0.1, -rng.uniform(5, 30, (T, C)), rng.randn(T, C) + 2)
    value = rng.randn(T, C) * 10.0 ** rng.uniform(-3, 4, (T, C))
    gate[7], value[7] = -30, rng.randn(C) * 1e-3                  # every channel lets go of its first state
    gate[T - 3:], value[T - 3:] = -25, rng.randn(3, C) * 1e-3
    gate, value, dh = (torch.from_numpy(t).to(dt).cuda() for t in (gate, value, rng.randn(T, C)))
    state = torch.from_numpy(rng.randn(1, C) * 1e6).float().cuda()
    n64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    want = _definition(n64(gate), n64(value), n64(state)[0], n64(dh), dt)
    rays = torch.tensor([[0, 0, T]], dtype=torch.int32, device="cuda")
    leaf = gate.clone().requires_grad_(True)
    h, last = ray_recurrence(leaf, value, rays, state=state)
    top = torch.finfo(dt).max                                     # (fp16 cannot hold the first states of 1e6: infinities there)
    held = np.abs(want["h"][0]) < top / 2
    within(torch.where(torch.from_numpy(held).cuda(), h, torch.zeros_like(h)), np.where(held, want["h"][0], 0), np.where(held, want["h"][1], 0), "h")
    within(last[0], *want["last"], "last")
    dgate, = torch.autograd.grad(h, [leaf], dh)
    held = np.abs(want["dgate"][0]) < top / 2
    within(torch.where(torch.from_numpy(held).cuda(), dgate, torch.zeros_like(dgate)), np.where(held, want["dgate"][0], 0), np.where(held, want["dgate"][1], 0), "dgate")


@pytest.mark.parametrize("state,gate,value", [(1e6, -30.0, 1e-3), (100.0, -20.0, 0.01), (3.0, -200.0, 1.2345e-5), (1.0, -18.0, 1e-3), (3e38, 0.0, -3e38), (-3e38, 1.0, 3e38), (3e38, -1.0, -3e38)])
def test_one_step_from_a_large_state(state, gate, value):
    """a h + (1 - a) v for single steps, and where v - h alone would be above the largest number"""
    from envidr_amd.blocks import ray_recurrence
    full = lambda v: torch.full((1, 4), v, device="cuda")  # noqa: E731
    _, last = ray_recurrence(full(gate), full(value), torch.tensor([[0, 0, 1]], dtype=torch.int32, device="cuda"), state=full(state))
    g, v, h = (float(torch.tensor(t)) for t in (gate, value, state))
    a, an = 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))
    want = a * h + an * v
    assert np.isfinite(float(last[0, 0])) and abs(float(last[0, 0]) - want) <= 16 * U * (a * abs(h) + an * abs(v)), (float(last[0, 0]), want)


@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_an_infinity_is_what_the_definition_makes_of_it(dt):
    """an infinite state stays one at gates whose sigmoid is above zero, and so does an infinite value's mark on it; opposite infinities meet in NaN"""
    from envidr_amd.blocks import ray_recurrence
    inf = float("inf")
    gates = torch.tensor([[-3.0], [0.0], [2.0], [-1.0], [5.0]], device="cuda").expand(5, 4).to(dt).contiguous()
    rays = torch.tensor([[0, 0, 5]], dtype=torch.int32, device="cuda")
    state = torch.tensor([[inf, -inf, 1.0, 1.0]], device="cuda")
    value = torch.ones(5, 4, device="cuda").to(dt)
    value[2, 2], value[1, 3], value[3, 3] = -inf, inf, -inf
    h, last = ray_recurrence(gates, value, rays, state=state)
    assert bool((h[:, 0] == inf).all()) and bool((h[:, 1] == -inf).all()) and last[0, :2].tolist() == [inf, -inf]
    assert bool(h[:2, 2].isfinite().all()) and bool((h[2:, 2] == -inf).all())
    assert bool(h[0, 3].isfinite()) and bool((h[1:3, 3] == inf).all()) and bool(h[3:, 3].isnan().all())
    flipped = ray_recurrence(gates, value, rays, state=state * -1)[0]
    assert bool((flipped[:, 0] == -inf).all()) and bool((flipped[:, 1] == inf).all())


@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_an_infinite_state_outlives_the_gates_product(dt):
    """along 1000 rows of gates near -3, whose product over a cut's rows is below the smallest number: infinite to the end, and the gradient of an
    infinite dlast back to the beginning"""
    from envidr_amd.blocks import ray_recurrence
    T, C, inf = 1000, 6, float("inf")
    g = torch.Generator(device="cuda").manual_seed(1)
    gate, value = ((torch.randn(T, C, generator=g, device="cuda") * 0.5 + shift).to(dt) for shift in (-3.0, 0.0))
    state = torch.tensor([inf, -inf] * 3, device="cuda").reshape(1, C).repeat(2, 1)
    rays = torch.tensor([[1, 400, 600], [0, 0, 390]], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (gate, value, state.clone())]
    h, last = ray_recurrence(leaves[0], leaves[1], rays, state=leaves[2])
    owned = [*range(390), *range(400, T)]
    assert torch.equal(last, state) and torch.equal(h[owned].float(), state[:1].expand(len(owned), C)) and not h[390:400].any()
    dvalue, dstate = torch.autograd.grad(last, leaves[1:], -state)
    assert torch.equal(dstate, -state) and torch.equal(dvalue[owned].float(), -state[:1].expand(len(owned), C)) and not dvalue[390:400].any()
