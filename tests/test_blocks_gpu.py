"""The block operators (envidr_amd.blocks, include/envidr_blocks.h) against their definitions in 64 bits, with the elementwise bounds of
tests/block_cases.py; strides, empty rows, captured graphs, streams, and all of them together as one block over packed ray samples."""
import zlib

import numpy as np
import pytest
import torch

from tests.block_cases import HALF_STEP, U, mlp64, philox_bits, scan64, within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _rand(g, dt, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)


def _mlp_inputs(g, dt, M, D, F, O):
    return _rand(g, dt, M, D), _rand(g, dt, F, D, scale=D ** -0.5), _rand(g, dt, F, D, scale=D ** -0.5), _rand(g, dt, O, F, scale=F ** -0.5), _rand(g, dt, M, O)


# ---- gated feed-forward block ---------------------------------------------------------------------------------------------------------------
# one row to many, around the few-row limit and the tile edges, widths of any remainder, one-wide layers, reductions that are split (over the rows;
# over the hidden layer), narrow layers whose weights stay in LDS
MLP_SHAPES = [(1, 1, 1, 1), (1, 512, 2048, 512), (2, 72, 256, 12), (15, 7, 33, 5), (16, 250, 1000, 250), (17, 64, 128, 64), (33, 90, 300, 20), (63, 130, 70, 9), (64, 256, 520, 256), (65, 256, 520, 256), (127, 72, 256, 12),
              (128, 128, 128, 128), (129, 8, 16, 8), (300, 257, 131, 259), (1000, 39, 64, 3), (4097, 72, 264, 16), (20011, 40, 72, 24),
              (40, 456, 944, 144), (200, 90, 2001, 77),
              (700, 128, 33, 64), (1000, 20, 900, 16), (33, 100, 250, 40),
              # narrow layers whose gradients' sums stay in registers: one to eight teams, the widest, and more rows than a round of workgroups takes
              (31, 96, 256, 32), (33, 96, 250, 17), (300, 65, 40, 1), (257, 33, 20, 17), (1031, 64, 100, 1), (600, 1, 64, 32), (20000, 24, 200, 8), (70000, 5, 30, 4)]


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("shape", MLP_SHAPES, ids=str)
def test_gated_mlp_forward_and_gradients(shape, dt):
    from envidr_amd.blocks import ACTIVATIONS, gated_mlp
    M, D, F, O = shape
    kind = list(ACTIVATIONS)[(M + D) % 4]
    x, wg, wu, wd, dy = _mlp_inputs(_gen(shape, str(dt)), dt, M, D, F, O)
    want = mlp64(x, wg, wu, wd, kind, dy)
    within(gated_mlp(x, wg, wu, wd, kind), *want["y"], "y without gradients")
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_mlp(*leaves, activation=kind)
    within(y, *want["y"], "y")
    for name, got in zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, leaves, dy)):
        assert got.dtype == dt
        within(got, *want[name], name)


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu", "sigmoid"])
def test_gated_mlp_gradient_is_the_difference_quotient(kind):
    """central differences of the operator itself (fp32): the loss moves along a random direction as its gradient says"""
    from envidr_amd.blocks import gated_mlp
    g = _gen(kind)
    leaves = [t.requires_grad_(True) for t in _mlp_inputs(g, torch.float32, 40, 24, 48, 16)[:4]]
    y = gated_mlp(*leaves, activation=kind)
    dy = _rand(g, torch.float32, *y.shape)
    grads = torch.autograd.grad(y, leaves, dy)
    move = [_rand(g, torch.float32, *t.shape) for t in leaves]
    loss = lambda s: float((gated_mlp(*[(t + s * m).detach() for t, m in zip(leaves, move)], activation=kind).double() * dy).sum())  # noqa: E731
    slope = sum(float((a.double() * m).sum()) for a, m in zip(grads, move))
    step = 1e-3
    quotient = (loss(step) - loss(-step)) / (2 * step)
    # the quotient's own error: u of the outputs' magnitude over the step, and its third-order term (checked to shrink with the step: 4 x for 2 x)
    wide = (loss(2 * step) - loss(-2 * step)) / (4 * step)
    noise = 64 * U * float((y.abs().double() * dy.abs()).sum()) / step
    assert abs(quotient - slope) <= noise + abs(wide - quotient), (quotient, slope, wide)


@pytest.mark.parametrize("M", [50, 100])
def test_gated_mlp_takes_any_strides_and_batch_shapes(M):
    from envidr_amd.blocks import gated_mlp
    g = _gen("strides")
    for dt in DTYPES:
        wide = _rand(g, dt, M, 3, 96)
        x = wide[:, 1, 5:77]                                    # rows 288 apart, 2 or 4 bytes off the 16-byte grid
        wg, wu, wd = _rand(g, dt, 72, 256).t(), _rand(g, dt, 300, 144)[20:276, :72], _rand(g, dt, 12, 2, 256)[:, 1]
        dy = _rand(g, dt, 12, M).t()
        want = mlp64(x, wg, wu, wd, "silu", dy)
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = gated_mlp(*leaves)
        within(y, *want["y"], "y")
        for name, got in zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, leaves, dy)):
            within(got, *want[name], name)
        # every row's gradient the same memory (sum().backward())
        y = gated_mlp(*leaves)
        one, = torch.autograd.grad(y.sum(0)[3], [leaves[0]])
        unit = torch.zeros_like(dy)
        unit[:, 3] = 1
        within(one, *mlp64(x, wg, wu, wd, "silu", unit)["dx"], "dx of a sum")
        assert gated_mlp(wide[:, :, :72].reshape(5, M // 5, 3, 72), wg, wu, wd).shape == (5, M // 5, 3, 12)


def test_gated_mlp_without_rows_and_with_only_some_gradients_wanted():
    from envidr_amd.blocks import gated_mlp
    for dt in DTYPES:
        x, wg, wu, wd, _ = _mlp_inputs(_gen("none"), dt, 0, 24, 40, 8)
        leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
        y = gated_mlp(*leaves)
        assert y.shape == (0, 8)
        got = torch.autograd.grad(y.sum(), leaves)
        assert got[0].shape == (0, 24) and all(float(t.abs().sum()) == 0 for t in got[1:])
        x, wg, wu, wd, dy = _mlp_inputs(_gen("some"), dt, 100, 24, 40, 8)
        want = mlp64(x, wg, wu, wd, "silu", dy)
        wu.requires_grad_(True)
        got, = torch.autograd.grad(gated_mlp(x, wg, wu, wd), [wu], dy)
        within(got, *want["dw_up"], "dw_up alone")
        x.requires_grad_(True)
        got, = torch.autograd.grad(gated_mlp(x, wg, wu.detach(), wd), [x], dy)
        within(got, *want["dx"], "dx alone")


def test_gated_mlp_keeps_a_bad_row_to_itself():
    """an infinity or a NaN in one row of x leaves the other rows' results as they were, bit for bit"""
    from envidr_amd.blocks import gated_mlp
    for dt in DTYPES:
        for M in (9, 200):
            x, wg, wu, wd, _ = _mlp_inputs(_gen("bad", M), dt, M, 64, 128, 32)
            good = gated_mlp(x, wg, wu, wd)
            x[4, 3], x[7, 60] = float("nan"), float("inf")
            bad = gated_mlp(x, wg, wu, wd)
            rest = [i for i in range(M) if i not in (4, 7)]
            assert torch.equal(bad[rest], good[rest]) and bad[4].isnan().all() and not bad[7].isfinite().any()


def test_gated_mlp_hidden_units_above_the_types_largest_number():
    """fp16, hidden units of 90000 and more: infinities of their sign, from few rows as from many"""
    from envidr_amd.blocks import gated_mlp
    for M in (1, 20, 33, 300):
        x = torch.full((M, 64), 300.0, dtype=torch.float16, device="cuda")
        w = torch.full((160, 64), 300.0 / (300 * 64), dtype=torch.float16, device="cuda")
        for sign in (1.0, -1.0):
            y = gated_mlp(x, w, sign * w, torch.full((80, 160), 0.01, dtype=torch.float16, device="cuda"), "relu")
            assert (y == sign * float("inf")).all()


def test_gated_mlp_single_rows_with_any_pitch():
    """a dimension of one has a stride that nothing steps by: zero, or as large as its tensor's"""
    from envidr_amd.blocks import gated_mlp
    g = _gen("one row")
    big = _rand(g, torch.bfloat16, 2, (1 << 21) + 64)
    wg, wu, wd = _rand(g, torch.bfloat16, 24, 40), _rand(g, torch.bfloat16, 24, 40), _rand(g, torch.bfloat16, 8, 24)
    for x in (big[1:, 16:56], big[1:, 16:56].as_strided((1, 40), (0, 1)), big[:1, :40].as_strided((1, 40), (7, 1))):
        within(gated_mlp(x, wg, wu, wd), *mlp64(x, wg, wu, wd, "silu")["y"], "y")
    x = _rand(g, torch.bfloat16, 50, 40)
    wg, wu = (big[i:i + 1, :40] for i in (0, 1))
    wd = _rand(g, torch.bfloat16, 1, 9).t()
    within(gated_mlp(x, wg, wu, wd), *mlp64(x, wg, wu, wd, "silu")["y"], "one hidden unit")


def test_gated_mlp_in_chunks_of_rows_adds_the_weights_gradients_up():
    """more rows than one chunk of hidden-layer operands holds (2 GiB: 71 k rows of three operands of 5000 units)"""
    from envidr_amd.blocks import gated_mlp
    M, D, F, O = 100000, 8, 5000, 8
    x, wg, wu, wd, dy = _mlp_inputs(_gen("chunks"), torch.bfloat16, M, D, F, O)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_mlp(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        some = torch.arange(0, M, 997, device="cuda")
        want = mlp64(x[some], wg, wu, wd, "silu", dy[some])
        within(y[some], *want["y"], "y")
        within(grads[0][some], *want["dx"], "dx")
        # the weights' gradients: the same sums in 64 bits, the rows in parts
        total = {}
        for part in torch.arange(M, device="cuda").split(9000):
            for name, (v, b) in mlp64(x[part], wg, wu, wd, "silu", dy[part]).items():
                if name.startswith("dw"):
                    a = total.setdefault(name, [0, 0])
                    a[0], a[1] = a[0] + v, a[1] + b
        # (a sum over all rows instead of a part's: M u of its magnitude more; the parts' own final roundings are in b already)
        for name, got in zip(("dw_gate", "dw_up", "dw_down"), grads[1:]):
            v, b = total[name]
            within(got, v, b * (1 + M * U / (9000 * U)), name)


# ---- recurrence -----------------------------------------------------------------------------------------------------------------------------
def _ray_table(rng, lengths, gaps, ids=None):
    """rays of the lengths, `gaps` rows of nobody in front of each, in a random order with random ids"""
    first = np.cumsum(np.asarray(lengths) + np.asarray(gaps)) - np.asarray(lengths)
    ids = rng.permutation(len(lengths)) if ids is None else ids
    rays = np.stack([ids, first, lengths], 1)[rng.permutation(len(lengths))]
    return rays.astype(np.int32), int(first[-1] + lengths[-1])


def _scan_lengths(kind, rng):
    return {"one": [1], "ones": [1] * 70, "row": [300], "some": [3, 0, 17, 1, 64, 5, 0, 33], "border": [256, 256, 1, 255, 257],
            "long": [1500, 2, 0, 900], "many": list(rng.randint(0, 40, 300)), "steps": [1, 0, 1, 1] * 40, "uneven": [1] * 200 + [2000] + [3] * 50}[kind]


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("C", [1, 3, 12, 64, 65, 200])
@pytest.mark.parametrize("kind", ["one", "ones", "row", "some", "border", "long", "many", "steps", "uneven"])
def test_ray_recurrence_forward_and_gradients(kind, C, dt):
    from envidr_amd.blocks import ray_recurrence
    rng = np.random.RandomState(zlib.crc32(repr((kind, C)).encode()))
    lengths = _scan_lengths(kind, rng)
    gaps = rng.randint(0, 3, len(lengths)) if kind in ("some", "many", "long") else np.zeros(len(lengths), int)
    rays, T = _ray_table(rng, lengths, gaps)
    T += 7                                                       # rows behind the last ray
    N, blend = len(rays), kind not in ("row", "many")
    half = lambda *s: torch.from_numpy(rng.randn(*s)).to(dt).cuda()  # noqa: E731
    gate, value, dh = half(T, C) + 1.5, half(T, C), half(T, C)
    state, dlast = (torch.from_numpy(rng.randn(N, C)).float().cuda() for _ in range(2))
    n64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    want = scan64(n64(gate), n64(value), rays, n64(state), blend, dt, n64(dh), n64(dlast))
    r = torch.from_numpy(rays).cuda()
    h, last = ray_recurrence(gate, value, r, state=state, blend=blend)
    within(h, *want["h"], "h without gradients")
    within(last, *want["last"], "last without gradients")
    leaves = [t.clone().requires_grad_(True) for t in (gate, value, state)]
    h, last = ray_recurrence(leaves[0], leaves[1], r, state=leaves[2], blend=blend)
    within(h, *want["h"], "h")
    within(last, *want["last"], "last")
    assert last.dtype == torch.float32 and h.dtype == dt
    for name, got in zip(("dgate", "dvalue", "dstate"), torch.autograd.grad([h, last], leaves, [dh, dlast])):
        within(got, *want[name], name)
    owned = np.zeros(T, bool)
    for _, off, cnt in rays:
        owned[off:off + cnt] = True
    assert float(h[torch.from_numpy(~owned).cuda()].abs().sum()) == 0


def test_ray_recurrence_goes_on_from_a_state():
    """a sequence in one call, and sample by sample with the state handed on: the same states (bf16 inputs, 32-bit states)"""
    from envidr_amd.blocks import ray_recurrence, rays_of_lengths
    g = _gen("steps")
    N, L, C = 5, 40, 24
    gate, value = _rand(g, torch.bfloat16, N, L, C), _rand(g, torch.bfloat16, N, L, C)
    rays = rays_of_lengths(torch.full((N,), L, device="cuda"))
    _, whole = ray_recurrence(gate.reshape(-1, C), value.reshape(-1, C), rays)
    one = rays_of_lengths(torch.ones(N, device="cuda"))
    state = None
    for t in range(L):
        _, state = ray_recurrence(gate[:, t], value[:, t], one, state=state)
    assert float((whole - state).abs().max()) <= 40 * 16 * U * float(value.abs().max())


def test_ray_recurrence_with_saturated_gates_and_with_bad_values_elsewhere():
    """gates of +-infinity hold or replace the state exactly; infinities and NaN in rows of nobody and of other rays do not reach a ray"""
    from envidr_amd.blocks import ray_recurrence
    inf = float("inf")
    for dt in DTYPES:
        T, C = 700, 5
        rays = torch.tensor([[1, 10, 400], [0, 420, 3], [2, 430, 0]], dtype=torch.int32, device="cuda")
        gate = torch.full((T, C), float("nan"), device="cuda", dtype=dt)
        value = torch.full((T, C), inf, device="cuda", dtype=dt)
        gate[10:410], value[10:410] = inf, 7.0
        gate[300], value[300] = -inf, 2.5
        gate[420:423], value[420:423] = torch.tensor([[0.0], [inf], [-inf]], device="cuda"), torch.tensor([[1.0], [5.0], [3.0]], device="cuda")
        state = torch.tensor([[4.0], [1.25], [9.0]], device="cuda").expand(3, C)
        h, last = ray_recurrence(gate, value, rays, state=state)
        want = torch.zeros(T, C)
        want[10:300], want[300:410] = 1.25, 2.5
        want[420:423] = torch.tensor([[2.5], [2.5], [3.0]])
        assert torch.equal(h.float().cpu(), want) and torch.equal(last.cpu(), torch.tensor([[3.0], [2.5], [9.0]]).expand(3, C))


@pytest.mark.parametrize("blend", [True, False], ids=["blend", "sum"])
def test_ray_recurrence_keeps_a_bad_value_along_its_own_ray_only(blend):
    """NaN and infinities in values, gates, states and gradients of long rays: from there on (backward: up to there) nothing of that ray and channel
    is finite, however small the gates' products get, and the rays before and behind it keep their bits"""
    from envidr_amd.blocks import ray_recurrence
    nan, inf, T, C = float("nan"), float("inf"), 3000, 4
    g = _gen("bad values")
    rays = torch.tensor([[2, 2000, 990], [0, 5, 900], [1, 910, 1080]], dtype=torch.int32, device="cuda")      # (910 .. 1989: the middle one)
    for shift in (0.0, -6.0):                                   # sigmoid(-6)^64 is below the smallest number
        gate, value, dh = (_rand(g, torch.float32, T, C) + (shift if i == 0 else 0.0) for i in range(3))
        state, dlast = _rand(g, torch.float32, 3, C), _rand(g, torch.float32, 3, C)

        def run():
            leaves = [t.clone().requires_grad_(True) for t in (gate, value, state)]
            out = ray_recurrence(leaves[0], leaves[1], rays, state=leaves[2], blend=blend)
            return [t.detach() for t in (*out, *torch.autograd.grad(out, leaves, (dh, dlast)))]

        good = run()
        value[1000, 0], gate[1100, 1], state[1, 2], dh[1800, 3] = nan, nan, inf, nan
        bad = run()
        others = [i for i in range(T) if not 910 <= i < 1990]
        for a, b in zip(good, bad):
            assert torch.equal(a[others] if len(a) == T else a[[0, 2]], b[others] if len(b) == T else b[[0, 2]])
        h, last, _, dvalue, dstate = bad
        for c, first in ((0, 1000), (1, 1100), (2, 910)):
            assert not h[first:1990, c].isfinite().any() and not last[1, c].isfinite() and h[910:first, c].isfinite().all()
        assert torch.equal(h[:, 3], good[0][:, 3])
        for c, behind in ((1, 1101), (3, 1801)):                # channel 1: the gradient passes the NaN gate at row 1100
            assert not dvalue[910:behind - 1, c].isfinite().any() and not dstate[1, c].isfinite() and torch.equal(dvalue[behind:, c], good[3][behind:, c])


def test_ray_recurrence_of_nothing_and_of_rays_that_do_not_fit():
    from envidr_amd.blocks import ray_recurrence
    z = torch.zeros(0, 4, device="cuda")
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    h, last = ray_recurrence(z, z, none)
    assert h.shape == (0, 4) and last.shape == (0, 4)
    state = torch.ones(2, 4, device="cuda").requires_grad_(True)
    empty = torch.tensor([[0, 0, 0], [1, 0, 0]], dtype=torch.int32, device="cuda")
    h, last = ray_recurrence(z, z, empty, state=state)
    assert torch.equal(last, state) and torch.equal(torch.autograd.grad(last.sum(), [state])[0], torch.ones(2, 4, device="cuda"))
    ones = torch.ones(9, 4, device="cuda")
    h, last = ray_recurrence(ones, ones, none)
    assert float(h.abs().sum()) == 0 and last.shape == (0, 4)
    # behind the rows, negative, an id of nobody: no rows, or rows without a state
    odd = torch.tensor([[0, 6, 4], [1, -1, 3], [77, 2, 2], [3, 5, -2]], dtype=torch.int32, device="cuda")
    state = torch.full((4, 4), 2.0, device="cuda")
    h, last = ray_recurrence(torch.zeros(9, 4, device="cuda"), ones, odd, state=state)
    assert torch.equal(last, state) and torch.equal(h[:, 0].cpu(), torch.tensor([0, 0, 0.5, 0.75, 0, 0, 0, 0, 0]))


def test_ray_recurrence_takes_the_marchers_rays():
    """the training marcher's own output: rays in the order of its counter, padded rows behind"""
    from envidr_amd.blocks import ray_recurrence
    from envidr_amd.raymarching import march_rays_train, near_far_from_aabb
    g = _gen("march")
    N = 500
    o = torch.randn(N, 3, generator=g, device="cuda") * 0.2 + torch.tensor([0, 0, 2.0], device="cuda")
    d = torch.nn.functional.normalize(torch.randn(N, 3, generator=g, device="cuda") * 0.3 - o, dim=-1)
    grid = torch.randint(0, 256, (32 ** 3 // 8,), generator=g, device="cuda", dtype=torch.uint8)
    nears, fars = near_far_from_aabb(o, d, torch.tensor([-1.0, -1, -1, 1, 1, 1], device="cuda"), 0.2)
    xyzs, _, _, rays = march_rays_train(o, d, 1, grid, 1, 32, nears, fars, align=128, max_steps=512)
    T, C = xyzs.shape[0], 12
    assert T > 2000
    gate, value = _rand(g, torch.float32, T, C), _rand(g, torch.float32, T, C)
    h, last = ray_recurrence(gate, value, rays)
    n64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    want = scan64(n64(gate), n64(value), rays.cpu().numpy(), np.zeros((N, C)), True, torch.float32)
    within(h, *want["h"], "h")
    within(last, *want["last"], "last")


# ---- dropout --------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7,), 0.1), ((8,), 0.0), ((61, 257), 0.1), ((3, 5, 64), 1.0), ((4099,), 0.9), ((1000, 72), 0.25)], ids=str)
def test_dropout_draws_the_published_stream(shape, p, dt):
    from envidr_amd.blocks import dropout
    g = _gen(shape, p, str(dt))
    x, res, dy = (_rand(g, dt, *shape) for _ in range(3))
    x = torch.where(x == 0, torch.ones_like(x), x)
    key, call = -0x123456789ABCDEF, 0x1F00000003
    rng = torch.tensor([key, call], dtype=torch.int64, device="cuda")
    limit = round(p * 65536)
    keep = philox_bits(key, call, x.numel()).reshape(shape) >= limit
    factor = np.where(keep, 65536 / max(65536 - limit, 1), 0.0)
    r = HALF_STEP[dt]
    n64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    y = dropout(x, p, rng)
    assert np.array_equal(n64(y) != 0, keep)
    want = n64(x) * factor
    within(y, want, (r + 2 * U) * np.abs(want) + 2.0 ** -25, "y")
    a, b = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
    y = dropout(a, p, rng, residual=b)
    sum64 = want + n64(res)
    within(y, sum64, (r + U) * np.abs(sum64) + 3 * U * np.abs(want) + 2.0 ** -25, "y + residual")
    da, db = torch.autograd.grad(y, [a, b], dy)
    assert torch.equal(db, dy)
    within(da, n64(dy) * factor, (r + 2 * U) * np.abs(n64(dy) * factor) + 2.0 ** -25, "dx")
    assert torch.equal(dropout(x.reshape(-1), p, rng).reshape(shape), dropout(x, p, rng))


def test_dropout_of_strided_empty_and_bad_values():
    from envidr_amd.blocks import dropout
    rng = torch.tensor([5, 9], dtype=torch.int64, device="cuda")
    for dt in DTYPES:
        x = _rand(_gen("strided"), dt, 40, 30).t()
        assert torch.equal(dropout(x, 0.3, rng, residual=x), dropout(x.contiguous(), 0.3, rng, residual=x.contiguous()))
        assert dropout(x[:0], 0.3, rng).shape == (0, 40)
        # what is dropped is zero whatever stood there
        y = dropout(torch.full((4096,), float("inf"), device="cuda", dtype=dt), 0.5, rng)
        assert bool(((y == 0) | y.isinf()).all()) and bool((y == 0).any()) and bool(y.isinf().any())


def test_counter_dropout_module_takes_a_new_mask_each_call():
    from envidr_amd.blocks import CounterDropout
    m = CounterDropout(0.5, seed=3).cuda().train()
    x = torch.ones(5000, device="cuda", requires_grad=True)
    y1, y2 = m(x), m(x)
    assert not torch.equal(y1, y2) and int(m.rng[1]) == 2
    g1, = torch.autograd.grad(y1.sum(), [x])                     # the first call's own mask, although another call came after it
    assert torch.equal(g1, y1)
    m.eval()
    assert m(x) is x and torch.equal(m(x, residual=x), x + x)
    assert "rng" in m.state_dict()


# ---- graphs, streams, repeats ---------------------------------------------------------------------------------------------------------------
def _block_pass(x, rays, leaves, dy, drop):
    """one recurrent block over packed samples: x + dropout(gated_mlp(recurrence)), and its gradients"""
    from envidr_amd.blocks import dropout, gated_mlp, ray_recurrence
    w_in, w_value, wg, wu, wd, state = leaves
    h, last = ray_recurrence(x @ w_in.t(), x @ w_value.t(), rays, state=state)
    y = dropout(gated_mlp(h, wg, wu, wd), 0.25, drop, residual=x)
    return y, last, *torch.autograd.grad([y, last], leaves, [dy, torch.ones_like(last)])


def _block_inputs(seed, dt, T=900, C=48, F=112):
    g = _gen("block", seed)
    lengths = torch.tensor([300, 1, 0, 520, 60, 9], device="cuda")
    from envidr_amd.blocks import rays_of_lengths
    rays = rays_of_lengths(lengths)
    leaves = [_rand(g, dt, C, C, scale=C ** -0.5) for _ in range(2)] + [_rand(g, dt, F, C, scale=C ** -0.5) for _ in range(2)] + [_rand(g, dt, C, F, scale=F ** -0.5)]
    leaves.append(torch.randn(6, C, generator=g, device="cuda"))
    return _rand(g, dt, T, C), rays, [t.requires_grad_(True) for t in leaves], _rand(g, dt, T, C), torch.tensor([11, seed], dtype=torch.int64, device="cuda")


def test_the_operators_together_match_the_definitions_in_64_bits():
    """the block in fp32 against the same block composed in 64 bits (torch's own derivatives): relative error of every result in the 2-norm.
    Each of the chain's stages is off by a few u sqrt(terms) of its norm (sums of <= 900 rows, 112 units, 48 channels) and passes its
    input's error on with a condition of a few units: 1e-5 leaves two decades to those figures."""
    x, rays, leaves, dy, drop = _block_inputs(1, torch.float32)
    got = _block_pass(x, rays, leaves, dy, drop)
    w = [t.detach().double().requires_grad_(True) for t in leaves]
    x64 = x.double()
    a, v = torch.sigmoid(x64 @ w[0].t()), x64 @ w[1].t()
    rows, last = [], [None] * 6
    for ident, off, cnt in rays.tolist():
        c = w[5][ident]
        for t in range(off, off + cnt):
            c = a[t] * c + (1 - a[t]) * v[t]
            rows.append(c)
        last[ident] = c
    h = torch.cat([torch.stack(rows), torch.zeros(900 - len(rows), 48, device="cuda", dtype=torch.float64)])
    y = (torch.nn.functional.silu(h @ w[2].t()) * (h @ w[3].t())) @ w[4].t()
    keep = torch.from_numpy(philox_bits(11, 1, y.numel()).reshape(y.shape) >= 16384).cuda()
    y = x64 + torch.where(keep, y * (65536 / 49152), 0)
    last = torch.stack(last)
    want = (y, last, *torch.autograd.grad([y, last], w, [dy.double(), torch.ones_like(last)]))
    for i, (p, q) in enumerate(zip(got, want)):
        off = float((p.double() - q).norm() / q.norm())
        assert off <= 1e-5, (i, off)


@pytest.mark.parametrize("width", [(48, 112), (24, 100)], ids=str)
@pytest.mark.parametrize("dt", DTYPES, ids=str)
def test_every_operator_gives_the_same_bits_again(dt, width):
    args = _block_inputs(2, dt, 900, *width)
    first = _block_pass(*args)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, _block_pass(*args)))


@pytest.mark.parametrize("C,F", [(48, 112), (24, 100)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_a_captured_block_replays_with_what_its_inputs_hold(dt, C, F):
    """forward and backward in one graph, replayed with other inputs and other call numbers between eager work: every replay equals the
    eager pass.  (The linear maps around the operators are torch's: left out of the graph.)"""
    from envidr_amd.blocks import dropout, gated_mlp, ray_recurrence

    def run(gate, value, rays, w, state, dy, rng):
        h, last = ray_recurrence(gate, value, rays, state=state)
        y = dropout(gated_mlp(h, *w), 0.25, rng, residual=value)
        return y, last, *torch.autograd.grad([y, last], [gate, value, state, *w], [dy, dlast])

    def inputs(seed):
        x, rays, leaves, dy, rng = _block_inputs(seed, dt, 900, C, F)
        return [x + 1, dy * 0.5, *[t.detach() for t in leaves[2:5]], leaves[5].detach(), dy, rng], rays

    held, rays = inputs(0)
    dlast = torch.ones(6, C, device="cuda")
    for t in held[:6]:
        t.requires_grad_(True)
    call = lambda: run(held[0], held[1], rays, held[2:5], held[5], held[6], held[7])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in (3, 4, 5, 6):
        fresh, _ = inputs(seed)
        with torch.no_grad():
            for t, f in zip(held, fresh):
                t.copy_(f)
        eager = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), seed


def test_two_streams_at_once_do_not_meet():
    a, b = _block_inputs(7, torch.bfloat16), _block_inputs(8, torch.bfloat16)
    alone = [_block_pass(*a), _block_pass(*b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    both = [[], []]
    for _ in range(5):
        for k, args in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                both[k].append(_block_pass(*args))
    torch.cuda.synchronize()
    for k in range(2):
        for got in both[k]:
            assert all(torch.equal(p, q) for p, q in zip(alone[k], got))


def test_gated_mlp_module_trains_with_dropout_and_a_residual():
    """the module's pass is the operators' composition, in training and in evaluation"""
    from envidr_amd.blocks import GatedMLP, dropout, gated_mlp
    m = GatedMLP(24, 64, residual=True, p=0.5, seed=2).cuda().train()
    x = _rand(_gen("module"), torch.float32, 500, 24)
    rng = m.drop.rng.clone()
    want = dropout(gated_mlp(x, m.w_gate, m.w_up, m.w_down), 0.5, rng, residual=x)
    y = m(x)
    assert torch.equal(y, want)
    y.square().sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
    m.eval()
    assert torch.equal(m(x), x + gated_mlp(x, m.w_gate, m.w_up, m.w_down))


def test_elements_beyond_32_bit_offsets():
    """tensors of more than 2^32 elements, empty but for their ends: the ends are computed as they are alone"""
    from envidr_amd.blocks import dropout, gated_mlp, ray_recurrence
    dt, g = torch.bfloat16, _gen("far")
    rows, D, F, O = (1 << 22) + 300, 1032, 64, 8
    assert rows * D > 1 << 32
    x, wg, wu, wd, dy = _mlp_inputs(g, dt, 300, D, F, O)
    far, fdy = torch.zeros(rows, D, dtype=dt, device="cuda"), torch.zeros(rows, O, dtype=dt, device="cuda")
    far[-300:], fdy[-300:] = x, dy
    want = mlp64(x, wg, wu, wd, "silu", dy)
    leaves = [t.requires_grad_(True) for t in (far, wg, wu, wd)]
    y = gated_mlp(*leaves)
    got = dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, leaves, fdy)))
    within(y[-300:], *want["y"], "y")
    within(got["dx"][-300:], *want["dx"], "dx")
    assert not y[:-300].any() and not got["dx"][:-300].any()
    for name in ("dw_gate", "dw_up", "dw_down"):                # (a row of zeros adds nothing, but a sum of more terms: + rows * U of what is there)
        value, bound = want[name]
        within(got[name], value, bound * (1 + rows * U), name)
    w = [t.detach() for t in (wg[:, :72].contiguous(), wu[:, :72].contiguous(), wd)]
    with torch.no_grad():                                       # a narrow layer of rows far apart
        y = gated_mlp(far[:, :72], *w)
        within(y[-300:], *mlp64(x[:, :72], *w, "silu")["y"], "narrow")
    assert not y[:-300].any()
    del far, leaves, got, y

    T, C, n = (1 << 20) + 500, 4104, 400
    assert T * C > 1 << 32
    gate, value = (torch.zeros(T, C, dtype=dt, device="cuda") for _ in range(2))
    gate[-n:], value[-n:] = _rand(g, dt, n, C), _rand(g, dt, n, C)
    rays = torch.tensor([[0, T - n, n]], dtype=torch.int32, device="cuda")
    alone = torch.tensor([[0, 0, n]], dtype=torch.int32, device="cuda")
    ends = [t[-n:].clone().requires_grad_(True) for t in (gate, value)]
    leaves = [t.requires_grad_(True) for t in (gate, value)]
    (h, last), (h1, last1) = ray_recurrence(*leaves, rays), ray_recurrence(*ends, alone)
    dlast = torch.ones_like(last)
    # (cut at other rows, so not the same bits: 64 steps' roundings at most of states below |value|)
    top = float(value.abs().max())
    assert not h[:-n].any() and float((h[-n:].float() - h1.float()).abs().max()) <= (2 ** -7 + 64 * 16 * U) * top and float((last - last1).abs().max()) <= 64 * 16 * U * top
    one, two = torch.autograd.grad(last, leaves, dlast), torch.autograd.grad(last1, ends, dlast)
    for a, b in zip(one, two):
        assert not a[:-n].any() and float((a[-n:].float() - b.float()).abs().max()) <= (2 ** -7 + 64 * 16 * U) * 2 * top
    del gate, value, leaves, h, one, a

    n, key = (1 << 32) + 4099, 77
    x = torch.ones(n, dtype=dt, device="cuda")
    y = dropout(x, 0.5, torch.tensor([key, 3], device="cuda"))
    first = (1 << 32) - 4096
    assert np.array_equal(y[first:].float().cpu().numpy(), np.where(philox_bits(key, 3, n - first, first) >= 32768, 2.0, 0.0))


def test_the_wrappers_refuse_what_does_not_fit_together():
    from envidr_amd import blocks
    from envidr_amd._lib import EnvidrError
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    for bad, text in ((lambda: blocks.gated_mlp(z(4, 8), z(16, 9), z(16, 9), z(8, 16)), "are wanted"), (lambda: blocks.gated_mlp(z(4, 8), z(16, 8), z(15, 8), z(8, 16)), "are wanted"),
                      (lambda: blocks.gated_mlp(z(4, 8), z(16, 8), z(16, 8), z(8, 15)), "are wanted"), (lambda: blocks.gated_mlp(z(4, 8), z(0, 8), z(0, 8), z(8, 0)), "zero"),
                      (lambda: blocks.gated_mlp(z(4, 8), z(16, 8, dt=torch.bfloat16), z(16, 8), z(8, 16)), "w_gate is"),
                      (lambda: blocks.gated_mlp(z(4, 8, dt=torch.float64), z(16, 8), z(16, 8), z(8, 16)), "not one of"), (lambda: blocks.gated_mlp(z(4, 8), z(16, 8), z(16, 8), z(8, 16), "tanh"), "tanh"),
                      (lambda: blocks.ray_recurrence(z(4, 8), z(4, 7), z(1, 3, dt=torch.int32)), "both"), (lambda: blocks.ray_recurrence(z(4, 8), z(4, 8), z(1, 3, dt=torch.int64)), "int32"),
                      (lambda: blocks.ray_recurrence(z(4, 8), z(4, 8), z(1, 3, dt=torch.int32).cpu()), "int32"),
                      (lambda: blocks.ray_recurrence(z(4, 8), z(4, 8), z(1, 3, dt=torch.int32), state=z(2, 8)), "state is"),
                      (lambda: blocks.ray_recurrence(z(4, 8, dt=torch.float16), z(4, 8, dt=torch.float16), z(1, 3, dt=torch.int32), state=z(1, 8, dt=torch.float16)), "state is"),
                      (lambda: blocks.dropout(z(4), 0.5, z(2)), "int64"), (lambda: blocks.dropout(z(4), 1.5, z(2, dt=torch.int64)), "probability"),
                      (lambda: blocks.dropout(z(4), 0.5, z(2, dt=torch.int64), residual=z(5)), "residual"), (lambda: blocks.CounterDropout().train()(z(4)), "move the module")):
        with pytest.raises(EnvidrError, match=text):
            bad()
