"""The block operators' boundary without a GPU: the library exports what include/envidr_blocks.h declares, the binding's table is the header's,
impossible arguments are refused before anything is launched, and the 64-bit definitions the GPU tests compare with agree with torch."""
import ctypes
import importlib
import re
from pathlib import Path

import numpy as np
import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


def _declarations():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "envidr_blocks.h").read_text(), flags=re.S)
    return {m.group(2): (m.group(1), [" ".join(p.split()) for p in m.group(3).split(",")]) for m in re.finditer(r"\b(int|uint64_t)\s+(envidr_\w+)\s*\((.*?)\)\s*;", text, flags=re.S)}


def test_the_binding_is_the_header():
    from envidr_amd.blocks import _bind
    lib = _bind.lib()
    declared = _declarations()
    assert set(declared) == set(_bind.SIGNATURES)
    kinds = {"uint32_t": ctypes.c_uint32, "uint64_t": ctypes.c_uint64, "int64_t": ctypes.c_int64, "int": ctypes.c_int, "double": ctypes.c_double, "envidr_stream_t": ctypes.c_void_p}
    for name, (result, params) in declared.items():
        want = [] if params == ["void"] else [ctypes.c_void_p if "*" in p else kinds[p.split()[0]] for p in params]
        assert _bind.SIGNATURES[name] == (kinds[result], want), name
        assert hasattr(lib, name)
    assert lib.envidr_blocks_abi_version() == 1


def _refused(rc, text):
    from envidr_amd.blocks import _bind
    assert rc == -1 and text in _bind.lib().envidr_last_error(), (rc, _bind.lib().envidr_last_error())


def test_gated_mlp_refuses_what_it_cannot_take():
    from envidr_amd.blocks import _bind
    lib = _bind.lib()
    p = ctypes.cast((ctypes.c_float * 4096)(), ctypes.c_void_p)
    p = ctypes.c_void_p((p.value + 63) // 64 * 64)

    def forward(M=4, D=8, F=8, O=8, dtype=1, act=0, x=p, ldx=8, ldg=8, ldy=8, ws=p, n=1 << 20):
        return lib.envidr_gated_mlp_forward(x, ldx, p, ldg, p, 8, p, 8, M, D, F, O, dtype, act, p, ldy, ws, n, None)

    assert forward(M=0, x=None, ws=None, n=0) == 0                                # no rows: nothing to do
    _refused(forward(dtype=3), b"unknown dtype")
    _refused(forward(act=4), b"unknown activation")
    _refused(forward(D=0), b"widths")
    _refused(forward(F=1 << 21), b"widths")
    _refused(forward(D=1 << 17, F=1 << 17), b"2^32")
    _refused(forward(x=None), b"null pointer")
    _refused(forward(ldx=-8), b"row pitch")
    _refused(forward(ldg=1 << 22), b"row pitch")
    _refused(forward(ldy=7), b"ldy=7 < O=8")
    _refused(forward(ws=None), b"workspace")
    _refused(forward(n=16), b"workspace")
    _refused(forward(ws=ctypes.c_void_p(p.value + 8)), b"workspace")

    def backward(M=4, D=8, F=8, O=8, dy=p, lddx=8, dx=p, lddy=8, n=1 << 20, dtype=1):
        return lib.envidr_gated_mlp_backward(dy, lddy, p, 8, p, 8, p, 8, p, 8, M, D, F, O, dtype, 0, dx, lddx, p, p, p, p, n, None)

    _refused(backward(dy=None), b"null pointer")
    _refused(backward(lddx=7), b"lddx=7 < D=8")
    _refused(backward(lddy=-1), b"row pitch")
    _refused(backward(n=100), b"workspace")
    _refused(backward(dtype=-1), b"unknown dtype")
    assert lib.envidr_gated_mlp_backward(None, 8, None, 8, None, 8, None, 8, None, 8, 0, 8, 8, 8, 1, 0, None, 8, None, None, None, None, 0, None) == 0
    assert lib.envidr_gated_mlp_workspace_bytes(0, 8, 8, 8, 1, 0) == 0 and lib.envidr_gated_mlp_workspace_bytes(4, 0, 8, 8, 1, 0) == 0
    # the hidden layer is held a chunk of rows at a time: the workspace stops growing with the rows
    few, many = (lib.envidr_gated_mlp_workspace_bytes(m, 64, 4096, 64, 1, 1) for m in (1 << 18, 1 << 30))
    assert many == few < 3 << 30


def test_ray_recurrence_refuses_what_it_cannot_take():
    from envidr_amd.blocks import _bind
    lib = _bind.lib()
    p = ctypes.cast((ctypes.c_float * 4096)(), ctypes.c_void_p)
    p = ctypes.c_void_p((p.value + 63) // 64 * 64)

    def forward(T=8, N=2, C=4, dtype=0, gate=p, rays=p, h=p, last=p, ws=p, n=1 << 20):
        return lib.envidr_ray_recurrence_forward(gate, p, rays, None, T, N, C, dtype, 1, h, last, None, ws, n, None)

    assert forward(T=0, N=0, gate=None, rays=None, h=None, last=None, ws=None, n=0) == 0
    _refused(forward(dtype=9), b"unknown dtype")
    _refused(forward(C=0), b"no channels")
    _refused(forward(T=1 << 31), b"too large")
    _refused(forward(C=(1 << 19) + 1), b"too large")
    _refused(forward(N=1 << 26), b"too large")                                    # 64 threads a ray: more than a launch holds
    _refused(forward(T=(1 << 31) - 1, N=33 << 20), b"too large")
    _refused(forward(T=(1 << 31) - 1, N=31 << 20), b"workspace")
    _refused(forward(gate=None), b"null pointer")
    _refused(forward(rays=None), b"null pointer")
    _refused(forward(last=None), b"null pointer")
    _refused(forward(n=8), b"workspace")
    _refused(forward(ws=None), b"workspace")

    def backward(T=8, N=2, C=4, dh=p, saved=p, rays=p, n=1 << 20):
        return lib.envidr_ray_recurrence_backward(dh, None, p, p, rays, None, saved, T, N, C, 0, 1, p, p, None, p, n, None)

    _refused(backward(dh=None), b"null pointer")
    _refused(backward(saved=None), b"null pointer")
    _refused(backward(rays=None), b"null pointer")
    _refused(backward(n=0), b"workspace")
    # states, marks and owners: in proportion to the rows
    assert lib.envidr_ray_recurrence_saved_floats(1 << 20, 4, 64) < (1 << 20) * (64 // 8 + 2)


def test_dropout_refuses_what_it_cannot_take():
    from envidr_amd.blocks import _bind
    lib = _bind.lib()
    p = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p)
    assert lib.envidr_dropout(None, None, None, 0, 0.5, 0, None, None) == 0
    _refused(lib.envidr_dropout(p, None, p, 8, 1.5, 0, p, None), b"probability")
    _refused(lib.envidr_dropout(p, None, p, 8, float("nan"), 0, p, None), b"probability")
    _refused(lib.envidr_dropout(p, None, p, 8, 0.5, 7, p, None), b"unknown dtype")
    for n in (1 << 35, (1 << 64) - 1):
        _refused(lib.envidr_dropout(p, None, p, n, 0.5, 1, p, None), b"too many")
    _refused(lib.envidr_dropout(None, None, p, 8, 0.5, 0, p, None), b"null pointer")
    _refused(lib.envidr_dropout(p, None, None, 8, 0.5, 0, p, None), b"null pointer")
    _refused(lib.envidr_dropout_step(None, p, None), b"null pointer")


def test_the_wrappers_refuse_cpu_tensors_and_wrong_shapes():
    from envidr_amd import blocks
    from envidr_amd._lib import EnvidrError
    x, w, d = torch.zeros(4, 8), torch.zeros(16, 8), torch.zeros(8, 16)
    with pytest.raises(EnvidrError, match="GPU"):
        blocks.gated_mlp(x, w, w, d)
    with pytest.raises(EnvidrError, match="GPU"):
        blocks.ray_recurrence(x, x, torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(EnvidrError, match="GPU"):
        blocks.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    gated_mlp, ray_recurrence = (importlib.import_module(f"envidr_amd.blocks.{n}") for n in ("gated_mlp", "ray_recurrence"))
    with pytest.raises(EnvidrError, match="M=4294967297 is too large"):
        gated_mlp._workspace_bytes((1 << 32) + 1, 8, 8, 8, 1, 0)
    with pytest.raises(EnvidrError, match="N=4294967296 is too large"):
        ray_recurrence._sizes(5, 1 << 32, 4)
    with pytest.raises(EnvidrError, match="residual"):
        blocks.GatedMLP(8, 16, 4, residual=True)
    with pytest.raises(EnvidrError, match="activation"):
        blocks.GatedMLP(8, 16, activation="tanh")
    with pytest.raises(EnvidrError, match="probability"):
        blocks.CounterDropout(-0.1)
    assert torch.equal(blocks.rays_of_lengths(torch.tensor([3, 0, 2])), torch.tensor([[0, 0, 3], [1, 3, 0], [2, 3, 2]], dtype=torch.int32))


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu", "sigmoid"])
def test_the_64_bit_block_is_torchs(kind):
    from tests.block_cases import mlp64
    g = torch.Generator().manual_seed(1)
    x, wg, wu, wd, dy = (torch.randn(*s, generator=g) for s in ((20, 9), (13, 9), (13, 9), (5, 13), (20, 5)))
    leaves = [t.double().requires_grad_(True) for t in (x, wg, wu, wd)]
    act = {"silu": torch.nn.functional.silu, "relu": torch.relu, "sigmoid": torch.sigmoid, "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[kind]
    F = torch.nn.functional
    y = F.linear(act(F.linear(leaves[0], leaves[1])) * F.linear(leaves[0], leaves[2]), leaves[3])
    want = [y, *torch.autograd.grad(y, leaves, dy.double())]
    got = mlp64(x, wg, wu, wd, kind, dy)
    for name, w in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), want):
        assert torch.allclose(got[name][0], w, rtol=1e-12, atol=1e-12)


def test_the_64_bit_recurrence_is_torchs():
    from tests.block_cases import scan64
    g = torch.Generator().manual_seed(2)
    T, C, rays = 12, 3, np.array([[1, 5, 4], [0, 0, 3], [2, 9, 0]])
    gate, value, dh = (torch.randn(T, C, generator=g).double().requires_grad_(True) for _ in range(3))
    state, dlast = (torch.randn(3, C, generator=g).double().requires_grad_(True) for _ in range(2))
    for blend in (True, False):
        a = torch.sigmoid(gate)
        rows, last = [torch.zeros(C).double()] * T, [state[i] for i in range(3)]
        for ident, off, cnt in rays:
            for t in range(off, off + cnt):
                last[ident] = rows[t] = a[t] * last[ident] + ((1 - a[t]) if blend else 1) * value[t]
        h, last = torch.stack(rows), torch.stack(last)
        want = [h, last, *torch.autograd.grad([h, last], [gate, value, state], [dh.detach(), dlast.detach()])]
        n = lambda t: t.detach().numpy()  # noqa: E731
        got = scan64(n(gate), n(value), rays, n(state), blend, torch.float32, n(dh), n(dlast))
        for name, w in zip(("h", "last", "dgate", "dvalue", "dstate"), want):
            assert np.allclose(got[name][0], n(w), rtol=1e-12, atol=1e-12), name
