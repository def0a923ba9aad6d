"""The backward pass outside autograd (raw_linear_bwd, raw_gated_linear_bwd): the same bits as through it, with z kept and formed again, for all gradients and for single ones."""
import pytest
import torch

from tests.test_gpu_head import BF16, F16, F32, gated_case, linear_case, rnd
from wast3d_amd import _lib, ops

pytestmark = pytest.mark.gpu

SIZES = [(40, 64, 24), (300, 99, 70), (784, 512, 512), (5000, 136, 264)]


def room(R, N, gated):
    return torch.empty(R, _lib.lib().w3d_linear_z_stride(N, gated), dtype=F32, device="cuda")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", SIZES)
def test_linear(R, K, N, dt, monkeypatch):
    for act, code in ((None, 0), ("relu", 1), ("silu", 3)):
        x, w, b, _ = linear_case(R, K, N, dt, act, True, False, seed=5)
        dy = rnd(R, N, seed=6, dtype=dt)
        for kept in (True, False) if code and dt != F32 else (code > 0,):
            monkeypatch.setattr(ops, "_KEEP_FROM", 1 if kept else 1 << 30)
            leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
            out = ops.linear(*leaves, activation=act)
            want = torch.autograd.grad(out, leaves, dy)
            y, z = torch.empty_like(out), room(R, N, 0) if kept else None
            ops.raw_linear(x, w, b, None, code, y, z)
            grads = [torch.empty_like(t) for t in (x, w, b)]
            ops.raw_linear_bwd(x, w, b, code, dy, z, *grads)
            assert torch.equal(y, out) and all(torch.equal(p, q) for p, q in zip(grads, want))
            for i in range(3):
                one = [None, None, None]
                one[i] = torch.empty_like(grads[i])
                ops.raw_linear_bwd(x, w, b, code, dy, z, *one)
                assert torch.equal(one[i], want[i])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", SIZES)
def test_gated_linear(R, K, N, dt, monkeypatch):
    case = gated_case(R, K, N, dt, bias=True, seed=7)
    dy = rnd(R, N, seed=8, dtype=dt)
    for kept in (True, False) if dt != F32 else (True,):
        monkeypatch.setattr(ops, "_KEEP_FROM", 1 if kept else 1 << 30)
        leaves = [t.clone().requires_grad_(True) for t in case]
        out = ops.gated_linear(*leaves, activation="gelu")
        want = torch.autograd.grad(out, leaves, dy)
        y, z = torch.empty_like(out), room(R, N, 1) if kept else None
        ops.raw_gated_linear(*case, 2, y, z)
        grads = [torch.empty_like(t) for t in case]
        ops.raw_gated_linear_bwd(*case, 2, dy, z, *grads)
        assert torch.equal(y, out) and all(torch.equal(p, q) for p, q in zip(grads, want))


def test_f32_rows_without_z_are_refused():
    x, w, b, _ = linear_case(40, 64, 24, F32, "relu", True, False)
    with pytest.raises(_lib.W3dError):
        ops.raw_linear_bwd(x, w, b, 1, rnd(40, 24), None, torch.empty_like(x))
    with pytest.raises(_lib.W3dError):
        ops.raw_linear_bwd(x, w, b, 0, rnd(40, 24))                                            # nothing wanted
