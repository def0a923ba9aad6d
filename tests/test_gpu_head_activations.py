"""The activations of the linear layers over their whole range.

One nonzero column in x and in the weights makes z an exact product: what is left is the activation's own part."""
import pytest
import torch

from tests.test_gpu_head import BF16, F16, F32
from wast3d_amd import ops

pytestmark = pytest.mark.gpu

# rows, inputs, outputs: few rows, 64 x 64 tiles, sliced, 256 x 256 tiles (16 bits)
SHAPES = [(40, 64, 24), (200, 64, 72), (200, 4096, 40), (4096, 128, 2048)]


def values(R):
    """z of every row: the whole range of interest, evenly, and single far ones."""
    z = torch.linspace(-13.0, 9.0, R, device="cuda")
    far = torch.tensor([-20.0, -87.0, -100.0, -1e4, 0.0, 1e-6, 30.0, 100.0, 1e4, -5.75, -5.8, -8.0], device="cuda")
    z[1:1 + len(far)] = far
    return z


def operands(R, K, N, dt):
    z = values(R).to(dt)
    x = torch.zeros(R, K, dtype=dt, device="cuda")
    x[:, K // 2] = z
    w = torch.zeros(N, K, dtype=dt, device="cuda")
    w[:, K // 2] = 1
    return z.double()[:, None].expand(R, N), x, w


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", SHAPES)
def test_relu_passes_no_gradient_where_it_is_off(R, K, N, dt, kept, monkeypatch):
    """dz is 0 where z <= 0, also where dy is infinite or not a number."""
    if dt != F32:
        monkeypatch.setattr(ops, "_KEEP_FROM", 1 if kept else 1 << 30)
    elif not kept:
        pytest.skip("f32 layers always keep z")
    z, x, w = operands(R, K, N, dt)
    on = z > 0
    x.requires_grad_(True), w.requires_grad_(True)
    b = torch.zeros(N, dtype=dt, device="cuda", requires_grad=True)
    dy = torch.full((R, N), 0.5, dtype=dt, device="cuda")
    bad = dy.clone()
    bad[~on] = float("inf")
    bad[0] = float("nan")                                  # z = -13
    for f in (lambda: ops.linear(x, w, b, activation="relu"),):
        for got, want in zip(torch.autograd.grad(f(), (x, w, b), bad), torch.autograd.grad(f(), (x, w, b), dy)):
            assert got.isfinite().all() and torch.equal(got, want)
    # gate off: nothing reaches the gate's weights and bias (the other half has dy act(g) = inf * 0)
    v = torch.zeros_like(w)
    for got, want in zip(torch.autograd.grad(ops.gated_linear(x, w, v, b, None, activation="relu"), (w, b), bad), torch.autograd.grad(ops.gated_linear(x, w, v, b, None, activation="relu"), (w, b), dy)):
        assert got.isfinite().all() and torch.equal(got, want)
