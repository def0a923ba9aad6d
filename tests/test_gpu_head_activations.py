"""The activations of the linear layers over their whole range, and their derivatives, to a relative bound.

One nonzero column in x and in the weights makes z an exact product: what is left is the activation's own error.  W = 2^-24.  An exponential of an argument a that was rounded has a relative error of
|a| W: gelu and gelu' of f32 layers evaluate exp(-z^2 / 2) (its argument rounded three times: 1.5 z^2 W) and a polynomial of relative error 1.4e-7 (2.4 W, 6 W in f32), silu and sigmoid exp(-|z|).
16-bit layers take a polynomial in the exponent for gelu's tail, fitted to less than half a step of the type: bf16 2.1e-3 of it up to z = -10.5,
f16 2.1e-4 up to -8, and less than all of it beyond (of 5e-25 and 5e-15); 2.5e-7 next to zero.  Outputs are rounded once; results whose exponential is below 2^-126 may be zero."""
import math

import pytest
import torch

from tests.test_gpu_head import BF16, F16, F32, W, half_step, tiny, within
from wast3d_amd import ops

pytestmark = pytest.mark.gpu


def act64(z, name):
    """act, act' in 64 bits (erfc and exp(-|z|): no cancellation anywhere)."""
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    e = torch.exp(-z.abs())
    s, q = torch.where(z < 0, e, 1.0) / (1 + e), torch.where(z < 0, 1.0, e) / (1 + e)
    return (z * s, s * (1 + z * q)) if name == "silu" else (s, s * q)


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


def forward_bound(z, a, act, dt):
    if act == "gelu":
        e = (16 + 2 * z * z) * W * a.abs()
        if dt != F32:
            e = e + torch.where(z < -1, (torch.where(z < -8, 1.0, 2.1e-4) if dt == F16 else torch.where(z < -10.5, 1.0, 2.1e-3)) * a.abs(), 2.5e-7)
        return e
    return (12 + 2 * z.abs()) * W * a.abs()


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("R,K,N", SHAPES)
def test_forward_values(R, K, N, act, dt):
    z, x, w = operands(R, K, N, dt)
    a, _ = act64(z, act)
    tol = forward_bound(z, a, act, dt)
    # (a 16-bit layer's exponentials leave f32's range at 2^-126 and 2^127: bf16 results below 2^-119 may be zero)
    tol = tol + half_step(dt) * (a.abs() + tol) + (2.0 ** -119 if dt == BF16 else tiny(dt))
    within(ops.linear(x, w, activation=act), a, tol, act)
    u = 1000.0 if dt == F16 else 2.0 ** 60
    v = torch.zeros_like(w)
    v[:, 0] = 1
    x2 = x.clone()
    x2[:, 0] = u                                           # the tail times a large factor
    y = ops.gated_linear(x2, w, v, activation=act)
    ref = a * u
    keep = ref.abs() < torch.finfo(dt).max / 2
    tol = forward_bound(z, a, act, dt) * u
    tol = tol + half_step(dt) * (ref.abs() + tol) + 4 * W * ref.abs() + tiny(dt) + 2.0 ** -119 * u
    within(torch.where(keep, y.double(), 0.0), torch.where(keep, ref, 0.0), tol, "gated " + act)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("R,K,N", SHAPES)
def test_derivatives(R, K, N, act, dt, kept, monkeypatch):
    """dx of one input column that reaches one output with weight 1, and the bias gradients' terms: the derivative itself."""
    if dt != F32:
        monkeypatch.setattr(ops, "_KEEP_FROM", 1 if kept else 1 << 30)
    elif not kept:
        pytest.skip("f32 layers always keep z")
    z, x, w = operands(R, K, N, dt)
    w[1:] = 0                                              # dx[:, K / 2] = dy[:, 0] act'(z)
    z, w = z[:, :1], w.requires_grad_(True)
    x.requires_grad_(True)
    dy = torch.ones(R, N, dtype=dt, device="cuda")
    dx, = torch.autograd.grad(ops.linear(x, w, activation=act), x, dy)
    a, d = act64(z, act)
    if act == "gelu":
        phi = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        tol = (16 + 2 * z * z) * W * (0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z.abs() * phi)
        if dt != F32:                                      # Phi's own error (half a step of the type; 1.1e-6 next to zero)
            rel = torch.where(z < -8, 1.0, 2.1e-4) if dt == F16 else torch.where(z < -10.5, 1.0, 2.1e-3)
            tol = tol + torch.where(z < -1, rel * 0.5 * torch.special.erfc(-z * math.sqrt(0.5)), 1.1e-6)
    elif act == "relu":
        tol = torch.zeros_like(z)
    else:
        s, q = act64(z, "sigmoid")[0], act64(-z, "sigmoid")[0]
        tol = (12 + 2 * z.abs()) * W * (s + z.abs() * s * q if act == "silu" else s * q)
    u = half_step(dt)
    tol = tol + 2 * u * (d.abs() + tol) + 2 * tiny(dt)     # dz is rounded, and dx
    within(dx[:, K // 2: K // 2 + 1], d, tol, act)


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


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid", "relu"])
def test_a_closed_gate_stays_closed(act, dt):
    """The other half of a gated layer is f32 inside and can be far past its type's range: 6e4 * 6e4 * 16 here, times act(z) of a closed gate."""
    for R, K, N in SHAPES:
        x, w, v = torch.zeros(R, K, dtype=dt, device="cuda"), torch.zeros(N, K, dtype=dt, device="cuda"), torch.zeros(N, K, dtype=dt, device="cuda")
        x[:, :16], v[:, :16] = 6e4, 6e4
        x[:, K - 1], w[:, K - 1] = -100.0, 1.0
        y = ops.gated_linear(x, w, v, activation=act).double()
        # silu's own value; gelu's and relu's is 0.  exp(-100) = 3.72e-44 lies among f32's subnormals, 2^-149 = 1.4e-45 apart: half a step is 2 % of it
        assert float(y.abs().max()) <= 100 * (math.exp(-100.0) + 2.0 ** -149) * 16 * 3.6e9 * 1.01
