"""rms_norm over the whole range of its rows' type: squares leave f32's range long before the rows do (1.8e19, and with eps = 0 below 1e-22).

Bounds as in test_gpu_head.py: W = 2^-24; the mean of d squares, root and products (d + 16) W; outputs half a step of their type."""
import pytest
import torch

from tests.test_gpu_head import BF16, F32, W, dequant, half_step, rnd, within
from wast3d_amd import ops

pytestmark = pytest.mark.gpu

WIDTHS = [(7, 64), (300, 300), (40, 2049), (5, 9000)]      # part of a wave, a wave, a block, rows that are read again


def rows(R, d, dt, size, seed):
    x = rnd(R, d, seed=seed) * size
    x[R // 2] = rnd(d, seed=seed + 1)                      # an ordinary row among them
    return x.to(dt)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("size,eps", [(1e20, 1e-6), (3e37, 1e-6), (1e-25, 0.0), (3e-30, 0.0)])
@pytest.mark.parametrize("R,d", WIDTHS)
def test_rows_far_from_one(R, d, size, eps, dt):
    x, w = rows(R, d, dt, size, 1), (1 + 0.2 * rnd(d, seed=3)).to(dt)
    x.requires_grad_(True), w.requires_grad_(True)
    y = ops.rms_norm(x, w, eps=eps)
    s, w64 = x.detach().double(), w.detach().double()
    rs = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + float(torch.tensor(eps)))
    unit, ef, u = s * rs, (d + 16) * W, half_step(dt)
    within(y, unit * w64, (u + ef) * (unit * w64).abs() + 2.0 ** -126, "y")
    assert torch.equal(ops.rms_norm(x.detach(), w.detach(), eps=eps), y)
    q, e = ops.rms_norm_fp8(x.detach(), w.detach(), eps=eps)
    scale = torch.exp2((e - 127).double())[:, None]
    within(dequant(q, e), unit * w64, (2.0 ** -4 + ef) * (unit * w64).abs() + 2.0 ** -10 * scale, "fp8")
    dy = rnd(R, d, seed=4, dtype=dt)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    mag = (dy.double() * unit).abs().sum(0)
    tol = (ef + 2 * W + (R + 8) * W) * mag
    ref = (dy.double() * unit).sum(0)
    within(dw, ref, tol + u * (ref.abs() + tol) + 2.0 ** -126, "dw")
    g = dy.double() * w64
    dot = (g * unit).mean(1, keepdim=True)
    ref = rs * (g - unit * dot)
    ex = ef + 2 * W
    edot = (g * unit).abs().mean(1, keepdim=True) * (ex + (d + 8) * W)
    tol = rs * (unit.abs() * edot + ex * (unit * dot).abs() + (ef + 4 * W) * (g.abs() + (unit * dot).abs()))
    live = (ref.abs() < 1e38) if dt == F32 else (ref.abs() < 3e38)      # (gradients of the smallest rows leave the type's range)
    tol = tol + u * (ref.abs() + tol) + 2.0 ** -126
    within(torch.where(live, dx.double(), 0.0), torch.where(live, ref, 0.0), tol, "dx")


@pytest.mark.parametrize("dt", [BF16, F32])
def test_the_largest_and_smallest_rows(dt):
    """Rows of one value each: +-1 whatever the value, up to the type's largest; eps = 0."""
    top = torch.finfo(dt).max
    for d in (48, 1000, 2050, 8200):
        sizes = torch.tensor([top, 1e30, 1.9e19, 1.0, 1e-19, 1e-23, 1e-30, 1e-37], dtype=torch.float64, device="cuda")
        x = (sizes[:, None] * torch.where(torch.arange(d, device="cuda") % 3 == 0, -1.0, 1.0)).to(dt)
        within(ops.rms_norm(x, eps=0.0), x.double().sign(), half_step(dt) + 80 * W)
        q, e = ops.rms_norm_fp8(x, eps=0.0)
        within(dequant(q, e), x.double().sign(), 2.0 ** -4)


def test_an_infinite_row_stays_as_it_was():
    for dt in (BF16, F32):
        x = rnd(4, 64, seed=9, dtype=dt)
        x[1, 3] = float("inf")
        x[2, 5] = float("nan")
        y = ops.rms_norm(x)
        assert y[2].isnan().all() and y[1, 3].isnan() and not y[1, :3].any() and y[0].isfinite().all() and y[3].isfinite().all()
