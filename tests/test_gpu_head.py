"""The layers of a feature head (rms_norm, linear, gated_linear and their 8-bit forms) against their definitions in 64 bits.

Bounds are derived, not tuned: u = half a step of the output's type (torch.finfo(t).eps / 2), w = 2^-24 for f32 arithmetic.
  * a sum of n products in f32, in any order: (n + 8) w times the sum of the products' magnitudes
  * an activation with |act'| <= 1.13 (gelu's largest slope): that many times the error of its argument, plus 4e-7 max(1, |z|) for its evaluation
    (polynomial of gelu: 1.5e-7; exponential and reciprocal: a few w)
  * derivatives: |act''| <= 0.8 (gelu at 0: 2 pdf(0)), evaluation 2e-6; relu jumps where |z| is below its own error
  * dz is rounded once to the operands' type: u |dz|
  * every output is rounded once: u |y|, or half the smallest subnormal of f16 (2^-25)
  * fp8 products: the scaled instruction keeps fewer guard bits than f32: 2^-14 of the sum of magnitudes
"""
import math

import pytest
import torch

from wast3d_amd import _lib, ops

pytestmark = pytest.mark.gpu

W = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ACTS = [None, "relu", "gelu", "silu", "sigmoid"]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == F16 else 2.0 ** -126


def rnd(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * len(shape) + sum(shape))
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def act64(z, name):
    """act, act' in 64 bits."""
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return (z * s, s * (1 + z * (1 - s))) if name == "silu" else (s, s * (1 - s))


def within(got, ref, tol, what=""):
    got, ref = got.detach().double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    over = ((got - ref).abs() - tol)
    assert torch.isfinite(got).all() and not (over > 0).any(), (what, "largest excess", float(over.max()), "at", int(over.argmax()), "of", got.numel())


def product64(x, w, b):
    """z, its magnitude sum, and the error bound of an f32 sum."""
    x, w = x.double(), w.double()
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    return z, mag, (x.shape[-1] + 8) * W * mag


def deriv_error(z, ez, name):
    e = 0.8 * ez + 2e-6
    return e + (z.abs() <= ez).double() if name == "relu" else (torch.zeros_like(e) if name is None else e)


# sizes: one element, odd everything, the boundaries of fragments (16), few-row form (64 / 65), tiles (128 / 256), sliced contractions, several tiles each way
SIZES = [(1, 1, 1), (1, 4096, 17), (3, 7, 5), (16, 64, 64), (17, 130, 33), (33, 40, 256), (64, 256, 48), (65, 128, 128), (100, 1000, 3), (129, 72, 200), (257, 515, 131), (300, 2048, 96),
         (1000, 64, 1024), (700, 999, 515), (4100, 136, 264)]
# 16-bit (and 8-bit) rows in numbers that take the 256 x 256 tile: whole tiles, odd edges everywhere, a contraction tail, sliced contractions
LARGE = [(4096, 512, 2048), (9001, 264, 1304), (16400, 72, 1032), (1030, 2056, 1016), (5000, 1032, 520), (6000, 520, 1301)]


def linear_case(R, K, N, dt, act, bias, res, seed=0, bias_dt=None):
    x = rnd(R, K, seed=seed, dtype=dt)
    w = rnd(N, K, seed=seed + 1, dtype=dt, scale=1 / math.sqrt(K))
    b = rnd(N, seed=seed + 2, dtype=bias_dt or dt) if bias else None
    r = rnd(R, N, seed=seed + 3, dtype=dt) if res else None
    return x, w, b, r


def check_linear(x, w, b, r, act, y):
    z, _, ez = product64(x, w, b)
    a, _ = act64(z, act)
    ref = a if r is None else a + r.double()
    tol = 1.13 * ez + 4e-7 * z.abs().clamp_min(1) + 4 * W * (a.abs() + ref.abs())
    within(y, ref, tol + half_step(y.dtype) * (ref.abs() + tol) + tiny(y.dtype), "y")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", SIZES)
def test_linear_forward(R, K, N, dt):
    for i, act in enumerate(ACTS):
        x, w, b, r = linear_case(R, K, N, dt, act, bias=i % 2 == 0, res=i % 3 == 0, bias_dt=F32 if i == 4 else None)
        check_linear(x, w, b, r, act, ops.linear(x, w, b, activation=act, residual=r))


@pytest.mark.parametrize("R,K,N", LARGE)
def test_large_forward(R, K, N):
    for i, (dt, act) in enumerate(((BF16, "gelu"), (F16, None))):
        x, w, b, r = linear_case(R, K, N, dt, act, bias=i == 0, res=i == 1)
        check_linear(x, w, b, r, act, ops.linear(x, w, b, activation=act, residual=r))
        c = gated_case(R, K, N, dt, bias=i == 1)
        check_gated(*c, "silu", ops.gated_linear(*c, activation="silu"))


# few rows that take tiles over a sliced contraction (long rows, many columns), next to ones that do not
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", [(1, 65536, 16), (3, 65544, 20), (16, 8192, 96), (33, 2048, 16400), (48, 4096, 520), (64, 8200, 64), (64, 16384, 33)])
def test_few_long_rows(R, K, N, dt):
    x, w, b, r = linear_case(R, K, N, dt, "gelu", True, True, seed=40)
    check_linear(x, w, b, r, "gelu", ops.linear(x, w, b, activation="gelu", residual=r))
    shift = torch.cat([w.new_zeros(1), w.reshape(-1)])[1:].view(N, K)                          # weights off the 16-byte grid: read in place
    check_linear(x, shift, b, r, "silu", ops.linear(x, shift, b, activation="silu", residual=r))
    c = gated_case(R, K, N, dt, bias=True, seed=41)
    check_gated(*c, "silu", ops.gated_linear(*c, activation="silu"))
    if dt != F32:
        fp8_layers(R, K, N, dt, [(1, "gelu")])


@pytest.mark.parametrize("R,K,N", LARGE)
def test_large_gradients(R, K, N):
    linear_gradients(R, K, N, BF16, [(2, "gelu")])
    linear_gradients(R, K, N, F16, [(0, None), (1, "relu")])
    gated_gradients(R, K, N, BF16, [(1, "silu")])
    gated_gradients(R, K, N, F16, [(0, "gelu")])


@pytest.mark.parametrize("R,K,N", LARGE)
def test_large_fp8(R, K, N):
    fp8_layers(R, K, N, BF16, [(0, None), (1, "gelu"), (2, "silu")])


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", SIZES)
def test_linear_gradients(R, K, N, dt):
    linear_gradients(R, K, N, dt, list(enumerate(ACTS)))


def linear_gradients(R, K, N, dt, acts):
    for i, act in acts:
        x, w, b, r = linear_case(R, K, N, dt, act, bias=i != 1, res=i % 2 == 1, bias_dt=F32 if i == 3 else None, seed=10)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
        y = ops.linear(x, w, b, activation=act, residual=r)
        dy = rnd(R, N, seed=20, dtype=dt)
        grads = dict(zip(["x", "w"] + (["b"] if b is not None else []) + (["r"] if r is not None else []), torch.autograd.grad(y, leaves, dy)))
        u = half_step(dt)
        x, w = x.detach(), w.detach()
        z, _, ez = product64(x, w, b.detach() if b is not None else None)
        _, d = act64(z, act)
        dz = dy.double() * d
        edz = dy.double().abs() * deriv_error(z, ez, act) + 2 * W * dz.abs()                    # before the rounding to the operands' type
        eop = edz + (u * (dz.abs() + edz) + tiny(dt) if act is not None else 0)
        xa, wa, dza = x.double().abs(), w.double().abs(), dz.abs()
        for name, ref, tol in (("x", dz @ w.double(), eop @ wa + (N + 8) * W * (dza @ wa)), ("w", dz.t() @ x.double(), eop.t() @ xa + (R + 8) * W * (dza.t() @ xa)),
                               ("b", dz.sum(0), edz.sum(0) + (R + 8) * W * dza.sum(0))):
            if name in grads:
                within(grads[name], ref, tol + half_step(grads[name].dtype) * (ref.abs() + tol) + tiny(grads[name].dtype), f"d{name} {act}")
        if r is not None:
            assert torch.equal(grads["r"], dy)


def gated_case(R, K, N, dt, bias, seed=0, bias_dt=None):
    x = rnd(R, K, seed=seed, dtype=dt)
    wg, wu = (rnd(N, K, seed=seed + i, dtype=dt, scale=1 / math.sqrt(K)) for i in (1, 2))
    bg, bu = (rnd(N, seed=seed + i, dtype=bias_dt or dt) if bias else None for i in (3, 4))
    return x, wg, wu, bg, bu


def check_gated(x, wg, wu, bg, bu, act, y, extra=0.0):
    g, mg, eg = product64(x, wg, bg)
    u, mu, eu = product64(x, wu, bu)
    eg, eu = eg + extra * mg, eu + extra * mu
    a, _ = act64(g, act)
    ref, ea = a * u, 1.13 * eg + 4e-7 * g.abs().clamp_min(1)
    tol = ea * (u.abs() + eu) + a.abs() * eu + 4 * W * ref.abs()
    within(y, ref, tol + half_step(y.dtype) * (ref.abs() + tol) + tiny(y.dtype), "y")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", SIZES)
def test_gated_forward(R, K, N, dt):
    for i, act in enumerate(ACTS):
        c = gated_case(R, K, N, dt, bias=i % 2 == 0, bias_dt=F32 if i == 2 else None)
        check_gated(*c, act, ops.gated_linear(*c, activation=act))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,K,N", SIZES)
def test_gated_gradients(R, K, N, dt):
    gated_gradients(R, K, N, dt, list(enumerate(ACTS)))


def gated_gradients(R, K, N, dt, acts):
    for i, act in acts:
        c = gated_case(R, K, N, dt, bias=i % 2 == 1, seed=30)
        leaves = [t.requires_grad_(True) for t in c if t is not None]
        y = ops.gated_linear(*c, activation=act)
        dy = rnd(R, N, seed=40, dtype=dt)
        grads = dict(zip(("x", "wg", "wu", "bg", "bu"), torch.autograd.grad(y, leaves, dy)))
        x, wg, wu, bg, bu = (t.detach() if t is not None else None for t in c)
        h = half_step(dt)
        g, _, eg = product64(x, wg, bg)
        u, _, eu = product64(x, wu, bu)
        a, d = act64(g, act)
        dyd = dy.double()
        dg, du = dyd * u * d, dyd * a
        edg = dyd.abs() * ((u.abs() + eu) * deriv_error(g, eg, act) + eu * d.abs()) + 3 * W * dg.abs()
        edu = dyd.abs() * (1.13 * eg + 4e-7 * g.abs().clamp_min(1)) + 2 * W * du.abs()
        og, ou = edg + h * (dg.abs() + edg) + tiny(dt), edu + h * (du.abs() + edu) + tiny(dt)
        xa, ga, ua = x.double().abs(), wg.double().abs(), wu.double().abs()
        checks = [("x", dg @ wg.double() + du @ wu.double(), og @ ga + ou @ ua + (2 * N + 8) * W * (dg.abs() @ ga + du.abs() @ ua)),
                  ("wg", dg.t() @ x.double(), og.t() @ xa + (R + 8) * W * (dg.abs().t() @ xa)), ("wu", du.t() @ x.double(), ou.t() @ xa + (R + 8) * W * (du.abs().t() @ xa)),
                  ("bg", dg.sum(0), edg.sum(0) + (R + 8) * W * dg.abs().sum(0)), ("bu", du.sum(0), edu.sum(0) + (R + 8) * W * du.abs().sum(0))]
        for name, ref, tol in checks:
            if name in grads:
                within(grads[name], ref, tol + h * (ref.abs() + tol) + tiny(dt), f"d{name} {act}")


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("R", [40, 700])
def test_any_subset_of_gradients(R, dt):
    """A call that wants only some of its gradients gets the same bits for them as one that wants all."""
    x, w, b, r = linear_case(R, 99, 70, dt, "silu", True, True, seed=170)
    v, c = rnd(70, 99, seed=171, dtype=dt, scale=0.1), rnd(70, seed=172, dtype=dt)
    dy = rnd(R, 70, seed=173, dtype=dt)
    calls = [(lambda x, w, b, r: ops.linear(x, w, b, activation="silu", residual=r), (x, w, b, r)), (lambda x, w, b: ops.linear(x, w, b), (x, w, b)),
             (lambda x, w, v, b, c: ops.gated_linear(x, w, v, b, c, activation="gelu"), (x, w, v, b, c)), (lambda x, w, r: sum(ops.rms_norm(x, w, residual=r)), (r, b, r * 0.5))]
    for f, args in calls:
        full = [a.clone().requires_grad_(True) for a in args]
        want = torch.autograd.grad(f(*full), full, dy)
        for mask in range(1, 2 ** len(args)):
            some = [a.clone().requires_grad_(bool(mask >> i & 1)) for i, a in enumerate(args)]
            live = [i for i in range(len(args)) if mask >> i & 1]
            got = torch.autograd.grad(f(*some), [some[i] for i in live], dy)
            assert all(torch.equal(g, want[i]) for g, i in zip(got, live)), (mask, live)


def test_gradients_accumulate_and_second_derivatives_are_refused():
    x, w = rnd(70, 64, seed=180).requires_grad_(True), rnd(48, 64, seed=181).requires_grad_(True)
    y = ops.linear(ops.rms_norm(x) + ops.rms_norm(x), w, activation="gelu")
    y.sum().backward()
    first = x.grad.clone(), w.grad.clone()
    ops.linear(ops.rms_norm(x) + ops.rms_norm(x), w, activation="gelu").sum().backward()
    assert torch.equal(x.grad, 2 * first[0]) and torch.equal(w.grad, 2 * first[1])
    g, = torch.autograd.grad(ops.linear(x, w, activation="gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


# ------------------------------------------------------------------------------------------------ 8-bit rows
def dequant(q, e):
    return torch.ldexp(q.view(torch.float8_e4m3fn).double(), (e - 127)[:, None].double())


@pytest.mark.parametrize("out", [BF16, F16])
@pytest.mark.parametrize("R,K,N", SIZES)
def test_fp8_layers(R, K, N, out):
    fp8_layers(R, K, N, out, list(enumerate(ACTS)))


def fp8_layers(R, K, N, out, acts):
    kp = -(-K // 4) * 4                                                                        # quantize_rows_fp8 takes multiples of 4; the layers any width
    rows = lambda n, seed, scale=1.0: (rnd(n, kp, seed=seed, scale=scale) * torch.exp2(rnd(n, 1, seed=seed + 1) * 3)).contiguous()  # noqa: E731
    q, wq, uq = (ops.quantize_rows_fp8(t) for t in (rows(R, 50), rows(N, 51, 1 / math.sqrt(K)), rows(N, 52, 1 / math.sqrt(K))))
    (q, e), (wq, we), (uq, ue) = ((a[:, :K].contiguous(), b) for a, b in (q, wq, uq))
    x, w, u = dequant(q, e), dequant(wq, we), dequant(uq, ue)
    for i, act in acts:
        b = rnd(N, seed=53, dtype=F32 if i == 1 else out) if i % 2 else None
        r = rnd(R, N, seed=54, dtype=out) if i % 3 == 0 else None
        y = ops.linear_fp8(q, e, wq, we, b, activation=act, residual=r, out_dtype=out)
        z, mag, ez = product64(x, w, b)
        ez = ez + 2.0 ** -14 * mag
        a, _ = act64(z, act)
        ref = a if r is None else a + r.double()
        big = torch.finfo(out).max
        ok = ref.abs() + 1.13 * ez < big / 2                                                   # f16: values past its range are infinite, and not looked at
        tol = 1.13 * ez + 4e-7 * z.abs().clamp_min(1) + 4 * W * (a.abs() + ref.abs())
        tol = tol + half_step(out) * (ref.abs() + tol) + tiny(out)
        assert bool(ok.float().mean() > 0.5)
        within(torch.where(ok, y.double(), 0.0), torch.where(ok, ref, 0.0), tol, act)
        y = ops.gated_linear_fp8(q, e, wq, we, uq, ue, b, b, activation=act, out_dtype=BF16 if b is None or b.dtype == F32 else out)
        if y.dtype == BF16:
            check_gated(x, w, u, b, b, act, y, extra=2.0 ** -14)


def test_fp8_scales_far_apart():
    """Exponents are added before they are applied: neither side's scale alone may overflow or vanish."""
    K, N = 64, 48
    for R in (5, 200):
        q, wq = (ops.quantize_rows_fp8(rnd(n, K, seed=60))[0] for n in (R, N))
        for ex, ew in ((1, 250), (250, 1), (127, 127), (3, 249)):
            e, we = torch.full((R,), ex, dtype=torch.int32, device="cuda"), torch.full((N,), ew, dtype=torch.int32, device="cuda")
            x, w = dequant(q, e), dequant(wq, we)
            z, mag, ez = product64(x, w, None)
            tol = ez + 2.0 ** -14 * mag
            within(ops.linear_fp8(q, e, wq, we), z, tol + half_step(BF16) * (z.abs() + tol) + 2.0 ** -126)


# ------------------------------------------------------------------------------------------------ norm
NORMS = [(1, 1), (5, 3), (1, 4096), (33, 8), (100, 60), (257, 256), (65, 255), (40, 500), (31, 513), (300, 1024), (17, 2047), (9, 2049), (12, 4099), (6, 8192), (5, 8193), (3, 20001), (70000, 64)]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,d", NORMS)
def test_rms_norm(R, d, dt):
    for res, weight in ((False, dt), (True, dt), (True, F32), (True, None), (False, None)):
        x = rnd(R, d, seed=1, dtype=dt) * 3
        r = rnd(R, d, seed=2, dtype=dt) if res else None
        w = (1 + 0.2 * rnd(d, seed=3)).to(weight) if weight is not None else None
        eps = 1e-5
        leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
        got = ops.rms_norm(x, w, residual=r, eps=eps)
        y, s = got if res else (got, None)
        u = half_step(dt)
        s64 = x.detach().double() + (r.detach().double() if res else 0.0)
        w64 = w.detach().double() if w is not None else torch.ones(d, dtype=torch.float64, device="cuda")
        rs = 1 / torch.sqrt((s64 * s64).mean(1, keepdim=True) + eps)
        unit = s64 * rs
        ef = (d + 16) * W                                                                      # f32: sum of d squares, root, two products
        within(y, unit * w64, (u + ef) * (unit * w64).abs() + tiny(dt), "y")
        if res:
            within(s, s64, (u + W) * s64.abs() + tiny(dt), "s")
        dy = rnd(R, d, seed=4, dtype=dt)
        ds = rnd(R, d, seed=5, dtype=dt) if res else None
        grads = torch.autograd.grad([y] + ([s] if res else []), leaves, [dy] + ([ds] if res else []))
        g = dy.double() * w64
        dot = (g * unit).mean(1, keepdim=True)
        dx = rs * (g - unit * dot) + (ds.double() if res else 0.0)
        ex = ef + 2 * W                                                                        # relative error of x^ (s is formed again, in f32)
        edot = (g * unit).abs().mean(1, keepdim=True) * (ex + (d + 8) * W)
        tol = rs * (unit.abs() * edot + ex * (unit * dot).abs() + (ef + 4 * W) * (g.abs() + (unit * dot).abs()))
        within(grads[0], dx, tol + u * (dx.abs() + tol) + tiny(dt), "dx")
        if res:
            assert torch.equal(grads[0], grads[1])
        if w is not None:
            dw, mag = (dy.double() * unit).sum(0), (dy.double() * unit).abs().sum(0)
            tol = (ex + (R + 8) * W) * mag
            uw = half_step(w.dtype)
            within(grads[-1], dw, tol + uw * (dw.abs() + tol) + tiny(w.dtype), "dw")
        plain = ops.rms_norm(x.detach(), w.detach() if w is not None else None, residual=r.detach() if res else None, eps=eps)
        assert torch.equal(plain[0] if res else plain, y)                                      # the call without gradients: the same bits


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("R,d", NORMS)
def test_rms_norm_fp8(R, d, dt):
    x, r, w = rnd(R, d, seed=1, dtype=dt), rnd(R, d, seed=2, dtype=dt), (1 + 0.2 * rnd(d, seed=3)).to(dt)
    if R > 4:
        x[2] = 0
        r[2] = 0                                                                               # a row of zeros: exponent 127, bytes 0
    q, e, s = ops.rms_norm_fp8(x, w, residual=r)
    assert torch.equal(s, ops.rms_norm(x, w, residual=r)[1])
    s64 = x.double() + r.double()
    y = s64 / torch.sqrt((s64 * s64).mean(1, keepdim=True) + 1e-6) * w.double()
    scale, top = torch.exp2((e - 127).double())[:, None], y.abs().amax(1, keepdim=True)
    ef = (d + 16) * W
    within(dequant(q, e), y, (2.0 ** -4 + ef) * y.abs() + 2.0 ** -10 * scale, "rows")
    live = top > 0
    assert bool((448 * scale * (1 + 2 * ef) >= top).all()) and bool((224 * scale * (1 - 2 * ef) < top)[live].all())      # the smallest power of two that holds the row
    if R > 4:
        assert int(e[2]) == 127 and int(q[2].max()) == 0
    if dt == F32 and d % 4 == 0:
        q2, e2 = ops.quantize_rows_fp8(ops.rms_norm(x + r, w))
        assert torch.equal(e, e2) and torch.equal(q.view(torch.float8_e4m3fn).float(), q2.view(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("R,d", [(200000, 256), (300, 2056), (40, 9000)])
def test_rms_norm_fp8_is_the_rounded_definition(R, d, dt):
    """8-bit rows are the 64-bit rows rounded to f32 and then to e4m3: no value falls on the other side of a border (the sums' orders differ by 2^-50)."""
    x, w = rnd(R, d, seed=51, dtype=dt), (1 + 0.1 * rnd(d, seed=52)).to(dt)
    q, e = ops.rms_norm_fp8(x, w)
    y = (x.double() * (1 / torch.sqrt(x.double().square().mean(1, keepdim=True) + float(torch.tensor(1e-6)))) * w.double()).float()
    m, ex = torch.frexp(y.abs().amax(1))
    assert torch.equal(e, torch.where(m <= 0.875, ex - 9, ex - 8) + 127)
    assert torch.equal(dequant(q, e), (y.double() * torch.exp2(127.0 - e.double())[:, None]).float().to(torch.float8_e4m3fn).double() * torch.exp2(e.double() - 127)[:, None])


def test_rms_norm_only_the_sum_is_used():
    x, r, w = (rnd(40, 96, seed=i).requires_grad_(True) for i in (1, 2, 3))
    w = rnd(96, seed=3).requires_grad_(True)
    s = ops.rms_norm(x, w, residual=r)[1]
    gs = rnd(40, 96, seed=9)
    gx, gr, gw = torch.autograd.grad(s, (x, r, w), gs)
    assert torch.equal(gx, gs) and torch.equal(gr, gs) and not gw.any()


def test_rms_norm_eps_zero_row_and_extremes():
    x = torch.zeros(4, 64, device="cuda", dtype=BF16)
    assert not ops.rms_norm(x, eps=1e-6).any()
    x[1] = float("inf")
    x[2, 3] = float("nan")
    y = ops.rms_norm(x)
    assert not y[0].any() and not y[3].any() and y[2].isnan().all() and y[1].isnan().all()     # inf * 0
    big = torch.full((2, 64), 1e18, device="cuda")
    within(ops.rms_norm(big), torch.ones(2, 64, device="cuda"), 80 * W)


# ------------------------------------------------------------------------------------------------ strides, alignment, neighbours in memory
@pytest.mark.parametrize("dt", [BF16, F32])
def test_strides_and_alignment(dt):
    for R, K, N in ((7, 64, 32), (200, 64, 96), (300, 100, 72)):
        x, w, b, r = linear_case(R, K, N, dt, "silu", True, True, seed=70)
        want = ops.linear(x, w, b, activation="silu", residual=r)
        shift = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731   (contiguous, one element off the allocation's start)
        assert shift(x).data_ptr() % 16 != 0
        for f in (lambda t: t.t().contiguous().t(), lambda t: torch.stack([t, t], -1)[..., 0]):    # columns first; every second element
            check_linear(x, w, b, r, "silu", ops.linear(f(x), f(w), b, activation="silu", residual=f(r)))
            assert torch.equal(want, ops.linear(f(x), f(w), b, activation="silu", residual=f(r)))
        check_linear(x, w, b, r, "silu", ops.linear(shift(x), shift(w), shift(b), activation="silu", residual=shift(r)))
        y3 = ops.linear(x.view(1, R, K).expand(2, R, K), w, b, activation="silu")               # leading dimensions, a broadcast one among them
        assert y3.shape == (2, R, N) and torch.equal(y3[0], y3[1])
        assert torch.equal(ops.rms_norm(shift(x)), ops.rms_norm(x)) and torch.equal(ops.rms_norm(x.t().contiguous().t()), ops.rms_norm(x))
        g = ops.gated_linear(shift(x), shift(w), w, shift(b), b, activation="gelu")
        check_gated(x, w, w, b, b, "gelu", g)


def test_broadcast_inputs_get_summed_gradients():
    x, w = rnd(1, 64, seed=1).requires_grad_(True), rnd(1, 48, seed=2).requires_grad_(True)
    y = ops.linear(x.expand(300, 64), rnd(48, 64, seed=3), residual=w.expand(300, 48))
    dy = rnd(300, 48, seed=4)
    gx, gr = torch.autograd.grad(y, (x, w), dy)
    ref = dy.double() @ rnd(48, 64, seed=3).double()
    within(gx, ref.sum(0, keepdim=True), 800 * W * ref.abs().sum(0, keepdim=True) + 1e-4)
    within(gr, dy.double().sum(0, keepdim=True), 800 * W * dy.double().abs().sum(0, keepdim=True))


@pytest.mark.parametrize("R,K,N", [(5, 64, 33), (130, 72, 200), (300, 999, 515), (300, 1024, 96)])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_rows_behind_the_last_stay(R, K, N, dt):
    x, w, b, _ = linear_case(R, K, N, dt, None, True, False, seed=80)
    room = torch.full((R * N + 512,), 7.0, dtype=dt, device="cuda")
    ops.raw_linear(x, w, b, None, 0, room[256:256 + R * N].view(R, N))
    assert bool((room[:256] == 7).all()) and bool((room[256 + R * N:] == 7).all())
    check_linear(x, w, b, None, None, room[256:256 + R * N].view(R, N))
    room.fill_(7.0)
    ops.raw_gated_linear(x, w, w, b, None, 3, room[256:256 + R * N].view(R, N))
    assert bool((room[:256] == 7).all()) and bool((room[256 + R * N:] == 7).all())
    room = torch.full((R * K + 512,), 7.0, dtype=dt, device="cuda")
    ops.raw_rms_norm(x, None, None, 1e-6, room[256:256 + R * K].view(R, K))
    assert bool((room[:256] == 7).all()) and bool((room[256 + R * K:] == 7).all())


@pytest.mark.parametrize("R", [9, 300])
def test_a_bad_row_stays_alone(R):
    """Infinities and NaN in one row of x (or of the weights) reach that row (column) of the output and nothing else, also where tiles read past an edge."""
    for K, N in ((96, 70), (99, 130)):
        x, w, b, _ = linear_case(R, K, N, BF16, "silu", True, False, seed=90)
        clean = ops.linear(x, w, b, activation="silu")
        x2, w2 = x.clone(), w.clone()
        x2[R - 1, 5], x2[2, 0], w2[N - 1, 3] = float("inf"), float("nan"), float("nan")
        y = ops.linear(x2, w2, b, activation="silu")
        keep = torch.ones(R, N, dtype=torch.bool, device="cuda")
        keep[R - 1], keep[2], keep[:, N - 1] = False, False, False
        assert torch.equal(y[keep], clean[keep]) and y[2].isnan().all() and y[:, N - 1].isnan().all()
        g = ops.gated_linear(x2, w, w2, activation="gelu")
        assert torch.equal(g[keep], ops.gated_linear(x, w, w, activation="gelu")[keep])


def test_bad_gradient_rows_stay_alone():
    """dx of a row depends on that row alone; padding columns of dz (70 is no multiple of a chunk) are zeros whatever the memory held."""
    x, w, b, _ = linear_case(150, 96, 70, BF16, "gelu", True, False, seed=95)
    x.requires_grad_(True)
    dy = rnd(150, 70, seed=96, dtype=BF16)
    bad = dy.clone()
    bad[149] = float("nan")
    junk = torch.full((1 << 22,), float("nan"), device="cuda")
    del junk                                                                                   # the next workspace is likely cut from this
    for f in (lambda: ops.linear(x, w, b, activation="gelu"), lambda: ops.gated_linear(x, w, w, activation="gelu")):
        a, = torch.autograd.grad(f(), x, dy)
        c, = torch.autograd.grad(f(), x, bad)
        assert a.isfinite().all() and torch.equal(a[:149], c[:149]) and c[149].isnan().all()


@pytest.mark.parametrize("N", [64, 70])
@pytest.mark.parametrize("act", ["relu", "sigmoid"])
def test_an_infinite_row_keeps_its_finite_gradient(act, N):
    """z = +-inf: the derivatives are 0 or 1 and dx finite; columns that only pad dz to whole chunks (70) must not add inf * 0."""
    x, w, _, _ = linear_case(150, 96, N, BF16, act, False, False, seed=97)
    x[149, 5] = float("inf")
    dy = rnd(150, N, seed=98, dtype=BF16)
    dx, = torch.autograd.grad(ops.linear(x.requires_grad_(True), w, activation=act), x, dy)
    d = (w[:, 5] > 0).double() if act == "relu" else torch.zeros(N, dtype=torch.float64, device="cuda")
    dz = dy[149].double() * d
    ref, mag = dz @ w.double(), dz.abs() @ w.double().abs()
    within(dx[149], ref, (N + 8) * W * mag + half_step(BF16) * ref.abs() + tiny(BF16))
    assert dx[:149].isfinite().all()


def test_rows_just_short_of_8_megabytes():
    """The longest rows there are (32-bit offsets inside a tile): the last columns hold everything, so that the definition is a small product."""
    K, used = (8 << 20) // 2 - 8, 512
    for R, N in ((100, 9), (1030, 264)):
        x, w = torch.zeros(R, K, dtype=BF16, device="cuda"), torch.zeros(N, K, dtype=BF16, device="cuda")
        xs, ws, b, _ = linear_case(R, used, N, BF16, None, True, False, seed=185)
        x[:, -used:], w[:, -used:] = xs, ws
        y = ops.linear(x.requires_grad_(True), w.requires_grad_(True), b)
        check_linear(xs, ws, b, None, None, y)
        dy = rnd(R, N, seed=186, dtype=BF16)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        for got, p, q, n in ((dx, dy, ws, N), (dw, dy.t(), xs, R)):
            ref, mag = p.double() @ q.double(), p.double().abs() @ q.double().abs()
            within(got[:, -used:], ref, (n + 8) * W * mag + half_step(BF16) * ref.abs() + tiny(BF16))
            assert not got[:, :-used].any()
        del x, w, y, dx, dw, got
    with pytest.raises(_lib.W3dError):
        ops.linear(torch.zeros(1, K + 8, dtype=BF16, device="cuda"), torch.zeros(1, K + 8, dtype=BF16, device="cuda"))


def test_rms_norm_widths_past_32_bits_are_refused():
    one = torch.ones(1, 1, dtype=BF16, device="cuda")
    for d in ((1 << 30) + 1, (1 << 31) + 5, (1 << 32) + 5):
        for f in (ops.rms_norm, ops.rms_norm_fp8):
            with pytest.raises(_lib.W3dError):
                f(one.expand(1, d))


def test_rms_norm_fp8_of_infinities():
    """An infinity behind the norm saturates, by the rule of quantize_rows_fp8; the other rows do not see it."""
    x, w = rnd(5, 64, seed=187), torch.ones(64, device="cuda")
    q0, e0 = ops.rms_norm_fp8(x, w)
    w[7] = float("inf")
    q, e = ops.rms_norm_fp8(x, w)
    q2, e2 = ops.quantize_rows_fp8(ops.rms_norm(x, w))
    assert torch.equal(q, q2) and torch.equal(e, e2)
    x[3] *= 3.0e38
    x[3, 9] = float("inf")
    q, e = ops.rms_norm_fp8(x)
    keep = torch.arange(5, device="cuda") != 3
    assert torch.equal(q[keep], q0[keep]) and torch.equal(e[keep], e0[keep])


def test_more_than_2_to_the_31_elements():
    """Rows whose elements are past 2^31 (and bytes past 2^32) from the first: the last rows of every output against the definition on those rows alone."""
    R, K, N, tail = 2_200_001, 1024, 128, 300
    x = torch.empty(R, K, dtype=BF16, device="cuda")
    x[: 1 << 16] = rnd(1 << 16, K, seed=190, dtype=BF16)
    for a in range(1 << 16, R, 1 << 16):
        x[a: a + (1 << 16)] = x[: min(1 << 16, R - a)]
    x[-tail:] = rnd(tail, K, seed=191, dtype=BF16)
    w, b = rnd(N, K, seed=192, dtype=BF16, scale=K ** -0.5), rnd(N, seed=193, dtype=BF16)
    y = ops.linear(x, w, b, activation="gelu")
    check_linear(x[-tail:], w, b, None, "gelu", y[-tail:])
    check_linear(x[:tail], w, b, None, "gelu", y[:tail])
    assert torch.equal(ops.rms_norm(x)[-tail:], ops.rms_norm(x[-tail:].clone()))
    q, e = ops.rms_norm_fp8(x)
    q1, e1 = ops.rms_norm_fp8(x[-tail:].clone())
    assert torch.equal(q[-tail:], q1) and torch.equal(e[-tail:], e1)
    check_linear(dequant(q[-tail:], e[-tail:]), dequant(*ops.quantize_rows_fp8(w)), None, None, None, ops.linear_fp8(q, e, *ops.quantize_rows_fp8(w))[-tail:])
    del q, e, y
    dy = torch.zeros(R, N, dtype=BF16, device="cuda")
    dy[-tail:] = rnd(tail, N, seed=194, dtype=BF16)
    w.requires_grad_(True)
    xg = x.requires_grad_(True)
    dx, dw = torch.autograd.grad(ops.linear(xg, w, b, activation="gelu"), (xg, w), dy)
    xt, wt = x.detach()[-tail:].clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    dxt, dwt = torch.autograd.grad(ops.linear(xt, wt, b, activation="gelu"), (xt, wt), dy[-tail:])
    # (the same products in another cut: two f32 sums of the same terms, rounded once)
    assert not dx[:-tail].any()
    for a, c in ((dx[-tail:], dxt), (dw, dwt)):
        within(a, c, 2 ** -7 * c.double().abs() + 1e-3 * float(c.double().abs().mean()))


# ------------------------------------------------------------------------------------------------ no rows, repeatability, streams, graphs
def test_no_rows():
    for dt in (BF16, F32):
        x = torch.empty(0, 64, device="cuda", dtype=dt, requires_grad=True)
        w, b = rnd(32, 64, seed=1, dtype=dt).requires_grad_(True), rnd(32, seed=2, dtype=dt).requires_grad_(True)
        for y, leaves in ((ops.linear(x, w, b, activation="relu"), (x, w, b)), (ops.gated_linear(x, w, w, b, b), (x, w, b)), (ops.rms_norm(x, rnd(64, seed=3, dtype=dt)), (x,))):
            assert y.shape[0] == 0 and y.dtype == dt
            for t, g in zip(leaves, torch.autograd.grad(y, leaves, torch.empty_like(y))):
                assert g.shape == t.shape and not g.any()
    q, e = ops.rms_norm_fp8(torch.empty(0, 128, device="cuda"))
    assert q.shape == (0, 128) and e.shape == (0,)
    wq, we = ops.quantize_rows_fp8(rnd(32, 128, seed=1))
    assert ops.linear_fp8(q, e, wq, we).shape == (0, 32) and ops.gated_linear_fp8(q, e, wq, we, wq, we).shape == (0, 32)


def step(x, w, wg, wu, wn, dy):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, wg, wu, wn)]
    a, b, c, d, e = leaves
    n, s = ops.rms_norm(a, e, residual=a * 0.5)
    y = ops.linear(ops.gated_linear(n, c, d, activation="silu"), b, activation="gelu", residual=s)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def step_inputs(dt, seed, R=300, K=128, H=352):
    return [rnd(R, K, seed=seed, dtype=dt), rnd(K, H, seed=seed + 1, dtype=dt, scale=H ** -0.5), rnd(H, K, seed=seed + 2, dtype=dt, scale=K ** -0.5),
            rnd(H, K, seed=seed + 3, dtype=dt, scale=K ** -0.5), (1 + 0.1 * rnd(K, seed=seed + 4)).to(dt), rnd(R, K, seed=seed + 5, dtype=dt)]


def test_no_rows_large_weights():
    """The weight gradient of no rows is zeros, also for more weights than a launch has threads / 16."""
    N, K = 20001, 16000
    dw = torch.full((N, K), 7.0, dtype=BF16, device="cuda")
    ops._launch("w3d_linear_bwd", 0, _lib.lib().w3d_linear_bwd, None, None, None, 0, None, None, 0, K, N, _lib.BF16, 0, None, dw.data_ptr(), None, None, 0)
    assert not dw.any()


def test_the_same_bits_every_time():
    for dt in (BF16, F32):
        a = step_inputs(dt, 100, R=1500)
        first = step(*a)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, step(*a)))


def test_two_streams_at_once():
    a, b = step_inputs(BF16, 110, R=2000), step_inputs(BF16, 120, R=700, H=1000)
    want = step(*a), step(*b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (st, args) in enumerate(((s1, a), (s2, b))):
            with torch.cuda.stream(st):
                got[i] = step(*args)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for g, w in zip(got, want) for p, q in zip(g, w))


def test_captured_step_replays():
    """Two captured training steps, replayed in turn with eager work between: every replay equals the eager step on the same inputs."""
    graphs = []
    for dt, seed in ((BF16, 130), (F32, 140)):
        static = step_inputs(dt, seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*static)
        graphs.append((g, static, out, dt))
    for turn in range(4):
        for g, static, out, dt in graphs:
            fresh = step_inputs(dt, 200 + turn)
            for t, f in zip(static, fresh):
                t.copy_(f)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, step(*fresh)))


def test_captured_serving_row_replays():
    wn = rnd(256, seed=1, dtype=BF16)
    wg, wu, wd = (ops.quantize_rows_fp8(rnd(*s, seed=2 + i, scale=0.06)) for i, s in enumerate(((512, 256), (512, 256), (256, 512))))

    def serve(x):
        q, e, s = ops.rms_norm_fp8(x, wn, residual=x)
        h = ops.gated_linear_fp8(q, e, *wg, *wu)
        return ops.linear_fp8(*ops.rms_norm_fp8(h), *wd, residual=s)

    for R in (1, 100):
        x = rnd(R, 256, seed=9, dtype=BF16)
        serve(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = serve(x)
        for turn in range(4):
            x.copy_(rnd(R, 256, seed=300 + turn, dtype=BF16))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, serve(x.clone()))


# ------------------------------------------------------------------------------------------------ together
def test_gradients_against_differences():
    """f32, a head's block: the gradient along random directions against central differences of the definition in 64 bits (step 1e-4: truncation below 1e-7 of curvatures of order one)."""
    x, w, wg, wu, wn, dy = step_inputs(F32, 150, R=70, K=48, H=40)
    grads = step(x, w, wg, wu, wn, dy)[1:]

    def loss(x, w, wg, wu, wn):
        s = 1.5 * x
        n = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-6) * wn
        h = act64(n @ wg.t(), "silu")[0] * (n @ wu.t())
        return ((act64(h @ w.t(), "gelu")[0] + s) * dy.double()).sum()

    args = [t.double() for t in (x, w, wg, wu, wn)]
    for i, g in enumerate(grads):
        for k in range(3):
            v = rnd(*args[i].shape, seed=400 + k).double()
            hi, lo = ([t + (h * v if j == i else 0.0) for j, t in enumerate(args)] for h in (1e-4, -1e-4))
            num = float((loss(*hi) - loss(*lo)) / 2e-4)
            got = float((g.double() * v).sum())
            mag = float((g.double() * v).abs().sum())
            assert abs(num - got) <= 2e-5 * mag + 1e-5, (i, k, num, got)


def test_a_head_in_front_of_the_match():
    """Descriptor-like rows of an odd width -> a learned head -> rows of 128 features -> knn_match_loss, and the gradients of every weight, against the same chain in 64 bits on the same
    neighbours."""
    R, M, K, H, D = 300, 500, 99, 192, 128
    x = rnd(R, K, seed=1, dtype=BF16)
    w0 = rnd(D, K, seed=2, dtype=BF16, scale=K ** -0.5)
    wg, wu = (rnd(H, D, seed=i, dtype=BF16, scale=D ** -0.5) for i in (3, 4))
    wd = rnd(D, H, seed=5, dtype=BF16, scale=H ** -0.5)
    wn, wo = ((1 + 0.1 * rnd(D, seed=i)).to(BF16) for i in (6, 7))
    leaves = [t.requires_grad_(True) for t in (w0, wg, wu, wd, wn, wo)]
    FY = ops.rms_norm(rnd(M, D, seed=8, dtype=BF16)).detach()
    s = ops.linear(x, w0)
    y = ops.linear(ops.gated_linear(ops.rms_norm(s, wn), wg, wu), wd, residual=s)
    FX = ops.rms_norm(y, wo)
    loss, idx = ops.knn_match_loss(FX, FY, k=5, weight=float(R * M))
    grads = torch.autograd.grad(loss, leaves)

    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    a0, ag, au, ad, an, ao = ref
    norm = lambda t, w: t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6) * w  # noqa: E731
    s64 = x.double() @ a0.t()
    n = norm(s64, an)
    y64 = s64 + (act64(n @ ag.t(), "silu")[0] * (n @ au.t())) @ ad.t()
    F64 = norm(y64, ao)
    loss64 = (F64[:, None] - FY.double()[idx.long()]).square().sum()
    want = torch.autograd.grad(loss64, ref)
    # each of the chain's six 16-bit tensors carries 2^-9 relative, and its gradient as many again: norms of the gradients agree to a few per cent at most
    assert abs(float(loss.detach()) - float(loss64.detach())) <= 0.01 * float(loss64.detach())
    for g, r in zip(grads, want):
        assert float((g.double() - r).norm()) <= 12 * 2.0 ** -8 * float(r.norm())


def test_8_bit_rows_into_the_match():
    """rms_norm_fp8 -> raw_knn_match_fp8: rows of equal norm, so the nearest rows are those of the largest cosine."""
    X, Y = rnd(400, 256, seed=1, dtype=BF16), rnd(900, 256, seed=2, dtype=BF16)
    (qx, ex), (qy, ey) = ops.rms_norm_fp8(X), ops.rms_norm_fp8(Y)
    idx, d2 = ops.raw_knn_match_fp8(qx, ex, qy, ey, 8)
    full = torch.cdist(dequant(qx, ex), dequant(qy, ey)).square()
    v, i = full.topk(8, 1, largest=False)
    assert float((d2.double().sort(1).values - v).abs().max()) <= 4e-5 * 3 * 256
    assert float((idx.long().sort(1).values == i.sort(1).values).float().mean()) > 0.98


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    x, w, b = rnd(4, 8), rnd(6, 8), rnd(6)
    bad = [lambda: ops.linear(x, rnd(6, 7)), lambda: ops.linear(x, w, rnd(5)), lambda: ops.linear(x, w, activation="tanh"), lambda: ops.linear(x, w, activation=["relu"]),
           lambda: ops.linear(x, w.half()), lambda: ops.linear(x.double(), w.double()), lambda: ops.linear(x.half(), w.half(), b.to(BF16)), lambda: ops.linear(x, w, residual=rnd(4, 5)),
           lambda: ops.linear(x, w, residual=rnd(1, 6)), lambda: ops.linear(x, w[0]), lambda: ops.linear(x, torch.empty(0, 8, device="cuda")),
           lambda: ops.linear(torch.empty(4, 0, device="cuda"), torch.empty(6, 0, device="cuda")), lambda: ops.linear(x, w.cpu()), lambda: ops.linear(x.cpu(), w.cpu()),
           lambda: ops.gated_linear(x, w, rnd(5, 8)), lambda: ops.gated_linear(x.half(), w.half(), w.half(), b, b.half()), lambda: ops.gated_linear(x, w, w, b, rnd(7)),
           lambda: ops.rms_norm(x, rnd(7)), lambda: ops.rms_norm(x, residual=rnd(4, 7)), lambda: ops.rms_norm(x, residual=rnd(4, 8).half()), lambda: ops.rms_norm(x, eps=-1.0),
           lambda: ops.rms_norm(x, eps=float("nan")), lambda: ops.rms_norm(x.int()), lambda: ops.rms_norm(torch.tensor(1.0, device="cuda")), lambda: ops.rms_norm_fp8(x.view(2, 2, 8)),
           lambda: ops.rms_norm_fp8(x.clone().requires_grad_(True))]
    q, e = ops.quantize_rows_fp8(x)
    wq, we = ops.quantize_rows_fp8(w)
    bad += [lambda: ops.linear_fp8(x, e, wq, we), lambda: ops.linear_fp8(q, e[:3], wq, we), lambda: ops.linear_fp8(q, e.long(), wq, we), lambda: ops.linear_fp8(q, e, wq[:, :4], we),
            lambda: ops.linear_fp8(q, e, wq, we, out_dtype=F32), lambda: ops.linear_fp8(q, e, wq, we, b.half()), lambda: ops.linear_fp8(q, e, wq, we, residual=rnd(4, 6)),
            lambda: ops.linear_fp8(q, e, wq, we, b.clone().requires_grad_(True)), lambda: ops.gated_linear_fp8(q, e, wq, we, wq[:5], we[:5])]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.W3dError):
            f()
            print("not refused:", i)
