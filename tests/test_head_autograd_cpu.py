"""How the feature-head layers meet torch's transformations (forward-mode AD, tracing), without a GPU: the launch is replaced by one that computes the norm or the product on the host."""
import ctypes as C

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

from wast3d_amd import _lib, ops

R, K, N = 5, 8, 6


def _array(p, *shape):
    return np.ctypeslib.as_array((C.c_float * int(np.prod(shape))).from_address(p)).reshape(shape)


def _norm(*a):
    x = _array(a[0], a[4], a[5])
    _array(a[8], a[4], a[5])[:] = x / np.sqrt((x * x).mean(1, keepdims=True) + a[7])
    return 0


def _linear(*a):
    _array(a[10], a[5], a[7])[:] = _array(a[0], a[5], a[6]) @ _array(a[1], a[7], a[6]).T
    return 0


def _gated(*a):
    g, u = (_array(a[0], a[6], a[7]) @ _array(p, a[8], a[7]).T for p in a[1:3])
    _array(a[11], a[6], a[8])[:] = g / (1 + np.exp(-g)) * u
    return 0


class _Library:
    """Entry points of f32 rows on the host (no bias, no activation but the gated layer's silu); the others do nothing."""

    def __init__(self):
        own = {"w3d_rms_norm_fwd": _norm, "w3d_linear_fwd": _linear, "w3d_gated_linear_fwd": _gated, "w3d_linear_z_stride": lambda n, gated: n * (1 + gated)}
        for name, (res, args) in _lib.SIGNATURES.items():
            if "norm" in name or "linear" in name or "clear" in name:
                setattr(self, name, C.CFUNCTYPE(res, *args)(own.get(name, lambda *a: 0)))


@pytest.fixture()
def host(monkeypatch):
    library = _Library()
    monkeypatch.setattr(ops, "lib", lambda: library)
    monkeypatch.setattr(ops, "_head_rows", lambda what, x: ops._DTYPE_CODES[x.dtype])
    monkeypatch.setattr(ops, "require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "clear_stale_hip_error", lambda: None)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(ops, "_forward_bytes", lambda *a: 0)


def _calls():
    g = torch.Generator().manual_seed(1)
    x, w, v = (torch.randn(s, generator=g) for s in ((R, K), (N, K), (N, K)))
    silu = torch.nn.functional.silu
    return x, [(lambda x: ops.rms_norm(x), lambda x: x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)), (lambda x: ops.linear(x, w), lambda x: x @ w.t()),
               (lambda x: ops.gated_linear(x, w, v), lambda x: silu(x @ w.t()) * (x @ v.t()))]


def _same(a, b):
    assert a.shape == b.shape and float((a - b).abs().max()) <= 2.0 ** -20 * float(b.abs().max() + 1)      # f32 sums of 8 terms, in two orders


def test_the_stand_in_computes(host):
    x, calls = _calls()
    for own, plain in calls:
        _same(own(x), plain(x))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(host, grad, no_grad):
    """There is no forward-mode derivative: a dual argument raises, whether or not it also asks for a gradient; other arguments of an open level are computed."""
    x, calls = _calls()
    with fwAD.dual_level(), torch.set_grad_enabled(not no_grad):
        for own, plain in calls:
            with pytest.raises((NotImplementedError, _lib.W3dError)):
                own(fwAD.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x)))
            _same(own(x), plain(x))


def test_a_dual_weight_bias_or_residual_is_refused(host):
    x, w, b, r = torch.randn(R, K), torch.randn(N, K), torch.randn(N), torch.randn(R, N)
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: ops.linear(x, dual(w)), lambda: ops.linear(x, w, dual(b)), lambda: ops.linear(x, w, b, residual=dual(r)), lambda: ops.rms_norm(x, dual(w[0])),
                  lambda: ops.rms_norm(x, residual=dual(x)), lambda: ops.gated_linear(x, w, dual(w)), lambda: ops.gated_linear(x, w, w, b, dual(b)),
                  lambda: ops.rms_norm_fp8(dual(x)), lambda: ops.rms_norm_fp8(x, dual(w[0])), lambda: ops.rms_norm_fp8(x, residual=dual(x))):
            with pytest.raises((NotImplementedError, _lib.W3dError)):
                f()
        q, e = torch.zeros(R, K, dtype=torch.uint8), torch.full((R,), 127, dtype=torch.int32)
        wq, we = torch.zeros(N, K, dtype=torch.uint8), torch.full((N,), 127, dtype=torch.int32)
        for f in (lambda: ops.linear_fp8(q, e, wq, we, dual(b.bfloat16())), lambda: ops.gated_linear_fp8(q, e, wq, we, wq, we, None, dual(b.bfloat16()))):
            with pytest.raises(_lib.W3dError):
                f()


def test_traced_calls_compute(host):
    """torch.jit.trace records the call itself, not the allocation of its output: the traced function computes on other rows, also where nothing asks for a gradient."""
    x, calls = _calls()
    other = torch.randn(R, K, generator=torch.Generator().manual_seed(2))
    for own, plain in calls:
        traced = torch.jit.trace(own, x, check_trace=False)
        assert any("^_" in str(n) for n in traced.graph.nodes())
        _same(traced(x), plain(x))
        _same(traced(other), plain(other))


def test_8_bit_calls_are_not_traced(host):
    """The 8-bit forms have no function that a trace could record."""
    q, e = torch.zeros(R, K, dtype=torch.uint8), torch.full((R,), 127, dtype=torch.int32)
    wq, we = torch.zeros(N, K, dtype=torch.uint8), torch.full((N,), 127, dtype=torch.int32)
    for f, args in ((lambda x: ops.rms_norm_fp8(x), (torch.randn(R, K),)), (lambda q: ops.linear_fp8(q, e, wq, we), (q,)), (lambda q: ops.gated_linear_fp8(q, e, wq, we, wq, we), (q,))):
        with pytest.raises(_lib.W3dError):
            torch.jit.trace(f, args, check_trace=False)


@pytest.mark.parametrize("grad", [False, True])
def test_symbolic_traces_are_refused(host, grad):
    """make_fx would record the allocation alone, with or without a gradient."""
    x, calls = _calls()
    for own, _ in calls + [(lambda x: ops.rms_norm_fp8(x.detach())[0], None)]:
        with pytest.raises(_lib.W3dError):
            make_fx(own)(x.clone().requires_grad_(grad))


def test_compiled_calls_compute(host):
    """torch.compile breaks its graph at the launch."""
    x, calls = _calls()
    for own, plain in calls:
        torch._dynamo.reset()
        _same(torch.compile(lambda t: own(2 * t) + 1, backend="eager")(x), plain(2 * x) + 1)


def test_nothing_is_kept_for_a_residual_alone(host):
    """A frozen layer on a stream that is trained: the residual's gradient is dy, and neither z nor the operands live until then."""
    x, w, b, dy = torch.randn(R, K), torch.randn(N, K), torch.randn(N), torch.randn(R, N)
    r = torch.randn(R, N, requires_grad=True)
    y = ops.linear(x, w, b, activation="gelu", residual=r)
    assert not [t for t in y.grad_fn.saved_tensors if t is not None]
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)
    for leaf in (x, w, b):                                 # any other gradient: the operands, and z (f32)
        y = ops.linear(*(t.detach().requires_grad_(t is leaf) for t in (x, w, b)), activation="gelu", residual=r)
        assert any(t is not None and t.shape == (R, N) for t in y.grad_fn.saved_tensors)
