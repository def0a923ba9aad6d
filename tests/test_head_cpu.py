"""Refusals of the feature-head entry points that need no GPU: error codes before anything touches the device."""
import ctypes as C

import pytest
import torch

from wast3d_amd import _lib, build, ops


@pytest.fixture(scope="module")
def L():
    build.build(verbose=False)
    return _lib.lib()


BUF = C.create_string_buffer(4096)
P = C.c_void_p((C.addressof(BUF) + 255) & ~255)
ARG, WS, UNSUP = -1, -3, -4


def test_rms_norm_arguments(L):
    f = L.w3d_rms_norm_fwd
    assert f(None, None, None, 0, 4, 8, 0, 1e-6, P, None, None, None) == ARG
    assert f(P, None, None, 0, 4, 8, 0, 1e-6, None, None, None, None) == ARG                    # no output
    assert f(P, None, None, 0, 4, 0, 0, 1e-6, P, None, None, None) == ARG
    assert f(P, None, None, 0, -1, 8, 0, 1e-6, P, None, None, None) == ARG
    assert f(P, None, None, 0, 4, 8, 3, 1e-6, P, None, None, None) == ARG                       # rows of 8 bits
    assert f(P, None, P, 2, 4, 8, 1, 1e-6, P, None, None, None) == ARG                          # weight f16 next to bf16
    assert f(P, None, None, 0, 4, 8, 0, -1.0, P, None, None, None) == ARG
    assert f(P, None, None, 0, 4, 8, 0, float("nan"), P, None, None, None) == ARG
    assert f(P, None, None, 0, 4, 8, 0, 1e-6, P, P, None, None) == ARG                          # a sum without a residual
    assert f(None, None, None, 0, 0, 8, 0, 1e-6, None, None, None, None) == 0                   # no rows
    assert L.w3d_rms_norm_fp8(P, None, None, 0, 4, 8, 0, 1e-6, P, None, None, None) == ARG
    assert f(P, None, None, 0, 4, (1 << 30) + 1, 0, 1e-6, P, None, None, None) == UNSUP
    b = L.w3d_rms_norm_bwd
    assert b(P, None, P, 0, P, P, None, 4, 8, 0, None, None, P, 4096, None) == ARG                    # nothing wanted
    assert b(P, None, P, 0, P, None, None, 4, 8, 0, P, P, P, 4096, None) == ARG
    assert b(P, None, P, 0, P, P, None, 4, 8, 0, P, P, P, 16, None) == WS
    assert b(P, None, P, 0, P, P, None, 4, 8, 0, P, P, None, 0, None) == WS
    assert L.w3d_rms_norm_bwd_workspace_bytes(0, 8) == 0 and L.w3d_rms_norm_bwd_workspace_bytes(4, 8) >= 32


def test_linear_arguments(L):
    def f(*a):                                                                                  # z: not kept
        return L.w3d_linear_fwd(*a[:11], None, *a[11:])

    assert f(None, P, None, 0, None, 4, 8, 6, 0, 0, P, None, 0, None) == ARG
    assert f(P, P, None, 0, None, 4, 0, 6, 0, 0, P, None, 0, None) == ARG
    assert f(P, P, None, 0, None, 4, 8, 0, 0, 0, P, None, 0, None) == ARG
    assert f(P, P, None, 0, None, -1, 8, 6, 0, 0, P, None, 0, None) == ARG
    assert f(P, P, None, 0, None, 4, 8, 6, 3, 0, P, None, 0, None) == ARG                       # 8-bit rows have their own entry point
    assert f(P, P, None, 0, None, 4, 8, 6, 0, 5, P, None, 0, None) == ARG                       # activation
    assert f(P, P, P, 1, None, 4, 8, 6, 2, 0, P, None, 0, None) == ARG                          # bias bf16 next to f16
    assert f(P, P, None, 0, None, 4, 1 << 22, 6, 0, 0, P, None, 0, None) == UNSUP               # rows of 16 MB
    assert f(None, None, None, 0, None, 0, 8, 6, 0, 0, None, None, 0, None) == 0                # no rows
    assert L.w3d_linear_workspace_bytes(300, 4096, 64, 1, 0, 0) > 0                                # few tiles, a long contraction: slices
    assert f(P, P, None, 0, None, 300, 4096, 64, 1, 0, P, None, 0, None) == WS
    assert L.w3d_linear_workspace_bytes(1, 4096, 64, 1, 0, 1) == 0
    assert L.w3d_linear_workspace_bytes(300, 64, 64, 1, 0, 1) >= 300 * 128 + 64 * 128 and L.w3d_linear_workspace_bytes(300, 63, 64, 1, 0, 0) >= 300 * 128 + 64 * 128      # aligned copies
    assert f(P, P, None, 0, None, 300, 63, 64, 1, 0, P, None, 0, None) == WS
    assert L.w3d_gated_linear_fwd(P, P, None, None, None, 0, 4, 8, 6, 0, 3, P, None, None, 0, None) == ARG
    assert L.w3d_linear_fwd(P, P, None, 0, None, 4, 8, 6, 1, 2, P, P.value + 4, None, 0, None) == ARG   # z off its 16 bytes
    assert L.w3d_linear_z_stride(515, 0) == 528 and L.w3d_linear_z_stride(515, 1) == 1056 and L.w3d_linear_z_stride(0, 0) == 0
    e = L.w3d_linear_fp8_fwd
    assert e(P, P, P, P, None, 0, None, 4, 8, 6, 0, 0, P, None, 0, None) == ARG                 # f32 output
    assert e(P, None, P, P, None, 0, None, 4, 8, 6, 1, 0, P, None, 0, None) == ARG
    assert L.w3d_gated_linear_fp8_fwd(P, P, P, P, P, None, None, None, 0, 4, 8, 6, 1, 0, P, None, 0, None) == ARG
    def b(*a):
        return L.w3d_linear_bwd(*a[:5], None, *a[5:])

    assert b(P, P, None, 0, P, 4, 8, 6, 0, 0, None, None, None, P, 4096, None) == ARG           # nothing wanted
    assert b(P, P, None, 0, None, 4, 8, 6, 0, 0, P, P, None, P, 4096, None) == ARG
    assert b(P, P, None, 0, P, 400, 8, 6, 1, 2, P, P, None, P, 16, None) == WS
    assert b(P, P, None, 0, P, 400, 8, 6, 0, 2, P, P, None, P, 1 << 20, None) == ARG             # f32: z is needed
    assert L.w3d_linear_bwd(P, P, None, 0, P, P.value + 4, 400, 8, 6, 1, 2, P, P, None, P, 1 << 20, None) == ARG
    assert L.w3d_linear_bwd_workspace_bytes(0, 8, 6, 0, 0, 0, 0, 0) == 0
    assert L.w3d_gated_linear_bwd(P, P, None, None, None, 0, P, None, 4, 8, 6, 0, 3, P, P, P, None, None, P, 4096, None) == ARG


def test_no_cpu_path():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for call in (lambda: ops.rms_norm(x), lambda: ops.rms_norm_fp8(x), lambda: ops.linear(x, w), lambda: ops.gated_linear(x, w, w),
                 lambda: ops.linear_fp8(x.to(torch.uint8), torch.zeros(4, dtype=torch.int32), w.to(torch.uint8), torch.zeros(6, dtype=torch.int32))):
        with pytest.raises(_lib.W3dError):
            call()
