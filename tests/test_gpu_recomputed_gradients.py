"""Gradients of 16-bit layers whose z is formed again in the backward pass, at every way that product can be cut (few rows, tiles of each size, sliced contractions), next to the same with z kept."""
import pytest
import torch

from tests.test_gpu_head import BF16, F16, LARGE, SIZES, gated_gradients, linear_gradients
from wast3d_amd import ops

pytestmark = pytest.mark.gpu

# contractions just short of the length from which z is kept by default, sliced; few and odd outputs
SLICED = [(122, 2, 836), (200, 13, 888), (100, 24, 840), (300, 5, 895), (65, 70, 872)]
ACTS = ["relu", "gelu", "silu", "sigmoid"]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("R,N,K", SLICED + [(R, N, K) for R, K, N in SIZES])
def test_gradients(R, N, K, kept, dt, monkeypatch):
    monkeypatch.setattr(ops, "_KEEP_FROM", 1 if kept else 1 << 30)
    linear_gradients(R, K, N, dt, [(i + 1, act) for i, act in enumerate(ACTS)])
    gated_gradients(R, K, N, dt, [(i, act) for i, act in enumerate([None] + ACTS)])


@pytest.mark.parametrize("R,K,N", LARGE)
def test_large_gradients(R, K, N, monkeypatch):
    monkeypatch.setattr(ops, "_KEEP_FROM", 1 << 30)
    linear_gradients(R, K, N, F16, [(2, "silu")])
    gated_gradients(R, K, N, BF16, [(1, "gelu")])


def test_the_default_sizes_slice():
    """The sizes above do cut the recomputing product: its partial tiles are part of the workspace."""
    from wast3d_amd import _lib
    L = _lib.lib()
    for i, (R, N, K) in enumerate(SLICED):
        for gated in (0, 1) if i in (0, 2) else (0,):
            again, kept = (L.w3d_linear_bwd_workspace_bytes(R, K, N, _lib.BF16, 2, gated, k, 0) for k in (0, 1))
            assert again > kept, (R, N, K, gated)
