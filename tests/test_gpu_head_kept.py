"""The feature-head tests of padding, infinities, streams, graphs and repeatability on 16-bit layers that keep z (their sizes are below the length from which it is kept by default)."""
import pytest

from tests import test_gpu_head as head
from wast3d_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def keep(monkeypatch):
    monkeypatch.setattr(ops, "_KEEP_FROM", 1)


def test_bad_rows():
    head.test_bad_gradient_rows_stay_alone()


@pytest.mark.parametrize("N", [64, 70])
@pytest.mark.parametrize("act", ["relu", "sigmoid"])
def test_an_infinite_row(act, N):
    head.test_an_infinite_row_keeps_its_finite_gradient(act, N)


@pytest.mark.parametrize("R", [40, 700])
def test_subsets(R):
    head.test_any_subset_of_gradients(R, head.BF16)


def test_no_rows():
    head.test_no_rows()


def test_the_same_bits():
    head.test_the_same_bits_every_time()


def test_two_streams():
    head.test_two_streams_at_once()


def test_captured_steps():
    head.test_captured_step_replays()


def test_in_front_of_the_match():
    head.test_a_head_in_front_of_the_match()
