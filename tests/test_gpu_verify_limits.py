"""The check of drafted tokens at the ends of its arguments' ranges."""

import pytest
import torch

from b200_attention import clear_device_errors
from test_gpu_verify import DEV, case, check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


@pytest.mark.parametrize("temperature", [1e-3, 1e-12, 1e-300, 50.0, 1e300])
@pytest.mark.parametrize("drafter", [True, False])
def test_temperatures(temperature, drafter):
    check(case(4, 6, 333, "tree", drafter, seed=3), temperature)


def test_temperatures_whose_reciprocal_is_not_finite_are_refused():
    for temperature in (1e-310, 5e-324):
        with pytest.raises(ValueError, match="reciprocal"):
            check(case(4, 6, 333, "tree", True, seed=3), temperature)


def test_equal_largest_logits_share_at_small_temperatures():
    c = case(6, 5, 64, "star", False, seed=4)
    c["logits"] = torch.where(torch.arange(64) % 9 == 2, 3.0, -2.0).expand(6, 5, 64).contiguous()
    for temperature in (1e-300, 1e-5, 0.0):
        check(c, temperature)


@pytest.mark.parametrize("V", [4096, 4097, 16384, 16385, 53248, 53249, 131071])
def test_vocabularies_at_the_borders_of_the_division(V):
    check(case(2, 4, V, "tree", True, seed=5))


def test_a_tree_of_many_nodes():
    check(case(2, 256, 40, "tree", True, seed=6))
    check(case(1, 200, 40, "star", False, seed=7))
