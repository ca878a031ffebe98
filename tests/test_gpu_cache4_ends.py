"""Ordinary scores of very small queries and very large keys, over committed and drafted tokens of a
4-bit cache."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors
from test_gpu_cache4 import BF16, DEV, check, ints, pools, tree_masks

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


# rows a key head: few, one tile of 128, two; contexts that end inside a tile, and drafted tokens that
# begin one
@pytest.mark.parametrize("T,group", [(4, 2), (24, 2), (40, 5)])
@pytest.mark.parametrize("committed", [0, 90, 128, 300])
@pytest.mark.parametrize("keys_up,queries_up,scale", [(116, -116, 0.125), (116, -110, 2.0 ** -9),
                                                      (122, -122, 0.125), (120, -109, 2.0 ** -14),
                                                      (60, -60, 0.125), (-60, 60, 0.125), (-110, 110, 0.125)])
def test_queries_and_keys_far_apart(T, group, committed, keys_up, queries_up, scale):
    """Their products, times the scale, are as usual, and so are the bounds."""
    gen = torch.Generator().manual_seed(T + committed)
    D, n = 64, committed + T
    k, v = pools(1, 24, 2, 16, D)
    table = torch.arange(24, dtype=torch.int32, device=DEV).view(1, 24)
    x = torch.randn(2, 1, 2, n, D, generator=gen)
    b2.b200_cache_append((x[0] * 2.0 ** keys_up).to(DEV), x[1].to(DEV), k[0], v[0], table, ints(0))
    q = (2 * torch.randn(1, 2 * group, T, D, generator=gen) * 2.0 ** queries_up).to(BF16).to(DEV)
    args = (q, k[0], v[0], table, ints(committed), tree_masks(1, T, gen).to(DEV), None, scale)
    out = b2.b200_tree_attention(*args)
    check_device_errors(DEV)
    assert torch.isfinite(out).all()
    check(out, *args)
