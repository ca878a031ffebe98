"""Pools whose bytes pass 32 bits, and long page tables: the same results as in a small pool."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors
from test_gpu_cache4 import BF16, DEV, FP16, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


def test_pages_behind_4_gigabytes():
    gen = torch.Generator().manual_seed(1)
    kv, page, D, n = 8, 64, 128, 300
    slots = 5
    many = 110_000  # 4.5 GB a pool
    far = torch.tensor([[many - 1, 3, many - 7, 52_500, many - 2], [many - 3, 0, 104_900, many - 5, 1]],
                       dtype=torch.int32, device=DEV)
    near = torch.arange(10, dtype=torch.int32, device=DEV).view(2, 5)
    shape = (kv, page, D // 2 + 16)
    large = [torch.empty(many, *shape, dtype=torch.uint8, device=DEV) for _ in range(2)]
    small = [torch.empty(10, *shape, dtype=torch.uint8, device=DEV) for _ in range(2)]
    x = torch.randn(2, 2, kv, n + 16, D, generator=gen).to(BF16).to(DEV)
    zero, lens = ints(0, 0), ints(n, n - 100)
    for pools, table in ((large, far), (small, near)):
        b2.b200_cache_append(x[0], x[1], *pools, table, zero)
    for ours, theirs in zip(b2.b200_cache_read(*large, far, zero, n + 16, D), b2.b200_cache_read(*small, near, zero, n + 16, D)):
        assert torch.equal(ours, theirs)
    for T, group, dtype in ((1, 4, BF16), (3, 4, FP16), (16, 1, BF16), (16, 4, BF16), (16, 12, BF16)):
        q = torch.randn(2, kv * group, T, D, generator=gen).to(dtype).to(DEV)
        assert torch.equal(b2.b200_tree_attention(q, *large, far, lens), b2.b200_tree_attention(q, *small, near, lens))
    check_device_errors(DEV)


@pytest.mark.parametrize("T,group", [(1, 2), (12, 3)])
def test_slots_that_are_not_used(T, group):
    """A table for a million keys of which a sequence holds a few hundred."""
    gen = torch.Generator().manual_seed(2)
    D, page = 64, 16
    table = torch.full((3, 65536), -1, dtype=torch.int32)
    for b in range(3):
        table[b, :20] = torch.arange(20 * b, 20 * b + 20)
    table = table.to(DEV)
    k, v = (torch.empty(60, 2, page, 48, dtype=torch.uint8, device=DEV) for _ in range(2))
    x = torch.randn(2, 3, 2, 320, D, generator=gen).to(BF16).to(DEV)
    b2.b200_cache_append(x[0], x[1], k, v, table, ints(0, 0, 0))
    q = torch.randn(3, 2 * group, T, D, generator=gen).to(BF16).to(DEV)
    lens = ints(300, 0, 17)
    out = b2.b200_tree_attention(q, k, v, table, lens)
    short = b2.b200_tree_attention(q, k, v, table[:, :20].contiguous(), lens)
    check_device_errors(DEV)
    assert torch.allclose(out.float(), short.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
