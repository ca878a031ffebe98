"""Drafted-token attention whose units are cut over many CTAs, for head groups that do not
divide the row tile, against a 64-bit implementation."""

import pytest
import torch

from b200_attention import b200_tree_attention, read_device_errors
from paged_reference import attention64, attention_bound
from test_gpu_tree_attention import make, random_tree

pytestmark = pytest.mark.gpu


def worst_case_bound(dtype, v, out, size, grow, head_dim, keys):
    """attention_bound with the errors of the rounded weights all pointing one way.

    With r = 2u the relative error of one rounding and weights p_i (1 + d_i), |d_i| <= r, over
    their own sum, the output is off by at most r (size + |out|) / (1 - r), and its rounding
    adds r |out|: 2u size + 4u |out|, where attention_bound has 2u size + u |out|.  Terms of
    second order are below 8u of the whole.  float16 weights below 2^-14 round to a multiple of
    2^-24 of the largest one's 1: half of that at most for each key, on its value and on the
    sum."""
    u = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}[dtype]
    bound = (1 + 8 * u) * (attention_bound(dtype, out, size, grow, head_dim, keys) + 3 * u * out.abs())
    if dtype == torch.float16:
        bound = bound + keys * 2.0 ** -25 * (float(v[v.isfinite()].abs().max()) + out.abs())
    return bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,group", [(64, 3), (64, 5), (64, 6), (64, 7), (32, 12), (43, 3), (100, 5)])
def test_groups_that_do_not_divide_the_row_tile(dtype, D, T, group):
    """More rows than one half of the row tile takes (128 / group whole tokens), so that the
    two halves' partial results lie side by side."""
    gen = torch.Generator().manual_seed(T + group)
    args = make([2900, 0, 1301], T, 1, group, D, 16, dtype, seed=D + T + group)
    q, k, v, table, lens = args
    mask = torch.stack([random_tree(T, gen) for _ in lens])
    want, size, grow = attention64(*args, mask)
    got = b200_tree_attention(*(t.cuda() for t in args), mask.cuda())
    assert read_device_errors(got.device) == 0
    bound = worst_case_bound(dtype, v, want, size, grow, D, 2900 + T)
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), f"off by {float((err / bound).max()):.2f} bounds"


@pytest.mark.parametrize("T,group", [(64, 3), (64, 7), (32, 12)])
def test_cut_units_give_the_same_bits_again(T, group):
    args = [t.cuda() for t in make([4000, 911], T, 2, group, 64, 32, torch.bfloat16, seed=T)]
    first = b200_tree_attention(*args)
    assert read_device_errors(first.device) == 0 and torch.isfinite(first).all()
    for _ in range(20):
        assert torch.equal(b200_tree_attention(*args), first)
