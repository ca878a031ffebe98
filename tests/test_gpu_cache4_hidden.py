"""Numbers of any finite size in drafted tokens that a row does not see leave the row as it is."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors
from test_gpu_cache4 import BF16, DEV, FP16, case, check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,group,D", [(3, 1, 64), (4, 2, 128), (5, 3, 40), (12, 4, 128), (10, 20, 64)])
@pytest.mark.parametrize("what", ["keys", "values"])
def test_huge_numbers_in_hidden_tokens(T, group, D, dtype, what):
    gen = torch.Generator().manual_seed(T + D)
    lens = (0, 9, 130, 700)
    q, k, v, table, lens_t, _, _ = case(4, 2, group, T, D, 16, lens, None, dtype, None)
    mask = torch.eye(T, dtype=torch.bool).repeat(4, 1, 1)
    mask[:, :, 0] = True     # all see the root, and themselves
    mask[:, T - 1, 1] = True  # the last one sees the huge one too
    mask = mask.to(DEV)
    x = torch.randn(2, 4, 2, T, D, generator=gen).to(BF16).to(DEV)
    huge = x.clone()
    huge[0 if what == "keys" else 1, :, :, 1] *= 2.0 ** 100
    others = [i for i in range(T) if i not in (1, T - 1)]
    outs = []
    for y in (x, huge):
        b2.b200_cache_append(y[0], y[1], k, v, table, lens_t)
        outs.append(b2.b200_tree_attention(q, k, v, table, lens_t, mask))
        check_device_errors(DEV)
        if y is x:
            check(outs[0], q, k, v, table, lens_t, mask)
    first, second = (o.cpu()[:, :, others] for o in outs)
    # The rows that do not see the token: within the bounds of each result, so off by twice that; here
    # simply by the rounding of the output and of the weights, 2^-8 and three of 2^-8 (bf16).
    assert torch.isfinite(second).all()
    bound = 2 * 2.0 ** -7 * (first.float().abs().amax(-1, keepdim=True) + 0.05)
    assert (first.float() - second.float()).abs().le(bound).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,group,D", [(4, 2, 64), (4, 4, 128), (9, 8, 128), (40, 5, 64)])
def test_a_query_that_is_not_finite_stays_in_its_row(T, group, D, dtype):
    q, k, v, table, lens, mask, _ = case(2, 2, group, T, D, 16, (50, 400), None, dtype, "tree")
    q = q.contiguous()
    want = b2.b200_tree_attention(q, k, v, table, lens, mask)
    odd = q.clone()
    odd[0, 1, 1, 3] = float("nan")
    odd[1, 0, 2, 0] = float("inf")
    out = b2.b200_tree_attention(odd, k, v, table, lens, mask)
    check_device_errors(DEV)
    assert torch.isnan(out[0, 1, 1]).all() and torch.isnan(out[1, 0, 2]).all()
    out[0, 1, 1], out[1, 0, 2] = want[0, 1, 1], want[1, 0, 2]
    if group * T <= 16:  # the order of a row's sums may follow its neighbours' steps
        assert torch.allclose(out.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    else:
        assert torch.allclose(out.float(), want.float(), rtol=2.0 ** -6, atol=2.0 ** -8)


@pytest.mark.parametrize("T,group", [(4, 2), (24, 2)])
def test_queries_and_keys_near_the_ends_of_the_type(T, group):
    """Large queries with small keys and the other way round: ordinary scores."""
    gen = torch.Generator().manual_seed(9)
    for up in (100, -100, 110):
        q, k, v, table, lens, mask, _ = case(2, 2, group, T, 64, 16, (0, 90), None, BF16, "tree")
        x = torch.randn(2, 2, 2, T, 64, generator=gen)
        lens = torch.zeros_like(lens)  # only these keys
        b2.b200_cache_append((x[0] * 2.0 ** -up).to(DEV), x[1].to(DEV), k, v, table, lens)
        args = ((q.float() * 2.0 ** up).to(BF16).contiguous(), k, v, table, lens, mask)
        check(b2.b200_tree_attention(*args), *args)
        check_device_errors(DEV)
