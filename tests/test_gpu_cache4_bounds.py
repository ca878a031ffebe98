"""Attention of more than 16 rows over the 4-bit cache within the bounds of what its kernel rounds:
keys, values and weights each on their own."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors
from cache4_reference import attention64, decode
from test_gpu_cache4 import BF16, CASES, DEV, FP16, case, ints, pools

GPU = pytest.mark.gpu
W = 2.0 ** -24


def sums(head_dim, keys, grow):
    """Scores (head_dim products and the factors), the exponential, normalising, sums over the keys: as
    for few rows; a weight that is the sum of two bf16 numbers is off by 2^-16 at most."""
    return 2 * ((head_dim + 12) * W * grow + 16 * W) + 2 * keys * W + 2.0 ** -16


def half_step(x):
    """Half a step of bf16 where x lies."""
    return 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -120))) - 8)


def beyond(out, exact, size, grow, head_dim, keys, rounded=0.0):
    """How many times its bound each number is off.  The rounding of the output is half a step, of the
    number or of what was rounded if that lies past a power of two; `rounded`: of operands."""
    off = (sums(head_dim, keys, grow) + rounded) * size
    return ((out.double() - exact).abs() - off) / half_step(exact.abs() + off)


def whole_numbers(T, group, committed, gen):
    """Keys and values that are whole numbers 0 to 15, which codes, fp16 and bf16 hold as they are; two
    drafted tokens a row to see, of one of which the value is 0."""
    D, n = 64, committed + T
    x = torch.randint(0, 16, (2, 1, 1, n, D), generator=gen).float()
    x[..., 0::16], x[..., 1::16] = 0.0, 15.0
    x[1, 0, 0, committed, 2:16] = 0.0
    x[1, 0, 0, committed, 18:32] = 0.0
    mask = torch.eye(T, dtype=torch.bool)
    mask[:, 0] = True
    q = (torch.randn(1, group, T, D, generator=gen) / 16).to(BF16)
    return q, x, mask


def single_weights(q, x, mask, group):
    """The same attention with weights that are one bf16 number each, relative to the row's largest, and
    their sum as it was before the rounding."""
    q, k, v = q.double(), x[0, 0, 0].double(), x[1, 0, 0].double()
    s = torch.where(mask, torch.einsum("hid,jd->hij", q[0], k) * 0.125, -torch.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    return ((w.to(BF16).double() @ v) / w.sum(-1, keepdim=True))[None].to(BF16)


def exact_attention(q, x, mask):
    q, k, v = q.double(), x[0, 0, 0].double(), x[1, 0, 0].double()
    s = torch.where(mask, torch.einsum("hid,jd->hij", q[0], k) * 0.125, -torch.inf)
    p = torch.softmax(s, -1)
    grow = torch.where(mask, torch.einsum("hid,jd->hij", q[0].abs(), k) * 0.125, 0.0).amax(-1, keepdim=True)
    return (p @ v)[None], (p @ v.abs())[None], grow[None]


@pytest.mark.parametrize("T,group", [(24, 2), (40, 5)])
def test_the_bound_tells_weights_of_one_number(T, group):
    q, x, mask = whole_numbers(T, group, 0, torch.Generator().manual_seed(T))
    exact, size, grow = exact_attention(q, x, mask)
    assert (beyond(single_weights(q, x, mask, group), exact, size, grow, 64, T) > 1.05).any()
    assert (beyond(exact.to(BF16), exact, size, grow, 64, T) <= 1).all()


@GPU
@pytest.mark.parametrize("T,group", [(24, 2), (40, 5)])
def test_weights_keep_two_numbers(T, group):
    q, x, mask = whole_numbers(T, group, 0, torch.Generator().manual_seed(T))
    k, v = pools(1, 4, 1, 16, 64)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(1, 4)
    b2.b200_cache_append(x[0].to(DEV), x[1].to(DEV), k[0], v[0], table, ints(0))
    assert torch.equal(decode(v[0], 64, False)[0].reshape(64, 64)[:T], x[1, 0, 0].double())
    out = b2.b200_tree_attention(q.to(DEV), k[0], v[0], table, ints(0), mask.to(DEV), None, 0.125)
    check_device_errors(DEV)
    exact, size, grow = exact_attention(q, x, mask)
    assert (beyond(out.cpu(), exact, size, grow, 64, T) <= 1).all()


@GPU
@pytest.mark.parametrize("B,kv,group,T,D,page,lens,drafts,mask",
                         [c for c in CASES if c[2] * c[3] > 16] + [(1, 2, 4, 30, 128, 64, (5000,), None, "tree")])
def test_many_rows(B, kv, group, T, D, page, lens, drafts, mask):
    """Keys are rounded to fp16 (a score is off by 2^-11 of sum |q k|, a weight by as much, and
    normalising doubles it) and values to bf16, 2^-8.  (More tokens than 64 under a mask take the kernel of
    few rows, which rounds a weight times a step to fp16 instead: less.)"""
    args = case(B, kv, group, T, D, page, lens, drafts, BF16, mask, seed=3)
    q, k, v, table, lens_t, m, d = args
    out = b2.b200_tree_attention(*args)
    check_device_errors(DEV)
    exact, size, grow = attention64(q, decode(k, D, True), decode(v, D, False), table, lens_t, m, d)
    far = beyond(out.cpu(), exact, size, grow, D, table.shape[1] * page, 2 * 2.0 ** -11 * grow + 2.0 ** -8)
    assert (far <= 1).all(), float(far.max())
    clear_device_errors(DEV)


@GPU
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,group", [(6, 2), (6, 1), (24, 2), (40, 5)])
def test_rows_that_see_nothing_are_zero(T, group, dtype):
    """Sequences without committed tokens: exactly the rows whose mask is empty are zero."""
    gen = torch.Generator().manual_seed(T)
    q, k, v, table, lens, mask, _ = case(3, 2, group, T, 128, 16, (0, 0, 0), None, dtype, "tree")
    empty = torch.rand(3, T, generator=gen) < 0.4
    empty[0, 2], empty[1, 0], empty[2, T - 1] = True, True, True
    mask[empty.to(DEV)] = False
    x = 1 + torch.rand(2, 3, 2, T, 128, generator=gen)  # values that do not add up to 0
    b2.b200_cache_append(x[0].to(DEV), x[1].to(DEV), k, v, table, lens)
    out = b2.b200_tree_attention(q.contiguous().fill_(1.0), k, v, table, lens, mask)
    check_device_errors(DEV)
    zero = (out == 0).cpu().transpose(1, 2)  # [B, T, H, D]
    assert zero[empty].all() and not zero[~empty].any()
