"""Attention of many rows over the 4-bit paged cache, on the tensor-memory kernel: layouts, units that
share a CTA, numbers of unlike size, graphs and bad numbers."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors, read_device_errors
from test_gpu_cache4 import BF16, DEV, case, check, ints, pools

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


# rows a key head: one tile of 128, and two
@pytest.mark.parametrize("T,group,D", [(24, 2, 128), (24, 2, 40), (40, 4, 128), (60, 3, 64)])
def test_layouts_and_output_in_the_queries_place(T, group, D):
    q, k, v, table, lens, mask, _ = case(3, 2, group, T, D, 16, (0, 40, 333), None, BF16, "tree")
    mask[0, 2] = False
    mask[1, :, 3:] = False
    out = b2.b200_tree_attention(q, k, v, table, lens, mask, None, 0.3, True)
    assert out.shape == (3, T, 2 * group, D)
    check(out.transpose(1, 2), q, k, v, table, lens, mask, None, 0.3)
    assert not out[0, 2].any()
    row = k.shape[-1]
    wide = [torch.full((*x.shape[:3], row + 32), 0xFF, dtype=torch.uint8, device=DEV) for x in (k, v)]
    for w, x in zip(wide, (k, v)):
        w[..., 16:16 + row] = x
    wk, wv = (w[..., 16:16 + row] for w in wide)
    turned = mask.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(b2.b200_tree_attention(q, wk, wv, table, lens, turned, None, 0.3), out.transpose(1, 2))
    place = q.contiguous()
    b2.b200_tree_attention(place, k, v, table, lens, mask, None, 0.3, out=place)
    assert torch.equal(place, out.transpose(1, 2))


@pytest.mark.parametrize("T,group", [(10, 4), (48, 3)])
def test_units_of_one_cta_and_values_that_are_not_finite(T, group):
    """More units than the GPU has SMs, a few tiles each: what a CTA keeps of one unit must not
    reach the next, nor a note of one be lost in the next one's."""
    gen = torch.Generator().manual_seed(T)
    B, kv, D = 48, 8, 64
    lens = torch.randint(0, 300, (B,), generator=gen).tolist()
    q, k, v, table, lens_t, mask, _ = case(B, kv, group, T, D, 32, lens, None, BF16, "tree", seed=2)
    x = torch.randn(2, B, kv, T, D, generator=gen).to(BF16).to(DEV)
    # one drafted token of some sequences has an infinite value in some heads
    at = torch.randint(1, T, (B, kv), generator=gen)
    odd = torch.rand(B, kv, generator=gen) < 0.6
    for b in range(B):
        for h in range(kv):
            if odd[b, h]:
                x[1, b, h, at[b, h], 20] = float("inf")
    b2.b200_cache_append(x[0], x[1], k, v, table, lens_t)
    mask[:, torch.arange(T), torch.arange(T)] = True
    out = b2.b200_tree_attention(q, k, v, table, lens_t, mask)
    for _ in range(2):
        assert torch.equal(b2.b200_tree_attention(q, k, v, table, lens_t, mask).view(torch.int16), out.view(torch.int16))
    check_device_errors(DEV)
    sees = mask.cpu()[torch.arange(B)[:, None], :, at].transpose(1, 2)  # [B, T, kv]: token sees the odd one
    bad = (sees & odd[:, None]).transpose(1, 2).repeat_interleave(group, 1)
    want = torch.zeros(B, kv * group, T, D, dtype=torch.bool)
    want[..., 16:32] = bad[..., None]
    assert torch.equal(torch.isnan(out).cpu(), want)
    # the same without those values, within the bounds
    x[1] = torch.where(torch.isinf(x[1]), 0.0, x[1])
    b2.b200_cache_append(x[0], x[1], k, v, table, lens_t)
    few = slice(0, 6)
    args = (q[few], k, v, table[few], lens_t[few], mask[few])
    clean = b2.b200_tree_attention(q, k, v, table, lens_t, mask)
    check(clean[few], *args)
    assert torch.equal(clean.cpu()[~want], out.cpu()[~want])


def test_values_of_unlike_size():
    """Values from 2^-90 to 2^90 in one context."""
    gen = torch.Generator().manual_seed(3)
    n, D = 200, 128
    k, v = pools(1, 16, 1, 16, D)
    table = torch.arange(16, dtype=torch.int32, device=DEV).view(1, 16)
    kn = torch.randn(1, 1, n, D, generator=gen)
    for sizes in (torch.logspace(-90, 90, n, base=2.0), torch.logspace(90, -90, n, base=2.0)):
        vn = torch.randn(1, 1, n, D, generator=gen) * sizes[None, None, :, None]
        vn[..., 32:64] += 1000
        b2.b200_cache_append(kn.to(DEV), vn.to(DEV), k[0], v[0], table, ints(0))
        for q in (torch.randn(1, 20, 5, D, generator=gen), 1e-30 * torch.randn(1, 20, 5, D, generator=gen),
                  torch.zeros(1, 20, 5, D)):
            args = (q.to(BF16).to(DEV), k[0], v[0], table, ints(n - 5))
            check(b2.b200_tree_attention(*args), *args)


@pytest.mark.parametrize("T,group", [(3, 2), (12, 1), (12, 4)])
def test_small_and_zero_queries_and_scales(T, group):
    """Scores next to nothing: all keys that a row sees have one weight, the others none."""
    q, k, v, table, lens, mask, _ = case(2, 1, group, T, 64, 16, (0, 70), None, BF16, "tree")
    q = q.contiguous()
    for size, scale in ((1e-6, None), (1e-12, 1.0), (0.0, 1e-20), (1.0, 1e-36), (1e-37, 1e-30)):
        args = ((q.float() * size).to(BF16), k, v, table, lens, mask, None, scale)
        check(b2.b200_tree_attention(*args), *args)


def test_keys_of_unlike_size():
    """Keys of 2^-10 to 2^10 times the ordinary ones, small and large beside each other."""
    gen = torch.Generator().manual_seed(4)
    n, D = 300, 64
    k, v = pools(1, 20, 1, 16, D)
    table = torch.arange(20, dtype=torch.int32, device=DEV).view(1, 20)
    sizes = 2.0 ** torch.randint(-10, 11, (n,), generator=gen)
    kn = torch.randn(1, 1, n, D, generator=gen) * sizes[:, None]
    vn = torch.randn(1, 1, n, D, generator=gen)
    b2.b200_cache_append(kn.to(DEV), vn.to(DEV), k[0], v[0], table, ints(0))
    q = (2.0 ** -8 * torch.randn(1, 24, 5, D, generator=gen)).to(BF16).to(DEV)
    args = (q, k[0], v[0], table, ints(n - 5))
    check(b2.b200_tree_attention(*args), *args)


@pytest.mark.parametrize("T,group,D", [(16, 4, 128), (64, 4, 64)])
def test_graphs_and_streams(T, group, D):
    """Two captured calls of different sizes, replayed after each other and beside eager ones."""
    one = case(3, 2, group, T, D, 16, (100, 1500, 7), None, BF16, "tree")
    two = case(5, 1, group, T, D, 32, (900, 0, 31, 64, 2100), None, BF16, "shared", seed=1)
    want = [b2.b200_tree_attention(*a) for a in (one, two)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = b2.b200_tree_attention(*one)
    here = b2.b200_tree_attention(*two)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, want[0]) and torch.equal(here, want[1])
    graphs, outs = [], []
    for a in (one, two):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(b2.b200_tree_attention(*a))
    for a in (one, two):
        a[0].neg_()
    fresh = [b2.b200_tree_attention(*a) for a in (one, two)]
    for i in (0, 1, 1, 0):
        outs[i].zero_()
        graphs[i].replay()
        assert torch.equal(outs[i], fresh[i])


def test_bad_numbers_are_reported_and_skipped():
    q, k, v, table, lens, _, _ = case(3, 1, 4, 12, 64, 16, (20, 40, 3), None, BF16, None)
    good = b2.b200_tree_attention(q, k, v, table, lens)

    def reported(*args):
        clear_device_errors(DEV)
        result = b2.b200_tree_attention(*args)
        torch.cuda.synchronize()
        assert read_device_errors(DEV)
        clear_device_errors(DEV)
        return result

    out = reported(q, k, v, table, ints(20, -1, 3))
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2]) and not out[1].any()
    out = reported(q, k, v, table, lens, None, ints(12, 13, 12))
    assert torch.equal(out[0], good[0]) and not out[1].any()
    missing = table.clone()
    missing[0, 0], missing[1, 0] = 1 << 20, -1
    out = reported(q, k, v, missing, lens)
    assert torch.equal(out[2], good[2]) and torch.isfinite(out).all()
