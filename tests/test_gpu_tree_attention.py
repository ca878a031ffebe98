"""Drafted-token attention over a paged cache against a 64-bit implementation."""

import pytest
import torch

from b200_attention import b200_tree_attention, read_device_errors
from b200_attention.fused_attention import DeviceError, clear_device_errors
from paged_reference import attention64, attention_bound

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def random_tree(T, gen):
    m = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        if i:
            m[i] = m[int(torch.randint(max(0, i - 5), i, (1,), generator=gen))]
        m[i, i] = True
    return m


def make(lens, T, kv_heads, group, D, page, dtype, drafts=None, seed=0, fill=float("nan"), spare=3):
    """A cache whose unused rows and pages hold `fill`, and queries."""
    gen = torch.Generator().manual_seed(seed)
    B = len(lens)
    drafts = [T] * B if drafts is None else drafts
    need = [-(-(n + d) // page) for n, d in zip(lens, drafts)]
    pages = sum(need) + spare
    table = torch.full((B, max(1, max(need))), -1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=gen).int(), 0
    k = torch.full((pages, kv_heads, page, D), fill).to(dtype)
    v = k.clone()
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        for t in range(lens[b] + drafts[b]):
            p, r = int(table[b, t // page]), t % page
            k[p, :, r] = torch.randn(kv_heads, D, generator=gen).to(dtype)
            v[p, :, r] = torch.randn(kv_heads, D, generator=gen).to(dtype)
    q = (2 * torch.randn(B, T, kv_heads * group, D, generator=gen)).to(dtype).transpose(1, 2)
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32)


def check(args, mask=None, drafts=None, scale=None, **kw):
    q, k, v, table, lens = args
    d = None if drafts is None else torch.tensor(drafts, dtype=torch.int32)
    want, size, grow = attention64(q, k, v, table, lens, mask, d, scale)
    cuda = [t.cuda() for t in args]
    got = b200_tree_attention(*cuda, None if mask is None else mask.cuda(),
                              None if d is None else d.cuda(), scale, **kw)
    assert read_device_errors(got.device) == 0
    if kw.get("output_bshd"):
        assert got.is_contiguous()
        got = got.transpose(1, 2)
    keys = int((lens + (torch.tensor(drafts) if drafts is not None else q.shape[2])).max())
    bound = attention_bound(q.dtype, want, size, grow, q.shape[3], keys)
    err = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"off by {float((err / bound.clamp(min=1e-300)).max()):.2f} bounds"
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 128])
@pytest.mark.parametrize("T,group", [(1, 1), (1, 8), (3, 4), (17, 1)])
def test_heads_types_and_token_counts(dtype, D, T, group):
    gen = torch.Generator().manual_seed(D + T)
    args = make([0, 1, 37, 150], T, 2, group, D, 16, dtype, seed=T)
    check(args, torch.stack([random_tree(T, gen) for _ in range(4)]))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("page", [1, 7, 8, 16, 24, 48, 64, 100, 128, 256])
def test_page_sizes(dtype, page):
    """Pages that end inside a tile, hold several tiles, and of one row."""
    args = make([5, 127, 128, 300], 9, 1, 3, 64, page, dtype, seed=page)
    check(args, random_tree(9, torch.Generator().manual_seed(page)))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [40, 72, 128])
@pytest.mark.parametrize("T,group", [(17, 1), (8, 4)])
def test_a_wider_table_changes_nothing(dtype, D, T, group):
    """Slots for more than 2048 keys change the kernel for 17 to 32 rows of narrow heads: both are
    within the bound of the same values, so within two of each other."""
    gen = torch.Generator().manual_seed(D)
    q, k, v, table, lens = make([0, 20, 190, 333], T, 2, group, D, 16, dtype, seed=D + T)
    mask = torch.stack([random_tree(T, gen) for _ in range(4)])
    wide = torch.full((4, 130), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    want, size, grow = attention64(q, k, v, table, lens, mask)
    bound = attention_bound(dtype, want, size, grow, D, 333 + T)
    got = [b200_tree_attention(q.cuda(), k.cuda(), v.cuda(), t.cuda(), lens.cuda(), mask.cuda())
           for t in (table, wide)]
    assert read_device_errors(got[0].device) == 0
    assert ((got[0].cpu().double() - got[1].cpu().double()).abs() <= 2 * bound).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [40, 72, 128])
@pytest.mark.parametrize("T,group", [(17, 1), (8, 4), (25, 3)])
def test_the_page_size_changes_nothing(dtype, D, T, group):
    """Odd pages go to the kernel of few rows in several row tiles, pages of 16 to that of
    many rows: both are within the bound of the same values, so within two of each other."""
    gen = torch.Generator().manual_seed(D)
    lens_of = [0, 20, 190, 333]
    q, k, v, table, lens = make(lens_of, T, 2, group, D, 16, dtype, seed=D + T + 1)
    mask = torch.stack([random_tree(T, gen) for _ in range(4)])
    other = make(lens_of, T, 2, group, D, 7, dtype, seed=D + T + 1)
    for b, n in enumerate(lens_of):
        for t in range(n + T):
            here, there = table[b, t // 16], other[3][b, t // 7]
            other[1][there, :, t % 7] = k[here, :, t % 16]
            other[2][there, :, t % 7] = v[here, :, t % 16]
    want, size, grow = attention64(q, k, v, table, lens, mask)
    bound = attention_bound(dtype, want, size, grow, D, 333 + T)
    got = [b200_tree_attention(q.cuda(), *(x.cuda() for x in c), lens.cuda(), mask.cuda())
           for c in ((k, v, table), other[1:4])]
    assert read_device_errors(got[0].device) == 0
    assert ((got[0].cpu().double() - got[1].cpu().double()).abs() <= 2 * bound).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,group,kv_heads", [(33, 1, 2), (16, 4, 1), (31, 3, 1), (64, 2, 1), (65, 4, 1),
                                              (130, 1, 1)])
def test_many_rows(dtype, T, group, kv_heads):
    """Row counts around the row tiles of the kernels, drafts cut short."""
    gen = torch.Generator().manual_seed(T)
    drafts = [T, T - 1, T // 2, 1, 0]
    args = make([70, 0, 129, 33, 12], T, kv_heads, group, 128, 32, dtype, drafts, seed=T)
    got = check(args, torch.stack([random_tree(T, gen) for _ in drafts]), drafts)
    for b, n in enumerate(drafts):
        assert (got[b, :, n:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("lens", [[1], [2047], [4001], [0, 3000, 0, 1, 700], [0], [15, 16, 17, 31, 32, 33]])
@pytest.mark.parametrize("T,group", [(1, 4), (8, 4), (40, 2)])
def test_lengths_and_splits(dtype, lens, T, group):
    """From an empty cache to lengths cut over many CTAs; no mask: a causal chain."""
    check(make(lens, T, 1, group, 64, 16, dtype, seed=len(lens)))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("T", [4, 40])
def test_rows_that_see_nothing_are_zero(dtype, T):
    mask = torch.zeros(2, T, T, dtype=torch.bool)
    mask[1, 1, 0] = True
    got = check(make([0, 0], T, 2, 2, 64, 16, dtype), mask)
    assert (got[0] == 0).all() and (got[1, :, 0] == 0).all() and (got[1, :, 2:] == 0).all()
    assert (got[1, :, 1] != 0).any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,group", [(6, 2), (40, 4), (50, 6)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_hidden_draft_rows_may_hold_anything(dtype, T, group, bad):
    """A drafted token with non-finite keys and values reaches those that see it only."""
    gen = torch.Generator().manual_seed(3)
    lens = [45, 0]
    args = make(lens, T, 1, group, 64, 16, dtype)
    q, k, v, table, _ = args
    mask = torch.stack([random_tree(T, gen) for _ in lens])
    mask[:, :, 3] = False
    mask[:, 3, 3] = True
    want = attention64(*args, mask)[0]
    for b, n in enumerate(lens):
        p, r = int(table[b, (n + 3) // 16]), (n + 3) % 16
        k[p, :, r] = bad
        v[p, :, r, ::3] = bad
    cuda = [t.cuda() for t in args]
    got = b200_tree_attention(*cuda, mask.cuda()).cpu()
    clean = torch.tensor([i for i in range(T) if i != 3])
    assert torch.isfinite(got[:, :, clean]).all()
    assert float((got[:, :, clean].double() - want[:, :, clean]).abs().max()) < 0.1
    assert not torch.isfinite(got[:, :, 3, ::3]).any()


@pytest.mark.parametrize("T,group", [(4, 2), (20, 4), (64, 4)])
def test_infinite_values_of_many_short_sequences(T, group):
    """Several units of one key tile to a CTA, each with an infinite value in its draft."""
    gen = torch.Generator().manual_seed(5)
    lens = [(7 * b) % 50 for b in range(40)]
    args = make(lens, T, 16, group, 64, 32, BF16, seed=6)
    q, k, v, table, _ = args
    mask = torch.stack([random_tree(T, gen) for _ in lens])
    for b, n in enumerate(lens):
        v[int(table[b, (n + 3) // 32]), :, (n + 3) % 32, ::3] = float("inf")
    got = b200_tree_attention(*(t.cuda() for t in args), mask.cuda()).cpu()
    for b in range(len(lens)):
        sees = mask[b, :, 3]
        assert torch.isfinite(got[b][:, ~sees]).all()
        assert (got[b][:, sees][..., ::3] == float("inf")).all()
        rest = torch.arange(64) % 3 != 0
        assert torch.isfinite(got[b][:, sees][..., rest]).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("T,group", [(3, 2), (40, 3)])
def test_strides_and_layouts(dtype, T, group):
    """Token-major pools, keys and values in one tensor, padded rows, both output
    layouts, a table that is part of a wider one, transposed masks."""
    args = make([100, 31, 64], T, 2, group, 64, 16, dtype)
    q, k, v, table, lens = (t.cuda() for t in args)
    gen = torch.Generator().manual_seed(5)
    mask = torch.stack([random_tree(T, gen) for _ in range(3)]).cuda()
    base = check(args, mask.cpu())
    both = torch.stack([k.transpose(1, 2), v.transpose(1, 2)], 1).contiguous()
    kk, vv = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    wide = torch.zeros(3, table.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    padded = torch.zeros(q.shape[:3] + (72,), dtype=dtype, device="cuda")
    padded[..., :64] = q
    flipped = mask.transpose(1, 2).contiguous().transpose(1, 2)
    got = b200_tree_attention(padded[..., :64], kk, vv, wide[:, :table.shape[1]], lens, flipped)
    assert torch.equal(got, base)
    out = torch.empty(3, T, q.shape[1], 64, dtype=dtype, device="cuda")
    got = b200_tree_attention(q, k, v, table, lens, mask, output_bshd=True, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got.transpose(1, 2), base)
    check(args, mask.cpu(), scale=0.3, output_bshd=True)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_same_bits_again_in_a_graph_and_on_a_side_stream(dtype):
    args = [t.cuda() for t in make([900, 3, 411], 5, 2, 4, 128, 16, dtype)]
    first = b200_tree_attention(*args)
    for _ in range(3):
        assert torch.equal(b200_tree_attention(*args), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = b200_tree_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = b200_tree_attention(*args)
    args[0].mul_(0.5)
    graph.replay()
    assert torch.equal(held, b200_tree_attention(*args))


def test_large_pool_offsets():
    """Rows past 2^31 elements of the pool."""
    page, kv, D = 128, 8, 128
    pages = (1 << 31) // (page * kv * D) + 64
    k = torch.zeros(pages, kv, page, D, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    gen = torch.Generator("cuda").manual_seed(1)
    used = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device="cuda")
    for p in used[0].tolist():
        k[p].normal_(generator=gen)
        v[p].normal_(generator=gen)
    q = torch.randn(1, 16, 2, D, generator=gen, device="cuda").to(BF16)
    lens = torch.tensor([350], dtype=torch.int32, device="cuda")
    got = b200_tree_attention(q, k, v, used, lens)
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    pick = used[0].long()
    assert torch.equal(got, b200_tree_attention(q, k[pick], v[pick], near, lens))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("T", [2, 40])
def test_bad_pages_and_lengths_are_reported_and_skipped(dtype, T):
    args = make([40, 60], T, 2, 2, 64, 16, dtype)
    q, k, v, table, lens = (t.cuda() for t in args)
    want, size, grow = attention64(*args)
    bound = attention_bound(dtype, want, size, grow, 64, 60 + T)
    for broken in ("page", "missing", "length", "drafts"):
        t, n = table.clone(), lens.clone()
        drafts = None
        if broken == "page":
            t[0, 1] = k.shape[0]
        elif broken == "missing":
            t[0, 1] = -1
        elif broken == "length":
            n[0] = 1 << 30
        else:
            drafts = torch.tensor([T + 1, T], dtype=torch.int32, device="cuda")
        try:
            got = b200_tree_attention(q, k, v, t, n, None, drafts)
            torch.cuda.synchronize()
            with pytest.raises(DeviceError, match="bounds"):
                b200_tree_attention(q, k, v, table, lens)
        finally:
            clear_device_errors(q.device)
        # the other sequence is unharmed (its keys may be cut differently, so not bit for bit)
        assert ((got[1].cpu().double() - want[1]).abs() <= bound[1]).all(), broken
