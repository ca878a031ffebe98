"""The paged cache held in 4 bits on the GPU: append, read back, page operations, and attention for
drafted tokens over it, against their definitions in 64 bits."""

import numpy as np
import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors, read_device_errors
from cache4_reference import attention64, attention_bound, decode, padded, quantise

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


def table_of(pages_of, slots, gen, spare=3):
    total = sum(pages_of) + spare
    order = torch.randperm(total, generator=gen)[:sum(pages_of)].int()
    table, at = torch.full((len(pages_of), slots), -1, dtype=torch.int32), 0
    for b, n in enumerate(pages_of):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEV), total


def pools(layers, total, kv, page, head_dim):
    shape = (layers, total, kv, page, padded(head_dim) // 2 + 16)
    return (torch.full(shape, 0xA5, dtype=torch.uint8, device=DEV),
            torch.full(shape, 0x5A, dtype=torch.uint8, device=DEV))


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("layers,kv,head_dim,page,lens,tokens,counts", [
    (1, 1, 8, 16, (0,), 1, None),
    (2, 3, 40, 16, (5, 0, 31), 19, (19, 0, 7)),
    (1, 4, 64, 48, (0, 47, 300), 70, (1, 70, 69)),
    (3, 2, 72, 1, (3, 0), 5, None),
    (1, 8, 96, 64, (63, 64), 130, (130, 128)),
    (2, 2, 128, 32, (0, 1, 31, 1000), 33, None),
])
def test_append_and_read(dtype, layers, kv, head_dim, page, lens, tokens, counts):
    gen = torch.Generator().manual_seed(head_dim + tokens)
    B = len(lens)
    given = [tokens] * B if counts is None else list(counts)
    table, total = table_of([-(-(n + c) // page) for n, c in zip(lens, given)],
                            -(-(max(lens) + tokens) // page) + 1, gen)
    k, v = pools(layers, total, kv, page, head_dim)
    shape = (layers, B, tokens, kv, head_dim)
    offset = 3 * torch.randn(1, 1, 1, kv, head_dim, generator=gen)
    kn = (torch.randn(shape, generator=gen) + offset).to(dtype).transpose(2, 3)
    vn = (torch.randn(shape, generator=gen) * torch.logspace(-6, 4, tokens)[:, None, None]).to(dtype).transpose(2, 3)
    before = k.clone(), v.clone()
    counts_t = None if counts is None else ints(*counts)
    b2.b200_cache_append(kn.to(DEV), vn.to(DEV), k, v, table, ints(*lens), counts_t)
    rk, rv = b2.b200_cache_read(k, v, table, ints(*lens), tokens, head_dim, FP32, counts_t)
    tk, tv = b2.b200_cache_read(k, v, table, ints(*lens), tokens, head_dim, dtype, counts_t)
    check_device_errors(DEV)
    touched = torch.zeros(total, page, dtype=torch.bool)
    dk, dv = decode(k, head_dim, True)[0], decode(v, head_dim, False)[0]
    for b in range(B):
        for j in range(tokens):
            if j >= given[b]:
                assert not rk[:, b, :, j].any() and not rv[:, b, :, j].any()
                continue
            at = lens[b] + j
            touched[table[b, at // page], at % page] = True
    for new, read, typed, pool, rows in ((kn, rk, tk, k, dk), (vn, rv, tv, v, dv)):
        want, step = quantise(new)
        for b in range(B):
            n = given[b]
            got = read[:, b, :, :n].cpu().double()
            # the very codes, steps and lows of the definition; the sum is rounded to fp32 once
            torch.testing.assert_close(got, want[:, b, :, :n], rtol=2.0 ** -24, atol=0)
            assert (got - new[:, b, :, :n].double()).abs().le(step[:, b, :, :n] * 0.5 * (1 + 2.0 ** -20) + 2.0 ** -24 * got.abs()).all()
            assert torch.equal(typed[:, b, :, :n], read[:, b, :, :n].to(dtype))
            for j in range(n):
                at = lens[b] + j
                torch.testing.assert_close(rows[:, table[b, at // page].long(), :, at % page],
                                           want[:, b, :, j], rtol=1e-12, atol=0)
    for pool, old in zip((k, v), before):  # rows that were not given are as they were
        same = (pool == old).all(-1).all(2).all(0).cpu()
        assert same[~touched].all()


def test_append_of_groups_that_are_constant_tiny_huge_or_not_finite():
    D, each = 64, 16
    x = torch.zeros(1, 1, 10, D)
    x[0, 0, 1] = 3.0                                # constant: exact
    x[0, 0, 2] = 1.0 + 2.0 ** -12                   # constant, not a bf16 number
    x[0, 0, 3, :each] = torch.linspace(0, 1e-37, each)
    x[0, 0, 4, each:2 * each] = float("inf")
    x[0, 0, 5, 0], x[0, 0, 6, 2 * each] = float("nan"), float("-inf")
    x[0, 0, 7, :each] = torch.linspace(-3e38, 3e38, each)   # the range overflows
    x[0, 0, 8, :each] = torch.linspace(-1e38, 1e38, each)
    x[0, 0, 9] = -torch.arange(D).float()
    k, v = pools(1, 1, 1, 16, D)
    table, zero = ints(0).view(1, 1), ints(0)
    b2.b200_cache_append(x.to(DEV), x.to(DEV), k[0], v[0], table, zero)
    check_device_errors(DEV)
    for got in b2.b200_cache_read(k[0], v[0], table, zero, 10, D, FP32):
        got = got.cpu().double()
        want, _ = quantise(x)
        want[0, 0, 7, :each] = float("nan")
        torch.testing.assert_close(got, want, rtol=2.0 ** -24, atol=0, equal_nan=True)
        assert torch.equal(got[0, 0, 1], x[0, 0, 1].double())


def test_ties_go_to_even():
    """Numbers halfway between two codes, exactly: low 0, step 1."""
    x = torch.tensor([0.0, 15.0] + [c + 0.5 for c in range(14)]).repeat(4)[None, None, None]
    k, v = pools(1, 1, 1, 16, 64)
    table, zero = ints(0).view(1, 1), ints(0)
    for dtype in (BF16, FP16, FP32):
        b2.b200_cache_append(x.to(dtype).to(DEV), x.to(dtype).to(DEV), k[0], v[0], table, zero)
        got = b2.b200_cache_read(k[0], v[0], table, zero, 1, 64, FP32)[0].cpu()
        assert torch.equal(got, torch.tensor(np.rint(x.numpy())))


def test_page_operations_move_4_bit_rows():
    """reserve, append, fork with copy on write, accept, free and compact over 4-bit pools."""
    gen = torch.Generator().manual_seed(5)
    cache = b2.PagedKVCache(2, 12, 2, 16, 40, 3, 4, bits=4)
    assert cache.k_pages.dtype == torch.uint8 and cache.k_pages.shape[-1] == 48
    assert int(cache.reserve(ints(20, 0, 9))) == 0
    x = torch.randn(2, 2, 3, 2, 20, 40, generator=gen).to(BF16).to(DEV)
    for layer in range(2):
        cache.append(layer, x[0, layer], x[1, layer], ints(20, 0, 9))
    cache.accept(torch.arange(20, dtype=torch.int32, device=DEV).expand(3, 20).contiguous(), ints(20, 0, 9))
    cache.fork(ints(0), ints(1))
    assert int(cache.reserve(ints(0, 5, 0))) == 0  # copies the four rows of the shared page
    y = torch.randn(2, 2, 3, 2, 5, 40, generator=gen).to(BF16).to(DEV)
    for layer in range(2):
        cache.append(layer, y[0, layer], y[1, layer], ints(0, 5, 0))
    cache.accept(ints(0, 0, 0, 0, 2, 4, 0, 0, 0).view(3, 3), ints(0, 3, 0))
    cache.free(ints(2))
    live = int(cache.compact())
    check_device_errors(DEV)
    assert live == 3 and cache.seq_lens.tolist() == [20, 23, 0]
    for layer in range(2):
        kept = [torch.cat([x[i, layer, :1], torch.zeros_like(x[i, layer, :1])]) for i in range(2)]
        for i, got in enumerate(cache.read(layer, ints(0, 0, 0), 23, ints(20, 23, 0))):
            want0 = quantise(x[i, layer, 0])[0]
            torch.testing.assert_close(got[0, :, :20].cpu(), want0.to(BF16), rtol=0, atol=0)
            torch.testing.assert_close(got[1, :, :20].cpu(), want0.to(BF16), rtol=0, atol=0)
            want1 = quantise(y[i, layer, 1])[0][:, [0, 2, 4]]
            torch.testing.assert_close(got[1, :, 20:].cpu(), want1.to(BF16), rtol=0, atol=0)
            assert not got[2].any()


# ------------------------------------------------------------------- attention
def random_rows(shape, head_dim, gen, keys):
    """A pool filled by append, one token a page row, from normal numbers with an offset."""
    total, kv, page = shape
    k, v = pools(1, total, kv, page, head_dim)
    table = torch.arange(total, dtype=torch.int32, device=DEV).view(1, total)
    x = torch.randn(1, kv, total * page, head_dim, generator=gen)
    off = torch.randn(1, kv, 1, head_dim, generator=gen)
    b2.b200_cache_append((x + off).to(BF16).to(DEV), x.roll(1, 2).to(BF16).to(DEV), k[0], v[0], table, ints(0))
    return k[0], v[0]


def tree_masks(B, T, gen):
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            if i:
                mask[b, i] = mask[b, int(torch.randint(max(0, i - 5), i, (1,), generator=gen))]
            mask[b, i, i] = True
    return mask


def case(B, kv, group, T, D, page, lens, drafts, dtype, mask, seed=0):
    gen = torch.Generator().manual_seed(1000 * seed + 7 * T + D)
    n = [T] * B if drafts is None else drafts
    table, total = table_of([-(-(a + c) // page) for a, c in zip(lens, n)],
                            max(1, -(-(max(lens) + T) // page)), gen)
    k, v = random_rows((total, kv, page), D, gen, None)
    q = (2 * torch.randn(B, T, kv * group, D, generator=gen)).to(dtype).to(DEV).transpose(1, 2)
    m = None if mask is None else (tree_masks(1, T, gen)[0] if mask == "shared" else tree_masks(B, T, gen))
    return q, k, v, table, ints(*lens), None if m is None else m.to(DEV), None if drafts is None else ints(*drafts)


def check(out, q, k, v, table, lens, mask=None, drafts=None, scale=None):
    D = q.shape[-1]
    want, size, grow = attention64(q, decode(k, D, True), decode(v, D, False), table, lens, mask, drafts, scale)
    err = (out.cpu().double() - want).abs()
    bound = attention_bound(q.dtype, want, size, grow, D, table.shape[1] * k.shape[2],
                            q.shape[2] * q.shape[1] // k.shape[1])
    assert (err <= bound).all(), f"off by {float((err / bound.clamp(min=1e-30)).max()):.2f} of the bound"


CASES = [
    # B, kv, group, T, D, page, lens, drafts, mask
    (1, 1, 1, 1, 64, 16, (0,), None, None),
    (1, 2, 1, 1, 128, 16, (1,), None, None),
    (3, 2, 4, 1, 128, 16, (0, 15, 700), None, None),
    (4, 1, 8, 1, 64, 32, (63, 64, 65, 0), (1, 1, 1, 0), None),
    (2, 3, 3, 5, 40, 16, (33, 257), (5, 2), "tree"),
    (3, 4, 1, 7, 64, 48, (601, 0, 1003), (7, 4, 0), "tree"),
    (2, 2, 2, 9, 96, 64, (128, 511), None, "shared"),
    (1, 1, 4, 16, 128, 64, (2001,), None, "tree"),
    (2, 2, 5, 13, 128, 1, (5, 70), (13, 12), None),
    (2, 1, 4, 33, 72, 24, (90, 400), (33, 20), "tree"),
    (1, 2, 3, 70, 64, 16, (130,), None, "tree"),
    # more than 16 rows: whole tokens to a row tile, one and two tiles of rows, small and large boxes
    (2, 2, 4, 8, 128, 16, (0, 300), None, "tree"),
    (3, 1, 1, 40, 64, 48, (127, 128, 5), (40, 0, 17), "tree"),
    (1, 2, 3, 64, 96, 64, (777,), None, "shared"),
    (2, 1, 5, 64, 128, 1, (40, 129), (64, 33), "tree"),
    (1, 1, 2, 150, 128, 128, (260,), None, None),
    (2, 1, 1, 300, 40, 32, (3, 0), (300, 1), None),
    (1, 1, 100, 3, 64, 32, (500,), None, "tree"),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,kv,group,T,D,page,lens,drafts,mask", CASES)
def test_attention(B, kv, group, T, D, page, lens, drafts, mask, dtype):
    args = case(B, kv, group, T, D, page, lens, drafts, dtype, mask)
    out = b2.b200_tree_attention(*args)
    check_device_errors(DEV)
    check(out, *args)


def test_long_context_split_over_the_gpu():
    args = case(1, 2, 2, 3, 128, 64, (20011,), None, BF16, "tree")
    check(b2.b200_tree_attention(*args), *args)
    args = case(1, 1, 1, 1, 64, 16, (9001,), None, FP16, None)
    check(b2.b200_tree_attention(*args), *args)
    for T, D in ((10, 128), (40, 64)):
        args = case(1, 1, 4, T, D, 64, (9001,), None, BF16, "tree")
        check(b2.b200_tree_attention(*args), *args)


def test_rows_that_see_nothing_and_layouts():
    q, k, v, table, lens, mask, _ = case(2, 2, 2, 6, 128, 16, (0, 40), None, BF16, "tree")
    mask[0, 2] = False
    mask[0, :, 3:] = False
    out = b2.b200_tree_attention(q, k, v, table, lens, mask, None, 0.3, True)
    assert out.shape == (2, 6, 4, 128)
    check(out.transpose(1, 2), q, k, v, table, lens, mask, None, 0.3)
    assert not out[0, 2].any() and not out[0, 3:].any() or mask[0, 3:].any()
    # pools with room between their rows, a mask read against its order, output in the queries' place
    wide = [torch.zeros(*x.shape[:3], 112, dtype=torch.uint8, device=DEV) for x in (k, v)]
    for w, x in zip(wide, (k, v)):
        w[..., 16:96] = x
    wk, wv = (w[..., 16:96] for w in wide)
    turned = mask.transpose(1, 2).contiguous().transpose(1, 2)
    again = b2.b200_tree_attention(q, wk, wv, table, lens, turned, None, 0.3)
    assert torch.equal(again, out.transpose(1, 2))
    place = q.contiguous()
    b2.b200_tree_attention(place, k, v, table, lens, mask, None, 0.3, out=place)
    assert torch.equal(place, again)


def test_nan_in_hidden_and_in_seen_rows():
    """Groups that are NaN reach the rows that see them, and no other."""
    for T, group in ((6, 1), (6, 2), (6, 4), (6, 48)):
        q, k, v, table, lens, _, _ = case(2, 1, group, T, 64, 16, (30, 0), None, BF16, None)
        nan = torch.full((2, 1, T, 64), float("nan"), dtype=BF16, device=DEV)
        x = torch.randn(2, 1, T, 64, dtype=BF16, device=DEV)
        vn = x.clone()
        vn[:, :, 2, 16:32] = float("inf")  # values of drafted token 2, one group
        kn = x.clone()
        kn[:, :, 4] = nan[:, :, 4]         # keys of drafted token 4
        b2.b200_cache_append(kn, vn, k, v, table, lens)
        mask = torch.eye(T, dtype=torch.bool, device=DEV)
        mask[5, 2] = True
        out = b2.b200_tree_attention(q, k, v, table, lens, mask).cpu().float()
        check_device_errors(DEV)
        bad = torch.zeros(T, 64, dtype=torch.bool)
        bad[2, 16:32] = bad[5, 16:32] = True
        bad[4] = True
        assert torch.equal(torch.isnan(out), bad.expand(out.shape))
    # behind the last drafted token anything may lie
    q, k, v, table, lens, _, _ = case(2, 1, 2, 4, 128, 16, (3, 17), (4, 2), BF16, None)
    clean = b2.b200_tree_attention(q, k, v, table, lens, None, ints(4, 2))
    for pool in (k, v):
        for b, n in ((0, 7), (1, 19)):
            pool[table[b, n // 16].long(), :, n % 16:] = 0xFF
    assert torch.equal(b2.b200_tree_attention(q, k, v, table, lens, None, ints(4, 2)), clean)


def test_steps_and_lows_of_unlike_size():
    """Steps from 2^-90 to 2^90 in one context: the products' common factor follows the largest."""
    gen = torch.Generator().manual_seed(3)
    n, D = 200, 128
    k, v = pools(1, 16, 1, 16, D)
    table = torch.arange(16, dtype=torch.int32, device=DEV).view(1, 16)
    kn = torch.randn(1, 1, n, D, generator=gen)
    for sizes in (torch.logspace(-90, 90, n, base=2.0), torch.logspace(90, -90, n, base=2.0)):
        vn = torch.randn(1, 1, n, D, generator=gen) * sizes[None, None, :, None]
        vn[..., 32:64] += 1000
        b2.b200_cache_append(kn.to(DEV), vn.to(DEV), k[0], v[0], table, ints(0))
        for q in (torch.randn(1, 2, 1, D, generator=gen).to(BF16).to(DEV),
                  (1e-30 * torch.randn(1, 2, 1, D, generator=gen)).to(BF16).to(DEV),
                  torch.zeros(1, 2, 1, D, dtype=BF16, device=DEV)):
            args = (q, k[0], v[0], table, ints(n - 1))
            check(b2.b200_tree_attention(*args), *args)


def test_graph_streams_and_same_results():
    args = case(3, 2, 4, 4, 128, 16, (100, 1500, 7), None, BF16, "tree")
    want = b2.b200_tree_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = b2.b200_tree_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b2.b200_tree_attention(*args)
    args[0].neg_()
    graph.replay()
    assert torch.equal(out, b2.b200_tree_attention(*args))
    for _ in range(3):
        assert torch.equal(b2.b200_tree_attention(*args), out)


def test_bad_numbers_are_reported_and_skipped():
    q, k, v, table, lens, _, _ = case(3, 1, 1, 2, 64, 16, (20, 40, 3), None, BF16, None)
    good = b2.b200_tree_attention(q, k, v, table, lens)
    x = torch.randn(3, 1, 2, 64, dtype=BF16, device=DEV)
    saved = k.clone()

    def reported(call):
        clear_device_errors(DEV)
        result = call()
        torch.cuda.synchronize()
        assert read_device_errors(DEV)
        clear_device_errors(DEV)
        return result

    bad_lens = ints(20, -1, 3)
    out = reported(lambda: b2.b200_tree_attention(q, k, v, table, bad_lens))
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2]) and not out[1].any()
    out = reported(lambda: b2.b200_tree_attention(q, k, v, table, lens, None, ints(2, 3, 2)))
    assert not out[1].any()
    missing = table.clone()
    missing[0, 0], missing[1, 0] = 1 << 20, -1
    out = reported(lambda: b2.b200_tree_attention(q, k, v, missing, lens))
    assert torch.equal(out[2], good[2])
    reported(lambda: b2.b200_cache_append(x, x, k, v, missing, ints(0, 0, 1 << 30)))
    assert torch.equal(k, saved)
    reported(lambda: b2.b200_cache_append(x, x, k, v, table, lens, ints(-1, 3, 0)))
    assert torch.equal(k, saved)
    rk, _ = reported(lambda: b2.b200_cache_read(k, v, missing, ints(0, 0, 0), 3, 64))
    assert not rk[:2].any() and rk[2].any()
    assert not reported(lambda: b2.b200_cache_read(k, v, table, ints(-5, 0, 0), 3, 64))[0][0].any()
