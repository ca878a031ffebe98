"""The page operations of the paged cache against a plain Python restatement."""

import pytest
import torch

from b200_attention import (PagedKVCache, b200_cache_accept, b200_cache_append, b200_cache_compact,
                            b200_cache_fork, b200_cache_free, b200_cache_reserve, read_device_errors)
from b200_attention.fused_attention import DeviceError, clear_device_errors
from paged_reference import CacheModel

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def filled(layers, pages, kv, page, D, batch, slots, dtype, seed=0):
    c = PagedKVCache(layers, pages, kv, page, D, batch, slots, dtype=dtype)
    gen = torch.Generator("cuda").manual_seed(seed)
    c.k_pages.copy_(torch.randn(c.k_pages.shape, generator=gen, device="cuda"))
    c.v_pages.copy_(torch.randn(c.v_pages.shape, generator=gen, device="cuda"))
    return c


def model_of(c):
    return CacheModel(c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)


def same(m, c):
    m.check(c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)
    assert read_device_errors(c.seq_lens.device) == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,kv,page,D", [(1, 1, 1, 8), (2, 3, 7, 40), (5, 2, 16, 64), (3, 4, 48, 128)])
def test_a_life_of_a_cache(dtype, layers, kv, page, D):
    """Random steps of every operation, compared after each one."""
    gen = torch.Generator().manual_seed(layers)
    B, slots = 6, 40
    c = filled(layers, 130, kv, page, D, B, slots, dtype)
    m = model_of(c)
    for step in range(14):
        T = int(torch.randint(1, 12, (1,), generator=gen))
        tokens = torch.randint(0, T + 1, (B,), generator=gen).tolist()
        assert int(c.reserve(i32(tokens))) == m.reserve(tokens)
        same(m, c)
        k_new = torch.randn(layers, B, T, kv, D, generator=gen).to(dtype).cuda().transpose(2, 3)
        v_new = torch.randn(layers, B, kv, T, D, generator=gen).to(dtype).cuda()
        b200_cache_append(k_new, v_new, c.k_pages, c.v_pages, c.page_table, c.seq_lens, i32(tokens))
        m.append(k_new, v_new, tokens)
        same(m, c)
        counts = [int(torch.randint(0, n + 1, (1,), generator=gen)) for n in tokens]
        paths = torch.zeros(B, T, dtype=torch.int32)
        for b in range(B):
            paths[b, :counts[b]] = torch.randperm(tokens[b], generator=gen)[:counts[b]].sort()[0]
        lens = m.accept(paths.tolist(), counts)
        before = c.seq_lens.clone()
        got = b200_cache_accept(c.k_pages, c.v_pages, c.page_table, c.seq_lens, paths.cuda(), i32(counts))
        assert torch.equal(c.seq_lens, before)
        c.seq_lens.copy_(got)
        m.lens = lens
        same(m, c)
        pick = torch.randperm(B, generator=gen).tolist()
        if step % 3 == 0:
            c.fork(i32([pick[0], pick[0], pick[1]]), i32(pick[3:6]))
            m.fork([pick[0], pick[0], pick[1]], pick[3:6])
            same(m, c)
        if step % 4 == 2:
            c.free(i32([pick[2], pick[2], pick[4]]))
            m.free([pick[2], pick[2], pick[4]])
            same(m, c)
        if step % 5 == 4:
            assert int(c.compact()) == m.compact()
            same(m, c)


def test_reserve_is_all_or_nothing():
    c = filled(1, 6, 1, 4, 8, 3, 4, torch.bfloat16)
    m = model_of(c)
    assert int(c.reserve(i32([9, 4, 4]))) == m.reserve([9, 4, 4]) == 0
    same(m, c)
    assert int(c.reserve(i32([9, 4, 12]))) == c.NO_PAGES == m.reserve([9, 4, 12])
    same(m, c)
    assert int(c.reserve(17)) == (c.ROW_FULL | 0)
    same(m, c)
    assert int(c.reserve(0)) == 0
    same(m, c)
    c.page_table[1, 0] = 6  # no such page
    before = [t.clone() for t in (c.page_table, c.page_refs, c.k_pages)]
    assert int(c.reserve(i32([0, 4, 4]))) == c.BAD_ENTRY
    for t, u in zip(before, (c.page_table, c.page_refs, c.k_pages)):
        assert torch.equal(t, u)


def test_reserve_of_long_prompts_and_many_sequences():
    """More slots and pages than one round of the planning CTA, and no page left over."""
    c = PagedKVCache(1, 5003 + 1100, 1, 2, 8, 1100, 5003, dtype=torch.bfloat16)
    m = model_of(c)
    tokens = [2 * 5003] + [1] * 1099
    assert int(c.reserve(i32(tokens))) == m.reserve(tokens) == 0
    same(m, c)
    c.free(i32(list(range(0, 1100, 2))))
    m.free(list(range(0, 1100, 2)))
    tokens = [5, 0] * 550
    assert int(c.reserve(i32(tokens))) == m.reserve(tokens) == 0
    same(m, c)
    assert int(c.compact()) == m.compact()
    same(m, c)


def test_writers_of_one_shared_page_each_get_a_copy():
    c = filled(2, 40, 2, 8, 64, 5, 6, torch.float16)
    m = model_of(c)
    for x in (c, m):
        x.reserve(i32([21, 0, 0, 0, 0]) if x is c else [21, 0, 0, 0, 0])
    c.seq_lens[0] = m.lens[0] = 19
    c.fork(i32([0, 0, 0, 0]), i32([1, 2, 3, 4]))
    m.fork([0] * 4, [1, 2, 3, 4])
    same(m, c)
    assert int(c.reserve(6)) == m.reserve([6] * 5) == 0
    same(m, c)
    # whole pages shared: no copy, a new page
    c.seq_lens.fill_(8)
    m.lens[:] = 8
    c.fork(i32([0]), i32([2]))
    m.fork([0], [2])
    assert int(c.reserve(i32([0, 0, 3, 0, 0]))) == m.reserve([0, 0, 3, 0, 0]) == 0
    same(m, c)


def test_strided_pools_and_rows():
    """Token-major pools with keys and values in one tensor, rows out of a fused projection."""
    gen = torch.Generator("cuda").manual_seed(0)
    L, P, kv, page, D, B, T = 3, 20, 2, 16, 64, 2, 20
    both = torch.randn(P, L, 2, page, kv, D, generator=gen, device="cuda").bfloat16()
    k, v = both[:, :, 0].permute(1, 0, 3, 2, 4), both[:, :, 1].permute(1, 0, 3, 2, 4)
    table = torch.full((B, 4), -1, dtype=torch.int32, device="cuda")
    lens, refs = i32([0, 0]), i32([0] * P)
    m = CacheModel(k, v, table, lens, refs)
    assert int(b200_cache_reserve(k, v, table, lens, refs, T)) == m.reserve([T] * B) == 0
    qkv = torch.randn(L, B, T, 3, kv, D, generator=gen, device="cuda").bfloat16()
    k_new, v_new = qkv[:, :, :, 1].transpose(2, 3), qkv[:, :, :, 2].transpose(2, 3)
    b200_cache_append(k_new, v_new, k, v, table, lens)
    m.append(k_new, v_new)
    m.check(k, v, table, lens, refs)
    paths, counts = i32([[2, 5, 19], [0, 1, 2]]), i32([3, 2])
    lens.copy_(b200_cache_accept(k, v, table, lens, paths, counts))
    m.lens = m.accept(paths.tolist(), counts.tolist())
    b200_cache_free(table, lens, refs, i32([0]))
    m.free([0])
    assert int(b200_cache_compact(k, v, table, refs)) == m.compact()
    m.check(k, v, table, lens, refs)


def test_long_paths_move_through_their_own_places():
    """Paths longer than one batch of moves, whose sources are later destinations."""
    c = filled(2, 8, 2, 16, 64, 2, 4, torch.bfloat16)
    m = model_of(c)
    c.reserve(40)
    m.reserve([40, 40])
    paths = [list(range(1, 31)), list(range(0, 30))]
    got = b200_cache_accept(c.k_pages, c.v_pages, c.page_table, c.seq_lens, i32(paths), i32([30, 17]))
    assert got.tolist() == m.accept(paths, [30, 17]).tolist()
    same(m, c)


def test_bad_numbers_on_the_device_are_reported():
    c = filled(1, 8, 1, 4, 8, 3, 2, torch.bfloat16)
    assert int(c.reserve(4)) == 0
    before = [t.clone() for t in (c.k_pages, c.page_table, c.page_refs, c.seq_lens)]
    rows = torch.randn(1, 3, 1, 9, 8, device="cuda").bfloat16()
    small = rows[:, :, :, :1]
    for bad in (lambda: b200_cache_append(rows, rows, c.k_pages, c.v_pages, c.page_table, i32([4, 8, 1 << 29])),
                lambda: b200_cache_append(small, small, c.k_pages, c.v_pages, c.page_table, i32([-1, -5, 1 << 30])),
                lambda: c.fork(i32([0]), i32([0])),
                lambda: c.fork(i32([3]), i32([1])),
                lambda: c.fork(i32([0, 0]), i32([1, 1])),
                lambda: c.free(i32([-1])),
                lambda: b200_cache_accept(c.k_pages, c.v_pages, c.page_table, c.seq_lens,
                                          i32([[-7], [1 << 30], [400]]), i32([1, 1, 1])),
                lambda: b200_cache_accept(c.k_pages, c.v_pages, c.page_table, c.seq_lens,
                                          i32([[0], [0], [0]]), i32([0, 2, -1]))):
        try:
            bad()
            torch.cuda.synchronize()
            with pytest.raises(DeviceError, match="bounds"):
                c.free(i32([0]))
        finally:
            clear_device_errors(c.seq_lens.device)
        for t, u in zip(before, (c.k_pages, c.page_table, c.page_refs, c.seq_lens)):
            assert torch.equal(t, u)


def test_a_step_in_a_graph():
    """Reserve, append, accept and the length update replayed without the host."""
    c = filled(2, 64, 2, 8, 64, 3, 16, torch.bfloat16)
    m = model_of(c)
    k_new = torch.randn(2, 3, 2, 5, 64, device="cuda").bfloat16()
    paths, counts = i32([[0, 2, 4], [1, 2, 3], [0, 0, 0]]), i32([3, 2, 0])
    ops = [t.clone() for t in (c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)]

    def step():
        status = c.reserve(5)
        b200_cache_append(k_new, k_new, c.k_pages, c.v_pages, c.page_table, c.seq_lens)
        c.accept(paths, counts)
        return status

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t, u in zip(ops, (c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)):
        u.copy_(t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        status = step()
    for _ in range(6):
        k_new.normal_()
        graph.replay()
        assert int(status) == m.reserve([5] * 3) == 0
        m.append(k_new, k_new)
        m.lens = m.accept(paths.tolist(), counts.tolist())
        same(m, c)
