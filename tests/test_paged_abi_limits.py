"""Sizes, limits and overlaps that the C entries of the paged cache look at on the host (no GPU
needed: nothing here is launched)."""

import ctypes

import pytest

from b200_attention import _native
from test_paged_abi import INVALID, OK, attn, cache, lib  # noqa: F401 (lib is a fixture)


@pytest.mark.parametrize("batch,slots,page,heads,group,D,tokens,rows", [
    (32, 128, 64, 8, 4, 128, 64, 256),
    (1, 2048, 64, 8, 4, 128, 64, 256),
    (1, 2048, 64, 8, 4, 128, 16, 128),
    (64, 512, 16, 8, 4, 128, 1, 16),
    (5, 512, 7, 16, 1, 64, 30, 32),
])
def test_workspace_is_that_of_the_runs_of_one_gpu(lib, batch, slots, page, heads, group, D, tokens, rows):  # noqa: F811
    """Two partial results of up to 256 rows for each CTA, on 160 SMs at most (two CTAs an SM
    for up to 16 rows), and 8 bytes a unit."""
    row, head = D, page * D
    kw = dict(batch=batch, slots=slots, table_stride=slots, page_size=page, kv_heads=heads, head_dim=D, pages=4096,
              k_stride=(0, heads * head, head, row), v_stride=(0, heads * head, head, row))
    t = attn(cache_kw=kw, heads=heads * group, tokens=tokens,
             q_stride=(heads * group * tokens * D, tokens * D, D), o_stride=(heads * group * tokens * D, tokens * D, D))
    size = lib.b200_tree_attn_workspace_bytes(ctypes.byref(t))
    ctas = 160 * (2 if rows == 16 else 1)
    units = batch * heads * -(-tokens * group // rows)
    assert 0 < size <= 2 * ctas * 4 * rows * (D + 2) + 8 * units + 16


def test_the_table_has_room_for_the_numbering_of_its_slots(lib):  # noqa: F811
    """The planning CTA steps over the slots wanted in rounds of 1024, in 32 bits: the end of
    the last round has to be below 2^31."""
    def check(batch, slots):
        return lib.b200_cache_check(ctypes.byref(cache(batch=batch, slots=slots, table_stride=slots, page_size=1)))

    assert 8192 * 262143 + 1024 < 1 << 31 and check(8192, 262143) == OK
    assert 7282 * 294903 == (1 << 31) - 2 and check(7282, 294903) == INVALID
    assert check(1, 1 << 24) == OK


def test_rows_of_a_page_in_all_layers_are_numbered_in_32_bits(lib):  # noqa: F811
    """Page moves number a page's (layer, keys or values, head) pieces in 32 bits."""
    def check(layers, heads):
        strides = (8 * heads, 8 * heads, 8, 8)
        return lib.b200_cache_check(ctypes.byref(cache(layers=layers, kv_heads=heads, page_size=1, head_dim=8,
                                                       k_stride=strides, v_stride=strides)))

    assert check(1 << 15, (1 << 15) - 1) == OK
    assert check(1 << 15, 1 << 15) == INVALID and check(1 << 15, 1 << 16) == INVALID


@pytest.mark.parametrize("out,code", [
    (0x30000000 + 8, INVALID),    # the lengths
    (0x30000000 - 8, INVALID),
    (0x700 + 8, INVALID),         # the counts
    (0x600 + 60, INVALID),        # the last entries of the paths
    (0x20000000 + 92, INVALID),   # the page table
])
def test_accept_refuses_new_lengths_over_what_it_reads(lib, out, code):  # noqa: F811
    """Blocks of one sequence read while those of another write."""
    p = ctypes.c_void_p
    got = lib.b200_cache_accept(ctypes.byref(cache()), p(0x600), 5, 6, p(0x700), p(out), None)
    assert got == code


def rows_at(q, o, q_stride, o_stride, **kw):
    return attn(q=q, o=o, q_stride=q_stride, o_stride=o_stride, **kw)


# attn(): 3 sequences, 8 heads, 5 tokens, D 64; a token of all heads is 1024 bytes
HEAD_MAJOR, TOKEN_MAJOR = (8 * 5 * 64, 5 * 64, 64), (8 * 5 * 64, 64, 8 * 64)
HALVES = (2 * 8 * 5 * 64, 64, 2 * 8 * 64)  # token-major, as one of two in a tensor
SIZE = 3 * 8 * 5 * 64 * 2


@pytest.mark.parametrize("q,o,qs,os,code", [
    (0x70000000, 0x70000000, HEAD_MAJOR, HEAD_MAJOR, OK),        # in place, element for element
    (0x70000000, 0x70000000, TOKEN_MAJOR, TOKEN_MAJOR, OK),
    (0x70000000, 0x70000000, TOKEN_MAJOR, HEAD_MAJOR, INVALID),  # in place in another order
    (0x70000000, 0x70000000 + 128, HEAD_MAJOR, HEAD_MAJOR, INVALID),
    (0x70000000, 0x70000000 + SIZE - 16, HEAD_MAJOR, HEAD_MAJOR, INVALID),
    (0x70000000, 0x70000000 + SIZE, HEAD_MAJOR, HEAD_MAJOR, OK),
    (0x70000000 + SIZE, 0x70000000, HEAD_MAJOR, HEAD_MAJOR, OK),
    (0x70000000, 0x70000000 + 1024, HALVES, HALVES, OK),         # side by side in one tensor
    (0x70000000 + 1024, 0x70000000, HALVES, HALVES, OK),
    (0x70000000, 0x70000000 + 1008, HALVES, HALVES, INVALID),
    (0x70000000, 0x70000000 + 1040, HALVES, HALVES, INVALID),
    (0x70000000, 0x70000000 + 1024, HALVES, HEAD_MAJOR, INVALID),
    (0x70000000, 0x10000000 + 2048, HEAD_MAJOR, HEAD_MAJOR, INVALID),   # in the keys
    (0x70000000, 0x100000000 - 128, HEAD_MAJOR, HEAD_MAJOR, INVALID),   # into the values
    (0x70000000, 0x20000000 - SIZE + 16, HEAD_MAJOR, HEAD_MAJOR, INVALID),  # into the table
    (0x70000000, 0x30000000 - SIZE + 16, HEAD_MAJOR, HEAD_MAJOR, INVALID),  # into the lengths
    (0x70000000, 0x80000000, HEAD_MAJOR, (0, 5 * 64, 64), INVALID),     # one row for all sequences
])
def test_output_may_not_lie_over_the_inputs(lib, q, o, qs, os, code):  # noqa: F811
    assert lib.b200_tree_attn_check(ctypes.byref(rows_at(q, o, qs, os))) == code


def test_output_may_not_lie_over_the_mask_or_the_draft_lengths(lib):  # noqa: F811
    mask = dict(mask=0x80000000 + 64, mask_stride=(0, 5, 1))
    for kw, code in ((mask, INVALID), (dict(mask, mask=0x80000000 - 25), OK), (dict(mask, mask=0x80000000 - 24), INVALID),
                     (dict(draft_lens=0x80000000 + SIZE), OK), (dict(draft_lens=0x80000000 + SIZE - 4), INVALID)):
        assert lib.b200_tree_attn_check(ctypes.byref(attn(**kw))) == code


def test_output_beside_the_pools_of_one_tensor(lib):  # noqa: F811
    """Keys, values and an output in the same rows of one tensor do not overlap."""
    # a row of 3 x 64 elements: keys, values, output; pages of 16 rows, 4 heads
    kw = dict(k=0x10000000, v=0x10000080, k_stride=(0, 4 * 16 * 192, 16 * 192, 192),
              v_stride=(0, 4 * 16 * 192, 16 * 192, 192))
    strides = (8 * 5 * 192, 5 * 192, 192)
    assert lib.b200_tree_attn_check(ctypes.byref(attn(cache_kw=kw, o=0x10000100, o_stride=strides))) == OK
    assert lib.b200_tree_attn_check(ctypes.byref(attn(cache_kw=kw, o=0x10000080, o_stride=strides))) == INVALID
