"""Lengths and counts on the device that do not fit: reported, and nothing of the sequence that
has them is touched, while the others are served."""

import pytest
import torch

from b200_attention import b200_cache_accept, b200_cache_append
from b200_attention.fused_attention import DeviceError, clear_device_errors
from test_gpu_paged_cache import filled, i32, model_of

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def reported(c, call):
    """The result of a call that reports a failed bounds check."""
    try:
        result = call()
        torch.cuda.synchronize()
        with pytest.raises(DeviceError, match="bounds"):
            c.free(i32([0]))
    finally:
        clear_device_errors(c.seq_lens.device)
    return result


def rows_of(c, T, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    layers, _, kv, _, D = c.k_pages.shape
    return [torch.randn(layers, c.page_table.shape[0], kv, T, D, generator=gen, device="cuda").to(c.k_pages.dtype)
            for _ in range(2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("negative", [(-1, -2), (-4, -5), (-7, -(1 << 31))])
def test_append_skips_negative_lengths(dtype, negative):
    """More rows than the length lies below zero: none may land on the tokens from 0 on."""
    c = filled(5, 20, 2, 4, 16, 3, 4, dtype)
    assert int(c.reserve(12)) == 0
    m = model_of(c)
    k_new, v_new = rows_of(c, 9, 1)
    reported(c, lambda: b200_cache_append(k_new, v_new, c.k_pages, c.v_pages, c.page_table, i32([*negative, 3])))
    m.lens[2] = 3
    m.append(k_new, v_new, [0, 0, 9])
    m.lens[2] = 0
    m.check(c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [(6, -1, 2), (1 << 30, -(1 << 31), 5), (6, 7, 0)])
def test_append_skips_counts_of_rows_that_were_not_given(dtype, counts):
    c = filled(2, 20, 2, 4, 16, 3, 4, dtype)
    assert int(c.reserve(12)) == 0
    m = model_of(c)
    k_new, v_new = rows_of(c, 5, 2)
    reported(c, lambda: b200_cache_append(k_new, v_new, c.k_pages, c.v_pages, c.page_table, c.seq_lens, i32(counts)))
    m.append(k_new, v_new, [0, 0, counts[2]])
    m.check(c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("paths", [[0, 1, 2, 3], [1, 2, 3, 4]])
def test_accept_does_not_grow_a_sequence_past_its_slots(dtype, paths):
    """The length stays as it is, and no row moves; a sequence may fill its slots exactly."""
    c = filled(2, 20, 2, 4, 16, 4, 4, dtype)
    assert int(c.reserve(16)) == 0
    c.seq_lens.copy_(i32([14, 16, 2, 12 if paths[0] == 0 else 11]))
    m = model_of(c)
    counts = i32([3, 1, 2, 4])
    got = reported(c, lambda: b200_cache_accept(c.k_pages, c.v_pages, c.page_table, c.seq_lens,
                                                i32([paths] * 4), counts))
    want = m.accept([paths] * 4, [0, 0, 2, 4])
    assert got.tolist() == want.tolist()
    m.check(c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)


@pytest.mark.parametrize("length", [-1, 17, (1 << 31) - 1])
def test_fork_does_not_hand_on_a_bad_length(length):
    c = filled(1, 20, 1, 4, 16, 4, 4, torch.bfloat16)
    assert int(c.reserve(6)) == 0
    c.seq_lens.copy_(i32([length, 6, 5, 5]))
    m = model_of(c)
    reported(c, lambda: c.fork(i32([0, 1]), i32([2, 3])))
    m.fork([1], [3])
    m.check(c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.page_refs)
