"""A copy of coded rows that never comes: the attention kernel of many rows over a 4-bit cache reports
the wait that ran out and ends by itself, whatever each of its warps has seen of it."""

import ctypes
import time

import pytest
import torch

import b200_attention as b2
from b200_attention import _native, check_device_errors, clear_device_errors, read_device_errors
from b200_attention.fused_attention import device_error_word
from test_gpu_cache4 import BF16, DEV, case, check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


def params_of(q, k, v, table, lens, out, word):
    p = _native.TreeAttnParams()
    c = p.cache
    c.k, c.v, c.page_table, c.seq_lens = k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr()
    c.layers, c.pages, c.kv_heads, c.page_size, c.head_dim = 1, *k.shape[:3], k.shape[3] // 2
    c.k_stride[:], c.v_stride[:] = ([0] + [x // 2 for x in t.stride()[:3]] for t in (k, v))
    c.batch, c.slots, c.table_stride = *table.shape, table.stride(0)
    c.dtype, c.error_word = _native.DTYPE_BF16, word
    p.q, p.o, p.heads, p.tokens, p.scale = q.data_ptr(), out.data_ptr(), q.shape[1], q.shape[2], 0.125
    p.q_stride[:], p.o_stride[:] = q.stride()[:3], out.stride()[:3]
    return p


# One row tile of 128 rows, whose two groups of warps meet at each segment's end, and one of 256; few
# units, each over several CTAs, and many short ones, several segments to a CTA.
@pytest.mark.parametrize("T,group", [(10, 4), (60, 4)])
@pytest.mark.parametrize("B,kv,lens,skipped", [(1, 2, [9000], 0), (40, 8, [130] * 40, 2), (24, 8, [300] * 24, 3)])
def test_a_copy_that_never_comes(T, group, B, kv, lens, skipped):
    args = case(B, kv, group, T, 128, 32, lens, None, BF16, None)
    q, k, v, table, lens_t = args[:5]
    want = b2.b200_tree_attention(*args)
    check_device_errors(DEV)
    lib = _native.load_library()
    q = q.contiguous()
    out = torch.empty_like(q)
    word = device_error_word(DEV).data_ptr()
    p = params_of(q, k, v, table, lens_t, out, word)
    size = lib.b200_cache4_attn_workspace_bytes(ctypes.byref(p), 128, _native.DTYPE_BF16)
    assert size > 0
    work = torch.empty(size, dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes = work.data_ptr(), size
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    began = time.perf_counter()
    rc = lib.b200_cache4_selftest_stall(ctypes.byref(p), 128, _native.DTYPE_BF16, skipped, stream)
    assert rc == _native.OK
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    assert read_device_errors(DEV) == _native.DEVERR_WAIT_TIMEOUT
    assert 0.5 < took < 20.0, took
    clear_device_errors(DEV)
    again = b2.b200_tree_attention(*args)
    check_device_errors(DEV)
    assert torch.equal(again, want)
    few = slice(0, 2)
    check(again[few], args[0][few], k, v, table[few], lens_t[few])
