"""Sequences whose length or draft does not fit: their rows are zero and reported, the others
are unharmed, whatever the workspace held before."""

import ctypes

import pytest
import torch

from b200_attention import _native, b200_tree_attention
from b200_attention.fused_attention import DeviceError, clear_device_errors
from paged_reference import attention64, attention_bound
from test_gpu_tree_attention import make

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
CODES = {BF16: _native.DTYPE_BF16, FP16: _native.DTYPE_FP16, FP32: _native.DTYPE_FP32}


def call(q, k, v, table, lens, drafts, fill, counters=None):
    """The C entry with a workspace of the words given, over and over; (output, error word)."""
    out = torch.full_like(q, float("nan"))
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = _native.TreeAttnParams()
    c = p.cache
    c.k, c.v, c.layers, c.error_word = k.data_ptr(), v.data_ptr(), 1, word.data_ptr()
    c.pages, c.kv_heads, c.page_size, c.head_dim = k.shape
    c.k_stride[1:], c.v_stride[1:] = k.stride()[:3], v.stride()[:3]
    c.page_table, c.table_stride, c.seq_lens = table.data_ptr(), table.stride(0), lens.data_ptr()
    c.batch, c.slots = table.shape
    c.dtype = CODES[q.dtype]
    p.q, p.o, p.heads, p.tokens, p.scale = q.data_ptr(), out.data_ptr(), q.shape[1], q.shape[2], q.shape[3] ** -0.5
    p.q_stride[:], p.o_stride[:] = q.stride()[:3], out.stride()[:3]
    p.draft_lens = None if drafts is None else drafts.data_ptr()
    p.counters = None if counters is None else counters.data_ptr()
    lib = _native.load_library()
    size = lib.b200_tree_attn_workspace_bytes(ctypes.byref(p))
    words = torch.tensor(fill, dtype=torch.int32, device="cuda")
    ws = words.repeat(size // (4 * len(fill)) + 1)
    p.workspace, p.workspace_bytes = ws.data_ptr(), size
    assert lib.b200_tree_attn_fwd(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == _native.OK
    torch.cuda.synchronize()
    return out, int(word)


# Cut differently, so not bit for bit: each within 2^-8 (size + 2 |out|) of the exact result in
# bfloat16, with size and |out| at most the largest |v|, below 5 for the values drawn here.
APART = 2 * 3 * 5 * 2.0 ** -8

# ranges of runs that a join would follow: far outside the workspace, inside it, and none
FILLS = [(0, 1 << 30), (1, 2), (-1, -1), (-(1 << 30), 1 << 30)]


@pytest.mark.parametrize("dtype,T,group,D,page,long", [
    (BF16, 40, 1, 64, 16, 300),    # 128 rows
    (FP16, 64, 4, 128, 32, 900),   # 256 rows, in several row tiles
    (BF16, 2, 2, 64, 16, 300),     # few rows, joined by a second kernel
    (BF16, 8, 1, 128, 16, 4000),   # few rows over a long context, joined four rows a block
    (BF16, 17, 1, 64, 7, 300),     # two row tiles
    (FP32, 2, 2, 64, 16, 300),
    (FP32, 40, 2, 64, 16, 300),
])
@pytest.mark.parametrize("bad", ["negative", "full", "huge", "more drafts", "negative drafts"])
def test_left_out_sequences_are_zero(dtype, T, group, D, page, long, bad):
    args = make([40, long, 70], T, 2, group, D, page, dtype)
    q, k, v, table, lens = (t.cuda() for t in args)
    want, size, grow = attention64(*args)
    bound = attention_bound(dtype, want, size, grow, D, long + T)
    drafts = torch.full((3,), T, dtype=torch.int32, device="cuda")
    if bad == "more drafts":
        drafts[0] = T + 1
    elif bad == "negative drafts":
        drafts[0] = -1
    else:
        lens[0] = {"negative": -1, "full": table.shape[1] * page - T + 1, "huge": 1 << 30}[bad]
    for fill in FILLS:
        got, word = call(q, k, v, table, lens, drafts, fill)
        assert word == _native.DEVERR_BOUNDS
        assert (got[0] == 0).all(), fill
        # (twice attention_bound holds if all its roundings point one way: 2u size + 4u |out|,
        # and |out| <= size)
        assert ((got[1:].cpu().double() - want[1:]).abs() <= 2 * bound[1:]).all(), fill


def test_more_units_than_counters():
    args = make([5, 300] * 150, 1, 4, 1, 64, 16, BF16, seed=2)
    q, k, v, table, lens = (t.cuda() for t in args)
    counters = torch.zeros(1024, dtype=torch.int32, device="cuda")
    good, word = call(q, k, v, table, lens, None, (-1, -1), counters)
    assert word == 0
    lens[::2] = -3
    for fill in FILLS:
        got, word = call(q, k, v, table, lens, None, fill, counters)
        assert word == _native.DEVERR_BOUNDS and not counters.any()
        assert (got[::2] == 0).all()
        assert float((got[1::2].float() - good[1::2].float()).abs().max()) < APART


@pytest.mark.parametrize("dtype,T", [(BF16, 1), (BF16, 40), (FP32, 3)])
def test_a_captured_step_goes_on_over_a_full_sequence(dtype, T):
    """A sequence grows past its slots between replays, as when nobody reads the status of
    the reservation."""
    args = make([40, 500, 70], T, 2, 2, 64, 16, dtype)
    q, k, v, table, lens = (t.cuda() for t in args)
    b200_tree_attention(q, k, v, table, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = b200_tree_attention(q, k, v, table, lens)
    graph.replay()
    good = held.clone()
    lens[1] = table.shape[1] * 16 - T + 1
    try:
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert (held[1] == 0).all()
        assert float((held[::2].float() - good[::2].float()).abs().max()) < APART
        with pytest.raises(DeviceError, match="bounds"):
            b200_tree_attention(q, k, v, table, lens)
    finally:
        clear_device_errors(q.device)
    lens[1] = 500
    graph.replay()
    assert torch.equal(held, good)
