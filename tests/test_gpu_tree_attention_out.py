"""Where the output of drafted-token attention may lie, and gradients asked for."""

import pytest
import torch

from b200_attention import b200_tree_attention, read_device_errors
from test_gpu_tree_attention import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,T,group,lens", [
    (torch.bfloat16, 1, 4, [1000]),
    (torch.bfloat16, 9, 1, [4000, 3]),
    (torch.float16, 40, 1, [2000, 0, 31]),
    (torch.bfloat16, 64, 3, [2500, 7]),
    (torch.float32, 5, 2, [900, 0]),
])
def test_in_the_place_of_the_queries(dtype, T, group, lens):
    """The same bits, with units cut over many CTAs and drafts cut short."""
    q, k, v, table, lens = (t.cuda() for t in make(lens, T, 2, group, 64, 16, dtype, seed=T))
    drafts = torch.full_like(lens, T)
    drafts[-1] = T // 2
    want = b200_tree_attention(q, k, v, table, lens, None, drafts)
    for _ in range(5):
        out = q.clone()
        got = b200_tree_attention(out, k, v, table, lens, None, drafts, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    # beside them in one tensor [B, T, 2, H, D]
    both = torch.stack([q.transpose(1, 2)] * 2, 2)
    side = both[:, :, 1].transpose(1, 2)
    got = b200_tree_attention(both[:, :, 0].transpose(1, 2), k, v, table, lens, None, drafts, out=side)
    assert torch.equal(got, want) and torch.equal(both[:, :, 0], q.transpose(1, 2))
    assert read_device_errors(q.device) == 0


def test_not_over_other_inputs():
    q, k, v, table, lens = (t.cuda() for t in make([40, 50], 4, 2, 2, 64, 16, torch.bfloat16))
    other = torch.empty(2, 4, 5, 64, dtype=q.dtype, device="cuda")
    other[:, :, :4] = q
    for queries, out in ((other[:, :, :4], other[:, :, 1:]), (q, k.view(-1)[:q.numel()].view(q.shape)),
                         (q, v.view(-1)[-q.numel():].view(q.shape)), (q, other[:1, :, :4].expand(2, 4, 4, 64))):
        with pytest.raises(ValueError):
            b200_tree_attention(queries, k, v, table, lens, out=out)


def test_gradients_through_a_cache_are_refused():
    """Of queries, pools and rows alike: the result would have none."""
    from b200_attention import b200_cache_accept, b200_cache_append, b200_cache_compact, b200_cache_reserve

    q, k, v, table, lens = (t.cuda() for t in make([40, 50], 1, 2, 2, 64, 16, torch.bfloat16))
    refs = torch.ones(k.shape[0], dtype=torch.int32, device="cuda")
    rows = torch.randn(2, 2, 1, 64, device="cuda").bfloat16()
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    for kk, vv in ((k.clone().requires_grad_(), v), (k, v.clone().requires_grad_())):
        for call in (lambda: b200_tree_attention(q, kk, vv, table, lens),
                     lambda: b200_cache_append(rows, rows, kk, vv, table, lens),
                     lambda: b200_cache_accept(kk, vv, table, lens, torch.zeros_like(table[:, :1]), one),
                     lambda: b200_cache_reserve(kk, vv, table, lens, refs, 0),
                     lambda: b200_cache_compact(kk, vv, table.clone(), refs.clone())):
            with pytest.raises(ValueError, match="inference-only"):
                call()
        with torch.no_grad():
            b200_tree_attention(q, kk, vv, table, lens)
    with pytest.raises(ValueError, match="inference-only"):
        b200_cache_append(rows.requires_grad_(), rows.detach(), k, v, table, lens)
    assert read_device_errors(q.device) == 0
