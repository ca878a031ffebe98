"""A step of speculative decoding as a user runs it: a decoder over a cache held in 4 bits, the check
of its drafted tree against its own probabilities, and the cache moved to the nodes kept."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors
from b200_attention.transformer import Decoder, DecoderConfig, init_normal_
from cache4_reference import verify64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
VOCAB = 5  # few tokens: drafts drawn at random are often kept


def model_of(heads, d_model):
    config = DecoderConfig(batch_size=3, seq_len=40, d_model=d_model, num_heads=heads, ffn_dim=2 * d_model,
                           num_layers=2, causal=True, vocab_size=VOCAB)
    return init_normal_(Decoder(config), std=0.1, seed=3).to("cuda", torch.bfloat16).eval()


def tree_of(nodes, gen):
    parents = torch.tensor([-1] + [int(torch.randint(max(0, i - 3), i, (1,), generator=gen)) for i in range(1, nodes)])
    mask = torch.zeros(nodes, nodes, dtype=torch.bool)
    for i in range(nodes):
        if i:
            mask[i] = mask[parents[i]]
        mask[i, i] = True
    return parents.int().to(DEV), mask.to(DEV)


def step(model, cache, drafted, mask, parents, uniforms):
    """What a user runs for each tree: no call of it waits for the host."""
    failed = cache.reserve(drafted.shape[1])
    hidden = model.cached_forward(drafted, cache, mask)
    logits = hidden.float() @ model.embed.weight.float().t()
    before = cache.seq_lens.clone()
    rows = [cache.read(layer, before, drafted.shape[1]) for layer in range(2)]
    paths, counts, following = b2.b200_verify_drafts(logits, drafted, uniforms, None, parents)
    cache.accept(paths, counts)
    return failed, logits, before, rows, paths, counts, following


@pytest.mark.parametrize("heads,d_model,nodes", [(2, 128, 6), (1, 128, 24)])
def test_a_step_over_a_4_bit_cache(heads, d_model, nodes):
    gen = torch.Generator().manual_seed(nodes)
    model = model_of(heads, d_model)
    parents, mask = tree_of(nodes, gen)
    prompts = torch.randint(0, VOCAB, (3, 20), generator=gen).to(DEV)
    given = torch.tensor([20, 7, 1], dtype=torch.int32, device=DEV)
    caches = [model.new_cache(3, 200, 16, bits=4) for _ in range(2)]
    with torch.no_grad():
        for cache in caches:
            assert int(cache.reserve(given)) == 0
            model.cached_forward(prompts, cache, None, given)
            cache.accept(torch.arange(20, dtype=torch.int32, device=DEV).expand(3, 20).contiguous(), given)
        drafted = torch.randint(0, VOCAB, (3, nodes), generator=gen).to(DEV)
        uniforms = torch.rand(3, nodes, generator=gen).to(DEV)
        graph, kept = None, 0
        for turn in range(5):
            failed, logits, before, rows, paths, counts, following = step(model, caches[0], drafted, mask, parents, uniforms)
            if turn == 0:  # the other cache takes its first step eagerly, the others from a graph
                twin = step(model, caches[1], drafted, mask, parents, uniforms)
            else:
                if graph is None:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        twin = step(model, caches[1], drafted, mask, parents, uniforms)
                graph.replay()
            check_device_errors(DEV)
            assert int(failed) == 0 and int(twin[0]) == 0
            want = verify64(logits, drafted, uniforms, None, parents.view(1, -1))
            assert torch.equal(paths.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
            assert torch.equal(following.cpu(), want[2])
            assert torch.equal(caches[0].seq_lens, before + counts)
            for layer in range(2):  # the kept nodes' rows, in order, behind what was there
                after = caches[0].read(layer, before, nodes, counts)
                for now, then in zip(after, rows[layer]):
                    at = paths.long().clamp(min=0)[:, None, :, None].expand_as(then)
                    there = (paths >= 0)[:, None, :, None]
                    assert torch.equal(now, torch.where(there, then.gather(2, at), 0))
            for x, y in zip((paths, counts, following, logits), (twin[4], twin[5], twin[6], twin[1])):
                assert torch.equal(x, y)
            for name in ("page_table", "seq_lens", "page_refs", "k_pages", "v_pages"):
                assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))
            kept += int(counts.sum())
            # the next tree: its root is the token that follows
            fresh = torch.randint(0, VOCAB, (3, nodes), generator=gen).to(DEV)
            fresh[:, 0] = following
            drafted.copy_(fresh)
            uniforms.copy_(torch.rand(3, nodes, generator=gen).to(DEV))
        assert kept > 15  # some drafts were kept
