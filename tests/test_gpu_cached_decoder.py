"""The decoder over a paged cache against its forward pass over whole sequences."""

import sys
from pathlib import Path

import pytest
import torch

from b200_attention import read_device_errors
from b200_attention.transformer import Decoder, DecoderConfig, init_normal_

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


def model_of(dtype, heads=4, d_model=256, layers=2):
    config = DecoderConfig(batch_size=3, seq_len=70, d_model=d_model, num_heads=heads,
                           ffn_dim=2 * d_model, num_layers=layers, causal=True, vocab_size=61)
    # std 0.1 gives softmaxes with weight on few keys
    return init_normal_(Decoder(config), std=0.1, seed=3).to("cuda", dtype).eval()


def reference(model, tokens):
    """Hidden states of whole sequences [B, S] in 64-bit torch operations."""
    x = model.embed(tokens).double()
    for layer in model.layers:
        at = layer.attention

        def lin(m, t):
            return t @ m.weight.double().t() + m.bias.double()

        def norm(m, t):
            return torch.nn.functional.layer_norm(t, t.shape[-1:], m.weight.double(),
                                                  m.bias.double(), m.eps)

        h = norm(layer.norm1, x)
        b, s, d = h.shape
        q, k, v = (lin(m, h).view(b, s, at.num_heads, at.head_dim).transpose(1, 2)
                   for m in (at.q_proj, at.k_proj, at.v_proj))
        scores = (q @ k.transpose(2, 3)) * at.scale
        scores = scores.masked_fill(torch.ones(s, s, dtype=torch.bool, device=h.device).triu(1),
                                    float("-inf"))
        x = x + lin(at.out_proj, (scores.softmax(-1) @ v).transpose(1, 2).reshape(b, s, d))
        x = x + lin(layer.ffn_out, torch.nn.functional.gelu(lin(layer.ffn_in, norm(layer.norm2, x))))
    return norm(model.final_norm, x)


# fp32: a few thousand operations of relative error 2^-24 on values of order 1 (the outputs
# are normalised).  16-bit: each block rounds about ten intermediate tensors (up to 2^-8 or
# 2^-11 relative, values up to 8 or so), which add up as independent errors.
BOUNDS = {torch.float32: 2e-4, torch.float16: 5e-2, torch.bfloat16: 3e-1}


@pytest.mark.parametrize("dtype", list(BOUNDS))
@pytest.mark.parametrize("page", [16, 24])
def test_prompt_then_tokens_then_trees(dtype, page):
    model = model_of(dtype)
    gen = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, 61, (3, 70), generator=gen).cuda()
    cache = model.new_cache(3, 120, page)
    with torch.no_grad():
        want = reference(model, tokens)
        # a prompt of 41 tokens
        assert int(cache.reserve(41)) == 0
        got = model.cached_forward(tokens[:, :41], cache)
        assert float((got.double() - want[:, :41]).abs().max()) < BOUNDS[dtype]
        chain = torch.arange(41, dtype=torch.int32, device="cuda").expand(3, 41).contiguous()
        cache.accept(chain, torch.full((3,), 41, dtype=torch.int32, device="cuda"))
        # one token a step
        first = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
        one = torch.ones(3, dtype=torch.int32, device="cuda")
        for t in range(41, 47):
            assert int(cache.reserve(1)) == 0
            got = model.cached_forward(tokens[:, t:t + 1], cache)
            assert float((got[:, 0].double() - want[:, t]).abs().max()) < BOUNDS[dtype]
            cache.accept(first, one)
        # a tree: the true next four tokens interleaved with wrong ones
        wrong = torch.randint(0, 61, (3, 4), generator=gen).cuda()
        drafted = torch.stack([tokens[:, 47:51], wrong], 2).reshape(3, 8)
        mask = torch.zeros(8, 8, dtype=torch.bool)
        for i in range(8):
            mask[i, i % 2:i + 1:2] = True
        assert int(cache.reserve(8)) == 0
        got = model.cached_forward(drafted, cache, mask.cuda())
        assert float((got[:, ::2].double() - want[:, 47:51]).abs().max()) < BOUNDS[dtype]
        wrong_seq = torch.cat([tokens[:, :47], wrong], 1)
        other = reference(model, wrong_seq)[:, 47:]
        assert float((got[:, 1::2].double() - other).abs().max()) < BOUNDS[dtype]
        cache.accept(torch.tensor([[0, 2, 4, 6]] * 3, dtype=torch.int32, device="cuda"),
                     torch.tensor([4, 2, 0], dtype=torch.int32, device="cuda"))
        # sequences of different lengths go on
        assert cache.seq_lens.tolist() == [51, 49, 47]
        assert int(cache.reserve(1)) == 0
        step = torch.stack([tokens[0, 51], tokens[1, 49], tokens[2, 47]])[:, None]
        got = model.cached_forward(step, cache)
        for b, t in enumerate((51, 49, 47)):
            assert float((got[b, 0].double() - want[b, t]).abs().max()) < BOUNDS[dtype]
    assert read_device_errors(tokens.device) == 0


def test_branches_of_one_prompt():
    """Fork, write different tokens, free one and close the gaps: the others go on."""
    model = model_of(torch.bfloat16)
    tokens = torch.randint(0, 61, (1, 30), generator=torch.Generator().manual_seed(2)).cuda()
    ends = torch.tensor([[5, 6], [7, 8], [9, 10]]).cuda()
    cache = model.new_cache(3, 64, 16)
    i32 = dict(dtype=torch.int32, device="cuda")
    with torch.no_grad():
        assert int(cache.reserve(torch.tensor([28, 0, 0], **i32))) == 0
        lens = torch.tensor([28, 0, 0], **i32)
        model.cached_forward(tokens[:, :28].expand(3, 28).contiguous(), cache, None, lens)
        cache.accept(torch.arange(28, **i32).expand(3, 28).contiguous(), lens)
        cache.fork(torch.tensor([0, 0], **i32), torch.tensor([1, 2], **i32))
        for j in range(2):
            assert int(cache.reserve(1)) == 0
            got = model.cached_forward(ends[:, j:j + 1], cache)
            cache.accept(torch.zeros(3, 1, **i32), torch.ones(3, **i32))
            if j == 0:
                cache.free(torch.tensor([1], **i32))
                assert int(cache.compact()) == int((cache.page_refs > 0).sum())
        want = reference(model, torch.cat([tokens[:, :28].expand(3, 28), ends], 1))[:, -1]
        for b in (0, 2):
            assert float((got[b, 0].double() - want[b]).abs().max()) < BOUNDS[torch.bfloat16]
    assert read_device_errors(tokens.device) == 0


def test_example_gives_the_same_tokens():
    import speculative_decode

    assert speculative_decode.main() == 0


def test_cache_refuses_models_that_look_ahead():
    config = DecoderConfig(batch_size=1, seq_len=8, d_model=64, num_heads=1, ffn_dim=64,
                           num_layers=1, causal=False)
    model = Decoder(config).cuda()
    with pytest.raises(ValueError, match="causal"):
        model.cached_forward(torch.zeros(1, 1, 64, device="cuda"), model.new_cache(1, 8))
