"""A decoder's cache in 4 bits: for the types whose attention reads one (no GPU needed)."""

import pytest
import torch

from b200_attention.transformer import Decoder, DecoderConfig


def model_of(dtype):
    return Decoder(DecoderConfig(batch_size=1, seq_len=8, d_model=64, num_heads=2, ffn_dim=64, num_layers=1,
                                 causal=True)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_types_that_have_it(dtype):
    cache = model_of(dtype).new_cache(1, 8, 16, bits=4)
    assert cache.k_pages.dtype == torch.uint8 and cache.dtype == dtype


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_others_are_refused_where_the_cache_is_made(dtype):
    with pytest.raises(TypeError, match="4-bit cache"):
        model_of(dtype).new_cache(1, 8, 16, bits=4)
    assert model_of(dtype).new_cache(1, 8, 16).k_pages.dtype == dtype  # pages of the model's type
