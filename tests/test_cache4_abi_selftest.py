"""The stall self-test of the 4-bit cache's attention refuses what it does not cover (no GPU needed)."""

import ctypes

import pytest

from b200_attention import _native
from b200_attention.build import build_native
from test_cache4_abi import BF16, FP16, UNSUPPORTED, attn


@pytest.fixture(scope="module")
def lib():
    build_native()
    return _native.load_library()


def test_selftest_refuses(lib):
    def call(head_dim=128, dtype=BF16, skipped=0, **kw):
        p = attn(cache_kw=dict(head_dim=40, **kw))
        return lib.b200_cache4_selftest_stall(ctypes.byref(p), head_dim, dtype, skipped, None)

    word = dict(error_word=0x900000000)
    assert call() == UNSUPPORTED                         # nowhere to report
    assert call(64, **word) == UNSUPPORTED and call(136, **word) == UNSUPPORTED
    assert call(dtype=FP16, **word) == UNSUPPORTED
    assert call(skipped=-1, **word) == UNSUPPORTED
    assert lib.b200_cache4_selftest_stall(None, 128, BF16, 0, None) == UNSUPPORTED
