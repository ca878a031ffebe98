"""Groups of a 4-bit cache whose numbers lie about as far apart as fp32 reaches."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors
from cache4_reference import quantise
from test_gpu_cache4 import BF16, DEV, FP32, ints, pools

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("D", [64, 128])
def test_spreads_up_to_fp32_and_past_it(dtype, D):
    each, most = D // 4, 2.0 ** 128
    x = torch.zeros(1, 1, 6, D, dtype=torch.float64)
    # -a..b in bf16 numbers, so that low is the smallest: largest - low is 2^128 (1 - 2^-8), its half...
    for row, (a, b) in enumerate([(most / 2, most / 2 * (1 - 2.0 ** -7)), (most / 4, most / 4),
                                  (0.0, most * (1 - 2.0 ** -8)), (most / 2, most / 2)]):
        x[0, 0, row, :each] = torch.linspace(-a, b, each, dtype=torch.float64)
    x[0, 0, 4, :each] = torch.linspace(-3e38, 3e38, each, dtype=torch.float64)
    x[0, 0, 5, :each] = -3.4e38  # below the lowest bf16 number in fp32; bf16 rounds it to -infinity
    x[0, 0, :, each:2 * each] = torch.arange(each)  # (their neighbours are as usual)
    x = x.to(dtype)
    k, v = pools(1, 1, 1, 16, D)
    table, zero = ints(0).view(1, 1), ints(0)
    b2.b200_cache_append(x.to(DEV), x.to(DEV), k[0], v[0], table, zero)
    want, _ = quantise(x)
    want[0, 0, 3:, :each] = float("nan")  # 2^128 and more
    assert torch.isfinite(want[0, 0, :3]).all()
    for got in b2.b200_cache_read(k[0], v[0], table, zero, 6, D, FP32):
        check_device_errors(DEV)
        torch.testing.assert_close(got.cpu().double(), want, rtol=2.0 ** -24, atol=0, equal_nan=True)
