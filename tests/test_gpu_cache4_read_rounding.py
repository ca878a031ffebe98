"""What a 4-bit cache holds, read back: each number is rounded once to the type asked for."""

import numpy as np
import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors
from cache4_reference import decode
from test_gpu_cache4 import BF16, DEV, FP16, FP32, ints, pools

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


def rounded(x, dtype):
    """float64 numbers, of bf16 and fp32 normal ones, rounded to nearest, ties to even, in one go."""
    x = x.numpy()
    bits = {BF16: 8, FP16: 11, FP32: 24}[dtype]
    ulp = 2.0 ** (np.floor(np.log2(np.abs(np.where(x == 0, 1.0, x)))) + 1 - bits)
    if dtype == FP16:  # numbers below the normal ones
        ulp = np.maximum(ulp, 2.0 ** -24)
    return torch.from_numpy(np.rint(x / ulp) * ulp)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [64, 128])
def test_next_to_a_border(dtype, D):
    """low = +-2^-30 or 0 and steps of 8 bits: many step * code lie halfway between two numbers of a
    16-bit type, and low says on which side the sum lies (or leaves a tie)."""
    each, codes = D // 4, torch.arange(16).float().repeat(D // 64)
    steps = torch.arange(129, 256, 2).float() / 256  # 64 of them, all 8 bits long
    low = torch.tensor([2.0 ** -30, -2.0 ** -30, 0.0, 2.0 ** -13])
    x = codes * steps[:, None, None]                                        # [64, 1, each]
    x = torch.where(codes == 15, x * (1 - 2.0 ** -12), x).expand(64, 4, each)
    x = torch.where(codes == 0, low[:, None], x).reshape(1, 1, 64, D)
    k, v = pools(1, 4, 1, 16, D)
    table, zero = torch.arange(4, dtype=torch.int32, device=DEV).view(1, 4), ints(0)
    for sign in (1, -1):  # (of negated groups low is the largest code's end)
        b2.b200_cache_append((sign * x).to(DEV), (sign * x).to(DEV), k[0], v[0], table, zero)
        got = b2.b200_cache_read(k[0], v[0], table, zero, 64, D, dtype)
        check_device_errors(DEV)
        for read, pool, keys in ((got[0], k, True), (got[1], v, False)):
            exact = decode(pool, D, keys)[0][0, :, 0].reshape(64, D)
            assert torch.equal(read[0, 0].cpu().double(), rounded(exact, dtype))
        if sign == 1 and dtype != FP32:  # the cases are there: rounding to fp32 first goes wrong
            twice = exact.float().to(dtype).double()
            assert (twice != rounded(exact, dtype)).any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_steps_and_lows_of_every_size(dtype):
    """Steps and lows of 8 bits, each up to 2^24 times the other, and numbers below the normal ones of
    fp16."""
    gen = torch.Generator().manual_seed(1)
    n, D = 4096, 64
    step = (torch.randint(128, 256, (n, 4, 1), generator=gen) / 128.0)
    low = (torch.randint(128, 256, (n, 4, 1), generator=gen) / 128.0) * (
        torch.randint(0, 2, (n, 4, 1), generator=gen) * 2 - 1)
    low = low * 2.0 ** torch.randint(-24, 25, (n, 4, 1), generator=gen)
    size = 2.0 ** (torch.randint(-30, -8, (n, 4, 1), generator=gen) if dtype == FP16 else
                   torch.randint(-60, 60, (n, 4, 1), generator=gen)).float()
    codes = torch.arange(16.0)
    codes[15] -= 2.0 ** -9  # the step is not rounded up from it
    # the sum itself has more bits than fp32: what matters is that the group has these ends
    x = ((low.double() + step.double() * codes) * size).float()
    x[..., 0] = (low * size)[..., 0]
    x = x.reshape(1, 1, n, D)
    k, v = pools(1, n // 16, 1, 16, D)
    table, zero = torch.arange(n // 16, dtype=torch.int32, device=DEV).view(1, -1), ints(0)
    b2.b200_cache_append(x.to(DEV), x.to(DEV), k[0], v[0], table, zero)
    got = b2.b200_cache_read(k[0], v[0], table, zero, n, D, dtype)
    check_device_errors(DEV)
    for read, pool, keys in ((got[0], k, True), (got[1], v, False)):
        exact = decode(pool, D, keys)[0][0, :, 0].reshape(n, D)
        assert torch.equal(read[0, 0].cpu().double(), rounded(exact, dtype))
