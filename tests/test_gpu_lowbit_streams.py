"""GPU: what a constructor puts on its stream is done when it returns, so that the first call may be on any stream."""
import pytest
import torch

import megaqwen_b200 as mq

pytestmark = pytest.mark.gpu
BUSY = 200_000_000                                      # clocks that the constructing stream is kept busy for (0.1 s)


def _rand(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").bfloat16()


def test_cache():
    x, zero = _rand((2, 60, 8, 128), 1), torch.zeros(2, dtype=torch.int32, device="cuda")
    want = mq.KV4Cache(1, 2, 60)
    want.append(0, x, x, zero)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(BUSY)
        c = mq.KV4Cache(1, 2, 60)                       # fills codes and scales behind the sleep
    c.append(0, x, x, zero)
    torch.cuda.synchronize()
    assert torch.equal(c.codes, want.codes) and torch.equal(c.scales, want.scales)
    c.check_device()


@pytest.mark.parametrize("k", [100, 96])
@pytest.mark.parametrize("m", [2, 40])
def test_linear(k, m):
    """k = 100: the weights are copied into padded rows."""
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-127, 128, (70, k), generator=g, device="cuda", dtype=torch.int8)
    s, x = torch.rand(140, generator=g, device="cuda")[::2], _rand((m, k), 2)
    want = mq.Int8Linear(w, s)(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(BUSY)
        lin = mq.Int8Linear(w, s)
    got = lin(x)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    lin.check_device()
