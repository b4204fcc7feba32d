"""GPU: attention over the 4-bit cache where the groups of a position, or the elements of a query, differ by large
powers of two, against 64 bits.

Bounds, before the output type's rounding (an ulp of bf16, 2^-8 |out|):
  * as everywhere 2^-10 sum_p w |v| (a weight's or product's rounding to 16 bits, and the scores');
  * up to 32 query rows for a KV head, the product of weight and V scale is held in fp16 with the row's largest at 2^7 at
    least, so what is below 2^-14 is off by up to 2^-25: n 7 2^-25 / 2^7 of the row's largest max_p(w s), n positions;
  * more rows: weights in fp16 with the largest at 2^7 at least, so a weight below 2^-14 is off by up to 2^-25:
    n 2^-32 max_p(w s) / s of a dim's own group in V, at most n 2^-32 max_p(w) max_p|v| for a dim.
"""
import pytest
import torch

import megaqwen_b200 as mq

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _held(x, group):
    """Values float64 [1][H][S][D] and the largest scale of each position [1][H][S] that the cache stands for."""
    y = x.cpu().double().unflatten(-1, (-1, group))
    s = (y.abs().amax(-1, keepdim=True).float() / 7).bfloat16().double()
    c = torch.where(s > 0, torch.round(y / s), torch.zeros_like(y)).clamp(-7, 7)
    return (c * s).flatten(-2).transpose(1, 2).contiguous(), s.squeeze(-1).amax(-1).transpose(1, 2)


def _compare(got, q, k, v, smax, scale, many):
    """got, q [1][T][Hq][D] causal at the end of k, v [1][H][n][D]; smax [1][H][n]."""
    _, T, Hq, D = q.shape
    H, n = k.shape[1], k.shape[2]
    share, q, got = Hq // H, q.cpu().double(), got.cpu().double()
    worst = 0.0
    for t in range(T):
        m = n - T + t + 1
        for h in range(H):
            w = torch.softmax(scale * q[0, t, h * share:(h + 1) * share] @ k[0, h, :m].t(), -1)
            ref, mag = w @ v[0, h, :m], w @ v[0, h, :m].abs()
            if many:
                flat = m * 2.0 ** -32 * w.amax(-1, keepdim=True) * v[0, h, :m].abs().amax(0)
            else:
                flat = m * 7 * 2.0 ** -32 * (w * smax[0, h, :m]).amax(-1, keepdim=True)
            bound = 2.0 ** -8 * ref.abs() + 2.0 ** -10 * mag + flat + 1e-30
            off = (got[0, t, h * share:(h + 1) * share] - ref).abs() / bound
            assert torch.isfinite(off).all()
            worst = max(worst, float(off.max()))
    assert worst <= 1.0, worst


# 2 rows and 16 in blocks of 8 and 16, 100 rows in a block of 128
@pytest.mark.parametrize("T", [1, 8, 50])
@pytest.mark.parametrize("D,group", [(128, 32), (128, 64), (64, 32)])
@pytest.mark.parametrize("down", [16, 20, 27])
def test_a_group_of_v_far_below_its_neighbours(T, D, group, down):
    S = 300
    c = mq.KV4Cache(1, 1, S, num_kv_heads=1, head_dim=D, group=group)
    k, v = _rand((1, S, 1, D), 1, torch.bfloat16), _rand((1, S, 1, D), 2)
    v[..., group:2 * group] *= 2.0 ** -down
    v = v.bfloat16()
    c.append(0, k, v, [0])
    q = _rand((1, T, 2, D), 3, torch.bfloat16)
    vv, smax = _held(v, group)
    _compare(c.attend(0, q, [S]), q, _held(k, group)[0], vv, smax, D ** -0.5, 2 * T > 32)


@pytest.mark.parametrize("T", [1, 8, 50])
@pytest.mark.parametrize("D,group", [(128, 32), (128, 64), (64, 32)])
@pytest.mark.parametrize("down", [12, 16, 20])
def test_a_group_of_k_far_below_its_neighbours(T, D, group, down):
    """The queries are as much larger in that group, so its part of the scores counts as much as the others'."""
    S = 40 + T
    c = mq.KV4Cache(1, 1, S, num_kv_heads=1, head_dim=D, group=group)
    k, q = _rand((1, S, 1, D), 1), _rand((1, T, 2, D), 3)
    k[..., group:2 * group] *= 2.0 ** -down
    q[..., group:2 * group] *= 2.0 ** down
    k, q = k.bfloat16(), q.bfloat16()
    v = _rand((1, S, 1, D), 2, torch.bfloat16)
    c.append(0, k, v, [0])
    vv, smax = _held(v, group)
    _compare(c.attend(0, q, [S], scale=0.2), q, _held(k, group)[0], vv, smax, 0.2, 2 * T > 32)


@pytest.mark.parametrize("T", [1, 8, 50])
@pytest.mark.parametrize("dtype,up", [(torch.bfloat16, 5), (torch.float16, 7), (torch.bfloat16, 9), (torch.bfloat16, 16), (torch.bfloat16, 20),
                                      (torch.float16, 12), (torch.float16, 14)])
def test_a_large_element_of_the_query(T, dtype, up):
    """One dim of the queries far above the others, where K is zero: the scores are the others' alone."""
    S, D = 40 + T, 128
    c = mq.KV4Cache(1, 1, S, num_kv_heads=1)
    k, q = _rand((1, S, 1, D), 1), _rand((1, T, 2, D), 3)
    k[..., 40] = 0.0
    q[..., 40] = 2.0 ** up
    k, q, v = k.bfloat16(), q.to(dtype), _rand((1, S, 1, D), 2, torch.bfloat16)
    c.append(0, k, v, [0])
    vv, smax = _held(v, 32)
    _compare(c.attend(0, q, [S], scale=0.2), q, _held(k, 32)[0], vv, smax, 0.2, 2 * T > 32)
