"""Windowed attention with scores so large that every rounding of one shows:
weights of different running maxima must be joined by differences in which these
roundings cancel."""

import pytest
import torch
from test_window_attention_gpu import F, HALF, _check, _mask, _rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch", [1, 80])
@pytest.mark.parametrize("heads,kv", [(4, 2), (3, 1)])
def test_scores_of_a_million(ms, dtype, batch, heads, kv):
    """Scores 2^20 + d with d in steps of 1/4: exact in float32. What is left are
    the roundings of differences: exponents x = c (s - max) from one fma of
    inputs that both sides of a join share, |x| 2^-23 for c and the fma each,
    2^-21 for ex2 and its joins, n 2^-24 for sums; one half step each for the
    weights and the result."""
    n, dim, window = 420, 64, 420
    q = torch.zeros(batch, n, heads, dim)
    k = torch.zeros(batch, n, kv, dim)
    gen = torch.Generator().manual_seed(5)
    q[..., 0], k[..., 0] = 1024.0, 1024.0
    q[..., 1] = 1.0
    # a few keys far above the others: the maximum in use rises
    d = torch.randint(0, 12, (batch, n, kv), generator=gen) * 0.25
    d[:, 130:135] += 7.0
    d[:, 300] += 14.0
    k[..., 1] = d
    q, k = q.to(dtype).cuda(), k.to(dtype).cuda()
    v = _rand((batch, n, kv, dim), dtype, 3)
    got = ms.window_attention(q, k, v, window=window, scale=1.0).double()
    u = 0.0 if dtype == torch.float32 else HALF[dtype]
    seen = _mask(n, n, window, 0)
    s = k[..., 1].double().permute(0, 2, 1).repeat_interleave(heads // kv, 1)[:, :, None, :].expand(-1, -1, n, -1)
    s = s.masked_fill(~seen, float("-inf"))
    p = torch.softmax(s, -1)
    vv = v.double().repeat_interleave(heads // kv, 2)
    value = torch.einsum("bhqk,bkhd->bqhd", p, vv)
    if dtype == torch.float32:  # the general kernels round every score times c by itself: |s c| 2^-24 a weight
        r = 2 * 2 ** 20 * 1.45 * F + (16 + n) * F
    else:
        r = (4 * 25 * 1.45 + 16 + n) * F
    spread = torch.einsum("bhqk,bkhd->bqhd", p, vv.abs())
    bar = (2 * r + u) * spread
    if dtype == torch.float16:
        bar = bar + 2.0 ** -25 * n * vv.abs().max()
    _check(got, (value, bar + HALF[dtype] * (value.abs() + bar)), "out")
