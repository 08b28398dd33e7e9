"""Windowed attention with more work than SMs: every CTA of the persistent
kernels takes several items one after another, in each of their forms.

The references and bars are those of ``test_window_attention_gpu``. The sizes
come from the SM count and are asserted to exceed it, so that no rule of
dispatch can leave these paths without a test.
"""

import pytest
import torch
from test_window_attention_gpu import HALF, _all, _check, _mask, _rand, _reference

pytestmark = pytest.mark.gpu

NAMES = ("out", "dq", "dk", "dv")


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


@pytest.fixture(scope="module")
def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _items(batch, q_len, heads, kv):
    """Work items of the forward kernel: two heads of one key head, or two query tiles where the group is odd."""
    tiles = -(-q_len // 128)
    return batch * (heads // 2 * tiles if heads // kv % 2 == 0 else heads * ((tiles + 1) // 2))


def _compare(got, q, k, v, g, seen, scale):
    """Key head by key head: the 64-bit scores of all heads at once would be tens of GB."""
    kv = k.shape[2]
    group = q.shape[2] // kv
    for h in range(kv):
        own, pair = slice(h * group, (h + 1) * group), slice(h, h + 1)
        refs = _reference(q[:, :, own], k[:, :, pair], v[:, :, pair], seen, scale, g[:, :, own])
        for x, ref, heads, name in zip(got, refs, (own, own, pair, pair), NAMES):
            _check(x[:, :, heads], ref, f"{name} of key head {h}")


# (entries for 3 items a CTA and some) q_len, k_len, q_heads, k_heads, dim, window, sinks
PROMPTS = [
    (700, 700, 8, 2, 64, 150, 3),     # pairs of heads
    (600, 600, 6, 2, 128, 200, 5),    # an odd group, an odd number of query tiles
    (520, 1500, 4, 1, 128, 300, 2),   # a chunk behind earlier keys
    (390, 1111, 3, 3, 72, 64, 70),
    (900, 400, 4, 2, 64, 100, 4),     # tiles that see nothing before the ones that do
    (900, 400, 5, 5, 128, 100, 0),
    (257, 257, 2, 1, 96, 0, 4),       # sinks alone
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", PROMPTS, ids=str)
def test_several_items_for_each_cta(ms, sms, shape, dtype):
    n, m, heads, kv, dim, window, sinks = shape
    batch = -(-(3 * sms + 5) // _items(1, n, heads, kv))
    assert _items(batch, n, heads, kv) > 3 * sms
    q, k, v = _rand((batch, n, heads, dim), dtype, 1), _rand((batch, m, kv, dim), dtype, 2), _rand((batch, m, kv, dim), dtype, 3)
    g = _rand(q.shape, dtype, 4)
    got = _all(ms, q, k, v, g, window=window, sinks=sinks)
    _compare(got, q, k, v, g, _mask(n, m, window, sinks), dim ** -0.5)
    with torch.no_grad():
        assert torch.equal(ms.window_attention(q, k, v, window=window, sinks=sinks), got[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(48, 12, 64), (44, 4, 128)])
def test_packed_items(ms, sms, heads, kv, dim, dtype):
    """The first and the last query tiles of every head see nothing and lie
    between the full ones of the heads before and after."""
    bounds, tokens, window, sinks = [140, 141, 500, 500, 1200, 1300, 1650, 1701], 1900, 130, 5
    assert _items(1, tokens, heads, kv) > 2 * sms
    q, g = _rand((tokens, heads, dim), dtype, 1), _rand((tokens, heads, dim), dtype, 4)
    k, v = _rand((tokens, kv, dim), dtype, 2), _rand((tokens, kv, dim), dtype, 3)
    got = _all(ms, q, k, v, g, window=window, sinks=sinks, indptr=torch.tensor(bounds).cuda())
    for x in got:
        assert (x[:140] == 0).all() and (x[1701:] == 0).all()
    _compare([x[None] for x in got], q[None], k[None], v[None], g[None], _mask(tokens, tokens, window, sinks, bounds),
             dim ** -0.5)


@pytest.mark.parametrize("dtype,heads,kv,dim", [(torch.bfloat16, 80, 40, 64), (torch.float16, 75, 25, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_hidden_values_between_items(ms, sms, dtype, heads, kv, dim, bad):
    """Poisoned tokens that some rows of a tile see and others do not: the
    rows that do not are computed again, and the items after them are as ever."""
    bounds, tokens, window, sinks = [0, 100, 170, 1020], 1040, 40, 2
    assert _items(1, tokens, heads, kv) > 2 * sms
    q, g = _rand((tokens, heads, dim), dtype, 1), _rand((tokens, heads, dim), dtype, 4)
    k, v = _rand((tokens, kv, dim), dtype, 2), _rand((tokens, kv, dim), dtype, 3)
    ptr = torch.tensor(bounds).cuda()
    clean = _all(ms, q, k, v, g, window=window, sinks=sinks, indptr=ptr)
    seen = _mask(tokens, tokens, window, sinks, bounds)
    hit = torch.zeros(tokens, dtype=torch.bool).cuda()
    hit[100:170] = True
    hit[1020:] = True
    hit[400] = True
    poisoned = [t.clone() for t in (q, k, v, g)]
    for t in poisoned:
        t[hit] = bad
    got = _all(ms, *poisoned, window=window, sinks=sinks, indptr=ptr)
    rows = ~(hit | (seen & hit[None, :]).any(1))
    keys = ~(hit | (seen & ~rows[:, None]).any(0))
    assert rows.sum() > 700 and keys.sum() > 700
    for x, y, keep, name in zip(got, clean, (rows, rows, keys, keys), NAMES):
        x, y = x[keep].double(), y[keep].double()
        assert torch.isfinite(x).all(), name
        # the same sums, in fp32 and with unrounded weights where a row is computed again: each side is off by
        # half a step of its weights and half a step of its result
        assert ((x - y).abs() <= 4 * HALF[dtype] * (y.abs() + y.abs().max())).all(), name
