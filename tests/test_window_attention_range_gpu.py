"""Windowed attention's gradients where values on the way are beyond what
float16 holds.

The references and bars are those of ``test_window_attention_gpu``.
"""

import pytest
import torch
from test_window_attention_gpu import _all, _check, _mask, _rand, _reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


# batch, tokens, q_heads, k_heads, dim, window, sinks
SCALED = [
    (2, 40, 4, 2, 64, 40, 0),
    (1, 300, 6, 2, 128, 100, 3),
    (3, 129, 2, 2, 72, 20, 1),
    (1, 1100, 2, 1, 128, 30, 16),     # far queries of the sinks
    (40, 300, 8, 2, 64, 60, 2),       # several items for each CTA
    (2, 60, 2, 1, 136, 60, 1),        # the general kernels
]


@pytest.mark.parametrize("shape", SCALED, ids=str)
@pytest.mark.parametrize("size", [8192.0, 14000.0])
def test_loss_scaled_gradients(ms, shape, size):
    """float16 with loss-scaled gradients: P (dP - delta) of single pairs is
    beyond the type's largest number, the gradients themselves are not."""
    b, n, heads, kv, dim, window, sinks = shape
    dtype = torch.float16
    q, k, v = (_rand((b, n, h, dim), dtype, s, x) for h, s, x in ((heads, 1, 0.25), (kv, 2, 0.25), (kv, 3, 3.0)))
    # heads that share a key add their gradients up: smaller ones keep the sums in range
    g = (_rand((b, n, heads, dim), torch.float32, 4) * size / (heads // kv) ** 0.5).clamp(-60000, 60000).to(dtype)
    seen = _mask(n, n, window, sinks)
    refs = _reference(q, k, v, seen, dim ** -0.5, g)
    big = [bool((value.abs() + bar).max() < 65504) for value, bar in refs]
    assert big[1] and big[2], "dq and dk must be in the type's range"
    got = _all(ms, q, k, v, g, window=window, sinks=sinks)
    for x, (value, bar), name in zip(got, refs, ("out", "dq", "dk", "dv")):
        fits = value.abs() + bar < 65504
        assert fits.float().mean() > 0.99
        _check(torch.where(fits, x.double(), 0.0), (torch.where(fits, value, 0.0), bar), name)


@pytest.mark.parametrize("shape", [(2, 300, 4, 2, 64, 90, 3), (60, 300, 4, 2, 64, 90, 3), (1, 1100, 2, 1, 128, 30, 16)],
                         ids=str)
def test_overflow_beside_a_diverged_row(ms, shape):
    """One query's gradient is infinite and others' are loss-scaled: what
    the first does not reach is computed as without it."""
    b, n, heads, kv, dim, window, sinks = shape
    q, k, v = (_rand((b, n, h, dim), torch.float16, s, x) for h, s, x in ((heads, 1, 0.25), (kv, 2, 0.25), (kv, 3, 3.0)))
    g = (_rand((b, n, heads, dim), torch.float32, 4) * 8192).clamp(-40000, 40000).half()
    g[:, 200] = 0
    seen = _mask(n, n, window, sinks)
    refs = _reference(q, k, v, seen, dim ** -0.5, g)
    g[:, 200, 1] = float("inf")
    got = _all(ms, q, k, v, g, window=window, sinks=sinks)
    rows = torch.arange(n).cuda() != 200
    keys = ~seen[200]
    for x, (value, bar), keep, name in zip(got, refs, (rows, rows, keys, keys), ("out", "dq", "dk", "dv")):
        fits = (value.abs() + bar < 65504)[:, keep]
        assert fits.float().mean() > 0.99
        _check(torch.where(fits, x[:, keep].double(), 0.0), (torch.where(fits, value[:, keep], 0.0), bar[:, keep]), name)
