"""Waits of the windowed-attention kernels that give up: the call ends, the
error is reported once, and what runs next is not touched by what the kernel had
in flight."""

import contextlib

import pytest
import torch
from test_window_attention_gpu import _all, _rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


@contextlib.contextmanager
def _wait_limit(ns):
    from mlx_sparse import _native

    L = _native.extension()
    try:
        _native.check(L.msx_debug_set_window_wait_limit(ns))
        yield
    finally:
        _native.check(L.msx_debug_set_window_wait_limit(-1))


# batch, tokens, q_heads, k_heads, dim, window, sinks
SHAPES = [
    (1, 200, 2, 1, 64, 90, 2),        # both slots of a CTA share the queries
    (40, 700, 4, 2, 128, 300, 3),     # pairs of heads, several items for each CTA
    (20, 900, 6, 2, 64, 100, 20),     # two query tiles a CTA; far queries of the sinks
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_waits_that_give_up(ms, shape, dtype):
    from mlx_sparse import _native

    b, n, heads, kv, dim, window, sinks = shape
    q, k, v, g = (_rand((b, n, h, dim), dtype, s) for h, s in ((heads, 1), (kv, 2), (kv, 3), (heads, 4)))
    want = _all(ms, q, k, v, g, window=window, sinks=sinks)
    ms.check_device_errors()
    fwd = _native.window_attention_forward(q, k, v, window, sinks, dim ** -0.5, with_lse=True)
    calls = (
        lambda: _native.window_attention_forward(q, k, v, window, sinks, dim ** -0.5, with_lse=False),
        lambda: _native.window_attention_forward(q, k, v, window, sinks, dim ** -0.5, with_lse=True),
        lambda: _native.window_attention_backward(q, k, v, *fwd, g, window, sinks, dim ** -0.5, want_kv=False),
        lambda: _native.window_attention_backward(q, k, v, *fwd, g, window, sinks, dim ** -0.5, want_q=False),
    )
    for call in calls:
        with _wait_limit(0):
            call()
        # right behind it, on the same SMs and the same shared memory
        for x, y in zip(_all(ms, q, k, v, g, window=window, sinks=sinks), want):
            assert torch.equal(x, y)
        with pytest.raises(RuntimeError, match="windowed-attention kernel's wait"):
            ms.check_device_errors()
        ms.check_device_errors()  # reported once


def test_a_short_limit_that_suffices(ms):
    """A tenth of a second is far more than these sizes take."""
    q, k, v, g = (_rand((2, 300, 2, 64), torch.bfloat16, s) for s in (1, 2, 3, 4))
    want = _all(ms, q, k, v, g, window=90, sinks=2)
    with _wait_limit(100_000_000):
        for x, y in zip(_all(ms, q, k, v, g, window=90, sinks=2), want):
            assert torch.equal(x, y)
    ms.check_device_errors()
