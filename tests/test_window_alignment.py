"""Alignment of what a C caller passes to windowed attention: the softmax
statistics and the workspace are refused where they are not 16-byte aligned
(answered before any CUDA call), outputs may lie anywhere."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from mlx_sparse import _native

    return _native.extension()


def test_statistics_and_workspace_must_be_aligned(lib):
    st = (ctypes.c_int64 * 3)(64, 64, 64)

    def head(dim=64):
        return [2, None, st, None, st, None, st, 0, 4, 4, 4, 2, dim, 2, 0, 1.0, 0, None, 0]

    def forward(lse):
        return lib.msx_window_attention_forward(*head(), None, None, lse, None)

    def backward(lse, work):
        return lib.msx_window_attention_backward(*head(), None, None, lse, None, work, None, None, None, None)

    for bad in (4, 8, 24, 4104):
        assert forward(bad) == 1 and b"16-byte aligned" in lib.msx_last_error()
        assert backward(bad, 16) == 1 and b"16-byte aligned" in lib.msx_last_error()
        assert backward(16, bad) == 1 and b"16-byte aligned" in lib.msx_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 200, 4, 2, 64, 50, 3), (30, 300, 4, 2, 128, 90, 2)], ids=str)
def test_outputs_anywhere(lib, shape, dtype):
    from mlx_sparse import _native
    from test_window_attention_gpu import _check, _mask, _rand, _reference

    b, n, heads, kv, dim, window, sinks = shape
    q, k, v, g = (_rand((b, n, h, dim), dtype, s) for h, s in ((heads, 1), (kv, 2), (kv, 3), (heads, 4)))
    refs = _reference(q, k, v, _mask(n, n, window, sinks), dim ** -0.5, g)
    lse = torch.empty(b, heads, (n + 127) // 128 * 128, device="cuda")
    floats = ctypes.c_int64()
    _native.check(lib.msx_window_attention_workspace(b, n, n, heads, kv, dim, window, sinks, ctypes.byref(floats)))
    work = torch.empty(floats.value, device="cuda")
    args, keep = _native._window_args(q, k, v, window, sinks, dim ** -0.5, None)
    stream = torch.cuda.current_stream().cuda_stream
    for moved in range(6):  # each of the outputs one element off in turn, then none
        def new(like, off):
            flat = torch.full((like.numel() + 24,), 7.0, dtype=dtype, device="cuda")
            return flat, flat[off:off + like.numel()].view(like.shape)

        flats, outs = zip(*(new(t, 8 + (i == moved)) for i, t in enumerate((q, q, q, k, k))))
        out, low, dq, dk, dv = outs
        _native.check(lib.msx_window_attention_forward(*args, out.data_ptr(), low.data_ptr(), lse.data_ptr(), stream))
        _native.check(lib.msx_window_attention_backward(*args, out.data_ptr(), low.data_ptr(), lse.data_ptr(),
                                                        g.data_ptr(), work.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                                                        dv.data_ptr(), stream))
        for x, ref, name in zip((out, dq, dk, dv), refs, ("out", "dq", "dk", "dv")):
            _check(x, ref, f"{name}, output {moved} moved")
        for i, (flat, t) in enumerate(zip(flats, outs)):  # nothing beside the outputs is written
            if dtype == torch.float32 and i == 1:
                continue  # not wanted
            first = 8 + (i == moved)
            assert (flat[:first] == 7).all() and (flat[first + t.numel():] == 7).all()
