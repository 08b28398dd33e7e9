"""Threads that call one operator at once, each on a stream of its own."""

import threading

import pytest
import torch
from test_window_attention_gpu import _all, _rand

pytestmark = pytest.mark.gpu


def _together(works):
    failed, start = [], threading.Barrier(len(works))

    def run(work):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                work()
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 - reported by the main thread
            failed.append(repr(e))

    threads = [threading.Thread(target=run, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[:3]


@pytest.mark.parametrize("dtype,dims", [(torch.float32, (256, 8)), (torch.float16, (250, 33)), (torch.bfloat16, (128, 64))])
def test_threads_with_different_head_sizes(dtype, dims):
    import mlx_sparse as ms

    def calls(dim):
        def work():
            q, k, v, g = (_rand((1, 20, 2, dim), dtype, s) for s in (1, 2, 3, 4))
            torch.cuda.synchronize()
            want = _all(ms, q, k, v, g, window=7, sinks=1)
            for _ in range(200):
                for a, b in zip(_all(ms, q, k, v, g, window=7, sinks=1), want):
                    assert torch.equal(a, b)

        return work

    _together([calls(d) for d in dims for _ in range(2)])


def test_threads_in_the_entry_point_itself():
    """Little but launches: one thread's head size must not change what another's launch may use."""
    from mlx_sparse import _native

    lib = _native.extension()

    def calls(dim):
        q = _rand((1, 16, 1, dim), torch.float32, 1)
        out = torch.empty_like(q)
        torch.cuda.synchronize()

        def work():
            args, keep = _native._window_args(q, q, q, 4, 0, 1.0, None)
            args += [out.data_ptr(), None, None, torch.cuda.current_stream().cuda_stream]
            call = lib.msx_window_attention_forward
            for _ in range(20000):
                if call(*args):
                    raise RuntimeError(lib.msx_last_error())

        return work

    _together([calls(d) for d in (256, 8, 256, 8)])
