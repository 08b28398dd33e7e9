"""Argument checks of the language-model operators that need no GPU: they
answer before any CUDA call."""

import pytest
import torch


def test_distillation_metadata():
    from mlx_sparse import _validation as v

    d, i, p = torch.zeros(2), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    z = torch.zeros(3, 5)
    v.validate_distillation_inputs(d, i, p, z, (3, 5), 1.0)
    with pytest.raises(ValueError, match="teacher's shape"):
        v.validate_distillation_inputs(d, i, p, z, (3, 6), 1.0)
    with pytest.raises(TypeError, match="same dtype"):
        v.validate_distillation_inputs(d, i, p, z.half(), (3, 5), 1.0)
    with pytest.raises(TypeError, match="dtype must be one of"):
        v.validate_distillation_inputs(d, i, p, z.double(), (3, 5), 1.0)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            v.validate_distillation_inputs(d, i, p, z, (3, 5), bad)
    with pytest.raises(ValueError, match="constant"):
        v.validate_distillation_inputs(d.requires_grad_(), i, p, z, (3, 5), 1.0)


def test_distillation_entry_points():
    from mlx_sparse import _native

    lib = _native.extension()

    def forward(vt=0, it=0, nnz=0, ld=5, rows=0, cols=5, temperature=1.0):
        return lib.msx_csr_distill_forward(vt, it, None, None, None, nnz, None, ld, rows, cols, temperature, None, None,
                                           None)

    assert forward(rows=-1) == 1 and b"non-negative" in lib.msx_last_error()
    assert forward(ld=4) == 1 and b"overlap" in lib.msx_last_error()
    assert forward(temperature=0.0) == 1 and b"temperature" in lib.msx_last_error()
    assert forward(vt=5) == 2 and forward(it=5) == 2
    assert forward(rows=2) == 1 and b"must not be null" in lib.msx_last_error()
    assert lib.msx_csr_distill_backward(0, 0, None, None, None, 0, None, 5, 2, 5, 1.0, None, None, None, None) == 1
    assert lib.msx_csr_distill_forward_backward(0, 0, None, None, None, 0, None, 5, 2, 5, 1.0, None, None, None,
                                                None) == 1


def test_window_metadata():
    from mlx_sparse import _validation as v

    q, k = torch.zeros(1, 4, 4, 8), torch.zeros(1, 4, 2, 8)

    def check(q=q, k=k, w=k, window=3, sinks=0, scale=None, rank=4):
        return v.validate_window_inputs(q, k, w, window, sinks, scale, rank=rank, name="window_attention")

    assert check() == (3, 0, 8 ** -0.5) and check(scale=2, window=2 ** 70, sinks=5) == (2 ** 31, 5, 2.0)
    for bad in (dict(q=q[0]), dict(w=k[:, :3]), dict(q=q[..., :4]), dict(q=q[:, :, :3]), dict(q=q[:, :, :0]),
                dict(window=-1), dict(sinks=-1), dict(scale=float("nan")), dict(rank=3),
                dict(q=q.repeat(1, 1, 1, 40), k=k.repeat(1, 1, 1, 40), w=k.repeat(1, 1, 1, 40))):
        with pytest.raises(ValueError):
            check(**bad)
    for bad in (dict(window=1.0), dict(sinks=True), dict(k=k.half()), dict(q=q.double(), k=k.double(), w=k.double())):
        with pytest.raises(TypeError):
            check(**bad)


def test_window_entry_points():
    import ctypes

    from mlx_sparse import _native

    lib = _native.extension()
    st = (ctypes.c_int64 * 3)(64, 64, 64)

    def forward(vt=2, strides=st, batch=0, q_len=4, k_len=4, hq=4, hk=2, dim=64, window=2, sinks=0, scale=1.0, it=0,
                indptr=None, n_seq=0):
        return lib.msx_window_attention_forward(vt, None, strides, None, st, None, st, batch, q_len, k_len, hq, hk, dim,
                                                window, sinks, scale, it, indptr, n_seq, None, None, None, None)

    for bad in (dict(batch=-1), dict(q_len=-1), dict(hq=3), dict(hk=0), dict(dim=0), dict(dim=257), dict(window=-1),
                dict(sinks=-1), dict(scale=float("nan")), dict(strides=None), dict(batch=1), dict(indptr=8, n_seq=1)):
        assert forward(**bad) == 1, bad
    assert forward(vt=3) == 2 and forward(it=9) == 2
    assert forward(batch=70000) == 3 and forward(k_len=2 ** 31) == 3
    assert lib.msx_window_attention_decode(2, None, None, None, st, None, st, 0, 4, 4, 2, 64, 2, 0, 1.0, 0, None, None,
                                           None) == 1
    assert lib.msx_window_attention_decode(2, None, st, None, st, None, st, 1, 4, 4, 2, 64, 2, 0, 1.0, 0, None, None,
                                           None) == 1


def test_window_operands_are_copied_only_where_they_must():
    from mlx_sparse import _native

    base = torch.zeros(2, 10, 6, 64, dtype=torch.bfloat16)
    assert _native.heads_of(base) is base and _native.heads_of(base[:, :, 2:4]).data_ptr() == base[:, :, 2:4].data_ptr()
    turned = base.permute(0, 2, 1, 3)
    assert _native.heads_of(turned).data_ptr() == base.data_ptr()
    for view in (base.transpose(-1, -2).contiguous().transpose(-1, -2), torch.zeros(2, 10, 6, 67).bfloat16()[..., :64],
                 base[:, :, :1].expand(-1, -1, 6, -1), torch.zeros(2 * 10 * 6 * 64 + 1).bfloat16()[1:].view(2, 10, 6, 64)):
        got = _native.heads_of(view)
        assert got.is_contiguous() and got.data_ptr() % 16 == 0 and torch.equal(got, view)
    assert _native._strides(torch.zeros(1, 5, 1, 8)) == [40, 8, 8]
    assert _native._strides(torch.zeros(4, 1, 6, 8)[:, :, ::2]) == [48, 24, 16]
    assert _native._strides(torch.zeros(2, 0, 3, 8)) == [24, 24, 8]
