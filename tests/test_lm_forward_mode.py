"""The language-model operators have no forward-mode derivatives: an input
with a tangent is refused (before any CUDA call), not computed without it."""

import pytest
import torch
from torch.autograd import forward_ad


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_attention_refuses_tangents():
    import mlx_sparse as ms

    q, k = torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8)
    with forward_ad.dual_level():
        for pick in range(3):
            args = [q, k, k]
            args[pick] = _dual(args[pick])
            with pytest.raises(ValueError, match="window_attention has no forward-mode"):
                ms.window_attention(*args, window=2)
            args[0] = _dual(q[:, 0]) if pick == 0 else q[:, 0]
            with pytest.raises(ValueError, match="window_attention_decode has no forward-mode"):
                ms.window_attention_decode(*args, torch.tensor([4]), window=2)


@pytest.mark.gpu
def test_tangents_and_none():
    import mlx_sparse as ms

    data, idx, ptr = torch.randn(4).cuda(), torch.tensor([0, 2, 1, 4]).cuda(), torch.tensor([0, 2, 4]).cuda()
    logits, w = torch.randn(2, 5).cuda(), torch.ones(2).cuda()
    teacher = ms.csr_array((data, idx, ptr), shape=(2, 5))
    q = torch.randn(1, 4, 2, 8).cuda()
    want = ms.csr_distillation_loss(teacher, logits), ms.window_attention(q, q, q, window=2)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="csr_distillation_loss has no forward-mode"):
            ms.csr_distillation_loss(teacher, _dual(logits))
        with pytest.raises(ValueError, match="csr_distillation_loss has no forward-mode"):
            ms.csr_distillation_loss(ms.csr_array((_dual(data), idx, ptr), shape=(2, 5)), logits)
        with pytest.raises(ValueError, match="loss_and_grad has no forward-mode"):
            ms.csr_distillation_loss_and_grad(teacher, _dual(logits))
        with pytest.raises(ValueError, match="loss_and_grad has no forward-mode"):
            ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=_dual(w))
        with pytest.raises(ValueError, match="window_attention has no forward-mode"):
            ms.window_attention(_dual(q.requires_grad_()), q, q, window=2)
        # what has no tangent is computed as ever, inside a level too
        q = q.detach()
        got = ms.csr_distillation_loss(teacher, logits), ms.window_attention(q, q, q, window=2)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    with pytest.raises(ValueError, match="window_attention has no forward-mode"):  # by the functional transform too
        torch.func.jvp(lambda x: ms.window_attention(x, x, x, window=2), (q,), (q,))
