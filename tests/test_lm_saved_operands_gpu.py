"""What a backward pass of the language-model operators reads is what the
forward pass read: an operand written to in between is an error."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_boundaries_written_before_the_backward_pass(ms, dtype):
    q, k, v = (torch.randn(90, 2, 64, device="cuda").to(dtype).requires_grad_() for _ in range(3))
    ptr = torch.tensor([0, 40, 90]).cuda()
    out = ms.window_attention(q, k, v, window=8, sinks=1, indptr=ptr)
    want = torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)
    for a, b in zip(want, torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)):
        assert torch.equal(a, b)
    ptr.copy_(torch.tensor([0, 10, 90]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("which", ["data", "indices", "indptr"])
def test_teacher_written_before_the_backward_pass(ms, which):
    parts = dict(data=torch.randn(6).cuda(), indices=torch.tensor([0, 3, 4, 1, 2, 8]).cuda(),
                 indptr=torch.tensor([0, 2, 3, 6]).cuda())
    logits = torch.randn(3, 9, device="cuda", requires_grad=True)
    teacher = ms.csr_array((parts["data"], parts["indices"], parts["indptr"]), shape=(3, 9))
    kept = getattr(teacher, which)
    loss = ms.csr_distillation_loss(teacher, logits)
    torch.autograd.grad(loss.sum(), logits, retain_graph=True)
    kept.copy_(kept.flip(0) if which != "indptr" else torch.tensor([0, 1, 2, 6]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()
