"""Distillation rows whose entries share columns, with probabilities over the
whole range of float32: the gradient of a column that the student gives next to
nothing is the sum of its entries' probabilities, to relative accuracy.

References and bars are those of ``test_distill_gpu``; the sum of a column's
entries adds one rounding, which the bar's slack of 8 covers.
"""

import numpy as np
import pytest
import torch
from test_distill_gpu import _check, _reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


def _case(rows, vocab, entries, columns, dtype, seed):
    """Rows of `entries` entries on at most `columns` different columns; every
    seventh row has none. The student gives the entries' columns very little."""
    rng = np.random.default_rng(seed)
    cols, ptr = [], [0]
    logits = rng.standard_normal((rows, vocab)).astype(np.float32)
    for i in range(rows):
        n = 0 if i % 7 == 6 else entries
        some = rng.choice(vocab, min(columns, vocab), replace=False)
        logits[i, some] = rng.uniform(-30, -20, len(some))
        cols.append(rng.choice(some, n))
        ptr.append(ptr[-1] + n)
    data = torch.from_numpy(rng.uniform(-12, 8, ptr[-1])).to(dtype).cuda()
    parts = (data, torch.from_numpy(np.concatenate(cols)).cuda(), torch.tensor(ptr).cuda())
    return parts, torch.from_numpy(logits).to(dtype).cuda()


# rows, vocab, entries, columns: slices kept in shared memory, spread over a cluster, read again
SHAPES = [(1, 40, 60, 9), (5, 5000, 64, 30), (9, 33, 1, 1), (3, 90000, 2000, 700), (400, 70001, 40, 25), (2, 900, 30000, 50)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sums_of_small_probabilities(ms, shape, dtype):
    rows, vocab, entries, columns = shape
    T = 0.25  # probabilities down to e^-80
    parts, logits = _case(rows, vocab, entries, columns, dtype, seed=vocab)
    teacher = ms.csr_array(parts, shape=(rows, vocab))
    w = torch.linspace(0.25, 1.0, rows)
    loss, bar, grad, gbar = _reference(parts, logits, T, w.double())
    one = ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=w.cuda(), temperature=T)
    _check(one[0], loss, bar, "one-pass loss")
    _check(one[1], grad, gbar, "one-pass gradient")
    leaf = logits.clone().requires_grad_()
    two = ms.csr_distillation_loss(teacher, leaf, temperature=T)
    (auto,) = torch.autograd.grad(two, leaf, w.cuda())
    _check(auto, grad, gbar, "gradient")
    again = ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=w.cuda(), temperature=T)
    assert torch.equal(again[0], one[0]) and torch.equal(again[1], one[1])


def test_entries_of_no_mass_and_of_no_number(ms):
    inf, nan = float("inf"), float("nan")
    data = torch.tensor([1.0, -inf, 2.0, -inf, -inf, nan, 1.0, 1.0, -inf, -inf, 0.0, 0.0]).cuda()
    idx = torch.tensor([3, 3, 7, 5, 5, 2, 2, 4, 1, 1, 6, 6]).cuda()
    ptr = torch.tensor([0, 5, 8, 10, 12]).cuda()
    logits = torch.zeros(4, 9).cuda()
    teacher = ms.csr_array((data, idx, ptr), shape=(4, 9))
    leaf = logits.clone().requires_grad_()
    (auto,) = torch.autograd.grad(ms.csr_distillation_loss(teacher, leaf).sum(), leaf)
    for grad in (ms.csr_distillation_loss_and_grad(teacher, logits)[1], auto):
        p = torch.softmax(torch.tensor([1.0, 2.0], dtype=torch.float64), 0)
        want = torch.full((9,), 1 / 9, dtype=torch.float64)
        want[3] -= p[0]
        want[7] -= p[1]
        assert ((grad[0].cpu().double() - want).abs() <= 40 * 2.0 ** -24).all()
        assert torch.isnan(grad[1, [2, 4]]).all() and torch.isnan(grad[2, 1])
        assert abs(float(grad[3, 6]) - (1 / 9 - 1)) <= 40 * 2.0 ** -24
