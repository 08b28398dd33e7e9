"""Distillation against a CSR matrix of teacher logits: loss, autograd and the
one-pass form against the definition in 64 bits.

Bars. Every exponent x = c z - max is formed by one fma from inputs that the
64-bit side shares, so it is off by (|x| + |c z|) 2^-24 for c's and the fma's
rounding; ex2.approx adds 2^-22, a sum of n positive terms kept by one thread
n 2^-24. With M the largest |x| of a row in base 2 and n = V / 256 + 32 adds a
thread, p, q and both logarithms are within
    e = (8 + 4 M + n) 2^-24
relative (p, q) or absolute (logarithms), the loss within T^2 e (sum p (|log p|
+ |log q|) + 2), and the gradient within w T (q + p) e plus half a step of its
type.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


def _case(rows, vocab, top, dtype, index=torch.int32, seed=0, empty=()):
    """Ragged rows of distinct columns in no order; rows in `empty` have none."""
    rng = np.random.default_rng(seed)
    cols, ptr = [], [0]
    for i in range(rows):
        k = 0 if i in empty else int(rng.integers(1, min(top, vocab) + 1))
        cols.append(rng.choice(vocab, k, replace=False) if vocab < 100000 else rng.permutation(
            np.unique(rng.integers(0, vocab, k))))
        ptr.append(ptr[-1] + len(cols[-1]))
    cols = np.concatenate(cols)
    data = torch.from_numpy(rng.standard_normal(len(cols)) * 3 + 4).to(dtype).cuda()
    logits = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 3).to(dtype).cuda()
    return (data, torch.from_numpy(cols).to(index).cuda(), torch.tensor(ptr).to(index).cuda()), logits


def _reference(parts, logits, T, w):
    """Loss, gradient and their bars, float64."""
    data, idx, ptr = (t.cpu() for t in parts)
    z = logits.detach().cpu().double()
    rows, vocab = z.shape
    loss, bar = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    grad, gbar = torch.zeros_like(z), torch.zeros_like(z)
    for i in range(rows):
        a, b = int(ptr[i]), int(ptr[i + 1])
        if a == b:
            continue
        c = idx[a:b].long()
        lp = torch.log_softmax(data[a:b].double() / T, 0)
        lq = torch.log_softmax(z[i] / T, 0)
        p, q = lp.exp(), lq.exp()
        finite, kept = (x[torch.isfinite(x)].tolist() + [0.0] for x in (z[i], data[a:b].double()))
        M = max(finite) - min(finite) + max(map(abs, finite)) + 2 * max(map(abs, kept))
        e = (8 + 4 * M / T * 1.4427 + vocab / 256 + 32) * 2.0 ** -24
        term = torch.where(p > 0, p * (lp - lq[c]), torch.zeros_like(p))
        loss[i] = T * T * term.sum()
        weight = torch.where(p > 0, p * (lp.abs() + lq[c].abs()), torch.zeros_like(p))
        bar[i] = T * T * e * (weight.sum() + 2)
        full = torch.zeros(vocab, dtype=torch.float64).index_add_(0, c, p)
        grad[i] = w[i] * T * (q - full)
        gbar[i] = abs(w[i]) * T * (q + full) * e
    half = HALF[logits.dtype]
    return loss, bar, grad, gbar + grad.abs() * half + TINY[logits.dtype]


def _check(got, want, bar, what):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    worst = ((got - want).abs() - bar).max()
    assert worst <= 0, f"{what}: {float(worst)} above its bar"


SHAPES = [(1, 1, 1), (3, 7, 2), (5, 33, 5), (7, 1031, 8), (4, 50021, 20), (700, 257, 3), (3, 128000, 300)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss_and_gradient(ms, shape, dtype):
    rows, vocab, top = shape
    T = 2.0
    index = torch.int64 if rows % 2 else torch.int32
    parts, logits = _case(rows, vocab, top, dtype, index, seed=vocab, empty=(1,) if rows > 2 else ())
    teacher = ms.csr_array(parts, shape=(rows, vocab))
    w = torch.linspace(0.25, 1.0, rows)
    loss, bar, grad, gbar = _reference(parts, logits, T, w.double())
    one, one_grad = ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=w.cuda(), temperature=T)
    _check(one, loss, bar, "one-pass loss")
    _check(one_grad, grad, gbar, "one-pass gradient")
    assert one.dtype == torch.float32 and one_grad.dtype == dtype
    leaf = logits.clone().requires_grad_()
    two = ms.csr_distillation_loss(teacher, leaf, temperature=T)
    _check(two, loss, bar, "loss")
    (two * w.cuda()).sum().backward()
    _check(leaf.grad, grad, gbar, "gradient")
    with torch.no_grad():
        _check(ms.csr_distillation_loss(teacher, leaf, temperature=T), loss, bar, "loss without a graph")


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 900001), (torch.bfloat16, 300007), (torch.float16, 13000003)])
def test_rows_beyond_one_sm(ms, dtype, vocab):
    """Rows that are read twice, and one too long for a bit a column in shared memory."""
    parts, logits = _case(2, vocab, 40, dtype, seed=3)
    teacher = ms.csr_array(parts, shape=(2, vocab))
    loss, bar, grad, gbar = _reference(parts, logits, 1.0, torch.ones(2, dtype=torch.float64))
    got, got_grad = ms.csr_distillation_loss_and_grad(teacher, logits)
    _check(got, loss, bar, "loss")
    _check(got_grad, grad, gbar, "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows_beyond_shared_memory(ms, dtype):
    """More rows than SMs: a cluster of two that reads each half row again."""
    rows, vocab = 400, 70001
    parts, logits = _case(rows, vocab, 12, dtype, seed=9, empty=(0, 17))
    teacher = ms.csr_array(parts, shape=(rows, vocab))
    w = torch.linspace(0.5, 1.0, rows)
    loss, bar, grad, gbar = _reference(parts, logits, 1.0, w.double())
    got, got_grad = ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=w.cuda())
    _check(got, loss, bar, "loss")
    _check(got_grad, grad, gbar, "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_logits(ms, dtype):
    rows, vocab = 6, 1003
    parts, logits = _case(rows, vocab, 9, dtype, seed=5)
    teacher = ms.csr_array(parts, shape=(rows, vocab))
    want = ms.csr_distillation_loss_and_grad(teacher, logits)
    for pad, shift in ((5, 1), (8, 3), (0, 0)):
        wide = torch.full((rows, vocab + pad), float("nan"), dtype=dtype, device="cuda")
        view = wide[:, shift:shift + vocab]
        view.copy_(logits)
        got = ms.csr_distillation_loss_and_grad(teacher, view)
        ref = _reference(parts, logits, 1.0, torch.ones(rows, dtype=torch.float64))
        _check(got[0], ref[0], ref[1], "loss")
        _check(got[1], ref[2], ref[3], "gradient")
        assert got[1].is_contiguous()
    turned = logits.t().contiguous().t()
    got = ms.csr_distillation_loss_and_grad(teacher, turned)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    same_row = logits[:1].expand(rows, vocab)  # stride 0 between rows
    assert ms.csr_distillation_loss(teacher, same_row).shape == (rows,)


def test_rows_left_out_and_infinities(ms):
    inf, nan = float("inf"), float("nan")
    rows, vocab = 6, 40
    data = torch.tensor([1.0, 2.0, 3.0, -inf, 0.5, 1.0, 2.0, 1.0, 1.0]).cuda()
    idx = torch.tensor([3, 7, 1, 39, 0, 5, 6, 2, 4], dtype=torch.int32).cuda()
    ptr = torch.tensor([0, 2, 2, 4, 6, 8, 9], dtype=torch.int32).cuda()
    logits = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(1)).cuda()
    logits[1] = nan          # no entries: zeros all the same
    logits[2, 39] = -inf     # the teacher gives it no mass either: 0 log 0 = 0
    logits[3, 10:20] = -inf  # masked vocabulary outside the entries
    logits[4, 6] = -inf      # the teacher wants it: infinite loss, finite gradient
    logits[5] = nan          # weight 0: gradient 0
    teacher = ms.csr_array((data, idx, ptr), shape=(rows, vocab))
    w = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 0.0]).cuda()
    loss, grad = ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=w)
    leaf = logits.clone().requires_grad_()
    two = ms.csr_distillation_loss(teacher, leaf)
    (auto,) = torch.autograd.grad(two, leaf, w)
    for lo, g in ((loss, grad), (two, auto)):
        assert lo[1] == 0 and (g[1] == 0).all()
        assert torch.isinf(lo[4]) and torch.isfinite(g[4]).all() and torch.isnan(lo[5]) and (g[5] == 0).all()
        assert (g[3, 10:20] == 0).all()
        keep = [0, 2, 3]
        ref = _reference((data, idx, ptr), logits, 1.0, torch.ones(rows, dtype=torch.float64))
        _check(lo[keep], ref[0][keep], ref[1][keep], "loss")
        _check(g[keep], ref[2][keep], ref[3][keep], "gradient")


def test_nan_stays_in_its_row(ms):
    parts, logits = _case(5, 3001, 6, torch.float32, seed=8)
    teacher = ms.csr_array(parts, shape=(5, 3001))
    clean = ms.csr_distillation_loss_and_grad(teacher, logits)
    logits[2, 1500] = float("nan")
    loss, grad = ms.csr_distillation_loss_and_grad(teacher, logits)
    assert torch.isnan(loss[2]) and torch.isnan(grad[2]).all()
    keep = [0, 1, 3, 4]
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(grad[keep], clean[1][keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeated_columns_add_up(ms, dtype):
    vocab = 70001
    rng = np.random.default_rng(4)
    idx = np.concatenate([[5, 5, 5, 69999, 5, 12, 69999], rng.integers(0, 50, 900)])
    ptr = torch.tensor([0, 7, 907], dtype=torch.int64).cuda()
    data = torch.from_numpy(rng.standard_normal(907)).to(dtype).cuda()
    logits = torch.from_numpy(rng.standard_normal((2, vocab)) * 2).to(dtype).cuda()
    parts = (data, torch.from_numpy(idx).cuda(), ptr)
    loss, bar, grad, gbar = _reference(parts, logits, 1.0, torch.ones(2, dtype=torch.float64))
    teacher = ms.csr_array(parts, shape=(2, vocab))
    first = ms.csr_distillation_loss_and_grad(teacher, logits)
    _check(first[0], loss, bar, "loss")
    _check(first[1], grad, gbar, "gradient")
    leaf = logits.clone().requires_grad_()
    (auto,) = torch.autograd.grad(ms.csr_distillation_loss(teacher, leaf).sum(), leaf)
    _check(auto, grad, gbar, "autograd gradient")
    for _ in range(5):
        again = ms.csr_distillation_loss_and_grad(teacher, logits)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_gradient_against_differences(ms):
    """Along a direction d with |d| <= 1 the third derivative of a row's loss
    is at most 8 / T: the central difference at step h is off by 8 h^2 / (6 T),
    and by the losses' own error over h."""
    rows, vocab, T, h = 4, 501, 1.5, 2.0 ** -5
    parts, logits = _case(rows, vocab, 10, torch.float32, seed=11)
    teacher = ms.csr_array(parts, shape=(rows, vocab))
    d = torch.rand(rows, vocab, generator=torch.Generator().manual_seed(2)).cuda() * 2 - 1
    leaf = logits.clone().requires_grad_()
    (g,) = torch.autograd.grad(ms.csr_distillation_loss(teacher, leaf, temperature=T).sum(), leaf)
    slope = (g.double() * d.double()).sum(1).cpu()
    up = ms.csr_distillation_loss(teacher, logits + h * d, temperature=T).double().cpu()
    down = ms.csr_distillation_loss(teacher, logits - h * d, temperature=T).double().cpu()
    bar = _reference(parts, logits, T, torch.ones(rows, dtype=torch.float64))[1]
    # logits + h d is rounded: 2^-23 of |z| <= 16 in each of two terms, weighted by |q - p| <= 2 in all
    tol = 8 * h * h / (6 * T) + 2 * bar / h + T * 2 * 16 * 2.0 ** -23 / h
    assert ((up - down) / (2 * h) - slope).abs().le(tol).all()


def test_bad_columns_and_offsets_do_not_reach_memory(ms):
    """Columns outside the vocabulary make their row NaN; offsets outside the
    arrays are clamped. The other rows keep their values."""
    data = torch.ones(6).cuda()
    idx = torch.tensor([1, 2, 50, -3, 0, 4]).cuda()
    logits = torch.randn(3, 10, generator=torch.Generator().manual_seed(1)).cuda()
    teacher = ms.csr_array((data, idx, torch.tensor([0, 2, 4, 6]).cuda()), shape=(3, 10))
    loss, grad = ms.csr_distillation_loss_and_grad(teacher, logits)
    assert torch.isnan(loss[1]) and torch.isfinite(loss[[0, 2]]).all() and torch.isfinite(grad).all()
    loose = ms.csr_array((data, idx, torch.tensor([-7, 2, 9, 5]).cuda()), shape=(3, 10))
    got, _ = ms.csr_distillation_loss_and_grad(loose, logits)
    assert got[0] == loss[0] and got[2] == 0


@pytest.mark.parametrize("rows,vocab", [(0, 50), (4, 0), (0, 0)])
def test_nothing_to_do(ms, rows, vocab):
    empty = torch.zeros(0).cuda()
    teacher = ms.csr_array((empty, empty.int(), torch.zeros(rows + 1, dtype=torch.int32).cuda()), shape=(rows, vocab))
    logits = torch.zeros(rows, vocab, device="cuda", requires_grad=True)
    loss, grad = ms.csr_distillation_loss_and_grad(teacher, logits)
    assert loss.tolist() == [0.0] * rows and grad.shape == (rows, vocab)
    ms.csr_distillation_loss(teacher, logits).sum().backward()
    assert logits.grad.shape == (rows, vocab)


def test_streams_and_graphs(ms):
    parts, logits = _case(64, 5003, 12, torch.bfloat16, seed=21)
    teacher = ms.csr_array(parts, shape=(64, 5003))
    want = ms.csr_distillation_loss_and_grad(teacher, logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ms.csr_distillation_loss_and_grad(teacher, logits)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    static = logits.clone().requires_grad_()

    def step():
        loss = ms.csr_distillation_loss(teacher, static)
        return loss.detach(), torch.autograd.grad(loss.sum(), static)[0]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step()
    for seed in (1, 2):
        new = torch.randn(64, 5003, generator=torch.Generator().manual_seed(seed)).cuda().bfloat16()
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        ref = step()
        assert torch.equal(loss, ref[0]) and torch.equal(grad, ref[1])


def test_refusals(ms):
    parts, logits = _case(3, 20, 4, torch.float32)
    teacher = ms.csr_array(parts, shape=(3, 20))
    with pytest.raises(TypeError, match="CSRArray"):
        ms.csr_distillation_loss(logits, logits)
    with pytest.raises(ValueError, match="teacher's shape"):
        ms.csr_distillation_loss(teacher, logits[:2])
    with pytest.raises(TypeError, match="same dtype"):
        ms.csr_distillation_loss(teacher, logits.half())
    with pytest.raises(ValueError, match="temperature"):
        ms.csr_distillation_loss_and_grad(teacher, logits, temperature=0.0)
    with pytest.raises(ValueError, match="cotangent must have shape"):
        ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=torch.ones(4).cuda())
    with pytest.raises(TypeError, match="cotangent must be float32"):
        ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=torch.ones(3).cuda().half())
    learnt = ms.csr_array((parts[0].clone().requires_grad_(),) + parts[1:], shape=(3, 20))
    with pytest.raises(ValueError, match="constant"):
        ms.csr_distillation_loss(learnt, logits)
