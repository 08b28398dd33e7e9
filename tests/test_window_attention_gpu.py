"""Windowed attention with sink keys: forward, backward and the single-token
form against the definition in 64 bits.

Bars, with u half a step of the inputs' type (0 for float32, whose products
are not rounded on the way), a = 2^-25 where that type is float16 (its smallest
step), f = 2^-24, and sums over the seen pairs:
  scores       e_ij = (dim + 8) f scale sum_d |q_d k_d| + 8 f |s_ij|; p is off by
               r_ij = 2 max e + 16 f + n f relative (n terms are added up)
  out          sum_j ((u + r) p_ij + a) |v_j| + half a step of the result
  delta        t_i = (half + dim f) sum_d |o_d g_d| + sum_d |g_d| err(o_d) (o is the rounded output)
  dS           x_ij = (u + r) |dS_ij| + p_ij (t_i + (dim + 4) f sum_d |g_d v_d|) (1 + u) + a
  dq           scale sum_j x_ij |k_j|, dk the same over i, dv sum_i ((u + r) p_ij + a) |g_i|,
               each plus half a step of the result.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
HALF = {torch.float32: F, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ALL = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ms():
    import mlx_sparse

    return mlx_sparse


def _rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()


def _mask(q_len, k_len, window, sinks, bounds=None):
    p = torch.arange(q_len).cuda()[:, None] + (k_len - q_len)
    j = torch.arange(k_len).cuda()[None, :]
    if bounds is None:
        return (j <= p) & (p >= 0) & ((p - j < window) | (j < sinks))
    seen = torch.zeros(q_len, k_len, dtype=torch.bool).cuda()
    for a, b in zip(bounds, bounds[1:]):
        seen[a:b, a:b] = _mask(b - a, b - a, window, sinks)
    return seen


def _reference(q, k, v, seen, scale, g=None):
    """(value, bar) of out and, with g, of dq, dk and dv; rank-4 operands. Rows
    of v, k, q and g that no pair touches are left out, whatever they hold."""
    dtype = q.dtype
    half, u = HALF[dtype], 0.0 if dtype == torch.float32 else HALF[dtype]
    a = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v = (t.detach().double() for t in (q, k, v))
    batch, n, heads, dim = q.shape
    kv = k.shape[2]
    group = heads // kv
    q = torch.where(seen.any(1)[None, :, None, None], q, torch.zeros_like(q))
    k, v = (torch.where(seen.any(0)[None, :, None, None], t, torch.zeros_like(t)) for t in (k, v))
    kk, vv = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    dot = lambda x, y: torch.einsum("bqhd,bkhd->bhqk", x, y)
    s = dot(q, kk) * scale
    e = (dim + 8) * F * abs(scale) * dot(q.abs(), kk.abs()) + 8 * F * s.abs()
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1).masked_fill(~seen, 0.0).masked_fill(~seen.any(1)[:, None], 0.0)
    r = 2 * (e * seen).amax(-1, keepdim=True) + (16 + seen.shape[1]) * F if seen.shape[1] else e
    pull = lambda x, y: torch.einsum("bhqk,bkhd->bqhd", x, y)
    push = lambda x, y: torch.einsum("bhqk,bqhd->bkhd", x, y)
    tiny = torch.finfo(dtype).tiny * half * 2
    out = pull(p, vv)
    out_bar = pull((u + r) * p + a * seen, vv.abs())
    out_bar = out_bar + half * (out.abs() + out_bar) + tiny
    if g is None:
        return [(out, out_bar)]
    g = torch.where(seen.any(1)[None, :, None, None], g.double(), torch.zeros_like(q))
    fold = lambda x: x.reshape(batch, -1, kv, group, dim).sum(3)
    dp = dot(g, vv)
    delta = (g * out).sum(-1).permute(0, 2, 1)[..., None]
    t = (dim * F * (g * out).abs().sum(-1) + (g.abs() * out_bar).sum(-1)).permute(0, 2, 1)[..., None]
    ds = p * (dp - delta)
    x = ((u + r) * ds.abs() + p * (t + (dim + 4) * F * dot(g.abs(), vv.abs())) * (1 + u + r) + a) * seen
    terms = (seen.shape[0] * group + 16) * F
    res = []
    for value, bar, size in (
        (pull(ds, kk) * scale, pull(x, kk.abs()) * abs(scale), pull(ds.abs(), kk.abs()) * abs(scale)),
        (fold(push(ds, q)) * scale, fold(push(x, q.abs())) * abs(scale), fold(push(ds.abs(), q.abs())) * abs(scale)),
        (fold(push(p, g)), fold(push((u + r) * p + a * seen, g.abs())), fold(push(p, g.abs()))),
    ):
        bar = bar + terms * size
        res.append((value, bar + half * (value.abs() + bar) + tiny))
    return [(out, out_bar)] + res


def _check(got, ref, what):
    value, bar = ref
    got = got.detach().double().reshape(value.shape)
    assert torch.isfinite(got).all(), f"{what} is not finite"
    over = (got - value).abs() - bar
    assert over.numel() == 0 or over.max() <= 0, f"{what}: {float(over.max())} above its bar"


def _all(ms, q, k, v, g, **kw):
    leaves = [t.detach().clone().requires_grad_() if t.is_contiguous() else t.detach().requires_grad_()
              for t in (q, k, v)]
    out = ms.window_attention(*leaves, **kw)
    return (out.detach(),) + torch.autograd.grad(out, leaves, g)


# batch, q_len, k_len, q_heads, k_heads, dim, window, sinks
SHAPES = [
    (1, 1, 1, 1, 1, 64, 1, 0),
    (2, 17, 17, 4, 2, 64, 8, 2),
    (1, 130, 130, 3, 1, 80, 200, 0),
    (2, 128, 128, 2, 2, 128, 128, 0),
    (1, 300, 701, 4, 1, 128, 100, 5),
    (1, 129, 40, 2, 1, 64, 16, 3),     # more queries than keys: the first see nothing
    (1, 257, 257, 2, 1, 32, 0, 0),     # nobody sees anything
    (1, 200, 200, 2, 1, 64, 0, 4),     # sinks alone
    (1, 513, 513, 8, 8, 96, 257, 130),  # more sinks than a tile of keys
    (3, 70, 70, 6, 2, 40, 1, 1),
    (1, 400, 400, 2, 2, 8, 64, 70),
    (1, 1, 900, 4, 2, 128, 1000, 0),
    (1, 1100, 1100, 2, 1, 128, 384, 16),
    (1, 900, 500, 2, 1, 64, 60, 3),     # sinks with queries in several chunks: more queries than keys,
    (2, 600, 1500, 4, 2, 64, 70, 4),   # fewer,
    (1, 1100, 1100, 3, 1, 128, 30, 100),  # sinks over most of a tile of keys
    (1, 95, 95, 2, 1, 33, 20, 1),      # head sizes that are the general kernels'
    (1, 40, 40, 2, 1, 256, 11, 2),
    (1, 50, 50, 1, 1, 1, 7, 0),
    (2, 33, 60, 5, 5, 136, 30, 2),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(ms, shape, dtype):
    b, n, m, heads, kv, dim, window, sinks = shape
    q, k, v = _rand((b, n, heads, dim), dtype, 1), _rand((b, m, kv, dim), dtype, 2), _rand((b, m, kv, dim), dtype, 3)
    g = _rand(q.shape, dtype, 4)
    scale = dim ** -0.5
    refs = _reference(q, k, v, _mask(n, m, window, sinks), scale, g)
    got = _all(ms, q, k, v, g, window=window, sinks=sinks)
    for x, ref, name in zip(got, refs, ("out", "dq", "dk", "dv")):
        assert x.dtype == dtype
        _check(x, ref, name)
    with torch.no_grad():
        assert torch.equal(ms.window_attention(q, k, v, window=window, sinks=sinks), got[0])


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("dim", [64, 128, 72, 17])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_packed_sequences(ms, dtype, dim, index):
    bounds = [3, 4, 4, 60, 61, 318, 330, 330, 741, 760]
    tokens, heads, kv, window, sinks = 777, 4, 2, 90, 3
    q, g = _rand((tokens, heads, dim), dtype, 1), _rand((tokens, heads, dim), dtype, 4)
    k, v = _rand((tokens, kv, dim), dtype, 2), _rand((tokens, kv, dim), dtype, 3)
    seen = _mask(tokens, tokens, window, sinks, bounds)
    refs = _reference(q[None], k[None], v[None], seen, dim ** -0.5, g[None])
    ptr = torch.tensor(bounds, dtype=index).cuda()
    got = _all(ms, q, k, v, g, window=window, sinks=sinks, indptr=ptr)
    for x, ref, name in zip(got, refs, ("out", "dq", "dk", "dv")):
        _check(x, ref, name)
        assert (x[:3] == 0).all() and (x[760:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bounds", [[0, 256, 900, 1030, 1800], [0, 250, 270, 1300, 1305, 1800], [100, 255, 257, 1700]])
@pytest.mark.parametrize("sinks", [1, 5, 128])
def test_sinks_of_long_packed_sequences(ms, dtype, bounds, sinks):
    """Sequences that start at, before and behind the 256-query chunks in which
    far queries reach their sinks."""
    tokens, dim = 1850, 64
    q, k, v, g = (_rand((tokens, 2, dim), dtype, s) for s in (1, 2, 3, 4))
    refs = _reference(q[None], k[None], v[None], _mask(tokens, tokens, 40, sinks, bounds), dim ** -0.5, g[None])
    got = _all(ms, q, k, v, g, window=40, sinks=sinks, indptr=torch.tensor(bounds).cuda())
    for x, ref, name in zip(got, refs, ("out", "dq", "dk", "dv")):
        _check(x, ref, name)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 64), (torch.float16, 128)])
def test_many_short_sequences(ms, dtype, dim):
    rng = np.random.default_rng(0)
    bounds = np.concatenate([[0], np.cumsum(rng.integers(0, 6, 300))]).tolist()
    tokens = bounds[-1]
    q, k, v, g = (_rand((tokens, 2, dim), dtype, s) for s in (1, 2, 3, 4))
    refs = _reference(q[None], k[None], v[None], _mask(tokens, tokens, 2, 1, bounds), dim ** -0.5, g[None])
    got = _all(ms, q, k, v, g, window=2, sinks=1, indptr=torch.tensor(bounds).cuda())
    for x, ref, name in zip(got, refs, ("out", "dq", "dk", "dv")):
        _check(x, ref, name)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_mask_hides_does_not_reach_the_rest(ms, dtype, dim, bad):
    """A poisoned sequence, a poisoned tail behind the last sequence, and a
    poisoned token of the same sequence: rows that do not see it, and gradients
    of keys and queries that are not paired with it, keep their values."""
    bounds, tokens, window, sinks = [0, 100, 170, 620], 640, 40, 2
    q, g = _rand((tokens, 4, dim), dtype, 1), _rand((tokens, 4, dim), dtype, 4)
    k, v = _rand((tokens, 2, dim), dtype, 2), _rand((tokens, 2, dim), dtype, 3)
    ptr = torch.tensor(bounds).cuda()
    clean = _all(ms, q, k, v, g, window=window, sinks=sinks, indptr=ptr)
    seen = _mask(tokens, tokens, window, sinks, bounds)
    poisoned = [t.clone() for t in (q, k, v, g)]
    hit = torch.zeros(tokens, dtype=torch.bool).cuda()
    hit[100:170] = True
    hit[620:] = True
    hit[400] = True
    for t in poisoned:
        t[hit] = bad
    got = _all(ms, *poisoned, window=window, sinks=sinks, indptr=ptr)
    rows = ~(hit | (seen & hit[None, :]).any(1))       # queries that see no poisoned key
    # a key's gradients hold from every query that sees it, whose weights depend on all it sees
    keys = ~(hit | (seen & ~rows[:, None]).any(0))
    assert rows.sum() > 300 and keys.sum() > 300
    half = HALF[dtype]
    for x, y, keep, name in zip(got, clean, (rows, rows, keys, keys), ("out", "dq", "dk", "dv")):
        x, y = x[keep].double(), y[keep].double()
        assert torch.isfinite(x).all(), name
        # the same sums in an order that may differ where a tile is recomputed without its hidden entries
        assert ((x - y).abs() <= 4 * half * (y.abs() + y.abs().max())).all(), name
    assert (got[0][620:] == 0).all() and (got[1][620:] == 0).all() and (got[2][620:] == 0).all()


@pytest.mark.parametrize("dtype", ALL)
def test_views_and_shared_heads(ms, dtype):
    b, n, heads, kv, dim = 2, 150, 6, 2, 64
    fused = _rand((b, n, heads + 2 * kv, dim), dtype, 1)
    q, k, v = fused.split((heads, kv, kv), 2)
    g = _rand((b, n, heads, dim), dtype, 4)
    want = _all(ms, q.contiguous(), k.contiguous(), v.contiguous(), g, window=50, sinks=1)
    for x, y in zip(_all(ms, q, k, v, g, window=50, sinks=1), want):
        assert torch.equal(x, y)
    turned = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]  # (batch, heads, tokens, dim)
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:1 + dim] for t in (q, k, v)]         # unaligned rows
    last = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v)]        # strided last dimension
    for views in (turned, odd, last):
        for x, y in zip(_all(ms, *views, g, window=50, sinks=1), want):
            assert torch.equal(x, y)
    # one key head for all, given as a broadcast view: its gradient adds up over the copies
    one = k[:, :, :1].contiguous().requires_grad_()
    vals = v[:, :, :1].contiguous().requires_grad_()
    out = ms.window_attention(q.contiguous(), one.expand(-1, -1, heads, -1), vals.expand(-1, -1, heads, -1), window=50,
                              sinks=1)
    dk, dv = torch.autograd.grad(out, (one, vals), g)
    refs = _reference(q, one, vals, _mask(n, n, 50, 1), dim ** -0.5, g)
    _check(out, refs[0], "out")
    # autograd rounds each head's gradient and their sum to the type
    for x, (value, bar) in ((dk, refs[2]), (dv, refs[3])):
        assert ((x.double() - value).abs() <= (heads + 2) * bar + 2 * heads * HALF[dtype] * value.abs().max()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_some_gradients_and_twice(ms, dtype):
    q, k, v = (_rand((1, 200, 2, 64), dtype, s) for s in (1, 2, 3))
    g = _rand(q.shape, dtype, 4)
    full = _all(ms, q, k, v, g, window=33, sinks=2)
    for pick in range(3):
        leaves = [t.clone() for t in (q, k, v)]
        leaves[pick].requires_grad_()
        out = ms.window_attention(*leaves, window=33, sinks=2)
        out.backward(g, retain_graph=True)
        assert torch.equal(leaves[pick].grad, full[1 + pick])
        out.backward(g)  # accumulates the same once more
        assert torch.equal(leaves[pick].grad, full[1 + pick] * 2)
    x = q.clone().requires_grad_()  # one tensor in all three places
    (d,) = torch.autograd.grad(ms.window_attention(x, x, x, window=33, sinks=2), x, g)
    assert torch.isfinite(d).all()
    for _ in range(3):
        for a, b in zip(_all(ms, q, k, v, g, window=33, sinks=2), full):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_gradients_one_at_a_time_and_output_in_place(ms, dtype):
    q, k, v = (_rand((200, heads, 64), dtype, s) for heads, s in ((4, 1), (2, 2), (2, 3)))
    g = _rand(q.shape, dtype, 4)
    args = dict(window=33, sinks=2, indptr=torch.tensor([0, 90, 200], device="cuda"))
    full = _all(ms, q, k, v, g, **args)
    for pick in range(3):
        leaves = [t.clone() for t in (q, k, v)]
        leaves[pick].requires_grad_()
        out = ms.window_attention(*leaves, **args)
        out.backward(g)
        assert torch.equal(out, full[0]) and torch.equal(leaves[pick].grad, full[1 + pick])
        # the output is a tensor of its own, not a view that refuses to be changed
        ms.window_attention(*leaves, **args).add_(1)
    fused = _rand((200, 8, 64), dtype, 5)
    parts = fused.split((4, 2, 2), 1)
    want = _all(ms, *(t.contiguous() for t in parts), g, **args)
    for x, y in zip(_all(ms, *parts, g, **args), want):
        assert torch.equal(x, y)


def test_gradient_against_differences(ms):
    """float32, along random directions. Each side's value is off by the
    forward's bar; the third derivative of sum(g * out) along a direction of
    unit size stays below 40 sum |g| max |v| for these scores (|ds| <= 4)."""
    b, n, heads, dim, h = 1, 40, 2, 16, 2.0 ** -7
    q, k, v = (_rand((b, n, heads, dim), torch.float32, s) for s in (1, 2, 3))
    g = _rand(q.shape, torch.float32, 4) / (n * heads * dim)
    grads = _all(ms, q, k, v, g, window=9, sinks=2)[1:]
    ins = [q, k, v]
    for pick in range(3):
        d = _rand(q.shape, torch.float32, 10 + pick)
        d = d / d.norm(dim=-1, keepdim=True)
        value = []
        for step in (h, -h):
            moved = list(ins)
            moved[pick] = ins[pick] + step * d
            value.append((ms.window_attention(*moved, window=9, sinks=2).double() * g.double()).sum())
        slope = (grads[pick].double() * d.double()).sum()
        bar = (_reference(q, k, v, _mask(n, n, 9, 2), dim ** -0.5)[0][1] * g.double().abs()).sum()
        tol = 40 * float(g.abs().sum() * v.abs().max()) * h * h / 6 + 2 * float(bar) / h + 1e-6
        assert abs(float((value[0] - value[1]) / (2 * h) - slope)) <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_extreme_scores(ms, dtype):
    """Scores of hundreds: the running maximum keeps every exponential in range."""
    q, k, v = _rand((1, 300, 2, 64), dtype, 1, 8.0), _rand((1, 300, 2, 64), dtype, 2, 8.0), _rand((1, 300, 2, 64), dtype, 3)
    got = ms.window_attention(q, k, v, window=200, sinks=2)
    _check(got, _reference(q, k, v, _mask(300, 300, 200, 2), 0.125)[0], "out")
    lowest = torch.finfo(dtype).min
    k2 = k.clone()
    k2[:, 5] = lowest  # scores of -inf or +inf in some rows: only rows that see it may change
    out = ms.window_attention(q, k2, v, window=20, sinks=0)
    want = ms.window_attention(q, k, v, window=20, sinks=0)
    keep = [i for i in range(300) if not 5 <= i < 25]
    assert torch.equal(out[:, keep], want[:, keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_streams_and_graphs(ms, dtype):
    def inputs(seed):
        return [_rand((2, 260, 4, 64), dtype, seed), _rand((2, 260, 2, 64), dtype, seed + 1),
                _rand((2, 260, 2, 64), dtype, seed + 2), _rand((2, 260, 4, 64), dtype, seed + 3)]

    q, k, v, g = inputs(0)
    want = _all(ms, q, k, v, g, window=70, sinks=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _all(ms, q, k, v, g, window=70, sinks=3)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs = []
    for seed in (10, 20):  # two graphs that live at once
        static = inputs(seed)
        leaves = [t.requires_grad_() for t in static[:3]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ms.window_attention(*leaves, window=70, sinks=3)
            grads = torch.autograd.grad(out, leaves, static[3])
        graphs.append((graph, static, (out.detach(),) + grads))
    for seed in (30, 40):
        for n, (graph, static, res) in enumerate(graphs):
            with torch.no_grad():
                for a, b in zip(static, inputs(seed + n)):
                    a.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for n, (graph, static, res) in enumerate(graphs):
            for a, b in zip(res, _all(ms, *(t.detach() for t in static), window=70, sinks=3)):
                assert torch.equal(a, b)


# batch, max_len, q_heads, k_heads, dim, window, sinks
DECODE = [
    (1, 1, 1, 1, 64, 1, 0),
    (5, 40, 4, 2, 64, 8, 2),
    (3, 700, 8, 1, 128, 300, 4),
    (7, 1500, 6, 2, 80, 2000, 0),
    (2, 4100, 32, 8, 128, 4096, 4),
    (4, 300, 3, 1, 128, 0, 5),
    (4, 300, 2, 2, 96, 0, 0),
    (2, 200, 40, 2, 64, 64, 130),
    (2, 130, 2, 1, 33, 20, 1),
    (2, 130, 4, 2, 256, 50, 2),
    (300, 65, 2, 1, 32, 17, 1),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("shape", DECODE, ids=str)
def test_decode(ms, shape, dtype):
    b, top, heads, kv, dim, window, sinks = shape
    rng = np.random.default_rng(top)
    lengths = rng.integers(0, top + 1, b)
    lengths[0] = top
    q, k, v = _rand((b, heads, dim), dtype, 1), _rand((b, top, kv, dim), dtype, 2), _rand((b, top, kv, dim), dtype, 3)
    for i, n in enumerate(lengths):  # what lies behind a sequence's end is not there yet
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    it = torch.int64 if b % 2 else torch.int32
    got = ms.window_attention_decode(q, k, v, torch.from_numpy(lengths).to(it).cuda(), window=window, sinks=sinks)
    assert got.shape == q.shape and got.dtype == dtype
    for i, n in enumerate(lengths.tolist()):
        if n == 0:
            assert (got[i] == 0).all()
            continue
        ref = _reference(q[i][None, None], k[i, :n][None], v[i, :n][None], _mask(1, n, window, sinks), dim ** -0.5)
        _check(got[i], ref[0], f"sequence {i}")


@pytest.mark.parametrize("dtype", ALL)
def test_decode_masked_tokens_views_and_lengths(ms, dtype):
    b, top, heads, kv, dim = 3, 500, 4, 2, 64
    q = _rand((b, heads, dim), dtype, 1)
    k, v = _rand((b, top, kv, dim), dtype, 2), _rand((b, top, kv, dim), dtype, 3)
    lengths = torch.tensor([500, 77, 301]).cuda()
    want = ms.window_attention_decode(q, k, v, lengths, window=60, sinks=3)
    # lengths outside the cache are clamped, NaN between sinks and window is not seen
    k2, v2 = k.clone(), v.clone()
    k2[0, 3:440], v2[0, 3:440] = float("nan"), float("nan")
    got = ms.window_attention_decode(q, k2, v2, torch.tensor([900, 77, 301]).cuda(), window=60, sinks=3)
    assert torch.equal(got, want)
    assert (ms.window_attention_decode(q, k, v, lengths - 1000, window=60, sinks=3) == 0).all()
    turned = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (k, v)]
    both = torch.stack((k, v), 2)  # keys and values of a token side by side
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:1 + dim] for t in (k, v)]
    for kk, vv in (turned, (both[:, :, 0], both[:, :, 1]), odd):
        assert torch.equal(ms.window_attention_decode(q, kk, vv, lengths, window=60, sinks=3), want)
    qq = _rand((b, heads + 2, dim), dtype, 9)
    qq[:, :heads] = q
    assert torch.equal(ms.window_attention_decode(qq[:, :heads], k, v, lengths, window=60, sinks=3), want)
    graph = torch.cuda.CUDAGraph()
    static = lengths.clone()
    with torch.cuda.graph(graph):
        out = ms.window_attention_decode(q, k, v, static, window=60, sinks=3)
    for new in ([500, 77, 301], [1, 0, 62]):
        static.copy_(torch.tensor(new))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ms.window_attention_decode(q, k, v, static, window=60, sinks=3))


def test_offsets_past_32_bits(ms):
    """A cache of more than 2^32 bytes and 2^31 elements; prompts over a view of it too."""
    b, top, kv, dim = 3, 1 << 20, 8, 128
    k = torch.zeros((b, top, kv, dim), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    tail = slice(top - 300, top)
    for t, seed in ((k, 2), (v, 3)):
        t[:, tail] = _rand((b, 300, kv, dim), torch.bfloat16, seed)
    q = _rand((b, 16, dim), torch.bfloat16, 1)
    lengths = torch.full((b,), top).cuda()
    got = ms.window_attention_decode(q, k, v, lengths, window=300)
    assert torch.equal(got, ms.window_attention_decode(q, k[:, tail], v[:, tail], torch.full((b,), 300).cuda(), window=300))
    chunk = _rand((b, 100, 16, dim), torch.bfloat16, 5)
    assert torch.equal(ms.window_attention(chunk, k, v, window=200),
                       ms.window_attention(chunk, k[:, tail], v[:, tail], window=200))


def test_prompt_then_tokens(ms):
    """Reading a prompt in chunks and then token by token from a cache gives
    what one call over the whole text gives, row by row."""
    n, heads, kv, dim, window, sinks = 230, 4, 2, 64, 50, 2
    q, k, v = (_rand((1, n, h, dim), torch.bfloat16, s) for h, s in ((heads, 1), (kv, 2), (kv, 3)))
    whole = _reference(q, k, v, _mask(n, n, window, sinks), dim ** -0.5)[0]
    rows = [ms.window_attention(q[:, a:b], k[:, :b], v[:, :b], window=window, sinks=sinks)
            for a, b in ((0, 100), (100, 101), (101, 200))]
    for i in range(200, n):
        rows.append(ms.window_attention_decode(q[:, i], k, v, torch.tensor([i + 1]).cuda(), window=window,
                                               sinks=sinks)[:, None])
    _check(torch.cat(rows, 1), whole, "chunks and tokens")


def test_student_learns_from_kept_logits(ms):
    """The operators as they are used together: packed texts through windowed
    attention into logits, the loss against a teacher's kept logits, gradients
    of every weight against 64-bit autograd of the same student."""
    rng = np.random.default_rng(3)
    bounds, vocab, width, heads, kv, dim, T = [0, 90, 91, 240], 331, 64, 4, 2, 32, 2.0
    tokens = bounds[-1]
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(tokens, width, generator=gen).cuda()
    weights = [(torch.randn(s, generator=gen) * s[0] ** -0.5).cuda()
               for s in ((width, (heads + 2 * kv) * dim), (heads * dim, vocab))]
    counts = rng.integers(0, 9, tokens)
    cols = np.concatenate([rng.choice(vocab, c, replace=False) for c in counts])
    ptr = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda()
    data = torch.from_numpy(rng.standard_normal(len(cols)).astype(np.float32) * 3).cuda()
    cot = torch.full((tokens,), 1.0 / tokens).cuda()

    def logits_of(w, attend):
        qkv = (x.to(w[0].dtype) @ w[0]).reshape(tokens, heads + 2 * kv, dim)
        return attend(*qkv.split((heads, kv, kv), 1)).reshape(tokens, heads * dim) @ w[1]

    leaves = [w.clone().requires_grad_() for w in weights]
    logits = logits_of(leaves, lambda q, k, v: ms.window_attention(q, k, v, window=30, sinks=1,
                                                                   indptr=torch.tensor(bounds).cuda()))
    teacher = ms.csr_array((data, torch.from_numpy(cols).cuda(), ptr), shape=(tokens, vocab))
    loss = ms.csr_distillation_loss(teacher, logits, temperature=T)
    got = torch.autograd.grad(loss, leaves, cot, retain_graph=True)
    # the one-pass form gives the same gradient of the logits
    one, g = ms.csr_distillation_loss_and_grad(teacher, logits, cotangent=cot, temperature=T)
    again = torch.autograd.grad(logits, leaves, g)

    wide = [w.double().requires_grad_() for w in weights]
    seen = _mask(tokens, tokens, 30, 1, bounds)

    def attend(q, k, v):
        s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(heads // kv, 1)) * dim ** -0.5
        return torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(~seen, -math.inf), -1),
                            v.repeat_interleave(heads // kv, 1))

    log_q = torch.log_softmax(logits_of(wide, attend) / T, 1)
    ref = torch.zeros(tokens, dtype=torch.float64).cuda()
    for i, (a, b) in enumerate(zip(ptr.tolist(), ptr.tolist()[1:])):
        if b > a:
            lp = torch.log_softmax(data[a:b].double() / T, 0)
            ref[i] = T * T * (lp.exp() * (lp - log_q[i, torch.from_numpy(cols[a:b]).cuda()])).sum()
    want = torch.autograd.grad(ref, wide, cot.double())
    # float32 throughout: sums of at most 240 * 331 terms, exponents below 2^6
    bar = 2.0 ** -24 * 2 ** 10
    assert ((loss.double() - ref).abs() <= bar * (1 + ref.abs())).all() and torch.equal(one, loss)
    for a, b, c in zip(got, again, want):
        scale = c.abs().max()
        assert ((a.double() - c).abs() <= bar * scale).all() and ((b.double() - c).abs() <= bar * scale).all()


@pytest.mark.parametrize("b,n,m", [(0, 5, 5), (2, 0, 4), (2, 3, 0), (1, 0, 0)])
def test_nothing_to_do(ms, b, n, m):
    q, k, v = (torch.ones((b, x, 2, 64), device="cuda", dtype=torch.bfloat16, requires_grad=True) for x in (n, m, m))
    out = ms.window_attention(q, k, v, window=3)
    assert out.shape == q.shape and (out == 0).all()
    out.sum().backward()
    assert (q.grad == 0).all() and (k.grad == 0).all() and (v.grad == 0).all()
    if n == 3:
        none = ms.window_attention_decode(q[:, 0].detach(), k.detach(), v.detach(), torch.tensor([0, 7]).cuda(), window=2)
        assert none.shape == (2, 2, 64) and (none == 0).all()
    if n == m == 5:
        empty = ms.window_attention_decode(q[:, 0].detach(), k.detach(), v.detach(), torch.zeros(0).cuda().int(), window=2)
        assert empty.shape == (0, 2, 64)


def test_boundaries_outside_the_tokens_do_not_reach_memory(ms):
    q, k, v = (_rand((50, 2, 64), torch.bfloat16, s) for s in (1, 2, 3))
    for ptr in ([0, 90], [-20, 30, 70], [10], [60, 80], [30, 10, 50], [0, 2 ** 31 - 1]):
        got = _all(ms, q, k, v, q, window=9, sinks=2, indptr=torch.tensor(ptr, dtype=torch.int32).cuda())
        assert all(torch.isfinite(t).all() for t in got)
    want = ms.window_attention(q, k, v, window=9, sinks=2, indptr=torch.tensor([0, 50]).cuda())
    assert torch.equal(ms.window_attention(q, k, v, window=9, sinks=2, indptr=torch.tensor([0, 90]).cuda()), want)


def test_windows_beyond_64_bits(ms):
    q, k = _rand((1, 70, 2, 64), torch.bfloat16, 1), _rand((1, 70, 2, 64), torch.bfloat16, 2)
    want = ms.window_attention(q, k, k, window=70, sinks=70)
    assert torch.equal(ms.window_attention(q, k, k, window=2 ** 64, sinks=2 ** 65), want)
    n = torch.tensor([70]).cuda()
    assert torch.equal(ms.window_attention_decode(q[:, 0], k, k, n, window=2 ** 64),
                       ms.window_attention_decode(q[:, 0], k, k, n, window=70))


def test_refusals(ms):
    q, k = torch.zeros(1, 4, 4, 64).cuda(), torch.zeros(1, 4, 2, 64).cuda()
    for bad in (dict(window=-1), dict(window=1, sinks=-2), dict(window=1, scale=float("inf"))):
        with pytest.raises(ValueError):
            ms.window_attention(q, k, k, **bad)
    with pytest.raises(TypeError, match="integer"):
        ms.window_attention(q, k, k, window=1.5)
    with pytest.raises(ValueError, match="batch size"):
        ms.window_attention(q, k.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), window=1)
    with pytest.raises(ValueError, match="as many queries"):
        ms.window_attention(q[0], k[0, :3], k[0, :3], window=1, indptr=torch.tensor([0, 3]).cuda())
    with pytest.raises(TypeError, match="indptr dtype"):
        ms.window_attention(q[0], k[0], k[0], window=1, indptr=torch.tensor([0.0, 3.0]).cuda())
    with pytest.raises(ValueError, match="batch size"):
        ms.window_attention_decode(q[:, 0], k, k, torch.tensor([1, 2]).cuda(), window=1)
    with pytest.raises(ValueError, match="no gradient"):
        ms.window_attention_decode(q[:, 0].requires_grad_(), k, k, torch.tensor([1]).cuda(), window=1)
