"""The language-model operators of mlx_sparse, as cases to measure.

Two families share the sparse structure that a windowed student model has on
both ends. ``window_attention`` (and ``window_attention_decode``) is attention
whose score matrix is a band plus a few always-visible first columns;
``csr_distillation_loss`` (and ``csr_distillation_loss_and_grad``) is the loss
against a teacher's stored top logits, a CSR matrix of tokens x vocabulary.

A case is a dict of plain values. ``prepare`` makes its inputs from a seed,
``run`` makes one pass, ``work`` counts what a pass cannot do without and
``exact`` computes the outputs in 64 bits. With ``own`` false ``run`` uses
elementary torch operations in 32 bits, with ``own`` true the calls of
``mlx_sparse``.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-sparse_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import mlx_sparse

    return mlx_sparse


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a prompt of a few words in a small model: nothing but latency
        dict(name="prefill_short", op="prefill", dtype="bfloat16", batch=1, q_len=17, k_len=17, heads=4, kv_heads=1,
             dim=64, window=8, sinks=2),
        # one chunk of a long prompt against the keys that came before it
        dict(name="prefill_chunk", op="prefill", dtype="float16", batch=1, q_len=512, k_len=6001, heads=16,
             kv_heads=4, dim=128, window=1024, sinks=4),
        # a whole long prompt at once
        dict(name="prefill_long", op="prefill", dtype="bfloat16", batch=1, q_len=32768, k_len=32768, heads=32,
             kv_heads=8, dim=128, window=4096, sinks=4),
        # a training step of a small model over short packed texts
        dict(name="train_packed_small", op="train", dtype="float16", tokens=1531, max_seq=300, heads=8, kv_heads=8,
             dim=64, window=128, sinks=1),
        # an ordinary training step: packed texts of ragged lengths
        dict(name="train_packed", op="train", dtype="bfloat16", tokens=16384, max_seq=4000, heads=16, kv_heads=4,
             dim=128, window=1024, sinks=4),
        # a training step over one long text
        dict(name="train_long", op="train", dtype="bfloat16", tokens=16384, max_seq=16384, heads=32, kv_heads=8,
             dim=128, window=2048, sinks=16),
        # one user's next token
        dict(name="decode_one", op="decode", dtype="bfloat16", batch=1, max_len=8192, min_len=5003, heads=32,
             kv_heads=8, dim=128, window=1024, sinks=4),
        # the next token of a full serving batch, caches of all lengths
        dict(name="decode_batch", op="decode", dtype="bfloat16", batch=128, max_len=8192, min_len=0, heads=32,
             kv_heads=8, dim=128, window=4096, sinks=4),
        # loss and gradient of a handful of tokens over a toy vocabulary
        dict(name="distill_small", op="loss_and_grad", dtype="float32", rows=7, vocab=1031, top=8, temperature=2.0,
             index="int32"),
        # a training step through autograd, 32-bit logits
        dict(name="distill_train", op="loss_train", dtype="float32", rows=2048, vocab=32000, top=32, temperature=2.0,
             index="int32"),
        # a large step over a large vocabulary: loss and gradient in one call
        dict(name="distill_large", op="loss_and_grad", dtype="bfloat16", rows=8192, vocab=128000, top=64,
             temperature=1.0, index="int64"),
        # evaluation on held-out text: the loss alone, a vocabulary of odd size
        dict(name="distill_eval", op="loss", dtype="bfloat16", rows=4096, vocab=50021, top=20, temperature=1.0,
             index="int32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefill", "train", "decode", "loss", "loss_train", "loss_and_grad"])
    if op.startswith("loss"):
        vocab = _log_int(rng, 500, 160000)
        rows = _log_int(rng, 1, max(1, min(8192, 2 ** 30 // vocab)))
        return dict(op=op, dtype=rng.choice(["float32", "float16", "bfloat16"]), rows=rows, vocab=vocab,
                    top=_log_int(rng, 1, min(256, vocab // 4)), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                    index=rng.choice(["int32", "int64"]))
    kv_heads = rng.choice([1, 2, 4, 8])
    case = dict(op=op, dtype=rng.choice(["float16", "bfloat16"]), heads=kv_heads * rng.choice([1, 2, 3, 4, 8]),
                kv_heads=kv_heads, dim=rng.choice([32, 64, 80, 96, 128]), window=_log_int(rng, 16, 4096),
                sinks=rng.choice([0, 1, 4, 7, 16, 64]))
    if op == "decode":
        max_len = _log_int(rng, 64, 8192)
        case.update(batch=_log_int(rng, 1, 128), max_len=max_len, min_len=rng.choice([0, max_len // 2, max_len]))
    elif op == "train":
        # at most the work of the largest listed training step
        tokens = _log_int(rng, 100, max(101, 2 ** 25 // max(case["window"] * case["heads"] // 16, 128)))
        tokens = min(tokens, 16384)
        case.update(tokens=tokens, max_seq=_log_int(rng, max(2, tokens // 32), tokens))
    else:
        batch = rng.choice([1, 1, 2, 4])
        k_len = min(32768, _log_int(rng, 16, max(17, 2 ** 26 // max(case["window"] * case["heads"] * batch // 16, 64))))
        case.update(batch=batch, k_len=k_len, q_len=rng.choice([k_len, k_len, max(1, k_len // 5)]))
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _sequence_lengths(case, seed):
    """Ragged lengths of packed texts; the last one takes what is left."""
    gen = torch.Generator().manual_seed(seed * 7919 + 17)
    left, out = case["tokens"], []
    while left > 0:
        n = min(left, int(torch.randint(1, case["max_seq"] + 1, (1,), generator=gen)))
        if case["max_seq"] >= case["tokens"]:
            n = left
        out.append(n)
        left -= n
    return out


def _cache_lengths(case, seed):
    gen = torch.Generator().manual_seed(seed * 6007 + 5)
    return torch.randint(case["min_len"], case["max_len"] + 1, (case["batch"],), generator=gen).tolist()


def _top_counts(case, seed):
    """Entries kept for each row: about `top`, none for rows that are not trained on (prompts, padding)."""
    gen = torch.Generator().manual_seed(seed * 104729 + 3)
    n = torch.randint(max(1, case["top"] // 2), case["top"] + case["top"] // 2 + 1, (case["rows"],), generator=gen)
    n = n.clamp(max=case["vocab"] // 2)
    if case["rows"] > 4:
        n[torch.rand(case["rows"], generator=gen) < 0.1] = 0
    return n


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    op = case["op"]
    state = dict(case=case)
    if op.startswith("loss"):
        counts = _top_counts(case, seed)
        index = torch.int32 if case["index"] == "int32" else torch.int64
        rows, vocab = case["rows"], case["vocab"]
        indptr = torch.zeros(rows + 1, dtype=torch.int64)
        indptr[1:] = torch.cumsum(counts, 0)
        row = torch.repeat_interleave(torch.arange(rows), counts).cuda()
        place = torch.arange(int(indptr[-1]), device="cuda") - indptr.cuda()[row]
        first = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        most = max(1, int(counts.max()))
        step = torch.randint(1, vocab // most + 1, (rows,), generator=gen, device="cuda")
        column = (first[row] + step[row] * place) % vocab  # distinct in a row, in no order
        # the teacher's logits fall off from the first to the last kept one
        data = 12.0 - 2.0 * torch.log1p(place.float()) + 0.3 * torch.randn(row.shape, generator=gen, device="cuda")
        logits = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.0
        logits.index_put_((row, column), 0.6 * data, accumulate=True)
        weights = torch.full((rows,), 1.0 / max(1, int((counts > 0).sum())), device="cuda")
        state.update(data=data.to(dtype), indices=column.to(index), indptr=indptr.to(index).cuda(),
                     logits=logits.to(dtype), weights=weights)
        if own:
            ms = _package()
            state["teacher"] = ms.csr_array((state["data"], state["indices"], state["indptr"]), shape=(rows, vocab))
            if op == "loss_train":
                state["logits"].requires_grad_()
        return state
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if op == "decode":
        lengths = _cache_lengths(case, seed)
        cache = (case["batch"], case["max_len"], kv_heads, dim)
        state.update(q=_normal(gen, (case["batch"], heads, dim), dtype), k=_normal(gen, cache, dtype),
                     v=_normal(gen, cache, dtype), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                     host_lengths=lengths)
        return state
    if op == "train":
        lengths = _sequence_lengths(case, seed)
        lead = (case["tokens"],)
        state["host_lengths"] = lengths
        ptr = torch.zeros(len(lengths) + 1, dtype=torch.int32)
        ptr[1:] = torch.cumsum(torch.tensor(lengths), 0)
        state["indptr"] = ptr.cuda()
        q_lead = k_lead = lead
    else:
        q_lead, k_lead = (case["batch"], case["q_len"]), (case["batch"], case["k_len"])
    state.update(q=_normal(gen, q_lead + (heads, dim), dtype), k=_normal(gen, k_lead + (kv_heads, dim), dtype),
                 v=_normal(gen, k_lead + (kv_heads, dim), dtype))
    if op == "train":
        state["grad"] = _normal(gen, q_lead + (heads, dim), dtype)
        if own:
            for name in "qkv":
                state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return _PLAIN[op](state)
    ms = _package()
    if op.startswith("loss"):
        if op == "loss_and_grad":
            return ms.csr_distillation_loss_and_grad(state["teacher"], state["logits"], cotangent=state["weights"],
                                                     temperature=case["temperature"])
        loss = ms.csr_distillation_loss(state["teacher"], state["logits"], temperature=case["temperature"])
        if op == "loss":
            return loss
        (grad,) = torch.autograd.grad(loss, state["logits"], state["weights"])
        return loss.detach(), grad
    band = dict(window=case["window"], sinks=case["sinks"])
    if op == "decode":
        return ms.window_attention_decode(state["q"], state["k"], state["v"], state["lengths"], **band)
    if op == "prefill":
        return ms.window_attention(state["q"], state["k"], state["v"], **band)
    out = ms.window_attention(state["q"], state["k"], state["v"], indptr=state["indptr"], **band)
    grads = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["grad"])
    return (out.detach(),) + grads


# ---------------------------------------------------------------------------
# Plain forms: elementary torch operations in 32 bits
# ---------------------------------------------------------------------------
def _chunks(q_len, k_len, window, sinks, size=512):
    """Query rows in chunks with the key positions that any of them sees."""
    for start in range(0, q_len, size):
        stop = min(q_len, start + size)
        position = torch.arange(start, stop, device="cuda") + (k_len - q_len)
        last = k_len - q_len + stop
        low = max(0, k_len - q_len + start - window + 1)
        keys = torch.arange(min(low, max(last, 0)), max(last, 0), device="cuda")
        keys = torch.cat((torch.arange(min(sinks, low, max(last, 0)), device="cuda"), keys))
        ahead = position[:, None] - keys[None, :]
        seen = (ahead >= 0) & ((ahead < window) | (keys[None, :] < sinks))
        yield slice(start, stop), keys, seen


def _weights(q, k, seen, scale):
    """Softmax over the seen keys, zero rows where none is seen: (kv_heads, group, queries, keys)."""
    s = torch.einsum("qhgd,khd->hgqk", q, k) * scale
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:-1] + (1,))
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _attend(q, k, v, window, sinks, grad=None):
    """One sequence: q (queries, heads, dim), k and v (keys, kv_heads, dim), 32 bits."""
    n, heads, dim = q.shape
    kv_heads = k.shape[1]
    scale = 1.0 / math.sqrt(dim)
    q = q.reshape(n, kv_heads, heads // kv_heads, dim)
    out = torch.zeros_like(q)
    if grad is not None:
        grad = grad.reshape(q.shape)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for rows, keys, seen in _chunks(n, k.shape[0], window, sinks):
        kc, vc = k[keys], v[keys]
        p = _weights(q[rows], kc, seen, scale)
        out[rows] = torch.einsum("hgqk,khd->qhgd", p, vc)
        if grad is None:
            continue
        g = grad[rows]
        dp = torch.einsum("qhgd,khd->hgqk", g, vc)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
        dq[rows] = torch.einsum("hgqk,khd->qhgd", ds, kc)
        dk.index_add_(0, keys, torch.einsum("hgqk,qhgd->khd", ds, q[rows]))
        dv.index_add_(0, keys, torch.einsum("hgqk,qhgd->khd", p, g))
    out = out.reshape(n, heads, dim)
    return out if grad is None else (out, dq.reshape(n, heads, dim), dk, dv)


def _plain_prefill(state):
    case = state["case"]
    q, k, v = (state[x].float() for x in "qkv")
    out = [_attend(q[b], k[b], v[b], case["window"], case["sinks"]) for b in range(case["batch"])]
    return torch.stack(out).to(state["q"].dtype)


def _plain_train(state):
    case = state["case"]
    dtype = state["q"].dtype
    parts, start = [], 0
    for n in state["host_lengths"]:
        rows = slice(start, start + n)
        q, k, v, g = (state[x][rows].float() for x in ("q", "k", "v", "grad"))
        parts.append(_attend(q, k, v, case["window"], case["sinks"], g))
        start += n
    return tuple(torch.cat(x).to(dtype) for x in zip(*parts))


def _plain_decode(state):
    case = state["case"]
    q = state["q"]
    out = torch.zeros_like(q)
    for b, n in enumerate(state["host_lengths"]):
        if n:
            low = max(0, n - case["window"])
            head = min(case["sinks"], low)
            k = torch.cat((state["k"][b, :head], state["k"][b, low:n])).float()
            v = torch.cat((state["v"][b, :head], state["v"][b, low:n])).float()
            seen = torch.ones((1, k.shape[0]), dtype=torch.bool, device="cuda")
            split = q[b:b + 1].float().reshape(1, case["kv_heads"], -1, case["dim"])
            p = _weights(split, k, seen, 1.0 / math.sqrt(case["dim"]))
            out[b] = torch.einsum("hgqk,khd->qhgd", p, v).reshape(case["heads"], case["dim"]).to(q.dtype)
    return out


def _plain_distill(state, want_loss=True, want_grad=True):
    case = state["case"]
    logits = state["logits"].detach()
    rows, vocab = logits.shape
    temperature = case["temperature"]
    indptr = state["indptr"].long()
    row = torch.repeat_interleave(torch.arange(rows, device="cuda"), indptr.diff())
    column = state["indices"].long()
    t = state["data"].float() / temperature
    top = torch.full((rows,), -math.inf, device="cuda").scatter_reduce(0, row, t, "amax")
    e = torch.exp(t - top[row])
    total = torch.zeros(rows, device="cuda").index_add_(0, row, e)
    p = e / total[row]
    log_p = t - top[row] - torch.log(total)[row]
    loss = torch.zeros(rows, device="cuda")
    grad = torch.empty_like(logits) if want_grad else None
    bounds = list(range(0, rows, 1024)) + [rows]
    cuts = indptr[torch.tensor(bounds, device="cuda")].tolist()
    for a, b, lo, hi in zip(bounds, bounds[1:], cuts, cuts[1:]):
        z = logits[a:b].float() / temperature
        peak = z.amax(1, keepdim=True)
        ez = torch.exp(z - peak)
        mass = ez.sum(1, keepdim=True)
        r, c, q = row[lo:hi] - a, column[lo:hi], p[lo:hi]
        log_q = z[r, c] - peak[r, 0] - torch.log(mass)[r, 0]
        loss[a:b].index_add_(0, r, q * (log_p[lo:hi] - log_q) * temperature * temperature)
        if want_grad:
            ez /= mass
            ez.index_put_((r, c), -q, accumulate=True)
            live = (indptr[a:b] < indptr[a + 1:b + 1]).float()
            grad[a:b] = (ez * (temperature * state["weights"][a:b] * live)[:, None]).to(logits.dtype)
    return loss, grad


_PLAIN = {
    "prefill": _plain_prefill,
    "train": _plain_train,
    "decode": _plain_decode,
    "loss": lambda s: _plain_distill(s, want_grad=False)[0],
    "loss_train": _plain_distill,
    "loss_and_grad": _plain_distill,
}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(q_len, k_len, window, sinks):
    """Visible (query, key) pairs and the keys that any query sees."""
    total = 0
    for i in range(q_len):
        p = i + k_len - q_len
        if p >= 0:
            low = max(0, p - window + 1)
            total += p + 1 - low + min(sinks, low)
    low = max(0, k_len - q_len - window + 1)
    return total, max(0, k_len - low) + min(sinks, low)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op = case["op"]
    if op.startswith("loss"):
        elements = case["rows"] * case["vocab"]
        kept = case["rows"] * case["top"]
        index = 4 if case["index"] == "int32" else 8
        bytes_ = elements * size + kept * (size + index) + case["rows"] * (index + 4)
        if op != "loss":
            bytes_ += elements * size + 4 * case["rows"]
        return {"bytes": bytes_, "flops": elements * (4 if op == "loss" else 6)}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    window, sinks = case["window"], case["sinks"]
    if op == "decode":
        mean = (case["min_len"] + case["max_len"]) // 2
        pairs, keys = _pairs(1, mean, window, sinks)
        return {"bytes": case["batch"] * size * dim * (2 * heads + 2 * keys * kv_heads) + 4 * case["batch"],
                "flops": 4 * case["batch"] * pairs * heads * dim}
    if op == "train":
        tokens = case["tokens"]
        pairs = sum(_pairs(n, n, window, sinks)[0] for n in _sequence_lengths(case, 0))
        # forward q k v -> out; backward reads them and out's gradient again and writes three gradients
        return {"bytes": size * dim * tokens * (4 * heads + 4 * kv_heads), "flops": (4 + 10) * pairs * heads * dim}
    pairs, keys = _pairs(case["q_len"], case["k_len"], window, sinks)
    return {"bytes": case["batch"] * size * dim * (2 * heads * case["q_len"] + 2 * kv_heads * keys),
            "flops": 4 * case["batch"] * pairs * heads * dim}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_head(q, k, v, window, sinks, grad=None, step=2048):
    """One head of one sequence from the definition: every score, masked."""
    q, k, v = q.double(), k.double(), v.double()
    n, m, scale = q.shape[0], k.shape[0], q.shape[1] ** -0.5
    j = torch.arange(m, device=q.device)
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for a in range(0, n, step):
        i = torch.arange(a, min(n, a + step), device=q.device) + m - n
        hi = int(i[-1]) + 1
        if hi <= 0:
            continue
        hidden = (j[:hi] > i[:, None]) | ((j[:hi] <= i[:, None] - window) & (j[:hi] >= sinks))
        x = (q[a:a + step] @ k[:hi].T * scale).masked_fill_(hidden, -math.inf)
        p = torch.softmax(x, 1).masked_fill_(hidden.all(1, keepdim=True), 0.0)
        out[a:a + step] = p @ v[:hi]
        if grad is not None:
            g = grad[a:a + step].double()
            d = p * (g @ v[:hi].T - (g * out[a:a + step]).sum(1, keepdim=True))
            dq[a:a + step] = d @ k[:hi] * scale
            dk[:hi] += d.T @ q[a:a + step] * scale
            dv[:hi] += p.T @ g
    return out, dq, dk, dv


def _exact_sequence(q, k, v, window, sinks, grad=None):
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(out), torch.zeros_like(k, dtype=torch.float64), torch.zeros_like(v, dtype=torch.float64)
    for h in range(q.shape[1]):
        g = None if grad is None else grad[:, h]
        o, a, b, c = _exact_head(q[:, h], k[:, h // group], v[:, h // group], window, sinks, g)
        out[:, h], dq[:, h] = o, a
        dk[:, h // group] += b
        dv[:, h // group] += c
    return out, dq, dk, dv


def _exact_distill(state):
    """Loss from the definition, its gradient by formula, a few rows at a time."""
    case = state["case"]
    T = case["temperature"]
    ptr = state["indptr"].tolist()
    logits = state["logits"].detach()
    loss = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    grad = torch.zeros(logits.shape, dtype=torch.float64, device="cuda") if case["op"] != "loss" else None
    for i in range(case["rows"]):
        a, b = ptr[i], ptr[i + 1]
        if a == b:
            continue
        column = state["indices"][a:b].long()
        log_p = torch.log_softmax(state["data"][a:b].double() / T, 0)
        log_q = torch.log_softmax(logits[i].double() / T, 0)
        loss[i] = T * T * torch.dot(torch.exp(log_p), log_p - log_q[column])
        if grad is not None:
            torch.exp(log_q, out=grad[i])
            grad[i].index_add_(0, column, -torch.exp(log_p))
            grad[i] *= T * state["weights"][i].double()
    return loss if grad is None else (loss, grad)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op.startswith("loss"):
        return _exact_distill(state)
    q, k, v = (state[x].detach() for x in "qkv")
    window, sinks = case["window"], case["sinks"]
    if op == "decode":
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for b, n in enumerate(state["host_lengths"]):
            j = torch.arange(n, device="cuda")
            j = j[(j >= n - window) | (j < sinks)]
            if len(j) == 0:
                continue
            kb = k[b, j].double().repeat_interleave(group, 1)
            vb = v[b, j].double().repeat_interleave(group, 1)
            x = (kb * q[b].double()).sum(2) * case["dim"] ** -0.5
            out[b] = (torch.softmax(x, 0)[:, :, None] * vb).sum(0)
        return out
    if op == "prefill":
        return torch.stack([_exact_sequence(q[b], k[b], v[b], window, sinks)[0] for b in range(case["batch"])])
    parts, start = [], 0
    for n in state["host_lengths"]:
        rows = slice(start, start + n)
        parts.append(_exact_sequence(q[rows], k[rows], v[rows], window, sinks, state["grad"][rows]))
        start += n
    return tuple(torch.cat(x) for x in zip(*parts))
