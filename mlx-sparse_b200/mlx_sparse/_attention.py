"""Windowed attention: products with a score matrix that is sparse by rule.

The score matrix of a sliding window is a band; a few first tokens ("sinks")
stay visible to every later query and add full columns. No pattern is stored:
the kernels walk the band and the sink columns only, as ``csr_matmul_data_vjp``
followed by ``csr_matmul`` would walk a stored pattern, with the softmax between
the two products kept on chip. Results are enqueued on the current CUDA stream
and nothing synchronises.
"""

from __future__ import annotations

import torch

from mlx_sparse import _native
from mlx_sparse._validation import check_index_dtype, check_rank1, ensure_array, refuse_tangents, validate_window_inputs


def window_attention(q, k, v, *, window: int, sinks: int = 0, scale=None, indptr=None):
    """``softmax(scale * q k^T) v`` over a sliding window and sink tokens.

    Query position ``p`` sees key ``j`` of its own sequence iff ``j <= p`` and
    (``p - j < window`` or ``j < sinks``, counted from the sequence's start). A
    query that sees nothing has output 0 and gradient 0.

    * Batched: ``q`` (batch, q_len, q_heads, dim), ``k`` and ``v`` (batch,
      k_len, k_heads, dim). Queries are the last ``q_len`` positions: query
      ``i`` is at ``i + k_len - q_len`` (a chunk of a prompt against the keys
      before it; with more queries than keys the first ones see nothing).
    * Packed: ``q`` (tokens, q_heads, dim), ``k`` and ``v`` (tokens, k_heads,
      dim) and ``indptr`` (sequences + 1 boundaries, int32 or int64, as a CSR
      row pointer): sequences lie one after another. Tokens before the first
      or behind the last boundary belong to none: they see nothing, are seen by
      none and get zeros. Boundaries are read on the device and not checked;
      they must not decrease.

    ``q_heads`` is a multiple of ``k_heads``; query head ``h`` reads key head
    ``h // (q_heads // k_heads)``. float32, float16 or bfloat16, head sizes up
    to 256; sums and the softmax are held in float32. 16-bit inputs with a head
    size that is a multiple of 8 up to 128 run on the tensor cores; these round
    the probabilities ``p``, and in the backward pass ``p * (dp - delta)`` too, to
    the inputs' type before the products that sum them (in float32). float16 rows
    where the latter is beyond the type's range are computed again in float32, which
    takes longer. ``scale`` defaults to ``dim ** -0.5``. Inputs may be strided
    views; a view whose last dimension is strided, or whose 16-bit rows do not
    start on 16-byte boundaries, is copied first.

    Differentiable (once, in reverse mode; inputs with forward-mode tangents are
    refused) in ``q``, ``k`` and ``v``. A training step can be captured
    into a CUDA graph under torch's rule for it: no eager graph of the same leaves
    may be alive meanwhile.
    """
    refuse_tangents("window_attention", q, k, v)
    q = ensure_array(q)
    k, v = ensure_array(k, device=q.device), ensure_array(v, device=q.device)
    if indptr is None:
        window, sinks, scale = validate_window_inputs(q, k, v, window, sinks, scale, rank=4, name="window_attention")
        if q.shape[0] != k.shape[0]:
            raise ValueError(f"window_attention q and k must have one batch size, got {q.shape[0]} and {k.shape[0]}.")
    else:
        window, sinks, scale = validate_window_inputs(q, k, v, window, sinks, scale, rank=3, name="window_attention")
        indptr = ensure_array(indptr, device=q.device)
        check_rank1("window_attention indptr", indptr)
        check_index_dtype("window_attention indptr", indptr)
        if indptr.shape[0] < 1:
            raise ValueError("window_attention indptr must hold at least one boundary.")
        if q.shape[0] != k.shape[0]:
            raise ValueError(
                f"window_attention with indptr needs as many queries as keys, got {q.shape[0]} and {k.shape[0]}."
            )
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        from mlx_sparse._autodiff import WindowAttention

        return WindowAttention.apply(q, k, v, window, sinks, scale, indptr)
    return _native.window_attention_forward(q, k, v, window, sinks, scale, indptr, with_lse=False)[0]


def window_attention_decode(q, k_cache, v_cache, lengths, *, window: int, sinks: int = 0, scale=None):
    """One next token for each sequence of a batch: ``window_attention`` of a
    single query at the end of its cache.

    ``q`` (batch, q_heads, dim); ``k_cache`` and ``v_cache`` (batch, max_len,
    k_heads, dim), of which sequence ``b`` holds its first ``lengths[b]`` tokens,
    the query's own among them; what lies behind is not read into the result.
    ``lengths`` (batch,) int32 or int64 is read on the device and clamped to
    ``[0, max_len]``; a sequence of length 0 gets zeros. Only the window and the
    sink tokens are read. Types, heads and scale as ``window_attention``. Not
    differentiable: it refuses inputs that require a gradient or carry a tangent.
    """
    name = "window_attention_decode"
    refuse_tangents(name, q, k_cache, v_cache)
    q = ensure_array(q)
    k_cache, v_cache = ensure_array(k_cache, device=q.device), ensure_array(v_cache, device=q.device)
    lengths = ensure_array(lengths, device=q.device)
    if q.ndim != 3 or k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError(f"{name} expects q of rank 3 and caches of rank 4, got {q.ndim}, {k_cache.ndim} and "
                         f"{v_cache.ndim}.")
    window, sinks, scale = validate_window_inputs(q.unsqueeze(1), k_cache, v_cache, window, sinks, scale, rank=4,
                                                  name=name)
    check_rank1(f"{name} lengths", lengths)
    check_index_dtype(f"{name} lengths", lengths)
    if not q.shape[0] == k_cache.shape[0] == lengths.shape[0]:
        raise ValueError(f"{name} q, caches and lengths must have one batch size, got {q.shape[0]}, "
                         f"{k_cache.shape[0]} and {lengths.shape[0]}.")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise ValueError(f"{name} has no gradient; use window_attention, or call it under torch.no_grad().")
    return _native.window_attention_decode(q, k_cache, v_cache, lengths, window, sinks, scale)
