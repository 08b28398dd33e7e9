// Windowed attention: what the general and the tensor-core kernels share.
//
// Queries and keys have positions; query position p sees key j iff they are of
// one sequence, j <= p, and p - j < window or j - start < sinks, where start is
// the sequence's first position. Unpacked: every batch entry is one sequence,
// query i is at p = i + k_len - q_len. Packed: batch 1, the sequences lie one
// after another along the tokens, query i is at p = i, and `indptr` holds the
// sequence boundaries; tokens outside them see nothing. With `lengths`, batch
// entry b has only the first lengths[b] of the k_len keys.
#pragma once
#include "common.cuh"
#include "ops.cuh"

namespace msx {

struct WindowProblem {
  WindowCall c;
  int group;    // query heads for each key head
  int offset;   // position of query 0
  int wide_ptr; // indptr or lengths are int64
  int window, sinks;  // clamped to k_len
};

// Sequence of a position: [start, end), empty (start = end) outside all.
__device__ __forceinline__ void sequence_of(const WindowProblem &w, int p, int &start, int &end) {
  start = 0, end = (int)w.c.k_len;
  if (w.c.indptr == nullptr) return;
  auto at = [&](int64_t r) -> int64_t {
    return w.wide_ptr ? static_cast<const int64_t *>(w.c.indptr)[r] : (int64_t) static_cast<const int32_t *>(w.c.indptr)[r];
  };
  int64_t lo = 0, hi = w.c.n_seq;  // boundary lo <= p, boundary hi > p
  if (hi < 1 || at(0) > p || at(hi) <= p) {
    start = end = 0;
    return;
  }
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (at(mid) <= p) lo = mid; else hi = mid;
  }
  start = (int)max((int64_t)0, at(lo));
  end = (int)min((int64_t)w.c.k_len, at(hi));
}

// What one query sees: [start, sink_end) and [low, p]; nothing if p < low.
struct QuerySpan {
  int start, sink_end, low, p;
  __device__ __forceinline__ bool sees(int j) const { return (j >= low && j <= p) || (j >= start && j < sink_end); }
  __device__ __forceinline__ bool empty() const { return p < low && sink_end <= start; }
};

__device__ __forceinline__ int key_count(const WindowProblem &w, int b) {
  if (w.c.lengths == nullptr) return (int)w.c.k_len;
  const int64_t n = w.wide_ptr ? static_cast<const int64_t *>(w.c.lengths)[b]
                               : (int64_t) static_cast<const int32_t *>(w.c.lengths)[b];
  return (int)max((int64_t)0, min(n, w.c.k_len));
}

__device__ __forceinline__ QuerySpan query_span(const WindowProblem &w, int b, int i) {
  QuerySpan s{0, 0, 0, -1};
  if (i >= w.c.q_len) return s;
  const int p = i + key_count(w, b) - (int)w.c.q_len;
  if (p < 0) return s;
  int start, end;
  sequence_of(w, p, start, end);
  if (start >= end) return s;
  s.start = start, s.p = p;
  s.low = max(start, p - w.window + 1);
  s.sink_end = min(start + w.sinks, s.low);
  return s;
}

// The query positions that see one key: [j, last]; nothing if last < j.
__device__ __forceinline__ int last_query(const WindowProblem &w, int j) {
  if (j >= w.c.k_len) return -1;
  int start, end;
  sequence_of(w, j, start, end);
  if (start >= end) return -1;
  return j - start < w.sinks ? end - 1 : min(end - 1, j + w.window - 1);
}

// Kernels for every type and head size (window_attention.cu) ...
void window_forward_general(const WindowProblem &w, int value_dtype, cudaStream_t s);
void window_backward_general(const WindowProblem &w, int value_dtype, cudaStream_t s);

}  // namespace msx
