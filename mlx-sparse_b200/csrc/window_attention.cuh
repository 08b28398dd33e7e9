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
  int64_t lse_row;    // floats of lse (delta) for each head: q_len rounded up to whole tiles; both negated
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

// The keys that the queries [first, last] see: [low, end) and, before it, the
// sink keys [sink0, sink_end) of the first query's sequence. (A sequence that
// starts further on has its sinks in [low, end).) Positions rise with the
// queries and so do the lower ends of their bands, so the ends decide.
struct KeyRange {
  int sink0, sink_end, low, end;
  __device__ __forceinline__ bool empty() const { return end <= low && sink_end <= sink0; }
  __device__ __forceinline__ bool touches(int j0, int j1) const {
    return (j0 < end && j1 > low && end > low) || (j0 < sink_end && j1 > sink0);
  }
};

__device__ __forceinline__ KeyRange key_range(const WindowProblem &w, int b, int first, int last) {
  const int shift = key_count(w, b) - (int)w.c.q_len;
  int lo = max(first, max(0, -shift)), hi = min(last, (int)w.c.q_len - 1);
  if (w.c.indptr != nullptr) {
    const int64_t n = w.c.n_seq;
    auto at = [&](int64_t r) -> int64_t {
      return w.wide_ptr ? static_cast<const int64_t *>(w.c.indptr)[r]
                        : (int64_t) static_cast<const int32_t *>(w.c.indptr)[r];
    };
    lo = (int)max((int64_t)lo, min(at(0), (int64_t)INT_MAX));
    hi = (int)min((int64_t)hi, max(at(n), (int64_t)0) - 1);
  }
  KeyRange r{0, 0, 0, 0};
  if (lo > hi) return r;
  const QuerySpan s = query_span(w, b, lo);
  if (s.p < 0) return r;
  r.low = s.low, r.end = hi + shift + 1;
  r.sink0 = s.start, r.sink_end = max(s.start, min(s.start + w.sinks, s.low));
  return r;
}

// A range as tiles of N keys: the sink keys' tiles, then the band's.
template <int N> struct KeyTiles {
  int sink0, low, n_sink, n;
  __device__ __forceinline__ explicit KeyTiles(const KeyRange &r)
      : sink0(r.sink0), low(r.low), n_sink((r.sink_end - r.sink0 + N - 1) / N),
        n(n_sink + (max(r.end - r.low, 0) + N - 1) / N) {}
  __device__ __forceinline__ int first(int t) const { return t < n_sink ? sink0 + t * N : low + (t - n_sink) * N; }
  // end of the tile's own keys: a sink tile stops where the band begins
  __device__ __forceinline__ int end(int t) const {
    const int e = first(t) + N;
    return t < n_sink ? min(e, low) : e;
  }
};

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
// ... and for the tensor cores (window_forward_tc.cu, window_backward_tc.cu).
bool window_tc_ok(const WindowProblem &w, int value_dtype);
void window_forward_tc(const WindowProblem &w, int value_dtype, cudaStream_t s);
void window_backward_tc(const WindowProblem &w, int value_dtype, cudaStream_t s);
int64_t window_backward_floats_tc(const WindowProblem &w);  // workspace behind delta
// One query for each sequence (window_decode.cu).
void window_decode(const WindowProblem &w, int value_dtype, cudaStream_t s);
void window_delta(const WindowProblem &w, int value_dtype, cudaStream_t s);

}  // namespace msx
