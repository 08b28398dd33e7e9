// Distillation against a teacher's stored top logits (a CSR matrix, tokens x
// vocabulary), forward, backward, and both in one pass over the logits.
//
// For a row with teacher entries t_e at columns c_e and student logits z:
//   p_e  = softmax_e(t_e / T)               over the row's stored entries
//   q_j  = softmax_j(z_j / T)               over the whole vocabulary
//   loss = T^2 sum_e p_e (log p_e - log q_{c_e})
//   dloss/dz_j = T (q_j - sum_{e: c_e = j} p_e)
// A row without entries has loss 0 and gradient 0 whatever its logits hold.
// Entries that share a column are terms of their own; their p add up in the
// gradient. Everything is computed in base 2 (c = log2(e) / T) and in fp32;
// the gradient is rounded once, to the logits' type.
//
// Bound: HBM (8192 x 128000 bf16: forward 0.34 ms, backward 0.67 ms, both in one
// pass 0.90 ms, where the special-function unit, with two exponentials and a
// conversion for each logit, is busy 63% of the time and DRAM moves 72% of what a copy
// does). Forward reads the logits once, the backward pass reads them
// again and writes the gradient. The one-pass form reads HBM about once and writes
// once, two thirds of the bytes of the two passes: a row's logits stay on chip
// between the sum of the exponentials and the gradient, in shared memory where
// they fit (spread over a cluster where there are too few rows to fill the SMs),
// else in L2, from where the CTA that summed the row reads it again (2048 x 128000
// bf16: 634 MB read from DRAM for 524 MB of logits, a fifth of the second reads miss).
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "ops.cuh"

namespace cg = cooperative_groups;

namespace msx {
namespace {

constexpr float kNegInf = -INFINITY;

// Per-row softmax statistics kept for the backward pass.
struct RowStats {
  float z_max, z_inv;  // c max_j z_j and 1 / sum_j 2^(c z_j - z_max)
  float t_max, t_inv;  // the same of the teacher's entries
};

constexpr int kMaxKept = 200 * 1024;  // dynamic shared memory, at most
constexpr int kKeepMost = 64 * 1024;  // slices up to this are kept in shared memory
// Longer ones are read again, in slices of 128 KB: four CTAs an SM then have few
// enough bytes between their two reads for L2 (8192 x 128000 bf16, in one series of
// runs: 860 us with a cluster of two, 947 with whole rows, all of whose second reads
// miss, 1095 with four slices and their waits; 900 on other days).
constexpr int kRereadMost = 128 * 1024;
constexpr int kRereadThreads = 384;

struct DistillArgs {
  const void *logits;
  int64_t ld;  // elements between rows of the logits
  const void *t_data, *t_idx, *t_ptr;
  int64_t nnz, rows, vocab;
  float c, temperature;
  const float *cot;  // null: ones
  float *loss;
  RowStats *stats;
  void *grad;  // contiguous (rows, vocab)
  int64_t slice;  // columns of a row for each CTA of its cluster
  int n_slices;
};

// ex2.approx: at most 2 ulp, results below 2^-126 flushed to zero; the
// probabilities lost there are below fp32's smallest normal number.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> struct Vec;  // 16 bytes of T
template <> struct Vec<float> {
  static constexpr int n = 4;
  __device__ static void unpack(const uint4 &v, float *f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float *f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  __device__ static void unpack(const uint4 &v, float *f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  __device__ static uint4 pack(const float *f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  __device__ static void unpack(const uint4 &v, float *f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 pack(const float *f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Running maximum m of the logits and sum of 2^(z c - b) with b = m c rounded. A sum
// that is still empty has m = -inf, b = 0 and sum 0; a NaN ends up in the sum. Sums
// over different maxima are joined by the difference of their rounded b: the
// product of an unrounded m c would leave the rounding's error in the sum, once
// for every join.
struct MaxSum {
  float m = kNegInf, b = 0.f, s = 0.f;
  __device__ void raise(float top, float c) {
    const float up = __fmul_rn(top, c);
    if (m != kNegInf) s *= exp2_fast(b - up);
    m = top, b = up;
  }
  template <int N> __device__ void add(const float *z, float c) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    if (top > m) raise(top, c);
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp2_fast(fmaf(z[i], c, -b));
  }
  __device__ void join(float m2, float s2, float c) {
    if (m2 > m) raise(m2, c);
    s += m2 == m || m2 == kNegInf ? s2 : s2 * exp2_fast(__fmul_rn(m2, c) - b);
  }
};

// Joins every thread's pair; thread order is fixed, so the result is too.
__device__ MaxSum block_join(MaxSum v, float c, float2 *warp_part) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float m2 = __shfl_xor_sync(~0u, v.m, d), s2 = __shfl_xor_sync(~0u, v.s, d);
    v.join(m2, s2, c);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) warp_part[warp] = make_float2(v.m, v.s);
  __syncthreads();
  MaxSum r;
  for (int w = 0; w < n; ++w) r.join(warp_part[w].x, warp_part[w].y, c);
  return r;
}

__device__ float block_sum(float v, float *warp_part) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) r += warp_part[w];
  return r;
}

// The row's entries, clamped into the arrays.
template <typename I> __device__ void row_range(const DistillArgs &a, int64_t row, int64_t &lo, int64_t &hi) {
  const I *ptr = static_cast<const I *>(a.t_ptr);
  lo = max((int64_t)0, min((int64_t)ptr[row], a.nnz));
  hi = max(lo, min((int64_t)ptr[row + 1], a.nnz));
}

template <typename T> __device__ MaxSum teacher_stats(const DistillArgs &a, int64_t lo, int64_t hi, float2 *part) {
  const T *t = static_cast<const T *>(a.t_data);
  MaxSum v;
  for (int64_t e = lo + threadIdx.x; e < hi; e += blockDim.x) {
    const float x = VT<T>::load(t[e]);
    v.add<1>(&x, a.c);
  }
  return block_join(v, a.c, part);
}

// T^2 sum_e p_e (log p_e - log q_{c_e}); entries with p = 0 add nothing (0 log
// 0 = 0), an entry outside the vocabulary makes the loss NaN.
template <typename T, typename I>
__device__ float row_loss(const DistillArgs &a, const T *z, int64_t lo, int64_t hi, const RowStats &st, float z_sum,
                          float t_sum, float *part) {
  const T *t = static_cast<const T *>(a.t_data);
  const I *idx = static_cast<const I *>(a.t_idx);
  const float lg_z = log2f(z_sum), lg_t = log2f(t_sum);
  float v = 0.f;
  for (int64_t e = lo + threadIdx.x; e < hi; e += blockDim.x) {
    const int64_t col = (int64_t)idx[e];
    const float lp = fmaf(VT<T>::load(t[e]), a.c, -st.t_max) - lg_t;
    const float p = exp2_fast(lp);
    if (col < 0 || col >= a.vocab) {
      v = NAN;
    } else if (!(p == 0.f)) {
      const float lq = fmaf(VT<T>::load(z[col]), a.c, -st.z_max) - lg_z;
      v = fmaf(p, lp - lq, v);
    }
  }
  return block_sum(v, part) * (a.temperature * a.temperature * 0.69314718055994531f);
}

// The columns [c0, c1) of a row as 16-byte vectors of the row's own alignment:
// `head` loose elements, `nvec` vectors, `tail` loose elements.
template <typename T> struct SliceShape {
  int head, tail, nvec;
  __device__ SliceShape(const T *p, int64_t n) {
    const int mis = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    head = (int)min((int64_t)(mis ? Vec<T>::n - mis : 0), n);
    nvec = (int)((n - head) / Vec<T>::n);
    tail = (int)(n - head - (int64_t)nvec * Vec<T>::n);
  }
};

// Subtracts the teacher's probabilities from the gradient of columns [c0, c1):
// the gradient of every entry's column is recomputed and rounded once. `bits`
// (a bit for each column) finds columns that occur twice; only then the
// probabilities are added up in `table`, some columns at a time and only those near
// a column that occurred twice: as integers, so that their order does not matter,
// of a step that follows the largest probability of the column, 2^52 or so steps
// for a thousand entries, so that sums of small ones keep fp32's accuracy.
constexpr int kSumBytes = 12;  // of the table for each column: the sum and the largest term

template <typename T, typename I>
__device__ void subtract_teacher(const DistillArgs &a, const T *z, T *g, int64_t lo, int64_t hi, int64_t c0,
                                 int64_t c1, const RowStats &st, float scale, uint32_t *bits, void *table,
                                 int64_t table_bytes) {
  __shared__ uint32_t near_twice[2];  // blocks of columns, modulo 64, with one that occurs twice
  const T *t = static_cast<const T *>(a.t_data);
  const I *idx = static_cast<const I *>(a.t_idx);
  const int64_t n = table_bytes / kSumBytes;
  unsigned long long *sum = static_cast<unsigned long long *>(table);
  uint32_t *top = reinterpret_cast<uint32_t *>(sum + n);
  const int words = (int)((c1 - c0 + 31) / 32);
  for (int w = threadIdx.x; w < words; w += blockDim.x) bits[w] = 0;
  if (threadIdx.x < 2) near_twice[threadIdx.x] = 0;
  __syncthreads();  // also: the gradient of this slice is written
  auto p_of = [&](int64_t e) { return exp2_fast(fmaf(VT<T>::load(t[e]), a.c, -st.t_max)) * st.t_inv; };
  auto put = [&](int64_t col, float p) {
    const float q = exp2_fast(fmaf(VT<T>::load(z[col]), a.c, -st.z_max)) * st.z_inv;
    g[col] = VT<T>::store((q - p) * scale);
  };
  int twice = 0;
  for (int64_t e = lo + threadIdx.x; e < hi; e += blockDim.x) {
    const int64_t col = (int64_t)idx[e];
    if (col < c0 || col >= c1) continue;
    const uint32_t bit = 1u << ((col - c0) & 31);
    if (atomicOr(&bits[(col - c0) >> 5], bit) & bit) {
      const int64_t block = (col - c0) / n;
      twice = 1;
      atomicOr(&near_twice[block >> 5 & 1], 1u << (block & 31));
    }
    put(col, p_of(e));
  }
  if (!__syncthreads_or(twice) || !isfinite(st.t_inv)) return;  // a row of NaN keeps the NaN that is there
  const int steps = 62 - (64 - __clzll(hi - lo));  // all entries' terms, each below 2^steps, fit 62 bits
  int64_t block = 0;
  for (int64_t b0 = c0; b0 < c1; b0 += n, ++block) {
    if (!(near_twice[block >> 5 & 1] >> (block & 31) & 1)) continue;
    const int64_t b1 = min(c1, b0 + n);
    auto each = [&](auto f) {
      for (int64_t e = lo + threadIdx.x; e < hi; e += blockDim.x) {
        const int64_t col = (int64_t)idx[e];
        if (col >= b0 && col < b1) f(col, (int)(col - b0), p_of(e));
      }
      __syncthreads();
    };
    for (int64_t j = threadIdx.x; j < b1 - b0; j += blockDim.x) sum[j] = 0, top[j] = 0;
    __syncthreads();
    each([&](int64_t, int j, float p) { atomicMax(&top[j], __float_as_uint(p)); });
    each([&](int64_t, int j, float p) {
      const float most = __uint_as_float(top[j]);  // below 2^(ilogb + 1)
      if (most > 0.f) atomicAdd(&sum[j], __double2ull_rn(ldexp((double)p, steps - 1 - ilogbf(most))));
    });
    each([&](int64_t col, int j, float) {
      const float most = __uint_as_float(top[j]);
      put(col, most > 0.f ? (float)ldexp((double)sum[j], ilogbf(most) + 1 - steps) : 0.f);
    });
  }
}

// Writes zeros to g[c0, c1).
template <typename T> __device__ void zero_slice(T *g, int64_t n) {
  const SliceShape<T> sh(g, n);
  for (int i = threadIdx.x; i < sh.head + sh.tail; i += blockDim.x) {
    const int64_t j = i < sh.head ? i : n - 1 - (i - sh.head);
    g[j] = VT<T>::store(0.f);
  }
  uint4 *v = reinterpret_cast<uint4 *>(g + sh.head);
  for (int i = threadIdx.x; i < sh.nvec; i += blockDim.x) __stcs(v + i, make_uint4(0, 0, 0, 0));
}

// Stores a vector of gradients at g (aligned like the logits or not).
template <typename T> __device__ __forceinline__ void store_vec(T *g, const float *f, bool aligned) {
  const uint4 v = Vec<T>::pack(f);
  if (aligned) {
    __stcs(reinterpret_cast<uint4 *>(g), v);
  } else {
    T e[Vec<T>::n];
    *reinterpret_cast<uint4 *>(e) = v;
#pragma unroll
    for (int i = 0; i < Vec<T>::n; ++i) g[i] = e[i];
  }
}

__device__ __forceinline__ void cp_async16(void *smem, const void *gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem)
               : "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kThreads = 256;
constexpr int kGroups = 4;  // commit groups of a slice: the sums start when the first quarter is there

// What a CTA does with its slice of a row after the sum: nothing (the forward
// pass alone), or the gradient, from the slice in shared memory or from a second
// read of it.
enum class Grad { none, kept, reread };
constexpr int kTableBytes = 8192;  // for repeated entries' sums, where the slice does not leave its space to them

// One cluster for each row, one slice of the row for each CTA. Registers are held to
// what lets 48 warps run on an SM where the loads are waited for (forward alone: 0.33
// ms against 0.37 at 32 warps).
template <typename T, typename I, Grad MODE, int TH>
__global__ void __launch_bounds__(TH, MODE == Grad::kept ? 1024 / TH : 1536 / TH) distill_row_kernel(const DistillArgs a) {
  constexpr bool KEEP = MODE == Grad::kept;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ float2 part[TH / 32];
  __shared__ float2 ranks[16];
  constexpr int N = Vec<T>::n;
  cg::cluster_group cluster = cg::this_cluster();
  const int n_ranks = a.n_slices;
  const int rank = (int)(blockIdx.x % n_ranks);
  const int64_t row = blockIdx.x / n_ranks;
  int64_t lo, hi;
  row_range<I>(a, row, lo, hi);
  const int64_t c0 = min(a.vocab, (int64_t)rank * a.slice), c1 = min(a.vocab, c0 + a.slice);
  T *g = MODE == Grad::none ? nullptr : static_cast<T *>(a.grad) + row * a.vocab;
  if (lo == hi) {  // every CTA of the cluster leaves
    if (rank == 0 && threadIdx.x == 0) {
      a.loss[row] = 0.f;
      if (a.stats) a.stats[row] = RowStats{0.f, 0.f, 0.f, 0.f};
    }
    if (MODE != Grad::none) zero_slice(g + c0, c1 - c0);
    return;
  }
  const T *z = static_cast<const T *>(a.logits) + row * a.ld;
  const SliceShape<T> sh(z + c0, c1 - c0);
  if (n_ranks > 1) cluster.barrier_arrive();  // waited for before the first access to another CTA's memory
  const uint4 *src = reinterpret_cast<const uint4 *>(z + c0 + sh.head);
  uint4 *kept = reinterpret_cast<uint4 *>(dyn);
  const int tid = threadIdx.x;

  MaxSum ms;
  float loose = 0.f;  // this thread's head or tail element
  const int64_t loose_col = tid < sh.head ? c0 + tid : c1 - 1 - (tid - sh.head);
  const bool has_loose = tid < sh.head + sh.tail;
  if (has_loose) loose = VT<T>::load(z[loose_col]);
  if (KEEP) {
    const int per = (sh.nvec + TH * kGroups - 1) / (TH * kGroups);
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      for (int it = q * per; it < (q + 1) * per; ++it) {
        const int i = tid + it * TH;
        if (i < sh.nvec) cp_async16(kept + i, src + i);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // each thread reads back only what it copied itself, so its own wait is enough
    auto take = [&](int q) {
      for (int it = q * per; it < (q + 1) * per; ++it) {
        const int i = tid + it * TH;
        if (i < sh.nvec) {
          float f[N];
          Vec<T>::unpack(kept[i], f);
          ms.add<N>(f, a.c);
        }
      }
    };
    cp_async_wait<3>(), take(0);
    cp_async_wait<2>(), take(1);
    cp_async_wait<1>(), take(2);
    cp_async_wait<0>(), take(3);
  } else {
    constexpr int U = 4;  // 16-byte loads in flight for each thread
    int i = tid;
    for (; i + (U - 1) * TH < sh.nvec; i += U * TH) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = MODE == Grad::none ? __ldcs(src + i + u * TH) : src[i + u * TH];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        Vec<T>::unpack(v[u], f);
        ms.add<N>(f, a.c);
      }
    }
    for (; i < sh.nvec; i += TH) {
      float f[N];
      Vec<T>::unpack(src[i], f);
      ms.add<N>(f, a.c);
    }
  }
  if (has_loose) ms.add<1>(&loose, a.c);
  MaxSum all = block_join(ms, a.c, part);
  const MaxSum ts = teacher_stats<T>(a, lo, hi, part);
  if (n_ranks > 1) {
    cluster.barrier_wait();
    if (tid < n_ranks) *cluster.map_shared_rank(&ranks[rank], tid) = make_float2(all.m, all.s);
    cluster.sync();
    all = MaxSum();
    for (int r = 0; r < n_ranks; ++r) all.join(ranks[r].x, ranks[r].y, a.c);
  }
  const RowStats st{all.b, 1.f / all.s, ts.b, 1.f / ts.s};
  if (rank == 0) {
    const float loss = row_loss<T, I>(a, z, lo, hi, st, all.s, ts.s, reinterpret_cast<float *>(part));
    if (tid == 0) {
      a.loss[row] = loss;
      if (a.stats) a.stats[row] = st;
    }
  }
  if (MODE == Grad::none) return;
  const float w = a.cot ? a.cot[row] : 1.f;
  if (w == 0.f) {
    zero_slice(g + c0, c1 - c0);
    return;
  }
  const float scale = w * a.temperature;
  const float qs = st.z_inv * scale;
  T *dst = g + c0 + sh.head;
  const bool aligned = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
  auto put = [&](int i, const uint4 &v) {
    float f[N];
    Vec<T>::unpack(v, f);
#pragma unroll
    for (int u = 0; u < N; ++u) f[u] = exp2_fast(fmaf(f[u], a.c, -st.z_max)) * qs;
    store_vec(dst + (int64_t)i * N, f, aligned);
  };
  if (KEEP) {
    for (int i = tid; i < sh.nvec; i += TH) put(i, kept[i]);
  } else {
    constexpr int U = 4;
    int i = tid;
    for (; i + (U - 1) * TH < sh.nvec; i += U * TH) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = __ldcs(src + i + u * TH);
#pragma unroll
      for (int u = 0; u < U; ++u) put(i + u * TH, v[u]);
    }
    for (; i < sh.nvec; i += TH) put(i, __ldcs(src + i));
  }
  if (has_loose) g[loose_col] = VT<T>::store(exp2_fast(fmaf(loose, a.c, -st.z_max)) * qs);
  __syncthreads();  // the slice in shared memory is done with: its space serves the teacher's entries
  const int64_t bits_bytes = (c1 - c0 + 127) / 128 * 16;
  subtract_teacher<T, I>(a, z, g, lo, hi, c0, c1, st, scale, reinterpret_cast<uint32_t *>(dyn), dyn + bits_bytes,
                         KEEP ? a.slice * (int64_t)sizeof(T) - bits_bytes : kTableBytes);
}

// The backward pass from the forward's statistics: one CTA for each slice.

template <typename T, typename I>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const DistillArgs a) {
  extern __shared__ __align__(16) unsigned char dyn[];
  constexpr int N = Vec<T>::n, U = 4;
  const int64_t row = blockIdx.x / a.n_slices;
  const int64_t c0 = (int64_t)(blockIdx.x % a.n_slices) * a.slice, c1 = min(a.vocab, c0 + a.slice);
  int64_t lo, hi;
  row_range<I>(a, row, lo, hi);
  T *g = static_cast<T *>(a.grad) + row * a.vocab;
  const float w = a.cot ? a.cot[row] : 1.f;
  if (lo == hi || w == 0.f) {
    zero_slice(g + c0, c1 - c0);
    return;
  }
  const RowStats st = a.stats[row];
  const T *z = static_cast<const T *>(a.logits) + row * a.ld;
  const SliceShape<T> sh(z + c0, c1 - c0);
  const uint4 *src = reinterpret_cast<const uint4 *>(z + c0 + sh.head);
  const int tid = threadIdx.x;
  const float scale = w * a.temperature, qs = st.z_inv * scale;
  T *dst = g + c0 + sh.head;
  const bool aligned = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
  auto put = [&](int i, const uint4 &v) {
    float f[N];
    Vec<T>::unpack(v, f);
#pragma unroll
    for (int u = 0; u < N; ++u) f[u] = exp2_fast(fmaf(f[u], a.c, -st.z_max)) * qs;
    store_vec(dst + (int64_t)i * N, f, aligned);
  };
  int i = tid;
  for (; i + (U - 1) * kThreads < sh.nvec; i += U * kThreads) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = __ldcs(src + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) put(i + u * kThreads, v[u]);
  }
  for (; i < sh.nvec; i += kThreads) put(i, __ldcs(src + i));
  if (tid < sh.head + sh.tail) {
    const int64_t col = tid < sh.head ? c0 + tid : c1 - 1 - (tid - sh.head);
    g[col] = VT<T>::store(exp2_fast(fmaf(VT<T>::load(z[col]), a.c, -st.z_max)) * qs);
  }
  subtract_teacher<T, I>(a, z, g, lo, hi, c0, c1, st, scale, reinterpret_cast<uint32_t *>(dyn + kTableBytes), dyn,
                         kTableBytes);
}

template <typename K>
void launch_rows(K kernel, const DistillArgs &a, int threads, size_t smem, cudaStream_t s) {
  const int64_t grid = a.rows * a.n_slices;
  if (grid > INT32_MAX) fail(MSX_ERR_OVERFLOW, "csr_distillation has too many rows for one call.");
  MSX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxKept));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.n_slices;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MSX_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
}

int64_t slice_columns(int64_t vocab, int64_t n) { return ceil_div(ceil_div(vocab, n), 32) * 32; }

// Slices of a row: enough of them that one is at most `most` bytes, and more
// while the rows alone leave SMs idle and a slice stays above 8 KB.
int64_t pick_slices(int64_t rows, int64_t row_bytes, int64_t most, int64_t max_slices) {
  int64_t n = 1;
  while (n < max_slices && ceil_div(row_bytes, n) > most) n *= 2;
  while (n < max_slices && rows * n < 2 * num_sms() && row_bytes / n > 16384) n *= 2;
  return n;
}

template <typename T, typename I> void run_typed(const DistillCall &call, cudaStream_t s) {
  DistillArgs a{};
  a.logits = call.logits, a.ld = call.ld;
  a.t_data = call.t_data, a.t_idx = call.t_indices, a.t_ptr = call.t_indptr;
  a.nnz = call.nnz, a.rows = call.rows, a.vocab = call.vocab;
  a.c = 1.4426950408889634f / call.temperature, a.temperature = call.temperature;
  a.cot = call.cotangent, a.loss = call.loss, a.stats = static_cast<RowStats *>(call.stats), a.grad = call.grad;
  if (a.rows == 0) return;
  const int64_t row_bytes = a.vocab * (int64_t)sizeof(T);
  auto split = [&](int64_t n) { a.n_slices = (int)n, a.slice = slice_columns(a.vocab, n); };
  auto backward = [&] {
    split(pick_slices(a.rows, row_bytes, 65536, 1 << 20));
    if (a.rows * a.n_slices > INT32_MAX) fail(MSX_ERR_OVERFLOW, "csr_distillation has too many rows for one call.");
    const size_t smem = kTableBytes + (size_t)(a.slice + 31) / 32 * 4;
    distill_backward_kernel<T, I><<<(unsigned)(a.rows * a.n_slices), kThreads, smem, s>>>(a);
    MSX_CHECK_LAUNCH();
  };
  // Short rows have few vectors for each thread and gain from more CTAs.
  const bool small = row_bytes <= 40960;
  if (call.loss == nullptr) return backward();
  if (call.grad == nullptr) {
    split(pick_slices(a.rows, row_bytes, INT64_MAX, 8));
    if (small) return launch_rows(distill_row_kernel<T, I, Grad::none, 128>, a, 128, 0, s);
    return launch_rows(distill_row_kernel<T, I, Grad::none, kThreads>, a, kThreads, 0, s);
  }
  split(pick_slices(a.rows, row_bytes, kRereadMost, 8));
  const int64_t kept = a.slice * (int64_t)sizeof(T);
  if (kept > kKeepMost) {
    const int64_t smem = ceil_div(a.slice, 128) * 16 + kTableBytes;
    if (smem <= kMaxKept)
      return launch_rows(distill_row_kernel<T, I, Grad::reread, kRereadThreads>, a, kRereadThreads, (size_t)smem, s);
    // a bit for each column of a slice does not fit (over 12 million columns): two passes
    Scratch stats(sizeof(RowStats) * (size_t)a.rows, s);
    a.stats = stats.as<RowStats>();
    launch_rows(distill_row_kernel<T, I, Grad::none, kThreads>, a, kThreads, 0, s);
    return backward();
  }
  if (small) return launch_rows(distill_row_kernel<T, I, Grad::kept, 128>, a, 128, (size_t)kept, s);
  launch_rows(distill_row_kernel<T, I, Grad::kept, kThreads>, a, kThreads, (size_t)kept, s);
}

}  // namespace

void distill_run(int value_dtype, int index_dtype, const DistillCall &call, cudaStream_t s) {
  dispatch_value(value_dtype, [&](auto v) {
    dispatch_index(index_dtype, [&](auto i) { run_typed<decltype(v), decltype(i)>(call, s); });
  });
}

}  // namespace msx
