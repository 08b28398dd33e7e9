// Windowed attention with sink keys, forward and backward: dispatch and the
// kernels for every type and head size, in fp32 arithmetic.
//
//   S = scale Q K^T,  P = softmax of a row's seen scores,  O = P V
//   dV = P^T dO,  dP = dO V^T,  delta_i = dO_i . O_i = sum_j P_ij dP_ij
//   dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q
// dK and dV add up over the query heads that share a key head.
//
// These kernels take float32 inputs and head sizes that the tensor-core
// kernels do not, and they skip unseen pairs one by one, so that nothing that
// a mask hides (a NaN in padding, another sequence) reaches a result. A warp
// owns a few rows, a lane one key (or query) of a tile of 32; the dot products
// run from shared memory and bound the kernel.
#include "window_attention.cuh"

#include <initializer_list>

namespace msx {
namespace {

constexpr int kTile = 32;     // keys (queries) of a tile: a lane each
constexpr int kRows = 16;     // rows of a CTA
constexpr int kWarps = 4;
constexpr int kRowsPerWarp = kRows / kWarps;
constexpr int kMaxDim = 256;
constexpr int kRegs = kMaxDim / 32;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
__device__ void load_rows(float *dst, int stride, const T *src, int64_t token_stride, int first, int limit, int n, int dim) {
  for (int x = threadIdx.x; x < n * dim; x += blockDim.x) {
    const int r = x / dim, d = x % dim, t = first + r;
    dst[r * stride + d] = t >= 0 && t < limit ? VT<T>::load(src[t * token_stride + d]) : 0.f;
  }
}

__device__ __forceinline__ float dot(const float *a, const float *b, int dim) {
  float s = 0.f;
  for (int d = 0; d < dim; ++d) s = fmaf(a[d], b[d], s);
  return s;
}

template <typename T> __global__ void __launch_bounds__(kWarps * 32) forward_kernel(const WindowProblem w) {
  extern __shared__ float sm[];
  const int dim = w.c.dim, ks = dim + 1;
  float *sk = sm, *sv = sk + kTile * ks, *sq = sv + kTile * ks;
  const int b = blockIdx.z, h = blockIdx.y, hk = h / w.group, i0 = blockIdx.x * kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T *q = static_cast<const T *>(w.c.q.ptr) + b * w.c.q.batch + h * w.c.q.head;
  const T *k = static_cast<const T *>(w.c.k.ptr) + b * w.c.k.batch + hk * w.c.k.head;
  const T *v = static_cast<const T *>(w.c.v.ptr) + b * w.c.v.batch + hk * w.c.v.head;
  load_rows(sq, dim, q, w.c.q.token, i0, (int)w.c.q_len, kRows, dim);
  const KeyTiles<kTile> tiles(key_range(w, b, i0, i0 + kRows - 1));
  QuerySpan span[kRowsPerWarp];
  float m[kRowsPerWarp], l[kRowsPerWarp], acc[kRowsPerWarp][kRegs];
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    span[r] = query_span(w, b, i0 + warp * kRowsPerWarp + r);
    m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
    for (int x = 0; x < kRegs; ++x) acc[r][x] = 0.f;
  }
  for (int t = 0; t < tiles.n; ++t) {
    const int j0 = tiles.first(t), j = j0 + lane, end = tiles.end(t);
    __syncthreads();
    load_rows(sk, ks, k, w.c.k.token, j0, (int)w.c.k_len, kTile, dim);
    load_rows(sv, ks, v, w.c.v.token, j0, (int)w.c.k_len, kTile, dim);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
      const bool seen = j < end && span[r].sees(j);
      const unsigned who = __ballot_sync(~0u, seen);
      if (!who) continue;
      const float s = seen ? dot(sq + (warp * kRowsPerWarp + r) * dim, sk + lane * ks, dim) * (w.c.scale * kLog2e)
                           : -INFINITY;
      float top = s;
#pragma unroll
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      top = fmaxf(top, m[r]);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2f(m[r] - base);
      const float p = seen ? exp2f(s - base) : 0.f;
      float sum = p;
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
      l[r] = l[r] * keep + sum, m[r] = top;
#pragma unroll
      for (int x = 0; x < kRegs; ++x) acc[r][x] *= keep;
      for (unsigned left = who; left; left &= left - 1) {
        const int kk = __ffs(left) - 1;
        const float pk = __shfl_sync(~0u, p, kk);
#pragma unroll
        for (int x = 0; x < kRegs; ++x)
          if (x * 32 + lane < dim) acc[r][x] = fmaf(pk, sv[kk * ks + x * 32 + lane], acc[r][x]);
      }
    }
  }
  T *out = static_cast<T *>(w.c.out);
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    const int i = i0 + warp * kRowsPerWarp + r;
    if (i >= w.c.q_len) continue;
    const bool empty = span[r].empty();
    const float inv = empty ? 0.f : 1.f / l[r];
#pragma unroll
    for (int x = 0; x < kRegs; ++x) {
      const int d = x * 32 + lane;
      if (d >= dim) continue;
      const int64_t at = ((b * w.c.q_len + i) * w.c.q_heads + h) * dim + d;
      const float o = empty ? 0.f : acc[r][x] * inv;
      out[at] = VT<T>::store(o);
      if (w.c.out_low) static_cast<T *>(w.c.out_low)[at] = VT<T>::store(o - VT<T>::load(out[at]));
    }
    // an empty row's -inf makes its probabilities 0 in the backward pass
    if (w.c.lse && lane == 0)
      w.c.lse[((int64_t)b * w.c.q_heads + h) * w.lse_row + i] = empty ? -INFINITY : -(m[r] + log2f(l[r]));
  }
}

// -delta_i = -dO_i . O_i, 16 lanes for each row and head, VEC elements at a time.
// Of a 16-bit output what its rounding took off is added back: the same error of
// delta reaches every key of a row, which would cost dQ and dK as much as all their
// other roundings where a row sees few keys.
template <typename T, int VEC> __global__ void delta_kernel(const WindowProblem w) {
  const int64_t x = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4;
  const int lane = threadIdx.x & 15;
  const bool inside = x < w.c.batch * w.c.q_len * w.c.q_heads;
  float s = 0.f;
  if (inside) {
    const T *o = static_cast<const T *>(w.c.out) + x * w.c.dim, *g = static_cast<const T *>(w.c.grad_out) + x * w.c.dim;
    const T *l = w.c.out_low ? static_cast<const T *>(w.c.out_low) + x * w.c.dim : nullptr;
    for (int d = lane * VEC; d < w.c.dim; d += 16 * VEC) {
      alignas(16) T a[VEC], b[VEC], c[VEC];
      if (VEC > 1) {
        *reinterpret_cast<uint4 *>(a) = __ldcs(reinterpret_cast<const uint4 *>(o + d));
        *reinterpret_cast<uint4 *>(b) = __ldcs(reinterpret_cast<const uint4 *>(g + d));
        *reinterpret_cast<uint4 *>(c) = l ? __ldcs(reinterpret_cast<const uint4 *>(l + d)) : make_uint4(0, 0, 0, 0);
      } else {
        a[0] = o[d], b[0] = g[d], c[0] = l ? l[d] : VT<T>::store(0.f);
      }
#pragma unroll
      for (int y = 0; y < VEC; ++y) s = fmaf(VT<T>::load(a[y]) + VT<T>::load(c[y]), VT<T>::load(b[y]), s);
    }
  }
#pragma unroll
  for (int d = 8; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  const int64_t h = x % w.c.q_heads, bi = x / w.c.q_heads, b = bi / w.c.q_len, i = bi % w.c.q_len;
  if (inside && lane == 0) w.c.delta[(b * w.c.q_heads + h) * w.lse_row + i] = -s;
}

template <typename T> __global__ void __launch_bounds__(kWarps * 32) dq_kernel(const WindowProblem w) {
  extern __shared__ float sm[];
  const int dim = w.c.dim, ks = dim + 1;
  float *sk = sm, *sv = sk + kTile * ks, *sq = sv + kTile * ks, *sg = sq + kRows * dim;
  const int b = blockIdx.z, h = blockIdx.y, hk = h / w.group, i0 = blockIdx.x * kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T *q = static_cast<const T *>(w.c.q.ptr) + b * w.c.q.batch + h * w.c.q.head;
  const T *k = static_cast<const T *>(w.c.k.ptr) + b * w.c.k.batch + hk * w.c.k.head;
  const T *v = static_cast<const T *>(w.c.v.ptr) + b * w.c.v.batch + hk * w.c.v.head;
  const int64_t head0 = (b * w.c.q_len * w.c.q_heads + h) * dim;
  load_rows(sq, dim, q, w.c.q.token, i0, (int)w.c.q_len, kRows, dim);
  load_rows(sg, dim, static_cast<const T *>(w.c.grad_out) + head0, (int64_t)w.c.q_heads * dim, i0, (int)w.c.q_len,
            kRows, dim);
  const KeyTiles<kTile> tiles(key_range(w, b, i0, i0 + kRows - 1));
  QuerySpan span[kRowsPerWarp];
  float lse[kRowsPerWarp], delta[kRowsPerWarp], acc[kRowsPerWarp][kRegs];
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    const int i = i0 + warp * kRowsPerWarp + r;
    span[r] = query_span(w, b, i);
    const int64_t at = ((int64_t)b * w.c.q_heads + h) * w.lse_row + i;
    lse[r] = i < w.c.q_len ? w.c.lse[at] : -INFINITY;
    delta[r] = i < w.c.q_len ? w.c.delta[at] : 0.f;
#pragma unroll
    for (int x = 0; x < kRegs; ++x) acc[r][x] = 0.f;
  }
  for (int t = 0; t < tiles.n; ++t) {
    const int j0 = tiles.first(t), j = j0 + lane, end = tiles.end(t);
    __syncthreads();
    load_rows(sk, ks, k, w.c.k.token, j0, (int)w.c.k_len, kTile, dim);
    load_rows(sv, ks, v, w.c.v.token, j0, (int)w.c.k_len, kTile, dim);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
      const bool seen = j < end && span[r].sees(j);
      const unsigned who = __ballot_sync(~0u, seen);
      if (!who) continue;
      float ds = 0.f;
      if (seen) {
        const int row = warp * kRowsPerWarp + r;
        const float s = dot(sq + row * dim, sk + lane * ks, dim) * (w.c.scale * kLog2e);
        ds = exp2f(s + lse[r]) * (dot(sg + row * dim, sv + lane * ks, dim) + delta[r]);
      }
      for (unsigned left = who; left; left &= left - 1) {
        const int kk = __ffs(left) - 1;
        const float x1 = __shfl_sync(~0u, ds, kk);
#pragma unroll
        for (int x = 0; x < kRegs; ++x)
          if (x * 32 + lane < dim) acc[r][x] = fmaf(x1, sk[kk * ks + x * 32 + lane], acc[r][x]);
      }
    }
  }
  T *dq = static_cast<T *>(w.c.dq) + head0;
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    const int64_t i = i0 + warp * kRowsPerWarp + r;
    if (i >= w.c.q_len) continue;
#pragma unroll
    for (int x = 0; x < kRegs; ++x)
      if (x * 32 + lane < dim)
        dq[i * w.c.q_heads * dim + x * 32 + lane] = VT<T>::store(acc[r][x] * w.c.scale);
  }
}

template <typename T> __global__ void __launch_bounds__(kWarps * 32) dkv_kernel(const WindowProblem w) {
  extern __shared__ float sm[];
  const int dim = w.c.dim, ks = dim + 1;
  float *sq = sm, *sg = sq + kTile * ks, *sk = sg + kTile * ks, *sv = sk + kRows * dim;
  const int b = blockIdx.z, hk = blockIdx.y, j0 = blockIdx.x * kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T *k = static_cast<const T *>(w.c.k.ptr) + b * w.c.k.batch + hk * w.c.k.head;
  const T *v = static_cast<const T *>(w.c.v.ptr) + b * w.c.v.batch + hk * w.c.v.head;
  load_rows(sk, dim, k, w.c.k.token, j0, (int)w.c.k_len, kRows, dim);
  load_rows(sv, dim, v, w.c.v.token, j0, (int)w.c.k_len, kRows, dim);
  int last = -1;
  for (int j = j0; j < j0 + kRows; ++j) last = max(last, last_query(w, j));
  int own_last[kRowsPerWarp];
  float ak[kRowsPerWarp][kRegs], av[kRowsPerWarp][kRegs];
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    own_last[r] = last_query(w, j0 + warp * kRowsPerWarp + r);
#pragma unroll
    for (int x = 0; x < kRegs; ++x) ak[r][x] = av[r][x] = 0.f;
  }
  const int first = max(0, j0 - w.offset), stop = min((int)w.c.q_len, last - w.offset + 1);
  for (int h = hk * w.group; h < (hk + 1) * w.group; ++h) {
    const T *q = static_cast<const T *>(w.c.q.ptr) + b * w.c.q.batch + h * w.c.q.head;
    const T *g = static_cast<const T *>(w.c.grad_out) + (b * w.c.q_len * w.c.q_heads + h) * dim;
    const int64_t at = ((int64_t)b * w.c.q_heads + h) * w.lse_row;
    for (int i0 = first; i0 < stop; i0 += kTile) {
      __syncthreads();
      load_rows(sq, ks, q, w.c.q.token, i0, (int)w.c.q_len, kTile, dim);
      load_rows(sg, ks, g, (int64_t)w.c.q_heads * dim, i0, (int)w.c.q_len, kTile, dim);
      __syncthreads();
      const int i = i0 + lane, p = i + w.offset;
      const float lse = i < w.c.q_len ? w.c.lse[at + i] : -INFINITY, delta = i < w.c.q_len ? w.c.delta[at + i] : 0.f;
#pragma unroll
      for (int r = 0; r < kRowsPerWarp; ++r) {
        const int row = warp * kRowsPerWarp + r;
        const bool seen = i < w.c.q_len && p >= j0 + row && p <= own_last[r];
        const unsigned who = __ballot_sync(~0u, seen);
        if (!who) continue;
        float pr = 0.f, ds = 0.f;
        if (seen) {
          pr = exp2f(dot(sk + row * dim, sq + lane * ks, dim) * (w.c.scale * kLog2e) + lse);
          ds = pr * (dot(sv + row * dim, sg + lane * ks, dim) + delta);
        }
        for (unsigned left = who; left; left &= left - 1) {
          const int ii = __ffs(left) - 1;
          const float p1 = __shfl_sync(~0u, pr, ii), d1 = __shfl_sync(~0u, ds, ii);
#pragma unroll
          for (int x = 0; x < kRegs; ++x)
            if (x * 32 + lane < dim) {
              av[r][x] = fmaf(p1, sg[ii * ks + x * 32 + lane], av[r][x]);
              ak[r][x] = fmaf(d1, sq[ii * ks + x * 32 + lane], ak[r][x]);
            }
        }
      }
    }
  }
  T *dk = static_cast<T *>(w.c.dk), *dv = static_cast<T *>(w.c.dv);
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    const int64_t j = j0 + warp * kRowsPerWarp + r;
    if (j >= w.c.k_len) continue;
#pragma unroll
    for (int x = 0; x < kRegs; ++x) {
      const int d = x * 32 + lane;
      if (d >= dim) continue;
      const int64_t at = ((b * w.c.k_len + j) * w.c.k_heads + hk) * dim + d;
      dk[at] = VT<T>::store(ak[r][x] * w.c.scale);
      dv[at] = VT<T>::store(av[r][x]);
    }
  }
}

template <typename K>
void launch_general(K kernel, const WindowProblem &w, int64_t rows, int64_t heads, int staged, cudaStream_t s) {
  const int64_t blocks = ceil_div(rows, kRows);
  if (blocks == 0 || heads == 0 || w.c.batch == 0) return;
  auto bytes = [&](int dim) { return sizeof(float) * ((size_t)2 * kTile * (dim + 1) + (size_t)staged * kRows * dim); };
  // The attribute is the kernel's, not the launch's: what the largest head size
  // needs, so that another thread's call cannot lower it before this launch.
  MSX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(kMaxDim)));
  kernel<<<dim3((unsigned)blocks, (unsigned)heads, (unsigned)w.c.batch), kWarps * 32, bytes(w.c.dim), s>>>(w);
  MSX_CHECK_LAUNCH();
}

}  // namespace

void window_forward_general(const WindowProblem &w, int value_dtype, cudaStream_t s) {
  dispatch_value(value_dtype, [&](auto v) {
    launch_general(forward_kernel<decltype(v)>, w, w.c.q_len, w.c.q_heads, 1, s);
  });
}

void window_delta(const WindowProblem &w, int value_dtype, cudaStream_t s) {
  const int64_t rows = w.c.batch * w.c.q_len * w.c.q_heads;
  if (rows == 0) return;
  const uintptr_t at = reinterpret_cast<uintptr_t>(w.c.out) | reinterpret_cast<uintptr_t>(w.c.grad_out) |
                       reinterpret_cast<uintptr_t>(w.c.out_low);
  dispatch_value(value_dtype, [&](auto v) {
    using T = decltype(v);
    constexpr int kVec = 16 / sizeof(T);
    const unsigned grid = (unsigned)ceil_div(rows, 16);
    if (w.c.dim % kVec == 0 && at % 16 == 0)
      delta_kernel<T, kVec><<<grid, 256, 0, s>>>(w);
    else
      delta_kernel<T, 1><<<grid, 256, 0, s>>>(w);
    MSX_CHECK_LAUNCH();
  });
}

void window_backward_general(const WindowProblem &w, int value_dtype, cudaStream_t s) {
  window_delta(w, value_dtype, s);
  dispatch_value(value_dtype, [&](auto v) {
    if (w.c.dq) launch_general(dq_kernel<decltype(v)>, w, w.c.q_len, w.c.q_heads, 2, s);
    if (w.c.dk) launch_general(dkv_kernel<decltype(v)>, w, w.c.k_len, w.c.k_heads, 2, s);
  });
}

static WindowProblem problem(const WindowCall &c) {
  WindowProblem w{};
  w.c = c;
  w.group = (int)(c.q_heads / c.k_heads);
  w.offset = (int)(c.k_len - c.q_len);
  w.wide_ptr = c.indptr_dtype == MSX_I64;
  w.lse_row = ceil_div(c.q_len, 128) * 128;
  w.window = (int)std::min(c.window, c.k_len);
  w.sinks = (int)std::min(c.sinks, c.k_len);
  return w;
}

int64_t window_backward_floats(const WindowCall &c) {
  const WindowProblem w = problem(c);
  return c.batch * c.q_heads * w.lse_row + window_backward_floats_tc(w);
}

// The tensor-core kernels write 16 bytes at a time; the general ones any element.
static bool aligned16(std::initializer_list<const void *> outputs) {
  uintptr_t at = 0;
  for (const void *p : outputs) at |= reinterpret_cast<uintptr_t>(p);
  return at % 16 == 0;
}

void window_forward_run(int value_dtype, const WindowCall &c, cudaStream_t s) {
  const WindowProblem w = problem(c);
  if (window_tc_ok(w, value_dtype) && aligned16({c.out, c.out_low}))
    window_forward_tc(w, value_dtype, s);
  else
    window_forward_general(w, value_dtype, s);
}

void window_decode_run(int value_dtype, const WindowCall &c, cudaStream_t s) {
  window_decode(problem(c), value_dtype, s);
}

void window_backward_run(int value_dtype, const WindowCall &c, cudaStream_t s) {
  const WindowProblem w = problem(c);
  if (window_tc_ok(w, value_dtype) && aligned16({c.grad_out, c.dq, c.dk, c.dv}))
    window_backward_tc(w, value_dtype, s);
  else
    window_backward_general(w, value_dtype, s);
}

}  // namespace msx
