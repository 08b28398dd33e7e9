// Windowed attention of one query for each sequence, at the end of its cache.
//
// The keys that the query sees, the sinks and then the window, are numbered
// through and split over the CTAs of a cluster; a CTA takes the query heads of
// one key head (up to 16), so that its keys and values are read once. Each warp
// keeps a running maximum, sum and output of its own; at the end the cluster's
// CTAs join all their warps' parts from each other's shared memory, each CTA a
// share of the output, in a fixed order.
//
// Nothing is masked: keys outside the numbering are not loaded (their rows are
// zeros), so nothing behind a sequence's end or between sinks and window reaches
// a result.
//
// Bound: HBM, 2 (window + sinks) dim elements for each sequence and key head.
#include <cooperative_groups.h>

#include <algorithm>

#include "window_tc.cuh"

namespace cg = cooperative_groups;

namespace msx {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 64;    // keys of a stage, 16 for each warp
constexpr int kHeads = 16;   // query heads of a CTA: the rows of an mma tile
constexpr int kMaxSplit = 16;

struct Params {
  WindowProblem w;
  int head_blocks, splits;
};

// The keys of sequence b, numbered 0..n-1: sinks first, then the window.
struct Keys {
  int sinks, gap, n;
  __device__ Keys(const WindowProblem &w, int b) {
    const int len = key_count(w, b);
    const int low = max(0, len - w.window);
    sinks = min(w.sinks, low);
    gap = low - sinks;
    n = len - gap;
  }
  __device__ int64_t at(int x) const { return x < sinks ? x : x + gap; }
};

// What a warp hands over: for each of `HEADS` heads maximum, sum and output.
template <int HEADS, int DIM> struct Part {
  float m[kWarps][HEADS], l[kWarps][HEADS], o[kWarps][HEADS][DIM];
};

// Joins the parts of all warps of all CTAs of the cluster and writes the output.
// A CTA that saw no key has maximum -inf and weight 0.
template <typename T, int HEADS, int DIM>
__device__ void join_parts(const Params &p, Part<HEADS, DIM> *mine, int b, int h0, int heads, int n_keys) {
  const WindowProblem &w = p.w;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), dim = w.c.dim, n = p.splits;
  if (n > 1) cluster.sync(); else __syncthreads();
  T *out = static_cast<T *>(w.c.out) + ((int64_t)b * w.c.q_heads + h0) * dim;
  for (int x = rank * blockDim.x + threadIdx.x; x < heads * dim; x += n * blockDim.x) {
    const int h = x / dim, d = x % dim;
    float top = -INFINITY, sum = 0.f, val = 0.f;
    for (int r = 0; r < n; ++r) {
      const Part<HEADS, DIM> *part = n > 1 ? cluster.map_shared_rank(mine, r) : mine;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) top = fmaxf(top, part->m[k][h]);
    }
    const float base = top == -INFINITY ? 0.f : top;
    for (int r = 0; r < n; ++r) {
      const Part<HEADS, DIM> *part = n > 1 ? cluster.map_shared_rank(mine, r) : mine;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float f = exp2_fast(part->m[k][h] - base);
        sum = fmaf(f, part->l[k][h], sum);
        val = fmaf(f, part->o[k][h][d], val);
      }
    }
    out[x] = VT<T>::store(n_keys > 0 ? val / sum : 0.f);
  }
  if (n > 1) cluster.sync();  // the parts stay until all have read them
}

// ---- 16-bit types, head sizes that are multiples of 8 up to 128 ------------------
// mma m16n8k16: 16 query heads (unused rows are zeros), 8 keys or 8 dims, 16 deep.
__device__ __forceinline__ void ldmatrix4(uint32_t *r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t *r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <bool BF16> __device__ __forceinline__ void mma(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kDecodeStages = 3;
template <int DIM> constexpr int kStageBytes = 2 * kTile * DIM * 2;

// DIM: 64 or 128, the head size padded with zeros. 16-byte chunks of a row are
// stored at chunk ^ (row % 8), which keeps ldmatrix free of bank conflicts.
template <typename T, int DIM>
__global__ void __launch_bounds__(kWarps * 32) decode_mma_kernel(const __grid_constant__ Params p) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int CH = DIM / 8, KS = DIM / 16;
  extern __shared__ __align__(128) unsigned char sm[];
  const WindowProblem &w = p.w;
  const int split = (int)(blockIdx.x % p.splits);
  int64_t x = blockIdx.x / p.splits;
  const int hb = (int)(x % p.head_blocks);
  x /= p.head_blocks;
  const int hk = (int)(x % w.c.k_heads), b = (int)(x / w.c.k_heads);
  const int h0 = hk * w.group + hb * kHeads, heads = min(kHeads, w.group - hb * kHeads);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const Keys keys(w, b);
  // whole tiles for every split, the first ones one more
  const int tiles = (keys.n + kTile - 1) / kTile;
  const int first = tiles * split / p.splits, last = tiles * (split + 1) / p.splits;
  const T *k = static_cast<const T *>(w.c.k.ptr) + b * w.c.k.batch + hk * w.c.k.head;
  const T *v = static_cast<const T *>(w.c.v.ptr) + b * w.c.v.batch + hk * w.c.v.head;
  const int chunks = w.c.dim / 8;

  if (chunks < CH)  // the padding of every stage, once
    for (int y = tid; y < kDecodeStages * 2 * kTile * CH; y += blockDim.x)
      reinterpret_cast<uint4 *>(sm)[y] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  auto load = [&](int tile, int stage) {
    if (tile < last) {
      unsigned char *base = sm + stage * kStageBytes<DIM>;
      const int c = tid % CH;
      if (c < chunks) {
#pragma unroll
        for (int r = tid / CH; r < kTile; r += kWarps * 32 / CH) {
          const int y = tile * kTile + r;
          const int64_t j = keys.at(min(y, keys.n - 1));
          const int bytes = y < keys.n ? 16 : 0;  // rows past the end are zeros
          const uint32_t dst = tc::smem_addr(base) + (r * CH + (c ^ (r & 7))) * 16;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(k + j * w.c.k.token + c * 8), "r"(bytes)
                       : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + kTile * DIM * 2),
                       "l"(v + j * w.c.v.token + c * 8), "r"(bytes)
                       : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kDecodeStages - 1; ++s) load(first + s, s);

  // query fragments, straight from global memory
  uint32_t q[KS][4];
  {
    const T *src = static_cast<const T *>(w.c.q.ptr) + b * w.c.q.batch + h0 * w.c.q.head;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = g + (e & 1) * 8, d = s * 16 + (e >> 1) * 8 + t * 2;
        q[s][e] = r < heads && d < w.c.dim ? *reinterpret_cast<const uint32_t *>(src + r * w.c.q.head + d) : 0u;
      }
  }
  const float c = w.c.scale * kLog2e;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[DIM / 8][4];
#pragma unroll
  for (int y = 0; y < DIM / 8; ++y) o[y][0] = o[y][1] = o[y][2] = o[y][3] = 0.f;

  const int mi = lane >> 3, mr = lane & 7;
  for (int tile = first, stage = 0; tile < last; ++tile) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kDecodeStages - 2) : "memory");
    __syncthreads();
    load(tile + kDecodeStages - 1, (stage + kDecodeStages - 1) % kDecodeStages);
    const uint32_t kb = tc::smem_addr(sm) + stage * kStageBytes<DIM>, vb = kb + kTile * DIM * 2;
    stage = (stage + 1) % kDecodeStages;
    const int key0 = tile * kTile + warp * 16;  // this warp's 16 keys
    float s[2][4] = {};
    {
      const int r = warp * 16 + (mi >> 1) * 8 + mr;
#pragma unroll
      for (int y = 0; y < KS; ++y) {
        uint32_t kf[4];
        ldmatrix4(kf, kb + (r * CH + ((2 * y + (mi & 1)) ^ (r & 7))) * 16);
        mma<BF16>(s[0], q[y], kf[0], kf[1]);
        mma<BF16>(s[1], q[y], kf[2], kf[3]);
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = key0 + n * 8 + t * 2 + (e & 1) < keys.n ? s[n][e] * c : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 2));
    }
    // the maximum in use is only raised by 2^8 or more
    if (__any_sync(~0u, top[0] - m[0] > 8.f || top[1] - m[1] > 8.f)) {
      float keep[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float up = fmaxf(m[r], top[r]);
        keep[r] = m[r] == -INFINITY ? 0.f : exp2_fast(m[r] - up);
        m[r] = up, l[r] *= keep[r];
      }
#pragma unroll
      for (int y = 0; y < DIM / 8; ++y)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[y][e] *= keep[e >> 1];
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2_fast(s[n][e] - base[e >> 1]);
        l[e >> 1] += s[n][e];
      }
    const uint32_t a[4] = {pack2<BF16>(s[0][0], s[0][1]), pack2<BF16>(s[0][2], s[0][3]), pack2<BF16>(s[1][0], s[1][1]),
                           pack2<BF16>(s[1][2], s[1][3])};
    {
      const int r = warp * 16 + (mi & 1) * 8 + mr;
#pragma unroll
      for (int y = 0; y < DIM / 16; ++y) {
        uint32_t vf[4];
        ldmatrix4_trans(vf, vb + (r * CH + ((2 * y + (mi >> 1)) ^ (r & 7))) * 16);
        mma<BF16>(o[2 * y], a, vf[0], vf[1]);
        mma<BF16>(o[2 * y + 1], a, vf[2], vf[3]);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // the stages are done with: their space takes the parts
  using P = Part<kHeads, DIM>;
  static_assert(sizeof(P) <= kDecodeStages * kStageBytes<DIM>, "the parts fit the stages");
  P *part = reinterpret_cast<P *>(sm);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(~0u, l[r], 1);
    l[r] += __shfl_xor_sync(~0u, l[r], 2);
    if (t == 0) part->m[warp][g + r * 8] = m[r], part->l[warp][g + r * 8] = l[r];
  }
#pragma unroll
  for (int y = 0; y < DIM / 8; ++y)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float2 *>(&part->o[warp][g + r * 8][y * 8 + t * 2]) = make_float2(o[y][2 * r], o[y][2 * r + 1]);
  join_parts<T>(p, part, b, h0, heads, keys.n);
}

// ---- every type and head size -------------------------------------------------------
// 8 lanes for each key, 4 keys at a time for each warp; lane u of a key has the
// dims u, u + 8, ...; a CTA takes HEADS query heads. fp32 arithmetic.
template <typename T, int HEADS, int DIM>
__global__ void __launch_bounds__(kWarps * 32) decode_general_kernel(const __grid_constant__ Params p) {
  constexpr int N = DIM / 8;
  extern __shared__ __align__(128) unsigned char sm[];
  const WindowProblem &w = p.w;
  const int split = (int)(blockIdx.x % p.splits);
  int64_t x = blockIdx.x / p.splits;
  const int hb = (int)(x % p.head_blocks);
  x /= p.head_blocks;
  const int hk = (int)(x % w.c.k_heads), b = (int)(x / w.c.k_heads);
  const int h0 = hk * w.group + hb * HEADS, heads = min(HEADS, w.group - hb * HEADS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, u = lane & 7, dim = w.c.dim;
  const Keys keys(w, b);
  const int first = (int)((int64_t)keys.n * split / p.splits), last = (int)((int64_t)keys.n * (split + 1) / p.splits);
  const T *k = static_cast<const T *>(w.c.k.ptr) + b * w.c.k.batch + hk * w.c.k.head;
  const T *v = static_cast<const T *>(w.c.v.ptr) + b * w.c.v.batch + hk * w.c.v.head;
  const T *src = static_cast<const T *>(w.c.q.ptr) + b * w.c.q.batch + h0 * w.c.q.head;
  const float c = w.c.scale * kLog2e;
  float q[HEADS][N], o[HEADS][N], m[HEADS], l[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
    for (int y = 0; y < N; ++y) {
      const int d = y * 8 + u;
      q[h][y] = h < heads && d < dim ? VT<T>::load(src[h * w.c.q.head + d]) : 0.f;
      o[h][y] = 0.f;
    }
  }
  for (int j = first + warp * 4; j < last; j += kWarps * 4) {
    const bool live = j + sub < last;
    const int64_t at = keys.at(min(j + sub, last - 1));
    float s[HEADS] = {}, row[N];
#pragma unroll
    for (int y = 0; y < N; ++y) {
      const int d = y * 8 + u;
      const float e = d < dim ? VT<T>::load(k[at * w.c.k.token + d]) : 0.f;
      row[y] = d < dim ? VT<T>::load(v[at * w.c.v.token + d]) : 0.f;
#pragma unroll
      for (int h = 0; h < HEADS; ++h) s[h] = fmaf(q[h][y], e, s[h]);
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      s[h] += __shfl_xor_sync(~0u, s[h], 1);
      s[h] += __shfl_xor_sync(~0u, s[h], 2);
      s[h] += __shfl_xor_sync(~0u, s[h], 4);
      s[h] *= c;
      if (!live) continue;  // its 8 lanes alike; no lane of the warp is waited for below
      const float top = fmaxf(m[h], s[h]), base = top == -INFINITY ? 0.f : top;
      const float keep = exp2f(m[h] - base), e = exp2f(s[h] - base);
      l[h] = l[h] * keep + e, m[h] = top;
#pragma unroll
      for (int y = 0; y < N; ++y) o[h][y] = fmaf(e, row[y], o[h][y] * keep);
    }
    __syncwarp();
  }
  using P = Part<HEADS, DIM>;
  P *part = reinterpret_cast<P *>(sm);
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    // the warp's four keys' parts
    float top = m[h];
    top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
    top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
    const float f = exp2f(m[h] - (top == -INFINITY ? 0.f : top));
    float sum = l[h] * f;
    sum += __shfl_xor_sync(~0u, sum, 8);
    sum += __shfl_xor_sync(~0u, sum, 16);
    if (lane == 0) part->m[warp][h] = top, part->l[warp][h] = sum;
#pragma unroll
    for (int y = 0; y < N; ++y) {
      float e = o[h][y] * f;
      e += __shfl_xor_sync(~0u, e, 8);
      e += __shfl_xor_sync(~0u, e, 16);
      if (sub == 0) part->o[warp][h][y * 8 + u] = e;
    }
  }
  join_parts<T>(p, part, b, h0, heads, keys.n);
}

template <typename K> void launch(K kernel, Params &p, int heads, int smem, int per_sm, cudaStream_t s) {
  const WindowProblem &w = p.w;
  p.head_blocks = (int)ceil_div(w.group, heads);
  const int64_t rows = w.c.batch * w.c.k_heads * p.head_blocks;
  if (rows == 0) return;
  // Splits: until every SM has its CTAs, while each keeps two tiles of keys.
  const int64_t most = std::min<int64_t>(w.c.k_len, (int64_t)w.window + w.sinks);
  p.splits = 1;
  while (p.splits < kMaxSplit && rows * p.splits < (int64_t)per_sm * num_sms() && most > 2 * kTile * p.splits)
    p.splits *= 2;
  if (rows * p.splits > INT32_MAX) fail(MSX_ERR_OVERFLOW, "window_attention_decode has too many heads for one call.");
  MSX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (p.splits > 8) MSX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * p.splits));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MSX_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<const Params &>(p)));
}

template <typename T> void run_general(Params &p, cudaStream_t s) {
  if (p.w.c.dim <= 128)
    launch(decode_general_kernel<T, 4, 128>, p, 4, (int)sizeof(Part<4, 128>), 4, s);
  else
    launch(decode_general_kernel<T, 2, 256>, p, 2, (int)sizeof(Part<2, 256>), 4, s);
}

template <typename T> void run_mma(Params &p, cudaStream_t s) {
  if (p.w.c.dim <= 64)
    launch(decode_mma_kernel<T, 64>, p, kHeads, kDecodeStages * kStageBytes<64>, 4, s);
  else
    launch(decode_mma_kernel<T, 128>, p, kHeads, kDecodeStages * kStageBytes<128>, 2, s);
}

}  // namespace

void window_decode(const WindowProblem &w, int value_dtype, cudaStream_t s) {
  Params p{};
  p.w = w;
  // 16-byte loads of whole rows
  auto rows16 = [](const WindowTensor &t) {
    return reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0 && t.batch % 8 == 0 && t.token % 8 == 0 && t.head % 8 == 0;
  };
  const bool mma_ok = w.c.dim % 8 == 0 && w.c.dim <= 128 && rows16(w.c.q) && rows16(w.c.k) && rows16(w.c.v);
  if (value_dtype == MSX_F32)
    run_general<float>(p, s);
  else if (value_dtype == MSX_F16)
    mma_ok ? run_mma<__half>(p, s) : run_general<__half>(p, s);
  else
    mma_ok ? run_mma<__nv_bfloat16>(p, s) : run_general<__nv_bfloat16>(p, s);
}

}  // namespace msx
