// Windowed attention, backward, on the tensor cores (float16 / bfloat16, head
// sizes that are multiples of 8 up to 128). Two kernels, so that every gradient
// is summed in one place and in one order:
//
//  dQ:    a query tile of 128 rows walks the tiles of 128 keys that it sees:
//         S = Q K^T, dP = dO V^T, dS = P (dP - delta), dQ += dS K.
//  dK/dV: a key tile of 128 rows walks the tiles of 128 queries that see it, of
//         every head that shares it: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO,
//         dK += dS^T Q.
//
// A sink key is seen by every later query of its sequence. Where that would make a
// few key tiles much longer than the rest, the queries are cut into chunks: the
// key tile itself takes the queries of its band and of the chunk that the sequence
// starts in, and every later chunk has a CTA of its own for the sinks of its first
// query's sequence (a sequence that starts later in the chunk is in its own first
// chunk). Their sums go to a workspace in fp32, a slot for each chunk, and the key
// tile adds them in the order of the chunks.
//
// P = 2^(c S - lse) is recomputed from the forward pass's log-sum-exp. That is 7
// products of 128 x 128 x dim for each tile pair where one kernel with atomic
// sums of dQ would make 5; atomics would change results from run to run.
//
// As in the forward pass one warp loads tiles by TMA, one warp issues
// tcgen05.mma, and some warpgroups do the arithmetic in between, straight from
// tensor memory, 32 or 64 columns of every row each. P and dS, rounded to the inputs'
// type for the second products (half a step each; the sums are fp32), take the
// place of the scores they came from. The products of one tile pair are issued
// between those of its neighbours, so that the tensor cores work while the
// exponentials of the next tile and the differences of this one are taken.
//
// Bound: the tensor cores, 4 x 520 (3 x 520) clocks for each tile pair at head
// size 128, against 128 x 128 / 16 = 1024 clocks of exponentials; the weights wait
// for the scores and the scores for the sums of the tile before, which makes it
// about 3700 (2900), with the tensor pipe busy 55% of the time. 16384 tokens, window
// 2048, 32 / 8 heads of 128, bf16: dQ 0.74-0.80 ms, dK and dV 1.03-1.14 ms, as the
// power cap lets the clock run.
//
// A masked P or dS is 0, but 0 times an infinity or NaN in a hidden row of dO, Q
// or K would reach the sums: rows that end not finite while something not finite
// hides in their tiles are computed again pair by pair.
//
// float16: dS is beyond the type's range where loss-scaled gradients of a few
// thousand meet few keys, while dQ and dK need not be. A row with such a dS ends
// not finite with finite log-sum-exp and delta, and is computed again in fp32 like
// those above. (A factor on dS before it is rounded would move the range's other
// end: gradients of 1e-5 already have dS among float16's smallest steps.)
#include <algorithm>

#include "window_tc.cuh"

namespace msx {

using namespace tc;

namespace {

constexpr int kT = 128;        // rows and columns of a tile pair
// Columns of a tile for each warpgroup of arithmetic. dQ of head sizes over 64 is
// 4% faster with fewer, busier warps, everything else up to 8% slower.
constexpr int kKvCols = 32;
template <int DB> constexpr int kQCols = DB == 2 ? 64 : 32;
constexpr int threads_for(int cols) { return 64 + kT / cols * 128; }  // loads, products, arithmetic
constexpr int kStages = 4;

struct Params {
  WindowProblem w;
  CUtensorMap q, k, v, g;
  int items, q_tiles;
  Watch watch;
  // far queries of the sinks: queries of a chunk (0: not cut), chunks, and sums
  // [batch][key head][chunk][sink][dV, dK][dim]
  int chunk, n_chunks;
  float *far;
};

// The first chunk that takes a sequence's queries away from the key tiles.
__device__ __forceinline__ int first_far_chunk(const Params &p, int start) {
  const int i = start - p.w.offset;
  return i < 0 ? 0 : i / p.chunk + 1;
}

// The last query position that a key's own tile takes (at least; it takes whole
// tiles of queries).
__device__ __forceinline__ int last_near_query(const Params &p, int j) {
  const WindowProblem &w = p.w;
  if (p.chunk == 0) return last_query(w, j);
  if (j >= w.c.k_len) return -1;
  int start, end;
  sequence_of(w, j, start, end);
  if (start >= end) return -1;
  int last = j + w.window - 1;
  if (j - start < w.sinks) last = max(last, first_far_chunk(p, start) * p.chunk - 1 + w.offset);
  return min(end - 1, last);
}

// The score of one pair times log2(e) and dO_i . V_j, from global memory.
template <typename T> struct PairDots {
  const T *q, *k, *g, *v;
  __device__ PairDots(const WindowProblem &w, int b, int h, int64_t i, int64_t j) {
    const int hk = h / w.group;
    q = static_cast<const T *>(w.c.q.ptr) + b * w.c.q.batch + h * w.c.q.head + i * w.c.q.token;
    g = static_cast<const T *>(w.c.grad_out) + ((b * w.c.q_len + i) * w.c.q_heads + h) * w.c.dim;
    k = static_cast<const T *>(w.c.k.ptr) + b * w.c.k.batch + hk * w.c.k.head + j * w.c.k.token;
    v = static_cast<const T *>(w.c.v.ptr) + b * w.c.v.batch + hk * w.c.v.head + j * w.c.v.token;
  }
  __device__ void weights(const WindowProblem &w, float lse, float delta, float &p, float &ds) const {
    float s = 0.f, dp = 0.f;
    for (int d = 0; d < w.c.dim; d += 8) {  // 16 bytes of each row
      alignas(16) T x[4][8];
      const T *rows[4] = {q, k, g, v};
#pragma unroll
      for (int r = 0; r < 4; ++r) *reinterpret_cast<uint4 *>(x[r]) = *reinterpret_cast<const uint4 *>(rows[r] + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s = fmaf(VT<T>::load(x[0][e]), VT<T>::load(x[1][e]), s);
        dp = fmaf(VT<T>::load(x[2][e]), VT<T>::load(x[3][e]), dp);
      }
    }
    p = exp2f(s * (w.c.scale * kLog2e) + lse);
    ds = p * (dp + delta);
  }
};

// One row of dQ again, by a warp, pair by pair; columns [d0, d1) are written.
template <typename T>
__device__ __noinline__ void repair_dq(const WindowProblem &w, int b, int h, int i, int d0, int d1) {
  const int lane = threadIdx.x & 31;
  const QuerySpan span = query_span(w, b, i);
  const int64_t at = ((int64_t)b * w.c.q_heads + h) * w.lse_row + i;
  const float lse = w.c.lse[at], delta = w.c.delta[at];
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < 2; ++part) {
    const int from = part ? span.low : span.start, end = part ? span.p + 1 : span.sink_end;
    for (int j0 = from; j0 < end; j0 += 32) {
      float p = 0.f, ds = 0.f;
      if (j0 + lane < end) PairDots<T>(w, b, h, i, j0 + lane).weights(w, lse, delta, p, ds);
#pragma unroll 8  // loads in flight
      for (int x = 0; x < min(32, end - j0); ++x) {
        const float e = __shfl_sync(~0u, ds, x);
        const T *k = PairDots<T>(w, b, h, i, j0 + x).k;
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (y * 32 + lane < w.c.dim) acc[y] = fmaf(e, VT<T>::load(k[y * 32 + lane]), acc[y]);
      }
    }
  }
  T *dq = static_cast<T *>(w.c.dq) + ((b * w.c.q_len + i) * w.c.q_heads + h) * w.c.dim;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const int d = y * 32 + lane;
    if (d >= d0 && d < d1 && d < w.c.dim) dq[d] = VT<T>::store(acc[y] * w.c.scale);
  }
}

// One row of dK (keys) or dV again, columns [d0, d1).
template <typename T>
__device__ __noinline__ void repair_dkv(const WindowProblem &w, int b, int hk, int j, bool keys, int d0, int d1) {
  const int lane = threadIdx.x & 31, shift = key_count(w, b) - (int)w.c.q_len;
  const int i0 = max(0, j - shift), i1 = min((int)w.c.q_len, last_query(w, j) - shift + 1);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int h = hk * w.group; h < (hk + 1) * w.group; ++h) {
    const int64_t at = ((int64_t)b * w.c.q_heads + h) * w.lse_row;
    for (int i = i0; i < i1; i += 32) {
      float p = 0.f, ds = 0.f;
      if (i + lane < i1)
        PairDots<T>(w, b, h, i + lane, j).weights(w, w.c.lse[at + i + lane], w.c.delta[at + i + lane], p, ds);
#pragma unroll 8  // loads in flight
      for (int x = 0; x < min(32, i1 - i); ++x) {
        const float e = __shfl_sync(~0u, keys ? ds : p, x);
        const PairDots<T> pair(w, b, h, i + x, j);
        const T *row = keys ? pair.q : pair.g;
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (y * 32 + lane < w.c.dim) acc[y] = fmaf(e, VT<T>::load(row[y * 32 + lane]), acc[y]);
      }
    }
  }
  T *out = static_cast<T *>(keys ? w.c.dk : w.c.dv) + ((b * w.c.k_len + j) * w.c.k_heads + hk) * w.c.dim;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const int d = y * 32 + lane;
    if (d >= d0 && d < d1 && d < w.c.dim) out[d] = VT<T>::store(acc[y] * (keys ? w.c.scale : 1.f));
  }
}

// After a wait gave up, by all threads at the kernel's end: see bar_settle. The
// phases armed last of the ring's barriers and of `once` are the bits of `armed`.
__device__ __forceinline__ void settle(uint64_t *ring, uint64_t *once, uint64_t *idle, uint32_t armed) {
  const int warp = (int)threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) bar_settle(&ring[s], armed >> s & 1);
    bar_settle(once, armed >> kStages & 1);
  }
  if (warp == 1) mma_commit((threadIdx.x & 31) == 0, idle), bar_settle(idle, 0);
}
constexpr uint32_t kNoneArmed = (2u << kStages) - 1;  // the ring's barriers, then the other one

// ---- dK and dV -------------------------------------------------------------------
struct KvBars {
  uint64_t kv_full, full[kStages], empty[kStages], s_full, dp_full, p_full, ds_full, done, idle;
  uint32_t tmem, armed;
  int stop, last;
};

// Key tiles that a sequence's sinks can touch.
__host__ __device__ inline int far_key_tiles(const WindowProblem &w) { return (w.sinks + kT - 2) / kT + 1; }

template <int DB> constexpr int kKvSmem = 1024 + (2 + kStages) * DB * kBox + 2 * 2 * kT * 4;

// FAR: the sinks of one sequence against one chunk of queries.
template <typename T, int DB, bool FAR>
__global__ void __launch_bounds__(threads_for(kKvCols), 1) dkv_tc_kernel(const __grid_constant__ Params p) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kTile = DB * kBox, kCols = kKvCols;
  extern __shared__ unsigned char raw[];
  unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ KvBars bars;
  unsigned char *k_tile = sm, *v_tile = sm + kTile, *ring = sm + 2 * kTile;
  float *row_stats = reinterpret_cast<float *>(ring + kStages * kTile);  // two of {lse[128], delta[128]}
  const WindowProblem &w = p.w;
  const int warp = __shfl_sync(~0u, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int shift = w.offset;
  int x = (int)blockIdx.x;
  const int hk = x % w.c.k_heads;
  x /= w.c.k_heads;
  const int b = x % (int)w.c.batch;
  x /= (int)w.c.batch;
  int j0, chunk = 0, far_start = 0, far_end = 0;
  if (FAR) {
    const int n_tiles = far_key_tiles(w);
    chunk = x / n_tiles;
    const int p0 = chunk * p.chunk + shift;
    if (p0 >= 0) sequence_of(w, p0, far_start, far_end);
    j0 = (far_start / kT + x % n_tiles) * kT;
    if (far_start >= far_end || first_far_chunk(p, far_start) > chunk || j0 >= min(far_start + w.sinks, far_end)) return;
  } else {
    j0 = x * kT;
  }
  volatile int *stop = &bars.stop;
  if (threadIdx.x == 0) {
    bar_init(&bars.kv_full, 1);
    for (int s = 0; s < kStages; ++s) bar_init(&bars.full[s], 1), bar_init(&bars.empty[s], 1);
    bar_init(&bars.s_full, 1), bar_init(&bars.dp_full, 1), bar_init(&bars.done, 1);
    bar_init(&bars.p_full, 4 * kT / kCols), bar_init(&bars.ds_full, 4 * kT / kCols);
    bar_init(&bars.idle, 1);
    bars.stop = 0, bars.last = -1, bars.armed = kNoneArmed;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // the tiles of queries that see any of these keys
  const int key = j0 + (warp & 3) * 32 + lane;
  if (warp >= 2 && warp < 6) {
    const int top = __reduce_max_sync(~0u, last_near_query(p, key));
    if (lane == 0) atomicMax(&bars.last, top);
  }
  __syncthreads();
  const int i_first = max(0, j0 - shift), i_stop = min((int)w.c.q_len, bars.last - shift + 1);
  int t0 = i_first / kT, n_tiles = i_stop > i_first ? (i_stop - t0 * kT + kT - 1) / kT : 0;
  const int near_end = (t0 + n_tiles) * kT;  // queries from here on are the chunks'
  int first_i = key - shift, last_i = min(last_query(w, key) - shift, (int)w.c.q_len - 1);
  if (FAR) {
    const int from = max(chunk * p.chunk, near_end), to = min((chunk + 1) * p.chunk, far_end - shift);
    if (from >= to) return;
    t0 = from / kT, n_tiles = (to - from + kT - 1) / kT;
    const bool sink = key >= far_start && key < min(far_start + w.sinks, far_end);
    first_i = sink ? from : INT_MAX, last_i = sink ? to - 1 : -1;
  }
  const int n = n_tiles * w.group;
  if (warp == 1) tmem_alloc(&bars.tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(~0u, bars.tmem, 0), t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;
  // the pair (head, query tile) that comes next: all tiles of a head, then the next head's
  struct Walk {
    int h, t, first, end;
    __device__ void next() {
      if (++t == end) t = first, ++h;
    }
  };
  const Walk first_pair{hk * w.group, t0, t0, t0 + n_tiles};

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      bar_expect(&bars.kv_full, 2 * kTile);
      uint32_t armed = kNoneArmed ^ 1u << kStages;
      for (int x = 0; x < DB; ++x) {
        tma_load_4d(k_tile + x * kBox, &p.k, &bars.kv_full, x * 64, j0, hk, b);
        tma_load_4d(v_tile + x * kBox, &p.v, &bars.kv_full, x * 64, j0, hk, b);
      }
      bool ok = true;
      Walk at_pair = first_pair;
      for (int e = 0; ok && e < 2 * n; ++e) {  // Q and dO of each pair in turn
        const int s = e % kStages, it = e >> 1;
        if (e > 0 && !(e & 1)) at_pair.next();
        const int h = at_pair.h, i0 = at_pair.t * kT;
        if (!(ok = bar_wait(&bars.empty[s], (e / kStages & 1) ^ 1, stop, &p.watch))) break;
        armed ^= 1u << s;
        if (e & 1) {
          bar_expect(&bars.full[s], kTile);
        } else {
          bar_expect(&bars.full[s], kTile + 2 * kT * 4);
          const int64_t at = ((int64_t)b * w.c.q_heads + h) * w.lse_row + i0;
          float *dst = row_stats + (it & 1) * 2 * kT;
          bulk_load(dst, w.c.lse + at, kT * 4, &bars.full[s]);
          bulk_load(dst + kT, w.c.delta + at, kT * 4, &bars.full[s]);
        }
        for (int x = 0; x < DB; ++x)
          tma_load_4d(ring + s * kTile + x * kBox, e & 1 ? &p.g : &p.q, &bars.full[s], x * 64, i0, h, b);
      }
      bars.armed = armed;
    }
  } else if (warp == 1) {
    if (n > 0) {
      const Products<DB, kCols> mm(BF16, w.c.dim);
      const uint32_t ka = smem_addr(k_tile), va = smem_addr(v_tile), ra = smem_addr(ring);
      bool ok = warp_wait(&bars.kv_full, 0, stop, &p.watch);
      auto ready = [&](int e) { return ok = ok && warp_wait(&bars.full[e % kStages], e / kStages & 1, stop, &p.watch); };
      auto tile = [&](int e) { return ra + (e % kStages) * kTile; };
      if (ready(0)) {
        fence_after();
        mm.scores(t_s, ka, tile(0));
        mma_commit(mm.leader, &bars.s_full);
      }
      if (ready(1)) {
        mm.scores(t_dp, va, tile(1));
        mma_commit(mm.leader, &bars.dp_full);
      }
      for (int it = 0; ok && it < n; ++it) {
        const int q = 2 * it, g = q + 1;
        if (!(ok = warp_wait(&bars.p_full, it & 1, stop, &p.watch))) break;
        fence_after();
        mm.sums(t_dv, t_s, tile(g), it > 0);
        mma_commit(mm.leader, &bars.empty[g % kStages]);
        if (it + 1 < n) {
          if (!ready(q + 2)) break;
          mm.scores(t_s, ka, tile(q + 2));
          mma_commit(mm.leader, &bars.s_full);
        }
        if (!(ok = warp_wait(&bars.ds_full, it & 1, stop, &p.watch))) break;
        fence_after();
        mm.sums(t_dk, t_dp, tile(q), it > 0);
        mma_commit(mm.leader, &bars.empty[q % kStages]);
        if (it + 1 < n) {
          if (!ready(g + 2)) break;
          mm.scores(t_dp, va, tile(g + 2));
          mma_commit(mm.leader, &bars.dp_full);
        }
      }
      mma_commit(mm.leader, &bars.done);
    }
  } else {
    const int part = (warp - 2) >> 2;
    const uint32_t at = ((uint32_t)(warp & 3) << 21) + part * kCols;
    const float c = w.c.scale * kLog2e;
    const float2 c2 = make_float2(c, c);
    // the queries that all 32 keys of this warp are seen by
    const int all_first = __reduce_max_sync(~0u, first_i), all_last = __reduce_min_sync(~0u, last_i);
    bool ok = true;
    Walk at_pair = first_pair;
    for (int it = 0; ok && it < n; ++it, at_pair.next()) {
      const int i0 = at_pair.t * kT + part * kCols;
      const float *lse = row_stats + (it & 1) * 2 * kT + part * kCols, *delta = lse + kT;
      const bool masked = !(i0 >= all_first && i0 + kCols - 1 <= all_last);
      const uint32_t seen = first_i > last_i ? 0 : bits(first_i - i0, last_i + 1 - i0, 0);
      // lse and delta came with Q's tile, which the products of s_full have read
      if (!(ok = warp_wait(&bars.full[2 * it % kStages], 2 * it / kStages & 1, stop, &p.watch))) break;
      if (!(ok = warp_wait(&bars.s_full, it & 1, stop, &p.watch))) break;
      fence_after();
      float2 pr[kCols / 2];
      auto weights = [&](auto mask) {
        uint32_t z[kCols], pk[kCols / 2];
#pragma unroll
        for (int x = 0; x < 2; ++x) tmem_ld16(t_s + at + x * 16, z + x * 16);
        wait_ld();
        tie32(z);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t *zz = z + x * 16;
          float4 stat;
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const int col = x * 16 + 2 * y;
            if (!(y & 1)) stat = *reinterpret_cast<const float4 *>(lse + col);
            float2 e = fma2(make_float2(__uint_as_float(zz[2 * y]), __uint_as_float(zz[2 * y + 1])), c2,
                            y & 1 ? make_float2(stat.z, stat.w) : make_float2(stat.x, stat.y));
            e.x = exp2_fast(e.x), e.y = exp2_fast(e.y);
            if (mask) {
              if (!(seen >> col & 1)) e.x = 0.f;
              if (!(seen >> col & 2)) e.y = 0.f;
            }
            pr[x * 8 + y] = e;
            pk[x * 8 + y] = pack2<BF16>(e.x, e.y);
          }
        }
        tmem_st16(t_s + at, pk);
      };
      if (masked) weights(std::true_type{}); else weights(std::false_type{});
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&bars.p_full);
      if (!(ok = warp_wait(&bars.dp_full, it & 1, stop, &p.watch))) break;
      fence_after();
      auto grads = [&](auto mask) {
        uint32_t z[kCols], pk[kCols / 2];
#pragma unroll
        for (int x = 0; x < 2; ++x) tmem_ld16(t_dp + at + x * 16, z + x * 16);
        wait_ld();
        tie32(z);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t *zz = z + x * 16;
          float4 stat;
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const int col = x * 16 + 2 * y;
            if (!(y & 1)) stat = *reinterpret_cast<const float4 *>(delta + col);
            float2 e = add2(make_float2(__uint_as_float(zz[2 * y]), __uint_as_float(zz[2 * y + 1])),
                            y & 1 ? make_float2(stat.z, stat.w) : make_float2(stat.x, stat.y));
            e = mul2(e, pr[x * 8 + y]);
            if (mask) {
              if (!(seen >> col & 1)) e.x = 0.f;
              if (!(seen >> col & 2)) e.y = 0.f;
            }
            pk[x * 8 + y] = pack2<BF16>(e.x, e.y);
          }
        }
        tmem_st16(t_dp + at, pk);
      };
      if (masked) grads(std::true_type{}); else grads(std::false_type{});
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&bars.ds_full);
    }
    if (ok && n > 0) ok = warp_wait(&bars.done, 0, stop, &p.watch);
    if (ok) {
      fence_after();
      // the first two warpgroups write dV, the others dK, half of the columns each
      const int half = part >> 1, d0 = (part & 1) * DB * 32;
      const bool inside = key < w.c.k_len;
      const uint32_t from = (half ? t_dk : t_dv) + ((uint32_t)(warp & 3) << 21);
      const float scale = half ? w.c.scale : 1.f;
      int start = 0, end = 0, c0 = 0, c1 = 0;  // the chunks that have sums for this key
      if (p.chunk && inside) {
        sequence_of(w, key, start, end);
        if (key < min(start + w.sinks, end) && near_end < end - shift) {
          c0 = max(first_far_chunk(p, start), near_end / p.chunk);
          c1 = min(p.n_chunks, (end - shift + p.chunk - 1) / p.chunk);
        }
      }
      float *far = nullptr;  // the sums of a chunk: far + chunk * far_step
      const int64_t far_step = (int64_t)w.sinks * 2 * w.c.dim;
      if (p.chunk) far = p.far + ((((int64_t)b * w.c.k_heads + hk) * p.n_chunks * w.sinks + key - start) * 2 + half) * w.c.dim;
      T *out = static_cast<T *>(half ? w.c.dk : w.c.dv) + ((b * w.c.k_len + key - lane) * w.c.k_heads + hk) * w.c.dim;
      bool bad = false;
#pragma unroll 1
      for (int d = d0; d < d0 + DB * 32; d += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld16(from + d, o), tmem_ld16(from + d + 16, o + 16);
          wait_ld();
          tie32(o);
        } else {
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = 0;
        }
        if (FAR) {
          if (first_i <= last_i)
#pragma unroll
            for (int y = 0; y < 32; y += 4)
              if (d + y < w.c.dim)
                *reinterpret_cast<float4 *>(far + chunk * far_step + d + y) =
                    make_float4(__uint_as_float(o[y]), __uint_as_float(o[y + 1]), __uint_as_float(o[y + 2]),
                                __uint_as_float(o[y + 3]));
          continue;
        }
        for (int c = c0; c < c1; ++c)
#pragma unroll
          for (int y = 0; y < 32; y += 4)
            if (d + y < w.c.dim) {
              const float4 f = *reinterpret_cast<const float4 *>(far + c * far_step + d + y);
              o[y] = __float_as_uint(__uint_as_float(o[y]) + f.x);
              o[y + 1] = __float_as_uint(__uint_as_float(o[y + 1]) + f.y);
              o[y + 2] = __float_as_uint(__uint_as_float(o[y + 2]) + f.z);
              o[y + 3] = __float_as_uint(__uint_as_float(o[y + 3]) + f.w);
            }
        bad = store32<T>(out, (int64_t)w.c.k_heads * w.c.dim, o, scale, d, w.c.dim, (int)w.c.k_len - (key - lane)) || bad;
      }
      if (!FAR && __any_sync(~0u, bad && inside)) {
        bool hidden = false;
        auto look_at = [&](int h, int i0, int first, int last) {
          const PairDots<T> row(w, b, h, 0, 0);
          for (int y = 0; y < kT; y += 32) {
            const bool odd = half ? row_not_finite(row.q, w.c.q.token, i0 + y + lane, w.c.q_len, w.c.dim)
                                  : row_not_finite(row.g, (int64_t)w.c.q_heads * w.c.dim, i0 + y + lane, w.c.q_len, w.c.dim);
            for (unsigned left = __ballot_sync(~0u, odd); left; left &= left - 1) {
              const int i = i0 + y + __ffs(left) - 1;
              hidden = hidden || i < first || i > last;
            }
          }
        };
        Walk look = first_pair;
        for (int it = 0; it < n; ++it, look.next())
          if (!(look.t * kT >= all_first && look.t * kT + kT - 1 <= all_last)) look_at(look.h, look.t * kT, first_i, last_i);
        // of a sink's far queries' tiles only the sequence's last holds other queries
        const int stop_i = c0 < c1 ? end - shift : 0, most = __reduce_max_sync(~0u, stop_i);
        if (most > 0)
          for (int h = hk * w.group; h < (hk + 1) * w.group; ++h)
            look_at(h, (most - 1) / kT * kT, 0, stop_i > 0 ? stop_i - 1 : INT_MAX);
        if (stop_i > 0 && stop_i < most) hidden = true;
        if (!BF16 && half && bad && inside && !hidden) {  // as in dQ, of all queries that see the key
          hidden = true;
          for (int h = hk * w.group; hidden && h < (hk + 1) * w.group; ++h) {
            const int64_t at = ((int64_t)b * w.c.q_heads + h) * w.lse_row;
            for (int i = max(0, first_i); hidden && i <= last_i; ++i)
              hidden = isfinite(w.c.lse[at + i]) && isfinite(w.c.delta[at + i]);
          }
        }
        for (unsigned left = __ballot_sync(~0u, bad && inside && hidden); left; left &= left - 1)
          repair_dkv<T>(w, b, hk, key - lane + __ffs(left) - 1, half != 0, d0, d0 + DB * 32);
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (*stop) settle(bars.full, &bars.kv_full, &bars.idle, bars.armed);
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 512);
}

// ---- dQ ---------------------------------------------------------------------------
struct QBars {
  uint64_t q_full, q_empty, full[kStages], empty[kStages], s_full[2], dp_full, ds_full, dq_full, idle;
  uint32_t tmem, armed;
  int stop;
};

template <int DB> constexpr int kQSmem = 1024 + (2 + kStages) * DB * kBox;

template <typename T, int DB>
__global__ void __launch_bounds__(threads_for(kQCols<DB>), 1) dq_tc_kernel(const __grid_constant__ Params p) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kTile = DB * kBox, kCols = kQCols<DB>;
  extern __shared__ unsigned char raw[];
  unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ QBars bars;
  unsigned char *q_tile = sm, *g_tile = sm + kTile, *ring = sm + 2 * kTile;
  const WindowProblem &w = p.w;
  const int warp = __shfl_sync(~0u, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int *stop = &bars.stop;
  if (threadIdx.x == 0) {
    bar_init(&bars.q_full, 1), bar_init(&bars.q_empty, 1);
    for (int s = 0; s < kStages; ++s) bar_init(&bars.full[s], 1), bar_init(&bars.empty[s], 1);
    bar_init(&bars.s_full[0], 1), bar_init(&bars.s_full[1], 1);
    bar_init(&bars.dp_full, 1), bar_init(&bars.ds_full, 4 * kT / kCols), bar_init(&bars.dq_full, 1);
    bar_init(&bars.idle, 1);
    bars.stop = 0, bars.armed = kNoneArmed;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&bars.tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(~0u, bars.tmem, 0), t_dp = tmem + 256, t_dq = tmem + 384;  // two score tiles before them
  auto item = [&](int x, int &b, int &h, int &i0) {  // heads of one key head side by side
    const int g = x % w.group;
    x /= w.group;
    i0 = x % p.q_tiles * kT;
    x /= p.q_tiles;
    h = x % w.c.k_heads * w.group + g;
    b = x / w.c.k_heads;
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, b, h, i0;
      uint32_t phase = 1, q_phase = 1, armed = kNoneArmed;
      bool ok = true;
      for (int x = blockIdx.x; ok && x < p.items; x += gridDim.x) {
        item(x, b, h, i0);
        const KeyTiles<kT> tiles(key_range(w, b, i0, i0 + kT - 1));
        if (tiles.n == 0) continue;
        if (!(ok = bar_wait(&bars.q_empty, q_phase, stop, &p.watch))) break;
        q_phase ^= 1;
        bar_expect(&bars.q_full, 2 * kTile);
        armed ^= 1u << kStages;
        for (int d = 0; d < DB; ++d) {
          tma_load_4d(q_tile + d * kBox, &p.q, &bars.q_full, d * 64, i0, h, b);
          tma_load_4d(g_tile + d * kBox, &p.g, &bars.q_full, d * 64, i0, h, b);
        }
        for (int e = 0; ok && e < 2 * tiles.n; ++e) {
          if (!(ok = bar_wait(&bars.empty[stage], phase, stop, &p.watch))) break;
          bar_expect(&bars.full[stage], kTile);
          armed ^= 1u << stage;
          for (int d = 0; d < DB; ++d)
            tma_load_4d(ring + stage * kTile + d * kBox, e & 1 ? &p.v : &p.k, &bars.full[stage], d * 64,
                        tiles.first(e >> 1), h / w.group, b);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
      }
      bars.armed = armed;
    }
  } else if (warp == 1) {
    {
      const Products<DB, kCols> mm(BF16, w.c.dim);
      const uint32_t qa = smem_addr(q_tile), ga = smem_addr(g_tile), ra = smem_addr(ring);
      uint32_t done = 0;  // tile pairs of earlier items: K of pair t is ring entry 2 (done + t), V the next
      uint32_t q_phase = 0;
      bool ok = true;
      auto ready = [&](uint32_t e) {
        return ok = ok && warp_wait(&bars.full[e % kStages], e / kStages & 1, stop, &p.watch);
      };
      auto tile = [&](uint32_t e) { return ra + e % kStages * kTile; };
      auto s_at = [&](uint32_t t) { return tmem + (t & 1) * 128; };
      for (int x = blockIdx.x; ok && x < p.items; x += gridDim.x) {
        int b, h, i0;
        item(x, b, h, i0);
        const KeyTiles<kT> tiles(key_range(w, b, i0, i0 + kT - 1));
        if (tiles.n == 0) continue;
        if (!(ok = warp_wait(&bars.q_full, q_phase, stop, &p.watch))) break;
        q_phase ^= 1;
        auto scores = [&](uint32_t t) {
          if (!ready(2 * t)) return;
          fence_after();
          mm.scores(s_at(t), qa, tile(2 * t));
          mma_commit(mm.leader, &bars.s_full[t & 1]);
        };
        auto grads = [&](uint32_t t, bool last) {
          if (!ready(2 * t + 1)) return;
          fence_after();
          mm.scores(t_dp, ga, tile(2 * t + 1));
          mma_commit(mm.leader, &bars.dp_full);
          mma_commit(mm.leader, &bars.empty[(2 * t + 1) % kStages]);
          if (last) mma_commit(mm.leader, &bars.q_empty);
        };
        scores(done);
        grads(done, tiles.n == 1);
        for (int t = 0; ok && t < tiles.n; ++t) {
          const uint32_t e = done + t;
          if (t + 1 < tiles.n) scores(e + 1);
          if (!(ok = ok && warp_wait(&bars.ds_full, e & 1, stop, &p.watch))) break;
          fence_after();
          mm.sums(t_dq, t_dp, tile(2 * e), t > 0);
          mma_commit(mm.leader, &bars.empty[2 * e % kStages]);
          if (t + 1 < tiles.n) grads(e + 1, t + 2 == tiles.n);
        }
        mma_commit(mm.leader, &bars.dq_full);
        done += tiles.n;
      }
    }
  } else {
    const int part = (warp - 2) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const float c = w.c.scale * kLog2e;
    const float2 c2 = make_float2(c, c);
    uint32_t done = 0;
    uint32_t dq_phase = 0;
    bool ok = true;
    for (int x = blockIdx.x; ok && x < p.items; x += gridDim.x) {
      int b, h, i0;
      item(x, b, h, i0);
      const KeyTiles<kT> tiles(key_range(w, b, i0, i0 + kT - 1));
      const int i = i0 + row;
      const bool inside = i < w.c.q_len;
      const QuerySpan span = query_span(w, b, i);
      const int all_low = __reduce_max_sync(~0u, span.p < 0 ? INT_MAX : span.low);
      const int all_end = __reduce_min_sync(~0u, span.p < 0 ? -1 : span.p) + 1;
      const int64_t stat = ((int64_t)b * w.c.q_heads + h) * w.lse_row + i;
      const float lse = inside ? w.c.lse[stat] : -INFINITY, delta = inside ? w.c.delta[stat] : 0.f;
      const float2 lse2 = make_float2(lse, lse), delta2 = make_float2(delta, delta);
      for (int t = 0; t < tiles.n; ++t) {
        const uint32_t e = done + t;
        const int j0 = tiles.first(t) + part * kCols, j1 = tiles.end(t);
        const bool masked = !(j0 >= all_low && j0 + kCols <= all_end && j1 - j0 >= kCols);
        uint32_t seen[kCols / 32];
        {
          const int b0 = span.low - j0, b1 = min(span.p + 1, j1) - j0, s0 = span.start - j0,
                    s1 = min(span.sink_end, j1) - j0;
          
#pragma unroll
          for (int y = 0; y < kCols / 32; ++y) seen[y] = bits(b0, b1, y * 32) | bits(s0, s1, y * 32);
        }
        if (!(ok = warp_wait(&bars.s_full[e & 1], e >> 1 & 1, stop, &p.watch))) break;
        fence_after();
        const uint32_t t_s = tmem + (e & 1) * 128 + lanes + part * kCols, t_d = t_dp + lanes + part * kCols;
        float2 pr[kCols / 2];
        auto weights = [&](auto mask) {
          uint32_t z[kCols];
#pragma unroll
          for (int y = 0; y < kCols; y += 16) tmem_ld16(t_s + y, z + y);
          wait_ld();
#pragma unroll
          for (int y = 0; y < kCols; y += 32) tie32(z + y);
#pragma unroll
          for (int y = 0; y < kCols / 16; ++y) {
            const uint32_t *zz = z + y * 16;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int col = y * 16 + 2 * u;
              float2 f = fma2(make_float2(__uint_as_float(zz[2 * u]), __uint_as_float(zz[2 * u + 1])), c2, lse2);
              f.x = exp2_fast(f.x), f.y = exp2_fast(f.y);
              if (mask) {
                if (!(seen[col >> 5] >> (col & 31) & 1)) f.x = 0.f;
                if (!(seen[col >> 5] >> (col & 31) & 2)) f.y = 0.f;
              }
              pr[y * 8 + u] = f;
            }
          }
        };
        if (masked) weights(std::true_type{}); else weights(std::false_type{});
        if (!(ok = warp_wait(&bars.dp_full, e & 1, stop, &p.watch))) break;
        fence_after();
        auto grads = [&](auto mask) {
          uint32_t z[kCols], pk[kCols / 2];
#pragma unroll
          for (int y = 0; y < kCols; y += 16) tmem_ld16(t_d + y, z + y);
          wait_ld();
#pragma unroll
          for (int y = 0; y < kCols; y += 32) tie32(z + y);
#pragma unroll
          for (int y = 0; y < kCols / 16; ++y) {
            const uint32_t *zz = z + y * 16;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int col = y * 16 + 2 * u;
              float2 f = add2(make_float2(__uint_as_float(zz[2 * u]), __uint_as_float(zz[2 * u + 1])), delta2);
              f = mul2(f, pr[y * 8 + u]);
              if (mask) {
                if (!(seen[col >> 5] >> (col & 31) & 1)) f.x = 0.f;
                if (!(seen[col >> 5] >> (col & 31) & 2)) f.y = 0.f;
              }
              pk[y * 8 + u] = pack2<BF16>(f.x, f.y);
            }
          }
#pragma unroll
          for (int y = 0; y < kCols / 2; y += 16) tmem_st16(t_d + y, pk + y);
        };
        if (masked) grads(std::true_type{}); else grads(std::false_type{});
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&bars.ds_full);
      }
      if (!ok) break;
      done += tiles.n;
      if (tiles.n > 0) {
        if (!(ok = warp_wait(&bars.dq_full, dq_phase, stop, &p.watch))) break;
        dq_phase ^= 1;
        fence_after();
      }
      T *dq = static_cast<T *>(w.c.dq) + ((b * w.c.q_len + i - lane) * w.c.q_heads + h) * w.c.dim;
      // this warpgroup's columns of dQ; of four only two have some at head sizes up to 64
      constexpr int kOut = DB == 2 ? DB * 64 * kCols / kT : 32;
      const int d0 = part * kOut;
      bool bad = false;
#pragma unroll 1
      for (int d = d0; d < d0 + kOut && d < DB * 64; d += 32) {
        uint32_t o[32];
        if (tiles.n > 0) {
          tmem_ld32(t_dq + lanes + d, o);
          wait_ld();
          tie32(o);
        } else {
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = 0;
        }
        bad = store32<T>(dq, (int64_t)w.c.q_heads * w.c.dim, o, w.c.scale, d, w.c.dim, (int)w.c.q_len - (i - lane)) || bad;
      }
      if (__any_sync(~0u, bad && inside)) {
        // float16: the row's own numbers are finite, a dS was beyond the type's range
        bool hidden = !BF16 && isfinite(lse) && isfinite(delta);
        const PairDots<T> pair(w, b, h, 0, 0);
        for (int t = 0; t < tiles.n; ++t) {
          const int j0 = tiles.first(t);
          if (j0 >= all_low && j0 + kT <= all_end && tiles.end(t) - j0 == kT) continue;
          for (int y = 0; y < kT; y += 32) {
            const bool odd = row_not_finite(pair.k, w.c.k.token, j0 + y + lane, w.c.k_len, w.c.dim);
            for (unsigned left = __ballot_sync(~0u, odd); left; left &= left - 1) {
              const int j = j0 + y + __ffs(left) - 1;
              hidden = hidden || j >= tiles.end(t) || !span.sees(j);
            }
          }
        }
        for (unsigned left = __ballot_sync(~0u, bad && inside && hidden); left; left &= left - 1)
          repair_dq<T>(w, b, h, i - lane + __ffs(left) - 1, d0, d0 + kOut);
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (*stop) settle(bars.full, &bars.q_full, &bars.idle, bars.armed);
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 512);
}

template <typename T, int DB> void launch(Params &p, cudaStream_t s) {
  const WindowProblem &w = p.w;
  if (w.c.dq && w.c.q_len > 0) {
    auto kernel = dq_tc_kernel<T, DB>;
    MSX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kQSmem<DB>));
    kernel<<<(unsigned)std::min(p.items, num_sms()), threads_for(kQCols<DB>), kQSmem<DB>, s>>>(p);
    MSX_CHECK_LAUNCH();
  }
  if (w.c.dk) {
    auto run = [&](auto kernel, int64_t grid) {
      grid *= w.c.batch * w.c.k_heads;
      if (grid > INT32_MAX) fail(MSX_ERR_OVERFLOW, "window_attention has too many key tiles for one call.");
      MSX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvSmem<DB>));
      kernel<<<(unsigned)grid, threads_for(kKvCols), kKvSmem<DB>, s>>>(p);
      MSX_CHECK_LAUNCH();
    };
    if (p.chunk) run(dkv_tc_kernel<T, DB, true>, (int64_t)p.n_chunks * far_key_tiles(w));
    run(dkv_tc_kernel<T, DB, false>, ceil_div(w.c.k_len, kT));
  }
}

// Queries of a chunk, a multiple of the tile: about 256 chunks over all sequences
// and key heads, of two tiles at least. 0 where one chunk would hold all queries,
// where no query lies outside the window, or with more sinks than a tile of keys
// (then their tiles are several, and the products over them no longer mostly idle).
int pick_chunk(const WindowProblem &w) {
  if (w.sinks == 0 || w.sinks > kT || w.window >= w.c.k_len) return 0;
  const int64_t tiles = ceil_div(w.c.q_len, kT);
  const int64_t n = std::max<int64_t>(2, ceil_div(tiles * w.c.batch * w.c.k_heads, 256));
  return n >= tiles ? 0 : (int)n * kT;
}

}  // namespace

int64_t window_backward_floats_tc(const WindowProblem &w) {
  const int chunk = pick_chunk(w);
  return chunk ? w.c.batch * w.c.k_heads * ceil_div(w.c.q_len, chunk) * w.sinks * 2 * w.c.dim : 0;
}

void window_backward_tc(const WindowProblem &w, int value_dtype, cudaStream_t s) {
  if (w.c.batch == 0) return;
  if (w.c.q_len == 0) return window_backward_general(w, value_dtype, s);  // zeros
  window_delta(w, value_dtype, s);
  Params p{};
  p.w = w;
  const bool bf16 = value_dtype == MSX_BF16;
  const int64_t heads = w.c.q_heads, dim = w.c.dim;
  const WindowTensor g{w.c.grad_out, w.c.q_len * heads * dim, heads * dim, dim};
  p.q = make_map(w.c.q, w.c.batch, w.c.q_len, heads, dim, bf16, kT);
  p.g = make_map(g, w.c.batch, w.c.q_len, heads, dim, bf16, kT);
  p.k = make_map(w.c.k, w.c.batch, w.c.k_len, w.c.k_heads, dim, bf16, kT);
  p.v = make_map(w.c.v, w.c.batch, w.c.k_len, w.c.k_heads, dim, bf16, kT);
  p.q_tiles = (int)ceil_div(w.c.q_len, kT);
  const int64_t items = w.c.batch * heads * p.q_tiles;
  if (items > INT32_MAX / 2) fail(MSX_ERR_OVERFLOW, "window_attention has too many queries and heads for one call.");
  p.items = (int)items;
  p.watch = window_watch();
  p.chunk = pick_chunk(w);
  p.n_chunks = p.chunk ? (int)ceil_div(w.c.q_len, p.chunk) : 0;
  p.far = w.c.delta + w.c.batch * heads * w.lse_row;
  if (bf16) {
    if (dim <= 64) launch<__nv_bfloat16, 1>(p, s); else launch<__nv_bfloat16, 2>(p, s);
  } else {
    if (dim <= 64) launch<__half, 1>(p, s); else launch<__half, 2>(p, s);
  }
}

}  // namespace msx
