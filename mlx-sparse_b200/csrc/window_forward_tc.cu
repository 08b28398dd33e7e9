// Windowed attention, forward, on the tensor cores (float16 / bfloat16, head
// sizes that are multiples of 8 up to 128).
//
// A persistent CTA takes work items of two "slots" of 128 queries each: two
// heads that share a key head, or two neighbouring query tiles of one head where
// the group is odd. It walks the tiles of 128 keys that they see, the sink
// tiles and then the band's, and no others. One warp loads Q, K and V tiles by
// TMA into a ring of shared memory; one warp issues tcgen05.mma; a warpgroup
// for each slot does its softmax, a query row for each thread, straight from
// tensor memory. Scores and output of a slot stay there (S 128 columns, O 128, two
// slots: all 512). The probabilities, rounded to the inputs' type for the second
// product (half a step each, against sums held in fp32), take the place of the
// scores and are read from there as its left operand. While one slot's softmax
// runs, the other slot's products do.
//
// The running maximum is only raised when a row's new maximum is 2^8 above the
// one in use, so the output is rescaled in tensor memory a few times at most;
// the probabilities stay below 2^8 and the sum is of the same unrounded values.
//
// A masked score is -inf before the softmax, whatever it was. Its probability
// is 0, but 0 times an infinite or NaN value row would still reach the second
// product: rows that end not finite are computed again pair by pair where
// something not finite hides among their tiles' other keys.
//
// Bound: the products (2 x 520 clocks for 128 x 128 scores at head size 128) and
// the exponentials (16 a clock and SM: 1024 clocks) take about the same time, side by
// side; beside a busy softmax a product takes about 700 clocks, and neither unit is
// busy half of the time. 32768 tokens, window 4096, 32 / 8 heads of 128, bf16: 2.22
// ms, 930 TFLOP/s. Ten warps leave a thread 168 registers; all variants spill, some 12
// loads and 6 stores for each warp and tile of keys.
#include <algorithm>
#include <atomic>

#include "window_tc.cuh"

namespace msx {

using namespace tc;

namespace {

__device__ int g_window_error;

constexpr int kM = 128;  // queries of a slot: the lanes of tensor memory
constexpr int kN = 128;  // keys of a tile
constexpr int kThreads = 64 + 2 * 128;  // loads, products, two softmax warpgroups

struct Bars {
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2];
  uint64_t kv_full[8], step[8], idle;
  uint32_t tmem, armed;  // armed: the last phases of kv_full (bits 0-7) and q_full (8, 9), see bar_settle
  int stop;
  float max1[kM], sum1[kM];  // the second slot's, where both share the queries
};

template <int DB> struct Shape {  // DB boxes of 64 elements cover the head size
  static constexpr int tile = DB * kBox;
  static constexpr int stages = DB == 2 ? 5 : 8;
  static constexpr int smem = (2 + stages) * tile + (int)sizeof(Bars);
};

struct Params {
  WindowProblem w;
  CUtensorMap q, k, v;
  int items, q_tiles, paired;
  Watch watch;
};

// One work item: the two slots' heads and first queries, and the keys of each
// and of both.
struct Item {
  int b, hk, head[2], i0[2];
  KeyRange range[2], both;
  int last[2];  // the last tile of keys that a slot takes part in, -1: none
};

template <bool SPLIT> __device__ __forceinline__ Item item_of(const Params &p, int n) {
  const WindowProblem &w = p.w;
  Item it;
  if (SPLIT) {
    it.i0[0] = it.i0[1] = n % p.q_tiles * kM;
    n /= p.q_tiles;
    it.head[0] = it.head[1] = n % w.c.q_heads;
    it.b = n / w.c.q_heads;
    it.hk = it.head[0] / w.group;
    it.both = it.range[0] = it.range[1] = key_range(w, it.b, it.i0[0], it.i0[0] + kM - 1);
    const int tiles = KeyTiles<kN>(it.both).n;
    it.last[0] = tiles == 0 ? -1 : (tiles - 1) & ~1;
    it.last[1] = tiles < 2 ? -1 : (tiles - 2) | 1;
  } else if (p.paired) {
    const int pairs = w.group / 2;
    const int pair = n % pairs;
    n /= pairs;
    it.i0[0] = it.i0[1] = n % p.q_tiles * kM;
    n /= p.q_tiles;
    it.hk = n % w.c.k_heads;
    it.b = n / w.c.k_heads;
    it.head[0] = it.hk * w.group + 2 * pair;
    it.head[1] = it.head[0] + 1;
    it.both = it.range[0] = it.range[1] = key_range(w, it.b, it.i0[0], it.i0[0] + kM - 1);
    it.last[0] = it.last[1] = KeyTiles<kN>(it.both).n - 1;
  } else {
    const int blocks = (p.q_tiles + 1) / 2;
    const int h = n / blocks % w.c.q_heads;
    it.b = n / blocks / w.c.q_heads;
    it.hk = h / w.group;
    it.head[0] = it.head[1] = h;
    it.i0[0] = n % blocks * 2 * kM;
    it.i0[1] = it.i0[0] + kM;
    it.both = key_range(w, it.b, it.i0[0], it.i0[1] + kM - 1);
    const KeyTiles<kN> tiles(it.both);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      it.range[s] = key_range(w, it.b, it.i0[s], it.i0[s] + kM - 1);
      it.last[s] = it.range[s].empty() ? -1 : tiles.n - 1;
      while (it.last[s] >= 0 && !it.range[s].touches(tiles.first(it.last[s]), tiles.end(it.last[s]))) --it.last[s];
    }
  }
  return it;
}

// One row again, by a warp, pair by pair: only what the query sees is touched.
template <typename T>
__device__ __noinline__ void repair_row(const WindowProblem &w, int b, int h, int i) {
  const int lane = threadIdx.x & 31, dim = w.c.dim, hk = h / w.group;
  const T *q = static_cast<const T *>(w.c.q.ptr) + b * w.c.q.batch + h * w.c.q.head + i * w.c.q.token;
  const T *k = static_cast<const T *>(w.c.k.ptr) + b * w.c.k.batch + hk * w.c.k.head;
  const T *v = static_cast<const T *>(w.c.v.ptr) + b * w.c.v.batch + hk * w.c.v.head;
  const QuerySpan span = query_span(w, b, i);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < 2; ++part) {
    const int from = part ? span.low : span.start, end = part ? span.p + 1 : span.sink_end;
    for (int j0 = from; j0 < end; j0 += 32) {
      const int j = j0 + lane;
      float s = -INFINITY;
      if (j < end) {
        s = 0.f;
        for (int d = 0; d < dim; ++d) s = fmaf(VT<T>::load(q[d]), VT<T>::load(k[j * w.c.k.token + d]), s);
        s *= w.c.scale * kLog2e;
      }
      float top = s;
#pragma unroll
      for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
      top = fmaxf(top, m);
      const float base = top == -INFINITY ? 0.f : top, keep = exp2f(m - base);
      const float p = j < end ? exp2f(s - base) : 0.f;
      float sum = p;
#pragma unroll
      for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
      l = l * keep + sum, m = top;
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[x] *= keep;
      for (int kk = 0; kk < min(32, end - j0); ++kk) {
        const float pk = __shfl_sync(~0u, p, kk);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (x * 32 + lane < dim) acc[x] = fmaf(pk, VT<T>::load(v[(j0 + kk) * w.c.v.token + x * 32 + lane]), acc[x]);
      }
    }
  }
  const int64_t at = ((b * w.c.q_len + i) * w.c.q_heads + h) * dim;
  T *out = static_cast<T *>(w.c.out) + at;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int d = x * 32 + lane;
    if (d >= dim) continue;
    out[d] = VT<T>::store(acc[x] / l);
    if (w.c.out_low) static_cast<T *>(w.c.out_low)[at + d] = VT<T>::store(acc[x] / l - VT<T>::load(out[d]));
  }
  if (w.c.lse && lane == 0) w.c.lse[((int64_t)b * w.c.q_heads + h) * w.lse_row + i] = -(m + log2f(l));
}

// SPLIT: both slots share the queries. LOW: what the rounding of the output takes
// off is kept too. (As run-time branches the two cost the other calls 10%.)
template <typename T, int DB, bool SPLIT, bool LOW>
__global__ void __launch_bounds__(kThreads, 1) forward_tc_kernel(const __grid_constant__ Params p) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  using Sh = Shape<DB>;
  extern __shared__ __align__(1024) unsigned char sm[];  // no static shared memory: all 227 KB are needed
  Bars &bars = *reinterpret_cast<Bars *>(sm + (2 + Sh::stages) * Sh::tile);
  unsigned char *q_tile = sm, *kv_tile = sm + 2 * Sh::tile;
  const WindowProblem &w = p.w;
  const int warp = __shfl_sync(~0u, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int *stop = &bars.stop;
  if (smem_addr(sm) % 1024 != 0) {  // the swizzle's atoms would not lie where they are read
    *p.watch.error = 1;
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      bar_init(&bars.q_full[s], 1), bar_init(&bars.q_empty[s], 1);
      bar_init(&bars.s_full[s], 1), bar_init(&bars.p_full[s], 4), bar_init(&bars.o_full[s], 1);
    }
    for (int s = 0; s < Sh::stages; ++s) bar_init(&bars.kv_full[s], 1);
    for (int s = 0; s < 8; ++s) bar_init(&bars.step[s], 1);
    bar_init(&bars.idle, 1);
    bars.stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&bars.tmem, 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(~0u, bars.tmem, 0);
  if (warp == 0) {
    // ---- loads -------------------------------------------------------------
    if (lane == 0) {
      uint32_t q_phase[2] = {1, 1};  // an empty barrier's first wait passes
      uint32_t armed = 0xff;
      // Step g of all tiles so far frees V of tile g, K of tile g + 1 and, where that
      // is an item's first, K of tile g: an item's entries of the ring, K and V in
      // turn, are free after the steps t - 1 (0 for the first) and t. `freed`: the
      // step that frees each stage's entry. It has barrier freed % 8, more than the
      // steps that the ring lets the products run ahead.
      int64_t base = 0, freed[Sh::stages];
#pragma unroll
      for (int x = 0; x < Sh::stages; ++x) freed[x] = -1;
      int stage = 0;
      bool ok = true;
      for (int n = blockIdx.x; ok && n < p.items; n += gridDim.x) {
        const Item it = item_of<SPLIT>(p, n);
        const KeyTiles<kN> tiles(it.both);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (it.last[s] < 0) continue;
          ok = ok && bar_wait(&bars.q_empty[s], q_phase[s], stop, &p.watch);
          if (!ok) break;
          q_phase[s] ^= 1;
          bar_expect(&bars.q_full[s], Sh::tile);
          for (int x = 0; x < DB; ++x)
            tma_load_4d(q_tile + s * Sh::tile + x * kBox, &p.q, &bars.q_full[s], x * 64, it.i0[s], it.head[s], it.b);
        }
        for (int t = 0; ok && t < tiles.n; ++t) {
          for (int kv = 0; kv < 2; ++kv) {
            const int64_t g = freed[stage];
            if (g >= 0 && !(ok = bar_wait(&bars.step[g & 7], (uint32_t)(g >> 3 & 1), stop, &p.watch))) break;
            freed[stage] = base + (kv || t == 0 ? t : t - 1);
            bar_expect(&bars.kv_full[stage], Sh::tile);
            armed ^= 1u << stage;
            for (int x = 0; x < DB; ++x)
              tma_load_4d(kv_tile + stage * Sh::tile + x * kBox, kv ? &p.v : &p.k, &bars.kv_full[stage], x * 64,
                          tiles.first(t), it.hk, it.b);
            if (++stage == Sh::stages) stage = 0;
          }
        }
        base += tiles.n;
      }
      bars.armed = armed | q_phase[0] << 8 | q_phase[1] << 9;
    }
  } else if (warp == 1) {
    // ---- products ------------------------------------------------------------
    const Products<DB> mm(BF16, w.c.dim);
    const uint32_t q_addr = smem_addr(q_tile), kv_addr = smem_addr(kv_tile);
    int stage = 0;
    uint32_t phase = 0, steps = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
    bool ok = true;
    auto need = [&](bool waited) { return ok = ok && waited; };
    auto next = [&] {
      if (++stage == Sh::stages) stage = 0, phase ^= 1;
    };
    for (int n = blockIdx.x; ok && n < p.items; n += gridDim.x) {
      const Item it = item_of<SPLIT>(p, n);
      const KeyTiles<kN> tiles(it.both);
      if (tiles.n == 0) continue;
      auto takes = [&](int s, int t) {
        return SPLIT ? (t & 1) == s : p.paired || it.range[s].touches(tiles.first(t), tiles.end(t));
      };
      auto scores = [&](int s, int st, bool last_one) {
        mm.scores(tmem + s * kN, q_addr + s * Sh::tile, kv_addr + st * Sh::tile);
        mma_commit(mm.leader, &bars.s_full[s]);
        if (last_one) mma_commit(mm.leader, &bars.q_empty[s]);
      };
      bool started[2] = {false, false};
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (it.last[s] >= 0) {
          need(warp_wait(&bars.q_full[s], q_phase[s], stop, &p.watch));
          q_phase[s] ^= 1;
        }
      // the stage of K_0 is now, V_t and K_{t+1} follow in turn
      if (!need(warp_wait(&bars.kv_full[stage], phase, stop, &p.watch))) break;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (takes(s, 0)) scores(s, stage, it.last[s] == 0);
      next();
      for (int t = 0; ok && t < tiles.n; ++t) {
        const int v_stage = stage;
        const uint32_t v_phase = phase;
        const bool more = t + 1 < tiles.n;
        if (SPLIT) {
          // the slots take turns: the other one's scores before this one's output
          next();
          if (more) {
            if (!need(warp_wait(&bars.kv_full[stage], phase, stop, &p.watch))) break;
#pragma unroll
            for (int s = 0; s < 2; ++s)
              if ((t & 1) != s) scores(s, stage, it.last[s] == t + 1);
          }
          need(warp_wait(&bars.kv_full[v_stage], v_phase, stop, &p.watch));
#pragma unroll
          for (int s = 0; s < 2; ++s)
            if ((t & 1) == s) {
              need(warp_wait(&bars.p_full[s], p_phase[s], stop, &p.watch));
              fence_after();
              mm.sums(tmem + 256 + s * 128, tmem + s * kN, kv_addr + v_stage * Sh::tile, started[s]);
              if (t == it.last[s]) mma_commit(mm.leader, &bars.o_full[s]);
              p_phase[s] ^= 1;
              started[s] = true;
            }
          mma_commit(mm.leader, &bars.step[steps++ & 7]);
          if (more) next();
          continue;
        }
        if (!need(warp_wait(&bars.kv_full[stage], phase, stop, &p.watch))) break;
        next();
        const int k_stage = stage;
        const bool now[2] = {takes(0, t), takes(1, t)}, then[2] = {more && takes(0, t + 1), more && takes(1, t + 1)};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (now[s]) {
            need(warp_wait(&bars.p_full[s], p_phase[s], stop, &p.watch));
            fence_after();
            mm.sums(tmem + 256 + s * 128, tmem + s * kN, kv_addr + v_stage * Sh::tile, started[s]);
            if (t == it.last[s]) mma_commit(mm.leader, &bars.o_full[s]);
            p_phase[s] ^= 1;
            started[s] = true;
          }
          if (s == 0 && more) need(warp_wait(&bars.kv_full[k_stage], phase, stop, &p.watch));
          if (then[s]) scores(s, k_stage, it.last[s] == t + 1);
        }
        mma_commit(mm.leader, &bars.step[steps++ & 7]);
        if (more) next();
      }
    }
  } else {
    // ---- softmax, a query row for each thread ------------------------------------
    const int s = (warp - 2) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t t_s = tmem + s * kN + lanes, t_o = tmem + 256 + s * 128 + lanes;
    const float c = w.c.scale * kLog2e;
    // What the exponents of a maximum are taken over. Weights of two maxima are
    // joined by the difference of these rounded products, in which their rounding,
    // |c m| 2^-24, cancels (as it would not in c times the difference).
    auto over = [&](float max) { return __fmul_rn(max, c); };
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    for (int n = blockIdx.x; ok && n < p.items; n += gridDim.x) {
      const Item it = item_of<SPLIT>(p, n);
      const KeyTiles<kN> tiles(it.both);
      const KeyRange range = s ? it.range[1] : it.range[0];
      const int i = (s ? it.i0[1] : it.i0[0]) + row, h = s ? it.head[1] : it.head[0];
      const QuerySpan span = query_span(w, it.b, i);
      // the keys that all 32 rows of this warp see: halves inside need no mask
      const int all_low = __reduce_max_sync(~0u, span.p < 0 ? INT_MAX : span.low);
      const int all_end = __reduce_min_sync(~0u, span.p < 0 ? -1 : span.p) + 1;
      float m = -INFINITY, l = 0.f;
      bool started = false;
      for (int t = 0; ok && t < tiles.n; ++t) {
        if (SPLIT ? (t & 1) != s : !p.paired && !range.touches(tiles.first(t), tiles.end(t))) continue;
        if (!(ok = warp_wait(&bars.s_full[s], s_phase, stop, &p.watch))) break;
        fence_after();
        const int j0 = tiles.first(t), j1 = tiles.end(t);
        const bool masked = !(j0 >= all_low && j0 + kN <= all_end && j1 - j0 >= kN);
        uint32_t pk[kN / 2];
        // Scores of the tile: their maximum and, with EXP, their exponentials over the
        // maximum in use, packed, and their sum.
        auto tile = [&](auto exp, auto mask) {
          const float base = m == -INFINITY ? 0.f : over(m);
          const float2 base2 = make_float2(-base, -base), c2 = make_float2(c, c);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          const int b0 = span.low - j0, b1 = min(span.p + 1, j1) - j0, s0 = span.start - j0,
                    s1 = min(span.sink_end, j1) - j0;
#pragma unroll
          for (int x = 0; x < kN; x += 32) {
            uint32_t z[32];
            tmem_ld16(t_s + x, z), tmem_ld16(t_s + x + 16, z + 16);
            wait_ld();
            tie32(z);
            if (mask) {
              const uint32_t seen = bits(b0, b1, x) | bits(s0, s1, x);
#pragma unroll
              for (int y = 0; y < 32; ++y)
                if (!(seen >> y & 1)) z[y] = 0xff800000u;  // -inf
            }
#pragma unroll
            for (int y = 0; y < 32; y += 2)
              tops[y >> 1 & 3] = max3(tops[y >> 1 & 3], __uint_as_float(z[y]), __uint_as_float(z[y + 1]));
            if (exp) {
#pragma unroll
              for (int y = 0; y < 16; ++y) {
                float2 e = fma2(make_float2(__uint_as_float(z[2 * y]), __uint_as_float(z[2 * y + 1])), c2, base2);
                e.x = exp2_fast(e.x), e.y = exp2_fast(e.y);
                sum[y & 1] = add2(sum[y & 1], e);
                pk[x / 2 + y] = pack2<BF16>(e.x, e.y);
              }
            }
          }
          return make_float2(fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]),
                             (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
        };
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        // Later tiles rarely raise the maximum in use: their exponentials are taken
        // at once and only taken again where it had to rise.
        float2 r = !started ? tile(no, yes) : masked ? tile(yes, yes) : tile(yes, no);
        const bool raise = (r.x - m) * c > 8.f;
        if (!started || __any_sync(~0u, raise)) {
          const float keep = raise ? (m == -INFINITY ? 0.f : exp2_fast(over(m) - over(r.x))) : 1.f;
          l *= keep;
          if (raise) m = r.x;
          if (started) {  // the tiles before are in the output: these scores were computed after them
#pragma unroll 1
            for (int x = 0; x < DB * 64; x += 16) {
              uint32_t o[16];
              tmem_ld16(t_o + x, o);
              wait_ld();
              tie16(o);
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * keep);
              tmem_st16(t_o + x, o);
            }
          }
          r = tile(yes, yes);
        }
        tmem_st32(t_s, pk), tmem_st32(t_s + kHalf, pk + 32);
        l += r.y;
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&bars.p_full[s]);
        started = true;
        s_phase ^= 1;
      }
      float keep0 = 1.f, keep1 = 0.f;
      if (SPLIT) {
        // One item a CTA. The first slot's warps write the row; they read the second's
        // output too. The barrier is met on every path.
        if (s == 1) bars.max1[row] = m, bars.sum1[row] = l;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (s == 1 || !ok) break;
        if (it.last[1] >= 0) {
          if (!(ok = warp_wait(&bars.o_full[1], 0, stop, &p.watch))) break;
          const float m1 = bars.max1[row], top = fmaxf(m, m1);
          keep0 = m == -INFINITY ? 0.f : exp2_fast(over(m) - over(top));
          keep1 = m1 == -INFINITY ? 0.f : exp2_fast(over(m1) - over(top));
          l = l * keep0 + bars.sum1[row] * keep1, m = top;
        }
      }
      if (!ok) break;
      if (started) {
        if (!(ok = warp_wait(&bars.o_full[s], o_phase, stop, &p.watch))) break;
        o_phase ^= 1;
        fence_after();
      }
      const bool inside = i < w.c.q_len, empty = span.empty();
      const float inv = empty ? 0.f : 1.f / l;
      const int64_t first = ((it.b * w.c.q_len + i - lane) * w.c.q_heads + h) * w.c.dim;
      T *out = static_cast<T *>(w.c.out) + first;
      bool bad = false;
#pragma unroll
      for (int x = 0; x < DB * 64; x += 32) {
        uint32_t o[32];
        if (started) {
          tmem_ld16(t_o + x, o), tmem_ld16(t_o + x + 16, o + 16);
          wait_ld();
          tie32(o);
          if (SPLIT && it.last[1] >= 0) {
            uint32_t o1[32];
            tmem_ld16(t_o + 128 + x, o1), tmem_ld16(t_o + 128 + x + 16, o1 + 16);
            wait_ld();
            tie32(o1);
#pragma unroll
            for (int y = 0; y < 32; ++y)
              o[y] = __float_as_uint(__uint_as_float(o[y]) * keep0 + __uint_as_float(o1[y]) * keep1);
          }
        }
        if (!started || empty) {
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = 0;
        }
        bad = store32<T>(out, (int64_t)w.c.q_heads * w.c.dim, o, inv, x, w.c.dim, (int)w.c.q_len - (i - lane)) || bad;
        if (LOW) {
#pragma unroll
          for (int y = 0; y < 32; ++y) {
            const float e = __uint_as_float(o[y]) * inv;
            o[y] = __float_as_uint(e - VT<T>::load(VT<T>::store(e)));
          }
          store32<T>(static_cast<T *>(w.c.out_low) + first, (int64_t)w.c.q_heads * w.c.dim, o, 1.f, x, w.c.dim,
                     (int)w.c.q_len - (i - lane));
        }
      }
      if (inside && w.c.lse)
        w.c.lse[((int64_t)it.b * w.c.q_heads + h) * w.lse_row + i] = empty ? -INFINITY : -(over(m) + log2f(l));
      if (__any_sync(~0u, bad && inside)) {
        // What the row sees may be at fault; recompute it only if something not
        // finite hides among the tiles' other keys.
        bool hidden = false;
        const T *v = static_cast<const T *>(w.c.v.ptr) + it.b * w.c.v.batch + it.hk * w.c.v.head;
        for (int t = 0; t < tiles.n; ++t) {
          const int j0 = tiles.first(t);
          if (!range.touches(j0, tiles.end(t)) ||
              (j0 >= all_low && j0 + kN <= all_end && tiles.end(t) - j0 == kN)) continue;
          for (int x = 0; x < kN; x += 32) {
            const unsigned flags = __ballot_sync(~0u, row_not_finite(v, w.c.v.token, j0 + x + lane, w.c.k_len, w.c.dim));
            for (unsigned left = flags; left; left &= left - 1) {
              const int j = j0 + x + __ffs(left) - 1;
              hidden = hidden || j >= tiles.end(t) || !span.sees(j);
            }
          }
        }
        for (unsigned left = __ballot_sync(~0u, bad && inside && hidden); left; left &= left - 1)
          repair_row<T>(w, it.b, h, i - lane + __ffs(left) - 1);
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (*stop) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < Sh::stages; ++s) bar_settle(&bars.kv_full[s], bars.armed >> s & 1);
      for (int s = 0; s < 2; ++s) bar_settle(&bars.q_full[s], bars.armed >> (8 + s) & 1);
    }
    if (warp == 1) mma_commit(lane == 0, &bars.idle), bar_settle(&bars.idle, 0);
  }
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 512);
}

template <typename T, int DB> void launch(Params &p, bool split, cudaStream_t s) {
  auto run = [&](auto kernel) {
    MSX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DB>::smem));
    kernel<<<(unsigned)std::min(p.items, num_sms()), kThreads, Shape<DB>::smem, s>>>(p);
    MSX_CHECK_LAUNCH();
  };
  const bool low = p.w.c.out_low != nullptr;
  if (split)
    low ? run(forward_tc_kernel<T, DB, true, true>) : run(forward_tc_kernel<T, DB, true, false>);
  else
    low ? run(forward_tc_kernel<T, DB, false, true>) : run(forward_tc_kernel<T, DB, false, false>);
}

}  // namespace

static std::atomic<long long> g_wait_ns{kWaitNs};

Watch window_watch() {
  Watch w{};
  MSX_CUDA(cudaGetSymbolAddress(reinterpret_cast<void **>(&w.error), g_window_error));
  w.limit_ns = (unsigned long long)g_wait_ns.load(std::memory_order_relaxed);
  w.polls = w.limit_ns ? 64 : 0;
  return w;
}

void window_set_wait_limit(long long ns) { g_wait_ns.store(ns < 0 ? kWaitNs : ns, std::memory_order_relaxed); }

bool window_take_error() {
  int v = 0;
  MSX_CUDA(cudaMemcpyFromSymbol(&v, g_window_error, sizeof(int)));
  if (v) {
    const int zero = 0;
    MSX_CUDA(cudaMemcpyToSymbol(g_window_error, &zero, sizeof(int)));
  }
  return v != 0;
}

// 16-bit types, head sizes and layouts that TMA can read; the running maximum
// of raw scores needs a positive scale.
bool window_tc_ok(const WindowProblem &w, int value_dtype) {
  return value_dtype != MSX_F32 && w.c.dim % 8 == 0 && w.c.dim <= 128 && w.c.scale > 0.f && w.c.k_len > 0 &&
         tma_ready(w.c.q) && tma_ready(w.c.k) && tma_ready(w.c.v);
}

void window_forward_tc(const WindowProblem &w, int value_dtype, cudaStream_t s) {
  if (w.c.batch == 0 || w.c.q_len == 0) return;
  Params p{};
  p.w = w;
  const bool bf16 = value_dtype == MSX_BF16;
  p.q = make_map(w.c.q, w.c.batch, w.c.q_len, w.c.q_heads, w.c.dim, bf16, kM);
  p.k = make_map(w.c.k, w.c.batch, w.c.k_len, w.c.k_heads, w.c.dim, bf16, kN);
  p.v = make_map(w.c.v, w.c.batch, w.c.k_len, w.c.k_heads, w.c.dim, bf16, kN);
  p.q_tiles = (int)ceil_div(w.c.q_len, kM);
  const bool split = w.c.batch * w.c.q_heads * p.q_tiles <= num_sms();
  p.paired = !split && w.group % 2 == 0;
  const int64_t items = split ? w.c.batch * w.c.q_heads * p.q_tiles
                        : p.paired ? w.c.batch * w.c.k_heads * p.q_tiles * (w.group / 2)
                                 : w.c.batch * w.c.q_heads * ((p.q_tiles + 1) / 2);
  if (items > INT32_MAX / 2) fail(MSX_ERR_OVERFLOW, "window_attention has too many queries and heads for one call.");
  p.items = (int)items;
  p.watch = window_watch();
  if (bf16) {
    if (w.c.dim <= 64) launch<__nv_bfloat16, 1>(p, split, s); else launch<__nv_bfloat16, 2>(p, split, s);
  } else {
    if (w.c.dim <= 64) launch<__half, 1>(p, split, s); else launch<__half, 2>(p, split, s);
  }
}

}  // namespace msx
