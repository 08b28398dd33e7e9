// What the tensor-core kernels of windowed attention share.
#pragma once
#include <cudaTypedefs.h>

#include <type_traits>

#include "tc.cuh"
#include "window_attention.cuh"

namespace msx {

constexpr int kBox = 128 * 128;  // bytes of a TMA box: 128 rows of 64 elements
constexpr float kLog2e = 1.4426950408889634f;

// ex2.approx: within 2 ulp; results below 2^-126 are flushed to 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations for one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// The largest of three numbers; NaNs are left out.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Bits [lo, hi) of the 32 that start at bit `from`.
__device__ __forceinline__ uint32_t bits(int lo, int hi, int from) {
  lo = max(lo - from, 0), hi = min(hi - from, 32);
  return hi <= lo ? 0u : (~0u >> (32 - hi)) & (~0u << lo);
}

// Products issued by a warp's leader, of 128 x 128 tiles of scores (64 columns
// would take nearly as long: 465 clocks against 530); DB boxes of 64 elements cover
// the head size. Scores: both operands K-major in shared memory. Sums: the left
// operand in tensor memory, where each run of W columns of scores holds its 16-bit
// values in its first W / 2; the right operand MN-major in shared memory. Unrolled: the issuing warp is on the critical path of
// every tile.
constexpr int kHalf = 64;                // columns of scores that are handled together
template <int DB, int W = 64> struct Products {
  bool leader;
  int k_steps;
  uint32_t scores_desc, sums_desc;
  __device__ Products(bool bf16, int dim) : leader((threadIdx.x & 31) == 0), k_steps((dim + 15) / 16) {
    scores_desc = tc::mma_desc(bf16, 128, 128, false, false);
    sums_desc = tc::mma_desc(bf16, 128, k_steps * 16, false, true);
  }
  __device__ __forceinline__ void scores(uint32_t d, uint32_t a, uint32_t b) const {
    const uint32_t x = tc::desc_k_major(a), y = tc::desc_k_major(b);
#pragma unroll
    for (int k = 0; k < DB * 4; ++k)
      if (k < k_steps) {
        const uint32_t off = ((k >> 2) * kBox + (k & 3) * 32) >> 4;
        tc::mma_ss(leader, d, x + off, y + off, scores_desc, k > 0);
      }
  }
  __device__ __forceinline__ void sums(uint32_t d, uint32_t left, uint32_t b, bool add) const {
    const uint32_t y = tc::desc_mn_major(b, kBox);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      tc::mma_ts(leader, d, left + k * 16 / W * W + k * 16 % W / 2, y + (k * 2048 >> 4), sums_desc, add || k > 0);
  }
};

// Writes 32 accumulator columns [d0, d0 + 32) of a warp's 32 rows, scaled and
// rounded; `first` is the first row, rows from `rows` on are left out. A thread
// has a row's columns; 4 threads exchange 16-byte pieces so that they write 64
// bytes of one row together (a row each would be 32 lines for each store: 4096
// clocks for two slots' tiles). True where a value of this thread's own row is not
// finite.
template <typename T>
__device__ __forceinline__ bool store32(T *first, int64_t row_stride, const uint32_t *o, float scale, int d0, int dim,
                                        int rows) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  const int lane = threadIdx.x & 31, c = lane & 3;
  float2 odd = make_float2(0.f, 0.f);  // 0 times an infinity or a NaN is NaN
  uint32_t v[4][4];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const bool inside = d0 + 8 * y < dim;  // whole 16-byte pieces
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      float2 a = make_float2(__uint_as_float(o[8 * y + 2 * z]), __uint_as_float(o[8 * y + 2 * z + 1]));
      if (!inside) a = make_float2(0.f, 0.f);
      a = mul2(a, make_float2(scale, scale));
      odd = fma2(a, make_float2(0.f, 0.f), odd);
      v[y][z] = pack2<BF16>(a.x, a.y);
    }
  }
  const bool bad = !(odd.x + odd.y == 0.f);
#pragma unroll
  for (int bit = 1; bit < 4; bit *= 2)
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (!(y & bit)) {
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const uint32_t got = __shfl_xor_sync(~0u, c & bit ? v[y][z] : v[y | bit][z], bit);
          if (c & bit) v[y][z] = got; else v[y | bit][z] = got;
        }
      }
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const int r = (lane & ~3) + y, d = d0 + 8 * c;
    if (r < rows && d < dim)
      *reinterpret_cast<uint4 *>(first + r * row_stride + d) = make_uint4(v[y][0], v[y][1], v[y][2], v[y][3]);
  }
  return bad;
}

// Whether row t of a 16-bit matrix (dim elements from `p`, a multiple of 8,
// 16-byte aligned) holds an infinity or a NaN; rows outside [0, limit) do not.
template <typename T> __device__ inline bool row_not_finite(const T *p, int64_t token_stride, int64_t t, int64_t limit, int dim) {
  if (t < 0 || t >= limit) return false;
  const uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  const uint4 *v = reinterpret_cast<const uint4 *>(p + t * token_stride);
  bool bad = false;
  for (int x = 0; x < dim / 8; ++x) {
    const uint4 u = v[x];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int y = 0; y < 4; ++y) bad = bad || (w[y] & e & 0xffffu) == (e & 0xffffu) || (w[y] & e & 0xffff0000u) == (e & 0xffff0000u);
  }
  return bad;
}

// ---- host ---------------------------------------------------------------------
tc::Watch window_watch();  // the current device's error flag and the limit of waits (window_forward_tc.cu)

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// Boxes of 64 elements by `rows` tokens of one head; what lies outside the
// tensor (elements past the head size, tokens past the end) reads as 0.
inline CUtensorMap make_map(const WindowTensor &t, int64_t batch, int64_t tokens, int64_t heads, int64_t dim, bool bf16,
                     int rows) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
  if (fn == nullptr) fail(MSX_ERR_RUNTIME, "the driver does not offer cuTensorMapEncodeTiled.");
  CUtensorMap map;
  const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)tokens, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)t.token * 2, (cuuint64_t)t.head * 2, (cuuint64_t)t.batch * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = fn(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                        const_cast<void *>(t.ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(MSX_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r) + ".");
  return map;
}

// Strides and base that a tensor map takes.
inline bool tma_ready(const WindowTensor &t) {
  const int64_t most = (int64_t)1 << 39;  // elements; strides stay below 2^40 bytes
  auto good = [&](int64_t x) { return x > 0 && x % 8 == 0 && x < most; };
  return reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0 && good(t.batch) && good(t.token) && good(t.head);
}

}  // namespace msx
