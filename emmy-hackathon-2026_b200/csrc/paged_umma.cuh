// Shared by the kernels of paged attention on the 5th-generation tensor cores
// (paged_umma.cu, paged_umma_wide.cu): 16-bit products with P in tensor memory,
// tiles of 128 keys by 64 elements with the 128-byte swizzle, tensor maps.
#pragma once

#include <math.h>

#include <algorithm>

#include "paged.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace umma {

using paged::Args;

constexpr int kRows = 128;    // rows of a tile
constexpr int kKeys = 128;    // keys of a tile
constexpr int kHalf = kKeys * 128;  // bytes of a tile's 64 columns: 128 rows of 128 bytes
constexpr int kMarks = 8;     // tiles whose key marks are kept

// 4-D tile load: (element, row of the page, head, page).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(sm100::smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// Two FP32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}

template <typename T>
struct Type;
template <>
struct Type<__half> {
  static constexpr uint32_t kFormat = 0;
  static constexpr float kLift = 6.0f, kSlack = 8.0f;  // 2^14 at most: within f16
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};
template <>
struct Type<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;
  static constexpr float kLift = 0.0f, kSlack = 8.0f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};

// Instruction descriptor, kind::f16, FP32 accumulate (fields as idesc_tf32).
template <typename T>
__device__ constexpr uint32_t idesc(int n, bool b_mn_major) {
  return (1u << 4) | (Type<T>::kFormat << 7) | (Type<T>::kFormat << 10) | (b_mn_major ? (1u << 16) : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
}

// MN-major 16-bit operand with the 128-byte swizzle: atoms of 64 MN-consecutive
// elements (128 bytes) by 8 K rows (1024 bytes); bits 16-29 the stride between
// atoms along MN, bits 32-45 along K.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t mn_stride, uint32_t k_stride) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | static_cast<uint64_t>((mn_stride >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>((k_stride >> 4) & 0x3FFFu) << 32 | static_cast<uint64_t>(1u) << 46 |
         static_cast<uint64_t>(2u) << 61;
}

// Four products D (+)= A B of 16 steps of K each, issued by one elected lane of a
// converged warp: A in shared memory, K-major like B, 32 bytes (2 units of a
// descriptor's address) a step; or A in tensor memory, eight columns a step,
// and B N-major, 2048 bytes a step.  The first overwrites D unless `accumulate`.
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
      "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p, t;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.s64 b1, %2, 128;\n\tadd.u32 a2, %1, 16;\n\tadd.s64 b2, %2, 256;\n\t"
      "add.u32 a3, %1, 24;\n\tadd.s64 b3, %2, 384;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}

// [pages][heads][page rows][d] of a cache in any order of strides, boxes of 64
// elements by a page's rows (128 at most).
template <typename T>
int make_map(b2k_ctx *ctx, CUtensorMap *map, const Args &a, bool keys) {
  auto encode = b2k::tensor_map_encoder();
  if (!encode) return b2k::fail(ctx, B2K_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  const void *base = keys ? a.k : a.v;
  const int64_t row = keys ? a.k_row : a.v_row, head = keys ? a.k_head : a.v_head, page = keys ? a.k_page : a.v_page;
  cuuint64_t dims[4] = {(cuuint64_t)a.d, (cuuint64_t)a.page_size, (cuuint64_t)a.kv_heads, (cuuint64_t)a.pages};
  cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)head * 2, (cuuint64_t)page * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)std::min(a.page_size, kKeys), 1, 1};
  cuuint32_t elem[4] = {1, 1, 1, 1};
  const CUresult res =
      encode(map, Type<T>::kFormat ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (res != CUDA_SUCCESS) return b2k::fail(ctx, B2K_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)res);
  return B2K_OK;
}

// Whether pages are boxes: whole swizzle atoms (8 rows) that tile 128 keys, or
// 128 keys a part of one; and strides and extents a tensor map can hold.
inline bool boxes_fit(const Args &a) {
  const int64_t most = (int64_t)1 << 38;  // 2^39 bytes
  return a.page_size >= 8 && (kKeys % a.page_size == 0 || a.page_size % kKeys == 0) && a.pages <= INT32_MAX &&
         a.k_row < most && a.k_head < most && a.k_page < most && a.v_row < most && a.v_head < most && a.v_page < most;
}

// Queries [tokens][heads][d], boxes of 64 elements by a cache head's query heads
// by the tokens that make 128 rows.
template <typename T>
int make_q_map(b2k_ctx *ctx, CUtensorMap *map, const Args &a) {
  auto encode = b2k::tensor_map_encoder();
  if (!encode) return b2k::fail(ctx, B2K_ECUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)a.d, (cuuint64_t)(a.kv_heads * a.group), (cuuint64_t)a.tokens};
  cuuint64_t strides[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_token * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(kRows / a.group)};
  cuuint32_t elem[3] = {1, 1, 1};
  const CUresult res =
      encode(map, Type<T>::kFormat ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
             const_cast<void *>(a.q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (res != CUDA_SUCCESS) return b2k::fail(ctx, B2K_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)res);
  return B2K_OK;
}

// Whether the queries are boxes of tokens by heads.  (A single head's stride is
// not used, but a tensor map wants one it can hold.)
inline bool query_boxes_fit(const Args &a) {
  const int64_t most = (int64_t)1 << 38;
  return kRows % a.group == 0 && a.q_head > 0 && a.q_token > 0 && a.q_head < most && a.q_token < most;
}

// A warp's 32 rows to memory, one a lane, 128 bytes of each at a time through 4 KB
// of shared memory, so that a store instruction writes whole lines of four rows
// (16 bytes of 32 rows each instead take about 4000 cycles more at a block's end).  `own`: the row's
// place in `out`, elements, -1 for none; load(c, w): its 128 bytes from element c.
template <typename E, typename Load>
__device__ __forceinline__ void store_rows(uint8_t *stage, E *out, int64_t own, int d, Load load) {
  constexpr int kPiece = 16 / sizeof(E);
  const int lane = threadIdx.x & 31, piece = lane & 7;
  int64_t to[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) to[i] = __shfl_sync(0xffffffffu, own, 4 * i + (lane >> 3));
  for (int c = 0; c < d; c += 8 * kPiece) {
    uint32_t w[32];
    __syncwarp();  // the last step's pieces have been read; the load is the whole warp's
    load(c, w);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      *reinterpret_cast<uint4 *>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) =
          make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 4 * i + (lane >> 3);
      const uint4 v = *reinterpret_cast<const uint4 *>(stage + row * 128 + ((piece ^ (row & 7)) << 4));
      if (to[i] >= 0 && c + piece * kPiece < d) *reinterpret_cast<uint4 *>(out + to[i] + c + piece * kPiece) = v;
    }
  }
}

// The same from the accumulator at o_at: rounded to T and times inv, or in FP32;
// zeros where `some` is false (a row without keys).  `filled`: the accumulator
// holds anything (the warp's).
template <typename T>
__device__ __forceinline__ void store_output(uint8_t *stage, T *out, int64_t own, int d, uint32_t o_at, bool filled, bool some, float inv) {
  store_rows(stage, out, own, d, [&](int c, uint32_t (&w)[32]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t ov[32];
      if (filled) {
        sm100::tmem_ld_32x32b_x32(o_at + c + 32 * half, ov);
        sm100::tmem_ld_wait();
      }
#pragma unroll
      for (int u = 0; u < 16; ++u)
        w[16 * half + u] = filled && some ? Type<T>::pack(__uint_as_float(ov[2 * u]) * inv, __uint_as_float(ov[2 * u + 1]) * inv) : 0u;
    }
  });
}
__device__ __forceinline__ void store_sums(uint8_t *stage, float *out, int64_t own, int d, uint32_t o_at, bool filled, bool some) {
  store_rows(stage, out, own, d, [&](int c, uint32_t (&w)[32]) {
    if (filled) {
      sm100::tmem_ld_32x32b_x32(o_at + c, w);
      sm100::tmem_ld_wait();
    }
#pragma unroll
    for (int u = 0; u < 32; ++u) w[u] = filled && some ? w[u] : 0u;
  });
}

}  // namespace umma
