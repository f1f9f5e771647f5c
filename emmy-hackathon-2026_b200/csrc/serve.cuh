// Shared by the operators of serving (rotary.cu, paged.cu, paged_umma.cu): 16-byte
// vectors of the element types, the page lookup and the checks of the
// descriptors.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace serve {

// Bit of the context's error word for an index out of bounds (b2k_stream_sync
// reports it as B2K_EINDEX; the bits below are the bounded waits' sites).
constexpr unsigned kErrIndex = 0x1000;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N elements of T moved as one access (N * sizeof(T) = 16, 8, 4 or 2 bytes).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

inline size_t type_size(int32_t dtype) { return dtype == B2K_F32 ? 4 : 2; }
inline bool type_ok(int32_t dtype) { return dtype == B2K_F32 || dtype == B2K_F16 || dtype == B2K_BF16; }

// Page holding `position`, or -1 for a position outside the table (lengths are
// 32-bit, so none is beyond that) or a page outside the cache.
__host__ __device__ __forceinline__ int64_t page_of(const int32_t *table_row, int32_t table_width, int64_t pages,
                                                    int32_t page_size, int64_t position) {
  if (position < 0 || position > INT32_MAX || position >= (int64_t)table_width * page_size) return -1;
  const int64_t page = table_row[(uint32_t)position / (uint32_t)page_size];
  return page >= 0 && page < pages ? page : -1;
}

// b2k_paged_cache / b2k_paged_batch / b2k_heads argument checks (rotary.cu).
int check_cache(b2k_ctx *ctx, const char *what, const b2k_paged_cache *cache);
int check_batch(b2k_ctx *ctx, const char *what, const b2k_paged_cache *cache, const b2k_paged_batch *batch);
int check_heads(b2k_ctx *ctx, const char *what, const char *name, const b2k_heads *x, int64_t tokens, int32_t d,
                int32_t dtype);
int check_output(b2k_ctx *ctx, const char *what, const char *name, const b2k_heads *x, int64_t tokens, int32_t d,
                 int32_t dtype);
int check_apart(b2k_ctx *ctx, const char *what, const char *name, const b2k_heads &out, const b2k_heads &other, bool same,
                int64_t tokens, int32_t d, int32_t dtype);

// Whether an array lies on its elements' boundary (a load off it faults).
inline bool on_boundary(const void *p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// Whether a tensor's base and strides allow accesses of `bytes` bytes.
inline bool vec_ok(const void *p, int64_t s0, int64_t s1, int64_t s2, size_t size, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (s0 * (int64_t)size) % (int64_t)bytes == 0 &&
         (s1 * (int64_t)size) % (int64_t)bytes == 0 && (s2 * (int64_t)size) % (int64_t)bytes == 0;
}

}  // namespace serve
