// Attention over a paged cache for f32 operands and few rows a cache head: the
// decode kernel's plan (paged_mma.cu) in FP32 arithmetic on the plain cores.  A
// block holds 4 or 8 rows and one split of the keys; each of its four warps
// streams tiles of its own, 1024 floats of keys and of values, through a ring
// that only it waits for.
//
// Bound: HBM for up to four rows, the FMA units for eight (16 FMA instructions a
// row for each 128 bytes of keys and values, a warp's).  TF32 tensor cores with
// the operands split in two would be faster there, but their sums are not
// rounded to nearest: over a head of 128 that leaves scores, and with them
// probabilities, off by 1e-6 of themselves and more, where FP32 is asked for.
//
// Scores: the lanes share a tile's keys, 2 to 8 lanes a key (head dim 64 to
// 256), each every second to eighth 16-byte piece of it; queries come as
// broadcasts from shared memory.  P V: lane = four dims (both halves of a warp
// take every other four keys at head dim 64), probabilities back as broadcasts
// of four keys.  Rows of a tile are swizzled by their key, so that the lanes of a
// quarter warp meet eight different pieces in both products.
#include <math.h>

#include <type_traits>

#include "paged.cuh"

namespace {

using paged::Args;

constexpr int kThreads = 128;
constexpr int kWarps = 4;
// and three blocks an SM (40 sequences of up to 1500 keys, 8 cache heads of 128: 81 us,
// 90 with three stages and two blocks; of 64 40 and 46; 9 x 2 tokens 14.5 and 13.3)
constexpr int kStages = 2;
constexpr int kTileFloats = 1024;  // of keys, and of values
constexpr int kStageFloats = 2 * kTileFloats;

template <int R, int DP>
constexpr int ring_floats() {
  constexpr int ring = kWarps * kStages * kStageFloats, sums = kWarps * R * (DP + 4);
  return ring > sums ? ring : sums;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on, uint64_t policy) {
  const int bytes = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int R, int DP>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 2 : 3) paged_f32_kernel(const __grid_constant__ Args a, const paged::Grid grid) {
  constexpr int kTile = kTileFloats / DP;   // keys of a warp's step: 16, 8, 4
  constexpr int kLanes = 32 / kTile;        // lanes of a key: 2, 4, 8
  constexpr int kChunks = DP / 4;           // 16-byte pieces of a row
  constexpr int kSides = DP == 64 ? 2 : 1;  // key groups of the second product
  constexpr int kDims = DP == 256 ? 2 : 1;  // pieces of a lane there
  constexpr int kLdo = DP + 4;
  extern __shared__ __align__(128) float smem[];
  __shared__ __align__(16) float qs[R][DP], ps[kWarps][R][kTile];
  __shared__ float2 ml[kWarps][R];
  __shared__ int64_t q_at[R];
  __shared__ uint32_t there_s[kWarps][kStages];
  paged::part_begin(a, grid.beside);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const paged::Block at = paged::this_block(a, grid);
  const bool prefix = at.prefix;
  const int head = at.head, split = at.split, b = at.sequence;
  paged::Sequence s = {0, 0, 0};
  if (prefix) s.n = paged::used_tokens(a);
  else s = paged::sequence(a, b);
  const int rows = s.n * a.group, row0 = at.row_block * R;
  if (row0 >= rows) return paged::part_end(grid.beside);
  const int last_token = (min(row0 + R, rows) - 1) / a.group;
  const int chunk = prefix ? a.prefix_chunk : a.own_chunk;
  const int key0 = split * chunk;
  const int key_end = paged::split_end(key0, chunk, prefix ? a.prefix_len : paged::own_limit(a, s, last_token));
  const bool direct = a.own_splits + a.prefix_splits == 1;
  if (key0 >= key_end && !(direct && key0 == 0)) return paged::part_end(grid.beside);
  const int q_heads = a.kv_heads * a.group;

  // --- this warp's tiles: keys key0 + kTile (warp + 4 i), as in the decode kernel -----
  float *ring_f = smem + warp * kStages * kStageFloats;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_f);
  const int tiles = (key_end - key0 + kTile - 1) / kTile;
  const int mine = (tiles - warp + kWarps - 1) / kWarps;
  const bool whole = a.page_size % kTile == 0 && (prefix || !a.joined || a.prefix_len % kTile == 0);
  int pages32 = 0;  // whole: lane i holds the page of this warp's tile 32 k + i
  const float *kc = static_cast<const float *>(a.k) + (int64_t)head * a.k_head;
  const float *vc = static_cast<const float *>(a.v) + (int64_t)head * a.v_head;
  uint64_t policy;  // streamed keys leave L2 first (paged_mma.cu)
  if (!prefix && grid.own_row_blocks == 1) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  else asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
  auto tile_key = [&](int i) { return key0 + (warp + kWarps * i) * kTile; };
  constexpr int kRowsAtOnce = kChunks >= 32 ? 1 : 32 / kChunks;  // rows of one pass over the lanes
  constexpr int kPieces = kChunks >= 32 ? kChunks / 32 : 1;
  constexpr int kPasses = kTile / kRowsAtOnce;
  const int lane_row = kChunks >= 32 ? 0 : lane / kChunks, lane_chunk = kChunks >= 32 ? lane : lane % kChunks;
  const bool full_width = a.d == DP;
  auto place = [](int r, int c) { return (r * kChunks + (c ^ ((r * kLanes) & 7))) * 16; };  // bytes in a tile
  auto issue = [&](int i) {
    if (i < mine) {
      const int key = tile_key(i), stage = i % kStages;
      const uint32_t kd = ring + stage * kStageFloats * 4, vd = kd + kTileFloats * 4;
      int page = -1, page_row = 0;
      if (whole) {
        if (i % 32 == 0) {
          int row;
          pages32 = i + lane < mine ? (int)paged::key_page(a, prefix, b, tile_key(i + lane), row) : -1;
        }
        page = __shfl_sync(0xffffffffu, pages32, i % 32);
        const int own = prefix || !a.joined || key < a.prefix_len ? key : key - a.prefix_len;
        page_row = (int)((unsigned)own % (unsigned)a.page_size);
      }
      constexpr uint32_t kAll = (1u << kTile) - 1u;
      if (whole && page >= 0 && key + kTile <= key_end && full_width) {
        // a whole tile of one page: the rows follow each other
        if (lane == 0) there_s[warp][stage] = kAll;
        const float *kp = kc + (page * a.k_page + (page_row + lane_row) * a.k_row + lane_chunk * 4);
        const float *vp = vc + (page * a.v_page + (page_row + lane_row) * a.v_row + lane_chunk * 4);
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          const int r = p * kRowsAtOnce + lane_row;
#pragma unroll
          for (int e = 0; e < kPieces; ++e) {
            copy16(kd + place(r, lane_chunk + 32 * e), kp + 128 * e, true, policy);
            copy16(vd + place(r, lane_chunk + 32 * e), vp + 128 * e, true, policy);
          }
          kp += kRowsAtOnce * a.k_row;
          vp += kRowsAtOnce * a.v_row;
        }
      } else {
        int64_t ko = 0, vo = 0;  // lane r < kTile: offsets of key + r
        bool on = key + (lane % kTile) < key_end;
        int row = page_row + lane % kTile;
        if (on) {
          if (!whole) page = (int)paged::key_page(a, prefix, b, key + lane % kTile, row);
          on = page >= 0;
          if (on) {
            ko = page * a.k_page + row * a.k_row;
            vo = page * a.v_page + row * a.v_row;
          }
        }
        const uint32_t there = __ballot_sync(0xffffffffu, on) & kAll;
        if (lane == 0) there_s[warp][stage] = there;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          const int r = p * kRowsAtOnce + lane_row;
          const int64_t rk = __shfl_sync(0xffffffffu, ko, r), rv = __shfl_sync(0xffffffffu, vo, r);
          const bool row_on = (there >> r) & 1u;
#pragma unroll
          for (int e = 0; e < kPieces; ++e) {
            const int c = lane_chunk + 32 * e;
            const bool yes = row_on && c * 4 < a.d;
            copy16(kd + place(r, c), kc + (yes ? rk + c * 4 : 0), yes, policy);
            copy16(vd + place(r, c), vc + (yes ? rv + c * 4 : 0), yes, policy);
          }
        }
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  // this block's queries, times log2(e) / scale, while the first tiles are on their way
  if (threadIdx.x < R) {
    const int row = row0 + threadIdx.x, j = row / a.group;
    q_at[threadIdx.x] =
        row < rows ? (int64_t)(s.first + j) * a.q_token + (int64_t)(head * a.group + row - j * a.group) * a.q_head : -1;
  }
  __syncthreads();
  {
    constexpr int kBatch = R * DP / kThreads;
    float x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = threadIdx.x + u * kThreads, r = i / DP, c = i % DP;
      const int64_t from = q_at[r];
      x[u] = from >= 0 && c < a.d ? static_cast<const float *>(a.q)[from + c] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) (&qs[0][0])[threadIdx.x + u * kThreads] = x[u] * a.scale_log2;
  }
  int limit[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i;
    limit[i] = row >= rows ? 0 : prefix ? a.prefix_len : paged::own_limit(a, s, row / a.group);
  }
  // keys below this are seen by every row of the block (rows that are not there see none)
  const int free_end = rows - row0 < R ? 0 : prefix ? a.prefix_len : paged::own_limit(a, s, row0 / a.group);
  __syncthreads();

  const int key_of = lane / kLanes, part = lane % kLanes;              // of a score
  const int side = kSides == 2 ? lane >> 4 : 0, dim = kSides == 2 ? lane & 15 : lane;  // of an output (pieces)
  float4 o[R][kDims];
  float m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < kDims; ++c) o[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }

  for (int i = 0; i < mine; ++i) {
    issue(i + kStages - 1);
    copy_wait<kStages - 1>();
    __syncwarp();
    const int stage = i % kStages, key = tile_key(i);
    const char *ks = reinterpret_cast<const char *>(ring_f + stage * kStageFloats), *vs = ks + kTileFloats * 4;
    float4 sum[R];
#pragma unroll
    for (int x = 0; x < R; ++x) sum[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int e = 0; e < kChunks / kLanes; ++e) {
      const int c = part + kLanes * e;
      const float4 kv = *reinterpret_cast<const float4 *>(ks + place(key_of, c));
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const float4 qv = *reinterpret_cast<const float4 *>(&qs[x][4 * c]);
        sum[x].x = fmaf(qv.x, kv.x, sum[x].x);
        sum[x].y = fmaf(qv.y, kv.y, sum[x].y);
        sum[x].z = fmaf(qv.z, kv.z, sum[x].z);
        sum[x].w = fmaf(qv.w, kv.w, sum[x].w);
      }
    }
    const uint32_t there = there_s[warp][stage];
    constexpr uint32_t kAll = (1u << kTile) - 1u;
    const bool open = there == kAll && key + kTile <= free_end;
    const bool key_there = (there >> key_of) & 1u;
#pragma unroll
    for (int x = 0; x < R; ++x) {
      float sc = (sum[x].x + sum[x].y) + (sum[x].z + sum[x].w);
#pragma unroll
      for (int n = 1; n < kLanes; n <<= 1) sc += __shfl_xor_sync(0xffffffffu, sc, n);
      if (!open && !(key_there && key + key_of < limit[x])) sc = -INFINITY;
      float mx = sc;
#pragma unroll
      for (int n = kLanes; n < 32; n <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, n));
      mx = fmaxf(m[x], mx);
      const float base = mx == -INFINITY ? 0.0f : mx;
      const float alpha = exp2_fast(m[x] - base), p = exp2_fast(sc - base);
      if (part == 0) ps[warp][x][key_of] = p;
      l[x] = l[x] * alpha + p;  // this lane's key; the keys' lanes are added at the end
      m[x] = mx;
#pragma unroll
      for (int c = 0; c < kDims; ++c) {
        o[x][c].x *= alpha;
        o[x][c].y *= alpha;
        o[x][c].z *= alpha;
        o[x][c].w *= alpha;
      }
    }
    __syncwarp();
    // the test of a masked key costs as much as its products: only where there is one
    auto values = [&](auto guarded) {
#pragma unroll
      for (int t0 = 0; t0 < kTile / kSides; t0 += 4) {
        const int t = t0 * kSides + 4 * side;
        float4 v[4][kDims];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < kDims; ++c) v[u][c] = *reinterpret_cast<const float4 *>(vs + place(t + u, dim + 32 * c));
#pragma unroll
        for (int x = 0; x < R; ++x) {
          const float4 p4 = *reinterpret_cast<const float4 *>(&ps[warp][x][t]);
          const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (decltype(guarded)::value && p[u] == 0.0f) continue;  // a masked value may be anything
#pragma unroll
            for (int c = 0; c < kDims; ++c) {
              o[x][c].x = fmaf(p[u], v[u][c].x, o[x][c].x);
              o[x][c].y = fmaf(p[u], v[u][c].y, o[x][c].y);
              o[x][c].z = fmaf(p[u], v[u][c].z, o[x][c].z);
              o[x][c].w = fmaf(p[u], v[u][c].w, o[x][c].w);
            }
          }
        }
      }
    };
    if (open) values(std::false_type{});
    else values(std::true_type{});
    __syncwarp();  // the stage, and the probabilities, may be written again
  }

  // --- the four warps' sums become one ------------------------------------------------
  copy_wait<0>();
#pragma unroll
  for (int x = 0; x < R; ++x) {
    float v = l[x];
#pragma unroll
    for (int n = kLanes; n < 32; n <<= 1) v += __shfl_xor_sync(0xffffffffu, v, n);
    if (lane == 0) ml[warp][x] = make_float2(m[x], v);
    if (kSides == 2) {
      o[x][0].x += __shfl_xor_sync(0xffffffffu, o[x][0].x, 16);
      o[x][0].y += __shfl_xor_sync(0xffffffffu, o[x][0].y, 16);
      o[x][0].z += __shfl_xor_sync(0xffffffffu, o[x][0].z, 16);
      o[x][0].w += __shfl_xor_sync(0xffffffffu, o[x][0].w, 16);
    }
  }
  __syncthreads();  // and nobody reads keys any more
#pragma unroll
  for (int x = 0; x < R; ++x)
#pragma unroll
    for (int c = 0; c < kDims; ++c)
      if (side == 0) *reinterpret_cast<float4 *>(smem + (warp * R + x) * kLdo + 4 * (dim + 32 * c)) = o[x][c];
  __syncthreads();
  for (int r = warp; r < R && row0 + r < rows; r += kWarps) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml[w][r].x);
    const float base = mx == -INFINITY ? 0.0f : mx;
    float f[kWarps], total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = exp2_fast(ml[w][r].x - base);
      total += ml[w][r].y * f[w];
    }
    const int j = (row0 + r) / a.group, qh = head * a.group + (row0 + r) - j * a.group;
    const int64_t token = s.first + j;
    const float inv = direct ? (total == 0.0f ? 0.0f : 1.0f / total) : 1.0f;
    const int64_t slot = (int64_t)(prefix ? a.own_splits + split : split) * a.tokens * q_heads + token * q_heads + qh;
    if (!direct && lane == 0) a.part_ml[slot] = make_float2(mx, total);
    float *out = direct ? static_cast<float *>(a.o) + token * a.o_token + (int64_t)qh * a.o_head : a.part_o + slot * a.d;
    for (int col = lane; col < a.d; col += 32) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = fmaf(smem[(w * R + r) * kLdo + col], f[w], v);
      out[col] = v * inv;
    }
  }
  paged::part_end(grid.beside);
}

template <int R, int DP>
int launch(b2k_ctx *ctx, const Args &a, const paged::Grid &g, unsigned blocks, cudaStream_t s) {
  auto kernel = paged_f32_kernel<R, DP>;
  constexpr int bytes = ring_floats<R, DP>() * sizeof(float);
  cudaError_t err = b2k::set_max_smem(ctx, (const void *)kernel, bytes);
  if (err == cudaSuccess) err = b2k::launch_kernel(a.pdl, kernel, dim3(blocks), dim3(kThreads), bytes, s, a, g);
  return err == cudaSuccess ? B2K_OK : b2k::cuda_fail(ctx, err, "paged_attention launch");
}

}  // namespace

namespace paged {

int f32_parts(b2k_ctx *ctx, const Args &a, bool with_prefix, bool with_own, int rows, bool beside, cudaStream_t s) {
  Grid g = {};
  const int64_t n = make_grid(ctx, a, with_prefix, with_own, rows, beside, g);
  if (n < 0) return B2K_EUNSUPPORTED;
  const unsigned blocks = (unsigned)n;
  if (rows == 4)
    return a.d <= 64    ? launch<4, 64>(ctx, a, g, blocks, s)
           : a.d <= 128 ? launch<4, 128>(ctx, a, g, blocks, s)
                        : launch<4, 256>(ctx, a, g, blocks, s);
  return a.d <= 64    ? launch<8, 64>(ctx, a, g, blocks, s)
         : a.d <= 128 ? launch<8, 128>(ctx, a, g, blocks, s)
                      : launch<8, 256>(ctx, a, g, blocks, s);
}

}  // namespace paged
