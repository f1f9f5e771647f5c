// Attention over a paged cache for f16 and bf16 operands and few rows a cache
// head: the decode kernel.  A block holds 16 or 32 rows (query heads of one
// cache head, tokens side by side) and one split of the keys; its four warps
// take 16 keys at a time in turn, each on its own.
//
// Bound: HBM, the cache read once, and with many rows the instructions about it.
// Each warp keeps a ring of two to four tiles of 16 keys and values in flight
// with 16-byte asynchronous copies that only it waits for (no block barrier
// until the end), two or three blocks an SM: about 96 KB on the way at any
// time, where the copy bandwidth times the latency of HBM is about 45 KB an SM.
// The third block is worth its tighter registers (33 sequences of 20 rows of
// 64: 30 us with two, 24 with three).  The products are 16 x 8 x 16 warp MMAs with the probabilities
// taken from the score registers as they lie; rows that are not there cost
// nothing that the loads would not hide, so the 16-row tile is not split
// further.  The tensor-memory instructions need 64 rows and more to one tile:
// their kernel (paged_umma.cu) takes the calls that have them.
//
// The probabilities are rounded to the operands' type for the second product
// (half a step of that type each, as the output's own rounding); f16 ones are
// kept 2^8 larger, so that a key 2^-22 below the largest still has all its bits.
#include <math.h>

#include <algorithm>

#include "paged.cuh"

namespace {

using paged::Args;

constexpr int kThreads = 128;
constexpr int kWarps = 4;
constexpr int kTile = 16;  // keys of a warp's step

// Tiles a warp has in its ring.  Two at head dim 128 with 16 rows leave room for
// a third block on an SM (128 sequences of up to 2000 keys behind 8192: 138 us, 143
// with two blocks of two or of three tiles; one sequence of 50001: 37.8, 37.2, 39.5).
template <int DP, int MT>
constexpr int stages() { return DP == 64 ? 4 : DP == 128 && MT == 1 ? 2 : 3; }
template <int DP>
constexpr int tile_bytes() { return kTile * DP * 2; }  // one of K, V
template <int DP, int MT>
constexpr int sums_bytes() { return kWarps * 16 * MT * (DP + 8) * 4; }  // at the end, where the keys were
template <int DP, int MT>
constexpr int smem_bytes() {
  return std::max(kWarps * stages<DP, MT>() * 2 * tile_bytes<DP>(), sums_bytes<DP, MT>());
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 16-byte copy global to shared; zeros where `on` is false (nothing is read).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on, uint64_t policy) {
  const int bytes = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T>
struct Type;
template <>
struct Type<__half> {
  static constexpr float kLift = 8.0f;  // probabilities are kept times 2^kLift
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};
template <>
struct Type<__nv_bfloat16> {
  static constexpr float kLift = 0.0f;
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
};

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 1 : DP == 128 && MT == 2 ? 2 : 3)
    paged_mma_kernel(const __grid_constant__ Args a, const paged::Grid grid) {
  constexpr int kStages = stages<DP, MT>();
  constexpr int kChunks = DP / 8;        // 16-byte pieces of a row
  constexpr int kRows = 16 * MT;
  constexpr int kLdo = DP + 8;           // row stride of the warps' sums in shared memory
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 ml[kWarps][kRows];
  __shared__ uint32_t there_s[kWarps][kStages];
  paged::part_begin(a, grid.beside);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const paged::Block at = paged::this_block(a, grid);
  const bool prefix = at.prefix;
  const int row_blocks = prefix ? grid.prefix_row_blocks : grid.own_row_blocks;
  const int block = at.row_block, head = at.head, split = at.split, b = at.sequence;

  paged::Sequence s = {0, 0, 0};
  if (prefix) s.n = paged::used_tokens(a);
  else s = paged::sequence(a, b);
  const int rows = s.n * a.group, row0 = block * kRows;
  if (row0 >= rows) return paged::part_end(grid.beside);
  const int last_token = (min(row0 + kRows, rows) - 1) / a.group;
  const int chunk = prefix ? a.prefix_chunk : a.own_chunk;
  const int key0 = split * chunk;
  const int key_end = paged::split_end(key0, chunk, prefix ? a.prefix_len : paged::own_limit(a, s, last_token));
  const bool direct = a.own_splits + a.prefix_splits == 1;
  if (key0 >= key_end && !(direct && key0 == 0)) return paged::part_end(grid.beside);
  const int q_heads = a.kv_heads * a.group;

  // keys below this are seen by every row of the block
  const int free_end = prefix ? a.prefix_len : paged::own_limit(a, s, row0 / a.group);

  float o[MT][DP / 8][4], m[MT][2], l[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][n][e] = 0.0f;
    m[i][0] = m[i][1] = -INFINITY;
    l[i][0] = l[i][1] = 0.0f;
  }

  // --- this warp's tiles: keys key0 + 16 (warp + 4 i) -------------------------
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * kStages * 2 * tile_bytes<DP>();
  const int tiles = (key_end - key0 + kTile - 1) / kTile;
  const int mine = (tiles - warp + kWarps - 1) / kWarps;
  // A tile lies in one page where pages are whole tiles and the part starts on
  // one (a joined part's own keys start where the prefix ends).
  const bool whole = a.page_size % kTile == 0 && (prefix || !a.joined || a.prefix_len % kTile == 0);
  int pages32 = 0;  // whole: lane i holds the page of this warp's tile 32 k + i
  const T *kc = static_cast<const T *>(a.k) + (int64_t)head * a.k_head;
  const T *vc = static_cast<const T *>(a.v) + (int64_t)head * a.v_head;
  auto tile_key = [&](int i) { return key0 + (warp + kWarps * i) * kTile; };
  // Keys that one block reads leave L2 first, and with them in it the shared
  // prefix, the parts' sums and what the caller keeps there are not driven out
  // (128 sequences behind 8192 tokens: 116 -> 112 us; one of 50001: 40 -> 38).
  uint64_t policy;
  if (!prefix && row_blocks == 1) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  else asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
  constexpr int kRowsAtOnce = kChunks >= 32 ? 1 : 32 / kChunks;  // rows of one pass over the lanes
  constexpr int kPieces = kChunks >= 32 ? kChunks / 32 : 1;
  constexpr int kPasses = kTile / kRowsAtOnce;
  const int lane_row = kChunks >= 32 ? 0 : lane / kChunks, lane_chunk = kChunks >= 32 ? lane : lane % kChunks;
  const bool full_width = a.d == DP;
  auto issue = [&](int i) {
    if (i < mine) {
      const int key = tile_key(i), stage = i % kStages;
      const uint32_t kd = ring + stage * 2 * tile_bytes<DP>(), vd = kd + tile_bytes<DP>();
      int page = -1, row0 = 0;
      if (whole) {
        if (i % 32 == 0) {
          int row;
          const int k = tile_key(i + lane);
          pages32 = i + lane < mine ? (int)paged::key_page(a, prefix, b, k, row) : -1;
        }
        page = __shfl_sync(0xffffffffu, pages32, i % 32);
        const int own = prefix || !a.joined || key < a.prefix_len ? key : key - a.prefix_len;
        row0 = (int)((unsigned)own % (unsigned)a.page_size);
      }
      if (whole && page >= 0 && key + kTile <= key_end && full_width) {
        // a whole tile of one page: the rows follow each other
        if (lane == 0) there_s[warp][stage] = 0xffffu;
        const T *kp = kc + (page * a.k_page + (row0 + lane_row) * a.k_row + lane_chunk * 8);
        const T *vp = vc + (page * a.v_page + (row0 + lane_row) * a.v_row + lane_chunk * 8);
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          const int r = p * kRowsAtOnce + lane_row;
#pragma unroll
          for (int e = 0; e < kPieces; ++e) {
            const uint32_t to = r * DP * 2 + (((lane_chunk + 32 * e) ^ (r & 7)) << 4);
            copy16(kd + to, kp + 256 * e, true, policy);
            copy16(vd + to, vp + 256 * e, true, policy);
          }
          kp += kRowsAtOnce * a.k_row;
          vp += kRowsAtOnce * a.v_row;
        }
      } else {
        int64_t ko = 0, vo = 0;  // lane r < 16: offsets of key + r
        int row = row0 + (lane & 15);
        const int k = key + (lane & 15);
        bool on = k < key_end;
        if (on) {
          if (!whole) page = (int)paged::key_page(a, prefix, b, k, row);
          on = page >= 0;
          if (on) {
            ko = page * a.k_page + row * a.k_row;
            vo = page * a.v_page + row * a.v_row;
          }
        }
        const uint32_t there = __ballot_sync(0xffffffffu, on) & 0xffffu;
        if (lane == 0) there_s[warp][stage] = there;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          const int r = p * kRowsAtOnce + lane_row;
          const int64_t rk = __shfl_sync(0xffffffffu, ko, r), rv = __shfl_sync(0xffffffffu, vo, r);
          const bool row_on = (there >> r) & 1u;
#pragma unroll
          for (int e = 0; e < kPieces; ++e) {
            const int c = lane_chunk + 32 * e;
            const uint32_t to = r * DP * 2 + ((c ^ (r & 7)) << 4);
            const bool yes = row_on && c * 8 < a.d;
            copy16(kd + to, kc + (yes ? rk + c * 8 : 0), yes, policy);
            copy16(vd + to, vc + (yes ? rv + c * 8 : 0), yes, policy);
          }
        }
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  // The first tiles are on their way.  Queries as A fragments, straight from global memory: thread (g, t) holds
  // rows g and g + 8 of each 16, columns 2t, 2t + 1 and 8 further.
  const int g = lane >> 2, t = lane & 3;
  uint32_t qf[MT][DP / 16][4];
  int limit[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = row0 + 16 * i + 8 * h + g;
      const bool on = row < rows;
      const int j = on ? row / a.group : 0;
      limit[i][h] = !on ? 0 : prefix ? a.prefix_len : paged::own_limit(a, s, j);
      const T *q = static_cast<const T *>(a.q) + (int64_t)(s.first + j) * a.q_token +
                   (int64_t)(head * a.group + (on ? row - j * a.group : 0)) * a.q_head;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const int c = kk * 16 + 2 * t;
        qf[i][kk][h] = on && c < a.d ? *reinterpret_cast<const uint32_t *>(q + c) : 0u;
        qf[i][kk][2 + h] = on && c + 8 < a.d ? *reinterpret_cast<const uint32_t *>(q + c + 8) : 0u;
      }
    }
  }

  const float c = a.scale_log2;
  const int id = lane >> 3, ir = lane & 7;
  for (int i = 0; i < mine; ++i) {
    issue(i + kStages - 1);
    copy_wait<kStages - 1>();
    __syncwarp();
    const int stage = i % kStages, key = tile_key(i);
    const uint32_t kd = ring + stage * 2 * tile_bytes<DP>(), vd = kd + tile_bytes<DP>();
    float sc[MT][2][4];
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[x][n][e] = 0.0f;
    {
      const int r = (id >> 1) * 8 + ir;
      const uint32_t base = kd + r * DP * 2;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t kf[4];
        ldm(kf, base + (((kk * 2 + (id & 1)) ^ (r & 7)) << 4));
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          Type<T>::mma(sc[x][0], qf[x][kk], kf[0], kf[1]);
          Type<T>::mma(sc[x][1], qf[x][kk], kf[2], kf[3]);
        }
      }
    }
    const uint32_t there = there_s[warp][stage];
    if (there != 0xffffu || key + kTile > free_end) {
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = n * 8 + 2 * t + (e & 1);
            if (!((there >> k) & 1u) || key + k >= limit[x][e >> 1]) sc[x][n][e] = -INFINITY;
          }
    }
    uint32_t pf[MT][4];
#pragma unroll
    for (int x = 0; x < MT; ++x) {
      float base[2], alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(fmaxf(sc[x][0][2 * h], sc[x][0][2 * h + 1]), fmaxf(sc[x][1][2 * h], sc[x][1][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(m[x][h], mx * c - Type<T>::kLift);
        base[h] = mx == -INFINITY ? 0.0f : mx;
        alpha[h] = exp2_fast(m[x][h] - base[h]);
        m[x][h] = mx;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[x][n][e] = exp2_fast(fmaf(sc[x][n][e], c, -base[e >> 1]));
#pragma unroll
      for (int h = 0; h < 2; ++h)
        l[x][h] = l[x][h] * alpha[h] + ((sc[x][0][2 * h] + sc[x][0][2 * h + 1]) + (sc[x][1][2 * h] + sc[x][1][2 * h + 1]));
      // the maximum seldom moves once a few tiles are through
      if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          o[x][n][0] *= alpha[0];
          o[x][n][1] *= alpha[0];
          o[x][n][2] *= alpha[1];
          o[x][n][3] *= alpha[1];
        }
      }
      pf[x][0] = Type<T>::pack(sc[x][0][0], sc[x][0][1]);
      pf[x][1] = Type<T>::pack(sc[x][0][2], sc[x][0][3]);
      pf[x][2] = Type<T>::pack(sc[x][1][0], sc[x][1][1]);
      pf[x][3] = Type<T>::pack(sc[x][1][2], sc[x][1][3]);
    }
    {
      const int r = (id & 1) * 8 + ir;
      const uint32_t base = vd + r * DP * 2;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        uint32_t vf[4];
        ldm_t(vf, base + (((n * 2 + (id >> 1)) ^ (r & 7)) << 4));
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          Type<T>::mma(o[x][2 * n], pf[x], vf[0], vf[1]);
          Type<T>::mma(o[x][2 * n + 1], pf[x], vf[2], vf[3]);
        }
      }
    }
    __syncwarp();  // the stage is free
  }

  // --- the four warps' sums become one -----------------------------------------
  copy_wait<0>();
#pragma unroll
  for (int x = 0; x < MT; ++x)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = l[x][h];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (t == 0) ml[warp][16 * x + 8 * h + g] = make_float2(m[x][h], v);
    }
  __syncthreads();  // and nobody reads keys any more
  float *sums = reinterpret_cast<float *>(smem);
#pragma unroll
  for (int x = 0; x < MT; ++x)
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2 *>(sums + (warp * kRows + 16 * x + 8 * h + g) * kLdo + 8 * n + 2 * t) =
            make_float2(o[x][n][2 * h], o[x][n][2 * h + 1]);
  __syncthreads();
  for (int r = warp; r < kRows && row0 + r < rows; r += kWarps) {
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
    const int64_t part = (int64_t)(prefix ? a.own_splits + split : split) * a.tokens * q_heads + token * q_heads + qh;
    if (!direct && lane == 0) a.part_ml[part] = make_float2(mx, total);
    for (int col = 2 * lane; col < a.d; col += 64) {
      float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 x = *reinterpret_cast<const float2 *>(sums + (w * kRows + r) * kLdo + col);
        v.x = fmaf(x.x, f[w], v.x);
        v.y = fmaf(x.y, f[w], v.y);
      }
      if (direct)
        *reinterpret_cast<uint32_t *>(static_cast<T *>(a.o) + token * a.o_token + (int64_t)qh * a.o_head + col) =
            Type<T>::pack(v.x * inv, v.y * inv);
      else
        *reinterpret_cast<float2 *>(a.part_o + part * a.d + col) = v;
    }
  }
  paged::part_end(grid.beside);
}

template <typename T, int DP, int MT>
cudaError_t launch(b2k_ctx *ctx, const Args &a, const paged::Grid &g, unsigned blocks, cudaStream_t s) {
  auto kernel = paged_mma_kernel<T, DP, MT>;
  cudaError_t err = b2k::set_max_smem(ctx, (const void *)kernel, smem_bytes<DP, MT>());
  if (err != cudaSuccess) return err;
  return b2k::launch_kernel(a.pdl, kernel, dim3(blocks), dim3(kThreads), smem_bytes<DP, MT>(), s, a, g);
}

template <typename T>
cudaError_t pick(b2k_ctx *ctx, const Args &a, const paged::Grid &g, unsigned blocks, int mt, cudaStream_t s) {
  if (a.d <= 64) return mt == 1 ? launch<T, 64, 1>(ctx, a, g, blocks, s) : launch<T, 64, 2>(ctx, a, g, blocks, s);
  if (a.d <= 128) return mt == 1 ? launch<T, 128, 1>(ctx, a, g, blocks, s) : launch<T, 128, 2>(ctx, a, g, blocks, s);
  return launch<T, 256, 1>(ctx, a, g, blocks, s);
}

}  // namespace

namespace paged {

// Up to 32 rows in one block, which reads the keys once: 33 sequences of 20 rows
// over up to 2500 keys of 64 and 500 shared ones 24.4 us, 25.3 in two blocks of 16.
// Longer keys are faster in two blocks of 16, three of them an SM instead of two,
// the second of which finds the keys in L2: 64 sequences of 24 rows over up to 2000 keys 82.5 us against
// 72.6 at head dim 128 and 55.5 against 46.5 at 64, 32 of 18 rows 53.6 against 44.3.
int mma_rows(int d, int64_t rows) { return d <= 128 && rows > 16 ? 32 : 16; }

int mma_parts(b2k_ctx *ctx, const Args &a, int32_t dtype, bool with_prefix, bool with_own, int rows, bool beside,
              cudaStream_t s) {
  Grid g = {};
  const int64_t n = make_grid(ctx, a, with_prefix, with_own, rows, beside, g);
  if (n < 0) return B2K_EUNSUPPORTED;
  const unsigned blocks = (unsigned)n;
  const int mt = rows / 16;
  const cudaError_t err =
      dtype == B2K_F16 ? pick<__half>(ctx, a, g, blocks, mt, s) : pick<__nv_bfloat16>(ctx, a, g, blocks, mt, s);
  return err == cudaSuccess ? B2K_OK : b2k::cuda_fail(ctx, err, "paged_attention launch");
}

}  // namespace paged
