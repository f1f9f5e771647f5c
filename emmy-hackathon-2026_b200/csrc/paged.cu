// Attention over a paged key / value cache: the plan of a call (which kernel
// takes the shared prefix and which the sequences' own keys, and how the keys
// are split), the FP32 kernel, and the merge of the parts (paged.cuh has the
// mathematics).
//
// paged_rows_kernel: FP32 arithmetic on the plain cores, for f32 operands and
// for any layout that the tensor-core kernels do not read (element strides
// and bases off 16 bytes, head dims off 8).  A block of four warps holds R = 4
// RW rows (query heads of one cache head, tokens side by side) and streams 32
// keys at a time through shared memory as FP32.  Scores: each warp its own RW
// rows, lane = key, or with 32 rows lane = two rows by four keys and two dims an
// instruction (prompts of 430 over 1430 keys, 12 / 4 heads, f32: 222 -> 214 us at
// 64 dims, 355 -> 357 at 128, 822 -> 795 at 256; FMA pipe and shared memory both
// near half there, with 4 to 12 warps an SM).  The next tile is on its way meanwhile (asynchronous
// copies where the cache is f32 in 16-byte pieces).  P V: lane = four
// dims, the probabilities read back four keys at a time as one broadcast
// (shuffled one by one they took two thirds of the kernel's instructions).  In a
// tile with masked keys a probability of exactly zero skips its key, so what a
// masked place of the cache holds (infinities and NaN too) has no effect.
#include <math.h>

#include <algorithm>
#include <new>
#include <vector>
#include <type_traits>

#include "paged.cuh"

namespace {

using paged::Args;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 32;  // keys

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two FP32 products and sums in one instruction.
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
// o += p v, p twice in pp
__device__ __forceinline__ void fma4(float4 &o, uint64_t pp, const float4 &v) {
  unpair(fma2(pp, pair(v.x, v.y), pair(o.x, o.y)), o.x, o.y);
  unpair(fma2(pp, pair(v.z, v.w), pair(o.z, o.w)), o.z, o.w);
}

// 16-byte copy global to shared.
__device__ __forceinline__ void copy16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

// DV: float4s of a head that a lane holds (head dim up to 128 DV; 0: up to 64,
// where the two halves of a warp take every other four keys and add up at the end).
// V: elements of one access to the cache (16 bytes, or 1).
// Tiles a block holds: one in use, the others on their way.
template <int DV0>
constexpr int rows_stages() { return DV0 == 0 ? 3 : 2; }

template <typename T, int RW, int DV0, int V>
__global__ void __launch_bounds__(kThreads)
    paged_rows_kernel(const __grid_constant__ Args a, const paged::Grid grid) {
  constexpr int R = RW * kWarps;
  constexpr int DV = DV0 == 0 ? 1 : DV0, kSides = DV0 == 0 ? 2 : 1;
  constexpr bool kAsync = sizeof(T) == 4 && V == 4;  // the cache's bytes are the tile's
  extern __shared__ __align__(16) float smem[];
  constexpr int kStages = rows_stages<DV0>(), kSlots = kStages + 1;
  static_assert(kStages * kTile <= kThreads, "a thread looks up one key of the first tiles");
  __shared__ int64_t k_at[kSlots][kTile], v_at[kSlots][kTile];  // offsets of a tile's rows; -1: no such key
  constexpr bool kSquare = RW == 8;  // scores: lane = two rows by four keys, else RW rows by one
  constexpr int kPs = kSquare ? kTile + 4 : kTile;
  __shared__ __align__(16) float ps[kWarps][RW][kPs];  // a warp's probabilities
  __shared__ __align__(16) float alphas[kWarps][RW];   // (kSquare) and what its rows' sums are scaled by
  __shared__ int64_t q_at[R];
  const int dp = (a.d + 3) / 4 * 4, ldk = dp + 4, ldq = dp + 4;
  const int stage_floats = kTile * (ldk + dp);  // keys, then values; the stages behind the queries
  float *qs = smem, *tiles = qs + R * ldq;
  paged::part_begin(a, grid.beside);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int side = kSides == 2 ? lane >> 4 : 0, col = 4 * (kSides == 2 ? lane & 15 : lane);  // of a lane's output
  const paged::Block at = paged::this_block(a, grid);
  const bool prefix = at.prefix;
  const int split = at.split, head = at.head, block = at.row_block, b = at.sequence;
  const int q_heads = a.kv_heads * a.group;
  paged::Sequence s = {0, 0, 0};
  if (prefix) s.n = paged::used_tokens(a);
  else s = paged::sequence(a, b);
  const int rows = s.n * a.group, row0 = block * R;
  if (row0 >= rows) return paged::part_end(grid.beside);
  const int last_token = (min(row0 + R, rows) - 1) / a.group;
  const int chunk = prefix ? a.prefix_chunk : a.own_chunk;
  const int key0 = split * chunk;
  const int key_end = paged::split_end(key0, chunk, prefix ? a.prefix_len : paged::own_limit(a, s, last_token));
  const bool direct = a.own_splits + a.prefix_splits == 1;
  if (key0 >= key_end && !(direct && key0 == 0)) return paged::part_end(grid.beside);
  const int n_tiles = (key_end - key0 + kTile - 1) / kTile;

  // A key's page is asked for one tile before its load is issued; the answer
  // is used at the end of the tile in between.
  int asked = 0, asked_row = 0;
  bool wanted = false;
  auto ask = [&](int tile, int i) {
    const int at = key0 + tile * kTile + i;
    wanted = at < key_end;
    if (wanted) asked = paged::key_entry(a, prefix, b, at, asked_row);
  };
  auto answer = [&](int tile, int i) {
    int64_t ko = -1, vo = -1;
    if (wanted && asked >= 0 && asked < a.pages) {
      ko = asked * a.k_page + asked_row * a.k_row + head * a.k_head;
      vo = asked * a.v_page + asked_row * a.v_row + head * a.v_head;
    } else if (wanted) {
      atomicOr(a.err, serve::kErrIndex);
    }
    k_at[tile % kSlots][i] = ko;
    v_at[tile % kSlots][i] = vo;
  };
  // a thread's first piece of a tile, and the step to its next one
  const int per_row = dp / V, r_first = threadIdx.x / per_row, c_first = threadIdx.x - r_first * per_row;
  const int r_step = kThreads / per_row, c_step = kThreads - r_step * per_row;
  auto load = [&](int i) {
    if (i >= n_tiles) return;
    float *ks = tiles + i % kStages * stage_floats, *vs = ks + kTile * ldk;
    for (int r = r_first, piece = c_first; r < kTile; r += r_step, piece += c_step) {
      if (piece >= per_row) {
        piece -= per_row;
        if (++r >= kTile) break;
      }
      const int c = piece * V;
      const int64_t ko = k_at[i % kSlots][r], vo = v_at[i % kSlots][r];
      const T *kx = static_cast<const T *>(a.k) + ko + c, *vx = static_cast<const T *>(a.v) + vo + c;
      if (kAsync) {
        if (ko >= 0) {
          copy16(ks + r * ldk + c, kx);
          copy16(vs + r * dp + c, vx);
        } else {
          *reinterpret_cast<float4 *>(ks + r * ldk + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          *reinterpret_cast<float4 *>(vs + r * dp + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      } else {
        serve::Pack<T, V> kp = {}, vp = {};
        if (ko >= 0 && c < a.d) {
          kp = *reinterpret_cast<const serve::Pack<T, V> *>(kx);
          vp = *reinterpret_cast<const serve::Pack<T, V> *>(vx);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          ks[r * ldk + c + e] = serve::to_f32(kp.v[e]);
          vs[r * dp + c + e] = serve::to_f32(vp.v[e]);
        }
      }
    }
  };
  if (threadIdx.x < kStages * kTile) {
    ask(threadIdx.x / kTile, threadIdx.x % kTile);
    answer(threadIdx.x / kTile, threadIdx.x % kTile);
  }

  // this block's queries, FP32, times log2(e) / scale; eight loads in flight
  if (threadIdx.x < R) {
    const int row = row0 + threadIdx.x, j = row / a.group;
    q_at[threadIdx.x] =
        row < rows ? (int64_t)(s.first + j) * a.q_token + (int64_t)(head * a.group + row - j * a.group) * a.q_head : -1;
  }
  __syncthreads();
  constexpr int kBatch = 8;
  for (int i0 = threadIdx.x; i0 < R * dp; i0 += kBatch * kThreads) {
    float x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * kThreads, r = (unsigned)i / (unsigned)dp, c = i - r * dp;
      const int64_t from = r < R ? q_at[r] : -1;
      x[u] = from >= 0 && c < a.d ? serve::to_f32(static_cast<const T *>(a.q)[from + c]) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (i0 + u * kThreads < R * dp) {
        const int i = i0 + u * kThreads, r = (unsigned)i / (unsigned)dp;
        qs[r * ldq + i - r * dp] = x[u] * a.scale_log2;
      }
  }
  int limit[RW];
  // the lane's rows of the scores, and their running maximum and sum of its keys
  constexpr int kOwn = kSquare ? 2 : RW;
  const int ty = lane >> 3, tx = lane & 7;
  int row_limit[2];
  float m[kOwn], l[kOwn];
  float4 o[RW][DV];
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int row = row0 + warp * RW + i;
    limit[i] = row >= rows ? 0 : prefix ? a.prefix_len : paged::own_limit(a, s, row / a.group);
#pragma unroll
    for (int c = 0; c < DV; ++c) o[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = row0 + warp * RW + 2 * ty + i;
    row_limit[i] = !kSquare || row >= rows ? 0 : prefix ? a.prefix_len : paged::own_limit(a, s, row / a.group);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    load(i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  for (int tile = 0; tile < n_tiles; ++tile) {
    const int key = key0 + tile * kTile;
    const float *ks = tiles + tile % kStages * stage_floats, *vs = ks + kTile * ldk;
    if (threadIdx.x < kTile) ask(tile + kStages, threadIdx.x);
    load(tile + kStages - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncthreads();

    // every key of the tile is seen by every row of the warp
    bool open = key + kTile <= key_end;
#pragma unroll
    for (int i = 0; i < RW; ++i) open = open && key + kTile <= limit[i];
    open = __all_sync(0xffffffffu, open && k_at[tile % kSlots][lane] >= 0);
    if constexpr (kSquare) {
      // lane = rows 2 ty, 2 ty + 1 by keys tx, tx + 8, ..: six cycles of shared memory for
      // 32 products, where a key a lane takes twelve; and a row's butterfly is
      // over 8 lanes
      uint64_t sum[2][4];  // of even and of odd dims
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = 0;
      const float *qr = qs + (warp * RW + 2 * ty) * ldq, *kr = ks + tx * ldk;
#pragma unroll 4
      for (int c = 0; c < dp; c += 4) {
        float4 qv[2], kv[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) qv[i] = *reinterpret_cast<const float4 *>(qr + i * ldq + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4 *>(kr + 8 * j * ldk + c);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sum[i][j] = fma2(pair(qv[i].x, qv[i].y), pair(kv[j].x, kv[j].y), sum[i][j]);
            sum[i][j] = fma2(pair(qv[i].z, qv[i].w), pair(kv[j].z, kv[j].w), sum[i][j]);
          }
      }
      bool there[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) there[j] = k_at[tile % kSlots][tx + 8 * j] >= 0;
      bool moved = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = m[i], score[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float even, odd;
          unpair(sum[i][j], even, odd);
          score[j] = there[j] && key + tx + 8 * j < row_limit[i] ? even + odd : -INFINITY;
          mx = fmaxf(mx, score[j]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float alpha = exp2_fast(m[i] - base);
        l[i] *= alpha;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2_fast(score[j] - base);
          ps[warp][2 * ty + i][tx + 8 * j] = p;
          l[i] += p;
        }
        m[i] = mx;
        moved = moved || alpha != 1.0f;
        if (tx == 0) alphas[warp][2 * ty + i] = alpha;
      }
      if (__any_sync(0xffffffffu, moved)) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          const float alpha = alphas[warp][i];
#pragma unroll
          for (int c = 0; c < DV; ++c) {
            o[i][c].x *= alpha;
            o[i][c].y *= alpha;
            o[i][c].z *= alpha;
            o[i][c].w *= alpha;
          }
        }
      }
    } else {
      float4 sum[RW];  // four chains a row: one would be as long as the head
#pragma unroll
      for (int i = 0; i < RW; ++i) sum[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int c = 0; c < dp; c += 4) {
        const float4 kv = *reinterpret_cast<const float4 *>(ks + lane * ldk + c);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          const float4 qv = *reinterpret_cast<const float4 *>(qs + (warp * RW + i) * ldq + c);
          sum[i].x = fmaf(qv.x, kv.x, sum[i].x);
          sum[i].y = fmaf(qv.y, kv.y, sum[i].y);
          sum[i].z = fmaf(qv.z, kv.z, sum[i].z);
          sum[i].w = fmaf(qv.w, kv.w, sum[i].w);
        }
      }
      const bool there = k_at[tile % kSlots][lane] >= 0;
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        const float sc = there && key + lane < limit[i] ? (sum[i].x + sum[i].y) + (sum[i].z + sum[i].w) : -INFINITY;
        const float mx = fmaxf(m[i], warp_max(sc));
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float alpha = exp2_fast(m[i] - base);
        const float p = exp2_fast(sc - base);
        ps[warp][i][lane] = p;
        l[i] = l[i] * alpha + p;  // this lane's keys; the lanes are added at the end
        m[i] = mx;
#pragma unroll
        for (int c = 0; c < DV; ++c) {
          o[i][c].x *= alpha;
          o[i][c].y *= alpha;
          o[i][c].z *= alpha;
          o[i][c].w *= alpha;
        }
      }
    }
    __syncwarp();
    // the test of a masked key costs as much as its products: only where there is one
    auto values = [&](auto guarded) {
      for (int t0 = 4 * side; t0 < kTile; t0 += 4 * kSides) {
        float4 vv[4][DV];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < DV; ++c)
            vv[u][c] = col + 128 * c < dp ? *reinterpret_cast<const float4 *>(vs + (t0 + u) * dp + col + 128 * c)
                                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          const float4 p4 = *reinterpret_cast<const float4 *>(&ps[warp][i][t0]);
          const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (decltype(guarded)::value && p[u] == 0.0f) continue;  // a masked value may be anything
#pragma unroll
            for (int c = 0; c < DV; ++c) {
              fma4(o[i][c], pair(p[u], p[u]), vv[u][c]);
            }
          }
        }
      }
    };
    if (open) values(std::false_type{});
    else values(std::true_type{});
    // (this tile's slot is not the one written: kSlots is one more than the stages)
    if (threadIdx.x < kTile) answer(tile + kStages, threadIdx.x);
    __syncthreads();  // the stage may be written again
  }

  if (kSquare) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
  }
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int row = row0 + warp * RW + i;
    float total, top;
    if constexpr (kSquare) {
      total = __shfl_sync(0xffffffffu, l[i & 1], i / 2 * 8);
      top = __shfl_sync(0xffffffffu, m[i & 1], i / 2 * 8);
    } else {
      total = warp_sum(l[i]);
      top = m[i];
    }
    if (kSides == 2) {
      o[i][0].x += __shfl_xor_sync(0xffffffffu, o[i][0].x, 16);
      o[i][0].y += __shfl_xor_sync(0xffffffffu, o[i][0].y, 16);
      o[i][0].z += __shfl_xor_sync(0xffffffffu, o[i][0].z, 16);
      o[i][0].w += __shfl_xor_sync(0xffffffffu, o[i][0].w, 16);
    }
    if (row >= rows || side == 1) continue;
    const int64_t token = s.first + row / a.group;
    const int qh = head * a.group + row % a.group;
    if (direct) {
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
      T *out = static_cast<T *>(a.o) + token * a.o_token + qh * a.o_head;
#pragma unroll
      for (int c = 0; c < DV; ++c) {
        const float x[4] = {o[i][c].x, o[i][c].y, o[i][c].z, o[i][c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + 128 * c + e < a.d) out[col + 128 * c + e] = serve::from_f32<T>(x[e] * inv);
      }
    } else {
      const int64_t at = (int64_t)(prefix ? a.own_splits + split : split) * a.tokens * q_heads + token * q_heads + qh;
      if (lane == 0) a.part_ml[at] = make_float2(top, total);
#pragma unroll
      for (int c = 0; c < DV; ++c) {
        const float x[4] = {o[i][c].x, o[i][c].y, o[i][c].z, o[i][c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + 128 * c + e < a.d) a.part_o[at * a.d + col + 128 * c + e] = x[e];
      }
    }
  }
  paged::part_end(grid.beside);
}

// Joins a row's parts, in an order that does not depend on which part ended
// first.  A row (token, query head) is one warp's, or, SHARED, a block's, whose
// warps take every fourth part: with many parts and too few rows to fill the
// GPU, a warp alone waits for one batch of loads after the other (36 parts of
// 32 rows: 41 us against 4).  Lanes over the dims, V at a time.
template <typename T, int V, bool SHARED>
__global__ void __launch_bounds__(kThreads) paged_merge_kernel(const __grid_constant__ Args a, bool vec_out) {
  constexpr int kPieces = B2K_MAX_HEAD_DIM / 32 / V;  // of a lane
  constexpr int kStep = SHARED ? kWarps : 1;          // parts from one of a warp's to the next
  constexpr int kAhead = SHARED ? 10 : 4;  // parts a warp has in flight: up to 40 of a row at once
  __shared__ float sums[SHARED ? kWarps : 1][SHARED ? B2K_MAX_HEAD_DIM : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_heads = a.kv_heads * a.group;
  const bool ready = paged::call_ready(a);
  if (!ready) grid_dependency_wait();
  const paged::Sequence s = paged::sequence(a, blockIdx.x);
  if (ready) grid_dependency_wait();
  grid_dependents_launch();
  const int64_t stride = a.tokens * q_heads;
  const int64_t step = (int64_t)gridDim.y * (SHARED ? 1 : kWarps);
  for (int64_t row = (int64_t)blockIdx.y * (SHARED ? 1 : kWarps) + (SHARED ? 0 : warp); row < (int64_t)s.n * q_heads;
       row += step) {
    const int j = (int)(row / q_heads), qh = (int)(row % q_heads);
    const int64_t at = (int64_t)(s.first + j) * q_heads + qh;
    // (rounded up without a sum: a split may be as long as the largest length)
    const int limit = paged::own_limit(a, s, j), own = limit > 0 ? (limit - 1) / a.own_chunk + 1 : 0;
    const int parts = own + a.prefix_splits;
    auto slot = [&](int i) { return (int64_t)(i < own ? i : a.own_splits + i - own) * stride + at; };
    // the first parts' sums are on their way while the weights are found
    serve::Pack<float, V> v[kAhead][kPieces];
    auto load = [&](int i0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kStep;
        if (i >= parts) break;
        const float *from = a.part_o + slot(i) * a.d;
#pragma unroll
        for (int c = 0; c < kPieces; ++c)
          if ((c * 32 + lane) * V < a.d) v[u][c] = *reinterpret_cast<const serve::Pack<float, V> *>(from + (c * 32 + lane) * V);
      }
    };
    const int mine = SHARED ? warp : 0;
    load(mine);
    float mx = -INFINITY, total = 0.0f;
    for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, a.part_ml[slot(i)].x);
    mx = warp_max(mx);
    const float base = mx == -INFINITY ? 0.0f : mx;
    for (int i = lane; i < parts; i += 32) {
      const float2 ml = a.part_ml[slot(i)];
      total += ml.y * exp2_fast(ml.x - base);
    }
    total = warp_sum(total);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    float x[kPieces][V];
#pragma unroll
    for (int c = 0; c < kPieces; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = 0.0f;
    for (int i0 = mine; i0 < parts; i0 += kAhead * kStep) {
      if (i0 != mine) load(i0);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kStep;
        if (i >= parts) break;
        const float w = exp2_fast(a.part_ml[slot(i)].x - base);
#pragma unroll
        for (int c = 0; c < kPieces; ++c)
          if ((c * 32 + lane) * V < a.d)
#pragma unroll
            for (int e = 0; e < V; ++e) x[c][e] = fmaf(v[u][c].v[e], w, x[c][e]);
      }
    }
    if (SHARED) {
      __syncthreads();  // the last row's readers are done
#pragma unroll
      for (int c = 0; c < kPieces; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) sums[warp][(c * 32 + lane) * V + e] = x[c][e];
      __syncthreads();
      T *out = static_cast<T *>(a.o) + (int64_t)(s.first + j) * a.o_token + qh * a.o_head;
      for (int c = threadIdx.x; c < a.d; c += kThreads)
        out[c] = serve::from_f32<T>(((sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c])) * inv);
    } else {
      T *out = static_cast<T *>(a.o) + (int64_t)(s.first + j) * a.o_token + qh * a.o_head;
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const int col = (c * 32 + lane) * V;
        if (col >= a.d) continue;
        serve::Pack<T, V> y;
#pragma unroll
        for (int e = 0; e < V; ++e) y.v[e] = serve::from_f32<T>(x[c][e] * inv);
        if (vec_out) {
          *reinterpret_cast<serve::Pack<T, V> *>(out + col) = y;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) out[col + e] = y.v[e];
        }
      }
    }
  }
}

template <typename T>
cudaError_t merge(const Args &a, int sms, cudaStream_t s) {
  const int64_t rows = (int64_t)a.max_new * a.kv_heads * a.group;
  // A block to a row where it has more parts than one warp's loads and the rows
  // leave SMs idle: 32 / 8 heads of 128, one sequence of 50001 keys 38.0 us, 44.6 with a
  // warp to a row, 4 of 8000 23.9 and 26.8, 8 of 4000 22.5 and 23.4; with four parts
  // and fewer a block to a row costs 2 us (32 of 4000: 62.0 against 60.1), and with
  // rows for all SMs neither is faster.
  const bool shared = a.own_splits + a.prefix_splits > 4 && rows * a.sequences < (int64_t)sms * 8;
  const int64_t blocks = shared ? rows : (rows + kWarps - 1) / kWarps;
  const dim3 grid(a.sequences, (unsigned)std::min<int64_t>(blocks, 65535));
  const bool vec_out = serve::vec_ok(a.o, a.o_token, a.o_head, 0, sizeof(T), 4 * sizeof(T));
  auto kernel = a.d % 4 == 0 ? (shared ? paged_merge_kernel<T, 4, true> : paged_merge_kernel<T, 4, false>)
                             : (shared ? paged_merge_kernel<T, 1, true> : paged_merge_kernel<T, 1, false>);
  return b2k::launch_kernel(a.pdl, kernel, grid, dim3(kThreads), 0, s, a, vec_out);
}

// The kernel of a part: paged_rows_kernel, warp MMAs (paged_mma.cu), the
// tensor-memory kernel (paged_umma.cu) or the f32 decode kernel (paged_f32.cu).
enum Path { kPlain, kMma, kUmma, kF32 };
// What a cache's type and alignment allow.
enum Reach { kNoPieces, kHalfPieces, kFloatPieces };

// What a call launches, from its host values alone.
struct Plan {
  int own_splits, own_chunk, prefix_splits, prefix_chunk, joined, joined_keys;
  Path own_path, prefix_path;
  int own_rows, prefix_rows;  // rows of a block
  size_t bytes;               // workspace
};

// Bytes of the parts' (m, l), which the sums follow on a 16-byte boundary.
size_t ml_bytes(size_t slots, int64_t tokens, int q_heads) {
  return (slots * (size_t)tokens * q_heads * sizeof(float2) + 15) / 16 * 16;
}

// The plain kernel's block, the fewest rows that hold them all: keys are read once,
// and rows that are not there cost what others do (40 sequences of up to 1500 keys,
// 8 cache heads of 100, bf16: 4 rows each 303 us in blocks of 4, 424 of 8, 530 of 32;
// 8 rows each 424 in 8 and 525 in 32; 16 rows each 527 in 32 and 679 in two of 8).
int plain_rows(int64_t rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : 32; }

// Whether the cache can be read in 16-byte pieces throughout, and of what.
Reach cache_pieces(const b2k_paged_cache &c) {
  const int size = c.dtype == B2K_F32 ? 4 : 2;
  if (c.d % (16 / size) || !serve::vec_ok(c.k, c.k_page, c.k_row, c.k_head, size, 16) ||
      !serve::vec_ok(c.v, c.v_page, c.v_row, c.v_head, size, 16))
    return kNoPieces;
  return size == 4 ? kFloatPieces : kHalfPieces;
}
bool rows_pieces(const b2k_heads &x) { return serve::vec_ok(x.data, x.stride_token, x.stride_head, 0, 2, 16); }

// Kernel for a part with `rows` rows and `keys` keys a cache head, in `units`
// such pairs.  Up to 32 rows fit one block of the warp kernel, which then reads
// the keys once as well, two or three blocks an SM; above that the tensor-memory
// kernel's 256 rows save re-reading them, and its products cost less, but its
// launch and its blocks' starts cost about 10 us.  By rows x keys x units: own
// parts are even near 3 million (16 / 4 heads; 2.3 million at head dim 128: 19 us
// with warps, 26 with tensor memory; 4.4 million: 31 and 20; 4.4 million at 64:
// 21 and 17, at 256: 56 and 27), a prefix, whose blocks run beside the own
// part's, near 1.5 million (2 million behind 32 single tokens: 25 and 22; 6.4
// million behind 100: 44 and 31; 0.5 million: even).  Head dims above 128 need
// pages that are boxes there.
// f32: up to 64 rows in the kernel that streams, eight to a block (42 rows of a
// prefix of 333: 15 us a call in it, 20 in the other), more in the one whose
// blocks hold 32 (160 rows of 1000: 64 us against 72; prompts of 430: 161
// against 353).  Up to 4 rows in blocks of 4 (40 sequences of 4 rows over up to 1500
// keys of 128: 81 us, 151 in blocks of 8).  Above, blocks of 8 read the keys half as
// often as two of 4, but the second of those, launched beside the first, finds them
// in L2: 8 rows each of the same 149 us in blocks of 8 against 105.
int g_kernel = 0;  // b2k_paged_attention_set_kernel

Path pick_path(Reach reach, const b2k_paged_cache &c, int64_t rows, int64_t keys, int64_t units, double repaid) {
  if (reach == kNoPieces || g_kernel == 1) return kPlain;
  if (reach == kFloatPieces) return rows <= 64 ? kF32 : kPlain;
  const bool umma = c.d <= 128 || paged::umma_boxes(c);
  if (g_kernel > 1) return g_kernel == 3 && umma ? kUmma : kMma;
  return umma && rows > 32 && (double)rows * keys * units > repaid ? kUmma : kMma;
}
int block_rows(Path path, int d, int64_t rows) {
  return path == kF32 ? (rows <= 4 ? 4 : 8) : path == kPlain ? plain_rows(rows) : path == kMma ? paged::mma_rows(d, rows) : paged::umma_rows(d);
}

// Splits of `keys` keys so that `units` independent row blocks become `want`
// blocks, each at least `least` keys long.
void split_keys(int64_t keys, int64_t units, int64_t want, int least, int tile, int &splits, int &chunk) {
  want = std::max<int64_t>(1, want / std::max<int64_t>(1, units));
  int64_t c = std::max<int64_t>(least, (keys + want - 1) / want);
  c = (c + tile - 1) / tile * tile;
  splits = (int)std::max<int64_t>(1, (keys + c - 1) / c);
  chunk = (int)c;
}

Plan make_plan(const b2k_paged_cache &c, const b2k_paged_batch &b, int q_heads, int sms, Reach reach) {
  Plan p = {};
  const int64_t group = q_heads / c.heads;
  const int64_t own = b.max_new * group, prefix = b.tokens * group;
  p.own_path = pick_path(reach, c, own, (int64_t)b.max_len + b.prefix_len, (int64_t)c.heads * b.sequences, 3e6);
  p.own_rows = block_rows(p.own_path, c.d, own);
  // Sequences whose own rows fill a block read the prefix with their own keys:
  // stacking the rows of several sequences would save no reads of it, and cost a
  // part and its merge (32 / 8 heads of 128, own up to 600 behind 2000: 8 sequences of
  // 64 tokens 49.5 us joined and 53.9 stacked, of 32, 128 rows, 39.4 and 41.2, of 16
  // 37.0 and 34.9; 32 of 16 behind 4000 175 and 76).  Few sequences behind a long
  // prefix lose by it, whose splits the own keys then bound: 4 of 32 behind 8000
  // 50.7 and 43.6.
  p.joined = b.prefix_len > 0 && own >= 128;
  // blocks that the GPU holds at once, and keys that make a block worth its start
  // (a third decode block an SM has room, but its splits cost more than it
  // brings: one sequence of 50001 keys 38 us with two, 41 with three; plain blocks,
  // heads of 100: one of 20000 keys 160 us with four, 196 with six or eight, 40 of up
  // to 1500 365, 303, 312).  The shortest split, plain: 8 sequences of up to 700 31 us
  // with 64 keys, 45 with 128; f32: 9 x 2 tokens of 700 and 333 12.7 with 64, 14.8
  // with 128, 18.5 with 256, one of 8000 or 40 of 1500 the same with each.
  auto wave = [&](Path path) { return (int64_t)sms * (path == kPlain ? 6 : path == kUmma || (path == kMma && c.d > 128) ? 1 : 2); };
  auto least = [&](Path path) { return path == kPlain ? 64 : path == kUmma ? 128 : path == kF32 ? 128 : c.d <= 64 ? 512 : 256; };
  auto tile = [](Path path) { return path == kUmma ? 128 : 64; };  // keys of a block's step
  // the tensor-memory kernel's tiles end with the prefix
  p.joined_keys = !p.joined ? 0 : p.own_path == kUmma ? (b.prefix_len + 127) / 128 * 128 : b.prefix_len;
  // Sequences of different lengths leave a single wave's blocks unequal: two
  // waves of shorter ones even that out (33 sequences of 625 to 2500 keys, 20
  // rows of 64: 38 us with one, 33 with two, 33 to 39 with four).
  const int64_t own_wave = wave(p.own_path) * (b.sequences > 1 && p.own_path != kUmma ? 2 : 1);
  split_keys((int64_t)b.max_len + p.joined_keys,
             (own + p.own_rows - 1) / p.own_rows * c.heads * b.sequences, own_wave, least(p.own_path),
             tile(p.own_path), p.own_splits, p.own_chunk);
  if (b.prefix_len > 0 && !p.joined) {
    p.prefix_path = pick_path(reach, c, prefix, b.prefix_len, c.heads, 1.5e6);
    p.prefix_rows = block_rows(p.prefix_path, c.d, prefix);
    // a few row blocks of the own part's height save a launch, at the price of
    // as many readings of the prefix
    if (p.prefix_path == p.own_path && p.own_path != kUmma && prefix <= 8 * p.own_rows) p.prefix_rows = p.own_rows;
    const int64_t units = (prefix + p.prefix_rows - 1) / p.prefix_rows * c.heads;
    int64_t want = wave(p.prefix_path);
    if (p.prefix_path == kUmma && p.own_path != kUmma) {
      // The prefix part's blocks, one an SM, run beside the own part, which
      // needs the other SMs' loads more than it needs the prefix part done:
      // the fewest splits that do not make it the last to end, by what both
      // take: a block 8 us and 2 us for each 128 keys; the own part the time of
      // its bytes at 5.4 TB/s.  The host knows of the lengths only that none is
      // above max_len: half of that stands for them, as for lengths spread evenly
      // below it (a max_len far above the lengths in use makes the splits too few).
      // 128 sequences of up to 1000 behind 8192 tokens, 32 units: 152 us with one
      // split, 95 with two, 102 with three, 109 with four.
      const double own_us = 0.5 * b.sequences * (double)b.max_len * c.heads * c.d * 4 / 5.4e6;
      for (int64_t s = 1; s * units < want; ++s) {
        const double block_us = 8.0 + 2.0 * ((b.prefix_len + s * 128 - 1) / (s * 128));
        if (block_us <= (units * s * block_us) / sms + own_us) want = s * units;
      }
    }
    split_keys(b.prefix_len, units, want, least(p.prefix_path), tile(p.prefix_path), p.prefix_splits, p.prefix_chunk);
  }
  const size_t slots = (size_t)p.own_splits + p.prefix_splits;
  if (slots > 1) p.bytes = ml_bytes(slots, b.tokens, q_heads) + slots * (size_t)b.tokens * q_heads * c.d * sizeof(float);
  return p;
}

template <typename T, int RW, int DV>
int launch_rows(b2k_ctx *ctx, const Args &a, bool vec, const paged::Grid &g, unsigned blocks, cudaStream_t s) {
  const int dp = (a.d + 3) / 4 * 4;
  const size_t smem = sizeof(float) * (size_t)(RW * kWarps * (dp + 4) + rows_stages<DV>() * kTile * (2 * dp + 4));
  constexpr int kFull = 16 / sizeof(T);
  auto kernel = vec ? paged_rows_kernel<T, RW, DV, kFull> : paged_rows_kernel<T, RW, DV, 1>;
  constexpr int kMost = DV == 0 ? 64 : 128 * DV;  // head dim
  constexpr int most = sizeof(float) * (RW * kWarps * (kMost + 4) + rows_stages<DV>() * kTile * (2 * kMost + 4));
  cudaError_t err = b2k::set_max_smem(ctx, (const void *)kernel, most);
  if (err == cudaSuccess) err = b2k::launch_kernel(a.pdl, kernel, dim3(blocks), dim3(kThreads), smem, s, a, g);
  return err == cudaSuccess ? B2K_OK : b2k::cuda_fail(ctx, err, "paged_attention launch");
}

template <typename T, int RW>
int rows_by_dim(b2k_ctx *ctx, const Args &a, bool vec, const paged::Grid &g, unsigned blocks, cudaStream_t s) {
  return a.d <= 64    ? launch_rows<T, RW, 0>(ctx, a, vec, g, blocks, s)
         : a.d <= 128 ? launch_rows<T, RW, 1>(ctx, a, vec, g, blocks, s)
                      : launch_rows<T, RW, 2>(ctx, a, vec, g, blocks, s);
}

template <typename T>
int rows_parts(b2k_ctx *ctx, const Args &a, bool with_prefix, bool with_own, int rows, bool beside, cudaStream_t s) {
  paged::Grid g = {};
  const int64_t n = paged::make_grid(ctx, a, with_prefix, with_own, rows, beside, g);
  if (n < 0) return B2K_EUNSUPPORTED;
  const size_t size = sizeof(T);
  const bool vec = a.d % (16 / (int)size) == 0 && serve::vec_ok(a.k, a.k_page, a.k_row, a.k_head, size, 16) &&
                   serve::vec_ok(a.v, a.v_page, a.v_row, a.v_head, size, 16);
  const unsigned blocks = (unsigned)n;
  return rows == 4   ? rows_by_dim<T, 1>(ctx, a, vec, g, blocks, s)
         : rows == 8 ? rows_by_dim<T, 2>(ctx, a, vec, g, blocks, s)
                     : rows_by_dim<T, 8>(ctx, a, vec, g, blocks, s);
}

// Two launches of a call being captured, as parallel branches of its graph: what
// the second depends on is set back to what the first did, and what follows
// depends on both.  Not active outside a capture.
class CapturedBranches {
 public:
  CapturedBranches(cudaStream_t s, bool wanted) : s_(s) { active_ = wanted && dependencies(before_); }
  bool active() const { return active_; }
  cudaError_t second() { return dependencies(first_) ? set(before_, cudaStreamSetCaptureDependencies) : cudaErrorUnknown; }
  cudaError_t join() { return set(first_, cudaStreamAddCaptureDependencies); }

 private:
  struct Set {
    std::vector<cudaGraphNode_t> nodes;
    std::vector<cudaGraphEdgeData> edges;
  };
  bool dependencies(Set &out) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    const cudaGraphNode_t *nodes = nullptr;
    const cudaGraphEdgeData *edges = nullptr;
    size_t n = 0;
    if (cudaStreamGetCaptureInfo_v3(s_, &status, nullptr, nullptr, &nodes, &edges, &n) != cudaSuccess) {
      cudaGetLastError();  // the legacy stream beside a capture in another: the launch itself says so
      return false;
    }
    if (status != cudaStreamCaptureStatusActive) return false;
    try {
      out.nodes.assign(nodes, nodes + n);
      out.edges.assign(n, cudaGraphEdgeData{});
      if (edges) out.edges.assign(edges, edges + n);
    } catch (const std::bad_alloc &) {
      return false;
    }
    return true;
  }
  cudaError_t set(Set &deps, unsigned flags) {
    return cudaStreamUpdateCaptureDependencies_v2(s_, deps.nodes.data(), deps.edges.data(), deps.nodes.size(), flags);
  }
  cudaStream_t s_;
  bool active_ = false;
  Set before_, first_;
};

template <typename T>
int run(b2k_ctx *ctx, Args &a, const Plan &p, int32_t dtype, cudaStream_t s) {
  int launches = 1, status = B2K_OK;
  const bool prefix = a.prefix_splits > 0, several = a.own_splits + a.prefix_splits > 1;
  CapturedBranches branches(s, several);
  if (several && !branches.active()) {
    a.call = ++ctx->order_calls;
    a.ready = ctx->order_words + a.call % b2k_ctx::kOrderWords;
  }
  auto parts = [&](Path path, bool pre, bool own, int rows, bool beside) {
    return path == kPlain ? rows_parts<T>(ctx, a, pre, own, rows, beside, s)
           : path == kMma ? paged::mma_parts(ctx, a, dtype, pre, own, rows, beside, s)
           : path == kF32 ? paged::f32_parts(ctx, a, pre, own, rows, beside, s)
                          : paged::umma_part(ctx, a, dtype, pre, s);
  };
  if (!prefix) {
    status = parts(p.own_path, false, true, p.own_rows, false);
  } else if (p.own_path == p.prefix_path && p.own_path != kUmma && p.own_rows == p.prefix_rows) {
    status = parts(p.own_path, true, true, p.own_rows, false);
  } else if (p.own_path != kUmma && branches.active()) {
    status = parts(p.prefix_path, true, false, p.prefix_rows, false);
    cudaError_t err = status == B2K_OK ? branches.second() : cudaSuccess;
    a.pdl = false;  // the own part's and the merge's dependences are whole
    if (status == B2K_OK && err == cudaSuccess) status = parts(p.own_path, false, true, p.own_rows, false);
    if (status == B2K_OK && err == cudaSuccess) err = branches.join();
    if (err != cudaSuccess) status = b2k::cuda_fail(ctx, err, "paged_attention capture");
    ++launches;
  } else {
    status = parts(p.prefix_path, true, false, p.prefix_rows, false);
    // (the tensor-memory kernel waits)
    if (status == B2K_OK) status = parts(p.own_path, false, true, p.own_rows, p.own_path != kUmma);
    ++launches;
  }
  if (status != B2K_OK) return status;
  if (a.own_splits + a.prefix_splits > 1) {
    const cudaError_t err = merge<T>(a, ctx->sm_count, s);
    if (err != cudaSuccess) return b2k::cuda_fail(ctx, err, "paged_attention launch");
    ++launches;
  }
  return b2k::check_launch(ctx, "paged_attention launch", launches);
}

int check_call(b2k_ctx *ctx, const b2k_paged_cache *cache, const b2k_paged_batch *batch, int32_t q_heads) {
  int status = serve::check_cache(ctx, "paged_attention", cache);
  if (status == B2K_OK) status = serve::check_batch(ctx, "paged_attention", cache, batch);
  if (status != B2K_OK) return status;
  if (q_heads < 1 || q_heads > 65535 || q_heads % cache->heads)
    return b2k::fail(ctx, B2K_EINVAL, "paged_attention: %d query heads for %d cache heads", q_heads, cache->heads);
  // the limits of a launch's grid, and of a row's 32-bit number
  constexpr int64_t kMost = INT32_MAX - 65536;  // sums of a row's or key's number and a block's stay within 32 bits
  if (batch->sequences > 65535 || batch->tokens * q_heads > kMost || (int64_t)batch->max_new * q_heads > kMost ||
      (int64_t)batch->max_len + batch->prefix_len > kMost)
    return b2k::fail(ctx, B2K_EUNSUPPORTED, "paged_attention: a batch of %d sequences, %lld rows is too large",
                     batch->sequences, (long long)(batch->tokens * q_heads));
  return B2K_OK;
}

}  // namespace

// Workspace of a call with these host values, whatever its q and o are: those
// off 16 bytes take the plain kernel, which splits otherwise.
static size_t workspace_bytes_of(const b2k_paged_cache &c, const b2k_paged_batch &b, int q_heads, int sms) {
  const Reach reach = cache_pieces(c);
  const size_t plain = make_plan(c, b, q_heads, sms, kNoPieces).bytes;
  return reach == kNoPieces ? plain : std::max(plain, make_plan(c, b, q_heads, sms, reach).bytes);
}

// Everything about a call's arguments but its workspace, and its plan.
static int check_operands(b2k_ctx *ctx, const b2k_paged_cache *cache, const b2k_paged_batch *batch, const b2k_heads *q,
                          const b2k_heads *o, int sms, Plan &p) {
  const char *what = "paged_attention";
  if (!q) return b2k::fail(ctx, B2K_EINVAL, "%s: no q", what);
  int status = check_call(ctx, cache, batch, q->heads);
  if (status == B2K_OK) status = serve::check_heads(ctx, what, "q", q, batch->tokens, cache->d, cache->dtype);
  if (status == B2K_OK) status = serve::check_output(ctx, what, "o", o, batch->tokens, cache->d, cache->dtype);
  if (status != B2K_OK) return status;
  if (q->heads != o->heads) return b2k::fail(ctx, B2K_EINVAL, "%s: %d heads in, %d out", what, q->heads, o->heads);
  if (q->data == o->data && batch->tokens > 0) return b2k::fail(ctx, B2K_EINVAL, "%s: o is q", what);
  Reach reach = cache_pieces(*cache);
  if (reach == kHalfPieces && !(rows_pieces(*q) && rows_pieces(*o))) reach = kNoPieces;
  p = make_plan(*cache, *batch, q->heads, sms, reach);
  return B2K_OK;
}

extern "C" int b2k_paged_attention_set_kernel(int mode) {
  if (mode < 0 || mode > 3) return B2K_EINVAL;
  g_kernel = mode;
  return B2K_OK;
}

extern "C" int b2k_paged_attention_plan(int32_t sms, const b2k_paged_cache *cache, const b2k_paged_batch *batch,
                                        const b2k_heads *q, const b2k_heads *o, b2k_paged_attention_plan_info *out) {
  if (sms < 1 || !out) return B2K_EINVAL;
  Plan p;
  const int status = check_operands(nullptr, cache, batch, q, o, sms, p);
  if (status != B2K_OK) return status;
  auto shown = [](Path path) { return path == kF32 ? 0 : (int32_t)path; };
  *out = {shown(p.own_path), p.prefix_splits > 0 ? shown(p.prefix_path) : -1, p.own_splits, p.own_chunk,
          p.prefix_splits, p.prefix_chunk, p.joined,
          (p.own_path == kF32 ? 1 : 0) + (p.prefix_splits > 0 && p.prefix_path == kF32 ? 2 : 0),
          (int64_t)workspace_bytes_of(*cache, *batch, q->heads, sms)};
  return B2K_OK;
}

extern "C" int b2k_paged_attention_workspace(b2k_ctx *ctx, const b2k_paged_cache *cache, const b2k_paged_batch *batch,
                                             int32_t q_heads, size_t *bytes) {
  if (!ctx) return B2K_EINVAL;
  if (!bytes) return b2k::fail(ctx, B2K_EINVAL, "paged_attention_workspace: null result");
  int status = check_call(ctx, cache, batch, q_heads);
  if (status != B2K_OK) return status;
  *bytes = workspace_bytes_of(*cache, *batch, q_heads, ctx->sm_count);
  return B2K_OK;
}

extern "C" int b2k_paged_attention(b2k_ctx *ctx, const b2k_paged_cache *cache, const b2k_paged_batch *batch,
                                   const b2k_heads *q, const b2k_heads *o, float scale_div, void *workspace,
                                   size_t workspace_bytes, void *stream) {
  B2K_CHECK_CTX(ctx);
  const char *what = "paged_attention";
  // (a subnormal scale's reciprocal is beyond FP32)
  const float scale_log2 = (float)(1.4426950408889634074 / scale_div);
  if (!(scale_div > 0.0f) || !isfinite(scale_div) || !isfinite(scale_log2))
    return b2k::fail(ctx, B2K_EINVAL, "%s: scale %g", what, scale_div);
  Plan p;
  int status = check_operands(ctx, cache, batch, q, o, ctx->sm_count, p);
  if (status == B2K_OK) status = serve::check_apart(ctx, what, "o", *o, *q, false, batch->tokens, cache->d, cache->dtype);
  if (status != B2K_OK) return status;
  if (batch->sequences == 0 || batch->tokens == 0 || batch->max_new == 0) return B2K_OK;
  const size_t needed = workspace_bytes_of(*cache, *batch, q->heads, ctx->sm_count);
  if (needed > 0 && (!workspace || workspace_bytes < needed))
    return b2k::fail(ctx, B2K_EINVAL, "%s: a workspace of %zu bytes where %zu are needed", what,
                     workspace ? workspace_bytes : (size_t)0, needed);
  if (needed > 0 && !b2k::aligned16(workspace))
    return b2k::fail(ctx, B2K_EINVAL, "%s: the workspace is not 16-byte aligned", what);
  Args a = {};
  a.q = q->data;
  a.o = o->data;
  a.q_token = q->stride_token;
  a.q_head = q->stride_head;
  a.o_token = o->stride_token;
  a.o_head = o->stride_head;
  a.k = cache->k;
  a.v = cache->v;
  a.k_page = cache->k_page;
  a.k_row = cache->k_row;
  a.k_head = cache->k_head;
  a.v_page = cache->v_page;
  a.v_row = cache->v_row;
  a.v_head = cache->v_head;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  a.kv_heads = cache->heads;
  a.group = q->heads / cache->heads;
  a.d = cache->d;
  a.sequences = batch->sequences;
  a.tokens = batch->tokens;
  a.first = batch->first;
  a.lengths = batch->lengths;
  a.table = batch->table;
  a.prefix_table = batch->prefix_table;
  a.table_stride = batch->table_stride;
  a.table_width = batch->table_width;
  a.prefix_len = batch->prefix_len;
  a.max_new = batch->max_new;
  a.max_len = batch->max_len;
  a.scale_log2 = scale_log2;
  a.err = ctx->error_flag;
  a.pdl = b2k::pdl_enabled();
  a.own_splits = p.own_splits;
  a.own_chunk = p.own_chunk;
  a.prefix_splits = p.prefix_splits;
  a.prefix_chunk = p.prefix_chunk;
  a.joined = p.joined;
  a.joined_keys = p.joined_keys;
  if (p.bytes > 0) {
    const size_t slots = (size_t)(p.own_splits + p.prefix_splits);
    a.part_ml = static_cast<float2 *>(workspace);
    a.part_o = reinterpret_cast<float *>(static_cast<char *>(workspace) + ml_bytes(slots, batch->tokens, q->heads));
  }
  cudaStream_t s = (cudaStream_t)stream;
  b2k::PhaseTimer timer(ctx, B2K_PHASE_PAGED, s);
  if (cache->dtype == B2K_F32) return run<float>(ctx, a, p, cache->dtype, s);
  if (cache->dtype == B2K_F16) return run<__half>(ctx, a, p, cache->dtype, s);
  return run<__nv_bfloat16>(ctx, a, p, cache->dtype, s);
}
