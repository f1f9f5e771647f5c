// Rotary positions, and the append of rotated keys (and values) to a paged
// cache: one kernel, since both move each element once and differ in where
// the result goes.
//
// Mathematics.  A pair (a, b) of a head turns by position * f_i.  The plan
// holds f_i / 2 pi as a 64-bit fraction of a turn, so position * turn_i in
// wrapping 64-bit integer arithmetic IS the angle modulo one turn; its top 32
// bits, as a signed number, give the angle in half turns for sincospif.  The
// angle's error is what those bits leave out (below 2^-32 turns), the rounding
// of that number to FP32 (at most 2^-25 half turns) and |position| times the
// fraction's own error (b2k_rope_plan: below 2^-62 turns, 2^-22 of a turn at
// position 2^40): no table of cosines is read, kept or outgrown, and no FP32
// product position * f loses the far positions.
//
// Bound: HBM (each element read and written once).  A warp takes a token, or
// some of its heads where tokens are few; nothing in a block waits for another
// warp.  The lanes share out the token's cosines and sines through shared memory
// while the first heads' loads are in flight; then every lane keeps one place
// of the head (16 bytes of each half of its pairs, its cosines in registers)
// and walks the heads, whose loads are all on their way by then.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "serve.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxPairs = B2K_ROPE_MAX_PAIRS;

enum Target : int { kLinear = 0, kKeys = 1, kValues = 2 };

// One tensor of the call: source, destination, and whether it is rotated.
struct Segment {
  const char *x;
  char *y;
  int64_t xt, xh;      // source strides in bytes: token, head
  int64_t yp, yt, yh;  // destination strides in bytes: page, token or row, head
  int heads, target, rotate;
};

struct RotaryArgs {
  Segment seg[3];
  int count, heads, d, rot, interleaved;  // heads: of all segments
  float magnitude, sine;  // sine: +magnitude, or -magnitude for the transpose
  int items;              // places of a head: a lane keeps one
  int warps_log2;         // of the warps that share a token (1, 2, 4 or 8)
  int64_t tokens;
  const int64_t *positions;  // unpaged
  // paged
  const int32_t *first, *lengths, *table;
  int64_t table_stride, pages;
  int table_width, page_size, prefix_len, max_new, max_len;
  unsigned *err;
  uint64_t turn[kMaxPairs];
};

// V values from and to T, two at a time where the type has such an instruction.
template <typename T, int V>
__device__ __forceinline__ void widen(const serve::Pack<T, V> &p, float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = serve::to_f32(p.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void narrow(const float (&x)[V], serve::Pack<T, V> &p) {
  if constexpr (V % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (std::is_same<T, __half>::value)
        *reinterpret_cast<__half2 *>(&p.v[i]) = __floats2half2_rn(x[i], x[i + 1]);
      else
        *reinterpret_cast<__nv_bfloat162 *>(&p.v[i]) = __floats2bfloat162_rn(x[i], x[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = serve::from_f32<T>(x[i]);
  }
}

// 16 bytes global to shared memory, for this thread alone.
__device__ __forceinline__ void copy16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

// Many tokens of 16-byte vectors: a lane's loads wait in shared memory, kSlots
// steps of two vectors of all the token's segments at once, and cost no
// registers: six blocks of four warps an SM have 190 KB on the way, where four
// heads ahead in registers are 64.  Calls back to back, from registers and staged:
// 16384 tokens x 40 heads of 128, bf16 57.5 and 55.9 us; 12 prompts into a cache,
// interleaved f16 46.6 and 43.0; but the gradient of 6001 x 32 heads of 64,
// interleaved f32, 18.0 and 19.0.
// Small blocks, a token a warp, keep the last wave short: blocks of eight warps
// 57.3, 44.5 and 19.5 us, the first with two tokens a warp 60, with four 71.
constexpr int kSlots = 8, kStagedWarps = 4;
template <typename T, int V, bool FLAT>
constexpr bool kStaged = !FLAT && V * sizeof(T) == 16;
template <typename T, int V, bool FLAT>
constexpr int block_warps() { return kStaged<T, V, FLAT> ? kStagedWarps : kWarps; }
template <typename T, int V, bool FLAT>
constexpr int staged_bytes() { return kStaged<T, V, FLAT> ? kStagedWarps * kSlots * 2 * 32 * 16 : 0; }

// FLAT, for few tokens with several warps to each: the heads of all segments in
// one walk through registers, so that the few heads a lane has of each load
// together (61 tokens into a cache: 5.5 -> 4.5 us); without it segment after
// segment, whose addresses are simple steps (16384 tokens: 60 -> 58 us).
template <typename T, int V, bool PAGED, bool FLAT>
__global__ void __launch_bounds__(32 * block_warps<T, V, FLAT>(), kStaged<T, V, FLAT> ? 24 / kStagedWarps : V * sizeof(T) == 16 && sizeof(T) == 2 ? 2 : 4) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  using P = serve::Pack<T, V>;
  constexpr int kAhead = V * sizeof(T) == 16 && sizeof(T) == 2 ? 4 : 2;  // heads a lane has in registers
  extern __shared__ uint4 slots[];  // staged: [warp][step][two vectors][lane]
  constexpr int kBlockWarps = block_warps<T, V, FLAT>();
  __shared__ __align__(16) float cs[kBlockWarps][kMaxPairs], sn[kBlockWarps][kMaxPairs];
  grid_dependency_wait();
  grid_dependents_launch();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tokens_per_block = kBlockWarps >> a.warps_log2;
  const int pairs = a.rot / 2;
  // rows of this block's sequence (paged) or of the call
  int64_t row_begin = 0, row_end = a.tokens, own0 = 0;
  if (PAGED) {
    const int b = blockIdx.x;
    row_begin = a.first[b];
    const int64_t n = (int64_t)a.first[b + 1] - row_begin;
    const int len = a.lengths[b];
    own0 = len - n;
    row_end = row_begin + n;
    if (row_begin < 0 || n < 0 || row_end > a.tokens || n > a.max_new || len < 0 || len > a.max_len) {
      if (threadIdx.x == 0) atomicOr(a.err, serve::kErrIndex);
      return;
    }
  }
  // A head has at most 32 places for a whole warp to walk several heads at once;
  // more (single elements) are walked 32 at a time, one head after the other.
  const int per_warp = a.items <= 32 ? 32 / a.items : 1;
  const int slot = a.items <= 32 ? lane / a.items : 0, j_first = a.items <= 32 ? lane - slot * a.items : lane;
  const int head_step = per_warp << a.warps_log2, h_first = (warp & ((1 << a.warps_log2) - 1)) * per_warp + slot;
  const int half_items = a.interleaved ? 0 : a.rot / 2 / V;

  const int64_t chunk0 = PAGED ? blockIdx.y : blockIdx.x, chunk_step = PAGED ? gridDim.y : gridDim.x;
  for (int64_t row = row_begin + chunk0 * tokens_per_block + (warp >> a.warps_log2); row < row_end; row += chunk_step * tokens_per_block) {
    int64_t page = -1;
    int page_row = 0;
    bool turned = false;  // cosines and sines are there
    for (int j = j_first; j < a.items; j += 32) {
      const bool on = slot < per_warp;
      // The two vectors of the head this lane moves, so that neighbouring lanes
      // move neighbouring vectors: the two halves of V pairs (half layout, rotated
      // part), or the j-th vectors of the two halves of what is left.
      int e0, e1;
      if (j < half_items) {
        e0 = j * V;
        e1 = e0 + a.rot / 2;
      } else if (V == 1 && a.interleaved) {
        e0 = 2 * j;  // a pair
        e1 = e0 + 1 < a.d ? e0 + 1 : -1;
      } else {
        e0 = (a.interleaved ? 0 : a.rot) + (j - half_items) * V;
        e1 = e0 + (a.items - half_items) * V;
        if (e1 >= a.d) e1 = -1;
      }
      P va[kAhead], vb[kAhead];
      const int h1 = a.count > 1 ? a.seg[0].heads : INT32_MAX, h2 = a.count > 2 ? h1 + a.seg[1].heads : INT32_MAX;
      // of head h of walk g: the segment's own, or (FLAT) that of the segment it falls into
      auto pick = [&](int h, auto own, auto first, auto second, auto third) {
        if constexpr (FLAT) return h >= h2 ? third : h >= h1 ? second : first;
        else return own;
      };
      const char *x0 = a.seg[0].x + row * a.seg[0].xt, *x1 = a.seg[1].x + row * a.seg[1].xt, *x2 = a.seg[2].x + row * a.seg[2].xt;
      auto load = [&](int g, int hb) {
        const Segment &s = a.seg[g];
        const int heads = FLAT ? a.heads : s.heads;
        const char *base = FLAT ? nullptr : s.x + row * s.xt;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int h = hb + u * head_step;
          if (h >= heads) break;
          const char *x = pick(h, base, x0, x1, x2) +
                          (h - pick(h, 0, 0, h1, h2)) * pick(h, s.xh, a.seg[0].xh, a.seg[1].xh, a.seg[2].xh);
          va[u] = *reinterpret_cast<const P *>(x + e0 * (int)sizeof(T));
          if (e1 >= 0) vb[u] = *reinterpret_cast<const P *>(x + e1 * (int)sizeof(T));
        }
      };
      uint4 *const slot_at = slots + threadIdx.x / 32 * (kSlots * 2 * 32) + lane;
      // walks the steps from (g, hb) on, at most kSlots: f(segment, head, step)
      auto walk = [&](int &g, int &hb, auto f) {
        for (int n = 0; g < a.count && n < kSlots; ++n) {
          const Segment &s = a.seg[g];
          if (on && hb + h_first < s.heads) f(s, hb + h_first, n);
          hb += head_step;
          if (hb >= s.heads) ++g, hb = 0;
        }
      };
      auto issue = [&](int g, int hb) {
        walk(g, hb, [&](const Segment &s, int h, int n) {
          const char *x = s.x + row * s.xt + h * s.xh;
          copy16(slot_at + 64 * n, x + e0 * (int)sizeof(T));
          if (e1 >= 0) copy16(slot_at + 64 * n + 32, x + e1 * (int)sizeof(T));
        });
      };
      if constexpr (kStaged<T, V, FLAT>) issue(0, 0);
      else if (on) load(0, h_first);
      if (!turned) {
        const int64_t own = own0 + (row - row_begin);
        const int64_t pos = PAGED ? a.prefix_len + own : pairs ? a.positions[row] : 0;
        if (PAGED) {
          // where this token's keys and values go
          page = serve::page_of(a.table + blockIdx.x * a.table_stride, a.table_width, a.pages, a.page_size, own);
          page_row = (int)((uint32_t)own % (uint32_t)a.page_size);
          if (page < 0) atomicOr(a.err, serve::kErrIndex);
        }
        __syncwarp();  // the last token's cosines have been read
        for (int p = lane; p < pairs; p += 32) {
          const uint64_t turns = a.turn[p] * (uint64_t)pos;
          float s, c;
          sincospif((float)(int32_t)(turns >> 32) * 4.656612873077392578125e-10f, &s, &c);  // 2^-31
          cs[warp][p] = c * a.magnitude;
          sn[warp][p] = s * a.sine;
        }
        __syncwarp();
        turned = true;
      }
      // this lane's V pairs: of the half layout, or V / 2 of each vector
      auto pair_of = [&](int i) {
        if (!a.interleaved) return j < half_items ? j * V + i : kMaxPairs;
        if (V == 1) return j;
        return (2 * i < V ? e0 : e1 < 0 ? 2 * kMaxPairs : e1) / 2 + i % (V > 1 ? V / 2 : 1);
      };
      float c[V], sv[V];
      bool turns = false;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int p = pair_of(i);
        const bool in = p < pairs;
        turns = turns || in;
        c[i] = in ? cs[warp][p] : 0.0f;
        sv[i] = in ? sn[warp][p] : 0.0f;
      }
      if (!on) continue;
      auto target = [&](const Segment &s) {
        return s.y + (PAGED && s.target != kLinear ? page * s.yp + page_row * s.yt : row * s.yt);
      };
      auto finish = [&](P &pa, P &pb, char *y, bool rotate) {
        if (turns && rotate) {
          float xa[V], xb[V];
          if (a.interleaved) {
            // neighbours a, b, a, b ...: pair i is in the first vector for i < V / 2
            float lo[V], hi[V];
            widen<T, V>(pa, lo);
            widen<T, V>(pb, hi);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              xa[i] = 2 * i < V ? lo[2 * i % V] : hi[2 * i % V];
              xb[i] = 2 * i + 1 < V ? lo[(2 * i + 1) % V] : hi[(2 * i + 1) % V];
            }
          } else {
            widen<T, V>(pa, xa);
            widen<T, V>(pb, xb);
          }
          float ya[V], yb[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            ya[i] = xa[i] * c[i] - xb[i] * sv[i];
            yb[i] = xb[i] * c[i] + xa[i] * sv[i];
          }
          if (a.interleaved) {
            float lo[V], hi[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
              (2 * i < V ? lo[2 * i % V] : hi[2 * i % V]) = ya[i];
              (2 * i + 1 < V ? lo[(2 * i + 1) % V] : hi[(2 * i + 1) % V]) = yb[i];
            }
            P ta, tb;
            narrow<T, V>(lo, ta);
            narrow<T, V>(hi, tb);
            // pairs behind the rotated part stay as they were, bit for bit: a NaN
            // would lose its sign and payload on the way through FP32
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (pair_of(i) < pairs) {
                (2 * i < V ? pa : pb).v[2 * i % V] = (2 * i < V ? ta : tb).v[2 * i % V];
                (2 * i + 1 < V ? pa : pb).v[(2 * i + 1) % V] = (2 * i + 1 < V ? ta : tb).v[(2 * i + 1) % V];
              }
          } else {
            narrow<T, V>(ya, pa);
            narrow<T, V>(yb, pb);
          }
        }
        *reinterpret_cast<P *>(y + e0 * (int)sizeof(T)) = pa;
        if (e1 >= 0) *reinterpret_cast<P *>(y + e1 * (int)sizeof(T)) = pb;
      };
      if constexpr (kStaged<T, V, FLAT>) {
        for (int g = 0, hb = 0; g < a.count;) {
          if (g > 0 || hb > 0) issue(g, hb);
          asm volatile("cp.async.wait_all;" ::: "memory");
          walk(g, hb, [&](const Segment &s, int h, int n) {
            if (PAGED && page < 0 && s.target != kLinear) return;
            P pa = *reinterpret_cast<const P *>(slot_at + 64 * n), pb = {};
            if (e1 >= 0) pb = *reinterpret_cast<const P *>(slot_at + 64 * n + 32);
            finish(pa, pb, target(s) + h * s.yh, s.rotate);
          });
        }
        continue;
      }
      char *y0 = nullptr, *y1 = nullptr, *y2 = nullptr;
      if (FLAT) y0 = target(a.seg[0]), y1 = target(a.seg[1]), y2 = target(a.seg[2]);
      for (int g = 0; g < (FLAT ? 1 : a.count); ++g) {
        const Segment &s = a.seg[g];
        const int heads = FLAT ? a.heads : s.heads;
        if (!FLAT && PAGED && page < 0 && s.target != kLinear) continue;
        char *base = FLAT ? nullptr : target(s);
        for (int hb = h_first; hb < heads; hb += kAhead * head_step) {
          if (g > 0 || hb != h_first) load(g, hb);
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const int h = hb + u * head_step;
            if (h >= heads) break;
            if (FLAT && PAGED && page < 0 && pick(h, 0, a.seg[0].target, a.seg[1].target, a.seg[2].target) != kLinear) continue;
            char *y = pick(h, base, y0, y1, y2) +
                      (h - pick(h, 0, 0, h1, h2)) * pick(h, s.yh, a.seg[0].yh, a.seg[1].yh, a.seg[2].yh);
            finish(va[u], vb[u], y, pick(h, s.rotate, a.seg[0].rotate, a.seg[1].rotate, a.seg[2].rotate));
          }
        }
      }
    }
  }
}

// Widest vector (elements) that every tensor of the call and the layout of
// its heads allow: 16 bytes, 8 bytes or single elements.
int pick_vector(const RotaryArgs &a, int count, size_t size) {
  for (int bytes = 16; bytes >= 8; bytes /= 2) {
    const int v = bytes / (int)size;
    bool ok = a.d % v == 0 && (a.interleaved || a.rot % (2 * v) == 0);
    for (int i = 0; ok && i < count; ++i) {
      const Segment &s = a.seg[i];
      ok = serve::vec_ok(s.x, s.xt, s.xh, 0, 1, bytes) && serve::vec_ok(s.y, s.yp, s.yt, s.yh, 1, bytes);
    }
    if (ok) return v;
  }
  return 1;
}

template <typename T, int V, bool PAGED>
cudaError_t launch(b2k_ctx *ctx, const RotaryArgs &a, dim3 grid, cudaStream_t s) {
  // few tokens, several warps to each: few heads a lane
  auto kernel = a.warps_log2 > 1 ? rotary_kernel<T, V, PAGED, true> : rotary_kernel<T, V, PAGED, false>;
  const int bytes = a.warps_log2 > 1 ? 0 : staged_bytes<T, V, false>();
  if (bytes > 0) {
    const cudaError_t err = b2k::set_max_smem(ctx, (const void *)kernel, bytes);
    if (err != cudaSuccess) return err;
  }
  return b2k::launch_kernel(b2k::pdl_enabled(), kernel, grid, dim3(32 * (bytes > 0 ? kStagedWarps : kWarps)), bytes, s, a);
}

template <typename T, bool PAGED>
cudaError_t launch(b2k_ctx *ctx, const RotaryArgs &a, int v, dim3 grid, cudaStream_t s) {
  constexpr int kFull = 16 / sizeof(T);
  if (v == kFull) return launch<T, kFull, PAGED>(ctx, a, grid, s);
  if (v == kFull / 2) return launch<T, kFull / 2, PAGED>(ctx, a, grid, s);
  return launch<T, 1, PAGED>(ctx, a, grid, s);
}

// Fill in the vector width and the block shape, and launch.  `tokens_each`:
// tokens of one blockIdx.x (paged: of a sequence).
template <bool PAGED>
int run(b2k_ctx *ctx, RotaryArgs &a, int count, int32_t dtype, int64_t tokens_each, unsigned sequences, int phase,
        cudaStream_t s, const char *what) {
  a.count = count;
  const size_t size = serve::type_size(dtype);
  const int v = pick_vector(a, count, size);
  a.items = a.interleaved ? (a.d + 2 * v - 1) / (2 * v) : a.rot / 2 / v + (a.d - a.rot + 2 * v - 1) / (2 * v);
  // A warp to a token once that fills the GPU (64 warps an SM); fewer tokens are
  // shared out, down to one batch of loads a lane.
  const int64_t all = PAGED ? tokens_each * sequences : tokens_each;
  const int per_warp = a.items <= 32 ? 32 / a.items : 1;
  int wpt = 1;
  a.warps_log2 = 0;
  while (wpt < kWarps && all * wpt < (int64_t)ctx->sm_count * 8 * kWarps && per_warp * wpt < a.heads) {
    wpt *= 2;
    ++a.warps_log2;
  }
  const int tokens_per_block = (a.warps_log2 <= 1 && v * size == 16 ? kStagedWarps : kWarps) / wpt;
  const int64_t chunks = (tokens_each + tokens_per_block - 1) / tokens_per_block;
  const dim3 grid = PAGED ? dim3(sequences, (unsigned)std::min<int64_t>(chunks, 65535))
                          : dim3((unsigned)std::min<int64_t>(chunks, INT32_MAX));
  b2k::PhaseTimer timer(ctx, phase, s);
  cudaError_t err = dtype == B2K_F32   ? launch<float, PAGED>(ctx, a, v, grid, s)
                    : dtype == B2K_F16 ? launch<__half, PAGED>(ctx, a, v, grid, s)
                                       : launch<__nv_bfloat16, PAGED>(ctx, a, v, grid, s);
  if (err != cudaSuccess) return b2k::cuda_fail(ctx, err, what);
  return b2k::check_launch(ctx, what);
}

int use_rope(b2k_ctx *ctx, const char *what, const b2k_rope *rope, int32_t d, int transpose, RotaryArgs &a) {
  if (rope->rot < 2 || rope->rot > 2 * kMaxPairs || rope->rot % 2 || rope->rot > d)
    return b2k::fail(ctx, B2K_EINVAL, "%s: %d rotated elements of a head of %d", what, rope->rot, d);
  a.rot = rope->rot;
  a.interleaved = rope->interleaved != 0;
  a.magnitude = rope->magnitude;
  a.sine = transpose ? -rope->magnitude : rope->magnitude;
  for (int i = 0; i < rope->rot / 2; ++i) a.turn[i] = rope->turn[i];
  return B2K_OK;
}

}  // namespace

namespace serve {

int check_heads(b2k_ctx *ctx, const char *what, const char *name, const b2k_heads *x, int64_t tokens, int32_t d,
                int32_t dtype) {
  if (!x) return b2k::fail(ctx, B2K_EINVAL, "%s: no %s", what, name);
  if (x->heads < 1 || x->heads > 65535) return b2k::fail(ctx, B2K_EINVAL, "%s: %s has %d heads", what, name, x->heads);
  if (tokens > 0 && !x->data) return b2k::fail(ctx, B2K_EINVAL, "%s: null %s", what, name);
  if (!on_boundary(x->data, type_size(dtype)))
    return b2k::fail(ctx, B2K_EINVAL, "%s: %s is off its elements' boundary", what, name);
  if (x->stride_token < 0 || x->stride_head < 0 || (x->heads > 1 && x->stride_head < d))
    return b2k::fail(ctx, B2K_EINVAL, "%s: %s has strides %lld, %lld", what, name, (long long)x->stride_token,
                     (long long)x->stride_head);
  return B2K_OK;
}

namespace {
using Wide = __int128;  // products of strides and counts
Wide floor_div(Wide a, Wide b) { return a / b - (a % b != 0 && (a < 0) != (b < 0)); }
}  // namespace

// Rows of d elements begin at t * st + h * sh, t < tokens, h < heads.
bool overlaps_itself(const b2k_heads &x, int64_t tokens, int32_t d) {
  const Wide st = x.stride_token, sh = x.stride_head;
  if ((tokens > 1 && st < d) || (x.heads > 1 && sh < d)) return true;
  if (tokens <= 1 || x.heads <= 1) return false;
  if (st >= (x.heads - 1) * sh + d || sh >= (tokens - 1) * st + d) return false;  // one axis within the other's step
  // h heads on and t tokens back, less than a row apart
  for (Wide h = 1; h < x.heads; ++h) {
    const Wide t = floor_div(h * sh, st);
    if ((t >= 1 && t < tokens && h * sh - t * st < d) || (t + 1 < tokens && (t + 1) * st - h * sh < d)) return true;
  }
  return false;
}

// The same of rows of two tensors, y's from y - x bytes on.  Exact where the
// tokens follow each other in both by the same step with a token's heads within
// it, or where both strides are the same; other tensors, whose extents cross, count
// as overlapping.
bool overlap(const b2k_heads &x, const b2k_heads &y, int64_t tokens, int32_t d, size_t size) {
  if (tokens == 0) return false;
  const Wide row = (Wide)d * size, n = size;
  const Wide from = (Wide)reinterpret_cast<uintptr_t>(y.data) - (Wide)reinterpret_cast<uintptr_t>(x.data);
  const Wide tx = x.stride_token == 0 ? 1 : tokens, ty = y.stride_token == 0 ? 1 : tokens;  // tokens apart
  Wide xt = x.stride_token * n, yt = y.stride_token * n, xh = x.stride_head * n, yh = y.stride_head * n;
  if (tx == 1) xt = yt;
  if (ty == 1) yt = xt;
  if (x.heads == 1) xh = yh;
  if (y.heads == 1) yh = xh;
  const Wide x_row = (x.heads - 1) * xh + row, y_row = (y.heads - 1) * yh + row;  // bytes of a token with its heads
  if (from >= (tx - 1) * xt + x_row || -from >= (ty - 1) * yt + y_row) return false;
  if (tx == 1 && ty == 1) xt = yt = std::max(x_row, y_row);
  if (xt != yt) return true;
  if (xt >= x_row && xt >= y_row) {
    // y's token t steps on from x's: the two walks over the heads, side by side
    for (Wide t = std::max(1 - tx, floor_div(-from - y_row, xt)); t < ty && from + t * xt < x_row; ++t) {
      const Wide off = from + t * xt;
      if (-off >= y_row) continue;
      for (int64_t i = 0, j = 0; i < x.heads && j < y.heads;) {
        const Wide apart = off + j * yh - i * xh;
        if (apart < row && -apart < row) return true;
        if (apart > 0) ++i;
        else ++j;
      }
    }
    return false;
  }
  if (xh != yh) return true;
  for (Wide h = 1 - x.heads; h < y.heads; ++h) {
    // the tokens t apart whose heads h apart are nearest, below and above
    const Wide off = from + h * xh, t = floor_div(-off, xt);
    for (Wide u : {t, t + 1}) {
      const Wide apart = off + std::min(std::max(u, 1 - tx), ty - 1) * xt;
      if (apart < row && -apart < row) return true;
    }
  }
  return false;
}

// check_heads, and no two rows of it in one place (an input may repeat a token).
int check_output(b2k_ctx *ctx, const char *what, const char *name, const b2k_heads *x, int64_t tokens, int32_t d,
                 int32_t dtype) {
  const int status = check_heads(ctx, what, name, x, tokens, d, dtype);
  if (status != B2K_OK || !overlaps_itself(*x, tokens, d)) return status;
  return b2k::fail(ctx, B2K_EINVAL, "%s: tokens or heads of %s overlap, strides %lld, %lld", what, name,
                   (long long)x->stride_token, (long long)x->stride_head);
}

// An output in an input's (or another output's) place: refused, but for the whole
// of `same`, the input it may replace.
int check_apart(b2k_ctx *ctx, const char *what, const char *name, const b2k_heads &out, const b2k_heads &other, bool same,
                int64_t tokens, int32_t d, int32_t dtype) {
  if (same && out.data == other.data && out.stride_token == other.stride_token && out.stride_head == other.stride_head)
    return B2K_OK;
  if (!overlap(other, out, tokens, d, type_size(dtype))) return B2K_OK;
  return b2k::fail(ctx, B2K_EINVAL, "%s: %s overlaps another operand", what, name);
}

int check_cache(b2k_ctx *ctx, const char *what, const b2k_paged_cache *c) {
  if (!c) return b2k::fail(ctx, B2K_EINVAL, "%s: no cache", what);
  if (!type_ok(c->dtype)) return b2k::fail(ctx, B2K_EINVAL, "%s: unknown element type %d", what, c->dtype);
  if (c->page_size < 1 || c->pages < 1 || c->heads < 1 || c->heads > 65535)
    return b2k::fail(ctx, B2K_EINVAL, "%s: a cache of %lld pages of %d tokens, %d heads", what, (long long)c->pages,
                     c->page_size, c->heads);
  if (c->d < 1 || c->d > B2K_MAX_HEAD_DIM) return b2k::fail(ctx, B2K_EINVAL, "%s: head dim %d", what, c->d);
  if (!c->k || !c->v) return b2k::fail(ctx, B2K_EINVAL, "%s: null cache", what);
  if (!on_boundary(c->k, type_size(c->dtype)) || !on_boundary(c->v, type_size(c->dtype)))
    return b2k::fail(ctx, B2K_EINVAL, "%s: the cache is off its elements' boundary", what);
  if (c->k_page < c->d || c->k_row < c->d || c->k_head < c->d || c->v_page < c->d || c->v_row < c->d ||
      c->v_head < c->d)
    return b2k::fail(ctx, B2K_EINVAL, "%s: a cache stride is below the head dim", what);
  return B2K_OK;
}

int check_batch(b2k_ctx *ctx, const char *what, const b2k_paged_cache *c, const b2k_paged_batch *b) {
  if (!b) return b2k::fail(ctx, B2K_EINVAL, "%s: no batch", what);
  if (b->sequences < 0 || b->tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->prefix_len < 0 || b->table_width < 0)
    return b2k::fail(ctx, B2K_EINVAL, "%s: negative extent", what);
  if (b->tokens > INT32_MAX) return b2k::fail(ctx, B2K_EINVAL, "%s: too many tokens", what);
  if (b->sequences == 0) return B2K_OK;
  if (!b->first || !b->lengths) return b2k::fail(ctx, B2K_EINVAL, "%s: null first or lengths", what);
  if (b->max_len > 0 && (!b->table || b->table_width < 1)) return b2k::fail(ctx, B2K_EINVAL, "%s: no page table", what);
  if (b->table_stride < b->table_width) return b2k::fail(ctx, B2K_EINVAL, "%s: table stride below its width", what);
  if (b->max_len > (int64_t)b->table_width * c->page_size)
    return b2k::fail(ctx, B2K_EINVAL, "%s: max_len %d is beyond the table's %d pages of %d", what, b->max_len,
                     b->table_width, c->page_size);
  if (!on_boundary(b->first, 4) || !on_boundary(b->lengths, 4) || !on_boundary(b->table, 4) ||
      !on_boundary(b->prefix_table, 4))
    return b2k::fail(ctx, B2K_EINVAL, "%s: first, lengths or a table is off 4 bytes", what);
  if (b->prefix_len > 0 && !b->prefix_table) return b2k::fail(ctx, B2K_EINVAL, "%s: no prefix table", what);
  return B2K_OK;
}

}  // namespace serve

extern "C" {

int b2k_rope_plan(const b2k_rope_params *p, b2k_rope *out) {
  if (!p || !out) return B2K_EINVAL;
  const int r = p->rot;
  const bool ramp = p->scaling == B2K_ROPE_RAMP || p->scaling == B2K_ROPE_LOG_RAMP;
  if (r < 2 || r > 2 * kMaxPairs || r % 2 || p->scaling < B2K_ROPE_NONE || p->scaling > B2K_ROPE_LOG_RAMP)
    return B2K_EINVAL;
  if (!(p->theta > 0) || !isfinite(p->theta) || !isfinite(p->magnitude)) return B2K_EINVAL;
  if (p->scaling != B2K_ROPE_NONE && (!(p->factor > 0) || !isfinite(p->factor))) return B2K_EINVAL;
  if (p->scaling == B2K_ROPE_BASE && r == 2) return B2K_EINVAL;
  if (ramp && (!(p->context > 0) || !isfinite(p->context) || !(p->low < p->high) || !isfinite(p->low) ||
               !isfinite(p->high) || (p->scaling == B2K_ROPE_LOG_RAMP && !(p->low > 0))))
    return B2K_EINVAL;
  // long double: 64 significant bits on this platform.  A power f = theta^-e
  // is off by f (|ln f| + 2) 2^-64 (its exponent's rounding, its own), the turn
  // by another two roundings and the last one to 2^-64: below 2^-63 for f <= 1,
  // and with the scalings' sums and quotients below 2^-62.
  const long double two_pi = 2.0L * acosl(-1.0L);
  const long double s = p->factor;
  long double theta = p->theta;
  if (p->scaling == B2K_ROPE_BASE) theta *= powl(s, (long double)r / (r - 2));
  b2k_rope rope = {};
  for (int i = 0; i < r / 2; ++i) {
    long double f = powl(theta, -2.0L * i / r);
    if (p->scaling == B2K_ROPE_LINEAR) f /= s;
    if (ramp) {
      const long double t = p->context * f / two_pi;
      long double w = p->scaling == B2K_ROPE_RAMP
                          ? (t - p->low) / ((long double)p->high - p->low)
                          : (logl(t) - logl(p->low)) / (logl(p->high) - logl(p->low));
      w = std::min(1.0L, std::max(0.0L, w));
      f = f * w + f * (1.0L - w) / s;
    }
    const long double turns = f / two_pi;
    if (!isfinite(turns)) return B2K_EINVAL;
    // the fraction of a turn, in units of 2^-64; 1 - 2^-65 and above is a whole turn
    const long double units = ldexpl(turns - floorl(turns), 64);
    rope.turn[i] = units >= 18446744073709551615.5L ? 0 : (uint64_t)(units + 0.5L);
  }
  rope.rot = r;
  rope.interleaved = p->interleaved != 0;
  rope.magnitude = (float)p->magnitude;
  *out = rope;
  return B2K_OK;
}

int b2k_heads_overlap(const b2k_heads *x, const b2k_heads *y, int64_t tokens, int32_t d, int32_t dtype) {
  if (!x || tokens < 0 || d < 1 || !serve::type_ok(dtype)) return -1;
  for (const b2k_heads *t : {x, y})
    if (t && (t->heads < 1 || t->stride_token < 0 || t->stride_head < 0)) return -1;
  const bool met = y ? serve::overlap(*x, *y, tokens, d, serve::type_size(dtype)) : serve::overlaps_itself(*x, tokens, d);
  return met ? 1 : 0;
}

int64_t b2k_paged_slot(const int32_t *table_row, int32_t table_width, int64_t pages, int32_t page_size,
                       int64_t position) {
  if (!table_row || table_width < 0 || page_size < 1) return -1;
  const int64_t page = serve::page_of(table_row, table_width, pages, page_size, position);
  return page < 0 ? -1 : page * page_size + position % page_size;
}

int b2k_rotary(b2k_ctx *ctx, const b2k_rope *rope, int32_t dtype, int32_t count, const b2k_heads *x,
               const b2k_heads *y, const int64_t *positions, int64_t tokens, int32_t d, int32_t transpose,
               void *stream) {
  B2K_CHECK_CTX(ctx);
  if (!rope || !x || !y) return b2k::fail(ctx, B2K_EINVAL, "rotary: null argument");
  if (!serve::type_ok(dtype)) return b2k::fail(ctx, B2K_EINVAL, "rotary: unknown element type %d", dtype);
  if (count < 1 || count > 3) return b2k::fail(ctx, B2K_EINVAL, "rotary: %d tensors", count);
  if (tokens < 0 || d < 1 || d > B2K_MAX_HEAD_DIM || (transpose != 0 && transpose != 1))
    return b2k::fail(ctx, B2K_EINVAL, "rotary: %lld tokens of head dim %d, transpose %d", (long long)tokens, d, transpose);
  RotaryArgs a = {};
  int status = use_rope(ctx, "rotary", rope, d, transpose, a);
  if (status != B2K_OK) return status;
  const int64_t size = (int64_t)serve::type_size(dtype);
  for (int i = 0; i < count; ++i) {
    if ((status = serve::check_heads(ctx, "rotary", "input", &x[i], tokens, d, dtype)) != B2K_OK) return status;
    if ((status = serve::check_output(ctx, "rotary", "output", &y[i], tokens, d, dtype)) != B2K_OK) return status;
    if (x[i].heads != y[i].heads)
      return b2k::fail(ctx, B2K_EINVAL, "rotary: tensor %d has %d heads in and %d out", i, x[i].heads, y[i].heads);
    if (x[i].data == y[i].data && (x[i].stride_token != y[i].stride_token || x[i].stride_head != y[i].stride_head))
      return b2k::fail(ctx, B2K_EINVAL, "rotary: tensor %d is rotated in place with other strides", i);
    a.seg[i] = {static_cast<const char *>(x[i].data), static_cast<char *>(y[i].data), x[i].stride_token * size,
                x[i].stride_head * size, 0, y[i].stride_token * size, y[i].stride_head * size, x[i].heads, kLinear, 1};
    a.heads += x[i].heads;
  }
  for (int i = 0; i < count; ++i)
    for (int j = 0; j < count; ++j) {
      status = serve::check_apart(ctx, "rotary", "an output", y[i], x[j], i == j, tokens, d, dtype);
      if (status == B2K_OK && j < i) status = serve::check_apart(ctx, "rotary", "an output", y[i], y[j], false, tokens, d, dtype);
      if (status != B2K_OK) return status;
    }
  if (tokens == 0) return B2K_OK;
  if (!positions || !serve::on_boundary(positions, 8))
    return b2k::fail(ctx, B2K_EINVAL, "rotary: positions are null or off 8 bytes");
  a.d = d;
  a.tokens = tokens;
  a.positions = positions;
  return run<false>(ctx, a, count, dtype, tokens, 1, B2K_PHASE_ROTARY, (cudaStream_t)stream, "rotary launch");
}

int b2k_paged_append(b2k_ctx *ctx, const b2k_rope *rope, const b2k_paged_cache *cache, const b2k_paged_batch *batch,
                     const b2k_heads *k, const b2k_heads *v, const b2k_heads *q, const b2k_heads *q_out,
                     void *stream) {
  B2K_CHECK_CTX(ctx);
  const char *what = "paged_append";
  int status = serve::check_cache(ctx, what, cache);
  if (status == B2K_OK) status = serve::check_batch(ctx, what, cache, batch);
  if (status == B2K_OK) status = serve::check_heads(ctx, what, "k", k, batch->tokens, cache->d, cache->dtype);
  if (status == B2K_OK) status = serve::check_heads(ctx, what, "v", v, batch->tokens, cache->d, cache->dtype);
  if (status != B2K_OK) return status;
  if (k->heads != cache->heads || v->heads != cache->heads)
    return b2k::fail(ctx, B2K_EINVAL, "%s: %d key and %d value heads for a cache of %d", what, k->heads, v->heads,
                     cache->heads);
  if (rope && cache->k == cache->v)  // (read for both, by attention, they may be one)
    return b2k::fail(ctx, B2K_EINVAL, "%s: rotated keys and values in one place", what);
  if (!q != !q_out || (q && !rope)) return b2k::fail(ctx, B2K_EINVAL, "%s: q needs q_out and a rope", what);
  RotaryArgs a = {};
  a.d = cache->d;
  if (rope && (status = use_rope(ctx, what, rope, cache->d, 0, a)) != B2K_OK) return status;
  if (!rope) a.rot = 0, a.interleaved = 1;  // nothing turns: plain copies of neighbouring vectors
  const int64_t size = (int64_t)serve::type_size(cache->dtype);
  int count = 0;
  if (q) {
    if ((status = serve::check_heads(ctx, what, "q", q, batch->tokens, cache->d, cache->dtype)) != B2K_OK) return status;
    if ((status = serve::check_output(ctx, what, "q_out", q_out, batch->tokens, cache->d, cache->dtype)) != B2K_OK) return status;
    if (q->heads != q_out->heads ||
        (q->data == q_out->data && (q->stride_token != q_out->stride_token || q->stride_head != q_out->stride_head)))
      return b2k::fail(ctx, B2K_EINVAL, "%s: q and q_out differ in heads, or in strides in place", what);
    for (const b2k_heads *in : {q, k, v})
      if ((status = serve::check_apart(ctx, what, "q_out", *q_out, *in, in == q, batch->tokens, cache->d, cache->dtype)) != B2K_OK)
        return status;
    a.seg[count++] = {static_cast<const char *>(q->data), static_cast<char *>(q_out->data), q->stride_token * size,
                      q->stride_head * size, 0, q_out->stride_token * size, q_out->stride_head * size, q->heads, kLinear, 1};
    a.heads += q->heads;
  }
  a.seg[count++] = {static_cast<const char *>(k->data), static_cast<char *>(cache->k), k->stride_token * size,
                    k->stride_head * size, cache->k_page * size, cache->k_row * size, cache->k_head * size, k->heads,
                    kKeys, rope != nullptr};
  a.heads += k->heads;
  a.seg[count++] = {static_cast<const char *>(v->data), static_cast<char *>(cache->v), v->stride_token * size,
                    v->stride_head * size, cache->v_page * size, cache->v_row * size, cache->v_head * size, v->heads,
                    kValues, 0};
  a.heads += v->heads;
  if (batch->sequences == 0 || batch->tokens == 0 || batch->max_new == 0) return B2K_OK;
  a.tokens = batch->tokens;
  a.first = batch->first;
  a.lengths = batch->lengths;
  a.table = batch->table;
  a.table_stride = batch->table_stride;
  a.table_width = batch->table_width;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  a.prefix_len = batch->prefix_len;
  a.max_new = batch->max_new;
  a.max_len = batch->max_len;
  a.err = ctx->error_flag;
  return run<true>(ctx, a, count, cache->dtype, batch->max_new, (unsigned)batch->sequences, B2K_PHASE_APPEND,
                   (cudaStream_t)stream, "paged_append launch");
}

}  // extern "C"
