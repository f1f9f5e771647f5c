// Attention over a paged cache for f16 and bf16, many rows a cache head and head
// dims of 136 to 256: the tensor-memory kernel (paged_umma.cu) for heads whose
// output fills half of the tensor memory.
//
// One block per SM holds one tile of 128 rows.  With one output of 256 columns
// there is room for two score buffers, so the tensor core computes S_{j+1} while
// the softmax works on S_j -- the other tile's part in the narrower kernel:
//
//   warps 0-3  softmax, one thread a row: S_j from its buffer, running maximum, P_j
//              back into the same columns; at the end the rows' output
//   warp 4     loads by TMA, in units of 128 keys by 128 dims (32 KB), five in a
//              ring: K_0, then K_{j+1}, V_j for each j, two units each; queries
//              as boxes of tokens by heads, or by the softmax warps where a cache
//              head's query heads do not divide 128
//   warp 5     MMA issuer: S_0, then for each j S_{j+1} and O += P_j V_j
//
// Softmax, bases of the exponents and marks of missing keys are the narrower
// kernel's.  Bound: the tensor core, 2048 cycles a tile at head dim 256 against
// about 1900 of the softmax.  All mbarrier waits are bounded (sm100.cuh).
#include "paged_umma.cuh"

namespace {

using namespace umma;

constexpr int kSoftmaxWarps = 4;
constexpr int kThreads = 32 * (kSoftmaxWarps + 2);
constexpr int kUnit = 2 * kHalf;  // bytes of 128 keys (or rows) by 128 dims
constexpr int kUnits = 5;
constexpr int kSmem = 2 * kUnit + kUnits * kUnit;  // queries, ring
constexpr uint32_t kColO = 256;   // S (then P) of even and odd tiles: columns 0, 128; O: 256 columns

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    paged_umma_wide_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const __grid_constant__ CUtensorMap map_q, const __grid_constant__ Args a, const bool prefix,
                           const int row_blocks, const bool q_boxes) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kUnits], empty[kUnits], q_full, s_full[2], p_full[2][2], pv_done, drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ uint32_t marks[kMarks][4];  // keys of a tile that are there

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort = &abort_word;
  if (threadIdx.x == 0) {
    // swizzled tiles need 1024-byte alignment: refuse to run (error word, no
    // work) rather than compute garbage
    abort_word = (sm100::smem_addr(smem) & 1023u) ? 1 : 0;
    if (abort_word) atomicOr(a.err, sm100::kSiteAttention);
    for (int i = 0; i < kUnits; ++i) {
      sm100::mbar_init(&full[i], 1);
      sm100::mbar_init(&empty[i], 1);
    }
    sm100::mbar_init(&q_full, q_boxes ? 1 : kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&s_full[i], 1);
      // P's first 64 keys, the others; of even and odd tiles apart, since a softmax
      // warp may be through with S_{j+1} before another has released P_j
      sm100::mbar_init(&p_full[i][0], kSoftmaxWarps);
      sm100::mbar_init(&p_full[i][1], kSoftmaxWarps);
    }
    sm100::mbar_init(&pv_done, 1);
    sm100::mbar_init(&drain, 1);
    sm100::fence_barrier_init();
  }
  if (threadIdx.x == 32 * kSoftmaxWarps) {
    sm100::prefetch_tensormap(&map_k);
    sm100::prefetch_tensormap(&map_v);
  }
  if (warp == kSoftmaxWarps + 1) sm100::tmem_alloc(&tmem_slot, 512);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  paged::part_begin(a, false);

  // --- this block's rows and keys ------------------------------------------------
  unsigned at = blockIdx.x;
  const int block = row_blocks - 1 - at % row_blocks;  // the longest of a causal part first
  at /= row_blocks;
  const int head = at % a.kv_heads;
  at /= a.kv_heads;
  const int splits = prefix ? a.prefix_splits : a.own_splits;
  const int split = at % splits;
  int b = at / splits;
  paged::Sequence s = {0, 0, 0};
  if (prefix) s.n = paged::used_tokens(a);
  else s = paged::sequence_by_length(a, b);  // the longest first: the last to start are short
  const int rows = s.n * a.group, row0 = block * kRows;
  const int chunk = prefix ? a.prefix_chunk : a.own_chunk;
  const int key0 = split * chunk;
  int key_end = key0;
  if (row0 < rows) {
    const int last = (min(row0 + kRows, rows) - 1) / a.group;
    key_end = max(key0, paged::split_end(key0, chunk, prefix ? a.prefix_len : paged::own_limit(a, s, last)));
  }
  const int tiles = (key_end - key0 + kKeys - 1) / kKeys;
  const bool direct = a.own_splits + a.prefix_splits == 1;
  const bool work = row0 < rows && (tiles > 0 || (direct && key0 == 0));
  const int tile0 = key0 / kKeys;                                         // of the part
  const int prefix_tiles = !prefix && a.joined ? a.joined_keys / kKeys : 0;  // of those, the prefix's
  auto valid = [&](int j) {  // keys of the block's tile j
    const int key = key0 + j * kKeys;
    return min(kKeys, (tile0 + j < prefix_tiles ? min(key_end, a.prefix_len) : key_end) - key);
  };
  uint8_t *const qs = smem, *const ring = smem + 2 * kUnit;

  if (work && warp == kSoftmaxWarps) {
    // ---------------- loads: lane i a tile's i-th box
    const int box = min(a.page_size, kKeys), boxes = kKeys / box;
    const int32_t *own_table = a.table + (int64_t)b * a.table_stride;
    auto is_prefix = [&](int j) { return prefix || tile0 + j < prefix_tiles; };
    auto key_of = [&](int j) { return (tile0 + j - (is_prefix(j) ? 0 : prefix_tiles)) * kKeys + lane * box; };
    auto wanted = [&](int j) { return j < tiles && lane < boxes && lane * box < valid(j); };
    auto look_up = [&](int j) {  // page of this lane's box, -1 behind the last key
      return wanted(j) ? (is_prefix(j) ? a.prefix_table : own_table)[(unsigned)key_of(j) / (unsigned)a.page_size] : -1;
    };
    bool ok = true;
    if (q_boxes && lane == 0 && tiles > 0) {
      sm100::mbar_arrive_expect_tx(&q_full, 2 * kUnit);
      for (int c = 0; c < 4; ++c)
        sm100::tma_load_3d(qs + c * kHalf, &map_q, &q_full, 64 * c, head * a.group, s.first + row0 / a.group);
    }
    __syncwarp();
    int n = 0;  // units issued
    auto load = [&](const CUtensorMap *map, int j, int page) {
      const int row = (int)((unsigned)key_of(j) % (unsigned)a.page_size);
      for (int half = 0; ok && half < 2; ++half, ++n) {
        const int unit = n % kUnits;
        if (n >= kUnits)
          ok = sm100::mbar_wait_warp(&empty[unit], ((n / kUnits) - 1) & 1, a.err, sm100::kSiteProducerEmpty, abort);
        if (!ok) break;
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive_expect_tx(&full[unit], kUnit);
        __syncwarp();
        if (lane < boxes) {
          const uint32_t to = sm100::smem_addr(ring + unit * kUnit) + lane * box * 128;
#pragma unroll
          for (int c = 0; c < 2; ++c)
            tma_load_4d(to + c * kHalf, map, &full[unit], 128 * half + 64 * c, row, head, page);
        }
      }
    };
    auto mark = [&](int j, int page) {  // checks the page; the page to load, and the keys that are there
      const bool there = wanted(j) && page >= 0 && page < a.pages;
      if (wanted(j) && !there) atomicOr(a.err, serve::kErrIndex);
      const uint32_t have = __ballot_sync(0xffffffffu, there);
      if (lane < 4) {
        uint32_t m = 0;
        for (int i = 0; i < 32; i += min(box, 32))
          if ((have >> ((32 * lane + i) / box)) & 1u) m |= (box >= 32 ? 0xffffffffu : ((1u << box) - 1u) << i);
        marks[j % kMarks][lane] = m;
      }
      return there ? page : -1;
    };
    int next = tiles > 0 ? mark(0, look_up(0)) : -1;
    if (tiles > 0) load(&map_k, 0, next);
    for (int j = 0; ok && j < tiles; ++j) {
      const int page = next;
      const int asked = look_up(j + 1);
      if (j + 1 < tiles) {
        next = mark(j + 1, asked);
        load(&map_k, j + 1, next);
      }
      if (ok) load(&map_v, j, page);
    }
    // loads in flight must land before the block leaves (budget only)
    int never = 0;
    if (!ok)
      for (int i = 0; i < kUnits; ++i) sm100::mbar_wait(&full[i], 0, a.err, sm100::kSiteDrain, &never, 1000000);
  } else if (work && warp == kSoftmaxWarps + 1) {
    // ---------------- MMA issuer
    const uint32_t id_s = idesc<T>(kKeys, false), id_o = idesc<T>(kKeys, true);
    const uint32_t q_addr = sm100::smem_addr(qs);
    bool ok = tiles == 0 || sm100::mbar_wait_warp(&q_full, 0, a.err, sm100::kSiteMmaFull, abort);
    int n = 0;  // units consumed
    auto wait_unit = [&]() {
      ok = ok && sm100::mbar_wait_warp(&full[n % kUnits], (n / kUnits) & 1, a.err, sm100::kSiteMmaFull, abort);
      sm100::tc_fence_after();
      return sm100::smem_addr(ring + (n % kUnits) * kUnit);
    };
    auto issue_s = [&](int j) {
      for (int half = 0; half < 2; ++half) {
        const uint32_t k = wait_unit();
        if (!ok) return;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          mma4_ss(tmem + (j & 1) * 128, sm100::desc_kmajor<128>(q_addr + (2 * half + c) * kHalf),
                  sm100::desc_kmajor<128>(k + c * kHalf), id_s, half != 0 || c != 0);
        sm100::mma_commit(&empty[n % kUnits]);
        ++n;
      }
      sm100::mma_commit(&s_full[j & 1]);
    };
    if (ok && tiles > 0) issue_s(0);
    for (int j = 0; ok && j < tiles; ++j) {
      // S_{j+1} takes the buffer that P_{j-1} was in; its product was issued before
      if (j + 1 < tiles) issue_s(j + 1);
      const uint32_t p = tmem + (j & 1) * 128;
      for (int half = 0; ok && half < 2; ++half) {  // 128 dims of V
        const uint32_t v = wait_unit();
        if (ok && valid(j) < kKeys) {
          // the values behind the last key (of the prefix, or of all) become
          // zeros: a page's unused rows may hold anything, and 0 x NaN is NaN
          uint8_t *vs = ring + (n % kUnits) * kUnit;
          for (int i = 8 * valid(j) + lane; i < 8 * kKeys; i += 32)
#pragma unroll
            for (int c = 0; c < 2; ++c) *reinterpret_cast<uint4 *>(vs + c * kHalf + 16 * i) = make_uint4(0, 0, 0, 0);
          sm100::fence_proxy_async_smem();
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 64 keys
          if (half == 0) {
            ok = ok && sm100::mbar_wait_warp(&p_full[j & 1][h], (j >> 1) & 1, a.err, sm100::kSiteMmaFull, abort);
            sm100::tc_fence_after();
          }
          if (ok) mma4_ts(tmem + kColO + half * 128, p + h * 32, desc_mn(v + h * 8192, kHalf, 1024), id_o, j != 0 || h != 0);
        }
        if (ok) sm100::mma_commit(&empty[n % kUnits]);
        ++n;
      }
      if (ok) sm100::mma_commit(&pv_done);
    }
    sm100::mma_commit(&drain);
    int never = 0;
    sm100::mbar_wait(&drain, 0, a.err, sm100::kSiteDrain, &never);
  } else if (work && warp < kSoftmaxWarps) {
    // ---------------- softmax, one thread a row
    const int r = threadIdx.x;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    if (!q_boxes) {
      // queries into shared memory, 16 bytes at a time, eight loads in flight
      constexpr int kPieces = 32, kBatch = 8;
      for (int i0 = threadIdx.x; i0 < kRows * kPieces; i0 += kBatch * kRows) {
        uint4 v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kRows, qr = i / kPieces, c = i % kPieces, row = row0 + qr;
          v[u] = make_uint4(0, 0, 0, 0);
          if (row < rows && c * 8 < a.d) {
            const int j = row / a.group;
            v[u] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (int64_t)(s.first + j) * a.q_token +
                                                    (int64_t)(head * a.group + row - j * a.group) * a.q_head + c * 8);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kRows, qr = i / kPieces, c = i % kPieces;
          *reinterpret_cast<uint4 *>(qs + (c >> 3) * kHalf + qr * 128 + (((c & 7) ^ (qr & 7)) << 4)) = v[u];
        }
      }
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&q_full);
    }
    const int row = row0 + r;
    const int j_row = row / a.group;
    const int limit = row >= rows ? 0 : min(prefix ? a.prefix_len : paged::own_limit(a, s, j_row), key_end);
    int free_end = limit;  // keys below this are seen by every row of the warp
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) free_end = min(free_end, __shfl_xor_sync(0xffffffffu, free_end, o));
    const float c = a.scale_log2;
    const uint32_t o_at = tmem + lane_base + kColO;
    float base = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      ok = ok && sm100::mbar_wait_warp(&s_full[j & 1], (j >> 1) & 1, a.err, sm100::kSiteAttention, abort);
      if (!ok) break;
      sm100::tc_fence_after();
      const uint32_t s_at = tmem + lane_base + (j & 1) * 128;
      uint32_t sr[kKeys];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sm100::tmem_ld_32x32b_x32(s_at + 32 * i, *reinterpret_cast<uint32_t(*)[32]>(&sr[32 * i]));
      sm100::tmem_ld_wait();
      const int key = key0 + j * kKeys, part_end = tile0 + j < prefix_tiles ? a.prefix_len : INT32_MAX;
      const uint32_t *mk = marks[j % kMarks];
      const uint32_t m0 = mk[0], m1 = mk[1], m2 = mk[2], m3 = mk[3];
      if (key + kKeys > min(free_end, part_end) || (m0 & m1 & m2 & m3) != 0xffffffffu) {
        const int lim = min(limit, part_end) - key;
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
          const uint32_t word = i < 32 ? m0 : i < 64 ? m1 : i < 96 ? m2 : m3;
          if (i >= lim || !((word >> (i & 31)) & 1u)) sr[i] = __float_as_uint(-INFINITY);
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kKeys; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(sr[i + 2 * e]), __uint_as_float(sr[i + 2 * e + 1]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c - Type<T>::kLift;
      if (__any_sync(0xffffffffu, top > base + Type<T>::kSlack || (base == -INFINITY && top > base))) {
        const float moved = fmaxf(base, top);
        const float alpha = moved == -INFINITY ? 1.0f : exp2_fast(base - moved);
        base = moved;
        l *= alpha;
        if (j > 0) {
          // the product before has to be complete for its sums to be scaled (the one
          // before that is: S_j was committed behind it)
          ok = sm100::mbar_wait_warp(&pv_done, (j - 1) & 1, a.err, sm100::kSiteAttention, abort);
          if (!ok) break;
          sm100::tc_fence_after();
#pragma unroll 4
          for (int i = 0; i < 256; i += 16) {
            uint32_t ov[16];
            sm100::tmem_ld_32x32b_x16(o_at + i, ov);
            sm100::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            sm100::tmem_st_32x32b_x16(o_at + i, ov);
          }
        }
      }
      const float from = base == -INFINITY ? 0.0f : base;
      uint64_t sum[2] = {0, 0};
      const uint64_t c2 = pair(c, c), from2 = pair(-from, -from);
      auto release = [&](int h) {  // the product of these keys may begin
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[j & 1][h]);
      };
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float p0, p1;
          unpair(fma2(pair(__uint_as_float(sr[32 * h + i]), __uint_as_float(sr[32 * h + i + 1])), c2, from2), p0, p1);
          p0 = exp2_fast(p0);
          p1 = exp2_fast(p1);
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pair(p0, p1));
          pk[i / 2] = Type<T>::pack(p0, p1);
        }
        if (h == 2) release(0);  // its stores have landed meanwhile
        sm100::tmem_st_32x32b_x16(s_at + 16 * h, pk);
      }
      release(1);
      float l0, l1;
      unpair(add2(sum[0], sum[1]), l0, l1);
      l += l0 + l1;
    }
    // ---------------- the row's output
    // the last two products, one after the other: with neither done, the
    // barrier's parity is that of the phase before both
    if (tiles > 0 || !q_boxes) ok = ok && sm100::mbar_wait_warp(&q_full, 0, a.err, sm100::kSiteEpilogueAccum, abort);
    for (int j = max(0, tiles - 2); j < tiles; ++j)
      ok = ok && sm100::mbar_wait_warp(&pv_done, j & 1, a.err, sm100::kSiteEpilogueAccum, abort);
    if (ok) {
      sm100::tc_fence_after();
      const int q_heads = a.kv_heads * a.group;
      const int64_t token = s.first + j_row;
      const int qh = head * a.group + row - j_row * a.group;
      const bool on = row < rows, some = l != 0.0f && tiles > 0;  // (NaN too)
      const float inv = !direct ? 1.0f : some ? 1.0f / l : 0.0f;
      const int64_t part = (int64_t)(prefix ? a.own_splits + split : split) * a.tokens * q_heads + token * q_heads + qh;
      // rows of a split that see none of its keys are not read by the merge
      if (!direct && on) a.part_ml[part] = make_float2(base, l);
      // (the queries' place in shared memory is free: the products with them are
      // complete, and all of them have arrived)
      uint8_t *const stage = qs + warp * 4096;
      if (direct)
        store_output<T>(stage, static_cast<T *>(a.o), on ? token * a.o_token + (int64_t)qh * a.o_head : -1, a.d, o_at, tiles > 0, some, inv);
      else
        store_sums(stage, a.part_o, on ? part * a.d : -1, a.d, o_at, tiles > 0, some);
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == kSoftmaxWarps + 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 512);
  }
}

template <typename T>
int launch(b2k_ctx *ctx, const Args &a, bool prefix, int row_blocks, unsigned blocks, cudaStream_t s) {
  auto kernel = paged_umma_wide_kernel<T>;
  CUtensorMap map_k = {}, map_v = {}, map_q = {};
  const bool q_boxes = query_boxes_fit(a);
  int status = make_map<T>(ctx, &map_k, a, true);
  if (status == B2K_OK) status = make_map<T>(ctx, &map_v, a, false);
  if (q_boxes && status == B2K_OK) status = make_q_map<T>(ctx, &map_q, a);
  if (status != B2K_OK) return status;
  cudaError_t err = b2k::set_max_smem(ctx, (const void *)kernel, kSmem);
  if (err == cudaSuccess)
    err = b2k::launch_kernel(a.pdl, kernel, dim3(blocks), dim3(kThreads), kSmem, s, map_k, map_v, map_q, a, prefix,
                             row_blocks, q_boxes);
  return err == cudaSuccess ? B2K_OK : b2k::cuda_fail(ctx, err, "paged_attention launch");
}

}  // namespace

namespace paged {

int umma_wide_part(b2k_ctx *ctx, const Args &a, int32_t dtype, bool prefix, int row_blocks, unsigned blocks, cudaStream_t s) {
  return dtype == B2K_F16 ? launch<__half>(ctx, a, prefix, row_blocks, blocks, s)
                          : launch<__nv_bfloat16>(ctx, a, prefix, row_blocks, blocks, s);
}

}  // namespace paged
