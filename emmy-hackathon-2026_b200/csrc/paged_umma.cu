// Attention over a paged cache for f16 and bf16 operands and many rows a cache
// head -- the shared prefix under the stacked rows of a batch, prompt chunks --
// on the 5th-generation tensor cores.
//
// One block per SM holds two tiles of 128 rows (A and B), so keys and values
// are read once for 256 rows, and the tensor core works on one tile while the
// softmax works on the other:
//
//   warps 0-3   softmax of tile A, one thread a row: S_j from tensor memory,
//   warps 4-7   (tile B the same) running maximum, P_j back into S_j's columns
//               in the operands' type, where the second product reads it;
//               at the end the rows' output
//   warp 8      loads: keys and values into 128-byte-swizzled tiles of 128 keys, in
//               the order K_0, V_0, K_1, V_1 ... through one ring, by TMA boxes
//               of a page (or 128 rows of one); pages outside the cache are
//               outside the tensor map and arrive as zeros.  Queries the same way,
//               as boxes of tokens by heads, where a cache head's query heads
//               divide 128 (row by row by the softmax warps they take 8000
//               cycles of a block's start)
//   warp 10     MMA issuer: S_j = Q K_j^T (128 x 128), then O += P_j V_j with P
//               from tensor memory and V as it lies (N-major), in the order O_A,
//               S_A, O_B, S_B: while one tile has the tensor core the other is in
//               its softmax (an issuer for each tile lets the two fall into step,
//               and each then waits for both: 3 to 5 % slower)
//   (pages that no box fits -- sizes that neither divide 128 nor are a multiple of
//               it, or below 8 -- are copied row by row by warps 8 and 9, 16 bytes a
//               lane; warp 11 passes on what has landed, since the tensor core sees
//               such copies behind a proxy fence alone.  Those copies' issue bounds the kernel then: 7000
//               cycles a pair of tiles)
//
// Mathematics: O stays in tensor memory over all tiles.  The exponents' base is
// the running maximum of the time when it was last moved: it moves only when a
// row's maximum has risen by more than 2^kSlack over it, and then the row's sums
// in tensor memory are scaled (a rare step after the first tiles).  Until
// then probabilities may exceed one; FP32 sums and the operands' range carry
// 2^kSlack.  f16 probabilities are lifted by 2^kLift, so that small ones keep
// their bits.
//
// Bound: tensor core and exponentials alike: a pair of 128 x 128 tiles takes
// 2 x 1024 tensor cycles at head dim 128 and 2 x 1024 of the special-function unit.
// It takes 3430, each tile's own chain of steps: scores seen 850 cycles after
// their products are issued, maximum 620 later, 128 exponentials a row 1800 (the
// other tile's beside them), the last products 350 after that.  5 prompt chunks
// of up to 1024 tokens over 1211 to 3500 keys and 1111 shared ones, 32 / 8 heads:
// 233 us, 766 TFLOP/s.
// All mbarrier waits are bounded (sm100.cuh).
#include "paged_umma.cuh"

namespace {

using namespace umma;

constexpr int kSoftmaxWarps = 8, kLoadWarps = 2;
constexpr int kThreads = 32 * (kSoftmaxWarps + kLoadWarps + 2);

template <int DP>
constexpr int tile_bytes() { return kHalf * (DP / 64); }
template <int DP>
constexpr int stages() { return DP == 64 ? 8 : 5; }
template <int DP>
constexpr int smem_bytes() { return 2 * tile_bytes<DP>() + stages<DP>() * tile_bytes<DP>(); }

// Tensor-memory columns.
constexpr uint32_t kColS = 0, kColO = 256;  // S (then P) of tile A, B: 128 each; O of A, B: 128 each

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on) {
  const int bytes = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrive on `bar` once every copy of this thread so far has landed.
__device__ __forceinline__ void copy_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sm100::smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <typename T, int DP, bool TMA>
__global__ void __launch_bounds__(kThreads, 1)
    paged_umma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CUtensorMap map_q, const __grid_constant__ Args a, const bool prefix,
                      const int row_blocks, const bool q_boxes) {
  constexpr int kStages = stages<DP>();
  constexpr int kTile = tile_bytes<DP>();
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t landed[kStages], full[kStages], empty[kStages], q_full, s_full[2], p_full[2][2], o_full[2], drain;
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
    for (int i = 0; i < kStages; ++i) {
      sm100::mbar_init(&landed[i], 32 * kLoadWarps);
      sm100::mbar_init(&full[i], 1);  // TMA: the bytes; else warp 11
      sm100::mbar_init(&empty[i], 1);
    }
    sm100::mbar_init(&q_full, q_boxes ? 1 : kSoftmaxWarps);
    sm100::mbar_init(&drain, 1);
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&s_full[i], 1);
      sm100::mbar_init(&p_full[i][0], 4);  // P's first 64 keys, the others
      sm100::mbar_init(&p_full[i][1], 4);
      sm100::mbar_init(&o_full[i], 1);
    }
    sm100::fence_barrier_init();
  }
  if (TMA && threadIdx.x == 32 * kSoftmaxWarps) {
    sm100::prefetch_tensormap(&map_k);
    sm100::prefetch_tensormap(&map_v);
    if (q_boxes) sm100::prefetch_tensormap(&map_q);
  }
  if (warp == kSoftmaxWarps + kLoadWarps) sm100::tmem_alloc(&tmem_slot, 512);
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
  const int rows = s.n * a.group, row0 = block * 2 * kRows;
  const int chunk = prefix ? a.prefix_chunk : a.own_chunk;
  const int key0 = split * chunk;
  // keys of a tile's rows [first, first + 128): up to its last row's
  auto keys_of = [&](int first) {
    if (first >= rows) return 0;
    const int last = (min(first + kRows, rows) - 1) / a.group;
    return max(0, paged::split_end(key0, chunk, prefix ? a.prefix_len : paged::own_limit(a, s, last)) - key0);
  };
  const int keys_a = keys_of(row0), keys_b = keys_of(row0 + kRows);
  const int tiles_a = (keys_a + kKeys - 1) / kKeys, tiles_b = (keys_b + kKeys - 1) / kKeys;
  const int key_end = key0 + max(keys_a, keys_b), tiles = max(tiles_a, tiles_b);
  const bool direct = a.own_splits + a.prefix_splits == 1;
  const bool work = row0 < rows && (tiles > 0 || (direct && key0 == 0));

  uint8_t *const qs = smem, *const ring = smem + 2 * kTile;

  const int tile0 = key0 / kKeys;                                         // of the part
  const int prefix_tiles = !prefix && a.joined ? a.joined_keys / kKeys : 0;  // of those, the prefix's
  // keys of the block's tile j
  auto valid = [&](int j) {
    const int key = key0 + j * kKeys;
    return min(kKeys, (tile0 + j < prefix_tiles ? min(key_end, a.prefix_len) : key_end) - key);
  };

  if (TMA && work && warp == kSoftmaxWarps) {
    // ---------------- loads: lane i the tile's i-th box
    const int box = min(a.page_size, kKeys), boxes = kKeys / box;
    const int32_t *own_table = a.table + (int64_t)b * a.table_stride;
    auto look_up = [&](int j) {  // page of this lane's box, -1 behind the last key
      const bool pre = prefix || tile0 + j < prefix_tiles;
      const int key = (tile0 + j - (pre ? 0 : prefix_tiles)) * kKeys + lane * box;
      return lane < boxes && lane * box < valid(j) ? (pre ? a.prefix_table : own_table)[(unsigned)key / (unsigned)a.page_size] : -1;
    };
    bool ok = true;
    if (q_boxes && lane == 0 && tiles > 0) {
      // a tile's rows are whole tokens: 128 / group of them, group heads each
      sm100::mbar_arrive_expect_tx(&q_full, 2 * kTile);
      for (int x = 0; x < 2; ++x)
        for (int half = 0; half < DP / 64; ++half)
          sm100::tma_load_3d(qs + x * kTile + half * kHalf, &map_q, &q_full, 64 * half, head * a.group,
                             s.first + (row0 + x * kRows) / a.group);
    }
    __syncwarp();
    int page = look_up(0);
    for (int j = 0; ok && j < tiles; ++j) {
      const bool pre = prefix || tile0 + j < prefix_tiles;
      const int key = (tile0 + j - (pre ? 0 : prefix_tiles)) * kKeys + lane * box;
      const int row = (int)((unsigned)key % (unsigned)a.page_size);
      const bool wanted = lane < boxes && lane * box < valid(j), there = wanted && page >= 0 && page < a.pages;
      if (wanted && !there) atomicOr(a.err, serve::kErrIndex);
      const uint32_t have = __ballot_sync(0xffffffffu, there);
      if (lane < 4) {
        uint32_t mark = 0;
        for (int i = 0; i < 32; i += min(box, 32))
          if ((have >> ((32 * lane + i) / box)) & 1u) mark |= (box >= 32 ? 0xffffffffu : ((1u << box) - 1u) << i);
        marks[j % kMarks][lane] = mark;
      }
      const int at_page = there ? page : -1;
      if (j + 1 < tiles) page = look_up(j + 1);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int n = 2 * j + kv, stage = n % kStages;
        if (n >= kStages)
          ok = ok && sm100::mbar_wait_warp(&empty[stage], ((n / kStages) - 1) & 1, a.err, sm100::kSiteProducerEmpty, abort);
        if (!ok) break;
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive_expect_tx(&full[stage], kTile);
        __syncwarp();
        if (lane < boxes) {
          const uint32_t to = sm100::smem_addr(ring + stage * kTile) + lane * box * 128;
#pragma unroll
          for (int half = 0; half < DP / 64; ++half)
            tma_load_4d(to + half * kHalf, kv ? &map_v : &map_k, &full[stage], 64 * half, row, head, at_page);
        }
      }
    }
    // loads in flight must land before the block leaves (budget only)
    int never = 0;
    if (!ok)
      for (int i = 0; i < kStages; ++i) sm100::mbar_wait(&full[i], 0, a.err, sm100::kSiteDrain, &never, 1000000);
  } else if (!TMA && work && warp >= kSoftmaxWarps && warp < kSoftmaxWarps + kLoadWarps) {
    // ---------------- loads row by row: warp w takes rows 64 w .. of every tile
    const int w = warp - kSoftmaxWarps;
    const T *kc = static_cast<const T *>(a.k) + (int64_t)head * a.k_head;
    const T *vc = static_cast<const T *>(a.v) + (int64_t)head * a.v_head;
    const int32_t *own_table = a.table + (int64_t)b * a.table_stride;
    // page and row of the two keys this lane looks up (64 w + lane, + 32)
    int page[2], row[2], next_page[2], next_row[2];
    auto look_up = [&](int j, int (&pg)[2], int (&rw)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool pre = prefix || tile0 + j < prefix_tiles;
        const int in = 64 * w + 32 * h + lane, k = (tile0 + j - (pre ? 0 : prefix_tiles)) * kKeys + in;
        pg[h] = -1;
        rw[h] = -1;
        if (in < valid(j)) {
          const int32_t *table = pre ? a.prefix_table : own_table;
          const int i = (int)((unsigned)k / (unsigned)a.page_size);
          rw[h] = k - i * a.page_size;
          pg[h] = table[i];
        }
      }
    };
    int n = 0;
    bool ok = true;
    auto issue = [&](bool keys, int j) {
      const int stage = n % kStages;
      if (n >= kStages)
        ok = __all_sync(0xffffffffu, sm100::mbar_wait(&empty[stage], ((n / kStages) - 1) & 1, a.err,
                                                      sm100::kSiteProducerEmpty, abort));
      if (!ok) return;
      const uint32_t to = sm100::smem_addr(ring + stage * kTile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        bool there = page[h] >= 0 && page[h] < a.pages;
        if (!there && row[h] >= 0) atomicOr(a.err, serve::kErrIndex);
        const int64_t off = !there ? -1 : keys ? page[h] * a.k_page + row[h] * a.k_row : page[h] * a.v_page + row[h] * a.v_row;
        if (keys) {
          const uint32_t mark = __ballot_sync(0xffffffffu, there);
          if (lane == 0) marks[j % kMarks][2 * w + h] = mark;
        }
        const T *from = keys ? kc : vc;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + (lane >> 3);           // row of these 32
          const int64_t o = __shfl_sync(0xffffffffu, off, r);
          const int rr = 64 * w + 32 * h + r;
#pragma unroll
          for (int half = 0; half < DP / 64; ++half) {
            const int c = lane & 7;
            const bool on = o >= 0 && half * 64 + c * 8 < a.d;
            copy16(to + half * kHalf + rr * 128 + ((c ^ (rr & 7)) << 4), from + (on ? o + half * 64 + c * 8 : 0), on);
          }
        }
      }
      copy_arrive(&landed[stage]);
      ++n;
    };
    look_up(0, page, row);
    for (int j = 0; ok && j < tiles; ++j) {
      issue(true, j);
      if (j + 1 < tiles) look_up(j + 1, next_page, next_row);
      if (ok) issue(false, j);
#pragma unroll
      for (int h = 0; h < 2; ++h) page[h] = next_page[h], row[h] = next_row[h];
    }
    copy_wait_all();
  } else if (!TMA && work && warp == kSoftmaxWarps + kLoadWarps + 1) {
    // ---------------- what has landed becomes visible to the tensor core
    bool ok = true;
    for (int i = 0; ok && i < 2 * tiles; ++i) {
      ok = sm100::mbar_wait_warp(&landed[i % kStages], (i / kStages) & 1, a.err, sm100::kSiteConvert, abort);
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (ok && lane == 0) sm100::mbar_arrive(&full[i % kStages]);
    }
  } else if (work && warp == kSoftmaxWarps + kLoadWarps) {
    // ---------------- MMA issuer
    const uint32_t id_s = idesc<T>(kKeys, false), id_o = idesc<T>(DP, true);
    const uint32_t q_addr = sm100::smem_addr(qs);
    bool ok = tiles == 0 || sm100::mbar_wait_warp(&q_full, 0, a.err, sm100::kSiteMmaFull, abort);
    auto wait_item = [&](int i) {  // K_j is item 2 j, V_j 2 j + 1
      ok = ok && sm100::mbar_wait_warp(&full[i % kStages], (i / kStages) & 1, a.err, sm100::kSiteMmaFull, abort);
      sm100::tc_fence_after();
    };
    auto item_addr = [&](int i) { return sm100::smem_addr(ring + (i % kStages) * kTile); };
    auto issue_s = [&](int x, int j) {
      const uint32_t k = item_addr(2 * j), q = q_addr + x * kTile, d = tmem + kColS + x * 128;
#pragma unroll
      for (int half = 0; half < DP / 64; ++half)
        mma4_ss(d, sm100::desc_kmajor<128>(q + half * kHalf), sm100::desc_kmajor<128>(k + half * kHalf), id_s, half != 0);
      sm100::mma_commit(&s_full[x]);
    };
    auto issue_o = [&](int x, int j, bool last) {
      const uint32_t v = item_addr(2 * j + 1), p = tmem + kColS + x * 128, d = tmem + kColO + x * 128;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        ok = ok && sm100::mbar_wait_warp(&p_full[x][half], j & 1, a.err, sm100::kSiteMmaFull, abort);
        if (!ok) return;
        sm100::tc_fence_after();
        mma4_ts(d, p + half * 32, desc_mn(v + half * 8192, kHalf, 1024), id_o, j != 0 || half != 0);
        // the keys of the next score, looked for while the second half is computed
        if (half == 0 && x == 0 && j + 1 < tiles) wait_item(2 * j + 2);
      }
      if (last) sm100::mma_commit(&o_full[x]);
    };
    auto tiles_of = [&](int x) { return x == 0 ? tiles_a : tiles_b; };
    if (ok && tiles > 0) {
      wait_item(0);
      for (int x = 0; ok && x < 2; ++x)
        if (tiles_of(x) > 0) issue_s(x, 0);
      if (ok) sm100::mma_commit(&empty[0]);
      for (int j = 0; ok && j < tiles; ++j) {
        wait_item(2 * j + 1);
        if (TMA && ok && valid(j) < kKeys) {
          // the values behind the last key (of the prefix, or of all) become
          // zeros: a page's unused rows may hold anything, and 0 x NaN is NaN
          uint8_t *v = ring + ((2 * j + 1) % kStages) * kTile;
          for (int i = 8 * valid(j) + lane; i < 8 * kKeys; i += 32)
#pragma unroll
            for (int half = 0; half < DP / 64; ++half)
              *reinterpret_cast<uint4 *>(v + half * kHalf + 16 * i) = make_uint4(0, 0, 0, 0);
          sm100::fence_proxy_async_smem();
          __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (ok && j < tiles_of(x)) issue_o(x, j, j + 1 == tiles_of(x));
          if (ok && x == 1) sm100::mma_commit(&empty[(2 * j + 1) % kStages]);
          if (ok && x == 0 && j >= tiles_of(0) && j + 1 < tiles) wait_item(2 * j + 2);
          if (ok && j + 1 < tiles_of(x)) issue_s(x, j + 1);
        }
        if (ok && j + 1 < tiles) sm100::mma_commit(&empty[(2 * j + 2) % kStages]);
      }
    }
    sm100::mma_commit(&drain);
    int never = 0;
    sm100::mbar_wait(&drain, 0, a.err, sm100::kSiteDrain, &never);
  } else if (work && warp < kSoftmaxWarps) {
    // ---------------- softmax, one thread a row
    const int x = warp >> 2;  // tile
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    if (!q_boxes) {
      // both tiles' queries into shared memory, 16 bytes at a time
      constexpr int kPieces = DP / 8;
      // eight loads in flight before the first is stored
      constexpr int kStep = 32 * kSoftmaxWarps, kBatch = 8;
      for (int i0 = threadIdx.x; i0 < 2 * kRows * kPieces; i0 += kBatch * kStep) {
        uint4 v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kStep, qr = i / kPieces, c = i % kPieces, row = row0 + qr;
          v[u] = make_uint4(0, 0, 0, 0);
          if (row < rows && c * 8 < a.d) {
            const int j = row / a.group;
            v[u] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (int64_t)(s.first + j) * a.q_token +
                                                    (int64_t)(head * a.group + row - j * a.group) * a.q_head + c * 8);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kStep, qr = i / kPieces, c = i % kPieces, tr = qr & 127;
          *reinterpret_cast<uint4 *>(qs + (qr >> 7) * kTile + (c >> 3) * kHalf + tr * 128 + (((c & 7) ^ (tr & 7)) << 4)) = v[u];
        }
      }
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&q_full);
    }
    const int row = row0 + x * kRows + r;
    const int j_row = row / a.group;
    const int limit = row >= rows ? 0 : min(prefix ? a.prefix_len : paged::own_limit(a, s, j_row), key_end);
    // keys below this are seen by every row of the warp
    int free_end = limit;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) free_end = min(free_end, __shfl_xor_sync(0xffffffffu, free_end, o));
    const int mine = x == 0 ? tiles_a : tiles_b;
    const float c = a.scale_log2;
    const uint32_t s_at = tmem + lane_base + kColS + x * 128, o_at = tmem + lane_base + kColO + x * 128;
    float base = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < mine; ++j) {
      ok = ok && sm100::mbar_wait_warp(&s_full[x], j & 1, a.err, sm100::kSiteAttention, abort);
      if (!ok) break;
      sm100::tc_fence_after();
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
          // S_j is complete, so is the product before it: O holds still
#pragma unroll
          for (int i = 0; i < DP; i += 16) {
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
      // (A third of the exponentials as a polynomial on the FMA units lengthens
      // the tile, 257 -> 282 us for prompt chunks: two warps a scheduler do not
      // hide its chains.)
      auto release = [&](int h) {  // the product of these keys may begin
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[x][h]);
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
    if (tiles > 0 || !q_boxes) ok = ok && sm100::mbar_wait_warp(&q_full, 0, a.err, sm100::kSiteEpilogueAccum, abort);
    if (mine > 0) ok = ok && sm100::mbar_wait_warp(&o_full[x], 0, a.err, sm100::kSiteEpilogueAccum, abort);
    if (ok && row0 + x * kRows < rows) {
      sm100::tc_fence_after();
      const int q_heads = a.kv_heads * a.group;
      const int64_t token = s.first + j_row;
      const int qh = head * a.group + row - j_row * a.group;
      const bool on = row < rows;
      const bool some = l != 0.0f;  // (NaN too)
      const float inv = !direct ? 1.0f : some ? 1.0f / l : 0.0f;
      const int64_t part = (int64_t)(prefix ? a.own_splits + split : split) * a.tokens * q_heads + token * q_heads + qh;
      // rows of a split that see none of its keys are not read by the merge
      if (!direct && on) a.part_ml[part] = make_float2(base, l);
      // (the queries' place in shared memory is free: the products with them are
      // complete, and all of them have arrived)
      uint8_t *const stage = qs + x * kTile + (warp & 3) * 4096;
      if (direct)
        store_output<T>(stage, static_cast<T *>(a.o), on ? token * a.o_token + (int64_t)qh * a.o_head : -1, a.d, o_at, mine > 0, some, inv);
      else
        store_sums(stage, a.part_o, on ? part * a.d : -1, a.d, o_at, mine > 0, some);
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == kSoftmaxWarps + kLoadWarps) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 512);
  }
}

template <typename T, int DP, bool TMA>
int launch(b2k_ctx *ctx, const Args &a, bool prefix, int row_blocks, unsigned blocks, cudaStream_t s) {
  auto kernel = paged_umma_kernel<T, DP, TMA>;
  CUtensorMap map_k = {}, map_v = {}, map_q = {};
  const bool q_boxes = TMA && query_boxes_fit(a);
  int status = B2K_OK;
  if (TMA) status = make_map<T>(ctx, &map_k, a, true);
  if (TMA && status == B2K_OK) status = make_map<T>(ctx, &map_v, a, false);
  if (q_boxes && status == B2K_OK) status = make_q_map<T>(ctx, &map_q, a);
  if (status != B2K_OK) return status;
  cudaError_t err = b2k::set_max_smem(ctx, (const void *)kernel, smem_bytes<DP>());
  if (err == cudaSuccess)
    err = b2k::launch_kernel(a.pdl, kernel, dim3(blocks), dim3(kThreads), smem_bytes<DP>(), s, map_k, map_v,
                             map_q, a, prefix, row_blocks, q_boxes);
  return err == cudaSuccess ? B2K_OK : b2k::cuda_fail(ctx, err, "paged_attention launch");
}

template <typename T>
int pick(b2k_ctx *ctx, const Args &a, bool prefix, int row_blocks, unsigned blocks, cudaStream_t s) {
  const bool tma = boxes_fit(a);
  if (a.d <= 64)
    return tma ? launch<T, 64, true>(ctx, a, prefix, row_blocks, blocks, s)
               : launch<T, 64, false>(ctx, a, prefix, row_blocks, blocks, s);
  return tma ? launch<T, 128, true>(ctx, a, prefix, row_blocks, blocks, s)
             : launch<T, 128, false>(ctx, a, prefix, row_blocks, blocks, s);
}

}  // namespace

namespace paged {

bool umma_boxes(const b2k_paged_cache &c) {
  Args a = {};
  a.page_size = c.page_size;
  a.pages = c.pages;
  a.k_row = c.k_row;
  a.k_head = c.k_head;
  a.k_page = c.k_page;
  a.v_row = c.v_row;
  a.v_head = c.v_head;
  a.v_page = c.v_page;
  return boxes_fit(a);
}

int umma_part(b2k_ctx *ctx, const Args &a, int32_t dtype, bool prefix, cudaStream_t s) {
  const int64_t rows = (prefix ? a.tokens : (int64_t)a.max_new) * a.group;
  const int block_rows = umma_rows(a.d);
  const int64_t row_blocks = (rows + block_rows - 1) / block_rows;
  const int64_t blocks = row_blocks * a.kv_heads * (prefix ? a.prefix_splits : (int64_t)a.own_splits * a.sequences);
  if (blocks > INT32_MAX) return b2k::fail(ctx, B2K_EUNSUPPORTED, "paged_attention: %lld blocks", (long long)blocks);
  if (a.d > 128) return umma_wide_part(ctx, a, dtype, prefix, (int)row_blocks, (unsigned)blocks, s);
  return dtype == B2K_F16 ? pick<__half>(ctx, a, prefix, (int)row_blocks, (unsigned)blocks, s)
                          : pick<__nv_bfloat16>(ctx, a, prefix, (int)row_blocks, (unsigned)blocks, s);
}

}  // namespace paged
