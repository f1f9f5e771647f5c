// Shared by the kernels of attention over a paged cache: what a launch of one
// part of the keys gets, and the partial sums that parts leave for the merge.
//
// Mathematics.  A row's softmax over a set of keys is (m, l, o): the largest
// score, the sum of exp(s - m) and the sum of exp(s - m) v.  Two disjoint sets
// join exactly: m = max(m1, m2), l and o each the sum of both sides' times
// exp(m_i - m).  So the keys are cut into parts -- the shared prefix, once for
// all sequences, and every sequence's own keys, each again into splits where
// the rows alone would not fill the GPU -- and a last kernel joins a row's
// parts.  Scores are kept times log2(e) / scale, exponentials are base 2.
#pragma once

#include "serve.cuh"

namespace paged {

struct Args {
  const void *q;
  void *o;
  int64_t q_token, q_head, o_token, o_head;  // strides, elements
  const void *k, *v;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;
  int64_t pages;
  int page_size, kv_heads, group, d;  // group: query heads of a cache head
  int sequences;
  int64_t tokens;
  const int32_t *first, *lengths, *table, *prefix_table;
  int64_t table_stride;
  int table_width, prefix_len, max_new, max_len;
  float scale_log2;  // log2(e) / scale
  unsigned *err;
  // the parts: own keys in `own_splits` splits of `own_chunk`, the prefix in
  // prefix_splits of prefix_chunk behind them (0: there is none, or own parts
  // begin with it: `joined`)
  int own_splits, own_chunk, prefix_splits, prefix_chunk;
  int joined;
  int joined_keys;   // where a joined part's own keys begin in its numbering: prefix_len, or that rounded up to whole tiles
  unsigned *ready;   // several kernels, not captured: the word that orders them (part_begin), and this
  unsigned call;     // call's value of it; ready is null otherwise
  bool pdl;          // launched with programmatic dependence on the kernel before
  float *part_o;   // [own_splits + prefix_splits][tokens * q heads][d]
  float2 *part_ml; // [own_splits + prefix_splits][tokens * q heads]: m, l
};

// A sequence's rows as its device-side numbers give them; n = 0 (and the error
// word set) where they leave the bounds the launch was sized by.
struct Sequence {
  int first, n, own0;  // own0: own position of its first new token
};
__device__ __forceinline__ Sequence sequence_of(const Args &a, int first, int next, int len) {
  Sequence s;
  s.first = first;
  s.n = next - first;
  s.own0 = len - s.n;
  if (s.first < 0 || s.n < 0 || (int64_t)s.first + s.n > a.tokens || s.n > a.max_new || len > a.max_len || len < 0) {
    atomicOr(a.err, serve::kErrIndex);
    s.n = 0;
  }
  return s;
}
__device__ __forceinline__ Sequence sequence(const Args &a, int b) {
  return sequence_of(a, a.first[b], a.first[b + 1], a.lengths[b]);
}
// The b-th longest of up to 32 sequences (in their own order above that; `b`
// becomes its number).  For whole warps; one round of loads, as for one sequence.
__device__ __forceinline__ Sequence sequence_by_length(const Args &a, int &b) {
  if (a.sequences > 32) return sequence(a, b);
  const int lane = threadIdx.x & 31;
  const bool in = lane < a.sequences;
  const int first = in ? a.first[lane] : 0, next = in ? a.first[lane + 1] : 0, len = in ? a.lengths[lane] : 0;
  int longer = 0;
  for (int i = 0; i < a.sequences; ++i) {
    const int other = __shfl_sync(0xffffffffu, len, i);
    longer += other > len || (other == len && i < lane);
  }
  b = __ffs(__ballot_sync(0xffffffffu, in && longer == b)) - 1;
  return sequence_of(a, __shfl_sync(0xffffffffu, first, b), __shfl_sync(0xffffffffu, next, b),
                     __shfl_sync(0xffffffffu, len, b));
}
// Packed rows in use.
__device__ __forceinline__ int used_tokens(const Args &a) {
  const int n = a.first[a.sequences];
  return (int)min((int64_t)max(n, 0), a.tokens);
}

// Keys of an own part that new token j may see, as the part numbers them: its
// prefix (joined; numbers from prefix_len to joined_keys name none) and own
// positions up to its own.
__device__ __forceinline__ int own_limit(const Args &a, const Sequence &s, int j) {
  const int own = max(0, s.own0 + j + 1);
  return !a.joined ? own : own > 0 ? a.joined_keys + own : a.prefix_len;
}

// A block's keys end: its split's, or where its last row sees no more.  (A split's
// end is not computed by itself: near the largest lengths it passes 32 bits.)
__device__ __forceinline__ int split_end(int key0, int chunk, int limit) { return key0 + min(chunk, limit - key0); }

// The page table's entry for a key, unchecked, and the key's row in that page.
// `at` counts from the start of the part: the prefix's keys, or the own keys
// behind the prefix's where the part is joined (joined_keys = prefix_len).
__device__ __forceinline__ int key_entry(const Args &a, bool prefix, int b, int at, int &row) {
  const int32_t *table = a.prefix_table;
  if (!prefix && (!a.joined || at >= a.prefix_len)) {
    table = a.table + (int64_t)b * a.table_stride;
    at -= a.joined ? a.prefix_len : 0;
  }
  const int i = (int)((unsigned)at / (unsigned)a.page_size);
  row = at - i * a.page_size;
  return table[i];
}
// The key's page; -1 (and the error word set) for one outside the cache.
__device__ __forceinline__ int64_t key_page(const Args &a, bool prefix, int b, int at, int &row) {
  const int64_t page = key_entry(a, prefix, b, at, row);
  if (page >= 0 && page < a.pages) return page;
  atomicOr(a.err, serve::kErrIndex);
  return -1;
}

// The own part runs beside the prefix part, the kernel before it in the stream,
// whose results it does not read: its blocks do not wait for that kernel, but
// what precedes the call (queries, cache, lengths, the workspace's last readers)
// has to be complete and visible to them.  The prefix part's first block waits
// for that and then releases the call's number to a word of the context; a
// thread of the own part that acquires this number is ordered behind that wait.
// One that does not find it yet waits for the prefix part itself: nothing spins.
// The merge reads the sequences' numbers ahead of its own wait in the same way.
// (Blocks of the prefix part let the next kernel start only behind their wait, so
// nearly all find it.)  A number comes again after 2^32 calls, which have written
// its word 2^26 times by then.  A captured call, whose number would come again at
// every replay, has the two parts as parallel branches of its graph instead
// (paged.cu).  128 single tokens behind 8192 shared ones: 102 us a call in a
// stream, 92 in a graph; with no ordering of the own part's reads 102 and 90, with
// the parts one after the other 142.
// The own part's last block waits for the prefix part at its end, so that the own
// part's end means the prefix part's too and the merge, which waits for the own
// part, has both.  (The last block alone: waiting blocks hold their place on an SM, and
// with all of them waiting the two parts all but took turns.)
__device__ __forceinline__ bool call_ready(const Args &a) {
  if (!a.ready) return false;
  unsigned seen;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(a.ready) : "memory");
  return seen == a.call;
}
__device__ __forceinline__ void part_begin(const Args &a, bool beside) {
  if (beside) {
    if (!call_ready(a)) grid_dependency_wait();
  } else {
    grid_dependency_wait();
    if (a.ready && blockIdx.x == 0 && threadIdx.x == 0)
      asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(a.ready), "r"(a.call) : "memory");
  }
  grid_dependents_launch();
}
__device__ __forceinline__ void part_end(bool beside) {
  if (beside && blockIdx.x == gridDim.x - 1) grid_dependency_wait();
}

// The blocks of a launch of one or both parts, in one dimension: the prefix
// part's first, then the sequences'; row blocks within heads within splits
// (within sequences).
struct Grid {
  unsigned prefix_blocks;  // 0: no prefix part in this launch
  int prefix_row_blocks, own_row_blocks;
  bool beside;  // the prefix part is the kernel before: run beside it (part_begin)
};
struct Block {
  bool prefix;
  int row_block, head, split, sequence;
};
__device__ __forceinline__ Block this_block(const Args &a, const Grid &g) {
  Block b;
  b.prefix = blockIdx.x < g.prefix_blocks;
  unsigned at = b.prefix ? blockIdx.x : blockIdx.x - g.prefix_blocks;
  const unsigned row_blocks = b.prefix ? g.prefix_row_blocks : g.own_row_blocks;
  b.row_block = at % row_blocks;
  at /= row_blocks;
  b.head = at % (unsigned)a.kv_heads;
  at /= (unsigned)a.kv_heads;
  const unsigned splits = b.prefix ? a.prefix_splits : a.own_splits;
  b.split = at % splits;
  b.sequence = at / splits;
  return b;
}
// Fills `g` for blocks of `rows` rows; the number of blocks, or -1 (error recorded).
inline int64_t make_grid(b2k_ctx *ctx, const Args &a, bool with_prefix, bool with_own, int rows, bool beside, Grid &g) {
  g.prefix_row_blocks = (int)((a.tokens * a.group + rows - 1) / rows);
  g.own_row_blocks = (int)(((int64_t)a.max_new * a.group + rows - 1) / rows);
  g.beside = beside;
  const int64_t prefix = with_prefix ? (int64_t)g.prefix_row_blocks * a.kv_heads * a.prefix_splits : 0;
  const int64_t own = with_own ? (int64_t)g.own_row_blocks * a.kv_heads * a.own_splits * a.sequences : 0;
  g.prefix_blocks = (unsigned)prefix;
  if (prefix + own <= INT32_MAX) return prefix + own;
  b2k::fail(ctx, B2K_EUNSUPPORTED, "paged_attention: %lld blocks", (long long)(prefix + own));
  return -1;
}

// paged_mma.cu: rows of a block (16 or 32) for `rows` rows of one cache head, and
// the launch of the prefix part, the sequences' own parts or both.
int mma_rows(int d, int64_t rows);
int mma_parts(b2k_ctx *ctx, const Args &a, int32_t dtype, bool with_prefix, bool with_own, int rows, bool beside,
              cudaStream_t s);

// paged_f32.cu: the same for f32 in 16-byte pieces, blocks of 4 or 8 rows.
int f32_parts(b2k_ctx *ctx, const Args &a, bool with_prefix, bool with_own, int rows, bool beside, cudaStream_t s);

// paged_umma.cu (and paged_umma_wide.cu for head dims above 128): rows of a block,
// whether a cache's pages can be loaded as boxes, which the wide kernel needs,
// and the launch of one part.
inline int umma_rows(int d) { return d <= 128 ? 256 : 128; }
bool umma_boxes(const b2k_paged_cache &c);
int umma_wide_part(b2k_ctx *ctx, const Args &a, int32_t dtype, bool prefix, int row_blocks, unsigned blocks, cudaStream_t s);
int umma_part(b2k_ctx *ctx, const Args &a, int32_t dtype, bool prefix, cudaStream_t s);

}  // namespace paged
