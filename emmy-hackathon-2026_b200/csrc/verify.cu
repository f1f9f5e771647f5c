// Verification of drafted tokens: how many of a sequence's drafts the target
// takes, and the token drawn behind them.
//
// Mathematics.  A draft x with drafter's probability q(x) is taken with
// probability min(1, p(x) / q(x)): u q(x) < p(x), a comparison of two
// products of FP32 numbers, exact in FP64.  The draw from the rest r =
// max(p - q, 0) is the inverse of its cumulative sum; FP64 sums of at most
// 2^31 FP32 terms leave an error near 1e-13 of the total, far below the
// spacing of the steps, so the order of the summation does not show.
//
// Bound: HBM, one row of p and one of q a sequence (2 * 4 * vocab bytes), in
// one launch: a cluster of eight CTAs takes a sequence, each an eighth of the
// row, each warp a contiguous run of that.  The runs' sums meet through
// distributed shared memory, every CTA finds the run that holds the
// threshold, and the CTA that owns it reads it again (from L2) in order, all
// its threads side by side.  Few sequences then still use eight SMs each, and
// nothing is kept in global memory between the two passes.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "serve.cuh"

namespace {

constexpr int kCluster = 8;
constexpr int kAhead = 8;   // elements a lane has in flight in the first pass
constexpr int kRun = 8;     // consecutive elements of a thread in the second

struct VerifyArgs {
  b2k_drafts d;
  int32_t *accepted, *tokens;
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Inclusive sum over the lanes, in a fixed order.
__device__ __forceinline__ double warp_scan(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += other;
  }
  return v;
}

// Of 32 lanes' sums v in order, `upto` their cumulative sums: the first whose
// cumulative sum passes the threshold, or the last that holds anything where
// rounding leaves none (-1: none does), and the sum before it.
__device__ __forceinline__ int pick(double v, double upto, double start, double threshold, double &before) {
  const unsigned over = __ballot_sync(0xffffffffu, v > 0.0 && start + upto > threshold);
  const unsigned held = __ballot_sync(0xffffffffu, v > 0.0);
  const int at = over ? __ffs(over) - 1 : held ? 31 - __clz(held) : -1;
  before = start + __shfl_sync(0xffffffffu, upto - v, at < 0 ? 0 : at);
  return at;
}

// The rest that the token is drawn from: max(p - q, 0), p where q is not
// there, and nothing of the rejected draft where that was certain.
struct Rest {
  const float *p, *q;
  int64_t without;
};

template <int kThreads>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) verify_kernel(const VerifyArgs a) {
  constexpr int kWarps = kThreads / 32;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double run_sum[kWarps], scan_sum[kWarps], slice_sum[2];
  __shared__ int taken_s;
  __shared__ int warp_hit[kWarps], warp_last[kWarps];
  grid_dependency_wait();
  grid_dependents_launch();

  const b2k_drafts &d = a.d;
  const int rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / kCluster;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = d.counts ? min(max(d.counts[b], 0), d.drafts) : d.drafts;
  const int32_t *drafted = d.drafted + b * d.drafts;

  if (warp == 0) {
    int taken = n;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool ok = true;
      if (i < n) {
        const int64_t x = drafted[i];
        ok = x >= 0 && x < d.vocab;
        if (ok) {
          const double p = d.target[(b * (d.drafts + 1) + i) * d.ld_target + x];
          const double q = d.draft ? (double)d.draft[(b * d.drafts + i) * d.ld_draft + x] : 1.0;
          ok = (double)d.u_accept[b * d.drafts + i] * q < p;
        }
      }
      const unsigned refused = __ballot_sync(0xffffffffu, !ok);
      if (refused) {
        taken = i0 + __ffs(refused) - 1;
        break;
      }
    }
    if (lane == 0) taken_s = taken;
  }
  __syncthreads();
  const int taken = taken_s;
  Rest rest;
  rest.p = d.target + (b * (d.drafts + 1) + taken) * d.ld_target;
  rest.q = taken < n && d.draft ? d.draft + (b * d.drafts + taken) * d.ld_draft : nullptr;
  rest.without = taken < n && !d.draft ? (int64_t)drafted[taken] : -1;

  // this warp's run [lo, hi) of the row
  const int64_t run = (d.vocab + kCluster * kWarps - 1) / (kCluster * kWarps);
  const int64_t lo = min(d.vocab, (rank * kWarps + warp) * run), hi = min(d.vocab, lo + run);

  int64_t token = -1;   // of the CTA that owns the draw
  bool owner = false;
  for (int pass = 0; pass < 2; ++pass) {  // the second only where the rest is zero everywhere
    // FP64 sums of the run's elements, four chains a lane.  HAS_Q and WITHOUT as
    // the rest has them: fewer comparisons where it has not.
    auto sum_run = [&](auto has_q, auto without) {
      constexpr bool kQ = decltype(has_q)::value, kWithout = decltype(without)::value;
      double s[4] = {0.0, 0.0, 0.0, 0.0};
      const float *p = rest.p + lane, *q = rest.q + (kQ ? lane : 0);
      const int skip = kWithout ? (int)(rest.without - lane) : 0;  // (vocab is below 2^31 - 2^16)
      int i = (int)lo;
      const int end = (int)hi;
      for (; i + 32 * kAhead <= end; i += 32 * kAhead) {
        float pv[kAhead], qv[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          pv[u] = __ldg(p + i + 32 * u);
          qv[u] = kQ ? __ldg(q + i + 32 * u) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (pv[u] > qv[u] && !(kWithout && i + 32 * u == skip)) s[u & 3] += kQ ? (double)pv[u] - (double)qv[u] : (double)pv[u];
      }
      if (i < end) {  // the rest of the run, all of it in flight too
        float pv[kAhead], qv[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const bool in = i + 32 * u + lane < end;
          pv[u] = in ? __ldg(p + i + 32 * u) : 0.0f;
          qv[u] = in && kQ ? __ldg(q + i + 32 * u) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (pv[u] > qv[u] && !(kWithout && i + 32 * u == skip)) s[u & 3] += kQ ? (double)pv[u] - (double)qv[u] : (double)pv[u];
      }
      return (s[0] + s[1]) + (s[2] + s[3]);
    };
    double sum = rest.q ? sum_run(std::true_type{}, std::false_type{})
                 : rest.without >= 0 ? sum_run(std::false_type{}, std::true_type{})
                                     : sum_run(std::false_type{}, std::false_type{});
    sum = warp_sum(sum);
    if (lane == 0) run_sum[warp] = sum;
    __syncthreads();
    const double mine_of = lane < kWarps ? run_sum[lane] : 0.0;  // each warp scans the runs' sums for itself
    const double mine_upto = warp_scan(mine_of), slice_total = __shfl_sync(0xffffffffu, mine_upto, 31);
    if (threadIdx.x == 0) slice_sum[pass] = slice_total;
    cluster.sync();
    const double slice = lane < kCluster ? *cluster.map_shared_rank(&slice_sum[pass], lane < kCluster ? lane : 0) : 0.0;
    const double slices_upto = warp_scan(slice), total = __shfl_sync(0xffffffffu, slices_upto, 31);
    if (!(total > 0.0) && pass == 0 && taken < n) {
      rest.q = nullptr;
      rest.without = -1;
      continue;
    }
    cluster.barrier_arrive();  // this thread has read; who leaves waits for all of them
    // the slice, then the run in it, whose cumulative sum first passes the
    // threshold; rounding may leave none, then the last one that holds anything
    const double threshold = (double)d.u_sample[b] * total;
    double start, run_start;
    const int slice_at = pick(slice, slices_upto, 0.0, threshold, start);
    if (slice_at == rank) {
      const int run_at = pick(mine_of, mine_upto, start, threshold, run_start);
      // run_at is one for the whole CTA: its elements in order, kRun a thread,
      // kRun * kThreads at a time
      owner = true;
      const int64_t run_lo = min(d.vocab, (rank * kWarps + run_at) * run), run_hi = min(d.vocab, run_lo + run);
      double base = run_start;
      for (int64_t i0 = run_lo; i0 < run_hi; i0 += kRun * kThreads) {
        const int64_t i = i0 + threadIdx.x * kRun;
        float pv[kRun], qv[kRun];
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
          const bool in = i + u < run_hi;
          pv[u] = in ? __ldg(rest.p + i + u) : 0.0f;
          qv[u] = in && rest.q ? __ldg(rest.q + i + u) : 0.0f;
        }
        double v[kRun], mine = 0.0;
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
          v[u] = pv[u] > qv[u] && i + u != rest.without ? (double)pv[u] - (double)qv[u] : 0.0;
          mine += v[u];
        }
        const double upto = warp_scan(mine);  // over the lanes, then over the warps
        if (lane == 31) scan_sum[warp] = upto;
        __syncthreads();
        const double warps = lane < kWarps ? scan_sum[lane] : 0.0, warps_upto = warp_scan(warps);
        double c = base + __shfl_sync(0xffffffffu, warps_upto - warps, warp) + (upto - mine);
        base += __shfl_sync(0xffffffffu, warps_upto, 31);
        int hit = -1, last = -1;
#pragma unroll
        for (int u = 0; u < kRun; ++u) {
          c += v[u];
          if (v[u] > 0.0) {
            last = (int)(i + u);
            if (hit < 0 && c > threshold) hit = (int)(i + u);
          }
        }
        const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), held = __ballot_sync(0xffffffffu, last >= 0);
        hit = hits ? __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1) : -1;
        last = held ? __shfl_sync(0xffffffffu, last, 31 - __clz(held)) : -1;
        if (lane == 0) {
          warp_hit[warp] = hit;
          warp_last[warp] = last;
        }
        __syncthreads();
        hit = lane < kWarps ? warp_hit[lane] : -1;
        last = lane < kWarps ? warp_last[lane] : -1;
        const unsigned hit_warps = __ballot_sync(0xffffffffu, hit >= 0), held_warps = __ballot_sync(0xffffffffu, last >= 0);
        if (hit_warps) {
          token = __shfl_sync(0xffffffffu, hit, __ffs(hit_warps) - 1);
          break;
        }
        if (held_warps) token = __shfl_sync(0xffffffffu, last, 31 - __clz(held_warps));
      }
    } else if (slice_at < 0) {
      owner = rank == 0;  // nothing above zero: token -1
    }
    break;
  }
  if (owner && threadIdx.x == 0) a.tokens[b * (d.drafts + 1) + taken] = (int32_t)token;
  if (rank == 0 && warp == 1) {
    if (lane == 0) a.accepted[b] = taken;
    for (int i = lane; i <= d.drafts; i += 32)
      if (i != taken) a.tokens[b * (d.drafts + 1) + i] = i < taken ? drafted[i] : -1;
  }
  cluster.barrier_wait();
}

}  // namespace

extern "C" int b2k_verify_drafts(b2k_ctx *ctx, const b2k_drafts *d, int32_t *accepted, int32_t *tokens, void *stream) {
  B2K_CHECK_CTX(ctx);
  if (!d) return b2k::fail(ctx, B2K_EINVAL, "verify_drafts: null drafts");
  if (d->batch < 0 || d->drafts < 0 || d->vocab < 1 || d->vocab > INT32_MAX - 65536)
    return b2k::fail(ctx, B2K_EINVAL, "verify_drafts: batch %lld, %d drafts, vocab %lld", (long long)d->batch, d->drafts,
                     (long long)d->vocab);
  if (d->batch > INT32_MAX / kCluster) return b2k::fail(ctx, B2K_EINVAL, "verify_drafts: too many sequences");
  if (d->ld_target < d->vocab || (d->draft && d->ld_draft < d->vocab))
    return b2k::fail(ctx, B2K_EINVAL, "verify_drafts: a row stride is below vocab");
  if (d->batch == 0) return B2K_OK;
  if (!d->target || !d->u_sample || !accepted || !tokens || (d->drafts > 0 && (!d->drafted || !d->u_accept)))
    return b2k::fail(ctx, B2K_EINVAL, "verify_drafts: null buffer");
  // every array's extent (elements of 4 bytes, rows of probabilities with what lies
  // between them), the outputs first
  const double rows = (double)d->batch * (d->drafts + 1.0), drafted = (double)d->batch * d->drafts;
  const struct {
    const void *p;
    double n;
  } arrays[] = {{accepted, (double)d->batch}, {tokens, rows}, {d->target, (rows - 1) * d->ld_target + d->vocab},
                {d->draft, drafted > 0 ? (drafted - 1) * d->ld_draft + d->vocab : 0.0}, {d->drafted, drafted},
                {d->counts, (double)d->batch}, {d->u_accept, drafted}, {d->u_sample, (double)d->batch}};
  for (const auto &x : arrays)
    if (!serve::on_boundary(x.p, 4)) return b2k::fail(ctx, B2K_EINVAL, "verify_drafts: a buffer is off 4 bytes");
  for (int i = 0; i < 2; ++i)
    for (const auto &x : arrays) {
      const auto &out = arrays[i];
      if (&x == &out || !x.p || x.n == 0.0) continue;
      const double apart = (double)(reinterpret_cast<uintptr_t>(x.p) / 4) - (double)(reinterpret_cast<uintptr_t>(out.p) / 4);
      if (apart < out.n && -apart < x.n)
        return b2k::fail(ctx, B2K_EINVAL, "verify_drafts: %s overlaps another array", i ? "tokens" : "accepted");
    }
  cudaStream_t s = (cudaStream_t)stream;
  b2k::PhaseTimer timer(ctx, B2K_PHASE_VERIFY, s);
  const VerifyArgs a{*d, accepted, tokens};
  // A few sequences leave an SM to each CTA, which wants many loads in flight for
  // a long row (131071: 7.0 us with 512 threads, 7.9 with 256) and fewer warps to
  // wait for for a short one (32000: 5.5 and 5.1); a batch wants all its CTAs
  // resident at once (64 sequences of 131071: 25 us with 512, 17.6 with 256).
  const bool few = d->batch * kCluster <= ctx->sm_count && d->vocab > 65536;
  cudaError_t err = b2k::launch_kernel(b2k::pdl_enabled(), few ? verify_kernel<512> : verify_kernel<256>,
                                       dim3((unsigned)(d->batch * kCluster)), dim3(few ? 512 : 256), 0, s, a);
  if (err != cudaSuccess) return b2k::cuda_fail(ctx, err, "verify_drafts launch");
  return b2k::check_launch(ctx, "verify_drafts launch");
}
