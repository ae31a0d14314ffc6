// Block tables, row positions and cache slots of a step, made on the device from the lengths of its requests.
//
// Sequence b holds start[b] tokens and brings n[b] more.  With held = ceil(start / block) and after = ceil((start + n) / block),
// its table gets the next after - held entries of the free list; sequences take theirs in order.  Row r of the step belongs to the
// sequence whose prefix sums of n enclose it, and lies at slot table[pos / block] * block + pos % block.
//
// Every CTA computes both prefix sums by itself (at most 16384 sequences, 128 KB of reads that the L2 serves) and then writes its
// share of the rows and tables, so that one launch does it all and no CTA waits for another.  The bytes are few; what bounds it is
// the latency of a launch, of one load and of the scan: 5 us a call for 8 sequences, 6 for 1024 with 65536 rows.
#include <algorithm>

#include "pi_kv8.cuh"

namespace {

constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32, kPlanMaxSeqs = 16384;   // at most

struct PlanParams {
  pi_step_arrays a;
  const int32_t *start, *n_tokens, *free_list;
  int n_seqs, n_free;
  pi_divisor by_block;
};

struct Totals {
  long long rows, need, spill;
};

__device__ __forceinline__ void plan_sequence(const PlanParams& p, int b, int& start, long long& n, int& held, int& after, long long& spill) {
  const int bs = p.a.block_size, wide = p.a.max_blocks;
  start = max(p.start[b], 0);
  n = max(p.n_tokens[b], 0);
  const long long end = (long long)start + n + bs - 1;
  const long long held_all = end < 0x7fffffffll ? p.by_block(start + bs - 1) : ((long long)start + bs - 1) / bs, after_all = end < 0x7fffffffll ? p.by_block((int)end) : end / bs;
  held = (int)min(held_all, (long long)wide);
  after = (int)min(after_all, (long long)wide);
  spill = after_all - max(held_all, (long long)after);   // blocks that the table's row has no room for
}

__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(const PlanParams p) {
  extern __shared__ int s_plan[];
  const int B = p.n_seqs, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5, bs = p.a.block_size, wide = p.a.max_blocks;
  int *s_cu = s_plan, *s_free = s_cu + B + 1, *s_start = s_free + B;   // first row, first entry of the free list, start
  __shared__ Totals s_warp[kPlanWarps];
  pi_grid_dependency_wait();

  // prefix sums: a run of sequences per thread, a scan of the runs' totals
  const int per = (B + threads - 1) / threads, b0 = min(tid * per, B), b1 = min(b0 + per, B);
  Totals mine = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    int start, held, after;
    long long n, spill;
    plan_sequence(p, b, start, n, held, after, spill);
    mine.rows += n;
    mine.need += after - held;
    mine.spill += spill;
  }
  Totals upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long r = __shfl_up_sync(0xffffffffu, upto.rows, o), f = __shfl_up_sync(0xffffffffu, upto.need, o);
    if (lane >= o) {
      upto.rows += r;
      upto.need += f;
    }
  }
  if (__any_sync(0xffffffffu, mine.spill != 0)) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) upto.spill += __shfl_xor_sync(0xffffffffu, upto.spill, o);
  }
  if (lane == 31) s_warp[warp] = upto;
  __syncthreads();
  // lane w looks at warp w
  Totals ahead = lane < warps ? s_warp[lane] : Totals{0, 0, 0}, total = ahead;
  if (lane >= warp) ahead.rows = ahead.need = 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o >= warps) continue;   // further lanes hold nothing
    ahead.rows += __shfl_xor_sync(0xffffffffu, ahead.rows, o);
    ahead.need += __shfl_xor_sync(0xffffffffu, ahead.need, o);
    total.rows += __shfl_xor_sync(0xffffffffu, total.rows, o);
    total.need += __shfl_xor_sync(0xffffffffu, total.need, o);
    total.spill += __shfl_xor_sync(0xffffffffu, total.spill, o);
  }
  if (warps < 32) {
    ahead.rows = __shfl_sync(0xffffffffu, ahead.rows, 0);
    ahead.need = __shfl_sync(0xffffffffu, ahead.need, 0);
    total.rows = __shfl_sync(0xffffffffu, total.rows, 0);
    total.need = __shfl_sync(0xffffffffu, total.need, 0);
    total.spill = __shfl_sync(0xffffffffu, total.spill, 0);
  }
  ahead.rows += upto.rows - mine.rows;
  ahead.need += upto.need - mine.need;
  const long long cap = p.a.max_rows;
  for (int b = b0; b < b1; ++b) {
    int start, held, after;
    long long n, spill;
    plan_sequence(p, b, start, n, held, after, spill);
    s_cu[b] = (int)min(ahead.rows, cap);
    s_free[b] = (int)min(ahead.need, (long long)p.n_free);
    s_start[b] = start;
    ahead.rows += n;
    ahead.need += after - held;
    if (blockIdx.x == 0) {
      p.a.cu_rows[b] = s_cu[b];
      p.a.lens[b] = after;
    }
  }
  if (tid == 0) {
    s_cu[B] = (int)min(total.rows, cap);
    if (blockIdx.x == 0) {
      const long long taken = min(total.need, (long long)p.n_free);
      p.a.cu_rows[B] = s_cu[B];
      p.a.counts[0] = (int)min(total.rows, 0x7fffffffll);
      p.a.counts[1] = (int)taken;
      p.a.counts[2] = (int)min(total.need - taken + total.spill, 0x7fffffffll);
    }
  }
  __syncthreads();

  // new table entries: a warp per sequence
  for (int b = blockIdx.x * warps + warp; b < B; b += gridDim.x * warps) {
    int start, held, after;
    long long n, spill;
    plan_sequence(p, b, start, n, held, after, spill);
    for (int j = lane; j < after - held; j += 32) {
      const long long f = (long long)s_free[b] + j;
      p.a.tables[(size_t)b * wide + held + j] = f < p.n_free ? p.free_list[f] : -1;
    }
  }
  // rows: entries below `held` are read from the table, the ones above from where they come from
  for (long long r = (long long)blockIdx.x * threads + tid; r < cap; r += (long long)gridDim.x * threads) {
    int seq = -1, pos = -1;
    long long slot = -1;
    if (r < s_cu[B]) {
      int lo = 0, hi = B;   // the last b with s_cu[b] <= r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= r) lo = mid;
        else hi = mid;
      }
      seq = lo;
      const long long at = (long long)s_start[seq] + (r - s_cu[seq]);
      const long long lb = at < 0x7fffffffll ? p.by_block((int)at) : at / bs;
      const long long before = (long long)s_start[seq] + bs - 1;
      const int held = (int)min(before < 0x7fffffffll ? (long long)p.by_block((int)before) : before / bs, (long long)wide);
      pos = (int)at;
      int block = -1;
      if (lb < held) block = p.a.tables[(size_t)seq * wide + lb];
      else if (lb < wide && s_free[seq] + (lb - held) < p.n_free) block = p.free_list[s_free[seq] + (lb - held)];
      if (block >= 0) slot = (long long)block * bs + (at - lb * bs);
    }
    p.a.row_seq[r] = seq;
    p.a.row_pos[r] = pos;
    p.a.slots[r] = slot;
  }
}

}  // namespace

extern "C" pi_status pi_step_plan(pi_ctx* ctx, const pi_step_arrays* a, const int32_t* start_dev, const int32_t* n_tokens_dev, int n_seqs, const int32_t* free_dev,
                                  int n_free) {
  PI_ENTER(ctx);
  PI_REQUIRE(ctx, a && start_dev && n_tokens_dev && (free_dev || n_free == 0), "null pointer");
  PI_REQUIRE(ctx, a->tables && a->lens && a->cu_rows && a->row_seq && a->row_pos && a->slots && a->counts, "a plan needs all of its arrays");
  PI_REQUIRE(ctx, a->block_size > 0 && a->max_blocks > 0 && a->max_rows >= 0 && n_free >= 0, "block size and table width must be positive, row and block counts not negative");
  PI_REQUIRE(ctx, n_seqs >= 1 && n_seqs <= a->max_seqs && n_seqs <= kPlanMaxSeqs, "%d sequences: the arrays have room for %d, a plan for %d", n_seqs, a->max_seqs, kPlanMaxSeqs);
  const size_t smem = (size_t)(3 * n_seqs + 1) * sizeof(int);
  static pi_smem_grant grant;
  if (smem > kSmemFree && smem > grant.of(ctx)) {
    const size_t most = (size_t)(3 * kPlanMaxSeqs + 1) * sizeof(int);
    PI_CUDA(ctx, cudaFuncSetAttribute(step_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    grant.of(ctx) = most;
  }
  // as many threads as there are rows or sequences, up to a whole CTA; more CTAs for more rows than that
  const int busy = std::max(n_seqs, std::min(a->max_rows, kPlanThreads)), threads = std::min(kPlanThreads, (busy + 31) / 32 * 32), warps = threads / 32;
  const long long shares = std::max<long long>({1, ((long long)a->max_rows + threads - 1) / threads, ((long long)n_seqs + warps - 1) / warps});
  pi_prof_scope prof(ctx, PI_PROF_OTHER);
  const PlanParams p = {*a, start_dev, n_tokens_dev, free_dev, n_seqs, n_free, pi_divisor(a->block_size)};
  PI_CUDA(ctx, pi_launch_chained(ctx, step_plan_kernel, dim3((unsigned)std::min<long long>(shares, ctx->sm_count)), dim3(threads), smem, 1, p));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}
