// A token per row of logits: temperature, top-k, min-p and top-p, from a given random number.
//
// With M the row's maximum and w(x) = exp((x - M) / T), tokens are ordered by logit, equal ones by index.  Kept are the first top_k of
// that order, of those the ones with w >= min_p, and of those the shortest beginning whose sum reaches top_p of the sum of all of
// them.  Out of the kept tokens, in the order of their indices, comes the first whose running sum of w exceeds u times their sum.
//
// Every set above is a beginning of the order, so it is (threshold, number of tokens that equal it); neither a sort nor a list of
// the kept tokens is needed.  The threshold is found digit by digit over the logits' ordered bit patterns: a histogram of 1024 bins
// over the range that is left, by count (top-k) or by weight (top-p).
//
// Weights are whole numbers, w 2^45 rounded to nearest, taken from an exponential in 64 bits.  Sums of whole numbers do not depend on
// their order: neither the atomics nor the number of CTAs change a result.  45 bits leave a row of 2^18 equal tokens room in 64 bits,
// and each of three 15-bit limbs of 2^16 tokens room in 32, which is what the histogram adds with the 32-bit atomics of shared memory.
//
// A cluster of CTAs takes a row: each holds its slice of the logits in shared memory, so that they are read once, and reads the
// others' histograms there.
#include <float.h>

#include <algorithm>

#include "pi_kv8.cuh"

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kBins = 1024, kMaxCluster = 8;
constexpr int kWeightBits = 45, kLimb = 15;
constexpr int kSliceFloats = 48 * 1024;   // logits that fit a CTA's shared memory beside the histograms

struct SampleParams {
  const void* logits;
  int dtype;
  size_t stride;
  int n, per;                // logits of a row, of a CTA's slice
  const float *temperature, *top_p, *min_p, *u;
  const int32_t* top_k;
  int32_t* ids;
  float* probs;
};

// What a CTA shows the others.
struct Shown {
  unsigned long long best;   // ordered logit << 32 | ~index
  unsigned long long weight; // above the threshold
  unsigned int ties;
};

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <typename T>
__device__ __forceinline__ T peer(const T* mine, uint32_t rank) {   // the same variable of another CTA
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  if (sizeof(T) == 8) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return (T)v;
  }
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return (T)v;
}
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Row {
  const SampleParams& p;
  const float* x;       // the slice
  int count;
  float most;
  double rate;          // log2(e) / T
  __device__ __forceinline__ unsigned long long weight(float v) const {
    if (v == most) return 1ull << kWeightBits;
    return __double2ull_rn(exp2(((double)v - (double)most) * rate) * (double)(1ull << kWeightBits));
  }
};

struct Shared {
  uint32_t hist[2][3][kBins];
  unsigned long long warp_a[kWarps];
  unsigned int warp_b[kWarps];
  Shown shown;
  unsigned long long above, total;
  int bin;
};

// The threshold of the tokens whose running amount (count, or weight) first reaches `want`, from the largest down, among those
// with `low` <= logit.  By weight, `want` comes from the sum of all of them, and of those that equal `low` only `ties` count.
// Returns false where all of them together hold less than `want`.
template <bool WEIGHT>
__device__ bool find_threshold(const Row& row, Shared& s, uint32_t low, uint32_t high, unsigned long long ties, double part, unsigned long long want, int& turn,
                               uint32_t& thr, unsigned long long& above) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ranks = cluster_size();
  uint32_t lo = low, hi = high;
  above = 0;
  const unsigned long long tie_weight = WEIGHT ? ties * row.weight(from_ordered(low)) : 0;
  for (bool first = true; first || lo < hi; first = false) {
    const uint32_t span = hi - lo;
    const int shift = max(0, 32 - __clz(span) - 10);
    uint32_t(*h)[kBins] = s.hist[turn & 1];
    ++turn;
    for (int i = tid; i < (WEIGHT ? 3 : 1) * kBins; i += kThreads) (&h[0][0])[i] = 0;
    __syncthreads();
    for (int i = tid; i < row.count; i += kThreads) {
      const float x = row.x[i];
      const uint32_t k = ordered(x);
      if (k < lo || k > hi) continue;
      const uint32_t b = (k - lo) >> shift;
      if (!WEIGHT) {
        atomicAdd(&h[0][b], 1u);
      } else if (k != low) {
        const unsigned long long w = row.weight(x);
        atomicAdd(&h[0][b], (uint32_t)w & 0x7fffu);
        atomicAdd(&h[1][b], (uint32_t)(w >> kLimb) & 0x7fffu);
        atomicAdd(&h[2][b], (uint32_t)(w >> 2 * kLimb));
      }
    }
    cluster_sync();
    // a bin per thread, the largest logits first
    const int bin = kBins - 1 - tid;
    unsigned long long v = 0;
    for (uint32_t r = 0; r < ranks; ++r) {
      v += peer(&h[0][bin], r);
      if (WEIGHT) v += ((unsigned long long)peer(&h[1][bin], r) << kLimb) + ((unsigned long long)peer(&h[2][bin], r) << 2 * kLimb);
    }
    if (WEIGHT && bin == 0 && lo == low) v += tie_weight;
    unsigned long long upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    if (lane == 31) s.warp_a[warp] = upto;
    __syncthreads();
    unsigned long long all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += s.warp_a[w];
      all += s.warp_a[w];
    }
    if (first) {
      if (WEIGHT) want = max(1ull, (unsigned long long)ceil(part * (double)all));
      if (all < want) {
        if (!WEIGHT) return false;
        want = all;   // rounding of part * all
      }
    }
    if (above + upto >= want && above + upto - v < want) {
      s.bin = bin;
      s.above = above + upto - v;
    }
    __syncthreads();
    above = s.above;
    lo += (uint32_t)s.bin << shift;
    hi = min(hi, lo + ((1u << shift) - 1));
    __syncthreads();
  }
  thr = lo;
  if (WEIGHT) s.total = want;
  __syncthreads();
  return true;
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  extern __shared__ float s_slice[];
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int r = blockIdx.x / ranks;
  const int from = min((int)rank * p.per, p.n), count = min(p.per, p.n - from);
  const size_t base = (size_t)r * p.stride + from;
  pi_grid_dependency_wait();

  // the slice, and the largest logit with the lowest index; NaN counts as minus infinity, -0 as 0
  unsigned long long best = 0;
  for (int i = tid; i < count; i += kThreads) {
    float x = pi_load_as_f32(p.logits, base + i, p.dtype);
    x = x == x ? x + 0.f : -INFINITY;
    s_slice[i] = x;
    best = max(best, (unsigned long long)ordered(x) << 32 | (uint32_t)~(from + i));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.warp_a[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) best = max(best, s.warp_a[w]);
    s.shown.best = best;
  }
  cluster_sync();
  best = 0;
  for (uint32_t k = 0; k < ranks; ++k) best = max(best, peer(&s.shown.best, k));
  const uint32_t high = (uint32_t)(best >> 32);
  const float most = from_ordered(high), temperature = p.temperature[r];
  if (!(temperature > 0.f) || most == -INFINITY) {   // the largest; a row without any
    if (rank == 0 && tid == 0) {
      p.ids[r] = most == -INFINITY ? -1 : (int32_t)~(uint32_t)best;
      if (p.probs) p.probs[r] = most == -INFINITY ? 0.f : 1.f;
    }
    cluster_sync();
    return;
  }
  const Row row = {p, s_slice, count, most, 1.4426950408889634 / (double)temperature};

  // tokens below `low` weigh less than half a unit, or less than min_p
  double bound = (double)most - 32.0 * (double)temperature;
  const float min_p = p.min_p[r];
  if (min_p > 0.f) bound = max(bound, (double)most + (double)temperature * log(min((double)min_p, 1.0)));
  uint32_t thr = ordered(most == INFINITY ? INFINITY : max(__double2float_ru(bound), -FLT_MAX));
  unsigned long long ties = ~0u, above;
  int turn = 0;
  const int k = p.top_k[r];
  if (k > 0 && k < p.n) {
    uint32_t t;
    if (find_threshold<false>(row, s, thr, high, 0, 0., (unsigned long long)k, turn, t, above)) {
      thr = t;
      ties = (unsigned long long)k - above;
    }
  }
  const float top_p = p.top_p[r];
  if (top_p < 1.f) {
    // how many equal the threshold, where all of them count
    if (ties == ~0u) {
      unsigned int c = 0;
      for (int i = tid; i < count; i += kThreads) c += ordered(s_slice[i]) == thr;
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) s.warp_b[warp] = c;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) c += s.warp_b[w];
        s.shown.ties = c;
      }
      cluster_sync();
      ties = 0;
      for (uint32_t q = 0; q < ranks; ++q) ties += peer(&s.shown.ties, q);
      cluster_sync();
    }
    uint32_t t;
    find_threshold<true>(row, s, thr, high, ties, (double)max(top_p, 0.f), 0, turn, t, above);
    thr = t;
    const unsigned long long w = row.weight(from_ordered(thr)), missing = s.total - above;
    ties = (missing + w - 1) / w;
  }

  // sums in the order of the indices: a run of the slice per warp
  const int run = ((count + kWarps * 32 - 1) / (kWarps * 32)) * 32, i0 = min(warp * run, count), i1 = min(i0 + run, count);
  unsigned long long sum = 0;
  unsigned int same = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t key = ordered(s_slice[i]);
    if (key > thr) sum += row.weight(s_slice[i]);
    same += key == thr;
  }
  sum = warp_sum(sum);
  same = __reduce_add_sync(0xffffffffu, same);
  if (lane == 0) {
    s.warp_a[warp] = sum;
    s.warp_b[warp] = same;
  }
  __syncthreads();
  if (tid == 0) {
    unsigned long long a = 0;
    unsigned int b = 0;
    for (int w = 0; w < kWarps; ++w) {
      a += s.warp_a[w];
      b += s.warp_b[w];
    }
    s.shown.weight = a;
    s.shown.ties = b;
  }
  cluster_sync();
  const unsigned long long w_thr = row.weight(from_ordered(thr));
  unsigned long long total = 0, ahead = 0, used = 0, used_here = 0;
  for (uint32_t q = 0; q < ranks; ++q) {
    const unsigned long long equal = min((unsigned long long)peer(&s.shown.ties, q), ties - used), v = peer(&s.shown.weight, q) + equal * w_thr;
    if (q < rank) ahead += v;
    if (q == rank) used_here = used;
    used += equal;
    total += v;
  }
  const float u = p.u[r];
  unsigned long long goal = u > 0.f ? (unsigned long long)floor((double)u * (double)total) : 0;
  goal = min(goal, total - 1);
  // the first token whose running sum exceeds the goal: the warp whose run holds it finds it
  unsigned long long mine = ahead, taken = used_here;
  for (int w = 0; w < warp; ++w) {
    const unsigned long long equal = min((unsigned long long)s.warp_b[w], ties - taken);
    mine += s.warp_a[w] + equal * w_thr;
    taken += equal;
  }
  const unsigned long long here = s.warp_a[warp] + min((unsigned long long)s.warp_b[warp], ties - taken) * w_thr;
  if (goal >= mine && goal < mine + here) {
    for (int i = i0 + lane; i - lane < i1; i += 32) {
      const uint32_t key = i < i1 ? ordered(s_slice[i]) : 0;
      const unsigned equal = __ballot_sync(0xffffffffu, i < i1 && key == thr);
      unsigned long long w = 0;
      if (i < i1 && key > thr) w = row.weight(s_slice[i]);
      if (i < i1 && key == thr && taken + __popc(equal & ((1u << lane) - 1)) < ties) w = w_thr;
      taken += __popc(equal);
      unsigned long long upto = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
      }
      const unsigned found = __ballot_sync(0xffffffffu, mine + upto > goal);
      if (found) {
        if (lane == __ffs(found) - 1) {
          p.ids[r] = from + i;
          if (p.probs) p.probs[r] = (float)((double)w / (double)total);
        }
        break;
      }
      mine += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  cluster_sync();   // nobody leaves while another one reads its memory
}

}  // namespace

extern "C" pi_status pi_sample(pi_ctx* ctx, const void* logits_dev, int dtype, size_t row_stride, int rows, int n, const float* temperature_dev, const int32_t* top_k_dev,
                               const float* top_p_dev, const float* min_p_dev, const float* u_dev, int32_t* ids_dev, float* probs_dev_or_null) {
  PI_ENTER(ctx);
  PI_REQUIRE(ctx, dtype == PI_F32 || dtype == PI_BF16 || dtype == PI_F16, "logits of kind %d: PI_F32, PI_BF16 or PI_F16 are wanted", dtype);
  PI_REQUIRE(ctx, rows >= 0, "negative row count");
  if (rows == 0) return PI_OK;
  PI_REQUIRE(ctx, logits_dev && temperature_dev && top_k_dev && top_p_dev && min_p_dev && u_dev && ids_dev, "null pointer");
  PI_REQUIRE(ctx, n >= 1 && n <= kMaxCluster * kSliceFloats, "%d logits a row: 1 to %d are taken", n, kMaxCluster * kSliceFloats);
  PI_REQUIRE(ctx, row_stride >= (size_t)n || rows == 1, "rows of %d logits cannot be %zu apart", n, row_stride);
  PI_REQUIRE(ctx, (uintptr_t)logits_dev % (dtype == PI_F32 ? 4 : 2) == 0, "logits must be aligned to their type");
  // a CTA per 16384 logits, which is half of what an SM can hold
  int cluster = 1;
  while (cluster < kMaxCluster && (n + cluster - 1) / cluster > 16384) cluster *= 2;
  SampleParams p = {logits_dev, dtype, row_stride, n, (n + cluster - 1) / cluster, temperature_dev, top_p_dev, min_p_dev, u_dev, top_k_dev, ids_dev, probs_dev_or_null};
  const size_t smem = (size_t)p.per * sizeof(float);
  static pi_smem_grant grant;
  if (smem > grant.of(ctx)) {
    PI_CUDA(ctx, cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceFloats * (int)sizeof(float)));
    grant.of(ctx) = kSliceFloats * sizeof(float);
  }
  pi_prof_scope prof(ctx, PI_PROF_OTHER);
  PI_CUDA(ctx, pi_launch_chained(ctx, sample_kernel, dim3((unsigned)rows * cluster), dim3(kThreads), smem, cluster, p));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}
