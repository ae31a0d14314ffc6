// A token per row of logits: temperature, top-k, min-p and top-p, from a given random number.
//
// With M the row's maximum and w(x) = exp((x - M) / T), tokens are ordered by logit, equal ones by index.  Kept are the first top_k of
// that order, of those the ones with w >= min_p, and of those the shortest beginning whose sum reaches top_p of the sum of all of
// them.  Out of the kept tokens, in the order of their indices, comes the first whose running sum of w exceeds u times their sum.
//
// Every set above is a beginning of the order, so it is (threshold, number of tokens that equal it); neither a sort nor a list of
// the kept tokens is needed.  The tokens that can matter (w above 2^-46, or min_p) are counted in 512 bins of equal width between
// the smallest and the largest of them.  Counts lead to the bin of the top_k-th token; counts times the weight in the middle of a
// bin lead to the three bins that should hold the end of the nucleus, which the one pass that takes the weights of all kept tokens
// confirms or moves.  Inside them the threshold is found digit by digit over the logits' ordered bit patterns, by exact sums.
//
// Weights are whole numbers, w 2^45 rounded to nearest, taken from an exponential in 64 bits.  Sums of whole numbers do not depend on
// their order: neither the atomics nor the number of CTAs change a result.  45 bits leave the sum of the longest row room in 64 bits,
// and each of three 15-bit limbs of the tokens of a CTA room in 32, which is what histograms of weights add with the 32-bit atomics
// of shared memory.
//
// A cluster of CTAs takes a row: each holds its slice of the logits in shared memory, so that they are read once, and reads the
// others' histograms there.
#include <float.h>

#include <algorithm>

#include "pi_kv8.cuh"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = kThreads, kBinBits = 9, kMaxCluster = 8;   // a bin per thread
constexpr int kWeightBits = 45, kLimb = 15;
constexpr int kSliceFloats = 48 * 1024;   // logits that fit a CTA's shared memory beside the histograms

struct SampleParams {
  const void* logits;
  int dtype;
  size_t stride;
  int n, per;                // logits of a row, of a CTA's slice
  bool wide;                 // slices can be loaded 16 bytes at a time
  const float *temperature, *top_p, *min_p, *u;
  const int32_t* top_k;
  int32_t* ids;
  float* probs;
};

// What a CTA shows the others.
struct Shown {
  unsigned long long best;            // ordered logit << 32 | ~index
  unsigned long long sums[2][3];      // of the kept weights: all, above the interval, in it (two buffers)
  unsigned long long weight;          // above the threshold
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

// 2^(j / 16), and ln(2)^k / k!
__device__ const double kRoots[16] = {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
                                      1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

struct Row {
  const float* x;       // the slice
  int count;
  float most, scale;    // bins per unit of logit
  double rate;          // log2(e) / T
  const double* roots;
  // 2^y for y = (v - most) rate <= 0: a sixteenth from the table, the rest g, |g| <= 1/32, by its series up to g^6 (the next term is below
  // 2^-51), as a multiple of 2^-45
  __device__ __forceinline__ unsigned long long weight(float v) const {
    if (v == most) return 1ull << kWeightBits;
    const double y = ((double)v - (double)most) * rate;
    if (!(y > -60.0)) return 0;
    const double shifted = y + 422212465065984.0;                  // 1.5 2^48: the low bits of the sum count sixteenths
    const int k = __double2loint(shifted);
    const double g = y - (shifted - 422212465065984.0);
    double e = 1.5403530393381608e-4;                              // ln(2)^6 / 6!
    e = fma(e, g, 1.3333558146428443e-3);
    e = fma(e, g, 9.618129107628477e-3);
    e = fma(e, g, 5.550410866482158e-2);
    e = fma(e, g, 2.402265069591007e-1);
    e = fma(e, g, 6.931471805599453e-1);
    const double root = roots[k & 15];
    e = fma(e * g, root, root);
    const int n = (k >> 4) + kWeightBits;                          // times 2^n, n >= -15
    const double w = __hiloint2double(__double2hiint(e) + (n << 20), __double2loint(e)) + 4503599627370496.0;   // 2^52: rounds to a whole number
    return (unsigned long long)__double_as_longlong(w) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ int bin(float v) const { return min(kBins - 1, (int)((most - v) * scale)); }   // never falls as v does
};

struct Shared {
  uint32_t hist[2][3][kBins];
  double roots[16];
  unsigned long long warp_a[kWarps], warp_sum[kWarps];
  unsigned long long warp_s[3][kWarps];
  float warp_f[kWarps];
  unsigned int warp_b[kWarps];
  Shown shown;
  unsigned long long above;
  int bin;
};

// Running sums over the threads of the CTA; `all`: of all of them.
template <typename T>
__device__ __forceinline__ T scan(T v, T* s_warp, T& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  all = 0;
  for (int w = 0; w < kWarps; ++w) {
    const T t = s_warp[w];
    if (w < warp) v += t;
    all += t;
  }
  __syncthreads();
  return v;
}

// The tokens of bins first .. last, ordered by their bit patterns k, lo <= k <= hi: the largest k for which `above` and the amounts (counts, or
// weights) of tokens of at least k reach `want`; `above` becomes the amount above k.  By weight, tokens that equal `low` are left
// out and `low_weight` stands for them.
template <bool WEIGHT>
__device__ uint32_t refine(const Row& row, Shared& s, int first, int last, uint32_t lo, uint32_t hi, uint32_t low, unsigned long long low_weight, unsigned long long want,
                           int& turn, unsigned long long& above) {
  const int tid = threadIdx.x;
  const uint32_t ranks = cluster_size();
  while (lo < hi) {
    const int shift = max(0, 32 - __clz(hi - lo) - kBinBits);
    uint32_t(*h)[kBins] = s.hist[turn & 1];
    ++turn;
#pragma unroll
    for (int i = 0; i < (WEIGHT ? 3 : 1); ++i) h[i][tid] = 0;
    __syncthreads();
    for (int i = tid; i < row.count; i += kThreads) {
      const float x = row.x[i];
      const uint32_t k = ordered(x);
      if (k < lo || k > hi) continue;
      const int b = row.bin(x);
      if (b < first || b > last) continue;
      const uint32_t digit = (k - lo) >> shift;
      if (!WEIGHT) {
        atomicAdd(&h[0][digit], 1u);
      } else if (k != low) {
        const unsigned long long w = row.weight(x);
        atomicAdd(&h[0][digit], (uint32_t)w & 0x7fffu);
        atomicAdd(&h[1][digit], (uint32_t)(w >> kLimb) & 0x7fffu);
        atomicAdd(&h[2][digit], (uint32_t)(w >> 2 * kLimb));
      }
    }
    cluster_sync();
    const int digit = kBins - 1 - tid;   // the largest first
    unsigned long long v = 0, all;
    for (uint32_t r = 0; r < ranks; ++r) {
      v += peer(&h[0][digit], r);
      if (WEIGHT) v += ((unsigned long long)peer(&h[1][digit], r) << kLimb) + ((unsigned long long)peer(&h[2][digit], r) << 2 * kLimb);
    }
    if (WEIGHT && digit == 0 && lo == low) v += low_weight;
    const unsigned long long upto = above + scan(v, s.warp_a, all);
    if (upto >= want && upto - v < want) {
      s.bin = digit;
      s.above = upto - v;
    }
    __syncthreads();
    above = s.above;
    lo += (uint32_t)s.bin << shift;
    hi = min(hi, lo + ((1u << shift) - 1));
    __syncthreads();
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) float s_slice[];
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int r = blockIdx.x / ranks;
  const int from = min((int)rank * p.per, p.n), count = min(p.per, p.n - from);
  const size_t base = (size_t)r * p.stride + from;
  if (tid < 16) s.roots[tid] = kRoots[tid];
  pi_grid_dependency_wait();

  // the slice, and the largest logit with the lowest index; NaN counts as minus infinity, -0 as 0
  unsigned long long best = 0;
  auto take = [&](int i, float x) {
    x = x == x ? x + 0.f : -INFINITY;
    s_slice[i] = x;
    best = max(best, (unsigned long long)ordered(x) << 32 | (uint32_t)~(from + i));
  };
  if (p.wide) {
    const int whole = count & ~3;
#pragma unroll 4
    for (int i = 4 * tid; i < whole; i += 4 * kThreads) {
      float x[4];
      pi_load4_as_f32(x, p.logits, base + i, p.dtype, 4, true);
#pragma unroll
      for (int e = 0; e < 4; ++e) take(i + e, x[e]);
    }
    if (whole + tid < count) take(whole + tid, pi_load_as_f32(p.logits, base + whole + tid, p.dtype));
  } else {
#pragma unroll 4
    for (int i = tid; i < count; i += kThreads) take(i, pi_load_as_f32(p.logits, base + i, p.dtype));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.warp_a[warp] = best;
  s.hist[0][0][tid] = 0;
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
  // tokens below `bound` weigh less than half a unit, or less than min_p
  double exact_bound = (double)most - 32.0 * (double)temperature;
  const float min_p = p.min_p[r];
  if (min_p > 0.f) exact_bound = max(exact_bound, (double)most + (double)temperature * log(min((double)min_p, 1.0)));
  const float bound = most == INFINITY ? INFINITY : max(__double2float_ru(exact_bound), -FLT_MAX);
  const Row row = {s_slice, count, most, (float)kBins / (most - bound), 1.4426950408889634 / (double)temperature, s.roots};

  const int k = p.top_k[r];
  const float top_p = p.top_p[r];
  const bool by_count = k > 0 && k < p.n, by_weight = top_p < 1.f;
  uint32_t thr = ordered(bound) - 1;           // kept: above thr, and the first `ties` that equal it
  unsigned long long ties = 0, above = 0;
  int turn = 1, first = 0;                     // bins in front of `first`: their weights are in warp_sum already
  unsigned long long interval_above = 0;
  if (tid < kWarps) s.warp_sum[tid] = 0;
  if (by_count || by_weight) {
    for (int i = tid; i < count; i += kThreads)
      if (s_slice[i] >= bound) atomicAdd(&s.hist[0][0][row.bin(s_slice[i])], 1u);
    cluster_sync();
    unsigned int here = 0, all;
    for (uint32_t q = 0; q < ranks; ++q) here += peer(&s.hist[0][0][tid], q);
    unsigned int upto = scan(here, s.warp_b, all);
    // logits at the edges of a bin, a little outside
    const float step = (most - bound) / (float)kBins, slack = fmaxf(fabsf(most), fabsf(bound)) * 1e-6f;
    auto upper = [&](int b) {
      const float x = most - (float)b * step + slack + 0.f;
      return b == 0 || !(x < most) ? high : ordered(x);
    };
    auto lower = [&](int b) {
      const float x = most - (float)(b + 1) * step - slack + 0.f;
      return b == kBins - 1 || !(x > bound) ? ordered(bound) : ordered(x);
    };
    int last_bin = kBins - 1;
    if (by_count && all > (unsigned int)k) {
      if (upto >= (unsigned int)k && upto - here < (unsigned int)k) {
        s.bin = tid;
        s.above = upto - here;
      }
      __syncthreads();
      last_bin = s.bin;
      above = s.above;
      __syncthreads();
      thr = refine<false>(row, s, last_bin, last_bin, lower(last_bin), upper(last_bin), 0, 0, (unsigned long long)k, turn, above);
      ties = (unsigned long long)k - above;
      const unsigned int before = min(upto - here, (unsigned int)k);
      here = min(upto, (unsigned int)k) - before;
    }
    if (by_weight) {
      // where the nucleus should end
      float sum;
      const float hint = (float)here * exp2f(-((float)tid + 0.5f) * step * (float)row.rate), hints = scan(hint, s.warp_f, sum);
      const unsigned long long low_weight = ties * row.weight(from_ordered(thr));
      const int low_bin = ties ? row.bin(from_ordered(thr)) : kBins;
      float goal = fmaxf(top_p, 0.f) * sum;   // identical in all CTAs, as all that steers them is
      unsigned long long want = 0, inside = 0;
      int last = 0;
      for (int round = 0;; ++round) {
        const int middle = min(__syncthreads_count(hints < goal), last_bin);
        first = max(0, middle - 1);
        last = min(last_bin, middle + 1);
        if (round >= 6) first = 0, last = last_bin;   // whatever the estimate says
        // exact sums: a run of the slice per warp, so that they serve the draw as well
        const int run = ((count + kWarps * 32 - 1) / (kWarps * 32)) * 32, i0 = min(warp * run, count), i1 = min(i0 + run, count);
        unsigned long long in_front = 0, in = 0, behind = 0;
        for (int i = i0 + lane; i < i1; i += 32) {
          const float x = s_slice[i];
          if (ordered(x) > thr) {
            const int b = row.bin(x);
            const unsigned long long w = row.weight(x);
            if (b < first) in_front += w;
            else if (b <= last) in += w;
            else behind += w;
          }
        }
        in_front = warp_sum(in_front);
        in = warp_sum(in);
        behind = warp_sum(behind);
        if (lane == 0) {
          s.warp_sum[warp] = in_front;
          s.warp_s[0][warp] = in_front + in + behind;
          s.warp_s[1][warp] = in_front;
          s.warp_s[2][warp] = in;
        }
        __syncthreads();
        if (tid < 3) {
          unsigned long long t = 0;
          for (int w = 0; w < kWarps; ++w) t += s.warp_s[tid][w];
          s.shown.sums[round & 1][tid] = t;
        }
        cluster_sync();
        unsigned long long t[3] = {low_weight, low_bin < first ? low_weight : 0, low_bin >= first && low_bin <= last ? low_weight : 0};
        for (uint32_t q = 0; q < ranks; ++q)
#pragma unroll
          for (int e = 0; e < 3; ++e) t[e] += peer(&s.shown.sums[round & 1][e], q);
        want = min(max(1ull, (unsigned long long)ceil((double)fmaxf(top_p, 0.f) * (double)t[0])), t[0]);
        interval_above = t[1];
        inside = t[2];
        if (interval_above < want && want <= interval_above + inside) break;
        // the estimate again, from the exact sum in front of the interval
        if (tid == first) s.warp_f[0] = hints - hint;
        __syncthreads();
        goal = s.warp_f[0] + ((float)((double)want - (double)interval_above)) * (1.f / (float)(1ull << kWeightBits));
        if (want <= interval_above) goal = fminf(goal, s.warp_f[0] * 0.9999999f);
        __syncthreads();
      }
      above = interval_above;
      const uint32_t low = thr;
      thr = refine<true>(row, s, first, last, max(low, last == last_bin ? low : lower(last)), upper(first), low, low_weight, want, turn, above);
      const unsigned long long w = row.weight(from_ordered(thr));
      ties = (want - above + w - 1) / w;
    }
  }

  // sums in the order of the indices: a run of the slice per warp
  const int run = ((count + kWarps * 32 - 1) / (kWarps * 32)) * 32, i0 = min(warp * run, count), i1 = min(i0 + run, count);
  unsigned long long sum = 0;
  unsigned int same = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const uint32_t key = ordered(s_slice[i]);
    if (key > thr && (first == 0 || row.bin(s_slice[i]) >= first)) sum += row.weight(s_slice[i]);
    same += key == thr;
  }
  sum = warp_sum(sum);
  same = __reduce_add_sync(0xffffffffu, same);
  __syncthreads();
  if (lane == 0) {
    s.warp_a[warp] = sum + (first > 0 ? s.warp_sum[warp] : 0);
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
  // a CTA per 16384 logits, two of which an SM has room for; shorter slices where there are few rows
  int cluster = 1;
  while (cluster < kMaxCluster && (n > 16384 * cluster || (n > 2048 * cluster && 2 * rows * cluster <= ctx->sm_count))) cluster *= 2;
  const int per = std::min((n + cluster * 8 - 1) / (cluster * 8) * 8, kSliceFloats);
  const size_t size = dtype == PI_F32 ? 4 : 2;
  const bool wide = (uintptr_t)logits_dev % (4 * size) == 0 && (rows == 1 || row_stride % 4 == 0);
  SampleParams p = {logits_dev, dtype, row_stride, n, per, wide, temperature_dev, top_p_dev, min_p_dev, u_dev, top_k_dev, ids_dev, probs_dev_or_null};
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
