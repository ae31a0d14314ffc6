// A token per row of logits: temperature, top-k, min-p and top-p, from a given random number.
//
// With M the row's maximum and w(x) = exp((x - M) / T), tokens are ordered by logit, equal ones by index.  Kept are the first top_k of
// that order, of those the ones with w >= min_p, and of those the shortest beginning whose sum reaches top_p of the sum of all of
// them.  Out of the kept tokens, in the order of their indices, comes the first whose running sum of w exceeds u times their sum.
//
// Every set above is a beginning of the order, so it is (threshold, number of tokens that equal it); neither a sort nor a list of
// the kept tokens is needed.  The tokens that can matter (w above 2^-46, or min_p) are counted in 1024 bins of equal width between
// the smallest and the largest of them.  Counts lead to the bin of the top_k-th token; counts times the weight in the middle of a
// bin lead to the three bins that should hold the end of the nucleus, which the one pass that takes the weights of all kept tokens
// confirms or moves.  Inside them the threshold is found digit by digit over the logits' ordered bit patterns, by exact sums.
//
// Weights are whole numbers, w 2^45 rounded to nearest, taken from an exponential in 64 bits.  Sums of whole numbers do not depend on
// their order: neither the atomics nor the number of CTAs change a result.  45 bits leave the sum of the longest row room in 64 bits,
// and each of three 15-bit limbs of the tokens of a CTA room in 32, which is what histograms of weights add with the 32-bit atomics
// of shared memory.
//
// A cluster of CTAs takes a row: each holds its slice of the logits in shared memory, so that they are read once.  A histogram is
// made in each CTA's own memory; then every bin has a home in one of them, to which the others add theirs, and everybody reads all
// bins from their homes.  (Reading all histograms of all eight CTAs instead: 143 us for 64 rows of 128256 when this took 82.)
//
// Bound: the barriers of the cluster and of the CTA, some eight and twenty-five of them with a pass over the slice between each two; the
// pass that takes the weights is the longest.  Measured: 1 row of 32000 logits 17 us, 64 of 128256 72 us.
#include <float.h>

#include <algorithm>

#include "pi_kv8.cuh"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2 * kThreads, kBinBits = 10, kMaxCluster = 8;   // two bins per thread
constexpr int kWeightBits = 45, kLimb = 15;
constexpr int kSliceFloats = 48 * 1024;   // logits that fit a CTA's shared memory beside the histograms
constexpr int kAtOnce = 4;                // weights that a thread takes at a time
constexpr int kTable = 64;                // floats that 32 doubles take

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
  unsigned int most;                  // ordered logit
  unsigned int at;                    // lowest index of the row's largest
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

__device__ __forceinline__ unsigned long long cluster_sum(unsigned long long v) {   // of eight neighbouring lanes
#pragma unroll
  for (int o = kMaxCluster / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 2^(j / 32)
__device__ const double kRoots[32] = {1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
                                      1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
                                      1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
                                      1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
                                      1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103,
                                      1.9152065613971474, 1.9571441241754002};

struct Row {
  const float* x;       // the slice
  int count;
  float most, scale;    // bins per unit of logit; 0: all tokens are in one bin
  double top, rate;     // `most`, log2(e) / T
  // 2^y for y = (v - most) rate <= 0: a 32nd from the table, the rest g, |g| <= 1/64, by its series up to g^5 (the next term is below 2^-48),
  // as a multiple of 2^-45; y above -60
  __device__ __forceinline__ double exponent(float v) const { return ((double)fminf(v, FLT_MAX) - top) * rate; }   // infinite logits: the largest alone
  __device__ __forceinline__ double power(double y) const {
    extern __shared__ __align__(16) float s_slice[];
    const double shifted = y + 211106232532992.0;                  // 1.5 2^47: the low bits of the sum count 32nds
    const int k = __double2loint(shifted);
    const double g = y - (shifted - 211106232532992.0);
    double e = 1.3333558146428441e-3;                              // ln(2)^5 / 5!
    e = fma(e, g, 9.618129107628477e-3);
    e = fma(e, g, 5.5504108664821576e-2);
    e = fma(e, g, 2.402265069591007e-1);
    e = fma(e, g, 6.931471805599453e-1);
    const double root = reinterpret_cast<const double*>(s_slice)[k & 31];   // times 2^45; the table lies in front of the slice
    e = fma(e * g, root, root);
    const double w = __hiloint2double(__double2hiint(e) + ((k & ~31) << 15), __double2loint(e));   // times 2^floor(y)
    return (w + 4503599627370496.0) - 4503599627370496.0;          // 2^52: rounds to a whole number
  }
  __device__ __forceinline__ unsigned long long weight(float v) const { return exponent(v) > -60.0 ? (unsigned long long)power(exponent(v)) : 0; }
  // use(logit, weight) for the tokens i, i + 32, ... below `end` with least < logit <= most_used, several at a time, so that the chains of
  // their weights overlap; they are at least `bound`, with a y above -47.  A thread's sums of weights are exact in f64: at most 96 of them, of
  // 2^45 at most.  The whole warp calls it.
  template <typename F>
  __device__ __forceinline__ void weigh(int i, int end, float least, float most_used, F use) const {
    const int lane = threadIdx.x & 31;
    for (; i - lane < end; i += 32 * kAtOnce) {
      float v[kAtOnce];
      bool in[kAtOnce], any = false;
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        v[e] = i + 32 * e < end ? x[i + 32 * e] : -INFINITY;
        any |= in[e] = v[e] > least && !(v[e] > most_used);
      }
      if (!__any_sync(0xffffffffu, any)) continue;
      double w[kAtOnce];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) w[e] = power(exponent(v[e]));
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e)
        if (in[e]) use(v[e], w[e]);
    }
  }
  // Never falls as v does.  The truncated sum's low bits are a whole number; the last bin for what is not a number (infinity minus itself).
  __device__ __forceinline__ int bin(float v) const { return min(kBins - 1, (int)(__float_as_uint(__fmaf_rz(most - v, scale, 8388608.f)) - 0x4b000000u)); }
};

struct Shared {
  uint32_t hist[3][kBins];             // of this CTA
  unsigned long long warp_a[kWarps], warp_sum[kWarps];
  unsigned long long warp_s[3][kWarps];
  float warp_f[kWarps];
  unsigned int warp_b[kWarps];
  Shown shown;
  unsigned long long above, taken;
  int bin;
  int2 dealt;
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
  T t = s_warp[lane & (kWarps - 1)];   // lanes 16 and up hold the same again
  T upto = t;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, upto, o, kWarps);
    if ((lane & (kWarps - 1)) >= o) upto += u;
  }
  all = __shfl_sync(0xffffffffu, upto, kWarps - 1);
  const T before = __shfl_sync(0xffffffffu, upto - t, warp);
  v += before;
  __syncthreads();
  return v;
}

// In dynamic shared memory: the table of roots, the cluster's totals of the bins that live here (three turns of kBins / CTAs), the slice.
__device__ __forceinline__ unsigned long long* home_bins() {
  extern __shared__ __align__(16) float s_slice[];
  return reinterpret_cast<unsigned long long*>(s_slice + kTable);
}

// Two bins per thread, the ones of thread 0 first: the CTA's amounts in, the cluster's out.  A turn's buffer is cleared a turn ahead:
// by then everybody has passed the barrier behind which nobody reads what it held two turns ago.
__device__ __forceinline__ void exchange(unsigned long long* v, int& turn) {
  const uint32_t tid = threadIdx.x, share = kBins / cluster_size(), home = 2 * tid / share;
  unsigned long long *homes = home_bins(), *at = homes + turn % 3 * share + (2 * tid - home * share);
  if (2 * tid < share) homes[(turn + 1) % 3 * share + 2 * tid] = homes[(turn + 1) % 3 * share + 2 * tid + 1] = 0;
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(home));
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (v[e]) asm volatile("red.relaxed.cluster.shared::cluster.add.u64 [%0], %1;" ::"r"(a + 8 * e), "l"(v[e]) : "memory");
  cluster_sync();
  asm volatile("ld.shared::cluster.v2.u64 {%0,%1}, [%2];" : "=l"(v[0]), "=l"(v[1]) : "r"(a) : "memory");
  ++turn;
}

// The tokens of bins first .. last, ordered by their bit patterns k, lo <= k <= hi: the largest k for which `above` and the amounts (counts, or
// weights) of tokens of at least k reach `want`; `above` becomes the amount above k.  By weight, tokens that equal `low` are left
// out and `low_weight` stands for them.
template <bool WEIGHT>
__device__ uint32_t refine(const Row& row, Shared& s, int first, int last, uint32_t lo, uint32_t hi, uint32_t low, unsigned long long low_weight, unsigned long long want,
                           int& turn, unsigned long long& above) {
  const int tid = threadIdx.x, digit = kBins - 1 - 2 * tid;   // the largest first
  while (lo < hi) {
    const int shift = max(0, 32 - __clz(hi - lo) - kBinBits);
#pragma unroll
    for (int i = 0; i < (WEIGHT ? 3 : 1); ++i) s.hist[i][tid] = s.hist[i][tid + kThreads] = 0;
    if (tid == 0) {   // amounts that do not reach `want` leave the smallest
      s.bin = 0;
      s.above = above;
    }
    __syncthreads();
    const float from = from_ordered(lo), to = from_ordered(hi);
#pragma unroll 4
    for (int i = tid; i < row.count; i += kThreads) {
      const float x = row.x[i];
      if (x >= from && x <= to) {
        const int b = row.bin(x);
        const uint32_t k = ordered(x), d = (k - lo) >> shift;
        if (b >= first && b <= last && k - lo <= hi - lo) {   // 0 passes for -0 above
          if (!WEIGHT) {
            atomicAdd(&s.hist[0][d], 1u);
          } else if (k != low) {
            const unsigned long long w = row.weight(x);
            atomicAdd(&s.hist[0][d], (uint32_t)w & 0x7fffu);
            atomicAdd(&s.hist[1][d], (uint32_t)(w >> kLimb) & 0x7fffu);
            atomicAdd(&s.hist[2][d], (uint32_t)(w >> 2 * kLimb));
          }
        }
      }
    }
    __syncthreads();
    unsigned long long v[2], all;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[e] = s.hist[0][digit - e];
      if (WEIGHT) v[e] += ((unsigned long long)s.hist[1][digit - e] << kLimb) + ((unsigned long long)s.hist[2][digit - e] << 2 * kLimb);
    }
    exchange(v, turn);
    if (WEIGHT && tid == kThreads - 1 && lo == low) v[1] += low_weight;
    unsigned long long upto = above + scan(v[0] + v[1], s.warp_a, all) - v[1];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (upto >= want && upto - v[e] < want) {
        s.bin = digit - e;
        s.above = upto - v[e];
      }
      upto += v[1];
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
  float* const slice = s_slice + kTable + 6 * kBins / ranks;
  if (tid < 32) reinterpret_cast<double*>(s_slice)[tid] = kRoots[tid] * (double)(1ull << kWeightBits);
  pi_grid_dependency_wait();
  const float temperature = p.temperature[r], min_p = p.min_p[r], top_p = p.top_p[r], u = p.u[r];
  const int k = p.top_k[r];

  // the slice, and the largest logit; NaN counts as minus infinity, -0 as 0
  float best = -INFINITY;
  if (p.wide) {
    const int whole = count & ~3;
#pragma unroll 4
    for (int i = 4 * tid; i < whole; i += 4 * kThreads) {
      float x[4];
      pi_load4_as_f32(x, p.logits, base + i, p.dtype, 4, true);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = fmaxf(x[e], -INFINITY) + 0.f;
        best = fmaxf(best, x[e]);
      }
      *reinterpret_cast<float4*>(slice + i) = make_float4(x[0], x[1], x[2], x[3]);
    }
    if (whole + tid < count) best = fmaxf(best, slice[whole + tid] = fmaxf(pi_load_as_f32(p.logits, base + whole + tid, p.dtype), -INFINITY) + 0.f);
  } else {
#pragma unroll 4
    for (int i = tid; i < count; i += kThreads) best = fmaxf(best, slice[i] = fmaxf(pi_load_as_f32(p.logits, base + i, p.dtype), -INFINITY) + 0.f);
  }
  best = pi_warp_max(best);
  if (lane == 0) s.warp_f[warp] = best;
  s.hist[0][tid] = s.hist[0][tid + kThreads] = 0;
  if (2 * tid < kBins / ranks) home_bins()[2 * tid] = home_bins()[2 * tid + 1] = 0;
  __syncthreads();
  if (warp == 0) {
    best = pi_warp_max(s.warp_f[lane & (kWarps - 1)]);
    if (lane == 0) {
      s.shown.most = ordered(best);
      s.shown.at = 0x7fffffff;
    }
  }
  cluster_sync();
  const uint32_t high = __reduce_max_sync(0xffffffffu, lane < ranks ? peer(&s.shown.most, lane) : 0);
  const float most = from_ordered(high);
  if (!(temperature > 0.f) || most == -INFINITY) {   // the largest, the lowest index of equal ones; a row without any
    for (int i = tid; i < count; i += kThreads)
      if (slice[i] == most) {
        atomicMin(&s.shown.at, (unsigned int)(from + i));
        break;
      }
    cluster_sync();
    if (rank == 0 && tid == 0) {
      unsigned int at = 0x7fffffff;
      for (uint32_t q = 0; q < ranks; ++q) at = min(at, peer(&s.shown.at, q));
      p.ids[r] = most == -INFINITY ? -1 : (int32_t)at;
      if (p.probs) p.probs[r] = most == -INFINITY ? 0.f : 1.f;
    }
    cluster_sync();
    return;
  }
  // tokens below `bound` weigh less than half a unit, or less than min_p
  double exact_bound = (double)most - 32.0 * (double)temperature;
  if (min_p > 0.f) exact_bound = max(exact_bound, (double)most + (double)temperature * log(min((double)min_p, 1.0)));
  const float bound = most == INFINITY ? INFINITY : max(__double2float_ru(exact_bound), -FLT_MAX) + 0.f;   // not -0
  const double rate = 1.4426950408889634 / (double)temperature;
  // An interval beyond a float's range is cut at that: what lies further down is in the last bin.  One so short (below 3e-36, with
  // temperatures below 1e-37) that a unit would hold more bins than a float can say is one bin.
  const float width = fminf(most - bound, FLT_MAX), bins = most > bound ? (float)kBins / width : 0.f;
  const Row row = {slice, count, most, bins <= FLT_MAX ? bins : 0.f, (double)fminf(most, FLT_MAX), rate};

  const bool by_count = k > 0 && k < p.n, by_weight = top_p < 1.f;
  // kept: above thr, and the first `ties` that equal it; the number below 0 is not -0, which equals it
  uint32_t thr = ordered(bound) - (bound == 0.f ? 2 : 1);
  unsigned long long ties = 0, above = 0;
  int turn = 0, first = 0;                     // bins in front of `first`: their weights are in warp_sum already
  unsigned long long interval_above = 0;
  if (tid < kWarps) s.warp_sum[tid] = 0;
  float sure = INFINITY;                       // logits above it lie in those bins
  if (by_count || by_weight) {
#pragma unroll 4
    for (int i = tid; i < count; i += kThreads) {
      const float x = slice[i];
      if (x >= bound) atomicAdd(&s.hist[0][row.bin(x)], 1u);
    }
    __syncthreads();
    unsigned long long v[2] = {s.hist[0][2 * tid], s.hist[0][2 * tid + 1]};
    exchange(v, turn);
    unsigned int here[2] = {(unsigned int)v[0], (unsigned int)v[1]}, upto[2], all;
    upto[1] = scan(here[0] + here[1], s.warp_b, all);
    upto[0] = upto[1] - here[1];
    // logits at the edges of a bin, a little outside
    const float step = width / (float)kBins, slack = fmaxf(fabsf(most), fabsf(bound)) * 1e-6f;
    auto upper = [&](int b) {
      const float x = most - (float)b * step + slack + 0.f;
      return b == 0 || row.scale == 0.f || !(x < most) ? high : ordered(x);
    };
    auto lower = [&](int b) {
      const float x = most - (float)(b + 1) * step - slack + 0.f;
      return b == kBins - 1 || row.scale == 0.f || !(x > bound) ? ordered(bound) : ordered(x);
    };
    int last_bin = kBins - 1;
    if (by_count && all > (unsigned int)k) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (upto[e] >= (unsigned int)k && upto[e] - here[e] < (unsigned int)k) {
          s.bin = 2 * tid + e;
          s.above = upto[e] - here[e];
        }
      __syncthreads();
      last_bin = s.bin;
      above = s.above;
      __syncthreads();
      thr = refine<false>(row, s, last_bin, last_bin, lower(last_bin), upper(last_bin), 0, 0, (unsigned long long)k, turn, above);
      ties = (unsigned long long)k - above;
#pragma unroll
      for (int e = 0; e < 2; ++e) here[e] = min(upto[e], (unsigned int)k) - min(upto[e] - here[e], (unsigned int)k);
    }
    if (by_weight) {
      // where the nucleus should end
      float sum;
      float hint[2], hints[2];
      const float fall = (float)((double)step * row.rate);
#pragma unroll
      for (int e = 0; e < 2; ++e) hint[e] = (float)here[e] * exp2f(-((float)(2 * tid + e) + 0.5f) * fall);
      hints[1] = scan(hint[0] + hint[1], s.warp_f, sum);
      hints[0] = hints[1] - hint[1];
      const unsigned long long low_weight = ties * row.weight(from_ordered(thr));
      const int low_bin = ties ? row.bin(from_ordered(thr)) : kBins;
      float goal = fmaxf(top_p, 0.f) * sum;   // identical in all CTAs, as all that steers them is
      unsigned long long want = 0, inside = 0;
      int last = 0;
      for (int round = 0;; ++round) {
        if (tid == 0) s.bin = 0;
        __syncthreads();
        const int under = __popc(__ballot_sync(0xffffffffu, hints[0] < goal)) + __popc(__ballot_sync(0xffffffffu, hints[1] < goal));
        if (lane == 0) atomicAdd(&s.bin, under);
        __syncthreads();
        const int middle = min(s.bin, last_bin);
        first = max(0, middle - 1);
        last = min(last_bin, middle + 1);
        if (round >= 6) first = 0, last = last_bin;   // whatever the estimate says
        // exact sums: a run of the slice per warp, so that they serve the draw as well
        const int run = ((count + kWarps * 32 - 1) / (kWarps * 32)) * 32, i0 = min(warp * run, count), i1 = min(i0 + run, count);
        double front_of = 0, in_of = 0, all_of = 0;
        const float least = from_ordered(thr);
        row.weigh(i0 + lane, i1, least, INFINITY, [&](float x, double w) {
          const int b = row.bin(x);
          all_of += w;
          if (b < first) front_of += w;
          if (b >= first && b <= last) in_of += w;
        });
        const unsigned long long in_front = warp_sum((unsigned long long)front_of), in = warp_sum((unsigned long long)in_of), in_all = warp_sum((unsigned long long)all_of);
        if (lane == 0) {
          s.warp_sum[warp] = in_front;
          s.warp_s[0][warp] = in_all;
          s.warp_s[1][warp] = in_front;
          s.warp_s[2][warp] = in;
        }
        __syncthreads();
        if (warp < 3) {
          const unsigned long long t = warp_sum(lane < kWarps ? s.warp_s[warp][lane] : 0);
          if (lane == 0) s.shown.sums[round & 1][warp] = t;
        }
        cluster_sync();
        unsigned long long t[3] = {low_weight, low_bin < first ? low_weight : 0, low_bin >= first && low_bin <= last ? low_weight : 0};
#pragma unroll
        for (int e = 0; e < 3; ++e) t[e] += cluster_sum((lane & 7) < ranks ? peer(&s.shown.sums[round & 1][e], lane & 7) : 0);
        want = min(max(1ull, (unsigned long long)ceil((double)fmaxf(top_p, 0.f) * (double)t[0])), t[0]);
        interval_above = t[1];
        inside = t[2];
        if ((interval_above < want && want <= interval_above + inside) || round == 7) break;   // from round 6 on it is all of them
        // the estimate again, from the exact sum in front of the interval
        if (tid == first / 2) s.warp_f[0] = hints[first & 1] - hint[first & 1];
        __syncthreads();
        goal = s.warp_f[0] + ((float)((double)want - (double)interval_above)) * (1.f / (float)(1ull << kWeightBits));
        if (want <= interval_above) goal = fminf(goal, s.warp_f[0] * 0.9999999f);
        __syncthreads();
      }
      above = interval_above;
      if (first > 0) sure = from_ordered(upper(first));
      const uint32_t low = thr;
      thr = refine<true>(row, s, first, last, max(low, last == last_bin ? low : lower(last)), upper(first), low, low_weight, want, turn, above);
      const unsigned long long w = row.weight(from_ordered(thr));
      ties = want - above <= w || w == 0 ? 1 : (want - above + w - 1) / w;
    }
  }

  // sums in the order of the indices, a run of start .. end per warp, of the tokens of bins from `ahead_of` on, which lie at or below `most_used`
  const float least = from_ordered(thr);
  int i0, i1;
  auto sum_run = [&](int start, int end, int ahead_of, float most_used) {
    const int run = (end - start + kThreads - 1) / kThreads * 32;
    i0 = min(start + warp * run, end), i1 = min(i0 + run, end);
    double sum_of = 0;
    unsigned int same = 0;
    row.weigh(i0 + lane, i1, least, most_used, [&](float x, double w) {
      if (row.bin(x) >= ahead_of) sum_of += w;
    });
    if (ties > 0)
#pragma unroll 4
      for (int i = i0 + lane; i < i1; i += 32) same += slice[i] == least;
    const unsigned long long sum = warp_sum((unsigned long long)sum_of);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) {
      s.warp_a[warp] = sum + (ahead_of > 0 ? s.warp_sum[warp] : 0);
      s.warp_b[warp] = same;
    }
  };
  __syncthreads();
  sum_run(0, count, first, sure);
  __syncthreads();
  if (warp == 0) {   // lane w looks at warp w
    const unsigned long long a = warp_sum(lane < kWarps ? s.warp_a[lane] : 0);
    const unsigned int b = __reduce_add_sync(0xffffffffu, lane < kWarps ? s.warp_b[lane] : 0);
    if (lane == 0) {
      s.shown.weight = a;
      s.shown.ties = b;
    }
  }
  cluster_sync();
  const unsigned long long w_thr = row.weight(from_ordered(thr));
  // lane q looks at CTA q: how many of its equal tokens are kept, and what it holds
  unsigned int equals = lane < ranks ? peer(&s.shown.ties, lane) : 0, upto_equals = equals;
#pragma unroll
  for (int o = 1; o < kMaxCluster; o <<= 1) {
    const unsigned int t = __shfl_up_sync(0xffffffffu, upto_equals, o);
    if (lane >= o) upto_equals += t;
  }
  const unsigned long long used = min((unsigned long long)(upto_equals - equals), ties), held = (lane < ranks ? peer(&s.shown.weight, lane) : 0) + (min((unsigned long long)upto_equals, ties) - used) * w_thr;
  const unsigned long long total = warp_sum(lane < ranks ? held : 0), ahead = warp_sum(lane < rank ? held : 0), used_here = __shfl_sync(0xffffffffu, used, rank), held_here = __shfl_sync(0xffffffffu, held, rank);
  unsigned long long goal = u > 0.f ? (unsigned long long)floor((double)u * (double)total) : 0;
  goal = min(goal, total - 1);
  // the first token whose running sum exceeds the goal: its CTA finds the warp whose run holds it, deals that run to all warps, and the
  // warp whose part holds it scans that.  (64 rows of 128256 without top-k or top-p:
  // 42 us, 60 where that warp scans its whole run.)
  if (goal >= ahead && goal < ahead + held_here) {
    unsigned long long before = ahead, taken = used_here;
    for (bool dealt = false;; dealt = true) {
      const unsigned long long in_warp = lane < kWarps ? s.warp_a[lane] : 0;
      const unsigned int equal_in_warp = lane < kWarps ? s.warp_b[lane] : 0;
      unsigned int upto_equal = equal_in_warp;
#pragma unroll
      for (int o = 1; o < kWarps; o <<= 1) {
        const unsigned int t = __shfl_up_sync(0xffffffffu, upto_equal, o);
        if (lane >= o) upto_equal += t;
      }
      const unsigned long long taken_before = min(taken + (upto_equal - equal_in_warp), ties), holds = in_warp + (min(taken + upto_equal, ties) - taken_before) * w_thr;
      unsigned long long holds_upto = holds;
#pragma unroll
      for (int o = 1; o < kWarps; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, holds_upto, o);
        if (lane >= o) holds_upto += t;
      }
      unsigned long long mine = before + __shfl_sync(0xffffffffu, holds_upto - holds, warp), taken_mine = __shfl_sync(0xffffffffu, taken_before, warp);
      const bool here = goal >= mine && goal < mine + __shfl_sync(0xffffffffu, holds, warp);
      if (dealt) {
        for (int i = i0 + lane; here && i - lane < i1; i += 32) {
          const float x = i < i1 ? slice[i] : -INFINITY;
          const unsigned equal = __ballot_sync(0xffffffffu, i < i1 && x == least);
          unsigned long long w = 0;
          if (x > least) w = row.weight(x);
          if (i < i1 && x == least && taken_mine + __popc(equal & ((1u << lane) - 1)) < ties) w = w_thr;
          taken_mine += __popc(equal);
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
        break;
      }
      if (here && lane == 0) {
        s.dealt = make_int2(i0, i1);
        s.above = mine;
        s.taken = taken_mine;
      }
      __syncthreads();
      before = s.above, taken = s.taken;
      const int2 dealt_run = s.dealt;
      sum_run(dealt_run.x, dealt_run.y, 0, INFINITY);
      __syncthreads();
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
  const size_t smem = (size_t)(kTable + 6 * kBins / cluster + p.per) * sizeof(float);
  constexpr int kMostShared = (kTable + 6 * kBins / kMaxCluster + kSliceFloats) * (int)sizeof(float);   // of the longest row; smaller clusters have shorter slices
  static pi_smem_grant grant;
  if (smem > grant.of(ctx)) {
    PI_CUDA(ctx, cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
    grant.of(ctx) = kMostShared;
  }
  pi_prof_scope prof(ctx, PI_PROF_OTHER);
  PI_CUDA(ctx, pi_launch_chained(ctx, sample_kernel, dim3((unsigned)rows * cluster), dim3(kThreads), smem, cluster, p));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}
