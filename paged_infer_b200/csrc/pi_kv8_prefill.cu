// Paged attention over the 8-bit cache for sequences that bring many rows (portions of prompts), on tcgen05: accumulators and the A
// operands in tensor memory, B operands in shared memory.  Head sizes that are stored in 64 or 128 bytes.
//
// A CTA owns 128 (row, query head) pairs of one sequence and KV head, one per TMEM lane, and walks the positions that they see in tiles
// of 128 columns (64 for heads of 128 with two planes): eight times 16 tokens, each of one block and with one pair of scales.  Codes are
// widened to f16, which holds them exactly; queries (brought to 2^14 to 2^15 by a power of two per row) and weights are f16 too, in two planes (22 bits) for f32 tensors:
//     scores  S = Q K^T        A = Q (written once),  B = codes of K, [token][channel]
//     output  O = P V          A = P,                 B = codes of V transposed, [channel][token]
// A row's thread multiplies the K scale in as it reads its scores, and weighs exp(score) by V scale / r, r a power of two above the
// largest product of weight and V scale in the tile, so that P stays in f16's range whatever the scales are, and what a large scale
// takes from a small one's bits it takes by what it adds to the result; the product of a tile is read
// back, multiplied by r and added to the row's f32 output in registers.  The running maximum may lag 2^3 behind, so that the output
// is seldom rescaled.
//
// Warps 0-7: two threads per row, each with half of a tile's columns and half of the output's channels; they share the row's running
// maximum through shared memory, once a tile (one thread per row leaves every scheduler one such warp: 151 us where two take 143).
// Warps 8-11 and 12-15: the codes of the first and of the second 64 tokens of every tile (with tiles of 64: of the even and of the odd
// tiles), into registers ahead of their turn, then widened into shared memory (V by byte permutes of eight tokens at a time).
// Warp 16: issues the products (17-19 are there because registers are dealt to four warps at a time); the scores of tile j + 1 run
// while the rows work on tile j.
// Hand-offs go through mbarriers; every wait is bounded and raises the context's error word instead of hanging, and the tile's rows
// become NaN.  Where there are few tiles of rows, a cluster shares the positions of one and joins its CTAs' outputs through shared memory.
//
// Bound: the rows' threads.  A tile of 128 by 128 needs 16384 exponentials, of which an SM makes 16 a clock: 1024 clocks, as long as
// both products of a head of 128 channels; around them come a multiplication, a maximum, an addition and half a conversion each, and
// reading back the tile's output.
//
// Measured: 512 rows behind 3584 positions, 32 query heads of 128 over 8, bf16: 108 us, 298 TFLOP/s; 16 sequences of 1 to 256 rows in a
// window of 1024, 32 over 4 of 64, f32 (two planes): 165 us.  Leaving out the exponentials, the widening, the products or the output's
// way back saved at most 8 % each (of 121 us, with slower waits): the chain of one tile of rows is what takes the time.  Tensor memory has no room
// for a second one in this layout (two buffers of scores, P, the tile's output and Q beside each other).  Heads of 128 keep 64 outputs and 64
// scores in a row thread's 152 registers, which spills some 150 bytes a thread (one plane; 50 with two, none at 64).
#include <math.h>

#include <algorithm>

#include "pi_kv8_widen.cuh"

namespace {

using namespace pi_kv8;

constexpr int kRowsP = 128, kPartP = 64, kThreadsP = 20 * 32, kMostStages = 4, kMostSplitsP = 8;   // a part: the tokens of a tile that four warps widen
constexpr long long kWaitLimitP = 1ll << 31;   // clocks of a wait: about a second

struct PrefillParams {
  pi_kv8_attn_params a;
  int rows_per_tile, min_cols;   // rows of a tile; sequences with fewer columns are another kernel's
  int* err_flag;
  long long wait_limit;          // clocks
};

// 16 tokens of a tile: first position, how many are there (0: not mapped), scale of K, scale of V as 2^v_exp 2^v_log, v_log in [0, 1).
struct Group {
  int base, valid;
  float k_scale;
  float v_exp, v_log;
};
constexpr float kNoScale = -100000.f;   // v_exp of a zero scale

__device__ __forceinline__ uint32_t s_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void st_shared(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {   // the same without suspending
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// A try may suspend the thread for a while that the hardware limits; tries end after `limit` clocks, or when the CTA gives up.
// Converters, who are ahead, sleep between theirs.
template <bool NAP = false>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit) {
  if (bar_test(bar, parity)) return true;
  const long long until = clock64() + limit;
  while (clock64() < until && !(abort_flag && *abort_flag)) {
    if (NAP) __nanosleep(200);
    if (bar_try(bar, parity)) return true;
  }
  return false;
}
// Every lane waits for itself: what was released to the barrier is then there for all of them (a shuffle of one lane's answer would
// order no memory).
template <bool NAP = false>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit) {
  return __all_sync(0xffffffffu, bar_wait<NAP>(bar, parity, abort_flag, limit));
}
// K-major, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d), "r"(tmem_a), "l"(b), "r"(idesc),
               "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void t_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
__device__ __forceinline__ void t_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7]));
}
__device__ __forceinline__ void t_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void t_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int HD, int PLANES>
struct Prefill {
  // columns of a tile: two buffers of scores, P, the output and Q have to fit the 512 columns of tensor memory
  static constexpr int tile = HD == 128 && PLANES == 2 ? 64 : 128, parts = tile / kPartP, groups = tile / 16;
  static constexpr int side = tile * HD * 2, stage = 2 * side;     // bytes of a tile's K, and as many of V
  static constexpr int stages = stage > 32768 ? 3 : 4;
  static constexpr int line = HD + 4;                              // floats of a row where the CTAs of a cluster meet
  static constexpr int rings = stages * stage, meet = kRowsP * line * 4 + kRowsP * 8;
  static constexpr int body = rings > meet ? rings : meet;
  // at least 120 KB: two of these CTAs, each of which takes all of tensor memory, never share an SM
  static constexpr int smem = (body > 119 * 1024 ? body : 119 * 1024) + 1024;
  // tensor memory: two buffers of scores, the planes of P, the tile's output, the planes of Q
  static constexpr uint32_t col_s = 0, col_p = 2 * tile, col_o = col_p + PLANES * tile / 2, col_q = col_o + HD;
  static_assert(col_q + PLANES * HD / 2 <= 512, "tensor memory");
};

template <int KIND, int HD, int PLANES>
__global__ void __launch_bounds__(kThreadsP, 1) kv8_prefill_kernel(const PrefillParams pp) {
  using L = Prefill<HD, PLANES>;
  constexpr int TILE = L::tile, STAGES = L::stages, PARTS = L::parts;
  const pi_kv8_attn_params& p = pp.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long bars[2 * kMostStages + 6];
  __shared__ Group s_group[kMostStages][8];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ float2 s_most[2][2][kRowsP];   // [tile parity][half][row]
  __shared__ int s_lo, s_hi, s_seq, s_first;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bs = p.block_size, G = p.group;
  uint32_t split, splits;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(split));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const int row_tile = (int)(blockIdx.x / splits) / p.kv_heads, kvh = (int)(blockIdx.x / splits) - row_tile * p.kv_heads;
  const uint32_t kv_full0 = s_u32(&bars[0]), kv_free0 = s_u32(&bars[kMostStages]), s_full0 = s_u32(&bars[2 * kMostStages]), p_full = s_u32(&bars[2 * kMostStages + 2]),
                 o_full = s_u32(&bars[2 * kMostStages + 3]), o_free = s_u32(&bars[2 * kMostStages + 4]), idle = s_u32(&bars[2 * kMostStages + 5]);
  pi_grid_dependency_wait_only();

  // the tile of rows: sequences' tiles are numbered through
  if (warp == 0) {
    int ahead = 0, seq = -1, first = 0;
    for (int b0 = 0; b0 < p.n_seqs && seq < 0; b0 += 32) {
      const int b = b0 + lane;
      int n = 0, begin = 0;
      if (b < p.n_seqs) {
        begin = max(0, min(p.cu_rows[b], p.n_rows));
        n = max(0, min(p.cu_rows[b + 1], p.n_rows) - begin);
      }
      const int tiles = n * G > pp.min_cols ? (n + pp.rows_per_tile - 1) / pp.rows_per_tile : 0;
      int upto = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
      }
      const int y = row_tile - ahead;
      const unsigned hit = __ballot_sync(0xffffffffu, y < upto && y >= upto - tiles);
      if (hit) {
        const int at = __ffs(hit) - 1;
        seq = b0 + at;
        // a sequence's last rows see most: they come first
        first = __shfl_sync(0xffffffffu, begin + (upto - 1 - y) * pp.rows_per_tile, at);
      }
      ahead += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      s_seq = seq;
      s_first = first;
      s_lo = 0x7fffffff;
      s_hi = -1;
      s_abort = 0;
      for (int i = 0; i < L::stages; ++i) {
        bar_init(kv_full0 + 8 * i, 4 * L::parts);   // one arrival per converter warp
        bar_init(kv_free0 + 8 * i, 1);   // tcgen05.commit
      }
      for (int i = 0; i < 2; ++i) bar_init(s_full0 + 8 * i, 1);
      bar_init(p_full, 8);               // one arrival per row warp
      bar_init(o_full, 1);
      bar_init(o_free, 8);
      bar_init(idle, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
  }
  __syncthreads();
  const int seq = s_seq;
  if (seq < 0) return;   // the whole cluster: fewer tiles than the grid allows for
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(&s_tmem)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // this thread's row (warps 0-7), and its half of it
  const int row_end = min(p.cu_rows[seq + 1], p.n_rows), m = tid & 127, half = tid >> 7, local = p.by_group(m), head = m - local * G;
  const bool live = warp < 8 && local < pp.rows_per_tile && s_first + local < row_end;
  int pos = -1, from = 0;
  if (live) {
    pos = p.row_pos[s_first + local];
    from = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    if (pos >= 0) {
      atomicMin(&s_lo, from);
      atomicMax(&s_hi, pos);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // the dependent grid is released only now that this CTA holds its tensor memory (a dependent CTA that took the SM's columns first
  // would keep them until this grid completes)
  pi_grid_launch_dependents();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s_tmem, smem_base = s_u32(smem), lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  const int lo_all = s_lo, hi_all = min(s_hi, max(0, min(p.lens[seq], p.max_blocks)) * bs - 1);
  const int per_block = (bs + 15) >> 4, first_block = hi_all < lo_all ? 0 : p.by_block(lo_all);
  const int groups = hi_all < lo_all ? 0 : (p.by_block(hi_all) - first_block + 1) * per_block, tiles_all = (groups + L::groups - 1) / L::groups;
  // this CTA's share of the positions: every splits-th tile
  const int ntiles = tiles_all > (int)split ? (tiles_all - (int)split + (int)splits - 1) / (int)splits : 0;
  const int32_t* table = p.tables + (size_t)seq * p.max_blocks;

  float factor = 0.f;
  if (warp < 8) {
    // the row's query, half of its channels a thread: two readings, the largest channel first
    const size_t at = live ? (size_t)(s_first + local) * p.q_stride + (size_t)(kvh * G + head) * p.head_dim : 0;
    float most = 0.f;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
      float x[4];
      pi_load4_as_f32(x, p.q, at + d, p.dtype, live ? p.head_dim - d : 0, p.q_wide);
#pragma unroll
      for (int b = 0; b < 4; ++b) most = fmaxf(most, fabsf(x[b]));
    }
    const uint32_t e = min(max(__float_as_uint(most) >> 23, 17u), 252u);   // both powers stay normal
    const float shrink = __uint_as_float((268u - e) << 23);
    factor = __uint_as_float((e - 14) << 23) * p.scale2;
#pragma unroll 2
    for (int d = half * (HD / 2); d < (half + 1) * (HD / 2); d += 16) {
      uint32_t hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[4];
        pi_load4_as_f32(x, p.q, at + d + 4 * i, p.dtype, live ? p.head_dim - d - 4 * i : 0, p.q_wide);
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] *= shrink;
        hi[2 * i] = pack_f16(x[0], x[1]);
        hi[2 * i + 1] = pack_f16(x[2], x[3]);
        if constexpr (PLANES == 2) {
          lo[2 * i] = pack_rest(x[0], x[1], hi[2 * i]);
          lo[2 * i + 1] = pack_rest(x[2], x[3], hi[2 * i + 1]);
        }
      }
      __syncwarp();
      t_st8(lane_addr + L::col_q + d / 2, hi);
      if constexpr (PLANES == 2) t_st8(lane_addr + L::col_q + HD / 2 + d / 2, lo);
    }
    t_wait_st();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  auto fail = [&](int code) {
    if (!s_abort) {
      s_abort = 1;
      if (pp.err_flag) atomicExch(pp.err_flag, code);
    }
  };

  float* s_out = reinterpret_cast<float*>(smem);   // where the CTAs of a cluster meet: outputs relative to their own maxima
  float2* s_stat = reinterpret_cast<float2*>(s_out + kRowsP * L::line);
  auto store = [&](int row_local, int h, int d, float4 v, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l, y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    if (d < p.head_dim)
      pi_store4_f32_as(y, p.out, (size_t)(s_first + row_local) * p.out_stride + (size_t)(kvh * G + h) * p.head_dim + d, p.dtype, p.head_dim - d, p.out_wide);
  };
  // of the 5 x 96 registers that the groups of four warps have at launch: 152 for each of rows, 64 for each of converters, 48 for the rest
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    constexpr int HALF = HD / 2;   // channels of this thread
    float acc[HALF], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < HALF; ++i) acc[i] = 0.f;
    // ---- rows -----------------------------------------------------------------------------------------------------------------
    float fold_keep = 1.f, fold_unit = 0.f;   // of the tile before: what became of the output so far, and its r
    bool alive = true;
    const int to = min(pos, hi_all);
    auto fold = [&](int j) -> bool {   // the product of tile j into the output
      if (!warp_wait(o_full, j & 1, &s_abort, pp.wait_limit)) {
        if (lane == 0) fail(22);
        return false;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const bool shrunk = __any_sync(0xffffffffu, fold_keep != 1.f);
#pragma unroll
      for (int c = 0; c < HALF; c += 32) {
        uint32_t o[32];
        t_ld16(lane_addr + L::col_o + half * HALF + c, o);
        t_ld16(lane_addr + L::col_o + half * HALF + c + 16, o + 16);
        t_wait_ld();
        if (shrunk) {
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c + i] *= fold_keep;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(fold_unit, __uint_as_float(o[i]), acc[c + i]);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(o_free);
      return true;
    };
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };   // the two halves' warps: once a tile, come what may
    for (int j = 0; j < ntiles; ++j) {
      const int buf = j & 1;
      if (!alive) {
        meet();
        continue;
      }
      // the groups, which the converters wrote (the products' thread has waited for them, but its commit hands on only what the products
      // did; the stage is not filled again before these warps have delivered the tile's weights), and the scores
      if (!__all_sync(0xffffffffu, bar_wait(kv_full0 + 8 * (j % STAGES), (j / STAGES) & 1, &s_abort, pp.wait_limit) && bar_wait(s_full0 + 8 * buf, (j >> 1) & 1, &s_abort, pp.wait_limit))) {
        if (lane == 0) fail(21);
        alive = false;
        meet();
        continue;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const Group* group = s_group[j % STAGES];
      constexpr int COLS = TILE / 2, GROUPS = COLS / 16;   // of this thread
      const uint32_t s_col = lane_addr + L::col_s + buf * TILE + half * COLS;
      // the tile as a whole: lane g looks at group g
      int lowest, highest;
      bool filled;
      {
        const Group q = group[lane < 2 * GROUPS ? lane : 0];
        lowest = __reduce_min_sync(0xffffffffu, q.base);
        highest = __reduce_max_sync(0xffffffffu, q.base + 15);
        filled = __all_sync(0xffffffffu, q.valid == 16);
      }
      const bool masks = !__all_sync(0xffffffffu, filled && from <= lowest && to >= highest);
      // where not all of it is seen: a bit per column of this thread's groups
      uint32_t seen[GROUPS];
      if (masks) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const Group q = group[half * GROUPS + g];
          const int f = max(0, from - q.base), l = min(to - q.base, q.valid - 1);
          seen[g] = f <= l ? (0xffffu >> (15 - l)) & (0xffffu << f) : 0;
        }
      }
      float w[COLS];
      {
        uint32_t raw[COLS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) t_ld16(s_col + g * 16, raw + g * 16);
        t_wait_ld();
#pragma unroll
        for (int i = 0; i < COLS; ++i) w[i] = __uint_as_float(raw[i]);
      }
      // the largest score of the tile, and of score and V scale together
      float most = -INFINITY, reach = -INFINITY;
      if (masks) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!(seen[g] & 1u << i)) w[g * 16 + i] = -INFINITY;
      }
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        float top2[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 16; ++i) top2[i & 1] = fmaxf(top2[i & 1], w[g * 16 + i]);
        const float t = fmaxf(top2[0], top2[1]);
        if (t > -INFINITY) {
          const float score = t * (factor * group[half * GROUPS + g].k_scale);
          most = fmaxf(most, score);
          reach = fmaxf(reach, score + group[half * GROUPS + g].v_exp);
        }
      }
      // the other half's; both threads come to the same maxima
      s_most[buf][half][m] = make_float2(most, reach);
      meet();
      {
        const float2 other = s_most[buf][half ^ 1][m];
        most = fmaxf(most, other.x);
        reach = fmaxf(reach, other.y);
      }
      float keep = 1.f;
      if (most > top + kLag) {
        keep = top == -INFINITY ? 1.f : exp2_fast(top - most);
        top = most;
      }
      sum *= keep;
      const float base = (top == -INFINITY ? 0.f : top) - kTopWeight;
      // r = 2^v_unit: a weight relative to 2^kTopWeight times its V scale is below it.  Where all that the row sees has V scales or weights of next to
      // nothing, r stays a normal number.
      const float v_unit = fminf(fmaxf(ceilf(reach - (base + kTopWeight)) + 1.f, -126.f), 127.f);
      uint32_t hi[COLS / 2], lo[PLANES == 2 ? COLS / 2 : 1];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const Group q = group[half * GROUPS + g];
        const float f = factor * q.k_scale;
        // weights times V scale / r; a zero scale's codes are zero, so that any factor does
        float shift = q.v_exp == kNoScale ? 0.f : q.v_exp - v_unit + q.v_log;
        if (shift < -100.f) shift = -100.f;   // 2^-100 of the largest in the tile; not a number stays that
        const float less = shift - base;
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) w[g * 16 + i] = exp2_fast(fmaf(w[g * 16 + i], f, less));
        if (masks && !(f > 0.f && f < INFINITY && less < INFINITY)) {   // minus infinity times f plus `less` is not minus infinity
#pragma unroll
          for (int i = 0; i < 16; ++i) w[g * 16 + i] = seen[g] & 1u << i ? w[g * 16 + i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i & 1] += w[g * 16 + i];
        if (!masks || seen[g]) sum = fmaf(part[0] + part[1], exp2_fast(-shift), sum);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hi[g * 8 + i] = pack_f16(w[g * 16 + 2 * i], w[g * 16 + 2 * i + 1]);
          if constexpr (PLANES == 2) lo[g * 8 + i] = pack_rest(w[g * 16 + 2 * i], w[g * 16 + 2 * i + 1], hi[g * 8 + i]);
        }
      }
      // the tile before is multiplied out by now: fold it in, which frees its output and the columns of P
      if (j > 0 && !fold(j - 1)) {
        alive = false;
        continue;
      }
      fold_keep = keep;
      fold_unit = exp2_fast(v_unit);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        t_st8(lane_addr + L::col_p + half * (COLS / 2) + g * 8, hi + g * 8);
        if constexpr (PLANES == 2) t_st8(lane_addr + L::col_p + TILE / 2 + half * (COLS / 2) + g * 8, lo + g * 8);
      }
      t_wait_st();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(p_full);
    }
    if (alive && ntiles > 0) alive = fold(ntiles - 1);
    if (!alive) sum = NAN;   // a wait ran out: the row's results say so, whatever CTA they come from
    // the halves' sums, in the buffer that the last tile did not use
    s_most[ntiles & 1][half][m].x = sum;
    meet();
    sum = s_most[ntiles & 1][0][m].x + s_most[ntiles & 1][1][m].x;
    if (splits == 1) {
      if (live) {
#pragma unroll
        for (int d = 0; d < HALF; d += 4) store(local, head, half * HALF + d, make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]), sum);
      }
    } else {   // where the rings were: the last product has read them
#pragma unroll
      for (int d = 0; d < HALF; d += 4) *reinterpret_cast<float4*>(s_out + m * L::line + half * HALF + d) = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
      if (half == 0) s_stat[m] = make_float2(top, sum);
    }
  } else if (warp < 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ---- converters -----------------------------------------------------------------------------------------------------------
    const int ct = tid & 127, cw = warp & 3, which = (warp - 8) >> 2;   // of two: a part of every tile, or every other tile of one part
    constexpr int EVERY = PARTS == 2 ? 1 : 2;
    const int part = PARTS == 2 ? which : 0, j0 = PARTS == 2 ? 0 : which;
    // K: half of a token's channels (HD bytes / 2); V: HD / 16 channels of eight tokens, a warp 32 neighbouring bytes at most of all 64
    constexpr int KW = HD / 8, VW = HD / 64;   // words of K, words per token of V
    const int k_token = ct >> 1, k_half = ct & 1, v_eight = lane & 7, v_part = (lane >> 3) + 4 * cw;
    struct Place {   // 16 tokens: physical block (-1: none), place in it, first position
      int id, sub, base;
    };
    auto locate = [&](int j, int group) -> Place {
      const int q = (j * (int)splits + (int)split) * L::groups + part * 4 + group, b = p.by_tiles(q);
      Place at = {-1, (q - b * per_block) * 16, 0};
      at.base = (first_block + b) * bs + at.sub;
      if (j < ntiles && q < groups) at.id = __ldg(table + first_block + b);
      return at;
    };
    struct Raw {
      uint32_t k[KW], v[8][VW];
      float2 k_scales;   // both scales of the group that this thread's token of K lies in
      float v_scale;
    };
    auto fetch = [&](const Place& k_at, const Place& v_at, Raw& r) {
#pragma unroll
      for (int i = 0; i < KW; ++i) r.k[i] = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int w = 0; w < VW; ++w) r.v[t][w] = 0;
      r.k_scales = make_float2(0.f, 0.f);
      r.v_scale = 0.f;
      if ((uint32_t)k_at.id < (uint32_t)p.num_blocks) {
        const unsigned long long id = (uint32_t)k_at.id;
        const uint8_t* k = p.codes + id * p.block_bytes + (size_t)kvh * 2 * p.side_bytes + (size_t)min(k_at.sub + (k_token & 15), bs - 1) * HD + k_half * (HD / 2);
#pragma unroll
        for (int i = 0; i < KW / 4; ++i) {
          const uint4 v = __ldcs(reinterpret_cast<const uint4*>(k) + i);
          r.k[4 * i] = v.x, r.k[4 * i + 1] = v.y, r.k[4 * i + 2] = v.z, r.k[4 * i + 3] = v.w;
        }
        r.k_scales = __ldg(reinterpret_cast<const float2*>(p.scales + (id * p.kv_heads + kvh) * 2));
      }
      if ((uint32_t)v_at.id < (uint32_t)p.num_blocks) {
        const unsigned long long id = (uint32_t)v_at.id;
        const uint8_t* v = p.codes + id * p.block_bytes + ((size_t)kvh * 2 + 1) * p.side_bytes + v_part * (HD / 16);
        const int off0 = (v_eight & 1) * 8;
        v += (size_t)(v_at.sub + off0) * HD;
        auto take = [&](int t) {
          if constexpr (VW == 2) {
            const uint2 x = __ldcs(reinterpret_cast<const uint2*>(v + t * HD));
            r.v[t][0] = x.x, r.v[t][1] = x.y;
          } else {
            r.v[t][0] = __ldcs(reinterpret_cast<const uint32_t*>(v + t * HD));
          }
        };
        if (v_at.sub + 16 <= bs && v_at.base >= lo_all && v_at.base + 15 <= hi_all) {
#pragma unroll
          for (int t = 0; t < 8; ++t) take(t);
        } else {   // tokens that no row sees stay zero: their bytes may be anything, also what e4m3 calls NaN
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if (v_at.sub + off0 + t < bs && v_at.base + off0 + t >= lo_all && v_at.base + off0 + t <= hi_all) take(t);
        }
        r.v_scale = __ldg(p.scales + (id * p.kv_heads + kvh) * 2 + 1);
      }
    };
    // the codes of a tile are requested as soon as this group's one before is stored, its table entries one tile earlier
    Raw cur;
    Place k_here = locate(j0, k_token >> 4), v_here = locate(j0, v_eight >> 1);
    fetch(k_here, v_here, cur);
    for (int j = j0; j < ntiles; j += EVERY) {
      const int stg = j % STAGES;
      const Place k_next = locate(j + EVERY, k_token >> 4);
      v_here = locate(j + EVERY, v_eight >> 1);
      if (!warp_wait<true>(kv_free0 + 8 * stg, ((j / STAGES) & 1) ^ 1, &s_abort, pp.wait_limit)) {
        if (lane == 0) fail(23);
        break;
      }
      // addresses of 16-byte chunks: the swizzle is an exclusive or with bits of the row, which are the thread's own
      const uint32_t kdst = smem_base + stg * L::stage + (part * kPartP + k_token) * 128 + ((k_token & 7) << 4);
      const uint32_t vdst = smem_base + stg * L::stage + L::side + part * (HD * 128) + v_part * (HD / 16) * 128 + ((v_eight ^ (v_part * (HD / 16) & 7)) << 4);
      if (lane == 0) {   // token 16 cw: this thread's token of K
        Group q;
        q.base = k_here.base;
        q.valid = (uint32_t)k_here.id < (uint32_t)p.num_blocks ? min(16, bs - k_here.sub) : 0;
        q.k_scale = cur.k_scales.x;
        const float sv = cur.k_scales.y;
        int e = 0;
        const float mant = frexpf(sv, &e);   // [0.5, 1)
        q.v_exp = sv == 0.f ? kNoScale : (float)(e - 1);
        q.v_log = sv == 0.f ? 0.f : (sv < INFINITY ? log2f(2.f * mant) : NAN);
        s_group[stg][part * 4 + cw] = q;
      }
      {   // K: two codes a word of f16, 16 bytes a store, [64 channels][token][128 bytes] swizzled
        constexpr int CHUNKS = KW / 2;   // of 8 channels
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const uint32_t a = unsign<KIND>(cur.k[2 * c]), b = unsign<KIND>(cur.k[2 * c + 1]);
          const int chunk = HD == 128 ? c : k_half * CHUNKS + c, sub = HD == 128 ? k_half : 0;
          st_shared((kdst ^ chunk << 4) + sub * (TILE * 128), widen<KIND>(a, false), widen<KIND>(a, true), widen<KIND>(b, false), widen<KIND>(b, true));
        }
      }
      {   // V: eight tokens of a channel are 16 bytes, [part][channel][128 bytes] swizzled
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t u[8];
#pragma unroll
          for (int t = 0; t < 8; ++t) u[t] = unsign<KIND>(cur.v_scale == 0.f ? 0 : cur.v[t][w]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t x[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) x[t] = __byte_perm(u[2 * t], u[2 * t + 1], half ? 0x7362 : 0x5140);
#pragma unroll
            for (int one = 0; one < 2; ++one) {
              const int i = w * 4 + half * 2 + one;   // of this thread's channels, which begin at a multiple of their number
              st_shared((vdst ^ i << 4) + i * 128, widen<KIND>(x[0], one), widen<KIND>(x[1], one), widen<KIND>(x[2], one), widen<KIND>(x[3], one));
            }
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // generic-proxy stores -> visible to the MMA's reads
      __syncwarp();
      if (lane == 0) bar_arrive(kv_full0 + 8 * stg);
      k_here = k_next;
      if (j + EVERY < ntiles) fetch(k_here, v_here, cur);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 16)
      if (pi_elect()) {   // a test of its own: behind a compound one the descriptors do not stay in uniform registers
    // ---- products ---------------------------------------------------------------------------------------------------------------
    auto idesc = [](uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((uint32_t)(kRowsP >> 4) << 24); };   // f16 x f16 -> f32
    auto scores = [&](int j) -> bool {
      const int stg = j % STAGES, buf = j & 1;
      if (s_abort || !bar_wait(kv_full0 + 8 * stg, (j / STAGES) & 1, &s_abort, pp.wait_limit)) {
        fail(24);
        return false;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t bd = desc_sw128(smem_base + stg * L::stage);
#pragma unroll
      for (int pl = PLANES - 1; pl >= 0; --pl)   // the smaller terms first
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
          mma_ts(tmem + L::col_s + buf * TILE, tmem + L::col_q + pl * (HD / 2) + ks * 8, bd + (uint64_t)(((ks >> 2) * (TILE * 128) + (ks & 3) * 32) >> 4), idesc(TILE),
                 pl == PLANES - 1 && ks == 0 ? 0u : 1u);
      mma_commit(s_full0 + 8 * buf);
      return true;
    };
    bool ok = ntiles > 0 && scores(0);
    for (int j = 0; j < ntiles && ok; ++j) {
      const int stg = j % STAGES;
      // the next tile's scores run while the row threads work on this tile's
      if (j + 1 < ntiles && !scores(j + 1)) break;
      if (s_abort || !bar_wait(p_full, j & 1, &s_abort, pp.wait_limit) || (j > 0 && !bar_wait(o_free, (j - 1) & 1, &s_abort, pp.wait_limit))) {
        fail(25);
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t bd = desc_sw128(smem_base + stg * L::stage + L::side);
#pragma unroll
      for (int pl = PLANES - 1; pl >= 0; --pl)
#pragma unroll
        for (int ks = 0; ks < TILE / 16; ++ks)
          mma_ts(tmem + L::col_o, tmem + L::col_p + pl * (TILE / 2) + ks * 8, bd + (uint64_t)(((ks >> 2) * (HD * 128) + (ks & 3) * 32) >> 4), idesc(HD), pl == PLANES - 1 && ks == 0 ? 0u : 1u);
      mma_commit(o_full);
      mma_commit(kv_free0 + 8 * stg);
    }
    // nobody frees tensor memory under a product, also where this thread or another one gave up
    mma_commit(idle);
    bar_wait(idle, 0, nullptr, kWaitLimitP);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 16) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
  if (splits == 1) return;
  // where a wait ran out, converters may have filled the rings over what the rows left there
  if (s_abort && tid < kRowsP) s_stat[tid] = make_float2(0.f, NAN);
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int share = kRowsP / (int)splits, rows_here = min(pp.rows_per_tile, row_end - s_first);
  for (int i = tid; i < share * (HD / 4); i += kThreadsP) {
    const int mm = (int)split * share + i / (HD / 4), d = i % (HD / 4) * 4, row_local = p.by_group(mm);
    if (row_local >= rows_here || d >= p.head_dim) continue;
    float all = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t r = 0; r < splits; ++r) all = fmaxf(all, peer2(s_stat + mm, r).x);
    for (uint32_t r = 0; r < splits; ++r) {
      const float2 st = peer2(s_stat + mm, r);
      const float4 x = peer4(s_out + mm * L::line + d, r);
      const float f = join_factor(st.x, st.y, all);
      v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
      l = fmaf(f, st.y, l);
    }
    store(row_local, mm - row_local * G, d, v, l);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int KIND, int HD, int PLANES>
pi_status launch_prefill(pi_ctx* ctx, const PrefillParams& p, dim3 grid, int splits) {
  constexpr int bytes = Prefill<HD, PLANES>::smem;
  auto kernel = kv8_prefill_kernel<KIND, HD, PLANES>;
  static pi_smem_grant grant;
  if (grant.of(ctx) == 0) {
    PI_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    grant.of(ctx) = bytes;
  }
  PI_CUDA(ctx, pi_launch_chained(ctx, kernel, grid, dim3(kThreadsP), bytes, splits, p));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}

}  // namespace

// Tiles of rows: each sequence ends with one that may not be full.
static long long prefill_tiles(const pi_kv8_attn_params& a) {
  const int rows = kRowsP / a.group;
  return ((long long)a.n_rows + rows - 1) / rows + std::min(a.n_seqs - 1, a.n_rows - 1);
}

bool pi_kv8_prefill_takes(const pi_kv8_pool* pool, const pi_kv8_attn_params& a) {
  return (pool->pitch == 64 || pool->pitch == 128) && a.group <= kRowsP && prefill_tiles(a) * a.kv_heads <= 0x7fffffffll / kMostSplitsP;   // CTAs of a grid
}

pi_status pi_launch_kv8_prefill(pi_ctx* ctx, const pi_kv8_pool* pool, const pi_kv8_attn_params& a, int min_cols, int max_context) {
  PrefillParams p = {};
  p.a = a;
  p.rows_per_tile = kRowsP / a.group;
  p.min_cols = min_cols;
  p.err_flag = ctx->dev_err;
  p.wait_limit = ctx->kv8_wait_limit ? ctx->kv8_wait_limit : kWaitLimitP;
  const long long full = ((long long)a.n_rows + p.rows_per_tile - 1) / p.rows_per_tile;
  // few tiles share their positions out among clusters, four tiles of them or more to a CTA
  const long long seen = a.window > 0 ? std::min<long long>(max_context, (long long)a.window + a.n_rows) : max_context;
  int splits = 1;
  while (splits < kMostSplitsP && full * a.kv_heads * splits * 2 <= ctx->sm_count && seen / 64 >= 8 * splits * 2) splits *= 2;
  const dim3 grid((unsigned)(prefill_tiles(a) * a.kv_heads * splits));   // a tile's heads side by side, a head's CTAs a cluster
  const bool two = a.dtype == PI_F32;
  if (pool->kind == PI_INT8) {
    if (pool->pitch == 64) return two ? launch_prefill<PI_INT8, 64, 2>(ctx, p, grid, splits) : launch_prefill<PI_INT8, 64, 1>(ctx, p, grid, splits);
    return two ? launch_prefill<PI_INT8, 128, 2>(ctx, p, grid, splits) : launch_prefill<PI_INT8, 128, 1>(ctx, p, grid, splits);
  }
  if (pool->pitch == 64) return two ? launch_prefill<PI_E4M3, 64, 2>(ctx, p, grid, splits) : launch_prefill<PI_E4M3, 64, 1>(ctx, p, grid, splits);
  return two ? launch_prefill<PI_E4M3, 128, 2>(ctx, p, grid, splits) : launch_prefill<PI_E4M3, 128, 1>(ctx, p, grid, splits);
}
