// Paged attention over the 8-bit cache for sequences that bring few rows: decoded tokens, short verify groups.  See
// pi_kv8_attention.cu for the dispatch; the instantiations are dealt to several files by their pitch.
//
// A warp takes 16 tokens of one block at a time, all with the same two scales.  Codes are whole numbers (or e4m3 values) that f16
// holds exactly, so both products run on the tensor cores (m16n8k16, f32 accumulators) with the CACHE as the wide operand:
//     S^T[16 tokens][8 columns] = K q^T,    O^T[dims][8 columns] += scale_v (V^T P^T),    a column = one query head of one row.
// A group of eight query heads fills a product; four need no more of them than eight would.  f32 queries, and the weights of f32
// outputs, are two f16 planes (22 bits); those of bf16 and f16 outputs are one.  Queries are brought to between 2^14 and 2^15 by a power
// of two per column, so that channels 2^29 below its largest are normal numbers of f16 still (2^17 with both planes' bits), weights to
// 2^15 at most; the scales stay in f32.
//
// Codes go from memory straight to the registers that feed the products: the k index of a product may be permuted at will, so a
// lane takes whole words of a token's codes for K, and, for V, of the four tokens whose weights it holds; pairs of tokens are put
// together by byte permutes.  The next tile's K codes are requested as soon as this tile's are used up, its V codes likewise, so that
// every warp has loads under way all the time without a second set of registers and without shared memory.
//
// int8 codes become f16 by a byte permute into the mantissa of 1024 (1024 + 128 + code), and 1152 is subtracted from every pair.  (Left in, with
// accumulators that start from -1152 times the sum of the other operand, it costs scores their precision beside a channel of large codes
// in which the query is small, and results theirs beside a token of nearly all the weight and small values; it takes longer, too: one
// context of 131072 108 us instead of 106.)
//
// Products add to their accumulators with truncation, up to an ulp of the sum each.  So the two planes of a query have accumulators of their
// own (terms of a code and 11 bits leave little to truncate, those of the second plane are small), and the first plane's sums are
// taken over 128 channels and added with rounding.  (f32 results against 64 bits in random calls: 0.9 times the error of f32 sums in torch in
// the median, 5.6e-7 of the result at most; with one accumulator 1.4 times and 1.2e-6.  64 sequences of heads of 64: 22.6 us, 22.3 with one.)
//
// The tokens of a sequence are dealt to the warps of a CTA and to the CTAs of a cluster; partial results are joined through shared
// memory, then through the cluster's: no scratch in device memory, and the order of the sums is fixed.
//
// Measured: 16 sequences of 3000 to 4096, 32 query heads of 128 over 8, bf16, e4m3: 30 us, 3.9 TB/s; 64 of 256 to 2048, 32 over 4 of 64, f32,
// int8: 22.6 us, 1.7 TB/s; one of 131072, 64 over 8 of 128: 106 us, 2.5 TB/s.  Bound: the latency of a warp's chain with sixteen warps an
// SM, and for few long sequences the 16 CTAs of a cluster.
#pragma once

#include <math.h>

#include <algorithm>

#include "pi_kv8_widen.cuh"

namespace pi_kv8 {

constexpr int kMaxSplit = 16, kMaxWarps = 8;   // CTAs of a cluster, warps of a CTA
__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_new(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // d = a b
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // of an 8 x 8 tile of 16-bit values, a row per four lanes
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Codes are read once.
template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t* to, const uint8_t* from) {
  if constexpr (BYTES == 16) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(from));
    to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = __ldcs(reinterpret_cast<const uint2*>(from));
    to[0] = v.x, to[1] = v.y;
  } else {
    to[0] = __ldcs(reinterpret_cast<const uint32_t*>(from));
  }
}

template <int PITCH>
struct Geometry {
  static constexpr int ksteps = PITCH / 16, mtiles = PITCH / 16;
  // K: a lane has PITCH / 4 channels of a token, in pieces of KB bytes that lie KB * 4 apart
  static constexpr int KB = PITCH % 64 == 0 ? 16 : 8, kpieces = PITCH / 4 / KB;
  // V: PITCH / 8 neighbouring channels of a token, in pieces of VB bytes
  static constexpr int VB = PITCH % 128 == 0 ? 16 : PITCH % 64 == 0 ? 8 : 4, vpieces = PITCH / 8 / VB;
};

// Tiles that a warp works on at a time, and CTAs of eight warps that an SM has registers for: sixteen warps hide the chain from load
// to product to exponential to product better than eight with longer steps (24 with 80 registers spill); wide heads and two groups
// of columns leave room for eight.
template <int PITCH, int NT>
struct Shape {
  static constexpr int TT = PITCH <= 64 && NT == 1 ? 2 : 1, min_ctas = PITCH <= 128 && NT == 1 ? 2 : 1, cols = 8 * NT;
  static constexpr int line = PITCH + 4;   // floats between columns where warps meet
};
// Shared memory: query fragments, per column (first and last position seen, factor), (max, sum) per warp, per CTA, partial results.
template <int PITCH, int PLANES, int NT>
struct Layout {
  static constexpr int cols = 8 * NT;
  static constexpr int queries = PITCH / 16 * PLANES * NT * 32 * 8;     // b fragments, 8 bytes a lane
  static constexpr int bytes(int warps) { return queries + cols * 12 + (warps + 1) * cols * 8 + (warps + 1) * cols * Shape<PITCH, NT>::line * 4; }
};

template <int KIND, int PITCH, int PLANES, int NT>
__global__ void __launch_bounds__(kMaxWarps * 32, Shape<PITCH, NT>::min_ctas) kv8_decode_kernel(const pi_kv8_attn_params p) {
  using G = Geometry<PITCH>;
  using S = Shape<PITCH, NT>;
  constexpr int COLS = S::cols, TT = S::TT, LINE = S::line;
  constexpr int RUN = PLANES == 2 ? 8 : G::ksteps;   // steps of 16 channels
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* s_queries = smem;
  int* s_lo = reinterpret_cast<int*>(smem + Layout<PITCH, PLANES, NT>::queries);
  int* s_hi = s_lo + COLS;
  float* s_factor = reinterpret_cast<float*>(s_hi + COLS);
  float2* s_stat = reinterpret_cast<float2*>(s_factor + COLS);   // of the CTA
  float2* s_warp = s_stat + COLS;                              // [warp][column]
  float* s_out = reinterpret_cast<float*>(s_warp + warps * COLS);   // [column][line] of the CTA
  float* s_part = s_out + COLS * LINE;                         // [warp][column][line]

  uint32_t split, splits;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(split));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const int kvh = blockIdx.x / splits, seq = blockIdx.y, bs = p.block_size;
  pi_grid_dependency_wait();
  const int row_begin = max(0, min(p.cu_rows[seq], p.n_rows)), row_end = min(p.cu_rows[seq + 1], p.n_rows);
  const int ncols = (row_end - row_begin) * p.group > p.max_cols ? 0 : (row_end - row_begin) * p.group;
  const int last_token = max(0, min(p.lens[seq], p.max_blocks)) * bs - 1;
  const int32_t* table = p.tables + (size_t)seq * p.max_blocks;
  // one tile of columns as the grid is cut; the loop is for sequences that bring more rows than the call said
  for (int col0 = blockIdx.z * COLS; col0 < ncols; col0 += gridDim.z * COLS) {
    // what the tile's columns see
    int lo_all = 0x7fffffff, hi_all = -1, lo_most = 0, hi_least = 0x7fffffff;
    const int first_row = row_begin + p.by_group(col0), last_row = row_begin + p.by_group(min(ncols, col0 + COLS) - 1);
    for (int r = first_row; r <= last_row; ++r) {
      const int pos = p.row_pos[r], from = p.window > 0 ? max(0, pos - p.window + 1) : 0;
      if (pos >= 0) lo_all = min(lo_all, from);
      hi_all = max(hi_all, pos);
      lo_most = max(lo_most, from);
      hi_least = min(hi_least, pos);
    }
    hi_all = min(hi_all, last_token);
    hi_least = min(hi_least, hi_all);

    // tiles: 16 tokens of a block; rounds of TT neighbouring ones are dealt to the warps of all CTAs in turn
    const int per_block = (bs + 15) >> 4;
    const int first_block = hi_all < lo_all ? 0 : p.by_block(lo_all), blocks = hi_all < lo_all ? 0 : p.by_block(hi_all) - first_block + 1;
    const int workers = (int)splits * warps, step_block = p.by_tiles(TT * workers), step_sub = TT * workers - step_block * per_block;
    int block[TT], sub[TT];   // of the tiles to look up next: from the first block, in the block
#pragma unroll
    for (int e = 0; e < TT; ++e) {
      const int first = TT * ((int)split * warps + warp) + e;
      block[e] = p.by_tiles(first);
      sub[e] = first - block[e] * per_block;
    }
    int next_id[TT], next_base[TT], next_sub[TT];   // looked up: physical block (-1: none), first token, place in the block
    auto look = [&]() {
#pragma unroll
      for (int e = 0; e < TT; ++e) {
        next_id[e] = -1;
        if (block[e] < blocks) next_id[e] = __ldg(table + first_block + block[e]);
        next_sub[e] = sub[e] * 16;
        next_base[e] = (first_block + block[e]) * bs + sub[e] * 16;
        block[e] += step_block;
        sub[e] += step_sub;
        if (sub[e] >= per_block) {
          sub[e] -= per_block;
          ++block[e];
        }
      }
    };
    const bool whole = (bs & 15) == 0;   // no tile reaches beyond its block
    const uint8_t* k_lane = p.codes + (size_t)kvh * 2 * p.side_bytes + t * G::KB;
    const uint8_t* v_lane = p.codes + ((size_t)kvh * 2 + 1) * p.side_bytes + g * (PITCH / 8);
    const float* scale_head = p.scales + kvh * 2;

    uint32_t kw[TT][2][PITCH / 16], vw[TT][4][PITCH / 32];
    float2 k_scale[TT];       // both scales of the tile whose K codes are in kw
    int id[TT], base[TT], place[TT];
    auto load_k = [&]() {     // of the tiles that were looked up last
#pragma unroll
      for (int e = 0; e < TT; ++e) {
        id[e] = (uint32_t)next_id[e] < (uint32_t)p.num_blocks ? next_id[e] : -1;
        base[e] = next_base[e];
        place[e] = next_sub[e];
        k_scale[e] = make_float2(0.f, 0.f);
        if (id[e] >= 0) {
          k_scale[e] = __ldg(reinterpret_cast<const float2*>(scale_head + (unsigned long long)(uint32_t)id[e] * (uint32_t)(p.kv_heads * 2)));
          const uint8_t* k = k_lane + (unsigned long long)(uint32_t)id[e] * p.block_bytes;
          if (whole) {
            k += (place[e] + g) * PITCH;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int c = 0; c < G::kpieces; ++c) load_words<G::KB>(&kw[e][r][c * G::KB / 4], k + r * 8 * PITCH + c * G::KB * 4);
          } else {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int c = 0; c < G::kpieces; ++c) load_words<G::KB>(&kw[e][r][c * G::KB / 4], k + min(place[e] + g + 8 * r, bs - 1) * PITCH + c * G::KB * 4);
          }
        }
      }
    };
    auto load_v = [&]() {     // of the tiles whose K codes were requested last
#pragma unroll
      for (int e = 0; e < TT; ++e)
        if (id[e] >= 0) {
          const uint8_t* v = v_lane + (unsigned long long)(uint32_t)id[e] * p.block_bytes;
          if (whole) {
            v += (place[e] + 2 * t) * PITCH;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int c = 0; c < G::vpieces; ++c) load_words<G::VB>(&vw[e][r][c * G::VB / 4], v + ((r & 1) + (r & 2) * 4) * PITCH + c * G::VB);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int c = 0; c < G::vpieces; ++c)
                load_words<G::VB>(&vw[e][r][c * G::VB / 4], v + min(place[e] + 2 * t + (r & 1) + (r & 2) * 4, bs - 1) * PITCH + c * G::VB);
          }
        }
    };
    const int tiles = blocks * per_block, rounds = (tiles + TT - 1) / TT, worker = (int)split * warps + warp;
    int mine = rounds > worker ? p.by_workers(rounds - worker - 1) + 1 : 0;
    look();
    load_k();
    load_v();
    look();

    // the first codes are under way; meanwhile the columns' queries become b fragments: eight lanes a column, four channels at a time,
    // each column times the power of two that brings its largest to 2^14 or more
    for (int c = tid >> 3; c < COLS; c += warps * 4) {
      const int l8 = lane & 7, rel = col0 + c < ncols ? p.by_group(col0 + c) : 0, row = row_begin + rel;
      const bool live = col0 + c < ncols;
      const size_t at = (size_t)row * p.q_stride + (size_t)(kvh * p.group + (col0 + c - rel * p.group)) * p.head_dim;
      float x[PITCH / 32][4], most = 0.f;
#pragma unroll
      for (int i = 0; i < PITCH / 32; ++i) {
        const int d = 4 * (l8 + 8 * i);
        pi_load4_as_f32(x[i], p.q, at + d, p.dtype, live ? p.head_dim - d : 0, p.q_wide);
#pragma unroll
        for (int b = 0; b < 4; ++b) most = fmaxf(most, fabsf(x[i][b]));
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      // 2^(e - 127) <= most < 2^(e - 126); both powers below stay normal
      const uint32_t e = min(max(__float_as_uint(most) >> 23, 17u), 252u);
      const float shrink = __uint_as_float((268u - e) << 23);   // 2^(141 - e)
#pragma unroll
      for (int i = 0; i < PITCH / 32; ++i) {
        const int d = 4 * (l8 + 8 * i), piece = d / (G::KB * 4), in = d % (G::KB * 4), to = (piece * (G::KB / 4) + in % G::KB / 4) * PLANES;
        float y[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) y[b] = x[i][b] * shrink;
        uint2 hi = make_uint2(pack_f16(y[0], y[1]), pack_f16(y[2], y[3]));
        uint2* frag = reinterpret_cast<uint2*>(s_queries) + ((size_t)to * NT + c / 8) * 32 + (c % 8) * 4 + in / G::KB;
        frag[0] = hi;
        if constexpr (PLANES == 2) frag[NT * 32] = make_uint2(pack_rest(y[0], y[1], hi.x), pack_rest(y[2], y[3], hi.y));
      }
      if (l8 == 0) {
        const int pos = live ? p.row_pos[row] : -1;
        s_lo[c] = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        s_hi[c] = pos;
        s_factor[c] = __uint_as_float((e - 14) << 23) * p.scale2;   // 2^(e - 141)
      }
    }
    __syncthreads();

    float out[NT][G::mtiles][4], top[NT][2], sum[NT][2], factor[NT][2];
    int lo[NT][2], hi[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = n * 8 + 2 * t + e;
        top[n][e] = -INFINITY;
        sum[n][e] = 0.f;
        factor[n][e] = s_factor[c];
        lo[n][e] = s_lo[c];
        hi[n][e] = min(s_hi[c], hi_all);
      }
#pragma unroll
      for (int m = 0; m < G::mtiles; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[n][m][e] = 0.f;
    }

    for (; mine > 0; --mine) {
      int valid[TT], token[TT];
      float2 scale[TT];
      bool all = true;   // every column sees every token
#pragma unroll
      for (int e = 0; e < TT; ++e) {
        valid[e] = id[e] >= 0 ? min(16, bs - place[e]) : 0;
        token[e] = base[e];
        all = all && valid[e] == 16 && token[e] >= lo_most && token[e] + 15 <= hi_least;
        scale[e] = k_scale[e];
      }
      if constexpr (KIND == PI_E4M3) {
        // bytes of tokens that nobody sees may be anything, also what e4m3 calls NaN; a weight of zero does not silence that
        if (!all) {
#pragma unroll
          for (int e = 0; e < TT; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int row = 2 * t + (r & 1) + (r & 2) * 4;
              const bool seen = row < valid[e] && token[e] + row >= lo_all && token[e] + row <= hi_all;
#pragma unroll
              for (int w = 0; w < PITCH / 32; ++w) vw[e][r][w] = seen ? vw[e][r][w] : 0;
            }
        }
      }
      float s[TT][NT][4], low[TT][NT][4], run[TT][NT][4];   // of the first plane of the queries, of the second, of the first since the last run
#pragma unroll
      for (int j = 0; j < G::ksteps; ++j) {
        uint32_t a[TT][4];
#pragma unroll
        for (int e = 0; e < TT; ++e) {
          const uint32_t w0 = unsign<KIND>(kw[e][0][j]), w1 = unsign<KIND>(kw[e][1][j]);
          a[e][0] = widen<KIND>(w0, false);
          a[e][1] = widen<KIND>(w1, false);
          a[e][2] = widen<KIND>(w0, true);
          a[e][3] = widen<KIND>(w1, true);
        }
#pragma unroll
        for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 b = reinterpret_cast<const uint2*>(s_queries)[((j * PLANES + pl) * NT + n) * 32 + lane];
#pragma unroll
            for (int e = 0; e < TT; ++e) {
              float* to = pl == 1 ? low[e][n] : j < RUN ? s[e][n] : run[e][n];
              if (pl == 1 ? j == 0 : j % RUN == 0) mma_f16_new(to, a[e][0], a[e][1], a[e][2], a[e][3], b.x, b.y);
              else mma_f16(to, a[e][0], a[e][1], a[e][2], a[e][3], b.x, b.y);
              if (pl == 0 && j >= RUN && (j % RUN == RUN - 1 || j == G::ksteps - 1)) {
#pragma unroll
                for (int c = 0; c < 4; ++c) s[e][n][c] += run[e][n][c];
              }
            }
          }
      }
      if constexpr (PLANES == 2) {
#pragma unroll
        for (int e = 0; e < TT; ++e)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[e][n][c] += low[e][n][c];
      }
      load_k();   // of the next round; the table's entries for the one behind it are on their way a whole round ahead
      look();

      // softmax: this lane has tokens g and g + 8 of every tile, columns 2 t and 2 t + 1
      uint32_t pw[TT][NT][2][PLANES];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < TT; ++e)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float f = factor[n][c] * scale[e].x;
            s[e][n][c] *= f;
            s[e][n][2 + c] *= f;
          }
        if (!all) {
#pragma unroll
          for (int e = 0; e < TT; ++e)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int row = g + (c >> 1) * 8, at_token = token[e] + row;
              if (row >= valid[e] || at_token < lo[n][c & 1] || at_token > hi[n][c & 1]) s[e][n][c] = -INFINITY;
            }
        }
        float most[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          most[c] = fmaxf(s[0][n][c], s[0][n][2 + c]);
#pragma unroll
          for (int e = 1; e < TT; ++e) most[c] = fmaxf(most[c], fmaxf(s[e][n][c], s[e][n][2 + c]));
        }
        // the first scores of a column exceed minus infinity by more than any lag
        if (__any_sync(0xffffffffu, most[0] > top[n][0] + kLag || most[1] > top[n][1] + kLag)) {
          float shrink[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) most[c] = fmaxf(most[c], __shfl_xor_sync(0xffffffffu, most[c], o));
            const float now = fmaxf(top[n][c], most[c]);
            shrink[c] = exp2_fast(top[n][c] - (now == -INFINITY ? 0.f : now));
            top[n][c] = now;
            sum[n][c] *= shrink[c];
          }
#pragma unroll
          for (int m = 0; m < G::mtiles; ++m) {
            out[n][m][0] *= shrink[0];
            out[n][m][1] *= shrink[1];
            out[n][m][2] *= shrink[0];
            out[n][m][3] *= shrink[1];
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float from = (top[n][c] == -INFINITY ? 0.f : top[n][c]) - kTopWeight;
#pragma unroll
          for (int e = 0; e < TT; ++e) {
            s[e][n][c] = exp2_fast(s[e][n][c] - from);
            s[e][n][2 + c] = exp2_fast(s[e][n][2 + c] - from);
            sum[n][c] += s[e][n][c] + s[e][n][2 + c];
          }
        }
#pragma unroll
        for (int e = 0; e < TT; ++e)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t h = pack_f16(s[e][n][2 * r], s[e][n][2 * r + 1]);
            pw[e][n][r][0] = transpose8(h);
            if constexpr (PLANES == 2) pw[e][n][r][1] = transpose8(pack_rest(s[e][n][2 * r], s[e][n][2 * r + 1], h));
          }
      }

#pragma unroll
      for (int e = 0; e < TT; ++e) {
        // the V scale per column; one that is not finite reaches the columns that see the tile and no others
        float unit[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            unit[n][c] = all || (token[e] + valid[e] > lo[n][c] && token[e] <= hi[n][c] && valid[e] > 0) ? scale[e].y : 0.f;
        }
#pragma unroll
        for (int w = 0; w < PITCH / 32; ++w) {
          const uint32_t v0 = unsign<KIND>(vw[e][0][w]), v1 = unsign<KIND>(vw[e][1][w]), v2 = unsign<KIND>(vw[e][2][w]), v3 = unsign<KIND>(vw[e][3][w]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x = __byte_perm(v0, v1, half ? 0x7362 : 0x5140), y = __byte_perm(v2, v3, half ? 0x7362 : 0x5140);
            const uint32_t a0 = widen<KIND>(x, false), a1 = widen<KIND>(x, true), a2 = widen<KIND>(y, false), a3 = widen<KIND>(y, true);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float d[4];
              mma_f16_new(d, a0, a1, a2, a3, pw[e][n][0][0], pw[e][n][1][0]);
              if constexpr (PLANES == 2) mma_f16(d, a0, a1, a2, a3, pw[e][n][0][1], pw[e][n][1][1]);
              float* o = out[n][2 * w + half];
#pragma unroll
              for (int c = 0; c < 4; ++c) o[c] = fmaf(unit[n][c & 1], d[c], o[c]);
            }
          }
        }
      }
      load_v();
    }

    // the warps' results meet: a common maximum, then sums in the order of the warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], o);
        if (g == 0) s_warp[warp * COLS + n * 8 + 2 * t + e] = make_float2(top[n][e], sum[n][e]);
      }
    __syncthreads();
    if (tid < COLS) {
      float m = -INFINITY, l = 0.f;
      for (int w = 0; w < warps; ++w) m = fmaxf(m, s_warp[w * COLS + tid].x);
      for (int w = 0; w < warps; ++w) {
        const float2 st = s_warp[w * COLS + tid];
        l = fmaf(join_factor(st.x, st.y, m), st.y, l);
      }
      s_stat[tid] = make_float2(m, l);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = n * 8 + 2 * t + e;
        float m = -INFINITY;
        for (int w = 0; w < warps; ++w) m = fmaxf(m, s_warp[w * COLS + c].x);
        const float f = join_factor(top[n][e], sum[n][e], m);
        float* to = s_part + (warp * COLS + c) * LINE + g * (PITCH / 8);
#pragma unroll
        for (int i = 0; i < PITCH / 32; ++i)
          *reinterpret_cast<float4*>(to + 4 * i) = make_float4(out[n][2 * i][e] * f, out[n][2 * i][2 + e] * f, out[n][2 * i + 1][e] * f, out[n][2 * i + 1][2 + e] * f);
      }
    __syncthreads();
    const int live = min(COLS, ncols - col0);
    auto store = [&](int c, int d, float4 v, float l) {
      const int rel = p.by_group(col0 + c);
      const float inv = l == 0.f ? 0.f : 1.f / l, y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
      pi_store4_f32_as(y, p.out, (size_t)(row_begin + rel) * p.out_stride + (size_t)(kvh * p.group + (col0 + c - rel * p.group)) * p.head_dim + d, p.dtype, p.head_dim - d, p.out_wide);
    };
    for (int i = tid; i < live * (PITCH / 4); i += warps * 32) {
      const int c = i / (PITCH / 4), d = i % (PITCH / 4) * 4;
      float4 v = *reinterpret_cast<const float4*>(s_part + c * LINE + d);
      for (int w = 1; w < warps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(s_part + (w * COLS + c) * LINE + d);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      if (splits > 1) *reinterpret_cast<float4*>(s_out + c * LINE + d) = v;
      else if (d < p.head_dim) store(c, d, v, s_stat[c].y);
    }
    if (splits > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      // every CTA of the cluster finishes its share of the columns' channels
      const int total = live * (PITCH / 4), share = (total + (int)splits - 1) / (int)splits;
      for (int i = (int)split * share + tid; i < min(total, ((int)split + 1) * share); i += warps * 32) {
        const int c = i / (PITCH / 4), d = i % (PITCH / 4) * 4;
        if (d >= p.head_dim) continue;
        float m = -INFINITY, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t r = 0; r < splits; ++r) m = fmaxf(m, peer2(s_stat + c, r).x);
        for (uint32_t r = 0; r < splits; ++r) {
          const float2 st = peer2(s_stat + c, r);
          const float4 x = peer4(s_out + c * LINE + d, r);
          const float f = join_factor(st.x, st.y, m);
          v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
          l = fmaf(f, st.y, l);
        }
        store(c, d, v, l);
      }
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
      __syncthreads();
    }
  }
}

template <int KIND, int PITCH, int PLANES, int NT>
pi_status launch_decode(pi_ctx* ctx, const pi_kv8_attn_params& p, dim3 grid, int splits, int warps) {
  static_assert(Layout<PITCH, PLANES, NT>::bytes(kMaxWarps) <= 227 * 1024, "shared memory");
  const int bytes = Layout<PITCH, PLANES, NT>::bytes(warps);
  auto kernel = kv8_decode_kernel<KIND, PITCH, PLANES, NT>;
  static pi_smem_grant grant;
  if (grant.of(ctx) == 0) {
    constexpr int most = Layout<PITCH, PLANES, NT>::bytes(kMaxWarps);
    PI_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    PI_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    grant.of(ctx) = most;
  }
  PI_CUDA(ctx, pi_launch_chained(ctx, kernel, grid, dim3(warps * 32), bytes, splits, p));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}

template <int PITCH>
pi_status launch_decode_pitch(pi_ctx* ctx, int kind, int planes, int nt, const pi_kv8_attn_params& p, dim3 grid, int splits, int warps) {
  if (kind == PI_INT8) {
    if (planes == 2) return nt == 1 ? launch_decode<PI_INT8, PITCH, 2, 1>(ctx, p, grid, splits, warps) : launch_decode<PI_INT8, PITCH, 2, 2>(ctx, p, grid, splits, warps);
    return nt == 1 ? launch_decode<PI_INT8, PITCH, 1, 1>(ctx, p, grid, splits, warps) : launch_decode<PI_INT8, PITCH, 1, 2>(ctx, p, grid, splits, warps);
  }
  if (planes == 2) return nt == 1 ? launch_decode<PI_E4M3, PITCH, 2, 1>(ctx, p, grid, splits, warps) : launch_decode<PI_E4M3, PITCH, 2, 2>(ctx, p, grid, splits, warps);
  return nt == 1 ? launch_decode<PI_E4M3, PITCH, 1, 1>(ctx, p, grid, splits, warps) : launch_decode<PI_E4M3, PITCH, 1, 2>(ctx, p, grid, splits, warps);
}
extern template pi_status launch_decode_pitch<32>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int, int);
extern template pi_status launch_decode_pitch<64>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int, int);
extern template pi_status launch_decode_pitch<96>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int, int);
extern template pi_status launch_decode_pitch<128>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int, int);
extern template pi_status launch_decode_pitch<192>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int, int);
extern template pi_status launch_decode_pitch<256>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int, int);

}  // namespace pi_kv8
