// Paged attention over the 8-bit cache for sequences that bring few rows: decoded tokens, short verify groups.  See
// pi_kv8_decode.cu for the dispatch; the instantiations are dealt to several files by their pitch.
//
// A warp takes 16 tokens of one block at a time, all with the same two scales.  Codes are whole numbers (or e4m3 values) that f16
// holds exactly, so both products run on the tensor cores (m16n8k16, f32 accumulators) with the CACHE as the wide operand:
//     S^T[16 tokens][8 columns] = K q^T,    O^T[dims][8 columns] += scale_v (V^T P^T),    a column = one query head of one row.
// A group of eight query heads fills a product; four need no more of them than eight would.  f32 queries, and the weights of f32
// outputs, are two f16 planes (22 bits); those of bf16 and f16 outputs are one.  Queries are brought to [-1, 1] by a power of two
// per column, weights to 2^14 at most, so that neither leaves f16's normal range; the scales stay in f32.
//
// Codes go from memory to registers without a shuffle: the k index of a product may be permuted at will, so a lane takes whole
// words of a token's codes for K, and, for V, of the four tokens whose weights it holds; pairs of tokens are put together by byte
// permutes.  The copies (cp.async) land where the same lane reads them, so a ring of tiles per warp needs no barrier.  Two 2 KB
// tiles at pitch 128 are 8 copies a lane.
//
// The tokens of a sequence are dealt to the warps of a CTA and to the CTAs of a cluster; partial results are joined through shared
// memory, then through the cluster's: no scratch in device memory, and the order of the sums is fixed.
#pragma once

#include <math.h>

#include <algorithm>

#include "pi_kv8.cuh"
#include "pi_mma.cuh"

namespace pi_kv8 {

constexpr int kWarpsD = 4, kStagesD = 4, kMaxSplit = 16;
constexpr float kTopWeight = 14.f;   // log2 of what the largest weight is stored as

__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // of an 8 x 8 tile of 16-bit values, a row per four lanes
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t* to, const unsigned char* from) {
  if constexpr (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(from);
    to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    to[0] = v.x, to[1] = v.y;
  } else {
    to[0] = *reinterpret_cast<const uint32_t*>(from);
  }
}
// How much a partial result (maximum, sum) counts beside the maximum of all: one that saw nothing does not, one that is not a
// number makes the whole one.
__device__ __forceinline__ float join_factor(float top, float sum, float all) {
  if (sum != sum) return sum;
  return top == -INFINITY ? 0.f : exp2_fast(top - all);
}
// Two codes as f16: bytes 0 and 1, or 2 and 3, of a word.  int8: 1024 + (code + 128) in the mantissa, less 1152.  e4m3: the bits of
// 2^-8 times the value, subnormals included.
template <int KIND>
__device__ __forceinline__ uint32_t widen(uint32_t w, uint32_t sel_int8, uint32_t sel_e4m3) {
  if (KIND == PI_INT8) {
    const uint32_t h = __byte_perm(w, 0x64646464u, sel_int8);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const uint32_t h = __byte_perm(w, 0, sel_e4m3);
  return (h & 0x80008000u) | (h >> 1 & 0x3f803f80u);
}
template <int KIND>
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
  return widen<KIND>(w, 0x4140, 0x1404);
}
template <int KIND>
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
  return widen<KIND>(w, 0x4342, 0x3424);
}
template <int KIND>
__device__ __forceinline__ uint32_t unsign(uint32_t w) {
  return KIND == PI_INT8 ? w ^ 0x80808080u : w;
}
template <int KIND>
constexpr float kUnit = KIND == PI_INT8 ? 1.f : 256.f;   // what a widened code of 1 stands for

// f16 pair of two values and the pair of what is left.
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_f16(a - f.x, b - f.y);
}

template <int PITCH>
struct Geometry {
  static constexpr int ksteps = PITCH / 16, mtiles = PITCH / 16;
  // K: a lane has PITCH / 4 channels of a token, in pieces of KB bytes that lie KB * 4 apart
  static constexpr int KB = PITCH % 64 == 0 ? 16 : 8, kpieces = PITCH / 4 / KB;
  // V: PITCH / 8 neighbouring channels of a token, in pieces of VB bytes
  static constexpr int VB = PITCH % 128 == 0 ? 16 : PITCH % 64 == 0 ? 8 : 4, vpieces = PITCH / 8 / VB;
  static constexpr int stage = 2 * 16 * PITCH + 256;   // both tiles, and 8 bytes of scales a lane
};

template <int KIND, int PITCH, int PLANES, int NT>
struct Layout {
  using G = Geometry<PITCH>;
  static constexpr int cols = 8 * NT;
  static constexpr int ring = kWarpsD * kStagesD * G::stage;
  static constexpr int queries = G::ksteps * PLANES * NT * 32 * 8;     // b fragments, 8 bytes a lane
  static constexpr int merge = kWarpsD * cols * PITCH * 4 + kWarpsD * cols * 8;
  static constexpr int body = ring > merge ? ring : merge;
  static constexpr int bytes = body + queries + cols * 16 + cols * PITCH * 4 + cols * 8;
};

template <int KIND, int PITCH, int PLANES, int NT>
__global__ void __launch_bounds__(kWarpsD * 32) kv8_decode_kernel(const pi_kv8_attn_params p) {
  using G = Geometry<PITCH>;
  using S = Layout<KIND, PITCH, PLANES, NT>;
  constexpr int COLS = S::cols;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* s_queries = smem + S::body;
  int* s_lo = reinterpret_cast<int*>(s_queries + S::queries);   // per column: first and last position seen, factor of the scores
  int* s_hi = s_lo + COLS;
  float* s_factor = reinterpret_cast<float*>(s_hi + COLS);
  float* s_out = s_factor + 2 * COLS;                           // this CTA's result [column][pitch], then (max, sum) per column
  float* s_stat = s_out + COLS * PITCH;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint32_t split, splits;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(split));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const int kvh = blockIdx.x / splits, seq = blockIdx.y, bs = p.block_size;
  const int row_begin = max(0, min(p.cu_rows[seq], p.n_rows)), row_end = min(p.cu_rows[seq + 1], p.n_rows);
  const int ncols = (row_end - row_begin) * p.group;
  // one tile of columns as the grid is cut; the loop is for sequences that bring more rows than the call said
  for (int col0 = blockIdx.z * COLS; col0 < ncols; col0 += gridDim.z * COLS) {
  // columns: what they see, and their queries as b fragments
  int lo_all = 0x7fffffff, hi_all = -1;
  for (int c = tid; c < COLS; c += kWarpsD * 32) {
    int lo = 0x7fffffff, hi = -1;
    if (col0 + c < ncols) {
      const int pos = p.row_pos[row_begin + (col0 + c) / p.group];
      lo = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
      hi = pos;
    }
    s_lo[c] = lo;
    s_hi[c] = hi;
  }
  // a warp per column: the power of two that brings its query to [-1, 1]
  for (int c = warp; c < COLS; c += kWarpsD) {
    float top = 0.f, x[(PITCH + 31) / 32];
    const bool live = col0 + c < ncols;
    const size_t at = live ? (size_t)(row_begin + (col0 + c) / p.group) * p.q_stride + (size_t)(kvh * p.group + (col0 + c) % p.group) * p.head_dim : 0;
#pragma unroll
    for (int i = 0; i < (PITCH + 31) / 32; ++i) {
      const int d = lane + 32 * i;
      x[i] = live && d < p.head_dim ? pi_load_as_f32(p.q, at + d, p.dtype) : 0.f;
      top = fmaxf(top, fabsf(x[i]));
    }
    top = pi_warp_max(top);
    // exponent e with 2^(e-1) <= top < 2^e; 2^e and 2^-e both have to be f32
    const int e = top > 0.f && top < INFINITY ? min(max(ilogbf(top) + 1, -126), 126) : 0;
    const float shrink = scalbnf(1.f, -e);
    if (lane == 0) s_factor[c] = scalbnf(1.f, e) * p.scale2;
#pragma unroll
    for (int i = 0; i < (PITCH + 31) / 32; ++i) {
      const int d = lane + 32 * i;
      if (d >= PITCH) continue;
      // channel d is byte b of word j of lane tt
      const int piece = d / (G::KB * 4), in = d % (G::KB * 4), tt = in / G::KB, j = piece * (G::KB / 4) + in % G::KB / 4, b = d & 3;
      const float v = x[i] * shrink;
      const __half hi = __float2half_rn(v);
#pragma unroll
      for (int pl = 0; pl < PLANES; ++pl) {
        __half* f = reinterpret_cast<__half*>(s_queries + ((((size_t)j * PLANES + pl) * NT + c / 8) * 32 + (c % 8) * 4 + tt) * 8);
        f[b] = pl == 0 ? hi : __float2half_rn(v - __half2float(hi));
      }
    }
  }
  __syncthreads();
  for (int c = 0; c < COLS; ++c)
    if (s_hi[c] >= 0) {
      lo_all = min(lo_all, s_lo[c]);
      hi_all = max(hi_all, s_hi[c]);
    }
  hi_all = min(hi_all, (int)min((long long)p.lens[seq], (long long)p.max_blocks) * bs - 1);

  // tiles: 16 tokens of a block, dealt to the warps of all CTAs in turn
  const int per_block = (bs + 15) / 16;
  const int first_block = lo_all / bs, tiles = hi_all < lo_all ? 0 : (hi_all / bs - first_block + 1) * per_block;
  const int worker = (int)split * kWarpsD + warp, workers = (int)splits * kWarpsD;
  const int mine = tiles > worker ? (tiles - worker + workers - 1) / workers : 0;
  const int32_t* table = p.tables + (size_t)seq * p.max_blocks;
  const uint32_t ring = pi_mma::smem_addr(smem) + (uint32_t)warp * kStagesD * G::stage;
  const size_t tile_bytes = (size_t)bs * PITCH;

  auto tile_block = [&](int i) -> int {   // the physical block of this warp's tile i, -1: not mapped
    if (i >= mine) return -1;
    const int b = __ldg(table + first_block + (worker + i * workers) / per_block);
    return b < p.num_blocks ? b : -1;
  };
  auto request = [&](int i, int block) {
    if (block >= 0) {
      const int sub = (worker + i * workers) % per_block * 16;
      const size_t tile = ((size_t)block * p.kv_heads + kvh) * 2;
      const uint8_t* k = p.codes + tile * tile_bytes;
      const uint8_t* v = k + tile_bytes;
      const uint32_t to = ring + (uint32_t)(i % kStagesD) * G::stage;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint8_t* row = k + (size_t)min(sub + g + 8 * r, bs - 1) * PITCH + t * G::KB;
#pragma unroll
        for (int c = 0; c < G::kpieces; ++c) copy_async<G::KB>(to + ((r * G::kpieces + c) * 32 + lane) * G::KB, row + c * G::KB * 4);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint8_t* row = v + (size_t)min(sub + 2 * t + (r & 1) + (r & 2) * 4, bs - 1) * PITCH + g * (PITCH / 8);
#pragma unroll
        for (int c = 0; c < G::vpieces; ++c) copy_async<G::VB>(to + 16 * PITCH + ((r * G::vpieces + c) * 32 + lane) * G::VB, row + c * G::VB);
      }
      copy_async<8>(to + 32 * PITCH + lane * 8, p.scales + tile);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

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

  int blocks[kStagesD];
#pragma unroll
  for (int i = 0; i < kStagesD - 1; ++i) {
    blocks[i] = tile_block(i);
    request(i, blocks[i]);
  }
  int ahead = tile_block(kStagesD - 1);
  for (int i = 0; i < mine; ++i) {
    blocks[kStagesD - 1] = ahead;
    request(i + kStagesD - 1, ahead);
    ahead = tile_block(i + kStagesD);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStagesD - 1) : "memory");
    const int block = blocks[0];
#pragma unroll
    for (int k = 0; k < kStagesD - 1; ++k) blocks[k] = blocks[k + 1];
    if (block < 0) continue;
    const unsigned char* at = smem + (size_t)warp * kStagesD * G::stage + (size_t)(i % kStagesD) * G::stage;
    const int tile = worker + i * workers, sub = tile % per_block * 16;
    const int base = (first_block + tile / per_block) * bs + sub, valid = min(16, bs - sub);
    const float2 scale = *reinterpret_cast<const float2*>(at + 32 * PITCH + lane * 8);

    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    {
      uint32_t kw[2][PITCH / 16];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < G::kpieces; ++c) {
          const unsigned char* from = at + ((r * G::kpieces + c) * 32 + lane) * G::KB;
          load_words<G::KB>(&kw[r][c * G::KB / 4], from);
        }
#pragma unroll
      for (int j = 0; j < G::ksteps; ++j) {
        const uint32_t w0 = unsign<KIND>(kw[0][j]), w1 = unsign<KIND>(kw[1][j]);
        const uint32_t a0 = widen_lo<KIND>(w0), a1 = widen_lo<KIND>(w1), a2 = widen_hi<KIND>(w0), a3 = widen_hi<KIND>(w1);
#pragma unroll
        for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 b = *reinterpret_cast<const uint2*>(s_queries + (((size_t)j * PLANES + pl) * NT + n) * 256 + lane * 8);
            mma_f16(s[n], a0, a1, a2, a3, b.x, b.y);
          }
      }
    }

    // softmax of the tile: this lane has tokens g and g + 8 of columns 2 t and 2 t + 1
    uint32_t pw[NT][2][PLANES];
    bool part = !(scale.y < INFINITY);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float most[2], shrink[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = factor[n][e] * (scale.x * kUnit<KIND>);
        const int t0 = base + g, t1 = t0 + 8;
        s[n][e] = t0 >= lo[n][e] && t0 <= hi[n][e] && g < valid ? s[n][e] * f : -INFINITY;
        s[n][2 + e] = t1 >= lo[n][e] && t1 <= hi[n][e] && g + 8 < valid ? s[n][2 + e] * f : -INFINITY;
        most[e] = fmaxf(s[n][e], s[n][2 + e]);
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        most[0] = fmaxf(most[0], __shfl_xor_sync(0xffffffffu, most[0], o));
        most[1] = fmaxf(most[1], __shfl_xor_sync(0xffffffffu, most[1], o));
      }
      bool grown = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float now = fmaxf(top[n][e], most[e]), zero = now == -INFINITY ? 0.f : now;
        shrink[e] = exp2_fast(top[n][e] - zero);
        grown |= now != top[n][e];
        top[n][e] = now;
        s[n][e] = exp2_fast(s[n][e] - zero + kTopWeight);
        s[n][2 + e] = exp2_fast(s[n][2 + e] - zero + kTopWeight);
        sum[n][e] = sum[n][e] * shrink[e] + (s[n][e] + s[n][2 + e]);
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int m = 0; m < G::mtiles; ++m) {
          out[n][m][0] *= shrink[0];
          out[n][m][1] *= shrink[1];
          out[n][m][2] *= shrink[0];
          out[n][m][3] *= shrink[1];
        }
      }
      const uint32_t h0 = pack_f16(s[n][0], s[n][1]), h1 = pack_f16(s[n][2], s[n][3]);
      pw[n][0][0] = transpose8(h0);
      pw[n][1][0] = transpose8(h1);
      if constexpr (PLANES == 2) {
        pw[n][0][1] = transpose8(pack_rest(s[n][0], s[n][1], h0));
        pw[n][1][1] = transpose8(pack_rest(s[n][2], s[n][3], h1));
      }
    }

    const float unit = scale.y * kUnit<KIND>;
    uint32_t vw[4][PITCH / 32];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < G::vpieces; ++c) {
        const unsigned char* from = at + 16 * PITCH + ((r * G::vpieces + c) * 32 + lane) * G::VB;
        load_words<G::VB>(&vw[r][c * G::VB / 4], from);
      }
#pragma unroll
    for (int w = 0; w < PITCH / 32; ++w) {
      const uint32_t v0 = unsign<KIND>(vw[0][w]), v1 = unsign<KIND>(vw[1][w]), v2 = unsign<KIND>(vw[2][w]), v3 = unsign<KIND>(vw[3][w]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t x = __byte_perm(v0, v1, half ? 0x7362 : 0x5140), y = __byte_perm(v2, v3, half ? 0x7362 : 0x5140);
        const uint32_t a0 = widen_lo<KIND>(x), a1 = widen_hi<KIND>(x), a2 = widen_lo<KIND>(y), a3 = widen_hi<KIND>(y);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) mma_f16(d, a0, a1, a2, a3, pw[n][0][pl], pw[n][1][pl]);
          float* o = out[n][2 * w + half];
          if (!part) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(unit, d[e], o[e]);
          } else {   // values that are not finite reach the columns that see them and no others
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (base + valid > lo[n][e & 1] && base <= hi[n][e & 1]) o[e] = fmaf(unit, d[e], o[e]);
          }
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // the ring becomes the place where the warps' results meet

  float* s_part = reinterpret_cast<float*>(smem);                    // [warp][column][pitch]
  float2* s_warp = reinterpret_cast<float2*>(s_part + kWarpsD * COLS * PITCH);   // (max, sum) [warp][column]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = sum[n][e];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      const int c = n * 8 + 2 * t + e;
      if (g == 0) s_warp[warp * COLS + c] = make_float2(top[n][e], l);
#pragma unroll
      for (int m = 0; m < G::mtiles; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) s_part[((size_t)warp * COLS + c) * PITCH + g * (PITCH / 8) + 2 * m + r] = out[n][m][2 * r + e];
    }
  __syncthreads();
  // the CTA's result, not yet divided by its sum
  for (int i = tid; i < COLS * PITCH; i += kWarpsD * 32) {
    const int c = i / PITCH;
    float m = -INFINITY, v = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarpsD; ++w) m = fmaxf(m, s_warp[w * COLS + c].x);
#pragma unroll
    for (int w = 0; w < kWarpsD; ++w) {
      const float2 st = s_warp[w * COLS + c];
      const float f = join_factor(st.x, st.y, m);
      if (f != 0.f) {
        v = fmaf(f, s_part[(size_t)w * COLS * PITCH + i], v);
        l = fmaf(f, st.y, l);
      }
    }
    s_out[i] = v;
    if (i % PITCH == 0) {
      s_stat[2 * c] = m;
      s_stat[2 * c + 1] = l;
    }
  }
  if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();

  auto peer = [&](const float* mine_at, uint32_t rank) -> float {
    uint32_t a;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(pi_mma::smem_addr(mine_at)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
  };
  // every CTA of the cluster finishes its share of the columns' channels
  const int live = min(COLS, ncols - col0), total = live * PITCH, share = (total + (int)splits - 1) / (int)splits;
  for (int i = (int)split * share + tid; i < min(total, ((int)split + 1) * share); i += kWarpsD * 32) {
    const int c = i / PITCH, d = i % PITCH;
    if (d >= p.head_dim) continue;
    float m = -INFINITY, v = 0.f, l = 0.f;
    for (uint32_t r = 0; r < splits; ++r) m = fmaxf(m, peer(s_stat + 2 * c, r));
    for (uint32_t r = 0; r < splits; ++r) {
      const float lr = peer(s_stat + 2 * c + 1, r), f = join_factor(peer(s_stat + 2 * c, r), lr, m);
      if (f != 0.f) {
        v = fmaf(f, peer(s_out + i, r), v);
        l = fmaf(f, lr, l);
      }
    }
    const int row = row_begin + (col0 + c) / p.group, head = kvh * p.group + (col0 + c) % p.group;
    pi_store_f32_as(p.out, (size_t)row * p.out_stride + (size_t)head * p.head_dim + d, p.dtype, l == 0.f ? 0.f : v / l);
  }
  if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
  }
}

template <int KIND, int PITCH, int PLANES, int NT>
pi_status launch_decode(pi_ctx* ctx, const pi_kv8_attn_params& p, dim3 grid, int splits) {
  constexpr int bytes = Layout<KIND, PITCH, PLANES, NT>::bytes;
  auto kernel = kv8_decode_kernel<KIND, PITCH, PLANES, NT>;
  static pi_smem_grant grant;
  if (grant.of(ctx) < (size_t)bytes) {
    PI_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    PI_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    grant.of(ctx) = bytes;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarpsD * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)splits, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  PI_CUDA(ctx, cudaLaunchKernelEx(&cfg, kernel, p));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}

template <int PITCH>
pi_status launch_decode_pitch(pi_ctx* ctx, int kind, int planes, int nt, const pi_kv8_attn_params& p, dim3 grid, int splits) {
  if (kind == PI_INT8) {
    if (planes == 2) return nt == 1 ? launch_decode<PI_INT8, PITCH, 2, 1>(ctx, p, grid, splits) : launch_decode<PI_INT8, PITCH, 2, 2>(ctx, p, grid, splits);
    return nt == 1 ? launch_decode<PI_INT8, PITCH, 1, 1>(ctx, p, grid, splits) : launch_decode<PI_INT8, PITCH, 1, 2>(ctx, p, grid, splits);
  }
  if (planes == 2) return nt == 1 ? launch_decode<PI_E4M3, PITCH, 2, 1>(ctx, p, grid, splits) : launch_decode<PI_E4M3, PITCH, 2, 2>(ctx, p, grid, splits);
  return nt == 1 ? launch_decode<PI_E4M3, PITCH, 1, 1>(ctx, p, grid, splits) : launch_decode<PI_E4M3, PITCH, 1, 2>(ctx, p, grid, splits);
}
extern template pi_status launch_decode_pitch<32>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int);
extern template pi_status launch_decode_pitch<64>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int);
extern template pi_status launch_decode_pitch<96>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int);
extern template pi_status launch_decode_pitch<128>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int);
extern template pi_status launch_decode_pitch<192>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int);
extern template pi_status launch_decode_pitch<256>(pi_ctx*, int, int, int, const pi_kv8_attn_params&, dim3, int);

}  // namespace pi_kv8
