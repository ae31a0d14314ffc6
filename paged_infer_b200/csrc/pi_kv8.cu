// The 8-bit KV cache: its pool and the write of a step's keys and values.
//
// One scale s per (block, head, K or V).  The rows of a step that fall into one block are a unit: with m the largest magnitude
// among them,
//     s = max(s of the tokens in front of them, m (1 / top)),  code = round(x / s),   top = 127 (int8) or 448 (e4m3),
// and where s has grown, the codes in front of them are encoded again: round(code s_old / s).  A block that is written from its
// first token on starts without a past.  All of it is IEEE f32 (1 / top as a constant, one product, one division, one rounding a code), so that codes do
// not depend on how the rows were dealt to warps.
//
// A warp takes a unit's one head and side, four neighbouring channels a lane, several rows at once where a row needs fewer lanes: the
// rows of a unit of up to 16 (8 for wide heads) are loaded together and stay in registers from their magnitudes to their codes;
// longer units are read twice.  Nothing is shared between warps.
//
// The quotient: q = x r with r = RN(1 / s), and one correction by the remainder, which is RN(x / s) by Markstein's theorem while
// the remainder is exact: for quotients that matter (2^-10 is the smallest border between two codes) a multiple of 2^-56 s, a number of f32 for s
// above 2^-93.  Scales outside 1e-20 to 1e30 take the division itself.
//
// Bound: latency, of the slots, then the rows, then the codes' stores, with the warps that registers leave room for: at heads of 65 to
// 128 channels 142 of them a thread, 12 warps an SM.  Measured: 4200 rows of 8 heads of 128, bf16 to e4m3: 15 us, 1.7 TB/s, 1200 CTAs on 444
// places (31 us with rows read twice and one load at a time).
#include <math.h>

#include <algorithm>
#include <new>

#include "pi_kv8.cuh"

namespace {

constexpr int kWriteWarps = 4;

struct WriteParams {
  const void *k, *v;
  size_t k_stride, v_stride;
  int dtype;
  bool wide;                 // four channels of a row can be loaded at once
  uint8_t* codes;            // of the layer
  float* scales;
  int num_blocks, block_size, kv_heads, head_dim, pitch;
  pi_divisor by_block;
  const int64_t* slots;
  int n_rows, rows_per_warp;   // a warp looks for units that begin in this many rows, at most 16
};

template <int KIND>
__device__ __forceinline__ uint32_t encode(float y) {   // any quotient
  if (KIND == PI_E4M3) return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)(int)fminf(fmaxf(roundf(y), -127.f), 127.f) & 0xffu;
}
template <int KIND>
__device__ __forceinline__ float decode(uint32_t code) {
  if (KIND == PI_E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
  return (float)(int8_t)code;
}
// Four codes under a scale; r = RN(1 / s) where s is in the middle of the normal range, 0 elsewhere.
template <int KIND>
__device__ __forceinline__ uint32_t encode4(const float* x, float s, float r) {
  if (r == 0.f) {
    if (!(s > 0.f)) return 0;   // an empty block, or one whose values are not finite
    return encode<KIND>(__fdiv_rn(x[0], s)) | encode<KIND>(__fdiv_rn(x[1], s)) << 8 | encode<KIND>(__fdiv_rn(x[2], s)) << 16 | encode<KIND>(__fdiv_rn(x[3], s)) << 24;
  }
  float y[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const float q = __fmul_rn(x[b], r);
    y[b] = __fmaf_rn(__fmaf_rn(-q, s, x[b]), r, q);
    if (KIND == PI_E4M3 && x[b] == 0.f) y[b] = x[b];   // the remainder has lost the sign of -0, which e4m3 has
  }
  if (KIND == PI_E4M3)
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3) << 16;
  // halves away from zero: |y| < 127.5, and the number below 1/2 added to a half makes the next whole one, to less than a half does not
  uint32_t c[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) c[b] = (uint32_t)(int)(y[b] + copysignf(0.49999997f, y[b]));
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// LANES of them to a row, GROUPS of four channels a lane.
template <int KIND, int LANES, int GROUPS>
__global__ void __launch_bounds__(kWriteWarps * 32) kv8_write_kernel(const WriteParams p) {
  constexpr int AT_ONCE = 32 / LANES, MOST = GROUPS == 1 ? 16 : 8, STEPS = MOST / AT_ONCE;   // rows at once, rows in registers
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bs = p.block_size, sub = lane / LANES, d0 = 4 * (lane % LANES);
  const long long job = (long long)blockIdx.x * kWriteWarps + warp;
  const int per_row = p.kv_heads * 2, hs = (int)(job % per_row), head = hs >> 1, side = hs & 1;
  const long long row0 = job / per_row * p.rows_per_warp;
  pi_grid_dependency_wait();
  if (row0 >= p.n_rows) return;
  const void* src = side ? p.v : p.k;
  const size_t stride = side ? p.v_stride : p.k_stride, col = (size_t)head * p.head_dim;

  // lane l looks at row row0 - 1 + l: its block, -1 where it has none
  auto place_of = [&](long long row, int& off) -> int {
    off = 0;
    if (row < 0 || row >= p.n_rows) return -1;
    const long long slot = p.slots[row];
    if (slot < 0) return -1;
    const long long b = slot < 0x7fffffffll ? p.by_block((int)slot) : slot / bs;
    off = (int)(slot - b * bs);
    return b < p.num_blocks ? (int)b : -1;
  };
  int my_off, other;
  const int mine = place_of(row0 - 1 + lane, my_off), before = __shfl_up_sync(0xffffffffu, mine, 1);
  unsigned leaders = __ballot_sync(0xffffffffu, lane >= 1 && lane <= p.rows_per_warp && mine >= 0 && mine != before);
  for (; leaders; leaders &= leaders - 1) {
    const int l0 = __ffs(leaders) - 1, block = __shfl_sync(0xffffffffu, mine, l0);
    const long long r = row0 - 1 + l0;
    // the unit: rows r .. r + n - 1, all in this block
    const unsigned out = __ballot_sync(0xffffffffu, lane > l0 && mine != block);
    long long n = (out ? __ffs(out) - 1 : 32) - l0;
    while (!out) {
      const unsigned more = __ballot_sync(0xffffffffu, place_of(r + n + lane, other) != block);
      n += more ? __ffs(more) - 1 : 32;
      if (more) break;
    }
    const int first = __shfl_sync(0xffffffffu, my_off, l0);
    const size_t tile = ((size_t)block * p.kv_heads + head) * 2 + side;
    uint8_t* codes = p.codes + tile * (size_t)bs * p.pitch;
    const float old = first > 0 ? p.scales[tile] : 0.f;
    float x[STEPS][GROUPS][4];
    const size_t start = (size_t)r * stride + col;
    auto load = [&](long long from) {   // up to MOST rows of the unit, their loads under way together
      if (p.wide && p.dtype == PI_F32) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const long long at = from + i * AT_ONCE + sub;
            const int d = d0 + g * 4 * LANES;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at < n && d < p.head_dim) v = *reinterpret_cast<const float4*>(static_cast<const float*>(src) + start + (size_t)at * stride + d);
            x[i][g][0] = v.x, x[i][g][1] = v.y, x[i][g][2] = v.z, x[i][g][3] = v.w;
          }
      } else if (p.wide) {
        uint2 raw[STEPS][GROUPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const long long at = from + i * AT_ONCE + sub;
            const int d = d0 + g * 4 * LANES;
            raw[i][g] = make_uint2(0, 0);
            if (at < n && d < p.head_dim) raw[i][g] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(src) + start + (size_t)at * stride + d);
          }
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const uint2 w = raw[i][g];
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
            const bool bf = p.dtype == PI_BF16;
            x[i][g][0] = bf ? __uint_as_float(w.x << 16) : a.x, x[i][g][1] = bf ? __uint_as_float(w.x & 0xffff0000u) : a.y;
            x[i][g][2] = bf ? __uint_as_float(w.y << 16) : b.x, x[i][g][3] = bf ? __uint_as_float(w.y & 0xffff0000u) : b.y;
          }
      } else {
#pragma unroll 1
        for (int i = 0; i < STEPS; ++i) {
          const long long at = from + i * AT_ONCE + sub;
          float y[GROUPS][4];
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) pi_load4_as_f32(y[g], src, start + (size_t)at * stride + d0 + g * 4 * LANES, p.dtype, at < n ? p.head_dim - d0 - g * 4 * LANES : 0, false);
#pragma unroll
          for (int e = 0; e < STEPS; ++e)
            if (e == i) {
#pragma unroll
              for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                for (int b = 0; b < 4; ++b) x[e][g][b] = y[g][b];
            }
        }
      }
    };
    float most = 0.f;
    bool odd = false;   // an infinity or NaN: the block's scale says so, whatever comes later
    for (long long from = 0; from < n; from += MOST) {
      load(from);
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            odd |= !(fabsf(x[i][g][b]) < INFINITY);
            most = fmaxf(most, fabsf(x[i][g][b]));
          }
    }
    most = pi_warp_max(most);
    odd = __any_sync(0xffffffffu, odd);
    float s = fmaxf(old, __fmul_rn(most, KIND == PI_E4M3 ? 1.f / 448.f : 1.f / 127.f));
    if (odd || old != old) s = __int_as_float(0x7fffffff);
    const float recip = s > 1e-20f && s < 1e30f ? __frcp_rn(s) : 0.f;
    if (s != old && s == s && first > 0)   // the tokens in front, in the larger scale
      for (int t = sub; t < first; t += AT_ONCE)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int d = d0 + g * 4 * LANES;
          if (d >= p.pitch) continue;
          uint32_t* w = reinterpret_cast<uint32_t*>(codes + (size_t)t * p.pitch + d);
          const uint32_t c = *w;
          const float y[4] = {__fmul_rn(decode<KIND>(c & 0xff), old), __fmul_rn(decode<KIND>(c >> 8 & 0xff), old), __fmul_rn(decode<KIND>(c >> 16 & 0xff), old),
                              __fmul_rn(decode<KIND>(c >> 24), old)};
          *w = encode4<KIND>(y, s, recip);
        }
    __syncwarp();
    for (long long from = 0; from < n; from += MOST) {
      if (n > MOST) load(from);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const long long at = from + i * AT_ONCE + sub;
        int off = __shfl_sync(0xffffffffu, my_off, (int)min(l0 + at, 31ll));
        if (at < n) {
          if (l0 + at > 31) off = (int)(p.slots[r + at] - (long long)block * bs);
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const int d = d0 + g * 4 * LANES;
            if (d < p.pitch) *reinterpret_cast<uint32_t*>(codes + (size_t)off * p.pitch + d) = encode4<KIND>(x[i][g], s, recip);
          }
        }
      }
      __syncwarp();
    }
    if (lane == 0) p.scales[tile] = s;
  }
}

template <int KIND>
cudaError_t launch_write(pi_ctx* ctx, const WriteParams& p, unsigned grid) {
  const dim3 g(grid), b(kWriteWarps * 32);
  if (p.pitch == 32) return pi_launch_chained(ctx, kv8_write_kernel<KIND, 8, 1>, g, b, 0, 1, p);
  if (p.pitch == 64) return pi_launch_chained(ctx, kv8_write_kernel<KIND, 16, 1>, g, b, 0, 1, p);
  if (p.pitch <= 128) return pi_launch_chained(ctx, kv8_write_kernel<KIND, 32, 1>, g, b, 0, 1, p);
  return pi_launch_chained(ctx, kv8_write_kernel<KIND, 32, 2>, g, b, 0, 1, p);
}

}  // namespace

extern "C" {

pi_status pi_kv8_pool_create(pi_ctx* ctx, const pi_kv_layout* layout, int kind, void* codes_dev_or_null, float* scales_dev_or_null, pi_kv8_pool** out) {
  PI_ENTER(ctx);
  PI_REQUIRE(ctx, layout && out, "null pointer");
  *out = nullptr;
  PI_REQUIRE(ctx, layout->num_layers > 0 && layout->num_blocks > 0 && layout->block_size > 0 && layout->num_kv_heads > 0 && layout->head_dim > 0,
             "KV layout fields must be positive");
  PI_REQUIRE(ctx, kind == PI_INT8 || kind == PI_E4M3, "codes of kind %d: an 8-bit cache holds PI_INT8 or PI_E4M3", kind);
  PI_REQUIRE(ctx, layout->head_dim <= 256 && layout->block_size <= 4096 && layout->num_kv_heads <= 1024,
             "an 8-bit cache takes head_dim <= 256, block_size <= 4096 and at most 1024 KV heads (got %d, %d, %d)", layout->head_dim, layout->block_size,
             layout->num_kv_heads);
  PI_REQUIRE(ctx, !codes_dev_or_null == !scales_dev_or_null, "codes and scales are either both the caller's or both the pool's");
  PI_REQUIRE(ctx, ((uintptr_t)codes_dev_or_null & 15) == 0 && ((uintptr_t)scales_dev_or_null & 7) == 0, "codes must lie on a 16-byte boundary, scales on an 8-byte one");
  const double bytes_wanted = (double)layout->num_layers * layout->num_blocks * layout->num_kv_heads * 2 * layout->block_size * pi_kv8_pitch_of(layout->head_dim);
  PI_REQUIRE(ctx, bytes_wanted < 1e15, "a pool of %g bytes", bytes_wanted);   // sizes and offsets fit 64 bits
  pi_kv8_pool* pool = new (std::nothrow) pi_kv8_pool();
  if (!pool) return pi_fail(ctx, PI_ERR_OOM, "host allocation failed");
  pool->L = *layout;
  pool->kind = kind;
  pool->pitch = pi_kv8_pitch_of(layout->head_dim);
  pool->codes = static_cast<uint8_t*>(codes_dev_or_null);
  pool->scales = scales_dev_or_null;
  if (!codes_dev_or_null) {
    pool->owns = true;
    cudaError_t e = cudaMalloc(&pool->codes, pool->code_bytes());
    if (e == cudaSuccess) e = cudaMalloc(&pool->scales, pool->scale_count() * sizeof(float));
    if (e != cudaSuccess) {
      const size_t bytes = pool->code_bytes();
      cudaGetLastError();
      pi_kv8_pool_destroy(pool);
      return pi_fail(ctx, PI_ERR_OOM, "allocating a %.2f GiB KV pool: %s", bytes / (double)(1 << 30), cudaGetErrorString(e));
    }
  }
  *out = pool;
  return PI_OK;
}

void pi_kv8_pool_destroy(pi_kv8_pool* pool) {
  if (!pool) return;
  if (pool->owns) {
    if (pool->codes) cudaFree(pool->codes);
    if (pool->scales) cudaFree(pool->scales);
  }
  delete pool;
}

size_t pi_kv8_pool_bytes(const pi_kv8_pool* pool) { return pool ? pool->code_bytes() + pool->scale_count() * sizeof(float) : 0; }
int pi_kv8_pool_pitch(const pi_kv8_pool* pool) { return pool ? pool->pitch : 0; }

pi_status pi_kv8_copy_block(pi_ctx* ctx, pi_kv8_pool* pool, int32_t src, int32_t dst) {
  PI_ENTER(ctx);
  PI_REQUIRE(ctx, pool, "null pool");
  PI_REQUIRE(ctx, src != dst, "copy_block called with src == dst");
  const pi_kv_layout& L = pool->L;
  PI_REQUIRE(ctx, src >= 0 && src < L.num_blocks && dst >= 0 && dst < L.num_blocks, "block %d -> %d outside the pool's %d blocks", src, dst, L.num_blocks);
  // a block is one span per layer
  for (const auto& [base, span] : {std::pair<uint8_t*, size_t>{pool->codes, (size_t)L.num_kv_heads * 2 * L.block_size * pool->pitch},
                                   std::pair<uint8_t*, size_t>{reinterpret_cast<uint8_t*>(pool->scales), (size_t)L.num_kv_heads * 2 * sizeof(float)}})
    for (int l = 0; l < L.num_layers; ++l) {
      uint8_t* layer = base + (size_t)l * L.num_blocks * span;
      PI_CUDA(ctx, cudaMemcpyAsync(layer + dst * span, layer + src * span, span, cudaMemcpyDeviceToDevice, ctx->stream));
    }
  return PI_OK;
}

pi_status pi_kv8_read_token(pi_ctx* ctx, const pi_kv8_pool* pool, int layer, int32_t block, int tok, float* k_host_out, float* v_host_out) {
  PI_ENTER(ctx);
  PI_REQUIRE(ctx, pool && k_host_out && v_host_out, "null pointer");
  const pi_kv_layout& L = pool->L;
  PI_REQUIRE(ctx, layer >= 0 && layer < L.num_layers && block >= 0 && block < L.num_blocks && tok >= 0 && tok < L.block_size,
             "KV address (layer %d, block %d, token %d) out of range", layer, block, tok);
  std::vector<uint8_t> codes;
  std::vector<float> scales;
  try {
    codes.resize((size_t)L.num_kv_heads * 2 * pool->pitch);
    scales.resize((size_t)L.num_kv_heads * 2);
  } catch (const std::bad_alloc&) {
    return pi_fail(ctx, PI_ERR_OOM, "host allocation failed");
  }
  const size_t tile = ((size_t)layer * L.num_blocks + block) * L.num_kv_heads * 2;
  PI_CUDA(ctx, cudaMemcpy2DAsync(codes.data(), pool->pitch, pool->codes + tile * L.block_size * pool->pitch + (size_t)tok * pool->pitch, (size_t)L.block_size * pool->pitch,
                                 pool->pitch, (size_t)L.num_kv_heads * 2, cudaMemcpyDeviceToHost, ctx->stream));
  PI_CUDA(ctx, cudaMemcpyAsync(scales.data(), pool->scales + tile, scales.size() * sizeof(float), cudaMemcpyDeviceToHost, ctx->stream));
  PI_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  for (int h = 0; h < L.num_kv_heads; ++h)
    for (int d = 0; d < L.head_dim; ++d)
      for (int side = 0; side < 2; ++side) {
        const uint8_t c = codes[((size_t)h * 2 + side) * pool->pitch + d];
        const float x = pool->kind == PI_INT8 ? (float)(int8_t)c : __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
        (side ? v_host_out : k_host_out)[(size_t)h * L.head_dim + d] = x * scales[h * 2 + side];
      }
  return PI_OK;
}

pi_status pi_kv8_write(pi_ctx* ctx, pi_kv8_pool* pool, int layer, int dtype, const void* k_dev, size_t k_stride, const void* v_dev, size_t v_stride,
                       const int64_t* slots_dev, int n_rows) {
  PI_ENTER(ctx);
  PI_REQUIRE(ctx, pool, "null pool");
  const pi_kv_layout& L = pool->L;
  PI_REQUIRE(ctx, layer >= 0 && layer < L.num_layers, "layer %d of %d", layer, L.num_layers);
  PI_REQUIRE(ctx, dtype == PI_F32 || dtype == PI_BF16 || dtype == PI_F16, "keys and values of kind %d: PI_F32, PI_BF16 or PI_F16 are wanted", dtype);
  PI_REQUIRE(ctx, n_rows >= 0, "negative row count");
  if (n_rows == 0) return PI_OK;
  PI_REQUIRE(ctx, k_dev && v_dev && slots_dev, "null pointer");
  const size_t row = (size_t)L.num_kv_heads * L.head_dim;
  PI_REQUIRE(ctx, (k_stride >= row && v_stride >= row) || n_rows == 1, "rows of %zu values cannot be %zu (K) and %zu (V) apart", row, k_stride, v_stride);
  const size_t size = dtype == PI_F32 ? 4 : 2;
  PI_REQUIRE(ctx, ((uintptr_t)k_dev | (uintptr_t)v_dev) % size == 0, "keys and values must be aligned to their type");
  WriteParams p = {};
  p.k = k_dev;
  p.v = v_dev;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.dtype = dtype;
  p.wide = L.head_dim % 4 == 0 && k_stride % 4 == 0 && v_stride % 4 == 0 && ((uintptr_t)k_dev | (uintptr_t)v_dev) % (4 * size) == 0;
  const size_t tiles = (size_t)L.num_blocks * L.num_kv_heads * 2;
  p.codes = pool->codes + (size_t)layer * tiles * L.block_size * pool->pitch;
  p.scales = pool->scales + (size_t)layer * tiles;
  p.num_blocks = L.num_blocks;
  p.block_size = L.block_size;
  p.kv_heads = L.num_kv_heads;
  p.head_dim = L.head_dim;
  p.pitch = pool->pitch;
  p.by_block = pi_divisor(L.block_size);
  p.slots = slots_dev;
  p.n_rows = n_rows;
  // a warp looks for units that begin in this many rows: one while that leaves the GPU room, more for prompts, where most rows begin none
  p.rows_per_warp = (int)std::min<long long>(16, std::max<long long>(1, (long long)n_rows * L.num_kv_heads * 2 / (ctx->sm_count * 32ll)));
  const long long jobs = ((long long)n_rows + p.rows_per_warp - 1) / p.rows_per_warp * L.num_kv_heads * 2;
  const long long grid = (jobs + kWriteWarps - 1) / kWriteWarps;
  PI_REQUIRE(ctx, grid <= 0x7fffffffll, "too many rows");
  pi_prof_scope prof(ctx, PI_PROF_ROPE_KV);
  PI_CUDA(ctx, pool->kind == PI_E4M3 ? launch_write<PI_E4M3>(ctx, p, (unsigned)grid) : launch_write<PI_INT8>(ctx, p, (unsigned)grid));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}

}  // extern "C"
