// The 8-bit KV cache: its pool and the write of a step's keys and values.
//
// One scale s per (block, head, K or V).  The rows of a step that fall into one block are a unit: with m the largest magnitude
// among them,
//     s = max(s of the tokens in front of them, m (1 / top)),  code = round(x / s),   top = 127 (int8) or 448 (e4m3),
// and where s has grown, the codes in front of them are encoded again: round(code s_old / s).  A block that is written from its
// first token on starts without a past.  All of it is IEEE f32 (1 / top as a constant, one product, one division, one rounding a code), so that codes do
// not depend on how the rows were dealt to warps.
//
// A warp takes a unit's one head and side: four channels a lane, the rows' magnitudes first, then the codes; the second reading
// comes from the caches.  Nothing is shared between warps.
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
  const int64_t* slots;
  int n_rows, rows_per_warp;
};

// Channels d .. d + 3 of the vector at element `at`, zeros behind the last.
__device__ __forceinline__ float4 load4(const WriteParams& p, const void* base, size_t at, int d) {
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d >= p.head_dim) return x;
  if (p.wide) {
    if (p.dtype == PI_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at + d);
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at + d);
    if (p.dtype == PI_BF16)
      return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  x.x = pi_load_as_f32(base, at + d, p.dtype);
  if (d + 1 < p.head_dim) x.y = pi_load_as_f32(base, at + d + 1, p.dtype);
  if (d + 2 < p.head_dim) x.z = pi_load_as_f32(base, at + d + 2, p.dtype);
  if (d + 3 < p.head_dim) x.w = pi_load_as_f32(base, at + d + 3, p.dtype);
  return x;
}

template <int KIND>
__device__ __forceinline__ uint32_t encode(float x, float s) {
  if (!(s > 0.f)) return 0;   // an empty block, or one whose values are not finite
  const float y = __fdiv_rn(x, s);
  if (KIND == PI_E4M3) return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)(int)fminf(fmaxf(roundf(y), -127.f), 127.f) & 0xffu;
}
template <int KIND>
__device__ __forceinline__ float decode(uint32_t code) {
  if (KIND == PI_E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
  return (float)(int8_t)code;
}
template <int KIND>
__device__ __forceinline__ uint32_t encode4(float4 x, float s) {
  return encode<KIND>(x.x, s) | encode<KIND>(x.y, s) << 8 | encode<KIND>(x.z, s) << 16 | encode<KIND>(x.w, s) << 24;
}

template <int KIND>
__global__ void __launch_bounds__(kWriteWarps * 32) kv8_write_kernel(const WriteParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bs = p.block_size;
  const long long job = (long long)blockIdx.x * kWriteWarps + warp;
  const int per_row = p.kv_heads * 2, hs = (int)(job % per_row), head = hs >> 1, side = hs & 1;
  const long long row0 = job / per_row * p.rows_per_warp;
  pi_grid_dependency_wait();
  if (row0 >= p.n_rows) return;
  const void* src = side ? p.v : p.k;
  const size_t stride = side ? p.v_stride : p.k_stride, col = (size_t)head * p.head_dim;
  const long long row_end = min(row0 + p.rows_per_warp, (long long)p.n_rows);

  long long before = row0 > 0 ? p.slots[row0 - 1] : -1;
  if (before >= 0) before /= bs;
  for (long long r = row0; r < row_end;) {
    const long long slot = p.slots[r], block = slot >= 0 ? slot / bs : -1;
    if (block < 0 || block >= p.num_blocks || block == before) {   // unmapped, or a unit that began further up
      before = block;
      ++r;
      continue;
    }
    // the unit: rows r .. end - 1, all in this block
    long long end = r + 1;
    while (true) {
      const long long i = end + lane;
      const long long there = i < p.n_rows ? p.slots[i] : -1;
      const unsigned out = __ballot_sync(0xffffffffu, there < block * bs || there >= (block + 1) * bs);
      if (out) {
        end += __ffs(out) - 1;
        break;
      }
      end += 32;
    }
    const int first = (int)(slot - block * bs);
    float most = 0.f;
    bool odd = false;   // an infinity or NaN: the block's scale says so, whatever comes later
    for (int d = 4 * lane; d < p.pitch; d += 128)
#pragma unroll 4
      for (long long i = r; i < end; ++i) {
        const float4 x = load4(p, src, (size_t)i * stride + col, d);
        const float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
        odd |= !(fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY && fabsf(x.z) < INFINITY && fabsf(x.w) < INFINITY);
        most = fmaxf(most, m);
      }
    most = pi_warp_max(most);
    odd = __any_sync(0xffffffffu, odd);
    const size_t tile = ((size_t)block * p.kv_heads + head) * 2 + side;
    const float old = first > 0 ? p.scales[tile] : 0.f;
    float s = fmaxf(old, __fmul_rn(most, KIND == PI_E4M3 ? 1.f / 448.f : 1.f / 127.f));
    if (odd || old != old) s = __int_as_float(0x7fffffff);
    uint8_t* codes = p.codes + tile * (size_t)bs * p.pitch;
    if (s != old && s == s && first > 0)
      for (int d = 4 * lane; d < p.pitch; d += 128)
#pragma unroll 4
        for (int t = 0; t < first; ++t) {
          uint32_t* w = reinterpret_cast<uint32_t*>(codes + (size_t)t * p.pitch + d);
          const uint32_t c = *w;
          *w = encode4<KIND>(make_float4(__fmul_rn(decode<KIND>(c & 0xff), old), __fmul_rn(decode<KIND>(c >> 8 & 0xff), old), __fmul_rn(decode<KIND>(c >> 16 & 0xff), old),
                                         __fmul_rn(decode<KIND>(c >> 24), old)), s);
        }
    for (int d = 4 * lane; d < p.pitch; d += 128)
#pragma unroll 4
      for (long long i = r; i < end; ++i) {
        const int off = (int)(p.slots[i] - block * bs);
        *reinterpret_cast<uint32_t*>(codes + (size_t)off * p.pitch + d) = encode4<KIND>(load4(p, src, (size_t)i * stride + col, d), s);
      }
    __syncwarp();
    if (lane == 0) p.scales[tile] = s;
    before = block;
    r = end;
  }
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
  std::vector<uint8_t> codes((size_t)L.num_kv_heads * 2 * pool->pitch);
  std::vector<float> scales((size_t)L.num_kv_heads * 2);
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
  p.slots = slots_dev;
  p.n_rows = n_rows;
  // a warp looks for units that begin in this many rows: one while that leaves the GPU room, more for prompts, where most rows begin none
  p.rows_per_warp = (int)std::min<long long>(16, std::max<long long>(1, (long long)n_rows * L.num_kv_heads * 2 / (ctx->sm_count * 32ll)));
  const long long jobs = ((long long)n_rows + p.rows_per_warp - 1) / p.rows_per_warp * L.num_kv_heads * 2;
  const long long grid = (jobs + kWriteWarps - 1) / kWriteWarps;
  PI_REQUIRE(ctx, grid <= 0x7fffffffll, "too many rows");
  pi_prof_scope prof(ctx, PI_PROF_ROPE_KV);
  PI_CUDA(ctx, pi_launch_chained(ctx, pool->kind == PI_E4M3 ? kv8_write_kernel<PI_E4M3> : kv8_write_kernel<PI_INT8>, dim3((unsigned)grid), dim3(kWriteWarps * 32), 0, 1, p));
  PI_CHECK_LAUNCH(ctx);
  return PI_OK;
}

}  // extern "C"
