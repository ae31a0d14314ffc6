// The 8-bit KV cache: declarations shared by its write, its attention kernels and the C ABI.
#pragma once

#include <cuda_fp8.h>

#include "pi_common.cuh"

// codes [layer][block][kv_head][k|v][token][pitch], scales [layer][block][kv_head][k|v]; a value is code * scale.
struct pi_kv8_pool {
  pi_kv_layout L;
  int kind = PI_INT8;        // PI_INT8 or PI_E4M3
  int pitch = 0;             // bytes from token to token, zeros behind head_dim
  uint8_t* codes = nullptr;
  float* scales = nullptr;
  bool owns = false;
  size_t code_bytes() const { return (size_t)L.num_layers * L.num_blocks * L.num_kv_heads * 2 * L.block_size * pitch; }
  size_t scale_count() const { return (size_t)L.num_layers * L.num_blocks * L.num_kv_heads * 2; }
};

// Bytes of a token's codes of one head: lanes of the attention kernels take equal shares of these widths in whole words.
inline int pi_kv8_pitch_of(int head_dim) {
  for (int p : {32, 64, 96, 128, 192, 256})
    if (p >= head_dim) return p;
  return 0;
}

// Division of 0 <= n < 2^31 by a constant: a product and a shift (Granlund and Montgomery, "Division by invariant integers using
// multiplication").
struct pi_divisor {
  uint32_t mul = 0, shift = 0;
  pi_divisor() = default;
  explicit pi_divisor(uint32_t d) {
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
#endif
};

// What the attention kernels get.  Columns of a CTA are (row, head) pairs: column c is head c % group of row c / group of its tile.
struct pi_kv8_attn_params {
  const void* q;
  void* out;
  size_t q_stride, out_stride;   // elements between rows
  int dtype;                     // PI_F32, PI_BF16 or PI_F16, of q and out
  const uint8_t* codes;          // of the layer
  const float* scales;
  int num_blocks, block_size, kv_heads, head_dim, group;
  uint32_t side_bytes, block_bytes;   // of K or V of a head, of a block
  bool q_wide, out_wide;         // four channels of a row can be moved at once
  pi_divisor by_group, by_block, by_tiles, by_workers;   // tiles: of 16 tokens in a block; workers: warps that share a sequence's head
  const int32_t *tables, *lens, *cu_rows, *row_pos;
  int max_blocks, n_seqs, n_rows;
  int window;                    // <= 0: none
  float scale2;                  // of the scores, times log2(e)
  int max_cols;                  // decode: sequences with more columns are another kernel's
};
// Sequences of at most max_cols columns (rows times group), and those of more than min_cols.
pi_status pi_launch_kv8_decode(pi_ctx* ctx, const pi_kv8_pool* pool, pi_kv8_attn_params& p, int max_seq_rows, int max_context, int max_cols);
bool pi_kv8_prefill_takes(const pi_kv8_pool* pool, const pi_kv8_attn_params& p);
pi_status pi_launch_kv8_prefill(pi_ctx* ctx, const pi_kv8_pool* pool, const pi_kv8_attn_params& p, int min_cols, int max_context);

// A launch on the context's stream that may begin while the kernel ahead of it ends (every kernel waits for that one before it touches
// memory), in clusters of `cluster` CTAs along x.
template <typename P>
cudaError_t pi_launch_chained(pi_ctx* ctx, void (*kernel)(const P), dim3 grid, dim3 block, size_t smem, int cluster, const P& params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (ctx->opt_pdl) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs++].val.clusterDim = {(unsigned)cluster, 1, 1};
  }
  return cudaLaunchKernelEx(&cfg, kernel, params);
}

#ifdef __CUDACC__
__device__ __forceinline__ float pi_load_as_f32(const void* base, size_t i, int dtype) {
  if (dtype == PI_F32) return static_cast<const float*>(base)[i];
  if (dtype == PI_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(static_cast<const __half*>(base)[i]);
}
// Four values from element i on, zeros behind the first `left`; wide: their address is a multiple of four elements.
__device__ __forceinline__ void pi_load4_as_f32(float* x, const void* base, size_t i, int dtype, int left, bool wide) {
  x[0] = x[1] = x[2] = x[3] = 0.f;
  if (left <= 0) return;
  if (wide) {
    if (dtype == PI_F32) {
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
      return;
    }
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
    if (dtype == PI_BF16) {
      x[0] = __uint_as_float(w.x << 16), x[1] = __uint_as_float(w.x & 0xffff0000u), x[2] = __uint_as_float(w.y << 16), x[3] = __uint_as_float(w.y & 0xffff0000u);
      return;
    }
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    return;
  }
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (b < left) x[b] = pi_load_as_f32(base, i + b, dtype);
}
__device__ __forceinline__ void pi_store_f32_as(void* base, size_t i, int dtype, float v) {
  if (dtype == PI_F32) static_cast<float*>(base)[i] = v;
  else if (dtype == PI_BF16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(base)[i] = __float2half_rn(v);
}
__device__ __forceinline__ void pi_store4_f32_as(const float* y, void* base, size_t i, int dtype, int left, bool wide) {
  if (wide) {
    if (dtype == PI_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = make_float4(y[0], y[1], y[2], y[3]);
    } else if (dtype == PI_BF16) {
      __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]), b = __floats2bfloat162_rn(y[2], y[3]);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    } else {
      __half2 a = __floats2half2_rn(y[0], y[1]), b = __floats2half2_rn(y[2], y[3]);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    }
    return;
  }
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (b < left) pi_store_f32_as(base, i + b, dtype, y[b]);
}
#endif
