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

// What the attention kernels get.  Columns of a CTA are (row, head) pairs: column c is head c % group of row c / group of its tile.
struct pi_kv8_attn_params {
  const void* q;
  void* out;
  size_t q_stride, out_stride;   // elements between rows
  int dtype;                     // PI_F32, PI_BF16 or PI_F16, of q and out
  const uint8_t* codes;          // of the layer
  const float* scales;
  int num_blocks, block_size, kv_heads, head_dim, group;
  const int32_t *tables, *lens, *cu_rows, *row_pos;
  int max_blocks, n_seqs, n_rows;
  int window;                    // <= 0: none
  float scale2;                  // of the scores, times log2(e)
};
pi_status pi_launch_kv8_decode(pi_ctx* ctx, const pi_kv8_pool* pool, const pi_kv8_attn_params& p, int max_seq_rows, int max_context);

#ifdef __CUDACC__
__device__ __forceinline__ float pi_load_as_f32(const void* base, size_t i, int dtype) {
  if (dtype == PI_F32) return static_cast<const float*>(base)[i];
  if (dtype == PI_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(static_cast<const __half*>(base)[i]);
}
__device__ __forceinline__ void pi_store_f32_as(void* base, size_t i, int dtype, float v) {
  if (dtype == PI_F32) static_cast<float*>(base)[i] = v;
  else if (dtype == PI_BF16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(base)[i] = __float2half_rn(v);
}
#endif
