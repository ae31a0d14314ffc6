// Attention over the 8-bit cache: the call's checks, and which kernel takes it.
#include "pi_kv8_decode.cuh"

using namespace pi_kv8;

namespace {
constexpr int kFewColumns = 64;
}

pi_status pi_launch_kv8_decode(pi_ctx* ctx, const pi_kv8_pool* pool, pi_kv8_attn_params& p, int max_seq_rows, int max_context, int max_cols) {
  p.max_cols = max_cols;
  // eight columns a product; sixteen where a sequence brings more, so that its codes are widened half as often
  const long long cols = (long long)max_seq_rows * p.group;
  const int nt = cols <= 8 ? 1 : 2, planes = p.dtype == PI_F32 ? 2 : 1;
  const long long col_tiles = (cols + 8 * nt - 1) / (8 * nt);
  // The warps that work on one sequence's head: about as many as give every SM fourteen (what registers leave room for is sixteen), with
  // a round or more for each.  Up to eight are one CTA, more are clusters of CTAs of four, of eight where a cluster is full.
  // 64 sequences of 256 to 2048 tokens, 4 KV heads of 64: 21.5 us with 8 warps, 30 with 4, 27 with 16; 16 of 3000 to 4096, 8 of 128:
  // 31 us with 16 (4 x 4), 44 with 8, 42 with 32.
  const long long base = (long long)p.kv_heads * p.n_seqs * col_tiles;
  const long long seen = p.window > 0 ? std::min<long long>(max_context, (long long)p.window + max_seq_rows) : max_context;
  const long long rounds = (seen / 16 + 1) / (pool->pitch <= 64 && nt == 1 ? 2 : 1);
  long long n = 4;
  while (n < kMaxSplit * kMaxWarps && base * n * 2 <= 16 * ctx->sm_count && rounds >= n * 2) n *= 2;
  const int splits = n <= kMaxWarps ? 1 : (int)std::min<long long>(kMaxSplit, n / 4), warps = (int)(n / splits);
  p.by_workers = pi_divisor(splits * warps);
  const dim3 grid((unsigned)(p.kv_heads * splits), (unsigned)p.n_seqs, (unsigned)std::min<long long>(col_tiles, 65535));   // its CTAs go on to the columns behind
  switch (pool->pitch) {
    case 32: return launch_decode_pitch<32>(ctx, pool->kind, planes, nt, p, grid, splits, warps);
    case 64: return launch_decode_pitch<64>(ctx, pool->kind, planes, nt, p, grid, splits, warps);
    case 96: return launch_decode_pitch<96>(ctx, pool->kind, planes, nt, p, grid, splits, warps);
    case 128: return launch_decode_pitch<128>(ctx, pool->kind, planes, nt, p, grid, splits, warps);
    case 192: return launch_decode_pitch<192>(ctx, pool->kind, planes, nt, p, grid, splits, warps);
    default: return launch_decode_pitch<256>(ctx, pool->kind, planes, nt, p, grid, splits, warps);
  }
}

extern "C" pi_status pi_kv8_attention(pi_ctx* ctx, const pi_kv8_pool* pool, int layer, int num_heads, int dtype, const void* q_dev, size_t q_stride, void* out_dev,
                                      size_t out_stride, const pi_step_arrays* a, int n_seqs, int n_rows, int max_seq_rows, int max_context, int window, float scale) {
  PI_ENTER(ctx);
  PI_REQUIRE(ctx, pool && a, "null pointer");
  const pi_kv_layout& L = pool->L;
  PI_REQUIRE(ctx, layer >= 0 && layer < L.num_layers, "layer %d of %d", layer, L.num_layers);
  PI_REQUIRE(ctx, num_heads > 0 && num_heads % L.num_kv_heads == 0, "%d query heads do not divide into %d KV heads", num_heads, L.num_kv_heads);
  PI_REQUIRE(ctx, dtype == PI_F32 || dtype == PI_BF16 || dtype == PI_F16, "queries of kind %d: PI_F32, PI_BF16 or PI_F16 are wanted", dtype);
  PI_REQUIRE(ctx, n_rows >= 0 && n_seqs >= 0, "negative row or sequence count");
  PI_REQUIRE(ctx, n_seqs <= 65535, "%d sequences: at most 65535", n_seqs);
  if (n_rows == 0 || n_seqs == 0) return PI_OK;
  PI_REQUIRE(ctx, q_dev && out_dev && a->tables && a->lens && a->cu_rows && a->row_pos, "null pointer");
  PI_REQUIRE(ctx, a->block_size == L.block_size, "the step's blocks hold %d tokens, the pool's %d", a->block_size, L.block_size);
  PI_REQUIRE(ctx, a->max_blocks > 0 && n_seqs <= a->max_seqs && n_rows <= a->max_rows, "%d sequences and %d rows: the step's arrays have room for %d and %d", n_seqs, n_rows,
             a->max_seqs, a->max_rows);
  PI_REQUIRE(ctx, (long long)n_rows * num_heads / L.num_kv_heads <= 0x7fffffffll - (1 << 21), "%d rows of %d query heads are too many", n_rows, num_heads);
  PI_REQUIRE(ctx, (long long)a->max_blocks * L.block_size <= 0x7fffffffll - 4096, "tables of %d blocks of %d tokens reach beyond position 2^31", a->max_blocks, L.block_size);
  const size_t row = (size_t)num_heads * L.head_dim, size = dtype == PI_F32 ? 4 : 2;
  PI_REQUIRE(ctx, (q_stride >= row && out_stride >= row) || n_rows == 1, "rows of %zu values cannot be %zu (queries) and %zu (results) apart", row, q_stride, out_stride);
  PI_REQUIRE(ctx, ((uintptr_t)q_dev | (uintptr_t)out_dev) % size == 0, "queries and results must be aligned to their type");
  PI_REQUIRE(ctx, max_seq_rows > 0 && max_context > 0, "the most rows of a sequence and the longest context must be positive");
  PI_REQUIRE(ctx, scale > 0.f && scale * 1.4426950408889634f < INFINITY, "a scale of %g", (double)scale);
  pi_kv8_attn_params p = {};
  p.q = q_dev;
  p.out = out_dev;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.dtype = dtype;
  const size_t tiles = (size_t)L.num_blocks * L.num_kv_heads * 2;
  p.codes = pool->codes + (size_t)layer * tiles * L.block_size * pool->pitch;
  p.scales = pool->scales + (size_t)layer * tiles;
  p.side_bytes = (uint32_t)(L.block_size * pool->pitch);
  p.block_bytes = (uint32_t)(L.num_kv_heads * 2 * p.side_bytes);
  const auto wide = [&](const void* at, size_t stride) { return L.head_dim % 4 == 0 && stride % 4 == 0 && (uintptr_t)at % (4 * size) == 0; };
  p.q_wide = wide(q_dev, q_stride);
  p.out_wide = wide(out_dev, out_stride);
  p.num_blocks = L.num_blocks;
  p.block_size = L.block_size;
  p.kv_heads = L.num_kv_heads;
  p.head_dim = L.head_dim;
  p.group = num_heads / L.num_kv_heads;
  p.by_group = pi_divisor(p.group);
  p.by_block = pi_divisor(L.block_size);
  p.by_tiles = pi_divisor((L.block_size + 15) / 16);
  p.tables = a->tables;
  p.lens = a->lens;
  p.cu_rows = a->cu_rows;
  p.row_pos = a->row_pos;
  p.max_blocks = a->max_blocks;
  p.n_seqs = n_seqs;
  p.n_rows = n_rows;
  p.window = window;
  p.scale2 = scale * 1.4426950408889634f;
  pi_prof_scope prof(ctx, PI_PROF_ATTENTION);
  max_seq_rows = std::min(max_seq_rows, n_rows);
  // Sequences of up to 64 columns beside longer portions: each kernel takes its own, whatever the lengths on the device are.  A sequence
  // alone is a portion.  4096 positions, 8 KV heads of 128: 4 sequences of 32 columns take 37 us on the one kernel and 94 on the other, one
  // of 128 columns 34 and 35.
  if ((long long)max_seq_rows * p.group <= kFewColumns || !pi_kv8_prefill_takes(pool, p)) return pi_launch_kv8_decode(ctx, pool, p, max_seq_rows, max_context, 0x7fffffff);
  if (n_seqs == 1) return pi_launch_kv8_prefill(ctx, pool, p, 0, max_context);
  if (p.group <= kFewColumns) PI_TRY(pi_launch_kv8_decode(ctx, pool, p, kFewColumns / p.group, max_context, kFewColumns));
  return pi_launch_kv8_prefill(ctx, pool, p, p.group <= kFewColumns ? kFewColumns : 0, max_context);
}
