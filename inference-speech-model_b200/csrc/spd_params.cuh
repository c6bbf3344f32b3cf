// spd_params.cuh — kernel parameter blocks shared by the kernels and the ABI layer.
// Passed to kernels by value (they live in the constant parameter bank).
#pragma once

#include <atomic>

#include "spd_common.cuh"

namespace spd {

// Raises kernel K's dynamic shared-memory limit, once per device (one bit each).
template <auto K>
inline bool allow_smem(size_t bytes) {
  static std::atomic<unsigned long long> seen{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = 1ull << (dev & 63);
  if (seen.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return false;
  seen.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

struct PagedParams {
  const void* q;
  void* k_pool;
  void* v_pool;
  const int* block_tables;
  const int* context_lens;
  void* out;
  const void* k_new;
  const void* v_new;
  int B, H, max_blocks, num_blocks;
  float scale_log2;  // scale * log2(e)
  int* err;          // workspace error word
  int* work;         // [0] next item to take, [1] CTAs done taking (both left at zero)
  int* counters;     // [B * H] ints kept in the workspace layout; the current kernels leave them unused
  float* partials;   // [B * ceil(max_blocks / kItemUnits) * H * (D + 8)]
  int stages;
  int table_in_smem;  // the whole block table is bulk-copied into shared memory
  unsigned long long wait_ns;  // bound on each wait that makes progress
};

struct CrossParams {
  const void* q;
  const void* k;
  const void* v;
  const int* valid_lens;
  void* out;
  int B, H, T_max;
  long long kv_batch_stride, kv_head_stride;  // elements
  float scale_log2;
  int* err;
  int* work;        // [0] next item to take, [1] CTAs done taking (both left at zero)
  float* partials;  // [B*H*kCrossMaxItems * (D + 2)]: one row per item
  int stages;
  int item_units;   // units (of the kernel's row chunk) per work item
  unsigned long long wait_ns;  // bound on each wait that makes progress
};

struct AppendParams {
  const unsigned char* k_src;
  const unsigned char* v_src;
  long long sb, sh, st;  // source strides in bytes
  unsigned char* k_pool;
  unsigned char* v_pool;
  const int* block_tables;
  const int* positions;
  int B, T, H, row_bytes, block_size, max_blocks, num_blocks;
  int* err;
};

struct AddLnParams {  // residual add + LayerNorm (decoder_layer_ops.cu)
  const void* x;
  const void* delta;  // or null: y = LayerNorm(x), x_out not written
  const void* gamma;
  const void* beta;
  void* x_out;
  void* y;
  int rows, cols;
  long long y_ld;  // elements between rows of y
  float eps;
};

struct ArgmaxParams {  // greedy token pick over rows (decoder_layer_ops.cu)
  const void* x;
  const void* skip;  // uint8 [cols] or null: columns scored as -inf
  long long* out;    // int64 [rows]
  int rows, cols;
  long long ld;      // elements between rows
  int vec;           // rows start 16-byte aligned: 16-byte loads
};

struct GatherParams {
  const unsigned char* pool;
  const int* block_tables;
  const int* seq_lens;
  unsigned char* out;
  int B, H, row_bytes, block_size, max_blocks, num_blocks, T_out, zero_pad;
  long long out_batch_stride;  // bytes
  int* err;
};

struct RopeAppendParams {  // rotation + K/V append (rope_kv_ops.cu)
  const void* q;  // or null
  const void* k;
  const void* v;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh;  // token and head strides (elements)
  void* q_out;                                   // [N][Hq][D]
  const float* cos;                              // [max_pos][rot / 2]
  const float* sin;
  void* k_pool;  // 16/32-bit pools, or the 4-bit pool with v_pool null
  void* v_pool;
  const int* block_tables;
  const int* positions;   // [B]
  const int* cu_seqlens;  // [B + 1] or null: token i belongs to sequence i
  int N, B, Hq, Hkv, D, rot, interleaved, max_pos;
  int block_size, max_blocks, num_blocks;
  int* err;
};

struct GatherInt4Params {  // tokens of a 4-bit pool back as packed k, v (rope_kv_ops.cu)
  const unsigned char* pool;
  const int* block_tables;
  const int* cu_seqlens;  // [B + 1]
  const int* starts;      // [B] or null: 0
  void* k_out;            // [N][Hkv][D]
  void* v_out;
  int N, B, Hkv, D, block_size, max_blocks, num_blocks;
  int* err;
};

struct PromptParams {  // attention of packed prompts (prompt_attn.cu)
  void* out;          // [Nq][Hq][D]
  const void* v;      // [Nk][Hkv][D], by token and head strides (elements)
  long long v_st, v_sh;
  const int* cu_q;    // [B + 1]
  const int* cu_k;    // [B + 1]
  int Nq, Nk, B, Hq, Hkv, D, causal;
  int pack;           // query heads of one key/value head that share a tile (a power of two)
  int ranked;         // items in the order of their length
  float scale_log2;   // scale * log2(e)
  int* err;
  unsigned long long wait_ns;
};

// How a 4-bit decode call is split: CTAs per (sequence, head tile) and the fewest tokens for one.
struct Int4Split {
  int chunks, least;
};

struct DecodeInt4Params {  // single-token attention over a 4-bit pool (paged_decode_attn_int4.cu)
  const void* q;
  const unsigned char* pool;
  const int* block_tables;
  const int* context_lens;
  void* out;
  int dtype;
  int B, Hq, Hkv, max_blocks, num_blocks;
  int least;          // tokens a CTA takes at least
  int chunks;         // CTAs per (sequence, head tile)
  float scale_log2;   // scale * log2(e)
  int* err;           // workspace error word
  int* counters;      // [B * Hkv * head tiles] arrivals, left at zero
  float* partials;    // [B * Hq][chunks][D + 4]
  unsigned long long wait_ns;
};

}  // namespace spd
