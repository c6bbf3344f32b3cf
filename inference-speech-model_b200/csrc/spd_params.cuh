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

// Launches kfn(args) with programmatic dependent launch: its CTAs may start as soon as those of the kernel
// before it on the stream have signalled, and wait (griddepcontrol.wait) for that kernel's results.
template <typename K, typename... Args>
inline int launch_dependent(K kfn, dim3 grid, dim3 block, size_t smem, cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kfn, args...) == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
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

struct SampleParams {  // a token a row by temperature, top-k, top-p, min-p (sample_rows.cu)
  const void* x;
  const unsigned char* skip;  // [cols] or null: columns that count as -inf
  const float* uniforms;      // [rows]
  const float* temperature;   // [rows], or null: the same for all; so the next three
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;
  long long* out;   // int64 [rows]
  float* logprobs;  // [rows] or null
  int rows, cols;
  long long ld;     // elements between rows
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

struct SpanParams {  // attention of groups of queries, each over the keys of its own span (span_attn.cu)
  const int* lens;    // [G] keys of each span
  const int* cu;      // [G + 1] queries of each group, or null: query g
  const int* tables;  // [G][max_blocks] of paged spans
  const int* slots;   // [G] planes of unpaged spans, or null: plane g
  int paged, max_keys;            // most keys a span can have
  int max_blocks, blocks;         // table columns; blocks of the pool (or planes)
  int bs_log2;                    // block size
  int N, G, Hq, Hkv, D;
  int per_tile;       // queries a tile: its rows are queries x the heads of one key/value head
  int q_rows;         // rows of a Q box
  float scale_log2;   // scale * log2(e)
  void* out;          // [N][Hq][D]; null: results stay partial
  float* whole;       // [N * Hq][D + 4] partial results of items in one piece (out null)
  int2* row_desc;     // [N * Hkv] where the pieces of a query's heads lie (out null)
  float* pieces;      // [2 * grid][rows][D + 4]
  ::int4* cta_desc;     // [grid] items that begin in a CTA and end in a later one (out given)
  int piece_rows;     // rows a piece has room for
  int* err;
  unsigned long long wait_ns;
};

struct SpanTensors {  // what a span call reads by TMA; strides in elements
  const void *q, *k, *v;
  long long q_st, q_sh;         // token and head
  long long kv_st, kv_sh, kv_sb;  // row, head and plane of unpaged keys and values
};

struct OwnParams {  // a sequence's own keys, joined with its prefix's results (own_attn.cu)
  const void* q;
  const void* k_pool;
  const void* v_pool;
  const int* block_tables;
  const int* context_lens;
  void* out;              // [B][Hq][D]
  long long q_st, q_sh;   // token and head strides of q (elements)
  int B, Hq, Hkv, D, max_blocks, num_blocks, bs_log2;
  int chunks, least;      // CTAs per (sequence, head tile), and the fewest tokens for one
  float scale_log2;
  int* counters;          // [B * Hkv * head tiles] arrivals, left at zero
  float* partials;        // [B * Hq][chunks][D + 4]
  int G;                  // groups that may have a prefix (0: none, and no kernel before this one)
  const int* cu_groups;
  const int* prefix_lens;
  const float* whole;
  const int2* row_desc;
  const float* pieces;
  int piece_rows, span_ctas;  // rows of a piece, and CTAs that left pieces
  int* err;
};

}  // namespace spd
