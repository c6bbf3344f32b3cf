// spd_int4.cuh — the page format of the 4-bit K/V pool, shared by the kernels that write
// and read it.
//
// Pool: uint8 [num_blocks][kv_heads][page_bytes].  A page holds one block's tokens of one
// key/value head as P = D / 64 planes of 64 dimensions, each with a scale and a zero point
// per token:
//   K codes   [P][block_size][32 bytes]   byte b: dimension 2b (low 4 bits) and 2b + 1
//   K params  [P][block_size]             (scale, zero), two fp16
//   V codes, V params                     the same
// A code c stands for c * scale + zero.  One (block, head) page is contiguous and a
// multiple of 16 bytes, so an attention kernel fetches keys, values and their parameters
// with one bulk copy.  64 dimensions per scale cost half a bit per value; they are what a
// quarter-warp's 8-byte shared-memory reads cover (32 bytes a token), so a tile of 8 tokens
// is read without bank conflicts.
#pragma once

#include <stddef.h>

namespace spd {
namespace int4 {

constexpr int kPlane = 64;     // dimensions that share one scale and zero point
constexpr int kRowBytes = 32;  // codes of one token in one plane
constexpr int kParamBytes = 4;

__host__ __device__ constexpr int half_bytes(int planes, int block_size) {
  return planes * block_size * (kRowBytes + kParamBytes);  // the K or the V part of a page
}
__host__ __device__ constexpr int page_bytes(int planes, int block_size) { return 2 * half_bytes(planes, block_size); }

}  // namespace int4
}  // namespace spd
