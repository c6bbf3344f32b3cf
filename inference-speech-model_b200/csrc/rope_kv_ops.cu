// rope_kv_ops.cu — rotary position embedding fused with the write of new keys and values
// into a paged cache (16/32-bit pools, or the 4-bit pool of spd_int4.cuh), and the read of
// cached tokens back out of the 4-bit pool.
//
// Rotation by position p over the first `rot` dimensions of a head, with r = rot / 2 angles
// a_i (cos and sin tables in fp32, [positions][r]):
//   y[i]     = x[i] * cos(a_i) - x[j] * sin(a_i)      j = i + r (halves) or the odd partner
//   y[j]     = x[j] * cos(a_i) + x[i] * sin(a_i)      of an even i (interleaved)
// in fp32 with separate products and sum, rounded once to the output type.  Dimensions past
// `rot` pass through.  Values and keys go to row (position % block_size) of block
// block_tables[b][position / block_size].
//
// 4 bits: each token's 64 consecutive dimensions of a head share
//   scale = fp16((max - min) / 15),  zero = fp16(min)      (saturated to the fp16 range)
//   code  = clamp(rint((x - zero) / scale), 0, 15),        0 where scale is 0
// computed from the fp32 rotated keys (no rounding to the model's type in between).  A NaN
// makes its 64 values NaN (through the parameters); an infinity saturates.
#include <limits>

#include "spd_int4.cuh"
#include "spd_params.cuh"

namespace spd {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxTokens = kThreads / 32;  // tokens per CTA: one warp looks each up

// Where a packed token lives: its position and the pool row block * block_size + offset.
struct Place {
  int pos, block, off, flag;  // block < 0: nothing there (no sequence, a skipped one, or `flag`)
};

// Looks `token` up by the whole warp.  The number of sequences that end at or before the token
// is its sequence: one load per lane and a population count for up to 32 sequences, instead of
// a chain of dependent loads.  cu null: token i is sequence i.
__device__ __forceinline__ Place find_place(int token, const int* cu, int B, const int* firsts, const int* tables,
                                            int max_blocks, int num_blocks, int block_size, int max_pos, int& b) {
  const int lane = threadIdx.x & 31;
  b = token;
  if (cu) {
    int ended = 0;
    for (int s = lane; s < B; s += 32) ended += cu[s + 1] <= token;
    b = __reduce_add_sync(0xffffffffu, ended);
    if (b >= B || token < cu[b]) b = -1;
  }
  Place w{0, -1, 0, 0};
  if (b < 0) return w;
  const int first = firsts ? firsts[b] : 0;
  if (first < 0) return w;
  const long long pos = (long long)first + (cu ? token - cu[b] : 0);
  const long long blk = pos / block_size;
  if (blk >= max_blocks || pos >= max_pos) {
    w.flag = SPD_DEVERR_LENGTH;
    return w;
  }
  const int id = tables[(long long)b * max_blocks + blk];
  if (id < 0 || id >= num_blocks) {
    w.flag = SPD_DEVERR_BLOCK_ID;
    return w;
  }
  w.pos = (int)pos;
  w.block = id;
  w.off = (int)(pos - blk * block_size);
  return w;
}

// minimum / maximum that give NaN when either side is NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&y)[8]) {
  alignas(16) T o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = Elem<T>::from_f(y[i]);
#pragma unroll
  for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
    reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(o)[i];
}

// Rotates the pair chunks lo and hi by the eight angles (cc, ss).
__device__ __forceinline__ void turn(float (&lo)[8], float (&hi)[8], const float (&cc)[8], const float (&ss)[8],
                                     bool interleaved) {
  if (interleaved) {  // the 16 elements are eight neighbouring pairs: four in lo, four in hi
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = lo[2 * k], b = lo[2 * k + 1], c = hi[2 * k], d = hi[2 * k + 1];
      lo[2 * k] = __fsub_rn(__fmul_rn(a, cc[k]), __fmul_rn(b, ss[k]));
      lo[2 * k + 1] = __fadd_rn(__fmul_rn(b, cc[k]), __fmul_rn(a, ss[k]));
      hi[2 * k] = __fsub_rn(__fmul_rn(c, cc[4 + k]), __fmul_rn(d, ss[4 + k]));
      hi[2 * k + 1] = __fadd_rn(__fmul_rn(d, cc[4 + k]), __fmul_rn(c, ss[4 + k]));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float a = lo[k], b = hi[k];
      lo[k] = __fsub_rn(__fmul_rn(a, cc[k]), __fmul_rn(b, ss[k]));
      hi[k] = __fadd_rn(__fmul_rn(b, cc[k]), __fmul_rn(a, ss[k]));
    }
  }
}

// Eight values of one 64-value group to a word of codes.
__device__ __forceinline__ uint32_t encode8(const float (&y)[8], float s, float z) {
  uint32_t word = 0;
  if (s > 0.f) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      word |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(y[k], z), s)), 0.f), 15.f) << (4 * k);
  }
  return word;
}

// A CTA owns `tokens` packed tokens; a thread owns a unit of 16 dimensions of a head row (q, k
// or v head of a token): the two chunks of eight that rotate into each other (d, d + rot / 2,
// or 16 neighbours when interleaved or not rotated), so every value is loaded once and shares
// its eight angles.
template <typename T, bool INT4>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const RopeAppendParams p, int tokens) {
  __shared__ Place place[kMaxTokens];
  const int token0 = blockIdx.x * tokens, n = min(tokens, p.N - token0);
  const int warp = threadIdx.x >> 5;
  if (warp < n) {
    int b;
    const Place w = find_place(token0 + warp, p.cu_seqlens, p.B, p.positions, p.block_tables, p.max_blocks, p.num_blocks,
                               p.block_size, p.max_pos, b);
    if ((threadIdx.x & 31) == 0) {
      place[warp] = w;
      if (w.flag) set_error(p.err, w.flag);
    }
  }
  const int upr = (p.D + 15) / 16;  // units per head row
  const int hq = p.q ? p.Hq : 0;
  const int rows = hq + 2 * p.Hkv;
  const int u = threadIdx.x % upr, step = kThreads / upr;  // rows per round
  const int turned = p.rot / 16, r = p.rot / 2;
  const bool halves = u < turned && !p.interleaved;
  const int d_rot = halves ? 8 * u : 16 * u, d_rot2 = halves ? 8 * u + r : 16 * u + 8;
  const bool usable = threadIdx.x < step * upr;
  __syncthreads();
  const int total = n * rows;
  const int rounds = (total + step - 1) / step;
#pragma unroll 2
  for (int it = 0; it < rounds; ++it) {
    const int i = it * step + threadIdx.x / upr;
    const bool live = usable && i < total;  // the same for all units of a row
    const int ti = live ? i / rows : 0, row = live ? i % rows : 0;
    const Place w = place[ti];
    const long long token = token0 + ti;
    const bool is_q = row < hq, is_k = !is_q && row < hq + p.Hkv;
    const int h = is_q ? row : is_k ? row - hq : row - hq - p.Hkv;
    const T* x = is_q ? reinterpret_cast<const T*>(p.q) + token * p.q_st + h * p.q_sh
                 : is_k ? reinterpret_cast<const T*>(p.k) + token * p.k_st + h * p.k_sh
                        : reinterpret_cast<const T*>(p.v) + token * p.v_st + h * p.v_sh;
    const bool rotates = u < turned && (is_q || is_k);
    const int d0 = rotates ? d_rot : 16 * u, d1 = rotates ? d_rot2 : 16 * u + 8;
    const bool second = INT4 || d1 < p.D;
    float lo[8] = {}, hi[8] = {};
    if (live && w.block >= 0) {
      load_to_float<T, 8>(x + d0, lo);
      if (second) load_to_float<T, 8>(x + d1, hi);
      if (rotates) {
        float cc[8], ss[8];
        const long long at = (long long)w.pos * r + 8 * u;
        load_to_float<float, 8>(p.cos + at, cc);
        load_to_float<float, 8>(p.sin + at, ss);
        turn(lo, hi, cc, ss, p.interleaved);
      }
    }
    if (is_q) {  // also the zeros of a token that is not written
      if (live) {
        T* o = reinterpret_cast<T*>(p.q_out) + (token * p.Hq + h) * p.D;
        store8(o + d0, lo);
        if (second) store8(o + d1, hi);
      }
    } else if (!INT4) {
      if (live && w.block >= 0) {
        T* o = reinterpret_cast<T*>(is_k ? p.k_pool : p.v_pool) +
               (((long long)w.block * p.block_size + w.off) * p.Hkv + h) * p.D;
        store8(o + d0, lo);
        if (second) store8(o + d1, hi);
      }
    }
    if constexpr (INT4) {
      // least and largest of each plane over the row's 4, 8 or 16 threads; a thread's two chunks
      // may lie in different planes
      const int planes = p.D / int4::kPlane, pl0 = d0 / int4::kPlane, pl1 = d1 / int4::kPlane;
      float mn0 = lo[0], mx0 = lo[0], mn1 = hi[0], mx1 = hi[0];
#pragma unroll
      for (int k = 1; k < 8; ++k) {
        mn0 = min_nan(mn0, lo[k]);
        mx0 = max_nan(mx0, lo[k]);
        mn1 = min_nan(mn1, hi[k]);
        mx1 = max_nan(mx1, hi[k]);
      }
      float a0 = 0.f, b0 = 0.f, a1 = 0.f, b1 = 0.f;  // (least, largest) of each chunk's plane
      for (int pl = 0; pl < planes; ++pl) {
        float mn = INFINITY, mx = -INFINITY;
        if (pl0 == pl) mn = mn0, mx = mx0;
        if (pl1 == pl) mn = min_nan(mn, mn1), mx = max_nan(mx, mx1);
        for (int o = 1; o < upr; o <<= 1) {
          mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
        if (pl0 == pl) a0 = mn, b0 = mx;
        if (pl1 == pl) a1 = mn, b1 = mx;
      }
      if (live && !is_q && w.block >= 0) {
        const int half = int4::half_bytes(planes, p.block_size);
        unsigned char* page = reinterpret_cast<unsigned char*>(p.k_pool) +
                              ((long long)w.block * p.Hkv + h) * (2 * half) + (is_k ? 0 : half);
        auto put = [&](const float (&y)[8], int d, float mn, float mx) {
          constexpr float kMax = 65504.f;
          float s = __fdiv_rn(__fsub_rn(mx, mn), 15.f);
          s = s > kMax ? kMax : s;  // a NaN stays
          float z = mn > kMax ? kMax : mn < -kMax ? -kMax : mn;
          const __half sh = __float2half_rn(s), zh = __float2half_rn(z);
          const int slot = (d / int4::kPlane) * p.block_size + w.off, in = d % int4::kPlane;
          *reinterpret_cast<uint32_t*>(page + slot * int4::kRowBytes + in / 2) =
              encode8(y, __half2float(sh), __half2float(zh));
          if (in == 0)
            *reinterpret_cast<__half2*>(page + planes * p.block_size * int4::kRowBytes + slot * int4::kParamBytes) =
                __halves2half2(sh, zh);
        };
        put(lo, d0, a0, b0);
        put(hi, d1, a1, b1);
      }
    }
  }
}

// Tokens of the 4-bit pool back as packed k and v; a thread owns one 4-byte word (8
// dimensions) of one head's K or V row, so a warp's stores are contiguous.
template <typename T>
__global__ void __launch_bounds__(kThreads) gather_int4_kernel(const GatherInt4Params p, int tokens) {
  __shared__ Place place[kMaxTokens];
  __shared__ int owner[kMaxTokens];
  const int token0 = blockIdx.x * tokens, n = min(tokens, p.N - token0);
  const int warp = threadIdx.x >> 5;
  if (warp < n) {
    int b;
    const Place w = find_place(token0 + warp, p.cu_seqlens, p.B, p.starts, p.block_tables, p.max_blocks, p.num_blocks,
                               p.block_size, 0x7fffffff, b);
    if ((threadIdx.x & 31) == 0) {
      place[warp] = w;
      owner[warp] = b;
      if (w.flag) set_error(p.err, w.flag);
    }
  }
  __syncthreads();
  const int cpr = p.D / 8;  // words per head row
  const int per_token = 2 * p.Hkv * cpr, total = n * per_token;
  const int planes = p.D / int4::kPlane;
  const int half = int4::half_bytes(planes, p.block_size);
#pragma unroll 4
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int ti = i / per_token, rest = i % per_token;
    const int row = rest / cpr, c = rest % cpr;
    const Place w = place[ti];
    if (owner[ti] < 0) continue;  // a row of no sequence
    const bool is_k = row < p.Hkv;
    const int h = is_k ? row : row - p.Hkv;
    float y[8] = {};  // a token that is not there
    if (w.block >= 0) {
      const unsigned char* page = p.pool + ((long long)w.block * p.Hkv + h) * (2 * half) + (is_k ? 0 : half);
      const int slot = (c / 8) * p.block_size + w.off;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(page + slot * int4::kRowBytes + (c & 7) * 4);
      const float2 sz = __half22float2(*reinterpret_cast<const __half2*>(
          page + planes * p.block_size * int4::kRowBytes + slot * int4::kParamBytes));
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = fmaf((float)((word >> (4 * k)) & 15u), sz.x, sz.y);
    }
    store8(reinterpret_cast<T*>(is_k ? p.k_out : p.v_out) + ((long long)(token0 + ti) * p.Hkv + h) * p.D + c * 8, y);
  }
}

}  // namespace rope

// Tokens per CTA: one while there are fewer tokens than 16 per SM, so that a step's few tokens
// spread over the SMs, up to eight, so that the look-up of a token's place is shared.
static int tokens_per_cta(int N, int sms) {
  const int t = N / (sms * 16);
  return t < 1 ? 1 : t > rope::kMaxTokens ? rope::kMaxTokens : t;
}

int rope_append_launch(const RopeAppendParams& p, int dtype, bool int4_pool, int sms, cudaStream_t st) {
  using namespace rope;
  const int tokens = tokens_per_cta(p.N, sms);
  const dim3 grid((unsigned)((p.N + tokens - 1) / tokens)), block(kThreads);
  auto run = [&](auto tag) {
    using T = decltype(tag);
    if (int4_pool) rope_append_kernel<T, true><<<grid, block, 0, st>>>(p, tokens);
    else rope_append_kernel<T, false><<<grid, block, 0, st>>>(p, tokens);
  };
  if (dtype == SPD_F32) run(float{});
  else if (dtype == SPD_F16) run(__half{});
  else run(__nv_bfloat16{});
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

int gather_int4_launch(const GatherInt4Params& p, int dtype, int sms, cudaStream_t st) {
  using namespace rope;
  const int tokens = tokens_per_cta(p.N, sms);
  const dim3 grid((unsigned)((p.N + tokens - 1) / tokens)), block(kThreads);
  if (dtype == SPD_F32) gather_int4_kernel<float><<<grid, block, 0, st>>>(p, tokens);
  else if (dtype == SPD_F16) gather_int4_kernel<__half><<<grid, block, 0, st>>>(p, tokens);
  else gather_int4_kernel<__nv_bfloat16><<<grid, block, 0, st>>>(p, tokens);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace spd
