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

// Sequence of packed token i: the b with cu[b] <= i < cu[b + 1], or -1 past the end.
__device__ __forceinline__ int sequence_of(const int* cu, int B, int i) {
  if (i < cu[0] || i >= cu[B]) return -1;
  int lo = 0, hi = B - 1;  // the largest b with cu[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
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

// One CTA per packed token; a thread owns 8 consecutive dimensions of one of the token's
// Hq + 2 * Hkv head rows (q heads, k heads, v heads).
template <typename T, bool INT4>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const RopeAppendParams p) {
  const int token = blockIdx.x;
  const int cpr = p.D / 8;  // chunks per head row
  const int hq = p.q ? p.Hq : 0;
  const int rows = hq + 2 * p.Hkv;
  const int total = rows * cpr;
  int b = token, flag = 0, phys = -1;
  if (p.cu_seqlens) b = sequence_of(p.cu_seqlens, p.B, token);
  const int first = b < 0 ? -1 : p.positions[b];  // < 0: no sequence, or a skipped one
  const long long pos = (long long)first + (p.cu_seqlens && b >= 0 ? token - p.cu_seqlens[b] : 0);
  const long long blk = pos / p.block_size;
  if (first >= 0) {
    if (blk >= p.max_blocks || pos >= p.max_pos) flag = SPD_DEVERR_LENGTH;
    else phys = p.block_tables[(long long)b * p.max_blocks + blk];
    if (!flag && (phys < 0 || phys >= p.num_blocks)) flag = SPD_DEVERR_BLOCK_ID;
  }
  if (first < 0 || flag) {  // nothing is written but zeros in the token's row of q_out
    if (flag && threadIdx.x == 0) set_error(p.err, flag);
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x; i < hq * cpr; i += kThreads)
      store8(reinterpret_cast<T*>(p.q_out) + (long long)token * p.Hq * p.D + i * 8, zero);
    return;
  }
  const int off = (int)(pos - blk * p.block_size);
  const int r = p.rot / 2;
  const float* cs = p.cos + pos * r;
  const float* sn = p.sin + pos * r;

  const int rounds = (total + kThreads - 1) / kThreads;
  for (int it = 0; it < rounds; ++it) {
    const int i = it * kThreads + threadIdx.x;
    const bool live = i < total;  // a 4-bit group of 8 threads is live or dead as a whole
    const int row = live ? i / cpr : 0, c = live ? i % cpr : 0;
    const int d0 = c * 8;
    const bool is_q = row < hq, is_k = !is_q && row < hq + p.Hkv;
    const int h = is_q ? row : is_k ? row - hq : row - hq - p.Hkv;
    const T* x = is_q ? reinterpret_cast<const T*>(p.q) + token * p.q_st + h * p.q_sh
                 : is_k ? reinterpret_cast<const T*>(p.k) + token * p.k_st + h * p.k_sh
                        : reinterpret_cast<const T*>(p.v) + token * p.v_st + h * p.v_sh;
    float y[8];
    load_to_float<T, 8>(x + d0, y);
    if ((is_q || is_k) && d0 < p.rot) {
      if (p.interleaved) {
        float cc[4], ss[4];
        load_to_float<float, 4>(cs + d0 / 2, cc);
        load_to_float<float, 4>(sn + d0 / 2, ss);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float a = y[2 * k], o = y[2 * k + 1];
          y[2 * k] = __fsub_rn(__fmul_rn(a, cc[k]), __fmul_rn(o, ss[k]));
          y[2 * k + 1] = __fadd_rn(__fmul_rn(o, cc[k]), __fmul_rn(a, ss[k]));
        }
      } else {
        float o[8], cc[8], ss[8];
        const bool low = d0 < r;
        const int a0 = low ? d0 : d0 - r;
        load_to_float<T, 8>(x + (low ? d0 + r : d0 - r), o);
        load_to_float<float, 8>(cs + a0, cc);
        load_to_float<float, 8>(sn + a0, ss);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          y[k] = low ? __fsub_rn(__fmul_rn(y[k], cc[k]), __fmul_rn(o[k], ss[k]))
                     : __fadd_rn(__fmul_rn(y[k], cc[k]), __fmul_rn(o[k], ss[k]));
      }
    }
    if (is_q) {
      if (live) store8(reinterpret_cast<T*>(p.q_out) + ((long long)token * p.Hq + h) * p.D + d0, y);
    } else if (!INT4) {
      if (live)
        store8(reinterpret_cast<T*>(is_k ? p.k_pool : p.v_pool) +
                   (((long long)phys * p.block_size + off) * p.Hkv + h) * p.D + d0, y);
    }
    if constexpr (INT4) {
      float mn = y[0], mx = y[0];
#pragma unroll
      for (int k = 1; k < 8; ++k) {
        mn = min_nan(mn, y[k]);
        mx = max_nan(mx, y[k]);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      }
      if (live && !is_q) {
        constexpr float kMax = 65504.f;
        float s = __fdiv_rn(__fsub_rn(mx, mn), 15.f);
        s = s > kMax ? kMax : s;  // a NaN stays
        float z = mn > kMax ? kMax : mn < -kMax ? -kMax : mn;
        const __half sh = __float2half_rn(s), zh = __float2half_rn(z);
        s = __half2float(sh);
        z = __half2float(zh);
        uint32_t word = 0;
        if (s > 0.f) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float t = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(y[k], z), s)), 0.f), 15.f);
            word |= (uint32_t)t << (4 * k);
          }
        }
        const int planes = p.D / int4::kPlane, plane = c / 8;
        const int half = int4::half_bytes(planes, p.block_size);
        unsigned char* page = reinterpret_cast<unsigned char*>(p.k_pool) + ((long long)phys * p.Hkv + h) * (2 * half) +
                              (is_k ? 0 : half);
        const int slot = plane * p.block_size + off;
        *reinterpret_cast<uint32_t*>(page + slot * int4::kRowBytes + (c & 7) * 4) = word;
        if ((c & 7) == 0)
          *reinterpret_cast<__half2*>(page + planes * p.block_size * int4::kRowBytes + slot * int4::kParamBytes) =
              __halves2half2(sh, zh);
      }
    }
  }
}

// Tokens of the 4-bit pool back as packed k and v: one CTA per packed token; a thread owns
// one 4-byte word (8 dimensions) of one head's K or V row.
template <typename T>
__global__ void __launch_bounds__(kThreads) gather_int4_kernel(const GatherInt4Params p) {
  const int token = blockIdx.x;
  const int cpr = p.D / 8;
  const int total = 2 * p.Hkv * cpr;
  const int b = sequence_of(p.cu_seqlens, p.B, token);
  if (b < 0) return;
  const int start = p.starts ? p.starts[b] : 0;
  const long long pos = (long long)max(start, 0) + (token - p.cu_seqlens[b]);
  const long long blk = pos / p.block_size;
  bool ok = start >= 0;  // a skipped sequence's rows are zeros
  int phys = 0;
  if (ok && blk >= p.max_blocks) {
    if (threadIdx.x == 0) set_error(p.err, SPD_DEVERR_LENGTH);
    ok = false;
  } else if (ok) {
    phys = p.block_tables[(long long)b * p.max_blocks + blk];
    if (phys < 0 || phys >= p.num_blocks) {
      if (threadIdx.x == 0) set_error(p.err, SPD_DEVERR_BLOCK_ID);
      ok = false;
    }
  }
  const int off = (int)(pos - blk * p.block_size);
  const int planes = p.D / int4::kPlane;
  const int half = int4::half_bytes(planes, p.block_size);
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int row = i / cpr, c = i % cpr;
    const bool is_k = row < p.Hkv;
    const int h = is_k ? row : row - p.Hkv;
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // a token the tables do not reach
    if (ok) {
      const unsigned char* page = p.pool + ((long long)phys * p.Hkv + h) * (2 * half) + (is_k ? 0 : half);
      const int slot = (c / 8) * p.block_size + off;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(page + slot * int4::kRowBytes + (c & 7) * 4);
      const float2 sz = __half22float2(*reinterpret_cast<const __half2*>(
          page + planes * p.block_size * int4::kRowBytes + slot * int4::kParamBytes));
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = fmaf((float)((word >> (4 * k)) & 15u), sz.x, sz.y);
    }
    store8(reinterpret_cast<T*>(is_k ? p.k_out : p.v_out) + ((long long)token * p.Hkv + h) * p.D + c * 8, y);
  }
}

}  // namespace rope

int rope_append_launch(const RopeAppendParams& p, int dtype, bool int4_pool, cudaStream_t st) {
  using namespace rope;
  const dim3 grid((unsigned)p.N), block(kThreads);
  auto run = [&](auto tag) {
    using T = decltype(tag);
    if (int4_pool) rope_append_kernel<T, true><<<grid, block, 0, st>>>(p);
    else rope_append_kernel<T, false><<<grid, block, 0, st>>>(p);
  };
  if (dtype == SPD_F32) run(float{});
  else if (dtype == SPD_F16) run(__half{});
  else run(__nv_bfloat16{});
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

int gather_int4_launch(const GatherInt4Params& p, int dtype, cudaStream_t st) {
  using namespace rope;
  const dim3 grid((unsigned)p.N), block(kThreads);
  if (dtype == SPD_F32) gather_int4_kernel<float><<<grid, block, 0, st>>>(p);
  else if (dtype == SPD_F16) gather_int4_kernel<__half><<<grid, block, 0, st>>>(p);
  else gather_int4_kernel<__nv_bfloat16><<<grid, block, 0, st>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace spd
