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
// makes its 64 values NaN (through the parameters), as 64 equal infinities do (max - min is one);
// an infinity among others saturates.
//
// What bounds them: HBM for prompts, since each value is read once and written once (a 4-bit row as
// 4.5 bits per value) and the rotation is a few operations; the latency of a few dependent loads
// (sequence, table, row) for a decode step.  So a CTA looks up the places of its tokens once, a thread
// keeps its dimensions for all of them, and for few tokens a CTA takes one.
// Measured in replayed graphs (a lone call in brackets): a step's 64 tokens, 12 heads of 64, fp16: 2.8 us
// (5.7); 16 prompts of 200 to 2,000 tokens, 32/8 heads of 128, bf16 (468 MB): 87 us (94), 5.4 TB/s, 0.82
// of a plain copy's rate.  Into 4 bits, 7 prompts of up to 4,001 tokens, 16/8 heads of 128 (199 MB): 55 us,
// 3.6 TB/s: the groups' exchanges and parameters are a chain that 28 warps an SM do not cover (66 % of the
// issue slots, no pipe full).  16 prefixes of 1,000 to 8,000 tokens out of 4 bits, 8 heads of 128
// (390 MB): 63 us (69), 6.1 TB/s.
#include "spd_int4.cuh"
#include "spd_params.cuh"

namespace spd {
namespace rope {

// Threads and most tokens of a CTA.  Small CTAs: rows of q are done before rows that are quantised,
// and a CTA's room is free as soon as its own rows are done (256 threads: 59 us in place of 55 for the
// 7 prompts above into 4 bits, 91 in place of 87 for the 16 into 16 bits).  Eight tokens share a
// look-up (four: 57 and 88 us; two: 64 and 93); where nothing but copying is left, four (the 16
// prefixes: 64 us, eight 71, sixteen 78).
constexpr int kThreads = 64, kMaxTokens = 8;
constexpr int kGatherThreads = 256, kGatherTokens = 4;

// Where a packed token lives: its position and the pool row block * block_size + offset.
struct Place {
  int pos, block, off, flag;  // block < 0: nothing there (no sequence, a skipped one, or `flag`)
};

// Looks up the packed tokens [token0, token0 + n), n <= 32, by the first warp, one per lane.  The
// number of sequences that end at or before token0 is its sequence (one load per lane and a
// sum for up to 32 sequences, instead of a chain of dependent loads); a later token's is found by
// stepping on from there.  cu null: token i is sequence i.  `owner`: the sequence or -1, or null.
__device__ __forceinline__ void find_places(int token0, int n, const int* cu, int B, const int* firsts,
                                            const int* tables, int max_blocks, int num_blocks, int block_size, int max_pos,
                                            int* err, Place* places, int* owner) {
  const int lane = threadIdx.x;
  if (lane >= 32) return;
  const int token = token0 + lane;
  int b = token;
  if (cu) {
    int ended = 0;
    for (int s = lane; s < B; s += 32) ended += cu[s + 1] <= token0;
    b = __reduce_add_sync(0xffffffffu, ended);
  }
  if (lane >= n) return;
  if (cu) {
    while (b < B && cu[b + 1] <= token) ++b;
    if (b >= B || token < cu[b]) b = -1;
  }
  Place w{0, -1, 0, 0};
  const int first = b < 0 ? -1 : firsts ? firsts[b] : 0;
  if (first >= 0) {
    const unsigned pos = (unsigned)first + (unsigned)(cu ? token - cu[b] : 0);  // below 2^32
    const unsigned blk = pos / (unsigned)block_size;
    if (blk >= (unsigned)max_blocks || pos >= (unsigned)max_pos) {
      w.flag = SPD_DEVERR_LENGTH;
    } else {
      const int id = tables[(long long)b * max_blocks + blk];
      if (id < 0 || id >= num_blocks) {
        w.flag = SPD_DEVERR_BLOCK_ID;
      } else {
        w.pos = (int)pos;
        w.block = id;
        w.off = (int)(pos - blk * (unsigned)block_size);
      }
    }
    if (w.flag) set_error(err, w.flag);
  }
  places[lane] = w;
  if (owner) owner[lane] = b;
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
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two values rounded to a 16-bit type, packed (one conversion).
template <typename T>
__device__ __forceinline__ uint32_t round2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Eight elements as loaded, and as fp32.
template <typename T> struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void floats(float (&y)[8]) const {
    const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = Elem<T>::to_f(e[i]);
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&y)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(y[0], y[1], y[2], y[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else {
    *reinterpret_cast<uint4*>(dst) = make_uint4(round2<T>(y[0], y[1]), round2<T>(y[2], y[3]), round2<T>(y[4], y[5]),
                                                round2<T>(y[6], y[7]));
  }
}

// Sixteen elements; of a 16-bit type with one 32-byte store where `wide` (dst 32-byte aligned).
template <typename T>
__device__ __forceinline__ void store16(T* dst, const float (&y)[16], bool wide) {
  if constexpr (sizeof(T) == 2) {
    if (!wide) {
#pragma unroll
      for (int i = 0; i < 16; i += 8)
        *reinterpret_cast<uint4*>(dst + i) = make_uint4(round2<T>(y[i], y[i + 1]), round2<T>(y[i + 2], y[i + 3]),
                                                        round2<T>(y[i + 4], y[i + 5]), round2<T>(y[i + 6], y[i + 7]));
      return;
    }
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(round2<T>(y[0], y[1])),
                 "r"(round2<T>(y[2], y[3])), "r"(round2<T>(y[4], y[5])), "r"(round2<T>(y[6], y[7])),
                 "r"(round2<T>(y[8], y[9])), "r"(round2<T>(y[10], y[11])), "r"(round2<T>(y[12], y[13])),
                 "r"(round2<T>(y[14], y[15]))
                 : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<float4*>(dst)[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
  }
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

// Eight values of one 64-value group to a word of codes, rint((y - z) / s) clamped to 0..15 each.
// One multiply-add per value gives v = 2^16 ((y - z) / s + 1/2) + 2 as a whole number in the low bits of
// 2^23 + v: byte 2 is the code, the low half says how far it is from the next one.  It is within 1.2
// of the quotient's own (three roundings of at most 1/2, 1/2 and 0.2 while |z| < 64 s), so a code may
// be another one only where the low half is at most 4: one value in 13,000, whose word is then made
// by division.  So is a word where s or z is saturated or s subnormal, or |z| >= 64 s: elsewhere the
// parameters' own rounding moves no quotient out of 0..15.
__device__ __forceinline__ uint32_t encode8(const float (&y)[8], float s, float z) {
  if (!(s > 0.f)) return 0u;
  const float inv = __frcp_rn(s), a = inv * 65536.f, c = fmaf(-z, a, 8388608.f + 32768.f + 2.f);
  uint32_t u[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = __float_as_uint(fmaf(y[k], a, c));
  auto least = [](uint32_t p, uint32_t q) {
    uint32_t r;
    asm("min.u16x2 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(q));
    return r;
  };
  auto lows = [&](int k) { return __byte_perm(u[k], u[k + 1], 0x5410); };
  const uint32_t low = least(least(lows(0), lows(2)), least(lows(4), lows(6)));
  auto codes = [&](int k) {  // of values k, k + 2, k + 4, k + 6
    return __byte_perm(__byte_perm(u[k], u[k + 2], 0x0062), __byte_perm(u[k + 4], u[k + 6], 0x0062), 0x5410);
  };
  uint32_t word = (codes(0) & 0x0F0F0F0Fu) | (codes(1) & 0x0F0F0F0Fu) << 4;
  const bool sure = s >= 6.103515625e-5f && s < 65504.f && fabsf(z) < 65504.f && fabsf(z * inv) < 64.f;
  if (!sure || min(low & 0xFFFFu, low >> 16) <= 4u) {
    word = 0;
#pragma unroll 1
    for (int k = 7; k >= 0; --k) {
      float v = y[0];
#pragma unroll
      for (int i = 1; i < 8; ++i)
        if (i == k) v = y[i];
      word = word * 16u + (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(v, z), s)), 0.f), 15.f);
    }
  }
  return word;
}

// A CTA owns `tokens` packed tokens and `rpc` of their head rows (q heads, then k, then v).  A thread
// owns the same unit of 16 dimensions of one row for all of the tokens: the two chunks of eight
// that rotate into each other (d, d + rot / 2, or 16 neighbours when interleaved or not rotated),
// so every value is loaded once, shares its eight angles, and all that depends on the row is worked
// out once.  The next tokens' values are loaded while one is worked on.
template <typename T, bool INT4>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 16 : INT4 ? 10 : 12)
    rope_append_kernel(const RopeAppendParams p, int tokens, int rpc) {
  __shared__ Place place[kMaxTokens];
  const int token0 = blockIdx.x * tokens, n = min(tokens, p.N - token0);
  const int upr = (p.D + 15) / 16;  // units per head row
  const int hq = p.q ? p.Hq : 0, rows = hq + 2 * p.Hkv;
  const int local = threadIdx.x / upr, u = threadIdx.x - local * upr, row = blockIdx.y * rpc + local;
  const bool live = local < rpc && row < rows;  // the same for all units of a row
  const bool is_q = row < hq, is_k = !is_q && row < hq + p.Hkv, is_v = !is_q && !is_k;
  const int h = is_q ? row : is_k ? row - hq : row - hq - p.Hkv;
  const int r = p.rot / 2;
  const bool turns = u < p.rot / 16 && !is_v, split = turns && !p.interleaved;
  const int d0 = split ? 8 * u : 16 * u, d1 = split ? 8 * u + r : 16 * u + 8;
  const bool second = INT4 || d1 < p.D;
  const long long st = is_q ? p.q_st : is_k ? p.k_st : p.v_st;
  const T* src = reinterpret_cast<const T*>(is_q ? p.q : is_k ? p.k : p.v) + token0 * st +
                 h * (is_q ? p.q_sh : is_k ? p.k_sh : p.v_sh);
  T* dst = reinterpret_cast<T*>(is_q ? p.q_out : is_k ? p.k_pool : p.v_pool) + (long long)h * p.D;
  const long long q_step = (long long)p.Hq * p.D;
  // planes of 64 dimensions share a scale: does every thread of this warp hold 16 dimensions of the
  // plane of its own four neighbours?  (Not where a rotation over more than 64 dimensions pairs planes.)
  const int planes = p.D / int4::kPlane;
  const bool one_plane =
      INT4 && __all_sync(0xffffffffu, !live || is_q || (d0 / int4::kPlane == u / 4 && d1 / int4::kPlane == u / 4));
  const float *cs = p.cos + 8 * u, *sn = p.sin + 8 * u;
  // tokens loaded ahead (of 16 bits one: 94 us against 91 for the 16 prompts above; into 4 bits two: 63 us
  // against 59, for want of registers)
  constexpr int kAhead = sizeof(T) == 2 && !INT4 ? 2 : 1;
  Raw8<T> lo_raw[kAhead], hi_raw[kAhead];
  auto load = [&](int t, int slot) {
    if (live && t < n) {
      lo_raw[slot].load(src + t * st + d0);
      if (second) hi_raw[slot].load(src + t * st + d1);
    }
  };
#pragma unroll
  for (int a = 0; a < kAhead; ++a) load(a, a);
  find_places(token0, n, p.cu_seqlens, p.B, p.positions, p.block_tables, p.max_blocks, p.num_blocks, p.block_size,
              p.max_pos, p.err, place, nullptr);
  __syncthreads();
  auto work = [&](int t, int slot) {
    const Place w = place[t];
    float lo[8] = {}, hi[8] = {};
    if (live && w.block >= 0) {
      lo_raw[slot].floats(lo);
      if (second) hi_raw[slot].floats(hi);
    }
    load(t + kAhead, slot);
    if (live && turns && w.block >= 0) {
      float cc[8], ss[8];
      const long long at = (long long)w.pos * r;
      load_to_float<float, 8>(cs + at, cc);
      load_to_float<float, 8>(sn + at, ss);
      turn(lo, hi, cc, ss, p.interleaved);
    }
    if (live && (is_q || (!INT4 && w.block >= 0))) {  // of q also the zeros of a token that is not written
      T* o = dst + (is_q ? (token0 + t) * q_step : ((long long)w.block * p.block_size + w.off) * p.Hkv * p.D);
      store8(o + d0, lo);
      if (second) store8(o + d1, hi);
    }
    if constexpr (INT4) {
      if (__any_sync(0xffffffffu, live && !is_q && w.block >= 0)) {
        float mn0 = min_nan(lo[0], lo[1]), mx0 = max_nan(lo[0], lo[1]), mn1 = min_nan(hi[0], hi[1]), mx1 = max_nan(hi[0], hi[1]);
#pragma unroll
        for (int k = 2; k < 8; k += 2) {
          mn0 = min_nan(mn0, lo[k], lo[k + 1]);
          mx0 = max_nan(mx0, lo[k], lo[k + 1]);
          mn1 = min_nan(mn1, hi[k], hi[k + 1]);
          mx1 = max_nan(mx1, hi[k], hi[k + 1]);
        }
        const bool writes = live && !is_q && w.block >= 0;
        const int half = int4::half_bytes(planes, p.block_size);
        unsigned char* page = reinterpret_cast<unsigned char*>(p.k_pool) + ((long long)w.block * p.Hkv + h) * (2 * half) +
                              (is_k ? 0 : half);
        // scale and zero of a group from its least and largest value; the rounded ones in s and z
        auto parameters = [](float mn, float mx, float& s, float& z) {
          constexpr float kMax = 65504.f;
          s = __fdiv_rn(__fsub_rn(mx, mn), 15.f);
          s = s > kMax ? kMax : s;  // a NaN stays
          z = mn > kMax ? kMax : mn < -kMax ? -kMax : mn;
          const __half2 h = __halves2half2(__float2half_rn(s), __float2half_rn(z));
          s = __low2float(h);
          z = __high2float(h);
          return h;
        };
        auto put = [&](const float (&y)[8], int d, __half2 sz, float s, float z) {
          const int slot = (d / int4::kPlane) * p.block_size + w.off, in = d % int4::kPlane;
          *reinterpret_cast<uint32_t*>(page + slot * int4::kRowBytes + in / 2) = encode8(y, s, z);
          if (in == 0)
            *reinterpret_cast<__half2*>(page + planes * p.block_size * int4::kRowBytes + slot * int4::kParamBytes) = sz;
        };
        float s, z;
        if (one_plane) {
          float mn = min_nan(mn0, mn1), mx = max_nan(mx0, mx1);
#pragma unroll
          for (int o = 1; o < 4; o <<= 1) {
            mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
            mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          }
          if (writes) {
            const __half2 sz = parameters(mn, mx, s, z);
            put(lo, d0, sz, s, z);
            put(hi, d1, sz, s, z);
          }
        } else {
          const int pl0 = d0 / int4::kPlane, pl1 = d1 / int4::kPlane;
          float a0 = 0.f, b0 = 0.f, a1 = 0.f, b1 = 0.f;  // (least, largest) of each chunk's plane
          for (int pl = 0; pl < planes; pl += 2) {        // two planes' exchanges beside each other
            float mn[2], mx[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              mn[i] = pl0 == pl + i ? mn0 : INFINITY;
              mx[i] = pl0 == pl + i ? mx0 : -INFINITY;
              if (pl1 == pl + i) mn[i] = min_nan(mn[i], mn1), mx[i] = max_nan(mx[i], mx1);
            }
            for (int o = 1; o < upr; o <<= 1)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                mn[i] = min_nan(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
                mx[i] = max_nan(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
              }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (pl0 == pl + i) a0 = mn[i], b0 = mx[i];
              if (pl1 == pl + i) a1 = mn[i], b1 = mx[i];
            }
          }
          if (writes) {
            __half2 sz = parameters(a0, b0, s, z);
            put(lo, d0, sz, s, z);
            sz = parameters(a1, b1, s, z);
            put(hi, d1, sz, s, z);
          }
        }
      }
    }
  };
#pragma unroll 1
  for (int t0 = 0; t0 < n; t0 += kAhead)
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (t0 + a < n) work(t0 + a, a);
}

// Tokens of the 4-bit pool back as packed k and v.  A CTA owns `tokens` tokens and `rpc` of their K and
// V head rows; a thread owns the same 32 dimensions of one row for all of them: 16 bytes of codes and
// their parameters in, 64 bytes of a 16-bit type out, U tokens in flight.  A masked code is an fp16
// subnormal (c * 2^-24, or 16c * 2^-24), so its conversion is exact and the powers of two go into
// the scale: c * scale + zero is one fp32 multiply-add whatever way c came.
template <typename T>
__global__ void __launch_bounds__(kGatherThreads) gather_int4_kernel(const GatherInt4Params p, int tokens, int rpc) {
  __shared__ Place place[kGatherTokens];
  __shared__ int owner[kGatherTokens];
  const int token0 = blockIdx.x * tokens, n = min(tokens, p.N - token0);
  find_places(token0, n, p.cu_seqlens, p.B, p.starts, p.block_tables, p.max_blocks, p.num_blocks, p.block_size,
              0x7fffffff, p.err, place, owner);
  const int upr = p.D / 32, planes = p.D / int4::kPlane, half = int4::half_bytes(planes, p.block_size);
  const int local = threadIdx.x / upr, u = threadIdx.x - local * upr, row = blockIdx.y * rpc + local;
  const bool is_k = row < p.Hkv;
  const int h = is_k ? row : row - p.Hkv;
  const unsigned char* src = p.pool + (long long)h * (2 * half) + (is_k ? 0 : half);
  const long long block_bytes = (long long)p.Hkv * (2 * half), step = (long long)p.Hkv * p.D;
  const int code_at = (u / 2) * p.block_size * int4::kRowBytes + (u & 1) * 16;
  const int param_at = planes * p.block_size * int4::kRowBytes + (u / 2) * p.block_size * int4::kParamBytes;
  T* dst = reinterpret_cast<T*>(is_k ? p.k_out : p.v_out) + token0 * step + (long long)h * p.D + 32 * u;
  const bool wide = (reinterpret_cast<uintptr_t>(dst) & 31) == 0;  // rows are multiples of 64 bytes
  __syncthreads();
  if (local >= rpc || row >= 2 * p.Hkv) return;
  constexpr int U = 2;
#pragma unroll 1
  for (int t0 = 0; t0 < n; t0 += U) {
    uint4 code[U];
    uint32_t param[U];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      code[q] = make_uint4(0, 0, 0, 0);
      param[q] = 0;  // zeros for a token that is not there
      if (t0 + q < n && place[t0 + q].block >= 0) {
        const Place w = place[t0 + q];
        const unsigned char* page = src + w.block * block_bytes;
        code[q] = __ldg(reinterpret_cast<const uint4*>(page + code_at + w.off * int4::kRowBytes));
        param[q] = __ldg(reinterpret_cast<const unsigned int*>(page + param_at + w.off * int4::kParamBytes));
      }
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (t0 + q >= n || owner[t0 + q] < 0) continue;  // past the end, or a row of no sequence
      const float2 sz = __half22float2(*reinterpret_cast<const __half2*>(&param[q]));
      const float s1 = sz.x * 16777216.f, s16 = sz.x * 1048576.f;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        float y[16];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t x = v ? (w ? code[q].w : code[q].z) : (w ? code[q].y : code[q].x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // dimensions i and i + 4 of the word's eight
            const uint32_t pair = (i < 2 ? x : x >> 8) & (i & 1 ? 0x00F000F0u : 0x000F000Fu);
            const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&pair));
            y[8 * w + i] = fmaf(c.x, i & 1 ? s16 : s1, sz.y);
            y[8 * w + 4 + i] = fmaf(c.y, i & 1 ? s16 : s1, sz.y);
          }
        }
        store16(dst + (t0 + q) * step + 16 * v, y, wide);
      }
    }
  }
}

}  // namespace rope

// Tokens per CTA: one while there are fewer tokens than 16 per SM, so that a step's few tokens
// spread over the SMs, up to `most`, so that the look-up of a token's place is shared.
static int tokens_per_cta(int N, int most, int sms) {
  const int t = N / (sms * 16);
  return t < 1 ? 1 : t > most ? most : t;
}

// Rows per CTA: as even a split of all rows as fits its threads, of `upr` units a row.
static int rows_per_cta(int rows, int upr, int threads) {
  const int most = threads / upr, parts = (rows + most - 1) / most;
  return (rows + parts - 1) / parts;
}

int rope_append_launch(const RopeAppendParams& p, int dtype, bool int4_pool, int sms, cudaStream_t st) {
  using namespace rope;
  const int tokens = tokens_per_cta(p.N, kMaxTokens, sms), upr = (p.D + 15) / 16, rows = (p.q ? p.Hq : 0) + 2 * p.Hkv;
  const int rpc = rows_per_cta(rows, upr, kThreads);
  const dim3 grid((unsigned)((p.N + tokens - 1) / tokens), (unsigned)((rows + rpc - 1) / rpc));
  const dim3 block((unsigned)((rpc * upr + 31) / 32 * 32));
  auto run = [&](auto tag) {
    using T = decltype(tag);
    if (int4_pool) rope_append_kernel<T, true><<<grid, block, 0, st>>>(p, tokens, rpc);
    else rope_append_kernel<T, false><<<grid, block, 0, st>>>(p, tokens, rpc);
  };
  if (dtype == SPD_F32) run(float{});
  else if (dtype == SPD_F16) run(__half{});
  else run(__nv_bfloat16{});
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

int gather_int4_launch(const GatherInt4Params& p, int dtype, int sms, cudaStream_t st) {
  using namespace rope;
  const int tokens = tokens_per_cta(p.N, kGatherTokens, sms), upr = p.D / 32, rpc = rows_per_cta(2 * p.Hkv, upr, kGatherThreads);
  const dim3 grid((unsigned)((p.N + tokens - 1) / tokens), (unsigned)((2 * p.Hkv + rpc - 1) / rpc));
  const dim3 block((unsigned)((rpc * upr + 31) / 32 * 32));
  if (dtype == SPD_F32) gather_int4_kernel<float><<<grid, block, 0, st>>>(p, tokens, rpc);
  else if (dtype == SPD_F16) gather_int4_kernel<__half><<<grid, block, 0, st>>>(p, tokens, rpc);
  else gather_int4_kernel<__nv_bfloat16><<<grid, block, 0, st>>>(p, tokens, rpc);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace spd
