// paged_decode_attn_int4.cu — single-token attention over the paged 4-bit K/V pool of
// spd_int4.cuh, with grouped heads (Hq = G * Hkv query heads):
//   out[b, h] = softmax_t(q[b, h] . k[t, h / G] * scale) . v[t, h / G],  t < context_lens[b]
// with k and v the values code * scale_t + zero_t of the pool.
//
// What bounds it: each cached token is read once (72 bytes per 64 dimensions, K and V
// together) for 4 * G * 64 operations, so HBM does, if the 4-bit codes reach the multipliers
// in few instructions.  They do so here without a conversion:
// * A code masked in place is an fp16 subnormal: bits 0..3 of a half are c * 2^-24, bits
//   4..7 are 16c * 2^-24.  The tensor core multiplies subnormals exactly, so a 32-bit word
//   of 8 codes becomes four fp16 pairs with one shift and four ANDs, and the powers of two
//   are taken out again in fp32 (and the 16 in the query's fragment or the output).
// * scores:  q . k = scale_t * (q . c) + zero_t * sum(q) per plane of 64 dimensions;
//   output:  sum_t p_t v_t = sum_t (p_t * scale_t) c_t + sum_t p_t * zero_t.
//   So scale and zero cost a few operations per token, not per value.
// * mma.sync m16n8k16 with tokens (scores) or head dimensions (output) as its 16 rows and
//   the group's query heads as its 8 columns: the products are a small part of the time at
//   single-token shapes, and tcgen05 (128 rows, operands through shared memory) would have
//   to write the unpacked codes back to shared memory first.
// * fp16 holds the query scaled by a power of two to below 2^11, and the weights p * scale_t
//   scaled by a running power of two to below 2^15: neither overflows, and the last bit of
//   what falls below fp16's normal numbers is 2^-30 of a weight of 1 at the largest value scale
//   met so far.  With up to four heads per tile (and for fp32 queries)
//   each head takes two columns, the value and its rounding remainder, so q and p keep 22
//   bits; with more, q keeps 11 bits (exact for fp16 and bf16 queries) and p 11.
//
// Work split: one CTA per (sequence, key/value head tile, chunk of tokens).  A CTA's four warps take
// every fourth step of 64 tokens, each fed by its own ring of shared-memory stages (one bulk copy per
// page, issued by the lanes in parallel, no CTA-wide barrier in the loop), with a running maximum that
// is raised only when a score passes it by 8 (p <= 2^8).  The warps are joined in shared memory, the
// chunks of a (sequence, head tile) by the last CTA to arrive, which adds them in their order: the
// result does not depend on who that is.
// Measured in replayed graphs: 32 contexts of 1,000 to 32,000 tokens, 32/8 heads of 128, bf16 (582 MB of
// pool): 129 us, 4.5 TB/s, 0.69 of a plain copy's rate (a lone call 140); copies alone took 108 us, the
// arithmetic alone 125.  No pipe and no issue slots are full (48 % of either): at three warps a scheduler,
// which is what registers allow, the arithmetic waits for its own fixed latencies and its loads.
// 128 contexts of up to 3,900, 12 heads of 64: 66 us; one of 32,000: 17.5 us; one of 448: 5.1 us, most
// of it the latency of table, page and join.  (Comparisons below are of the forms of their time, before
// pages could be left out.)
#include "spd_int4.cuh"
#include "spd_params.cuh"

#include <algorithm>

namespace spd {
namespace dec4 {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kLazy = 8.f;  // log2 units a score may pass the reference maximum by

// Tokens per warp step, stages per warp and CTAs per SM: as many warps as their registers allow.  At
// D = 128 12 warps an SM, each with two stages of 9,216 bytes (8 warps with three: 139 us for the 32
// contexts above in place of 126); at D = 64 16 warps (12: 70 us for the 128 contexts, 66 with 16).
template <int P> constexpr int step_tokens() { return P == 4 ? 32 : 64; }
template <int P> constexpr int stages() { return P == 1 ? 3 : 2; }
template <int P> constexpr int ctas_per_sm() { return P == 1 ? 4 : P == 2 ? 3 : 2; }
template <int P> constexpr int step_bytes() { return int4::page_bytes(P, step_tokens<P>()); }
template <int P> constexpr int ring_bytes() { return kWarps * stages<P>() * step_bytes<P>(); }

// D += A * B (m16n8k16, fp16 in, fp32 accumulation).  Not volatile: the compiler may interleave the
// chains of different accumulators, which hides each product's latency.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (round(x), round(x - round(x)))
__device__ __forceinline__ uint32_t pack_split(float x) {
  const float hi = __half2float(__float2half_rn(x));
  return pack_half(hi, x - hi);
}
__device__ __forceinline__ float2 unpack_half(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// P consecutive (scale, zero) pairs of one token
template <int P>
__device__ __forceinline__ void load_par(const float2* at, float2 (&v)[P]) {
  if constexpr (P == 1) {
    v[0] = *at;
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      const float4 x = *reinterpret_cast<const float4*>(at + i);
      v[i] = make_float2(x.x, x.y);
      v[i + 1] = make_float2(x.z, x.w);
    }
  }
}

// 16 consecutive query elements as fp32
__device__ __forceinline__ void load_q16(const void* q, int dtype, long long at, float* o) {
  if (dtype == SPD_F32) load_to_float<float, 16>(reinterpret_cast<const float*>(q) + at, o);
  else if (dtype == SPD_F16) load_to_float<__half, 16>(reinterpret_cast<const __half*>(q) + at, o);
  else load_to_float<__nv_bfloat16, 16>(reinterpret_cast<const __nv_bfloat16*>(q) + at, o);
}
__device__ __forceinline__ void store_out4(void* out, int dtype, long long at, float4 v) {
  if (dtype == SPD_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = v;
  } else if (dtype == SPD_F16) {
    alignas(8) __half o[4] = {__float2half_rn(v.x), __float2half_rn(v.y), __float2half_rn(v.z), __float2half_rn(v.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(out) + at) = *reinterpret_cast<const uint2*>(o);
  } else {
    alignas(8) __nv_bfloat16 o[4] = {__float2bfloat16_rn(v.x), __float2bfloat16_rn(v.y), __float2bfloat16_rn(v.z),
                                     __float2bfloat16_rn(v.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(out) + at) = *reinterpret_cast<const uint2*>(o);
  }
}

// P: planes (D / 64); BS: block size; SPLIT: two columns per head.
template <int P, int BS, bool SPLIT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<P>()) decode_int4_kernel(const DecodeInt4Params p) {
  constexpr int D = P * int4::kPlane;
  constexpr int kHeads = SPLIT ? 4 : 8;  // heads per column tile
  constexpr int kStages = stages<P>(), kStep = step_tokens<P>(), kSubs = kStep / 16;
  constexpr int kPage = int4::page_bytes(P, BS), kHalf = int4::half_bytes(P, BS);
  constexpr int kPages = kStep / BS;
  constexpr int kParams = P * BS * int4::kRowBytes;  // offset of the parameters in a half page
  constexpr int kRow = D + 4;  // floats per partial row: D values, m, l, two unused
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ float stat_m[kWarps][8], stat_l[kWarps][8];
  __shared__ uint32_t missing[kWarps][kStages];  // pages of a stage whose tokens are left out, a bit each
  __shared__ int last_flag;
  __shared__ float* joined[kWarps];  // where each warp left its result, [heads][D]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = p.Hq / p.Hkv;
  const int tiles = (G + kHeads - 1) / kHeads, Y = p.Hkv * tiles;

  // all heads of a sequence's chunk together: their pages lie side by side
  const int y = (int)(blockIdx.x % (unsigned)Y), rest = (int)(blockIdx.x / (unsigned)Y);
  const int chunk = rest % p.chunks, b = rest / p.chunks;
  const int tile = y % tiles, kvh = y / tiles;
  const int heads = min(kHeads, G - tile * kHeads);  // of this tile
  const long long head0 = (long long)b * p.Hq + kvh * G + tile * kHeads;  // row of q and out
  int ctx = p.context_lens[b];
  if ((long long)ctx > (long long)p.max_blocks * BS) {
    if (tid == 0) set_error(p.err, SPD_DEVERR_LENGTH);
    ctx = p.max_blocks * BS;
  }
  if (ctx <= 0) {
    if (chunk == 0)
#pragma unroll 1
      for (int i = tid; i < heads * D / 4; i += kThreads)
        store_out4(p.out, p.dtype, head0 * D + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  // the sequence's own chunks: as many as there are CTAs for it, but of `least` tokens or more
  // (unsigned: contexts reach 2^31 - 1)
  const int size = max(p.least, (int)((((unsigned)ctx + p.chunks - 1) / p.chunks + kStep - 1) / kStep * kStep));
  const long long first = (long long)chunk * size;
  if (first >= ctx) return;
  const int t0 = (int)first;
  const int t1 = ctx - t0 > size ? t0 + size : ctx;
  const int parts = (ctx - 1) / size + 1;
  const int steps = (t1 - t0 + kStep - 1) / kStep;
  const int* table = p.block_tables + (long long)b * p.max_blocks;

  unsigned char* ring = smem + (size_t)warp * kStages * step_bytes<P>();
  const uint64_t policy = l2_policy_evict_first();
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[warp][s], 1), missing[warp][s] = 0;
    fence_barrier_init();
  }
  __syncwarp();

  // Copies run ahead of the arithmetic: `id` is this lane's page of the step `ahead` that is fetched next
  // (its table entry is loaded one step early).  Block 0 is fetched in place of an id out of range, and
  // the page's bit in `missing` keeps its tokens out: a load and two branches a step, 1.3 % of the 32
  // contexts' time and nothing of the one's (a vote a step and a flag: 1.9 %; with both loops' conditions
  // in one: 0.7 %, but 4 % of the one's).
  const unsigned char* pool_h = p.pool + (long long)kvh * kPage;
  const long long block_stride = (long long)p.Hkv * kPage;
  int ahead = warp, id = 0, pages = 0, fetched = 0;
  auto look_up = [&]() {
    if (ahead >= steps) return;
    const int tok = t0 + ahead * kStep;
    pages = min(kPages, (t1 - tok + BS - 1) / BS);
    id = lane < pages ? __ldg(table + tok / BS + lane) : 0;
  };
  auto fetch = [&]() {
    if (ahead >= steps) return;
    const int st = fetched % kStages;
    if (lane == 0) mbar_arrive_expect_tx(&bars[warp][st], (uint32_t)(pages * kPage));
    __syncwarp();
    if (lane < pages) {
      if (id < 0 || id >= p.num_blocks) {
        set_error(p.err, SPD_DEVERR_BLOCK_ID);
        atomicOr(&missing[warp][st], 1u << lane);
        id = 0;
      }
      bulk_copy_g2s_hint(ring + (size_t)st * step_bytes<P>() + lane * kPage, pool_h + id * block_stride, kPage,
                         &bars[warp][st], policy);
    }
    ++fetched;
    ahead += kWarps;
    look_up();
  };
  look_up();
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) fetch();
  __syncwarp();  // marks of this warp's lanes in `missing`

  // Row r of an 8-token group holds token r ^ (r >> 2): with it both the rows that a
  // half-warp reads for the scores (r = 0..3, 4..7) and those that a warp reads for the output
  // (even or odd r) fall on four different quarters of the 32 banks.
  const int tok_k = g ^ (g >> 2);
  const int tok_v0 = (2 * t) ^ (t >> 1), tok_v1 = (2 * t + 1) ^ (t >> 1);
  auto place = [](int tok) { return (tok / BS) * kPage + (tok % BS) * int4::kRowBytes; };

  constexpr int C = SPLIT ? 1 : 2;  // heads of this lane's two columns
  static_assert(kHeads * D * 4 <= step_bytes<P>(), "a segment's result fits in a stage");
  int used = 0;
  bool fine = true;

  // ---- the query fragments: column g, k = this lane's 16 dimensions of each plane --------
  uint32_t qb[P][4][2];
  float f, qsa[P], qsb[P];  // score factor, and sums of q of this lane's columns 2t, 2t + 1
  {
    const int hq = SPLIT ? g >> 1 : g;
    float qv[P][16];
    float amax = 0.f, qs[P];
#pragma unroll
    for (int pl = 0; pl < P; ++pl) {
      if (hq < heads) load_q16(p.q, p.dtype, (head0 + hq) * D + pl * 64 + 16 * t, qv[pl]);
      else
#pragma unroll
        for (int i = 0; i < 16; ++i) qv[pl][i] = 0.f;
      qs[pl] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a = fabsf(qv[pl][i]);
        amax = fmaxf(amax, a < INFINITY ? a : 0.f);
        qs[pl] += qv[pl][i];
      }
      qs[pl] += __shfl_xor_sync(0xffffffffu, qs[pl], 1);
      qs[pl] += __shfl_xor_sync(0xffffffffu, qs[pl], 2);
      qs[pl] *= p.scale_log2;
    }
    amax = warp_max(amax);  // of the tile's finite queries
    // |q| * 2^k < 2^11; k is limited so that both 2^k and 2^(24 - k) are normal numbers
    const int k = amax > 0.f ? max(-100, min(100, 10 - ((__float_as_int(amax) >> 23) - 127))) : 0;
    const float up = pow2(k);
#pragma unroll
    for (int pl = 0; pl < P; ++pl)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int base = 8 * (s >> 1) + 2 * (s & 1);
        float x[4] = {qv[pl][base] * up, qv[pl][base + 4] * up, qv[pl][base + 1] * up, qv[pl][base + 5] * up};
        if (SPLIT) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float hi = __half2float(__float2half_rn(x[i]));
            x[i] = (g & 1) ? x[i] - hi : hi;
          }
        }
        qb[pl][s][0] = pack_half(x[0], x[1]);
        qb[pl][s][1] = pack_half(x[2] * 0.0625f, x[3] * 0.0625f);  // meets codes that read as 16c
      }
    f = pow2(24 - k) * p.scale_log2;
#pragma unroll
    for (int pl = 0; pl < P; ++pl) {
      qsa[pl] = __shfl_sync(0xffffffffu, qs[pl], 8 * t);
      qsb[pl] = __shfl_sync(0xffffffffu, qs[pl], 8 * t + 4);
    }
  }

  float o[P][4][4], zacc[P][C], l[C], m[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    l[c] = 0.f;
    m[c] = -INFINITY;
#pragma unroll
    for (int pl = 0; pl < P; ++pl) zacc[pl][c] = 0.f;
  }
#pragma unroll
  for (int pl = 0; pl < P; ++pl)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[pl][i >> 2][i & 3] = 0.f;
  int lift = -15;  // exponent of the largest value scale seen; weights carry 2^(6 - lift)

#pragma unroll 1
  for (int i = warp; i < steps && fine; i += kWarps) {
    const int st = used % kStages;
    const bool ok = mbar_wait_suspend(&bars[warp][st], (uint32_t)((used / kStages) & 1), p.err, p.wait_ns);
    fine = __all_sync(0xffffffffu, ok);
    if (!fine) break;
    ++used;
    unsigned char* buf = ring + (size_t)st * step_bytes<P>();
    const int left = t1 - (t0 + i * kStep);  // valid tokens of this step (>= 1)
    const uint32_t gone = missing[warp][st];
    auto hole = [&](int tok) { return (gone >> (tok / BS) & 1u) != 0; };

    // ---- the values' parameters, lane = token: zero past the end; the largest scale -----------
    uint32_t raw[kStep / 32][P], top = 0;
#pragma unroll
    for (int h = 0; h < kStep / 32; ++h) {
      const int tok = h * 32 + lane;
      const unsigned char* at = buf + kHalf + (tok / BS) * kPage + kParams + (tok % BS) * int4::kParamBytes;
#pragma unroll
      for (int pl = 0; pl < P; ++pl) {
        raw[h][pl] = tok < left ? *reinterpret_cast<const uint32_t*>(at + pl * BS * int4::kParamBytes) : 0u;
        top = max(top, raw[h][pl] & 0x7FFFu);
      }
    }
    if (gone) {
      top = 0;
#pragma unroll
      for (int h = 0; h < kStep / 32; ++h)
#pragma unroll
        for (int pl = 0; pl < P; ++pl) {
          if (hole(h * 32 + lane)) raw[h][pl] = 0u;
          top = max(top, raw[h][pl] & 0x7FFFu);
        }
    }
    if (__any_sync(0xffffffffu, (int)(top >> 10) - 15 > lift)) {  // a larger value scale than any before
      const int up = min(15, (int)(__reduce_max_sync(0xffffffffu, top) >> 10) - 15);
      const float w = pow2(lift - up);
      lift = up;
#pragma unroll
      for (int pl = 0; pl < P; ++pl)
#pragma unroll
        for (int k = 0; k < 16; ++k) o[pl][k >> 2][k & 3] *= w;
    }
    const float wscale = pow2(6 - lift);

    // ---- scores ----------------------------------------------------------------------
    // products of all 16-token tiles and planes first, their accumulator chains interleaved
    float acc[kSubs][P][4];
    {
      uint2 wa[kSubs][P], wb[kSubs][P];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
        for (int pl = 0; pl < P; ++pl) {
          const unsigned char* at = buf + pl * BS * int4::kRowBytes + 8 * t;
          wa[sub][pl] = *reinterpret_cast<const uint2*>(at + place(sub * 16 + tok_k));
          wb[sub][pl] = *reinterpret_cast<const uint2*>(at + place(sub * 16 + 8 + tok_k));
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[sub][pl][i] = 0.f;
        }
      // The key codes are in registers: over them go the values' parameters as fp32, (scale *
      // 2^(6 - lift), zero) of P planes per token.
      __syncwarp();
#pragma unroll
      for (int h = 0; h < kStep / 32; ++h) {
        const int tok = h * 32 + lane;
        float2* par = reinterpret_cast<float2*>(buf + (tok / BS) * kPage + (tok % BS) * (8 * P));
#pragma unroll
        for (int pl = 0; pl < P; ++pl) {
          const float2 v = unpack_half(raw[h][pl]);
          par[pl] = make_float2(v.x * wscale, v.y);
        }
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int pl = 0; pl < P; ++pl) {
            uint32_t xa = s < 2 ? wa[sub][pl].x : wa[sub][pl].y, xb = s < 2 ? wb[sub][pl].x : wb[sub][pl].y;
            if (s & 1) xa >>= 8, xb >>= 8;
            mma(acc[sub][pl], xa & 0x000F000Fu, xb & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x00F000F0u, qb[pl][s][0],
                qb[pl][s][1]);
          }
    }
    float sc[kSubs][2 * C];  // per 16 tokens: tokens tok_k and tok_k + 8 of each head
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      const int ta = sub * 16 + tok_k, tb = ta + 8;
#pragma unroll
      for (int pl = 0; pl < P; ++pl) {
        const float* a = acc[sub][pl];
        const unsigned char* at = buf + kParams + pl * BS * int4::kParamBytes;
        float2 ka = unpack_half(*reinterpret_cast<const uint32_t*>(at + (ta / BS) * kPage + (ta % BS) * int4::kParamBytes));
        float2 kb = unpack_half(*reinterpret_cast<const uint32_t*>(at + (tb / BS) * kPage + (tb % BS) * int4::kParamBytes));
        ka.x *= f;
        kb.x *= f;
        auto add = [&](int i, float x, float2 kp, float qs) {
          sc[sub][i] = fmaf(kp.x, x, pl ? fmaf(kp.y, qs, sc[sub][i]) : kp.y * qs);
        };
        if (SPLIT) {
          add(0, a[0] + a[1], ka, qsa[pl]);
          add(C, a[2] + a[3], kb, qsa[pl]);
        } else {
          add(0, a[0], ka, qsa[pl]);
          add(C - 1, a[1], ka, qsb[pl]);
          add(C, a[2], kb, qsa[pl]);
          add(2 * C - 1, a[3], kb, qsb[pl]);
        }
      }
      if (left < kStep)  // the sequence's last step
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (ta >= left) sc[sub][c] = -INFINITY;
          if (tb >= left) sc[sub][C + c] = -INFINITY;
        }
    }
    if (gone)
#pragma unroll
      for (int i = 0; i < 2 * kSubs; ++i)
        if (hole(i * 8 + tok_k))
#pragma unroll
          for (int c = 0; c < C; ++c) sc[i / 2][i % 2 * C + c] = -INFINITY;

    // ---- running maximum: raised when a score passes it by kLazy -----------------------------
    float mx[C];
    bool raise = false;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      mx[c] = fmaxf(sc[0][c], sc[0][C + c]);
#pragma unroll
      for (int sub = 1; sub < kSubs; ++sub) mx[c] = fmaxf(mx[c], fmaxf(sc[sub][c], sc[sub][C + c]));
      raise |= mx[c] > m[c] + kLazy;
    }
    if (__any_sync(0xffffffffu, raise)) {
      float fm[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], x));
        const float mn = fmaxf(m[c], mx[c]);
        fm[c] = m[c] == mn ? 1.f : ex2_approx(m[c] - mn);  // also when both are -inf
        m[c] = mn;
        l[c] *= fm[c];
#pragma unroll
        for (int pl = 0; pl < P; ++pl) zacc[pl][c] *= fm[c];
      }
#pragma unroll
      for (int pl = 0; pl < P; ++pl)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[pl][k][0] *= fm[0];
          o[pl][k][1] *= fm[C - 1];
          o[pl][k][2] *= fm[0];
          o[pl][k][3] *= fm[C - 1];
        }
    }
    float mm[C];  // a head whose scores are all -inf so far keeps m = -inf: its weights are 0
#pragma unroll
    for (int c = 0; c < C; ++c) mm[c] = m[c] == -INFINITY ? 0.f : m[c];

    // ---- output ------------------------------------------------------------------------
    __syncwarp();  // the values' parameters are written
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      const int ta = sub * 16 + tok_k, tb = ta + 8;
      float2 va[P], vb[P];
      load_par<P>(reinterpret_cast<const float2*>(buf + (ta / BS) * kPage + (ta % BS) * (8 * P)), va);
      load_par<P>(reinterpret_cast<const float2*>(buf + (tb / BS) * kPage + (tb % BS) * (8 * P)), vb);
      float pr[2 * C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        pr[c] = ex2_approx(sc[sub][c] - mm[c]);
        pr[C + c] = ex2_approx(sc[sub][C + c] - mm[c]);
        l[c] += pr[c] + pr[C + c];
      }
#pragma unroll
      for (int pl = 0; pl < P; ++pl) {
        uint32_t b0, b1;
        if (SPLIT) {
          b0 = movmatrix_trans(pack_split(pr[0] * va[pl].x));
          b1 = movmatrix_trans(pack_split(pr[1] * vb[pl].x));
          zacc[pl][0] += pr[0] * va[pl].y + pr[1] * vb[pl].y;
        } else {
          // what the rounding of a weight takes from the middle code (7.5) is put back, so that
          // its error meets codes of both signs, as an output's own rounding would
          const float unscale = 7.5f * pow2(lift - 6);
          const float w0 = pr[0] * va[pl].x, w1 = pr[C - 1] * va[pl].x, w2 = pr[C] * vb[pl].x, w3 = pr[2 * C - 1] * vb[pl].x;
          const uint32_t ha = pack_half(w0, w1), hb = pack_half(w2, w3);
          b0 = movmatrix_trans(ha);
          b1 = movmatrix_trans(hb);
          const float2 ra = unpack_half(ha), rb = unpack_half(hb);
          zacc[pl][0] += pr[0] * va[pl].y + pr[C] * vb[pl].y + unscale * ((w0 - ra.x) + (w2 - rb.x));
          zacc[pl][C - 1] += pr[C - 1] * va[pl].y + pr[2 * C - 1] * vb[pl].y + unscale * ((w1 - ra.y) + (w3 - rb.y));
        }
        const unsigned char* vb_ = buf + kHalf + pl * BS * int4::kRowBytes + 4 * g;
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + tok_v0));
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + tok_v1));
        const uint32_t w2 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + 8 + tok_v0));
        const uint32_t w3 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + 8 + tok_v1));
        // dimensions 8g..8g+3 (lo) and 8g+4..8g+7 (hi) of a pair of tokens per register
        uint32_t lo0 = __byte_perm(w0, w1, 0x5410), hi0 = __byte_perm(w0, w1, 0x7632);
        uint32_t lo1 = __byte_perm(w2, w3, 0x5410), hi1 = __byte_perm(w2, w3, 0x7632);
        mma(o[pl][0], lo0 & 0x000F000Fu, hi0 & 0x000F000Fu, lo1 & 0x000F000Fu, hi1 & 0x000F000Fu, b0, b1);
        mma(o[pl][1], lo0 & 0x00F000F0u, hi0 & 0x00F000F0u, lo1 & 0x00F000F0u, hi1 & 0x00F000F0u, b0, b1);
        lo0 >>= 8; hi0 >>= 8; lo1 >>= 8; hi1 >>= 8;
        mma(o[pl][2], lo0 & 0x000F000Fu, hi0 & 0x000F000Fu, lo1 & 0x000F000Fu, hi1 & 0x000F000Fu, b0, b1);
        mma(o[pl][3], lo0 & 0x00F000F0u, hi0 & 0x00F000F0u, lo1 & 0x00F000F0u, hi1 & 0x00F000F0u, b0, b1);
      }
    }
    // every lane has read this stage; what it wrote there comes before the next copy into it
    fence_proxy_async_smem();
    if (gone && lane == 0) missing[warp][st] = 0;
    __syncwarp();
    fetch();
  }
  // a wait that gave up: let this warp's copies in flight land
#pragma unroll 1
  for (; used < fetched; ++used)
    (void)mbar_wait_suspend(&bars[warp][used % kStages], (uint32_t)((used / kStages) & 1), nullptr);

  // ---- join the warps ---------------------------------------------------------------------
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
#pragma unroll
      for (int pl = 0; pl < P; ++pl) zacc[pl][c] += __shfl_xor_sync(0xffffffffu, zacc[pl][c], x);
    }
  const bool had_step = warp < steps;
  float* mine = reinterpret_cast<float*>(ring);  // the ring is drained
  if (lane == 0) joined[warp] = mine;
  if (had_step) {
    // out of the fp16 scaling: 2^24 / 2^(6 - lift), and / 16 where the codes read as 16c
    const float f1 = pow2(18 + lift), f16 = pow2(14 + lift);
#pragma unroll
    for (int pl = 0; pl < P; ++pl) {
      const int d = pl * 64 + 8 * g;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float4 a, e;
        auto val = [&](int k, int row) {
          const float x = SPLIT ? o[pl][k][2 * row] + o[pl][k][2 * row + 1] : o[pl][k][2 * row + c];
          return x * ((k & 1) ? f16 : f1) + zacc[pl][c];
        };
        a = make_float4(val(0, 0), val(1, 0), val(2, 0), val(3, 0));
        e = make_float4(val(0, 1), val(1, 1), val(2, 1), val(3, 1));
        float* row = mine + (C * t + c) * D + d;
        *reinterpret_cast<float4*>(row) = a;
        *reinterpret_cast<float4*>(row + 4) = e;
      }
    }
    if (g == 0)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        stat_m[warp][C * t + c] = m[c];
        stat_l[warp][C * t + c] = l[c];
      }
  }
  __syncthreads();
#pragma unroll 1
  for (int e = tid; e < heads * D / 4; e += kThreads) {
    const int h = e / (D / 4), d = (e % (D / 4)) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < steps) mm = fmaxf(mm, stat_m[w][h]);
    float ll = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w >= steps) break;  // a warp without a step
      const float f = stat_m[w][h] == mm ? 1.f : ex2_approx(stat_m[w][h] - mm);
      const float4 v = *reinterpret_cast<const float4*>(joined[w] + h * D + d);
      ll += f * stat_l[w][h];
      s.x += f * v.x; s.y += f * v.y; s.z += f * v.z; s.w += f * v.w;
    }
    if (parts == 1) {
      const float r = ll != 0.f ? 1.f / ll : 0.f;  // no weight at all: zeros
      store_out4(p.out, p.dtype, (head0 + h) * D + d, make_float4(s.x * r, s.y * r, s.z * r, s.w * r));
    } else {
      float* row = p.partials + ((head0 + h) * p.chunks + chunk) * kRow;
      *reinterpret_cast<float4*>(row + d) = s;
      if (d == 0) *reinterpret_cast<float2*>(row + D) = make_float2(mm, ll);
    }
  }
  if (parts == 1) return;

  // ---- join the chunks: the last CTA of this (sequence, head tile) to arrive ---------------
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int* counter = p.counters + (long long)b * Y + y;
    last_flag = atomicAdd(counter, 1) == parts - 1;
    if (last_flag) *counter = 0;
  }
  __syncthreads();
  if (!last_flag) return;
  __threadfence();
#pragma unroll 1
  for (int e = tid; e < heads * D / 4; e += kThreads) {
    const int h = e / (D / 4), d = (e % (D / 4)) * 4;
    const float* rows = p.partials + (head0 + h) * p.chunks * kRow;
    float mm = -INFINITY, ll = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int c = 0; c < parts; ++c) mm = fmaxf(mm, __ldcg(rows + (long long)c * kRow + D));
#pragma unroll 8
    for (int c = 0; c < parts; ++c) {
      const float* row = rows + (long long)c * kRow;
      const float2 st = __ldcg(reinterpret_cast<const float2*>(row + D));
      const float4 v = __ldcg(reinterpret_cast<const float4*>(row + d));
      const float f = st.x == mm ? 1.f : ex2_approx(st.x - mm);
      ll += f * st.y;
      a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
    }
    const float r = ll != 0.f ? 1.f / ll : 0.f;
    store_out4(p.out, p.dtype, (head0 + h) * D + d, make_float4(a.x * r, a.y * r, a.z * r, a.w * r));
  }
}

template <int P, int BS, bool SPLIT>
int launch(const DecodeInt4Params& p, unsigned grid, cudaStream_t st) {
  if (!allow_smem<decode_int4_kernel<P, BS, SPLIT>>(ring_bytes<P>())) return SPD_ERR_CUDA;
  decode_int4_kernel<P, BS, SPLIT><<<grid, kThreads, ring_bytes<P>(), st>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace dec4

// Heads per column tile: four with two columns each, or eight.
static int dec4_heads(int dtype, int G) { return (dtype == SPD_F32 || G <= 4) ? 4 : 8; }
static long long dec4_tiles(int Hq, int Hkv, int dtype) {
  const int G = Hq / Hkv, heads = dec4_heads(dtype, G);
  return (long long)Hkv * ((G + heads - 1) / heads);
}

// CTAs for each (sequence, head tile), from the longest contexts that the tables hold.  With up to 4096
// tokens for each CTA slot of the device all CTAs run at once, in chunks of 1024 tokens (four steps a
// warp) or more: less makes the join cost more than it saves (one context of 32,000 tokens, 8 key/value
// heads of 128: 17.5 us in chunks of 1024, 20.6 of 640, 22.0 of 1536; one of 448, 12 heads of 64:
// 5.3 us in one chunk, 7.1 in two; 12 of 8,000 to 16,000, 8 heads of 128: 44.7 us at once, 48.9 in
// chunks of 2048).  Beyond that, chunks of 2048 to 4096 tokens, half a slot's share within these: the
// SMs' rates differ by up to a third, and CTAs that are dealt out as slots fall free even that out
// (the 32 contexts above: one equal share per slot 132 us, chunks of 512 tokens 192, 1024 146, 2048
// 126, 4096 128; the 128 contexts: 97, 102, 80, 70, 66).
Int4Split decode_int4_split(int B, int Hq, int Hkv, int D, int dtype, int max_ctx, int sms) {
  using namespace dec4;
  constexpr int kLeast = 1024, kChunk = 2048;
  const int per_sm = D == 64 ? ctas_per_sm<1>() : D == 128 ? ctas_per_sm<2>() : ctas_per_sm<4>();
  const long long slots = (long long)sms * per_sm, pairs = B * dec4_tiles(Hq, Hkv, dtype);
  const long long share = max_ctx * pairs / slots;  // tokens
  if (share <= 2 * kChunk) return {(int)std::max(1ll, std::min(slots / pairs, (max_ctx + kLeast - 1ll) / kLeast)), kLeast};
  const long long c = std::min(std::max(share / 2, (long long)kChunk), 2ll * kChunk);
  return {(int)((max_ctx + c - 1) / c), kChunk};
}

int decode_int4_launch(const DecodeInt4Params& p, int D, int bs, cudaStream_t st) {
  using namespace dec4;
  const long long grid = (long long)p.chunks * p.B * dec4_tiles(p.Hq, p.Hkv, p.dtype);
  if (grid > 0x7fffffffll) return SPD_ERR_UNSUPPORTED;
  auto by_bs = [&](auto planes, auto split) -> int {
    constexpr int P = decltype(planes)::value;
    constexpr bool S = decltype(split)::value;
    switch (bs) {
      case 8: return launch<P, 8, S>(p, (unsigned)grid, st);
      case 16: return launch<P, 16, S>(p, (unsigned)grid, st);
      case 32: return launch<P, 32, S>(p, (unsigned)grid, st);
      default: return SPD_ERR_UNSUPPORTED;
    }
  };
  auto by_planes = [&](auto split) -> int {
    switch (D) {
      case 64: return by_bs(std::integral_constant<int, 1>{}, split);
      case 128: return by_bs(std::integral_constant<int, 2>{}, split);
      case 256: return by_bs(std::integral_constant<int, 4>{}, split);
      default: return SPD_ERR_UNSUPPORTED;
    }
  };
  return dec4_heads(p.dtype, p.Hq / p.Hkv) == 4 ? by_planes(std::true_type{}) : by_planes(std::false_type{});
}

}  // namespace spd
