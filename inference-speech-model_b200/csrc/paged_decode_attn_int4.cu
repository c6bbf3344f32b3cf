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
//   scaled by a running power of two to below 2^15: neither overflows, and what underflows
//   is below 2^-20 of the largest.  With up to four heads per tile (and for fp32 queries)
//   each head takes two columns, the value and its rounding remainder, so q and p keep 22
//   bits; with more, q keeps 11 bits (exact for fp16 and bf16 queries) and p 11.
//
// Work split: one CTA per (chunk of tokens, key/value head, sequence); each of its four
// warps takes every fourth step of 64 tokens, fed by its own ring of shared-memory stages
// (one bulk copy per page, issued by the lanes in parallel, no CTA-wide barrier in the
// loop), with a running maximum that is raised only when a score passes it by 8 (p <= 2^8).
// The warps' results are joined in shared memory, and the chunks' by the last CTA of a
// (sequence, head) to arrive.
#include "spd_int4.cuh"
#include "spd_params.cuh"

namespace spd {
namespace dec4 {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 64;  // tokens per warp step
constexpr float kLazy = 8.f;  // log2 units a score may pass the reference maximum by

template <int P> constexpr int stages() { return P == 1 ? 4 : 3; }
template <int P> constexpr int step_bytes() { return int4::page_bytes(P, kStep); }
template <int P> constexpr size_t smem_bytes() { return (size_t)kWarps * stages<P>() * step_bytes<P>() + 1024; }

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
__global__ void __launch_bounds__(kThreads) decode_int4_kernel(const DecodeInt4Params p) {
  constexpr int D = P * int4::kPlane;
  constexpr int kHeads = SPLIT ? 4 : 8;  // heads per column tile
  constexpr int kStages = stages<P>();
  constexpr int kPage = int4::page_bytes(P, BS), kHalf = int4::half_bytes(P, BS);
  constexpr int kPages = kStep / BS;
  constexpr int kParams = P * BS * int4::kRowBytes;  // offset of the parameters in a half page
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ float stat_m[kWarps][8], stat_l[kWarps][8];
  __shared__ int last_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int b = blockIdx.z, split = blockIdx.x;
  const int G = p.Hq / p.Hkv;
  const int tiles = (G + kHeads - 1) / kHeads;
  const int kvh = (int)blockIdx.y / tiles, tile = (int)blockIdx.y % tiles;
  const int heads = min(kHeads, G - tile * kHeads);  // of this tile
  const long long head0 = (long long)b * p.Hq + kvh * G + tile * kHeads;  // row of q and out

  int ctx = p.context_lens[b];
  if ((long long)ctx > (long long)p.max_blocks * BS) {
    if (tid == 0) set_error(p.err, SPD_DEVERR_LENGTH);
    ctx = p.max_blocks * BS;
  }
  if (ctx <= 0) {
    if (split == 0)
      for (int i = tid; i < heads * D / 4; i += kThreads)
        store_out4(p.out, p.dtype, head0 * D + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int t0 = split * p.chunk;
  if (t0 >= ctx) return;
  const int t1 = min(ctx, t0 + p.chunk);
  const int nsplit = (ctx + p.chunk - 1) / p.chunk;
  const int steps = (t1 - t0 + kStep - 1) / kStep;
  const int my_steps = steps > warp ? (steps - warp + kWarps - 1) / kWarps : 0;

  unsigned char* ring = smem + (size_t)warp * kStages * step_bytes<P>();
  const int* table = p.block_tables + (long long)b * p.max_blocks;
  const unsigned char* pool_h = p.pool + (long long)kvh * kPage;
  const long long block_stride = (long long)p.Hkv * kPage;
  const uint64_t policy = l2_policy_evict_first();
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[warp][s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  // Copies the pages of this warp's i-th step into its stage.
  auto issue = [&](int i) {
    const int tok = t0 + (warp + i * kWarps) * kStep;
    const int n = min(kPages, (t1 - tok + BS - 1) / BS);
    uint64_t* bar = &bars[warp][i % kStages];
    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(n * kPage));
    __syncwarp();
    if (lane < n) {
      int id = table[tok / BS + lane];
      if (id < 0 || id >= p.num_blocks) {
        set_error(p.err, SPD_DEVERR_BLOCK_ID);
        id = 0;
      }
      bulk_copy_g2s_hint(ring + (size_t)(i % kStages) * step_bytes<P>() + lane * kPage, pool_h + id * block_stride, kPage,
                         bar, policy);
    }
  };
  for (int i = 0; i < kStages && i < my_steps; ++i) issue(i);

  // ---- the query fragments: column g, k = this lane's 16 dimensions of each plane --------
  uint32_t qb[P][4][2];
  float fa, fb, qsa[P], qsb[P];  // score factors and sums of q of this lane's columns 2t, 2t + 1
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
        amax = fmaxf(amax, fabsf(qv[pl][i]));
        qs[pl] += qv[pl][i];
      }
      qs[pl] += __shfl_xor_sync(0xffffffffu, qs[pl], 1);
      qs[pl] += __shfl_xor_sync(0xffffffffu, qs[pl], 2);
      qs[pl] *= p.scale_log2;
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
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
    const float f = pow2(24 - k) * p.scale_log2;
    fa = __shfl_sync(0xffffffffu, f, 8 * t);
    fb = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
    for (int pl = 0; pl < P; ++pl) {
      qsa[pl] = __shfl_sync(0xffffffffu, qs[pl], 8 * t);
      qsb[pl] = __shfl_sync(0xffffffffu, qs[pl], 8 * t + 4);
    }
  }

  constexpr int C = SPLIT ? 1 : 2;  // heads of this lane's two columns
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

  // Row r of an 8-token group holds token r ^ (r >> 2): with it both the rows that a
  // half-warp reads for the scores (r = 0..3, 4..7) and those that a warp reads for the output
  // (even or odd r) fall on four different quarters of the 32 banks.
  const int tok_k = g ^ (g >> 2);
  const int tok_v0 = (2 * t) ^ (t >> 1), tok_v1 = (2 * t + 1) ^ (t >> 1);
  auto place = [](int tok) { return (tok / BS) * kPage + (tok % BS) * int4::kRowBytes; };

  int i = 0;
  for (; i < my_steps; ++i) {
    const int st = i % kStages;
    const bool ok = mbar_wait_bounded(&bars[warp][st], (uint32_t)((i / kStages) & 1), p.err, p.wait_ns);
    if (!__all_sync(0xffffffffu, ok)) break;
    const unsigned char* buf = ring + (size_t)st * step_bytes<P>();
    const int left = t1 - (t0 + (warp + i * kWarps) * kStep);  // valid tokens of this step (>= 1)

    // ---- scores ----------------------------------------------------------------------
    float sc[4][2 * C];      // per 16 tokens: tokens tok_k and tok_k + 8 of each head
    uint32_t vp[4][2][P];    // the value parameters of those tokens, zero past the end
    uint32_t smax = 0;
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
#pragma unroll
      for (int c = 0; c < 2 * C; ++c) sc[sub][c] = 0.f;
      const int ta = sub * 16 + tok_k, tb = ta + 8;
      const bool va = ta < left, vb = tb < left;
#pragma unroll
      for (int pl = 0; pl < P; ++pl) {
        const uint2 wa = *reinterpret_cast<const uint2*>(buf + place(ta) + pl * BS * int4::kRowBytes + 8 * t);
        const uint2 wb = *reinterpret_cast<const uint2*>(buf + place(tb) + pl * BS * int4::kRowBytes + 8 * t);
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t xa = w ? wa.y : wa.x, xb = w ? wb.y : wb.x;
          mma_16816<__half>(acc, xa & 0x000F000Fu, xb & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x00F000F0u, qb[pl][2 * w][0],
                            qb[pl][2 * w][1]);
          mma_16816<__half>(acc, (xa >> 8) & 0x000F000Fu, (xb >> 8) & 0x000F000Fu, (xa >> 8) & 0x00F000F0u,
                            (xb >> 8) & 0x00F000F0u, qb[pl][2 * w + 1][0], qb[pl][2 * w + 1][1]);
        }
        const int pa = (ta / BS) * kPage + kParams + (pl * BS + ta % BS) * int4::kParamBytes;
        const int pb = (tb / BS) * kPage + kParams + (pl * BS + tb % BS) * int4::kParamBytes;
        const float2 ka = unpack_half(*reinterpret_cast<const uint32_t*>(buf + pa));
        const float2 kb = unpack_half(*reinterpret_cast<const uint32_t*>(buf + pb));
        if (SPLIT) {
          sc[sub][0] += fa * ka.x * (acc[0] + acc[1]) + qsa[pl] * ka.y;
          sc[sub][1] += fa * kb.x * (acc[2] + acc[3]) + qsa[pl] * kb.y;
        } else {
          sc[sub][0] += fa * ka.x * acc[0] + qsa[pl] * ka.y;
          sc[sub][C - 1] += fb * ka.x * acc[1] + qsb[pl] * ka.y;
          sc[sub][C] += fa * kb.x * acc[2] + qsa[pl] * kb.y;
          sc[sub][2 * C - 1] += fb * kb.x * acc[3] + qsb[pl] * kb.y;
        }
        vp[sub][0][pl] = va ? *reinterpret_cast<const uint32_t*>(buf + kHalf + pa) : 0u;
        vp[sub][1][pl] = vb ? *reinterpret_cast<const uint32_t*>(buf + kHalf + pb) : 0u;
        smax = max(smax, max(vp[sub][0][pl] & 0x7FFFu, vp[sub][1][pl] & 0x7FFFu));
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (!va) sc[sub][c] = -INFINITY;
        if (!vb) sc[sub][C + c] = -INFINITY;
      }
    }

    // ---- running maximum and weight exponent: raised for the whole warp when needed --------
    float mx[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      mx[c] = -INFINITY;
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) mx[c] = fmaxf(mx[c], fmaxf(sc[sub][c], sc[sub][C + c]));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], x));
    }
    const int new_lift = min(15, (int)(__reduce_max_sync(0xffffffffu, smax) >> 10) - 15);
    bool raise = new_lift > lift;
#pragma unroll
    for (int c = 0; c < C; ++c) raise |= mx[c] > m[c] + kLazy;
    if (__any_sync(0xffffffffu, raise)) {
      const int up = max(lift, new_lift);
      const float w = pow2(lift - up);
      lift = up;
      float f[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float mn = fmaxf(m[c], mx[c]);
        f[c] = m[c] == mn ? 1.f : ex2_approx(m[c] - mn);  // also when both are -inf
        m[c] = mn;
        l[c] *= f[c];
#pragma unroll
        for (int pl = 0; pl < P; ++pl) zacc[pl][c] *= f[c];
        f[c] *= w;
      }
#pragma unroll
      for (int pl = 0; pl < P; ++pl)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[pl][k][0] *= f[0];
          o[pl][k][1] *= f[C - 1];
          o[pl][k][2] *= f[0];
          o[pl][k][3] *= f[C - 1];
        }
    }
    const float wscale = pow2(6 - lift);
    constexpr float mid = 7.5f;
    const float unscale = mid * pow2(lift - 6);

    // ---- output ------------------------------------------------------------------------
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
      float pr[2 * C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        // a head whose scores are all -inf so far keeps m = -inf: its weights are 0
        pr[c] = ex2_approx(sc[sub][c] - (m[c] == -INFINITY ? 0.f : m[c]));
        pr[C + c] = ex2_approx(sc[sub][C + c] - (m[c] == -INFINITY ? 0.f : m[c]));
        l[c] += pr[c] + pr[C + c];
      }
#pragma unroll
      for (int pl = 0; pl < P; ++pl) {
        const float2 a = unpack_half(vp[sub][0][pl]), bq = unpack_half(vp[sub][1][pl]);
        const float sa = a.x * wscale, sb = bq.x * wscale;
        uint32_t b0, b1;
        if (SPLIT) {
          b0 = movmatrix_trans(pack_split(pr[0] * sa));
          b1 = movmatrix_trans(pack_split(pr[1] * sb));
          zacc[pl][0] += pr[0] * a.y + pr[1] * bq.y;
        } else {
          // what the rounding of a weight takes from the middle code (7.5) is put back, so that
          // its error meets codes of both signs, as an output's own rounding would
          const uint32_t ha = pack_half(pr[0] * sa, pr[C - 1] * sa), hb = pack_half(pr[C] * sb, pr[2 * C - 1] * sb);
          b0 = movmatrix_trans(ha);
          b1 = movmatrix_trans(hb);
          const float2 ra = unpack_half(ha), rb = unpack_half(hb);
          zacc[pl][0] += pr[0] * (a.y + mid * a.x) - ra.x * unscale + pr[C] * (bq.y + mid * bq.x) - rb.x * unscale;
          zacc[pl][C - 1] += pr[C - 1] * (a.y + mid * a.x) - ra.y * unscale + pr[2 * C - 1] * (bq.y + mid * bq.x) - rb.y * unscale;
        }
        const unsigned char* vb_ = buf + kHalf + pl * BS * int4::kRowBytes + 4 * g;
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + tok_v0));
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + tok_v1));
        const uint32_t w2 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + 8 + tok_v0));
        const uint32_t w3 = *reinterpret_cast<const uint32_t*>(vb_ + place(sub * 16 + 8 + tok_v1));
        // dimensions 8g..8g+3 (lo) and 8g+4..8g+7 (hi) of a pair of tokens per register
        uint32_t lo0 = __byte_perm(w0, w1, 0x5410), hi0 = __byte_perm(w0, w1, 0x7632);
        uint32_t lo1 = __byte_perm(w2, w3, 0x5410), hi1 = __byte_perm(w2, w3, 0x7632);
        mma_16816<__half>(o[pl][0], lo0 & 0x000F000Fu, hi0 & 0x000F000Fu, lo1 & 0x000F000Fu, hi1 & 0x000F000Fu, b0, b1);
        mma_16816<__half>(o[pl][1], lo0 & 0x00F000F0u, hi0 & 0x00F000F0u, lo1 & 0x00F000F0u, hi1 & 0x00F000F0u, b0, b1);
        lo0 >>= 8; hi0 >>= 8; lo1 >>= 8; hi1 >>= 8;
        mma_16816<__half>(o[pl][2], lo0 & 0x000F000Fu, hi0 & 0x000F000Fu, lo1 & 0x000F000Fu, hi1 & 0x000F000Fu, b0, b1);
        mma_16816<__half>(o[pl][3], lo0 & 0x00F000F0u, hi0 & 0x00F000F0u, lo1 & 0x00F000F0u, hi1 & 0x00F000F0u, b0, b1);
      }
    }
    __syncwarp();  // every lane has read this stage
    if (i + kStages < my_steps) issue(i + kStages);
  }
  if (i < my_steps)  // a wait gave up: let this warp's copies in flight land before the CTA can exit
    for (int k = i; k < my_steps && k < i + kStages; ++k)
      (void)mbar_wait_bounded(&bars[warp][k % kStages], (uint32_t)((k / kStages) & 1), nullptr);

  // ---- join the warps ---------------------------------------------------------------------
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
#pragma unroll
      for (int pl = 0; pl < P; ++pl) zacc[pl][c] += __shfl_xor_sync(0xffffffffu, zacc[pl][c], x);
    }
  __syncwarp();
  float* mine = reinterpret_cast<float*>(ring);  // [head][D]; the ring is drained
  {
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
  constexpr int kRow = D + 4;  // floats per partial row: D values, m, l, two unused
  for (int e = tid; e < heads * D / 4; e += kThreads) {
    const int h = e / (D / 4), d = (e % (D / 4)) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, stat_m[w][h]);
    float ll = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (steps <= w) break;  // a warp without a step
      const float f = stat_m[w][h] == mm ? 1.f : ex2_approx(stat_m[w][h] - mm);
      const float4 v = *reinterpret_cast<const float4*>(smem + (size_t)w * kStages * step_bytes<P>() + (h * D + d) * 4);
      ll += f * stat_l[w][h];
      s.x += f * v.x; s.y += f * v.y; s.z += f * v.z; s.w += f * v.w;
    }
    if (nsplit == 1) {
      const float r = ll != 0.f ? 1.f / ll : 0.f;  // no weight at all: zeros
      store_out4(p.out, p.dtype, (head0 + h) * D + d, make_float4(s.x * r, s.y * r, s.z * r, s.w * r));
    } else {
      float* row = p.partials + ((head0 + h) * p.splits + split) * kRow;
      *reinterpret_cast<float4*>(row + d) = s;
      if (d == 0) *reinterpret_cast<float2*>(row + D) = make_float2(mm, ll);
    }
  }
  if (nsplit == 1) return;

  // ---- join the chunks: the last CTA of this (sequence, head tile) to arrive ---------------
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int* counter = p.counters + (long long)b * gridDim.y + blockIdx.y;
    const int n = atomicAdd(counter, 1);
    last_flag = n == nsplit - 1;
    if (last_flag) *counter = 0;
  }
  __syncthreads();
  if (!last_flag) return;
  __threadfence();
  for (int e = tid; e < heads * D / 4; e += kThreads) {
    const int h = e / (D / 4), d = (e % (D / 4)) * 4;
    const float* rows = p.partials + (head0 + h) * p.splits * kRow;
    float mm = -INFINITY;
    for (int s = 0; s < nsplit; ++s) mm = fmaxf(mm, __ldcg(rows + s * kRow + D));
    float ll = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < nsplit; ++s) {
      const float2 st = __ldcg(reinterpret_cast<const float2*>(rows + s * kRow + D));
      const float4 v = __ldcg(reinterpret_cast<const float4*>(rows + s * kRow + d));
      const float f = st.x == mm ? 1.f : ex2_approx(st.x - mm);
      ll += f * st.y;
      a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
    }
    const float r = ll != 0.f ? 1.f / ll : 0.f;
    store_out4(p.out, p.dtype, (head0 + h) * D + d, make_float4(a.x * r, a.y * r, a.z * r, a.w * r));
  }
}

template <int P, int BS, bool SPLIT>
int launch(const DecodeInt4Params& p, dim3 grid, cudaStream_t st) {
  if (!allow_smem<decode_int4_kernel<P, BS, SPLIT>>(smem_bytes<P>())) return SPD_ERR_CUDA;
  decode_int4_kernel<P, BS, SPLIT><<<grid, kThreads, smem_bytes<P>(), st>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace dec4

// Heads per column tile: four with two columns each, or eight.
static int dec4_heads(int dtype, int G) { return (dtype == SPD_F32 || G <= 4) ? 4 : 8; }

// Tokens per CTA: enough CTAs for four rounds of two per SM, each at least one step per warp
// and at most 4096 tokens (which bounds what the slowest CTA of a ragged batch does alone).
int decode_int4_chunk(int B, int Hq, int Hkv, int dtype, int max_ctx, int sms) {
  const int G = Hq / Hkv, kHeads = dec4_heads(dtype, G);
  const long long pairs = (long long)B * Hkv * ((G + kHeads - 1) / kHeads);
  const long long unit = dec4::kWarps * dec4::kStep;
  long long c = ((long long)max_ctx * pairs / (sms * 8) + unit - 1) / unit * unit;
  return (int)(c < unit ? unit : c > 4096 ? 4096 : c);
}

int decode_int4_launch(const DecodeInt4Params& p, int D, int bs, cudaStream_t st) {
  using namespace dec4;
  const int G = p.Hq / p.Hkv, kHeads = dec4_heads(p.dtype, G);
  const dim3 grid((unsigned)p.splits, (unsigned)(p.Hkv * ((G + kHeads - 1) / kHeads)), (unsigned)p.B);
  auto by_bs = [&](auto planes, auto split) -> int {
    constexpr int P = decltype(planes)::value;
    constexpr bool S = decltype(split)::value;
    switch (bs) {
      case 8: return launch<P, 8, S>(p, grid, st);
      case 16: return launch<P, 16, S>(p, grid, st);
      case 32: return launch<P, 32, S>(p, grid, st);
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
  return kHeads == 4 ? by_planes(std::true_type{}) : by_planes(std::false_type{});
}

}  // namespace spd
