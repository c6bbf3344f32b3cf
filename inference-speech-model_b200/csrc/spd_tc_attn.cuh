// spd_tc_attn.cuh — pieces shared by the attention kernels on tcgen05 (prompt_attn.cu, span_attn.cu):
// issue of products four at a time, TMEM loads and stores of 32 columns, the exponentials of a score
// tile (special-function unit and polynomial side by side), rings of stages.
#pragma once

#include "spd_tc.cuh"

namespace spd {
namespace tc {

constexpr float kLazy = 8.f;  // log2 units a score may pass the reference maximum by

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

// Has phase `parity` completed?  (Does not wait.)
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// One lane of a converged warp (the same one each time).
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}

// Four products of 16 k each, issued back to back: an operand's descriptors are its first one plus
// a constant, so that the issue takes fewer cycles than the products (64 each at N = 128).
// D[128 x N] (+)= A B, both in shared memory: k advances by 32 bytes inside the swizzle row.
__device__ __forceinline__ void umma4_ss(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, 1;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, 1;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, 1;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[128 x N] (+)= A B with A in TMEM (16-bit pairs, 8 columns per 16 k) and B MN-major: 16 k-rows
// of 128 bytes further.
__device__ __forceinline__ void umma4_ts(uint32_t d_tmem, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
      "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, 1;\n\t}" ::"r"(d_tmem),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// MN-major operand with 128-byte swizzle: 8 k-rows of 64 consecutive elements form a 1024-byte
// atom; atoms follow each other along k (stride 1024) and 64-element blocks every block_bytes.
__device__ __forceinline__ uint64_t smem_desc_mn(const void* tile, uint32_t block_bytes) {
  const uint64_t addr = smem_addr(tile);
  uint64_t d = 0;
  d |= (addr >> 4) & 0x3FFFull;
  d |= (uint64_t)(block_bytes >> 4) << 16;  // leading byte offset: next 64 elements
  d |= (uint64_t)(1024 >> 4) << 32;         // stride byte offset: next 8 k-rows
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// Waits for the loads issued so far; ties the 32 registers to the wait so that no use of them
// is scheduled before it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// the largest of three, NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ---- pairs of fp32 in one instruction ----------------------------------------------------
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^x of a pair on the fp32 pipes, for x <= 100; below -125 it stays at 2^-125.  x is split into a
// whole number n (adding 1.5 * 2^23 rounds it to the low bits) and f in [-1/2, 1/2]; 2^f is a
// polynomial whose largest relative error is least (fitted by the Remez exchange to 2^f on that
// interval: 7.5e-5 at degree 3, 2.6e-6 at degree 4), and n is added to its exponent field.  The
// special-function unit gives 4 results a cycle and quarter SM, a quarter of what the softmax
// needs; degree 3 is under a bf16 weight's rounding (2^-9), degree 4 under fp16's (2^-12).
template <int DEG>
__device__ __forceinline__ float2 exp2_poly(f32x2 x) {
  float2 v = unpair(x);
  x = pair(fmaxf(v.x, -125.f), fmaxf(v.y, -125.f));
  const f32x2 t = add2(x, pair(12582912.f, 12582912.f));
  const f32x2 f = fma2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), x);
  f32x2 q;
  if constexpr (DEG == 3) {
    q = fma2(pair(0.0551716691f, 0.0551716691f), f, pair(0.242611122f, 0.242611122f));
    q = fma2(q, f, pair(0.693260985f, 0.693260985f));
    q = fma2(q, f, pair(0.999928074f, 0.999928074f));
  } else {
    q = fma2(pair(0.00957010191f, 0.00957010191f), f, pair(0.0559178603f, 0.0559178603f));
    q = fma2(q, f, pair(0.240247448f, 0.240247448f));
    q = fma2(q, f, pair(0.693121815f, 0.693121815f));
    q = fma2(q, f, pair(0.999999261f, 0.999999261f));
  }
  const float2 n = unpair(t), p = unpair(q);
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(n.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(n.y) << 23)));
}

constexpr int kPoly = 2;  // of 8 pairs, to the polynomial
// Weights of 2 * PAIRS keys: p = 2^(s * c - m) rounded to T and packed, sums added.  EXACT: all on the
// special-function unit, so that a masked score (-inf) gives an exact zero and a NaN a NaN; otherwise kPoly of
// each 8 pairs go to the polynomial (0: 151 us, 1: 146, 2: 145, 4: 162 for the 8 x 1500 when last swept, and 516,
// 518, 519 and 532 in long runs of the 8192 tokens, 493, 485, 484 and 496 of an earlier form in short
// ones: the polynomial's six packed fp32 instructions soon cost more than they free).
template <typename T, bool EXACT, int PAIRS>
__device__ __forceinline__ void weights(const uint32_t* s, f32x2 c, f32x2 neg_m, uint32_t* pk, f32x2 (&sum)[2]) {
  constexpr int kDeg = std::is_same<T, __half>::value ? 4 : 3;
#pragma unroll
  for (int k = 0; k < PAIRS; ++k) {
    const f32x2 x = fma2(pair(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), c, neg_m);
    float2 e;
    if (!EXACT && (k * kPoly) % 8 < kPoly) {  // spread evenly
      e = exp2_poly<kDeg>(x);
    } else {
      const float2 v = unpair(x);
      e = make_float2(ex2_approx(v.x), ex2_approx(v.y));
    }
    sum[k & 1] = add2(sum[k & 1], pair(e.x, e.y));
    pk[k] = pack2<T>(e.x, e.y);
  }
}

// scores of keys at or past `seen` to -inf
template <int N>
__device__ __forceinline__ void mask(uint32_t* s, int seen) {
#pragma unroll
  for (int c = 0; c < N; ++c)
    if (c >= seen) s[c] = 0xff800000u;
}
// four running maxima over N scores
template <int N, bool FIRST>
__device__ __forceinline__ void max4(const uint32_t* s, float (&m)[4]) {
  if (FIRST)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __uint_as_float(s[i]);
#pragma unroll
  for (int c = FIRST ? 4 : 0; c < N; c += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m[i] = max3_nan(m[i], __uint_as_float(s[c + i]), __uint_as_float(s[c + 4 + i < N ? c + 4 + i : c + i]));
}

// Position in a ring of stages: the slot, and how often the ring has come round.
struct Ring {
  int slot = 0, round = 0;
  __device__ __forceinline__ uint32_t phase() const { return (uint32_t)(round & 1); }
  __device__ __forceinline__ void next(int stages) {
    if (++slot == stages) slot = 0, ++round;
  }
  __device__ __forceinline__ void back(int stages) {
    if (--slot < 0) slot = stages - 1, --round;
  }
  __device__ __forceinline__ void skip(int n, int stages) {
    slot += n;
    round += slot / stages;
    slot %= stages;
  }
};

}  // namespace tc
}  // namespace spd
