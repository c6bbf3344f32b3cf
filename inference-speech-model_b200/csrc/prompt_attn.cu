// prompt_attn.cu — attention of whole packed prompts:
//   out[i, h] = softmax_j(q[i, h] . k[j, h / G] * scale) . v[j, h / G]
// for the queries i and keys j of each of B sequences packed along the token axis
// (cu_q, cu_k: prefix sums of their lengths), with Hq = G * Hkv query heads.  A sequence may
// have more keys than queries (a cached prefix); with `causal` query i sees the keys
// j <= i + Tk - Tq, and a query that sees none gives zeros.
//
// Bounded by the tensor cores and, beside them, by the exponentials: a 128 x 128 score tile
// at D = 128 is 8.4 MFLOP (about 1,020 cycles of an SM's dense 16-bit rate) and 16,384
// exponentials (1,024 cycles of its special-function units); at D = 64 the exponentials
// take twice the products' time.
//
// sm_100a design:
// * A CTA owns two tiles of 128 query rows (A and B).  `pack` heads that share a key/value
//   head sit in one tile (row = token * pack + head), so K and V are read once for all of
//   them and short prompts fill the rows.
// * Warp 0 loads Q, K and V tiles by TMA (3-D maps over [tokens][heads][D], any strides;
//   128-byte swizzle).  One lane of warp 1 issues every tcgen05.mma, four at a time, with nothing
//   else in its step: S = Q K^T into TMEM and O += P V with P read from TMEM (it overwrites S)
//   and V as the MN-major operand, so nothing is transposed or written back to shared memory.
// * Warps 4-7 and 8-11 are the softmax of tiles A and B: one row per thread, so the row
//   maximum and sum need no shuffles.  While one tile's softmax runs, the tensor cores work on
//   the other tile; weights are handed over 64 keys at a time.  The running maximum is raised
//   only when a score passes it by 8 (in log2), so O in TMEM is rescaled rarely; P is at most
//   2^8 and rounded to the input type (its 8 or 11 bits are what the tensor core takes), the row
//   sum is taken in fp32 before the rounding.  A quarter of the exponentials is a polynomial on
//   the fp32 pipes.  (Both the lazy maximum and the polynomial are published techniques of
//   attention kernels on this architecture.)
// * Where a key does not count its weight is zero, but 0 * NaN is not.  So warp 2 sets rows of V past a
//   sequence's last key to zero in shared memory before they are multiplied, and, among keys that some
//   rows of the CTA do not see, every element that is not finite; rows that do see such a key add it
//   at the end.  What another sequence or a later key holds never reaches a result.  The tile is
//   handed to warp 2 a step ahead, so that its look (one multiply-add a pair) is mostly over in time
//   (graphs of the calls below with it and without: short prompts 10.4 and 10.2 us, the 8 x 1500, where
//   it looks at nothing, 147 and 143, ragged grouped prompts the same).
// * Steps are of 128 keys with one CTA an SM; at D <= 64, where TMEM holds four tiles, of 64 keys
//   with two CTAs an SM, unless no SM gets a second item.
// * One CTA is launched for each item (tile pair and head group), ranked by length; a running CTA
//   takes over the items of CTAs that have not started (warp 3 calls off their launch), so tiles
//   follow one another in it without a gap and the longest come first.  Every wait is bounded, and
//   waits suspend the thread, which leaves the issue slots to the softmax warps.
//
// Measured in replayed graphs (bf16, 32 query and 8 key/value heads of 128, causal): 8192 tokens 450 us in
// the first 60 ms of replays, at 1,965 MHz, 1.22 PFLOP/s and 0.75 of the library product's rate in a
// short run; 507 us from then on, under the power cap at 1.6 to 1.7 GHz; a lone call 523 us.  A
// step of 128 keys of both tiles takes about 3,250 cycles against 2,050 of products: a tile's chain
// (scores, their maximum, 128 exponentials a thread, weights, P V, next scores) is 1.5 times as long
// as the other tile's products can cover.  fp16, 20 heads of 64, 8 x 1500 tokens, not causal: 147 us,
// 0.63 PFLOP/s, where exponentials alone take 63 to 84.  The figures below compared forms when each was
// chosen, in short runs; the later one's present time may be another.  64 keys and two CTAs against 128 and
// one at D = 64: 143 against 166 us there, 202 against 224 for 4 x 4096 causal tokens of 16 heads, but 11.5 against
// 10.3 for 6 short prompts of 12 heads, one item an SM at most.  Items dealt out in fixed turns instead of taken
// over: 147 (forwards) and 163 us (forwards and backwards) for the 8 x 1500, 215 and 210 for the 4 x
// 4096.  Slower at D = 128: steps of 64 keys with two score buffers a tile, so that scores are there
// before the last weights are used (544 us; products of 64 columns read shared memory 1.5 times as
// often, and each step's hand-over is paid twice); two threads a row, two issuing lanes (the tiles
// fall into step) and a second read of S in place of 128 registers (579, 565 and 525 us when this one
// took 485).
#include "spd_tc.cuh"

#include <algorithm>

namespace spd {
namespace pa {
using namespace tc;

constexpr int BM = 128;  // query rows per tile (two tiles per CTA)
constexpr int kThreads = 384;
constexpr int kItems = 2;   // item slots
// Key steps before an item's end (counted by its loads) that the next one is asked for: late enough that
// the CTA that is done first takes the longest, early enough to hide the search.  2, 4 and 8 for the 8 x
// 1500 above: 143, 143, 145 us; for ragged grouped prompts 226, 222, 222; for 16 of up to 700 tokens
// 27.6, 28.0, 31.
constexpr int kAhead = 4;
constexpr float kLazy = 8.f;  // log2 units a score may pass the reference maximum by

// DP: head size, padded to 64 or 128; BN: keys per step.
template <int DP, int BN> struct Cfg {
  static constexpr int kCtas = BN == 128 ? 1 : 2;         // CTAs per SM
  static constexpr int kBoxes = DP / 64;                  // 64-column boxes of a row
  static constexpr int kQBox = 128 * 128;                 // 128 rows of 128 bytes
  static constexpr int kQBytes = kBoxes * kQBox;          // one Q tile
  static constexpr int kKvBox = BN * 128;
  static constexpr int kKvBytes = kBoxes * kKvBox;        // one K or V tile
  static constexpr int kParts = BN / 64;                  // weights are handed over 64 keys at a time
  static constexpr int kStages = DP == 128 ? 5 : 8;       // K and V tiles in flight
  static constexpr int kBarBytes = 512;
  static constexpr size_t kSmem = 1024 + 2 * (size_t)kQBytes + (size_t)kStages * kKvBytes + kBarBytes;
  static constexpr uint32_t kO = 2 * BN;                  // TMEM column of O_A; S_A at 0, S_B at BN
  static constexpr uint32_t kTmemCols = BN == 128 ? 512 : 256;
  // registers of the softmax threads and of the others; their sum is within what the launch gives to
  // all 384 (168 or 80 each, checked at the launch)
  static constexpr int kSoftmaxRegs = BN == 128 ? 216 : 96, kOtherRegs = BN == 128 ? 72 : 48;
  static constexpr int kAllRegs = 256 * kSoftmaxRegs + 128 * kOtherRegs;
  static_assert(kO + 2 * DP <= kTmemCols, "scores and outputs fit in TMEM");
};
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

// NaN in either half of the result if any of the eight values is not finite (or acc had one).
template <typename T>
__device__ __forceinline__ uint32_t odd_acc(uint4 v, uint32_t acc) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value)
      asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w[i]), "r"(0u));
    else
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w[i]), "r"(0u));
  }
  return acc;
}
// A pair of 16-bit values with those that are not finite set to zero.
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  if ((w & kExp) == kExp) w &= 0xFFFF0000u;
  if ((w >> 16 & kExp) == kExp) w &= 0x0000FFFFu;
  return w;
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

// One unit of work: 2 x 128 query rows (tokens [tok0, tok0 + 256 / pack) of one sequence for
// `pack` heads from h0).
struct Item {
  int q0, Tq, k0, Tk;  // the sequence's first query/key row and its lengths
  int tok0;            // first token of the CTA's tiles within the sequence
  int h0, kvh;
  int n[2];            // key steps of tiles A and B
  int there;           // 0 past the last item
};

// Asks for the next CTA that has not started yet: its index arrives in `response`, and its launch is
// called off.
__device__ __forceinline__ void ask_for_cta(void* response, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_addr(response)),
               "r"(smem_addr(bar))
               : "memory");
}
// The index of the CTA that was called off, or -1 if none was left.
__device__ __forceinline__ int called_off(const void* response) {
  uint32_t yes, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(yes), "=r"(x)
      : "r"(smem_addr(response))
      : "memory");
  return yes ? (int)x : -1;
}

// Sequence s of the packed batch: its query and key rows, clamped to what there is, and its tiles.
struct Span {
  int q0, Tq, k0, Tk, tiles;
  __device__ __forceinline__ Span(const PromptParams& p, int s, int tokens) {
    q0 = max(0, min(p.Nq, p.cu_q[s]));
    Tq = max(q0, min(p.Nq, p.cu_q[s + 1])) - q0;
    k0 = max(0, min(p.Nk, p.cu_k[s]));
    Tk = max(k0, min(p.Nk, p.cu_k[s + 1])) - k0;
    tiles = (Tq + tokens - 1) / tokens;
  }
  // How many of its tiles (the last ones) take t key steps or more.
  template <int BN>
  __device__ __forceinline__ int longer(const PromptParams& p, int t, int tokens) const {
    if (t <= 0 || tiles == 0) return tiles;
    const int need = (t - 1) * BN + 1;  // keys
    if (Tk < need) return 0;
    if (!p.causal) return tiles;
    return tiles - max(0, min(tiles - 1, (need - (Tk - Tq) + tokens - 1) / tokens - 1));
  }
};

// The it-th item, found by the whole warp from the prefix sums; false past the last one.  Heads come
// fastest.  With `ranked` the tiles come in the order of their key steps, the longest first: the
// number of steps that `tile` others have is searched for by halving, counting over the sequences.
// Otherwise (every item starts at once) they come sequence by sequence.
template <int BN>
__device__ __forceinline__ bool find_item(const PromptParams& p, int it, Item& w) {
  const int lane = threadIdx.x & 31;
  const int tokens = 2 * BM / p.pack, groups = p.Hq / p.pack;
  const int tile = it / groups, grp = it % groups;
  int steps = 0;  // of the tile; the tiles that have more come before
  int before = 0, b = -1, lvl = 0;
  if (p.ranked) {
    int most = 0;
    for (int base = 0; base < p.B; base += 32)
      if (base + lane < p.B) most = max(most, Span(p, base + lane, tokens).Tk);
    int none = (int)(__reduce_max_sync(0xffffffffu, (unsigned)most) + BN - 1) / BN + 1;  // nothing is as long
    while (none - steps > 1) {
      const int mid = (steps + none) / 2;
      int n = 0;
      for (int base = 0; base < p.B; base += 32)
        if (base + lane < p.B) n += Span(p, base + lane, tokens).longer<BN>(p, mid, tokens);
      n = __reduce_add_sync(0xffffffffu, n);
      if (n > tile) {
        steps = mid;
      } else {
        none = mid;
        before = n;
      }
    }
  }
  for (int base = 0; base < p.B; base += 32) {
    int tiles = 0, first = 0;
    if (base + lane < p.B) {
      const Span s(p, base + lane, tokens);
      const int n = p.ranked ? s.longer<BN>(p, steps, tokens) : s.tiles;
      first = s.tiles - n;
      tiles = p.ranked ? n - s.longer<BN>(p, steps + 1, tokens) : n;
    }
    int incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, tile < before + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      b = base + src;
      lvl = __shfl_sync(0xffffffffu, first - (incl - tiles), src) + tile - before;
      break;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (b < 0) return false;
  const Span s(p, b, tokens);
  w.q0 = s.q0;
  w.Tq = s.Tq;
  w.k0 = s.k0;
  w.Tk = s.Tk;
  w.tok0 = lvl * tokens;
  w.h0 = grp * p.pack;
  w.kvh = w.h0 / (p.Hq / p.Hkv);
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int first = w.tok0 + x * (tokens / 2), last = min(w.Tq, first + tokens / 2) - 1;
    int keys = 0;  // that the tile's last token sees
    if (first < w.Tq) keys = p.causal ? min(w.Tk, last + 1 + w.Tk - w.Tq) : w.Tk;
    w.n[x] = keys > 0 ? (keys + BN - 1) / BN : 0;
  }
  return true;
}

// Keys that every row of the item sees: the first ones.
__device__ __forceinline__ int seen_by_all(const PromptParams& p, const Item& w) {
  return p.causal ? max(0, min(w.Tk, w.tok0 + 1 + w.Tk - w.Tq)) : w.Tk;
}

template <typename T, int DP, int BN>
__global__ void __launch_bounds__(kThreads, Cfg<DP, BN>::kCtas)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const PromptParams p) {
  using C = Cfg<DP, BN>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Item items[kItems];
  __shared__ __align__(16) unsigned char response[16];
  __shared__ __align__(8) uint64_t item_wanted, asked;
  __shared__ int gave_up;    // a wait has run out
  __shared__ int left[4];    // the loader's place in its ring, and how often it loaded each Q tile, at its end
  __shared__ int odd_v;      // warp 2 has set elements of V to zero that are not finite
  __shared__ int stored[8];  // then: items whose rows each softmax warp has stored
  __shared__ __align__(8) uint64_t item_full[kItems], item_empty[kItems];
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  unsigned char* q_tiles = smem;                        // [2]
  unsigned char* kv_tiles = smem + 2 * C::kQBytes;   // [kStages]
  uint64_t* bars = reinterpret_cast<uint64_t*>(kv_tiles + C::kStages * C::kKvBytes);
  uint64_t* kv_full = bars;                    // [kStages]
  uint64_t* kv_empty = kv_full + C::kStages;   // [kStages]
  uint64_t* q_full = kv_empty + C::kStages;    // [2]
  uint64_t* q_empty = q_full + 2;              // [2]
  uint64_t* s_full = q_empty + 2;              // [2] scores ready (and all earlier products done)
  uint64_t* p_full = s_full + 2;               // [2 tiles][kParts] weights written (and the output rescaled)
  uint64_t* o_full = p_full + 2 * C::kParts;   // [2] output complete
  uint64_t* o_empty = o_full + 2;              // [2] output read
  uint64_t* v_landed = o_empty + 2;            // a V tile with keys that some row does not see is there
  uint64_t* v_fixed = v_landed + 1;            // and only what may be multiplied is left of them
  uint64_t* done = v_fixed + 1;                // every MMA has completed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  if (tid == 0) {
    gave_up = odd_v = 0;
    for (int i = 0; i < 8; ++i) stored[i] = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 1);
      mbar_init(&q_empty[x], 1);
      mbar_init(&s_full[x], 1);
      for (int h = 0; h < C::kParts; ++h) mbar_init(&p_full[C::kParts * x + h], 4);  // one arrival per warp
      mbar_init(&o_full[x], 1);
      mbar_init(&o_empty[x], 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 11);
    }
    mbar_init(&item_wanted, 1);
    mbar_init(&asked, 1);
    mbar_init(v_landed, 1);
    mbar_init(v_fixed, 1);
    mbar_init(done, 1);
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Item w;
  // The next item as warp 3 found it, for a whole warp; false past the last one or after a wait that gave up.
  auto next_item = [&](int it, bool& ok, Item& w) {
    const int slot = it % kItems;
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspend(&item_full[slot], (uint32_t)((it / kItems) & 1), p.err, p.wait_ns));
    if (!ok) return false;
    w = items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[slot]);
    return w.there != 0;
  };

  if (warp < 4) {
    regs_down<C::kOtherRegs>();
    if (warp == 0) {
      // ---- TMA: Q tiles, then K and V tiles of each step, through one ring ------------------
      const int half_tok = BM / p.pack;
      int q_use[2] = {0, 0};
      Ring ring;
      bool ok = true;
      auto load_kv = [&](const CUtensorMap* map, int kv_row) {
        if (ring.round) ok = mbar_wait_suspend(&kv_empty[ring.slot], ring.phase() ^ 1u, p.err, p.wait_ns);
        if (!ok) return;
        mbar_arrive_expect_tx(&kv_full[ring.slot], C::kKvBytes);
        for (int c = 0; c < C::kBoxes; ++c)
          tma_load_3d(kv_tiles + ring.slot * C::kKvBytes + c * C::kKvBox, map, 64 * c, w.kvh, kv_row,
                      &kv_full[ring.slot]);
        ring.next(C::kStages);
      };
      for (int it = 0; next_item(it, ok, w); ++it) {
        if (lane == 0) {
          const int n = max(w.n[0], w.n[1]);
          auto load_q = [&](int x) {
            if (!w.n[x] || !ok) return;
            if (q_use[x] > 0) ok = mbar_wait_suspend(&q_empty[x], (uint32_t)((q_use[x] - 1) & 1), p.err, p.wait_ns);
            if (!ok) return;
            ++q_use[x];
            mbar_arrive_expect_tx(&q_full[x], C::kQBytes);
            for (int c = 0; c < C::kBoxes; ++c)
              tma_load_3d(q_tiles + x * C::kQBytes + c * C::kQBox, &tm_q, 64 * c, w.h0,
                          w.q0 + w.tok0 + x * half_tok, &q_full[x]);
          };
          load_q(0);
          if (n == 0) mbar_arrive(&item_wanted);
          for (int j = 0; j < n && ok; ++j) {
            if (j == max(0, n - kAhead)) mbar_arrive(&item_wanted);
            load_kv(&tm_k, w.k0 + j * BN);
            if (j == 0) load_q(1);
            if (ok) load_kv(&tm_v, w.k0 + j * BN);
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      }
      if (lane == 0) {
        left[0] = ring.slot;
        left[1] = ring.round;
        left[2] = q_use[0];
        left[3] = q_use[1];
      }
      if (!ok) gave_up = 1;
    } else if (warp == 1) {
      // ---- MMA issuer: one lane, with nothing but waits and issues in its step -----------------
      constexpr uint32_t idesc_s = instr_desc_f16(kBf16, BM, BN);
      constexpr uint32_t idesc_o = instr_desc_f16(kBf16, BM, DP) | (1u << 16);  // B is MN-major
      constexpr uint32_t kQ16 = C::kQBytes >> 4, kQBox16 = C::kQBox >> 4, kKv16 = C::kKvBytes >> 4, kKvBox16 = C::kKvBox >> 4;
      // descriptors of the first Q tile, and of the ring's first tile as K and as V
      const uint64_t q_desc = smem_desc_sw128(q_tiles), kv_desc = smem_desc_sw128(kv_tiles),
                     v_desc = smem_desc_mn(kv_tiles, C::kKvBox);
      const bool leader = elect_one();
      const int leader_lane = __ffs(__ballot_sync(0xffffffffu, leader)) - 1;
      uint32_t q_ph[2] = {0, 0}, p_ph[2] = {0, 0}, o_ph[2] = {1, 1}, fix_ph = 0;
      Ring ring;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t phase) {
        if (ok) ok = mbar_wait_suspend(bar, phase, p.err, p.wait_ns);
      };
      auto scores = [&](int x, int slot) {  // S_x = Q_x K^T
#pragma unroll
        for (int c = 0; c < C::kBoxes; ++c)
          umma4_ss(tmem + x * BN, q_desc + (uint64_t)(x * kQ16 + c * kQBox16),
                   kv_desc + (uint64_t)(slot * kKv16 + c * kKvBox16), idesc_s, c != 0);
        umma_commit(&s_full[x]);
      };
      for (int it = 0; next_item(it, ok, w); ++it) {
        const int n = max(w.n[0], w.n[1]);
        const int first_fixed = seen_by_all(p, w) / BN;  // the first step with keys that some row does not see
        bool told = false;                               // warp 2 has been told of this step's V
        if (n > 0 && leader) {
          int kslot = ring.slot;
          wait(&kv_full[kslot], ring.phase());
          ring.next(C::kStages);
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (w.n[x]) {
              wait(&q_full[x], q_ph[x]);
              q_ph[x] ^= 1;
              if (!ok) break;
              tc_fence_after();
              scores(x, kslot);
              if (w.n[x] == 1) umma_commit(&q_empty[x]);
            }
          // A tile is given back only if its products were issued: after a wait that gave up its copy may still
          // be in flight, and the loader must not arm its barrier again.
          if (ok) umma_commit(&kv_empty[kslot]);
          for (int j = 0; j < n && ok; ++j) {
            const int vslot = ring.slot;
            wait(&kv_full[vslot], ring.phase());
            ring.next(C::kStages);
            if (j >= first_fixed && !told && ok) mbar_arrive(v_landed);
            kslot = ring.slot;
            if (j + 1 < n) {
              wait(&kv_full[kslot], ring.phase());
              ring.next(C::kStages);
            }
            if (j >= first_fixed) {
              wait(v_fixed, fix_ph);
              fix_ph ^= 1;
            }
            told = j + 1 < n && j + 1 >= first_fixed && ok && mbar_test(&kv_full[ring.slot], ring.phase());
            if (told) mbar_arrive(v_landed);
            const uint64_t dv = v_desc + (uint64_t)(vslot * kKv16);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (j >= w.n[x] || !ok) continue;
              if (j == 0) {
                wait(&o_empty[x], o_ph[x]);  // passes at once the first time
                o_ph[x] ^= 1;
              }
              // O_x += P_x V, each 64 of the keys when their weights are there
#pragma unroll
              for (int h = 0; h < C::kParts; ++h) {
                wait(&p_full[C::kParts * x + h], p_ph[x]);
                if (!ok) break;
                tc_fence_after();
                umma4_ts(tmem + C::kO + x * DP, tmem + x * BN + 32 * h, dv + h * 4 * 128, idesc_o, j != 0 || h);
              }
              p_ph[x] ^= 1;
              if (!ok) continue;
              if (j + 1 < w.n[x]) {
                scores(x, kslot);
                if (j + 2 == w.n[x]) umma_commit(&q_empty[x]);
              } else {
                umma_commit(&o_full[x]);
              }
            }
            if (ok) {
              umma_commit(&kv_empty[vslot]);
              if (j + 1 < n) umma_commit(&kv_empty[kslot]);
            }
          }
        }
        __syncwarp();
        ok = __shfl_sync(0xffffffffu, (int)ok, leader_lane) != 0;
      }
      if (!ok) gave_up = 1;
      if (leader) umma_commit(done);
      __syncwarp();
      (void)mbar_wait_suspend(done, 0, p.err);
      __syncwarp();
    } else if (warp == 2) {
      // ---- V of keys that some row does not see: zero where it must not be multiplied -------------
      // (told by the MMA lane that the tile is there: this warp does not see every phase of the ring)
      Ring ring;
      uint32_t ph = 0;
      bool ok = true;
      for (int it = 0; next_item(it, ok, w); ++it) {
        const int n = max(w.n[0], w.n[1]), all = seen_by_all(p, w);
        int passed = 0;    // tiles of this item
        int odd = n;       // the first step in which something was set to zero that is not finite
        for (int j = all / BN; j < n; ++j) {
          ok = __all_sync(0xffffffffu, mbar_wait_suspend(v_landed, ph, p.err, p.wait_ns));
          if (!ok) break;
          ph ^= 1;
          ring.skip(2 * j + 1 - passed, C::kStages);
          passed = 2 * j + 1;
          (void)mbar_test(&kv_full[ring.slot], ring.phase());  // complete: its copy is visible here too
          unsigned char* vt = kv_tiles + ring.slot * C::kKvBytes;
          // rows [lo, hi): seen by some rows of the CTA; from hi on: past the last key
          const int hi = min(BN, w.Tk - j * BN), lo = p.causal ? max(0, min(hi, all - j * BN)) : hi;
#pragma unroll
          for (int c = 0; c < C::kBoxes; ++c) {
            uint4* rows = reinterpret_cast<uint4*>(vt + c * C::kKvBox);
            uint32_t acc[4] = {0, 0, 0, 0};
#pragma unroll 1
            for (int i = lo * 8 + lane; i < hi * 8; i += 128)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (i + 32 * k < hi * 8) acc[k] = odd_acc<T>(rows[i + 32 * k], acc[k]);
            uint32_t any = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) any |= acc[k] & 0x7FFF7FFFu;  // 0 + x * 0: zero, or NaN
            if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll 1
              for (int i = lo * 8 + lane; i < hi * 8; i += 32) {
                const uint4 v = rows[i];
                rows[i] = make_uint4(finite_only<T>(v.x), finite_only<T>(v.y), finite_only<T>(v.z), finite_only<T>(v.w));
              }
              odd = min(odd, j);
              odd_v = 1;
            }
            for (int i = hi * 8 + lane; i < BN * 8; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(v_fixed);
        }
        if (!ok) break;
        ring.skip(2 * n - passed, C::kStages);
        if (odd < n) {
          // Once the rows are stored, what was taken out goes to those that see its key: an infinity or a
          // NaN, to which the finite rest adds nothing.  (Softmax warps doing so for their own rows cost
          // 3 % of the 8 x 1500's time, in which nothing is taken out: their loop is short of registers.)
          const unsigned long long t0 = global_ns();
          for (bool there = false; !there;) {
            int items_done = it + 1;
            if (lane < 8 && (lane < 4 ? w.n[0] : w.n[1]) > odd)  // (the other tile sees none of it)
              asm volatile("ld.acquire.cta.shared::cta.b32 %0, [%1];" : "=r"(items_done) : "r"(smem_addr(&stored[lane])) : "memory");
            there = __all_sync(0xffffffffu, items_done > it);
            if (!there && __any_sync(0xffffffffu, global_ns() - t0 > p.wait_ns)) {
              set_error(p.err, SPD_DEVERR_TIMEOUT);
              ok = false;
              break;
            }
          }
          if (!ok) break;
          // A lane takes every 32nd dimension; along the rows the keys seen only grow.
          const int last = min(w.Tq, w.tok0 + 2 * BM / p.pack), cleared = min(w.Tk, n * BN);
#pragma unroll 1
          for (int d = lane; d < p.D; d += 32) {
            const T* v = reinterpret_cast<const T*>(p.v) + w.k0 * p.v_st + w.kvh * p.v_sh + d;
            float sum = 0.f;
            int key = all;
#pragma unroll 1
            for (int t = w.tok0; t < last; ++t) {
#pragma unroll 1
              for (; key < min(cleared, t + 1 + w.Tk - w.Tq); ++key) {
                const float f = Elem<T>::to_f(v[key * p.v_st]);
                if (!(fabsf(f) < INFINITY)) sum += f;
              }
              if (sum == 0.f) continue;
              T* o = reinterpret_cast<T*>(p.out) + ((long long)(w.q0 + t) * p.Hq + w.h0) * p.D + d;
#pragma unroll 1
              for (int h = 0; h < p.pack; ++h, o += p.D) *o = Elem<T>::from_f(Elem<T>::to_f(*o) + sum);
            }
          }
          __syncwarp();
        }
      }
      if (!ok) gave_up = 1;
    } else {
      // ---- this CTA's items, found ahead of their use: its own, then those of CTAs that have not
      // started, whose launch it calls off
      bool ok = true;
      int index = (int)blockIdx.x;
      for (int it = 0; ok; ++it) {
        const int slot = it % kItems;
        if (it > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait_suspend(&item_wanted, (uint32_t)((it - 1) & 1), p.err, p.wait_ns));
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&asked, 16);
            ask_for_cta(response, &asked);
          }
          ok = __all_sync(0xffffffffu, mbar_wait_suspend(&asked, (uint32_t)((it - 1) & 1), p.err, p.wait_ns));
          if (!ok) {  // let the answer land before the CTA can exit
            (void)mbar_wait_suspend(&asked, (uint32_t)((it - 1) & 1), nullptr);
            break;
          }
          index = called_off(response);
          fence_proxy_async_smem();  // read before the next answer is written
          __syncwarp();
        }
        w.there = index >= 0 && find_item<BN>(p, index, w);
        if (it >= kItems)
          ok = __all_sync(0xffffffffu, mbar_wait_suspend(&item_empty[slot], (uint32_t)((it / kItems - 1) & 1), p.err, p.wait_ns));
        if (!ok) break;
        if (lane == 0) {
          items[slot] = w;
          mbar_arrive(&item_full[slot]);
        }
        if (!w.there) break;
      }
      if (!ok) gave_up = 1;
    }
  } else {
    // ---- softmax and epilogue of tile x: thread = query row = TMEM lane --------------------
    regs_up<C::kSoftmaxRegs>();
    const int x = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + x * BN, o_col = tmem + lanes + C::kO + x * DP;
    const int half_tok = BM / p.pack;
    int s_use = 0, o_use = 0;
    bool ok = true;
    for (int it = 0; next_item(it, ok, w); ++it) {
      const int tok = w.tok0 + x * half_tok + row / p.pack;  // of this row, within the sequence
      const int first = w.tok0 + x * half_tok;
      const int off = w.Tk - w.Tq;
      // keys this row sees, and the fewest any row of the tile sees
      const int limit = p.causal ? min(w.Tk, tok + 1 + off) : w.Tk;
      const int least = p.causal ? min(w.Tk, first + 1 + off) : w.Tk;
      const bool live = tok < w.Tq;
      float m = -INFINITY, l = 0.f;
      const int n = w.n[x];
      for (int j = 0; j < n; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait_suspend(&s_full[x], (uint32_t)(s_use & 1), p.err, p.wait_ns));
        ++s_use;
        if (!ok) break;
        tc_fence_after();
        constexpr int kHeld = BN == 128 ? 128 : 32;  // scores held in registers at a time
        uint32_t s[kHeld];
        const int base = j * BN, seen = limit - base;
        const bool edge = base + BN > least;  // some row of the tile does not see all of these keys
        float mx4[4];
        if constexpr (BN == 128) {
          tmem_ld32_nowait(s_col, s);
          tmem_ld32_nowait(s_col + 32, s + 32);
          tmem_ld_wait(s);
          tmem_ld_wait(s + 32);
          tmem_ld32_nowait(s_col + 64, s + 64);
          tmem_ld32_nowait(s_col + 96, s + 96);
          if (edge) {
            tmem_ld_wait(s + 64);
            tmem_ld_wait(s + 96);
            mask<BN>(s, seen);
          }
          max4<64, true>(s, mx4);  // while the other half is on its way
          if (!edge) {
            tmem_ld_wait(s + 64);
            tmem_ld_wait(s + 96);
          }
          max4<64, false>(s + 64, mx4);
        } else {
#pragma unroll
          for (int c = 0; c < BN; c += 32) {
            tmem_ld32_nowait(s_col + c, s);
            tmem_ld_wait(s);
            if (edge) mask<32>(s, seen - c);
            if (c == 0) max4<32, true>(s, mx4);
            else max4<32, false>(s, mx4);
          }
          tmem_ld32_nowait(s_col, s);
        }
        const float mx = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * p.scale_log2;
        // Also for a NaN and for infinite scores, which only the exact exponentials treat as they are.  Rows
        // past the sequence's end have no say: what they hold changes no rounding of the others.
        const bool raise = live && !(mx < m + kLazy);
        bool exact = edge;
        if (__any_sync(0xffffffffu, raise)) {
          exact |= __any_sync(0xffffffffu, live && !(fabsf(mx) < INFINITY));
          const float mn = fmaxf(m, mx);
          const float f = m == mn ? 1.f : ex2_approx(m - mn);
          m = mn;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              uint32_t o[32];
              tmem_ld32_nowait(o_col + c, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st32(o_col + c, o);
            }
          }
        }
        const float mm = m == -INFINITY ? 0.f : m;
        const f32x2 c2 = pair(p.scale_log2, p.scale_log2), nm2 = pair(-mm, -mm);
        f32x2 sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
        // 64 keys at a time, handed to the tensor cores when they are written
#pragma unroll
        for (int h = 0; h < C::kParts; ++h) {
          
          uint32_t pk[kHeld == 128 ? 32 : 16];
          if constexpr (BN == 128) {
            if (exact) weights<T, true, 32>(s + 64 * h, c2, nm2, pk, sum);
            else weights<T, false, 32>(s + 64 * h, c2, nm2, pk, sum);
            tmem_st32(s_col + 32 * h, pk);
          } else {
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
              tmem_ld_wait(s);
              if (edge) mask<32>(s, seen - c);
              if (exact) weights<T, true, 16>(s, c2, nm2, pk, sum);
              else weights<T, false, 16>(s, c2, nm2, pk, sum);
              if (c + 32 < BN) tmem_ld32_nowait(s_col + c + 32, s);
              tmem_st16(s_col + c / 2, pk);
            }
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[C::kParts * x + h]);
        }
        const float2 t2 = unpair(add2(sum[0], sum[1]));
        l += t2.x + t2.y;
      }
      if (!ok) break;
      T* out = reinterpret_cast<T*>(p.out) +
               ((long long)(w.q0 + tok) * p.Hq + w.h0 + row % p.pack) * p.D;
      if (n > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait_suspend(&o_full[x], (uint32_t)(o_use & 1), p.err, p.wait_ns));
        ++o_use;
        if (!ok) break;
        tc_fence_after();
        const float r = l != 0.f ? 1.f / l : 0.f;  // a row that sees no key: zeros
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32_nowait(o_col + c, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (live && c + k < p.D) {
              uint4 v;
              v.x = pack2<T>(__uint_as_float(o[k]) * r, __uint_as_float(o[k + 1]) * r);
              v.y = pack2<T>(__uint_as_float(o[k + 2]) * r, __uint_as_float(o[k + 3]) * r);
              v.z = pack2<T>(__uint_as_float(o[k + 4]) * r, __uint_as_float(o[k + 5]) * r);
              v.w = pack2<T>(__uint_as_float(o[k + 6]) * r, __uint_as_float(o[k + 7]) * r);
              *reinterpret_cast<uint4*>(out + c + k) = v;
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&o_empty[x]);
          if (p.causal && *(volatile int*)&odd_v)  // set before this item's products were issued, if by it
            asm volatile("st.release.cta.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&stored[warp - 4])), "r"(it + 1)
                         : "memory");
        }
      } else if (live) {
        for (int c = 0; c < p.D; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(0, 0, 0, 0);
      }
    }
    if (!ok) gave_up = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (gave_up) {
    // Some warp gave up, perhaps on a copy that is still in flight: all land before the CTA exits.
    if (tid == 0) {
      Ring ring{left[0], left[1]};
      for (int k = 0; k < C::kStages; ++k) {
        ring.back(C::kStages);
        if (ring.round >= 0) (void)mbar_wait_suspend(&kv_full[ring.slot], ring.phase(), nullptr);
      }
      for (int x = 0; x < 2; ++x)
        if (left[2 + x]) (void)mbar_wait_suspend(&q_full[x], (uint32_t)((left[2 + x] - 1) & 1), nullptr);
    }
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::kTmemCols);
}

// Without a key anywhere: zeros in the rows that belong to a sequence.
__global__ void no_keys_kernel(const PromptParams p) {
  const int first = max(0, min(p.Nq, p.cu_q[0])), last = max(first, min(p.Nq, p.cu_q[p.B]));
  const long long row = (long long)p.Hq * p.D / 8;  // in 16 bytes
  uint4* out = reinterpret_cast<uint4*>(p.out);
  for (long long i = first * row + (long long)blockIdx.x * blockDim.x + threadIdx.x; i < last * row;
       i += (long long)gridDim.x * blockDim.x)
    out[i] = make_uint4(0, 0, 0, 0);
}

struct PromptTensors {
  const void *q, *k, *v;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh;
};

// [tokens][heads][D] of 16-bit elements with any token and head strides, box [rows][heads][64].
static bool make_map3(CUtensorMap* map, const void* base, int D, int heads, int tokens, long long sh, long long st,
                      int box_heads, int box_tokens, bool bf16) {
  auto enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)sh * 2, (cuuint64_t)st * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
             dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, int BN>
static int launch(PromptParams p, const PromptTensors& t, long long items, int sms, cudaStream_t st) {
  using C = Cfg<DP, BN>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap tq, tk, tv;
  if (!make_map3(&tq, t.q, p.D, p.Hq, p.Nq, t.q_sh, t.q_st, p.pack, BM / p.pack, kBf16) ||
      !make_map3(&tk, t.k, p.D, p.Hkv, p.Nk, t.k_sh, t.k_st, 1, BN, kBf16) ||
      !make_map3(&tv, t.v, p.D, p.Hkv, p.Nk, t.v_sh, t.v_st, 1, BN, kBf16))
    return SPD_ERR_CUDA;
  p.ranked = items > (long long)sms * C::kCtas;
  p.v = t.v;
  p.v_st = t.v_st;
  p.v_sh = t.v_sh;
  if (!allow_smem<prompt_attn_kernel<T, DP, BN>>(C::kSmem)) return SPD_ERR_CUDA;
  static const bool enough = [] {  // a warpgroup that asks for more registers than the CTA has would wait for good
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, prompt_attn_kernel<T, DP, BN>) == cudaSuccess && a.numRegs * kThreads >= C::kAllRegs;
  }();
  if (!enough) return SPD_ERR_CUDA;
  prompt_attn_kernel<T, DP, BN><<<(unsigned)items, kThreads, C::kSmem, st>>>(tq, tk, tv, p);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace pa

int prompt_attn_launch(PromptParams p, const void* q, const void* k, const void* v, long long q_st, long long q_sh,
                       long long k_st, long long k_sh, long long v_st, long long v_sh, int dtype, int sms,
                       cudaStream_t st) {
  using namespace pa;
  const bool bf16 = dtype == SPD_BF16;
  if (p.Nk == 0) {
    const long long blocks = ((long long)p.Nq * p.Hq * p.D / 8 + 255) / 256;
    no_keys_kernel<<<(unsigned)std::min(blocks, 8ll * sms), 256, 0, st>>>(p);
    return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
  }
  // heads of one group in a tile: the largest power of two that divides G (up to 128)
  const int G = p.Hq / p.Hkv;
  p.pack = G & -G;
  if (p.pack > BM) p.pack = BM;
  const int tokens = 2 * BM / p.pack;
  const long long items = ((long long)p.Nq / tokens + p.B) * (p.Hq / p.pack);  // at most
  if (items > 0x7fffffffll) return SPD_ERR_UNSUPPORTED;
  const PromptTensors t{q, k, v, q_st, q_sh, k_st, k_sh, v_st, v_sh};
  auto by_d = [&](auto tag) -> int {
    using T = decltype(tag);
    if (p.D > 64) return launch<T, 128, 128>(p, t, items, sms, st);
    // two CTAs an SM with 64 keys a step, unless there is no second item for any SM (both measured above)
    return items <= sms ? launch<T, 64, 128>(p, t, items, sms, st) : launch<T, 64, 64>(p, t, items, sms, st);
  };
  return bf16 ? by_d(__nv_bfloat16{}) : by_d(__half{});
}

}  // namespace spd
