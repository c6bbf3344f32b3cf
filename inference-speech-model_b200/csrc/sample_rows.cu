// sample_rows.cu — a token a row by temperature, top-k, top-p and min-p from a given random number, and its
// log-probability.  With a row's values x (suppressed columns -inf), their largest m, w = exp((x - m) / t):
//   top-k leaves the k largest (equal ones by their place), top-p of those, in that order, the ones before which less
//   than p of their weight lies, min-p the ones with x >= m + t log(min_p); the token is the first column, by
//   its place, at which the weight left so far passes u times all of it.
//
// What bounds it: a row is read once from memory, 2 or 4 bytes a column, and again from shared memory by each later pass.
// What takes the time is that a row's passes follow one another, with clusters' barriers and remote reads between them, in the
// few rows that the SMs hold at once (37 of the last case below: three waves of them).  The passes' instructions, some 60
// a column in all, would be 31 of its 224 us.  Rows are not sorted:
// * A cluster of up to 8 CTAs shares a row.  A cut (the k-th largest, or the value at which the weight reaches p) is
//   found by histograms.  The first counts columns by their distance from m (one atomic a column).  For the k-th largest
//   the cut lies in one of its bins.  For p each bin's weight is known to within 2 %, and
//   their sums, by the law of large numbers, to some hundred-thousandths, so the cut nearly always lies in one or two; the
//   next pass adds up the weights above, in and below these, and only the columns in them enter a histogram of weights.
//   (If it lies elsewhere, which the sums show, the bins are taken anew from what is certain.  At once from that, a cut
//   far down a flat row had a tenth of the columns to put in their bins.)  Later passes look at the order-preserving
//   integers of the values in the bin that holds the cut, until a bin holds one value.  Equal values that the cut
//   divides count by their place.
// * Where 512 columns or fewer are left, above the cut and in its bins, the first CTA gets these and puts them in order, by
//   their ranks: cuts and the draw are then sums before a thread.
// * Every sum of weights is an integer (units of 2^-44 of the largest weight), so no order of atomics or threads changes a
//   result, and cumulative sums are exact in their weights.
// * Weights are fp32 polynomials of an argument in two parts, good to 2^-26.4.  A decision that an error of 2^-25.4 of the
//   whole could turn is taken again with weights in fp64 (one row in a hundred where two hundred thousand columns
//   weigh alike, else next to none), so that the token is the one that fp64 arithmetic gives.  (With 2^-23.8, and a fifth
//   fewer instructions a weight, it was one row in twenty, and the slowest row took twice as long.)
// * A CTA's columns lie in its shared memory, and what is known of the row beside them: passes are functions that are
//   called, so that none holds another's registers.  (In one function the state went to local memory, whose traffic
//   was twice that of the columns: 87 us in place of 64 for the second case below, then.)
// * The log-probability's sum is fp32, of special-function exponentials: some 10^-7 off.  No decision uses it.
// Measured on a B200, in CUDA graphs: one fp32 row of 51,865 columns by top-p 33 us (29 to 37, by the row), 64 fp16 rows of
// them by all settings 47, 192 bf16 rows of 128,257 by top-k 100, 96 fp32 rows of 200,019 by top-p 224 (their reading alone: 0.04, 1.0, 7.5, 12).  A
// row's CTAs spend some 50,000 cycles on a cut: 4,500 until the columns are there, 6,000 to 40,000 for passes, 9,500 for
// each barrier-bound search of a histogram.
#include "spd_params.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace spd {
namespace pick {
namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kFirst = 2048;      // bins of the first histogram (counts)
constexpr int kBins = 512;        // of the later ones (counts and weights)
constexpr int kList = kThreads;   // columns that one CTA puts in order
constexpr int kMaxChunks = 256;   // of a CTA's columns
constexpr int kCtas = 8;          // of a cluster, at most
constexpr int kScale = 44;        // a weight of 1 is 2^44: sums of 2^19 columns fit in 64 bits

// a value's place among all values: the larger, the larger (values of 16 bits leave low bits unused)
template <typename T> constexpr int unused_bits() { return sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16; }
template <typename T> __device__ __forceinline__ unsigned place_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);  // (-0 is 0)
  return (b & 0x80000000u ? ~b : b | 0x80000000u) >> unused_bits<T>();
}
template <typename T> __device__ __forceinline__ float value_of(unsigned place) {  // of a place that some value has
  const unsigned k = place << unused_bits<T>();
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~(k | ((1u << unused_bits<T>()) - 1u)));
}

// What CTAs of a cluster tell one another: written before, read after a cluster barrier.
struct Told {
  float mx, z;
  int count, first, last;
  u64 sum, inside, below;
  float least, most;
};
// The bin that holds a cut, and what lies above it.
struct Cut {
  int bin;  // -1: none, all is left
  int above, inside;
  u64 sum_above, sum_inside;
  int open;  // the decision could be another with exact weights
};

// What a pass over the row does with its columns.
enum Pass { kMax, kSeek, kCount, kWeigh, kRefine, kSum, kGather, kDone };

// What is known of the row: the same in all CTAs of its cluster but for the first line.
struct State {
  int rank, first_column, vectors, chunk, chunks;
  int ctas, k;
  float t, top_p, min_p;
  double u;
  Pass pass;
  int token;
  bool by_count, exact, z_due;
  bool sure, missed;      // the cut's bins are taken from certain bounds; they were not, and did not hold it
  float m, xmin, hi, lo;  // the largest value, the least that min-p leaves, 2 log2(e) / t in two parts
  float xt, xt0, xt_k;    // what is left: values above xt, and the first `ties` columns that have it;
  int ties, ties0, ties_k;  // as the cut under way found it; as top-k left it
  // the cut under way: bins [first, last] of the first histogram, places [from, to] among them, `shift` bits of a bin's
  int k_left, first, last, shift;
  unsigned from, to;
  float inv;
  u64 whole, above;
  double target;
};
// A CTA's columns follow it: vectors of 16 bytes that lie on 16-byte boundaries of the row (so the first may begin before
// it), in chunks of a warp, 32 vectors at a time.  Suppressed columns, and those that there are not, hold -inf.
struct Shared {
  State st;
  Cut cut;
  Told told[4];
  float z[kWarps], floats[3][kWarps];
  int counts[4][kWarps];
  int listed;  // columns in `list`
  u64 sums[3][kWarps];
  union {  // the first histogram, and what comes after it: the later ones and the chunks' sums, or the columns that are left
    unsigned first_count[kFirst];
    u64 list[2][kList];  // place << 32 | ~column; and in their order
    struct {
      u64 chunk_sum[kMaxChunks];
      int chunk_ties[kMaxChunks];
      unsigned count[kBins], low[kBins], high[kBins];
    };
  };
};
constexpr size_t kSharedBytes = (sizeof(Shared) + 127) / 128 * 128;
constexpr size_t kMostBytes = 226 * 1024, kGoodBytes = 112 * 1024;  // of a CTA's shared memory
extern __shared__ __align__(128) unsigned char shared_bytes[];
__device__ __forceinline__ Shared& shared() { return *reinterpret_cast<Shared*>(shared_bytes); }

// The weight of a value, in units of 2^-44: 2^y with y = (x - m) log2(e) / t = n + f, |f| <= 1/2.
// In fp64: the Taylor series of 2^f to the 12th power (2e-16).
__device__ __noinline__ u64 exact_weight(double y) {
  const double n = fmax(rint(y), -100.0), f = fmax(y - n, -1.0) * 0.69314718055994530942;
  double q = 1.0 / 479001600.0;
  q = fma(q, f, 1.0 / 39916800.0);
  q = fma(q, f, 1.0 / 3628800.0);
  q = fma(q, f, 1.0 / 362880.0);
  q = fma(q, f, 1.0 / 40320.0);
  q = fma(q, f, 1.0 / 5040.0);
  q = fma(q, f, 1.0 / 720.0);
  q = fma(q, f, 1.0 / 120.0);
  q = fma(q, f, 1.0 / 24.0);
  q = fma(q, f, 1.0 / 6.0);
  q = fma(q, f, 0.5);
  q = fma(q, f, 1.0);
  q = fma(q, f, 1.0);
  // in units of 2^-60, rounded, and then to their place
  const u64 bits = (u64)__double2ll_rn(q * 0x1p60);
  const int down = 60 - kScale - (int)n;
  return down < 63 ? (bits + (1ull << (down - 1))) >> down : 0;
}
template <typename T> struct Weight {
  float m, hi, lo;  // the largest value, and 2 log2(e) / t in two parts
  double temperature;
  bool exact;
  __device__ __forceinline__ explicit Weight(const State& st)
      : m(st.m), hi(st.hi), lo(st.lo), temperature(st.t), exact(st.exact) {}
  __device__ __forceinline__ u64 operator()(float x) const { return exact ? of<true>(x) : of<false>(x); }
  template <bool EXACT> __device__ __forceinline__ u64 of(float x) const {
    if (EXACT) return exact_weight(((double)x - (double)m) / temperature * 1.4426950408889634074);
    const float h = 0.5f * m, d = fmaf(0.5f, x, -h);  // <= 0: half the distance, which fits where the whole one would not
    // y = n + f + rest: f is exact (no contraction of its product), the rest what roundings left over
    const float y = __fmul_rn(d, hi), n = fmaxf(rintf(y), -63.f), f = fmaxf(y - n, -1.f);
    // (what the subtraction rounds off matters for 16-bit values too: of small ones beside m = 8 it is up to 2^-22)
    const float b = fmaf(-0.5f, x, d), a = d - b;
    const float rest = fmaf(fmaf(0.5f, x, -a) - (h + b), hi, fmaf(d, lo, fmaf(d, hi, -y)));
    // 2^f = 1 + f ln 2 + f^2 s(f), s a polynomial that interpolates (2^f - 1 - f ln 2) / f^2 at the Chebyshev nodes of
    // [-1/2, 1/2] (4e-10), and 2^rest = 1 + rest ln 2.  f ln 2 in two parts, and what is added to 1 in units of 2^-30.
    // Off by less than 2^-26.4 of itself (the half steps of s, f^2, the sum that holds the small terms, over 2^-1/2;
    // 2^-26.9 at the worst of 10^8 arguments) and a unit of 2^-44 that the shift drops.
    float s = fmaf(1.529094879515469e-05f, f, 0.00015453163359779865f);
    s = fmaf(s, f, 0.0013333521783351898f);
    s = fmaf(s, f, 0.009618083015084267f);
    s = fmaf(s, f, 0.05550410971045494f);
    s = fmaf(s, f, 0.24022650718688965f);
    constexpr float c = 0.6931471824645996f, c_rest = -1.9046542121259336e-09f;  // ln 2
    const float p = __fmul_rn(f, c), u = f * f, r = rest * c;
    const float low = fmaf(f, c_rest, fmaf(f, c, -p)) + fmaf(r, fmaf(u, s, p), r), t = fmaf(u, s, low);
    const unsigned bits = (1u << 30) + (unsigned)__float2int_rn(p * 0x1p30f) + (unsigned)__float2int_rn(t * 0x1p30f);
    return ((u64)bits << (kScale - 30)) >> -(int)n;
  }
};

template <typename V> __device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// (of 63 bits, 21 at a time: one instruction each in place of ten)
template <> __device__ __forceinline__ u64 warp_total<u64>(u64 v) {
  const unsigned low = (unsigned)v & 0x1fffffu, mid = (unsigned)(v >> 21) & 0x1fffffu, high = (unsigned)(v >> 42);
  return __reduce_add_sync(0xffffffffu, low) + ((u64)__reduce_add_sync(0xffffffffu, mid) << 21) +
         ((u64)__reduce_add_sync(0xffffffffu, high) << 42);
}
template <> __device__ __forceinline__ int warp_total<int>(int v) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)v); }
template <typename V> __device__ __forceinline__ V warp_inclusive(V v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

// What lies before this thread's v in the CTA, and the whole of it (slots: one a warp).
template <typename V> __device__ __forceinline__ V before_thread(V v, V* slots, V& whole) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const V incl = warp_inclusive(v);
  if (lane == 31) slots[warp] = incl;
  __syncthreads();
  const V of_warps = warp_inclusive(lane < kWarps ? slots[lane] : V(0));
  whole = __shfl_sync(0xffffffffu, of_warps, 31);
  const V before = __shfl_sync(0xffffffffu, of_warps, max(warp - 1, 0));
  return (warp ? before : V(0)) + incl - v;
}

// All CTAs of the cluster, and what they wrote before.
__device__ __forceinline__ void together(int ctas) {
  if (ctas > 1) cg::this_cluster().sync();
  else __syncthreads();
}
// The shared memory of CTA i.
__device__ __forceinline__ Shared& of_cta(int i) { return *cg::this_cluster().map_shared_rank(&shared(), i); }

// f(column, value) for the columns of this CTA, and g(chunk) after each chunk
template <typename T, typename F, typename G> __device__ __forceinline__ void each(F&& f, G&& g) {
  constexpr int E = 16 / sizeof(T);
  const State& st = shared().st;
  const uint4* at = reinterpret_cast<const uint4*>(shared_bytes + kSharedBytes);
  const int lane = threadIdx.x & 31, vectors = st.vectors, chunk = st.chunk, chunks = st.chunks, first = st.first_column;
#pragma unroll 1
  for (int ch = threadIdx.x >> 5; ch < chunks; ch += kWarps) {
    const int end = min(vectors, (ch + 1) * chunk);
#pragma unroll 1
    for (int j = ch * chunk + lane; j < end; j += 32) {
      const uint4 w = at[j];
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int k = 0; k < E; ++k) f(first + E * j + k, Elem<T>::to_f(e[k]));
    }
    __syncwarp();
    g(ch);
  }
}
struct Nothing {
  __device__ __forceinline__ void operator()(int) const {}
};
// The sum of exp(x - m), added up by the first pass that looks at the values again.
struct Z {
  float m, z = 0.f;
  bool due;
  __device__ __forceinline__ explicit Z(const State& st) : m(st.m), due(st.z_due) {}
  __device__ __forceinline__ void add(float v) {
    if (due) z += ex2_approx((v - m) * 1.4426950408889634f);
  }
  __device__ __forceinline__ void keep() {
    if (!due) return;
    z = warp_sum(z);
    if ((threadIdx.x & 31) == 0) shared().z[threadIdx.x >> 5] = z;
  }
};
// (half the distance: the whole one may be beyond fp32's range)
__device__ __forceinline__ int bin_of(float v, float m, float inv) {
  return (int)fminf(fmaf(-0.5f, v, 0.5f * m) * (2.f * inv), (float)(kFirst - 1));
}
__device__ __forceinline__ void put(int bin, unsigned n, u64 w) {
  Shared& sh = shared();
  atomicAdd(&sh.count[bin], n);
  if (w) {
    const unsigned l = (unsigned)w, old = atomicAdd(&sh.low[bin], l), h = (unsigned)(w >> 32) + (old + l < old);
    if (h) atomicAdd(&sh.high[bin], h);
  }
}
__device__ __forceinline__ void clear_bins() {
  Shared& sh = shared();
  for (int i = threadIdx.x; i < kBins; i += kThreads) sh.count[i] = sh.low[i] = sh.high[i] = 0;
  __syncthreads();
}
__device__ __forceinline__ int sub_of(unsigned place, const State& st) {
  return place >= st.from && place <= st.to ? (int)((st.to - place) >> st.shift) : -1;
}

// ---- passes ----------------------------------------------------------------------------------------
template <typename T> __device__ __noinline__ void pass_max() {
  float m = -INFINITY;
  each<T>([&](int, float v) { asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(v)); }, Nothing{});
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, m, o);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(w));
  }
  if ((threadIdx.x & 31) == 0) shared().floats[0][threadIdx.x >> 5] = m;
}
// the first column that has the largest value, or the first NaN
template <typename T> __device__ __noinline__ void pass_seek() {
  Z z(shared().st);
  const float m = z.m;
  int at = 0x7fffffff;
  each<T>([&](int c, float v) {
    z.add(v);
    if (v == m || v != v) at = min(at, max(c, 0));  // (a row without a finite value: its first column)
  }, Nothing{});
  z.keep();
  at = (int)__reduce_min_sync(0xffffffffu, (unsigned)at);
  if ((threadIdx.x & 31) == 0) shared().counts[0][threadIdx.x >> 5] = at;
}
// columns by their distance from the largest
template <typename T> __device__ __noinline__ void pass_count() {
  Shared& sh = shared();
  const float m = sh.st.m, inv = sh.st.inv, xt0 = sh.st.xt0;
  for (int i = threadIdx.x; i < kFirst; i += kThreads) sh.first_count[i] = 0;
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  if (!sh.st.by_count && xt0 > -INFINITY && sh.st.rank == 0 && threadIdx.x == 0)  // columns that have xt0 itself, by their number
    sh.first_count[bin_of(xt0, m, inv)] = (unsigned)sh.st.ties0;
  __syncthreads();
  each<T>([&](int, float v) {
    if (v > xt0) atomicAdd(&shared().first_count[bin_of(v, m, inv)], 1u);
  }, Nothing{});
}
// weights: above the cut's bins (chunk by chunk, too), in them (by their place) and below
template <typename T, bool EXACT> __device__ __noinline__ void pass_weigh() {
  Shared& sh = shared();
  const State& st = sh.st;
  const Weight<T> weight(st);
  const bool cut = st.top_p < 1.f;
  const float m = st.m, inv = st.inv, xt0 = st.xt0, xmin = st.xmin;
  const int first = cut ? st.first : kFirst, last = cut ? st.last : kFirst, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (cut) clear_bins();
  u64 all = 0, above = 0, inside = 0, mine = 0;
  if (cut && xt0 > -INFINITY && st.rank == 0 && threadIdx.x == 0) {  // columns that have xt0 itself, by their number
    const int bin = bin_of(xt0, m, inv);
    const u64 w = weight(xt0) * (u64)st.ties0;
    all = w;
    if (bin < first) {
      above = w;
    } else if (bin <= last) {
      inside = w;
      put(sub_of(place_of<T>(xt0), st), (unsigned)st.ties0, w);
    }
  }
  Z z(st);
  each<T>([&](int, float v) {
    z.add(v);
    const u64 w = v > xt0 ? weight.template of<EXACT>(v) : 0;
    const int bin = bin_of(v, m, inv);  // (the last one for -inf, which weighs nothing)
    all += w;
    above += bin < first ? w : 0;
    mine += bin < first && v >= xmin ? w : 0;
    if (bin >= first && bin <= last && v > xt0) {  // few
      inside += w;
      const int sub = sub_of(place_of<T>(v), shared().st);
      if (sub >= 0) put(sub, 1, w);
    }
  }, [&](int ch) {
    mine = warp_total(mine);
    if (lane == 0) shared().chunk_sum[ch] = mine;
    mine = 0;
  });
  z.keep();
  const u64 below = warp_total(all - above - inside);
  above = warp_total(above), inside = warp_total(inside);
  if (lane == 0) sh.sums[0][warp] = above, sh.sums[1][warp] = inside, sh.sums[2][warp] = below;
}
template <typename T> __device__ __noinline__ void pass_refine() {
  Shared& sh = shared();
  const State& st = sh.st;
  const Weight<T> weight(st);
  const float m = st.m, inv = st.inv, xt0 = st.xt0;
  const bool by_count = st.by_count;
  const int first = st.first, last = st.last, shift = st.shift;
  const unsigned from = st.from, to = st.to;
  clear_bins();
  auto look = [&](float v, unsigned n) {
    const unsigned place = place_of<T>(v);
    if (place < from || place > to) return;
    const int bin = bin_of(v, m, inv);
    if (bin >= first && bin <= last) put((int)((to - place) >> shift), n, by_count ? 0 : weight(v) * (u64)n);
  };
  if (!by_count && xt0 > -INFINITY && st.rank == 0 && threadIdx.x == 0) look(xt0, (unsigned)st.ties0);
  each<T>([&](int, float v) {
    if (v > xt0) look(v, 1);
  }, Nothing{});
}
// the columns that are left, or above and in the bins of the cut: they fit in one CTA's list
template <typename T> __device__ __noinline__ void pass_gather() {
  Shared& sh = shared();
  const State& st = sh.st;
  const Weight<T> weight(st);
  const bool by_count = st.by_count;
  const float m = st.m, inv = st.inv;
  const int last = st.last;
  u64 all = 0;
  Z z(st);
  each<T>([&](int c, float v) {
    z.add(v);
    if (!by_count) all += v > -INFINITY ? weight.template of<false>(v) : 0;
    if (bin_of(v, m, inv) > last || !(v > -INFINITY)) return;
    const int at = atomicAdd(&shared().listed, 1);
    if (at < kList) shared().list[0][at] = (u64)place_of<T>(v) << 32 | (unsigned)~c;
  }, Nothing{});
  z.keep();
  all = warp_total(all);
  if ((threadIdx.x & 31) == 0) sh.sums[0][threadIdx.x >> 5] = all;
}
// the chunks' sums completed by what is left of the cut's bins, and the columns that have xt itself
template <typename T> __device__ __noinline__ void pass_sum() {
  Shared& sh = shared();
  const State& st = sh.st;
  const Weight<T> weight(st);
  const float m = st.m, inv = st.inv, xt = st.xt, xmin = st.xmin;
  const int first = st.first, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  u64 mine = 0, all = 0;
  int n = 0, all_n = 0;
  each<T>([&](int, float v) {
    if (!(v >= xt && v >= xmin && v > -INFINITY)) return;
    if (v == xt) ++n;
    else if (first < kFirst && bin_of(v, m, inv) >= first) mine += weight(v);
  }, [&](int ch) {
    mine = warp_total(mine);
    n = (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
    mine += shared().chunk_sum[ch];
    __syncwarp();
    if (lane == 0) shared().chunk_sum[ch] = mine, shared().chunk_ties[ch] = n;
    all += mine, all_n += n;
    mine = 0, n = 0;
  });
  if (lane == 0) sh.sums[0][warp] = all, sh.counts[0][warp] = all_n;
}

// ---- what follows from them (thread 0 writes the state; every CTA of the cluster comes to the same) ---
__device__ __forceinline__ void begin_cut(State& st, bool by_count) {
  st.by_count = by_count;
  st.xt0 = st.xt;
  st.ties0 = st.ties;
  st.k_left = st.k;
  st.inv = (float)(kFirst - 1) / (by_count ? 32.f : 40.f * st.t);
  st.pass = kCount;
}
__device__ __forceinline__ void again_exactly(State& st) {
  st.exact = true;
  st.xt = st.xt_k;
  st.ties = st.ties_k;
  begin_cut(st, false);
  if (!(st.top_p < 1.f)) st.pass = kWeigh, st.first = kFirst;
}
// How far a sum and a target of it may be off: twice 2^-26.4 of the whole, and a unit for each column in both.
__device__ __forceinline__ double guard(const State& st, u64 whole) {
  return st.exact ? 0.0 : (double)whole * 0x1.84p-26 + 0x1p20;
}
// the largest value, and what comes first
__device__ __noinline__ void after_max() {
  Shared& sh = shared();
  State& st = sh.st;
  const int lane = threadIdx.x & 31;
  __syncthreads();
  float m = sh.floats[0][lane % kWarps];
  auto of_warp = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float w = __shfl_xor_sync(0xffffffffu, m, o);
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(w));
    }
  };
  of_warp();
  if (st.ctas > 1) {
    if (threadIdx.x == 0) sh.told[0].mx = m;
    together(st.ctas);
    m = lane < st.ctas ? of_cta(lane).told[0].mx : -INFINITY;
    of_warp();
  }
  if (threadIdx.x) return;
  const double per = 2.0 * 1.4426950408889634 / (double)st.t;
  st.m = m;
  st.hi = (float)per;
  st.lo = (float)(per - st.hi);
  bool pick_first = !(fabsf(m) < INFINITY) || !(st.t > 0.f);
  if (st.min_p > 0.f && !pick_first) {
    st.xmin = __double2float_ru((double)m + (double)st.t * log((double)st.min_p));
    pick_first = !(st.xmin <= m);
  }
  if (pick_first) st.pass = kSeek;
  else if (st.k > 0) begin_cut(st, true);
  else if (st.top_p < 1.f) begin_cut(st, false);
  else st.pass = kWeigh, st.first = kFirst;
}
__device__ __noinline__ void after_seek() {
  Shared& sh = shared();
  const int lane = threadIdx.x & 31;
  __syncthreads();
  int at = (int)__reduce_min_sync(0xffffffffu, (unsigned)sh.counts[0][lane % kWarps]);
  if (threadIdx.x == 0) sh.told[1].count = at;
  together(sh.st.ctas);
  at = (int)__reduce_min_sync(0xffffffffu, lane < sh.st.ctas ? (unsigned)of_cta(lane).told[1].count : 0x7fffffffu);
  if (threadIdx.x == 0) sh.st.token = at, sh.st.pass = kDone;
}
// The bins of the first histogram that hold the cut.  Each CTA looks at a share of them and tells the others.  (With every CTA
// reading all histograms and two barriers less, 96 rows of 200,019 took 273 us against 251, one of 51,865 34.4 against 32.3, then.)
template <typename T> __device__ __noinline__ void after_count() {
  Shared& sh = shared();
  State& st = sh.st;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = st.ctas, rank = st.rank, k_left = st.k_left;
  const bool by_count = st.by_count;
  together(C);
  // A thread has 4, 2 or 1 bins of the rank's share of them (or, of eight CTAs, every other thread one).  Their weights are
  // sums of most and least, or (not sure) in `least` of the middles and in `most` of the squares of these.
  const int share = kFirst / C, per = tid * max(1, share / kThreads) < share ? max(1, share / kThreads) : 0;
  const int at0 = rank * share + tid * per;
  constexpr float step = 1.4426950408889634f * 40.f / (kFirst - 1);  // of weights by a bin, as an exponent of 2
  auto most_of = [&](int bin) { return bin ? ex2_approx(-bin * step) * (1.f + 2e-5f) : 1.f; };
  const bool sure = st.sure;
  const float half = ex2_approx(-0.5f * step);  // the middle of a bin against its upper end
  auto least_at = [&](int bin) {
    return !sure ? most_of(bin) * half : bin + 1 == kFirst ? 0.f : most_of(bin + 1) * (1.f - 6e-5f);
  };
  auto most_at = [&](int bin) { return sure ? most_of(bin) : least_at(bin) * least_at(bin); };
  int n[4], all_n = 0;
  float least = 0.f, most = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    n[j] = 0;
    if (j < per) {
      unsigned c[kCtas];
#pragma unroll
      for (int i = 0; i < kCtas; ++i) c[i] = i < C ? of_cta(i).first_count[at0 + j] : 0;
#pragma unroll
      for (int i = 0; i < kCtas; ++i) n[j] += (int)c[i];
      all_n += n[j];
      most += n[j] * most_at(at0 + j);
      least += n[j] * least_at(at0 + j);
    }
  }
  int all;
  float all_least, all_most;
  int above_n = before_thread(all_n, sh.counts[0], all);
  float a_least = before_thread(least, sh.floats[0], all_least), a_most = before_thread(most, sh.floats[1], all_most);
  if (C > 1) {
    if (tid == 0) sh.told[1].count = all, sh.told[1].least = all_least, sh.told[1].most = all_most;
    together(C);
    const Told& o = of_cta(min(lane, C - 1)).told[1];
    const int o_n = lane < C ? o.count : 0;
    const float o_least = lane < C ? o.least : 0.f, o_most = lane < C ? o.most : 0.f;
    above_n += warp_total(lane < rank ? o_n : 0), a_least += warp_total(lane < rank ? o_least : 0.f);
    a_most += warp_total(lane < rank ? o_most : 0.f);
    all = warp_total(o_n), all_least = warp_total(o_least), all_most = warp_total(o_most);
  }
  // The bins before the cut's: how many there are in all.  (Sums of fp32 here are off by less than 1e-5 of the whole.  A
  // column lies off the middle of its bin by a factor whose standard deviation is 0.0057: three of the sum's are allowed.)
  const float off = sure ? 2e-5f * all_most : 4e-5f * all_least + 3.f * 0.0057f * sqrtf(all_most);
  const float t_least = st.top_p * all_least - off, t_most = st.top_p * (sure ? all_most : all_least) + off;
  int not_yet = 0, below_cut = 0, n_before = 0;  // n_before: columns above the cut's bin, if it is this thread's
  int n_left = 0;                                // and those above and in the cut's bins
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j >= per) break;
    if (by_count) {
      if (above_n + n[j] < k_left) ++not_yet;
      else if (above_n < k_left) n_before = above_n;
      if (above_n < k_left) n_left += n[j];
    } else {
      const bool may = a_least < t_most || above_n == 0;  // begin below the target
      below_cut += may;
      if (may) n_left += n[j];
      a_most += n[j] * most_at(at0 + j);
      a_least += n[j] * least_at(at0 + j);
      not_yet += (sure ? a_most : a_least) < t_least || above_n + n[j] == 0;  // surely ends below it
    }
    above_n += n[j];
  }
  not_yet = (int)__reduce_add_sync(0xffffffffu, (unsigned)not_yet);
  below_cut = (int)__reduce_add_sync(0xffffffffu, (unsigned)below_cut);
  n_before = (int)__reduce_max_sync(0xffffffffu, (unsigned)n_before);
  n_left = (int)__reduce_add_sync(0xffffffffu, (unsigned)n_left);
  if (lane == 0) {
    sh.counts[0][warp] = not_yet, sh.counts[1][warp] = below_cut;
    sh.counts[2][warp] = n_before, sh.counts[3][warp] = n_left;
  }
  __syncthreads();
  if (warp) return;
  int first = (int)__reduce_add_sync(0xffffffffu, lane < kWarps ? (unsigned)sh.counts[0][lane] : 0u);
  int last = (int)__reduce_add_sync(0xffffffffu, lane < kWarps ? (unsigned)sh.counts[1][lane] : 0u);
  int n_above = (int)__reduce_max_sync(0xffffffffu, (unsigned)sh.counts[2][lane % kWarps]);
  n_left = (int)__reduce_add_sync(0xffffffffu, lane < kWarps ? (unsigned)sh.counts[3][lane] : 0u);
  if (lane) return;
  sh.told[2].inside = (u64)n_left;
  sh.told[2].first = first, sh.told[2].last = last, sh.told[2].count = n_above;
  sh.told[2].mx = (float)(by_count && all < k_left);
}
template <typename T> __device__ __noinline__ void after_count_together() {
  Shared& sh = shared();
  State& st = sh.st;
  together(st.ctas);
  if (threadIdx.x) return;
  int first = 0, last = 0, n_above = 0, n_left = 0;
#pragma unroll
  for (int i = 0; i < kCtas; ++i)
    if (i < st.ctas) {
      const Told& o = of_cta(i).told[2];
      first += o.first, last += o.last, n_above = max(n_above, o.count), n_left += (int)o.inside;
    }
  if (sh.told[2].mx != 0.f) {  // fewer than k: all of it
    if (st.top_p < 1.f) begin_cut(st, false);
    else st.by_count = false, st.pass = kWeigh, st.first = kFirst;
    return;
  }
  if (st.by_count) {
    last = first;
    st.k_left -= n_above;
  } else {
    first = min(first, kFirst - 1);
    last = max(first, min(last, kFirst) - 1);
  }
  if (n_left <= kList && st.xt0 == -INFINITY && !st.exact) {
    st.last = last;
    st.pass = kGather;
    return;
  }
  // the places of the values in these bins
  const double slack = 1.0 + 0x1p-21, m = st.m, inv = st.inv;
  const float upper = first ? fminf(st.m, __double2float_ru(m - first / slack / inv)) : st.m;
  const float lower = last == kFirst - 1 ? -INFINITY : __double2float_rd(m - (last + 1) * slack / inv);
  unsigned to = place_of<T>(upper), from = place_of<T>(fmaxf(lower, -3.402823466e38f));
  if (unused_bits<T>()) ++to, from -= from > 0;  // (a bound may lie between two values of 16 bits)
  int shift = 0;
  while ((to - from) >> shift >= (unsigned)kBins) ++shift;
  st.first = first, st.last = last, st.to = to, st.from = from, st.shift = shift;
  st.above = 0;
  st.pass = st.by_count ? kRefine : kWeigh;
}
// The first bin, of the histograms of all CTAs added, at which the counts reach k_left or the sums the target.
__device__ __noinline__ void find_bin() {
  Shared& sh = shared();
  const State& st = sh.st;
  const int tid = threadIdx.x, lane = tid & 31, C = st.ctas, rank = st.rank, k_left = st.k_left;
  const bool by_count = st.by_count, weighed = st.pass == kWeigh;
  if (weighed) {
    __syncthreads();
    const u64 a = warp_total(lane < kWarps ? sh.sums[0][lane] : 0), b = warp_total(lane < kWarps ? sh.sums[1][lane] : 0),
              c = warp_total(lane < kWarps ? sh.sums[2][lane] : 0);
    if (tid == 0) sh.told[0].sum = a, sh.told[0].inside = b, sh.told[0].below = c;
  }
  if (tid == 0) sh.cut.bin = -1;  // (the last one was read before this pass)
  together(C);
  const int per = kBins / C, at0 = rank * per + tid;  // a thread a bin of the rank's share
  int n = 0;
  u64 s = 0;
  if (tid < per) {
    unsigned a[kCtas], b[kCtas], c[kCtas];
#pragma unroll
    for (int i = 0; i < kCtas; ++i)
      if (i < C) a[i] = of_cta(i).count[at0], b[i] = of_cta(i).low[at0], c[i] = of_cta(i).high[at0];
#pragma unroll
    for (int i = 0; i < kCtas; ++i)
      if (i < C) n += (int)a[i], s += ((u64)c[i] << 32) + b[i];
  }
  u64 whole = st.whole, above = st.above, inside = 0;
  double target = st.target;
  if (weighed) {
    const Told& o = of_cta(min(lane, C - 1)).told[0];
    above = warp_total(lane < C ? o.sum : 0);
    inside = warp_total(lane < C ? o.inside : 0);
    whole = above + inside + warp_total(lane < C ? o.below : 0);
    target = (double)st.top_p * (double)whole;
  }
  int all;
  u64 all_s;
  int at = before_thread(n, sh.counts[0], all);
  u64 at_s = before_thread(s, sh.sums[0], all_s);
  if (C > 1) {
    if (tid == 0) sh.told[1].count = all, sh.told[1].sum = all_s;
    together(C);
    const Told& o = of_cta(min(lane, C - 1)).told[1];
    const int o_n = lane < C ? o.count : 0;
    const u64 o_s = lane < C ? o.sum : 0;
    at += warp_total(lane < rank ? o_n : 0), at_s += warp_total(lane < rank ? o_s : 0);
    all = warp_total(o_n);
  }
  if (n > 0) {
    const int to_n = at + n;
    const u64 to_s = at_s + s;
    const double a = (double)(above + at_s), b = (double)(above + to_s);
    const bool final = to_n == all;  // the cut lies here at the latest
    const bool starts = by_count ? at < k_left : at == 0 || a < target, ends = by_count ? to_n >= k_left : b >= target || final;
    if (starts && ends) {
      const double g = guard(st, whole);
      const int open = !by_count && ((above + at_s > 0 && fabs(a - target) <= g) ||
                                     (to_s + above < whole && fabs(b - target) <= g));
      const Cut f{at0, at, n, at_s, s, open};
#pragma unroll 1
      for (int i = 0; i < C; ++i) of_cta(i).cut = f;
    }
  }
  __syncthreads();  // (the state is read above)
  if (tid == 0 && weighed) {
    sh.st.whole = whole, sh.st.above = above, sh.st.target = target;
    sh.st.missed = !st.sure && ((above > 0 && (double)above >= target) ||
                                (inside < whole - above && (double)(above + inside) < target));
  }
}
template <typename T> __device__ __noinline__ void after_bin() {
  Shared& sh = shared();
  State& st = sh.st;
  together(st.ctas);
  if (threadIdx.x) return;
  const Cut f = sh.cut;
  if (st.missed) {
    st.missed = false;
    st.sure = true;
    begin_cut(st, false);
    return;
  }
  bool open = f.open && !st.exact && !(st.shift == 0 && f.inside > 1);  // (one value: its columns are counted below)
  const unsigned to = st.to - ((unsigned)f.bin << st.shift), from = st.shift ? max(st.from, to - ((1u << st.shift) - 1u)) : to;
  st.to = to, st.from = from;
  st.k_left -= f.above;
  st.above += f.sum_above;
  if (!open && from == to) {  // one value: how many of the columns that have it
    st.xt = value_of<T>(to);
    if (st.by_count) {
      st.ties = st.k_left;
      st.xt_k = st.xt0 = st.xt;
      st.ties_k = st.ties0 = st.ties;
      if (st.top_p < 1.f) begin_cut(st, false);
      else st.by_count = false, st.pass = kWeigh, st.first = kFirst;
      return;
    }
    const u64 w = Weight<T>(st)(st.xt);
    const double need = w ? (st.target - (double)st.above) / (double)w : 1.0, g = w ? guard(st, st.whole) / (double)w : 0.0;
    const double left = fmin(fmax(ceil(need), 1.0), (double)f.inside);
    open = !st.exact && ((left > 1.0 && fabs(need - (left - 1.0)) <= g) || (left < f.inside && fabs(need - left) <= g));
    st.ties = (int)left;
    if (!open) {
      st.pass = kSum;
      return;
    }
  }
  if (open) {  // again with exact weights, from this cut's start
    again_exactly(st);
  } else {
    int shift = 0;
    while ((to - from) >> shift >= (unsigned)kBins) ++shift;
    st.shift = shift;
    st.pass = kRefine;
  }
}
// The tid-th largest of the n elements that threads have, element tid each; all differ.  A thread finds a part of one
// element's rank, which is what a sorting network's many short steps lose to (340 cycles each; 114 elements 9,400).
__device__ __noinline__ u64 nth_largest(u64 element, int n) {
  const int tid = threadIdx.x;
  u64 (&list)[2][kList] = shared().list;
  int parts = 1;  // of the list, a thread each
  while (parts < 32 && 2 * parts * n <= kThreads) parts *= 2;
  __syncthreads();
  if (tid < n) list[0][tid] = element;
  __syncthreads();
  const int i = tid / parts, part = tid % parts;
  int rank = 0;
  if (tid / 32 * 32 < n * parts) {
    const u64 mine = list[0][min(i, n - 1)];
#pragma unroll 4
    for (int j = part; j < n; j += parts) rank += list[0][j] > mine;
    for (int o = 1; o < parts; o *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (i < n && part == 0) list[1][rank] = mine;
  }
  __syncthreads();
  return tid < n ? list[1][tid] : 0;
}
// The first CTA puts the gathered columns in order, finds the cuts by the sums before each, puts what is left in the order of
// its places, and draws.  Of top-k's columns weights are taken in fp64 at once; top-p alone has its whole from
// all columns, in fp32 as elsewhere.
template <typename T> __device__ __noinline__ void finish() {
  Shared& sh = shared();
  State& st = sh.st;
  const int tid = threadIdx.x, lane = tid & 31, C = st.ctas;
  const bool by_count = st.by_count;
  __syncthreads();
  const u64 mine = warp_total(lane < kWarps ? sh.sums[0][lane] : 0);
  if (tid == 0) sh.told[3].sum = mine, sh.told[3].count = min(sh.listed, kList);
  together(C);
  if (st.rank == 0) {
    const Told& o = of_cta(min(lane, C - 1)).told[3];
    const int upto = warp_inclusive(lane < C ? o.count : 0), n = min(kList, __shfl_sync(0xffffffffu, upto, 31));
    u64 whole = warp_total(lane < C ? o.sum : 0);
    int from = 0, cta = 0;  // whose list holds element tid
#pragma unroll 1
    for (int i = 0; i + 1 < C; ++i) {
      const int end = __shfl_sync(0xffffffffu, upto, i);
      if (tid >= end) from = end, cta = i + 1;
    }
    u64 e = nth_largest(tid < n ? of_cta(cta).list[0][tid - from] : 0, n);
    Weight<T> weight(st);
    weight.exact |= by_count;
    const int k = by_count ? st.k : n;
    const float x = value_of<T>((unsigned)(e >> 32));
    u64 w = tid < k ? weight(x) : 0, all;
    const u64 before = before_thread(w, sh.sums[1], all);
    if (by_count) whole = all;
    const double target = st.top_p < 1.f ? (double)st.top_p * (double)whole : INFINITY, g = by_count ? 0.0 : guard(st, whole);
    const bool beyond = !by_count && all < whole && (double)all < target, missed = beyond && !st.sure;
    bool open = beyond || (!by_count && all < whole && fabs((double)all - target) <= g);
    if (tid > 0 && tid < k) open |= !by_count && fabs((double)before - target) <= g;
    const bool keep = tid < k && x >= st.xmin && (tid == 0 || (double)before < target);
    open = __syncthreads_or(open);
    const int kept = __syncthreads_count(keep);  // the first ones
    e = nth_largest(e << 32 | e >> 32, kept);    // by their places
    w = e ? weight(value_of<T>((unsigned)e)) : 0;
    const u64 at = before_thread(w, sh.sums[2], all), to = at + w;
    const double goal = st.u * (double)all;
    if (w && (double)to > goal && (at == 0 || (double)at <= goal)) {
      open |= !by_count && ((at > 0 && fabs((double)at - goal) <= g) || (to < all && fabs((double)to - goal) <= g));
      const Cut f{(int)~(unsigned)(e >> 32), missed, 0, 0, 0, open};
#pragma unroll 1
      for (int i = 0; i < C; ++i) of_cta(i).cut = f;
    }
  }
  together(C);
  if (tid) return;
  if (sh.cut.above) {
    st.sure = true;
    begin_cut(st, false);
  } else if (sh.cut.open) {
    again_exactly(st);
  } else {
    st.token = sh.cut.bin;
    st.pass = kDone;
  }
}
// The CTA, the chunk and the column at which the sum passes u times the whole.
template <typename T> __device__ __noinline__ void draw() {
  Shared& sh = shared();
  State& st = sh.st;
  constexpr int E = 16 / sizeof(T);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = st.ctas, rank = st.rank, ties = st.ties;
  const float xt = st.xt, xmin = st.xmin;
  const Weight<T> weight(st);
  __syncthreads();
  const u64 mine = warp_total(lane < kWarps ? sh.sums[0][lane] : 0);
  const int mine_n = warp_total(lane < kWarps ? sh.counts[0][lane] : 0);
  if (tid == 0) sh.told[3].sum = mine, sh.told[3].count = mine_n, sh.cut.bin = -1;
  together(C);
  if (warp == 0) {
    const u64 w_tie = xt > -INFINITY ? weight(xt) : 0;
    const Told& o = of_cta(min(lane, C - 1)).told[3];
    const int o_n = lane < C ? o.count : 0, o_before = warp_inclusive(o_n) - o_n;
    const u64 o_s = lane < C ? o.sum + w_tie * (u64)max(0, min(o_n, ties - o_before)) : 0, o_incl = warp_inclusive(o_s);
    const u64 whole = __shfl_sync(0xffffffffu, o_incl, 31), before = __shfl_sync(0xffffffffu, o_incl - o_s, rank),
              here = __shfl_sync(0xffffffffu, o_s, rank);
    const int ties_before = __shfl_sync(0xffffffffu, o_before, rank);
    const double goal = st.u * (double)whole, g = guard(st, whole);
    if (here > 0 && (before == 0 || (double)before <= goal) && (double)(before + here) > goal) {
      u64 at = before;
      int had = ties_before, found = -1;
#pragma unroll 1
      for (int ch0 = 0; ch0 < st.chunks && found < 0; ch0 += 32) {  // 32 chunks at a time
        const int ch = ch0 + lane, n = ch < st.chunks ? sh.chunk_ties[ch] : 0;
        const int n_incl = warp_inclusive(n), kept = max(0, min(n, ties - (had + n_incl - n)));
        const u64 s = (ch < st.chunks ? sh.chunk_sum[ch] : 0) + w_tie * (u64)kept, incl = warp_inclusive(s);
        const unsigned hit = __ballot_sync(0xffffffffu, (double)(at + incl) > goal);
        const int src = hit ? __ffs(hit) - 1 : 31;
        at += __shfl_sync(0xffffffffu, hit ? incl - s : incl, src);
        had += __shfl_sync(0xffffffffu, hit ? n_incl - n : n_incl, src);
        if (hit) found = ch0 + src;
      }
      int column = -1, open = 0;
      const int end = min(st.vectors, (found + 1) * st.chunk);
#pragma unroll 1
      for (int j0 = found * st.chunk; found >= 0 && j0 < end && column < 0; j0 += 32) {
        const int j = j0 + lane;
        const uint4 bits = reinterpret_cast<const uint4*>(shared_bytes + kSharedBytes)[min(j, end - 1)];
        const T* e = reinterpret_cast<const T*>(&bits);
        auto value = [&](int k) { return j < end ? Elem<T>::to_f(e[k]) : -INFINITY; };
        auto is_tie = [&](float x) { return x == xt && x >= xmin && x > -INFINITY; };
        int n = 0;
#pragma unroll
        for (int k = 0; k < E; ++k) n += is_tie(value(k));
        const int n_incl = warp_inclusive(n);
        // this thread's sum, and then, from what lies before it, the column
        u64 sum = 0, incl = 0;
        int src = -1;
#pragma unroll 1
        for (int round = 0; round < 2; ++round) {
          int rank_tie = had + n_incl - n;
#pragma unroll
          for (int k = 0; k < E; ++k) {
            const float x = value(k);
            u64 w = 0;
            if (x >= xmin && x > xt) w = weight(x);
            else if (is_tie(x) && rank_tie++ < ties) w = w_tie;
            if (lane == src && column < 0 && w && (double)(sum + w) > goal) {
              column = st.first_column + E * j + k;
              open = (sum > 0 && fabs((double)sum - goal) <= g) || (sum + w < whole && fabs((double)(sum + w) - goal) <= g);
            }
            sum += w;
          }
          if (round) break;
          incl = warp_inclusive(sum);
          const unsigned hit = __ballot_sync(0xffffffffu, (double)(at + incl) > goal);
          if (!hit) break;
          src = __ffs(hit) - 1;
          sum = at + incl - sum;
        }
        if (src >= 0) {
          column = __shfl_sync(0xffffffffu, column, src);
          open = __shfl_sync(0xffffffffu, open, src);
        }
        at += __shfl_sync(0xffffffffu, incl, 31);
        had += __shfl_sync(0xffffffffu, n_incl, 31);
      }
      if (lane == 0 && column >= 0) {
        const Cut f{column, 0, 0, 0, 0, open && !st.exact};
#pragma unroll 1
        for (int i = 0; i < C; ++i) of_cta(i).cut = f;
      }
    }
  }
  together(C);
  if (tid) return;
  if (sh.cut.bin >= 0 && sh.cut.open) {
    again_exactly(st);
  } else {
    st.token = max(sh.cut.bin, 0);  // (a column is always found: the largest has weight)
    st.pass = kDone;
  }
}

// Copies this CTA's part of the row to shared memory, and clears what does not take part.
template <typename T> __device__ __forceinline__ void load_row(const SampleParams& p, const T* x) {
  constexpr int E = 16 / sizeof(T);
  State& st = shared().st;
  const int tid = threadIdx.x, C = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
  const int shift = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));  // columns between the boundary and the row
  const int all = (p.cols + shift + E - 1) / E, per = ((all + C - 1) / C + 31) / 32 * 32, lo = min(all, rank * per);
  const int vectors = min(all, lo + per) - lo, first_column = E * lo - shift;
  uint4* columns = reinterpret_cast<uint4*>(shared_bytes + kSharedBytes);
  // (whole vectors: the row's ends share theirs with columns that are not its own)
  const uint4* from = reinterpret_cast<const uint4*>(x - shift) + lo;
#pragma unroll 4
  for (int j = tid; j < vectors; j += kThreads)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(columns + j)), "l"(from + j) : "memory");
  if (tid == 0) {
    st.rank = rank, st.ctas = C;
    st.first_column = first_column, st.vectors = vectors;
    st.chunk = (per / 32 / kMaxChunks + 1) * 32;
    st.chunks = (vectors + st.chunk - 1) / st.chunk;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  T* own = reinterpret_cast<T*>(columns);
  const T none = Elem<T>::from_f(-INFINITY);
  if (tid < 2 * E) {
    const int i = tid < E ? tid : E * vectors - 2 * E + tid;
    if (i >= 0 && i < E * vectors && (first_column + i < 0 || first_column + i >= p.cols)) own[i] = none;
  }
  if (p.skip) {
    const int begin = max(0, first_column), end = min(p.cols, first_column + E * vectors);
    // 16 columns a thread where the mask allows it
    const int head = max(0, min(end - begin, (int)((16 - (reinterpret_cast<uintptr_t>(p.skip + begin) & 15)) & 15)));
    const int wide = max(0, end - begin - head) / 16;
#pragma unroll 1
    for (int j = tid; j < wide; j += kThreads) {
      const int c = begin + head + 16 * j;
      const uint4 w = *reinterpret_cast<const uint4*>(p.skip + c);
      if (w.x | w.y | w.z | w.w)
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
          if (p.skip[c + i]) own[c + i - first_column] = none;
    }
#pragma unroll 1
    for (int i = tid; i < end - begin - 16 * wide; i += kThreads) {
      const int c = begin + (i < head ? i : 16 * wide + i);
      if (p.skip[c]) own[c - first_column] = none;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const SampleParams p) {
  Shared& sh = shared();
  State& st = sh.st;
  const int tid = threadIdx.x, lane = tid & 31;
  const long long r = (long long)blockIdx.x / cg::this_cluster().num_blocks();
  const T* x = reinterpret_cast<const T*>(p.x) + r * p.ld;
  if (tid == 0) {
    const int k = p.top_k ? p.top_k[r] : p.top_k_all;
    const float t = p.temperature ? p.temperature[r] : p.temperature_all;
    st.t = t > 0.f ? fmaxf(t, 0x1p-100f) : t;  // (below that its inverse would not be finite)
    st.k = k < p.cols ? k : 0;
    st.top_p = p.top_p ? p.top_p[r] : p.top_p_all;
    st.min_p = p.min_p ? p.min_p[r] : p.min_p_all;
    st.u = fmin(fmax((double)p.uniforms[r], 0.0), 1.0 - 0x1p-52);  // (a NaN counts as 0, 1 as a little less)
    st.z_due = p.logprobs != nullptr;
    st.by_count = st.exact = st.sure = st.missed = false;
    st.xmin = st.xt = st.xt0 = st.xt_k = -INFINITY;
    st.ties = st.ties0 = st.ties_k = 0x7fffffff;
    st.first = kFirst, st.last = -1, st.token = 0;
    st.pass = kMax;
  }
  load_row<T>(p, x);
  __syncthreads();
#pragma unroll 1
  for (Pass pass = kMax; pass != kDone;) {
    if (pass == kMax) {
      pass_max<T>();
      after_max();
    } else if (pass == kSeek) {
      pass_seek<T>();
      after_seek();
    } else if (pass == kCount) {
      pass_count<T>();
      after_count<T>();
      after_count_together<T>();
    } else if (pass == kGather) {
      pass_gather<T>();
      finish<T>();
    } else if (pass == kSum) {
      pass_sum<T>();
      draw<T>();
    } else {
      const bool weigh = pass == kWeigh;
      if (!weigh) pass_refine<T>();
      else if (st.exact) pass_weigh<T, true>();
      else pass_weigh<T, false>();
      if (weigh && !(st.top_p < 1.f)) {
        __syncthreads();
        if (tid == 0) st.pass = kSum;
      } else {
        find_bin();
        after_bin<T>();
      }
    }
    __syncthreads();
    if (tid == 0 && (pass == kSeek || pass == kWeigh || pass == kGather)) st.z_due = false;
    pass = st.pass;
  }

  // ---- the token and its log-probability ------------------------------------------------------------
  float z = 0.f;
  if (p.logprobs) {
    z = warp_sum(lane < kWarps ? sh.z[lane] : 0.f);
    if (tid == 0) sh.told[2].z = z;
  }
  together(st.ctas);
  if (st.rank == 0 && tid == 0) {
    p.out[r] = st.token;
    if (p.logprobs) {
      z = 0.f;
#pragma unroll 1
      for (int i = 0; i < st.ctas; ++i) z += of_cta(i).told[2].z;
      const float v = p.skip && p.skip[st.token] ? -INFINITY : Elem<T>::to_f(x[st.token]);
      p.logprobs[r] = v - st.m - logf(z);
    }
  }
  together(st.ctas);  // no CTA leaves while another reads what it told
}

template <typename T>
static int launch(const SampleParams& p, int cluster, size_t bytes, cudaStream_t st) {
  if (!allow_smem<sample_rows_kernel<T>>(kMostBytes)) return SPD_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = bytes;
  cfg.gridDim = dim3((unsigned)(p.rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, p) == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace pick

// Columns that fit in the shared memory of a cluster, whatever the row's place.
int sample_rows_most_cols(int dtype) {
  const int e = dtype == SPD_F32 ? 4 : 8, vectors = (int)(pick::kMostBytes - pick::kSharedBytes) / 512 * 32 * pick::kCtas;
  return std::min(1 << 19, (vectors - 1) * e);  // (2^19: sums of weights fit in 64 bits)
}

// CTAs that share a row: as many as it takes for each one's part to leave room for a second CTA on its SM (or for the part to
// fit at all), and as let all rows run at once with 2,048 columns each or more.
int sample_rows_launch(const SampleParams& p, int dtype, int sms, cudaStream_t st) {
  const int e = dtype == SPD_F32 ? 4 : 8;
  auto bytes = [&](int cluster) {  // of a CTA's shared memory (a vector more than the columns fill, for a row off the boundary)
    const long long vectors = ((long long)p.cols + e - 1) / e + 1;
    return pick::kSharedBytes + (size_t)(((vectors + cluster - 1) / cluster + 31) / 32 * 32 * 16);
  };
  int cluster = 1;
  while (cluster < pick::kCtas && (bytes(cluster) > pick::kGoodBytes ||
                                   ((long long)p.rows * cluster < sms && p.cols >= 4096 * cluster)))
    cluster *= 2;
  if ((long long)p.rows * cluster > 0x7fffffffll) return SPD_ERR_UNSUPPORTED;
  switch (dtype) {
    case SPD_F32: return pick::launch<float>(p, cluster, bytes(cluster), st);
    case SPD_F16: return pick::launch<__half>(p, cluster, bytes(cluster), st);
    case SPD_BF16: return pick::launch<__nv_bfloat16>(p, cluster, bytes(cluster), st);
    default: return SPD_ERR_UNSUPPORTED;
  }
}

}  // namespace spd
