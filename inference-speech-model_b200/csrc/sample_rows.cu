// sample_rows.cu — a token a row by temperature, top-k, top-p and min-p from a given random number, and its
// log-probability.  With a row's values x (suppressed columns -inf), their largest m, w = exp((x - m) / t):
//   top-k leaves the k largest (equal ones by their place), top-p of those, in that order, the ones before which less
//   than p of their weight lies, min-p the ones with x >= m + t log(min_p); the token is the first column, by
//   its place, at which the weight left so far passes u times all of it.
//
// What bounds it: a row is read once from memory, 2 or 4 bytes a column, and again from L1 or L2 by each later pass; the
// work is a few dozen instructions a column.  Nothing is sorted:
// * A cluster of up to 8 CTAs shares a row.  A cut (the k-th largest, or the value at which the weight reaches p)
//   is found by histograms: 1,024 bins over the distance from m, then over the order-preserving integers of the values in
//   the bin that holds the cut, until a bin holds one value.  Equal values that the cut divides count by their place.
// * Every sum of weights is an integer (units of 2^-44 of the largest weight), so no order of atomics or threads changes a
//   result, and cumulative sums are exact in their weights.
// * Weights are computed twice as precisely as fp32 needs where it matters: the exponent's argument in fp64, then the
//   hardware's 2^f (2^-22).  A decision that an error of 2^-20 of the whole could turn is
//   taken again with weights in fp64 (a few rows in a hundred where a hundred thousand columns are alike, else next to
//   none), so that the token is the one that fp64 arithmetic gives.
#include "spd_params.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace spd {
namespace pick {
namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kMaxChunks = 1024;  // of a CTA's columns
constexpr int kScale = 44;        // a weight of 1 is 2^44: sums of 2^19 columns fit in 64 bits

// a value's place among all values: the larger, the larger (values of 16 bits leave low bits unused)
template <typename T> constexpr int unused_bits() { return sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16; }
template <typename T> __device__ __forceinline__ unsigned place_of(float x) {
  const unsigned b = __float_as_uint(x);
  return (b & 0x80000000u ? ~b : b | 0x80000000u) >> unused_bits<T>();
}
template <typename T> __device__ __forceinline__ float value_of(unsigned place) {  // of a place that some value has
  const unsigned k = place << unused_bits<T>();
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~(k | ((1u << unused_bits<T>()) - 1u)));
}

struct Best {
  float v;
  int i;
};
// a beats b: NaN over numbers, larger value, then the lower index
__device__ __forceinline__ bool better(Best a, Best b) {
  const bool an = a.v != a.v, bn = b.v != b.v;
  if (an || bn) return an && (!bn || a.i < b.i);
  return a.v > b.v || (a.v == b.v && a.i < b.i);
}

// What CTAs of a cluster tell one another: written before, read after a cluster barrier.
struct Told {
  Best best;
  int count;
  u64 sum;
  float z;
};
// The bin that holds a cut, and what lies above it.
struct Cut {
  int bin;  // -1: none, all is left
  int above, inside;
  u64 sum_above, sum_inside;
  int open;  // the decision could be another with exact weights
};

// The E columns that a thread loads at a time, taken one by one (`next`): the code that looks at a column exists once
// a pass, not E times (unrolled, the kernel had 380 KB).
template <typename T> struct Columns {
  static constexpr int E = 16 / sizeof(T);
  u64 a, b, skip;
  __device__ __forceinline__ float next() {
    float v;
    if constexpr (sizeof(T) == 4) {
      v = __uint_as_float((unsigned)a);
      a = a >> 32 | b << 32;
      b >>= 32;
    } else {
      const unsigned short h = (unsigned short)a;
      v = Elem<T>::to_f(*reinterpret_cast<const T*>(&h));
      a = a >> 16 | b << 48;
      b >>= 16;
    }
    if (skip & 0xff) v = -INFINITY;
    skip >>= 8;
    return v + 0.f;  // no -0
  }
};
// A row's columns of one CTA, in chunks of a warp (32 * E columns at a time).
template <typename T> struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  const unsigned char* mask;
  int lo, hi, chunk, chunks;
  bool vec, mask_vec;  // loads of 16 bytes, of E mask bytes
  // columns c .. c + E - 1; those past the end count as suppressed
  __device__ __forceinline__ Columns<T> load(int c) const {
    Columns<T> v{0, 0, 0};
    const bool whole = c + E <= hi;
    if (vec && whole) {
      const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(x + c);
      v.a = w.x;
      v.b = w.y;
    } else {
#pragma unroll 1
      for (int k = E - 1; k >= 0; --k) {
        unsigned bits = 0;
        if (c + k < hi) {
          if constexpr (sizeof(T) == 4) bits = *reinterpret_cast<const unsigned*>(x + c + k);
          else bits = *reinterpret_cast<const unsigned short*>(x + c + k);
        } else {
          v.skip |= 0xffull << (8 * k);
        }
        constexpr int kBits = 8 * sizeof(T);
        v.b = v.b << kBits | v.a >> (64 - kBits);
        v.a = v.a << kBits | bits;
      }
    }
    if (mask) {
      if (mask_vec && whole) {
        if constexpr (E == 4) v.skip = *reinterpret_cast<const unsigned*>(mask + c);
        else v.skip = *reinterpret_cast<const u64*>(mask + c);
      } else {
#pragma unroll 1
        for (int k = 0; k < E && c + k < hi; ++k)
          if (mask[c + k]) v.skip |= 0xffull << (8 * k);
      }
    }
    return v;
  }
};

// The weight of a value, in units of 2^-44.
__device__ __noinline__ u64 exact_weight(double below, double t) {
  return (u64)(exp(below / t) * (double)(1ull << kScale) + 0.5);
}
struct Weight {
  double m, per, t;  // the largest value, log2(e) / t, t
  bool exact;
  __device__ __forceinline__ u64 operator()(float x) const {
    const double below = (double)x - m;  // <= 0
    if (exact) return exact_weight(below, t);
    const double y = fmax(below * per, -100.0);
    const int n = __double2int_rn(y);
    const unsigned b = __float_as_uint(ex2_approx((float)(y - (double)n)));  // in [2^-1/2, 2^1/2]
    const int shift = kScale - 23 + n + (int)(b >> 23) - 127;
    const u64 bits = (b & 0x7fffffu) | 0x800000u;
    return shift >= 0 ? bits << shift : shift > -25 ? bits >> -shift : 0;
  }
  // How far a sum may be off, seen against the whole of it.
  __device__ __forceinline__ double guard(u64 whole) const { return exact ? 0.0 : (double)whole * 0x1p-20; }
};

template <typename V> __device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V> __device__ __forceinline__ V warp_inclusive(V v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

// What a pass over the row does with its columns.
enum Pass { kMax, kBin, kSum, kLog };

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const SampleParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ unsigned count[kBins], low[kBins], high[kBins];
  __shared__ u64 chunk_sum[kMaxChunks];
  __shared__ int chunk_ties[kMaxChunks];
  __shared__ Told told[4];
  __shared__ Cut cut_here;
  __shared__ Best bests[kWarps];
  __shared__ float zs[kWarps];
  __shared__ u64 sums[kWarps];
  __shared__ int counts[kWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long r = (long long)blockIdx.x / C;
  constexpr int E = Row<T>::E, kUnit = 32 * E;
  Row<T> row;
  row.x = reinterpret_cast<const T*>(p.x) + r * p.ld;
  row.mask = p.skip;
  row.vec = p.vec;
  row.mask_vec = p.skip_vec;
  {
    const int per = ((p.cols + C - 1) / C + kUnit - 1) / kUnit * kUnit;  // columns of a CTA
    row.lo = (int)min((long long)p.cols, (long long)rank * per);
    row.hi = (int)min((long long)p.cols, (long long)row.lo + per);
    row.chunk = ((per / kUnit + kMaxChunks - 1) / kMaxChunks) * kUnit;
    row.chunks = (row.hi - row.lo + row.chunk - 1) / row.chunk;
  }
  const float t = p.temperature ? p.temperature[r] : p.temperature_all;
  const int k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;

  int token = -1;  // known to every thread once it is
  Best best{-INFINITY, 0x7fffffff};
  float m = 0.f, z = 0.f;  // the largest value; sum of exp(x - m)
  bool z_due = p.logprobs != nullptr;
  float xmin = -INFINITY;  // min-p
  float xt = -INFINITY;    // what is left: values above xt, and the first `ties` columns that have it
  int ties = 0x7fffffff;
  Weight weight{0.0, 0.0, 1.0, false};
  // a cut under way
  bool by_count = false;
  float xt0 = xt, xt_k = xt, inv = 0.f;
  int ties0 = ties, ties_k = ties, k_left = 0, bin1 = -1, shift = 0;
  unsigned from = 0, to = 0;
  u64 whole = 0, above = 0;
  double target = 0.0;

  auto bin_of = [&](float v) { return (int)fminf((m - v) * inv, (float)(kBins - 1)); };
  // this value's bin in the present histogram, or -1
  auto place_in = [&](float v) {
    const int bin = bin_of(v);
    if (bin1 < 0) return bin;
    const unsigned place = place_of<T>(v);
    return bin == bin1 && place >= from && place <= to ? (int)((to - place) >> shift) : -1;
  };
  auto put = [&](int bin, unsigned n, u64 w) {
    atomicAdd(&count[bin], n);
    if (w) {
      const unsigned l = (unsigned)w, old = atomicAdd(&low[bin], l), h = (unsigned)(w >> 32) + (old + l < old);
      if (h) atomicAdd(&high[bin], h);
    }
  };
  auto begin_cut = [&](bool count_them) {
    by_count = count_them;
    xt0 = xt;
    ties0 = ties;
    k_left = k;
    bin1 = -1;
    whole = above = 0;
    inv = (float)(kBins - 1) / (by_count ? 32.f : 40.f * t);
  };

  Pass pass = kMax;
#pragma unroll 1
  while (true) {
    // ---- one pass over the row ----------------------------------------------------------------------
    if (pass == kBin) {
#pragma unroll 1
      for (int i = tid; i < kBins; i += kThreads) count[i] = low[i] = high[i] = 0;
      __syncthreads();
      if (!by_count && xt0 > -INFINITY && rank == 0 && tid == 0) {  // columns that have xt0 itself, by their number
        const int bin = place_in(xt0);
        if (bin >= 0) put(bin, (unsigned)ties0, weight(xt0) * (u64)ties0);
      }
    }
    u64 mine = 0;
    int mine_ties = 0;
#pragma unroll 1
    for (int ch = warp; ch < row.chunks; ch += kWarps) {
      u64 s = 0;
      int n = 0;
      const int end = min(row.hi, row.lo + (ch + 1) * row.chunk);
#pragma unroll 1
      for (int c = row.lo + ch * row.chunk + lane * E; c < end; c += kUnit) {
        Columns<T> v4 = row.load(c);
#pragma unroll 1
        for (int e = 0; e < E; ++e) {
          const float v = v4.next();
          if (pass == kMax) {
            const Best b{v, c + e};
            if (c + e < row.hi && better(b, best)) best = b;
            continue;
          }
          if (z_due) z += ex2_approx((v - m) * 1.4426950408889634f);
          if (pass == kBin) {
            const int bin = v > xt0 ? place_in(v) : -1;
            if (bin >= 0) put(bin, 1, by_count ? 0 : weight(v));
          } else if (pass == kSum && v >= xmin) {
            if (v > xt) s += weight(v);
            n += v == xt && xt > -INFINITY;
          }
        }
      }
      if (pass == kSum) {
        s = warp_total(s);
        n = warp_total(n);
        if (lane == 0) chunk_sum[ch] = s, chunk_ties[ch] = n;
        mine += s;
        mine_ties += n;
      }
    }
    if (pass != kMax) z_due = false;

    // ---- and what follows from it -------------------------------------------------------------------
    if (pass == kMax) {
      auto best_of_warp = [&]() {
#pragma unroll 1
        for (int o = 16; o > 0; o >>= 1) {
          const Best b{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)};
          if (better(b, best)) best = b;
        }
      };
      best_of_warp();
      if (lane == 0) bests[warp] = best;
      __syncthreads();
      best = lane < kWarps ? bests[lane] : Best{-INFINITY, 0x7fffffff};
      best_of_warp();
      if (tid == 0) told[0].best = best;
      cluster.sync();
#pragma unroll 1
      for (int i = 0; i < C; ++i) {
        const Best b = cluster.map_shared_rank(told, i)[0].best;
        if (better(b, best)) best = b;
      }
      m = best.v;
      weight = Weight{(double)m, 1.4426950408889634 / (double)t, (double)t, false};
      if (!(fabsf(m) < INFINITY) || !(t > 0.f)) token = best.i;
      if (min_p > 0.f && token < 0) {
        xmin = __double2float_ru((double)m + (double)t * log((double)min_p));
        if (!(xmin <= m)) token = best.i;
      }
      if (token >= 0) {
        pass = kLog;
        if (!z_due) break;
      } else if (k > 0 && k < p.cols) {
        begin_cut(true);
        pass = kBin;
      } else if (top_p < 1.f) {
        begin_cut(false);
        pass = kBin;
      } else {
        pass = kSum;
      }
    } else if (pass == kBin) {
      // The first bin, of the histograms of all CTAs added, at which the counts reach k_left or the sums the target.
      cluster.sync();
      const int per = kBins / C;  // bins of a rank: 1024 (two a thread), 512, 256 or 128
      const int bins = per > kThreads ? 2 : tid < per ? 1 : 0, first = rank * per + (per > kThreads ? 2 * tid : tid);
      int n = 0, n0 = 0;
      u64 s = 0, s0 = 0;
#pragma unroll 1
      for (int j = 0; j < bins; ++j) {
        n0 = n;
        s0 = s;
#pragma unroll 1
        for (int i = 0; i < C; ++i) {
          n += (int)cluster.map_shared_rank(count, i)[first + j];
          s += (u64)cluster.map_shared_rank(low, i)[first + j] + ((u64)cluster.map_shared_rank(high, i)[first + j] << 32);
        }
      }
      int incl = warp_inclusive(n);
      u64 incl_s = warp_inclusive(s);
      if (lane == 31) counts[warp] = incl, sums[warp] = incl_s;
      __syncthreads();
      int all = 0;
      u64 all_s = 0;
#pragma unroll 1
      for (int i = 0; i < kWarps; ++i) {
        if (i == warp) incl += all, incl_s += all_s;
        all += counts[i];
        all_s += sums[i];
      }
      if (tid == 0) {
        told[1].count = all;
        told[1].sum = all_s;
        cut_here.bin = -1;
      }
      cluster.sync();  // every CTA's totals are there, and no cut found before is read any more
      int before = 0;
      u64 before_s = 0;
      all = 0;
      all_s = 0;
#pragma unroll 1
      for (int i = 0; i < C; ++i) {
        if (i == rank) before = all, before_s = all_s;
        const Told& o = cluster.map_shared_rank(told, i)[1];
        all += o.count;
        all_s += o.sum;
      }
      if (bin1 < 0 && !by_count) {
        whole = all_s;
        target = (double)top_p * (double)whole;
      }
      int at = before + incl - n;  // above this thread's bins, of this histogram
      u64 at_s = before_s + incl_s - s;
#pragma unroll 1
      for (int j = 0; j < bins; ++j) {
        const int to_n = before + incl - (j + 1 < bins ? n - n0 : 0);
        const u64 to_s = before_s + incl_s - (j + 1 < bins ? s - s0 : 0);
        if (to_n > at) {
          const double a = (double)(above + at_s), b = (double)(above + to_s);
          const bool last = to_n == all;  // the cut lies here at the latest
          const bool starts = by_count ? at < k_left : at == 0 || a < target, ends = by_count ? to_n >= k_left : b >= target || last;
          if (starts && ends) {
            const double g = weight.guard(whole);
            const int open = !by_count && ((at > 0 && fabs(a - target) <= g) || (!last && fabs(b - target) <= g));
            const Cut f{first + j, at, to_n - at, at_s, to_s - at_s, open};
#pragma unroll 1
            for (int i = 0; i < C; ++i) cluster.map_shared_rank(&cut_here, i)[0] = f;
          }
        }
        at = to_n;
        at_s = to_s;
      }
      cluster.sync();
      const Cut f = cut_here;
      bool cut_done = f.bin < 0;  // fewer than k: all of it
      bool open = !cut_done && f.open && !weight.exact;
      if (!cut_done) {
        if (bin1 < 0) {  // the first histogram, over distances: the places of the values in the bin lie in [from, to]
          bin1 = f.bin;
          const double slack = 1.0 + 0x1p-21;
          const float top = bin1 ? fminf(m, __double2float_ru((double)m - bin1 / slack / (double)inv)) : m;
          const float bottom = bin1 == kBins - 1 ? -INFINITY : __double2float_rd((double)m - (bin1 + 1) * slack / (double)inv);
          to = place_of<T>(top);
          from = place_of<T>(fmaxf(bottom, -3.402823466e38f));
          if (unused_bits<T>()) ++to, from -= from > 0;  // (a bound may lie between two values of 16 bits)
        } else {
          // (of one value, the columns that are left are counted below)
          if (shift == 0 && f.inside > 1) open = false;
          to -= (unsigned)f.bin << shift;
          from = shift ? max(from, to - ((1u << shift) - 1u)) : to;
        }
        k_left -= f.above;
        above += f.sum_above;
        if (from == to && !open) {  // one value: how many of the columns that have it
          xt = value_of<T>(to);
          if (by_count) {
            ties = k_left;
          } else {
            const u64 w = weight(xt);
            const double need = w ? (target - (double)above) / (double)w : 1.0, g = w ? weight.guard(whole) / (double)w : 0.0;
            const double left = fmin(fmax(ceil(need), 1.0), (double)f.inside);
            open = !weight.exact && ((left > 1.0 && fabs(need - (left - 1.0)) <= g) || (left < f.inside && fabs(need - left) <= g));
            ties = (int)left;
          }
          cut_done = true;
        } else {
          shift = 0;
          while ((to - from) >> shift >= (unsigned)kBins) ++shift;
        }
      }
      if (open) {  // again with exact weights, from this cut's start (decided alike by every thread of the cluster)
        weight.exact = true;
        xt = xt_k;
        ties = ties_k;
        begin_cut(false);
      } else if (cut_done) {
        if (by_count) {
          xt_k = xt;
          ties_k = ties;
        }
        if (by_count && top_p < 1.f) begin_cut(false);
        else pass = kSum;
      }
    } else if (pass == kSum) {
      // The CTA, the chunk and the column at which the sum passes u times the whole.
      if (lane == 0) sums[warp] = mine, counts[warp] = mine_ties;
      __syncthreads();
      if (tid == 0) {
        u64 s = 0;
        int n = 0;
#pragma unroll 1
        for (int i = 0; i < kWarps; ++i) s += sums[i], n += counts[i];
        told[2].sum = s;
        told[2].count = n;
        cut_here.bin = -1;
      }
      cluster.sync();
      const u64 w_tie = xt > -INFINITY ? weight(xt) : 0;
      u64 before = 0, here = 0;
      int ties_before = 0, seen = 0;
      whole = 0;
#pragma unroll 1
      for (int i = 0; i < C; ++i) {
        const Told& o = cluster.map_shared_rank(told, i)[2];
        const int n = max(0, min(o.count, ties - seen));
        const u64 s = o.sum + w_tie * (u64)n;
        if (i == rank) before = whole, here = s, ties_before = seen;
        whole += s;
        seen += o.count;
      }
      const double u = fmax((double)p.uniforms[r], 0.0);  // (a NaN counts as 0)
      const double goal = u < 1.0 ? u * (double)whole : (double)whole - 0.5, guard = weight.guard(whole);
      if (warp == 0 && here > 0 && (before == 0 || (double)before <= goal) && (double)(before + here) > goal) {
        u64 at = before;
        int had = ties_before, found = -1;
#pragma unroll 1
        for (int ch0 = 0; ch0 < row.chunks && found < 0; ch0 += 32) {  // 32 chunks at a time
          const int ch = ch0 + lane, n = ch < row.chunks ? chunk_ties[ch] : 0;
          const int n_incl = warp_inclusive(n), kept = max(0, min(n, ties - (had + n_incl - n)));
          const u64 s = (ch < row.chunks ? chunk_sum[ch] : 0) + w_tie * (u64)kept, incl = warp_inclusive(s);
          const unsigned hit = __ballot_sync(0xffffffffu, (double)(at + incl) > goal);
          const int src = hit ? __ffs(hit) - 1 : 31;
          at += __shfl_sync(0xffffffffu, hit ? incl - s : incl, src);
          had += __shfl_sync(0xffffffffu, hit ? n_incl - n : n_incl, src);
          if (hit) found = ch0 + src;
        }
        int column = -1, open = 0;
        const int end = min(row.hi, row.lo + (found + 1) * row.chunk);
#pragma unroll 1
        for (int c0 = row.lo + found * row.chunk; found >= 0 && c0 < end && column < 0; c0 += kUnit) {
          const int c = c0 + lane * E;
          const Columns<T> v4 = c < end ? row.load(c) : Columns<T>{0, 0, ~0ull};
          int n = 0;
          Columns<T> v = v4;
#pragma unroll 1
          for (int e = 0; e < E; ++e) {
            const float x = v.next();
            n += x == xt && x >= xmin && xt > -INFINITY;
          }
          const int n_incl = warp_inclusive(n);
          // the sum of this thread's columns, then the column: the second time over from the sum before them
          u64 incl = 0, s = 0;
          unsigned hit = 0;
          int src = 0;
#pragma unroll 1
          for (int round = 0; round < 2; ++round) {
            int rank_tie = had + n_incl - n;
            u64 sum = round ? at + incl - s : 0;
            v = v4;
#pragma unroll 1
            for (int e = 0; e < E; ++e) {
              const float x = v.next();
              u64 w = 0;
              if (x >= xmin && x > xt) w = weight(x);
              else if (x >= xmin && x == xt && xt > -INFINITY && rank_tie++ < ties) w = w_tie;
              if (round && lane == src && column < 0 && w && (double)(sum + w) > goal) {
                column = c + e;
                open = (sum > 0 && fabs((double)sum - goal) <= guard) || (sum + w < whole && fabs((double)(sum + w) - goal) <= guard);
              }
              sum += w;
            }
            if (round == 0) {
              s = sum;
              incl = warp_inclusive(s);
              hit = __ballot_sync(0xffffffffu, (double)(at + incl) > goal);
              if (!hit) break;
              src = __ffs(hit) - 1;
            }
          }
          if (hit) {
            column = __shfl_sync(0xffffffffu, column, src);
            open = __shfl_sync(0xffffffffu, open, src);
          }
          at += __shfl_sync(0xffffffffu, incl, 31);
          had += __shfl_sync(0xffffffffu, n_incl, 31);
        }
        if (lane == 0 && column >= 0) {
          const Cut f{column, 0, 0, 0, 0, open && !weight.exact};
#pragma unroll 1
          for (int i = 0; i < C; ++i) cluster.map_shared_rank(&cut_here, i)[0] = f;
        }
      }
      cluster.sync();
      if (cut_here.bin >= 0 && cut_here.open) {
        weight.exact = true;
        if (top_p < 1.f) {
          xt = xt_k;
          ties = ties_k;
          begin_cut(false);
          pass = kBin;
        }
        cluster.sync();  // (read by all before it is written again)
      } else {
        token = cut_here.bin >= 0 ? cut_here.bin : best.i;
        break;
      }
    } else {
      break;
    }
  }

  // ---- the token and its log-probability ------------------------------------------------------------
  if (p.logprobs) {
    z = warp_sum(z);
    if (lane == 0) zs[warp] = z;
    __syncthreads();
    if (tid == 0) {
      float s = 0.f;
#pragma unroll 1
      for (int i = 0; i < kWarps; ++i) s += zs[i];
      told[3].z = s;
    }
    cluster.sync();
  }
  if (rank == 0 && tid == 0) {
    p.out[r] = token;
    if (p.logprobs) {
      float s = 0.f;
#pragma unroll 1
      for (int i = 0; i < C; ++i) s += cluster.map_shared_rank(told, i)[3].z;
      const bool skipped = p.skip && p.skip[token];
      const float x = skipped ? -INFINITY : Elem<T>::to_f(row.x[token]);
      p.logprobs[r] = x - m - logf(s);
    }
  }
  cluster.sync();  // no CTA leaves while another reads what it told
}

template <typename T>
static int launch(const SampleParams& p, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
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

// CTAs that share a row: as many as let all rows run at once (four CTAs an SM), with 4,096 columns each or more.
int sample_rows_launch(const SampleParams& p, int dtype, int sms, cudaStream_t st) {
  int cluster = 8;
  while (cluster > 1 && ((long long)p.rows * cluster > 4ll * sms || p.cols < 4096 * cluster)) cluster /= 2;
  if ((long long)p.rows * cluster > 0x7fffffffll) return SPD_ERR_UNSUPPORTED;
  switch (dtype) {
    case SPD_F32: return pick::launch<float>(p, cluster, st);
    case SPD_F16: return pick::launch<__half>(p, cluster, st);
    case SPD_BF16: return pick::launch<__nv_bfloat16>(p, cluster, st);
    default: return SPD_ERR_UNSUPPORTED;
  }
}

}  // namespace spd
