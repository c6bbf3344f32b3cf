// own_attn.cu — single-token attention with grouped heads over a paged 16-bit cache, for sequences that
// also share a prefix with their group:
//   out[b, h] = softmax(q[b, h] . [prefix keys, own keys]) . [prefix values, own values]
// The prefix's part (output, maximum and sum a row, in one piece or several) comes from span_attn.cu, which
// reads it once for the whole group; this kernel attends each sequence's own tokens and adds the two.
//
// What bounds it: a key and its value are read once for 4 * G operations for each of their 4 bytes: HBM, or
// with short contexts the latency of lengths, table, rows and join.
// * mma.sync m16n8k16 with the group's heads as its 16 rows: at a row count of 1 to 16 the products are a
//   small part of the time.  (tcgen05 has 128 rows.)  With up to 8 heads the other 8 rows of the weights hold
//   their rounding remainders, so that weights keep 16 bits and more at no cost.  With more heads all 16 rows are
//   heads and weights are rounded to the input's type, as span_attn.cu does: 8 heads a CTA would read the keys twice as often.
// * A CTA takes a chunk of one sequence for one key/value head (16 heads of it), a warp every fourth step of
//   `kKeys` keys, by cp.async into a ring of its own: any block size, rows of a block out of range as zeros.
// * It is launched with programmatic dependent launch behind span_attn.cu, which hides its launch: its CTAs start as
//   those of the spans leave their SMs (which they fill with registers) and wait for the whole kernel only to join.  The
//   chunks of a sequence are joined by the last CTA to arrive, in their order.
// Measured on a B200, in CUDA graphs, with the prefixes' kernel: groups with ragged prefixes and own tokens 65 us (36 for
// their bytes at a copy's rate), two groups of 64 over prefixes of 32,000 tokens 132 (83), one request's candidates
// 12.7: some 8 us of dependent loads (lengths, table, rows, join) and the launches.  By itself, from cold caches: 42 us for
// the 136 MB of the first (0.50 of a copy), 62 us for the 282 MB of the second (0.70).
#include "spd_tc_attn.cuh"

#include <algorithm>

namespace spd {
namespace own {
using tc::pack2;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 2;
constexpr int kStageBytes = 8192;  // keys and values of a step

template <int DP> struct Cfg {
  static constexpr int kKeys = kStageBytes / (4 * DP);  // 16 at 128, 32 at 64
  static constexpr int kRow = 2 * DP;                   // bytes
  static constexpr size_t kSmem = (size_t)kWarps * kStages * kStageBytes;
  static_assert(16 * DP * 4 <= kStages * kStageBytes, "a warp's result fits in its ring");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

// A weighted sum of partial results of one row: values [d, d + 4), maximum and sum.
struct Sum {
  float m = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float4 v, float vm, float vl) {
    const float mm = fmaxf(m, vm);
    const float f0 = m == mm ? 1.f : ex2_approx(m - mm), f1 = vm == mm ? 1.f : ex2_approx(vm - mm);
    m = mm;
    l = l * f0 + vl * f1;
    a.x = a.x * f0 + v.x * f1;
    a.y = a.y * f0 + v.y * f1;
    a.z = a.z * f0 + v.z * f1;
    a.w = a.w * f0 + v.w * f1;
  }
};

// SPLIT: rows 8 to 15 hold the rounding remainders of the weights of rows 0 to 7.
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 3) own_attn_kernel(const OwnParams p) {
  using C = Cfg<DP>;
  constexpr int kKeys = C::kKeys, kHeads = SPLIT ? 8 : 16, kTiles = DP / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t there[kWarps][kStages];  // tokens of a step that count, a bit each
  __shared__ float stat_m[kWarps][16], stat_l[kWarps][16];
  __shared__ int last_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int Gq = p.Hq / p.Hkv;
  const int tiles = (Gq + kHeads - 1) / kHeads, Y = p.Hkv * tiles;
  const int y = (int)(blockIdx.x % (unsigned)Y), rest = (int)(blockIdx.x / (unsigned)Y);
  const int b = rest % p.B, chunk = rest / p.B;  // first chunks first
  const int tile = y % tiles, kvh = y / tiles;
  const int heads = min(kHeads, Gq - tile * kHeads);
  const long long head0 = (long long)b * p.Hq + kvh * Gq + tile * kHeads;  // row of out
  const int step = p.D + 4;  // floats of a partial result

  int ctx = max(0, p.context_lens[b]);
  if ((long long)ctx > (long long)p.max_blocks << p.bs_log2) {
    if (tid == 0) set_error(p.err, SPD_DEVERR_LENGTH);
    ctx = p.max_blocks << p.bs_log2;
  }
  const int size = max(p.least, (int)((((unsigned)ctx + p.chunks - 1) / p.chunks + kKeys - 1) / kKeys * kKeys));
  const int parts = max(1, (ctx - 1) / size + 1);
  if (chunk >= parts) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int t0 = chunk * size, t1 = ctx - t0 > size ? t0 + size : ctx;
  const int steps = (t1 - t0 + kKeys - 1) / kKeys;
  const int* table = p.block_tables + (long long)b * p.max_blocks;

  unsigned char* ring = smem + (size_t)warp * kStages * kStageBytes;
  const uint32_t ring_at = smem_addr(ring);
  const T* k_pool = reinterpret_cast<const T*>(p.k_pool) + (long long)kvh * p.D;
  const T* v_pool = reinterpret_cast<const T*>(p.v_pool) + (long long)kvh * p.D;
  const long long row_stride = (long long)p.Hkv * p.D;

  // Copies run ahead: lane `i` looks up the block of token i of the step `ahead`, one step before its copy.
  int ahead = warp, id = 0, fetched = 0;
  auto look_up = [&]() {
    const int tok = t0 + ahead * kKeys + lane;
    id = ahead < steps && lane < kKeys && tok < t1 ? __ldg(table + (tok >> p.bs_log2)) : -1;
  };
  auto fetch = [&]() {  // (a group is committed also when nothing is left, so that waits count alike)
    if (ahead < steps) {
      const int st = fetched % kStages, tok0 = t0 + ahead * kKeys;
      const bool inside = lane < kKeys && tok0 + lane < t1, good = inside && id >= 0 && id < p.num_blocks;
      if (inside && !good) set_error(p.err, SPD_DEVERR_BLOCK_ID);
      const uint32_t counts = __ballot_sync(0xffffffffu, good);
      if (lane == 0) there[warp][st] = counts;
      // rows of this warp's tokens in the pools
      const long long place = good ? ((long long)id << p.bs_log2) + ((tok0 + lane) & ((1 << p.bs_log2) - 1)) : 0;
      const uint32_t base = ring_at + st * kStageBytes;
      constexpr int kChunks = DP / 8, kPer = 32 / kChunks;  // 16-byte chunks of a row; rows a pass
      const int c = lane % kChunks;
#pragma unroll
      for (int r0 = 0; r0 < kKeys; r0 += kPer) {
        const int r = r0 + lane / kChunks;
        const long long row = __shfl_sync(0xffffffffu, place, r);
        const bool copy = (counts >> r & 1) && c * 8 < p.D;
        const long long from = copy ? row * row_stride + c * 8 : 0;
        const uint32_t to = base + r * C::kRow + ((c ^ (r & 7)) << 4);
        cp_async16(to, k_pool + from, copy);
        cp_async16(to + kKeys * C::kRow, v_pool + from, copy);
      }
      ++fetched;
      ahead += kWarps;
      look_up();
    }
    cp_commit();
  };
  look_up();

  // ---- the group whose prefix this sequence shares (by 32 starts at once: 1,024 groups of two 249 -> 187 us)
  int group = -1;
  {
    int first = 0, n = p.G;  // the groups that it may be
#pragma unroll 1
    while (n > 32) {  // 32 starts a step, the last that is not past it
      const int every = (n + 31) / 32, i = lane * every;
      const int before = __popc(__ballot_sync(0xffffffffu, i < n && p.cu_groups[first + i] <= b));
      const int skip = max(before - 1, 0) * every;
      first += skip;
      n = min(every, n - skip);
    }
    const int i = first + lane;
    const uint32_t hit = __ballot_sync(0xffffffffu, lane < n && p.cu_groups[i] <= b && b < p.cu_groups[i + 1]);
    if (hit) group = first + __ffs(hit) - 1;
  }
  if (group >= 0 && p.prefix_lens[group] <= 0) group = -1;

  // ---- query fragments: rows g and g + 8, pairs of dimensions 2t and 2t + 8 of each 16 ----------
  uint32_t qa[DP / 16][4];
  {
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_st + (kvh * Gq + tile * kHeads) * p.q_sh;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = g + 8 * (i & 1), d = 16 * s + 2 * t + 8 * (i >> 1);
        qa[s][i] = r < heads && d < p.D ? *reinterpret_cast<const uint32_t*>(q + r * p.q_sh + d) : 0u;
      }
  }
  float o[kTiles][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.f;

  int used = 0;
#pragma unroll 1
  for (int i = warp - (kStages - 1) * kWarps; i < steps; i += kWarps) {
    fetch();
    if (i < 0) continue;  // the first copies
    cp_wait<kStages - 1>();
    __syncwarp();
    const int st = used % kStages;
    ++used;
    const uint32_t k_at = ring_at + st * kStageBytes, v_at = k_at + kKeys * C::kRow;
    const uint32_t counts = there[warp][st];
    // ---- scores: [16 rows][keys] -------------------------------------------------------------
    float sc[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
    for (int n = 0; n < kKeys / 8; n += 2)
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        // matrices: keys 8n.. and 8n + 8.., dimensions 16s.. and 16s + 8..
        const int r = 8 * n + (lane & 7) + 8 * (lane >> 4), c = 2 * s + (lane >> 3 & 1);
        uint32_t kb[4];
        ldmatrix4(k_at + r * C::kRow + ((c ^ (r & 7)) << 4), kb);
        mma_16816<T>(sc[n], qa[s][0], qa[s][1], qa[s][2], qa[s][3], kb[0], kb[1]);
        mma_16816<T>(sc[n + 1], qa[s][0], qa[s][1], qa[s][2], qa[s][3], kb[2], kb[3]);
      }
    constexpr uint32_t kAll = kKeys == 32 ? 0xffffffffu : (1u << kKeys) - 1;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[n][e] *= p.scale_log2;
        if (counts != kAll && !(counts >> (8 * n + 2 * t + (e & 1)) & 1)) sc[n][e] = -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], sc[n][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (SPLIT && r) break;
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], x));
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || (!SPLIT && mx[1] > m[1]))) {
      float f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float mn = fmaxf(m[r], mx[r]);
        f[r] = m[r] == mn ? 1.f : ex2_approx(m[r] - mn);
        if (SPLIT && r) f[1] = f[0];
        else m[r] = mn;
        l[r] *= f[r];
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        o[j][0] *= f[0];
        o[j][1] *= f[0];
        o[j][2] *= f[1];
        o[j][3] *= f[1];
      }
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
    // ---- weights and output ------------------------------------------------------------------
#pragma unroll
    for (int n = 0; n < kKeys / 8; n += 2) {
      uint32_t pa[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float* s = sc[n + h];
        const float p0 = ex2_approx(s[0] - m0), p1 = ex2_approx(s[1] - m0);
        l[0] += p0 + p1;
        pa[2 * h] = pack2<T>(p0, p1);
        if constexpr (SPLIT) {
          const T* r = reinterpret_cast<const T*>(&pa[2 * h]);
          pa[2 * h + 1] = pack2<T>(p0 - Elem<T>::to_f(r[0]), p1 - Elem<T>::to_f(r[1]));
        } else {
          const float p2 = ex2_approx(s[2] - m1), p3 = ex2_approx(s[3] - m1);
          l[1] += p2 + p3;
          pa[2 * h + 1] = pack2<T>(p2, p3);
        }
      }
#pragma unroll
      for (int j = 0; j < kTiles; j += 2) {
        // matrices: keys 8n.. and 8n + 8.., dimensions 8j.. and 8j + 8..
        const int r = 8 * n + (lane & 15), c = j + (lane >> 4);
        uint32_t vb[4];
        ldmatrix4_trans(v_at + r * C::kRow + ((c ^ (r & 7)) << 4), vb);
        mma_16816<T>(o[j], pa[0], pa[1], pa[2], pa[3], vb[0], vb[1]);
        mma_16816<T>(o[j + 1], pa[0], pa[1], pa[2], pa[3], vb[2], vb[3]);
      }
    }
    __syncwarp();  // every lane has read this stage
  }
  cp_wait<0>();

  // ---- join the warps ---------------------------------------------------------------------------
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
  __syncwarp();
  float* mine = reinterpret_cast<float*>(ring);  // [heads][DP]; the ring is drained
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
    const int d = 8 * j + 2 * t;
    if constexpr (SPLIT) {
      // (over an infinite value a remainder, of any sign or zero, says nothing that its weight has not said)
      auto finite = [](float x) { return fabsf(x) < INFINITY ? x : 0.f; };
      *reinterpret_cast<float2*>(mine + g * DP + d) = make_float2(o[j][0] + finite(o[j][2]), o[j][1] + finite(o[j][3]));
    } else {
      *reinterpret_cast<float2*>(mine + g * DP + d) = make_float2(o[j][0], o[j][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * DP + d) = make_float2(o[j][2], o[j][3]);
    }
  }
  if (t == 0) {
    stat_m[warp][g] = m[0];
    stat_l[warp][g] = l[0];
    if (!SPLIT) {
      stat_m[warp][g + 8] = m[1];
      stat_l[warp][g + 8] = l[1];
    }
  }
  __syncthreads();
  const int quads = p.D / 4;
  auto of_warps = [&](Sum& s, int h, int d) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < steps)
        s.add(reinterpret_cast<const float4*>(smem + (size_t)w * kStages * kStageBytes)[(h * DP + d) / 4], stat_m[w][h], stat_l[w][h]);
  };
  // the n partial results of a row
  auto of_memory = [&](Sum& s, const float* row, long long next, int n, int d) {
#pragma unroll 4
    for (int c = 0; c < n; ++c, row += next) {
      const float2 st = __ldcg(reinterpret_cast<const float2*>(row + p.D));
      s.add(__ldcg(reinterpret_cast<const float4*>(row + d)), st.x, st.y);
    }
  };
  if (parts > 1) {
    // ---- the chunks of a sequence are joined by the last CTA of this (sequence, head tile) to arrive ----
#pragma unroll 1
    for (int e = tid; e < heads * quads; e += kThreads) {
      const int h = e / quads, d = e % quads * 4;
      Sum s;
      of_warps(s, h, d);
      float* row = p.partials + ((head0 + h) * p.chunks + chunk) * step;
      *reinterpret_cast<float4*>(row + d) = s.a;
      if (d == 0) *reinterpret_cast<float2*>(row + p.D) = make_float2(s.m, s.l);
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      int* counter = p.counters + (long long)b * Y + y;
      last_flag = atomicAdd(counter, 1) == parts - 1;
      if (last_flag) *counter = 0;
    }
    __syncthreads();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (parts > 1) {
    if (!last_flag) return;
    __threadfence();
  }
  // ---- and with the group's prefix ---------------------------------------------------------------
  int2 desc = make_int2(0, 0);
  if (group >= 0) {
    desc = __ldcg(p.row_desc + (long long)b * p.Hkv + kvh);
    // What a prefix's kernel that gave up waiting did not write is not followed.
    const int row0 = (int)((unsigned)desc.y >> 16), count = desc.y & 0xffff;
    if (desc.x < -1 || desc.x > p.span_ctas - count || row0 + Gq > p.piece_rows || (desc.x < 0 && count > 1)) desc.y = 0;
  }
  const int pieces = desc.y & 0xffff, first_cta = desc.x;
  const long long piece = (long long)p.piece_rows * step;
#pragma unroll 1
  for (int e = tid; e < heads * quads; e += kThreads) {
    const int h = e / quads, d = e % quads * 4;
    Sum s;
    if (parts == 1) of_warps(s, h, d);
    else of_memory(s, p.partials + (head0 + h) * p.chunks * step, step, parts, d);
    // the first piece lies in the second place of its CTA, the others in the first place of theirs
    const long long row = (long long)((unsigned)desc.y >> 16) + tile * kHeads + h;
    const float* at = first_cta < 0 ? p.whole + (head0 + h) * step : p.pieces + (2 * first_cta + 1) * piece + row * step;
    of_memory(s, at, 0, min(pieces, 1), d);
    of_memory(s, at + piece, 2 * piece, pieces - 1, d);
    const float r = s.l != 0.f ? 1.f / s.l : 0.f;  // no weight at all: zeros
    T* out = reinterpret_cast<T*>(p.out) + (head0 + h) * p.D + d;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(s.a.x * r, s.a.y * r), pack2<T>(s.a.z * r, s.a.w * r));
  }
}

template <typename T, int DP, bool SPLIT>
static int launch(const OwnParams& p, unsigned grid, cudaStream_t st) {
  using C = Cfg<DP>;
  if (!allow_smem<own_attn_kernel<T, DP, SPLIT>>(C::kSmem)) return SPD_ERR_CUDA;
  // dependent only on the prefixes' kernel: whatever else comes before may write what this one reads first
  if (p.G > 0) return launch_dependent(own_attn_kernel<T, DP, SPLIT>, dim3(grid), dim3(kThreads), C::kSmem, st, p);
  own_attn_kernel<T, DP, SPLIT><<<grid, kThreads, C::kSmem, st>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace own

// Heads of a CTA: up to eight with their weights' remainders, or sixteen.
static int own_heads(int Gq) { return Gq <= 8 ? 8 : 16; }
int own_attn_tiles(int Hq, int Hkv) {
  const int Gq = Hq / Hkv;
  return Hkv * ((Gq + own_heads(Gq) - 1) / own_heads(Gq));
}

// CTAs for each (sequence, head tile), from the longest context that the tables hold (the lengths are on the
// device): all at once if a slot's share is small, otherwise chunks of half a share that are dealt out as
// slots fall free.
Int4Split own_attn_split(int B, int Hq, int Hkv, int max_ctx, int sms) {
  constexpr int kLeast = 512, kChunk = 1024;
  const long long slots = 3ll * sms, pairs = (long long)B * own_attn_tiles(Hq, Hkv);
  const long long share = max_ctx * pairs / slots;
  if (share <= 2 * kChunk) return {(int)std::max(1ll, std::min(slots / pairs, (max_ctx + kLeast - 1ll) / kLeast)), kLeast};
  const long long c = std::min(std::max(share / 2, (long long)kChunk), 4ll * kChunk);
  return {(int)((max_ctx + c - 1) / c), kChunk};
}

int own_attn_launch(const OwnParams& p, int dtype, cudaStream_t st) {
  using namespace own;
  const long long grid = (long long)p.chunks * p.B * own_attn_tiles(p.Hq, p.Hkv);
  if (grid > 0x7fffffffll) return SPD_ERR_UNSUPPORTED;
  const bool split = p.Hq / p.Hkv <= 8;
  auto by_d = [&](auto tag) -> int {
    using T = decltype(tag);
    if (p.D > 64) return split ? launch<T, 128, true>(p, (unsigned)grid, st) : launch<T, 128, false>(p, (unsigned)grid, st);
    return split ? launch<T, 64, true>(p, (unsigned)grid, st) : launch<T, 64, false>(p, (unsigned)grid, st);
  };
  return dtype == SPD_BF16 ? by_d(__nv_bfloat16{}) : by_d(__half{});
}

}  // namespace spd
