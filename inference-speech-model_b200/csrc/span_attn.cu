// span_attn.cu — attention of groups of queries, each group over the keys of its own span:
//   out[i, h] = softmax_t(q[i, h] . k[t, h / Gq] * scale) . v[t, h / Gq],  t < lens[g],
// for the queries i of group g (cu[g] <= i < cu[g + 1]).  Every query of a group sees every key of its
// span, which lies in a paged pool (a prefix that candidates share) or in one plane a head (a
// request's encoder keys and values).
//
// What bounds it: a key and its value are read once for all rows of a tile (queries x the Gq heads that
// share them), 4 * rows operations for each of their 4 bytes.  With few rows that is HBM; with 256 rows
// a key and more the tensor cores and, beside them, the exponentials.
//
// sm_100a design:
// * Rows are cut into tiles of 128 (query-major, all Gq heads of a key/value head together), keys into
//   steps of 128.  S = Q K^T into TMEM, one thread a row for the softmax, P over S in TMEM, O += P V:
//   the products of prompt_attn.cu, whose pieces they share.
// * Two streams of scores a CTA, so that the tensor cores work on one while the exponentials of the
//   other run.  An item with more than 128 rows takes two tiles over the same steps; one with fewer has
//   a single tile whose steps go to the streams in turn, each with its own maximum, sum and output, which
//   are added when the item is stored.
// * Few items with many keys must fill the device: all steps of all items are laid end to end (a step of
//   two tiles costs 3, of one tile 2) and dealt to the CTAs in equal shares.  An item that a
//   share's end cuts leaves one partial result (output, maximum, sum, fp32) a piece; whoever reads
//   them adds them in their order.  A CTA has two such pieces at most, its first and its last.
// * The two streams have a ring of K and V tiles, a warp that loads and a warp that issues products each: with
//   one of either for both, their chains of instructions (some 1,000 cycles a tile) set the pace.  Loads are TMA
//   boxes of a page (or of 128 keys of a plane) and 64 dimensions, one lane a box, table entries fetched a
//   step ahead.  The issuing warp also zeroes the rows of V tiles that are past the span's end or
//   belong to a block id out of range.
// * Every wait is bounded; a CTA whose wait runs out lets its copies land before it exits.
// * Weights go into P V in the input's type, off by half a step of it (2^-8 bf16, 2^-11 fp16); maxima, sums and outputs are
//   fp32, and the sums take the weights unrounded.  Results are 1.3 times as far from 64 bits as with weights of
//   32 bits (0.0022 of 0.0017 relative in bf16, 0.00028 of 0.00021 in fp16: the output's own rounding is the rest).  The
//   remainders would take a second P V, and a second conversion and store of every weight in the chain that sets the pace.
// Measured on a B200, in CUDA graphs, with the join: 32 requests of 5 beams over up to 1,500 positions (20 heads of 64,
// bf16) 52 us, 0.45 of a copy's rate; 24 prompts of up to 448 tokens over them (fp16) 68 us, where the products alone would
// take 20 and the chain of a tile (scores, maximum, exponentials, weights, product) sets the pace; one request of 5 beams 13.0 to
// 13.7 us, of which 4 are the start and 3 to 4 the join.  Two prefixes of 32,000 tokens for 64 candidates each (bf16, 8 key/value
// heads of 128): 83 us of this kernel alone, 27 steps of two tiles a CTA at some 5,800 cycles, of which the products are 2,050.
#include "spd_tc_attn.cuh"

#include <algorithm>

namespace spd {
namespace span {
using namespace tc;

// Code size counts here: roles side by side miss the instruction cache, and each miss waits in L2 behind the
// K/V stream.  So waits are one small loop each, and the error word is set once at the end.  (32 x 5 beams over 1,500
// positions took 101 us with 134 KB of code; with this and four threads a row for few rows 51.)

// Waits for phase `parity` of `bar`, suspended, for `limit_ns` at most; false if it ran out.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, unsigned long long limit_ns) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 t0, t;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "@p bra DONE;\n\t"
      "mov.u64 t0, %%globaltimer;\n\t"
      "add.s64 t0, t0, %4;\n"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "@p bra DONE;\n\t"
      "mov.u64 t, %%globaltimer;\n\t"
      "setp.lt.u64 q, t, t0;\n\t"
      "@q bra AGAIN;\n"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity), "r"(kSuspendNs), "l"(limit_ns)
      : "memory");
  return done != 0;
}

constexpr int BM = 128;  // rows of a tile
constexpr int BN = 128;  // keys of a step
constexpr int kThreads = 384;
constexpr int kItems = 4;       // pieces known ahead, and the present one
constexpr int kHoles = 8;       // steps whose missing pages are remembered, of each kind (see Holes)
// What an item costs: so much, and so much a step of it.
constexpr int kCostItem = 4, kCostPair = 3, kCostSingle = 2;
// of a CTA, at least (one request of 5 beams 13.0 to 13.7 us, with 12 14.0; of 8 candidates 12.7, with 12 12.4; with 20 17 us each)
constexpr int kMinShare = 8;

template <int DP> struct Cfg {
  static constexpr int kBoxes = DP / 64;             // 64-column boxes of a row
  static constexpr int kBox = 128 * 128;             // 128 rows of 128 bytes
  static constexpr int kTile = kBoxes * kBox;        // a Q, K or V tile
  static constexpr int kStages = DP == 128 ? 2 : 4;  // tiles of each of the two rings (a power of two)
  static constexpr size_t kSmem = 1024 + (size_t)(2 + 2 * kStages) * kTile;
  static constexpr uint32_t kO = 2 * BN;             // TMEM column of O_0; S_0 at 0, S_1 at BN
  static constexpr uint32_t kTmemCols = 512;
  // registers of the softmax threads and of the others; their sum is within what the launch gives to
  // all 384 (168 each, checked at the launch)
  static constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
  static constexpr int kAllRegs = 256 * kSoftmaxRegs + 128 * kOtherRegs;
  static_assert(kO + 2 * DP <= kTmemCols, "scores and outputs fit in TMEM");
  static_assert(kStages + 2 <= kHoles, "an entry is free when it is written");
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar)), "l"(policy)
      : "memory");
}

// 16 rows of TMEM (from the address's lane) and 8 * 8 columns: thread t has rows t / 4 (r[4i], r[4i + 1]) and t / 4 + 8
// (r[4i + 2], r[4i + 3]), columns 8i + 2 (t % 4) and the next.
__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// The same rows, 8 * 4 columns: r[2i] is row t / 4, r[2i + 1] row t / 4 + 8, of column 4i + t % 4.
__device__ __forceinline__ void tmem_st_16x128b_x8(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Group g: its queries, clamped to what there is, and the keys they see.
struct Group {
  int tok0, tokens, len, steps, pairs, single;
  __device__ __forceinline__ Group(const SpanParams& p, int g) {
    tok0 = p.cu ? max(0, min(p.N, p.cu[g])) : g;
    tokens = p.cu ? max(tok0, min(p.N, p.cu[g + 1])) - tok0 : 1;
    len = max(0, min(p.lens[g], p.max_keys));
    if (!p.paged && p.slots && (p.slots[g] < 0 || p.slots[g] >= p.blocks)) len = 0;
    const int tiles = (tokens + p.per_tile - 1) / p.per_tile;
    steps = len / BN + (len % BN != 0);
    pairs = tiles >> 1;
    single = tiles & 1;
  }
  // of one key/value head
  __device__ __forceinline__ int cost() const {
    return steps ? pairs * (kCostItem + steps * kCostPair) + single * (kCostItem + steps * kCostSingle) : 0;
  }
};

__device__ __forceinline__ int pages_of(const SpanParams& p, int keys) {  // that a step of so many keys reads
  return (min(keys, BN) + (1 << p.bs_log2) - 1) >> p.bs_log2;
}

// One piece of work: steps [j0, j1) of one or two tiles of a group, for one key/value head.
struct Piece {
  int group, kvh, len;
  int tok0, tokens;   // queries of its tiles
  int j0, j1;
  int pair;           // two tiles over the same steps; otherwise one tile, its steps in turns
  int q_slot;         // Q tile of a single one
  int cut;            // 0: the whole item; 1: it ends here and began in an earlier CTA, or goes on; 2: it begins here
  int count;          // CTAs that share the item
  int there;          // 0 past the last one
};
// The steps of stream x: t = first, first + by, .. below n.
struct Steps {
  int n, first, by, last;
  __device__ __forceinline__ Steps(const Piece& w, int x)
      : n(w.j1 - w.j0), first(w.pair ? 0 : x), by(w.pair ? 1 : 2), last(w.pair ? n - 1 : n - 1 - ((n - 1 - x) & 1)) {}
};

// Where the missing pages of a step are remembered: single tiles' steps by stream, steps of two tiles in a third place.
// The streams of a single tile do not wait for one another before its end, so neither may use the other's entries.  An
// entry is read for the last time before its step's product of weights is issued.  A loader writes one when it
// has loaded the step before, that is, when a tile kStages further back has been given back: of single tiles that
// is a V tile, so kStages / 2 + 2 entries are in use; of two tiles' steps a K tile, given back by both streams after the
// product of the step before it, so kStages + 2 are.
struct Holes {
  int own = 0, pair = 0;  // steps before this item
  __device__ __forceinline__ int at(const Piece& w, int x, int t) const {
    return w.pair ? 2 * kHoles + (pair + t) % kHoles : x * kHoles + (own + (t >> 1)) % kHoles;
  }
  __device__ __forceinline__ void next(const Piece& w, int x) {
    const int n = w.j1 - w.j0;
    if (w.pair) pair += n;
    else own += (n + 1 - x) >> 1;
  }
};

// A row's output in TMEM times f (a row a lane).
template <int DP>
__device__ __forceinline__ void rescale(uint32_t o_col, float f) {
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

template <typename T, int DP, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1)
    span_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const SpanParams p) {
  using C = Cfg<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Piece items[kItems];
  __shared__ int gave_up;     // a wait has run out
  __shared__ int left[2][2];  // tiles that a loader copied into its ring ([1][1]: Q tiles), at its end
  __shared__ volatile uint32_t holes[3 * kHoles];  // pages of a step whose keys are left out, a bit each
  __shared__ float2 other[BM];                 // maximum and sum of the second stream's rows
  __shared__ __align__(8) uint64_t item_full[kItems], item_empty[kItems], other_full, other_empty;
  __shared__ __align__(8) uint64_t kv_full[2][C::kStages], kv_empty[2][C::kStages];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2];
  __shared__ __align__(8) uint64_t s_full[2];     // scores ready (and all earlier products of the stream done)
  __shared__ __align__(8) uint64_t p_full[2][2];  // weights written, 64 keys each (and the output rescaled)
  __shared__ __align__(8) uint64_t o_full[2], o_empty[2];  // output complete, output read
  __shared__ __align__(8) uint64_t turn[C::kStages];       // of two tiles' steps: the first stream's products are issued
  __shared__ __align__(8) uint64_t meet;          // both issuing warps are here
  __shared__ __align__(8) uint64_t done;          // every MMA has completed
  __shared__ uint32_t tmem_slot;
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  unsigned char* q_tiles = smem;                   // [2]
  unsigned char* kv_tiles = smem + 2 * C::kTile;   // [2 rings][kStages]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Gq = p.Hq / p.Hkv;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 1) tmem_alloc(&tmem_slot, C::kTmemCols);
  if (tid < 3 * kHoles) holes[tid] = 0;
  if (tid == 0) {
    gave_up = 0;
    left[0][0] = left[0][1] = left[1][0] = left[1][1] = 0;
  }
  {  // a thread a barrier
    const int i = tid - 64;
    auto init = [&](int first, int n, uint64_t* bar, uint32_t count) {
      if (i >= first && i < first + n) mbar_init(bar + (i - first), count);
    };
    init(0, 2 * C::kStages, &kv_full[0][0], 1);
    init(8, 2 * C::kStages, &kv_empty[0][0], 2);  // both streams
    init(16, 2, q_full, 1);
    init(18, 2, q_empty, 2);
    init(20, 2, s_full, 1);
    init(22, 4, &p_full[0][0], 4);  // one arrival per warp
    init(26, 2, o_full, 1);
    init(28, 2, o_empty, 4);
    init(32, kItems, item_full, 1);
    init(36, kItems, item_empty, 11);
    init(40, 1, &other_full, 4);
    init(41, 1, &other_empty, 4);
    init(42, 1, &done, 2);
    init(43, C::kStages, turn, 1);
    init(43 + C::kStages, 1, &meet, 2);
    if (i >= 0 && i < 64) fence_barrier_init();
  }
  // Warp 0 finds its share meanwhile.
  int total = 0, lo = 0, hi = 0, share = 1, g = 0, base = 0;
  if (warp == 0) {
    auto cost_of = [&](int i) { return i < p.G ? Group(p, i).cost() * p.Hkv : 0; };
    // The host refuses calls whose sum could reach 2^31 with each query in one group.  If groups overlap and it does, no
    // work is done.
    int mine = cost_of(lane);  // of group `lane`
    unsigned sum = (unsigned)mine;
    bool over = false;
#pragma unroll 4
    for (int i = lane + 32; i < p.G; i += 32) {
      sum += (unsigned)cost_of(i);
      over |= sum >> 31;
      sum &= 0x7fffffffu;
    }
    over = __any_sync(0xffffffffu, over) || __reduce_add_sync(0xffffffffu, sum >> 8) >= (1u << 23) - 32;
    total = over ? 0 : (int)__reduce_add_sync(0xffffffffu, sum);
    if (over && blockIdx.x == 0) set_error(p.err, SPD_DEVERR_LENGTH);
    const int shares = max(1, min((int)gridDim.x, total / kMinShare));
    share = max(1, (total + shares - 1) / shares);  // more than a step if there are two: every CTA between has one
    lo = (int)min((long long)total, (long long)blockIdx.x * share);
    hi = (int)min((long long)total, (long long)lo + share);
#pragma unroll 1
    for (int first = 0; lo < hi && first < p.G; first += 32) {
      if (first) mine = cost_of(first + lane);
      int incl = mine;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > lo);
      if (hit) {
        const int src = __ffs(hit) - 1;
        g = first + src;
        base += __shfl_sync(0xffffffffu, incl - mine, src);
        break;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;  // of the whole warp: no wait has run out
  auto wait = [&](uint64_t* bar, uint32_t phase) {
    if (ok) ok = __all_sync(0xffffffffu, wait_on(bar, phase & 1u, p.wait_ns));
    return ok;
  };
  Piece w;
  // The next piece as warp 0 dealt it, for a whole warp; false past the last one or after a wait that gave up.
  auto next_item = [&](int it) {
    const int slot = it % kItems;
    if (!ok || !wait(&item_full[slot], (uint32_t)(it / kItems))) return false;
    w = items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[slot]);
    return w.there != 0;
  };

  if (warp < 4) {
    regs_down<C::kOtherRegs>();
    if (warp == 0 || warp == 3) {
      // ---- TMA: K and V tiles.  Ring x has the tiles of stream x, K and V in turn; for two tiles of rows, which share
      // them, K tiles in ring 0 and V tiles in ring 1.  Warp 0 deals the pieces besides, two ahead.
      const int x = warp == 0 ? 0 : 1;
      const uint64_t policy = l2_policy_evict_first();  // (the code, the pieces and the tables stay in L2)
      const int bl7 = p.bs_log2 + 7;  // log2 of a page's bytes in one box
      unsigned char* const ring = kv_tiles + x * C::kStages * C::kTile;
      int used = 0;
      Holes hole;
      uint32_t q_seen = 0, q_odd = 0;  // of the Q tiles, a bit each: loaded before, an odd number of times

      // the share [lo, hi) of all items laid end to end: the present item starts at `at`
      int at = lo < hi ? base : hi, kvh = 0, tile2 = 0, singles = 0, dealt = 0;
      bool more = true;
      ::int4 mine = make_int4(0, 0, 0, 0);  // the item that begins here and ends in a later CTA
      Group s(p, min(g, max(0, p.G - 1)));
      if (x == 0 && lo < hi) {  // the item that `lo` lies in
        const int head = s.cost(), pair_cost = kCostItem + s.steps * kCostPair;
        kvh = (lo - at) / head;
        at += kvh * head;
        tile2 = min(s.pairs, (lo - at) / pair_cost);
        at += tile2 * pair_cost;
      }
      auto deal = [&]() {
        const int slot = dealt % kItems;
        if (dealt >= kItems && !wait(&item_empty[slot], (uint32_t)(dealt / kItems - 1))) return;
        Piece d;
        d.there = 0;
#pragma unroll 1
        while (at < hi && !d.there) {
          if (tile2 >= s.pairs + s.single || s.steps == 0) {  // the next head, or the next group with keys
            tile2 = 0;
            if (s.steps == 0 || s.tokens == 0 || ++kvh == p.Hkv) {
              kvh = 0;
              s = Group(p, ++g);  // (there is one: `hi` is not reached)
            }
            continue;
          }
          const bool pair = tile2 < s.pairs;
          const int unit = pair ? kCostPair : kCostSingle;
          // step j lies at begin + j * unit
          const int begin = at + kCostItem, end = begin + s.steps * unit;
          d.group = g;
          d.kvh = kvh;
          d.len = s.len;
          d.tok0 = s.tok0 + tile2 * 2 * p.per_tile;
          d.tokens = min(s.tok0 + s.tokens - d.tok0, 2 * p.per_tile);
          d.j0 = lo > begin ? (lo - begin + unit - 1) / unit : 0;
          d.j1 = hi < end ? max(0, hi - begin + unit - 1) / unit : s.steps;
          d.pair = pair;
          d.count = begin >= lo && end <= hi ? 1 : (end - unit) / share - begin / share + 1;
          d.cut = d.count == 1 ? 0 : d.j0 == 0 ? 2 : 1;
          d.q_slot = singles & 1;
          at = end;
          ++tile2;
          if (d.j0 >= d.j1) continue;
          singles += !pair;
          if (d.cut == 2) mine = make_int4(d.count, d.tok0, d.tokens, kvh);
          d.there = 1;
        }
        more = d.there != 0;
        if (lane == 0) {
          items[slot] = d;
          mbar_arrive(&item_full[slot]);
        }
        __syncwarp();
        ++dealt;
      };
#pragma unroll 1
      for (int it = 0; ok; ++it) {
        if (x == 0) {
          if (more && dealt == it) deal();
          if (!ok) break;
          w = items[it % kItems];
          if (!w.there) break;
        } else if (!next_item(it)) {
          break;
        }
        const Steps st(w, x);
        const int* table = PAGED ? p.tables + (long long)w.group * p.max_blocks + lane : nullptr;
        const int plane = PAGED ? 0 : p.slots ? p.slots[w.group] : w.group;
        auto look_up = [&](int t) {  // the block of page `lane` of step t, a step ahead of its use
          return PAGED && t < st.n && lane < pages_of(p, w.len - (w.j0 + t) * BN)
                     ? __ldg(table + (w.j0 + t) * (BN >> p.bs_log2)) : 0;
        };
        int id = look_up(st.first);
        if (x == 0)
#pragma unroll 1
          for (int q = w.pair ? 0 : w.q_slot; q <= (w.pair ? 1 : w.q_slot); ++q) {
            if ((q_seen >> q & 1u) && !wait(&q_empty[q], (q_odd >> q & 1u) ^ 1u)) break;
            q_seen |= 1u << q;
            q_odd ^= 1u << q;
            if (lane == 0) mbar_arrive_expect_tx(&q_full[q], (uint32_t)(C::kBoxes * p.q_rows * 128));
            __syncwarp();
            if (lane < C::kBoxes)
              tma_load_3d(q_tiles + q * C::kTile + lane * C::kBox, &tm_q, 64 * lane, w.kvh * Gq,
                          w.tok0 + (w.pair ? q * p.per_tile : 0), &q_full[q]);
          }
#pragma unroll 1
        for (int t = st.first; t < st.n && ok; t += st.by) {
          const int id_next = look_up(t + st.by);
          uint32_t bytes = C::kTile, gone = 0;  // gone: pages whose block id is out of range, a bit each
          int pages = 1;
          if constexpr (PAGED) {
            pages = pages_of(p, w.len - (w.j0 + t) * BN);
            const bool bad = lane < pages && (id < 0 || id >= p.blocks);
            gone = __ballot_sync(0xffffffffu, bad);
            if (bad) set_error(p.err, SPD_DEVERR_BLOCK_ID);
            bytes = (uint32_t)((pages - __popc(gone)) * C::kBoxes) << bl7;
            // known before K is armed, to all that wait for it
            if (lane == 0 && !(w.pair && x)) holes[hole.at(w, x, t)] = gone;
          }
#pragma unroll 1
          for (int kind = w.pair ? x : 0; kind <= (w.pair ? x : 1); ++kind) {
            const int slot = used % C::kStages;
            if (used >= C::kStages && !wait(&kv_empty[x][slot], (uint32_t)(used / C::kStages - 1))) break;
            unsigned char* tile = ring + slot * C::kTile;
            const CUtensorMap* map = kind ? &tm_v : &tm_k;
            if (lane == 0) mbar_arrive_expect_tx(&kv_full[x][slot], bytes);
            ++used;
            __syncwarp();
            // One lane issues, page after page: lanes with a page each would have their operands made uniform one by one
            // (2,600 cycles a tile of 8 pages).
#pragma unroll 1
            for (int page = 0; page < pages; ++page) {
              const int block = PAGED ? __shfl_sync(0xffffffffu, id, page) : plane;
              if ((gone >> page & 1u) || lane) continue;
#pragma unroll
              for (int box = 0; box < C::kBoxes; ++box) {
                unsigned char* to = tile + box * C::kBox + (PAGED ? page << bl7 : 0);
                if constexpr (PAGED) tma_load_4d(to, map, 64 * box, w.kvh, 0, block, &kv_full[x][slot], policy);
                else tma_load_4d(to, map, 64 * box, (w.j0 + t) * BN, w.kvh, block, &kv_full[x][slot], policy);
              }
            }
            __syncwarp();
          }
          id = id_next;
          if (x == 0 && more && dealt < it + 3) deal();  // two ahead, between copies
        }
        hole.next(w, x);
      }
      if (p.cta_desc && x == 0 && blockIdx.x == 0)  // what the lengths and slots have wrong
#pragma unroll 1
        for (int i = lane; i < p.G; i += 32)
          if (!PAGED && p.slots && (p.slots[i] < 0 || p.slots[i] >= p.blocks)) set_error(p.err, SPD_DEVERR_BLOCK_ID);
      if (x == 1 && blockIdx.x == 0)
#pragma unroll 1
        for (int i = lane; i < p.G; i += 32)
          if (p.lens[i] > p.max_keys) set_error(p.err, SPD_DEVERR_LENGTH);
      if (lane == 0) {
        left[x][0] = used;
        if (x == 0) left[1][1] = (int)(q_seen | (q_odd ^ 3u) << 2);  // Q tiles loaded, and the phases of their last loads
        if (x == 0 && p.cta_desc) p.cta_desc[blockIdx.x] = mine;
      }
      if (!ok) gave_up = 1;
    } else {
      // ---- MMA issue of stream x, by one lane ------------------------------------------------------
      const int x = warp - 1;
      constexpr uint32_t idesc_s = instr_desc_f16(kBf16, BM, BN);
      constexpr uint32_t idesc_o = instr_desc_f16(kBf16, BM, DP) | (1u << 16);  // B is MN-major
      constexpr uint32_t kTile16 = C::kTile >> 4, kBox16 = C::kBox >> 4;
      // descriptors of the first Q tile, and of the first ring's first tile as K and as V
      const uint64_t q_desc = smem_desc_sw128(q_tiles), kv_desc = smem_desc_sw128(kv_tiles),
                     v_desc = smem_desc_mn(kv_tiles, C::kBox);
      const bool leader = elect_one();
      uint32_t q_odd = 0, p_odd = 0, o_odd = 1;  // phases (q: a bit each)
      int u0 = 0, u1 = 0;                        // tiles of the two rings before this item
      Holes hole;
      bool single_before = false;
      int turns = 0, meets = 0;  // steps of two tiles; times that the two warps have met
      // A tile is given back only if its products were issued: after a wait that gave up its copy may still be in
      // flight, and the loader must not arm its barrier again.
      auto give_back = [&](uint64_t* bar) {
        umma_commit(bar);
        if (!w.pair) mbar_arrive(bar);  // for the stream that does not use it
      };
#pragma unroll 1
      for (int it = 0; next_item(it); ++it) {
        const Steps st(w, x);
        const int q = w.pair ? x : w.q_slot;
        // Each barrier's phases must be seen one by one.  Q: of both tiles, whoever uses them; a tile that this stream
        // does not use it gives back itself, once it has seen it.  (Were it given back by the stream that uses it, the
        // next copy could land, and a phase pass, before this warp came to look.)  Rings: the one that only the
        // other stream used is known to have landed once that stream's warp is here.
        if (w.pair && single_before) {
          if (lane == 0) mbar_arrive(&meet);
          if (!wait(&meet, (uint32_t)meets++)) break;
        }
        single_before = !w.pair;
#pragma unroll 1
        for (int r = w.pair ? 0 : q; r <= (w.pair ? 1 : q) && ok; ++r) {
          if (wait(&q_full[r], q_odd >> r) && lane == 0 && (r != q || st.first >= st.n)) mbar_arrive(&q_empty[r]);
          q_odd ^= 1u << r;
        }
        int k_at = w.pair ? u0 : x ? u1 : u0, v_at = w.pair ? u1 : k_at + 1;  // of the step's tiles in their rings
        const int k_ring = w.pair ? 0 : x, v_ring = w.pair ? 1 : x;
#pragma unroll 1
        for (int t = st.first - st.by; st.first < st.n && t < st.n && ok; t += st.by, v_at += st.by) {
          // The scores of the next step follow the product of this one's weights, which lie over them.  All that they
          // need is waited for before.
          const bool begin = t < st.first, more = t + st.by < st.n;
          const int k_slot = k_at % C::kStages, v_slot = v_at % C::kStages;
          // (with few tiles to a ring the next K is loaded late, and the product does not wait for it)
          const bool early = C::kStages > 2 || w.pair;
          if ((early || begin) && more && !wait(&kv_full[k_ring][k_slot], (uint32_t)(k_at / C::kStages))) break;
          if (begin) {
            v_at -= st.by;
          } else {
            const int keys = w.len - (w.j0 + t) * BN;
            if (!wait(&kv_full[v_ring][v_slot], (uint32_t)(v_at / C::kStages))) break;
            const uint32_t gone = holes[hole.at(w, x, t)];
            if (keys < BN || gone) {
              // A weight of zero does not silence an infinity or a NaN: rows that do not count become zero.  (Of two
              // tiles of rows over one V tile both streams do so.)
              unsigned char* tile = kv_tiles + (v_ring * C::kStages + v_slot) * C::kTile;
#pragma unroll 1
              for (int r = lane >> 3; r < BN; r += 4)
                if (r >= keys || (gone >> (r >> p.bs_log2) & 1))
#pragma unroll 1
                  for (int c = 0; c < C::kBoxes; ++c)
                    *reinterpret_cast<uint4*>(tile + c * C::kBox + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
              fence_proxy_async_smem();
              __syncwarp();
            }
            if (t == st.first) {
              if (!wait(&o_empty[x], o_odd)) break;  // passes at once the first time
              o_odd ^= 1;
            }
            // Two tiles over the same keys would keep in step, both at their exponentials and then both at their products
            // (4,350 cycles a step at D = 128): the second one's products go behind the first one's.
            if (w.pair && x && !wait(&turn[turns % C::kStages], (uint32_t)(turns / C::kStages))) break;
            // O += P V, each 64 of the keys when their weights are there
#pragma unroll 1
            for (int h = 0; h < 2 && wait(&p_full[x][h], p_odd); ++h)
              if (leader) {
                tc_fence_after();
                umma4_ts(tmem + C::kO + x * DP, tmem + x * BN + 32 * h,
                         v_desc + (uint64_t)((v_ring * C::kStages + v_slot) * kTile16 + h * 4 * 128), idesc_o, t != st.first || h);
              }
            if (!ok) break;
            p_odd ^= 1;
          }
          if (!early && !begin) {
            if (leader) give_back(&kv_empty[v_ring][v_slot]);
            if (more && !wait(&kv_full[k_ring][k_slot], (uint32_t)(k_at / C::kStages))) break;
          }
          if (leader) {
            if (more) {  // S = Q K^T
              if (begin || !early) tc_fence_after();
#pragma unroll
              for (int c = 0; c < C::kBoxes; ++c)
                umma4_ss(tmem + x * BN, q_desc + (uint64_t)(q * kTile16 + c * kBox16),
                         kv_desc + (uint64_t)((k_ring * C::kStages + k_slot) * kTile16 + c * kBox16), idesc_s, c != 0);
              umma_commit(&s_full[x]);
              give_back(&kv_empty[k_ring][k_slot]);
              if (t + st.by == st.last) umma_commit(&q_empty[q]);
            } else {
              umma_commit(&o_full[x]);
            }
            if (!begin) {
              if (early) give_back(&kv_empty[v_ring][v_slot]);
              if (w.pair && !x) mbar_arrive(&turn[turns % C::kStages]);
            }
          }
          turns += w.pair && !begin;
          k_at += st.by;
          __syncwarp();
        }
        u0 += w.pair ? st.n : (st.n + 1) & ~1;
        u1 += w.pair ? st.n : st.n & ~1;
        hole.next(w, x);
      }
      if (!ok) gave_up = 1;
      if (leader) umma_commit(&done);
      __syncwarp();
      (void)wait_on(&done, 0, SPD_WAIT_NS);
      __syncwarp();
    }
  } else {
    // ---- softmax and epilogue of stream x: thread = row = TMEM lane ---------------------------
    regs_up<C::kSoftmaxRegs>();
    const int x = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + x * BN, o_col = tmem + lanes + C::kO + x * DP;
    const int row_tok = row / Gq, row_head = row % Gq;
    int s_use = 0, others = 0;
    Holes hole;
    uint32_t o0 = 0, o1 = 0;  // outputs completed before, of each stream
    if (p.out) {  // queries of groups without keys: zeros
      const int per = p.Hq * p.D / 8;
#pragma unroll 1
      for (int g = (int)blockIdx.x; g < p.G; g += (int)gridDim.x) {
        const Group s(p, g);
        if (s.len > 0) continue;
        uint4* o = reinterpret_cast<uint4*>(p.out) + (long long)s.tok0 * per;
#pragma unroll 1
        for (long long i = tid - 128; i < (long long)s.tokens * per; i += 256) o[i] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll 1
    for (int it = 0; next_item(it); ++it) {
      const int n = w.j1 - w.j0;
      const int tile_tok = w.pair ? x * p.per_tile : 0;  // of this stream's tile
      const bool live = row_tok < p.per_tile && tile_tok + row_tok < w.tokens;
      const bool rows_here = __any_sync(0xffffffffu, live);
      // Up to 16 rows, all in the first warp: four threads share a row, so that it takes 32 exponentials a thread (64
      // with more than 8 rows) in place of 128, which alone take an SM quarter 1,024 cycles.
      const int rows = min(w.tokens - tile_tok, p.per_tile) * Gq;
      const bool few = rows <= 16, both = rows > 8;
      float m = -INFINITY, l = 0.f, mb = -INFINITY, lb = 0.f;  // few: of rows lane / 4 and lane / 4 + 8
      const int stride = w.pair ? 1 : 2;
      const int t0 = w.pair ? 0 : x;
#pragma unroll 1
      for (int t = t0; t < n; t += stride) {
        wait(&s_full[x], (uint32_t)(s_use));
        ++s_use;
        if (!ok) break;
        if (!rows_here) {  // nothing of this warp's rows is read: what its weights hold does not matter
          if (lane == 0) mbar_arrive(&p_full[x][0]), mbar_arrive(&p_full[x][1]);
          continue;
        }
        tc_fence_after();
        uint32_t s[128];
        const int seen = w.len - (w.j0 + t) * BN;
        const uint32_t gone = holes[hole.at(w, x, t)];
        const bool edge = seen < BN || gone;
        if (few) {
          tmem_ld_16x256b_x8(s_col, s);
          tmem_ld_16x256b_x8(s_col + 64, s + 32);
          tmem_ld_wait(s);
          tmem_ld_wait(s + 32);
          const int col = 2 * (lane & 3);
          if (edge)
#pragma unroll
            for (int c = 0; c < BN; c += 8) {
              const bool out = gone >> (c >> p.bs_log2) & 1;
              if (out || c + col >= seen) s[c / 2] = s[c / 2 + 2] = 0xff800000u;
              if (out || c + col + 1 >= seen) s[c / 2 + 1] = s[c / 2 + 3] = 0xff800000u;
            }
          auto val = [&](int i) { return __uint_as_float(s[i]); };
          float mx[2] = {val(0), val(2)};
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            mx[0] = max3_nan(mx[0], val(i), val(i + 1));
            mx[1] = max3_nan(mx[1], val(i + 2), val(i + 3));
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            mx[r] = max3_nan(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1), mx[r]);
            mx[r] = max3_nan(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2), mx[r]) * p.scale_log2;
          }
          const int quad = lane >> 2;
          if (__any_sync(0xffffffffu, (quad < rows && !(mx[0] < m + kLazy)) || (quad + 8 < rows && !(mx[1] < mb + kLazy)))) {
            const float ma = fmaxf(m, mx[0]), mc = fmaxf(mb, mx[1]);
            const float fa = m == ma ? 1.f : ex2_approx(m - ma), fb = mb == mc ? 1.f : ex2_approx(mb - mc);
            m = ma;
            mb = mc;
            l *= fa;
            lb *= fb;
            if (t > t0) {
              const float ga = __shfl_sync(0xffffffffu, fa, 4 * (lane & 7)), gb = __shfl_sync(0xffffffffu, fb, 4 * (lane & 7));
              rescale<DP>(o_col, lane < 8 ? ga : gb);
            }
          }
          const float na = m == -INFINITY ? 0.f : -m, nb = mb == -INFINITY ? 0.f : -mb;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int e = 32 * h + 4 * i;
              const float p0 = ex2_approx(fmaf(val(e), p.scale_log2, na)), p1 = ex2_approx(fmaf(val(e + 1), p.scale_log2, na));
              l += p0 + p1;
              pk[2 * i] = pack2<T>(p0, p1);
              pk[2 * i + 1] = 0;
            }
            if (both)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int e = 32 * h + 4 * i + 2;
                const float p0 = ex2_approx(fmaf(val(e), p.scale_log2, nb)), p1 = ex2_approx(fmaf(val(e + 1), p.scale_log2, nb));
                lb += p0 + p1;
                pk[2 * i + 1] = pack2<T>(p0, p1);
              }
            tmem_st_16x128b_x8(s_col + 32 * h, pk);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[x][h]);
          }
          continue;
        }
        float mx4[4];
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
          if (gone)
#pragma unroll
            for (int c = 0; c < BN; c += 8)  // (a page is 8 keys at least)
              if (gone >> (c >> p.bs_log2) & 1)
#pragma unroll
                for (int k = 0; k < 8; ++k) s[c + k] = 0xff800000u;
        }
        max4<64, true>(s, mx4);  // while the other half is on its way
        if (!edge) {
          tmem_ld_wait(s + 64);
          tmem_ld_wait(s + 96);
        }
        max4<64, false>(s + 64, mx4);
        const float mx = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * p.scale_log2;
        // (also for a NaN; rows that belong to no query have no say)
        const bool raise = live && !(mx < m + kLazy);
        if (__any_sync(0xffffffffu, raise)) {
          const float mn = fmaxf(m, mx);
          const float f = m == mn ? 1.f : ex2_approx(m - mn);
          m = mn;
          l *= f;
          if (t > t0) rescale<DP>(o_col, f);
        }
        const float mm = m == -INFINITY ? 0.f : m;
        const f32x2 c2 = pair(p.scale_log2, p.scale_log2), nm2 = pair(-mm, -mm);
        f32x2 sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
        // 64 keys at a time, handed to the tensor cores when they are written
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
          weights<T, true, 32>(s + 64 * h, c2, nm2, pk, sum);
          tmem_st32(s_col + 32 * h, pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[x][h]);
        }
        const float2 t2 = unpair(add2(sum[0], sum[1]));
        l += t2.x + t2.y;
      }
      if (!ok) break;
      hole.next(w, x);
      if (few) {  // back to a row a lane
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          l += __shfl_xor_sync(0xffffffffu, l, o);
          lb += __shfl_xor_sync(0xffffffffu, lb, o);
        }
        const int from = 4 * (lane & 7);
        const float ma = __shfl_sync(0xffffffffu, m, from), mc = __shfl_sync(0xffffffffu, mb, from);
        const float la = __shfl_sync(0xffffffffu, l, from), lc = __shfl_sync(0xffffffffu, lb, from);
        m = lane < 8 ? ma : mc;
        l = lane < 8 ? la : lc;
      }
      // A single tile's second stream leaves its output in TMEM, maximum and sum in shared memory, to the first.
      const bool two = !w.pair && n > 1;
      if (!w.pair && x == 1) {
        if (two) {
          if (others > 0) wait(&other_empty, (uint32_t)(others - 1));
          if (!ok) break;
          other[row] = make_float2(m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(&other_full);
          ++others;
          ++o1;
        }
        ++o0;
        continue;
      }
      wait(&o_full[x], (uint32_t)((x ? o1 : o0)));
      if (!ok) break;
      float f0 = 1.f, f1 = 0.f;
      if (two) {
        wait(&other_full, (uint32_t)(others));
        if (ok) wait(&o_full[1], (uint32_t)(o1));
        if (!ok) break;
        const float2 st = other[row];
        ++others;
        __syncwarp();
        if (lane == 0) mbar_arrive(&other_empty);
        const float mm = fmaxf(m, st.x);
        f0 = m == mm ? 1.f : ex2_approx(m - mm);
        f1 = st.x == mm ? 1.f : ex2_approx(st.x - mm);
        m = mm;
        l = l * f0 + st.y * f1;
      }
      ++o0;
      if (w.pair || two) ++o1;
      tc_fence_after();
      const int tok = w.tok0 + tile_tok + row_tok, head = w.kvh * Gq + row_head;
      const bool direct = p.out && w.cut == 0;
      if (direct) {
        const float r = l != 0.f ? 1.f / l : 0.f;  // every weight zero: zeros
        f0 *= r;
        f1 *= r;
      }
      T* out = reinterpret_cast<T*>(p.out) + ((long long)tok * p.Hq + head) * p.D;
      float* part = w.cut == 0 ? p.whole + ((long long)tok * p.Hq + head) * (p.D + 4)
                               : p.pieces + ((long long)(2 * (int)blockIdx.x + (w.cut == 2)) * p.piece_rows +
                                             (tile_tok + row_tok) * Gq + row_head) * (p.D + 4);
#pragma unroll 1
      for (int c = 0; c < (rows_here ? DP : 0); c += 32) {
        uint32_t o[32];
        tmem_ld32_nowait(o_col + c, o);
        tmem_ld_wait(o);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f0);
        if (two) {
          uint32_t o1[32];
          tmem_ld32_nowait(o_col + DP + c, o1);
          tmem_ld_wait(o1);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(o1[k]), f1, __uint_as_float(o[k])));
        }
#pragma unroll
        for (int k = 0; k < 32; k += 8)
          if (live && c + k < p.D) {
            if (direct) {
              uint4 v;
              v.x = pack2<T>(__uint_as_float(o[k]), __uint_as_float(o[k + 1]));
              v.y = pack2<T>(__uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
              v.z = pack2<T>(__uint_as_float(o[k + 4]), __uint_as_float(o[k + 5]));
              v.w = pack2<T>(__uint_as_float(o[k + 6]), __uint_as_float(o[k + 7]));
              *reinterpret_cast<uint4*>(out + c + k) = v;
            } else {
              *reinterpret_cast<uint4*>(part + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
              *reinterpret_cast<uint4*>(part + c + k + 4) = make_uint4(o[k + 4], o[k + 5], o[k + 6], o[k + 7]);
            }
          }
      }
      if (live && !direct) {
        *reinterpret_cast<float2*>(part + p.D) = make_float2(m, l);
        if (p.row_desc && row_head == 0 && w.cut != 1)
          p.row_desc[(long long)tok * p.Hkv + w.kvh] =
              make_int2(w.count == 1 ? -1 : (int)blockIdx.x, w.count | ((tile_tok + row_tok) * Gq) << 16);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&o_empty[x]);
        if (two) mbar_arrive(&o_empty[1]);
      }
    }
    if (!ok) gave_up = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (gave_up) {
    // Some warp gave up, perhaps on a copy that is still in flight: all land before the CTA exits.
    if (tid == 0) {
      set_error(p.err, SPD_DEVERR_TIMEOUT);
#pragma unroll 1
      for (int x = 0; x < 2; ++x) {
#pragma unroll 1
        for (int u = max(0, left[x][0] - C::kStages); u < left[x][0]; ++u)
          (void)wait_on(&kv_full[x][u % C::kStages], (uint32_t)(u / C::kStages) & 1u, SPD_WAIT_NS);
        if (left[1][1] >> x & 1) (void)wait_on(&q_full[x], (uint32_t)(left[1][1] >> (2 + x)) & 1u, SPD_WAIT_NS);
      }
    }
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::kTmemCols);
}

// The items that shares cut: their pieces, added in the CTAs' order.  CTAs (c, .) take the item that begins in CTA c
// of the attention kernel, a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) span_join_kernel(const SpanParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ::int4 d = p.cta_desc[blockIdx.x];  // CTAs, first query, queries, key/value head
  if (d.x < 2) return;
  const int Gq = p.Hq / p.Hkv, lane = threadIdx.x & 31, step = p.D + 4, at = min(lane * 4, p.D - 4);
  const long long next = 2ll * p.piece_rows * step;
#pragma unroll 1
  for (int row = (int)(blockIdx.y * 8 + (threadIdx.x >> 5)); row < d.z * Gq; row += 8 * (int)gridDim.y) {
    const float* first = p.pieces + ((long long)(2 * (int)blockIdx.x + 1) * p.piece_rows + row) * step;
    const float* rest = first + (1ll * p.piece_rows) * step;  // of the next CTA
    float mm = -INFINITY;
#pragma unroll 1
    for (int i = lane; i < d.x; i += 32) mm = fmaxf(mm, (i ? rest + (i - 1) * next : first)[p.D]);
    mm = warp_max(mm);
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* r = first;
#pragma unroll 4
    for (int i = 0; i < d.x; ++i) {
      const float2 st = *reinterpret_cast<const float2*>(r + p.D);
      const float4 v = *reinterpret_cast<const float4*>(r + at);
      r = rest + i * next;
      const float f = st.x == mm ? 1.f : ex2_approx(st.x - mm);
      l += f * st.y;
      a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
    }
    const float s = l != 0.f ? 1.f / l : 0.f;  // no weight at all: zeros
    T* out = reinterpret_cast<T*>(p.out) + ((long long)(d.y + row / Gq) * p.Hq + d.w * Gq + row % Gq) * p.D + at;
    if (lane * 4 < p.D) *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(a.x * s, a.y * s), pack2<T>(a.z * s, a.w * s));
  }
}

// A 16-bit tensor of up to four dimensions (strides in elements), box of 64 elements of the first.
static bool make_map4(CUtensorMap* map, const void* base, const long long (&dims)[4], const long long (&strides)[3],
                      const int (&box)[4], int rank, bool bf16) {
  auto enc = encode_fn();
  if (!enc) return false;
  cuuint64_t d[4], st[3];
  cuuint32_t b[4], estr[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) d[i] = (cuuint64_t)dims[i], b[i] = (cuuint32_t)box[i];
  for (int i = 0; i < 3; ++i) st[i] = (cuuint64_t)strides[i] * 2;
  return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank,
             const_cast<void*>(base), d, st, b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, bool PAGED>
static int launch(const SpanParams& p, const SpanTensors& t, int grid, cudaStream_t st) {
  using C = Cfg<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap tq, tk, tv;
  if (!make_map4(&tq, t.q, {p.D, p.Hq, p.N, 1}, {t.q_sh, t.q_st, 0}, {64, p.Hq / p.Hkv, p.q_rows / (p.Hq / p.Hkv), 1}, 3, kBf16))
    return SPD_ERR_CUDA;
  for (int i = 0; i < 2; ++i) {
    CUtensorMap* m = i ? &tv : &tk;
    const void* base = i ? t.v : t.k;
    const bool fine =
        p.paged ? make_map4(m, base, {p.D, p.Hkv, 1ll << p.bs_log2, p.blocks},
                            {p.D, (long long)p.Hkv * p.D, ((long long)p.Hkv * p.D) << p.bs_log2}, {64, 1, 1 << p.bs_log2, 1}, 4,
                            kBf16)
                : make_map4(m, base, {p.D, p.max_keys, p.Hkv, p.blocks}, {t.kv_st, t.kv_sh, t.kv_sb}, {64, BN, 1, 1}, 4, kBf16);
    if (!fine) return SPD_ERR_CUDA;
  }
  if (!allow_smem<span_attn_kernel<T, DP, PAGED>>(C::kSmem)) return SPD_ERR_CUDA;
  static const bool enough = [] {  // a warpgroup that asks for more registers than the CTA has would wait for good
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, span_attn_kernel<T, DP, PAGED>) == cudaSuccess && a.numRegs * kThreads >= C::kAllRegs;
  }();
  if (!enough) return SPD_ERR_CUDA;
  span_attn_kernel<T, DP, PAGED><<<grid, kThreads, C::kSmem, st>>>(tq, tk, tv, p);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace span

// Queries of a tile, and rows of a piece's result: two tiles, or all there are.
int span_per_tile(int Gq) { return span::BM / Gq; }
int span_piece_rows(int N, int Gq) { return std::min(2 * span_per_tile(Gq), N) * Gq; }

// Whether positions in the line of all steps stay below 2^31, whatever the lengths.
bool span_fits(int N, int G, int Hq, int Hkv, int max_keys) {
  const double tiles = G + (double)N / span_per_tile(Hq / Hkv), steps = max_keys / span::BN + 1;
  return Hkv * tiles * (steps * span::kCostPair + span::kCostItem) < 2147483647.0 - (1 << 20);
}

// The attention of all spans.  With p.out set a second kernel joins the items that were cut; otherwise the
// results stay partial, for a kernel that is launched with programmatic dependent launch.
int span_attn_launch(SpanParams p, const SpanTensors& t, int dtype, int sms, cudaStream_t st) {
  using namespace span;
  const int Gq = p.Hq / p.Hkv;
  p.per_tile = span_per_tile(Gq);
  if (!span_fits(p.N, p.G, p.Hq, p.Hkv, p.max_keys)) return SPD_ERR_UNSUPPORTED;
  p.q_rows = std::min(p.per_tile, p.N) * Gq;
  p.piece_rows = span_piece_rows(p.N, Gq);
  const bool bf16 = dtype == SPD_BF16;
  auto by_d = [&](auto tag, auto paged) -> int {
    using E = decltype(tag);
    constexpr bool P = decltype(paged)::value;
    return p.D > 64 ? launch<E, 128, P>(p, t, sms, st) : launch<E, 64, P>(p, t, sms, st);
  };
  auto by_place = [&](auto tag) { return p.paged ? by_d(tag, std::true_type{}) : by_d(tag, std::false_type{}); };
  const int rc = bf16 ? by_place(__nv_bfloat16{}) : by_place(__half{});
  if (rc != SPD_OK || !p.out) return rc;
  const dim3 grid((unsigned)sms, (unsigned)std::min(16, (p.piece_rows + 7) / 8));
  return bf16 ? launch_dependent(span_join_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p)
              : launch_dependent(span_join_kernel<__half>, grid, dim3(256), 0, st, p);
}

}  // namespace spd
