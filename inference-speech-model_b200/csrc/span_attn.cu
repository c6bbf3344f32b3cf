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
// * Warp 0 loads: Q by TMA (3-D map), K and V by TMA boxes of a page (or of 128 keys of a plane) and 64
//   dimensions, one lane a box, table entries fetched a step ahead.  Warp 1 issues all products, warp 2
//   zeroes the rows of V tiles that are past the span's end or belong to a block id out of range (a weight
//   of zero does not silence an infinity or a NaN there), warp 3 deals the pieces.
// * Every wait is bounded; a CTA whose wait runs out lets its copies land before it exits.
#include "spd_tc_attn.cuh"

#include <algorithm>

namespace spd {
namespace span {
using namespace tc;

constexpr int BM = 128;  // rows of a tile
constexpr int BN = 128;  // keys of a step
constexpr int kThreads = 384;
constexpr int kItems = 3;       // pieces known ahead
constexpr int kFix = 8;         // requests to clean a V tile: at most one for each tile of the ring
constexpr int kHoles = 16;      // steps whose missing pages are remembered: more than can be under way
constexpr int kCostPair = 3, kCostSingle = 2;  // of a step
constexpr int kMinSteps = 4;    // steps of a share, at least

template <int DP> struct Cfg {
  static constexpr int kBoxes = DP / 64;             // 64-column boxes of a row
  static constexpr int kBox = 128 * 128;             // 128 rows of 128 bytes
  static constexpr int kTile = kBoxes * kBox;        // a Q, K or V tile
  static constexpr int kStages = DP == 128 ? 5 : 8;  // K and V tiles in flight
  static constexpr int kBarBytes = 320;
  static constexpr size_t kSmem = 1024 + (size_t)(2 + kStages) * kTile + kBarBytes;
  static constexpr uint32_t kO = 2 * BN;             // TMEM column of O_0; S_0 at 0, S_1 at BN
  static constexpr uint32_t kTmemCols = 512;
  // registers of the softmax threads and of the others; their sum is within what the launch gives to
  // all 384 (168 each, checked at the launch)
  static constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
  static constexpr int kAllRegs = 256 * kSoftmaxRegs + 128 * kOtherRegs;
  static_assert(kO + 2 * DP <= kTmemCols && kStages <= kFix, "outputs fit in TMEM, requests in their ring");
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
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
  __device__ __forceinline__ long long cost() const { return (long long)steps * (pairs * kCostPair + single * kCostSingle); }
};

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

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    span_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const SpanParams p) {
  using C = Cfg<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Piece items[kItems];
  __shared__ int gave_up;  // a wait has run out
  __shared__ int left[4];  // the loader's place in its ring, and how often it loaded each Q tile, at its end
  __shared__ volatile uint32_t holes[kHoles];  // pages of a step whose keys are left out, a bit each
  __shared__ int4 fix_what[kFix];              // ring slot, phase, first row to clear, pages to clear
  __shared__ float2 other[BM];                 // maximum and sum of the second stream's rows
  __shared__ __align__(8) uint64_t item_full[kItems], item_empty[kItems], fix_wanted[kFix], fixed[kFix], other_full, other_empty;
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  unsigned char* q_tiles = smem;                   // [2]
  unsigned char* kv_tiles = smem + 2 * C::kTile;   // [kStages]
  uint64_t* bars = reinterpret_cast<uint64_t*>(kv_tiles + C::kStages * C::kTile);
  uint64_t* kv_full = bars;                    // [kStages]
  uint64_t* kv_empty = kv_full + C::kStages;   // [kStages]
  uint64_t* q_full = kv_empty + C::kStages;    // [2]
  uint64_t* q_empty = q_full + 2;              // [2]
  uint64_t* s_full = q_empty + 2;              // [2] scores ready (and all earlier products done)
  uint64_t* p_full = s_full + 2;               // [2 streams][2] weights written, 64 keys each (and the output rescaled)
  uint64_t* o_full = p_full + 4;               // [2] output complete
  uint64_t* o_empty = o_full + 2;              // [2] output read
  uint64_t* done = o_empty + 2;                // every MMA has completed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Gq = p.Hq / p.Hkv;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  if (tid == 0) {
    gave_up = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 1);
      mbar_init(&q_empty[x], 1);
      mbar_init(&s_full[x], 1);
      for (int h = 0; h < 2; ++h) mbar_init(&p_full[2 * x + h], 4);  // one arrival per warp
      mbar_init(&o_full[x], 1);
      mbar_init(&o_empty[x], 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 11);
    }
    for (int i = 0; i < kFix; ++i) {
      mbar_init(&fix_wanted[i], 1);
      mbar_init(&fixed[i], 1);
    }
    mbar_init(&other_full, 4);
    mbar_init(&other_empty, 4);
    mbar_init(done, 1);
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Piece w;
  // The next piece as warp 3 dealt it, for a whole warp; false past the last one or after a wait that gave up.
  auto next_item = [&](int it, bool& ok, Piece& w) {
    const int slot = it % kItems;
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspend(&item_full[slot], (uint32_t)((it / kItems) & 1), p.err, p.wait_ns));
    if (!ok) return false;
    w = items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[slot]);
    return w.there != 0;
  };
  const int page_mask = (1 << p.bs_log2) - 1;
  auto pages_of = [&](int keys) { return (min(keys, BN) + page_mask) >> p.bs_log2; };

  if (warp < 4) {
    regs_down<C::kOtherRegs>();
    if (warp == 0) {
      // ---- TMA: K and V tiles of each step through one ring, in the order of their first use ------
      int q_use[2] = {0, 0}, fixes = 0, hole_at = 0;
      Ring ring;
      bool ok = true;
      for (int it = 0; next_item(it, ok, w); ++it) {
        const int n = w.j1 - w.j0;
        const int* table = p.paged ? p.tables + (long long)w.group * p.max_blocks : nullptr;
        const int plane = p.paged ? 0 : p.slots ? p.slots[w.group] : w.group;
        // lane `l` of a paged step: box l % kBoxes of page l / kBoxes
        auto look_up = [&](int j) {
          if (!p.paged || j >= w.j1) return 0;
          const int page = lane / C::kBoxes;
          return page < pages_of(w.len - j * BN) ? __ldg(table + ((j * (BN >> p.bs_log2)) + page)) : 0;
        };
        // arms the slot and copies the tile of step j (K or V); `id`: this lane's block
        auto load = [&](const CUtensorMap* map, int j, int id, uint32_t gone) {
          if (ring.round) ok = __all_sync(0xffffffffu, mbar_wait_suspend(&kv_empty[ring.slot], ring.phase() ^ 1u, p.err, p.wait_ns));
          if (!ok) return;
          unsigned char* tile = kv_tiles + ring.slot * C::kTile;
          if (p.paged) {
            const int pages = pages_of(w.len - j * BN), box = lane % C::kBoxes;
            // (pages of 8 tokens with two boxes each fill the warp exactly)
            const int page = lane / C::kBoxes;
            const bool fine = page < pages && id >= 0 && id < p.blocks;
            if (lane == 0)
              mbar_arrive_expect_tx(&kv_full[ring.slot], (uint32_t)((pages - __popc(gone)) * C::kBoxes) << (p.bs_log2 + 7));
            __syncwarp();
            if (fine) tma_load_4d(tile + box * C::kBox + (page << (p.bs_log2 + 7)), map, 64 * box, w.kvh, 0, id, &kv_full[ring.slot]);
          } else {
            if (lane == 0) mbar_arrive_expect_tx(&kv_full[ring.slot], C::kTile);
            __syncwarp();
            if (lane < C::kBoxes) tma_load_4d(tile + lane * C::kBox, map, 64 * lane, j * BN, w.kvh, plane, &kv_full[ring.slot]);
          }
          __syncwarp();
        };
        // pages of step j whose block id is out of range, a bit each
        auto missing = [&](int j, int id) {
          uint32_t gone = 0;
          if (p.paged) {
            const bool bad = lane / C::kBoxes < pages_of(w.len - j * BN) && (id < 0 || id >= p.blocks);
            const uint32_t all = __ballot_sync(0xffffffffu, bad && lane % C::kBoxes == 0);
            if (all) {
              if (bad) set_error(p.err, SPD_DEVERR_BLOCK_ID);
              for (int q = 0; q < 32 / C::kBoxes; ++q) gone |= (all >> (q * C::kBoxes) & 1u) << q;
            }
          }
          return gone;
        };
        auto load_k = [&](int j, int id) {
          const uint32_t gone = missing(j, id);
          // known before the tile is armed, to all that wait for it
          if (lane == 0) holes[(hole_at + j - w.j0) % kHoles] = gone;
          load(&tm_k, j, id, gone);
          if (ok) ring.next(C::kStages);
        };
        auto load_v = [&](int j, int id) {
          const uint32_t gone = missing(j, id);
          load(&tm_v, j, id, gone);
          if (!ok) return;
          const int keys = w.len - j * BN;
          if (keys < BN || gone) {  // have it cleaned
            if (lane == 0) {
              fix_what[fixes % kFix] = make_int4(ring.slot, (int)ring.phase(), keys, (int)gone);
              mbar_arrive(&fix_wanted[fixes % kFix]);
            }
            ++fixes;
          }
          ring.next(C::kStages);
        };
        auto load_q = [&](int x, int tok) {
          if (!ok) return;
          if (q_use[x] > 0) ok = __all_sync(0xffffffffu, mbar_wait_suspend(&q_empty[x], (uint32_t)((q_use[x] - 1) & 1), p.err, p.wait_ns));
          if (!ok) return;
          ++q_use[x];
          if (lane == 0) mbar_arrive_expect_tx(&q_full[x], (uint32_t)(C::kBoxes * p.q_rows * 128));
          __syncwarp();
          if (lane < C::kBoxes)
            tma_load_3d(q_tiles + x * C::kTile + lane * C::kBox, &tm_q, 64 * lane, w.kvh * Gq, tok, &q_full[x]);
          __syncwarp();
        };
        int id = look_up(w.j0), id_next = look_up(w.j0 + 1);
        if (w.pair) {
          load_q(0, w.tok0);
          for (int j = w.j0; j < w.j1 && ok; ++j) {
            const int ahead = look_up(j + 2);
            load_k(j, id);
            if (j == w.j0) load_q(1, w.tok0 + p.per_tile);
            if (ok) load_v(j, id);
            id = id_next;
            id_next = ahead;
          }
        } else {
          load_q(w.q_slot, w.tok0);
          if (ok) load_k(w.j0, id);
          for (int j = w.j0; j < w.j1 && ok; ++j) {
            const int ahead = look_up(j + 2);
            if (j == w.j0 && n > 1) load_k(j + 1, id_next);
            if (ok) load_v(j, id);
            if (ok && j + 2 < w.j1) load_k(j + 2, ahead);
            id = id_next;
            id_next = ahead;
          }
        }
        hole_at += n;
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
      constexpr uint32_t kTile16 = C::kTile >> 4, kBox16 = C::kBox >> 4;
      // descriptors of the first Q tile, and of the ring's first tile as K and as V
      const uint64_t q_desc = smem_desc_sw128(q_tiles), kv_desc = smem_desc_sw128(kv_tiles),
                     v_desc = smem_desc_mn(kv_tiles, C::kBox);
      const bool leader = elect_one();
      const int leader_lane = __ffs(__ballot_sync(0xffffffffu, leader)) - 1;
      uint32_t q_ph[2] = {0, 0}, p_ph[2] = {0, 0}, o_ph[2] = {1, 1};
      int fixes = 0, hole_at = 0;
      Ring ring;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t phase) {
        if (ok) ok = mbar_wait_suspend(bar, phase, p.err, p.wait_ns);
      };
      auto take = [&]() {  // the ring's next tile, once it is there
        const int slot = ring.slot;
        wait(&kv_full[slot], ring.phase());
        ring.next(C::kStages);
        return slot;
      };
      auto wait_q = [&](int x) {
        wait(&q_full[x], q_ph[x]);
        q_ph[x] ^= 1;
      };
      auto scores = [&](int x, int q, int slot) {  // S_x = Q K^T
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::kBoxes; ++c)
          umma4_ss(tmem + x * BN, q_desc + (uint64_t)(q * kTile16 + c * kBox16),
                   kv_desc + (uint64_t)(slot * kTile16 + c * kBox16), idesc_s, c != 0);
        umma_commit(&s_full[x]);
      };
      auto output = [&](int x, int slot, bool first) {  // O_x (+)= P_x V, each 64 of the keys when their weights are there
        const uint64_t dv = v_desc + (uint64_t)(slot * kTile16);
        if (first) {
          wait(&o_empty[x], o_ph[x]);  // passes at once the first time
          o_ph[x] ^= 1;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          wait(&p_full[2 * x + h], p_ph[x]);
          if (!ok) break;
          tc_fence_after();
          umma4_ts(tmem + C::kO + x * DP, tmem + x * BN + 32 * h, dv + h * 4 * 128, idesc_o, !first || h);
        }
        p_ph[x] ^= 1;
      };
      for (int it = 0; next_item(it, ok, w); ++it) {
        const int n = w.j1 - w.j0;
        if (leader) {
          // the V tile of step j, cleaned
          auto take_v = [&](int t) {
            const int slot = take();
            if (ok && (w.len - (w.j0 + t) * BN < BN || holes[(hole_at + t) % kHoles])) {
              wait(&fixed[fixes % kFix], (uint32_t)((fixes / kFix) & 1));
              ++fixes;
            }
            return slot;
          };
          // A tile is given back only if its products were issued: after a wait that gave up its copy may still
          // be in flight, and the loader must not arm its barrier again.
          if (w.pair) {
            int k = take();
            for (int x = 0; x < 2; ++x) {
              wait_q(x);
              if (!ok) break;
              scores(x, x, k);
              if (n == 1) umma_commit(&q_empty[x]);
            }
            if (ok) umma_commit(&kv_empty[k]);
            for (int t = 0; t < n && ok; ++t) {
              const int v = take_v(t);
              if (t + 1 < n) k = take();
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                if (!ok) continue;
                output(x, v, t == 0);
                if (!ok) continue;
                if (t + 1 < n) {
                  scores(x, x, k);
                  if (t + 2 == n) umma_commit(&q_empty[x]);
                } else {
                  umma_commit(&o_full[x]);
                }
              }
              if (ok) {
                umma_commit(&kv_empty[v]);
                if (t + 1 < n) umma_commit(&kv_empty[k]);
              }
            }
          } else {
            const int q = w.q_slot;
            wait_q(q);
            for (int t = 0; t < min(2, n) && ok; ++t) {
              const int k = take();
              if (!ok) break;
              scores(t, q, k);
              umma_commit(&kv_empty[k]);
              if (t + 1 == n) umma_commit(&q_empty[q]);
            }
            for (int t = 0; t < n && ok; ++t) {
              const int x = t & 1, v = take_v(t);
              output(x, v, t < 2);
              if (!ok) break;
              umma_commit(&kv_empty[v]);
              if (t + 2 < n) {
                const int k = take();
                if (!ok) break;
                scores(x, q, k);
                umma_commit(&kv_empty[k]);
                if (t + 3 == n) umma_commit(&q_empty[q]);
              } else {
                umma_commit(&o_full[x]);
              }
            }
          }
          hole_at += n;
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
      // ---- V tiles: zero where a key does not count ---------------------------------------------
      // (asked by the loader: a request's ring slot is not loaded again before its tile is cleaned and used)
      bool ok = true;
      int fixes = 0;
      for (int it = 0; next_item(it, ok, w); ++it) {
        // as many requests as the loader makes for this piece
        for (int j = w.j0; j < w.j1; ++j) {
          const int keys = w.len - j * BN;
          bool asked = keys < BN;
          if (!asked && p.paged) {
            const int* table = p.tables + (long long)w.group * p.max_blocks + j * (BN >> p.bs_log2);
            const int id = lane < (BN >> p.bs_log2) ? __ldg(table + lane) : 0;
            asked = __any_sync(0xffffffffu, id < 0 || id >= p.blocks);
          }
          if (!asked) continue;
          ok = __all_sync(0xffffffffu, mbar_wait_suspend(&fix_wanted[fixes % kFix], (uint32_t)((fixes / kFix) & 1), p.err, p.wait_ns));
          if (!ok) break;
          const int4 what = fix_what[fixes % kFix];
          ok = __all_sync(0xffffffffu, mbar_wait_suspend(&kv_full[what.x], (uint32_t)what.y, p.err, p.wait_ns));
          if (!ok) break;
          unsigned char* tile = kv_tiles + what.x * C::kTile;
          for (int r = lane >> 3; r < BN; r += 4)
            if (r >= what.z || (what.w >> (r >> p.bs_log2) & 1))
              for (int c = 0; c < C::kBoxes; ++c)
                *reinterpret_cast<uint4*>(tile + c * C::kBox + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&fixed[fixes % kFix]);
          ++fixes;
        }
        if (!ok) break;
      }
      if (!ok) gave_up = 1;
    } else {
      // ---- this CTA's share of all steps, piece by piece -----------------------------------------
      bool ok = true;
      int it = 0;
      auto hand = [&](const Piece& w) {
        const int slot = it % kItems;
        if (it >= kItems)
          ok = __all_sync(0xffffffffu, mbar_wait_suspend(&item_empty[slot], (uint32_t)((it / kItems - 1) & 1), p.err, p.wait_ns));
        if (!ok) return;
        if (lane == 0) {
          items[slot] = w;
          mbar_arrive(&item_full[slot]);
        }
        ++it;
      };
      long long total = 0;
      for (int g = lane; g < p.G; g += 32) {
        const Group s(p, g);
        total += s.cost();
        if (blockIdx.x == 0) {
          if (p.lens[g] > p.max_keys) set_error(p.err, SPD_DEVERR_LENGTH);
          if (!p.paged && p.slots && (p.slots[g] < 0 || p.slots[g] >= p.blocks)) set_error(p.err, SPD_DEVERR_BLOCK_ID);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      total *= p.Hkv;
      const int shares = (int)max(1ll, min((long long)gridDim.x, total / (kMinSteps * kCostSingle)));
      const int cta = (int)blockIdx.x;
      long long lo = 0, hi = 0;
      if (cta < shares) {
        lo = range_start(cta, shares, total);
        hi = range_start(cta + 1, shares, total);
      }
      int4 mine = make_int4(0, 0, 0, 0);  // the item that begins here and ends in a later CTA
      // the group that position `lo` lies in
      int g = p.G;
      long long base = 0;
      if (lo < hi)
        for (int first = 0; first < p.G; first += 32) {
          const long long c = first + lane < p.G ? Group(p, first + lane).cost() * p.Hkv : 0;
          long long incl = c;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
          }
          const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > lo);
          if (hit) {
            const int src = __ffs(hit) - 1;
            g = first + src;
            base += __shfl_sync(0xffffffffu, incl - c, src);
            break;
          }
          base += __shfl_sync(0xffffffffu, incl, 31);
        }
      int singles = 0;
      for (long long at = lo; at < hi && g < p.G && ok;) {
        const Group s(p, g);
        const long long head = s.cost();
        if (head == 0 || at >= base + head * p.Hkv) {
          base += head * p.Hkv;
          ++g;
          continue;
        }
        const int kvh = (int)((at - base) / head);
        const long long in_head = at - base - kvh * head, pair_cost = (long long)s.steps * kCostPair;
        const int tile2 = (int)min((long long)s.pairs, in_head / pair_cost);
        const bool pair = tile2 < s.pairs;
        const int unit = pair ? kCostPair : kCostSingle;
        const long long begin = base + kvh * head + tile2 * pair_cost, end = begin + (long long)s.steps * unit;
        // steps whose position begin + j * unit lies in [lo, hi)
        w.group = g;
        w.kvh = kvh;
        w.len = s.len;
        w.tok0 = s.tok0 + tile2 * 2 * p.per_tile;
        w.tokens = min(s.tok0 + s.tokens - w.tok0, 2 * p.per_tile);
        w.j0 = lo > begin ? (int)((lo - begin + unit - 1) / unit) : 0;
        w.j1 = hi < end ? (int)((hi - begin + unit - 1) / unit) : s.steps;
        w.pair = pair;
        const int first_cta = cta_of_unit(begin, shares, total), last_cta = cta_of_unit(end - unit, shares, total);
        w.count = last_cta - first_cta + 1;
        w.cut = w.count == 1 ? 0 : w.j0 == 0 ? 2 : 1;
        w.q_slot = singles & 1;
        w.there = 1;
        at = end;
        if (w.j0 >= w.j1) continue;
        if (!pair) ++singles;
        if (w.cut == 2) mine = make_int4(w.count, w.tok0, w.tokens, kvh);
        hand(w);
      }
      w.there = 0;
      if (ok) hand(w);
      if (p.cta_desc && lane == 0) p.cta_desc[cta] = mine;
      if (!ok) gave_up = 1;
    }
  } else {
    // ---- softmax and epilogue of stream x: thread = row = TMEM lane ---------------------------
    regs_up<C::kSoftmaxRegs>();
    const int x = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + x * BN, o_col = tmem + lanes + C::kO + x * DP;
    const int row_tok = row / Gq, row_head = row % Gq;
    int s_use = 0, o_use[2] = {0, 0}, others = 0, hole_at = 0;  // o_use: outputs completed before, of each stream
    bool ok = true;
    if (p.out) {  // queries of groups without keys: zeros
      const int per = p.Hq * p.D / 8;
      for (int g = (int)blockIdx.x; g < p.G; g += (int)gridDim.x) {
        const Group s(p, g);
        if (s.len > 0) continue;
        uint4* o = reinterpret_cast<uint4*>(p.out) + (long long)s.tok0 * per;
        for (long long i = tid - 128; i < (long long)s.tokens * per; i += 256) o[i] = make_uint4(0, 0, 0, 0);
      }
    }
    for (int it = 0; next_item(it, ok, w); ++it) {
      const int n = w.j1 - w.j0;
      const int tile_tok = w.pair ? x * p.per_tile : 0;  // of this stream's tile
      const bool live = row_tok < p.per_tile && tile_tok + row_tok < w.tokens;
      float m = -INFINITY, l = 0.f;
      const int stride = w.pair ? 1 : 2;
      const int t0 = w.pair ? 0 : x;
      for (int t = t0; t < n; t += stride) {
        ok = __all_sync(0xffffffffu, mbar_wait_suspend(&s_full[x], (uint32_t)(s_use & 1), p.err, p.wait_ns));
        ++s_use;
        if (!ok) break;
        tc_fence_after();
        uint32_t s[128];
        const int seen = w.len - (w.j0 + t) * BN;
        const uint32_t gone = holes[(hole_at + t) % kHoles];
        const bool edge = seen < BN || gone;
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
        // Also for a NaN and for infinite scores, which only the exact exponentials treat as they are.  Rows
        // that belong to no query have no say: what they hold changes no rounding of the others.
        const bool raise = live && !(mx < m + kLazy);
        bool exact = edge;
        if (__any_sync(0xffffffffu, raise)) {
          exact |= __any_sync(0xffffffffu, live && !(fabsf(mx) < INFINITY));
          const float mn = fmaxf(m, mx);
          const float f = m == mn ? 1.f : ex2_approx(m - mn);
          m = mn;
          l *= f;
          if (t > t0) {
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
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
          if (exact) weights<T, true, 32>(s + 64 * h, c2, nm2, pk, sum);
          else weights<T, false, 32>(s + 64 * h, c2, nm2, pk, sum);
          tmem_st32(s_col + 32 * h, pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * x + h]);
        }
        const float2 t2 = unpair(add2(sum[0], sum[1]));
        l += t2.x + t2.y;
      }
      if (!ok) break;
      hole_at += n;
      // A single tile's second stream leaves its output in TMEM, maximum and sum in shared memory, to the first.
      const bool two = !w.pair && n > 1;
      if (!w.pair && x == 1) {
        if (two) {
          if (others > 0) ok = __all_sync(0xffffffffu, mbar_wait_suspend(&other_empty, (uint32_t)((others - 1) & 1), p.err, p.wait_ns));
          if (!ok) break;
          other[row] = make_float2(m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(&other_full);
          ++others;
          ++o_use[1];
        }
        ++o_use[0];
        continue;
      }
      ok = __all_sync(0xffffffffu, mbar_wait_suspend(&o_full[x], (uint32_t)(o_use[x] & 1), p.err, p.wait_ns));
      if (!ok) break;
      float f0 = 1.f, f1 = 0.f;
      if (two) {
        ok = __all_sync(0xffffffffu, mbar_wait_suspend(&other_full, (uint32_t)(others & 1), p.err, p.wait_ns));
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_suspend(&o_full[1], (uint32_t)(o_use[1] & 1), p.err, p.wait_ns));
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
      ++o_use[0];
      if (w.pair || two) ++o_use[1];
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
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
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

// The items that shares cut: their pieces, added in the CTAs' order.  CTA (c, y) takes 8 rows of the item that
// begins in CTA c of the attention kernel, a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) span_join_kernel(const SpanParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 d = p.cta_desc[blockIdx.x];  // CTAs, first query, queries, key/value head
  const int Gq = p.Hq / p.Hkv, lane = threadIdx.x & 31;
  const int row = (int)(blockIdx.y * 8 + (threadIdx.x >> 5));
  if (d.x < 2 || row >= d.z * Gq) return;
  const int step = p.D + 4;
  const float* first = p.pieces + ((long long)(2 * (int)blockIdx.x + 1) * p.piece_rows + row) * step;
  const float* rest = p.pieces + ((long long)(2 * ((int)blockIdx.x + 1)) * p.piece_rows + row) * step;
  const long long next = 2ll * p.piece_rows * step;
  auto piece = [&](int i) { return i == 0 ? first : rest + (i - 1) * next; };
  float mm = -INFINITY;
  for (int i = lane; i < d.x; i += 32) mm = fmaxf(mm, piece(i)[p.D]);
  mm = warp_max(mm);
  float l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const int at = min(lane * 4, p.D - 4);
#pragma unroll 8
  for (int i = 0; i < d.x; ++i) {
    const float* r = piece(i);
    const float2 st = *reinterpret_cast<const float2*>(r + p.D);
    const float4 v = *reinterpret_cast<const float4*>(r + at);
    const float f = st.x == mm ? 1.f : ex2_approx(st.x - mm);
    l += f * st.y;
    a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
  }
  const float r = l != 0.f ? 1.f / l : 0.f;  // no weight at all: zeros
  if (lane * 4 >= p.D) return;
  T* out = reinterpret_cast<T*>(p.out) + ((long long)(d.y + row / Gq) * p.Hq + d.w * Gq + row % Gq) * p.D + at;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(a.x * r, a.y * r), pack2<T>(a.z * r, a.w * r));
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

template <typename T, int DP>
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
  if (!allow_smem<span_attn_kernel<T, DP>>(C::kSmem)) return SPD_ERR_CUDA;
  static const bool enough = [] {  // a warpgroup that asks for more registers than the CTA has would wait for good
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, span_attn_kernel<T, DP>) == cudaSuccess && a.numRegs * kThreads >= C::kAllRegs;
  }();
  if (!enough) return SPD_ERR_CUDA;
  span_attn_kernel<T, DP><<<grid, kThreads, C::kSmem, st>>>(tq, tk, tv, p);
  return cudaPeekAtLastError() == cudaSuccess ? SPD_OK : SPD_ERR_CUDA;
}

}  // namespace span

// Queries of a tile, and rows of a piece's result: two tiles, or all there are.
int span_per_tile(int Gq) { return span::BM / Gq; }
int span_piece_rows(int N, int Gq) { return std::min(2 * span_per_tile(Gq), N) * Gq; }

// The attention of all spans.  With p.out set a second kernel joins the items that were cut; otherwise the
// results stay partial, for a kernel that is launched with programmatic dependent launch.
int span_attn_launch(SpanParams p, const SpanTensors& t, int dtype, int sms, cudaStream_t st) {
  using namespace span;
  const int Gq = p.Hq / p.Hkv;
  p.per_tile = span_per_tile(Gq);
  p.q_rows = std::min(p.per_tile, p.N) * Gq;
  p.piece_rows = span_piece_rows(p.N, Gq);
  const bool bf16 = dtype == SPD_BF16;
  const int rc = p.D > 64 ? (bf16 ? launch<__nv_bfloat16, 128>(p, t, sms, st) : launch<__half, 128>(p, t, sms, st))
                          : (bf16 ? launch<__nv_bfloat16, 64>(p, t, sms, st) : launch<__half, 64>(p, t, sms, st));
  if (rc != SPD_OK || !p.out) return rc;
  const dim3 grid((unsigned)sms, (unsigned)((p.piece_rows + 7) / 8));
  return bf16 ? launch_dependent(span_join_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p)
              : launch_dependent(span_join_kernel<__half>, grid, dim3(256), 0, st, p);
}

}  // namespace spd
