// Attention of drafted tokens over a paged cache for many query rows a key head (cache_attention.cu has the operator, the kernel for few
// rows and the join of shared items): tcgen05 over tiles of 128 rows.
//
// A (sequence, key head) has new tokens times query heads rows; a unit is 64 keys of one tile of 128 rows, or of two tiles
// that share the K and V (PAIR).  Each CTA has two softmax groups of four warps (thread = row) and an MMA-issuing warp for either:
//   * PAIR: group g has row tile g, both take every key tile;
//   * else one row tile, whose key tiles the groups take in turn, each with scores, O and statistics of its own, put together at the end
//     of the CTA's part of the item.
// S = Q.K^T into one of two TMEM buffers a group, P back over its scores as 16-bit pairs, O += P.V from there.  S runs two key tiles ahead of
// P.V, and a ring stage holds what an MMA warp takes in one step: V of key tile b and K of tile b + 2.
//
// Stages are filled by TMA, page by page.  Key tiles that reach behind lengths[b] are checked by a warp of their own before their values
// are used: rows behind the last key become zeros, and so do infinities and NaN, because their product with a weight of zero would reach
// rows that do not see them; if there were any, rows that do see them get them back when O is stored.
//
// 8-bit caches: the products take the codes as they are (kind::f8f6f4), and what meets them is written as a sum of 8-bit values, one
// MMA each.  A query row, scaled by a power of two to at most 256, becomes two e4m3 terms (bf16) or three (fp16) whose sum is the query but
// for what lies 2^-17 below the row's largest element.  A weight becomes a half, 2^12.75 at the reference A, and the half three e5m2 terms
// (bf16; 2^-9 of the weight in all, where bf16 weights have 2^-8) or four (fp16; exact).  e5m2 has the half's exponents: what is lost of a
// small weight is 2^-17, 2^-29.75 of the weight at A, so that thousands of keys beside a dominant one keep theirs.  (Two e4m3 terms end at
// 2^-15.75 of it: the rest of 2000 keys, e^-11 each, vanished.  They took 120 us where this takes 129, 16 x 6000 keys, 96 rows a head.)
// A moves when the maximum grew by more than 2^3.  Converting the codes to halves instead took four warps 1.6 us a tile (2.5 us a tile of
// 64 rows in all).
// Keys' scales multiply the scores; values' scales the weights, w = 2^(s + v - A): v is the tile's largest, as one number in the exponent,
// and a factor for every key relative to it.  The row sum has no part in the values' scales and is kept in units of 2^B of its own.  The
// checking warp prepares the scales.
//
// In the common path A goes by the tile's largest score and largest scale, which may be of two keys: what is lost of a weight is then up to
// 2^-24.75 of the largest.  8-bit tiles whose values' scales span more than 2^5 ("wide"), or lie 2^100 below A, take a path of rolled loops
// over tensor memory, which takes 2.4 times as long (16 x 6000 keys, 96 rows a head, scales all over: 316 us).  (Code that runs once an
// item has to be fetched: unrolled for masked tiles, too, it cost up to 20 us a tile.)
//
// What bounds it: up to 128 rows HBM, 0.77 us a 16-bit tile of 64 keys a SM (32 sequences of 8000 keys, 64 rows a head 180 us); else the
// softmax groups (some 1700 clk for 64 keys of 256 rows, of which 1024 exponentials: 64 new tokens over 8 x 32000 keys 422 us in short
// bursts, 502 under load).  At 8 bits the softmax groups throughout, 1.16 us a tile, for the terms of their weights (16 x 6000 keys, 96
// rows a head 129 us).
// Every mbarrier wait is bounded (ptx.cuh); no TMA load uses cluster multicast.
#include <algorithm>
#include <cfloat>

#include "attention_common.cuh"
#include "cache_attention.cuh"
#include "work_split.cuh"

namespace fb {
namespace {
using namespace attn;
using namespace cache;

constexpr int BN = kTileKeys;
constexpr int kThreadsTiles = 384;  // warps 0-3, 4-7: softmax groups; 8: TMA; 9, 10: MMA; 11: checks values, prepares scales
constexpr int kWarpFix = 11;
constexpr int kInfos = 8;            // key tiles whose scales are kept, for either group
constexpr uint32_t kNarrow = 5;      // log2: scales of a tile's values that lie this close share a reference, up to that much above any weight
constexpr float kTop8 = 12.75f;      // log2 of the 8-bit weight at the reference
constexpr float kRescale8 = 3.f;     // 8-bit: the reference moves when the maximum grew by more than this (together 2^15.75, e5m2 ends at 2^15.8)

// the scales of a key tile, 8-bit caches
struct alignas(16) TileInfo {
  float k[64];     // of the keys
  float v[64];     // of the values, relative to 2^v_log2
  float log2_v[64];  // log2 of the scales of the values
  float v_log2;
  int wide;
  int pad[2];
};

template <bool QBF16, bool E4M3, int D, bool PAIR>
struct TilesSmem {
  static constexpr int kElem = E4M3 ? 1 : 2;
  static constexpr int kTerms = E4M3 ? (QBF16 ? 2 : 3) : 1;  // of a query
  static constexpr int kQTile = BM * D * kElem;              // a term of a row tile
  static constexpr int kKv = BN * D * kElem;                 // a K or V tile
  static constexpr int kStage = 2 * kKv;                     // K, then V
  static constexpr int kQTiles = PAIR ? 2 : 1;
  static constexpr int kStages = E4M3 ? (PAIR ? 6 : 8) : (D == 128 ? (PAIR ? 4 : 6) : 8);
  static constexpr int kRing = kQTiles * kTerms * kQTile;
  static constexpr int kScales = kRing + kStages * kStage;  // [stages][128] exponents of the K tile's keys and values
  static constexpr int kInfo = kScales + (E4M3 ? kStages * 128 : 0);
  static constexpr int kBar = kInfo + (E4M3 ? 2 * kInfos * (int)sizeof(TileInfo) : 0);
  static constexpr int kTotal = kBar + 1024 + 1024;
  static_assert(kTotal <= 232448, "ring and tiles must fit");
};

// Shared-memory descriptor of rows of 128 or 64 bytes in the swizzle of that width: K-major, 8 rows apart; MN-major, 8 k apart
template <int ROW>
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(1) << 16) | (static_cast<uint64_t>(8 * ROW >> 4) << 32) |
         (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(ROW == 128 ? 2 : 4) << 61);
}
// byte `at` of a tile of such rows
template <int ROW>
__device__ __forceinline__ uint32_t swizzled(uint32_t at) {
  return at ^ (ROW == 128 ? ((at >> 7) & 7) << 4 : ((at >> 7) & 3) << 4);
}
// Four halves (not negative) as sums of TERMS e5m2 values.  An e5m2 value is the upper byte of a half, so every term but the last is what
// three bits hold of the rest, and the rest is exact.  Four terms hold the half's 11 bits, three are off by 2^-9 of it at most, and
// either by half of the smallest e5m2 step, 2^-17.
template <int TERMS>
__device__ __forceinline__ void terms_of(uint32_t ha, uint32_t hb, uint32_t (&term)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS - 1; ++t) {
    term[t] = __byte_perm(ha, hb, 0x7531);
    const uint32_t ba = ha & 0xff00ff00u, bb = hb & 0xff00ff00u;
    const __half2 ra = __hsub2(*reinterpret_cast<const __half2*>(&ha), *reinterpret_cast<const __half2*>(&ba));
    const __half2 rb = __hsub2(*reinterpret_cast<const __half2*>(&hb), *reinterpret_cast<const __half2*>(&bb));
    ha = *reinterpret_cast<const uint32_t*>(&ra);
    hb = *reinterpret_cast<const uint32_t*>(&rb);
  }
  if (TERMS == 4) {  // (two bits are left, or what lies below the smallest step)
    term[TERMS - 1] = __byte_perm(ha + 0x00800080u, hb + 0x00800080u, 0x7531);
  } else {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "cvt.rn.satfinite.e5m2x2.f16x2 a, %1;\n\t"
        "cvt.rn.satfinite.e5m2x2.f16x2 b, %2;\n\t"
        "mov.b32 %0, {a, b};\n\t}\n"
        : "=r"(term[TERMS - 1])
        : "r"(ha), "r"(hb));
  }
}

template <bool QBF16, bool E4M3, int D, bool PAIR>
__global__ void __launch_bounds__(kThreadsTiles, 1)
    cache_attention_tiles_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                                 const CacheAttnParams p) {
  using L = TilesSmem<QBF16, E4M3, D, PAIR>;
  constexpr int kRows = PAIR ? 2 * BM : BM;
  constexpr bool OWN_KV = !PAIR;  // each MMA warp has key tiles, and stages of the ring, of its own
  constexpr int kBoxes = E4M3 ? 1 : D / 64, kBoxBytes = BM * 128, kKvBoxBytes = BN * 128;  // (16-bit: column blocks of 128 bytes)
  constexpr int kStages = L::kStages, kOwnStages = OWN_KV ? kStages / 2 : kStages;
  constexpr int kElem = L::kElem;
  constexpr int kPTerms = !E4M3 ? 1 : QBF16 ? 3 : 4;  // of a weight
  constexpr int kPWords = E4M3 ? kPTerms : 2;         // of four weights, or of two and two
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* kv_full = bars;            // [8]
  uint64_t* kv_empty = bars + 8;       // [8]
  uint64_t* fixed = bars + 16;         // [8] the stage's values are checked, the scales of its keys prepared
  uint64_t* s_full = bars + 32;        // [2 groups][2 buffers] the scores of a key tile are complete
  uint64_t* p_ready = bars + 36;       // [2 groups][2 buffers] its probabilities are written
  uint64_t* o_done = bars + 40;        // [2 groups][2] of an item all P.V but the last, all P.V are complete
  uint64_t* q_full = bars + 44;        // [2]
  uint64_t* turn = bars + 46;          // [2] the MMA warps issue in turn
  uint64_t* xchg = bars + 48;          // [1] the two softmax groups meet
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 49);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* bad_values = tmem_slot + 2;  // [8] by item: number + 1 of one in which infinities or NaN were taken out of values
  int* tokens = reinterpret_cast<int*>(bars + 56);  // [8 key tiles][4 pieces of 16 keys] where they are in the cache
  PlanShared* plan_shared = reinterpret_cast<PlanShared*>(bars + 72);
  static_assert(72 * 8 + sizeof(PlanShared) <= 1024, "barriers and plan must fit");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto ring_stage = [](int n, int group) -> int { return (OWN_KV ? group * kOwnStages : 0) + n % kOwnStages; };
  auto ring_phase = [](int n) -> uint32_t { return (n / kOwnStages) & 1; };

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], E4M3 ? 1 + 32 : 1);         // (the lanes that copy exponents arrive, too)
      mbar_init(&kv_empty[i], (OWN_KV ? 1 : 2) + 1);  // MMA warps that read the stage, and the checking warp
      mbar_init(&fixed[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], PAIR ? 128 : 256);
      mbar_init(&turn[i], 1);
    }
    mbar_init(xchg, 256);
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) bad_values[i] = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == kWarpMma) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Plan plan = make_plan<kThreadsTiles>(p, kRows, plan_shared);

  // What the roles agree on about an item: key tiles [tile0, tile0 + n), of which group g takes every one, or every second.
  struct Work {
    int tile0, n, keys, rows, nq[2], first_masked;
  };
  auto work_of = [&](const Cursor& c) {
    Work w;
    w.tile0 = c.tile;
    w.n = c.tiles_here();
    w.keys = c.seq.length + c.seq.count;
    w.rows = min(kRows, c.seq.count * p.group - c.rt * kRows);
    w.nq[0] = PAIR ? w.n : (w.n + 1) / 2;
    w.nq[1] = PAIR ? (w.rows > BM ? w.n : 0) : w.n / 2;
    w.first_masked = c.seq.length / BN;  // key tiles from this one on are not seen whole by every row
    return w;
  };
  // key tile of group g's b-th
  auto tile_of = [](const Work& w, int b, int g) { return w.tile0 + (PAIR ? b : 2 * b + g); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kWarpTma) {
      // ------------------------------------------------------------------ TMA producer
      // K's tiles come in order, and V's after them: the tokens of the last eight are kept for V.
      int loaded[2] = {0, 0};  // stages filled so far, over all items; OWN_KV: for either MMA warp
      bool ok = true;
      const int box = min(p.t.page, BN);  // rows a load brings
      PageWalk walk;
      for (Cursor c(p, plan, kRows); c.left > 0 && ok; c.next_item(p, kRows)) {
        const Work w = work_of(c);
        walk.enter(p, p.t.table + c.b * p.t.stride, w.keys, c.h, w.tile0, lane);
        for (int b = -2; b < w.nq[0] && ok; ++b) {
#pragma unroll
          for (int g = 0; g < (OWN_KV ? 2 : 1); ++g) {
            const bool has_k = b + 2 < w.nq[g], has_v = b >= 0 && b < w.nq[g];
            if (!ok || !(has_k || has_v)) continue;
            const int k_tile = tile_of(w, b + 2, g), v_tile = tile_of(w, b, g);
            int k_token = 0;
            if (has_k) {
              k_token = walk.token(p, k_tile, lane);
              if (k_tile + 1 < w.tile0 + w.n) walk.look_up(p, k_tile + 1, lane);
              if (lane < 4) tokens[(k_tile & 7) * 4 + lane] = k_token;
            }
            const int v_token = has_v ? tokens[(v_tile & 7) * 4 + (lane & 3)] : 0;
            const int st = ring_stage(loaded[g], g);
            uint64_t* const full = &kv_full[st];
            ok = mbar_wait_warp(&kv_empty[st], ring_phase(loaded[g]) ^ 1, abort_flag, p.status, ST_CACHE_KV);
            if (!ok) continue;
            ++loaded[g];
            const int k_boxes = has_k ? min(BN / box, (w.keys - k_tile * BN + box - 1) / box) : 0;
            const int v_boxes = has_v ? min(BN / box, (w.keys - v_tile * BN + box - 1) / box) : 0;
            if (elect_one()) mbar_expect_tx(full, (uint32_t)((k_boxes + v_boxes) * box * D * kElem));
            __syncwarp();
            unsigned char* at = smem + L::kRing + st * L::kStage;
            if (E4M3) {
              if (lane < 8 && has_k && k_tile * BN + (lane & 3) * 16 < w.keys)
                copy16(smem + L::kScales + st * 128 + lane * 16, (lane < 4 ? p.k_exponent : p.v_exponent) + k_token);
              copies_arrive(full);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (i >= (x ? v_boxes : k_boxes)) break;
                const int token = uniform_of(x ? v_token : k_token, i * (box >> 4), lane);
                if (elect_one()) {
#pragma unroll
                  for (int d = 0; d < kBoxes; ++d)
                    tma_load_2d(at + x * L::kKv + d * kKvBoxBytes + i * box * (E4M3 ? D : 128), x ? &tmap_v : &tmap_k, full, d * 64, token);
                }
              }
            __syncwarp();
          }
        }
      }
    } else if (warp == kWarpMma || warp == kWarpMma + 1) {
      // ------------------------------------------------------------------ MMA issuers, one warp per softmax group
      // tcgen05 operations of ONE thread execute in issue order: S(b + 2) overwrites P(b) after P(b).V(b) has read it.  With 16-bit caches the
      // two warps issue in turn, so that one's waits lie behind the other's MMAs (64 new tokens over 8 x 32000 keys 462 -> 424 us); with 8-bit
      // ones the softmax groups are slower than the MMAs, and turns would tie them together (24 over 16 x 6000 keys 115 -> 121).  One
      // elected lane issues.
      const int mq = __shfl_sync(0xffffffffu, warp - kWarpMma, 0);
      // (kind::f8f6f4 has the fields of kind::f16; type 0 is e4m3 there, and 1, of the weights, e5m2)
      constexpr uint32_t idesc_s = umma_idesc_f16(BM, BN, QBF16 && !E4M3, false, false);
      constexpr uint32_t idesc_o = umma_idesc_f16(BM, D, QBF16 && !E4M3, false, true) | (E4M3 ? 1u << 7 : 0u);
      const uint32_t q_tile = smem_u32(smem) + (PAIR ? mq * L::kTerms * L::kQTile : 0);
      const uint64_t dq = E4M3 ? desc_rows<D>(q_tile) : umma_desc_kmajor_sw128(q_tile);
      const uint64_t dk = E4M3 ? desc_rows<D>(smem_u32(smem + L::kRing)) : umma_desc_kmajor_sw128(smem_u32(smem + L::kRing));
      const uint64_t dv = E4M3 ? desc_rows<D>(smem_u32(smem + L::kRing + L::kKv))
                               : umma_desc_mnmajor_sw128(smem_u32(smem + L::kRing + L::kKv), kKvBoxBytes, 1024);
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
      const uint32_t t_sq = tmem + mq * 128;        // the two buffers of scores, 64 columns each
      const uint32_t t_oq = tmem + 256 + mq * 128;  // O
      int turns = 0, taken = 0, begun = 0, finished = 0, items = 0;
      bool ok = true;
      for (Cursor c(p, plan, kRows); c.left > 0 && ok; c.next_item(p, kRows)) {
        const Work w = work_of(c);
        const int n_mine = w.nq[mq], n_max = OWN_KV ? n_mine : w.n;  // key tiles: used, followed
        const int n_steps = w.nq[0];                                  // the same for both MMA warps
        const bool in_turn = !E4M3 && w.nq[1] > 0;                    // a lone warp issues as it comes
        // (a barrier whose item has no key tile for this warp is neither arrived on nor waited for: the warp could be items behind)
        if (n_mine > 0) {
          ok = mbar_wait_warp(&q_full[mq], items & 1, abort_flag, p.status, ST_CACHE_Q);
          ++items;
        }
        for (int b = -2; b < n_steps && ok; ++b) {
          const bool staged = b + 2 < n_max || (b >= 0 && b < n_max);  // a stage of the ring comes with this step
          const bool use_p = b >= 0 && b < n_mine, use_s = b + 2 < n_mine;
          const int st = ring_stage(taken, mq), buf = finished & 1;
          // (8-bit: every stage passes the checking warp, which prepares the scales)
          uint64_t* const stage_bar = E4M3 ? &fixed[st] : &kv_full[st];
          if (use_p && staged)
            ok = mbar_wait_both(&p_ready[2 * mq + buf], (finished >> 1) & 1, stage_bar, ring_phase(taken), abort_flag, p.status, ST_CACHE_P,
                                ST_CACHE_KV);
          else if (staged)
            ok = mbar_wait(stage_bar, ring_phase(taken), abort_flag, p.status, ST_CACHE_KV);
          if (!E4M3 && ok && use_p && tile_of(w, b, mq) >= w.first_masked)
            ok = mbar_wait(&fixed[st], ring_phase(taken), abort_flag, p.status, ST_CACHE_KV);
          if (ok && in_turn) ok = mbar_wait(&turn[mq], (turns & 1) ^ (mq ^ 1), abort_flag, p.status, ST_CACHE_S);
          turns += in_turn;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t at = static_cast<uint64_t>((st * L::kStage) >> 4);
          if (use_p) {
            ++finished;
            if (elect_one()) {
              if (E4M3) {
#pragma unroll
                for (int t = 0; t < kPTerms; ++t)
#pragma unroll
                  for (int kk = 0; kk < BN / 32; ++kk)
                    umma_f8_ts(t_oq, t_sq + buf * BN + t * 16 + kk * 8, dv + at + static_cast<uint64_t>((kk * 32 * D) >> 4), idesc_o,
                               (b > 0 || t > 0 || kk > 0) ? 1u : 0u);
              } else {
#pragma unroll
                for (int kk = 0; kk < BN / 16; ++kk)
                  umma_f16_ts(t_oq, t_sq + buf * BN + kk * 8, dv + at + static_cast<uint64_t>((kk * 2048) >> 4), idesc_o,
                              (b > 0 || kk > 0) ? 1u : 0u);
              }
            }
          }
          if (use_s) {
            const int s_buf = begun & 1;
            ++begun;
            if (elect_one()) {
              if (E4M3) {
#pragma unroll
                for (int t = 0; t < L::kTerms; ++t)
#pragma unroll
                  for (int kk = 0; kk < D / 32; ++kk)
                    umma_f8_ss(t_sq + s_buf * BN, dq + static_cast<uint64_t>((t * L::kQTile + kk * 32) >> 4),
                               dk + at + static_cast<uint64_t>((kk * 32) >> 4), idesc_s, t > 0 || kk > 0);
              } else {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                  umma_f16_ss(t_sq + s_buf * BN, dq + static_cast<uint64_t>(((kk / 4) * kBoxBytes + (kk % 4) * 32) >> 4),
                              dk + at + static_cast<uint64_t>(((kk / 4) * kKvBoxBytes + (kk % 4) * 32) >> 4), idesc_s, kk != 0);
              }
              if (in_turn) mbar_arrive(&turn[mq ^ 1]);
              umma_commit(&s_full[2 * mq + s_buf]);
            }
          } else if (in_turn && elect_one()) {
            mbar_arrive(&turn[mq ^ 1]);
          }
          if (use_p && b >= n_mine - 2 && elect_one()) umma_commit(&o_done[2 * mq + (b == n_mine - 1)]);
          if (staged) {
            if (elect_one()) {
              if (use_p || use_s) umma_commit(&kv_empty[st]); else mbar_arrive(&kv_empty[st]);
            }
            ++taken;
          }
        }
      }
    } else if (warp == kWarpFix) {
      // ------------------------------------------------------------------ values that not every row sees; scales
      // It follows every stage, since the parity of a phase two back reads like its own, and releases it too.
      int followed[2] = {0, 0}, infos[2] = {0, 0}, items = 0;
      bool ok = true;
      for (Cursor c(p, plan, kRows); c.left > 0 && ok; c.next_item(p, kRows)) {
        const Work w = work_of(c);
        for (int b = -2; b < w.nq[0] && ok; ++b) {
#pragma unroll 1
          for (int g = 0; g < (OWN_KV ? 2 : 1); ++g) {
            const bool has_k = b + 2 < w.nq[g], has_v = b >= 0 && b < w.nq[g];
            if (!ok || !(has_k || has_v)) continue;
            const int st = ring_stage(followed[g], g);
            ok = mbar_wait_warp(&kv_full[st], ring_phase(followed[g]), abort_flag, p.status, ST_CACHE_KV);
            if (!ok) continue;
            ++followed[g];
            if (E4M3 && has_k) {
              // (The place is free: the tile eight before this one is long done, since S runs two tiles ahead of P.V, and the ring's
              // stages bring few more.)
              TileInfo* info = reinterpret_cast<TileInfo*>(smem + L::kInfo) + g * kInfos + (infos[g] + b + 2) % kInfos;
              const uint8_t* scales = smem + L::kScales + st * 128;
              const int left = w.keys - tile_of(w, b + 2, g) * BN;
              // Rows of zeros, and what is no larger than 2^-117, have the least scale: it does not make a tile wide.
              uint32_t e[2], top = 0, low = 255;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int key = lane + 32 * i;
                e[i] = key < left ? scales[64 + key] : 1u;
                top = max(top, e[i]);
                low = min(low, e[i] <= 1u ? 255u : e[i]);
                info->k[key] = key < left ? scale_of(scales[key]) : 1.f;
                info->log2_v[key] = e[i] == 255u ? __uint_as_float(0x7fc00000u) : (float)((int)e[i] - 127);
              }
              top = __reduce_max_sync(0xffffffffu, top);
              low = __reduce_min_sync(0xffffffffu, low);
              if (top <= 1u) top = low = 127;
#pragma unroll
              for (int i = 0; i < 2; ++i) info->v[lane + 32 * i] = __uint_as_float((uint32_t)max((int)e[i] - (int)top + 127, 0) << 23);
              if (lane == 0) {
                info->v_log2 = (float)((int)top - 127);
                info->wide = top - low > kNarrow || top > 187u || low < 67u;
              }
            }
            const int tile = tile_of(w, b, g);
            if (has_v && tile >= w.first_masked) {
              const int left = w.keys - tile * BN;  // rows of the tile that are keys
              bool bad = false;
              unsigned char* v = smem + L::kRing + st * L::kStage + L::kKv;
#pragma unroll 1
              for (int e0 = lane; e0 < L::kKv / 16; e0 += 32 * 8) {
                uint4 x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4*>(v + (e0 + 32 * i) * 16);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  // (the swizzle moves 16-byte pieces inside lines of 128 bytes; the line tells the key, of 64-byte rows the piece too)
                  const uint32_t at = swizzled<E4M3 ? D : 128>((e0 + 32 * i) * 16);
                  const int key = E4M3 ? at / D : at % kKvBoxBytes / 128;
                  uint32_t* y = reinterpret_cast<uint32_t*>(&x[i]);
                  uint32_t take = 0;
#pragma unroll
                  for (int n = 0; n < 4; ++n) {
                    const uint32_t m = key < left ? (E4M3 ? __vcmpeq4(y[n] & 0x7f7f7f7fu, 0x7f7f7f7fu)
                                                          : __vcmpeq2(y[n] & (QBF16 ? 0x7f807f80u : 0x7c007c00u), QBF16 ? 0x7f807f80u : 0x7c007c00u))
                                                  : 0xffffffffu;
                    bad |= key < left && m != 0;
                    y[n] &= ~m;
                    take |= m;
                  }
                  if (take) *reinterpret_cast<uint4*>(v + (e0 + 32 * i) * 16) = x[i];
                }
              }
              fence_proxy_async_smem();
              if (bad) bad_values[items & 7] = items + 1;
            }
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&fixed[st]);
              mbar_arrive(&kv_empty[st]);
            }
          }
        }
        infos[0] += w.nq[0];
        infos[1] += w.nq[1];
        ++items;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ------------------------------------------------------------------ softmax groups
    const int q = warp >> 2;    // this group: its row tile, or its share of the key tiles
    const int quad = warp & 3;  // TMEM lane quadrant this warp may touch
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem_base + q * 128 + lane_addr;
    const uint32_t t_o = tmem_base + 256 + q * 128 + lane_addr;
    int steps = 0;         // key tiles of this group so far, over all items: buffer and phase of s_full
    int ends[2] = {0, 0};  // items with two key tiles or more, with one or more so far: the phases of o_done
    int meets = 0, items = 0;
    int infos = 0;  // key tiles of the items before: the places of their scales
    bool ok = true;
    auto meet = [&]() {  // of the two groups
      tc_fence_before_sync();
      mbar_arrive(xchg);
      if (ok) ok = mbar_wait_warp(xchg, meets & 1, abort_flag, p.status, ST_CACHE_O);
      ++meets;
      tc_fence_after_sync();
    };
    // A row's query: 16 bytes a piece.  Where the groups share a tile, each brings half of every row (of an 8-bit cache it reads the whole,
    // whose largest element sets the scale).  Halves are loaded while the item before ends (32 sequences of 8000 keys, 64 rows a head: 11
    // of 187 us); whole rows would take registers that the epilogue needs.
    constexpr int kPieces = D / 8 / (PAIR ? 1 : 2), kLoads = E4M3 ? D / 8 : kPieces;
    constexpr bool kEarly = !E4M3 && !PAIR;
    const int first = PAIR ? 0 : q * kPieces;
    struct Place {
      int r, i_new, head;
      bool valid;
    };
    auto place_of = [&](const Cursor& c) {  // this thread's row of the item
      Place at;
      at.r = c.rt * kRows + (PAIR ? q * BM : 0) + row;  // of the (sequence, key head)
      at.valid = at.r < c.seq.count * p.group;
      at.i_new = at.valid ? at.r / p.group : 0;  // its new token
      at.head = c.h * p.group + (at.valid ? at.r - at.i_new * p.group : 0);
      return at;
    };
    auto load_query = [&](uint4 (&x)[kLoads], const Cursor& c) {
      const Place at = place_of(c);
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + (int64_t)(c.seq.first + at.i_new) * p.q_row +
                                                        (int64_t)at.head * p.q_head);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) x[i] = at.valid ? __ldg(src + (E4M3 ? 0 : first) + i) : make_uint4(0, 0, 0, 0);
    };
    Cursor c(p, plan, kRows);
    uint4 early[kLoads];
    if (kEarly && c.left > 0) load_query(early, c);
    while (c.left > 0 && ok) {
      const Work w = work_of(c);
      const Seq seq = c.seq;
      const int n_tiles = w.nq[q];
      const Place at = place_of(c);
      const bool valid = at.valid;
      const int i_new = at.i_new;

      // ---- the query, to its place in the swizzled tile.  (The products that read the tile before are complete: all of their scores have
      // been read, by both groups where they share it.)  A scale of zero is one of queries of zeros, so that -inf stays what it is.
      float row_scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
      {
        unsigned char* tile = smem + (PAIR ? q * L::kTerms * L::kQTile : 0);
        const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a negative scale goes into the queries)
        uint4 x[kLoads];
        if (!kEarly) load_query(x, c);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          if (kEarly) x[i] = early[i];
          if (p.scale_log2 == 0.f) x[i] = make_uint4(0, 0, 0, 0);
        }
        if (!E4M3) {
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const int n = first + i;
            *reinterpret_cast<uint4*>(tile + (n >> 3) * kBoxBytes + row * 128 + (((n & 7) ^ (row & 7)) << 4)) =
                make_uint4(x[i % kLoads].x ^ flip, x[i % kLoads].y ^ flip, x[i % kLoads].z ^ flip, x[i % kLoads].w ^ flip);
          }
        } else {
          auto pair_of = [&](uint32_t y) {
            return QBF16 ? make_float2(__uint_as_float(y << 16), __uint_as_float(y & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&y));
          };
          uint32_t most = 0;  // magnitudes of 16-bit floats compare as integers
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const uint32_t y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int n = 0; n < 4; ++n) most = __vmaxu2(most, y[n] & 0x7fff7fffu);
          }
          most = max(most & 0xffffu, most >> 16);
          // scaled by a power of two to a largest magnitude in [128, 256)
          const uint32_t e = min(max(__float_as_uint(pair_of(most).x) >> 23, 9u), 253u);
          const float up = __uint_as_float((254u + 7u - e) << 23);
          row_scale *= __uint_as_float((e - 7u) << 23);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {  // 16 elements: 16 bytes of every term
            if (!PAIR && i / (D / 32) != q) continue;
            const uint4 y0 = x[2 * i % kLoads], y1 = x[(2 * i + 1) % kLoads];
            const uint32_t y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
            uint32_t term[3][4] = {};
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              float2 left = pair_of(y[n] ^ flip);
              left = make_float2(left.x * up, left.y * up);
              // (infinities would saturate: NaN, as their scores are)
              if (!(fabsf(left.x) <= FLT_MAX)) left.x = __uint_as_float(0x7fc00000u);
              if (!(fabsf(left.y) <= FLT_MAX)) left.y = __uint_as_float(0x7fc00000u);
#pragma unroll
              for (int t = 0; t < L::kTerms; ++t) {
                const uint32_t codes = float2_to_e4m3x2(left.x, left.y);
                const uint32_t back = e4m3x2_to_half2(codes);
                const float2 is = __half22float2(*reinterpret_cast<const __half2*>(&back));
                left = make_float2(left.x - is.x, left.y - is.y);
                term[t][n >> 1] |= codes << (16 * (n & 1));
              }
            }
#pragma unroll
            for (int t = 0; t < L::kTerms; ++t)
              *reinterpret_cast<uint4*>(tile + t * L::kQTile + swizzled<D>(row * D + i * 16)) =
                  make_uint4(term[t][0], term[t][1], term[t][2], term[t][3]);
          }
        }
        fence_proxy_async_smem();
        if (!PAIR || n_tiles > 0) mbar_arrive(&q_full[PAIR ? q : 0]);
        if (!PAIR && w.nq[1] > 0) mbar_arrive(&q_full[1]);
      }

      float a_ref = -FLT_MAX;  // log2: what the stored weights and O are relative to
      float l_sum = 0.f, b_ref = -FLT_MAX;  // the row sum is l_sum * 2^b_ref (16-bit caches: b_ref stands for a_ref)
      uint32_t sr[2][32];                   // the scores of a key tile
      auto load_scores = [&]() {            // of step `steps`
        tc_fence_after_sync();
#pragma unroll
        for (int x = 0; x < 2; ++x) tmem_ld_32x32b_x32(t_s + (steps & 1) * BN + x * 32, sr[x]);
      };
      auto wait_scores = [&]() {
        if (ok) ok = mbar_wait_warp(&s_full[2 * q + (steps & 1)], (steps >> 1) & 1, abort_flag, p.status, ST_CACHE_S);
        if (ok) load_scores();
      };
      if (n_tiles > 0) wait_scores();
      for (int i = 0; i < n_tiles && ok; ++i) {
        const int buf = steps & 1, tile = tile_of(w, i, q);
        const TileInfo* info = reinterpret_cast<const TileInfo*>(smem + L::kInfo) + (PAIR ? 0 : q) * kInfos + (infos + i) % kInfos;
        ++steps;
        tmem_ld_wait();
        const bool more = i + 1 < n_tiles;
        const bool masked = tile >= w.first_masked;
        constexpr float kThreshold = E4M3 ? kRescale8 : kRescaleThreshold;
        constexpr float kTop = E4M3 ? kTop8 : QBF16 ? kTopWide : kTopHalf;  // log2 of the weight at the reference
        // Takes a new reference where it grew by more than the threshold: rare.  O is rescaled in tensor memory.
        auto settle = [&](float most) {
          const float a_new = fmaxf(a_ref, most);
          if (!__any_sync(0xffffffffu, a_new - a_ref > kThreshold)) return;
          const float factor = ex2f(a_ref - a_new);
          a_ref = a_new;
          if (!E4M3) l_sum *= factor;
          if (i == 0) return;  // (nothing is there yet)
          // O must be complete up to the key tile before this one (the scores of the next one come after that product)
          ok = more ? mbar_wait_warp(&s_full[2 * q + (buf ^ 1)], (steps >> 1) & 1, abort_flag, p.status, ST_CACHE_S)
                    : mbar_wait_warp(&o_done[2 * q], ends[0] & 1, abort_flag, p.status, ST_CACHE_O);
          if (!ok) return;
          tc_fence_after_sync();
#pragma unroll 1
          for (int x = 0; x < D / 32; ++x) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_o + x * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(scaled(__uint_as_float(o[e]), factor));
            tmem_st_32x32b_x32(t_o + x * 32, o);
          }
        };
        auto add_sum = [&](float sum, float unit) {  // sum * 2^unit to the row sum, 8-bit
          if (sum == 0.f) unit = b_ref;  // (the row sees nothing of the tile, whose unit may be far above)
          if (unit > b_ref) {
            l_sum *= ex2f(b_ref - unit);
            b_ref = unit;
          }
          l_sum = fmaf(sum, ex2f(unit - b_ref), l_sum);
        };
        uint32_t pk[kPWords][16];  // the weights' first and second 32 keys (16-bit), or their terms
        // What the row sees of the tile's keys, a bit a key.  The warp's rows belong to a few neighbouring tokens: the warp reads each one's
        // mask side by side, eight tokens' at a time.
        auto look = [&](uint32_t (&see)[2]) {
          const int a0 = tile * BN - seq.length + lane, a1 = a0 + 32;  // the lane's two keys, counted from the first new token
          const int width = p.mask ? min(p.mask_width, seq.count) : seq.count;
          const bool may0 = a0 >= 0 && a0 < width, may1 = a1 >= 0 && a1 < width;
          const int t0 = __shfl_sync(0xffffffffu, i_new, 0), t1 = __reduce_max_sync(0xffffffffu, i_new);
          see[0] = see[1] = 0;
#pragma unroll 1
          for (int t = min(t0, t1); t <= t1; t += 8) {
            bool lo[8], hi[8];
            const uint8_t* m = p.mask + (int64_t)(seq.first + t) * p.mask_stride;
#pragma unroll
            for (int n = 0; n < 8; ++n, m += p.mask_stride) {
              const bool there = t + n <= t1;
              lo[n] = a0 < 0 || (there && may0 && (p.mask ? __ldg(m + a0) != 0 : a0 <= t + n));
              hi[n] = a1 < 0 || (there && may1 && (p.mask ? __ldg(m + a1) != 0 : a1 <= t + n));
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const uint32_t l = __ballot_sync(0xffffffffu, lo[n]), h = __ballot_sync(0xffffffffu, hi[n]);
              if (t + n == i_new) {
                see[0] = l;
                see[1] = h;
              }
            }
          }
          __syncwarp();
        };
        // Masked tiles: by selection in the common path where the groups share the rows (32 sequences of 8000 keys, 64 rows a head: 2 us
        // less), in the rolled path where they do not, whose common path is the slower for it (64 new tokens over 8 x 32000 keys 425 -> 461).
        const bool inline_mask = !PAIR && masked;
        bool rolled = (PAIR && masked) || (E4M3 && info->wide != 0);
        uint32_t see[2] = {0xffffffffu, 0xffffffffu};
        if (inline_mask) look(see);
        float mx = -INFINITY;  // the largest score
        if (!rolled) {
          if (E4M3) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 f = *reinterpret_cast<const float4*>(info->k + x * 32 + e * 4);
                const float2 lo = mul2_rn(make_float2(__uint_as_float(sr[x][4 * e]), __uint_as_float(sr[x][4 * e + 1])), make_float2(f.x, f.y));
                const float2 hi = mul2_rn(make_float2(__uint_as_float(sr[x][4 * e + 2]), __uint_as_float(sr[x][4 * e + 3])), make_float2(f.z, f.w));
                sr[x][4 * e] = __float_as_uint(lo.x); sr[x][4 * e + 1] = __float_as_uint(lo.y);
                sr[x][4 * e + 2] = __float_as_uint(hi.x); sr[x][4 * e + 3] = __float_as_uint(hi.y);
              }
          }
          if (inline_mask) {  // (the row's scale is positive: -inf stays -inf)
#pragma unroll
            for (int e = 0; e < 32; ++e)
#pragma unroll
              for (int x = 0; x < 2; ++x)
                if (!((see[x] >> e) & 1u)) sr[x][e] = 0xff800000u;
          }
          float mxc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains of the row maximum
#pragma unroll
          for (int e = 0; e < 16; ++e)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              mxc[2 * x + (e & 1)] = max3f(mxc[2 * x + (e & 1)], __uint_as_float(sr[x][2 * e]), __uint_as_float(sr[x][2 * e + 1]));
          mx = max3f(mxc[0], mxc[1], fmaxf(mxc[2], mxc[3])) * row_scale;
          const float most = E4M3 ? mx + info->v_log2 : mx;
          // The common path has one exponential for the weight and the row sum.  Where A stands 2^100 above the tile's weights (values of
          // tiles before were that much larger), the exponentials would leave 32 bits' range, and the sum with them: rolled.
          constexpr float kFar = 100.f, kMid = (kFar - kThreshold) / 2.f;
          if (!E4M3) {
            settle(most);
          } else if (__any_sync(0xffffffffu, fabsf(most - a_ref + kMid) > kMid + kThreshold)) {  // (one vote for both)
            rolled = __any_sync(0xffffffffu, mx > -FLT_MAX && a_ref - most > kFar);
            if (!rolled) settle(most);
          }
          if (!ok) break;
        }
        if (!rolled) {
          const float v_log2 = E4M3 ? info->v_log2 : 0.f;
          const float unit = a_ref - v_log2 - kTop;  // the exponentials are 2^(score - unit)
          const float2 scale2 = make_float2(row_scale, row_scale), neg2 = make_float2(-unit, -unit);
          float2 sa = make_float2(0.f, 0.f), sb = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            // 16-bit: a pair of either half; 8-bit: four neighbouring keys
            const int xa = E4M3 ? e >> 3 : 0, xb = E4M3 ? e >> 3 : 1, ya = E4M3 ? (e & 7) * 4 : 2 * e, yb = E4M3 ? ya + 2 : 2 * e;
            const float2 ta = fma2(make_float2(__uint_as_float(sr[xa][ya]), __uint_as_float(sr[xa][ya + 1])), scale2, neg2);
            const float2 tb = fma2(make_float2(__uint_as_float(sr[xb][yb]), __uint_as_float(sr[xb][yb + 1])), scale2, neg2);
            float2 ea = make_float2(ex2f(ta.x), ex2f(ta.y));
            float2 eb = make_float2(ex2f(tb.x), ex2f(tb.y));
            sa = add2(sa, ea);
            sb = add2(sb, eb);
            if (!E4M3) {
              pk[0][e] = pack16<QBF16>(ea.x, ea.y);
              pk[1][e] = pack16<QBF16>(eb.x, eb.y);
            } else {
              const float4 f = *reinterpret_cast<const float4*>(info->v + e * 4);
              ea = mul2_rn(ea, make_float2(f.x, f.y));
              eb = mul2_rn(eb, make_float2(f.z, f.w));
              uint32_t term[kPWords];
              terms_of(pack16<false>(ea.x, ea.y), pack16<false>(eb.x, eb.y), term);
#pragma unroll
              for (int t = 0; t < kPWords; ++t) pk[t][e] = term[t];
            }
          }
          const float2 tot = add2(sa, sb);
          if (E4M3) add_sum(tot.x + tot.y, unit); else l_sum += tot.x + tot.y;
        } else {
          if (PAIR && masked) look(see);
          // In rolled loops over 16 keys: the scores, scaled, in tensor memory again, -inf for what the row does not see; their maxima.
          mx = -INFINITY;
          float mw = -INFINITY;  // largest score plus scale of the value
#pragma unroll 1
          for (int x = 0; x < BN / 16; ++x) {
            uint32_t y[16];
            __syncwarp();
            tmem_ld_32x32b_x16(t_s + buf * BN + x * 16, y);
            tmem_ld_wait();
            const uint32_t bits = (x & 2 ? see[1] : see[0]) >> (16 * (x & 1));
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float v = __uint_as_float(y[e]) * (E4M3 ? info->k[x * 16 + e] * row_scale : row_scale);
              if (!((bits >> e) & 1u)) v = -INFINITY;
              y[e] = __float_as_uint(v);
              mx = fmaxf(mx, v);
              if (E4M3) mw = fmaxf(mw, v + info->log2_v[x * 16 + e]);
            }
            tmem_st_32x32b_x16(t_s + buf * BN + x * 16, y);
          }
          __syncwarp();
          tmem_st_wait();
          settle(E4M3 ? mw : mx);
          if (!ok) break;
          if (E4M3 && mx > b_ref) {
            l_sum *= ex2f(b_ref - mx);
            b_ref = mx;
          }
          // the weights; what the loop makes of 16 keys is put into its place by selection, since P is written where scores still are
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e)
#pragma unroll
            for (int t = 0; t < kPWords; ++t) pk[t][e] = 0;
#pragma unroll 1
          for (int x = 0; x < BN / 16; ++x) {
            uint32_t y[16], a[8];
            __syncwarp();
            tmem_ld_32x32b_x16(t_s + buf * BN + x * 16, y);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float wgt[2];
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float v = __uint_as_float(y[2 * e + n]);
                const float pr = ex2f(v - (E4M3 ? b_ref : a_ref - kTop));
                sum += pr;
                // (what is not seen weighs nothing, whatever its value's scale is)
                wgt[n] = !E4M3 ? pr : v == -INFINITY ? 0.f : ex2f(v + info->log2_v[x * 16 + 2 * e + n] - a_ref + kTop);
              }
              a[e] = pack16<QBF16 && !E4M3>(wgt[0], wgt[1]);
            }
            if (E4M3) {
              uint32_t term[4][kPWords];
#pragma unroll
              for (int e = 0; e < 4; ++e) terms_of(a[2 * e], a[2 * e + 1], term[e]);
#pragma unroll
              for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int t = 0; t < kPWords; ++t) pk[t][e] = e / 4 == x ? term[e % 4][t] : pk[t][e];
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                pk[0][e] = e / 8 == x ? a[e % 8] : pk[0][e];
                pk[1][e] = e / 8 + 2 == x ? a[e % 8] : pk[1][e];
              }
            }
          }
          l_sum += sum;
        }
        // (the scores read ahead take the registers of this tile's)
        const bool ahead = __all_sync(0xffffffffu, more && mbar_test(&s_full[2 * q + (steps & 1)], (steps >> 1) & 1));
        if (ahead) load_scores();
        // P is written over the scores it comes from
#pragma unroll
        for (int t = 0; t < kPWords; ++t) tmem_st_32x32b_x16(t_s + buf * BN + t * 16, pk[t]);
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(&p_ready[2 * q + buf]);
        if (more && !ahead) wait_scores();
      }
      Cursor next = c;
      next.next_item(p, kRows);
      if (kEarly && next.left > 0) load_query(early, next);
      if (ok && n_tiles > 0) ok = mbar_wait_warp(&o_done[2 * q + 1], ends[1] & 1, abort_flag, p.status, ST_CACHE_O);
      if (!ok) break;
      tc_fence_after_sync();
      ends[0] += n_tiles > 1;
      ends[1] += n_tiles > 0;

      // ---- O: scaled to the units of the row sum, and out: whole, or as a part for the join
      const float m_mine = E4M3 ? b_ref : a_ref;
      float f[2] = {E4M3 ? ex2f(a_ref - kTop8 - b_ref + kTopWide) : 1.f, 0.f}, m = m_mine;
      if (E4M3) l_sum *= kUnitWide;
      float l = l_sum;
      if (l_sum == 0.f) f[0] = 0.f;
      if (!PAIR) {
        meet();  // all scores have been read: the statistics take the queries' place
        float4* stat = reinterpret_cast<float4*>(smem);
        stat[q * BM + row] = make_float4(m_mine, l_sum, f[0], 0.f);
        meet();
        if (!ok) break;
        const float4 s0 = stat[row], s1 = stat[BM + row];
        // a half that saw no key counts for nothing
        const float m0 = s0.y == 0.f ? -INFINITY : s0.x, m1 = s1.y == 0.f ? -INFINITY : s1.x;
        m = fmaxf(m0, m1);
        const float w0 = s0.y == 0.f ? 0.f : ex2f(m0 - m), w1 = s1.y == 0.f ? 0.f : ex2f(m1 - m);
        l = s0.y * w0 + s1.y * w1;
        f[0] = s0.z * w0;
        f[1] = s1.z * w1;
      } else if (l == 0.f) {
        m = -INFINITY;
      }
      const bool whole = w.tile0 == 0 && w.n == c.kt;
      float* part = p.partials + ((size_t)blockIdx.x * 2 + (c.first_item ? 0 : 1)) * partial_floats(kRows, D);
      const int part_row = (PAIR ? q * BM : 0) + row;
      const bool has_rows = PAIR ? q * BM < w.rows : true;
      if (has_rows) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        uint16_t* const out = static_cast<uint16_t*>(p.out) + (int64_t)(seq.first + i_new) * p.out_row +
                              (int64_t)at.head * p.out_head;
        const bool bad = bad_values[items & 7] == (uint32_t)items + 1;
        constexpr int kChunks = D / 32 / (PAIR ? 1 : 2);  // of 32 columns: each group stores half where they share the rows
        for (int x = PAIR ? 0 : q * kChunks; x < (PAIR ? kChunks : (q + 1) * kChunks); ++x) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_32x32b_x32(tmem_base + 256 + (PAIR ? q * 128 : 0) + lane_addr + x * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(scaled(__uint_as_float(o[e]), f[0]));  // (NaN stays, however small its weight)
          if (!PAIR && w.nq[1] > 0) {
            uint32_t o1[32];
            tmem_ld_32x32b_x32(tmem_base + 256 + 128 + lane_addr + x * 32, o1);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(__uint_as_float(o[e]) + scaled(__uint_as_float(o1[e]), f[1]));
          }
          if (bad && valid) {
            // infinities and NaN that were taken out of the values of partly seen tiles: rows that see them get them
            for (int key = max(w.tile0, w.first_masked) * BN; key < min(w.keys, (w.tile0 + w.n) * BN); ++key) {
              if (!sees(p, seq, i_new, key - seq.length)) continue;
              const int page = __ldg(p.t.table + c.b * p.t.stride + (key >> p.t.page_log2));
              if (page < 0 || page >= p.t.pages) continue;
              const int64_t at = ((((int64_t)page * p.t.heads + c.h) << p.t.page_log2) + (key & (p.t.page - 1))) * D + x * 32;
              for (int e = 0; e < 32; ++e) {
                float v = 0.f;
                if (E4M3) {
                  if ((__ldg(static_cast<const uint8_t*>(p.v_pages) + at + e) & 0x7f) == 0x7f) v = __uint_as_float(0x7fc00000u);
                } else {
                  const uint16_t bits = __ldg(static_cast<const uint16_t*>(p.v_pages) + at + e);
                  const uint16_t expo = QBF16 ? 0x7f80 : 0x7c00;
                  if ((bits & expo) == expo) v = QBF16 ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits));
                }
                if (v != 0.f) {
#pragma unroll
                  for (int y = 0; y < 32; ++y)
                    if (y == e) o[y] = __float_as_uint(__uint_as_float(o[y]) + v);
                }
              }
            }
          }
          if (valid) {
            if (whole) {
              store_row32<QBF16, E4M3>(out, x, o, inv);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) store32(part + (size_t)part_row * D + x * 32 + e * 8, o + e * 8);
            }
          }
        }
        if (!whole && valid && (PAIR || q == 0)) {
          __stcg(part + (size_t)kRows * D + part_row, m);
          __stcg(part + (size_t)kRows * D + kRows + part_row, l);
        }
      }
      ++items;
      infos += PAIR ? w.n : n_tiles;
      c = next;
      if (!PAIR) meet();  // both groups are done with the statistics, the queries and both O
    }
  }

  // ------------------------------------------------------------------ teardown
  if (*abort_flag) {
    unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kWarpMma) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

template <bool QBF16, bool E4M3, int D, bool PAIR>
int launch_tiles(frisk_b200_ctx* ctx, const CacheAttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, unsigned grid, cudaStream_t s) {
  auto kern = cache_attention_tiles_kernel<QBF16, E4M3, D, PAIR>;
  using L = TilesSmem<QBF16, E4M3, D, PAIR>;
  static PerDeviceOnce opt_in;
  const int rc = opt_in(ctx->device, [&] {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != cudaSuccess) return (int)FRISK_B200_E_CUDA;
    // setmaxnreg.inc waits until the CTA's own registers hold the request: what the launch brings must cover both shares
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kern) != cudaSuccess) return (int)FRISK_B200_E_CUDA;
    return a.numRegs * kThreadsTiles >= 256 * kRegsSoftmax + (kThreadsTiles - 256) * kRegsOther ? 0 : (int)FRISK_B200_E_UNSUPPORTED;
  });
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait) itself
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreadsTiles);
  cfg.dynamicSmemBytes = L::kTotal;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FB_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, tk, tv, p));
  return 0;
}

template <bool PAIR>
int launch_any(frisk_b200_ctx* ctx, const CacheAttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, unsigned grid, bool bf16, bool e4m3,
               int D, cudaStream_t s) {
  if (D == 64)
    return bf16 ? (e4m3 ? launch_tiles<true, true, 64, PAIR>(ctx, p, tk, tv, grid, s) : launch_tiles<true, false, 64, PAIR>(ctx, p, tk, tv, grid, s))
                : (e4m3 ? launch_tiles<false, true, 64, PAIR>(ctx, p, tk, tv, grid, s) : launch_tiles<false, false, 64, PAIR>(ctx, p, tk, tv, grid, s));
  return bf16 ? (e4m3 ? launch_tiles<true, true, 128, PAIR>(ctx, p, tk, tv, grid, s) : launch_tiles<true, false, 128, PAIR>(ctx, p, tk, tv, grid, s))
              : (e4m3 ? launch_tiles<false, true, 128, PAIR>(ctx, p, tk, tv, grid, s) : launch_tiles<false, false, 128, PAIR>(ctx, p, tk, tv, grid, s));
}

}  // namespace

int launch_cache_attention_tiles(frisk_b200_ctx* ctx, const cache::CacheAttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv,
                                 unsigned grid, bool bf16, bool e4m3, int D, int tile_rows, cudaStream_t s) {
  return tile_rows == 256 ? launch_any<true>(ctx, p, tk, tv, grid, bf16, e4m3, D, s) : launch_any<false>(ctx, p, tk, tv, grid, bf16, e4m3, D, s);
}

}  // namespace fb
