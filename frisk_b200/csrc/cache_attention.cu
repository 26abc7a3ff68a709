// Attention of drafted tokens over a paged cache: for every packed query row i of sequence b and head h
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),   m = max_j scale q.k_j,
//
// over the keys j of sequence b that row i sees: all those before the new tokens, and of the new ones those that the mask names (or
// those up to itself).  The new tokens' keys are in the cache already.  Queries of one key head share its keys: the rows of a (sequence,
// key head) are its new tokens times its query heads, in tiles of 16.  A row that sees no key is zero.
//
// One pass: a running reference for the exponent that moves when the maximum grew by more than 2^8, fp32 scores, statistics and
// products.  Probabilities are rounded to 16 bits before they meet V, the rate of whose products is the reason: what is lost is half a step
// of each (bf16: results are off by 0.0023 of their norm, by 0.0017 with 32-bit probabilities).
//
// 8-bit caches (value = code * 2^(e - 127), an e for every key): codes become halves exactly, a key's scale multiplies its score, and a
// value's scale joins the exponent of its weight: w_j = 2^(s_j + e_j - A) with a reference A of its own, so that a weight's half step
// is measured against the largest weight times scale and not against the largest probability.  bf16 queries become halves too, scaled
// by a power of two a row.
//
// Bound by HBM at 16 bits, since every key and value is read once (per row tile): 32 sequences of 8000 keys, 8 heads of 128, 4 rows a head
// take 147 us, 6.0 TB/s of the 6.5 that a copy reaches.  At 8 bits by the conversion of the codes, several instructions for two of them:
// 123 us for the same keys, 3.6 TB/s.  (mma.sync on the codes themselves took 1151 instructions for 32 keys of a warp, 182 us.)
// The (sequence, head, row tile, 64-key tile) units are numbered in this order and CTA c takes a contiguous range, whatever the lengths:
// every SM streams the same number of bytes.  The lengths live on the device, so each CTA sums up the units itself.  What a CTA holds of a
// shared item goes to the workspace with the record of the item, and a second kernel, launched early and waiting, joins the parts in
// order: no tickets, nothing to be zero beforehand, no CTA waits for another, and the result does not depend on who comes first.
// K and V tiles arrive by TMA, page by page, in a ring; four warps take 16 keys of a tile each (mma.sync 16x8x16).
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

constexpr int kKeys = 64;  // of a tile
constexpr int kRows = 16;  // query rows, padded

// Consumer warps: four share a tile; with 8-bit caches two fours take the tiles in turn, since a tile comes in half the time and has
// its codes to convert (32 sequences of 8000 keys, 4 rows a head: 240 us with one four, 123 with two, 159 with three of 152 registers a thread).
template <bool E4M3> constexpr int warps_of() { return E4M3 ? 8 : 4; }
// Threads of a CTA.  8-bit: the warp that loads is one of a group of four, which gives its registers to the other two groups: a ninth warp
// of its own would leave 168 registers a thread to all, and spills (141 us).
template <bool E4M3> constexpr int threads_of() { return 32 * (warps_of<E4M3>() + (E4M3 ? 4 : 1)); }
constexpr int kRegsConsumer = 224, kRegsProducer = 56;  // 256 * 224 + 128 * 56 = 384 * 168, what the CTA was launched with

// ones in the elements of `w` (codes, or 16-bit floats) that are infinite or NaN
template <bool E4M3, bool BF16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if (E4M3) return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
  const uint32_t mask = BF16 ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(w & mask, mask);
}
template <bool BF16>
__device__ __forceinline__ float unpack1(uint16_t w) {
  return BF16 ? __uint_as_float((uint32_t)w << 16) : __half2float(__ushort_as_half(w));
}

template <int D, bool E4M3>
struct RowSmem {
  static constexpr int kWarps = warps_of<E4M3>();
  static constexpr int kTile = kKeys * D * (E4M3 ? 1 : 2);
  static constexpr int kStage = 2 * kTile;
  static constexpr int kFloats = kWarps * kRows * D;            // fp32 O of the warps, where they meet
  static constexpr int kRoom = 232448 - 1024 - 512 - kFloats * 4 - 2 * kWarps * kRows * 4;
  static constexpr int kFit = kRoom / (kStage + (E4M3 ? 128 : 0));
  static constexpr int kStages = kFit > 12 ? 12 : E4M3 ? kFit / 2 * 2 : kFit;  // (8-bit: a stage belongs to one of the two fours)
  static constexpr int kExp = kStages * kStage;                 // [stages][K 64, V 64] exponents
  static constexpr int kO = kExp + (E4M3 ? kStages * 128 : 0);
  static constexpr int kStat = kO + kFloats * 4;                // [warps][rows] maxima, [warps][rows] sums
  static constexpr int kBar = kStat + 2 * kWarps * kRows * 4;
  static constexpr int kTotal = kBar + 512 + 1024;
  static_assert(kTotal <= 232448 && kStages >= 4 && kStages <= 12, "ring and reduction area must fit");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// QBF16: type of the queries and results.  E4M3: 8-bit cache, products in halves; else the cache has the queries' type.
template <bool QBF16, bool E4M3, int D>
__global__ void __launch_bounds__(threads_of<E4M3>(), 1)
    cache_attention_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                           const CacheAttnParams p) {
  using L = RowSmem<D, E4M3>;
  constexpr bool MBF16 = QBF16 && !E4M3;  // type of the products' operands
  constexpr float kTop = E4M3 ? 0.f : QBF16 ? kTopWide : kTopHalf;  // log2 of the probabilities (16-bit: weights) at the reference
  constexpr int kWarps = L::kWarps, kThreads = threads_of<E4M3>();
  constexpr int kBoxes = E4M3 ? 1 : D / 64, kBoxBytes = kKeys * 128;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* empty_bar = full_bar + L::kStages;
  uint64_t* meet_bar = empty_bar + L::kStages;  // the consumer threads among themselves
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(meet_bar + 1);
  PlanShared* plan_shared = reinterpret_cast<PlanShared*>(meet_bar + 2);
  static_assert((2 * L::kStages + 3) * 8 + sizeof(PlanShared) <= 512, "barriers and plan must fit");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full_bar[i], E4M3 ? 1 + 32 : 1);  // (the lanes that copy exponents arrive, too)
      mbar_init(&empty_bar[i], 4);
    }
    mbar_init(meet_bar, kWarps * 32);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  // Launched with programmatic stream serialization: the set-up above may overlap the kernel before this one.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Plan plan = make_plan<kThreads>(p, kRows, plan_shared);

  if (warp >= kWarps) {
    if (E4M3) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsProducer));
    // ------------------------------------------------------------------ TMA producer
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const int box = min(p.t.page, kKeys);  // rows a load brings
    PageWalk walk;
    for (Cursor c(p, plan, kRows); warp == kWarps && c.left > 0 && ok; c.next_item(p, kRows)) {
      const int end = c.tile + c.tiles_here(), keys = c.seq.length + c.seq.count;
      walk.enter(p, p.t.table + c.b * p.t.stride, keys, c.h, c.tile, lane);
      for (int tile = c.tile; tile < end; ++tile) {
        const int token = walk.token(p, tile, lane);
        if (tile + 1 < end) walk.look_up(p, tile + 1, lane);
        const int n_boxes = min(kKeys / box, (keys - tile * kKeys + box - 1) / box);
        if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.status, ST_CACHE_KV)) {
          ok = false;
          break;
        }
        unsigned char* sk = smem + stage * L::kStage;
        if (elect_one()) mbar_expect_tx(&full_bar[stage], (uint32_t)n_boxes * box * 2 * D * (E4M3 ? 1 : 2));
        __syncwarp();
        if (E4M3) {
          unsigned char* se = smem + L::kExp + stage * 128;
          if (lane < 8 && tile * kKeys + (lane & 3) * 16 < keys)
            copy16(se + lane * 16, (lane < 4 ? p.k_exponent : p.v_exponent) + token);
          copies_arrive(&full_bar[stage]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (x >= n_boxes) break;
          const int at = uniform_of(token, x * (box >> 4), lane);
          const int row = E4M3 && D == 64 ? at / 2 : at;  // (two 64-byte rows make a line of the 8-bit map)
          const int off = x * box * (E4M3 ? D : 128);
          if (elect_one()) {
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) {
              tma_load_2d(sk + b * kBoxBytes + off, &tmap_k, &full_bar[stage], b * 64, row);
              tma_load_2d(sk + L::kTile + b * kBoxBytes + off, &tmap_v, &full_bar[stage], b * 64, row);
            }
          }
        }
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else {
    if (E4M3) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsConsumer));
    // ------------------------------------------------------------------ consumers
    const int g = lane >> 2, tq = lane & 3;  // fragment coordinates: rows g and g + 8, column pair tq
    const int four = warp >> 2, part_keys = (warp & 3) * 16;  // which tiles, which of their keys
    float* s_o = reinterpret_cast<float*>(smem + L::kO);
    float* s_m = reinterpret_cast<float*>(smem + L::kStat);
    float* s_l = s_m + kWarps * kRows;
    uint32_t meet_phase = 0;
    bool ok = true;
    auto meet = [&]() {  // bounded meeting point of the consumer threads
      mbar_arrive(meet_bar);
      if (ok) ok = mbar_wait_warp(meet_bar, meet_phase, abort_flag, p.status, ST_TIMEOUT_MISC);
      meet_phase ^= 1;
    };
    // Which of its 8 keys a column of a score tile is.  8-bit keys of 128 bytes: a quarter-warp reads 16 bytes of two keys, which the
    // 128-byte swizzle keeps in different banks where the keys are 4 apart; keys of 64 bytes lie side by side in a line.
    auto key_of = [](int col) { return E4M3 && D == 128 ? ((col & 1) << 2) | (col >> 1) : col; };
    // Column of element i of product tile n, first or second of the lane's pair (8-bit: see below)
    auto column_of = [&](int n, int i) { return E4M3 ? (n >> 1) * 16 + 4 * tq + 2 * (i & 1) + (n & 1) : n * 8 + 2 * tq + (i & 1); };
    const int mat = lane >> 3, mrow = lane & 7;
    const int k_row = part_keys + (mat >> 1) * 8 + mrow, v_row = part_keys + (mat & 1) * 8 + mrow;  // 16-bit ldmatrix rows
    unsigned ring = 0;  // stages so far, over all items

    for (Cursor c(p, plan, kRows); c.left > 0 && ok; c.next_item(p, kRows)) {
      const int tile0 = c.tile, tile1 = c.tile + c.tiles_here();
      const Seq seq = c.seq;
      const int keys = seq.length + seq.count;
      const int rows_here = min(kRows, seq.count * p.group - c.rt * kRows);
      const int row0 = c.rt * kRows;

      uint32_t qf[D / 16][4];
      float row_scale[2];  // of scores, to log2 units
      int token[2];        // the row's new token, in its sequence
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = h * 8 + g, r = row0 + row;
        const int i = r / p.group;
        const bool real = row < rows_here;
        token[h] = real ? i : 0;
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + (int64_t)(seq.first + i) * p.q_row +
                            (int64_t)(c.h * p.group + r - i * p.group) * p.q_head;
        row_scale[h] = p.scale_log2;
        if (!E4M3) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x) qf[kk][h + 2 * x] = real ? __ldg(reinterpret_cast<const uint32_t*>(q) + kk * 8 + x * 4 + tq) : 0u;
        } else {
          // this lane's elements of the row: 16 from every 64, so that 16 neighbouring bytes of a key are its part of four products
          uint32_t w[D / 64][8];
#pragma unroll
          for (int b = 0; b < D / 64; ++b) {
            const uint4* from = reinterpret_cast<const uint4*>(q + b * 64 + tq * 16);
            const uint4 lo = real ? __ldg(from) : make_uint4(0, 0, 0, 0), hi = real ? __ldg(from + 1) : make_uint4(0, 0, 0, 0);
            w[b][0] = lo.x; w[b][1] = lo.y; w[b][2] = lo.z; w[b][3] = lo.w;
            w[b][4] = hi.x; w[b][5] = hi.y; w[b][6] = hi.z; w[b][7] = hi.w;
          }
          if (QBF16) {
            // to halves, with the row's largest magnitude in [1, 2): what is 2^14 below it loses bits, at 2^-25 of it
            uint32_t most = 0;
#pragma unroll
            for (int b = 0; b < D / 64; ++b)
#pragma unroll
              for (int n = 0; n < 8; ++n) most = max(most, max(w[b][n] & 0x7fffu, (w[b][n] >> 16) & 0x7fffu));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const uint32_t e = min(max(most >> 7, 1u), 253u);
            const float down = __uint_as_float((254u - e) << 23);
            row_scale[h] *= __uint_as_float(e << 23);
#pragma unroll
            for (int b = 0; b < D / 64; ++b)
#pragma unroll
              for (int n = 0; n < 8; ++n)
                w[b][n] = pack16<false>(__uint_as_float(w[b][n] << 16) * down, __uint_as_float(w[b][n] & 0xffff0000u) * down);
          }
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int n = 0; n < 8; ++n) qf[b * 4 + (n >> 1)][h + 2 * (n & 1)] = w[b][n];
        }
      }
      float o[D / 8][4];
      float m_ref[2], l_sum[2], a_ref[2];  // rows g and g + 8 (l: this lane's columns; a_ref: what 2^0 of a weight stands for)
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        m_ref[h] = a_ref[h] = -INFINITY;
        l_sum[h] = 0.f;
      }

      for (int tile = tile0; tile < tile1; ++tile, ++ring) {
        if (E4M3 && (ring & 1) != (unsigned)four) continue;
        const int stage = (int)(ring % L::kStages);
        if (!mbar_wait_warp(&full_bar[stage], (ring / L::kStages) & 1, abort_flag, p.status, ST_CACHE_KV)) {
          ok = false;
          break;
        }
        const uint32_t sk = smem_u32(smem + stage * L::kStage), sv = sk + L::kTile;
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
        float v_exp[2][2];  // 8-bit: log2 of the scale of this lane's values, by n and column
        // 8-bit values, transposed pairs of codes: a register has the codes of columns 2n, 2n + 1 for two keys.  They are read along with
        // the keys, since what follows has latency enough.
        uint32_t vf8[E4M3 ? D / 32 : 1][4];
        auto load_values = [&]() {
          const int key = part_keys + (mat & 1) * 8 + key_of(mrow);
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const uint32_t at = key * D + (2 * j + (mat >> 1)) * 16;
            ldsm4_trans(vf8[j], sv + (at ^ (((at >> 7) & 7) << 4)));
          }
        };
        if (!E4M3) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t kf[4];
            ldsm4(kf, sk + (kk >> 2) * kBoxBytes + k_row * 128 + ((((kk & 3) * 2 + (mat & 1)) ^ mrow) << 4));
            mma16816<MBF16>(s[0], qf[kk], kf[0], kf[1]);
            mma16816<MBF16>(s[1], qf[kk], kf[2], kf[3]);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] *= row_scale[i >> 1];
        } else {
          uint4 raw[2][D / 64];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
              const uint32_t at = (part_keys + n * 8 + key_of(g)) * D + b * 64 + tq * 16;
              raw[n][b] = lds128(sk + (at ^ (((at >> 7) & 7) << 4)));
            }
          load_values();
          float k_scale[2][2];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const unsigned char* se = smem + L::kExp + stage * 128 + part_keys + n * 8 + key_of(2 * tq + x);
              k_scale[n][x] = scale_of(se[0]);
              const unsigned e = se[64];
              v_exp[n][x] = e == 255u ? __uint_as_float(0x7fc00000u) : (float)((int)e - 127);
            }
          float s2[2][4];  // (two chains of products for either n)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s2[n][i] = 0.f;
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const uint32_t w = i == 0 ? raw[n][b].x : i == 1 ? raw[n][b].y : i == 2 ? raw[n][b].z : raw[n][b].w;
                mma16816<false>(i & 1 ? s2[n] : s[n], qf[b * 4 + i], e4m3x2_to_half2(w), e4m3x2_to_half2_hi(w));
              }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = (s[n][i] + s2[n][i]) * k_scale[n][i & 1] * row_scale[i >> 1];
        }
        // Scores are in log2 units now.  What a row does not see is -inf, whatever its key holds.  This warp's values are its own: rows
        // behind the last key become zeros in place, and so do a new token's infinities and NaN, which reach only the rows that see
        // them: those get them now.  (Their sum is infinite or NaN whatever is added later.)
        if ((tile + 1) * kKeys > seq.length) {
          bool see[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              see[n][i] = sees(p, seq, token[i >> 1], tile * kKeys + part_keys + n * 8 + key_of(2 * tq + (i & 1)) - seq.length);
              if (!see[n][i]) s[n][i] = -INFINITY;
            }
          unsigned char* v = smem + stage * L::kStage + L::kTile;
          constexpr int kRowBytes = E4M3 ? D : 2 * D;
          bool bad = false;
          for (int e = lane; e < 16 * kRowBytes / 16; e += 32) {
            const int key = part_keys + e / (kRowBytes / 16), col = e % (kRowBytes / 16) * 16;
            const uint32_t at = E4M3 ? key * D + col : (col >> 7) * kBoxBytes + key * 128 + (col & 127);
            uint4* at16 = reinterpret_cast<uint4*>(v + (at ^ (((at >> 7) & 7) << 4)));
            const uint4 x = *at16;
            const uint32_t y[4] = {x.x, x.y, x.z, x.w};
            if (tile * kKeys + key >= keys) {
              *at16 = make_uint4(0, 0, 0, 0);
            } else {
              uint32_t any = 0;
#pragma unroll
              for (int i = 0; i < 4; ++i) any |= not_finite<E4M3, MBF16>(y[i]);
              bad |= any != 0;
            }
          }
          if (__any_sync(0xffffffffu, bad)) {
            __syncwarp();
#pragma unroll 1
            for (int key = part_keys; key < part_keys + 16; ++key) {
              const int ahead = tile * kKeys + key - seq.length;
              const bool sees0 = sees(p, seq, token[0], ahead), sees1 = sees(p, seq, token[1], ahead);
#pragma unroll
              for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const int col = column_of(n, i) * (E4M3 ? 1 : 2);
                  const uint32_t at = E4M3 ? key * D + col : (col >> 7) * kBoxBytes + key * 128 + (col & 127);
                  const unsigned char* from = v + (at ^ (((at >> 7) & 7) << 4));
                  float x;
                  if (E4M3) x = (*from & 0x7f) == 0x7f ? __uint_as_float(0x7fc00000u) : 0.f;
                  else x = unpack1<MBF16>(*reinterpret_cast<const uint16_t*>(from));
                  if (!(fabsf(x) <= FLT_MAX)) {
                    if (sees0) o[n][i] += x;
                    if (sees1) o[n][2 + i] += x;
                  }
                }
            }
            __syncwarp();
            for (int e = lane; e < 16 * kRowBytes / 16; e += 32) {
              const int key = part_keys + e / (kRowBytes / 16), col = e % (kRowBytes / 16) * 16;
              const uint32_t at = E4M3 ? key * D + col : (col >> 7) * kBoxBytes + key * 128 + (col & 127);
              uint4* at16 = reinterpret_cast<uint4*>(v + (at ^ (((at >> 7) & 7) << 4)));
              const uint4 x = *at16;
              *at16 = make_uint4(x.x & ~not_finite<E4M3, MBF16>(x.x), x.y & ~not_finite<E4M3, MBF16>(x.y), x.z & ~not_finite<E4M3, MBF16>(x.z),
                                 x.w & ~not_finite<E4M3, MBF16>(x.w));
            }
          }
          fence_proxy_async_smem();  // (the stage's next load comes after these)
          __syncwarp();
          if (E4M3) load_values();
        }
        float m_new[2], a_new[2];
        bool grow = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
          float mw = -INFINITY;
          if (E4M3) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int x = 0; x < 2; ++x) mw = fmaxf(mw, s[n][2 * h + x] + v_exp[n][x]);
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          if (E4M3) mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          m_new[h] = fmaxf(m_ref[h], mx);
          grow |= m_new[h] - m_ref[h] > kRescaleThreshold;  // (false while no key has been seen: -inf - -inf)
          if (E4M3) {
            mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, 2));
            a_new[h] = fmaxf(a_ref[h], mw - kTopHalf);
            grow |= a_new[h] - a_ref[h] > kRescaleThreshold;
          }
        }
        if (__any_sync(0xffffffffu, grow)) {
          float f[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            f[h] = m_ref[h] == -INFINITY ? 0.f : ex2f(m_ref[h] - m_new[h]);
            m_ref[h] = m_new[h];
            l_sum[h] *= f[h];
            if (E4M3) {
              f[h] = a_ref[h] == -INFINITY ? 0.f : ex2f(a_ref[h] - a_new[h]);
              a_ref[h] = a_new[h];
            }
          }
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][0] = scaled(o[n][0], f[0]); o[n][1] = scaled(o[n][1], f[0]);
            o[n][2] = scaled(o[n][2], f[1]); o[n][3] = scaled(o[n][3], f[1]);
          }
        }
        uint32_t pf[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // (a row that sees no key yet: keep it finite)
          const float m0 = (m_ref[h] == -INFINITY ? 0.f : m_ref[h]) - kTop, a0 = a_ref[h] == -INFINITY ? 0.f : a_ref[h];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            float w[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float sc = s[n][2 * h + x], pr = ex2f(sc - m0);
              l_sum[h] += pr;
              // (what is not seen weighs nothing, whatever its value's scale is)
              w[x] = !E4M3 ? pr : sc == -INFINITY ? 0.f : ex2f(sc + v_exp[n][x] - a0);
            }
            pf[n * 2 + h] = pack16<MBF16>(w[0], w[1]);
          }
        }
        if (!E4M3) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            uint32_t vf[4];
            ldsm4_trans(vf, sv + (j >> 2) * kBoxBytes + v_row * 128 + ((((j & 3) * 2 + (mat >> 1)) ^ mrow) << 4));
            mma16816<MBF16>(o[2 * j], pf, vf[0], vf[1]);
            mma16816<MBF16>(o[2 * j + 1], pf, vf[2], vf[3]);
          }
        } else {
          // Even and odd columns go to product tiles of their own: tile 2u has the columns 16u + 2n, tile 2u + 1 the columns 16u + 2n + 1.
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t r0 = __byte_perm(vf8[j][2 * u], 0, 0x3120), r1 = __byte_perm(vf8[j][2 * u + 1], 0, 0x3120);
              mma16816<false>(o[(2 * j + u) * 2], pf, e4m3x2_to_half2(r0), e4m3x2_to_half2(r1));
              mma16816<false>(o[(2 * j + u) * 2 + 1], pf, e4m3x2_to_half2_hi(r0), e4m3x2_to_half2_hi(r1));
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty_bar[stage]);
      }
      if (!ok) break;

      // ---- the warps' results meet in shared memory
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = l_sum[h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int row = h * 8 + g;
        if (tq == 0) {
          s_m[warp * kRows + row] = m_ref[h];
          s_l[warp * kRows + row] = E4M3 ? l * kUnitWide : l;
        }
        // columns in blocks of 8, block index xor a function of the row: rows that are stored together fall into different banks
        float* out = s_o + (warp * kRows + row) * D;
        if (!E4M3) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(out + ((n ^ (row & 3)) << 3) + 2 * tq) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        } else {
          const float f = m_ref[h] == -INFINITY ? 1.f : ex2f(a_ref[h] - m_ref[h] + kTopWide);  // from A's units to m's
#pragma unroll
          for (int u = 0; u < D / 16; ++u)
            *reinterpret_cast<float4*>(out + (((2 * u + (tq >> 1)) ^ (row & 3)) << 3) + (tq & 1) * 4) =
                make_float4(o[2 * u][2 * h] * f, o[2 * u + 1][2 * h] * f, o[2 * u][2 * h + 1] * f, o[2 * u + 1][2 * h + 1] * f);
        }
      }
      meet();
      if (!ok) break;
      const bool whole = tile0 == 0 && tile1 == c.kt;
      // a CTA leaves at most two parts: slot 0 for the item its range begins in, slot 1 for the one it ends in
      float* part = p.partials + ((size_t)blockIdx.x * 2 + (c.first_item ? 0 : 1)) * partial_floats(kRows, D);
      for (int e = threadIdx.x; e < rows_here * (D / 4); e += kWarps * 32) {
        const int row = e / (D / 4), c4 = e % (D / 4);
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_m[w * kRows + row]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float mw = s_m[w * kRows + row];
          if (mw == -INFINITY && s_l[w * kRows + row] == 0.f) continue;  // this warp saw no key of the row
          const float f = mw == -INFINITY ? 1.f : ex2f(mw - m);
          const float4 v =
              *reinterpret_cast<const float4*>(s_o + (w * kRows + row) * D + (((c4 >> 1) ^ (row & 3)) << 3) + (c4 & 1) * 4);
          l = fmaf(s_l[w * kRows + row], f, l);
          acc.x += scaled(v.x, f); acc.y += scaled(v.y, f);
          acc.z += scaled(v.z, f); acc.w += scaled(v.w, f);
        }
        if (whole) {
          store_row4<QBF16, E4M3>(p, seq.first, c.h, row0 + row, c4, acc, l);
        } else {
          __stcg(reinterpret_cast<float4*>(part) + e, acc);
          if (c4 == 0) {
            __stcg(part + kRows * D + row, m);
            __stcg(part + kRows * D + kRows + row, l);
          }
        }
      }
      meet();  // the reduction area may be written again
    }
  }

  // ------------------------------------------------------------------ teardown
  if (*abort_flag) {
    unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();
}

// Joins the parts of the items that several CTAs worked on.  Block (c, y): rows 8 y .. of the item that CTA c began and others
// finished, a warp each, or several, which take their shares of the parts, where there are fewer rows.  (A warp each for four rows
// and 125 parts took 20 us of 33.  Blocks of 16 warps: 4 rows of 32000 keys 22 us for 24, but 24 tokens over 16 x 6000 keys 121 for 120.)
constexpr int kJoinWarps = 8, kJoinAhead = 8;  // parts that a lane has in flight
template <bool QBF16, bool E4M3, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) cache_attention_join_kernel(const CacheAttnParams p, int tile_rows) {
  __shared__ float4 sums[kJoinWarps][D / 4];
  __shared__ float sums_l[kJoinWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ItemRecord rec = p.records[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t floats = partial_floats(tile_rows, D);
  // the item's first part is the CTA's last item; the others' is their first
  auto slot = [&](int i) { return p.partials + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? rec.first_slot : 0)) * floats; };
  const int rows = min(rec.rows - (int)blockIdx.y * kJoinWarps, kJoinWarps);
  if (rows <= 0) return;  // (rec.rows is 0 where the CTA shares no item that it began)
  const int split = kJoinWarps >> (32 - __clz(rows - 1));  // warps a row
  const int local = warp / split, row = blockIdx.y * kJoinWarps + local;
  const int share = (rec.parts + split - 1) / split, part0 = warp % split * share, part1 = min(part0 + share, rec.parts);
  constexpr int N = D / 32;  // columns a lane: 4 or 2
  float acc[N] = {}, l = 0.f;
  if (local < rows) {
    float m = -INFINITY;
    for (int i = lane; i < rec.parts; i += 32) m = fmaxf(m, __ldcg(slot(i) + tile_rows * D + row));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    for (int i0 = part0; i0 < part1; i0 += 32) {
      float f = 0.f, lc = 0.f;
      if (i0 + lane < part1) {
        const float* s = slot(i0 + lane) + tile_rows * D + row;
        const float mc = __ldcg(s);
        lc = __ldcg(s + tile_rows);
        f = mc == -INFINITY ? (lc == 0.f ? 0.f : 1.f) : ex2f(mc - m);
      }
      const int here = min(32, part1 - i0);
#pragma unroll 1
      for (int i = 0; i < here; i += kJoinAhead) {
        float v[kJoinAhead][N];
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
          if (i + u >= here) break;
          const float* from = slot(i0 + i + u) + row * D + lane * N;
          if (N == 4) *reinterpret_cast<float4*>(v[u]) = __ldcg(reinterpret_cast<const float4*>(from));
          else *reinterpret_cast<float2*>(v[u]) = __ldcg(reinterpret_cast<const float2*>(from));
        }
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
          const float fi = __shfl_sync(0xffffffffu, f, i + u), li = __shfl_sync(0xffffffffu, lc, i + u);
          if (i + u >= here) break;
          if (fi == 0.f && li == 0.f) continue;  // saw no key of the row
          l = fmaf(li, fi, l);
#pragma unroll
          for (int x = 0; x < N; ++x) acc[x] += scaled(v[u][x], fi);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < N; ++x) reinterpret_cast<float*>(sums[warp])[lane * N + x] = acc[x];
    if (lane == 0) sums_l[warp] = l;
  }
  __syncthreads();
  // a row's shares in order, four columns a lane
  const int r = warp * (32 / (D / 4)) + lane / (D / 4), c4 = lane % (D / 4);
  if (r >= rows) return;
  float4 sum = sums[r * split][c4];
  l = sums_l[r * split];
  for (int i = 1; i < split; ++i) {
    const float4 x = sums[r * split + i][c4];
    sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
    l += sums_l[r * split + i];
  }
  store_row4<QBF16, E4M3>(p, rec.first_row, rec.head, rec.row0 + blockIdx.y * kJoinWarps + r, c4, sum, l);
}

template <bool QBF16, bool E4M3, int D>
int launch_rows(frisk_b200_ctx* ctx, const CacheAttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, unsigned grid, cudaStream_t s) {
  auto kern = cache_attention_kernel<QBF16, E4M3, D>;
  using L = RowSmem<D, E4M3>;
  static PerDeviceOnce opt_in;
  const int rc = opt_in(ctx->device, [&] {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != cudaSuccess) return (int)FRISK_B200_E_CUDA;
    if (!E4M3) return 0;
    // setmaxnreg.inc waits until the CTA's own registers hold the request: what the launch brings must cover both shares
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kern) != cudaSuccess) return (int)FRISK_B200_E_CUDA;
    return a.numRegs * threads_of<E4M3>() >= L::kWarps * 32 * kRegsConsumer + 128 * kRegsProducer ? 0 : (int)FRISK_B200_E_UNSUPPORTED;
  });
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernels wait (griddepcontrol.wait) themselves
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads_of<E4M3>());
  cfg.dynamicSmemBytes = L::kTotal;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FB_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, tk, tv, p));
  return 0;
}

template <bool QBF16, bool E4M3, int D>
int launch_all(frisk_b200_ctx* ctx, const CacheAttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, unsigned grid, int tile_rows,
               cudaStream_t s) {
  const int rc = tile_rows == kRows ? launch_rows<QBF16, E4M3, D>(ctx, p, tk, tv, grid, s)
                                    : launch_cache_attention_tiles(ctx, p, tk, tv, grid, QBF16, E4M3, D, tile_rows, s);
  if (rc || p.whole) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid, (unsigned)(tile_rows / kJoinWarps));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FB_CUDA(ctx, cudaLaunchKernelEx(&cfg, cache_attention_join_kernel<QBF16, E4M3, D>, p, tile_rows));
  return 0;
}

// Whether items are dealt out whole, which saves their joining and a launch (some seven key tiles' time) and costs the SMs that end early.
// Measured whole and shared, one query row: 8 heads x 200 keys 7.0 and 8.9 us, 128 heads x 500 10.0 and 15.1, 512 x 200 21.0 and 24.4, 1024 x
// 500 54.9 and 61.0.  It goes by the table's width, and for up to 32 key tiles, since the sequences may differ.
bool whole_items(const frisk_b200_cache_desc* c, const frisk_b200_cache_attn_desc* a) {
  const int64_t per = a->max_new > 0 ? a->max_new : (c->rows + c->batch - 1) / c->batch;
  const int64_t items = (int64_t)c->batch * c->heads * ((per * (a->heads_q / c->heads) + kRows - 1) / kRows);
  const int64_t tiles = ((int64_t)c->table_width * c->page + kKeys - 1) / kKeys;
  const int64_t rounds = (items + kNumSMsDefault - 1) / kNumSMsDefault;
  return tiles <= 32 && rounds * tiles * kNumSMsDefault <= items * tiles + 7 * kNumSMsDefault;
}

int check_attention(const frisk_b200_cache_desc* c, const frisk_b200_cache_attn_desc* a) {
  int rc = cache_validate(c);
  if (rc) return rc;
  if (!a) return FRISK_B200_E_ARG;
  if (a->dtype != FRISK_B200_F16 && a->dtype != FRISK_B200_BF16) return FRISK_B200_E_CACHE_TYPE;
  if (c->dtype != FRISK_B200_E4M3 && c->dtype != a->dtype) return FRISK_B200_E_CACHE_TYPE;
  if (a->heads_q < 1 || a->heads_q > 65536 || a->heads_q % c->heads || a->max_new < 0 || a->mask_width < 0 || a->mask_stride < 0)
    return FRISK_B200_E_CACHE_SHAPE;
  if (!(a->scale == a->scale) || a->scale * 0.f != 0.f) return FRISK_B200_E_ARG;
  if (a->tile_rows != 0 && a->tile_rows != kRows && a->tile_rows != 128 && a->tile_rows != 256) return FRISK_B200_E_ARG;
  // units are counted in 32 bits (16 rows and 64 keys at least)
  const double tiles = ((double)c->table_width * c->page + kKeys - 1) / kKeys, group = a->heads_q / c->heads;
  if (tiles * c->heads * (c->rows * group / 16 + c->batch) > 2147483647.0 || (double)c->table_width * c->page > 2147483647.0 - 4 * kKeys ||
      (double)c->rows * group > 2147483647.0)
    return FRISK_B200_E_TOO_LARGE;
  return 0;
}

// Query rows a tile, by the rows that a sequence is said to have for a key head.  (A sequence with more than a tile's rows takes several
// tiles, so a hint that is too low costs time only.)  Up to 16 rows this file's kernel; from 129 on tiles of 256.  In between it is
// weighed: this kernel reads the keys once for every 16 rows, the tiles of 128 once, at a higher cost of beginning and ending an item.  In
// us, with n key tiles a SM: 16 rows 0.74 n (16-bit, D = 128), 0.40 (D = 64), 0.55 and 0.45 (8-bit); tiles 0.77, 0.71, 1.16 and 1.10 n and 10
// (8-bit 14) more.  Measured, this kernel and tiles: 8 sequences of 4000 keys at D = 128, 32 rows a head 43.3 and 46.1, 8-bit 46.0 and
// 65.6, 48 rows 57.3 and 62.6, 64 rows 64.7 and 61.0; of 1000 keys, 32 rows 15.1 and 27.9, 17.2 and 36.0, 48 rows 27.7 and 29.3, 31.4 and
// 36.4; 32 sequences of 8000 keys, 32 rows, 8-bit 242 and 281, at D = 64 172 and 154, 8-bit 195 and 257.  n goes by the table's width, the longest that the sequences can be.
int tile_rows_of(const frisk_b200_cache_desc* c, const frisk_b200_cache_attn_desc* a) {
  const int64_t per = a->max_new > 0 ? a->max_new : c->batch > 0 ? (c->rows + c->batch - 1) / c->batch : 1;
  const int64_t rows = per * (a->heads_q / c->heads);
  if (a->tile_rows) return a->tile_rows;
  if (rows <= kRows) return kRows;
  if (rows > 128) return 256;
  const bool e4m3 = c->dtype == FRISK_B200_E4M3;
  const double n = (double)c->batch * c->heads * ((double)c->table_width * c->page / kKeys) / kNumSMsDefault;
  const double few = e4m3 ? (c->D == 128 ? 0.55 : 0.45) : (c->D == 128 ? 0.74 : 0.40);
  const double tiles = e4m3 ? (c->D == 128 ? 1.16 : 1.10) : (c->D == 128 ? 0.77 : 0.71);
  return (rows + kRows - 1) / kRows * few * n < tiles * n + (e4m3 ? 14 : 10) ? kRows : 128;
}

}  // namespace
}  // namespace fb

using namespace fb;
using namespace fb::cache;

extern "C" int frisk_b200_cache_attention_tile_rows(const frisk_b200_cache_desc* c, const frisk_b200_cache_attn_desc* a) {
  const int rc = check_attention(c, a);
  return rc ? rc : tile_rows_of(c, a);
}

extern "C" size_t frisk_b200_cache_attention_workspace_bytes(const frisk_b200_cache_desc* c, const frisk_b200_cache_attn_desc* a) {
  if (check_attention(c, a)) return 0;
  return kRecordBytes + (size_t)kNumSMsDefault * 2 * partial_floats(tile_rows_of(c, a), c->D) * sizeof(float);
}

extern "C" int frisk_b200_cache_attention(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, const frisk_b200_cache_attn_desc* a,
                                          const frisk_b200_packed* q, const frisk_b200_packed* out, const uint8_t* mask,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!ctx) return FRISK_B200_E_ARG;
  int rc = check_attention(c, a);
  if (rc) return rc;
  if (c->rows == 0 || c->batch == 0) return 0;
  if ((rc = cache_pointers(c))) return rc;
  if (!q || !out || !q->ptr || !out->ptr) return FRISK_B200_E_ARG;
  for (const frisk_b200_packed* x : {q, out}) {
    if (x->row_stride < 0 || x->head_stride < 0) return FRISK_B200_E_CACHE_SHAPE;
    if ((reinterpret_cast<uintptr_t>(x->ptr) & 15u) || (c->rows > 1 && x->row_stride % 8) || (a->heads_q > 1 && x->head_stride % 8))
      return FRISK_B200_E_ALIGN;
  }
  if (!packed_distinct(*out, c->rows, a->heads_q, c->D)) return FRISK_B200_E_CACHE_SHAPE;
  const size_t need = frisk_b200_cache_attention_workspace_bytes(c, a);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 31u)) return FRISK_B200_E_WORKSPACE;
  const size_t ob = packed_span(*out, c->rows, a->heads_q, c->D, 2), qb = packed_span(*q, c->rows, a->heads_q, c->D, 2);
  const size_t mb = mask && a->mask_width ? (size_t)((c->rows - 1) * a->mask_stride + a->mask_width) : 0;
  for (int w = 0; w < 2; ++w) {  // what is written: the results and the workspace
    const void* ptr = w ? workspace : out->ptr;
    const size_t n = w ? need : ob;
    const bool queries = w ? ranges_overlap(ptr, n, q->ptr, qb) : !packed_apart(*out, a->heads_q, *q, a->heads_q, c->rows, c->D, 2);
    if (queries || (mb && ranges_overlap(ptr, n, mask, mb)) || cache_overlaps(c, ptr, n) || tables_overlap(c, ptr, n))
      return FRISK_B200_E_OVERLAP;
  }
  if (ranges_overlap(workspace, need, out->ptr, ob)) return FRISK_B200_E_OVERLAP;

  FB_DEVICE(ctx);
  const bool e4m3 = c->dtype == FRISK_B200_E4M3, bf16 = a->dtype == FRISK_B200_BF16;
  const int tile_rows = tile_rows_of(c, a);
  // Lines of 128 bytes: one key or half of one at 16 bits, one or two at 8.  (The tensor core wants 8-bit keys of 64 bytes in lines of
  // their own and the swizzle of that width.)
  const uint64_t tokens = (uint64_t)c->pages * c->heads * c->page;
  const int box_rows = std::min(c->page, kKeys);
  CUtensorMap tk, tv;
  const int map_type = e4m3 ? FRISK_B200_F16 : c->dtype;
  const bool narrow = e4m3 && c->D == 64 && tile_rows > kRows;
  const uint64_t inner = narrow ? 32 : e4m3 ? 64 : c->D, outer = e4m3 && !narrow ? tokens * c->D / 128 : tokens;
  const uint32_t box = e4m3 && !narrow ? box_rows * c->D / 128 : box_rows;
  const TmapSwizzle swizzle = narrow ? TmapSwizzle::k64 : TmapSwizzle::k128;
  rc = encode_tmap_2d(ctx, &tk, map_type, c->k, inner, outer, inner * 2, narrow ? 32 : 64, box, swizzle);
  if (!rc) rc = encode_tmap_2d(ctx, &tv, map_type, c->v, inner, outer, inner * 2, narrow ? 32 : 64, box, swizzle);
  if (rc) {
    ctx->last_cuda = rc;
    return FRISK_B200_E_CUDA;
  }
  CacheAttnParams p{};
  p.t = cache_tables(c);
  p.q = q->ptr;
  p.q_row = q->row_stride;
  p.q_head = q->head_stride;
  p.out = out->ptr;
  p.out_row = out->row_stride;
  p.out_head = out->head_stride;
  p.k_exponent = c->k_exponent;
  p.v_exponent = c->v_exponent;
  p.v_pages = c->v;
  p.mask = mask;
  p.mask_stride = a->mask_stride;
  p.mask_width = a->mask_width;
  p.group = a->heads_q / c->heads;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.records = static_cast<ItemRecord*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + kRecordBytes);
  p.status = ctx->d_status;
  p.whole = tile_rows == kRows && whole_items(c, a);
  const unsigned grid = (unsigned)std::min(ctx->num_sms, kNumSMsDefault);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->D == 64)
    return bf16 ? (e4m3 ? launch_all<true, true, 64>(ctx, p, tk, tv, grid, tile_rows, s) : launch_all<true, false, 64>(ctx, p, tk, tv, grid, tile_rows, s))
                : (e4m3 ? launch_all<false, true, 64>(ctx, p, tk, tv, grid, tile_rows, s) : launch_all<false, false, 64>(ctx, p, tk, tv, grid, tile_rows, s));
  return bf16 ? (e4m3 ? launch_all<true, true, 128>(ctx, p, tk, tv, grid, tile_rows, s) : launch_all<true, false, 128>(ctx, p, tk, tv, grid, tile_rows, s))
              : (e4m3 ? launch_all<false, true, 128>(ctx, p, tk, tv, grid, tile_rows, s) : launch_all<false, false, 128>(ctx, p, tk, tv, grid, tile_rows, s));
}
