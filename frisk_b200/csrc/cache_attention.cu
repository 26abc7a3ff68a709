// Attention of drafted tokens over a paged cache: for every packed query row i of sequence b and head h
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),   m = max_j scale q.k_j,
//
// over the keys j of sequence b that row i sees: all those before the new tokens, and of the new ones those that the mask names (or
// those up to itself).  The new tokens' keys are in the cache already.  Queries of one key head share its keys: the rows of a (sequence,
// key head) are its new tokens times its query heads, in tiles of 16 or 32.  A row that sees no key is zero.
//
// One pass: a running reference for the exponent that moves when the maximum grew by more than 2^8, fp32 scores, statistics and
// products.  Probabilities are rounded to 16 bits before they meet V, the rate of whose products is the reason; relative to the
// reference, so what is lost is half a step of each.
//
// 8-bit caches (value = code * 2^(e - 127), an e for every key): codes become halves exactly, a key's scale multiplies its score, and a
// value's scale joins the exponent of its weight: w_j = 2^(s_j + e_j - A) with a reference A of its own, so that a weight's half step
// is measured against the largest weight times scale and not against the largest probability.  bf16 queries become halves too, scaled
// by a power of two a row.
//
// Bound by HBM up to some 60 query rows a key head: every key and value is read once (per row tile).  The (sequence, head, row tile,
// 64-key tile) units are numbered in this order and CTA c takes a contiguous range, whatever the lengths: every SM streams the same number
// of bytes.  The lengths live on the device, so each CTA sums up the units itself.  What a CTA holds of a shared item goes to the
// workspace with the record of the item, and a second kernel, launched early and waiting, joins the parts in order: no
// tickets, nothing to be zero beforehand, no CTA waits for another, and the result does not depend on who comes first.
// K and V tiles arrive by TMA, page by page, in a ring; four warps take 16 keys of a tile each (mma.sync 16x8x16).
// Every mbarrier wait is bounded (ptx.cuh); no TMA load uses cluster multicast.
#include <algorithm>

#include "attention_common.cuh"
#include "cache_attention.cuh"
#include "work_split.cuh"

namespace fb {
namespace {
using namespace attn;
using namespace cache;

constexpr int kKeys = 64;    // of a tile
constexpr int kWarps = 4;    // consumers
constexpr int kThreadsRow = 32 * (kWarps + 1);

template <int D, bool E4M3, int MT>
struct RowSmem {
  static constexpr int kRows = 16 * MT;
  static constexpr int kTile = kKeys * D * (E4M3 ? 1 : 2);
  static constexpr int kStage = 2 * kTile;
  static constexpr int kFloats = kWarps * kRows * D;            // fp32 O of the four warps, where they meet
  static constexpr int kRoom = 232448 - 1024 - 2048 - kFloats * 4 - 2 * kWarps * kRows * 4;
  static constexpr int kStages = (kRoom / (kStage + (E4M3 ? 128 : 0))) > 12 ? 12 : kRoom / (kStage + (E4M3 ? 128 : 0));
  static constexpr int kExp = kStages * kStage;                 // [stages][K 64, V 64] exponents
  static constexpr int kO = kExp + (E4M3 ? kStages * 128 : 0);
  static constexpr int kStat = kO + kFloats * 4;                // [4][rows] maxima, [4][rows] sums
  static constexpr int kBar = kStat + 2 * kWarps * kRows * 4;
  static constexpr int kTotal = kBar + 1024 + 1024;
  static_assert(kTotal <= 232448 && kStages >= 3 && kStages <= 12, "ring and reduction area must fit");
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

// 0xffff in the halves of `w` that are infinite or NaN
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  const uint32_t mask = BF16 ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(w & mask, mask);
}
// 1.0 in the halves that `m` selects
template <bool BF16>
__device__ __forceinline__ uint32_t ones_of(uint32_t m) {
  return m & (BF16 ? 0x3f803f80u : 0x3c003c00u);
}

// QBF16: type of the queries and results.  E4M3: 8-bit cache, products in halves; else the cache has the queries' type.
template <bool QBF16, bool E4M3, int D, int MT>
__global__ void __launch_bounds__(kThreadsRow, 1)
    cache_attention_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                           const CacheAttnParams p) {
  using L = RowSmem<D, E4M3, MT>;
  constexpr bool MBF16 = QBF16 && !E4M3;  // type of the products' operands
  constexpr int kRows = L::kRows;
  constexpr int kBoxes = E4M3 ? 1 : D / 64, kBoxBytes = kKeys * 128;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* empty_bar = full_bar + L::kStages;
  uint64_t* meet_bar = empty_bar + L::kStages;  // the 128 consumer threads among themselves
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(meet_bar + 1);
  PlanShared* plan_shared = reinterpret_cast<PlanShared*>(meet_bar + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], kWarps);
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
  const Plan plan = make_plan<kThreadsRow>(p, kRows, plan_shared);

  if (warp == kWarps) {
    // ------------------------------------------------------------------ TMA producer: the warp reads the table, lane 0 loads
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const int box = min(p.t.page, kKeys);  // rows a load brings
    for (Cursor c(p, plan, kRows); c.left > 0 && ok; c.next_item(p, kRows)) {
      const int tiles = c.tiles_here();
      const int keys = c.seq.length + c.seq.count;
      const int* row = p.t.table + c.b * p.t.stride;
      int ids = 0, ids_from = -32;  // pages ids_from + lane
      for (int tile = c.tile; tile < c.tile + tiles; ++tile) {
        const int n_boxes = min(kKeys / box, (keys - tile * kKeys + box - 1) / box);
        if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.status, ST_CACHE_KV)) {
          ok = false;
          break;
        }
        unsigned char* sk = smem + stage * L::kStage;
        unsigned char* se = smem + L::kExp + stage * 128;
        if (lane == 0) mbar_expect_tx(&full_bar[stage], (uint32_t)n_boxes * box * 2 * (D * (E4M3 ? 1 : 2) + (E4M3 ? 1 : 0)));
        for (int x = 0; x < n_boxes; ++x) {
          const int key = tile * kKeys + x * box, at = key >> p.t.page_log2;
          if (at < ids_from || at >= ids_from + 32) {
            ids_from = at;
            ids = at + lane < p.t.width ? __ldg(row + at + lane) : 0;
          }
          int page = __shfl_sync(0xffffffffu, ids, at - ids_from);
          if (page < 0 || page >= p.t.pages) {  // (page 0 is read in its place)
            if (lane == 0) atomicCAS(p.status, 0u, ST_CACHE_PAGE);
            page = 0;
          }
          if (lane == 0) {
            const int token = ((page * p.t.heads + c.h) << p.t.page_log2) + (key & (p.t.page - 1));
            const int at_row = E4M3 && D == 64 ? token / 2 : token;  // (two 64-byte rows make a line of the 8-bit map)
            const int off = x * box * (E4M3 ? D : 128);
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) {
              tma_load_2d(sk + b * kBoxBytes + off, &tmap_k, &full_bar[stage], b * 64, at_row);
              tma_load_2d(sk + L::kTile + b * kBoxBytes + off, &tmap_v, &full_bar[stage], b * 64, at_row);
            }
            if (E4M3) {
              bulk_load(se + x * box, p.k_exponent + token, box, &full_bar[stage]);
              bulk_load(se + 64 + x * box, p.v_exponent + token, box, &full_bar[stage]);
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
    // ------------------------------------------------------------------ consumers
    const int g = lane >> 2, tq = lane & 3;  // fragment coordinates: rows g and g + 8, column pair tq
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
    const int mat = lane >> 3, mrow = lane & 7;
    const int k_row = warp * 16 + (mat >> 1) * 8 + mrow, v_row = warp * 16 + (mat & 1) * 8 + mrow;  // 16-bit ldmatrix rows
    int stage = 0;
    uint32_t phase = 0;

    for (Cursor c(p, plan, kRows); c.left > 0 && ok; c.next_item(p, kRows)) {
      const int tile0 = c.tile, tile1 = c.tile + c.tiles_here();
      const Seq seq = c.seq;
      const int keys = seq.length + seq.count;
      const int rows_here = min(kRows, seq.count * p.group - c.rt * kRows);
      const int row0 = c.rt * kRows;

      uint32_t qf[MT][D / 16][4];
      float row_scale[MT][2];  // of scores, to log2 units
      int token[MT][2];        // the row's new token, in its sequence
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = mt * 16 + h * 8 + g, r = row0 + row;
          const int i = r / p.group;
          const bool real = row < rows_here;
          token[mt][h] = real ? i : 0;
          const uint16_t* q = static_cast<const uint16_t*>(p.q) + (int64_t)(seq.first + i) * p.q_row +
                              (int64_t)(c.h * p.group + r - i * p.group) * p.q_head;
          row_scale[mt][h] = p.scale_log2;
          if (!E4M3) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
              for (int x = 0; x < 2; ++x)
                qf[mt][kk][h + 2 * x] = real ? __ldg(reinterpret_cast<const uint32_t*>(q) + kk * 8 + x * 4 + tq) : 0u;
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
              row_scale[mt][h] *= __uint_as_float(e << 23);
#pragma unroll
              for (int b = 0; b < D / 64; ++b)
#pragma unroll
                for (int n = 0; n < 8; ++n)
                  w[b][n] = pack16<false>(__uint_as_float(w[b][n] << 16) * down, __uint_as_float(w[b][n] & 0xffff0000u) * down);
            }
#pragma unroll
            for (int b = 0; b < D / 64; ++b)
#pragma unroll
              for (int n = 0; n < 8; ++n) qf[mt][b * 4 + (n >> 1)][h + 2 * (n & 1)] = w[b][n];
          }
        }
      float o[MT][D / 8][4];
      float m_ref[MT][2], l_sum[MT][2], a_ref[MT][2];  // rows g and g + 8 (l: this lane's columns)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          m_ref[mt][h] = a_ref[mt][h] = -INFINITY;
          l_sum[mt][h] = 0.f;
        }
      }

      for (int tile = tile0; tile < tile1; ++tile) {
        if (!mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.status, ST_CACHE_KV)) {
          ok = false;
          break;
        }
        const uint32_t sk = smem_u32(smem + stage * L::kStage), sv = sk + L::kTile;
        float s[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[mt][n][i] = 0.f;
        float v_exp[2][2];  // 8-bit: log2 of the scale of this lane's values, by n and column
        if (!E4M3) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t kf[4];
            ldsm4(kf, sk + (kk >> 2) * kBoxBytes + k_row * 128 + ((((kk & 3) * 2 + (mat & 1)) ^ mrow) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma16816<MBF16>(s[mt][0], qf[mt][kk], kf[0], kf[1]);
              mma16816<MBF16>(s[mt][1], qf[mt][kk], kf[2], kf[3]);
            }
          }
        } else {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int key = warp * 16 + n * 8 + key_of(g);
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
              const uint32_t at = key * D + b * 64 + tq * 16;
              const uint4 raw = lds128(sk + (at ^ (((at >> 7) & 7) << 4)));
              const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t b0 = e4m3x2_to_half2(w[i]), b1 = e4m3x2_to_half2_hi(w[i]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) mma16816<false>(s[mt][n], qf[mt][b * 4 + i], b0, b1);
              }
            }
            const unsigned char* se = smem + L::kExp + stage * 128 + warp * 16 + n * 8;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int at = key_of(2 * tq + x);
              const float k_scale = scale_of(se[at]);
              const unsigned e = se[64 + at];
              v_exp[n][x] = e == 255u ? __uint_as_float(0x7fc00000u) : (float)((int)e - 127);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                s[mt][n][x] *= k_scale;
                s[mt][n][2 + x] *= k_scale;
              }
            }
          }
        }
        // to log2 units; what a row does not see is -inf, whatever its key holds
        const bool masked = (tile + 1) * kKeys > seq.length;
        uint32_t seen = 0xffffffffu;  // bit mt * 8 + n * 4 + i
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[mt][n][i] *= row_scale[mt][i >> 1];
        if (masked) {
          seen = 0;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int ahead = tile * kKeys + warp * 16 + n * 8 + key_of(2 * tq + (i & 1)) - seq.length;
                const bool see = sees(p, seq, token[mt][i >> 1], ahead);
                seen |= (see ? 1u : 0u) << (mt * 8 + n * 4 + i);
                if (!see) s[mt][n][i] = -INFINITY;
              }
        }
        float m_new[MT][2];
        bool grow = false;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float mx = fmaxf(fmaxf(s[mt][0][2 * h], s[mt][0][2 * h + 1]), fmaxf(s[mt][1][2 * h], s[mt][1][2 * h + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            m_new[mt][h] = fmaxf(m_ref[mt][h], mx);
            grow |= m_new[mt][h] - m_ref[mt][h] > kRescaleThreshold;  // (false while no key has been seen: -inf - -inf)
          }
        float a_new[MT][2];
        if (E4M3) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float mx = -INFINITY;
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x) mx = fmaxf(mx, s[mt][n][2 * h + x] + v_exp[n][x]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
              a_new[mt][h] = fmaxf(a_ref[mt][h], mx);
              grow |= a_new[mt][h] - a_ref[mt][h] > kRescaleThreshold;
            }
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              f[h] = m_ref[mt][h] == -INFINITY ? 0.f : ex2f(m_ref[mt][h] - m_new[mt][h]);
              m_ref[mt][h] = m_new[mt][h];
              l_sum[mt][h] *= f[h];
              if (E4M3) {
                f[h] = a_ref[mt][h] == -INFINITY ? 0.f : ex2f(a_ref[mt][h] - a_new[mt][h]);
                a_ref[mt][h] = a_new[mt][h];
              }
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              o[mt][n][0] *= f[0]; o[mt][n][1] *= f[0];
              o[mt][n][2] *= f[1]; o[mt][n][3] *= f[1];
            }
          }
        }
        uint32_t pf[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // (a row that sees no key yet: keep it finite)
            const float m0 = m_ref[mt][h] == -INFINITY ? 0.f : m_ref[mt][h], a0 = a_ref[mt][h] == -INFINITY ? 0.f : a_ref[mt][h];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              float w[2];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float sc = s[mt][n][2 * h + x], pr = ex2f(sc - m0);
                l_sum[mt][h] += pr;
                // (what is not seen weighs nothing, whatever its value's scale is)
                w[x] = !E4M3 ? pr : sc == -INFINITY ? 0.f : ex2f(sc + v_exp[n][x] - a0);
              }
              pf[mt][n * 2 + h] = pack16<MBF16>(w[0], w[1]);
            }
          }
        }
        // Values behind the last key count as zeros, and a new token's infinities and NaN reach only the rows that see it: they are
        // taken out of the product, and a product of what each row sees with where they are tells which results they make.
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if (masked) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int key = tile * kKeys + warp * 16 + n * 8;
            keep[n] = (key + key_of(2 * tq) < keys ? 0xffffu : 0u) | (key + key_of(2 * tq + 1) < keys ? 0xffff0000u : 0u);
          }
        }
        auto times_v = [&](float (&o0)[MT][D / 8][4], int n0, uint32_t b0, uint32_t b1) {
          if (masked) {
            b0 &= keep[0];
            b1 &= keep[1];
            const uint32_t x0 = not_finite<MBF16>(b0), x1 = not_finite<MBF16>(b1);
            if (__any_sync(0xffffffffu, (x0 | x1) != 0)) {
              const uint32_t frac = MBF16 ? 0x007f007fu : 0x03ff03ffu;
              const uint32_t n_0 = x0 & ~__vcmpeq2(b0 & frac, 0), n_1 = x1 & ~__vcmpeq2(b1 & frac, 0);  // NaN: of both signs
              const uint32_t s_0 = __vcmpgtu2(b0 & 0x80008000u, 0), s_1 = __vcmpgtu2(b1 & 0x80008000u, 0);
              const uint32_t pos0 = ones_of<MBF16>(x0 & (~s_0 | n_0)), pos1 = ones_of<MBF16>(x1 & (~s_1 | n_1));
              const uint32_t neg0 = ones_of<MBF16>(x0 & (s_0 | n_0)), neg1 = ones_of<MBF16>(x1 & (s_1 | n_1));
              const float inf = __uint_as_float(0x7f800000u);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                uint32_t sf[4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const uint32_t two = (seen >> (mt * 8 + n * 4 + 2 * h)) & 3u;
                    sf[n * 2 + h] = ones_of<MBF16>(((two & 1u) ? 0xffffu : 0u) | ((two & 2u) ? 0xffff0000u : 0u));
                  }
                float up[4] = {0.f, 0.f, 0.f, 0.f}, down[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816<MBF16>(up, sf, pos0, pos1);
                mma16816<MBF16>(down, sf, neg0, neg1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if (up[i] > 0.f) o0[mt][n0][i] += inf;
                  if (down[i] > 0.f) o0[mt][n0][i] -= inf;
                }
              }
              b0 &= ~x0;
              b1 &= ~x1;
            }
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma16816<MBF16>(o0[mt][n0], pf[mt], b0, b1);
        };
        if (!E4M3) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            uint32_t vf[4];
            ldsm4_trans(vf, sv + (j >> 2) * kBoxBytes + v_row * 128 + ((((j & 3) * 2 + (mat >> 1)) ^ mrow) << 4));
            times_v(o, 2 * j, vf[0], vf[1]);
            times_v(o, 2 * j + 1, vf[2], vf[3]);
          }
        } else {
          // transposed pairs of codes: a register has the codes of columns 2n, 2n + 1 for two keys.  Even and odd columns go to
          // product tiles of their own: tile 2u has the columns 16u + 2n, tile 2u + 1 the columns 16u + 2n + 1.
          const int key = warp * 16 + (mat & 1) * 8 + key_of(mrow);
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const uint32_t at = key * D + (2 * j + (mat >> 1)) * 16;
            uint32_t vf[4];
            ldsm4_trans(vf, sv + (at ^ (((at >> 7) & 7) << 4)));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t r0 = __byte_perm(vf[2 * u], 0, 0x3120), r1 = __byte_perm(vf[2 * u + 1], 0, 0x3120);
              times_v(o, (2 * j + u) * 2, e4m3x2_to_half2(r0), e4m3x2_to_half2(r1));
              times_v(o, (2 * j + u) * 2 + 1, e4m3x2_to_half2_hi(r0), e4m3x2_to_half2_hi(r1));
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty_bar[stage]);
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;

      // ---- the four warps' results meet in shared memory
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float l = l_sum[mt][h];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          const int row = mt * 16 + h * 8 + g;
          if (tq == 0) {
            s_m[warp * kRows + row] = m_ref[mt][h];
            s_l[warp * kRows + row] = l;
          }
          // columns in blocks of 8, block index xor a function of the row: rows that are stored together fall into different banks
          float* out = s_o + (warp * kRows + row) * D;
          if (!E4M3) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              *reinterpret_cast<float2*>(out + ((n ^ (row & 3)) << 3) + 2 * tq) = make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
          } else {
            const float f = m_ref[mt][h] == -INFINITY ? 0.f : ex2f(a_ref[mt][h] - m_ref[mt][h]);  // from A's units to m's
#pragma unroll
            for (int u = 0; u < D / 16; ++u)
              *reinterpret_cast<float4*>(out + (((2 * u + (tq >> 1)) ^ (row & 3)) << 3) + (tq & 1) * 4) =
                  make_float4(o[mt][2 * u][2 * h] * f, o[mt][2 * u + 1][2 * h] * f, o[mt][2 * u][2 * h + 1] * f,
                              o[mt][2 * u + 1][2 * h + 1] * f);
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
          acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
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

// Joins the parts of the items that several CTAs worked on.  Block (c, y): rows 4 y .. of the item that CTA c began and others
// finished, a warp each, and those gridDim.y blocks on.
template <bool QBF16, bool E4M3, int D>
__global__ void __launch_bounds__(128) cache_attention_join_kernel(const CacheAttnParams p, int tile_rows) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ItemRecord rec = p.records[blockIdx.x];
  const int lane = threadIdx.x & 31;
  const size_t floats = partial_floats(tile_rows, D);
  // the item's first part is the CTA's last item; the others' is their first
  auto slot = [&](int i) { return p.partials + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? rec.first_slot : 0)) * floats; };
  // (rec.rows is 0 where the CTA shares no item that it began)
  for (int row = blockIdx.y * 4 + (threadIdx.x >> 5); row < rec.rows; row += gridDim.y * 4) {
    float m = -INFINITY;
    for (int i = lane; i < rec.parts; i += 32) m = fmaxf(m, __ldcg(slot(i) + tile_rows * D + row));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    constexpr int N = D / 32;  // columns a lane: 4 or 2
    float acc[N] = {}, l = 0.f;
    for (int i0 = 0; i0 < rec.parts; i0 += 32) {
      float f = 0.f, lc = 0.f;
      if (i0 + lane < rec.parts) {
        const float* s = slot(i0 + lane) + tile_rows * D + row;
        const float mc = __ldcg(s);
        lc = __ldcg(s + tile_rows);
        f = mc == -INFINITY ? (lc == 0.f ? 0.f : 1.f) : ex2f(mc - m);
      }
      const int here = min(32, rec.parts - i0);
#pragma unroll 4
      for (int i = 0; i < here; ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, i), li = __shfl_sync(0xffffffffu, lc, i);
        const float* from = slot(i0 + i) + row * D + lane * N;
        float v[N];
        if (N == 4) *reinterpret_cast<float4*>(v) = __ldcg(reinterpret_cast<const float4*>(from));
        else *reinterpret_cast<float2*>(v) = __ldcg(reinterpret_cast<const float2*>(from));
        if (fi == 0.f && li == 0.f) continue;  // saw no key of the row
        l = fmaf(li, fi, l);
#pragma unroll
        for (int x = 0; x < N; ++x) acc[x] = fmaf(v[x], fi, acc[x]);
      }
    }
    if (N == 4) {
      store_row4<QBF16, E4M3>(p, rec.first_row, rec.head, rec.row0 + row, lane, make_float4(acc[0], acc[1], acc[N - 2], acc[N - 1]), l);
    } else {
      const float ox = __shfl_down_sync(0xffffffffu, acc[0], 1), oy = __shfl_down_sync(0xffffffffu, acc[1], 1);
      if (!(lane & 1)) store_row4<QBF16, E4M3>(p, rec.first_row, rec.head, rec.row0 + row, lane >> 1, make_float4(acc[0], acc[1], ox, oy), l);
    }
  }
}

template <bool QBF16, bool E4M3, int D, int MT>
int launch_rows(frisk_b200_ctx* ctx, const CacheAttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, unsigned grid, cudaStream_t s) {
  auto kern = cache_attention_kernel<QBF16, E4M3, D, MT>;
  using L = RowSmem<D, E4M3, MT>;
  static PerDeviceOnce opt_in;
  if (opt_in(ctx->device, [&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) == cudaSuccess ? 0 : 1;
      }))
    return FRISK_B200_E_CUDA;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernels wait (griddepcontrol.wait) themselves
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreadsRow);
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
  const int rc = tile_rows == 16   ? launch_rows<QBF16, E4M3, D, 1>(ctx, p, tk, tv, grid, s)
                 : tile_rows == 32 ? launch_rows<QBF16, E4M3, D, 2>(ctx, p, tk, tv, grid, s)
                                   : launch_cache_attention_tiles(ctx, p, tk, tv, grid, QBF16, E4M3, D, tile_rows, s);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid, (unsigned)std::min(tile_rows / 4, 16));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FB_CUDA(ctx, cudaLaunchKernelEx(&cfg, cache_attention_join_kernel<QBF16, E4M3, D>, p, tile_rows));
  return 0;
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
  // units are counted in 32 bits (16 rows and 64 keys at least)
  const double tiles = ((double)c->table_width * c->page + kKeys - 1) / kKeys, group = a->heads_q / c->heads;
  if (tiles * c->heads * (c->rows * group / 16 + c->batch) > 2147483647.0 || (double)c->table_width * c->page > 2147483647.0 ||
      (double)c->rows * group > 2147483647.0)
    return FRISK_B200_E_TOO_LARGE;
  return 0;
}

// Query rows a tile, by the rows that a sequence is said to have for a key head.  (A sequence with more than a tile's rows takes several
// tiles, so a hint that is too low costs time only.)
int tile_rows_of(const frisk_b200_cache_desc* c, const frisk_b200_cache_attn_desc* a) {
  const int64_t per = a->max_new > 0 ? a->max_new : c->batch > 0 ? (c->rows + c->batch - 1) / c->batch : 1;
  const int64_t rows = per * (a->heads_q / c->heads);
  return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 128 ? 128 : 256;
}

}  // namespace
}  // namespace fb

using namespace fb;
using namespace fb::cache;

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
  if ((a->heads_q > 1 && out->head_stride < c->D) || (c->rows > 1 && out->row_stride < (a->heads_q - 1) * out->head_stride + c->D))
    return FRISK_B200_E_CACHE_SHAPE;
  const size_t need = frisk_b200_cache_attention_workspace_bytes(c, a);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return FRISK_B200_E_WORKSPACE;
  const size_t ob = packed_span(*out, c->rows, a->heads_q, c->D, 2), qb = packed_span(*q, c->rows, a->heads_q, c->D, 2);
  const size_t mb = mask ? (size_t)((c->rows - 1) * a->mask_stride + a->mask_width) : 0;
  for (int w = 0; w < 2; ++w) {  // what is written: the results and the workspace
    const void* ptr = w ? workspace : out->ptr;
    const size_t n = w ? need : ob;
    if (ranges_overlap(ptr, n, q->ptr, qb) || (mask && ranges_overlap(ptr, n, mask, mb)) || cache_overlaps(c, ptr, n) || tables_overlap(c, ptr, n))
      return FRISK_B200_E_OVERLAP;
  }
  if (ranges_overlap(workspace, need, out->ptr, ob)) return FRISK_B200_E_OVERLAP;

  FB_DEVICE(ctx);
  const bool e4m3 = c->dtype == FRISK_B200_E4M3, bf16 = a->dtype == FRISK_B200_BF16;
  // lines of 128 bytes: one key or half of one at 16 bits, one or two at 8
  const uint64_t tokens = (uint64_t)c->pages * c->heads * c->page;
  const int box_rows = std::min(c->page, kKeys);
  CUtensorMap tk, tv;
  const int map_type = e4m3 ? FRISK_B200_F16 : c->dtype;
  const uint64_t inner = e4m3 ? 64 : c->D, outer = e4m3 ? tokens * c->D / 128 : tokens;
  const uint32_t box = e4m3 ? box_rows * c->D / 128 : box_rows;
  rc = encode_tmap_2d(ctx, &tk, map_type, c->k, inner, outer, inner * 2, 64, box, true);
  if (!rc) rc = encode_tmap_2d(ctx, &tv, map_type, c->v, inner, outer, inner * 2, 64, box, true);
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
  const unsigned grid = (unsigned)std::min(ctx->num_sms, kNumSMsDefault);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rows = tile_rows_of(c, a);
  if (c->D == 64)
    return bf16 ? (e4m3 ? launch_all<true, true, 64>(ctx, p, tk, tv, grid, rows, s) : launch_all<true, false, 64>(ctx, p, tk, tv, grid, rows, s))
                : (e4m3 ? launch_all<false, true, 64>(ctx, p, tk, tv, grid, rows, s) : launch_all<false, false, 64>(ctx, p, tk, tv, grid, rows, s));
  return bf16 ? (e4m3 ? launch_all<true, true, 128>(ctx, p, tk, tv, grid, rows, s) : launch_all<true, false, 128>(ctx, p, tk, tv, grid, rows, s))
              : (e4m3 ? launch_all<false, true, 128>(ctx, p, tk, tv, grid, rows, s) : launch_all<false, false, 128>(ctx, p, tk, tv, grid, rows, s));
}
