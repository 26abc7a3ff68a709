// Low-rank adapters over long sequences, on tcgen05: two launches.
//
// sums      x A^T of 128 rows: a cluster of eight CTAs shares K, each brings its part of x and A through a TMA ring to tcgen05.mma; the parts meet
//           through distributed shared memory, 16 rows a CTA, and leave as 16-bit terms (adapters.cu) for the second launch: R terms a row
//           where x has K, so they stay in the L2.  It also writes the table of tiles.
// columns   c + terms B^T: items of 128 rows x 128 columns, dealt out in order, so a CTA keeps the terms of its rows in shared memory while it
//           goes along the columns.  One warp brings B, one issues, eight add c, which they load while the product is made, and store.
//
// Why not in one: the columns need all of K, and a CTA that made the sums for itself would read x as often as there are CTAs along the columns.  Why not mma.sync:
// at R = 64 its rate is the whole time (7000 rows, K 4096, N 8192: 43 us, the floor at HBM's rate too; the kernel of adapters.cu took 330, with loads that nothing hid).
//
// Bound by HBM (x, c and the result once) and by a chain of barriers, MMAs and adding warps beside it: 71 us for these rows, 17 the sums (3.3 TB/s: 236 CTAs on 148 SMs, and 5
// us of tables, meeting and terms), 49 the columns (4.7 TB/s).
#include <algorithm>

#include "adapters.cuh"
#include "box_rows.cuh"
#include "gemm_common.cuh"

namespace fb {
namespace {
using namespace adapter;

enum : unsigned { ST_SUMS_EMPTY = 0x311, ST_SUMS_FULL = 0x312, ST_SUMS_PART = 0x313, ST_COLUMNS = 0x314 };  // waits

constexpr int kRows = 128;          // of a tile
constexpr int kBoxBytes = kRows * 128;  // 128 rows of 64 16-bit elements
constexpr int kMostCtas = 8;        // share the K of a tile

// The workspace: terms [terms][rows][R], what undoes the rows' powers of two [rows], tiles [most], their number
struct Work {
  uint16_t* terms;
  float* down;
  int4* tiles;  // first row, rows, adapter
  int* count;
};
int64_t most_tiles(int64_t rows, int64_t batch) { return std::min<int64_t>(rows, rows / kRows + batch); }
size_t up(size_t n) { return (n + 255) / 256 * 256; }
Work work_of(void* ws, int64_t rows, int R, int64_t batch) {
  uint8_t* at = static_cast<uint8_t*>(ws);
  Work w;
  w.terms = reinterpret_cast<uint16_t*>(at);
  at += up((size_t)rows * R * kTerms * 2);
  w.down = reinterpret_cast<float*>(at);
  at += up((size_t)rows * 4);
  w.tiles = reinterpret_cast<int4*>(at);
  at += up((size_t)most_tiles(rows, batch) * 16);
  w.count = reinterpret_cast<int*>(at);
  return w;
}

__device__ __forceinline__ void land(volatile uint32_t* abort_flag) {
  if (!*abort_flag) return;
  const unsigned long long t0 = globaltimer();  // a wait ran out somewhere: give copies that are still in flight time to land
  while (globaltimer() - t0 < 200000ull) __nanosleep(1000);
}

// ------------------------------------------------------------------------------------------------ sums
constexpr int kSumStages = 4, kAdders = 8, kSumThreads = 64 + 32 * kAdders;
// The tensor cores cut what an addition leaves below 24 bits, always towards zero, so a chain of n additions is off by some 2e-8 n of its result (K = 8192 in
// two CTAs: 5e-6).  So no accumulator takes more than 8 steps of 16, and the adders sum up what they leave, rounding to nearest (3e-7).
constexpr int kChain = 2;  // stages that an accumulator takes
struct SumsLayout {  // of `width` columns, R rounded up to a multiple of 16
  static __host__ __device__ int stage_bytes(int width) { return kBoxBytes + width * 128; }
  static __host__ __device__ int pitch(int width) { return width + 4; }  // of rows of sums, floats
  static __host__ __device__ int bytes(int width) { return kSumStages * stage_bytes(width) + 1024; }
};

template <typename T, int kMost>  // kMost: the rank at most, 64 or 128
__global__ void __launch_bounds__(kSumThreads)
    adapter_sums_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ AdapterParams p,
                        const __grid_constant__ Work work) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full_bar[kSumStages], empty_bar[kSumStages], part_full[2], part_empty[2];
  __shared__ uint32_t tmem_slot, abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ctas = p.cluster, rank = (int)cluster_ctarank(), tile = blockIdx.x / ctas;
  const int width = (p.R + 15) / 16 * 16, columns = width <= 16 ? 32 : width <= 32 ? 64 : width <= 64 ? 128 : 256, stage_bytes = SumsLayout::stage_bytes(width);
  if (tid == 0) {
    for (int i = 0; i < kSumStages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&part_full[i], 1);
      mbar_init(&part_empty[i], kAdders);
    }
    abort_word = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_a);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Tile found = find_tile<kSumThreads>(p, tile, kRows, tile == 0);
  // (no more than there are places: sequences behind one whose rows are out of range may name rows again)
  if (tile == 0 && rank == 0 && tid == 0) *work.count = min(found.counted, (int)gridDim.x / ctas);
  if (found.seq < 0) return;  // (the whole cluster, here and below)
  const int which = found.which;
  if (rank == 0 && tid == 0) work.tiles[tile] = make_int4(found.row, found.rows, which, 0);
  if (which < 0) return;
  if (warp == 1) {
    tmem_alloc(&tmem_slot, columns);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const int blocks = (p.K + 63) / 64, k0 = (int)((int64_t)blocks * rank / ctas), n_k = (int)((int64_t)blocks * (rank + 1) / ctas) - k0;

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < n_k; ++i) {
        const int stage = i % kSumStages;
        if (i >= kSumStages && !mbar_wait(&empty_bar[stage], (i / kSumStages - 1) & 1, abort_flag, p.status, ST_SUMS_EMPTY)) break;
        unsigned char* at = smem + stage * stage_bytes;
        mbar_expect_tx(&full_bar[stage], stage_bytes);
        tma_load_2d(at, &map_x, &full_bar[stage], (k0 + i) * 64, found.row);
        tma_load_3d(at + kBoxBytes, &map_a, &full_bar[stage], (k0 + i) * 64, 0, which);
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_f16(kRows, width, kBf16, false, false), d = __shfl_sync(0xffffffffu, tmem, 0);
    for (int i = 0; i < n_k; ++i) {
      const int stage = i % kSumStages, chain = i / kChain, acc = chain & 1;
      if (i % kChain == 0 && chain >= 2 && !mbar_wait_warp(&part_empty[acc], (chain / 2 - 1) & 1, abort_flag, p.status, ST_SUMS_PART)) break;
      if (!mbar_wait_warp(&full_bar[stage], (i / kSumStages) & 1, abort_flag, p.status, ST_SUMS_FULL)) break;
      tc_fence_after_sync();
      const uint32_t at = smem_u32(smem + stage * stage_bytes);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16_ss(d + acc * (columns / 2), umma_desc_kmajor_sw128(at + k * 32), umma_desc_kmajor_sw128(at + kBoxBytes + k * 32), idesc, i % kChain > 0 || k > 0 ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
        if (i % kChain == kChain - 1 || i + 1 == n_k) umma_commit(&part_full[acc]);
      }
      __syncwarp();
    }
  } else {
    // lane = row; a warp has every other 16 columns
    constexpr int kGroups = kMost / 32;
    const int row = (warp & 3) * 32 + lane, half = (warp - 2) >> 2, pitch = SumsLayout::pitch(width);
    float sum[kGroups][16];
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[g][i] = 0.f;
    const int chains = (n_k + kChain - 1) / kChain;
    for (int chain = 0; chain < chains; ++chain) {
      const int acc = chain & 1;
      if (!mbar_wait_warp(&part_full[acc], (chain >> 1) & 1, abort_flag, p.status, ST_SUMS_PART)) break;
      tc_fence_after_sync();
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int c = (2 * g + half) * 16;
        if (c >= width) break;
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + acc * (columns / 2) + c + ((uint32_t)((warp & 3) * 32) << 16), v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[g][i] += __uint_as_float(v[i]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&part_empty[acc]);
    }
    // this CTA's part into the ring, all of which has been read
    float* mine = reinterpret_cast<float*>(smem) + row * pitch;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int c = (2 * g + half) * 16;
      if (c >= width) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(mine + c + 4 * i) = make_float4(sum[g][4 * i], sum[g][4 * i + 1], sum[g][4 * i + 2], sum[g][4 * i + 3]);
    }
  }
  __syncwarp();
  cluster_sync_all();  // every part is there (all roles of all CTAs end: their waits are bounded)
  if (warp >= 2) {
    // Eight threads a row, four neighbours each in turns of 32; the parts in the order of the CTAs.
    const int t = tid - 64, quads = width / 4, pitch = SumsLayout::pitch(width), each = kRows / ctas;
#pragma unroll 1
    for (int row = rank * each + (t >> 3); row < (rank + 1) * each; row += 4 * kAdders) {
      const bool valid = row < found.rows;
      float4 v[kMaxRank / 32];
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < kMaxRank / 32; ++j) {
        const int quad = (t & 7) + 8 * j;
        v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (valid && quad < quads) {
          const uint32_t at = smem_u32(smem) + (row * pitch + quad * 4) * 4;
          float4 part[kMostCtas];
#pragma unroll
          for (int r = 0; r < kMostCtas; ++r) part[r] = r < ctas ? ld_cluster_f4(mapa_addr(at, r)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int r = 0; r < kMostCtas; ++r) {
            v[j].x += part[r].x; v[j].y += part[r].y; v[j].z += part[r].z; v[j].w += part[r].w;
          }
          most = fmaxf(fmaxf(fmaxf(most, finite_magnitude(v[j].x)), finite_magnitude(v[j].y)), fmaxf(finite_magnitude(v[j].z), finite_magnitude(v[j].w)));
        }
      }
      float up = 1.f;
      if (!kBf16) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        up = row_power(most);
      }
      if (valid && (t & 7) == 0) work.down[found.row + row] = 1.f / up;  // (of a power of two: exact)
#pragma unroll
      for (int j = 0; j < kMaxRank / 32; ++j) {
        const int k = ((t & 7) + 8 * j) * 4;
        if (!valid || k >= p.R) continue;
        uint32_t lo[kTerms], hi[kTerms];
        split<T>(v[j].x * up, v[j].y * up, lo);
        split<T>(v[j].z * up, v[j].w * up, hi);
#pragma unroll
        for (int n = 0; n < kTerms; ++n) *reinterpret_cast<uint2*>(work.terms + ((int64_t)n * p.rows + found.row + row) * p.R + k) = make_uint2(lo[n], hi[n]);
      }
    }
  }
  __syncwarp();
  cluster_sync_all();  // nobody reads a peer any more
  land(abort_flag);
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, columns);
  }
}

// ------------------------------------------------------------------------------------------------ columns
constexpr int kColumns = 128;   // of an item
constexpr int kWriters = 16;    // warps that add c and store, eight an item in turn
constexpr int kColThreads = 64 + 32 * kWriters;
constexpr int kBox = 32 * 128;   // bytes of a writer's box of c and results: 32 rows of 128 bytes

template <int kHalves>  // halves: 64 of R each
struct ColumnsLayout {
  static constexpr int kTermBytes = kTerms * kHalves * kBoxBytes;
  static constexpr int kStages = 2;
  static constexpr int kStageBytes = kHalves * kBoxBytes;
  static constexpr int kBoxes = kHalves == 1 ? 2 : 1;  // of a writer, in flight or at work
  static constexpr int kBoxOffset = kTermBytes + kStages * kStageBytes;
  static constexpr int kBytes = kBoxOffset + kWriters * kBoxes * kBox + 1024;
  static_assert(kBytes <= 232448 - 1024, "shared memory of a CTA");
};

// A writer's way through its CTA's items, every other one: 32 rows and 64 columns of each, in boxes of `wide` columns.  Boxes that hold nothing are left out.
struct Way {
  const AdapterParams& p;
  const int4* tiles;
  int across, quarter, half, wide, n_items;
  bool in_place;
  int item, tile, column, box, held;
  int4 t;       // the tile: first row, rows, adapter
  int left, rows, col, cols;  // of the box: the tile's rows from its first on; rows and columns that are there
  __device__ __forceinline__ Way(const AdapterParams& p, const int4* tiles, int across, int quarter, int half, int wide, int n_items, int tile, int column, int turn)
      : p(p), tiles(tiles), across(across), quarter(quarter), half(half), wide(wide), n_items(n_items), in_place(p.c == p.out), item(turn), tile(tile), column(column + turn), box(-1),
        held(-1), t(make_int4(0, 0, -1, 0)) {
    wrap();
  }
  __device__ __forceinline__ void wrap() {
    while (column >= across) {
      column -= across;
      ++tile;
    }
  }
  __device__ __forceinline__ bool item_read() {  // the item's tile
    if (item >= n_items) return false;
    if (held != tile) {
      held = tile;
      t = tiles[tile];
      left = t.y - quarter * 32;
      rows = left <= 0 ? 0 : left >= 32 ? 32 : left;
    }
    return true;
  }
  __device__ __forceinline__ void next_item() {
    item += 2;
    column += 2;
    box = -1;
    wrap();
  }
  // the next box of the item, if it has one
  __device__ __forceinline__ bool next_box() {
    if (rows == 0 || (t.z < 0 && in_place) || ++box == 64 / wide) return false;
    col = column * kColumns + half * 64 + box * wide;
    cols = min(wide, p.N - col);
    return cols > 0;
  }
  // the next box of all
  __device__ __forceinline__ bool next() {
    while (item_read()) {
      if (next_box()) return true;
      next_item();
    }
    return false;
  }
};

template <typename T, typename C, int kHalves>
__global__ void __launch_bounds__(kColThreads, 1)
    adapter_columns_kernel(const __grid_constant__ CUtensorMap map_t, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c,
                           const __grid_constant__ CUtensorMap map_out, const __grid_constant__ AdapterParams p, const __grid_constant__ Work work, const bool c_by_tma,
                           const bool out_by_tma) {
  using L = ColumnsLayout<kHalves>;
  constexpr int kStages = L::kStages;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t terms_full, terms_empty, b_full[kStages], b_empty[kStages], acc_full[2], acc_empty[2], box_full[kWriters * L::kBoxes];
  __shared__ uint32_t tmem_slot, abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&terms_full, 1);
    mbar_init(&terms_empty, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&b_full[i], 1);
      mbar_init(&b_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kWriters / 2);
    }
    for (int i = 0; i < kWriters * L::kBoxes; ++i) mbar_init(&box_full[i], 1);
    abort_word = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_t);
    tma_prefetch_desc(&map_b);
    if (c_by_tma) tma_prefetch_desc(&map_c);
    if (out_by_tma) tma_prefetch_desc(&map_out);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 2 * kColumns);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  // this CTA's items: tile by tile, along the columns
  const int across = (p.N + kColumns - 1) / kColumns;
  const int64_t items = (int64_t)*work.count * across;
  const int64_t first = items * blockIdx.x / gridDim.x, last = items * (blockIdx.x + 1) / gridDim.x;
  const int tile0 = (int)(first / across), col0 = (int)(first - (int64_t)tile0 * across);
  const int n_items = (int)(last - first);

  if (warp == 0) {
    if (lane == 0) {
      int tile = tile0, column = col0, held = -1, which = -1, row = 0, stage = 0;
      uint32_t phase = 0, terms_phase = 0;
      for (int i = 0; i < n_items; ++i) {
        if (held != tile) {
          const int4 t = work.tiles[tile];
          held = tile;
          which = t.z;
          row = t.x;
          if (which >= 0) {
            if (!mbar_wait(&terms_empty, terms_phase ^ 1, abort_flag, p.status, ST_COLUMNS)) break;
            terms_phase ^= 1;
            mbar_expect_tx(&terms_full, L::kTermBytes);
#pragma unroll
            for (int n = 0; n < kTerms; ++n)
#pragma unroll
              for (int h = 0; h < kHalves; ++h) tma_load_3d(smem + (n * kHalves + h) * kBoxBytes, &map_t, &terms_full, 64 * h, row, n);
          }
        }
        if (which >= 0) {
          if (!mbar_wait(&b_empty[stage], phase ^ 1, abort_flag, p.status, ST_COLUMNS)) break;
          mbar_expect_tx(&b_full[stage], L::kStageBytes);
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            tma_load_3d(smem + L::kTermBytes + stage * L::kStageBytes + h * kBoxBytes, &map_b, &b_full[stage], 64 * h, column * kColumns, which);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (++column == across) {
          column = 0;
          ++tile;
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc_f16(kRows, kColumns, std::is_same<T, __nv_bfloat16>::value, false, false);
    const uint32_t d = __shfl_sync(0xffffffffu, tmem, 0);
    const int steps = (p.R + 15) / 16;
    int tile = tile0, column = col0, held = -1, which = -1, stage = 0;
    uint32_t phase = 0, terms_phase = 0, acc_phases = 0;
    for (int i = 0; i < n_items; ++i) {
      if (held != tile) {
        held = tile;
        which = work.tiles[tile].z;
        if (which >= 0) {
          if (!mbar_wait_warp(&terms_full, terms_phase, abort_flag, p.status, ST_COLUMNS)) break;
          terms_phase ^= 1;
        }
      }
      if (which >= 0) {
        const int acc = i & 1;  // (whose writers take the item)
        if (!mbar_wait_warp(&acc_empty[acc], (acc_phases >> acc & 1) ^ 1, abort_flag, p.status, ST_COLUMNS)) break;
        acc_phases ^= 1u << acc;
        if (!mbar_wait_warp(&b_full[stage], phase, abort_flag, p.status, ST_COLUMNS)) break;
        tc_fence_after_sync();
        const uint32_t at = smem_u32(smem), b = at + L::kTermBytes + stage * L::kStageBytes;
        if (elect_one()) {
#pragma unroll
          for (int n = kTerms - 1; n >= 0; --n)  // (the smallest first: what the additions cut off them is the less)
            for (int k = 0; k < steps; ++k) {
              const uint32_t in = (k >> 2) * kBoxBytes + (k & 3) * 32;
              umma_f16_ss(d + acc * kColumns, umma_desc_kmajor_sw128(at + n * kHalves * kBoxBytes + in), umma_desc_kmajor_sw128(b + in), idesc, n < kTerms - 1 || k > 0 ? 1u : 0u);
            }
          umma_commit(&b_empty[stage]);
          umma_commit(&acc_full[acc]);
          if (column + 1 == across) umma_commit(&terms_empty);  // the tile's last item
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (++column == across) {
        column = 0;
        ++tile;
      }
    }
  } else {
    // Eight warps have the even items, eight the odd ones (one after the other they would take the time of each box's chain of waits, 1.9 us, for each item).  A warp
    // has 32 rows (its quarter of tensor memory) and 64 columns.  Boxes of c come by TMA, the next while one is at work; a lane adds the results of its row
    // where c stands; eight rows leave at a time, by TMA, and those of a tile that ends among eight one by one.
    const int quarter = warp & 3, half = (warp - 2) >> 2 & 1, acc = (warp - 2) >> 3;
    constexpr int U = 128 / (int)sizeof(C), kBoxes = L::kBoxes;
    unsigned char* boxes = smem + L::kBoxOffset + (warp - 2) * kBoxes * kBox;
    uint64_t* bars = box_full + (warp - 2) * kBoxes;
    const C* const c = static_cast<const C*>(p.c);
    C* const out = static_cast<C*>(p.out);
    Way now(p, work.tiles, across, quarter, half, U, n_items, tile0, col0, acc), ahead(p, work.tiles, across, quarter, half, U, n_items, tile0, col0, acc);
    int slot = 0, ahead_slot = 0;
    uint32_t phases = 0, acc_phase = 0;
    bool ok = true, more = c_by_tma;
    auto fetch = [&]() {  // the next box ahead, into a slot that has been read and stored from
      if (!more || !(more = ahead.next())) return;
      if (lane == 0) {
        mbar_expect_tx(&bars[ahead_slot], kBox);
        tma_load_2d(boxes + ahead_slot * kBox, &map_c, &bars[ahead_slot], ahead.col, ahead.t.x + quarter * 32);
      }
      ahead_slot = ahead_slot + 1 == kBoxes ? 0 : ahead_slot + 1;
    };
#pragma unroll 1
    for (int i = 0; i < kBoxes; ++i) fetch();
    int held = -1;
    float scale = 1.f, down = 1.f;  // (one after the other: their product may leave fp32's range)
    for (; ok && now.item_read(); now.next_item()) {
      const bool product = now.t.z >= 0;
      if (held != now.tile) {
        held = now.tile;
        scale = product && p.scales ? p.scales[now.t.z] : 1.f;
        down = std::is_same<T, __half>::value && product && lane < now.rows ? work.down[now.t.x + quarter * 32 + lane] : 1.f;
      }
      if (product) {
        if (!mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag, p.status, ST_COLUMNS)) break;
        tc_fence_after_sync();
      }
      const uint32_t results = tmem + acc * kColumns + half * 64 + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      while (now.next_box()) {
        unsigned char* box = boxes + slot * kBox;
        uint4* const mine = reinterpret_cast<uint4*>(box + lane * 128);
        const int64_t row0 = now.t.x + quarter * 32;
        if (c_by_tma) {
          ok = mbar_wait_warp(&bars[slot], (phases >> slot) & 1, abort_flag, p.status, ST_COLUMNS);
          if (!ok) break;
          phases ^= 1u << slot;
        } else {
          load_box_rows(c + row0 * p.ldc + now.col, p.ldc, now.rows, now.cols, lane, [&](int r, uint32_t w) {
            *reinterpret_cast<uint32_t*>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = w;
          });
        }
        __syncwarp();
        if (product) {
          constexpr int kEach = 16 / (int)sizeof(C);  // columns of 16 bytes
#pragma unroll
          for (int h = 0; h < U / 32; ++h) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(results + now.box * U + h * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32 / kEach; ++j) {
              uint4& at = mine[(h * (32 / kEach) + j) ^ (lane & 7)];
              const uint4 old = at;
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float2 f = gemm_detail::unpack_out<C>(word(old, e));
                constexpr int kIn = kEach / 4;  // columns of a word
                const float d0 = __uint_as_float(v[j * kEach + e * kIn]), d1 = __uint_as_float(v[j * kEach + e * kIn + kIn - 1]);
                f.x = fmaf(scale, std::is_same<T, __half>::value ? d0 * down : d0, f.x);
                f.y = fmaf(scale, std::is_same<T, __half>::value ? d1 * down : d1, f.y);
                w[e] = gemm_detail::pack_out<C>(f.x, f.y);
              }
              at = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        // (`rows` is not clamped by max(0, min(32, left)): nvcc 12.9 made left <= 32 of a comparison of that with 32)
        const int by_tma = out_by_tma ? now.rows & ~7 : 0;
        if (lane < 4 && 8 * lane < by_tma) {
          tma_store_2d(&map_out, box + lane * 1024, now.col, (int)row0 + 8 * lane);
          tma_store_commit();
        }
        if (by_tma < now.rows) {
          store_box_rows(out + (row0 + by_tma) * p.ldo + now.col, p.ldo, now.rows - by_tma, now.cols, lane, [&](int r) {
            return *reinterpret_cast<const uint32_t*>(box + (by_tma + r) * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
          });
          fence_proxy_async_smem();
        }
        if (lane < 4) tma_store_wait_read<0>();
        __syncwarp();
        slot = slot + 1 == kBoxes ? 0 : slot + 1;
        fetch();
      }
      if (product) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
        acc_phase ^= 1;
      }
    }
    if (lane < 4) tma_store_wait<0>();  // the boxes are read and written out before the CTA leaves
  }
  __syncwarp();
  land(abort_flag);
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, 2 * kColumns);
  }
}

// ------------------------------------------------------------------------------------------------ launches
template <typename... A>
cudaError_t launch(void (*kernel)(A...), int64_t blocks, int threads, int cluster, int smem, cudaStream_t s, const typename std::common_type<A>::type&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernels wait (griddepcontrol.wait) themselves
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename K>
cudaError_t allow(PerDeviceOnce& once, int device, K kernel, int smem) {
  cudaError_t e = cudaSuccess;
  once(device, [&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    return e == cudaSuccess ? 0 : 1;
  });
  return e;
}

template <typename T, typename C, int kHalves>
int launch_both(frisk_b200_ctx* ctx, AdapterParams p, const Work& work, cudaStream_t s) {
  constexpr int dtype = std::is_same<T, __half>::value ? FRISK_B200_F16 : FRISK_B200_BF16;
  using L = ColumnsLayout<kHalves>;
  const int width = (p.R + 15) / 16 * 16;
  CUtensorMap map_x, map_a, map_t, map_b, map_c{}, map_out{};
  const int64_t a_step = p.count > 1 ? p.a_step : p.lda * p.R, b_step = p.count > 1 ? p.b_step : p.ldb * p.N;
  int bad = encode_tmap_2d(ctx, &map_x, dtype, p.x, p.K, p.rows, p.ldx * 2, 64, kRows, true);
  bad |= encode_tmap_3d(ctx, &map_a, dtype, p.a, p.K, p.R, p.count, p.lda * 2, a_step * 2, 64, width, 1, true);
  bad |= encode_tmap_3d(ctx, &map_t, dtype, work.terms, p.R, p.rows, kTerms, p.R * 2, p.rows * p.R * 2, 64, kRows, 1, true);
  bad |= encode_tmap_3d(ctx, &map_b, dtype, p.b, p.R, p.N, p.count, p.ldb * 2, b_step * 2, 64, kColumns, 1, true);
  // c comes by TMA, and results leave by it, where rows begin on 16 bytes; a store clips at 16 bytes too
  constexpr int dtype_c = sizeof(C) == 4 ? FRISK_B200_F32 : dtype, U = 128 / (int)sizeof(C);
  const bool c_by_tma = (reinterpret_cast<uintptr_t>(p.c) & 15u) == 0 && p.ldc * (int64_t)sizeof(C) % 16 == 0;
  const bool out_by_tma = (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0 && p.ldo * (int64_t)sizeof(C) % 16 == 0 && p.N * (int64_t)sizeof(C) % 16 == 0;
  if (c_by_tma) bad |= encode_tmap_2d(ctx, &map_c, dtype_c, p.c, p.N, p.rows, p.ldc * sizeof(C), U, 32, true);
  if (out_by_tma) bad |= encode_tmap_2d(ctx, &map_out, dtype_c, p.out, p.N, p.rows, p.ldo * sizeof(C), U, 8, true);
  if (bad) return FRISK_B200_E_CUDA;
  static PerDeviceOnce once_sums, once_columns;
  auto sums = adapter_sums_kernel<T, 64 * kHalves>;
  auto columns = adapter_columns_kernel<T, C, kHalves>;
  FB_CUDA(ctx, allow(once_sums, ctx->device, sums, SumsLayout::bytes(64 * kHalves)));
  FB_CUDA(ctx, allow(once_columns, ctx->device, columns, L::kBytes));
  const int64_t tiles = most_tiles(p.rows, p.batch), items = tiles * ((p.N + kColumns - 1) / kColumns);
  p.cluster = kMostCtas;
  while (p.cluster > 2 && tiles * p.cluster > 2 * ctx->num_sms) p.cluster /= 2;
  FB_CUDA(ctx, launch(sums, tiles * p.cluster, kSumThreads, p.cluster, SumsLayout::bytes(width), s, map_x, map_a, p, work));
  FB_CUDA(ctx, launch(columns, std::min<int64_t>(items, ctx->num_sms), kColThreads, 1, L::kBytes, s, map_t, map_b, map_c, map_out, p, work, c_by_tma, out_by_tma));
  return 0;
}

}  // namespace

// Long sequences, if adapters lie one behind the other (no tensor map has a step of 0).  How long is measured, K = N = 4096, 4 to 64 adapters, here and in adapters.cu, us:
// rank 32, 16-bit results 100 sequences of 48 rows 56 and 67, 64 of 64 rows 44 and 38, 64 of 100 rows 53 and 67; 32-bit ones 128 of 32 rows 74 and 67, 64 of 64 rows 55 and 65;
// rank 64, 64 of 24 rows 43 and 41, 128 of 32 rows 67 and 80; rank 128, 64 of 16 rows 58 and 49, of 24 rows 53 and 63, 24 of 24 rows 39 and 27 to 60.
// No border of the mean is right everywhere (the first pair is on the wrong side of it), and one long sequence beside many short ones is taken whole by either kernel: lengths are
// known on the device only.  2000 rows and 60 tokens, rank 32 and 64: 33 and 51, in two calls 20 + 11 and 22 + 12; 4096 rows and 255 tokens, rank 64 and 128: 82 and 119,
// in two calls 33 + 19 and 56 + 24.
size_t adapter_tiles_workspace_bytes(const frisk_b200_adapter_desc& d) {
  const int64_t longest = d.rank > 64 ? 20 : d.rank > 32 ? 28 : d.dtype_c == FRISK_B200_F32 ? 40 : 64;  // mean rows that adapters.cu takes
  if (d.batch < 1 || d.rows < 512 || d.rows <= longest * d.batch || d.count < 1) return 0;
  if (d.count > 1 && (d.a_step < d.lda || d.b_step < d.ldb)) return 0;
  if (most_tiles(d.rows, d.batch) * ((d.N + kColumns - 1) / kColumns) > INT32_MAX || d.rows * (int64_t)d.rank > INT32_MAX) return 0;
  return up((size_t)d.rows * d.rank * kTerms * 2) + up((size_t)d.rows * 4) + up((size_t)most_tiles(d.rows, d.batch) * 16) + 256;
}

int launch_adapter_tiles(frisk_b200_ctx* ctx, const frisk_b200_adapter_desc& d, const AdapterParams& p, void* workspace, cudaStream_t s) {
  const bool f32 = d.dtype_c == FRISK_B200_F32, half = d.dtype == FRISK_B200_F16;
  const Work work = work_of(workspace, p.rows, p.R, p.batch);
  if (p.R <= 64) {
    if (half) return f32 ? launch_both<__half, float, 1>(ctx, p, work, s) : launch_both<__half, __half, 1>(ctx, p, work, s);
    return f32 ? launch_both<__nv_bfloat16, float, 1>(ctx, p, work, s) : launch_both<__nv_bfloat16, __nv_bfloat16, 1>(ctx, p, work, s);
  }
  if (half) return f32 ? launch_both<__half, float, 2>(ctx, p, work, s) : launch_both<__half, __half, 2>(ctx, p, work, s);
  return f32 ? launch_both<__nv_bfloat16, float, 2>(ctx, p, work, s) : launch_both<__nv_bfloat16, __nv_bfloat16, 2>(ctx, p, work, s);
}

}  // namespace fb
