// Low-rank adapters over long sequences, on tcgen05: two launches.
//
// sums      x A^T of 128 rows: a cluster of eight CTAs shares K, each brings its part of x and A through a TMA ring to tcgen05.mma; the parts meet
//           through distributed shared memory, 16 rows a CTA, and leave as 16-bit terms (adapters.cu) for the second launch: R terms a row
//           where x has K, so they stay in the L2.  It also writes the table of tiles.
// columns   c + terms B^T: items of 128 rows x 128 columns, dealt out in order, so a CTA keeps the terms of its rows in shared memory while it
//           goes along the columns.  One warp brings B, one issues, eight add c, which they load while the product is made, and store.
//
// Bound by HBM (x, c, out once): mma.sync would need the whole time for the products at R = 64 (7000 rows, K 4096, N 8192: 43 us at its rate, which is the
// floor too; a kernel of adapters.cu's kind took 330).
#include <algorithm>

#include "adapters.cuh"

namespace fb {
namespace {
using namespace adapter;

enum : unsigned { ST_SUMS_EMPTY = 0x311, ST_SUMS_FULL = 0x312, ST_SUMS_DONE = 0x313, ST_COLUMNS = 0x314 };  // waits

constexpr int kRows = 128;          // of a tile
constexpr int kBoxBytes = kRows * 128;  // 128 rows of 64 16-bit elements
constexpr int kCtas = 8;            // share the K of a tile

// The workspace: terms [terms][rows][R], what undoes the rows' powers of two [rows], tiles [most], their number
struct Work {
  uint16_t* terms;
  float* down;
  int4* tiles;  // first row, rows, adapter
  int* count;
};
int64_t most_tiles(int64_t rows, int64_t batch) { return std::min<int64_t>(rows, rows / kRows + batch); }
size_t up(size_t n) { return (n + 255) / 256 * 256; }
Work work_of(void* ws, int64_t rows, int R, int terms, int64_t batch) {
  uint8_t* at = static_cast<uint8_t*>(ws);
  Work w;
  w.terms = reinterpret_cast<uint16_t*>(at);
  at += up((size_t)rows * R * terms * 2);
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
constexpr int kSumStages = 4, kSumThreads = 192;
struct SumsLayout {  // of `width` columns, R rounded up to a multiple of 16
  static __host__ __device__ int stage_bytes(int width) { return kBoxBytes + width * 128; }
  static __host__ __device__ int pitch(int width) { return width + 4; }  // of rows of sums, floats
  static __host__ __device__ int bytes(int width) { return kSumStages * stage_bytes(width) + 1024; }
};

template <typename T, int kTerms>
__global__ void __launch_bounds__(kSumThreads) __cluster_dims__(kCtas, 1, 1)
    adapter_sums_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ AdapterParams p,
                        const __grid_constant__ Work work) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full_bar[kSumStages], empty_bar[kSumStages], done_bar;
  __shared__ uint32_t tmem_slot, abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster_ctarank(), tile = blockIdx.x / kCtas;
  const int width = (p.R + 15) / 16 * 16, columns = width <= 32 ? 32 : width <= 64 ? 64 : 128, stage_bytes = SumsLayout::stage_bytes(width);
  if (tid == 0) {
    for (int i = 0; i < kSumStages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    mbar_init(&done_bar, 1);
    abort_word = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_a);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Tile found = find_tile<kSumThreads>(p, tile, kRows, tile == 0);
  if (tile == 0 && rank == 0 && tid == 0) *work.count = found.counted;
  if (found.seq < 0) return;  // (the whole cluster, here and below)
  const int which = adapter_of(p, found.seq);
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
  const int blocks = (p.K + 63) / 64, k0 = (int)((int64_t)blocks * rank / kCtas), n_k = (int)((int64_t)blocks * (rank + 1) / kCtas) - k0;

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
      const int stage = i % kSumStages;
      if (!mbar_wait_warp(&full_bar[stage], (i / kSumStages) & 1, abort_flag, p.status, ST_SUMS_FULL)) break;
      tc_fence_after_sync();
      const uint32_t at = smem_u32(smem + stage * stage_bytes);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16_ss(d, umma_desc_kmajor_sw128(at + k * 32), umma_desc_kmajor_sw128(at + kBoxBytes + k * 32), idesc, i > 0 || k > 0 ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
        if (i + 1 == n_k) umma_commit(&done_bar);
      }
      __syncwarp();
    }
  } else {
    // this CTA's part into the ring, all of which has been read: lane = row
    const int row = (warp & 3) * 32 + lane, pitch = SumsLayout::pitch(width);
    float* mine = reinterpret_cast<float*>(smem) + row * pitch;
    const bool there = n_k > 0 && mbar_wait_warp(&done_bar, 0, abort_flag, p.status, ST_SUMS_DONE);
    tc_fence_after_sync();
    for (int c = 0; c < width; c += 16) {
      uint32_t v[16];
      if (there) {
        tmem_ld_32x32b_x16(tmem + c + ((uint32_t)((warp & 3) * 32) << 16), v);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(mine + c + 4 * i) =
            make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
    }
    tc_fence_before_sync();
  }
  __syncwarp();
  cluster_sync_all();  // every part is there (all roles of all CTAs end: their waits are bounded)
  if (warp >= 2) {
    // eight threads a row, four neighbours each in turns of 32; the parts in the order of the CTAs
    const int t = tid - 64, row = rank * (kRows / kCtas) + (t >> 3), quads = width / 4, pitch = SumsLayout::pitch(width);
    const bool valid = row < found.rows;
    float4 v[kMaxRank / 32];
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < kMaxRank / 32; ++j) {
      const int quad = (t & 7) + 8 * j;
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (valid && quad < quads) {
        const uint32_t at = smem_u32(smem) + (row * pitch + quad * 4) * 4;
        float4 part[kCtas];
#pragma unroll
        for (int r = 0; r < kCtas; ++r) part[r] = ld_cluster_f4(mapa_addr(at, r));
#pragma unroll
        for (int r = 0; r < kCtas; ++r) {
          v[j].x += part[r].x; v[j].y += part[r].y; v[j].z += part[r].z; v[j].w += part[r].w;
        }
        most = fmaxf(fmaxf(fmaxf(most, fabsf(v[j].x)), fabsf(v[j].y)), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
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
constexpr int kWriters = 8;     // warps that add c and store
constexpr int kColThreads = 64 + 32 * kWriters;
constexpr int kPitch = 36;      // floats of a row of 32 results on their way from lane = row to rows of lanes

template <int kTerms, int kHalves>  // halves: 64 of R each
struct ColumnsLayout {
  static constexpr int kTermBytes = kTerms * kHalves * kBoxBytes;
  static constexpr int kStages = 2;
  static constexpr int kStageBytes = kHalves * kBoxBytes;
  static constexpr int kTurnOffset = kTermBytes + kStages * kStageBytes;
  static constexpr int kBytes = kTurnOffset + kWriters * 32 * kPitch * 4 + 1024;
};

template <typename T, typename C, int kHalves>
__global__ void __launch_bounds__(kColThreads, sizeof(C) == 2 && kHalves == 1 ? 2 : 1)
    adapter_columns_kernel(const __grid_constant__ CUtensorMap map_t, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ AdapterParams p,
                           const __grid_constant__ Work work) {
  constexpr int kTerms = kTermsOf<T, C>;
  using L = ColumnsLayout<kTerms, kHalves>;
  constexpr int kStages = L::kStages;
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t terms_full, terms_empty, b_full[kStages], b_empty[kStages], acc_full[2], acc_empty[2];
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
      mbar_init(&acc_empty[i], kWriters);
    }
    abort_word = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_t);
    tma_prefetch_desc(&map_b);
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
    int tile = tile0, column = col0, held = -1, which = -1, stage = 0, acc = 0;
    uint32_t phase = 0, terms_phase = 0, acc_phase = 0;
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
        if (!mbar_wait_warp(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.status, ST_COLUMNS)) break;
        if (!mbar_wait_warp(&b_full[stage], phase, abort_flag, p.status, ST_COLUMNS)) break;
        tc_fence_after_sync();
        const uint32_t at = smem_u32(smem), b = at + L::kTermBytes + stage * L::kStageBytes;
        if (elect_one()) {
#pragma unroll
          for (int n = 0; n < kTerms; ++n)
            for (int k = 0; k < steps; ++k) {
              const uint32_t in = (k >> 2) * kBoxBytes + (k & 3) * 32;
              umma_f16_ss(d + acc * kColumns, umma_desc_kmajor_sw128(at + n * kHalves * kBoxBytes + in), umma_desc_kmajor_sw128(b + in), idesc, n > 0 || k > 0 ? 1u : 0u);
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
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (++column == across) {
        column = 0;
        ++tile;
      }
    }
  } else {
    // A warp has 32 rows (its quarter of tensor memory) and 64 columns of an item, in two turns of 32.  In a turn a lane has a row's results out of tensor
    // memory, then, through shared memory, 8 neighbours of rows lane / 4, lane / 4 + 8, ...: 64 bytes of a row are 4 lanes' accesses.
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    float* turn = reinterpret_cast<float*>(smem + L::kTurnOffset) + (warp - 2) * 32 * kPitch;
    const C* const c = static_cast<const C*>(p.c);
    C* const out = static_cast<C*>(p.out);
    const bool in_place = p.c == p.out;
    int tile = tile0, column = col0, held = -1, acc = 0;
    uint32_t acc_phase = 0;
    int4 t = make_int4(0, 0, -1, 0);
    float scale = 1.f, down[4] = {1.f, 1.f, 1.f, 1.f};  // (one after the other: their product may leave fp32's range)
    for (int i = 0; i < n_items; ++i) {
      if (held != tile) {
        held = tile;
        t = work.tiles[tile];
        scale = t.z >= 0 && p.scales ? p.scales[t.z] : 1.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int r = quarter * 32 + 8 * n + (lane >> 2);
          if (std::is_same<T, __half>::value && t.z >= 0 && r < t.y) down[n] = work.down[t.x + r];
        }
      }
      const int first_col = column * kColumns + half * 64 + (lane & 3) * 8;
      Eight<C> old[2][4];
      if (t.z >= 0 || !in_place) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int r = quarter * 32 + 8 * n + (lane >> 2), col = first_col + 32 * u;
            old[u][n].load(c + (t.x + r) * p.ldc + col, r < t.y ? p.N - col : 0, p.wide);
          }
      }
      if (t.z >= 0) {
        if (!mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag, p.status, ST_COLUMNS)) break;
        tc_fence_after_sync();
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (t.z >= 0) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(tmem + acc * kColumns + half * 64 + 32 * u + ((uint32_t)(quarter * 32) << 16), v);
          tmem_ld_wait();
          if (u == 1) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(turn + lane * kPitch + 4 * j) =
                make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
          __syncwarp();
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int r = quarter * 32 + 8 * n + (lane >> 2), col = first_col + 32 * u;
          if (r >= t.y || col >= p.N || (t.z < 0 && in_place)) continue;
          float y[8];
          if (t.z >= 0) {
            const float4* from = reinterpret_cast<const float4*>(turn + (8 * n + (lane >> 2)) * kPitch + (lane & 3) * 8);
            const float4 a = from[0], b = from[1];
            const float d[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = fmaf(scale, std::is_same<T, __half>::value ? d[j] * down[n] : d[j], old[u][n][j]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = old[u][n][j];
          }
          store_eight<C>(out + (t.x + r) * p.ldo + col, y, p.N - col, p.wide);
        }
      }
      if (t.z >= 0 && ++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
      if (++column == across) {
        column = 0;
        ++tile;
      }
    }
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
cudaError_t launch(void (*kernel)(A...), int64_t blocks, int threads, int smem, cudaStream_t s, const typename std::common_type<A>::type&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernels wait (griddepcontrol.wait) themselves
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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
int launch_both(frisk_b200_ctx* ctx, const AdapterParams& p, const Work& work, cudaStream_t s) {
  constexpr int kTerms = kTermsOf<T, C>, dtype = std::is_same<T, __half>::value ? FRISK_B200_F16 : FRISK_B200_BF16;
  using L = ColumnsLayout<kTerms, kHalves>;
  const int width = (p.R + 15) / 16 * 16;
  CUtensorMap map_x, map_a, map_t, map_b;
  const int64_t a_step = p.count > 1 ? p.a_step : p.lda * p.R, b_step = p.count > 1 ? p.b_step : p.ldb * p.N;
  int bad = encode_tmap_2d(ctx, &map_x, dtype, p.x, p.K, p.rows, p.ldx * 2, 64, kRows, true);
  bad |= encode_tmap_3d(ctx, &map_a, dtype, p.a, p.K, p.R, p.count, p.lda * 2, a_step * 2, 64, width, 1, true);
  bad |= encode_tmap_3d(ctx, &map_t, dtype, work.terms, p.R, p.rows, kTerms, p.R * 2, p.rows * p.R * 2, 64, kRows, 1, true);
  bad |= encode_tmap_3d(ctx, &map_b, dtype, p.b, p.R, p.N, p.count, p.ldb * 2, b_step * 2, 64, kColumns, 1, true);
  if (bad) return FRISK_B200_E_CUDA;
  static PerDeviceOnce once_sums, once_columns;
  auto sums = adapter_sums_kernel<T, kTerms>;
  auto columns = adapter_columns_kernel<T, C, kHalves>;
  FB_CUDA(ctx, allow(once_sums, ctx->device, sums, SumsLayout::bytes(kMaxRank)));
  FB_CUDA(ctx, allow(once_columns, ctx->device, columns, L::kBytes));
  const int64_t tiles = most_tiles(p.rows, p.batch), items = tiles * ((p.N + kColumns - 1) / kColumns);
  FB_CUDA(ctx, launch(sums, tiles * kCtas, kSumThreads, SumsLayout::bytes(width), s, map_x, map_a, p, work));
  FB_CUDA(ctx, launch(columns, std::min<int64_t>(items, (int64_t)ctx->num_sms * (L::kBytes <= 113 * 1024 && sizeof(C) == 2 ? 2 : 1)), kColThreads, L::kBytes, s, map_t, map_b,
                      p, work));
  return 0;
}

}  // namespace

// Sequences of more than 48 rows in the mean, if adapters lie one behind the other (no tensor map has a step of 0)
size_t adapter_tiles_workspace_bytes(const frisk_b200_adapter_desc& d) {
  if (d.batch < 1 || d.rows <= 48 * (int64_t)d.batch || d.count < 1) return 0;
  if (d.count > 1 && (d.a_step < d.lda || d.b_step < d.ldb)) return 0;
  if (most_tiles(d.rows, d.batch) * ((d.N + kColumns - 1) / kColumns) > INT32_MAX || d.rows * (int64_t)d.rank > INT32_MAX) return 0;
  const int terms = d.dtype_c == FRISK_B200_F32 && d.dtype == FRISK_B200_BF16 ? 3 : 2;
  return up((size_t)d.rows * d.rank * terms * 2) + up((size_t)d.rows * 4) + up((size_t)most_tiles(d.rows, d.batch) * 16) + 256;
}

int launch_adapter_tiles(frisk_b200_ctx* ctx, const frisk_b200_adapter_desc& d, const AdapterParams& p, void* workspace, cudaStream_t s) {
  const bool f32 = d.dtype_c == FRISK_B200_F32, half = d.dtype == FRISK_B200_F16;
  const Work work = work_of(workspace, p.rows, p.R, f32 && !half ? 3 : 2, p.batch);
  if (p.R <= 64) {
    if (half) return f32 ? launch_both<__half, float, 1>(ctx, p, work, s) : launch_both<__half, __half, 1>(ctx, p, work, s);
    return f32 ? launch_both<__nv_bfloat16, float, 1>(ctx, p, work, s) : launch_both<__nv_bfloat16, __nv_bfloat16, 1>(ctx, p, work, s);
  }
  if (half) return f32 ? launch_both<__half, float, 2>(ctx, p, work, s) : launch_both<__half, __half, 2>(ctx, p, work, s);
  return f32 ? launch_both<__nv_bfloat16, float, 2>(ctx, p, work, s) : launch_both<__nv_bfloat16, __nv_bfloat16, 2>(ctx, p, work, s);
}

}  // namespace fb
