// The kernel of adapters.cu and its launches; each 16-bit type is a source of its own (adapters_rows_f16.cu, adapters_rows_bf16.cu), which are compiled side by side.
#pragma once
#include <algorithm>

#include "adapters.cuh"

namespace fb {
namespace {
using namespace adapter;

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMostGrouped = 8 * kThreads;  // sequences that are brought together
constexpr int kChain = 4;  // blocks of 32 of the inner index that an accumulator takes
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8 elements from `at` on, of which the first `n` are there (others zero)
__device__ __forceinline__ uint4 load8(const uint16_t* at, int n) {
  if (n >= 8) return __ldg(reinterpret_cast<const uint4*>(at));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i >> 1] |= (uint32_t)__ldg(at + i) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The tile of kRows rows that is number `tile`.  Where it is asked for, sequences are brought together by adapter, kThreads of them at a time: the rows of those that share
// one lie behind one another, in the order of the sequences, and the groups in that of their first ones.  (Rows that come together read the adapter once: 99 tokens over
// 21 adapters of rank 64, K 4096, N 7744, 32-bit results 19 us, a tile for each 46.)  Else a sequence has tiles of its own.
struct Rows {
  int count, which;  // rows of the tile (0: there are fewer tiles), their adapter
};
template <int kRows>
__device__ __forceinline__ Rows gather_tile(const AdapterParams& p, int tile, int (&row_of)[kRows]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (!p.grouped) {
    const Tile t = find_tile<kThreads>(p, tile, kRows, false);
    if (tid < kRows) row_of[tid] = t.row + tid;
    __syncthreads();
    return Rows{t.seq < 0 ? 0 : t.rows, t.which};
  }
  __shared__ __align__(16) int keys[kThreads], many[kThreads];
  __shared__ int sums[kWarps], found[3];
  constexpr int kNone = -2;  // a sequence without rows
#pragma unroll 1
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + tid;
    int lo = 0, n = 0, key = kNone;
    if (b < p.batch) {
      lo = p.starts[b];
      key = p.adapters[b];
      const int64_t count = (int64_t)p.starts[b + 1] - lo;
      if (lo < 0 || count < 0 || lo + count > p.rows) atomicCAS(p.status, 0u, cache::ST_CACHE_ROWS);
      else n = (int)count;
      if (n > 0 && key >= p.count) atomicCAS(p.status, 0u, cache::ST_ADAPTER);
      key = n == 0 ? kNone : key < p.count ? max(key, -1) : -1;
    }
    keys[tid] = key;
    many[tid] = n;
    if (tid < 3) found[tid] = 0;
    __syncthreads();
    int before = 0, all = 0;  // rows of this adapter in the sequences before, and in all
    if (key != kNone) {
      const int last = min(kThreads, p.batch - b0);
#pragma unroll 4
      for (int s = 0; s < last; s += 4) {
        const int4 k = *reinterpret_cast<const int4*>(keys + s), m = *reinterpret_cast<const int4*>(many + s);
        const int a = k.x == key ? m.x : 0, b = k.y == key ? m.y : 0, c = k.z == key ? m.z : 0, d = k.w == key ? m.w : 0;
        all += (a + b) + (c + d);
        before += (s < tid ? a : 0) + (s + 1 < tid ? b : 0) + (s + 2 < tid ? c : 0) + (s + 3 < tid ? d : 0);
      }
    }
    const int mine = key != kNone && before == 0 ? (all + kRows - 1) / kRows : 0;  // (tiles of the group, at its first sequence)
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int at = upto - mine, total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) at += sums[i];
      total += sums[i];
    }
    if (tile >= at && tile < at + mine) {
      found[0] = min(kRows, all - (tile - at) * kRows);
      found[1] = key;
      found[2] = (tile - at) * kRows;
    }
    __syncthreads();
    const int rows = found[0], which = found[1], first = found[2];
    if (rows > 0 && key == which) {
      for (int i = max(first, before); i < min(first + rows, before + n); ++i) row_of[i - first] = lo + i - before;
    }
    __syncthreads();
    if (rows > 0) return Rows{rows, which};
    tile -= total;
  }
  return Rows{0, -1};
}

// MW: groups of 16 rows a warp has; MWARPS: warps side by side over rows (the others share the inner index, then the columns)
template <typename T, typename C, int RMAX, int MW, int MWARPS>
struct Plan {
  static constexpr int kRows = 16 * MW * MWARPS, kShare = kWarps / MWARPS;
  static constexpr int kTiles = RMAX / 8, kBlocks = (RMAX + 31) / 32;
  static constexpr int kPitch = RMAX + 8;  // of rows of sums, floats (lanes of a fragment meet no bank twice)
  static constexpr size_t kSumBytes = (size_t)kShare * kRows * kPitch * 4;
  static constexpr size_t kFullBytes = (size_t)kRows * kPitch * 4;
  static constexpr size_t kTermBytes = (size_t)MW * MWARPS * kBlocks * 2 * kTerms * 32 * 16;
  static constexpr size_t kFirstBytes = kSumBytes > kTermBytes ? kSumBytes : kTermBytes;  // (sums are done with where terms begin)
  static constexpr size_t kBytes = kFirstBytes + kFullBytes + kRows * 4;
};

template <typename T, typename C, int RMAX, int MW, int MWARPS, bool WIDE>
__global__ void __launch_bounds__(kThreads) adapter_kernel(const AdapterParams p) {
  using P = Plan<T, C, RMAX, MW, MWARPS>;
  extern __shared__ __align__(16) uint8_t memory[];
  float* sums = reinterpret_cast<float*>(memory);                                   // [share][row][pitch]
  uint4* terms = reinterpret_cast<uint4*>(memory);                                  // later: [16 rows][32 of R][half][term][lane]
  float* full = reinterpret_cast<float*>(memory + P::kFirstBytes);                  // [row][pitch]
  float* row_scale = reinterpret_cast<float*>(memory + P::kFirstBytes + P::kFullBytes);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int C_ = p.cluster, rank = (int)cluster_ctarank(), tile = blockIdx.x / C_;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  __shared__ int row_of[P::kRows];
  const Rows found = gather_tile<P::kRows>(p, tile, row_of);
  if (found.count == 0) return;  // (the whole cluster: there are fewer tiles than clusters)
  const int rows = found.count, which = found.which;
  const C* c = static_cast<const C*>(p.c);
  C* out = static_cast<C*>(p.out);
  const int blocks_n = (p.N + 31) / 32, n0 = (int)((int64_t)blocks_n * rank / C_), n1 = (int)((int64_t)blocks_n * (rank + 1) / C_);
  if (which < 0) {  // no adapter (the whole cluster)
    if (p.out != p.c) {
      const int pieces = (n1 - n0) * 4;
      for (int i = tid; i < rows * pieces; i += kThreads) {
        const int r = i / pieces, col = n0 * 32 + (i - r * pieces) * 8;
        if (col >= p.N) continue;
        Eight<C, WIDE> old;
        old.load(c + row_of[r] * p.ldc + col, p.N - col, p.begins);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = old[j];
        store_eight<C, WIDE>(out + row_of[r] * p.ldo + col, v, p.N - col, p.begins);
      }
    }
    return;
  }
  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  const uint16_t* a = static_cast<const uint16_t*>(p.a) + which * p.a_step;
  const uint16_t* bw = static_cast<const uint16_t*>(p.b) + which * p.b_step;
  const int mw = warp % MWARPS, share = warp / MWARPS;  // the warp's rows; its part of the inner index, then of the columns
  const int my_row = mw * 16 * MW;
  int row[MW][2];  // of this lane, in memory
#pragma unroll
  for (int m = 0; m < MW; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = my_row + 16 * m + 8 * h + g;
      row[m][h] = row_of[min(r, rows - 1)];
    }

  // ---- x A^T over this CTA's part of K, shared by kShare warps in turns of 32
  // (The tensor cores cut what an addition leaves below 24 bits, always towards zero, some 2e-8 of the result each time.  So an accumulator
  // takes kChain blocks, and the parts are summed up rounding to nearest, in shared memory.)
  const int blocks_k = (p.K + 31) / 32, k0 = (int)((int64_t)blocks_k * rank / C_), k1 = (int)((int64_t)blocks_k * (rank + 1) / C_);
  int kb = my_row < rows ? k0 + share : k1;
  bool begun = false;
  do {
    float acc[MW][P::kTiles][4];
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
      for (int t = 0; t < P::kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][t][i] = 0.f;
    const int end = min(k1, kb + kChain * P::kShare);
#pragma unroll 2
    for (; kb < end; kb += P::kShare) {
      const int k = kb * 32 + q * 8, left = p.K - k;
      uint4 xa[MW][2], w[P::kTiles];
#pragma unroll
      for (int m = 0; m < MW; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = my_row + 16 * m + 8 * h + g;
          xa[m][h] = load8(x + row[m][h] * p.ldx + k, r < rows ? left : 0);
        }
#pragma unroll
      for (int t = 0; t < P::kTiles; ++t) w[t] = load8(a + (8 * t + g) * p.lda + k, 8 * t < p.R ? left : 0);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < MW; ++m) {
          const uint32_t fa[4] = {word(xa[m][0], 2 * s), word(xa[m][1], 2 * s), word(xa[m][0], 2 * s + 1), word(xa[m][1], 2 * s + 1)};
#pragma unroll
          for (int t = 0; t < P::kTiles; ++t) mma<T>(acc[m][t], fa, word(w[t], 2 * s), word(w[t], 2 * s + 1));
        }
    }
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
      for (int t = 0; t < P::kTiles; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2* to = reinterpret_cast<float2*>(sums + (share * P::kRows + my_row + 16 * m + 8 * h + g) * P::kPitch + 8 * t + 2 * q);
          const float2 old = begun ? *to : make_float2(0.f, 0.f);
          *to = make_float2(old.x + acc[m][t][2 * h], old.y + acc[m][t][2 * h + 1]);
        }
    begun = true;
  } while (kb < k1);
  __syncthreads();
  // ---- parts added up: the CTA's warps, then the CTAs, each in their order
  const int quads = RMAX / 4, n_quads = rows * quads;
  for (int i = tid; i < n_quads; i += kThreads) {
    float* at = sums + i / quads * P::kPitch + i % quads * 4;
    float4 s = *reinterpret_cast<const float4*>(at);
#pragma unroll
    for (int j = 1; j < P::kShare; ++j) {
      const float4 o = *reinterpret_cast<const float4*>(at + j * P::kRows * P::kPitch);
      s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
    }
    *reinterpret_cast<float4*>(at) = s;
  }
  __syncwarp();
  cluster_sync_all();
  for (int i = rank * kThreads + tid; i < n_quads; i += C_ * kThreads) {
    const int offset = i / quads * P::kPitch + i % quads * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < C_; ++r) {
      const float4 o = ld_cluster_f4(mapa_addr(smem_u32(sums + offset), r));
      s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
    }
    for (int r = 0; r < C_; ++r) st_cluster_f4(mapa_addr(smem_u32(full + offset), r), s);
  }
  __syncwarp();
  cluster_sync_all();  // (from here on no CTA reads or writes another's memory)
  // ---- as terms, in the order in which the second product takes them
  if (std::is_same<T, __half>::value) {
    for (int r = warp; r < rows; r += kWarps) {
      float most = 0.f;
      for (int i = lane; i < RMAX; i += 32) most = fmaxf(most, finite_magnitude(full[r * P::kPitch + i]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (lane == 0) row_scale[r] = row_power(most);
    }
    __syncthreads();
  }
  for (int i = warp; i < MW * MWARPS * P::kBlocks * 2; i += kWarps) {
    const int s = i & 1, kb = (i >> 1) % P::kBlocks, m = (i >> 1) / P::kBlocks;
    if (16 * m >= rows) continue;
    uint32_t f[kTerms][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 16 * m + g + 8 * (j & 1), k = 32 * kb + 8 * q + 4 * s + 2 * (j >> 1);
      float v[2] = {0.f, 0.f};
      if (r < rows && k < p.R) {
        const float2 two = *reinterpret_cast<const float2*>(full + r * P::kPitch + k);
        const float up = std::is_same<T, __half>::value ? row_scale[r] : 1.f;
        v[0] = two.x * up;
        v[1] = two.y * up;
      }
      uint32_t both[kTerms];
      split<T>(v[0], v[1], both);
#pragma unroll
      for (int t = 0; t < kTerms; ++t) f[t][j] = both[t];
    }
#pragma unroll
    for (int t = 0; t < kTerms; ++t) terms[(i * kTerms + t) * 32 + lane] = make_uint4(f[t][0], f[t][1], f[t][2], f[t][3]);
  }
  __syncthreads();
  // ---- times B^T, 32 columns a step
  if (my_row >= rows) return;
  const float alpha = p.scales ? p.scales[which] : 1.f;
  float up[MW][2];
#pragma unroll
  for (int m = 0; m < MW; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = my_row + 16 * m + 8 * h + g;
      up[m][h] = std::is_same<T, __half>::value && r < rows ? 1.f / row_scale[r] : 1.f;  // (of a power of two: exact)
    }
  const int first = 8 * (g >> 1) + (g & 1);  // of the rows of B that this lane's columns of the four tiles are: first + 2 j
  for (int nb = n0 + share; nb < n1; nb += P::kShare) {
    const int col = nb * 32 + 8 * q, left = p.N - col;
    Eight<C, WIDE> old[MW][2];
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = my_row + 16 * m + 8 * h + g;
        old[m][h].load(c + row[m][h] * p.ldc + col, r < rows ? left : 0, p.begins);
      }
    // (the smaller terms apart, so that chains of cut additions are half as long)
    float d[MW][4][4], low[MW][4][4];
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[m][j][i] = low[m][j][i] = 0.f;
        }
#pragma unroll
    for (int kb = 0; kb < P::kBlocks; ++kb) {
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = nb * 32 + first + 2 * j, k = 32 * kb + 8 * q;
        w[j] = load8(bw + (int64_t)n * p.ldb + k, n < p.N ? p.R - k : 0);
      }
#pragma unroll
      for (int m = 0; m < MW; ++m)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int t = 0; t < kTerms; ++t) {
            const uint4 f = terms[((((my_row / 16 + m) * P::kBlocks + kb) * 2 + s) * kTerms + t) * 32 + lane];
            const uint32_t fa[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) mma<T>(t > 0 ? low[m][j] : d[m][j], fa, word(w[j], 2 * s), word(w[j], 2 * s + 1));
          }
    }
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = my_row + 16 * m + 8 * h + g;
        if (r >= rows) continue;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float sum = d[m][j / 2][2 * h + j % 2] + low[m][j / 2][2 * h + j % 2];
          y[j] = fmaf(alpha, sum * up[m][h], old[m][h][j]);
        }
        store_eight<C, WIDE>(out + row[m][h] * p.ldo + col, y, left, p.begins);
      }
  }
}

// at most: of sequences that share an adapter or have none, kThreads sequences at a time
int64_t groups_of(const AdapterParams& p) { return (p.batch + kThreads - 1) / kThreads * ((int64_t)p.count + 1); }

template <typename T, typename C, int RMAX, int MW, int MWARPS, bool WIDE>
struct Launch {
  using P = Plan<T, C, RMAX, MW, MWARPS>;
  static int capacity(int device, int cluster) {
    static ClusterCapacity known;
    return known(device, adapter_kernel<T, C, RMAX, MW, MWARPS, WIDE>, kThreads, (int)P::kBytes, cluster);
  }
  // (at most: every sequence, or group of sequences that share an adapter or have none, may end with a tile that is not full)
  static int64_t tiles(const AdapterParams& p) { return std::min<int64_t>(p.rows, p.rows / P::kRows + (p.grouped ? groups_of(p) : p.batch)); }
  static cudaError_t allow(int device) {
    static PerDeviceOnce once;
    cudaError_t e = cudaSuccess;
    once(device, [&] {
      e = cudaFuncSetAttribute(adapter_kernel<T, C, RMAX, MW, MWARPS, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kBytes);
      return e == cudaSuccess ? 0 : 1;
    });
    return e;
  }
  // whether all tiles run at once in the largest clusters
  static bool fits(int device, const AdapterParams& p) { return allow(device) == cudaSuccess && capacity(device, kMaxCluster) >= tiles(p); }
};

template <typename T, typename C, int RMAX, int MW, int MWARPS, bool WIDE>
cudaError_t launch(frisk_b200_ctx* ctx, AdapterParams p, cudaStream_t s) {
  using L = Launch<T, C, RMAX, MW, MWARPS, WIDE>;
  using P = typename L::P;
  auto kernel = adapter_kernel<T, C, RMAX, MW, MWARPS, WIDE>;
  const cudaError_t e = L::allow(ctx->device);
  if (e != cudaSuccess) return e;
  const int64_t tiles = L::tiles(p);
  // The most CTAs a tile with which all tiles run at once (64 requests of a token, rank 128: clusters of eight 57 us, of four 33).
  p.cluster = kMaxCluster;
  while (p.cluster > 2 && L::capacity(ctx->device, p.cluster) < tiles) p.cluster /= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait) itself
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(tiles * p.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = P::kBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, typename C, int RMAX, bool WIDE>
cudaError_t launch_rows(frisk_b200_ctx* ctx, const AdapterParams& p, cudaStream_t s) {
  // Sequences that share an adapter come together where there are more tiles than run at once in the largest clusters, and fewer if they do (us, 72 tokens over 5 adapters of
  // rank 16 24 -> 13; where they all run the more clusters the better: 37 tokens over 2 adapters 14.5, brought together 17.5, and 5 of 19 rows of one adapter 7.3 and 9.1).
  // Which adapters are named is known on the device only, so the bound on groups goes by all that are there: 256 tokens over 4 adapters of rank 64 are 17 us, of 64 adapters that are
  // there 27, of 256, which leaves each its own tile, 53.
  const int64_t mean = (p.rows + p.batch - 1) / p.batch;  // rows of a sequence
  AdapterParams g = p;
  g.grouped = p.batch <= kMostGrouped && groups_of(p) < p.batch && p.rows < (1 << 23);  // (rows are counted in 32 bits, even if sequences out of range name some again)
  if (g.grouped && !(mean <= 16 ? Launch<T, C, RMAX, 1, 1, WIDE>::fits(ctx->device, p) : Launch<T, C, RMAX, 2, 1, WIDE>::fits(ctx->device, p)))
    return p.rows <= 16 * groups_of(p) ? launch<T, C, RMAX, 1, 1, WIDE>(ctx, g, s) : launch<T, C, RMAX, 2, 1, WIDE>(ctx, g, s);
  if (mean <= 16) return launch<T, C, RMAX, 1, 1, WIDE>(ctx, p, s);
  return launch<T, C, RMAX, 2, 1, WIDE>(ctx, p, s);
}
template <typename T, typename C, bool WIDE>
cudaError_t launch_rank(frisk_b200_ctx* ctx, const AdapterParams& p, cudaStream_t s) {
  if (p.R <= 16) return launch_rows<T, C, 16, WIDE>(ctx, p, s);
  if (p.R <= 32) return launch_rows<T, C, 32, WIDE>(ctx, p, s);
  if (p.R <= 64) return launch_rows<T, C, 64, WIDE>(ctx, p, s);
  return launch_rows<T, C, 128, WIDE>(ctx, p, s);
}
// (Rows that do not begin on 16 bytes have kernels of their own: the check in one took registers, 64 tokens of 40 adapters 12.2 -> 13.5 us; one by one their elements
// took twice the time, 93 sequences of 42 rows, N 2420, 79 us for 38.)
template <typename T, typename C>
cudaError_t launch_types(frisk_b200_ctx* ctx, const AdapterParams& p, cudaStream_t s) {
  return p.begins == 16 ? launch_rank<T, C, true>(ctx, p, s) : launch_rank<T, C, false>(ctx, p, s);
}

}  // namespace
}  // namespace fb
