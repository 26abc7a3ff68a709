// Pieces shared by the kernels of low-rank adapters: parameters, the 16-bit types, eight neighbours of c and the result.
#pragma once
#include <cfloat>
#include <type_traits>

#include "cache_common.cuh"

namespace fb {
namespace adapter {

constexpr int kMaxRank = 128;

struct AdapterParams {
  const void *x, *a, *b, *c;
  void* out;
  const float* scales;
  const int *starts, *adapters;
  int64_t ldx, lda, a_step, ldb, b_step, ldc, ldo, rows;
  int K, N, R, count, batch;
  int cluster;
  int begins;    // bytes that c's and out's rows begin on: 16, 8, 4, or 0 (an element)
  bool grouped;  // sequences are brought together by adapter
  unsigned* status;
};

template <typename T> struct Terms;  // the 16-bit types
template <> struct Terms<__half> {
  static __device__ __forceinline__ float value(uint16_t w) { return __half2float(__ushort_as_half(w)); }
  static __device__ __forceinline__ uint16_t round(float x) { return __half_as_ushort(__float2half_rn(x)); }
};
template <> struct Terms<__nv_bfloat16> {
  static __device__ __forceinline__ float value(uint16_t w) { return __uint_as_float((uint32_t)w << 16); }
  static __device__ __forceinline__ uint16_t round(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
};

// The 16-bit terms that a sum between the products becomes: all of its 24 bits, whatever the result's type.  (Two hold 16 bits of a bf16 sum and 22 of an fp16 one:
// less than the result where columns cancel, or c the product.)
constexpr int kTerms = 3;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= FLT_MAX; }
// fp16: the power of two that brings a row's largest finite sum, most = 1.m * 2^(e - 127), to 2^14.  (Infinities stay; a row of zeros or subnormals
// stands at 2^126.)
__device__ __forceinline__ float finite_magnitude(float x) { return finite(x) ? fabsf(x) : 0.f; }
__device__ __forceinline__ float row_power(float most) {
  const int e = (int)(__float_as_uint(most) >> 23);
  return __uint_as_float((uint32_t)min(254, 268 - max(e, 15)) << 23);
}
// A sum's terms: all of its sign, and none of them 0, so that the three products with an infinite weight add up to the infinity that the formula has.  (Terms rounded to
// nearest may be 0, or of the other sign: NaN.)  With w the weight of the sum's last bit, each of the first two is what fits of the rest below 2 w and w: multiples of w, exact;
// in bf16 the third has 1 to 256 w.  fp16 terms are multiples of 2^-24.  Of fp16 sums below 3 2^-24 (their row's largest is 2^14), and bf16 ones
// below 2^-100, the terms are rounded to nearest.
template <typename T>
__device__ __forceinline__ void terms_of(float v, uint16_t (&terms)[kTerms]) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  const float a = fabsf(v);
  const uint32_t last = (__float_as_uint(a) >> 23) << 23;  // 2^23 w
  const float w = kHalf ? fmaxf(__uint_as_float(last) * 0x1p-23f, 0x1p-24f) : __uint_as_float(last) * 0x1p-23f;
  const uint16_t sign = (uint16_t)(__float_as_uint(v) >> 16 & 0x8000u);
  auto below = [](float x) -> uint16_t {
    if (kHalf) return __half_as_ushort(__float2half_rz(x));
    return (uint16_t)(__float_as_uint(x) >> 16);
  };
  // (by selection: with a branch for each, one after the other, a token took 7.9 us for 7.5)
  const bool usual = finite(v) && a >= (kHalf ? 3 * 0x1p-24f : 0x1p-100f);
  const uint16_t first = usual ? below(a - 2.f * w) : Terms<T>::round(a);
  const float rest = a - Terms<T>::value(first);
  const uint16_t second = usual ? below(rest - w) : Terms<T>::round(rest), third = Terms<T>::round(rest - Terms<T>::value(second));
  terms[0] = first ^ sign;
  terms[1] = (finite(v) ? second : first) ^ sign;
  terms[2] = (finite(v) ? third : first) ^ sign;
}
// two neighbours as words of terms
template <typename T>
__device__ __forceinline__ void split(float a, float b, uint32_t (&words)[kTerms]) {
  uint16_t lo[kTerms], hi[kTerms];
  terms_of<T>(a, lo);
  terms_of<T>(b, hi);
#pragma unroll
  for (int t = 0; t < kTerms; ++t) words[t] = lo[t] | (uint32_t)hi[t] << 16;
}

__device__ __forceinline__ uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// Eight neighbours of c, as they are in memory, of which the first n are there
// WIDE: rows begin on 16 bytes; else on `begins`: 8, 4, or 0 (an element)
template <typename C, bool WIDE>
struct Eight {
  uint4 w[sizeof(C) / 2];
  __device__ __forceinline__ void load(const C* at, int n, int begins) {
    if (WIDE && n >= 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(C) / 2; ++i) w[i] = *(reinterpret_cast<const uint4*>(at) + i);
    } else if (!WIDE && begins == 8 && n >= 8) {
      uint2 v[sizeof(C)];
#pragma unroll
      for (int i = 0; i < (int)sizeof(C); ++i) v[i] = *(reinterpret_cast<const uint2*>(at) + i);
#pragma unroll
      for (int i = 0; i < (int)sizeof(C) / 2; ++i) w[i] = make_uint4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
    } else if (!WIDE && sizeof(C) == 2 && begins == 4 && n >= 8) {
      const uint32_t* v = reinterpret_cast<const uint32_t*>(at);
      w[0] = make_uint4(v[0], v[1], v[2], v[3]);
    } else {
      alignas(16) C v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? at[i] : C(0.f);
#pragma unroll
      for (int i = 0; i < (int)sizeof(C) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(v)[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if (sizeof(C) == 4) return __uint_as_float(word(w[i / 4 % (sizeof(C) / 2)], i % 4));
    using T = typename std::conditional<sizeof(C) == 2, C, __half>::type;
    return Terms<T>::value((uint16_t)(word(w[0], i / 2) >> (16 * (i & 1))));
  }
};
template <typename C, bool WIDE>
__device__ __forceinline__ void store_eight(C* at, const float (&v)[8], int n, int begins) {
  constexpr int kWords = 2 * (int)sizeof(C);
  uint32_t w[kWords];
  if (sizeof(C) == 4) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __float_as_uint(v[i % 8]);
  } else {
    using T = typename std::conditional<sizeof(C) == 2, C, __half>::type;
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = Terms<T>::round(v[2 * i % 8]) | (uint32_t)Terms<T>::round(v[(2 * i + 1) % 8]) << 16;
  }
  if (WIDE && n >= 8) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  } else if (!WIDE && begins == 8 && n >= 8) {
#pragma unroll
    for (int i = 0; i < kWords / 2; ++i) reinterpret_cast<uint2*>(at)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
  } else if (!WIDE && sizeof(C) == 2 && begins == 4 && n >= 8) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint32_t*>(at)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) at[i] = (C)v[i];
  }
}

// The tile of `tile_rows` packed rows that is number `tile` over all sequences.  Counted by a block of kThreads threads, a sequence each; the answer
// is the same in all of them.  `everything`: all tiles are counted.
struct Tile {
  int seq, row, rows;  // seq < 0: there are fewer
  int which;           // the sequence's adapter; -1: none
  int counted;         // tiles up to here; all, where `everything` is asked for
};
template <int kThreads>
__device__ __forceinline__ Tile find_tile(const AdapterParams& p, int tile, int tile_rows, bool everything) {
  __shared__ int sums[kThreads / 32], found[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) found[0] = -1;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + tid;
    int lo = 0, n = 0, which = -1;
    if (b < p.batch) {
      lo = p.starts[b];
      which = p.adapters[b];  // (on its way at the same time)
      const int64_t many = (int64_t)p.starts[b + 1] - lo;
      if (lo < 0 || many < 0 || lo + many > p.rows) atomicCAS(p.status, 0u, cache::ST_CACHE_ROWS);
      else n = (int)many;
    }
    const int mine = (n + tile_rows - 1) / tile_rows;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int at = before + upto - mine;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) at += sums[i];
      before += sums[i];
    }
    before = min(before, 1 << 30);  // (2^26 rows are at most 2^30 tiles of 16 for 256 sequences, and less than 2^28 of 128 for 320)
    if (tile >= at && tile < at + mine) {
      found[0] = b;
      found[1] = lo + (tile - at) * tile_rows;
      found[2] = min(tile_rows, n - (tile - at) * tile_rows);
      found[3] = which < p.count ? max(which, -1) : -1;
      if (which >= p.count) atomicCAS(p.status, 0u, cache::ST_ADAPTER);
    }
    if (before > tile && !everything) break;  // (the same in all threads)
  }
  __syncthreads();
  return Tile{found[0], found[1], found[2], found[3], before};
}

}  // namespace adapter

// few rows a sequence (adapters_rows.cuh), and whether c has 32 bits
cudaError_t launch_adapter_rows_f16(frisk_b200_ctx* ctx, const adapter::AdapterParams& p, bool f32, cudaStream_t s);
cudaError_t launch_adapter_rows_bf16(frisk_b200_ctx* ctx, const adapter::AdapterParams& p, bool f32, cudaStream_t s);
// long sequences (adapters_tiles.cu)
size_t adapter_tiles_workspace_bytes(const frisk_b200_adapter_desc& d);  // 0: adapters.cu takes it
int launch_adapter_tiles(frisk_b200_ctx* ctx, const frisk_b200_adapter_desc& d, const adapter::AdapterParams& p, void* workspace, cudaStream_t s);

}  // namespace fb
