// Pieces shared by the kernels of the paged key/value cache: the packed rows they work on, where a row lies in the pages, and the
// 8-bit form of a row.
//
// A cache is K and V of [pages, heads, page, D]; table[b][i] names the page that holds keys i * page .. of sequence b.  Packed rows
// starts[b] .. starts[b + 1] - 1 belong to sequence b and sit behind lengths[b] keys: row starts[b] + i has position lengths[b] + i.
// These tables live on the device, so they are checked there: what they name outside its range is skipped, and the status word says so.
//
// 8-bit rows: e4m3 codes and one exponent byte e for a token and head, value = code * 2^(e - 127).  The scale is the least power of two
// that brings the row's largest magnitude to 448 or less.  With a power of two the quotient is exact, so a code depends on one
// rounding only and no rounding of a scale; an 8-bit float loses nothing by it, since the scale moves its exponent and not its three
// bits.  e = 255 marks a row that held an infinity or a NaN: it reads back as NaN throughout.
#pragma once
#include "common.cuh"
#include "ptx.cuh"

namespace fb {
namespace cache {

// device status words of the tables (first one wins)
enum : unsigned {
  ST_CACHE_ROWS = 0x301,    // starts not ascending, or beyond the packed rows
  ST_CACHE_LENGTH = 0x302,  // a negative length, or more keys than the table's width holds
  ST_CACHE_PAGE = 0x303,    // a page outside the cache
  ST_CACHE_KV = 0x304,      // (a wait) key tiles
  ST_CACHE_S = 0x305, ST_CACHE_P = 0x306, ST_CACHE_O = 0x307, ST_CACHE_Q = 0x309,
};

struct Tables {
  const int* table;  // [batch][stride]
  const int* starts;
  const int* lengths;
  int64_t stride;
  int batch, width;
  int64_t rows;    // packed rows
  int64_t pages;
  int page, page_log2, heads;
};

struct Seq {
  int first, count, length;  // packed rows, keys before them
  bool ok;
};
__device__ __forceinline__ Seq check_seq(const Tables& t, int lo, int hi, int length, unsigned* status) {
  Seq s;
  s.length = length;
  s.first = lo;
  s.count = hi - lo;
  const bool rows_ok = lo >= 0 && hi >= lo && hi <= t.rows;
  const bool length_ok = length >= 0 && (int64_t)length + s.count <= (int64_t)t.width * t.page;
  s.ok = rows_ok && length_ok;
  if (!s.ok) {
    atomicCAS(status, 0u, rows_ok ? ST_CACHE_LENGTH : ST_CACHE_ROWS);
    s.count = 0;
  }
  return s;
}
__device__ __forceinline__ Seq load_seq(const Tables& t, int b, unsigned* status) {
  return check_seq(t, __ldg(t.starts + b), __ldg(t.starts + b + 1), __ldg(t.lengths + b), status);
}

// 2^(e - 127) of an exponent byte
__device__ __forceinline__ float scale_of(unsigned e) {
  return e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(e ? e << 23 : 0x00400000u);
}

// at most the largest finite fp16 or bf16 value in magnitude; NaN stays
template <bool BF16>
__device__ __forceinline__ float saturated(float x) {
  const float most = BF16 ? __uint_as_float(0x7f7f0000u) : 65504.f;
  return x > most ? most : x < -most ? -most : x;
}

// two e4m3 codes (the low 16 bits) as two halves: exact
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "mov.b32 {lo, hi}, %1;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t}\n"
      : "=r"(h)
      : "r"(codes));
  return h;
}
__device__ __forceinline__ uint32_t e4m3x2_to_half2_hi(uint32_t codes) {
  uint32_t h;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "mov.b32 {lo, hi}, %1;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, hi;\n\t}\n"
      : "=r"(h)
      : "r"(codes));
  return h;
}
__device__ __forceinline__ uint16_t float2_to_e4m3x2(float lo, float hi) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
  return c;
}

}  // namespace cache
}  // namespace fb
