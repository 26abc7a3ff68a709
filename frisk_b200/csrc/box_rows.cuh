// Boxes of 32 rows x 128 bytes of a matrix that the TMA unit cannot address, on their way to and from shared memory.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace fb {

// A 32-row box (128 bytes a row, a 32-bit word a lane) of a C that the TMA unit cannot address: its rows begin on a multiple
// of the element's size and no more.  16-bit elements go in pairs wherever they lie on 4 bytes: of a row that begins
// there lane l has elements 2l and 2l + 1, of an odd row 2l + 1 and 2l + 2, and its first and last element go by themselves.
// Which rows are odd is one of four patterns, the same for the whole box: an epilogue warp has its scheduler to itself, so its
// time is the number of instructions, and rows that decide for themselves took 1200 of them a box (1.9 us).  With 2-byte accesses
// 4000 x 4092 x 512 took 51.7 us, 33.3 so, 22.9 with 4096 columns by TMA; 4095 columns 51.7 and 39.8.  The old values used to be
// loaded one after the other, each behind the shared-memory store of the one before: two panels of 6543 x 4546 x 2296
// 872 us, 359 so; fp32 3000 x 2055 x 1032 186 and 73.
struct BoxRows {
  bool first_odd, second_odd;
  template <typename TO>
  __device__ __forceinline__ BoxRows(const TO* row, int64_t pitch)
      : first_odd(sizeof(TO) == 2 && (reinterpret_cast<uintptr_t>(row) & 2u)),
        second_odd(sizeof(TO) == 2 && (reinterpret_cast<uintptr_t>(row + pitch) & 2u)) {}
  // f(first row odd, second row odd), the answers as types
  template <typename F>
  __device__ __forceinline__ void pattern(F&& f) const {
    if (first_odd) {
      if (second_odd) f(std::true_type(), std::true_type()); else f(std::true_type(), std::false_type());
    } else {
      if (second_odd) f(std::false_type(), std::true_type()); else f(std::false_type(), std::false_type());
    }
  }
};
// the old values of a box, cols x rows of which lie in C (all loads on their way before the first is used), into its image:
// put(r, word of row r)
template <typename TO, typename Put>
__device__ __forceinline__ void load_box_rows(const TO* row, int64_t pitch, int rows, int cols, int lane, Put&& put) {
  uint32_t w[32];
  if (sizeof(TO) == 4) {
#pragma unroll
    for (int r = 0; r < 32; ++r) w[r] = r < rows && lane < cols ? *reinterpret_cast<const uint32_t*>(row + r * pitch + lane) : 0u;
#pragma unroll
    for (int r = 0; r < 32; ++r) put(r, w[r]);
    return;
  }
  const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
  // lane r: the first element of row r
  const uint32_t firsts = lane < rows ? p[lane * pitch] : 0u;
  BoxRows(row, pitch).pattern([&](auto odd0, auto odd1) {
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const bool odd = r % 2 ? decltype(odd1)::value : decltype(odd0)::value;
      const int j = 2 * lane + (odd ? 1 : 0);
      w[r] = 0u;
      if (r < rows && j + 1 < cols) w[r] = *reinterpret_cast<const uint32_t*>(p + r * pitch + j);
      if (r < rows && j + 1 == cols) w[r] = p[r * pitch + j];
    }
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const bool odd = r % 2 ? decltype(odd1)::value : decltype(odd0)::value;
      if (odd) {
        const uint32_t before = __shfl_up_sync(0xffffffffu, w[r], 1), first = __shfl_sync(0xffffffffu, firsts, r);
        w[r] = (lane == 0 ? first : before >> 16) | (w[r] << 16);
      }
      put(r, w[r]);
    }
  });
}
// a box back to C: get(r) gives this lane's word of row r
template <typename TO, typename Get>
__device__ __forceinline__ void store_box_rows(TO* row, int64_t pitch, int rows, int cols, int lane, Get&& get) {
  constexpr int kStep = 8;
  if (sizeof(TO) == 4) {
#pragma unroll 1
    for (int r = 0; r < rows; r += kStep, row += kStep * pitch) {
      uint32_t w[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) w[i] = get(r + i);
#pragma unroll
      for (int i = 0; i < kStep; ++i)
        if (r + i < rows && lane < cols) *reinterpret_cast<uint32_t*>(row + i * pitch + lane) = w[i];
    }
    return;
  }
  unsigned short* p = reinterpret_cast<unsigned short*>(row);
  // an odd row's pairs, and what is left over: lane 0 has the first element, the lane of the last column the last where cols is even
  const bool pair_even = 2 * lane + 1 < cols, pair_odd = 2 * lane + 2 < cols, one_even = 2 * lane + 1 == cols;
  const bool one_odd = lane == 0 || 2 * lane + 2 == cols;
  const int one_at = lane == 0 ? 0 : 2 * lane + 1;
  BoxRows(row, pitch).pattern([&](auto odd0, auto odd1) {
#pragma unroll 1
    for (int r = 0; r < rows; r += kStep, p += kStep * pitch) {
      uint32_t w[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) w[i] = get(r + i);
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const bool odd = i % 2 ? decltype(odd1)::value : decltype(odd0)::value;
        unsigned short* q = p + i * pitch;
        const bool in = r + i < rows;
        if (odd) {
          const uint32_t after = __shfl_down_sync(0xffffffffu, w[i], 1);
          if (in && pair_odd) *reinterpret_cast<uint32_t*>(q + 2 * lane + 1) = __funnelshift_r(w[i], after, 16);
          if (in && one_odd) q[one_at] = (unsigned short)(lane == 0 ? w[i] : w[i] >> 16);
        } else {
          if (in && pair_even) *reinterpret_cast<uint32_t*>(q + 2 * lane) = w[i];
          if (in && one_even) q[2 * lane] = (unsigned short)w[i];
        }
      }
    }
    // (cols = 2: lane 0 has both ends of an odd row)
    if (cols == 2 && (decltype(odd0)::value || decltype(odd1)::value)) {
      unsigned short* q = reinterpret_cast<unsigned short*>(row);
      for (int r = 0; r < rows; ++r) {
        const uint32_t w = get(r);
        if (lane == 0 && (r % 2 ? decltype(odd1)::value : decltype(odd0)::value)) q[r * pitch + 1] = (unsigned short)(w >> 16);
      }
    }
  });
}

}  // namespace fb
