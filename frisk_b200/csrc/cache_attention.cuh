// What the kernels of attention over a paged cache share: parameters, how the work is dealt to CTAs, which keys a row sees, how a
// row's results leave.
#pragma once
#include <cfloat>

#include "attention_common.cuh"
#include "cache_common.cuh"
#include "work_split.cuh"

namespace fb {

int cache_validate(const frisk_b200_cache_desc* c);
int cache_pointers(const frisk_b200_cache_desc* c);
cache::Tables cache_tables(const frisk_b200_cache_desc* c);
bool cache_overlaps(const frisk_b200_cache_desc* c, const void* ptr, size_t bytes);
bool tables_overlap(const frisk_b200_cache_desc* c, const void* ptr, size_t bytes);
size_t packed_span(const frisk_b200_packed& x, int64_t rows, int heads, int D, size_t es);

namespace cache {

// An item (the rows of a tile, one key head, all keys) that the CTA of this index began and later ones finished; rows = 0: none.
struct ItemRecord {
  int rows, parts, first_slot;  // its query rows, the CTAs that hold a part, which of the first one's two slots
  int first_row, head, row0;    // the sequence's first packed row, the key head, the first row of the tile
  int pad[2];
};
constexpr size_t kRecordBytes = (kNumSMsDefault * sizeof(ItemRecord) + 255) / 256 * 256;
// a part: O [rows][D], reference maxima [rows], sums [rows]
__host__ __device__ constexpr size_t partial_floats(int rows, int D) { return (size_t)rows * D + 2 * rows; }

struct CacheAttnParams {
  Tables t;
  const void* q;
  void* out;
  int64_t q_row, q_head, out_row, out_head;
  const uint8_t *k_exponent, *v_exponent;
  const void* v_pages;
  const uint8_t* mask;
  int64_t mask_stride;
  int mask_width, group;
  int whole;  // items are not shared: a unit is an item
  float scale_log2;
  ItemRecord* records;
  float* partials;
  unsigned* status;
};

constexpr int kTileKeys = 64;

// log2 of a weight held as a half where the score is the reference, which a score passes by 2^8 at most: halves end just below 2^16 and at
// 2^-25 of nothing is left, so that 2^-32 of the reference is held of every key, however many there are.  (With 2^0 there, 60 thousand keys
// 17 or 18 below a dominant one in the exponent came out doubled or not at all.)
constexpr float kTopHalf = 7.f;
// The same for bf16 weights, and for the row sums and results of 8-bit caches: four million values near the end of the type's range, 2^8
// times weighted, add up to less than 32 bits' end.  (What is lost of values is below 2^-96.)
constexpr float kTopWide = -30.f, kUnitWide = 1.f / (1 << 30);

__device__ __forceinline__ int key_tiles(const Seq& s) { return (s.length + s.count + kTileKeys - 1) / kTileKeys; }
__device__ __forceinline__ int row_tiles(const CacheAttnParams& p, const Seq& s, int tile_rows) {
  return (s.count * p.group + tile_rows - 1) / tile_rows;
}
__device__ __forceinline__ unsigned units_of(const CacheAttnParams& p, const Seq& s, int tile_rows) {
  return (unsigned)p.t.heads * (unsigned)row_tiles(p, s, tile_rows) * (p.whole ? 1u : (unsigned)key_tiles(s));
}

struct PlanShared {
  unsigned warp_sum[16], warp_most[16];
  unsigned first_b, first_off;
};
struct Plan {
  unsigned begin, end;  // this CTA's units
  int b;                // the sequence that holds the first of them
  unsigned off;         // and its index there
};

// A call has fewer than 2^31 units, unless `starts` descends somewhere and sequences share rows: then sums end here, and nothing is done.
constexpr unsigned kTooMany = 0xffffffffu;
__device__ __forceinline__ unsigned add_units(unsigned a, unsigned b) { return a > kTooMany - b ? kTooMany : a + b; }

// The units of all sequences, summed up by the whole CTA; its range of them; the record of the item it shares with the CTAs behind it.
template <int THREADS>
__device__ __forceinline__ Plan make_plan(const CacheAttnParams& p, int tile_rows, PlanShared* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = (p.t.batch + THREADS - 1) / THREADS;
  const int b_lo = min((int)threadIdx.x * chunk, p.t.batch), b_hi = min(b_lo + chunk, p.t.batch);
  unsigned mine = 0, most = 0;  // units; key tiles of the longest sequence
  for (int b = b_lo; b < b_hi; ++b) {
    const Seq s = load_seq(p.t, b, p.status);
    mine = add_units(mine, units_of(p, s, tile_rows));
    if (s.count > 0) most = max(most, (unsigned)key_tiles(s));
  }
  unsigned upto = mine;  // of the warp's threads up to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned other = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto = add_units(upto, other);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 31) {
    sh->warp_sum[warp] = upto;
    sh->warp_most[warp] = most;
  }
  __syncthreads();
  unsigned before = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const unsigned n = sh->warp_sum[w];
    before += w < warp ? n : 0;
    total = add_units(total, n);
    most = max(most, sh->warp_most[w]);
  }
  if (total == kTooMany) {
    atomicCAS(p.status, 0u, ST_CACHE_ROWS);
    total = 0;
  }
  // Little work goes to fewer CTAs: the parts of an item of n key tiles cost as much to join as their tiles take where a CTA has some sqrt(n /
  // 10) tiles.  (One key head, dealt to 148 CTAs and so: 4 rows, 3000 keys 12.4 and 10.8 us, 8000 17.9 and 12.4, 32000 at 8 bits 32.6 and 24.1;
  // 200 rows, 9500 keys at 8 bits 47.9 and 38.5.)
  const unsigned least = p.whole ? 1u : max(1u, (unsigned)sqrtf((float)most * 0.1f));
  const unsigned workers = max(1u, min(gridDim.x, total / least));
  const WorkSplit work{total / workers, total % workers};
  Plan plan;
  plan.begin = min(work.start(blockIdx.x), total);
  plan.end = min(work.start(blockIdx.x + 1), total);
  auto holds = [&](unsigned u) { return before <= u && u - before < mine; };
  if (plan.begin < plan.end) {
    if (holds(plan.begin)) {
      unsigned at = before;
      for (int b = b_lo; b < b_hi; ++b) {
        const unsigned n = units_of(p, load_seq(p.t, b, p.status), tile_rows);
        if (plan.begin - at < n) {
          sh->first_b = (unsigned)b;
          sh->first_off = plan.begin - at;
          break;
        }
        at += n;
      }
    }
    if (!p.whole && holds(plan.end - 1)) {
      unsigned at = before;
      for (int b = b_lo; b < b_hi; ++b) {
        const Seq s = load_seq(p.t, b, p.status);
        const unsigned n = units_of(p, s, tile_rows);
        if (plan.end - 1 - at < n) {
          const unsigned kt = (unsigned)key_tiles(s), item = (plan.end - 1 - at) / kt;
          const unsigned from = at + item * kt, to = from + kt;
          ItemRecord r{};
          if (to > plan.end && from >= plan.begin) {
            const int rt = row_tiles(p, s, tile_rows), h = (int)item / rt;
            r.row0 = ((int)item - h * rt) * tile_rows;
            r.rows = min(tile_rows, s.count * p.group - r.row0);
            r.parts = (int)(work.worker_of(to - 1) - blockIdx.x) + 1;
            r.first_slot = from == plan.begin ? 0 : 1;
            r.first_row = s.first;
            r.head = h;
          }
          p.records[blockIdx.x] = r;
          break;
        }
        at += n;
      }
    }
  } else if (!p.whole && threadIdx.x == 0) {
    p.records[blockIdx.x] = ItemRecord{};
  }
  __syncthreads();
  plan.b = (int)sh->first_b;
  plan.off = sh->first_off;
  return plan;
}

// Walks a CTA's items.
struct Cursor {
  int b, h, rt, tile, kt, n_rt;
  unsigned left;  // units
  bool whole;
  bool first_item;
  Seq seq;
  __device__ __forceinline__ void enter(const CacheAttnParams& p, int tile_rows) {
    seq = load_seq(p.t, b, p.status);
    kt = key_tiles(seq);
    n_rt = row_tiles(p, seq, tile_rows);
  }
  __device__ __forceinline__ Cursor(const CacheAttnParams& p, const Plan& plan, int tile_rows) : left(plan.end - plan.begin), whole(p.whole != 0), first_item(true) {
    if (left == 0) return;
    b = plan.b;
    enter(p, tile_rows);
    const unsigned each = whole ? 1u : (unsigned)kt;
    const int item = (int)(plan.off / each);
    tile = (int)(plan.off - (unsigned)item * each);
    h = item / n_rt;
    rt = item - h * n_rt;
  }
  __device__ __forceinline__ int tiles_here() const { return whole ? kt : (int)min((unsigned)(kt - tile), left); }
  __device__ __forceinline__ void next_item(const CacheAttnParams& p, int tile_rows) {
    left -= whole ? 1u : (unsigned)tiles_here();
    first_item = false;
    tile = 0;
    if (left == 0 || ++rt < n_rt) return;
    rt = 0;
    if (++h < p.t.heads) return;
    h = 0;
    do {
      if (++b >= p.t.batch) {
        left = 0;
        return;
      }
      enter(p, tile_rows);
    } while (n_rt == 0);
  }
};

// whether new token i of the sequence sees key length + ahead
__device__ __forceinline__ bool sees(const CacheAttnParams& p, const Seq& s, int i, int ahead) {
  if (ahead < 0) return true;
  if (ahead >= s.count) return false;
  if (!p.mask) return ahead <= i;
  return ahead < p.mask_width && __ldg(p.mask + (int64_t)(s.first + i) * p.mask_stride + ahead) != 0;
}

// x * f, but that what is infinite or NaN stays so where f has vanished
__device__ __forceinline__ float scaled(float x, float f) { return f == 0.f ? (fabsf(x) <= FLT_MAX ? 0.f : x) : x * f; }

// A result that rounded weights brought beyond the type's range is its largest finite value.  Infinities of 16-bit values stay; 8-bit ones
// have none, but may lie beyond the range themselves.
template <bool BF16, bool E4M3>
__device__ __forceinline__ float in_range(float x) {
  return E4M3 || fabsf(x) <= FLT_MAX ? saturated<BF16>(x) : x;
}

// four results of row r (of the sequence and key head), acc / l; a row that saw nothing is zero
template <bool QBF16, bool E4M3>
__device__ __forceinline__ void store_row4(const CacheAttnParams& p, int first, int h, int r, int c4, float4 acc, float l) {
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  float x[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = in_range<QBF16, E4M3>(x[i]);
  const int i = r / p.group;
  uint16_t* out = static_cast<uint16_t*>(p.out) + (int64_t)(first + i) * p.out_row + (int64_t)(h * p.group + r - i * p.group) * p.out_head;
  *reinterpret_cast<uint2*>(out + c4 * 4) = make_uint2(attn::pack16<QBF16>(x[0], x[1]), attn::pack16<QBF16>(x[2], x[3]));
}

// 32 bytes in one access: a warp whose lanes write rows of their own takes a cycle for every line it touches, however little of it
__device__ __forceinline__ void store32(void* at, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// columns 32 x .. of a row of results, o * inv
template <bool QBF16, bool E4M3>
__device__ __forceinline__ void store_row32(uint16_t* row, int x, const uint32_t (&o)[32], float inv) {
  uint32_t y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float a = in_range<QBF16, E4M3>(__uint_as_float(o[2 * i]) * inv), b = in_range<QBF16, E4M3>(__uint_as_float(o[2 * i + 1]) * inv);
    y[i] = attn::pack16<QBF16>(a, b);
  }
  uint16_t* at = row + x * 32;
  if ((reinterpret_cast<uintptr_t>(at) & 31u) == 0) {
    store32(at, y);
    store32(at + 16, y + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(at + 8 * i) = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
  }
}

// 16 bytes from global to shared memory, and this thread's arrival on `bar` (one of its count) when its copies so far are there
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Where a warp that loads key tiles finds their tokens.  A page holds 16 keys at least, so lane l looks up piece l % 4 of 16 keys;
// the table is read one tile ahead.  What a lane knows becomes an operand of a load by a reduction, whose result the compiler knows
// to be the same for all lanes (a load costs the issuing warp 60 clk so, 110 with a shuffled operand and one lane's branch).
struct PageWalk {
  const int* row;  // of the table
  int keys, head, id;
  __device__ __forceinline__ void look_up(const CacheAttnParams& p, int tile, int lane) {
    const int key = tile * kTileKeys + (lane & 3) * 16;
    id = key < keys ? __ldg(row + (key >> p.t.page_log2)) : 0;
  }
  __device__ __forceinline__ void enter(const CacheAttnParams& p, const int* table_row, int n_keys, int h, int tile, int lane) {
    row = table_row;
    keys = n_keys;
    head = h;
    look_up(p, tile, lane);
  }
  // the token index (page, head, offset) of this lane's piece of the tile
  __device__ __forceinline__ int token(const CacheAttnParams& p, int tile, int lane) const {
    const int key = tile * kTileKeys + (lane & 3) * 16;
    int page = id;
    if (page < 0 || page >= p.t.pages) {  // (page 0 is read in its place)
      atomicCAS(p.status, 0u, ST_CACHE_PAGE);
      page = 0;
    }
    return ((page * p.t.heads + head) << p.t.page_log2) + (key & (p.t.page - 1));
  }
};
// lane `from`'s value (not negative), known to be uniform
__device__ __forceinline__ int uniform_of(int value, int from, int lane) {
  return (int)__reduce_max_sync(0xffffffffu, lane == from ? (unsigned)value : 0u);
}

}  // namespace cache

// tiles of 128 or 256 rows on tcgen05 (cache_attention_tiles.cu); without the join
int launch_cache_attention_tiles(frisk_b200_ctx* ctx, const cache::CacheAttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv,
                                 unsigned grid, bool bf16, bool e4m3, int D, int tile_rows, cudaStream_t s);

}  // namespace fb
