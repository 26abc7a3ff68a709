// Writing new rows into the paged cache, quantised on the way where it holds 8-bit floats, and reading rows back.
//
// A head's row is D elements: 16 of them a lane, D / 16 neighbouring lanes a row, so the largest magnitude of a row takes two or three
// shuffles and nothing passes through shared memory.  Bound by HBM: each side is read or written once.  A block takes
// up to 16 packed rows: a thread finds the place of each (its sequence by bisection of `starts`, then the page; a chain of dependent
// loads), then all threads move the pieces of all of them, two at a time.  (One row at a time, 52 thousand rows of 4 heads of 64 took
// 102 us.)  Fewer rows a block where that leaves SMs idle: a few rows cost the chain starts -> lengths -> table and little else.
#include <algorithm>

#include "cache_common.cuh"

namespace fb {
namespace {
using namespace cache;

constexpr int kThreads = 256;
constexpr int kMaxRows = 16;  // packed rows a block
constexpr int kCopied = 512;  // sequences whose tables fit into shared memory
constexpr int kAhead = 2;     // pieces a thread has in flight

struct Side {  // packed rows outside the cache, 16-bit
  void* ptr;
  int64_t row, head;
};
struct RowsParams {
  Tables t;
  Side k, v;
  void *ck, *cv;           // pages
  uint8_t *ek, *ev;        // exponents
  int64_t rows;
  int rows_block;
  unsigned* status;
};

// The index of packed row r among the cache's token slots of head 0, (page * heads) * P + offset; -1: it has none.
// `starts`, `lengths`: the tables, or copies of them in shared memory.
__device__ __forceinline__ int64_t locate(const Tables& t, const int* starts, const int* lengths, int64_t r, unsigned* status) {
  // the last b with starts[b] <= r; where starts does not ascend, some b that does not hold r
  int lo = 0, hi = t.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= r) lo = mid; else hi = mid;
  }
  const Seq s = check_seq(t, starts[lo], starts[lo + 1], lengths[lo], status);
  const int64_t i = r - s.first;
  if (!s.ok || i < 0 || i >= s.count) return -1;  // (rows before the first sequence and behind the last belong to none)
  const int64_t pos = s.length + i;
  const int page = __ldg(t.table + lo * t.stride + (pos >> t.page_log2));
  if (page < 0 || page >= t.pages) {
    atomicCAS(status, 0u, ST_CACHE_PAGE);
    return -1;
  }
  return ((int64_t)page * t.heads << t.page_log2) + (pos & (t.page - 1));
}

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool BF16, int D, bool E4M3, bool WRITE>
__global__ void __launch_bounds__(kThreads) cache_rows_kernel(const RowsParams p) {
  constexpr int kLanes = D / 16;  // of a row
  __shared__ int64_t bases[kMaxRows];
  __shared__ int starts[kCopied + 1], lengths[kCopied];
  const int64_t row0 = (int64_t)blockIdx.x * p.rows_block;
  const int here = (int)min((int64_t)p.rows_block, p.rows - row0);
  const int per_row = 2 * p.t.heads * kLanes;  // pieces of a token: keys, then values
  const int total = here * per_row;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.t.batch <= kCopied) {  // (one latency for the tables instead of one a step of the bisection)
    for (int b = threadIdx.x; b <= p.t.batch; b += kThreads) {
      starts[b] = __ldg(p.t.starts + b);
      if (b < p.t.batch) lengths[b] = __ldg(p.t.lengths + b);
    }
    __syncthreads();
    if ((int)threadIdx.x < here) bases[threadIdx.x] = locate(p.t, starts, lengths, row0 + threadIdx.x, p.status);
  } else if ((int)threadIdx.x < here) {
    bases[threadIdx.x] = locate(p.t, p.t.starts, p.t.lengths, row0 + threadIdx.x, p.status);
  }
  __syncthreads();
  // (whole groups of kLanes threads have the same head's row, and whole warps the same number of rounds: the shuffles below need them)
  const int sub = threadIdx.x % kLanes;
  int r_next = threadIdx.x / per_row, piece = threadIdx.x - r_next * per_row;  // of the next piece: its row, its place there
  const int r_step = kThreads / per_row, piece_step = kThreads - r_step * per_row;
  for (int e0 = 0; e0 < total; e0 += kThreads * kAhead) {
    uint4 x[kAhead][2];    // the 16-bit side, or the cache's piece
    uint32_t e_byte[kAhead];
    int64_t token[kAhead];  // -1: nothing to do
    uint4* packed[kAhead];
    bool values[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      if (e0 + n * kThreads >= total) break;
      const int e = e0 + n * kThreads + threadIdx.x;
      const bool mine = e < total;
      const int r = mine ? r_next : 0, unit = piece / kLanes;
      r_next += r_step;
      piece += piece_step;
      if (piece >= per_row) {
        piece -= per_row;
        ++r_next;
      }
      values[n] = unit >= p.t.heads;
      const int h = values[n] ? unit - p.t.heads : unit;
      const Side& side = values[n] ? p.v : p.k;
      packed[n] = reinterpret_cast<uint4*>(static_cast<uint16_t*>(side.ptr) + (row0 + r) * side.row + h * side.head) + 2 * sub;
      const int64_t base = bases[r];
      token[n] = mine && base >= 0 ? base + ((int64_t)h << p.t.page_log2) : -1;
      x[n][0] = x[n][1] = make_uint4(0, 0, 0, 0);
      e_byte[n] = 0;
      if (token[n] < 0) continue;
      const void* pages = values[n] ? p.cv : p.ck;
      if (WRITE) {
        x[n][0] = __ldcs(packed[n]);
        x[n][1] = __ldcs(packed[n] + 1);
      } else if (!E4M3) {
        const uint4* held = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(pages) + token[n] * D) + 2 * sub;
        x[n][0] = __ldcs(held);
        x[n][1] = __ldcs(held + 1);
      } else {
        x[n][0] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(pages) + token[n] * D) + sub);
        e_byte[n] = __ldg((values[n] ? p.ev : p.ek) + token[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      if (e0 + n * kThreads >= total) break;
      void* pages = values[n] ? p.cv : p.ck;
      if (!E4M3) {
        if (token[n] < 0) continue;
        if (WRITE) {
          uint4* held = reinterpret_cast<uint4*>(static_cast<uint16_t*>(pages) + token[n] * D) + 2 * sub;
          held[0] = x[n][0];
          held[1] = x[n][1];
        } else {
          __stcs(packed[n], x[n][0]);
          __stcs(packed[n] + 1, x[n][1]);
        }
      } else if (WRITE) {
        const uint32_t w[8] = {x[n][0].x, x[n][0].y, x[n][0].z, x[n][0].w, x[n][1].x, x[n][1].y, x[n][1].z, x[n][1].w};
        uint32_t most = 0;  // magnitudes of 16-bit floats compare as integers; infinities and NaN are the largest
#pragma unroll
        for (int i = 0; i < 8; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
        most = max(most & 0xffffu, most >> 16);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        most = __float_as_uint(unpack16<BF16>(most).x);
        // most = 1.m * 2^(E - 127) and 448 = 1.75 * 2^8: the least e with most <= 448 * 2^(e - 127)
        int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0);
        e = most >= 0x7f800000u ? 255 : max(e, 1);
        if (token[n] < 0) continue;
        uint32_t code[4] = {0, 0, 0, 0};
        if (e != 255) {
          const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 two = unpack16<BF16>(w[i]);
            code[i >> 1] |= (uint32_t)float2_to_e4m3x2(two.x * inv, two.y * inv) << (16 * (i & 1));
          }
        }
        reinterpret_cast<uint4*>(static_cast<uint8_t*>(pages) + token[n] * D)[sub] = make_uint4(code[0], code[1], code[2], code[3]);
        if (sub == 0) (values[n] ? p.ev : p.ek)[token[n]] = (uint8_t)e;
      } else {
        if (token[n] < 0) continue;
        const float scale = scale_of(e_byte[n]);
        const uint32_t c[4] = {x[n][0].x, x[n][0].y, x[n][0].z, x[n][0].w};
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t h2 = i & 1 ? e4m3x2_to_half2_hi(c[i >> 1]) : e4m3x2_to_half2(c[i >> 1]);
          const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&h2));
          // a row near the end of the type's range may have been rounded beyond it
          o[i] = pack16<BF16>(saturated<BF16>(two.x * scale), saturated<BF16>(two.y * scale));
        }
        __stcs(packed[n], make_uint4(o[0], o[1], o[2], o[3]));
        __stcs(packed[n] + 1, make_uint4(o[4], o[5], o[6], o[7]));
      }
    }
  }
}

template <bool BF16, int D, bool E4M3, bool WRITE>
cudaError_t launch(const RowsParams& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait) itself
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((p.rows + p.rows_block - 1) / p.rows_block));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, cache_rows_kernel<BF16, D, E4M3, WRITE>, p);
}
template <bool WRITE>
cudaError_t launch_any(const RowsParams& p, bool bf16, int D, bool e4m3, cudaStream_t s) {
  if (D == 64)
    return bf16 ? (e4m3 ? launch<true, 64, true, WRITE>(p, s) : launch<true, 64, false, WRITE>(p, s))
                : (e4m3 ? launch<false, 64, true, WRITE>(p, s) : launch<false, 64, false, WRITE>(p, s));
  return bf16 ? (e4m3 ? launch<true, 128, true, WRITE>(p, s) : launch<true, 128, false, WRITE>(p, s))
              : (e4m3 ? launch<false, 128, true, WRITE>(p, s) : launch<false, 128, false, WRITE>(p, s));
}

}  // namespace
}  // namespace fb

using namespace fb;

namespace fb {

int cache_validate(const frisk_b200_cache_desc* c) {
  if (!c) return FRISK_B200_E_ARG;
  if (c->dtype != FRISK_B200_F16 && c->dtype != FRISK_B200_BF16 && c->dtype != FRISK_B200_E4M3) return FRISK_B200_E_CACHE_TYPE;
  if (c->pages < 1 || c->page < 16 || c->page > 1024 || (c->page & (c->page - 1)) || c->heads < 1 || c->heads > 4096 ||
      (c->D != 64 && c->D != 128) || c->batch < 0 || c->table_width < 0 || c->rows < 0 || c->rows > INT32_MAX ||
      (c->batch > 1 && c->table_stride < c->table_width) || c->pages > INT32_MAX || c->pages * c->heads > (INT32_MAX / c->page))
    return FRISK_B200_E_CACHE_SHAPE;
  return 0;
}

// pointers of a cache that a call is going to use
int cache_pointers(const frisk_b200_cache_desc* c) {
  if (!c->k || !c->v || !c->starts || !c->lengths || (!c->table && c->table_width > 0)) return FRISK_B200_E_ARG;
  if (c->dtype == FRISK_B200_E4M3 && (!c->k_exponent || !c->v_exponent)) return FRISK_B200_E_ARG;
  const uintptr_t all = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) |
                        (c->dtype == FRISK_B200_E4M3 ? reinterpret_cast<uintptr_t>(c->k_exponent) | reinterpret_cast<uintptr_t>(c->v_exponent) : 0);
  if (all & 15u) return FRISK_B200_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(c->starts) | reinterpret_cast<uintptr_t>(c->lengths) | reinterpret_cast<uintptr_t>(c->table)) & 3u)
    return FRISK_B200_E_ALIGN;
  return 0;
}

cache::Tables cache_tables(const frisk_b200_cache_desc* c) {
  cache::Tables t{};
  t.table = c->table;
  t.starts = c->starts;
  t.lengths = c->lengths;
  t.stride = c->table_stride;
  t.batch = c->batch;
  t.width = c->table_width;
  t.rows = c->rows;
  t.pages = c->pages;
  t.page = c->page;
  t.heads = c->heads;
  while ((1 << t.page_log2) < c->page) ++t.page_log2;
  return t;
}

// bytes of the cache's tensors, which outputs must not overlap
bool cache_overlaps(const frisk_b200_cache_desc* c, const void* ptr, size_t bytes) {
  const size_t tokens = (size_t)c->pages * c->heads * c->page, held = tokens * c->D * (c->dtype == FRISK_B200_E4M3 ? 1 : 2);
  return ranges_overlap(ptr, bytes, c->k, held) || ranges_overlap(ptr, bytes, c->v, held) ||
         (c->dtype == FRISK_B200_E4M3 &&
          (ranges_overlap(ptr, bytes, c->k_exponent, tokens) || ranges_overlap(ptr, bytes, c->v_exponent, tokens)));
}
bool tables_overlap(const frisk_b200_cache_desc* c, const void* ptr, size_t bytes) {
  return ranges_overlap(ptr, bytes, c->starts, ((size_t)c->batch + 1) * 4) || ranges_overlap(ptr, bytes, c->lengths, (size_t)c->batch * 4) ||
         (c->batch > 0 && c->table_width > 0 && ranges_overlap(ptr, bytes, c->table, (size_t)((c->batch - 1) * c->table_stride + c->table_width) * 4));
}
size_t packed_span(const frisk_b200_packed& x, int64_t rows, int heads, int D, size_t es) {
  return (size_t)((rows - 1) * x.row_stride + (heads - 1) * x.head_stride + D) * es;
}

}  // namespace fb

static int check_side(const frisk_b200_packed* x, int heads, int D, int64_t rows, bool written) {
  if (!x || !x->ptr) return FRISK_B200_E_ARG;
  if (x->row_stride < 0 || x->head_stride < 0) return FRISK_B200_E_CACHE_SHAPE;
  if (written && !packed_distinct(*x, rows, heads, D)) return FRISK_B200_E_CACHE_SHAPE;
  if ((reinterpret_cast<uintptr_t>(x->ptr) & 15u) || (rows > 1 && x->row_stride % 8) || (heads > 1 && x->head_stride % 8)) return FRISK_B200_E_ALIGN;
  return 0;
}

static int cache_rows(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, int32_t dtype, const frisk_b200_packed* k,
                      const frisk_b200_packed* v, bool write, void* stream) {
  if (!ctx) return FRISK_B200_E_ARG;
  int rc = cache_validate(c);
  if (rc) return rc;
  if (dtype != FRISK_B200_F16 && dtype != FRISK_B200_BF16) return FRISK_B200_E_CACHE_TYPE;
  if (c->dtype != FRISK_B200_E4M3 && c->dtype != dtype) return FRISK_B200_E_CACHE_TYPE;
  if (c->rows == 0 || c->batch == 0) return 0;
  if ((rc = cache_pointers(c))) return rc;
  if ((rc = check_side(k, c->heads, c->D, c->rows, !write)) || (rc = check_side(v, c->heads, c->D, c->rows, !write))) return rc;
  const size_t kb = packed_span(*k, c->rows, c->heads, c->D, 2), vb = packed_span(*v, c->rows, c->heads, c->D, 2);
  if (cache_overlaps(c, k->ptr, kb) || cache_overlaps(c, v->ptr, vb)) return FRISK_B200_E_OVERLAP;
  if (!write && (!packed_apart(*k, c->heads, *v, c->heads, c->rows, c->D, 2) || tables_overlap(c, k->ptr, kb) || tables_overlap(c, v->ptr, vb)))
    return FRISK_B200_E_OVERLAP;
  if (write) {  // the cache's tensors apart from one another and from the tables
    const size_t tokens = (size_t)c->pages * c->heads * c->page, held = tokens * c->D * (c->dtype == FRISK_B200_E4M3 ? 1 : 2);
    struct { const void* p; size_t n; } part[4] = {{c->k, held}, {c->v, held}, {c->k_exponent, tokens}, {c->v_exponent, tokens}};
    const int n = c->dtype == FRISK_B200_E4M3 ? 4 : 2;
    for (int i = 0; i < n; ++i) {
      if (tables_overlap(c, part[i].p, part[i].n)) return FRISK_B200_E_OVERLAP;
      for (int j = i + 1; j < n; ++j)
        if (ranges_overlap(part[i].p, part[i].n, part[j].p, part[j].n)) return FRISK_B200_E_OVERLAP;
    }
  }
  RowsParams p{};
  p.t = cache_tables(c);
  p.k = Side{k->ptr, k->row_stride, k->head_stride};
  p.v = Side{v->ptr, v->row_stride, v->head_stride};
  p.ck = c->k;
  p.cv = c->v;
  p.ek = c->k_exponent;
  p.ev = c->v_exponent;
  p.rows = c->rows;
  p.status = ctx->d_status;
  p.rows_block = 1;
  // up to 1024 pieces a block, four a thread (13 thousand rows of 8 heads of 128, 8 rows a block: write and read 41 us, with 16 rows 48; 52
  // thousand of 4 heads of 64: 16 rows 21.6, with 8 23.1), and at least four blocks a SM
  const int pieces = 2 * c->heads * c->D / 16;
  while (p.rows_block < kMaxRows && 2 * p.rows_block * pieces <= 4 * kThreads && c->rows / (2 * p.rows_block) >= 4 * ctx->num_sms)
    p.rows_block *= 2;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == FRISK_B200_BF16, e4m3 = c->dtype == FRISK_B200_E4M3;
  FB_CUDA(ctx, write ? launch_any<true>(p, bf16, c->D, e4m3, s) : launch_any<false>(p, bf16, c->D, e4m3, s));
  return 0;
}

extern "C" {
int frisk_b200_cache_write(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, int32_t dtype, const frisk_b200_packed* k,
                           const frisk_b200_packed* v, void* stream) {
  return cache_rows(ctx, c, dtype, k, v, true, stream);
}
int frisk_b200_cache_read(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, int32_t dtype, const frisk_b200_packed* k,
                          const frisk_b200_packed* v, void* stream) {
  return cache_rows(ctx, c, dtype, k, v, false, stream);
}
}
