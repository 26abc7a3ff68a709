// Low-rank adapters of many requests, added to a shared projection:
//
//   out[r] = c[r] + scale[w] * (x[r] A_w^T) B_w^T,   w: the adapter of row r's sequence, A_w [R, K], B_w [N, R]
//
// One launch.  A cluster has up to kRows rows of one sequence, or of sequences that share an adapter.  Its CTAs share K: each makes the products of its part of x and A, and the
// parts are added up through distributed shared memory, in order, into all of the cluster's CTAs.  Then they share N: each multiplies the R sums of a row by its
// part of B and adds c.  So nothing between the two products leaves the SMs, and no order of threads changes a result.
//
// Bound by memory for the ranks of adapters: an element of x, c or out takes R multiplications (R = 64 at 6.5 TB/s: 0.2 PFLOP/s).  So the products
// are mma.sync's, operands go from memory to registers without a stop, and no tensor memory is set up.  For a few rows the adapters
// themselves are what is read, each by a cluster of its own; then the time is a chain: tables, x and A, two meetings of the cluster, B and c (one token, rank 16,
// K = N = 4096: 7.5 us with the launch; 64 tokens over 40 adapters of rank 32, N 5120: 12.9, 25 MB).  Long sequences have kernels of their own (adapters_tiles.cu).
//
// Order of a product's inner index is free if both sides have the same, so a lane takes 16 bytes of it at once: of 32 neighbouring elements lane q of
// four has 8 q .. 8 q + 7, which serve two steps of 16.  Columns of a result are permuted the same way: a lane ends up with 8 neighbours.
//
// Sums are 32-bit.  Before the second product they become sums of three 16-bit terms, which hold all 24 bits (fp16 terms stand at a power of two that brings a row's
// largest to 2^14, so that sums beyond fp16's range keep their value, and go down to 2^-38 of it).  The terms have the sum's sign, so that an infinite weight makes
// the infinity that the formula has.  With two terms, 16 bits in bf16 and 22 in fp16, times are 2 to 5 % less (one
// token 7.2 for 7.45 us, 64 over 40 adapters 12.6 for 13.3, 7000 rows 68 for 70.6), but columns in which sums cancel lose what is left of them.
#include <algorithm>

#include "adapters.cuh"

using namespace fb;
using namespace fb::adapter;

constexpr int64_t kMostRows = 1 << 26, kMostColumns = 1 << 28;
static int check_sizes(const frisk_b200_adapter_desc* d) {
  if (d->dtype != FRISK_B200_F16 && d->dtype != FRISK_B200_BF16) return FRISK_B200_E_CACHE_TYPE;
  if (d->dtype_c != d->dtype && d->dtype_c != FRISK_B200_F32) return FRISK_B200_E_CACHE_TYPE;
  if (d->rows < 0 || d->rows > INT32_MAX || d->batch < 0 || d->count < 0 || d->K < 1 || d->N < 1 || d->K > INT32_MAX - 64 || d->N > INT32_MAX - 64 || d->rank < 8 ||
      d->rank > kMaxRank || d->rank % 8)
    return FRISK_B200_E_CACHE_SHAPE;
  // (tiles over all sequences, and a tile's 16-byte pieces, are counted in 32 bits)
  if (d->rows > kMostRows || d->N > kMostColumns || (std::min<int64_t>(d->rows, d->rows / 16 + d->batch)) * kMaxCluster > INT32_MAX) return FRISK_B200_E_TOO_LARGE;
  return 0;
}

extern "C" size_t frisk_b200_adapter_workspace_bytes(const frisk_b200_adapter_desc* d) {
  return !d || check_sizes(d) || d->rows == 0 || d->batch == 0 ? 0 : adapter_tiles_workspace_bytes(*d);
}

extern "C" int frisk_b200_adapter_gemm(frisk_b200_ctx* ctx, const frisk_b200_adapter_desc* d, const void* x, const void* a, const void* b, const void* c,
                                       const float* scales, const int32_t* starts, const int32_t* adapters, void* out, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  if (!ctx || !d) return FRISK_B200_E_ARG;
  const int rc = check_sizes(d);
  if (rc) return rc;
  if (d->rows == 0 || d->batch == 0) return 0;
  if (!x || !c || !out || !starts || !adapters || (d->count > 0 && (!a || !b))) return FRISK_B200_E_ARG;
  const int64_t rows = d->rows;
  if ((rows > 1 && (d->ldx < d->K || d->ldc < d->N || d->ldo < d->N)) || d->lda < d->K || d->ldb < d->rank || (d->count > 1 && (d->a_step < 0 || d->b_step < 0)))
    return FRISK_B200_E_CACHE_SHAPE;
  const size_t es = 2, cs = dtype_size(d->dtype_c);
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) || (rows > 1 && d->ldx % 8) || d->lda % 8 || d->ldb % 8 ||
      (d->count > 1 && (d->a_step % 8 || d->b_step % 8)))
    return FRISK_B200_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(out)) % cs ||
      ((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(starts) | reinterpret_cast<uintptr_t>(adapters)) & 3u))
    return FRISK_B200_E_ALIGN;
  // out apart from everything but a c in its own place; x, c and out may be columns of one buffer
  auto bytes = [](const void* p, int64_t ld, size_t e) { return frisk_b200_packed{const_cast<void*>(p), ld * (int64_t)e, 0}; };
  const frisk_b200_packed po = bytes(out, d->ldo, cs);
  auto apart = [&](const frisk_b200_packed& y, int64_t width) {
    // (as rows of bytes of one width: the wider of the two would do, but ends apart are told by their own)
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(po.ptr), o1 = o0 + (rows - 1) * po.row_stride + d->N * cs, y0 = reinterpret_cast<uintptr_t>(y.ptr),
                    y1 = y0 + (rows - 1) * y.row_stride + width;
    if (o1 <= y0 || y1 <= o0) return true;
    if (rows == 1 || po.row_stride != y.row_stride) return false;
    const int64_t m = po.row_stride, at = ((int64_t)(y0 - o0) % m + m) % m;  // where y's columns begin in out's rows
    return at >= (int64_t)(d->N * cs) && at + width <= m;
  };
  const bool in_place = out == c && (rows == 1 || d->ldo == d->ldc);
  if (!in_place && !apart(bytes(c, d->ldc, cs), d->N * cs)) return FRISK_B200_E_OVERLAP;
  if (!apart(bytes(x, d->ldx, es), d->K * es)) return FRISK_B200_E_OVERLAP;
  const size_t out_bytes = (size_t)((rows - 1) * d->ldo + d->N) * cs;
  auto weights = [&](int64_t step, int64_t ld, int64_t n, int64_t width) { return d->count ? (size_t)((d->count - 1) * step + (n - 1) * ld + width) * es : 0; };
  const size_t a_bytes = weights(d->a_step, d->lda, d->rank, d->K), b_bytes = weights(d->b_step, d->ldb, d->N, d->rank);
  if ((a_bytes && ranges_overlap(out, out_bytes, a, a_bytes)) || (b_bytes && ranges_overlap(out, out_bytes, b, b_bytes)) ||
      (scales && d->count && ranges_overlap(out, out_bytes, scales, (size_t)d->count * 4)) || ranges_overlap(out, out_bytes, starts, ((size_t)d->batch + 1) * 4) ||
      ranges_overlap(out, out_bytes, adapters, (size_t)d->batch * 4))
    return FRISK_B200_E_OVERLAP;
  const size_t need = adapter_tiles_workspace_bytes(*d);
  if (need) {
    if (!workspace || workspace_bytes < need) return FRISK_B200_E_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return FRISK_B200_E_ALIGN;
    const size_t x_bytes = (size_t)((rows - 1) * d->ldx + d->K) * es, c_bytes = (size_t)((rows - 1) * d->ldc + d->N) * cs;
    if (ranges_overlap(workspace, need, out, out_bytes) || ranges_overlap(workspace, need, x, x_bytes) || ranges_overlap(workspace, need, c, c_bytes) ||
        (a_bytes && ranges_overlap(workspace, need, a, a_bytes)) || (b_bytes && ranges_overlap(workspace, need, b, b_bytes)) ||
        (scales && d->count && ranges_overlap(workspace, need, scales, (size_t)d->count * 4)) ||
        ranges_overlap(workspace, need, starts, ((size_t)d->batch + 1) * 4) || ranges_overlap(workspace, need, adapters, (size_t)d->batch * 4))
      return FRISK_B200_E_OVERLAP;
  }
  AdapterParams p{};
  p.x = x;
  p.a = a;
  p.b = b;
  p.c = c;
  p.out = out;
  p.scales = scales;
  p.starts = starts;
  p.adapters = adapters;
  p.ldx = d->ldx;
  p.lda = d->lda;
  p.a_step = d->a_step;
  p.ldb = d->ldb;
  p.b_step = d->b_step;
  p.ldc = d->ldc;
  p.ldo = d->ldo;
  p.rows = rows;
  p.K = (int)d->K;
  p.N = (int)d->N;
  p.R = d->rank;
  p.count = d->count;
  p.batch = d->batch;
  const uint64_t begins = reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(out) | (rows > 1 ? (uint64_t)((d->ldc | d->ldo) * (int64_t)cs) : 0);
  p.begins = begins % 16 == 0 ? 16 : begins % 8 == 0 ? 8 : begins % 4 == 0 ? 4 : 0;
  p.status = ctx->d_status;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (need) return launch_adapter_tiles(ctx, *d, p, workspace, s);
  const bool f32 = d->dtype_c == FRISK_B200_F32;
  FB_CUDA(ctx, d->dtype == FRISK_B200_F16 ? launch_adapter_rows_f16(ctx, p, f32, s) : launch_adapter_rows_bf16(ctx, p, f32, s));
  return 0;
}
