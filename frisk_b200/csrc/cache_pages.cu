// Pages of a cache that sequences share: forked, handed out, given back, moved together; pages copied; accepted rows moved together.
//
// users[p] is the number of table entries that name page p, 0 where it is free; a table entry below 0 names none.  All tables live on the
// device, so that a captured step is replayed with other contents, and every result follows from them alone: pages are taken lowest
// first, by sequences in their order, whatever the order of threads.
//
// fork     row b of the table becomes the old row parents[b], its entries behind the last key -1; users follow by integer atomics.  A cluster reads all
//          and then writes all, or (larger tables) two launches and a workspace do
// grow     one CTA plans: the slots that new tokens touch, in order of (sequence, slot), take the free pages in order (block scans); then
//          a second kernel copies the keys of last pages that were shared
// compact  one CTA pairs the k-th used page behind the first n (n: used pages) with the k-th free one among them, by one scan; then all copy
// keep     a block a sequence; a thread has one 16-byte column of the rows and moves it row by row: row kept[i] >= i comes to row i, so
//          no store meets a row that is still to be read
//
// Bound by HBM where pages are copied (1400 pages of 256 KB: 128 us, 5.7 TB/s read and written; 2000 of 9000 pages of 33 KB moved together: 31 us, 22 of them
// the copy at 6.1 TB/s, the rest the plan), else by launches and chains of dependent loads (fork of 16 rows 4.5 us; grow of 16 sequences 8.8 with its
// copies, of 192 14.6).
#include <algorithm>

#include "cache_common.cuh"

namespace fb {
int cache_validate(const frisk_b200_cache_desc* c);
cache::Tables cache_tables(const frisk_b200_cache_desc* c);
bool cache_overlaps(const frisk_b200_cache_desc* c, const void* ptr, size_t bytes);

namespace {
using namespace cache;

constexpr int kPlan = 1024;    // threads of a planning CTA
constexpr int kMove = 256;     // of one that copies
constexpr int kAhead = 4;      // pieces of 16 bytes a thread has in flight
constexpr int kSearched = 2048;  // sequences whose offsets fit into shared memory

struct Held {  // a cache's tensors as bytes
  uint8_t* part[4];     // keys, values, exponents of both
  uint32_t pieces[4];   // 16-byte pieces of a page
};
struct PageTables {
  const int *users, *table, *lengths, *starts, *parents;
  int *users_out, *table_out, *lengths_out;
  int64_t stride, out_stride;
  int batch, width;
  int pages, page, page_log2;
  int* ws;
  unsigned* status;
};

__device__ __forceinline__ void pdl_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void flag(unsigned* status, unsigned what) { atomicCAS(status, 0u, what); }

// The exclusive sum of `x` over the block's threads in order, and the sum of all.  Every thread of the block calls it.
__device__ __forceinline__ int block_scan(int x, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  __syncthreads();  // (the sums of the call before have been read)
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int s = lane < kPlan / 32 ? sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += up;
  }
  *total = __shfl_sync(0xffffffffu, s, kPlan / 32 - 1);
  const int before = __shfl_sync(0xffffffffu, s, warp ? warp - 1 : 0);
  return incl - x + (warp ? before : 0);
}

// What is not done in place, eight entries in flight: the compiler cannot tell that a store does not change what is still to be read.
constexpr int kDeep = 8;
__device__ __forceinline__ void copy_users(const PageTables& t, int64_t first, int64_t step) {
  if (t.users_out == t.users) return;
  for (int64_t p0 = first; p0 < t.pages; p0 += kDeep * step) {
    int x[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      if (p0 + j * step < t.pages) x[j] = t.users[p0 + j * step];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      if (p0 + j * step < t.pages) t.users_out[p0 + j * step] = x[j];
  }
}
__device__ __forceinline__ void copy_table(const PageTables& t, int64_t first, int64_t step) {
  if (t.table_out == t.table) return;
  const uint32_t slots = (uint32_t)t.batch * t.width, width = max(t.width, 1);
  for (uint32_t i0 = (uint32_t)first; i0 < slots; i0 += kDeep * (uint32_t)step) {
    int x[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const uint32_t i = i0 + j * (uint32_t)step, b = i / width;
      if (i < slots) x[j] = t.table[b * t.stride + i - b * width];
    }
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const uint32_t i = i0 + j * (uint32_t)step, b = i / width;
      if (i < slots) t.table_out[b * t.out_stride + i - b * width] = x[j];
    }
  }
}

// ------------------------------------------------------------------------------------------------ fork
// The row that slot `slot` of row b comes from, of its parent and the parent's length; -1: from none
__device__ __forceinline__ int forked_from(const PageTables& t, int b, int slot, int parent, int length) {
  if (parent < -1 || parent >= t.batch) return b;  // (said where the lengths are made)
  if (parent < 0) return -1;
  if (length < 0 || length > (int64_t)t.width * t.page) return b;
  return (int64_t)slot << t.page_log2 >= length ? -1 : parent;
}
__device__ __forceinline__ int forked_length(const PageTables& t, int b) {
  const int parent = t.parents[b];
  const bool known = parent >= -1 && parent < t.batch;
  const int length = t.lengths[known && parent >= 0 ? parent : b];
  const bool ok = known && (parent < 0 || (length >= 0 && length <= (int64_t)t.width * t.page));
  if (!ok) flag(t.status, known ? ST_CACHE_LENGTH : ST_CACHE_ROWS);
  return !ok ? t.lengths[b] : parent < 0 ? 0 : length;
}
__device__ __forceinline__ void apply_fork(const PageTables& t, int b, int slot, int old, int entry) {
  if (old != entry) {
    if (old >= t.pages || entry >= t.pages) flag(t.status, ST_CACHE_PAGE);
    if (old >= 0 && old < t.pages) atomicSub(t.users_out + old, 1);
    if (entry >= 0 && entry < t.pages) atomicAdd(t.users_out + entry, 1);
  }
  t.table_out[b * t.out_stride + slot] = entry;
}

// Tables that one cluster's threads can hold: all is read, then all is written.  (16 rows of 34 pages 5.7 us, in two launches 6.4 and more of the host; 192 rows of
// 378 pages 13.9, in two launches 7.8: eight SMs have too many instructions to do.)
constexpr int kTogether = 8, kHeldSlots = 4;
constexpr int64_t kForkTogether = (int64_t)kTogether * kPlan * kHeldSlots;
__global__ void __launch_bounds__(kPlan) fork_kernel(const PageTables t) {
  pdl_begin();
  constexpr int kStep = kTogether * kPlan;
  const int first = blockIdx.x * kPlan + threadIdx.x, slots = t.batch * t.width;
  copy_users(t, first, kStep);
  // (in steps of their own, so that the loads of all slots are on their way at once)
  int old[kHeldSlots], entry[kHeldSlots], parent[kHeldSlots];
#pragma unroll
  for (int j = 0; j < kHeldSlots; ++j) {
    const int i = first + j * kStep, b = i / max(t.width, 1);
    if (i < slots) parent[j] = t.parents[b];
  }
#pragma unroll
  for (int j = 0; j < kHeldSlots; ++j) {
    const int i = first + j * kStep, b = i / max(t.width, 1);
    if (i < slots) {
      old[j] = t.table[b * t.stride + i - b * t.width];
      entry[j] = t.lengths[parent[j] >= 0 && parent[j] < t.batch ? parent[j] : b];
    }
  }
#pragma unroll
  for (int j = 0; j < kHeldSlots; ++j) {
    const int i = first + j * kStep, b = i / max(t.width, 1);
    if (i < slots) {
      const int slot = i - b * t.width, from = forked_from(t, b, slot, parent[j], entry[j]);
      entry[j] = from < 0 ? -1 : max(t.table[from * t.stride + slot], -1);
    }
  }
  const int length = first < t.batch ? forked_length(t, first) : 0;
  __syncwarp();
  cluster_sync_all();
  if (first < t.batch) t.lengths_out[first] = length;
#pragma unroll
  for (int j = 0; j < kHeldSlots; ++j) {
    const int i = first + j * kStep;
    if (i >= slots) break;
    const int b = i / t.width;
    apply_fork(t, b, i - b * t.width, old[j], entry[j]);
  }
}

// Larger ones.  The new table into the workspace: [batch][width], then the lengths [batch].  (The old one is still read, by other rows too.)
__global__ void __launch_bounds__(kMove) fork_stage_kernel(const PageTables t) {
  pdl_begin();
  const int64_t i = (int64_t)blockIdx.x * kMove + threadIdx.x, slots = (int64_t)t.batch * t.width;
  if (t.users_out != t.users)
    for (int64_t p = i; p < t.pages; p += (int64_t)gridDim.x * kMove) t.users_out[p] = t.users[p];
  if (i < t.batch) t.ws[slots + i] = forked_length(t, (int)i);
  if (i >= slots) return;
  const int b = (int)(i / t.width), slot = (int)(i - (int64_t)b * t.width), parent = t.parents[b];
  const int from = forked_from(t, b, slot, parent, t.lengths[parent >= 0 && parent < t.batch ? parent : b]);
  t.ws[i] = from < 0 ? -1 : max(t.table[from * t.stride + slot], -1);
}
__global__ void __launch_bounds__(kMove) fork_apply_kernel(const PageTables t) {
  pdl_begin();
  const int64_t i = (int64_t)blockIdx.x * kMove + threadIdx.x, slots = (int64_t)t.batch * t.width;
  if (i < t.batch) t.lengths_out[i] = t.ws[slots + i];
  if (i >= slots) return;
  const int b = (int)(i / t.width), slot = (int)(i - (int64_t)b * t.width);
  apply_fork(t, b, slot, t.table[b * t.stride + slot], t.ws[i]);
}

// ------------------------------------------------------------------------------------------------ grow
__global__ void __launch_bounds__(kMove) copy_tables_kernel(const PageTables t) {
  pdl_begin();
  copy_users(t, (int64_t)blockIdx.x * kMove + threadIdx.x, (int64_t)gridDim.x * kMove);
  copy_table(t, (int64_t)blockIdx.x * kMove + threadIdx.x, (int64_t)gridDim.x * kMove);
}

// What becomes of a touched slot
enum : int { KEEP = 0, KEEP_AS_LAST = 1, TAKE = 2, SWAP = 3 };  // (the last that has a page keeps it, if the others take theirs)

// Places of the workspace, in ints.  T = batch * width bounds the touched slots.
struct GrowWork {
  int *copies;       // [batch][3]: page to copy from (-1: none), to, keys
  int *offset;       // [batch + 1]: first touched slot, in order of (sequence, slot)
  int *depends;      // [batch]
  int *kind, *before;  // [T], [T + 1]: what becomes of the slot; pages taken by those before it
  int *shared, *page;  // [T]: touched slots whose page others have too, and the page
  int *free;           // [T]
  int *holders, *last; // [pages]: of the touched slots whose page others have too, those with that page, and the last
  static constexpr int kSmall = 1536;  // touched slots whose lists are in shared memory
  __host__ __device__ static int64_t ints(int64_t batch, int64_t width, int64_t pages) { return 5 * batch + 1 + 5 * batch * width + 1 + 2 * pages; }
  __device__ GrowWork(int* ws, int64_t batch, int64_t width, int64_t pages) {
    const int64_t slots = batch * width;
    copies = ws;
    offset = copies + 3 * batch;
    depends = offset + batch + 1;
    kind = depends + batch;
    before = kind + slots;
    shared = before + slots + 1;
    page = shared + slots;
    free = page + slots;
    holders = free + slots;
    last = holders + pages;
  }
};

// COPIES: beside the planning CTA, the others of its cluster copy the tables that are not changed in place.  (The plan is made from the old ones; only what
// it changes waits for the copies.)
template <bool COPIES>
__global__ void __launch_bounds__(kPlan) grow_plan_kernel(const PageTables t) {
  __shared__ int sums[32], any_refused;
  __shared__ int near[kSearched + 1];  // offsets, where they fit
  extern __shared__ int lists[];       // five of kSmall, and one place
  GrowWork w(t.ws, t.batch, t.width, t.pages);
  const int tid = threadIdx.x, lane = tid & 31;
  pdl_begin();
  if (COPIES && blockIdx.x > 0) {
    copy_users(t, (int64_t)(blockIdx.x - 1) * kPlan + tid, (int64_t)(gridDim.x - 1) * kPlan);
    copy_table(t, (int64_t)(blockIdx.x - 1) * kPlan + tid, (int64_t)(gridDim.x - 1) * kPlan);
    __syncwarp();
    cluster_sync_all();
    return;
  }
  // (the first pages that may be free are looked at meanwhile)
  constexpr int kEach = 8;
  const int own = (tid >> 5) * 32 * kEach + lane;  // of a round of kPlan * kEach pages, the first that this thread looks at
  int ahead[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) ahead[j] = own + 32 * j < t.pages ? t.users[own + 32 * j] : 1;
  // 1. the slots that each sequence's new tokens touch
  if (tid == 0) any_refused = 0;
  int all = 0;
  for (int b0 = 0; b0 < t.batch; b0 += kPlan) {
    const int b = b0 + tid;
    int n = 0;
    if (b < t.batch) {
      const int lo = t.starts[b], hi = t.starts[b + 1], length = t.lengths[b];
      const int64_t count = (int64_t)hi - lo;
      const bool rows_ok = lo >= 0 && count >= 0, ok = rows_ok && length >= 0 && length + count <= (int64_t)t.width * t.page;
      if (!ok) flag(t.status, rows_ok ? ST_CACHE_LENGTH : ST_CACHE_ROWS);
      if (ok && count > 0) n = (int)(((length + count - 1) >> t.page_log2) - (length >> t.page_log2)) + 1;
      w.copies[3 * b] = -1;
      w.depends[b] = 0;
      t.lengths_out[b] = ok ? (int)count : 0;  // (granted; taken back below)
    }
    int total;
    const int at = all + block_scan(n, sums, &total);
    if (b < t.batch) {
      w.offset[b] = at;
      if (b < kSearched) near[b] = at;
    }
    all += total;
  }
  if (tid == 0) {
    w.offset[t.batch] = all;
    if (t.batch <= kSearched) near[t.batch] = all;
  }
  __syncthreads();
  const int* offset = t.batch <= kSearched ? near : w.offset;
  if (all <= GrowWork::kSmall) {
    w.kind = lists;
    w.before = w.kind + GrowWork::kSmall;
    w.shared = w.before + GrowWork::kSmall + 1;
    w.page = w.shared + GrowWork::kSmall;
    w.free = w.page + GrowWork::kSmall;
  }
  auto owner = [&](int i) {  // the last b with offset[b] <= i: the one whose slot it is
    int lo = 0, hi = t.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (offset[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
  };
  auto refused = [&](int b) { return *const_cast<volatile int*>(t.lengths_out + b) == 0; };
  // 2. what they name; those that others name too are listed.  A sequence that names a page without users gets nothing: it is told, and all is listed again without its slots.
  int n_shared = 0;
  bool again = false;
  while (true) {
    for (int i0 = 0; i0 < all; i0 += kPlan) {
      const int i = i0 + tid;
      int entry = -1;
      bool shared = false;
      if (i < all) {
        const int b = owner(i), slot = (t.lengths[b] >> t.page_log2) + i - offset[b];
        entry = t.table[b * t.stride + slot];
        const bool there = entry >= 0 && entry < t.pages, left = again && refused(b);
        const int users = there ? t.users[entry] : 0;
        if (entry >= t.pages) flag(t.status, ST_CACHE_PAGE);
        if (there && users <= 0) {
          flag(t.status, ST_CACHE_PAGE);
          t.lengths_out[b] = 0;
          any_refused = 1;
        }
        shared = users > 1 && !left;
        const bool alone = users == 1 && !left;
        w.kind[i] = entry < 0 && !left ? TAKE : KEEP;
        w.free[i] = alone ? entry : -1;
        if (alone) __stcg(w.last + entry, i);  // (any of those that name it)
      }
      int total;
      const int at = n_shared + block_scan(shared, sums, &total);
      if (shared) {
        w.shared[at] = i;
        w.page[at] = entry;
      }
      n_shared += total;
    }
    __syncthreads();
    if (again || !any_refused) break;
    again = true;
    n_shared = 0;
  }
  // 3. of the sequences that are going to write into a page, all take one of their own but the last that has it, if no one else does
  auto decide = [&](int k, int page, int holders, bool last) {  // of the touched slots with that page: how many, and whether k is the last
    const int users = t.users[page];
    if (users < holders) flag(t.status, ST_CACHE_PAGE);  // (it has more users than are said: left)
    else if (users > holders || !last) w.kind[w.shared[k]] = SWAP;
    else w.kind[w.shared[k]] = KEEP_AS_LAST;
  };
  if (all <= GrowWork::kSmall) {
    for (int k = tid; k < n_shared; k += kPlan) {
      const int page = w.page[k];
      int holders = 0, later = 0;
#pragma unroll 8
      for (int j = 0; j < n_shared; ++j) {
        const int same = w.page[j] == page;
        holders += same;
        later += same & (int)(j > k);
      }
      decide(k, page, holders, later == 0);
    }
  } else {  // (pair by pair, 10^5 of them would take seconds)
    for (int k = tid; k < n_shared; k += kPlan) {
      w.holders[w.page[k]] = 0;
      w.last[w.page[k]] = -1;
    }
    __syncthreads();
    for (int k = tid; k < n_shared; k += kPlan) {
      atomicAdd(w.holders + w.page[k], 1);
      atomicMax(w.last + w.page[k], k);
    }
    __syncthreads();
    for (int k = tid; k < n_shared; k += kPlan) {
      const int page = w.page[k];
      decide(k, page, __ldcg(w.holders + page), __ldcg(w.last + page) == k);
    }
  }
  __syncthreads();
  // 4. how many pages are taken before each slot
  int taken = 0;
  for (int i0 = 0; i0 < all; i0 += kPlan) {
    const int i = i0 + tid, kind = i < all ? w.kind[i] : KEEP, alone = i < all ? w.free[i] : -1;
    const int who = alone >= 0 ? __ldcg(w.last + alone) : i;  // (on its way meanwhile)
    int total;
    const int at = taken + block_scan(kind >= TAKE, sums, &total);
    if (i < all) w.before[i] = at;
    if (who != i) flag(t.status, ST_CACHE_PAGE);  // two slots name a page of one user: left, as above
    if (kind == SWAP || kind == KEEP_AS_LAST) w.depends[owner(i)] = 1;  // (all that write it, write 1)
    taken += total;
  }
  if (tid == 0) w.before[all] = taken;
  // 5. that many free pages, lowest first: a warp looks at 256 pages a round, 32 at a time.  (Not those that a refused sequence names: they are marked.)
  if (again) {
    for (int p = tid; p < t.pages; p += kPlan) w.last[p] = 0;
    __syncthreads();
    for (int i = tid; i < all; i += kPlan) {
      const int b = owner(i), entry = t.table[b * t.stride + (t.lengths[b] >> t.page_log2) + i - offset[b]];
      if (refused(b) && entry >= 0 && entry < t.pages) w.last[entry] = 1;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (own + 32 * j < t.pages && __ldcg(w.last + own + 32 * j)) ahead[j] = 1;
  }
  int found = 0;
  for (int p0 = 0; p0 < t.pages && found < taken; p0 += kPlan * kEach) {
    const int first = p0 + own;
    if (p0 > 0) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) ahead[j] = first + 32 * j < t.pages ? t.users[first + 32 * j] : 1;
      if (again) {
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          if (first + 32 * j < t.pages && __ldcg(w.last + first + 32 * j)) ahead[j] = 1;
      }
    }
    unsigned masks[kEach];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      masks[j] = __ballot_sync(0xffffffffu, ahead[j] == 0);
      mine += __popc(masks[j]);
    }
    int total;
    int at = found + __shfl_sync(0xffffffffu, block_scan(lane == 0 ? mine : 0, sums, &total), 0);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int k = at + __popc(masks[j] & ((1u << lane) - 1u));
      if ((masks[j] >> lane & 1u) && k < taken) w.free[k] = first + 32 * j;
      at += __popc(masks[j]);
    }
    found += total;
  }
  __syncthreads();
  // 6. a sequence gets all it needs or, with those behind it, nothing
  for (int b = tid; b < t.batch; b += kPlan) {
    const int need = w.before[offset[b + 1]] - w.before[offset[b]];
    const bool granted = !(again && refused(b)) && (w.before[offset[b + 1]] <= found || (need == 0 && !w.depends[b]));
    if (!granted) t.lengths_out[b] = 0;
    w.depends[b] = granted;
  }
  __syncthreads();
  if (COPIES) {
    __syncwarp();
    cluster_sync_all();
  }
  for (int i = tid; i < all; i += kPlan) {
    const int kind = w.kind[i];
    if (kind < TAKE) continue;
    const int b = owner(i);
    if (!w.depends[b]) continue;
    const int length = t.lengths[b], nth = i - offset[b], page = w.free[w.before[i]];
    const int64_t slot = (length >> t.page_log2) + nth;
    if (kind == SWAP) {
      const int old = t.table[b * t.stride + slot];
      atomicSub(t.users_out + old, 1);
      if (nth == 0 && (length & (t.page - 1))) {  // its keys come along
        w.copies[3 * b] = old;
        w.copies[3 * b + 1] = page;
        w.copies[3 * b + 2] = length & (t.page - 1);
      }
    }
    t.table_out[b * t.out_stride + slot] = page;
    t.users_out[page] = 1;
  }
}

// A block a sequence and head.  row: 16-byte pieces of a head's row
__global__ void __launch_bounds__(kMove) grow_copy_kernel(const int* copies, uint4* k, uint4* v, uint8_t* ek, uint8_t* ev, int heads, int page, int row) {
  pdl_begin();
  const int b = blockIdx.x / heads, h = blockIdx.x - b * heads;
  const int from = copies[3 * b], to = copies[3 * b + 1], keys = copies[3 * b + 2];
  if (from < 0) return;
  const int64_t src = ((int64_t)from * heads + h) * page, dst = ((int64_t)to * heads + h) * page;
  const int pieces = keys * row;
  for (int i = threadIdx.x; i < pieces; i += kMove) {
    const uint4 x = __ldcs(k + src * row + i), y = __ldcs(v + src * row + i);
    k[dst * row + i] = x;
    v[dst * row + i] = y;
  }
  if (ek)
    for (int i = threadIdx.x; i < keys; i += kMove) {
      ek[dst + i] = ek[src + i];
      ev[dst + i] = ev[src + i];
    }
}

// ------------------------------------------------------------------------------------------------ whole pages
// The workspace of compact: moves, then from [pages], to [pages], goes [pages].  With n used pages, u(p) of them before page p, a free page p < n is hole
// p - u(p), and a used one p >= n is move u(p) - u(n): one scan gives both.  A warp has neighbouring pages, 32 at a time, the first kHold of these
// words in registers (up to 16384 pages are read once).  2000 of 9000 pages of 33 KB: 31.4 us with the move; in two scans, with lists in memory, 33.5.
constexpr int kHold = 16;
constexpr int kNear = 2560;  // moves whose lists are in shared memory too
__global__ void __launch_bounds__(kPlan) compact_plan_kernel(const PageTables t) {
  __shared__ int sums[32], near_from[kNear], near_to[kNear], near_users[kNear], at_border;
  constexpr int kEach = 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int words = (t.pages + 31) / 32, per = (words + kPlan / 32 - 1) / (kPlan / 32), word0 = min(words, warp * per), word1 = min(words, word0 + per);
  int *from = t.ws + 1, *to = from + t.pages, *goes = to + t.pages;  // (goes[k], k below the moves and so below n: the users of the page that moves)
  pdl_begin();
  auto look = [&](int word) { return word < word1 && word * 32 + lane < t.pages ? t.users[word * 32 + lane] : 0; };
  int held[kHold], mine = 0, used;
#pragma unroll
  for (int j = 0; j < kHold; ++j) held[j] = look(word0 + j);
#pragma unroll
  for (int j = 0; j < kHold; ++j) mine += held[j] != 0;
  for (int w = word0 + kHold; w < word1; w += kEach) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) mine += look(w + j) != 0;
  }
  const int start = __shfl_sync(0xffffffffu, block_scan(mine, sums, &used), 0);  // used pages before the warp's
  const int border = used >> 5;  // the word of page n
  if (border >= word0 && border < word1) {
    int before = 0;
#pragma unroll
    for (int j = 0; j < kHold; ++j) before += held[j] != 0 && (word0 + j < border || (word0 + j == border && lane < (used & 31)));
    for (int w = word0 + kHold; w <= border; ++w) before += look(w) != 0 && (w < border || lane < (used & 31));
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) at_border = start + before;
  } else if (border == words && tid == 0) {  // (all are used)
    at_border = used;
  }
  __syncthreads();
  const int stay = at_border, moves = used - stay;
  int u = start;
  auto place = [&](int word, int users) {
    const unsigned mask = __ballot_sync(0xffffffffu, users != 0);
    const int p = word * 32 + lane, before = u + __popc(mask & ((1u << lane) - 1u));
    u += __popc(mask);
    if (p >= t.pages) return;
    if (p < used) {
      if (users == 0) {
        to[p - before] = p;
        if (p - before < kNear) near_to[p - before] = p;
      } else if (t.users_out != t.users) {
        t.users_out[p] = users;
      }
    } else {
      const int k = before - stay;
      if (users == 0) {
        goes[p] = -1;
      } else {
        from[k] = p;
        if (k < kNear) {
          near_from[k] = p;
          near_users[k] = users;
        } else {
          goes[k] = users;
        }
      }
      t.users_out[p] = 0;
    }
  };
#pragma unroll
  for (int j = 0; j < kHold; ++j)
    if (word0 + j < word1) place(word0 + j, held[j]);
  for (int w = word0 + kHold; w < word1; w += kEach) {
    int users[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) users[j] = look(w + j);
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (w + j < word1) place(w + j, users[j]);
  }
  __syncthreads();
  for (int k = tid; k < moves; k += kPlan) {  // (as many holes as moves)
    const bool near = k < kNear;
    const int p = near ? near_from[k] : from[k], q = near ? near_to[k] : to[k];
    t.users_out[q] = near ? near_users[k] : goes[k];
    goes[p] = q;
  }
  if (tid == 0) {
    t.ws[0] = moves;
    t.lengths_out[0] = used;
  }
}

// Copies page from[i] of `src` to page to[i] of `dst`, i < n (or *n_device): 16 bytes a lane, kAhead in flight.
__device__ __forceinline__ void move_pages(const Held& src, const Held& dst, const int* from, const int* to, int64_t n, int src_pages, int dst_pages, unsigned* status) {
  const uint32_t c1 = src.pieces[0], c2 = c1 + src.pieces[1], c3 = c2 + src.pieces[2], each = c3 + src.pieces[3];
  const int64_t total = n * each, step = (int64_t)gridDim.x * kMove * kAhead;
  for (int64_t base = (int64_t)blockIdx.x * kMove * kAhead; base < total; base += step) {
    const int64_t k0 = base / each;
    const uint32_t rest = (uint32_t)(base - k0 * each);
    uint4 x[kAhead];
    uint4* at[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      at[j] = nullptr;
      const uint32_t local = rest + threadIdx.x + j * kMove, more = local / each;
      if (base + threadIdx.x + j * kMove >= total) continue;
      const int64_t k = k0 + more;
      uint32_t piece = local - more * each;
      const int p = __ldg(from + k), q = __ldg(to + k);
      if (p < 0 || p >= src_pages || q < 0 || q >= dst_pages) {
        flag(status, ST_CACHE_PAGE);
        continue;
      }
      const int part = piece < c1 ? 0 : piece < c2 ? 1 : piece < c3 ? 2 : 3;
      piece -= part == 0 ? 0 : part == 1 ? c1 : part == 2 ? c2 : c3;
      const uint32_t size = part < 2 ? c1 : src.pieces[2];
      uint8_t* a = part == 0 ? src.part[0] : part == 1 ? src.part[1] : part == 2 ? src.part[2] : src.part[3];
      uint8_t* d = part == 0 ? dst.part[0] : part == 1 ? dst.part[1] : part == 2 ? dst.part[2] : dst.part[3];
      x[j] = __ldcs(reinterpret_cast<const uint4*>(a) + (int64_t)p * size + piece);
      at[j] = reinterpret_cast<uint4*>(d) + (int64_t)q * size + piece;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (at[j]) __stcs(at[j], x[j]);
  }
}
__global__ void __launch_bounds__(kMove) copy_pages_kernel(const Held src, const Held dst, const int* from, const int* to, int64_t n, int src_pages, int dst_pages,
                                                           unsigned* status) {
  pdl_begin();
  move_pages(src, dst, from, to, n, src_pages, dst_pages, status);
}
__global__ void __launch_bounds__(kMove) compact_move_kernel(const Held held, const PageTables t) {
  pdl_begin();
  const int *from = t.ws + 1, *to = from + t.pages, *goes = to + t.pages;
  const int used = t.lengths_out[0];
  const int64_t slots = (int64_t)t.batch * t.width;
  for (int64_t i = (int64_t)blockIdx.x * kMove + threadIdx.x; i < slots; i += (int64_t)gridDim.x * kMove) {
    const int64_t b = i / t.width, slot = i - b * t.width;
    int entry = t.table[b * t.stride + slot];
    if (entry >= used) {
      const int now = entry < t.pages ? goes[entry] : -1;
      if (now < 0) flag(t.status, ST_CACHE_PAGE);  // a page that is not there, or that nobody is said to use: left
      else entry = now;
    }
    t.table_out[b * t.out_stride + slot] = entry;
  }
  move_pages(held, held, from, to, t.ws[0], t.pages, t.pages, t.status);
}

// ------------------------------------------------------------------------------------------------ accepted rows
struct KeepParams {
  Tables t;
  const int *kept, *counts;
  int64_t kept_stride;
  int kept_width;
  int* lengths_out;
  uint4 *k, *v;
  uint8_t *ek, *ev;
  int row;  // 16-byte pieces of a head's row
  unsigned* status;
};
constexpr int kKeepRows = 128;  // rows whose places are in shared memory at a time

__global__ void __launch_bounds__(kMove) keep_kernel(const KeepParams p) {
  __shared__ int64_t come[kKeepRows], go[kKeepRows];  // token slots of head 0
  pdl_begin();
  const int b = blockIdx.x, tid = threadIdx.x;
  const Seq s = load_seq(p.t, b, p.status);
  const int count = p.counts[b];
  const int* kept = p.kept + b * p.kept_stride;
  bool fine = s.ok && count >= 0 && count <= p.kept_width && count <= s.count;
  if (fine) {
    bool mine = true;
    for (int i = tid; i < count; i += kMove) {
      const int at = kept[i];
      mine = mine && at >= 0 && at < s.count && (i == 0 || kept[i - 1] < at);
    }
    fine = __syncthreads_and(mine);
  }
  if (!fine) {
    if (tid == 0) {
      flag(p.status, ST_CACHE_ROWS);
      p.lengths_out[b] = s.length;
    }
    return;
  }
  const int columns = 2 * p.t.heads * p.row, bytes = p.ek ? 2 * p.t.heads : 0;
  for (int i0 = 0; i0 < count; i0 += kKeepRows) {
    const int n = min(kKeepRows, count - i0);
    __syncthreads();
    if (tid < n) {
      const int64_t from = (int64_t)s.length + kept[i0 + tid], to = (int64_t)s.length + i0 + tid;
      const int* row = p.t.table + b * p.t.stride;
      const int a = row[from >> p.t.page_log2], c = row[to >> p.t.page_log2];
      const bool there = a >= 0 && a < p.t.pages && c >= 0 && c < p.t.pages;
      if (!there) flag(p.status, ST_CACHE_PAGE);
      const bool moves = there && from != to;
      come[tid] = moves ? (((int64_t)a * p.t.heads) << p.t.page_log2) + (from & (p.t.page - 1)) : -1;
      go[tid] = moves ? (((int64_t)c * p.t.heads) << p.t.page_log2) + (to & (p.t.page - 1)) : -1;
    }
    __syncthreads();
    // (rows that are read here are not among those stored before: kept[i] >= i, ascending; so loads may run ahead of stores)
    for (int e = tid; e < columns; e += kMove) {
      const int unit = e / p.row, sub = e - unit * p.row, h = unit >= p.t.heads ? unit - p.t.heads : unit;
      uint4* x = unit >= p.t.heads ? p.v : p.k;
      const int64_t head = (int64_t)h << p.t.page_log2;
      for (int i = 0; i < n; i += kAhead) {
        uint4 y[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (i + j < n && come[i + j] >= 0) y[j] = x[(come[i + j] + head) * p.row + sub];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (i + j < n && come[i + j] >= 0) x[(go[i + j] + head) * p.row + sub] = y[j];
      }
    }
    for (int e = tid; e < bytes; e += kMove) {
      const int h = e >= p.t.heads ? e - p.t.heads : e;
      uint8_t* x = e >= p.t.heads ? p.ev : p.ek;
      const int64_t head = (int64_t)h << p.t.page_log2;
      for (int i = 0; i < n; ++i)
        if (come[i] >= 0) x[go[i] + head] = x[come[i] + head];
    }
  }
  if (tid == 0) p.lengths_out[b] = s.length + count;  // (the block has read its own: lengths_out may be lengths)
}

// ------------------------------------------------------------------------------------------------ launches
template <typename... A>
cudaError_t launch_with(void (*kernel)(A...), int64_t blocks, int threads, int smem, cudaStream_t s, typename std::common_type<A>::type... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernels wait (griddepcontrol.wait) themselves
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;  // planning CTAs, where there are several
  attr[1].val.clusterDim.x = kTogether;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = threads == kPlan && blocks == kTogether ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... A>
cudaError_t launch(void (*kernel)(A...), int64_t blocks, int threads, cudaStream_t s, typename std::common_type<A>::type... args) {
  return launch_with(kernel, blocks, threads, 0, s, args...);
}

size_t element(const frisk_b200_cache_desc* c) { return c->dtype == FRISK_B200_E4M3 ? 1 : 2; }

Held held_of(const frisk_b200_cache_desc* c) {
  Held h{};
  const size_t tokens = (size_t)c->heads * c->page, e = element(c);
  h.part[0] = static_cast<uint8_t*>(c->k);
  h.part[1] = static_cast<uint8_t*>(c->v);
  h.pieces[0] = h.pieces[1] = (uint32_t)(tokens * c->D * e / 16);
  if (c->dtype == FRISK_B200_E4M3) {
    h.part[2] = c->k_exponent;
    h.part[3] = c->v_exponent;
    h.pieces[2] = h.pieces[3] = (uint32_t)(tokens / 16);
  }
  return h;
}

int check_cache(const frisk_b200_cache_desc* c) {
  if (!c->k || !c->v || (c->dtype == FRISK_B200_E4M3 && (!c->k_exponent || !c->v_exponent))) return FRISK_B200_E_ARG;
  const uintptr_t all = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) |
                        (c->dtype == FRISK_B200_E4M3 ? reinterpret_cast<uintptr_t>(c->k_exponent) | reinterpret_cast<uintptr_t>(c->v_exponent) : 0);
  return all & 15u ? FRISK_B200_E_ALIGN : 0;
}
// a cache that is written: its tensors apart from one another
bool parts_overlap(const frisk_b200_cache_desc* c) {
  const Held h = held_of(c);
  const int n = c->dtype == FRISK_B200_E4M3 ? 4 : 2;
  for (int i = 0; i < n; ++i)
    for (int j = i + 1; j < n; ++j)
      if (ranges_overlap(h.part[i], (size_t)c->pages * h.pieces[i] * 16, h.part[j], (size_t)c->pages * h.pieces[j] * 16)) return true;
  return false;
}

struct Range {
  const void* p;
  size_t n;
  bool written;
  const void* own;  // the input that this output may be
};
// Outputs apart from one another and from all inputs but their own
int check_ranges(const Range* r, int n) {
  for (int i = 0; i < n; ++i) {
    if (r[i].n == 0) continue;
    if (!r[i].p) return FRISK_B200_E_ARG;
    if (reinterpret_cast<uintptr_t>(r[i].p) & 3u) return FRISK_B200_E_ALIGN;
    for (int j = 0; j < n; ++j) {
      if (j == i || r[j].n == 0 || !r[i].written || (r[j].written && j < i)) continue;
      if (!r[j].written && r[i].own == r[j].p && r[i].p == r[j].p) continue;
      if (ranges_overlap(r[i].p, r[i].n, r[j].p, r[j].n)) return FRISK_B200_E_OVERLAP;
    }
  }
  return 0;
}
size_t table_bytes(int64_t batch, int64_t width, int64_t stride) { return batch > 0 && width > 0 ? (size_t)((batch - 1) * stride + width) * 4 : 0; }

enum Which { FORK, GROW, COMPACT };
constexpr int64_t kCopiedTogether = 1 << 17;  // entries that a cluster copies in a few microseconds
int64_t workspace_ints(const frisk_b200_cache_desc* c, int which) {
  const int64_t batch = c->batch, width = c->table_width;
  if (which == FORK && batch * width <= kForkTogether && batch <= kTogether * kPlan && c->pages <= kCopiedTogether) return 0;
  return which == FORK ? batch * width + batch : which == GROW ? GrowWork::ints(batch, width, c->pages) : 1 + 3 * c->pages;
}
int check_sizes(const frisk_b200_cache_desc* c, int which) {
  const int rc = cache_validate(c);
  if (rc) return rc;
  if (which < FORK || which > COMPACT) return FRISK_B200_E_ARG;
  // (table slots are counted, and tokens of a sequence, in 32 bits)
  if ((int64_t)c->batch * c->table_width > INT32_MAX / 8 || c->pages > INT32_MAX / 4 || (int64_t)c->table_width * c->page > INT32_MAX) return FRISK_B200_E_CACHE_SHAPE;
  return 0;
}

int prepare(const frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, const frisk_b200_page_tables* t, int which, const int32_t* parents, void* ws, size_t ws_bytes,
            PageTables* out) {
  if (!ctx || !c || !t) return FRISK_B200_E_ARG;
  int rc = check_sizes(c, which);
  if (rc) return rc;
  if (c->batch > 1 && t->table_out_stride < c->table_width) return FRISK_B200_E_CACHE_SHAPE;
  if (t->table_out == c->table && c->batch > 1 && c->table_width > 0 && t->table_out_stride != c->table_stride) return FRISK_B200_E_OVERLAP;
  const size_t need = (size_t)workspace_ints(c, which) * 4, batch = (size_t)c->batch * 4, pages = (size_t)c->pages * 4;
  if (need && (!ws || ws_bytes < need)) return FRISK_B200_E_WORKSPACE;
  const Range all[] = {
      {t->users, pages, false, nullptr},
      {c->table, table_bytes(c->batch, c->table_width, c->table_stride), false, nullptr},
      {c->lengths, which == COMPACT ? 0 : batch, false, nullptr},
      {c->starts, which == GROW ? batch + 4 : 0, false, nullptr},
      {parents, which == FORK ? batch : 0, false, nullptr},
      {t->users_out, pages, true, t->users},
      {t->table_out, table_bytes(c->batch, c->table_width, t->table_out_stride), true, c->table},
      {t->lengths_out, which == COMPACT ? 4 : batch, true, which == FORK ? c->lengths : nullptr},
      {ws, need, true, nullptr},
  };
  if ((rc = check_ranges(all, (int)(sizeof(all) / sizeof(all[0]))))) return rc;
  if (which != FORK) {
    if ((rc = check_cache(c))) return rc;
    if (parts_overlap(c)) return FRISK_B200_E_OVERLAP;
    for (const Range& r : all)
      if (r.n && cache_overlaps(c, r.p, r.n)) return FRISK_B200_E_OVERLAP;
  }
  PageTables p{};
  p.users = t->users;
  p.table = c->table;
  p.lengths = c->lengths;
  p.starts = c->starts;
  p.parents = parents;
  p.users_out = t->users_out;
  p.table_out = t->table_out;
  p.lengths_out = t->lengths_out;
  p.stride = c->table_stride;
  p.out_stride = t->table_out_stride;
  p.batch = c->batch;
  p.width = c->table_width;
  p.pages = (int)c->pages;
  p.page = c->page;
  p.page_log2 = cache_tables(c).page_log2;
  p.ws = static_cast<int*>(ws);
  p.status = ctx->d_status;
  *out = p;
  return 0;
}

int64_t blocks_for(int64_t n) { return (n + kMove - 1) / kMove; }
// of the kernels that loop: enough to fill the GPU
int64_t blocks_up_to(const frisk_b200_ctx* ctx, int64_t blocks) { return std::max<int64_t>(1, std::min<int64_t>(blocks, 8 * ctx->num_sms)); }

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" {

size_t frisk_b200_cache_pages_workspace_bytes(const frisk_b200_cache_desc* c, int32_t which) {
  return check_sizes(c, which) ? 0 : (size_t)workspace_ints(c, which) * 4;
}

int frisk_b200_cache_fork(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, const frisk_b200_page_tables* tables, const int32_t* parents, void* workspace,
                          size_t workspace_bytes, void* stream) {
  PageTables t;
  const int rc = prepare(ctx, c, tables, FRISK_B200_PAGES_FORK, parents, workspace, workspace_bytes, &t);
  if (rc) return rc;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t slots = (int64_t)t.batch * t.width, work = std::max<int64_t>(slots, t.batch);
  if (workspace_ints(c, FORK) == 0) {
    FB_CUDA(ctx, launch(fork_kernel, kTogether, kPlan, s, t));
    return 0;
  }
  FB_CUDA(ctx, launch(fork_stage_kernel, std::max<int64_t>(blocks_for(work), blocks_up_to(ctx, t.users_out != t.users ? blocks_for(t.pages) : 1)), kMove, s, t));
  FB_CUDA(ctx, launch(fork_apply_kernel, std::max<int64_t>(1, blocks_for(work)), kMove, s, t));
  return 0;
}

int frisk_b200_cache_grow(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, const frisk_b200_page_tables* tables, void* workspace, size_t workspace_bytes, void* stream) {
  PageTables t;
  const int rc = prepare(ctx, c, tables, FRISK_B200_PAGES_GROW, nullptr, workspace, workspace_bytes, &t);
  if (rc) return rc;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t slots = (int64_t)t.batch * t.width;
  const bool copies = t.users_out != t.users || t.table_out != t.table, together = copies && t.pages + slots <= kCopiedTogether;
  if (copies && !together) FB_CUDA(ctx, launch(copy_tables_kernel, blocks_up_to(ctx, blocks_for(std::max<int64_t>(t.pages, slots))), kMove, s, t));
  constexpr int kLists = (5 * GrowWork::kSmall + 1) * 4;
  static_assert(kLists + (kSearched + 1) * 4 + 256 <= 48 * 1024, "what any kernel may have");
  if (together) FB_CUDA(ctx, launch_with(grow_plan_kernel<true>, kTogether, kPlan, kLists, s, t));
  else FB_CUDA(ctx, launch_with(grow_plan_kernel<false>, 1, kPlan, kLists, s, t));
  const Held h = held_of(c);
  if (t.batch > 0 && t.width > 0)
    FB_CUDA(ctx, launch(grow_copy_kernel, (int64_t)t.batch * c->heads, kMove, s, t.ws, reinterpret_cast<uint4*>(h.part[0]), reinterpret_cast<uint4*>(h.part[1]), h.part[2],
                        h.part[3], c->heads, c->page, (int)(c->D * element(c) / 16)));
  return 0;
}

int frisk_b200_cache_compact(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, const frisk_b200_page_tables* tables, void* workspace, size_t workspace_bytes,
                             void* stream) {
  PageTables t;
  const int rc = prepare(ctx, c, tables, FRISK_B200_PAGES_COMPACT, nullptr, workspace, workspace_bytes, &t);
  if (rc) return rc;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FB_CUDA(ctx, launch(compact_plan_kernel, 1, kPlan, s, t));
  const Held h = held_of(c);
  const int64_t pieces = c->pages * (int64_t)(h.pieces[0] + h.pieces[1] + h.pieces[2] + h.pieces[3]) / 2;  // (no more than half of the pages move)
  FB_CUDA(ctx, launch(compact_move_kernel, blocks_up_to(ctx, blocks_for(std::max<int64_t>(pieces / kAhead, (int64_t)t.batch * t.width))), kMove, s, h, t));
  return 0;
}

int frisk_b200_cache_copy(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* from, const frisk_b200_cache_desc* into, const int32_t* source, const int32_t* target, int64_t count,
                          void* stream) {
  if (!ctx || !from || !into) return FRISK_B200_E_ARG;
  int rc = cache_validate(from);
  if (rc || (rc = cache_validate(into))) return rc;
  if (count < 0 || count > INT32_MAX) return FRISK_B200_E_CACHE_SHAPE;
  if (from->dtype != into->dtype) return FRISK_B200_E_CACHE_TYPE;
  if (from->page != into->page || from->heads != into->heads || from->D != into->D) return FRISK_B200_E_CACHE_SHAPE;
  if (count == 0) return 0;
  if (!source || !target) return FRISK_B200_E_ARG;
  if ((reinterpret_cast<uintptr_t>(source) | reinterpret_cast<uintptr_t>(target)) & 3u) return FRISK_B200_E_ALIGN;
  if ((rc = check_cache(from)) || (rc = check_cache(into))) return rc;
  const Held a = held_of(from), d = held_of(into);
  const int n = from->dtype == FRISK_B200_E4M3 ? 4 : 2;
  bool same = true;
  for (int i = 0; i < n; ++i) same = same && a.part[i] == d.part[i];
  if (!same)
    for (int i = 0; i < n; ++i)
      if (cache_overlaps(into, a.part[i], (size_t)from->pages * a.pieces[i] * 16)) return FRISK_B200_E_OVERLAP;
  if (parts_overlap(into) || cache_overlaps(into, source, (size_t)count * 4) || cache_overlaps(into, target, (size_t)count * 4)) return FRISK_B200_E_OVERLAP;
  FB_DEVICE(ctx);
  const int64_t pieces = count * (int64_t)(a.pieces[0] + a.pieces[1] + a.pieces[2] + a.pieces[3]);
  FB_CUDA(ctx, launch(copy_pages_kernel, blocks_up_to(ctx, blocks_for(pieces / kAhead + 1)), kMove, static_cast<cudaStream_t>(stream), a, d, source, target, count,
                      (int)from->pages, (int)into->pages, ctx->d_status));
  return 0;
}

int frisk_b200_cache_keep(frisk_b200_ctx* ctx, const frisk_b200_cache_desc* c, const int32_t* kept, int64_t kept_stride, int32_t kept_width, const int32_t* counts,
                          int32_t* lengths_out, void* stream) {
  if (!ctx) return FRISK_B200_E_ARG;
  int rc = cache_validate(c);
  if (rc) return rc;
  if (kept_width < 0 || (c->batch > 1 && kept_stride < kept_width)) return FRISK_B200_E_CACHE_SHAPE;
  if (c->batch == 0) return 0;
  if ((rc = check_cache(c))) return rc;
  const size_t batch = (size_t)c->batch * 4;
  const Range all[] = {
      {c->lengths, batch, false, nullptr},
      {c->starts, batch + 4, false, nullptr},
      {c->table, table_bytes(c->batch, c->table_width, c->table_stride), false, nullptr},
      {kept, table_bytes(c->batch, kept_width, kept_stride), false, nullptr},
      {counts, batch, false, nullptr},
      {lengths_out, batch, true, c->lengths},
  };
  if ((rc = check_ranges(all, (int)(sizeof(all) / sizeof(all[0]))))) return rc;
  if (parts_overlap(c)) return FRISK_B200_E_OVERLAP;
  for (const Range& r : all)
    if (r.n && cache_overlaps(c, r.p, r.n)) return FRISK_B200_E_OVERLAP;
  FB_DEVICE(ctx);
  const Held h = held_of(c);
  KeepParams p{};
  p.t = cache_tables(c);
  p.kept = kept;
  p.counts = counts;
  p.kept_stride = kept_stride;
  p.kept_width = kept_width;
  p.lengths_out = lengths_out;
  p.k = reinterpret_cast<uint4*>(h.part[0]);
  p.v = reinterpret_cast<uint4*>(h.part[1]);
  p.ek = h.part[2];
  p.ev = h.part[3];
  p.row = (int)(c->D * element(c) / 16);
  p.status = ctx->d_status;
  FB_CUDA(ctx, launch(keep_kernel, c->batch, kMove, static_cast<cudaStream_t>(stream), p));
  return 0;
}

}  // extern "C"
