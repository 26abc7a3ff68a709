// Which drafted tokens stand, and the token after them, from the target's probabilities and given random numbers.
//
// The nodes of a sequence are its packed rows: node 0 the token sampled last, node i > 0 a drafted one that follows node parent[i] < i.
// target[row] is the distribution of the token behind that row, draft[row] the one its children were drawn from.  From node 0 on, with
// weights w = target[node] and a mass S = 1, the children x of the node in their order:
//
//   x stands where w(x) > 0 and u S q(x) < w(x): the walk goes on from it, with its own w and S = 1
//   else the draft's distribution is taken off:  w <- max(w - S q, 0),  S <- the sum of w
//
// Where no child is left the next token is the first one at which the running sum of w passes u times its sum.  So tokens come out
// distributed as the target's, whatever the draft.  Without draft distributions q is a whole at x: w loses x, and S <- max(S - w(x), 0).
// No quotient is taken: weights stand for themselves over S.
//
// All in 64 bits: in 32 the sums over 10^5 tokens would move borders between tokens by more than many tokens have.
//
// A cluster of up to eight CTAs has a sequence, its warps neighbouring parts of the vocabulary.  A tested child costs two single values, fetched for
// all nodes at once; whole rows are read only for a rejection (with a draft) and for the last sum, and come out of the L2 when the node's next child is
// rejected.  The parts' sums go to all CTAs, so that each decides by itself, and the token is found by descending: the warp's part, an eighth of it,
// 256 values, a lane.
//
// Bound by HBM where there are many sequences (64 chains of 6 tokens over 128000 fp32 values: 21 us, 49 MB read), else by the chain starts -> tokens ->
// values -> row -> sums -> row (one chain over 32000: 6 us with the launch) and, where much is rejected, by conversions to and products in 64 bits (16
// trees of 24 over 50001 bf16 values: 19 to 29 us, some 3 a rejected child).  Weights are not kept: the j-th child of one node that is rejected takes j products and differences of every
// entry of the row, so m of them take some m^2 / 2 (16 such nodes over 50001: 2 children 13 us, 8 58, 32 535, 128 7400; without a draft they take none).
#include <cfloat>

#include "cache_common.cuh"

namespace fb {
namespace {

constexpr int kMostCtas = 8;  // of a cluster
constexpr int kWarps = 8, kThreads = 32 * kWarps, kMostParts = kMostCtas * kWarps;
constexpr int kAhead = 4;  // steps a warp has in flight
constexpr int kLane = 8, kStep = 32 * kLane;  // values a lane and a warp look at in a step
constexpr int kMaxNodes = 1024;
enum : unsigned { ST_VERIFY = 0x315 };  // a wait

struct VerifyParams {
  const void* tokens;
  const int *parents, *starts;
  const void *target, *draft;
  int64_t target_stride, draft_stride;
  const float *accept, *sample;
  int *kept, *counts;
  void* next;
  int64_t rows;
  int tokens64, max_new, vocab, ctas;
  unsigned* status;
};

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// what a probability weighs: NaN and what is below zero nothing, an infinity the largest finite value
__device__ __forceinline__ float weight(float x) { return fminf(fmaxf(x, 0.f), FLT_MAX); }

// kLane values of a row, as they are
template <typename T>
struct Values {
  uint4 w[sizeof(T) / 2];
  // from an address on 16 bytes
  __device__ __forceinline__ void load(const T* at) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
  }
  // from index `at` of a row of n on: those before and behind the row are zero
  __device__ __forceinline__ void load_any(const T* row, int at, int n) {
    alignas(16) T v[kLane];
#pragma unroll
    for (int i = 0; i < kLane; ++i) v[i] = at + i >= 0 && at + i < n ? row[at + i] : T(0.f);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(v)[i];
  }
  __device__ __forceinline__ float operator[](int i) const { return weight(to_float<T>(reinterpret_cast<const T*>(w)[i])); }
};

// what is left of a weight w
__device__ __forceinline__ double less(double w, double mass, double q) {
  const double x = __dsub_rn(w, __dmul_rn(mass, q));
  return x > 0.0 ? x : 0.0;
}

// x to a CTA of the cluster, and its 8 bytes to a barrier there
__device__ __forceinline__ void send(uint32_t addr, double x, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(addr), "l"(__double_as_longlong(x)), "r"(bar) : "memory");
}
// A bounded wait of a whole warp for what the cluster sends.
__device__ __forceinline__ bool received(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}
__device__ __forceinline__ void wait_for(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, unsigned* status) {
  if (received(bar, parity)) return;
  const unsigned long long t0 = globaltimer();
  for (uint32_t spins = 1; !received(bar, parity); ++spins) {
    if (spins & 63u) continue;
    bool stop = *abort_flag != 0;
    if (!stop && globaltimer() - t0 > kWaitBudgetNs) {
      *abort_flag = 1;
      atomicCAS(status, 0u, ST_VERIFY);
      stop = true;
    }
    if (__any_sync(0xffffffffu, stop)) {
      const unsigned long long t1 = globaltimer();  // what is still in flight has time to land
      while (globaltimer() - t1 < 200000ull) __nanosleep(1000);
      return;
    }
  }
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) int nodes[];  // of every node: token, parent, weight there, the draft's, random number; then masses or tokens taken off
  __shared__ double part_sums[2][kMostParts], eighths[kWarps];
  __shared__ uint64_t arrived[2];  // all parts of a sum
  __shared__ uint32_t abort_word;
  __shared__ int n_off;
  int *token = nodes, *parent = token + p.max_new;
  float *at_target = reinterpret_cast<float*>(parent + p.max_new), *at_draft = at_target + p.max_new, *random = at_draft + p.max_new;
  // (doubles: behind five arrays of 32 bits, rounded up)
  double* masses = reinterpret_cast<double*>(nodes + (5 * p.max_new + 1) / 2 * 2);  // two sets, of one node with rejections and the next
  int* off = reinterpret_cast<int*>(masses);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x / p.ctas;
  const int rank = (int)cluster_ctarank();
  if (tid == 0) {
    mbar_init(&arrived[0], 1);
    mbar_init(&arrived[1], 1);
    abort_word = 0;
    mbar_fence_init();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int first = p.starts[b], last = p.starts[b + 1];
  const int64_t many = (int64_t)last - first;
  const bool ok = first >= 0 && many >= 0 && last <= p.rows && many <= p.max_new;
  const int n = ok ? (int)many : 0;
  int* kept = p.kept + (int64_t)b * p.max_new;
  if (n == 0) {  // (the whole cluster)
    if (rank == 0) {
      if (!ok && tid == 0) atomicCAS(p.status, 0u, cache::ST_CACHE_ROWS);
      for (int i = tid; i < p.max_new; i += kThreads) kept[i] = -1;
      if (tid == 0) {
        p.counts[b] = 0;
        if (p.tokens64) static_cast<int64_t*>(p.next)[b] = -1;
        else static_cast<int*>(p.next)[b] = -1;
      }
    }
    return;
  }
  const T* target = static_cast<const T*>(p.target) + first * p.target_stride;
  const T* draft = static_cast<const T*>(p.draft) + (DRAFT ? first * p.draft_stride : 0);
  for (int i = tid; i < n; i += kThreads) {
    const int64_t x = p.tokens64 ? static_cast<const int64_t*>(p.tokens)[first + i] : static_cast<const int*>(p.tokens)[first + i];
    const int up = p.parents ? p.parents[first + i] : i - 1;
    const bool there = i > 0 && up >= 0 && up < i && x >= 0 && x < p.vocab;
    token[i] = there ? (int)x : -1;
    parent[i] = there ? up : -1;  // (what is nobody's child is never tested)
    at_target[i] = there ? weight(to_float<T>(target[up * p.target_stride + x])) : 0.f;
    at_draft[i] = DRAFT && there ? weight(to_float<T>(draft[up * p.draft_stride + x])) : 1.f;
    random[i] = p.accept[first + i];
  }
  __syncwarp();
  cluster_sync_all();  // (and no CTA is written to before it runs)

  // Steps are cut where the row's addresses are multiples of 16, so a row may begin up to kLane - 1 values into the first.
  const int steps = (p.vocab + kLane - 1 + kStep - 1) / kStep, parts = p.ctas * kWarps, each = (steps + parts - 1) / parts;
  int node = 0, taken_off = 0;  // distributions taken off, at this node
  double* mine_off = masses;
  // the weights of a step, of the values x and q
  auto weights = [&](double (&w)[kLane], const Values<T>& x, const Values<T>& q, int at) {
#pragma unroll
    for (int i = 0; i < kLane; ++i) w[i] = x[i];
    if (DRAFT) {
      if (taken_off == 0) return;
      double d[kLane];
#pragma unroll
      for (int i = 0; i < kLane; ++i) d[i] = q[i];
#pragma unroll 1
      for (int j = 0; j < taken_off; ++j) {
        const double mass = mine_off[j];
#pragma unroll
        for (int i = 0; i < kLane; ++i) w[i] = less(w[i], mass, d[i]);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < taken_off; ++j) {
        const int d = off[j] - at;
        if (d >= 0 && d < kLane) {
#pragma unroll
          for (int i = 0; i < kLane; ++i)
            if (d == i) w[i] = 0.0;
        }
      }
    }
  };
  auto total_of = [](const double (&w)[kLane]) { return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])); };
  auto shift_of = [&]() { return (int)((reinterpret_cast<uintptr_t>(target + node * p.target_stride) & 15u) / sizeof(T)); };
  // the sum of a lane's weights in step s, and the weights
  auto one_step = [&](double (&w)[kLane], int s) {
    const int at = s * kStep + lane * kLane - shift_of();
    Values<T> x, q;
    x.load_any(target + node * p.target_stride, at, p.vocab);
    if (DRAFT && taken_off) q.load_any(draft + node * p.draft_stride, at, p.vocab);
    weights(w, x, q, at);
    return total_of(w);
  };
  // the sum of a lane's weights in steps [from, to)
  auto lane_sum = [&](int from, int to) {
    const T *row = target + node * p.target_stride, *others = DRAFT ? draft + node * p.draft_stride : row;
    const int shift = shift_of();
    // steps that lie in the row and begin on 16 bytes: kAhead at a time
    const bool even = !DRAFT || ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(others)) & 15u) == 0;
    const int whole0 = even ? max(from, shift ? 1 : 0) : to, whole1 = even ? min(to, (p.vocab + shift) / kStep) : to;
    double total = 0.0, w[kLane];
#pragma unroll 1
    for (int s0 = whole0; s0 < whole1; s0 += kAhead) {
      Values<T> x[kAhead], q[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s0 + u >= whole1) break;
        const int at = (s0 + u) * kStep + lane * kLane - shift;
        x[u].load(row + at);
        if (DRAFT && taken_off) q[u].load(others + at);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s0 + u >= whole1) break;
        weights(w, x[u], q[u], (s0 + u) * kStep + lane * kLane - shift);
        total += total_of(w);
      }
    }
#pragma unroll 1
    for (int s = from; s < to; ++s) {
      if (s == whole0 && whole0 < whole1) s = whole1 - 1;  // (done)
      else total += one_step(w, s);
    }
    return total;
  };
  const int step0 = min(steps, (rank * kWarps + warp) * each), step1 = min(steps, step0 + each);
  int turn = 0;
  uint32_t phases = 0;
  // The sum of the weights; the parts' stay in part_sums[turn ^ 1].  The whole cluster calls it.
  auto sum = [&]() {
    const double part = warp_sum(lane_sum(step0, step1));
    if (tid == 0) mbar_expect_tx(&arrived[turn], parts * 8);
    if (lane < p.ctas) send(mapa_addr(smem_u32(&part_sums[turn][rank * kWarps + warp]), lane), part, mapa_addr(smem_u32(&arrived[turn]), lane));
    __syncwarp();
    wait_for(&arrived[turn], phases >> turn & 1, &abort_word, p.status);
    phases ^= 1u << turn;
    double all = 0.0;
    for (int i = lane; i < parts; i += 32) all += part_sums[turn][i];
    all = warp_sum(all);
    turn ^= 1;  // (two sets: a warp may be one call ahead)
    return all;
  };

  // The walk: every warp takes the same steps.
  int length = 1, at = 0, set = 0;
  double mass = 1.0, whole = -1.0;  // whole: the sum of the weights as they are, if it is known
  if (rank == 0 && tid == 0) kept[0] = 0;
  while (true) {
    int child = n;  // the next one of this node
    for (int i = at + 1; i < n; i += 32) {
      const unsigned found = __ballot_sync(0xffffffffu, i + lane < n && parent[i + lane] == node);
      if (found) {
        child = i + __ffs(found) - 1;
        break;
      }
    }
    if (child == n) break;
    at = child;
    const double q = at_draft[child];
    double w = at_target[child];
    if (DRAFT) {
      for (int j = 0; j < taken_off; ++j) w = less(w, mine_off[j], q);
    } else {  // the same token again: nothing is left of it
      for (int i = node + 1; i < child; i += 32)
        if (__any_sync(0xffffffffu, i + lane < child && parent[i + lane] == node && token[i + lane] == token[child])) w = 0.0;
    }
    if (w > 0.0 && __dmul_rn(__dmul_rn((double)random[child], mass), q) < w) {
      node = child;
      if (rank == 0 && tid == 0) kept[length] = child;
      ++length;
      mass = 1.0;
      whole = -1.0;
      taken_off = 0;
    } else if (DRAFT) {
      // All warps write the same.  A warp may be ahead of others by less than one sum, so with a node's first rejection it may overwrite what
      // they still read of the node before, if there were not two sets.
      if (taken_off == 0) {
        mine_off = masses + set * p.max_new;
        set ^= 1;
      }
      __syncwarp();
      if (lane == 0) mine_off[taken_off] = mass;
      __syncwarp();
      ++taken_off;
      mass = whole = sum();
    } else {
      mass = fmax(mass - w, 0.0);
    }
  }
  if (!DRAFT) {  // all children of the node are off
    if (warp == 0) {
      int count = 0;
      for (int i = node + 1; i < n; i += 32) {
        const bool child = i + lane < n && parent[i + lane] == node;
        const unsigned found = __ballot_sync(0xffffffffu, child);
        if (child) off[count + __popc(found & ((1u << lane) - 1u))] = token[i + lane];
        count += __popc(found);
      }
      if (lane == 0) n_off = count;
    }
    __syncthreads();
    taken_off = n_off;
  }
  if (whole < 0.0) whole = sum();
  if (whole == 0.0 && taken_off) {  // nothing is left but by rounding: the target's own
    taken_off = 0;
    whole = sum();
  }
  if (rank == 0) {
    for (int i = length + tid; i < p.max_new; i += kThreads) kept[i] = -1;
    if (tid == 0) p.counts[b] = length;
  }
  auto answer = [&](int x) {
    if (p.tokens64) static_cast<int64_t*>(p.next)[b] = x;
    else static_cast<int*>(p.next)[b] = x;
  };
  if (whole == 0.0) {
    if (rank == 0 && tid == 0) answer(-1);
    return;
  }
  // The first part whose running sum passes the border; where rounding leaves none, the last one that weighs anything.
  const double border = (double)p.sample[b] * whole;
  double start = 0.0;  // the weights before the part
  auto pick = [&](const double* sums, int count) {  // (kMostParts / 32 a lane)
    constexpr int kEach = kMostParts / 32;
    double x[kEach], own = 0.0;
    int mine = -1;  // the lane's first that passes, or its last that weighs anything
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      x[i] = kEach * lane + i < count ? sums[kEach * lane + i] : 0.0;
      own += x[i];
    }
    double upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    double run = start + (upto - own), before = run;
    bool passed = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (!passed && x[i] > 0.0) {
        passed = run + x[i] > border;
        mine = i;
        before = run;
      }
      run += x[i];
    }
    const unsigned hits = __ballot_sync(0xffffffffu, passed), some = __ballot_sync(0xffffffffu, mine >= 0);
    const int who = hits ? __ffs(hits) - 1 : 31 - __clz(some);
    start = __shfl_sync(0xffffffffu, before, who);
    return kEach * who + __shfl_sync(0xffffffffu, mine, who);
  };
  const int part = pick(part_sums[turn ^ 1], parts);
  if (part / kWarps != rank) return;  // (nobody writes into a CTA that has gone: it has received all parts of the last sum)
  // its eighths, a warp each
  const int from = min(steps, part * each), to = min(steps, from + each), piece = (to - from + kWarps - 1) / kWarps;
  const int mine0 = min(to, from + warp * piece), mine1 = min(to, mine0 + piece);
  const double eighth = warp_sum(lane_sum(mine0, mine1));
  if (lane == 0) eighths[warp] = eighth;
  __syncthreads();
  if (pick(eighths, kWarps) != warp) return;
  int best = -1;
  for (int s = mine0; s < mine1; ++s) {
    double w[kLane];
    const double own = one_step(w, s);
    double upto = own;  // of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    double run = start + (upto - own);
    int here = -1, latest = -1;  // the first that passes; the last that weighs anything
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      run += w[i];
      if (w[i] > 0.0) {
        latest = i;
        if (here < 0 && run > border) here = i;
      }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, here >= 0), some = __ballot_sync(0xffffffffu, latest >= 0);
    if (hits || some) {
      const int who = hits ? __ffs(hits) - 1 : 31 - __clz(some);
      best = s * kStep + who * kLane - shift_of() + __shfl_sync(0xffffffffu, hits ? here : latest, who);
    }
    if (hits) break;
    start += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) answer(best);
}

template <typename T>
cudaError_t launch(VerifyParams p, int batch, cudaStream_t s) {
  // As many CTAs a sequence as run at once, two a SM (64 sequences, 128000 tokens: with four 23 us, with eight of half the registers
  // and one step in flight 30).  Sixteen warps a CTA where one runs a SM gave nothing (16 trees of 24 over 50001 tokens 23.7 us, with eight 23.1).
  p.ctas = kMostCtas;
  while (p.ctas > 1 && (int64_t)batch * p.ctas > 2 * kNumSMsDefault) p.ctas /= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait) itself
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)batch * p.ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)((5 * p.max_new + 1) / 2 * 2) * 4 + (size_t)p.max_new * 16;  // (36 KB at most)
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return p.draft ? cudaLaunchKernelEx(&cfg, verify_kernel<T, true>, p) : cudaLaunchKernelEx(&cfg, verify_kernel<T, false>, p);
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" int frisk_b200_draft_verify(frisk_b200_ctx* ctx, const frisk_b200_verify_desc* d, const void* tokens, const int32_t* parents, const int32_t* starts,
                                       const void* target, const void* draft, const float* accept, const float* sample, int32_t* kept, int32_t* counts,
                                       void* next, void* stream) {
  if (!ctx || !d) return FRISK_B200_E_ARG;
  if (!dtype_ok(d->dtype)) return FRISK_B200_E_CACHE_TYPE;
  if (d->rows < 0 || d->rows > INT32_MAX || d->batch < 0 || d->batch > INT32_MAX / kMostCtas || d->max_new < 1 || d->max_new > kMaxNodes || d->vocab < 1 ||
      d->vocab > INT32_MAX - 2 * kStep || (d->rows > 1 && (d->target_stride < 0 || d->draft_stride < 0)))
    return FRISK_B200_E_CACHE_SHAPE;
  if (d->batch == 0) return 0;
  if (!starts || !sample || !kept || !counts || !next || (d->rows > 0 && (!tokens || !target || !accept))) return FRISK_B200_E_ARG;
  const size_t es = dtype_size(d->dtype), ts = d->tokens64 ? 8 : 4, rows = (size_t)d->rows, batch = (size_t)d->batch;
  auto span = [&](int64_t stride) { return rows ? ((rows - 1) * (size_t)stride + (size_t)d->vocab) * es : 0; };
  struct Part {
    const void* p;
    size_t n, align;
  };
  const Part in[] = {{tokens, rows * ts, ts}, {parents, parents ? rows * 4 : 0, 4}, {starts, (batch + 1) * 4, 4}, {target, span(d->target_stride), es},
                     {draft, draft ? span(d->draft_stride) : 0, es}, {accept, rows * 4, 4}, {sample, batch * 4, 4}};
  const Part out[] = {{kept, batch * d->max_new * 4, 4}, {counts, batch * 4, 4}, {next, batch * ts, ts}};
  for (const Part& x : in)
    if (reinterpret_cast<uintptr_t>(x.p) % x.align) return FRISK_B200_E_ALIGN;
  for (int i = 0; i < 3; ++i) {
    if (reinterpret_cast<uintptr_t>(out[i].p) % out[i].align) return FRISK_B200_E_ALIGN;
    for (const Part& x : in)
      if (x.n && ranges_overlap(out[i].p, out[i].n, x.p, x.n)) return FRISK_B200_E_OVERLAP;
    for (int j = 0; j < i; ++j)
      if (ranges_overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return FRISK_B200_E_OVERLAP;
  }
  VerifyParams p{};
  p.tokens = tokens;
  p.parents = parents;
  p.starts = starts;
  p.target = target;
  p.draft = draft;
  p.target_stride = d->target_stride;
  p.draft_stride = d->draft_stride;
  p.accept = accept;
  p.sample = sample;
  p.kept = kept;
  p.counts = counts;
  p.next = next;
  p.rows = d->rows;
  p.tokens64 = d->tokens64;
  p.max_new = d->max_new;
  p.vocab = d->vocab;
  p.status = ctx->d_status;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FB_CUDA(ctx, d->dtype == FRISK_B200_F32   ? launch<float>(p, d->batch, s)
               : d->dtype == FRISK_B200_F16 ? launch<__half>(p, d->batch, s)
                                            : launch<__nv_bfloat16>(p, d->batch, s));
  return 0;
}
