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
// A cluster of eight CTAs has a sequence, its CTAs neighbouring parts of the vocabulary, their warps neighbouring parts of those.  A tested child
// costs two single values, fetched for all nodes at once; whole rows are read only for a rejection (with a draft) and for the last sum.
// The sums of a part stay in shared memory, so the token is found by descending: CTA, warp, 256 values, lane.  Bound by
// HBM where there are many sequences, else by the chain starts -> tokens -> values -> row -> exchange of sums.
#include <cfloat>

#include "cache_common.cuh"

namespace fb {
namespace {

constexpr int kCluster = 8;
constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr int kLane = 8, kStep = 32 * kLane;  // values a lane and a warp look at in a step
constexpr int kMaxNodes = 1024;

struct VerifyParams {
  const void* tokens;
  const int *parents, *starts;
  const void *target, *draft;
  int64_t target_stride, draft_stride;
  const float *accept, *sample;
  int *kept, *counts;
  void* next;
  int64_t rows;
  int tokens64, max_new, vocab;
  unsigned* status;
};

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// what a probability weighs: NaN and what is below zero nothing, an infinity the largest finite value
__device__ __forceinline__ float weight(float x) { return fminf(fmaxf(x, 0.f), FLT_MAX); }

// kLane values from `at` on, of which the first `n` are there
template <typename T>
__device__ __forceinline__ void load_lane(float (&x)[kLane], const T* at, int n) {
  if (n >= kLane && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
    uint4 w[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
    const T* v = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < kLane; ++i) x[i] = weight(to_float<T>(v[i]));
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) x[i] = i < n ? weight(to_float<T>(at[i])) : 0.f;
  }
}

__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double x) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(x) : "memory"); }

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kThreads) __cluster_dims__(kCluster, 1, 1) verify_kernel(const VerifyParams p) {
  extern __shared__ int nodes[];  // of every node: token, parent, weight there, the draft's, random number; masses or tokens taken off
  __shared__ double warp_sums[kWarps], cta_sums[2][kCluster];
  __shared__ int n_off;
  int *token = nodes, *parent = token + p.max_new;
  float *at_target = reinterpret_cast<float*>(parent + p.max_new), *at_draft = at_target + p.max_new, *random = at_draft + p.max_new;
  // (doubles: behind five arrays of 32 bits, rounded up)
  double* masses = reinterpret_cast<double*>(nodes + (5 * p.max_new + 1) / 2 * 2);
  int* off = reinterpret_cast<int*>(masses);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x / kCluster;
  const uint32_t rank = cluster_ctarank();
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
  cluster_sync_all();  // (and no CTA is written to before it runs)

  // this warp's part of the vocabulary: steps [step0, step1)
  const int steps = (p.vocab + kStep - 1) / kStep, each = (steps + kCluster * kWarps - 1) / (kCluster * kWarps);
  const int step0 = min(steps, ((int)rank * kWarps + warp) * each), step1 = min(steps, step0 + each);

  int node = 0, taken_off = 0;  // distributions taken off, at this node
  // the kLane weights of step s that are this lane's
  auto weights = [&](double (&w)[kLane], int s) {
    const int at = s * kStep + lane * kLane;
    float x[kLane];
    load_lane<T>(x, target + node * p.target_stride + at, p.vocab - at);
    if (DRAFT) {
      float q[kLane];
      if (taken_off) load_lane<T>(q, draft + node * p.draft_stride + at, p.vocab - at);
#pragma unroll
      for (int i = 0; i < kLane; ++i) w[i] = x[i];
      for (int j = 0; j < taken_off; ++j) {
        const double mass = masses[j];
#pragma unroll
        for (int i = 0; i < kLane; ++i) w[i] = fmax(__dsub_rn(w[i], __dmul_rn(mass, (double)q[i])), 0.0);
      }
    } else {
      for (int j = 0; j < taken_off; ++j) {
        const int d = off[j] - at;
#pragma unroll
        for (int i = 0; i < kLane; ++i)
          if (d == i) x[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kLane; ++i) w[i] = x[i];
    }
  };
  int turn = 0;
  // The sum of the weights; those of the warps and CTAs stay in warp_sums and cta_sums[turn ^ 1].  The whole cluster calls it.
  auto sum = [&]() {
    double mine = 0.0;
#pragma unroll 2
    for (int s = step0; s < step1; ++s) {
      double w[kLane];
      weights(w, s);
#pragma unroll
      for (int i = 0; i < kLane; ++i) mine += w[i];
    }
    mine = warp_sum(mine);
    __syncthreads();  // (the sums of the call before have been read)
    if (lane == 0) warp_sums[warp] = mine;
    __syncthreads();
    if (warp == 0) {
      double cta = warp_sum(lane < kWarps ? warp_sums[lane] : 0.0);
      if (lane < kCluster) st_cluster_f64(mapa_addr(smem_u32(&cta_sums[turn][rank]), lane), cta);
    }
    cluster_sync_all();
    double all = 0.0;
#pragma unroll
    for (int r = 0; r < kCluster; ++r) all += cta_sums[turn][r];
    turn ^= 1;  // (two sets: a CTA may be one call ahead)
    return all;
  };

  // The walk: every warp takes the same steps.
  int length = 1, at = 0;
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
      for (int j = 0; j < taken_off; ++j) w = fmax(__dsub_rn(w, __dmul_rn(masses[j], q)), 0.0);
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
      __syncthreads();  // (all have read the masses that are there; those of another node are overwritten)
      if (tid == 0) masses[taken_off] = mass;
      __syncthreads();
      ++taken_off;
      mass = whole = sum();
    } else {
      mass = fmax(mass - w, 0.0);
    }
  }
  if (!DRAFT) {  // all children of the node are off
    __syncthreads();
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
  } else {
    // The first part whose running sum passes the border; where rounding leaves none, the last one that weighs anything.
    const double border = (double)p.sample[b] * whole;
    const double* ctas = cta_sums[turn ^ 1];
    double before = 0.0, start = 0.0;
    int part = -1;
    bool passed = false;
    for (int r = 0; r < kCluster && !passed; ++r) {
      const double x = ctas[r];
      passed = before + x > border;
      if (passed || x > 0.0) {
        part = r;
        start = before;
      }
      before += x;
    }
    if (part == (int)rank) {
      int chosen = -1;
      double from = start;
      before = start;
      passed = false;
      for (int r = 0; r < kWarps && !passed; ++r) {
        const double x = warp_sums[r];
        passed = before + x > border;
        if (passed || x > 0.0) {
          chosen = r;
          from = before;
        }
        before += x;
      }
      if (chosen == warp) {
        int best = -1;
        bool done = false;
        for (int s = step0; s < step1 && !done; ++s) {
          double w[kLane], lane_sum = 0.0;
          weights(w, s);
#pragma unroll
          for (int i = 0; i < kLane; ++i) lane_sum += w[i];
          double upto = lane_sum;  // of the lanes up to this one
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
          }
          double run = from + (upto - lane_sum);
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
          if (hits) {
            const int who = __ffs(hits) - 1;
            best = s * kStep + who * kLane + __shfl_sync(0xffffffffu, here, who);
            done = true;
          } else if (some) {
            const int who = 31 - __clz(some);
            best = s * kStep + who * kLane + __shfl_sync(0xffffffffu, latest, who);
          }
          from += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) answer(best);
      }
    }
  }
  // (the last exchange of sums was behind a barrier of the cluster: nobody writes into a CTA that has gone)
}

template <typename T>
cudaError_t launch(const VerifyParams& p, int batch, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait) itself
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)batch * kCluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)((5 * p.max_new + 1) / 2 * 2) * 4 + (size_t)p.max_new * 8;  // (28 KB at most)
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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
  if (d->rows < 0 || d->rows > INT32_MAX || d->batch < 0 || d->batch > INT32_MAX / kCluster || d->max_new < 1 || d->max_new > kMaxNodes || d->vocab < 1 ||
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
