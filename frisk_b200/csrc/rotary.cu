// Rotary positions on the queries and keys of a batch of tokens, in one launch, and the gradients.
//
//   (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),   t = position * frequency of the pair
//
// Pairs are (i, i + dim/2) or, interleaved, (2i, 2i + 1) of the first `dim` elements of a head; the others pass.  The map is linear,
// so its backward is the transposed rotation: the same with -sin.
//
// t grows to 10^6 and more, where 32 bits keep no digit of a turn behind the point that matters: the product and the reduction to one
// turn are made in 64 bits, then sine and cosine of at most half a turn in 32.  A block does this once for every (token, pair) and
// uses it for all heads of queries and keys, whose products are rounded once.
//
// Bound by HBM: every element is read and written once, 16 bytes a thread and access where addresses and sizes allow, else one
// element.  A block takes the tokens whose angles make about one a thread, or a single one where that leaves SMs idle.
#include <algorithm>

#include "common.cuh"
#include "ptx.cuh"

namespace fb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;
constexpr int kAhead = 4;  // units a thread has in flight

struct Part {  // queries or keys
  const void* in;
  void* out;
  int64_t in_row, in_head, out_row, out_head;
  int heads;
};
struct RotaryParams {
  Part part[2];
  const void* positions;
  const double* frequencies;
  int64_t rows;
  int D, half, tokens;  // half = dim / 2; tokens a block
  int positions64;
  float amplitude, sign;
};

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ float to(float x) { return x; }
  static __device__ float from(float x) { return x; }
};
template <> struct Elem<__half> {
  static __device__ float to(__half x) { return __half2float(x); }
  static __device__ __half from(float x) { return __float2half_rn(x); }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// V elements an access: 16 bytes, or 1 where something is not aligned to that
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 angles[];  // [tokens][half]
  using E = Elem<T>;
  const int64_t row0 = (int64_t)blockIdx.x * p.tokens;
  const int here = (int)min((int64_t)p.tokens, p.rows - row0);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int e = threadIdx.x; e < here * p.half; e += kThreads) {
    const int t = e / p.half, i = e - t * p.half;
    const double pos = p.positions64 ? (double)static_cast<const long long*>(p.positions)[row0 + t]
                                     : (double)static_cast<const int*>(p.positions)[row0 + t];
    const double turns = pos * p.frequencies[i] * 0.15915494309189535;  // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    angles[e] = make_float2(c * p.amplitude, s * p.amplitude * p.sign);
  }
  __syncthreads();
  // units: the V-element groups of a head.  A pair of groups (half layout) or one group (interleaved) is rotated, others are copied.
  constexpr int kPairs = INTERLEAVED ? V / 2 : V;  // pairs a unit rotates
  const int n_rot = V == 1 && INTERLEAVED ? p.half : p.half / (kPairs > 0 ? kPairs : 1);
  const int n_pass = (p.D - 2 * p.half) / V;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Part& part = p.part[which];
    const bool copy = part.in != part.out;  // in place, what passes stays
    const int per_head = n_rot + (copy ? n_pass : 0);
    const int total = here * part.heads * per_head;
    if (total == 0) continue;
    // this thread's unit, head and token, and what a step of all threads adds to them
    int u = threadIdx.x % per_head, h = threadIdx.x / per_head % part.heads, t = threadIdx.x / per_head / part.heads;
    const int du = kThreads % per_head, dh = kThreads / per_head % part.heads, dt = kThreads / per_head / part.heads;
#pragma unroll 1
    for (int e0 = threadIdx.x; e0 < total; e0 += kThreads * kAhead) {
      Vec<T, V> x[kAhead], y[kAhead];
      int us[kAhead];
      T* out[kAhead];
      const float2* cs[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        us[n] = e0 + n * kThreads < total ? u : -1;
        if (us[n] >= 0) {
          const T* in = static_cast<const T*>(part.in) + (row0 + t) * part.in_row + h * part.in_head;
          out[n] = static_cast<T*>(part.out) + (row0 + t) * part.out_row + h * part.out_head;
          cs[n] = angles + t * p.half;
          const bool rotated = u < n_rot;
          if (V == 1 && INTERLEAVED && rotated) {
            x[n].v[0] = in[2 * u];
            y[n].v[0] = in[2 * u + 1];
          } else {
            x[n] = *reinterpret_cast<const Vec<T, V>*>(in + (rotated ? u * V : 2 * p.half + (u - n_rot) * V));
            if (!INTERLEAVED && rotated) y[n] = *reinterpret_cast<const Vec<T, V>*>(in + p.half + u * V);
          }
        }
        u += du;
        h += dh;
        t += dt;
        if (u >= per_head) {
          u -= per_head;
          ++h;
        }
        if (h >= part.heads) {
          h -= part.heads;
          ++t;
        }
      }
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int un = us[n];
        if (un < 0) continue;
        if (un >= n_rot) {
          *reinterpret_cast<Vec<T, V>*>(out[n] + 2 * p.half + (un - n_rot) * V) = x[n];
        } else if (INTERLEAVED && V > 1) {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            const float2 r = cs[n][un * (V / 2) + i];
            const float a = E::to(x[n].v[2 * i]), b = E::to(x[n].v[2 * i + 1]);
            x[n].v[2 * i] = E::from(a * r.x - b * r.y);
            x[n].v[2 * i + 1] = E::from(b * r.x + a * r.y);
          }
          *reinterpret_cast<Vec<T, V>*>(out[n] + un * V) = x[n];
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 r = cs[n][un * V + i];
            const float a = E::to(x[n].v[i]), b = E::to(y[n].v[i]);
            x[n].v[i] = E::from(a * r.x - b * r.y);
            y[n].v[i] = E::from(b * r.x + a * r.y);
          }
          *reinterpret_cast<Vec<T, V>*>(out[n] + (INTERLEAVED ? 2 * un : un * V)) = x[n];
          *reinterpret_cast<Vec<T, V>*>(out[n] + (INTERLEAVED ? 2 * un + 1 : p.half + un * V)) = y[n];
        }
      }
    }
  }
}

template <typename T, int V>
cudaError_t launch(const RotaryParams& p, bool interleaved, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait) itself
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((p.rows + p.tokens - 1) / p.tokens));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)p.tokens * p.half * sizeof(float2);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return interleaved ? cudaLaunchKernelEx(&cfg, rotary_kernel<T, V, true>, p)
                     : cudaLaunchKernelEx(&cfg, rotary_kernel<T, V, false>, p);
}

template <typename T>
cudaError_t launch_type(const RotaryParams& p, bool interleaved, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  // 16 bytes an access where every group of V elements begins on 16 bytes
  bool wide = p.half % (interleaved ? V / 2 : V) == 0 && (p.D - 2 * p.half) % V == 0;
  for (const Part& x : p.part) {
    if (x.heads == 0) continue;
    wide = wide && ((reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out)) & 15u) == 0 &&
           ((x.in_row | x.out_row) % V == 0) && (x.heads == 1 || (x.in_head | x.out_head) % V == 0);
  }
  return wide ? launch<T, V>(p, interleaved, s) : launch<T, 1>(p, interleaved, s);
}

// bytes a tensor of packed rows spans
size_t span(const frisk_b200_packed& x, int64_t rows, int heads, int D, size_t es) {
  return (size_t)((rows - 1) * x.row_stride + (heads - 1) * x.head_stride + D) * es;
}
// Two tensors that share a buffer of rows, each with its columns of every row: the same row pitch, and the ranges of a row apart.
bool apart(const frisk_b200_packed& a, int a_heads, const frisk_b200_packed& b, int b_heads, int64_t rows, int D, size_t es) {
  if (!ranges_overlap(a.ptr, span(a, rows, a_heads, D, es), b.ptr, span(b, rows, b_heads, D, es))) return true;
  if (a.row_stride != b.row_stride || rows < 2) return false;
  const int64_t pitch = a.row_stride * (int64_t)es;
  const int64_t a_len = ((a_heads - 1) * a.head_stride + D) * (int64_t)es, b_len = ((b_heads - 1) * b.head_stride + D) * (int64_t)es;
  if (pitch <= 0 || a_len > pitch || b_len > pitch) return false;
  const int64_t delta = (int64_t)(reinterpret_cast<intptr_t>(b.ptr) - reinterpret_cast<intptr_t>(a.ptr));
  const int64_t at = ((delta % pitch) + pitch) % pitch;  // where b's range begins in a's rows
  return at >= a_len && at + b_len <= pitch;
}
bool same(const frisk_b200_packed& a, const frisk_b200_packed& b) {
  return a.ptr == b.ptr && a.row_stride == b.row_stride && a.head_stride == b.head_stride;
}

}  // namespace
}  // namespace fb

using namespace fb;

extern "C" int frisk_b200_rotary(frisk_b200_ctx* ctx, const frisk_b200_rotary_desc* d, const void* positions,
                                 const double* frequencies, const frisk_b200_packed* q, const frisk_b200_packed* k,
                                 const frisk_b200_packed* q_out, const frisk_b200_packed* k_out, void* stream) {
  if (!ctx || !d || !q || !q_out) return FRISK_B200_E_ARG;
  if (!dtype_ok(d->dtype)) return FRISK_B200_E_CACHE_TYPE;
  if (d->rows < 0 || d->rows > INT32_MAX || d->heads_q < 1 || d->heads_k < 0 || d->D < 1 || d->D > 1024 || d->dim < 2 || d->dim % 2 ||
      d->dim > d->D || d->heads_q > 65536 || d->heads_k > 65536)
    return FRISK_B200_E_CACHE_SHAPE;
  if (d->rows == 0) return 0;
  if (!positions || !frequencies || !q->ptr || !q_out->ptr) return FRISK_B200_E_ARG;
  if (d->heads_k && (!k || !k_out || !k->ptr || !k_out->ptr)) return FRISK_B200_E_ARG;
  const size_t es = dtype_size(d->dtype);
  const frisk_b200_packed *in[2] = {q, k}, *out[2] = {q_out, k_out};
  const int heads[2] = {d->heads_q, d->heads_k}, n = d->heads_k ? 2 : 1;
  for (int i = 0; i < n; ++i)
    for (const frisk_b200_packed* x : {in[i], out[i]}) {
      if (x->row_stride < 0 || x->head_stride < 0) return FRISK_B200_E_CACHE_SHAPE;
      if (reinterpret_cast<uintptr_t>(x->ptr) % es) return FRISK_B200_E_ALIGN;
    }
  for (int i = 0; i < n; ++i) {
    // what is written: rows and heads apart from one another, from the other tensor's, and from every input but its own
    const frisk_b200_packed& o = *out[i];
    const int64_t row_len = (heads[i] - 1) * o.head_stride + d->D;
    if ((heads[i] > 1 && o.head_stride < d->D) || (d->rows > 1 && o.row_stride < row_len)) return FRISK_B200_E_CACHE_SHAPE;
    if (ranges_overlap(o.ptr, span(o, d->rows, heads[i], d->D, es), positions, (size_t)d->rows * (d->positions64 ? 8 : 4)) ||
        ranges_overlap(o.ptr, span(o, d->rows, heads[i], d->D, es), frequencies, (size_t)d->dim / 2 * 8))
      return FRISK_B200_E_OVERLAP;
    for (int j = 0; j < n; ++j) {
      if (!(i == j && same(o, *in[i])) && !apart(o, heads[i], *in[j], heads[j], d->rows, d->D, es)) return FRISK_B200_E_OVERLAP;
      if (i < j && !apart(o, heads[i], *out[j], heads[j], d->rows, d->D, es)) return FRISK_B200_E_OVERLAP;
    }
  }
  RotaryParams p{};
  for (int i = 0; i < n; ++i)
    p.part[i] = Part{in[i]->ptr, out[i]->ptr, in[i]->row_stride, in[i]->head_stride, out[i]->row_stride, out[i]->head_stride, heads[i]};
  p.positions = positions;
  p.frequencies = frequencies;
  p.rows = d->rows;
  p.D = d->D;
  p.half = d->dim / 2;
  p.positions64 = d->positions64;
  p.amplitude = d->amplitude;
  p.sign = d->inverse ? -1.f : 1.f;
  p.tokens = std::max(1, std::min(kMaxTokens, kThreads / p.half));
  while (p.tokens > 1 && d->rows / p.tokens < 4 * ctx->num_sms) p.tokens /= 2;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FB_CUDA(ctx, d->dtype == FRISK_B200_F32   ? launch_type<float>(p, d->interleaved != 0, s)
               : d->dtype == FRISK_B200_F16 ? launch_type<__half>(p, d->interleaved != 0, s)
                                            : launch_type<__nv_bfloat16>(p, d->interleaved != 0, s));
  return 0;
}
