// Rotary positions on the queries and keys of a batch of tokens, in one launch, and the gradients.
//
//   (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),   t = position * frequency of the pair
//
// Pairs are (i, i + dim/2) or, interleaved, (2i, 2i + 1) of the first `dim` elements of a head; the others pass.  The map is linear,
// so its backward is the transposed rotation: the same with -sin.
//
// t grows to 10^6 and more, where 32 bits keep no digit of a turn behind the point that matters: the product and the reduction to one
// turn are made in 64 bits, then sine and cosine of at most half a turn in 32.  Each product is rounded once to its type.
//
// Bound by HBM: every element is read and written once, 16 bytes a lane and access where addresses and sizes allow, else one element.
// A warp has a token, or some of its heads where there are few tokens: it makes the token's angles once, one a lane, passes them
// through shared memory and uses them for all its heads of queries and keys; the first heads are on their way meanwhile, and no warp
// waits for another.
#include <algorithm>

#include "common.cuh"
#include "ptx.cuh"

namespace fb {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kAhead = 2;       // heads a lane has in flight

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
  int D, half;      // half = dim / 2
  int chunk, chunks;  // heads a warp, warps a token
  int positions64;
  float amplitude, sign;
};

// A unit's group: V elements, as 32-bit words where there are several (two 16-bit elements a word).
template <typename T, int V>
struct Group {
  static constexpr int kWords = V == 1 ? 1 : V * (int)sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* from) {
    if (V == 1) {
      w[0] = sizeof(T) == 4 ? *reinterpret_cast<const uint32_t*>(from) : *reinterpret_cast<const uint16_t*>(from);
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(from);
      w[0] = x.x; w[1 % kWords] = x.y; w[2 % kWords] = x.z; w[3 % kWords] = x.w;
    }
  }
  __device__ __forceinline__ void store(T* to) const {
    if (V == 1) {
      if (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(to) = w[0];
      else *reinterpret_cast<uint16_t*>(to) = (uint16_t)w[0];
    } else {
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1 % kWords], w[2 % kWords], w[3 % kWords]);
    }
  }
};
// the two elements of a word (of the first only, where V == 1: the second is zero), and back
template <typename T> __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(__uint_as_float(w), 0.f); }
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint32_t pack(float2 x) { return __float_as_uint(x.x); }
template <> __device__ __forceinline__ uint32_t pack<__half>(float2 x) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float2 x) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (rounded step by step as written, so that the kernels for aligned and other rows agree to the bit)
__device__ __forceinline__ float2 turned(float a, float b, float2 cs) {
  return make_float2(__fmaf_rn(a, cs.x, -__fmul_rn(b, cs.y)), __fmaf_rn(b, cs.x, __fmul_rn(a, cs.y)));
}

// V elements an access: 16 bytes, or 1 where something is not aligned to that
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 all_angles[];  // [warps][half]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float2* angles = all_angles + warp * p.half;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t task = (int64_t)blockIdx.x * kWarps + warp, row = task / p.chunks;
  if (row >= p.rows) return;
  {
    const double pos = p.positions64 ? (double)static_cast<const long long*>(p.positions)[row]
                                     : (double)static_cast<const int*>(p.positions)[row];
    for (int i = lane; i < p.half; i += 32) {
      const double turns = pos * p.frequencies[i] * 0.15915494309189535;  // 1 / (2 pi)
      float s, c;
      sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
      angles[i] = make_float2(c * p.amplitude, s * p.amplitude * p.sign);
    }
    __syncwarp();
  }
  // Units: the V-element groups of a head.  A pair of groups (half layout) or one group (interleaved) is rotated, others are copied.  A
  // lane has one unit of several heads.
  using G = Group<T, V>;
  constexpr bool kTwo = !(INTERLEAVED && V > 1);         // a unit has two groups
  constexpr int kPairs = kTwo ? V : V / 2;               // pairs a unit rotates
  auto rotate = [](G& x, G& y, const float2 (&cs)[kPairs]) {
    if (!kTwo) {
#pragma unroll
      for (int i = 0; i < G::kWords; ++i) {
        if (sizeof(T) == 2) {
          const float2 ab = unpack<T>(x.w[i]);
          x.w[i] = pack<T>(turned(ab.x, ab.y, cs[i % kPairs]));
        } else if (i % 2 == 0) {
          const float2 r = turned(__uint_as_float(x.w[i]), __uint_as_float(x.w[(i + 1) % G::kWords]), cs[i / 2 % kPairs]);
          x.w[i] = __float_as_uint(r.x);
          x.w[(i + 1) % G::kWords] = __float_as_uint(r.y);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < G::kWords; ++i) {
        constexpr int kEach = sizeof(T) == 2 && V > 1 ? 2 : 1;  // elements a word
        const float2 a = unpack<T>(x.w[i]), b = unpack<T>(y.w[i]);
        const float2 r = turned(a.x, b.x, cs[i * kEach]);
        const float2 q = kEach == 2 ? turned(a.y, b.y, cs[(i * kEach + 1) % kPairs]) : make_float2(0.f, 0.f);
        x.w[i] = pack<T>(make_float2(r.x, q.x));
        y.w[i] = pack<T>(make_float2(r.y, q.y));
      }
    }
  };
  const int n_rot = p.half / kPairs, n_units = n_rot + (p.D - 2 * p.half) / V;
  const int first = (int)(task - row * p.chunks) * p.chunk, last = first + p.chunk;  // its heads, queries before keys
  const int width = min(n_units, 32), slots = 32 / width, slot = lane / width;
  if (slot >= slots) return;
  for (int u = lane - slot * width; u < n_units; u += width) {
    const bool rotated = u < n_rot;
    const int at = !rotated ? 2 * p.half + (u - n_rot) * V : INTERLEAVED && V == 1 ? 2 * u : u * V;  // the unit's first element
    const int other = INTERLEAVED ? at + 1 : at + p.half;                                             // its second group
    float2 cs[kPairs];
    if (rotated) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) cs[i] = angles[u * kPairs + i];
    }
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      const Part& part = p.part[which];
      if (!rotated && part.in == part.out) continue;  // (in place, what passes stays)
      const int skip = which ? p.part[0].heads : 0, begin = max(first - skip, 0) + slot, end = min(last - skip, part.heads);
      const T* in = static_cast<const T*>(part.in) + row * part.in_row + begin * part.in_head + at;
      T* out = static_cast<T*>(part.out) + row * part.out_row + begin * part.out_head + at;
      const int64_t in_step = slots * part.in_head, out_step = slots * part.out_head;
      for (int h = begin; h < end; h += slots * kAhead) {
        G x[kAhead], y[kAhead];  // (all loads before the first store: the compiler cannot tell that they are apart)
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
          if (h + n * slots < end) {
            x[n].load(in + n * in_step);
            if (kTwo && rotated) y[n].load(in + n * in_step + (other - at));
          }
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
          if (h + n * slots >= end) break;
          if (rotated) {
            rotate(x[n], y[n], cs);
            if (kTwo) y[n].store(out + n * out_step + (other - at));
          }
          x[n].store(out + n * out_step);
        }
        in += kAhead * in_step;
        out += kAhead * out_step;
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
  cfg.gridDim = dim3((unsigned)((p.rows * p.chunks + kWarps - 1) / kWarps));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)kWarps * p.half * sizeof(float2);  // (32 KB at most)
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
  if (reinterpret_cast<uintptr_t>(positions) % (d->positions64 ? 8 : 4) || reinterpret_cast<uintptr_t>(frequencies) % 8) return FRISK_B200_E_ALIGN;
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
    if (!packed_distinct(o, d->rows, heads[i], d->D)) return FRISK_B200_E_CACHE_SHAPE;
    if (ranges_overlap(o.ptr, span(o, d->rows, heads[i], d->D, es), positions, (size_t)d->rows * (d->positions64 ? 8 : 4)) ||
        ranges_overlap(o.ptr, span(o, d->rows, heads[i], d->D, es), frequencies, (size_t)d->dim / 2 * 8))
      return FRISK_B200_E_OVERLAP;
    for (int j = 0; j < n; ++j) {
      if (!(i == j && same(o, *in[i])) && !packed_apart(o, heads[i], *in[j], heads[j], d->rows, d->D, es)) return FRISK_B200_E_OVERLAP;
      if (i < j && !packed_apart(o, heads[i], *out[j], heads[j], d->rows, d->D, es)) return FRISK_B200_E_OVERLAP;
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
  // all heads of a token to one warp, or fewer where that leaves SMs with less than 16 warps
  const int all = d->heads_q + d->heads_k;
  p.chunk = all;
  while (p.chunk > 2 && d->rows * ((all + p.chunk - 1) / p.chunk) < 16 * ctx->num_sms) p.chunk = (p.chunk + 1) / 2;
  p.chunks = (all + p.chunk - 1) / p.chunk;
  if (d->rows * (int64_t)p.chunks > (int64_t)INT32_MAX * kWarps) return FRISK_B200_E_TOO_LARGE;
  FB_DEVICE(ctx);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FB_CUDA(ctx, d->dtype == FRISK_B200_F32   ? launch_type<float>(p, d->interleaved != 0, s)
               : d->dtype == FRISK_B200_F16 ? launch_type<__half>(p, d->interleaved != 0, s)
                                            : launch_type<__nv_bfloat16>(p, d->interleaved != 0, s));
  return 0;
}
