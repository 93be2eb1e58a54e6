// Rotary positions with several axes (time, height, width) on the queries and keys of a token list
// (sm_100a).
//
// Pair i of every head turns by the angle pos[token, axis(i)] * theta^(-2 j / d_axis), j being the
// pair's place among its axis's d_axis / 2 pairs.  Pairs are neighbouring elements (2i, 2i + 1) or
// halves (i, i + pairs); what lies behind 2 * pairs passes through.  The angle is formed in units of a
// turn in fp64 and reduced to [-1/2, 1/2] before it becomes fp32, so far positions keep their phase:
// pos * f errs by 2^-53 of the turns made, 1e-7 of a turn at a billion turns.  The rotation is fp32,
// rounded once to the tensors' type.
//
// A block takes a few tokens: its threads form the cosines and sines of their pairs once, in shared
// memory, for all heads of queries and keys.  Bound by HBM (each element read and written once).
#include "elem.cuh"
#include "kernels.h"

namespace ds {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double position(const RopeAxesArgs& a, int64_t row, int axis) {
  const int64_t i = (row % a.pos_rows) * a.pos_stride + axis * a.axis_stride;
  switch (a.pos_type) {
    case 0: return static_cast<double>(reinterpret_cast<const long long*>(a.pos)[i]);
    case 1: return static_cast<double>(reinterpret_cast<const int*>(a.pos)[i]);
    case 2: return static_cast<double>(reinterpret_cast<const float*>(a.pos)[i]);
    default: return reinterpret_cast<const double*>(a.pos)[i];
  }
}

// V > 1: 16-byte vectors of V elements; V = 1: one pair (or one unrotated element) at a time.
template <typename T, int V, bool kHalf>
__device__ __forceinline__ void rotate(const RopeTensor& t, const float2* cs, int64_t row0, int tokens, int head_dim,
                                       int pairs) {
  const T* x = reinterpret_cast<const T*>(t.x);
  T* y = reinterpret_cast<T*>(t.y);
  if constexpr (V > 1) {
    // one item = one vector (halves: two, i and i + pairs); behind the pairs: copied vectors
    const int rot = kHalf ? pairs / V : 2 * pairs / V;
    const int per_head = rot + (head_dim - 2 * pairs) / V;
    const int per_token = per_head * t.heads;
    for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
      const int tok = i / per_token, r = i - tok * per_token;
      const int head = r / per_head, v = r - head * per_head;
      const int64_t at = (row0 + tok) * t.x_stride + head * head_dim;
      const int64_t to = (row0 + tok) * t.y_stride + head * head_dim;
      if (v >= rot) {
        const int c = 2 * pairs + (v - rot) * V;
        *reinterpret_cast<uint4*>(y + to + c) = *reinterpret_cast<const uint4*>(x + at + c);
      } else if constexpr (kHalf) {
        float f[V], g[V];
        load_vec<T, V>(x + at + v * V, f);
        load_vec<T, V>(x + at + pairs + v * V, g);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 c = cs[tok * pairs + v * V + e];
          const float p = f[e] * c.x - g[e] * c.y;
          g[e] = f[e] * c.y + g[e] * c.x;
          f[e] = p;
        }
        store_vec<T, V>(y + to + v * V, f);
        store_vec<T, V>(y + to + pairs + v * V, g);
      } else {
        float f[V];
        load_vec<T, V>(x + at + v * V, f);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 c = cs[tok * pairs + (v * V + e) / 2];
          const float p = f[e] * c.x - f[e + 1] * c.y;
          f[e + 1] = f[e] * c.y + f[e + 1] * c.x;
          f[e] = p;
        }
        store_vec<T, V>(y + to + v * V, f);
      }
    }
  } else {
    const int per_head = head_dim - pairs;
    const int per_token = per_head * t.heads;
    for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
      const int tok = i / per_token, r = i - tok * per_token;
      const int head = r / per_head, v = r - head * per_head;
      const int64_t at = (row0 + tok) * t.x_stride + head * head_dim;
      const int64_t to = (row0 + tok) * t.y_stride + head * head_dim;
      if (v >= pairs) {
        y[to + pairs + v] = x[at + pairs + v];
      } else {
        const int i0 = kHalf ? v : 2 * v, i1 = kHalf ? v + pairs : 2 * v + 1;
        const float f = to_float(x[at + i0]), g = to_float(x[at + i1]);
        const float2 c = cs[tok * pairs + v];
        y[to + i0] = from_float<T>(f * c.x - g * c.y);
        y[to + i1] = from_float<T>(f * c.y + g * c.x);
      }
    }
  }
}

template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a, int tokens) {
  extern __shared__ float2 cs[];  // [tokens][pairs]
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * tokens;
  const int n = static_cast<int>(a.rows - row0 < tokens ? a.rows - row0 : tokens);
  for (int i = threadIdx.x; i < n * a.pairs; i += kThreads) {
    const int tok = i / a.pairs, p = i - tok * a.pairs;
    double turns = position(a, row0 + tok, a.axis[p]) * a.turns[p];
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * static_cast<float>(turns), &s, &c);
    cs[i] = make_float2(c, a.inverse ? -s : s);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (a.t[k].heads > 0) rotate<T, V, kHalf>(a.t[k], cs, row0, n, a.head_dim, a.pairs);
}

template <typename T, int V>
void launch_vec(const RopeAxesArgs& a, cudaStream_t s) {
  const int tokens = a.pairs >= 128 ? 2 : 4;
  const int64_t blocks = (a.rows + tokens - 1) / tokens;
  if (blocks > 0x7fffffff) throw std::runtime_error("rope_axes: too many rows");
  const size_t smem = static_cast<size_t>(tokens) * a.pairs * sizeof(float2);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (a.half) rope_axes_kernel<T, V, true><<<grid, kThreads, smem, s>>>(a, tokens);
  else rope_axes_kernel<T, V, false><<<grid, kThreads, smem, s>>>(a, tokens);
}

template <typename T>
void launch_type(const RopeAxesArgs& a, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  // vectors need heads, rotated parts and rows that start on 16 bytes
  bool vec = a.head_dim % V == 0 && (a.half ? a.pairs % V == 0 : 2 * a.pairs % V == 0);
  for (const RopeTensor& t : a.t) {
    if (t.heads == 0) continue;
    vec = vec && reinterpret_cast<uintptr_t>(t.x) % 16 == 0 && reinterpret_cast<uintptr_t>(t.y) % 16 == 0 &&
          t.x_stride % V == 0 && t.y_stride % V == 0;
  }
  if (vec) launch_vec<T, V>(a, s);
  else launch_vec<T, 1>(a, s);
}

}  // namespace

void launch_rope_axes(const RopeAxesArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return;
  switch (a.type) {
    case kBF16: launch_type<__nv_bfloat16>(a, s); break;
    case kFP16: launch_type<__half>(a, s); break;
    case kFP32: launch_type<float>(a, s); break;
    default: throw std::runtime_error("rope_axes: unsupported type");
  }
}

}  // namespace ds
