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
// A block takes a few tokens and forms the cosines and sines of their pairs once, in shared memory.  A thread takes
// one piece of a token's heads (a 16-byte vector, with halves two; or one pair), keeps that piece's angles in
// registers and turns the piece in every head of queries and keys, or in every so manieth,
// asking for kBatch heads at a time and for the first ones before the angles are formed.  Bound by HBM (each element
// read and written once): the queries and keys of 32760 tokens, 12 heads of 128 in bf16, take 72 us (5.6 TB/s; a copy
// of as many bytes runs at 5.5), with halves 68.  Small blocks, so that many are at different stages on an SM: 256
// threads and 8 heads at a time took 100 us, and items of (token, head, vector) found by division 89.
#include <algorithm>
#include <type_traits>

#include "elem.cuh"
#include "kernels.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace ds {
namespace {

constexpr int kThreads = 64, kBatch = 3;

__device__ __forceinline__ double position(const RopeAxesArgs& a, int64_t row, int axis) {
  const int64_t i = (row < a.pos_rows ? row : row % a.pos_rows) * a.pos_stride + axis * a.axis_stride;
  switch (a.pos_type) {
    case 0: return static_cast<double>(reinterpret_cast<const long long*>(a.pos)[i]);
    case 1: return static_cast<double>(reinterpret_cast<const int*>(a.pos)[i]);
    case 2: return static_cast<double>(reinterpret_cast<const float*>(a.pos)[i]);
    default: return reinterpret_cast<const double*>(a.pos)[i];
  }
}

struct Shape {
  int pieces;         // of a head
  int lanes;          // threads that share a head's pieces: all of them, at most kThreads
  int spread;         // threads that share a piece's heads
  int tokens;         // of a block
  FastDiv by_lane, by_spread, by_pair;
};

// cosine and sine of one pair of a token
__device__ __forceinline__ float2 angle(const RopeAxesArgs& a, int64_t row, int pair) {
  double turns = position(a, row, a.axis[pair]) * a.turns[pair];
  turns -= rint(turns);
  float s, c;
  sincospif(2.f * static_cast<float>(turns), &s, &c);
  return make_float2(c, a.inverse ? -s : s);
}

// V elements as they are stored: a 16-byte vector, or one element
template <typename T, int V>
struct Piece {
  typename std::conditional<V == 1, T, uint4>::type u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const decltype(u)*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<decltype(u)*>(p) = u; }
};

// V = 1: a piece is one pair.  V > 1: vectors of V elements, with halves (kHalf) the
// vectors of both elements of V pairs.  Pieces behind the pairs are copied.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a, Shape sh) {
  extern __shared__ float2 angles[];           // [tokens][pairs]
  constexpr bool kTwo = kHalf || V == 1;       // two loads a piece
  constexpr int kPairs = kTwo ? V : V / 2;     // pairs of a piece
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * sh.tokens;
  const int tokens = static_cast<int>(a.rows - row0 < sh.tokens ? a.rows - row0 : sh.tokens);
  const int group = sh.by_lane.div(threadIdx.x), tok = sh.by_spread.div(group);
  const int hg = group - tok * sh.spread;
  const bool here = tok < tokens;
  const int64_t row = row0 + (here ? tok : 0);
  const int heads0 = a.t[0].heads, heads = heads0 + a.t[1].heads;
  const T* x0 = reinterpret_cast<const T*>(a.t[0].x) + row * a.t[0].x_stride;
  const T* x1 = reinterpret_cast<const T*>(a.t[1].x) + row * a.t[1].x_stride;
  T* y0 = reinterpret_cast<T*>(a.t[0].y) + row * a.t[0].y_stride;
  T* y1 = reinterpret_cast<T*>(a.t[1].y) + row * a.t[1].y_stride;
  const int turned = a.pairs / kPairs;         // pieces that turn
  bool ready = false;
  for (int p0 = 0; p0 < sh.pieces; p0 += sh.lanes) {
    const int p = p0 + threadIdx.x - group * sh.lanes;
    const bool mine = here && p < sh.pieces, copy = p >= turned;
    // first and second load of the piece, from the head's first element on
    const int e0 = copy ? 2 * a.pairs + (p - turned) * V : (V == 1 && !kHalf ? 2 * p : p * V);
    const int e1 = kHalf ? e0 + a.pairs : e0 + 1;
    float2 cs[kPairs];
    for (int h = hg; h < heads || !ready; h += sh.spread * kBatch) {
      Piece<T, V> u[kBatch], w[kTwo ? kBatch : 1];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int hh = h + b * sh.spread;
        if (mine && hh < heads) {
          const T* x = hh < heads0 ? x0 + hh * a.head_dim : x1 + (hh - heads0) * a.head_dim;
          u[b].load(x + e0);
          if (kTwo && !copy) w[b].load(x + e1);
        }
      }
      if (!ready) {
        for (int i = threadIdx.x; i < tokens * a.pairs; i += blockDim.x) {
          const int k = sh.by_pair.div(i);
          angles[i] = angle(a, row0 + k, i - k * a.pairs);
        }
        __syncthreads();
        ready = true;
      }
      if (h == hg && mine && !copy) {
#pragma unroll
        for (int e = 0; e < kPairs; ++e) cs[e] = angles[tok * a.pairs + p * kPairs + e];
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int hh = h + b * sh.spread;
        if (mine && hh < heads) {
          T* to = hh < heads0 ? y0 + hh * a.head_dim : y1 + (hh - heads0) * a.head_dim;
          if (!copy) {
            if constexpr (V == 1) {
              const float f = to_float(u[b].u), g = to_float(w[b].u);
              u[b].u = from_float<T>(f * cs[0].x - g * cs[0].y);
              w[b].u = from_float<T>(f * cs[0].y + g * cs[0].x);
            } else if constexpr (kHalf) {
              float f[V], g[V];
              load_vec<T, V>(reinterpret_cast<const T*>(&u[b].u), f);
              load_vec<T, V>(reinterpret_cast<const T*>(&w[b].u), g);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float q = f[e] * cs[e].x - g[e] * cs[e].y;
                g[e] = f[e] * cs[e].y + g[e] * cs[e].x;
                f[e] = q;
              }
              store_vec<T, V>(reinterpret_cast<T*>(&u[b].u), f);
              store_vec<T, V>(reinterpret_cast<T*>(&w[b].u), g);
            } else {
              float f[V];
              load_vec<T, V>(reinterpret_cast<const T*>(&u[b].u), f);
#pragma unroll
              for (int e = 0; e < V; e += 2) {
                const float q = f[e] * cs[e / 2].x - f[e + 1] * cs[e / 2].y;
                f[e + 1] = f[e] * cs[e / 2].y + f[e + 1] * cs[e / 2].x;
                f[e] = q;
              }
              store_vec<T, V>(reinterpret_cast<T*>(&u[b].u), f);
            }
          }
          u[b].store(to + e0);
          if (kTwo && !copy) w[b].store(to + e1);
        }
      }
    }
  }
}

template <typename T, int V>
void launch_pieces(const RopeAxesArgs& a, cudaStream_t s) {
  Shape sh;
  const int turned = V == 1 ? a.pairs : (a.half ? a.pairs / V : 2 * a.pairs / V);
  sh.pieces = turned + (a.head_dim - 2 * a.pairs) / V;
  sh.lanes = std::min(sh.pieces, kThreads);
  const int64_t heads = a.t[0].heads + a.t[1].heads;
  // a thread takes the heads of one batch of loads, fewer while that leaves SMs with less than 512 threads, more where
  // a block's threads do not allow it
  int64_t spread = std::max((heads + kBatch - 1) / kBatch, 512 * device_sm_count() / (a.rows * sh.lanes));
  spread = std::max<int64_t>(1, std::min<int64_t>({spread, heads, kThreads / sh.lanes}));
  sh.spread = static_cast<int>(spread);
  sh.tokens = std::max(1, kThreads / (sh.lanes * sh.spread));
  sh.by_lane = FastDiv(sh.lanes);
  sh.by_spread = FastDiv(sh.spread);
  sh.by_pair = FastDiv(a.pairs);
  const int64_t blocks = (a.rows + sh.tokens - 1) / sh.tokens;
  if (blocks > 0x7fffffff) throw std::runtime_error("rope_axes: too many rows");
  const int threads = (sh.tokens * sh.lanes * sh.spread + 31) / 32 * 32;
  const size_t smem = static_cast<size_t>(sh.tokens) * a.pairs * sizeof(float2);
  auto kern = a.half ? rope_axes_kernel<T, V, true> : rope_axes_kernel<T, V, false>;
  kern<<<static_cast<unsigned>(blocks), threads, smem, s>>>(a, sh);
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
  if (vec) launch_pieces<T, V>(a, s);
  else launch_pieces<T, 1>(a, s);
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
