// Root-mean-square norm with the residual's addition in front and an 8-bit output behind (sm_100a).
//
//   h = round_T(x + r)                 the new residual stream, stored in x's type T
//   y = h * rsqrt(mean(h^2) + eps) * w   in fp32, from the stored h
//   s = max(max|y| / 448, 1e-30)         one fp32 scale a row, 448 = the largest e4m3
//   q = e4m3(y / s)                      rounded to nearest even
//
// The sum over a row, the norm and the scale are fp32.  Two roundings to fewer bits: h, because the
// next layer reads the same stored stream, and q, which is the output.  A NaN or an infinity in a
// row makes its scale and all its q NaN (the maximum passes NaN on).  The factors come in another order than above, h w
// once for maximum and output, then rstd, then 1 / s: y / s errs by some 2^-22 of itself, so a code whose value lies
// that close to the border of two steps may be either.
//
// One pass over memory: a row stays in registers between its sum of squares, its maximum and its
// quantisation, so an element costs its own read(s), the stored h and one byte.  Bound by HBM: 32760 x 1536 in bf16
// with a residual takes 57 us in a graph (6.2 TB/s), 60 call by call (a copy of as many bytes: 63).  Without a residual
// instructions bound it, the weights' two conversions a row among them: 35 us (4.3 TB/s).  Rows that start off 16 bytes
// go in pieces of 4 bytes (1530 wide: 100 us) or single elements (1531: 142 us).  Measured and not kept: cutting such
// rows' vectors out of two aligned ones, stores put together across lanes (148 and 158 us call by call).
#include <cuda_fp8.h>

#include "elem.cuh"
#include "kernels.h"

namespace ds {
namespace {

constexpr float kE4M3Max = 448.f;
constexpr float kScaleMin = 1e-30f;

template <bool kWarp>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (!kWarp) {
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <bool kWarp>
__device__ __forceinline__ float row_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (!kWarp) {
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) red[32 + (threadIdx.x >> 5)] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < warps ? red[32 + (threadIdx.x & 31)] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}

template <int V>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&y)[V], float inv) {
  if constexpr (V == 1) {
    *p = __nv_cvt_float_to_fp8(y[0] * inv, __NV_SATFINITE, __NV_E4M3);
  } else {
    uint16_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      w[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * inv, y[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    if constexpr (V == 2)
      *reinterpret_cast<uint16_t*>(p) = w[0];
    else if constexpr (V == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | (uint32_t(w[1]) << 16), w[2] | (uint32_t(w[3]) << 16));
    else
      *reinterpret_cast<uint32_t*>(p) = w[0] | (uint32_t(w[1]) << 16);
  }
}

// V consecutive elements as they are stored: a 16-byte vector, or one element
template <typename T, int V>
struct Raw {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = u; }
  __device__ __forceinline__ void clear() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 t = unpack2(T(), w[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
      else w[i] = pack2(T(), f[2 * i], f[2 * i + 1]);
    }
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct Raw<T, 2> {  // 16-bit elements in rows that start on 4 bytes only
  uint32_t u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint32_t*>(p) = u; }
  __device__ __forceinline__ void clear() { u = 0; }
  __device__ __forceinline__ void get(float (&f)[2]) const {
    const float2 t = unpack2(T(), u);
    f[0] = t.x;
    f[1] = t.y;
  }
  __device__ __forceinline__ void set(const float (&f)[2]) { u = pack2(T(), f[0], f[1]); }
};
template <typename T>
struct Raw<T, 1> {
  T u;
  __device__ __forceinline__ void load(const T* p) { u = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = u; }
  __device__ __forceinline__ void clear() { u = from_float<T>(0.f); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_float(u); }
  __device__ __forceinline__ void set(const float (&f)[1]) { u = from_float<T>(f[0]); }
};

// A row in registers, as it is stored (floats would double them and halve the rows in flight): kN vectors of V
// elements a thread.  kWarp: a warp a row (no shared memory), else a block a row.
template <typename T, int V, int kN, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 128 : (kN == 8 ? 512 : 1024)) norm_quant_kernel(NormQuantArgs a) {
  __shared__ float red[64];
  const int64_t row = kWarp ? (static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)) : blockIdx.x;
  if (row >= a.rows) return;
  const int t = kWarp ? (threadIdx.x & 31) : threadIdx.x;
  const int step = kWarp ? 32 : blockDim.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  Raw<T, V> v[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int c = (i * step + t) * V;
    if (c < a.dim) v[i].load(x + c);
    else v[i].clear();
  }
  float ss = 0.f;
  if (a.residual != nullptr) {
    const T* r = reinterpret_cast<const T*>(a.residual) + row * a.r_stride;
    T* h = reinterpret_cast<T*>(a.h) + row * a.h_stride;
    Raw<T, V> w[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = (i * step + t) * V;
      if (c < a.dim) w[i].load(r + c);
      else w[i].clear();
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = (i * step + t) * V;
      float f[V], g[V];
      v[i].get(f);
      w[i].get(g);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] += g[e];
      v[i].set(f);
      if (c < a.dim) v[i].store(h + c);
    }
  }
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    float f[V];
    v[i].get(f);
#pragma unroll
    for (int e = 0; e < V; ++e) ss += f[e] * f[e];
  }
  const float rstd = rsqrtf(row_sum<kWarp>(ss, red) / static_cast<float>(a.dim) + a.eps);
  const T* w = reinterpret_cast<const T*>(a.weight);
  // h * w of vector i; formed twice, for the maximum and for the output
  auto weighted = [&](int i, int c, float (&f)[V]) {
    v[i].get(f);
    if (w != nullptr) {
      Raw<T, V> u;
      float g[V];
      u.load(w + c);
      u.get(g);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= g[e];
    }
  };
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int c = (i * step + t) * V;
    if (c < a.dim) {
      float f[V];
      weighted(i, c, f);
#pragma unroll
      for (int e = 0; e < V; ++e) top = max_nan(top, fabsf(f[e]));
    }
  }
  const float scale = max_nan(row_max<kWarp>(top, red) * rstd / kE4M3Max, kScaleMin);
  const float inv = 1.f / scale;
  uint8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int c = (i * step + t) * V;
    if (c < a.dim) {
      float f[V];
      weighted(i, c, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= rstd;
      store_e4m3<V>(q + c, f, inv);
    }
  }
  if (t == 0) a.scale[row * a.scale_stride] = scale;
}

// Rows too long for registers: a block a row, three passes (the later two read h, or x without a
// residual, mostly from L2).
template <typename T>
__global__ void __launch_bounds__(1024) norm_quant_long_kernel(NormQuantArgs a) {
  __shared__ float red[64];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  const T* w = reinterpret_cast<const T*>(a.weight);
  const T* r = reinterpret_cast<const T*>(a.residual) + (a.residual ? row * a.r_stride : 0);
  T* h = reinterpret_cast<T*>(a.h) + (a.residual ? row * a.h_stride : 0);
  float ss = 0.f;
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
    float f = to_float(x[c]);
    if (a.residual != nullptr) {
      const T s = from_float<T>(f + to_float(r[c]));
      h[c] = s;
      f = to_float(s);
    }
    ss += f * f;
  }
  const float rstd = rsqrtf(row_sum<false>(ss, red) / static_cast<float>(a.dim) + a.eps);
  const T* s = a.residual != nullptr ? h : x;  // each thread reads back what it wrote itself
  auto y = [&](int c) {
    const float f = to_float(s[c]) * rstd;
    return w != nullptr ? f * to_float(w[c]) : f;
  };
  float top = 0.f;
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x) top = max_nan(top, fabsf(y(c)));
  const float scale = max_nan(row_max<false>(top, red) / kE4M3Max, kScaleMin);
  const float inv = 1.f / scale;
  uint8_t* q = a.q + row * a.q_stride;
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x)
    q[c] = __nv_cvt_float_to_fp8(y(c) * inv, __NV_SATFINITE, __NV_E4M3);
  if (threadIdx.x == 0) a.scale[row * a.scale_stride] = scale;
}

template <typename T, int V>
void launch_rows(const NormQuantArgs& a, cudaStream_t s) {
  const int vecs = (a.dim + V - 1) / V;
  const bool many = a.rows >= 148 * 8;
  // many rows: a warp a row up to 8 vectors a lane, then a block a row with 4 vectors (8 short pieces) a thread, small
  // blocks of which several run on an SM: while one row waits for its sums others load.  20000 x 512 bf16 takes 21 us
  // against 24 with blocks, 6000 x 8192 64 us against 71 with 8 vectors a thread and 79 with one.  Few rows: a block a
  // row with as few vectors a thread as 1024 threads allow, since a row's latency counts
  if (many && vecs <= 32 * 8) {
    const int64_t blocks = (a.rows + 3) / 4;
    const dim3 grid(static_cast<unsigned>(blocks));
    const int n = (vecs + 31) / 32;
    if (n <= 1) norm_quant_kernel<T, V, 1, true><<<grid, 128, 0, s>>>(a);
    else if (n <= 2) norm_quant_kernel<T, V, 2, true><<<grid, 128, 0, s>>>(a);
    else if (n <= 4) norm_quant_kernel<T, V, 4, true><<<grid, 128, 0, s>>>(a);
    else if (n <= 6) norm_quant_kernel<T, V, 6, true><<<grid, 128, 0, s>>>(a);
    else norm_quant_kernel<T, V, 8, true><<<grid, 128, 0, s>>>(a);
    return;
  }
  const dim3 grid(static_cast<unsigned>(a.rows));
  const int n = many ? (V > 2 ? 4 : 8) : (vecs + 1023) / 1024;
  const int per = n <= 1 ? 1 : n <= 2 ? 2 : (n <= 4 || vecs > 512 * 8) ? 4 : 8;
  const int threads = ((vecs + per - 1) / per + 31) / 32 * 32;
  if (threads > (per == 8 ? 512 : 1024)) norm_quant_long_kernel<T><<<grid, 1024, 0, s>>>(a);
  else if (per == 1) norm_quant_kernel<T, V, 1, false><<<grid, threads, 0, s>>>(a);
  else if (per == 2) norm_quant_kernel<T, V, 2, false><<<grid, threads, 0, s>>>(a);
  else if (per == 4) norm_quant_kernel<T, V, 4, false><<<grid, threads, 0, s>>>(a);
  else if constexpr (V <= 2) norm_quant_kernel<T, V, 8, false><<<grid, threads, 0, s>>>(a);
}

bool aligned(const void* p, int64_t stride_bytes, int bytes) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride_bytes % bytes == 0);
}

template <typename T>
void launch_type(const NormQuantArgs& a, cudaStream_t s) {
  constexpr int V = kVec16<T>;
  const int64_t e = sizeof(T);
  // 16-byte vectors when every row of every operand starts on one (q: V bytes)
  const bool vec = a.dim % V == 0 && aligned(a.x, a.x_stride * e, 16) && aligned(a.residual, a.r_stride * e, 16) &&
                   aligned(a.h, a.h_stride * e, 16) && aligned(a.weight, 0, 16) && aligned(a.q, a.q_stride, V);
  if (vec) {
    launch_rows<T, V>(a, s);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (a.dim % 2 == 0 && aligned(a.x, a.x_stride * e, 4) && aligned(a.residual, a.r_stride * e, 4) &&
        aligned(a.h, a.h_stride * e, 4) && aligned(a.weight, 0, 4) && aligned(a.q, a.q_stride, 2)) {
      launch_rows<T, 2>(a, s);
      return;
    }
  }
  launch_rows<T, 1>(a, s);
}

}  // namespace

void launch_norm_quant(const NormQuantArgs& a, cudaStream_t s) {
  if (a.rows <= 0 || a.dim <= 0) return;
  if (a.rows > 0x7fffffff) throw std::runtime_error("rms_norm_quant: too many rows");
  switch (a.type) {
    case kBF16: launch_type<__nv_bfloat16>(a, s); break;
    case kFP16: launch_type<__half>(a, s); break;
    case kFP32: launch_type<float>(a, s); break;
    default: throw std::runtime_error("rms_norm_quant: unsupported type");
  }
}

}  // namespace ds
