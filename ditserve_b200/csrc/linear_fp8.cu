// Linear layer on 8-bit operands (sm_100a):
//
//   y[m, n] = epilogue(sx[m] * sw[n] * sum_k x[m, k] * w[n, k] + b[n])
//
// x and w are e4m3 with one fp32 scale a row (a token, an output channel); sums are fp32.
#include "elem.cuh"
#include "kernels.h"
#include "mma_sync.cuh"
#include "sm100.cuh"

namespace ds {
namespace {

// bias, activation, gate and residual of one output value; v is the scaled sum
template <typename T>
__device__ __forceinline__ float finish(const LinearFp8Args& a, float v, int m, int n, const float* gate_row) {
  if (a.bias != nullptr) v += to_float(reinterpret_cast<const T*>(a.bias)[n]);
  if (a.gelu) {
    if constexpr (sizeof(T) == 4) {
      // fp32 outputs take the full-precision form of gelu_tanh: x / (1 + exp(-2u))
      const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
      v = v / (1.f + expf(-2.f * u));
    } else {
      v = gelu_tanh(v);
    }
  }
  if (a.residual != nullptr) {
    if (gate_row != nullptr) v *= gate_row[n];
    v += to_float(reinterpret_cast<const T*>(a.residual)[static_cast<int64_t>(m) * a.ldr + n]);
  }
  return v;
}

__device__ __forceinline__ const float* gate_of(const LinearFp8Args& a, int m) {
  if (a.gate == nullptr) return nullptr;
  int b = a.row_batch != nullptr ? a.row_batch[m] : m / a.rows_per_batch;
  b = b < 0 ? 0 : (b >= a.batches ? a.batches - 1 : b);
  return a.gate + static_cast<int64_t>(b) * a.gate_stride;
}

// 16 bytes of a row at column k; bytes at or behind K read as zero and are not touched
__device__ __forceinline__ uint4 load16(const uint8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i >> 2] |= static_cast<uint32_t>(row[k + i]) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Few rows: a block takes 16 output channels and 8 * kM rows of x; its warps split K in chunks of 64
// and join their sums in shared memory.  The weights are the product's A operand straight from
// global memory, read once: bound by HBM.
constexpr int kRowWarps = 8;

template <typename T, int kM>
__global__ void __launch_bounds__(32 * kRowWarps) linear_rows_kernel(LinearFp8Args a) {
  __shared__ float part[kRowWarps][kM * 8][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (8 * kM);
  // rows behind the last are read as the last one and their sums dropped
  const uint8_t* w0 = a.w + static_cast<int64_t>(min(n0 + g, a.N - 1)) * a.ldw;
  const uint8_t* w1 = a.w + static_cast<int64_t>(min(n0 + g + 8, a.N - 1)) * a.ldw;
  float acc[kM][4] = {};
  for (int k = warp * 64 + t * 16; k - t * 16 < a.K; k += 64 * kRowWarps) {
    const uint4 u = load16(w0, k, a.K), v = load16(w1, k, a.K);
#pragma unroll
    for (int i = 0; i < kM; ++i) {
      const int m = min(m0 + i * 8 + g, a.M - 1);
      const uint4 b = load16(a.x + static_cast<int64_t>(m) * a.ldx, k, a.K);
      mma16832_e4m3(acc[i], u.x, v.x, u.y, v.y, b.x, b.y);
      mma16832_e4m3(acc[i], u.z, v.z, u.w, v.w, b.z, b.w);
    }
  }
#pragma unroll
  for (int i = 0; i < kM; ++i) {
    part[warp][i * 8 + 2 * t][g] = acc[i][0];
    part[warp][i * 8 + 2 * t + 1][g] = acc[i][1];
    part[warp][i * 8 + 2 * t][g + 8] = acc[i][2];
    part[warp][i * 8 + 2 * t + 1][g + 8] = acc[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kM * 8 * 16; i += 32 * kRowWarps) {
    const int m = m0 + i / 16, n = n0 + i % 16;
    if (m >= a.M || n >= a.N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) v += part[w][i / 16][i % 16];
    v *= a.sx[m * a.sx_stride] * a.sw[n * a.sw_stride];
    reinterpret_cast<T*>(a.y)[static_cast<int64_t>(m) * a.ldy + n] = from_float<T>(finish<T>(a, v, m, n, gate_of(a, m)));
  }
}

template <typename T>
void launch_type(const LinearFp8Args& a, cudaStream_t s) {
  const unsigned gx = (a.N + 15) / 16;
  if (a.M <= 8) {
    linear_rows_kernel<T, 1><<<dim3(gx, 1), 32 * kRowWarps, 0, s>>>(a);
  } else if (a.M <= 16) {
    linear_rows_kernel<T, 2><<<dim3(gx, 1), 32 * kRowWarps, 0, s>>>(a);
  } else {
    linear_rows_kernel<T, 4><<<dim3(gx, (a.M + 31) / 32), 32 * kRowWarps, 0, s>>>(a);
  }
}

}  // namespace

void launch_linear_fp8(const LinearFp8Args& a, cudaStream_t s) {
  if (a.M <= 0 || a.N <= 0) return;
  switch (a.out_type) {
    case kBF16: launch_type<__nv_bfloat16>(a, s); break;
    case kFP16: launch_type<__half>(a, s); break;
    case kFP32: launch_type<float>(a, s); break;
    default: throw std::runtime_error("linear_fp8: unsupported output type");
  }
}

}  // namespace ds
