// Attention of queries to an encoder's states of another length (sm_100a): padded, masked contexts.
//
//   o[b, i, h] = sum_j p_ij v[b, j, hk] / sum_j p_ij,  p_ij = exp(scale q_i k_j - max_j), j over the keys of
//   batch entry b that its valid length and its key mask leave; nothing left: o = 0 and lse = -inf.
//
// Scores, the running maximum and sum and the output's sums are fp32; p is rounded to the values'
// type for the second product, as its operand has to be.  Keys that are masked never reach a product
// with their value: their v is replaced by zero, so that NaN or infinities in padding do no harm.
#include <cooperative_groups.h>

#include "elem.cuh"
#include "kernels.h"
#include "mma_sync.cuh"
#include "sm100.cuh"

namespace ds {
namespace {

namespace cg = cooperative_groups;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int valid_keys(const CrossAttnArgs& a, int b) {
  if (a.kv_lens == nullptr) return a.seq_k;
  const int n = a.kv_lens[b];
  return n < 0 ? 0 : (n < a.seq_k ? n : a.seq_k);
}

__device__ __forceinline__ bool key_allowed(const CrossAttnArgs& a, int b, int j, int valid) {
  return j < valid && (a.key_mask == nullptr || a.key_mask[b * a.mask_row + j * a.mask_col] != 0);
}

// Few queries: a cluster of up to 8 blocks takes 16 query rows of one key head (a row is a query of
// one of the heads that share the key head) and splits the keys over its warps, 16 at a time; their
// maxima, sums and outputs are joined in shared memory, then over the cluster.  K and V go from global
// memory straight to the products' operands in 16-byte pieces: bound by latency, then HBM.
constexpr int kFewWarps = 4;

template <int D>
struct FewSmem {
  float o[16][D + 4];
  float m[16], l[16];
  float wm[kFewWarps][16], wl[kFewWarps][16];
};

template <typename T, int D>
__global__ void __launch_bounds__(32 * kFewWarps) cross_few_kernel(CrossAttnArgs a, int split) {
  __shared__ FewSmem<D> sm;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int part = blockIdx.x % split;  // the cluster's blocks are neighbours in x
  const int rows0 = blockIdx.x / split * 16;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int group = a.heads / a.heads_kv;
  const int rows = a.seq_q * group;
  const int valid = valid_keys(a, b);
  const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_batch;
  const T* k = reinterpret_cast<const T*>(a.k) + b * a.k_batch + hk * D;
  const T* v = reinterpret_cast<const T*>(a.v) + b * a.v_batch + hk * D;
  // query operands: lane (g, t) holds elements t * 8 .. t * 8 + 7 of every 32 of rows g and g + 8
  uint4 qa[D / 32], qb[D / 32];
  {
    const int r0 = min(rows0 + g, rows - 1), r1 = min(rows0 + g + 8, rows - 1);
    const T* q0 = q + (r0 / group) * a.q_row + (hk * group + r0 % group) * D + t * 8;
    const T* q1 = q + (r1 / group) * a.q_row + (hk * group + r1 % group) * D + t * 8;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      qa[s] = *reinterpret_cast<const uint4*>(q0 + s * 32);
      qb[s] = *reinterpret_cast<const uint4*>(q1 + s * 32);
    }
  }
  float o[D / 8][4] = {};
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const float sl2 = a.scale * kLog2e;
  const int stride = split * kFewWarps * 16;
  for (int j0 = (part * kFewWarps + warp) * 16; j0 < valid; j0 += stride) {
    float s[2][4] = {};
    // V of this lane's four keys (2t, 2t + 1, 2t + 8, 2t + 9), zero where masked
    uint4 vv[4][D / 64];
    bool ok[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + 2 * t + (i & 1) + (i >> 1) * 8;
      const bool on = key_allowed(a, b, j, valid);
      ok[i >> 1][i & 1] = on;
      const T* row = v + static_cast<int64_t>(min(j, valid - 1)) * a.v_row + g * 8;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        vv[i][c] = on ? *reinterpret_cast<const uint4*>(row + c * 64) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const T* row = k + static_cast<int64_t>(min(j0 + n * 8 + g, valid - 1)) * a.k_row + t * 8;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(row + i * 32);
        mma16816(T(), s[n], qa[i].x, qb[i].x, qa[i].y, qb[i].y, u.x, u.y);
        mma16816(T(), s[n], qa[i].z, qb[i].z, qa[i].w, qb[i].w, u.z, u.w);
      }
    }
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][e] = ok[n][e] ? s[n][e] * sl2 : -INFINITY;
        s[n][2 + e] = ok[n][e] ? s[n][2 + e] * sl2 : -INFINITY;
        x0 = max_nan(x0, s[n][e]);
        x1 = max_nan(x1, s[n][2 + e]);
      }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      x0 = max_nan(x0, __shfl_xor_sync(0xffffffffu, x0, d));
      x1 = max_nan(x1, __shfl_xor_sync(0xffffffffu, x1, d));
    }
    const float n0 = max_nan(m0, x0), n1 = max_nan(m1, x1);
    // nothing allowed so far: subtract zero, every p is 2^-inf = 0
    const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
    const float c0 = exp2f(m0 - b0), c1 = exp2f(m1 - b1);
    m0 = n0;
    m1 = n1;
    l0 *= c0;
    l1 *= c1;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][e] = exp2f(s[n][e] - b0);
        s[n][2 + e] = exp2f(s[n][2 + e] - b1);
        l0 += s[n][e];
        l1 += s[n][2 + e];
      }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      o[i][0] *= c0;
      o[i][1] *= c0;
      o[i][2] *= c1;
      o[i][3] *= c1;
    }
    const uint32_t p0 = pack2(T(), s[0][0], s[0][1]), p1 = pack2(T(), s[0][2], s[0][3]);
    const uint32_t p2 = pack2(T(), s[1][0], s[1][1]), p3 = pack2(T(), s[1][2], s[1][3]);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vv[0][c]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vv[1][c]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vv[2][c]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vv[3][c]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // element 2e and 2e + 1 of the lanes' eight: output column c * 64 + 8 * (column of the product) + element
        mma16816(T(), o[c * 8 + 2 * e], p0, p1, p2, p3, __byte_perm(v0[e], v1[e], 0x5410), __byte_perm(v2[e], v3[e], 0x5410));
        mma16816(T(), o[c * 8 + 2 * e + 1], p0, p1, p2, p3, __byte_perm(v0[e], v1[e], 0x7632),
                 __byte_perm(v2[e], v3[e], 0x7632));
      }
    }
  }
  // the four lanes of a row hold different keys' sums
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, d);
    l1 += __shfl_xor_sync(0xffffffffu, l1, d);
  }
  if (t == 0) {
    sm.wm[warp][g] = m0;
    sm.wm[warp][g + 8] = m1;
    sm.wl[warp][g] = l0;
    sm.wl[warp][g + 8] = l1;
  }
  for (int i = threadIdx.x; i < 16 * (D + 4); i += 32 * kFewWarps) (&sm.o[0][0])[i] = 0.f;
  __syncthreads();
  if (threadIdx.x < 16) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) m = max_nan(m, sm.wm[w][threadIdx.x]);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float x = m == -INFINITY ? 0.f : exp2f(sm.wm[w][threadIdx.x] - m);
      l += x * sm.wl[w][threadIdx.x];
      sm.wl[w][threadIdx.x] = x;  // from here on the warp's factor
    }
    sm.m[threadIdx.x] = m;
    sm.l[threadIdx.x] = l;
  }
  __syncthreads();
  // the warps add in turn: the order of the sums is fixed
  for (int w = 0; w < kFewWarps; ++w) {
    if (warp == w) {
      const float f0 = sm.wl[w][g], f1 = sm.wl[w][g + 8];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const int col = (i >> 3) * 64 + (i & 7);
        sm.o[g][col + 16 * t] += f0 * o[i][0];
        sm.o[g][col + 16 * t + 8] += f0 * o[i][1];
        sm.o[g + 8][col + 16 * t] += f1 * o[i][2];
        sm.o[g + 8][col + 16 * t + 8] += f1 * o[i][3];
      }
    }
    __syncthreads();
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  // every block of the cluster finishes its share of the rows
  for (int i = part * 32 * kFewWarps + threadIdx.x; i < 16 * (D / 8); i += split * 32 * kFewWarps) {
    const int r = i / (D / 8), c = i % (D / 8) * 8;
    const int row = rows0 + r;
    if (row >= rows) continue;
    float m = -INFINITY;
    for (int p = 0; p < split; ++p) m = max_nan(m, cluster.map_shared_rank(&sm, p)->m[r]);
    float l = 0.f, f[8] = {};
    for (int p = 0; p < split; ++p) {
      const FewSmem<D>* other = cluster.map_shared_rank(&sm, p);
      const float x = m == -INFINITY ? 0.f : exp2f(other->m[r] - m);
      l += x * other->l[r];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += x * other->o[r][c + e];
    }
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= inv;
    const int i_q = row / group, h = hk * group + row % group;
    store_vec<T, 8>(reinterpret_cast<T*>(a.o) + b * a.o_batch + i_q * a.o_row + h * D + c, f);
    if (c == 0 && a.lse != nullptr)
      a.lse[(static_cast<int64_t>(b) * a.heads + h) * a.seq_q + i_q] = (m + log2f(l)) * 0.6931471805599453f;
  }
  cluster.sync();  // no block leaves while another reads its shared memory
}

template <typename T, int D>
void launch_few(const CrossAttnArgs& a, cudaStream_t s) {
  const int64_t tiles = (static_cast<int64_t>(a.seq_q) * (a.heads / a.heads_kv) + 15) / 16;
  const int64_t units = tiles * a.heads_kv * a.batch;
  // split the keys while the blocks do not fill the SMs twice and every warp keeps 16 keys
  int split = 1;
  while (split < 8 && units * split < 2 * 148 && split * kFewWarps * 16 < a.seq_k) split *= 2;
  if (tiles * split > 0x7fffffff) throw std::runtime_error("cross_attention: too many queries");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * split), a.heads_kv, a.batch);
  cfg.blockDim = dim3(32 * kFewWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, cross_few_kernel<T, D>, a, split);
}

template <typename T>
void launch_type(const CrossAttnArgs& a, cudaStream_t s) {
  if (a.head_dim == 128) launch_few<T, 128>(a, s);
  else launch_few<T, 64>(a, s);
}

}  // namespace

void launch_cross_attention(const CrossAttnArgs& a, cudaStream_t s) {
  if (a.batch <= 0 || a.seq_q <= 0 || a.heads <= 0) return;
  if (a.head_dim != 64 && a.head_dim != 128) throw std::runtime_error("cross_attention: head_dim must be 64 or 128");
  switch (a.type) {
    case kBF16: launch_type<__nv_bfloat16>(a, s); break;
    case kFP16: launch_type<__half>(a, s); break;
    default: throw std::runtime_error("cross_attention: unsupported type");
  }
}

}  // namespace ds
