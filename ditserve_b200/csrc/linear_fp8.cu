// Linear layer on 8-bit operands (sm_100a):
//
//   y[m, n] = epilogue(sx[m] * sw[n] * sum_k x[m, k] * w[n, k] + b[n])
//
// x and w are e4m3 with one fp32 scale a row (a token, an output channel); sums are fp32.
#include <cooperative_groups.h>

#include <algorithm>

#include "elem.cuh"
#include "kernels.h"
#include "mma_sync.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace ds {
namespace {

namespace cg = cooperative_groups;

// GELU with the tanh approximation (Hendrycks & Gimpel 2016) for every type of output: 0.5 x (1 + tanh u) =
// x / (1 + exp(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3), by the hardware's power of two and quotient.  With w = 2^-24 an
// fp32 rounding and a = 2u: the exponent errs by at most 7 |a| w, the power and the quotient by 4 w of themselves, the sum
// by w: (7 |a| + 9) w of the value, 2^-18 at x = -3; below |x| 2^-126 it is 0.  The hardware's tanh would take one function
// less (32760 x 8960 from 1536 values 318 us for 339), but leaves |x| 2^-12 beside a value that goes to 0 (all of it at
// x = -4.9), more than the 16-bit types' own rounding.
constexpr double kGeluExp = -2.0 * 0.79788456080286541 * 1.44269504088896341;  // the exponent of 2 for x + ...
__device__ __forceinline__ float gelu(float x) {
  constexpr float k = static_cast<float>(kGeluExp);
  return __fdividef(x, 1.f + ex2_approx(k * (x + 0.044715f * x * x * x)));
}

// bias, activation, gate and residual of one output value; v is the scaled sum
template <typename T>
__device__ __forceinline__ float finish(const LinearFp8Args& a, float v, int m, int n, const float* gate_row) {
  if (a.bias != nullptr) v += to_float(reinterpret_cast<const T*>(a.bias)[n]);
  if (a.gelu) v = gelu(v);
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
  if (k >= K) return make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i >> 2] |= static_cast<uint32_t>(row[k + i]) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Few rows: a block takes 16 output channels and 8 * kM rows of x; its warps split K in chunks of 64, and so do up
// to 8 blocks of a cluster where channels are few and K is long.  The weights are the product's A operand
// straight from global memory, read once; sums are joined in shared memory, in a fixed order.  Bound by HBM, for
// small weights by latency: 2 rows to 9216 channels from 1536 values take 4.7 us on the device, 1 row to 256 channels
// from 8192 values 3.5 (7.5 with K in one block's warps alone).
constexpr int kRowWarps = 8;

template <int kM>
struct RowSmem {
  float part[kRowWarps][kM * 8][17];
  float in[8][kM * 8][16];  // rank 0: the cluster's sums
};

template <typename T, int kM>
__global__ void __launch_bounds__(32 * kRowWarps) linear_rows_kernel(LinearFp8Args a, int split) {
  extern __shared__ __align__(16) uint8_t row_smem[];
  RowSmem<kM>& sm = *reinterpret_cast<RowSmem<kM>*>(row_smem);
  cg::cluster_group cluster = cg::this_cluster();
  if (split > 1) cluster.barrier_arrive();  // waited for below: no push before all blocks have started
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % split;  // the cluster's blocks are neighbours in x
  const int n0 = blockIdx.x / split * 16, m0 = blockIdx.y * (8 * kM);
  // channels and rows behind the last are read as the last one and their sums dropped
  const uint8_t* w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = a.w + static_cast<int64_t>(min(n0 + i * 8 + g, a.N - 1)) * a.ldw;
  const uint8_t* x[kM];
#pragma unroll
  for (int i = 0; i < kM; ++i) x[i] = a.x + static_cast<int64_t>(min(m0 + i * 8 + g, a.M - 1)) * a.ldx;
  float acc[kM][4] = {};
  const int step = 64 * kRowWarps * split;
  for (int k0 = (rank * kRowWarps + warp) * 64; k0 < a.K; k0 += 2 * step) {
    uint4 wf[2][2], xf[2][kM];
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // the loads of two chunks before the products of the first
      const int k = k0 + u * step + t * 16;
#pragma unroll
      for (int i = 0; i < 2; ++i) wf[u][i] = load16(w[i], k, a.K);
#pragma unroll
      for (int i = 0; i < kM; ++i) xf[u][i] = load16(x[i], k, a.K);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < kM; ++i) {
        const uint4 p = wf[u][0], q = wf[u][1], b = xf[u][i];
        mma16832_e4m3(acc[i], p.x, q.x, p.y, q.y, b.x, b.y);
        mma16832_e4m3(acc[i], p.z, q.z, p.w, q.w, b.z, b.w);
      }
  }
#pragma unroll
  for (int i = 0; i < kM; ++i) {
    sm.part[warp][i * 8 + 2 * t][g] = acc[i][0];
    sm.part[warp][i * 8 + 2 * t + 1][g] = acc[i][1];
    sm.part[warp][i * 8 + 2 * t][g + 8] = acc[i][2];
    sm.part[warp][i * 8 + 2 * t + 1][g + 8] = acc[i][3];
  }
  __syncthreads();
  if (split > 1) cluster.barrier_wait();
  const int rows = min(8 * kM, a.M - m0);
  auto store = [&](int r, int c, float v) {
    const int m = m0 + r, n = n0 + c;
    v *= a.sx[m * a.sx_stride] * a.sw[n * a.sw_stride];
    reinterpret_cast<T*>(a.y)[static_cast<int64_t>(m) * a.ldy + n] = from_float<T>(finish<T>(a, v, m, n, gate_of(a, m)));
  };
  RowSmem<kM>* to = split > 1 ? cluster.map_shared_rank(&sm, 0) : &sm;
  for (int i = threadIdx.x; i < rows * 16; i += 32 * kRowWarps) {
    const int r = i / 16, c = i % 16;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kRowWarps; ++q) v += sm.part[q][r][c];
    if (split > 1) to->in[rank][r][c] = v;
    else if (n0 + c < a.N) store(r, c, v);
  }
  if (split == 1) return;
  cluster.sync();
  if (rank != 0) return;
  for (int i = threadIdx.x; i < rows * 16; i += 32 * kRowWarps) {
    const int r = i / 16, c = i % 16;
    if (n0 + c >= a.N) continue;
    float v = 0.f;
    for (int p = 0; p < split; ++p) v += sm.in[p][r][c];
    store(r, c, v);
  }
}

// Blocks that share K: more while the blocks leave SMs without one and every warp keeps two chunks
int row_split(int64_t blocks, int K) {
  int split = 1;
  while (split < 8 && 2 * blocks * split <= device_sm_count() && 2 * split * kRowWarps * 128 <= K) split *= 2;
  return split;
}

template <typename T, int kM>
void launch_rows(const LinearFp8Args& a, cudaStream_t s) {
  auto kern = linear_rows_kernel<T, kM>;
  constexpr int kSmem = sizeof(RowSmem<kM>);
  static_assert(kSmem <= 48 * 1024, "more needs an opt-in");
  const int64_t gx = (static_cast<int64_t>(a.N) + 15) / 16, gy = (a.M + 8 * kM - 1) / (8 * kM);
  const int split = row_split(gx * gy, a.K);
  if (gx * split > 0x7fffffff) throw std::runtime_error("linear_fp8: too many channels");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(gx * split), static_cast<unsigned>(gy));
  cfg.blockDim = dim3(32 * kRowWarps);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, a, split);
}

// ---------------------------------------------------------------------------
// Many rows: persistent, warp-specialised tcgen05 product (kind::f8f6f4).  A tile is 128 rows of x per
// CTA and bn output channels (whole 64-byte units of y up to 256, a launch parameter).  Warp 0 streams 128-byte
// k-blocks of both operands with TMA (128-byte swizzle) through a ring of stages, warp 1 issues the
// products into one of two TMEM accumulators, warps 2..17 scale, finish and store the other.
// kPair: two CTAs share one 256-row tile (cta_group::2), each staging its rows of x and half of the
// channels; the leader issues for both, and no operand byte is staged twice in the pair.
constexpr int kBM = 128, kBK = 128;
constexpr int kEpiWarps = 16, kEpiParts = kEpiWarps / 4;
constexpr int kTileThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxBn = 256;

// An epilogue warp stages 32 rows x 64 bytes of y at a time, from which a tile store takes them (whole
// sectors), and keeps the scales and biases of its quarter of the tile's columns.  What shared memory is
// left holds as many k-blocks as fit (at most kMaxStages): a stage's round trip takes about 2000 cycles,
// its products 512 at most (twins 1024), so a narrow tile needs the deeper ring.
constexpr int kOutBytes = 32 * 64, kCols = kMaxBn / kEpiParts, kColBytes = 2 * kCols * 4;
constexpr int kMaxStages = 10;
constexpr int kSmemBytes = 227 * 1024;
constexpr int kSmemFixed = kEpiWarps * (kOutBytes + kColBytes) + 1024 /*align*/ + 512 /*barriers*/;

struct TileShape {
  int bn, num_m, num_n, num_k;
  int twin;  // 1: a CTA takes two neighbouring tiles at once, one accumulator each, on the same rows of x
  int stages, stage_bytes;
  int fast;  // y and the residual have separate rows on 16 bytes, gate rows too: tile stores and loads
};

// two floats at once on the packed datapath
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
}

// gelu of two values, the exponent as x (k + k c x^2)
__device__ __forceinline__ float2 gelu2(float2 x) {
  constexpr float k = static_cast<float>(kGeluExp), kc = static_cast<float>(kGeluExp * 0.044715);
  const float2 p = mul2(x, fma2(mul2(x, x), make_float2(kc, kc), make_float2(k, k)));
  return make_float2(__fdividef(x.x, 1.f + ex2_approx(p.x)), __fdividef(x.y, 1.f + ex2_approx(p.y)));
}

// kU accumulator columns of an output row: scale, bias, activation.  cols holds the columns' scales, then (at kCols)
// their biases.
template <typename T, int kU>
__device__ __forceinline__ void scale_unit(const LinearFp8Args& a, const uint32_t (&acc)[kU], const float* cols, float sx,
                                           float (&v)[kU]) {
  const float2 sx2 = make_float2(sx, sx);
#pragma unroll
  for (int j = 0; j < kU; j += 4) {
    const float4 s = *reinterpret_cast<const float4*>(cols + j);
    const float4 b = *reinterpret_cast<const float4*>(cols + kCols + j);
    float2 x = fma2(make_float2(__uint_as_float(acc[j]), __uint_as_float(acc[j + 1])), mul2(sx2, make_float2(s.x, s.y)),
                    make_float2(b.x, b.y));
    float2 y = fma2(make_float2(__uint_as_float(acc[j + 2]), __uint_as_float(acc[j + 3])),
                    mul2(sx2, make_float2(s.z, s.w)), make_float2(b.z, b.w));
    if (a.gelu) {
      x = gelu2(x);
      y = gelu2(y);
    }
    v[j] = x.x;
    v[j + 1] = x.y;
    v[j + 2] = y.x;
    v[j + 3] = y.y;
  }
}

// 16-byte piece q of a lane's row in a warp's staging buffer (the 64-byte swizzle's place)
__device__ __forceinline__ uint8_t* piece(uint8_t* b, int lane, int q) {
  return b + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16);
}

// gate and residual of kU columns from channel n on; the residual's tile lies in the staging buffer
template <typename T, int kU>
__device__ __forceinline__ void add_residual(const LinearFp8Args& a, uint8_t* b, int lane, int n, const float* gate_row,
                                             float (&v)[kU]) {
  constexpr int V = kVec16<T>;
  if (gate_row != nullptr) {
#pragma unroll
    for (int j = 0; j < kU; j += 4) {
      if (n + j + 4 <= a.N) {
        const float4 g = *reinterpret_cast<const float4*>(gate_row + n + j);
        v[j] *= g.x;
        v[j + 1] *= g.y;
        v[j + 2] *= g.z;
        v[j + 3] *= g.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + j + e < a.N) v[j + e] *= gate_row[n + j + e];
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float f[V];
    load_vec<T, V>(reinterpret_cast<const T*>(piece(b, lane, q)), f);
#pragma unroll
    for (int e = 0; e < V; ++e) v[q * V + e] += f[e];
  }
}

template <typename T, bool kPair>
__global__ void __launch_bounds__(kTileThreads, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmR, LinearFp8Args a,
                       TileShape sh) {
  constexpr int kCtas = kPair ? 2 : 1;
  const int ST = sh.stages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // barriers, staged outputs and columns first (1024-byte aligned as a whole), then the ring: a stage is
  // 128 rows of x and this CTA's channels
  uint8_t* sOut = smem;
  float* sCol = reinterpret_cast<float*>(sOut + kEpiWarps * kOutBytes);
  uint8_t* ring = reinterpret_cast<uint8_t*>(sCol) + kEpiWarps * kColBytes;
  constexpr int kABytes = kBM * kBK;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + ST * sh.stage_bytes);  // pair: the leader's
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;
  uint64_t* acc_empty = acc_full + 2;  // pair: the leader's
  uint64_t* res_full = acc_empty + 2;  // [epilogue warp]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + kEpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = kPair ? blockIdx.x >> 1 : blockIdx.x, step = kPair ? gridDim.x >> 1 : gridDim.x;
  const int tiles = sh.num_m * sh.num_n, items = tiles >> sh.twin;
  // the i-th tile of this CTA
  auto tile_at = [&](int i) {
    const int item = first + (i >> sh.twin) * step;
    return item < items ? (item << sh.twin) + (i & sh.twin) : tiles;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpiWarps * kCtas);  // one arrival per epilogue warp
    }
    for (int i = 0; i < kEpiWarps; ++i) mbar_init(&res_full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    if constexpr (kPair) tmem_alloc_pair<512>(tmem_slot);
    else tmem_alloc<512>(tmem_slot);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync_all();  // the leader's barriers are ready before the peer signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      const int b_rows = sh.bn / kCtas;
      const uint32_t bytes = kCtas * sh.stage_bytes;
      for (int item = first; item < items; item += step) {
        const int tile = item << sh.twin;
        const int m0 = (tile / sh.num_n) * (kCtas * kBM) + rank * kBM;
        const int n0 = (tile % sh.num_n) * sh.bn + rank * b_rows;
        for (int kb = 0; kb < sh.num_k; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, a.status, 310)) goto producer_done;
          if constexpr (kPair) {
            const uint32_t leader = mapa_shared(smem_u32(&full[stage]), 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
            tma_load_2d_pair(ring + stage * sh.stage_bytes, &tmX, kb * kBK, m0, leader);
            tma_load_2d_pair(ring + stage * sh.stage_bytes + kABytes, &tmW, kb * kBK, n0, leader);
            if (sh.twin)
              tma_load_2d_pair(ring + stage * sh.stage_bytes + kABytes + b_rows * kBK, &tmW, kb * kBK, n0 + sh.bn, leader);
          } else {
            mbar_arrive_expect_tx(&full[stage], bytes);
            tma_load_2d(ring + stage * sh.stage_bytes, &tmX, kb * kBK, m0, &full[stage]);
            tma_load_2d(ring + stage * sh.stage_bytes + kABytes, &tmW, kb * kBK, n0, &full[stage]);
            if (sh.twin)
              tma_load_2d(ring + stage * sh.stage_bytes + kABytes + b_rows * kBK, &tmW, kb * kBK, n0 + sh.bn, &full[stage]);
          }
          if (++stage == ST) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    producer_done:;
    }
  } else if (warp == 1) {
    if (rank == 0) {  // the whole warp walks the loop, one lane issues
      const bool one = elect_sync();
      constexpr uint32_t kHi = umma_desc_hi_sw128(1024);
      const uint32_t ring_lo = umma_desc_lo(smem_u32(ring), 16);
      const uint32_t idesc = umma_idesc_e4m3(kCtas * kBM, sh.bn);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      const uint32_t twin_lo = (sh.bn / kCtas * kBK) >> 4;
      for (int item = first; item < items; item += step, local += 1 + sh.twin) {
        const int acc = local & 1;  // of twins the first's: 0
        for (int g = 0; g <= sh.twin; ++g)
          if (!mbar_wait_warp(&acc_empty[acc + g], ((local >> 1) & 1) ^ 1, abort_flag, a.status, 311)) goto mma_done;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * kMaxBn;
        for (int kb = 0; kb < sh.num_k; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, abort_flag, a.status, 312)) goto mma_done;
          tc_fence_after();
          const uint32_t a_lo = ring_lo + stage * (sh.stage_bytes >> 4), b_lo = a_lo + (kABytes >> 4);
          if (one) {
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k) {
              // 32 bytes onwards inside the swizzle atom: 2 in the address field
              if constexpr (kPair) umma_f8_ss_pair(d, a_lo + 2 * k, kHi, b_lo + 2 * k, kHi, idesc, (kb | k) != 0);
              else umma_f8_ss(d, a_lo + 2 * k, kHi, b_lo + 2 * k, kHi, idesc, (kb | k) != 0);
            }
            if (sh.twin) {
#pragma unroll
              for (int k = 0; k < kBK / 32; ++k) {
                const uint32_t t_lo = b_lo + twin_lo + 2 * k;
                if constexpr (kPair) umma_f8_ss_pair(d + kMaxBn, a_lo + 2 * k, kHi, t_lo, kHi, idesc, (kb | k) != 0);
                else umma_f8_ss(d + kMaxBn, a_lo + 2 * k, kHi, t_lo, kHi, idesc, (kb | k) != 0);
              }
            }
            if constexpr (kPair) umma_commit_pair(&empty[stage]);
            else umma_commit(&empty[stage]);
          }
          if (++stage == ST) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (one) {
          for (int g = 0; g <= sh.twin; ++g) {
            if constexpr (kPair) umma_commit_pair(&acc_full[acc + g]);
            else umma_commit(&acc_full[acc + g]);
          }
        }
      }
    mma_done:;
    }
  } else {
    constexpr int kU = 64 / sizeof(T);        // columns of a unit (64 bytes of y)
    const int quarter = warp & 3;             // the TMEM lanes this warp may read
    const int part = (warp - 2) >> 2;         // the warps of a quarter take turns at the units
    uint8_t* b = sOut + (warp - 2) * kOutBytes;
    float* cols = sCol + (warp - 2) * (kColBytes / 4);
    // a tile's parameters of this lane: its row's scale, its two columns' scales and biases.  They are
    // fetched one tile ahead
    float p_sx = 0.f, p_sw[kCols / 32] = {}, p_b[kCols / 32] = {};
    auto fetch = [&](int tile) {
      if (tile >= tiles) return;
      const int m = (tile / sh.num_n) * (kCtas * kBM) + rank * kBM + quarter * 32 + lane;
      p_sx = m < a.M ? a.sx[m * a.sx_stride] : 0.f;
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        const int k = i * 32 + lane;                                       // this warp's k-th column of the tile
        const int c = (kEpiParts * (k / kU) + part) * kU + k % kU, n = (tile % sh.num_n) * sh.bn + c;
        const bool on = c < sh.bn && n < a.N;
        p_sw[i] = on ? a.sw[n * a.sw_stride] : 0.f;
        p_b[i] = on && a.bias != nullptr ? to_float(reinterpret_cast<const T*>(a.bias)[n]) : 0.f;
      }
    };
    // the accumulator goes back as soon as this warp's last columns are in registers
    auto hand_back = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair) mbar_arrive_remote(mapa_shared(smem_u32(&acc_empty[acc]), 0));
        else mbar_arrive(&acc_empty[acc]);
      }
    };
    // the residual of the next unit comes as a tile into the staging buffer, once the last store has read it: rows read
    // by their threads in 16-byte pieces took 64 us where this takes 46 (25528 x 768 in fp32 from 639 values)
    const bool by_tile = sh.fast && a.residual != nullptr;
    uint64_t* res_bar = &res_full[warp - 2];
    uint32_t res_phase = 0;
    auto ask = [&](int n, int m) {
      if (lane == 0) {
        tma_store_wait_read<0>();
        mbar_arrive_expect_tx(res_bar, kOutBytes);
        tma_load_2d(b, &tmR, n, m, res_bar);
      }
    };
    fetch(tile_at(0));
    for (int local = 0;; ++local) {
      const int tile = tile_at(local);
      if (tile >= tiles) break;
      const int acc = local & 1;
      const int m0 = (tile / sh.num_n) * (kCtas * kBM) + rank * kBM + quarter * 32;
      const int m = m0 + lane;
      const int n0 = (tile % sh.num_n) * sh.bn;
      const bool row_ok = m < a.M;
      const float sx = p_sx;
      const float* gate_row = row_ok ? gate_of(a, m) : nullptr;
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        cols[i * 32 + lane] = p_sw[i];
        cols[kCols + i * 32 + lane] = p_b[i];
      }
      fetch(tile_at(local + 1));
      if (by_tile && part * kU < sh.bn) ask(n0 + part * kU, m0);  // on its way while the accumulator is waited for
      if (!sh.fast && a.residual != nullptr && row_ok) {     // off 16 bytes at least on its way into the L2
        const T* res = reinterpret_cast<const T*>(a.residual) + static_cast<int64_t>(m) * a.ldr + n0;
        for (int c = part * kU; c < sh.bn && n0 + c < a.N; c += kEpiParts * kU)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(res + c));
      }
      __syncwarp();
      if (!mbar_wait_warp(&acc_full[acc], (local >> 1) & 1, abort_flag, a.status, 313)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kMaxBn;
#pragma unroll 1
      for (int c = part * kU; c < sh.bn; c += kEpiParts * kU) {
        uint32_t r[kU];
        if constexpr (kU == 32) tmem_ld32(taddr + c, r);
        else tmem_ld16(taddr + c, r);
        tmem_wait_ld();
        if (c + kEpiParts * kU >= sh.bn) hand_back(acc);
        float v[kU];
        const int n = n0 + c;
        scale_unit<T, kU>(a, r, cols + (c / kU / kEpiParts) * kU, sx, v);
        if (sh.fast) {
          if (by_tile) {
            if (!mbar_wait_warp(res_bar, res_phase, abort_flag, a.status, 314)) goto epilogue_done;
            res_phase ^= 1;
            add_residual<T, kU>(a, b, lane, n, gate_row, v);
          } else {
            if (lane == 0) tma_store_wait_read<0>();  // the last store has read the buffer
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)
            store_vec<T, kVec16<T>>(reinterpret_cast<T*>(piece(b, lane, q)),
                                    *reinterpret_cast<const float(*)[kVec16<T>]>(&v[q * kVec16<T>]));
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (m0 < a.M && n < a.N) tma_store_2d(&tmY, n, m0, b);
            tma_store_commit();
          }
          if (by_tile && c + kEpiParts * kU < sh.bn) ask(n + kEpiParts * kU, m0);
        } else {
          // rows off 16 bytes: 16 columns at a time through the buffer, so that a warp's store is of two rows' neighbours
#pragma unroll
          for (int h = 0; h < kU; h += 16) {
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<float4*>(b + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16)) =
                  make_float4(v[h + 4 * q], v[h + 4 * q + 1], v[h + 4 * q + 2], v[h + 4 * q + 3]);
            __syncwarp();
            const int col = lane & 15, n1 = n + h + col;
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += 16) {  // the residuals of eight stores first
              float y[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int k = r0 + 2 * i + (lane >> 4);
                const float* g = reinterpret_cast<const float*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(gate_row), k));
                y[i] = *reinterpret_cast<const float*>(b + k * 64 + (((col >> 2) ^ ((k >> 1) & 3)) * 16) + (col & 3) * 4);
                if (a.residual != nullptr && m0 + k < a.M && n1 < a.N)
                  y[i] = fmaf(y[i], g != nullptr ? g[n1] : 1.f,
                              to_float(reinterpret_cast<const T*>(a.residual)[static_cast<int64_t>(m0 + k) * a.ldr + n1]));
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int k = r0 + 2 * i + (lane >> 4);
                if (m0 + k < a.M && n1 < a.N)
                  reinterpret_cast<T*>(a.y)[static_cast<int64_t>(m0 + k) * a.ldy + n1] = from_float<T>(y[i]);
              }
            }
          }
        }
      }
      if (part * kU >= sh.bn) hand_back(acc);  // a narrow tile has no unit for this warp
    }
  epilogue_done:
    if (lane == 0) tma_store_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    // copies that may still be in flight get time to land
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  if constexpr (kPair) cluster_sync_all();  // no CTA leaves while its partner may still address its memory
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kPair) tmem_dealloc_pair<512>(tmem_base);
    else tmem_dealloc<512>(tmem_base);
  }
}

// Width of the tiles: the multiple of a unit whose rounds over the SMs cost least.  A k-block takes about 0.29 us +
// 0.1 us * bn / 256 (8960 x 1536 channels at 32760 rows: 0.39, 0.355 and 0.325 us for 256, 192 and 128
// channels), bound by the L2's traffic into shared memory more than by the products, so few wide rounds
// beat many narrow ones, and a single round takes the narrowest tile that keeps it one.  32760 rows to 8960 channels from
// 1536 values take 311 to 322 us as a single launch without an activation, 339 to 351 with GELU (0.88 and 0.81 of twice
// the measured 16-bit rate; the 8-bit rate itself is not measured), 365 to 450 in a row of them under the power limit.
// The cost knows no epilogue: where K is short it is the time (474 rows to 6656 channels from 64 values with a gated
// residual 9.4 us).
// `unit` (16 or 32) keeps whole 64-byte units of the output in a tile, which is how the epilogue goes through it.
// More tiles than CTAs, but fewer than twice as many: twins bring them into one round, and a k-block of x then serves
// both (the tiles' outputs leave behind one another, which a second round would not spare either): 512 rows to 10240
// channels from 4096 values 22.6 us against 23.6.
struct TilePlan {
  int bn, twin;
  int64_t rounds;
};

TilePlan plan_tiles(int64_t num_m, int N, int slots, int unit) {
  TilePlan best = {kMaxBn, 0, 1};
  int64_t cost = INT64_MAX;
  for (int twin = 0; twin < 2; ++twin) {
    if (twin && best.rounds == 1) break;
    for (int bn = kMaxBn; bn >= 32; bn -= unit) {
      const int width = bn << twin;
      const int64_t items = num_m * ((N + width - 1) / width), rounds = (items + slots - 1) / slots;
      if (twin && rounds > 1) break;
      const int64_t c = rounds * (width + 740);
      if (c < cost) {
        cost = c;
        best = {bn, twin, rounds};
      }
    }
  }
  return best;
}

template <typename T, bool kPair>
void launch_tiles(const LinearFp8Args& a, const TilePlan& plan, cudaStream_t s) {
  const int bn = plan.bn;
  constexpr int kCtas = kPair ? 2 : 1;
  auto kern = linear_tile_kernel<T, kPair>;
  static std::atomic<uint64_t> allowed{0};
  allow_smem(kern, kSmemBytes, allowed);
  const CUtensorMap tmX = make_tmap_u8_2d(a.x, a.M, a.K, a.ldx, kBM);
  const CUtensorMap tmW = make_tmap_u8_2d(a.w, a.N, a.K, a.ldw, bn / kCtas);
  auto at = [](const void* p, int64_t bytes, int n) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % n == 0 && bytes % n == 0);
  };
  const int64_t e = sizeof(T);
  TileShape sh;
  sh.bn = bn;
  sh.num_m = (a.M + kCtas * kBM - 1) / (kCtas * kBM);
  sh.twin = plan.twin;
  sh.num_n = (a.N + bn - 1) / bn;
  if (sh.twin) sh.num_n += sh.num_n & 1;  // twins are of one row of tiles
  sh.num_k = (a.K + kBK - 1) / kBK;
  sh.stage_bytes = (kBM + (bn << sh.twin) / kCtas) * kBK;
  sh.stages = std::min(kMaxStages, (kSmemBytes - kSmemFixed) / sh.stage_bytes);
  sh.fast = at(a.y, a.ldy * e, 16) && at(a.residual, a.ldr * e, 16) && at(a.gate, a.gate_stride * 4, 16) &&
            (a.residual == nullptr || a.ldr >= a.N);
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  const CUtensorMap tmY = sh.fast ? make_tmap_out_2d(a.y, type, sizeof(T), a.M, a.N, a.ldy, 32) : tmX;
  const CUtensorMap tmR =
      sh.fast && a.residual != nullptr
          ? make_tmap_out_2d(const_cast<void*>(a.residual), type, sizeof(T), a.M, a.N, a.ldr, 32)
          : tmX;
  const int64_t tiles = static_cast<int64_t>(sh.num_m) * sh.num_n;
  if (tiles > 0x3fffffff) throw std::runtime_error("linear_fp8: too many tiles");
  const int slots = device_sm_count() / kCtas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCtas * static_cast<unsigned>(std::min<int64_t>(tiles >> sh.twin, slots)));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, tmX, tmW, tmY, tmR, a, sh);
}

// Whether the few-row form takes less time, by what both were measured to take in us (in a graph, 12 to 256 rows, 64 to
// 10240 channels and values; up to 16 rows the first form always):
//   rows    2 (3.5 with K split over blocks) + the operands' bytes out of L2, 16 + 8 kM rows a block, at 4.8 TB/s
//   tiles   3.2 + rounds * (k-blocks * (0.24 + 0.1 bn / 256) + 0.6)
// e.g. 32 rows to 1024 channels from 4096 values 6.4 and 11.3, to 9216 from 1536 10.3 and 8.2.  Neither knows epilogues
// or warps without a chunk of K, which count where K is short: 100 rows to 4544 channels from 128 values with a
// residual take 11.1 in the first form, where the rule expects 3.5.
bool rows_are_faster(const LinearFp8Args& a) {
  if (a.M <= 16 || a.M > 4096) return a.M <= 16;
  const int rows = 32;
  const int64_t blocks = (static_cast<int64_t>(a.N) + 15) / 16 * ((a.M + rows - 1) / rows);
  const double few = (row_split(blocks, a.K) > 1 ? 3.5 : 2.0) + static_cast<double>(blocks) * (16 + rows) * a.K / 4.8e6;
  const int m = a.M <= kBM ? kBM : 2 * kBM, slots = device_sm_count() * kBM / m;
  const int64_t num_m = (a.M + m - 1) / m;
  const TilePlan p = plan_tiles(num_m, a.N, slots, a.out_type == kFP32 ? 16 : 32);
  const double blocks_k = static_cast<double>((a.K + kBK - 1) / kBK);
  return few < 3.2 + static_cast<double>(p.rounds) * (blocks_k * (0.24 + 0.1 * (p.bn << p.twin) / 256) + 0.6 * (1 + p.twin));
}

template <typename T>
void launch_type(const LinearFp8Args& a, cudaStream_t s) {
  if (a.M <= 8) {
    launch_rows<T, 1>(a, s);
  } else if (rows_are_faster(a)) {
    if (a.M <= 16) launch_rows<T, 2>(a, s);
    else launch_rows<T, 4>(a, s);
  } else {
    const int sms = device_sm_count();
    constexpr int kUnit = 64 / sizeof(T);
    if (a.M <= kBM) launch_tiles<T, false>(a, plan_tiles(1, a.N, sms, kUnit), s);
    else launch_tiles<T, true>(a, plan_tiles((a.M + 2 * kBM - 1) / (2 * kBM), a.N, sms / 2, kUnit), s);
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
