// Attention of queries to an encoder's states of another length (sm_100a): padded, masked contexts.
//
//   o[b, i, h] = sum_j p_ij v[b, j, hk] / sum_j p_ij,  p_ij = exp(scale q_i k_j - max_j), j over the keys of
//   batch entry b that its valid length and its key mask leave; nothing left: o = 0 and lse = -inf.
//
// Scores, the running maximum and sum (Milakov and Gimelshein, "Online normalizer calculation for softmax", 2018) and the
// output's sums are fp32.  p is rounded to the values' type for the second product, whose operands have 16 bits: half
// a step of each weight, while the sum below keeps 32 bits.  Against 64 bits the output errs 1.2 to 1.4 times as much as
// with weights of 32 bits (bf16 0.0023 of it for 0.0017, fp16 0.00028 for 0.00021), and fp16 weights below 2^-25 of the
// largest count in the sum alone.  Keys that are masked never reach a product with their value: their v is replaced by
// zero, so that NaN or infinities in padding do no harm.
#include <cooperative_groups.h>

#include <type_traits>

#include "elem.cuh"
#include "kernels.h"
#include "mma_sync.cuh"
#include "sm100.cuh"
#include "tma_host.h"

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

// Few queries: a cluster of up to 8 blocks takes 16 query rows of one key head (a row is a query of one of the heads
// that share the key head) and splits the keys over its warps, 16 at a time.  K and V go from global memory
// straight to the products' operands in 16-byte pieces; a warp's maximum, sum and output are joined with the
// others' through shared memory, then each row with the other blocks' in the block that finishes it: partials are
// pushed there, one cluster barrier behind the pushes, sums in a fixed order.  Bound by latency:
// one query of 2 x 12 heads over 512 keys takes 5.2 us (8.1 with the warps adding in turn and remote reads).
constexpr int kFewWarps = 8, kFewThreads = 32 * kFewWarps, kFewRows = 16;

template <int D>
struct FewSmem {
  float o[kFewWarps][kFewRows][D + 4];
  float m[kFewWarps][kFewRows], l[kFewWarps][kFewRows];
  float in[kFewRows][D + 4];  // [source block][row / split]: the cluster's partials of the rows finished here
  float2 in_ml[kFewRows];
};

template <typename T, int D>
__global__ void __launch_bounds__(kFewThreads) cross_few_kernel(CrossAttnArgs a, int split) {
  extern __shared__ __align__(16) uint8_t few_smem[];
  FewSmem<D>& sm = *reinterpret_cast<FewSmem<D>*>(few_smem);
  cg::cluster_group cluster = cg::this_cluster();
  if (split > 1) cluster.barrier_arrive();  // waited for below: no push before all blocks have started
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int part = blockIdx.x % split;  // the cluster's blocks are neighbours in x
  const int rows0 = blockIdx.x / split * kFewRows;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int group = a.heads / a.heads_kv;
  const int rows = a.seq_q * group;
  const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_batch;
  const T* k = reinterpret_cast<const T*>(a.k) + b * a.k_batch + hk * D;
  const T* v = reinterpret_cast<const T*>(a.v) + b * a.v_batch + hk * D;
  const int valid = valid_keys(a, b);
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
  for (int j0 = (part * kFewWarps + warp) * 16; j0 < a.seq_k; j0 += stride) {
    // all loads of the 16 keys first, whatever the lengths say: keys behind the last are read as the last
    uint4 kk[2][D / 32], vv[4][D / 64];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const T* row = k + static_cast<int64_t>(min(j0 + n * 8 + g, a.seq_k - 1)) * a.k_row + t * 8;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) kk[n][i] = *reinterpret_cast<const uint4*>(row + i * 32);
    }
    // V of this lane's four keys (2t, 2t + 1, 2t + 8, 2t + 9)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* row = v + static_cast<int64_t>(min(j0 + 2 * t + (i & 1) + (i >> 1) * 8, a.seq_k - 1)) * a.v_row + g * 8;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) vv[i][c] = *reinterpret_cast<const uint4*>(row + c * 64);
    }
    bool ok[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + 2 * t + (i & 1) + (i >> 1) * 8;
      ok[i >> 1][i & 1] = j < a.seq_k && key_allowed(a, b, j, valid);
    }
    if (j0 >= valid) break;
    float s[2][4] = {};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        mma16816(T(), s[n], qa[i].x, qb[i].x, qa[i].y, qb[i].y, kk[n][i].x, kk[n][i].y);
        mma16816(T(), s[n], qa[i].z, qb[i].z, qa[i].w, qb[i].w, kk[n][i].z, kk[n][i].w);
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
    const float c0 = ex2_approx(m0 - b0), c1 = ex2_approx(m1 - b1);
    m0 = n0;
    m1 = n1;
    l0 *= c0;
    l1 *= c1;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[n][e] = ex2_approx(s[n][e] - b0);
        s[n][2 + e] = ex2_approx(s[n][2 + e] - b1);
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
    // a masked key's value never meets a product, whatever its slot holds
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        if (!ok[i >> 1][i & 1]) vv[i][c] = make_uint4(0, 0, 0, 0);
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
    sm.m[warp][g] = m0;
    sm.m[warp][g + 8] = m1;
    sm.l[warp][g] = l0;
    sm.l[warp][g + 8] = l1;
  }
  const int here = min(kFewRows, rows - rows0);  // rows of this tile
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const int col = (i >> 3) * 64 + (i & 7) + 16 * t;
    if (g < here) {
      sm.o[warp][g][col] = o[i][0];
      sm.o[warp][g][col + 8] = o[i][1];
    }
    if (g + 8 < here) {
      sm.o[warp][g + 8][col] = o[i][2];
      sm.o[warp][g + 8][col + 8] = o[i][3];
    }
  }
  __syncthreads();
  auto finish = [&](int r, int c, float m, float l, float4 f) {
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    const int row = rows0 + r, i_q = row / group, h = hk * group + row % group;
    uint2 w = make_uint2(pack2(T(), f.x * inv, f.y * inv), pack2(T(), f.z * inv, f.w * inv));
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.o) + b * a.o_batch + i_q * a.o_row + h * D + c) = w;
    if (c == 0 && a.lse != nullptr)
      a.lse[(static_cast<int64_t>(b) * a.heads + h) * a.seq_q + i_q] = (m + log2f(l)) * 0.6931471805599453f;
  };
  if (split > 1) cluster.barrier_wait();
  for (int i = threadIdx.x; i < here * (D / 4); i += kFewThreads) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) m = max_nan(m, sm.m[w][r]);
    float l = 0.f;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float x = m == -INFINITY ? 0.f : ex2_approx(sm.m[w][r] - m);
      const float4 p = *reinterpret_cast<const float4*>(&sm.o[w][r][c]);
      l += x * sm.l[w][r];
      f.x += x * p.x;
      f.y += x * p.y;
      f.z += x * p.z;
      f.w += x * p.w;
    }
    if (split == 1) {
      finish(r, c, m, l, f);
    } else {
      FewSmem<D>* to = cluster.map_shared_rank(&sm, r % split);
      const int slot = part * (kFewRows / split) + r / split;
      *reinterpret_cast<float4*>(&to->in[slot][c]) = f;
      if (c == 0) to->in_ml[slot] = make_float2(m, l);
    }
  }
  if (split == 1) return;
  cluster.sync();
  for (int i = threadIdx.x; i < kFewRows / split * (D / 4); i += kFewThreads) {
    const int at = i / (D / 4), r = at * split + part, c = i % (D / 4) * 4;
    if (r >= here) continue;
    float m = -INFINITY;
    for (int p = 0; p < split; ++p) m = max_nan(m, sm.in_ml[p * (kFewRows / split) + at].x);
    float l = 0.f;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < split; ++p) {
      const int slot = p * (kFewRows / split) + at;
      const float2 ml = sm.in_ml[slot];
      const float4 y = *reinterpret_cast<const float4*>(&sm.in[slot][c]);
      const float x = m == -INFINITY ? 0.f : ex2_approx(ml.x - m);
      l += x * ml.y;
      f.x += x * y.x;
      f.y += x * y.y;
      f.z += x * y.z;
      f.w += x * y.w;
    }
    finish(r, c, m, l, f);
  }
}

// Blocks of the few-row form that run at once: its registers leave room for one an SM at 128 values a head, two at 64
int64_t few_slots(int d) { return static_cast<int64_t>(device_sm_count()) * (d == 64 ? 2 : 1); }

// Blocks that share a tile's keys: more while all of them still run at once and every warp keeps 16 keys
int few_split(int64_t units, int seq_k, int d) {
  int split = 1;
  while (split < 8 && 2 * units * split <= few_slots(d) && split * kFewWarps * 16 < seq_k) split *= 2;
  return split;
}

template <typename T, int D>
void launch_few(const CrossAttnArgs& a, cudaStream_t s) {
  auto kern = cross_few_kernel<T, D>;
  constexpr int kSmem = sizeof(FewSmem<D>);
  static std::atomic<uint64_t> allowed{0};
  allow_smem(kern, kSmem, allowed);
  const int64_t tiles = (static_cast<int64_t>(a.seq_q) * (a.heads / a.heads_kv) + kFewRows - 1) / kFewRows;
  const int64_t units = tiles * a.heads_kv * a.batch;
  const int split = few_split(units, a.seq_k, D);
  if (tiles * split > 0x7fffffff) throw std::runtime_error("cross_attention: too many queries");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * split), a.heads_kv, a.batch);
  cfg.blockDim = dim3(kFewThreads);
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
// Many queries: persistent CTAs on the tensor cores (tcgen05).  A unit of work is two 128-row tiles A and B of
// the query rows that read one key head (its heads' tiles in turn), against all key tiles of the batch entry.
//   warp 0        TMA: Q of both tiles, K one tile ahead of V
//   warp 1        products, in the order S_A(i+1) after PV_A(i), S_B(i+1) after PV_B(i), straight on over the
//                 end of a unit: the next unit's first scores are formed while this one's output leaves
//   warp 2        puts zeros in the values of masked keys (only with lengths or a mask)
//   warps 4..7    softmax and output of tile A, a row a thread; warps 8..11 of tile B
// TMEM: S_A [0, 128), S_B [128, 256), O_A [256, 256 + D), O_B [384, 384 + D).  P is written over the first
// half of its S as the second product's TMEM operand, in two chunks of 64 keys.  The maximum that is
// subtracted may lag, since a common factor cancels in the quotient (a known variant): O is rescaled only when it has
// grown by more than 2^8; P then is at most 256, which both types hold.
// Bound by the chain softmax (2000 cycles a step), P to PV, PV, next S (1400) of a tile, which two tiles in turn cover to
// about 60 % of the tensor pipe's time, and at a unit's end by its output (2500).  32760 queries of 12 heads over 4096
// keys take 690 to 765 us from one B200 to another (1190 to 1080 TFLOP/s), 2 x 32760 over 512 keys 207 to 220 (1000 to 940).
// Measured and not kept (against the form of the day, measured alike): P through shared memory
// with the next scores formed during the exponentials (268 us against 240 at 4096 x 4096: operands, P and loads together
// exceed the shared memory's rate), two threads a row (213 against 197), output warps of their own, every fourth pair of
// exponentials as a polynomial (238 against 197), a product warp a tile (218 against 197), key tiles of 64 with the scores
// formed two ahead (266 against 218; with a product warp a tile 256): a barrier's wait takes 200 cycles behind the other
// tile's exponentials in the queue, and smaller tiles wait twice as often.  A ragged last key tile costs what a full one
// does, and units of one key head's rows are not split over keys where they leave SMs without one: 4 x 288 queries over
// 764 keys of 12 heads of 64 take 15.6 us (floor 2.0), 2 x 845 over 1654 of 24 heads 53 (10.9).
constexpr int kQT = 128, kKT = 128, kPChunks = 2;
constexpr int kTileThreads = 384;

// a softmax warp stages 32 rows x 128 bytes of O at a time, from which a tile store takes them: stores of whole
// rows by their threads took 3700 cycles of 18400 a unit of four key tiles
constexpr int kOutBytes = 32 * 128;

// Batch entries whose keys a block lists, and bytes of mask it reads for that at most
constexpr int kListed = 64, kListedMask = 1 << 16;

template <int D>
struct TileCfg {
  static constexpr int kAtoms = D / 64;
  static constexpr int kQBytes = kQT * D * 2;
  static constexpr int kKvBytes = kKT * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;  // of K and of V
  static constexpr int kSmemBytes = 2 * kQBytes + 2 * kStages * kKvBytes + 8 * kOutBytes + kListed * 4 + 1024 + 512;
};

struct TileMaps {
  CUtensorMap q, k, v, o;
};

struct TileShape {
  int units, tiles, group;                  // unit = (b * heads_kv + hk) * pairs + pair of a key head's row tiles
  FastDiv pairs, heads_kv, q_tiles;
  int k_shared, v_shared, q_shared;  // batch stride 0: one entry read by all
  int listed;                        // the block lists the keys of every batch entry first
};

__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  return (static_cast<uint64_t>(__float_as_uint(hi)) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& lo, float& hi) {
  lo = __uint_as_float(static_cast<uint32_t>(v));
  hi = __uint_as_float(static_cast<uint32_t>(v >> 32));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

struct Unit {
  int b, hk, pair;   // batch entry, key head, pair of row tiles
  int valid, n;      // keys up to the last one that is left, and their tiles
  bool two;          // tile B has rows
};

// `ends`: the batch entries' keys, where the block has listed them
__device__ __forceinline__ Unit unit_of(const CrossAttnArgs& a, const TileShape& sh, const int* ends, int u) {
  Unit x;
  const int bh = sh.pairs.div(u);
  x.pair = u - bh * sh.pairs.d;
  x.b = sh.heads_kv.div(bh);
  x.hk = bh - x.b * a.heads_kv;
  x.valid = sh.listed ? ends[x.b] : valid_keys(a, x.b);
  x.n = (x.valid + kKT - 1) / kKT;
  x.two = 2 * x.pair + 1 < sh.tiles;
  return x;
}

// head and first query of tile t of a unit
__device__ __forceinline__ int2 tile_of(const CrossAttnArgs& a, const TileShape& sh, const Unit& x, int t) {
  const int i = 2 * x.pair + t, g = sh.q_tiles.div(i);
  return make_int2(x.hk * sh.group + g, (i - g * sh.q_tiles.d) * kQT);
}

// One key tile of one unit; walks a CTA's units in order, leaving out those without keys.  base + j counts the key
// tiles so far: the place in the K and V rings.
struct Step {
  int u, j = 0, base = 0;
  Unit x;
  __device__ __forceinline__ bool settle(const CrossAttnArgs& a, const TileShape& sh, const int* ends) {
    for (; u < sh.units; u += gridDim.x) {
      x = unit_of(a, sh, ends, u);
      if (x.n > 0) return true;
    }
    return false;
  }
  __device__ __forceinline__ bool advance(const CrossAttnArgs& a, const TileShape& sh, const int* ends) {
    if (++j < x.n) return true;
    j = 0;
    base += x.n;
    u += gridDim.x;
    return settle(a, sh, ends);
  }
};

// bit i of word w: key tile * 128 + 32 w + i may be attended to.  All lanes of the warp call it.
__device__ __forceinline__ void tile_mask(const CrossAttnArgs& a, int b, int tile, int valid, uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __ballot_sync(0xffffffffu, key_allowed(a, b, tile * kKT + i * 32 + (threadIdx.x & 31), valid));
}

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    cross_tile_kernel(const __grid_constant__ TileMaps maps, CrossAttnArgs a, TileShape sh) {
  using Cfg = TileCfg<D>;
  constexpr int ST = Cfg::kStages;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * Cfg::kQBytes;
  uint8_t* sV = sK + ST * Cfg::kKvBytes;
  uint8_t* sOut = sV + ST * Cfg::kKvBytes;                               // [8 warps]
  int* ends = reinterpret_cast<int*>(sOut + 8 * kOutBytes);              // [kListed]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ends + kListed);        // [2] a tile
  uint64_t* q_empty = q_full + 2;
  uint64_t* k_full = q_empty + 2;   // [ST]
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_ready = v_full + ST;  // masked values cleared
  uint64_t* v_empty = v_ready + ST;
  uint64_t* s_full = v_empty + ST;           // [2]
  uint64_t* p_full = s_full + 2;             // [2][kPChunks]
  uint64_t* pv_done = p_full + 2 * kPChunks;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool masked_kv = a.kv_lens != nullptr || a.key_mask != nullptr;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < 2 * kPChunks; ++i) mbar_init(&p_full[i], 4);  // one arrival a warp
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ready[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc<512>(tmem_slot);
  if (sh.listed) {
    // keys up to the last one that length and mask leave: padding given by a mask alone is left out, too
    for (int b = warp; b < a.batch; b += kTileThreads / 32) {
      int end = valid_keys(a, b);
      if (a.key_mask != nullptr) {
        int last = 0;
#pragma unroll 8
        for (int j = lane; j < end; j += 32)
          if (a.key_mask[b * a.mask_row + j * a.mask_col] != 0) last = j + 1;
        end = __reduce_max_sync(0xffffffffu, last);
      }
      if (lane == 0) ends[b] = end;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp < 4) {
    if (warp == 0) {
      if (lane == 0) {
        // ---------------- TMA ----------------
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
        int q_count[2] = {0, 0}, kc = 0, vc = 0;
        auto load_q = [&](const Unit& x) -> bool {
          for (int t = 0; t < (x.two ? 2 : 1); ++t) {
            if (!mbar_wait(&q_empty[t], (q_count[t] & 1) ^ 1, abort_flag, a.status, 410 + t)) return false;
            ++q_count[t];
            mbar_arrive_expect_tx(&q_full[t], Cfg::kQBytes);
            const int2 at = tile_of(a, sh, x, t);
#pragma unroll
            for (int i = 0; i < Cfg::kAtoms; ++i)
              tma_load_3d(sQ + t * Cfg::kQBytes + i * (kQT * 128), &maps.q, at.x * D + i * 64, at.y,
                          sh.q_shared ? 0 : x.b, &q_full[t]);
          }
          return true;
        };
        auto load_kv = [&](const Step& s, const CUtensorMap* map, int shared, uint8_t* base, uint64_t* full, uint64_t* empty,
                           int& count, int site) -> bool {
          const int st = count % ST;
          if (!mbar_wait(&empty[st], ((count / ST) & 1) ^ 1, abort_flag, a.status, site)) return false;
          ++count;
          mbar_arrive_expect_tx(&full[st], Cfg::kKvBytes);
#pragma unroll
          for (int i = 0; i < Cfg::kAtoms; ++i)
            tma_load_3d(base + st * Cfg::kKvBytes + i * (kKT * 128), map, s.x.hk * D + i * 64, s.j * kKT,
                        shared ? 0 : s.x.b, &full[st]);
          return true;
        };
        Step cur;
        cur.u = blockIdx.x;
        // K before Q: the first tile's scores need K and that tile's Q alone
        bool ok = cur.settle(a, sh, ends) && load_kv(cur, &maps.k, sh.k_shared, sK, k_full, k_empty, kc, 412) && load_q(cur.x);
        while (ok) {
          Step next = cur;
          const bool more = next.advance(a, sh, ends);
          if (more && !load_kv(next, &maps.k, sh.k_shared, sK, k_full, k_empty, kc, 412)) break;
          if (!load_kv(cur, &maps.v, sh.v_shared, sV, v_full, v_empty, vc, 413)) break;
          // the next unit's Q, which waits for the last scores, behind all that this unit needs
          if (more && next.j == 0 && !load_q(next.x)) break;
          cur = next;
          ok = more;
        }
      }
    } else if (warp == 1) {
      // ---------------- products (the whole warp walks the loop, one lane issues) ----------------
      const bool one = elect_sync();
      constexpr uint32_t idesc_s = kBf16 ? umma_idesc_bf16(kQT, kKT, false) : umma_idesc_fp16(kQT, kKT, false);
      constexpr uint32_t idesc_o = kBf16 ? umma_idesc_bf16(kQT, D, true) : umma_idesc_fp16(kQT, D, true);
      constexpr uint32_t kHi = umma_desc_hi_sw128(1024);
      const uint32_t q_lo = umma_desc_lo(smem_u32(sQ), 16), k_lo = umma_desc_lo(smem_u32(sK), 16);
      const uint32_t v_lo = umma_desc_lo(smem_u32(sV), kKT * 128);  // 64-value blocks of V lie a tile's rows apart
      uint64_t* v_go = masked_kv ? v_ready : v_full;
      int units[2] = {0, 0}, steps[2] = {0, 0};
      // S_t = Q_t K^T of a step
      auto issue_s = [&](int t, const Step& s) -> bool {
        const int i = s.base + s.j, st = i % ST;
        if (s.j == 0) {
          if (!mbar_wait_warp(&q_full[t], units[t] & 1, abort_flag, a.status, 420 + t)) return false;
          ++units[t];
        }
        if (t == 0 && !mbar_wait_warp(&k_full[st], (i / ST) & 1, abort_flag, a.status, 422)) return false;
        tc_fence_after();
        if (one) {
          const uint32_t q_at = q_lo + t * (Cfg::kQBytes >> 4), k_at = k_lo + st * (Cfg::kKvBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * (kQT * 128) + (kk & 3) * 32) >> 4;
            umma_f16_ss(tmem_base + t * kKT, q_at + off, kHi, k_at + off, kHi, idesc_s, kk != 0);
          }
          umma_commit(&s_full[t]);
          if (t == 1 || !s.x.two) umma_commit(&k_empty[st]);
          if (s.j + 1 == s.x.n) umma_commit(&q_empty[t]);
        }
        return true;
      };
      // O_t (+)= P_t V of a step
      auto issue_pv = [&](int t, const Step& s) -> bool {
        const int i = s.base + s.j, st = i % ST;
        const uint32_t v_at = v_lo + st * (Cfg::kKvBytes >> 4);
        if (t == 0 && !mbar_wait_warp(&v_go[st], (i / ST) & 1, abort_flag, a.status, 423)) return false;
#pragma unroll
        for (int c = 0; c < kPChunks; ++c) {
          if (!mbar_wait_warp(&p_full[t * kPChunks + c], steps[t] & 1, abort_flag, a.status, 424 + t)) return false;
          tc_fence_after();
          constexpr int kPer = kKT / 16 / kPChunks;
          if (one) {
#pragma unroll
            for (int kk = c * kPer; kk < (c + 1) * kPer; ++kk)
              umma_f16_ts(tmem_base + 256 + t * 128, tmem_base + t * kKT + kk * 8, v_at + kk * (16 * 128 / 16), kHi, idesc_o,
                          (s.j | kk) != 0);
          }
        }
        ++steps[t];
        if (one) {
          umma_commit(&pv_done[t]);
          if (t == 1 || !s.x.two) umma_commit(&v_empty[st]);
        }
        return true;
      };
      Step cur;
      cur.u = blockIdx.x;
      bool ok = cur.settle(a, sh, ends) && issue_s(0, cur) && (!cur.x.two || issue_s(1, cur));
      while (ok) {
        Step next = cur;
        const bool more = next.advance(a, sh, ends);
        if (!issue_pv(0, cur) || (more && !issue_s(0, next))) break;
        if (cur.x.two && !issue_pv(1, cur)) break;
        if (more && next.x.two && !issue_s(1, next)) break;
        cur = next;
        ok = more;
      }
    } else if (warp == 2) {
      if (masked_kv) {
        // ---------------- values of masked keys ----------------
        Step s;
        s.u = blockIdx.x;
        int vc = 0;
        for (bool ok = s.settle(a, sh, ends); ok; ok = s.advance(a, sh, ends), ++vc) {
          const int st = vc % ST;
          uint32_t w[4];
          tile_mask(a, s.x.b, s.j, s.x.valid, w);
          // every lane waits, so that what TMA wrote is ordered before its stores
          if (!mbar_wait_warp(&v_full[st], (vc / ST) & 1, abort_flag, a.status, 430)) break;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!((w[i] >> lane) & 1)) {
#pragma unroll
              for (int c = 0; c < Cfg::kAtoms; ++c) {
                // a key's 64 values are one 128-byte row of the atom, however its pieces are swizzled
                uint4* row = reinterpret_cast<uint4*>(sV + st * Cfg::kKvBytes + c * (kKT * 128) + (i * 32 + lane) * 128);
#pragma unroll
                for (int e = 0; e < 8; ++e) row[(e + lane) & 7] = make_uint4(0, 0, 0, 0);
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ready[st]);
        }
      }
    }
  } else {
    // ---------------- softmax and output of tile t ----------------
    const int t = (warp >> 2) - 1;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_col = tmem_base + lane_addr + t * kKT;
    const uint32_t o_col = tmem_base + lane_addr + 256 + t * 128;
    const float sl2 = a.scale * kLog2e;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    auto hand_over = [&](int c) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t * kPChunks + c]);
    };
    uint8_t* out = sOut + (warp - 4) * kOutBytes;
    int step = 0;  // key tiles of tile t so far: the phase of its barriers
    bool ok = true;
    for (int u = blockIdx.x; ok && u < sh.units; u += gridDim.x) {
      const Unit x = unit_of(a, sh, ends, u);
      if (t == 1 && !x.two) continue;
      const int valid = x.valid;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < x.n; ++j, ++step) {
        uint32_t w[4];
        bool masked = valid - j * kKT < kKT;
        if (a.key_mask != nullptr) {
          tile_mask(a, x.b, j, valid, w);
          masked = (w[0] & w[1] & w[2] & w[3]) != 0xffffffffu;
        } else if (masked) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int left = valid - j * kKT - i * 32;
            w[i] = left >= 32 ? 0xffffffffu : (left > 0 ? (1u << left) - 1 : 0u);
          }
        }
        if (!mbar_wait_warp(&s_full[t], step & 1, abort_flag, a.status, 440 + t)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[kKT];
#pragma unroll
        for (int c = 0; c < kKT / 32; ++c) tmem_ld32(s_col + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
        tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int c = 0; c < kKT; ++c)
            if (!((w[c / 32] >> (c % 32)) & 1)) s[c] = 0xff800000u;  // -inf
        }
        float mc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mc[i] = __uint_as_float(s[i]);
#pragma unroll
        for (int c = 8; c < kKT; c += 8)
#pragma unroll
          for (int i = 0; i < 8; ++i) mc[i] = fmaxf(mc[i], __uint_as_float(s[c + i]));
        const float mx = fmaxf(fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])), fmaxf(fmaxf(mc[4], mc[5]), fmaxf(mc[6], mc[7])));
        const float m_new = fmaxf(m_run, mx);
        // true where a row sees its first key; false (a NaN) while it has seen none
        const bool need = (m_new - m_run) * sl2 > 8.0f;
        float alpha = 1.f;
        if (need) {
          alpha = ex2_approx((m_run - m_new) * sl2);
          m_run = m_new;
        }
        if (j > 0) {
          // the product before has read P and written O
          if (!mbar_wait_warp(&pv_done[t], (step - 1) & 1, abort_flag, a.status, 442 + t)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        l_run *= alpha;
        const float neg = m_run == -INFINITY ? 0.f : -m_run * sl2;
        const uint64_t negx2 = f2_pack(neg, neg);
        float ls[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        // a rescale of O has to come before the products that follow; without one the chunks of P go at once
        const bool rescale = j > 0 && __any_sync(0xffffffffu, need);
        constexpr int kChunk = kKT / kPChunks;
        uint32_t pk[8];
#pragma unroll
        for (int c = 0; c < kKT; c += 2) {
          float x0, x1;
          const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sl2x2, negx2);
          f2_unpack(x2, x0, x1);
          x0 = ex2_approx(x0);
          x1 = ex2_approx(x1);
          ls[c & 7] += x0;
          ls[(c & 7) + 1] += x1;
          pk[(c / 2) & 7] = pack2(T(), x0, x1);
          if ((c & 15) == 14) tmem_st8(s_col + (c >> 4) * 8, pk);
          if ((c + 2) % kChunk == 0 && c + 2 < kKT && !rescale) hand_over((c + 2) / kChunk - 1);
        }
        l_run += ((ls[0] + ls[1]) + (ls[2] + ls[3])) + ((ls[4] + ls[5]) + (ls[6] + ls[7]));
        if (rescale) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_col + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(o_col + c, o);
          }
          for (int c = 0; c < kPChunks - 1; ++c) hand_over(c);
        }
        hand_over(kPChunks - 1);
      }
      if (!ok) break;
      const int2 at = tile_of(a, sh, x, t);
      const int i_q = at.y + row;
      const bool row_ok = i_q < a.seq_q;
      // no key left: zeros and -inf.  A row of NaN scores has no maximum either, but a sum of NaN, which is its result
      const bool none = m_run == -INFINITY && l_run == 0.f;
      const float inv = none ? 0.f : 1.f / l_run;
      if (x.n > 0) {
        if (!mbar_wait_warp(&pv_done[t], (step - 1) & 1, abort_flag, a.status, 444 + t)) break;
        tc_fence_after();
      }
      uint32_t o[D];
      if (x.n > 0) {
#pragma unroll
        for (int c = 0; c < D; c += 32) tmem_ld32(o_col + c, *reinterpret_cast<uint32_t(*)[32]>(&o[c]));
        tmem_wait_ld();
        tc_fence_before();  // O may be written again once the next P is handed over
      } else {
#pragma unroll
        for (int c = 0; c < D; ++c) o[c] = 0;
      }
#pragma unroll
      for (int c = 0; c < D; c += 64) {
        if (lane == 0) tma_store_wait_read<0>();  // the last store has read the buffer
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {  // 16-byte pieces in the 128-byte swizzle's places
          uint32_t p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            p[e] = pack2(T(), __uint_as_float(o[c + 8 * q + 2 * e]) * inv, __uint_as_float(o[c + 8 * q + 2 * e + 1]) * inv);
          *reinterpret_cast<uint4*>(out + lane * 128 + ((q ^ (lane & 7)) * 16)) = make_uint4(p[0], p[1], p[2], p[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (at.y + quarter * 32 < a.seq_q) tma_store_3d(&maps.o, at.x * D + c, at.y + quarter * 32, x.b, out);
          tma_store_commit();
        }
      }
      if (row_ok && a.lse != nullptr)
        a.lse[(static_cast<int64_t>(x.b) * a.heads + at.x) * a.seq_q + i_q] =
            none ? -INFINITY : m_run * a.scale + logf(l_run);
    }
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
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<512>(tmem_base);
  }
}

template <typename T, int D>
void launch_tiles(const CrossAttnArgs& a, cudaStream_t s) {
  using Cfg = TileCfg<D>;
  auto kern = cross_tile_kernel<T, D>;
  static std::atomic<uint64_t> allowed{0};
  allow_smem(kern, Cfg::kSmemBytes, allowed);
  TileMaps maps;
  TileShape sh;
  // a dimension of one entry, or a batch stride of 0, reads entry 0 alone: its stride is not used
  auto map = [&](const void* p, int rows, int heads, int64_t row, int64_t batch, uint32_t box, int& shared) {
    shared = a.batch == 1 || batch == 0;
    const uint64_t width = static_cast<uint64_t>(heads) * D;
    const uint64_t r = rows == 1 ? width : row;
    return make_tmap_16bit_3d(p, shared ? 1 : a.batch, rows, width, r, shared ? r * rows : batch, box);
  };
  maps.q = map(a.q, a.seq_q, a.heads, a.q_row, a.q_batch, kQT, sh.q_shared);
  maps.k = map(a.k, a.seq_k, a.heads_kv, a.k_row, a.k_batch, kKT, sh.k_shared);
  maps.v = map(a.v, a.seq_k, a.heads_kv, a.v_row, a.v_batch, kKT, sh.v_shared);
  const uint64_t width = static_cast<uint64_t>(a.heads) * D;
  const uint64_t o_row = a.seq_q == 1 ? width : a.o_row;
  maps.o = make_tmap_16bit_3d(a.o, a.batch, a.seq_q, width, o_row, a.batch == 1 ? o_row * a.seq_q : a.o_batch, 32);
  const int q_tiles = (a.seq_q + kQT - 1) / kQT;
  sh.group = a.heads / a.heads_kv;
  sh.tiles = q_tiles * sh.group;
  const int pairs = (sh.tiles + 1) / 2;
  const int64_t units = static_cast<int64_t>(pairs) * a.heads_kv * a.batch;
  if (units > 0x3fffffff) throw std::runtime_error("cross_attention: too many queries");
  sh.units = static_cast<int>(units);
  sh.pairs = FastDiv(pairs);
  sh.heads_kv = FastDiv(a.heads_kv);
  sh.q_tiles = FastDiv(q_tiles);
  sh.listed = (a.kv_lens != nullptr || a.key_mask != nullptr) && a.batch <= kListed &&
              (a.key_mask == nullptr || static_cast<int64_t>(a.batch) * a.seq_k <= kListedMask);
  const int sms = device_sm_count();
  kern<<<units < sms ? sh.units : sms, kTileThreads, Cfg::kSmemBytes, s>>>(maps, a, sh);
}

// The form that takes less time, by what both were measured to take in us (in a graph, 1 to 5 batch entries, 4 to 24
// heads of 64 and 128, 1 to 300 queries, 64 to 4096 keys):
//   few rows   1.5 (3 with split keys) + waves * (2 + passes over 128 keys)
//   tiles      3.2 + rounds of units * (1.2 + 1.65 a key tile)
// e.g. 64 queries of 2 x 12 heads over 1024 keys 12.2 and 17.9, 300 queries of 4 heads over 300 keys 7.6 and 11.2, 128
// queries of 2 x 12 heads over 300 keys 13.2 and 10.1.
bool few_is_faster(const CrossAttnArgs& a) {
  const int group = a.heads / a.heads_kv;
  const int64_t heads = static_cast<int64_t>(a.heads_kv) * a.batch;
  const int64_t few = (static_cast<int64_t>(a.seq_q) * group + kFewRows - 1) / kFewRows * heads;
  const int split = few_split(few, a.seq_k, a.head_dim);
  const int64_t slots = few_slots(a.head_dim), sms = device_sm_count();
  const double waves = static_cast<double>((few * split + slots - 1) / slots);
  const double passes = (a.seq_k + split * kFewWarps * 16 - 1) / (split * kFewWarps * 16);
  const int64_t units = ((static_cast<int64_t>(a.seq_q) + kQT - 1) / kQT * group + 1) / 2 * heads;
  const double rounds = static_cast<double>((units + sms - 1) / sms);
  return (split > 1 ? 3.0 : 1.5) + waves * (2.0 + passes) < 3.2 + rounds * (1.2 + 1.65 * ((a.seq_k + kKT - 1) / kKT));
}

template <typename T, int D>
void launch_dim(const CrossAttnArgs& a, cudaStream_t s) {
  if (few_is_faster(a)) launch_few<T, D>(a, s);
  else launch_tiles<T, D>(a, s);
}

template <typename T>
void launch_type(const CrossAttnArgs& a, cudaStream_t s) {
  if (a.head_dim == 128) launch_dim<T, 128>(a, s);
  else launch_dim<T, 64>(a, s);
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
