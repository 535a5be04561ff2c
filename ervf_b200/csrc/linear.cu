// linear.cu -- dense projection with its epilogue on the sm_100a tensor cores:
//
//   out[t][r] = act(sum_k W[r][k] x[t][k] + bias[r]) + resid[t][r]
//
// W, x bf16, products exact, sums and the whole epilogue in f32, one rounding
// to the output's type.  Both operands are K-major, so one kernel serves both
// orientations: the MMA's 128 rows are tokens and its columns features, or
// (few tokens) its rows are features and its columns tokens.
//
// Warp specialised, one CTA per SM; a k-block is 64 columns (128 bytes of a
// row, the swizzle's width):
//   warp 0      producer: TMA of both operands' tiles into a ring of stages
//   warp 1      one lane issues the tcgen05.mma of each stage into one of two
//               accumulator buffers in tensor memory
//   the others  epilogue: tcgen05.ld of a finished buffer (two warps a quarter
//               of its lanes, half the columns each), bias, activation,
//               residual, store -- while the next tile's MMAs run; bias and
//               residual are loaded one step ahead
// Three forms of it:
//   few tokens (rows = features): bound by reading W from HBM.  Each of a
//     k-block's four MMAs has an accumulator of its own, added in the epilogue:
//     the tensor core's sums lose a little with every step (4.4e-6 of the results'
//     norm over 4096 columns in one chain, 1.0e-6 in four).
//   more tokens than 64: 128 x 128 or 128 x 256 tiles.  Where these are fewer
//     than the SMs, a tile's k-blocks are dealt to a cluster of CTAs, whose sums
//     meet in shared memory and are added in rank order.  Bound by what L2
//     delivers to an SM (about 55 bytes a clock) and a start and end of 4 to 6 us
//     (512 x 3712 x 64: 4.5 and 5.7 us).
//   many tokens: a pair of CTAs computes a 256 x 256 tile (cta_group::2); each
//     holds its 128 rows of x and half of W's.  Bound by the tensor cores and
//     by what L2 delivers: 64 bytes a clock and SM at full rate, where a single
//     CTA's 128 x 256 tile takes 96.
// Every wait is bounded: one that runs out records kErrTimeout, marks the CTA
// dead, and every role drains before tensor memory is freed.
#include <cuda.h>  // CUtensorMap and the encode function's types (driver entry point)
#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "ssm_dev.cuh"

namespace ervf {

namespace {

constexpr int kLinM = 128, kLinKB = 64;
constexpr int kLinEpi = 8, kLinThreads = (2 + kLinEpi) * 32;
constexpr int kLinATile = kLinM * kLinKB * 2;
constexpr int kLinStage = 4096, kLinPitch = 20;  // an epilogue warp's staging, bytes; its row in lin_ragged, floats
constexpr int kLinPart = 32 * 32 * 4;            // a part of a tile's sums, 32 x 32

template <int BN, int CH>
struct LinShape {
  static constexpr int kBTile = BN * kLinKB * 2;
  static constexpr int kStage = kLinATile + kBTile;  // both multiples of 1024 bytes (swizzle period)
  static constexpr int kStages = (200 * 1024) / kStage > 8 ? 8 : (200 * 1024) / kStage;
  static constexpr int kSmem = 1024 + 1024 + kStages * kStage + kLinEpi * kLinStage;  // barriers, alignment slack, ring, staging
  static constexpr int kTmemCols = 2 * CH * BN;  // buffer d, chain c at columns (d CH + c) BN
  static_assert(BN % 16 == 0 && BN <= 256 && kTmemCols >= 32 && kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0,
                "tile");
  // ceil(parts / splits) splits parts, 8 splits at most
  static_assert((BN / 8 + 7) * kLinPart <= kStages * kStage, "a split's sums fit the ring");
};

struct LinTile {
  const float* bias;
  const void* resid;
  void* out;
  long long resid_stride, out_stride;
  int rows, cols, tokens;
  int act;
  int nkb, mtiles, ntiles, splits;
  int vec;  // out and resid take 16-byte accesses at every 16th feature
  int whole;  // features in whole 16-byte pieces
};

// Unit u's tile: along bands of eight tiles of M, so that the tiles in work at a
// time share both operands' rows in L2.
__device__ __forceinline__ void lin_place(const LinTile& a, int u, int& mt, int& nt) {
  constexpr int kBand = 8;
  const int per = kBand * a.ntiles, band = u / per, first = band * kBand, size = min(a.mtiles - first, kBand);
  u -= band * per;
  nt = u / size;
  mt = first + u - nt * size;
}

__device__ __forceinline__ uint64_t lin_desc(uint32_t saddr) {
  // K-major, 128-byte swizzle: 8-row groups 1024 bytes apart
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void lin_tma(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void lin_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("{\n .reg .b64 st;\n mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n}"
               ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void lin_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// The wait in the same statement: nothing may use the registers before it.
__device__ __forceinline__ void lin_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr) : "memory");
}

// Bounded wait that also gives up when another role of the CTA died.
__device__ __noinline__ bool lin_wait_slow(uint32_t bar, uint32_t parity, volatile int* dead) {
  const long long t0 = clock64();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if (*dead) return false;
    if (clock64() - t0 > 2000000000LL) {
      atomicExch(&g_device_error, kErrTimeout);
      *dead = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool lin_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok || lin_wait_slow(bar, parity, dead);
}
__device__ __forceinline__ bool lin_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  return lin_wait(smem_u32(bar), parity, dead);
}
// The same for a whole warp: one decision.  Warps that work as one look at
// `dead` nowhere else, or a lane could leave a loop without the others and the
// next warp-wide instruction wait for ever.
__device__ __forceinline__ bool lin_wait_w(uint64_t* bar, uint32_t parity, volatile int* dead) {
  return __all_sync(0xffffffffu, lin_wait(bar, parity, dead));
}

// A place in a ring of N stages: the producer's and the issuing thread's loops
// are one thread's, so their few instructions a k-block are what a k-block
// costs at least.
template <int N>
struct Ring {
  uint32_t s = 0, parity;
  __device__ explicit Ring(uint32_t p) : parity(p) {}
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      parity ^= 1;
    }
  }
};

// One branch for all N values.
template <int N>
__device__ __forceinline__ void lin_act(float (&v)[N], int act) {
  if (act == kActRelu2) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float r = v[i] < 0.0f ? 0.0f : v[i];  // a NaN stays one
      v[i] = r * r;
    }
  } else if (act == kActSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = silu(v[i]);
  } else if (act == kActGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.70710678118654752f));
  }
}

template <typename T>
__device__ __forceinline__ float lin_get(const T* p) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(*p);
  else return *p;
}
template <typename T>
__device__ __forceinline__ void lin_put(T* p, float v) {
  if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(v);
  else *p = v;
}

// The bias of 32 features from r, a lane's one.
__device__ __forceinline__ float lin_bias(const LinTile& a, int r) {
  r += threadIdx.x & 31;
  return a.bias && r < a.rows ? a.bias[r] : 0.0f;
}

// The epilogue of 16 features of one token, a lane's; the residual is loaded
// ahead of the sums.
template <typename T>
struct LinEdge {
  static constexpr int kWords = 16 * sizeof(T) / 4;
  uint32_t resid[kWords];
  __device__ __forceinline__ void load(const LinTile& a, int t, int r) {
    if (!a.vec) return;
    const bool whole = r + 16 <= a.rows;
    if (a.resid && t < a.tokens) {
      const T* q = static_cast<const T*>(a.resid) + (size_t)t * a.resid_stride + r;
      if (whole) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
          const uint4 v = reinterpret_cast<const uint4*>(q)[i / 4];
          resid[i] = v.x; resid[i + 1] = v.y; resid[i + 2] = v.z; resid[i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          if constexpr (sizeof(T) == 2) {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(q) + 2 * i;
            resid[i] = (r + 2 * i < a.rows ? h[0] : 0u) | (r + 2 * i + 1 < a.rows ? (uint32_t)h[1] << 16 : 0u);
          } else {
            resid[i] = r + i < a.rows ? reinterpret_cast<const uint32_t*>(q)[i] : 0u;
          }
        }
      }
    }
  }
  // the 16 results, as they lie in memory; their bias from lane 16 h on
  __device__ __forceinline__ void finish(const LinTile& a, float bias, int h, float (&f)[16],
                                         uint32_t (&w)[kWords]) const {
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] += __shfl_sync(0xffffffffu, bias, 16 * h + i);
    }
    lin_act(f, a.act);
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 2) {
        if (a.resid) {
          f[2 * i] += __uint_as_float(resid[i] << 16);
          f[2 * i + 1] += __uint_as_float(resid[i] & 0xFFFF0000u);
        }
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
      } else {
        w[i] = __float_as_uint(a.resid ? f[i] + __uint_as_float(resid[i]) : f[i]);
      }
    }
  }
};

// 16 features r.. of a warp's tokens t0 .. t0 + 31 where rows have any
// alignment: from shared memory, 16 lanes to a token, an element each.  Against
// tensor stores: 509 x 3712 x 2688 21 us instead of 17, 8192 x 2688 x 3712 134 instead
// of 115 in bf16, 150 instead of 116 in f32 (GPU time).
template <typename T>
__device__ __noinline__ void lin_ragged(const LinTile& a, int t0, int r, const float* stage) {
  const int lane = threadIdx.x & 31;
  if (r + (lane & 15) < a.rows) {
    const int f = r + (lane & 15), t = t0 + (lane >> 4);
    const float b = a.bias ? a.bias[f] : 0.0f;
    const T* q = a.resid ? static_cast<const T*>(a.resid) + (size_t)t * a.resid_stride + f : nullptr;
    T* o = static_cast<T*>(a.out) + (size_t)t * a.out_stride + f;
#pragma unroll 1
    for (int i = 0; i < 16; i += 8) {
      float v[8], res[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        res[k] = q && t + 2 * (i + k) < a.tokens ? lin_get(q + (size_t)(2 * (i + k)) * a.resid_stride) : 0.0f;
        v[k] = stage[(2 * (i + k) + (lane >> 4)) * kLinPitch + (lane & 15)] + b;
      }
      lin_act(v, a.act);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (t + 2 * (i + k) < a.tokens) lin_put(o + (size_t)(2 * (i + k)) * a.out_stride, q ? v[k] + res[k] : v[k]);
    }
  }
  __syncwarp();
}

// 16 features r.. of a warp's 32 tokens, the first (h 0) or second half of 32
// that leave by one tensor store, which cuts them at the output's edges: a row
// of 32 lies in the staging buffer as the store's swizzle has it (64 bytes of
// bf16, 128 of f32).  Stores from registers, 32 bytes a row, took 1000 clocks for
// what takes 570 so: their addresses and branches, with two to four warps a
// scheduler to hide them (18944 x 1024 x 64: 21.8 -> 15.1 us).
template <typename T>
__device__ __forceinline__ void lin_store(const LinTile& a, const CUtensorMap* map, const LinEdge<T>& e, float bias,
                                          int t0, int r, int h, float (&f)[16], uint8_t* stage) {
  const int lane = threadIdx.x & 31;
  if (!a.vec) {
    float* p = reinterpret_cast<float*>(stage);
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<float4*>(p + lane * kLinPitch + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    __syncwarp();
    lin_ragged<T>(a, t0, r, p);
    return;
  }
  uint32_t w[LinEdge<T>::kWords];
  e.finish(a, bias, h, f, w);
  if (h == 0) {  // the store before has read the buffer
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
  }
  constexpr int kRow = 32 * sizeof(T), kHalf = kRow / 32;  // 16-byte pieces of 16 features
  const int turn = kRow == 64 ? (lane >> 1) & 3 : lane & 7;
#pragma unroll
  for (int i = 0; i < kHalf; ++i)
    *reinterpret_cast<uint4*>(stage + lane * kRow + (((kHalf * h + i) ^ turn) << 4)) =
        make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  if (h == 1) {
    // a tensor store cuts at 16 bytes: the features behind the last whole piece
    // are stored one by one
    if (a.whole < a.rows && a.whole >= r - 16 && a.whole < r + 16 && t0 + lane < a.tokens) {
      const uint8_t* row = stage + lane * kRow;
      T* o = static_cast<T*>(a.out) + (size_t)(t0 + lane) * a.out_stride;
      const int piece = (a.whole - (r - 16)) * (int)sizeof(T) / 16 ^ turn;
#pragma unroll 1
      for (int i = a.whole; i < a.rows; ++i) o[i] = reinterpret_cast<const T*>(row + piece * 16)[i - a.whole];
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0 && t0 < a.tokens && r - 16 < a.whole)
      asm volatile(
          "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n"
          "cp.async.bulk.commit_group;"
          ::"l"(map), "r"(r - 16), "r"(t0), "r"(smem_u32(stage)) : "memory");
  }
}
// Behind a warp's last store: shared memory may go.
__device__ __forceinline__ void lin_stored() {
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}

// Feature m of token t, behind its activation.
template <typename T>
__device__ __forceinline__ void lin_one(const LinTile& a, int t, int m, float v) {
  if (a.resid) v += lin_get(static_cast<const T*>(a.resid) + (size_t)t * a.resid_stride + m);
  lin_put(static_cast<T*>(a.out) + (size_t)t * a.out_stride + m, v);
}

__device__ __forceinline__ float lin_remote(const float* p, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
// A cluster shares a tile's k-blocks.  Of the tile's parts of 32 x 32 (part
// 4 c + q: 32 columns, rows 32 q ..) CTA (or pair) k % splits gets everyone's sums
// of the k-th, in its ring, whose tiles are used up by then: four columns of a
// row together.  Half h of part k's columns of a lane's row, sent there:
__device__ __forceinline__ void lin_send(const uint8_t* ring, int k, int h, int splits, int from, int to_rank,
                                         const float (&f)[16]) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(at)
      : "r"(smem_u32(ring) + (k / splits * splits + from) * kLinPart + h * (kLinPart / 2) + (threadIdx.x & 31) * 16),
        "r"(to_rank));
#pragma unroll
  for (int i = 0; i < 16; i += 4)
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                 ::"r"(at + i * 128), "f"(f[i]), "f"(f[i + 1]), "f"(f[i + 2]), "f"(f[i + 3]) : "memory");
}
// and the sum of this CTA's i-th part, in the order of the CTAs
__device__ __forceinline__ void lin_sum(const uint8_t* ring, int i, int h, int splits, float (&f)[16]) {
  const uint8_t* at = ring + i * splits * kLinPart + h * (kLinPart / 2) + (threadIdx.x & 31) * 16;
#pragma unroll
  for (int j = 0; j < 16; ++j) f[j] = 0.0f;
#pragma unroll 2
  for (int r = 0; r < splits; ++r, at += kLinPart) {
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const float4 v = *reinterpret_cast<const float4*>(at + j * 128);
      f[j] += v.x; f[j + 1] += v.y; f[j + 2] += v.z; f[j + 3] += v.w;
    }
  }
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CH accumulator chains a buffer; SPLIT: a cluster shares one tile's k-blocks.
template <int BN, int CH, bool SWAP, bool SPLIT, typename T>
__global__ void __launch_bounds__(kLinThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map,
                  const __grid_constant__ CUtensorMap out_map, const __grid_constant__ LinTile a) {
  using Sh = LinShape<BN, CH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + Sh::kStages;
  uint64_t* dfull = empty + Sh::kStages;
  uint64_t* dempty = dfull + 2;
  uint64_t* mma_done = dempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 512);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + 516);
  uint8_t* ring = smem + 1024;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) |
                             ((uint32_t)(kLinM >> 4) << 24);

  if (tid == 0) {
    for (int i = 0; i < Sh::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&dfull[i], 1);
      mbar_init(&dempty[i], kLinEpi);
    }
    mbar_init(mma_done, 1);
    *dead = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(tmem_slot)), "r"(Sh::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  // SPLIT: one unit a cluster, this CTA's share of its k-blocks
  const int rank = SPLIT ? (int)(blockIdx.x % a.splits) : 0;
  const int units = a.mtiles * a.ntiles, u0 = SPLIT ? blockIdx.x / a.splits : blockIdx.x;
  const int step = SPLIT ? units : (int)gridDim.x;
  const int kb0 = SPLIT ? a.nkb * rank / a.splits : 0, kb1 = SPLIT ? a.nkb * (rank + 1) / a.splits : a.nkb;

  const uint32_t ring_at = smem_u32(ring), full_at = smem_u32(full), empty_at = smem_u32(empty);
  if (warp == 0) {
    if (lane == 0) {
      Ring<Sh::kStages> r(1);
      uint32_t loads = 0;
      for (int u = u0; u < units && !*dead; u += step) {
        const int my = u % a.mtiles * kLinM, ny = u / a.mtiles * BN;
#pragma unroll 1
        for (int kb = kb0; kb < kb1; ++kb, r.next(), ++loads) {
          if (!lin_wait(empty_at + 8 * r.s, r.parity, dead)) break;
          const uint32_t bar = full_at + 8 * r.s, st = ring_at + r.s * Sh::kStage;
          lin_expect(bar, Sh::kStage);
          lin_tma(st, &a_map, kb * kLinKB, my, bar);
          lin_tma(st + kLinATile, &b_map, kb * kLinKB, ny, bar);
        }
      }
      // leave no tensor copy in flight, in a dead CTA neither: these waits, bounded
      // too, end by the copies' arrival and not by the flag
      for (uint32_t k = loads > (uint32_t)Sh::kStages ? loads - Sh::kStages : 0; k < loads; ++k)
        mbar_wait(&full[k % Sh::kStages], (k / Sh::kStages) & 1, 200000000LL);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      Ring<Sh::kStages> r(0);
      const uint64_t da0 = lin_desc(ring_at), db0 = lin_desc(ring_at + kLinATile);
      int nu = 0;
      for (int u = u0; u < units && !*dead; u += step, ++nu) {
        const int d = nu & 1;
        if (!lin_wait(&dempty[d], ((nu >> 1) & 1) ^ 1, dead)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        bool ok = true;
#pragma unroll 1
        for (int kb = kb0; kb < kb1; ++kb, r.next()) {
          if (!lin_wait(full_at + 8 * r.s, r.parity, dead)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t da = da0 + r.s * (Sh::kStage >> 4), db = db0 + r.s * (Sh::kStage >> 4);
#pragma unroll
          for (int j = 0; j < kLinKB / 16; ++j) {
            const uint32_t acc = kb > kb0 || j >= CH ? 1u : 0u;
            asm volatile(
                "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                ::"r"(tmem + (uint32_t)((d * CH + j % CH) * BN)), "l"(da + 2 * j), "l"(db + 2 * j), "r"(idesc),
                  "r"(acc) : "memory");
          }
          lin_commit(empty_at + 8 * r.s);
        }
        if (!ok) break;
        lin_commit(smem_u32(&dfull[d]));
      }
      // every MMA is complete before tensor memory is freed
      lin_commit(smem_u32(mma_done));
      mbar_wait(mma_done, 0, 2000000000LL);
    }
  } else {
    const int q = warp & 3;  // tensor-memory lanes 32 q ..
    uint8_t* stage = ring + Sh::kStages * Sh::kStage + (warp - 2) * kLinStage;
    // 16 columns of buffer d, its chains added in order
    auto sums = [&](int d, int c, float (&f)[16]) {
#pragma unroll
      for (int h = 0; h < CH; ++h) {
        uint32_t v[16];
        lin_ld16(tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)((d * CH + h) * BN + c), v);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = h ? f[i] + __uint_as_float(v[i]) : __uint_as_float(v[i]);
      }
    };
    constexpr int kCols = BN >= 32 ? BN / 2 : BN;  // columns of a warp
    const int c0 = (warp - 2) / 4 * kCols;
    if constexpr (SPLIT && !SWAP) {
      const bool ok = lin_wait_w(&dfull[0], 0, dead);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      cluster_sync();  // every CTA's ring is used up
#pragma unroll 1
      for (int c = c0; ok && c < c0 + kCols; c += 16) {
        float f[16];
        sums(0, c, f);
        const int k = c / 32 * 4 + q;
        lin_send(ring, k, (c >> 4) & 1, a.splits, rank, k % a.splits, f);
      }
      cluster_sync();
      const int mt = u0 % a.mtiles, nt = u0 / a.mtiles;
      for (int i = warp - 2, k; (k = i * a.splits + rank) < BN / 8; i += kLinEpi)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t0 = mt * kLinM + 32 * (k & 3), r = nt * BN + (k >> 2) * 32 + 16 * h;
          LinEdge<T> e;
          e.load(a, t0 + lane, r);
          const float bias = lin_bias(a, r - 16 * h);
          float f[16];
          lin_sum(ring, i, h, a.splits, f);
          lin_store<T>(a, &out_map, e, bias, t0, r, h, f, stage);
        }
      lin_stored();
    } else {
      int nu = 0;
      for (int u = u0; u < units; u += step, ++nu) {
        const int mt = u % a.mtiles, nt = u / a.mtiles, d = nu & 1;
        const int m = mt * kLinM + 32 * q + lane;
        LinEdge<T> pre;
        float bias = 0.0f;
        if constexpr (!SPLIT) {
          if constexpr (SWAP) bias = a.bias && m < a.rows ? a.bias[m] : 0.0f;
          else pre.load(a, m, nt * BN + c0), bias = lin_bias(a, nt * BN + c0);
        }
        if (!lin_wait_w(&dfull[d], (nu >> 1) & 1, dead)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (SWAP) {
#pragma unroll 1
          for (int c = c0; c < c0 + kCols; c += 16) {
            float f[16];
            sums(d, c, f);
            if constexpr (SPLIT) {
              // all MMAs are done: the ring holds the sums, [column][row]
              float* part = reinterpret_cast<float*>(ring) + (size_t)c * kLinM + 32 * q + lane;
#pragma unroll
              for (int i = 0; i < 16; ++i) part[i * kLinM] = f[i];
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i] += bias;
              lin_act(f, a.act);
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (m < a.rows && nt * BN + c + i < a.tokens) lin_one<T>(a, nt * BN + c + i, m, f[i]);
            }
            __syncwarp();
          }
        } else {
#pragma unroll 1
          for (int c = c0; c < c0 + kCols; c += 32) {
            const float b = bias;
            if (c + 32 < c0 + kCols) bias = lin_bias(a, nt * BN + c + 32);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = nt * BN + c + 16 * h;
              LinEdge<T> ahead;
              if (c + 16 * h + 16 < c0 + kCols) ahead.load(a, m, r + 16);
              float f[16];
              sums(d, c + 16 * h, f);
              lin_store<T>(a, &out_map, pre, b, m - lane, r, h, f, stage);
              pre = ahead;
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&dempty[d]);  // the buffer is read
      }
      if constexpr (!SWAP) lin_stored();
    }
  }
  if constexpr (SPLIT && !SWAP) {
    if (warp < 2) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else if constexpr (SPLIT) {
    __syncwarp();
    cluster_sync();
    if (warp >= 2) {
      // this rank's share of the tile's columns, dealt to its warps
      const int q = warp & 3, mt = u0 % a.mtiles, nt = u0 / a.mtiles, m = mt * kLinM + 32 * q + lane;
      const int who = rank + a.splits * ((warp - 2) / 4), all = a.splits * (kLinEpi / 4);
      const float* part = reinterpret_cast<const float*>(ring) + 32 * q + lane;
      const int cols = min(BN, a.tokens - nt * BN);
      const float bias = a.bias && m < a.rows ? a.bias[m] : 0.0f;
      for (int c = who; c < cols; c += all) {
        float v[8], f[1] = {0.0f};
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = r < a.splits ? lin_remote(part + (size_t)c * kLinM, r) : 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) f[0] += v[r];  // in rank order
        f[0] += bias;
        lin_act(f, a.act);
        if (m < a.rows) lin_one<T>(a, nt * BN + c, m, f[0]);
      }
    }
    __syncwarp();
    cluster_sync();  // the others have read this CTA's sums
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::kTmemCols) : "memory");
}

// ------------------------------------------------------- a pair of CTAs

// One 256 x 256 tile by two CTAs: each loads its 128 rows of x and half of the
// tile's 256 rows of W; the even one issues the MMAs of both.
// Eight epilogue warps leave room for a sixth stage and have registers enough
// (8192 x 2688 x 3712 with bias and f32 residual: 159 us with sixteen, 144 with
// eight); a split's sums, which nothing overlaps, are faster with sixteen (509 x
// 3712 x 2688: 19.0 us instead of 19.9).
constexpr int kPairTile = 128 * kLinKB * 2;  // x's part in one CTA
constexpr int kPairStage = kPairTile + 128 * kLinKB * 2;
template <bool SPLIT>
struct PairShape {
  static constexpr int kEpi = SPLIT ? 16 : 8, kThreads = (2 + kEpi) * 32, kStages = SPLIT ? 5 : 6;
  static constexpr int kSmem = 2048 + kStages * kPairStage + kEpi * kLinStage;
  static_assert((256 / 8 + 3) * kLinPart <= kStages * kPairStage, "a split's sums fit the ring");
};

__device__ __forceinline__ uint32_t remote_addr(const void* p, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  return at;
}
// This GPU's own memory only, into this CTA; the bytes count at the even CTA's barrier.
__device__ __forceinline__ void pair_tma(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// Arrives at the same barrier of both CTAs, the even one of which is `lead`.
__device__ __forceinline__ void pair_commit(uint32_t bar, int lead) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"((uint16_t)(3 << lead)) : "memory");
}

// SPLIT: a cluster of pairs shares one tile's k-blocks.
template <bool SPLIT, typename T>
__global__ void __launch_bounds__(PairShape<SPLIT>::kThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map,
                       const __grid_constant__ CUtensorMap out_map, const __grid_constant__ LinTile a) {
  constexpr int BN = 256, kPairEpi = PairShape<SPLIT>::kEpi, kPairStages = PairShape<SPLIT>::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);  // counted at the even CTA
  uint64_t* empty = full + kPairStages;                // one each
  uint64_t* dfull = empty + kPairStages;               // one each
  uint64_t* dempty = dfull + 2;                        // counted at the even CTA
  uint64_t* mma_done = dempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 512);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + 516);
  uint8_t* ring = smem + 1024;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x & 1;
  // its pair's place in the cluster, and the even CTA's rank there
  const int pair = SPLIT ? (int)(blockIdx.x / 2 % a.splits) : 0, lead = 2 * pair;
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) |
                             (16u << 24);  // M 256

  if (tid == 0) {
    for (int i = 0; i < kPairStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&dfull[i], 1);
      mbar_init(&dempty[i], 2 * kPairEpi);
    }
    mbar_init(mma_done, 1);
    *dead = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(tmem_slot)), "r"(2 * BN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // the other CTA's barriers are there
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int units = a.mtiles * a.ntiles, u0 = SPLIT ? blockIdx.x / (2 * a.splits) : blockIdx.x >> 1;
  const int step = SPLIT ? units : (int)(gridDim.x >> 1);
  const int kb0 = SPLIT ? a.nkb * pair / a.splits : 0, kb1 = SPLIT ? a.nkb * (pair + 1) / a.splits : a.nkb;

  const uint32_t ring_at = smem_u32(ring), full_at = smem_u32(full), empty_at = smem_u32(empty);
  if (warp == 0) {
    if (lane == 0) {
      Ring<kPairStages> r(1);
      const uint32_t lead_full = remote_addr(full, lead);
      uint32_t loads = 0;
      for (int u = u0; u < units && !*dead; u += step) {
        int mt, nt;
        lin_place(a, u, mt, nt);
        const int my = (2 * mt + rank) * 128, ny = nt * BN + rank * (BN / 2);
#pragma unroll 1
        for (int kb = kb0; kb < kb1; ++kb, r.next(), ++loads) {
          if (!lin_wait(empty_at + 8 * r.s, r.parity, dead)) break;
          if (rank == 0) lin_expect(full_at + 8 * r.s, 2 * kPairStage);
          const uint32_t bar = lead_full + 8 * r.s, st = ring_at + r.s * kPairStage;
          pair_tma(st, &x_map, kb * kLinKB, my, bar);
          pair_tma(st + kPairTile, &w_map, kb * kLinKB, ny, bar);
        }
      }
      // leave no tensor copy in flight: each stage's release follows its arrival
      for (uint32_t k = loads > (uint32_t)kPairStages ? loads - kPairStages : 0; k < loads; ++k)
        lin_wait(empty_at + 8 * (k % kPairStages), (k / kPairStages) & 1, dead);
      if (*dead) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      Ring<kPairStages> r(0);
      const uint64_t da0 = lin_desc(ring_at), db0 = lin_desc(ring_at + kPairTile);
      int nu = 0;
      for (int u = u0; u < units && !*dead; u += step, ++nu) {
        const int d = nu & 1;
        if (!lin_wait(&dempty[d], ((nu >> 1) & 1) ^ 1, dead)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        bool ok = true;
#pragma unroll 1
        for (int kb = kb0; kb < kb1; ++kb, r.next()) {
          if (!lin_wait(full_at + 8 * r.s, r.parity, dead)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t da = da0 + r.s * (kPairStage >> 4), db = db0 + r.s * (kPairStage >> 4);
#pragma unroll
          for (int j = 0; j < kLinKB / 16; ++j) {
            asm volatile(
                "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                ::"r"(tmem + (uint32_t)(d * BN)), "l"(da + 2 * j), "l"(db + 2 * j), "r"(idesc), "r"((uint32_t)((kb - kb0) | j))
                : "memory");
          }
          pair_commit(empty_at + 8 * r.s, lead);
        }
        if (!ok) break;
        pair_commit(smem_u32(&dfull[d]), lead);
      }
      // every MMA is complete before tensor memory is freed
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                   ::"r"(smem_u32(mma_done)) : "memory");
      mbar_wait(mma_done, 0, 2000000000LL);
    }
  } else {
    const int q = warp & 3;  // tensor-memory lanes 32 q ..
    constexpr int kCols = BN / (kPairEpi / 4);  // columns of a warp
    const int c0 = (warp - 2) / 4 * kCols;
    uint8_t* stage = ring + kPairStages * kPairStage + (warp - 2) * kLinStage;
    const auto sums = [&](int d, int c, float (&f)[16]) {
      uint32_t v[16];
      lin_ld16(tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(d * BN + c), v);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
    };
    if constexpr (SPLIT) {
      const bool ok = lin_wait_w(&dfull[0], 0, dead);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      cluster_sync();  // every CTA's ring is used up
#pragma unroll 1
      for (int c = c0; ok && c < c0 + kCols; c += 16) {
        float f[16];
        sums(0, c, f);
        const int k = c / 32 * 4 + q;
        lin_send(ring, k, (c >> 4) & 1, a.splits, pair, 2 * (k % a.splits) + rank, f);
      }
      cluster_sync();
      int mt, nt;
      lin_place(a, u0, mt, nt);
      for (int i = warp - 2, k; (k = i * a.splits + pair) < BN / 8; i += kPairEpi)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t0 = (2 * mt + rank) * 128 + 32 * (k & 3), r = nt * BN + (k >> 2) * 32 + 16 * h;
          LinEdge<T> e;
          e.load(a, t0 + lane, r);
          const float bias = lin_bias(a, r - 16 * h);
          float f[16];
          lin_sum(ring, i, h, a.splits, f);
          lin_store<T>(a, &out_map, e, bias, t0, r, h, f, stage);
        }
    } else {
      int nu = 0;
      for (int u = u0; u < units; u += step, ++nu) {
        const int d = nu & 1;
        int mt, nt;
        lin_place(a, u, mt, nt);
        const int m = (2 * mt + rank) * 128 + 32 * q + lane;
        LinEdge<T> pre;
        pre.load(a, m, nt * BN + c0);
        float bias = lin_bias(a, nt * BN + c0);
        if (!lin_wait_w(&dfull[d], (nu >> 1) & 1, dead)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
        for (int c = c0; c < c0 + kCols; c += 32) {
          const float b = bias;
          if (c + 32 < c0 + kCols) bias = lin_bias(a, nt * BN + c + 32);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = nt * BN + c + 16 * h;
            LinEdge<T> ahead;
            if (c + 16 * h + 16 < c0 + kCols) ahead.load(a, m, r + 16);
            float f[16];
            sums(d, c + 16 * h, f);
            lin_store<T>(a, &out_map, pre, b, m - lane, r, h, f, stage);
            pre = ahead;
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0)  // the buffer is read
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_addr(&dempty[d], lead)) : "memory");
      }
    }
    lin_stored();
  }
  if constexpr (SPLIT) {
    if (warp < 2) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  __syncwarp();
  cluster_sync();  // nothing of the other CTA reads or signals here any more
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
}

// ------------------------------------------------------------------- host

typedef CUresult (*LinEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

LinEncodeFn lin_encode_fn() {
  static LinEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (LinEncodeFn) nullptr;
    return reinterpret_cast<LinEncodeFn>(p);
  }();
  return fn;
}

// bf16 [rows][cols] with rows `stride` elements apart, boxes of box_rows x 64
// columns, 128-byte swizzle, zeros past the edges.
int lin_map(CUtensorMap* map, const uint16_t* p, int rows, int cols, long long stride, int box_rows) {
  LinEncodeFn enc = lin_encode_fn();
  if (!enc) return kErrLaunch;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t box[2] = {kLinKB, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t*>(p), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? kOk
             : kErrArg;
}

int lin_whole(const LinearArgs& l) { return l.rows & ~(l.out_type == kTypeBF16 ? 7 : 3); }

// The output, boxes of 32 tokens x 32 features, swizzled by their row's width.
// Where its rows are not on 16-byte boundaries the kernel takes none.
int lin_out_map(CUtensorMap* map, const LinearArgs& l, const CUtensorMap& other, bool vec) {
  if (!vec) {
    *map = other;
    return kOk;
  }
  LinEncodeFn enc = lin_encode_fn();
  if (!enc) return kErrLaunch;
  const bool half = l.out_type == kTypeBF16;
  const cuuint64_t dims[2] = {(cuuint64_t)lin_whole(l), (cuuint64_t)l.tokens};
  const cuuint64_t strides[1] = {(cuuint64_t)l.out_stride * (half ? 2 : 4)};
  const cuuint32_t box[2] = {32, 32};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, half ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, l.out, dims, strides,
             box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, half ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? kOk
             : kErrArg;
}

int lin_vec(const LinearArgs& l) {
  const unsigned long long e = l.out_type == kTypeBF16 ? 2 : 4;
  const unsigned long long all = reinterpret_cast<uintptr_t>(l.out) | reinterpret_cast<uintptr_t>(l.resid) |
                                 l.out_stride * e | (l.resid ? l.resid_stride * e : 0);
  return (all & 15) == 0;
}

template <int BN, int CH, bool SWAP, bool SPLIT, typename T>
int linear_run(const LinearArgs& l, int splits, cudaStream_t stream) {
  using Sh = LinShape<BN, CH>;
  LinTile a{l.bias, l.resid, l.out, l.resid_stride, l.out_stride, l.rows, l.cols, l.tokens, l.act, 0, 0, 0, splits, 0, lin_whole(l)};
  a.vec = lin_vec(l) && a.whole > 0;
  a.nkb = (l.cols + kLinKB - 1) / kLinKB;
  const int ma = SWAP ? l.rows : l.tokens, nb = SWAP ? l.tokens : l.rows;
  a.mtiles = (ma + kLinM - 1) / kLinM;
  a.ntiles = (nb + BN - 1) / BN;
  CUtensorMap wm, xm, om;
  if (int e = lin_map(&wm, l.W, l.rows, l.cols, l.cols, SWAP ? kLinM : BN)) return e;
  if (int e = lin_map(&xm, l.x, l.tokens, l.cols, l.x_stride, SWAP ? BN : kLinM)) return e;
  if (int e = lin_out_map(&om, l, xm, !SWAP && a.vec)) return e;
  auto fn = linear_kernel<BN, CH, SWAP, SPLIT, T>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem) != cudaSuccess)
    return kErrLaunch;
  const long long units = (long long)a.mtiles * a.ntiles;
  if (units > 0x3fffffffLL) return kErrShape;
  const int sms = device_sm_count();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(SPLIT ? units * splits : units < sms ? units : sms));
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = Sh::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = SPLIT ? splits : 1;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = SPLIT ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, fn, SWAP ? wm : xm, SWAP ? xm : wm, om, a) == cudaSuccess ? kOk : kErrLaunch;
}

template <bool SPLIT, typename T>
int linear_pair(const LinearArgs& l, int splits, cudaStream_t stream) {
  LinTile a{l.bias, l.resid, l.out, l.resid_stride, l.out_stride, l.rows, l.cols, l.tokens, l.act, 0, 0, 0, splits, 0, lin_whole(l)};
  a.vec = lin_vec(l) && a.whole > 0;
  a.nkb = (l.cols + kLinKB - 1) / kLinKB;
  a.mtiles = (l.tokens + 255) / 256;
  a.ntiles = (l.rows + 255) / 256;
  const long long units = (long long)a.mtiles * a.ntiles;
  if (units > 0x3fffffffLL) return kErrShape;
  CUtensorMap wm, xm, om;
  if (int e = lin_map(&wm, l.W, l.rows, l.cols, l.cols, 128)) return e;
  if (int e = lin_map(&xm, l.x, l.tokens, l.cols, l.x_stride, 128)) return e;
  if (int e = lin_out_map(&om, l, xm, a.vec)) return e;
  using Sh = PairShape<SPLIT>;
  auto fn = linear_pair_kernel<SPLIT, T>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem) != cudaSuccess)
    return kErrLaunch;
  const int pairs = device_sm_count() / 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * (unsigned)(SPLIT ? units * splits : units < pairs ? units : pairs));
  cfg.blockDim = dim3(Sh::kThreads);
  cfg.dynamicSmemBytes = Sh::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2 * splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, xm, wm, om, a) == cudaSuccess ? kOk : kErrLaunch;
}

// Clusters of s CTAs (one an SM) that the current device runs at a time: SMs
// lie in groups that a cluster does not cross, so 21 clusters of 7 do not fit
// 148 SMs at once, though 147 CTAs do.
int linear_clusters(int s) {
  static std::atomic<int> known[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const bool keep = dev < 64;
  if (keep && known[dev][s].load()) return known[dev][s].load() - 1;
  auto fn = linear_kernel<32, 4, true, true, float>;
  constexpr int smem = LinShape<32, 4>::kSmem;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(s);
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = s;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (keep) known[dev][s].store(n + 1);
  return n;
}

// CTAs, or pairs of them (`each` 2), that share a tile's k-blocks: the most (8
// CTAs are a portable cluster) whose clusters all run at once, each CTA with two
// k-blocks or more.
int linear_splits(long long units, int cols, int each = 1) {
  const int nkb = (cols + kLinKB - 1) / kLinKB, most = 8 / each;
  for (int s = nkb / 2 < most ? nkb / 2 : most; s > 1; --s)
    if (units * s * each <= device_sm_count() && units <= linear_clusters(s * each)) return s;
  return 1;
}

template <int BN, int CH, bool SWAP, typename T>
int linear_single(const LinearArgs& l, cudaStream_t stream) {
  const long long ma = SWAP ? l.rows : l.tokens, nb = SWAP ? l.tokens : l.rows;
  const int splits = linear_splits(((ma + kLinM - 1) / kLinM) * ((nb + BN - 1) / BN), l.cols);
  return splits > 1 ? linear_run<BN, CH, SWAP, true, T>(l, splits, stream)
                    : linear_run<BN, CH, SWAP, false, T>(l, 1, stream);
}

template <typename T>
int linear_pick(const LinearArgs& l, cudaStream_t stream) {
  if (l.tokens <= 32) return linear_single<32, 4, true, T>(l, stream);
  if (l.tokens <= 64) return linear_single<64, 4, true, T>(l, stream);
  // Three tiles, by their time in units of 10 ns: a start and an epilogue, the
  // k-blocks that one CTA (pair) goes through, and a split's sums through the
  // cluster.  Measured with W in L2, tokens x features x columns, for 128 x 128,
  // 128 x 256 and pairs' 256 x 256:
  //   96 x 3712 x 2688     10.1   11.7   13.4 us
  //   384 x 3712 x 2688    17.1   14.7   16.0
  //   512 x 2688 x 5376    29.0   21.2   20.0
  //   1024 x 3712 x 2688   31.5   22.2   19.9
  //   2048 x 2688 x 5376   86.0   68.6   60.0
  // Pairs of 256 x 128 were within 5% of the best of these at best.
  const long long sms = device_sm_count(), nkb = (l.cols + kLinKB - 1) / kLinKB;
  const long long t128 = (l.tokens + 127LL) / 128, t256 = (l.tokens + 255LL) / 256;
  const long long r128 = (l.rows + 127LL) / 128, r256 = (l.rows + 255LL) / 256;
  const auto cost = [&](long long units, int each, int start, int kblock, int sums) {
    const int s = linear_splits(units, l.cols, each);
    return start + (units * each + sms - 1) / sms * ((nkb + s - 1) / s) * kblock + (s > 1 ? sums : 0);
  };
  const long long small = cost(t128 * r128, 1, 450, 30, 220), single = cost(t128 * r256, 1, 570, 46, 330);
  const long long pairs = cost(t256 * r256, 2, 680, 33, 330);
  if (pairs <= small && pairs <= single) {
    const int s = linear_splits(t256 * r256, l.cols, 2);
    return s > 1 ? linear_pair<true, T>(l, s, stream) : linear_pair<false, T>(l, 1, stream);
  }
  return small <= single ? linear_single<128, 2, false, T>(l, stream) : linear_single<256, 1, false, T>(l, stream);
}

}  // namespace

int launch_linear(const LinearArgs& l, cudaStream_t stream) {
  return l.out_type == kTypeBF16 ? linear_pick<__nv_bfloat16>(l, stream) : linear_pick<float>(l, stream);
}

int read_linear_device_error(bool clear) { return read_unit_error(clear); }

}  // namespace ervf
