// ssm_chunk.cu -- the selective scan of bf16 prompts on the sm_100a tensor
// cores, in chunks of Q = 128 tokens:
//
//   P[t][s] = (C_t . B_s) exp(c_t - c_s) d_s  for s <= t, + D on the diagonal
//   y_t     = sum_s P[t][s] x_s + exp(c_t) S C_t
//   S'      = exp(c_Q) S + sum_s exp(c_Q - c_s) d_s x_s B_s^T
//
// with c the running sum of d A inside the chunk and S the state before it.
// One CTA per SM walks a list of (head pair, sequence, chunk) steps and carries
// the two heads' state in registers; C B^T is shared by the pair.  The list
// is cut into equal pieces, one per CTA, wherever the cuts fall:
//   pass 1  (WHOLE = false) a CTA whose piece ends inside a sequence computes
//           the state that its own part of that sequence adds, and its decay;
//   pass 2  joins these along each sequence, in order;
//   pass 3  (WHOLE = true) every CTA runs its piece from its true start state.
// Exponents are sums of numbers of one sign (distances within blocks of 32
// tokens plus whole blocks), so no difference of two long sums is taken but
// inside a block.  Products meet the tensor cores in bf16: B, C and x are bf16
// already; P and S are split into two bf16 numbers (off by 2^-16 of the
// value, the output's own rounding is 2^-8), the state's new terms into three
// (2^-24: states stay f32).
//
// Warps, and what bounds them at 128 state columns (clocks per step of two
// heads, measured tcgen05 rates):
//   0..3   P: C B^T from tensor memory, weighted, split, back to tensor memory
//          as an A operand; scales S C by exp(c_t) in tensor memory
//   4..11  states: x scaled and split into the B operand of the state's new
//          terms; the f32 state (64 registers a thread), split for S C
//   12..15 y: tensor memory -> bf16 -> coalesced rows
//   16     TMA of the B, C and x tiles
//   17     all MMAs: C B^T 8 x 65, S C 16 x 69, P x 32 x 68, states 24 x 69
//          = 5460 clocks, which is the step's bound
//   18     steps: softplus, running sums, weights; clears rows behind a
//          sequence's end, so that a neighbour's NaN meets no zero weight
// Every wait is bounded: one that runs out records kErrTimeout, marks the CTA
// dead, and every role leaves; copies and MMAs are drained first.
#include <cuda.h>  // CUtensorMap and the encode function's types (driver entry point)
#include <cuda_bf16.h>

#include "kernels.h"
#include "ssm_dev.cuh"

namespace ervf {

namespace {

constexpr int kQ = 128, kP = 64;          // tokens per chunk, head_dim
constexpr int kPanel = kQ * 128;          // 128 rows of 64 bf16, 128-byte swizzle
constexpr int kHalfPanel = 64 * 128;
constexpr int kChWarps = 19, kChThreads = kChWarps * 32;
constexpr int kMaxCtas = 148;
// tensor-memory columns
constexpr int kTmCB = 0, kTmP = 128, kTmY = 256, kTmS = 384;

struct ChunkArgs {
  Packing pk;
  const __nv_bfloat16* dt;
  const float *A, *D, *dt_bias;
  float* state;
  __nv_bfloat16* y;
  long long dt_stride, y_stride;
  int heads, hpg, ppg, pairs;  // heads, heads and pairs per group, pairs in all
  int n;                       // d_state
  float* local;                // [ctas][2][kP][n]: pass 1's states, joined in place by pass 2
  float* init;                 // [ctas][2][kP][n]: carried states of sequences that are cut
  float* decay;                // [ctas][2]
  int* meta;                   // [ctas]: 0 no cut, 1 from a sequence's start, 2 continued
};

struct Barriers {
  uint64_t raw_b, raw_c, raw_x;   // TMA bytes landed
  uint64_t rdy_b, rdy_x;          // and rows behind the end cleared
  uint64_t sc_full[2], sc_free[2];
  uint64_t cb_full, cb_free, cs_done, p_full, px_done[2], y_free;
  uint64_t w_full[3], w_free[3], ds_done, ds_free, s_full, x_read, mma_done;
};

// Per-token numbers of one head, base-2 exponents.
struct alignas(16) Steps {
  float lp[kQ];  // running sum inside the token's block of 32, inclusive
  float d[kQ];   // softplus step, 0 behind the end
  float v[kQ];   // d exp2(distance to the end of the token's block)
  float w[kQ];   // d exp2(distance to the end of the chunk)
  float blk[4];  // sums of the blocks
  float all;     // exp2(sum of the chunk)
};

template <int N>
struct ChunkSmem {
  static constexpr int kTile = N / 64 * kPanel;    // B or C
  static constexpr int kB = 0, kC = kB + kTile, kX = kC + kTile;
  static constexpr int kS = kX + 2 * kPanel;       // [hi, lo][head][N rows]
  static constexpr int kSPanel = N * 128;
  static constexpr int kW = kS + 4 * kSPanel;      // 3 parts x [head][64 rows]
  static constexpr int kY = kW + 6 * kHalfPanel;   // 4 warps x 2 KB
  static constexpr int kSteps = kY + 4 * 2048;     // [2 buffers][2 heads]
  static constexpr int kBar = (kSteps + 4 * (int)sizeof(Steps) + 15) / 16 * 16;
  static constexpr int kBytes = 1024 + kBar + 512;
};
static_assert(ChunkSmem<128>::kBytes <= 232448, "shared memory");

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Swizzled shared-memory descriptor.  K-major: 8-row groups 1024 bytes apart
// (lbo unused).  MN-major: 64-element panels lbo bytes apart along M or N,
// groups of 8 along K 1024 bytes apart.
__device__ __forceinline__ uint64_t sw_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
constexpr uint32_t ch_idesc(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         ((uint32_t)(n >> 3) << 17) | (8u << 24);  // bf16 x bf16 -> f32, M = 128
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, 1, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(db), "r"(idesc) : "memory");
}
__device__ __forceinline__ void ch_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
               ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t t, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(t));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t t, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
        "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
        "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t t, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void ch_tma(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}

// Bounded wait of one thread; gives up too when another role died.
__device__ __forceinline__ bool ch_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait_sleep(bar, parity, 200)) {
    if (*dead) return false;
    if (clock64() - t0 > 2000000000LL) {
      atomicExch(&g_device_error, kErrTimeout);
      *dead = 1;
      return false;
    }
  }
  return true;
}
// The same for a whole warp: one decision.
__device__ __forceinline__ bool ch_wait_w(uint64_t* bar, uint32_t parity, volatile int* dead) {
  return __all_sync(0xffffffffu, ch_wait(bar, parity, dead));
}
__device__ __forceinline__ void ch_arrive_w(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ int chunks_of(int len) { return (len + kQ - 1) / kQ; }

// A place in the list of steps.
struct Walk {
  int pair, seq, chunk, begin, len, nch;
  __device__ void at(const Packing& pk, int pair_, int seq_, int chunk_) {
    pair = pair_;
    seq = seq_;
    chunk = chunk_;
    seq_range(pk, seq, begin, len);
    nch = chunks_of(len);
  }
  // the next step; there is one
  __device__ void next(const Packing& pk) {
    if (++chunk < nch) return;
    chunk = 0;
    do {
      if (++seq == pk.seqs) {
        seq = 0;
        ++pair;
      }
      seq_range(pk, seq, begin, len);
      nch = chunks_of(len);
    } while (nch == 0);
  }
  __device__ int row0() const { return begin + chunk * kQ; }
  __device__ int valid() const { return min(kQ, len - chunk * kQ); }
};

// First and one-past-last step of CTA c out of g.
__device__ __forceinline__ long long cut(long long steps, int c, int g) { return steps * c / g; }

template <int N, bool WHOLE>
__global__ void __launch_bounds__(kChThreads, 1)
    scan_chunk_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap b_map,
                      const __grid_constant__ CUtensorMap c_map, ChunkArgs a) {
  using Sm = ChunkSmem<N>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  Barriers& br = *reinterpret_cast<Barriers*>(smem + Sm::kBar);
  static_assert(sizeof(Barriers) <= 400, "barrier block");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Sm::kBar + 400);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + Sm::kBar + 404);
  int* first = reinterpret_cast<int*>(smem + Sm::kBar + 408);  // pair, seq, chunk, steps, piece before
  Steps* steps = reinterpret_cast<Steps*>(smem + Sm::kSteps);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, ctas = gridDim.x;

  if (warp == 0) {
    // this CTA's piece of the list
    int seq = 0, nth = 0, total = 0;
    find_tile(a.pk, -1, kQ, 0, seq, nth, total);
    const long long all = (long long)total * a.pairs;
    const long long f0 = cut(all, cta, ctas), f1 = cut(all, cta + 1, ctas);
    int n = (int)(f1 - f0), pair = 0, before = cta - 1;
    if (n > 0)  // the piece before this one: pieces may be empty
      while (before > 0 && cut(all, before, ctas) == f0) --before;
    if (n > 0) {
      int t;
      if (WHOLE) {
        pair = (int)(f0 / total);
        find_tile(a.pk, (int)(f0 - (long long)pair * total), kQ, 0, seq, nth, t);
      } else {
        // its part of the sequence that its piece ends in, if that goes on
        pair = (int)((f1 - 1) / total);
        find_tile(a.pk, (int)(f1 - 1 - (long long)pair * total), kQ, 0, seq, nth, t);
        int b, len;
        seq_range(a.pk, seq, b, len);
        if (nth == chunks_of(len) - 1) {
          n = 0;
        } else {
          n = (int)min((long long)(nth + 1), f1 - f0);
          nth = nth + 1 - n;
        }
      }
    }
    if (lane == 0) {
      first[0] = pair;
      first[1] = seq;
      first[2] = nth;
      first[3] = n;
      first[4] = before;
      if (!WHOLE) a.meta[cta] = n == 0 ? 0 : nth == 0 ? 1 : 2;
      const int cons = WHOLE ? 12 : 8;  // warps that read the steps
      mbar_init(&br.raw_b, 1);
      mbar_init(&br.raw_c, 1);
      mbar_init(&br.raw_x, 1);
      mbar_init(&br.rdy_b, 1);
      mbar_init(&br.rdy_x, 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&br.sc_full[i], 1);
        mbar_init(&br.sc_free[i], cons);
        mbar_init(&br.px_done[i], 1);
      }
      mbar_init(&br.cb_full, 1);
      mbar_init(&br.cb_free, 4);
      mbar_init(&br.cs_done, 1);
      mbar_init(&br.p_full, 4);
      mbar_init(&br.y_free, 4);
      for (int i = 0; i < 3; ++i) {
        mbar_init(&br.w_full[i], 8);
        mbar_init(&br.w_free[i], 1);
      }
      mbar_init(&br.ds_done, 1);
      mbar_init(&br.ds_free, 8);
      mbar_init(&br.s_full, 8);
      mbar_init(&br.x_read, 8);
      mbar_init(&br.mma_done, 1);
      *dead = 0;
      fence_mbar_init();
    }
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_slot;
  const int count = first[3];
  Walk wk;
  if (count > 0) wk.at(a.pk, first[0], first[1], first[2]);
  // heads of a pair; an odd group's last pair has its head twice
  auto head_of = [&](int pair, int h) {
    const int grp = pair / a.ppg, k = (pair - grp * a.ppg) * 2 + h;
    return grp * a.hpg + min(k, a.hpg - 1);
  };
  auto two = [&](int pair) { return (pair % a.ppg) * 2 + 1 < a.hpg; };

  if (warp < 4) {
    // ------------------------------------------------------------------ P
    if (WHOLE && count > 0) {
      const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16);
      {
        // columns behind the diagonal block stay zero
        uint32_t z[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0;
        for (int j = warp + 1; j < 4; ++j) {
          tm_st16(lanes + kTmP + 16 * j, z);
          tm_st16(lanes + kTmP + 64 + 16 * j, z);
        }
        tm_wait_st();
      }
      for (int it = 0; it < count; ++it) {
        const uint32_t ph = it & 1;
        const Steps* st2 = steps + 2 * ph;
        if (!ch_wait_w(&br.sc_full[ph], (it >> 1) & 1, dead)) break;
        if (!ch_wait_w(&br.cb_full, ph, dead)) break;
        tc_after();
        bool ok = true;
        for (int h = 0; h < 2; ++h) {
          const Steps& st = st2[h];
          const int t = 32 * warp + lane;
          const float lp = st.lp[t];
          // the P buffer is free: the last product of it is done
          if (!ch_wait_w(&br.px_done[h ^ 1], h ? ph : ph ^ 1, dead)) {
            ok = false;
            break;
          }
          tc_after();
          float before = lp;  // distance from the end of block j to t
          for (int j = warp; j >= 0; --j) {
            uint32_t v[32], hi[16], lo[16];
            tm_ld32(lanes + kTmCB + 32 * j, v);
            if (j == warp) {
              const float D = a.D ? a.D[head_of(wk.pair, h)] : 0.0f;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float p = __uint_as_float(v[i]) * (st.d[32 * j + i] * ex2(lp - st.lp[32 * j + i]));
                v[i] = __float_as_uint(i < lane ? p : i == lane ? p + D : 0.0f);
              }
            } else {
              const float u = ex2(before);
              before += st.blk[j];
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 q = *reinterpret_cast<const float4*>(&st.v[32 * j + i]);
                v[i] = __float_as_uint(__uint_as_float(v[i]) * (u * q.x));
                v[i + 1] = __float_as_uint(__uint_as_float(v[i + 1]) * (u * q.y));
                v[i + 2] = __float_as_uint(__uint_as_float(v[i + 2]) * (u * q.z));
                v[i + 3] = __float_as_uint(__uint_as_float(v[i + 3]) * (u * q.w));
              }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float e = __uint_as_float(v[2 * i]), o = __uint_as_float(v[2 * i + 1]);
              hi[i] = pack2(e, o);
              lo[i] = pack2(e - lo_f(hi[i]), o - hi_f(hi[i]));
            }
            tm_st16(lanes + kTmP + 16 * j, hi);
            tm_st16(lanes + kTmP + 64 + 16 * j, lo);
          }
          if (h == 1) {
            tc_before();
            ch_arrive_w(&br.cb_free);
          }
          // S C of this head times exp(c_t)
          if (h == 0 && !ch_wait_w(&br.cs_done, ph, dead)) {
            ok = false;
            break;
          }
          tc_after();
          const float e = ex2(before);  // every block before t's, and t's own part
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t v[32];
            tm_ld32(lanes + kTmY + 64 * h + c, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * e);
            tm_st32(lanes + kTmY + 64 * h + c, v);
          }
          tm_wait_st();
          tc_before();
          ch_arrive_w(&br.p_full);
        }
        if (!ok) break;
        ch_arrive_w(&br.sc_free[ph]);
        if (it + 1 < count) wk.next(a.pk);
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------- states
    const int q = warp & 3, half = (warp - 4) >> 2;  // state rows 32 q .., columns 32 half ..
    const int n = 32 * q + lane, wt = tid - 128;
    const bool own = n < N;
    float s[2][32];
    auto put_s = [&]() {
      // both parts of both heads' state as the B operand of S C
      if (own) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = s[h][8 * c + 2 * i], o = s[h][8 * c + 2 * i + 1];
              hi[i] = pack2(e, o);
              lo[i] = pack2(e - lo_f(hi[i]), o - hi_f(hi[i]));
            }
            uint8_t* p = smem + Sm::kS + h * Sm::kSPanel + n * 128 + (((4 * half + c) ^ (n & 7)) << 4);
            *reinterpret_cast<uint4*>(p) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(p + 2 * Sm::kSPanel) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
      }
      to_async();
      ch_arrive_w(&br.s_full);
    };
    // this thread's elements of a pair of states [2][kP][N] or of the heads' slots
    auto elem = [&](float* base, int h, int i) { return base + ((size_t)h * kP + 32 * half + i) * N + n; };
    for (int it = 0; it < count; ++it) {
      const uint32_t ph = it & 1;
      const Steps* st2 = steps + 2 * ph;
      if (wk.chunk == 0 || it == 0) {
        // where the state before this chunk comes from
        const int slot = a.state ? seq_slot(a.pk, wk.seq) : -1;
        const bool carried = slot >= 0 && a.pk.has && a.pk.has[wk.seq];
        const float* src = nullptr;
        bool slots = false;
        if (wk.chunk > 0) {
          if (WHOLE) src = a.local + (size_t)first[4] * 2 * kP * N;
        } else if (carried) {
          // a sequence that another CTA finishes may already have its new state in the slot
          const bool is_cut = WHOLE && wk.nch - wk.chunk > count - it;
          if (is_cut) src = a.init + (size_t)cta * 2 * kP * N;
          else slots = true;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* p = slots ? a.state + ((size_t)slot * a.heads + head_of(wk.pair, h)) * kP * N
                                 : src ? src + (size_t)h * kP * N : nullptr;
#pragma unroll
          for (int i = 0; i < 32; ++i) s[h][i] = p && own ? p[(size_t)(32 * half + i) * N + n] : 0.0f;
          if (!WHOLE && slots && own) {
#pragma unroll
            for (int i = 0; i < 32; ++i) *elem(a.init + (size_t)cta * 2 * kP * N, h, i) = s[h][i];
          }
        }
        if (WHOLE) {
          if (!ch_wait_w(&br.cs_done, ph ^ 1, dead)) break;
          put_s();
        }
      }
      if (!ch_wait_w(&br.sc_full[ph], (it >> 1) & 1, dead)) break;
      if (!ch_wait_w(&br.rdy_x, ph, dead)) break;
      bool ok = true;
      for (int hf = 0; hf < 2; ++hf) {
        // x rows 64 hf .., scaled to the chunk's end, in three bf16 parts
        for (int i = 0; i < 3 && ok; ++i) ok = ch_wait_w(&br.w_free[i], hf ^ 1, dead);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int id = i * 256 + wt, h = id >> 9, r = (id >> 3) & 63, ch = id & 7;
          const int row = 64 * hf + r;
          const float w = st2[h].w[row];
          const uint32_t at = (uint32_t)((ch ^ (r & 7)) << 4);
          const uint4 xv = *reinterpret_cast<const uint4*>(smem + Sm::kX + h * kPanel + row * 128 + at);
          const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
          uint32_t p0[4], p1[4], p2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float e = lo_f(xs[j]) * w, o = hi_f(xs[j]) * w;
            p0[j] = pack2(e, o);
            e -= lo_f(p0[j]);
            o -= hi_f(p0[j]);
            p1[j] = pack2(e, o);
            e -= lo_f(p1[j]);
            o -= hi_f(p1[j]);
            p2[j] = pack2(e, o);
          }
          uint8_t* dst = smem + Sm::kW + h * kHalfPanel + r * 128 + at;
          *reinterpret_cast<uint4*>(dst) = make_uint4(p0[0], p0[1], p0[2], p0[3]);
          *reinterpret_cast<uint4*>(dst + 2 * kHalfPanel) = make_uint4(p1[0], p1[1], p1[2], p1[3]);
          *reinterpret_cast<uint4*>(dst + 4 * kHalfPanel) = make_uint4(p2[0], p2[1], p2[2], p2[3]);
        }
        to_async();
        __syncwarp();
        if (lane == 0)
          for (int i = 0; i < 3; ++i) mbar_arrive(&br.w_full[i]);
      }
      if (!ok) break;
      ch_arrive_w(&br.x_read);
      if (!ch_wait_w(&br.ds_done, ph, dead)) break;
      tc_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[32];
        __syncwarp();
        tm_ld32(tmem + ((uint32_t)(32 * q) << 16) + kTmS + 64 * h + 32 * half, v);
        const float da = st2[h].all;
#pragma unroll
        for (int i = 0; i < 32; ++i) s[h][i] = fmaf(da, s[h][i], __uint_as_float(v[i]));
      }
      tc_before();
      ch_arrive_w(&br.ds_free);
      ch_arrive_w(&br.sc_free[ph]);
      if (WHOLE && wk.chunk == wk.nch - 1) {
        const int slot = a.state ? seq_slot(a.pk, wk.seq) : -1;
        if (slot >= 0 && own)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (h == 0 || two(wk.pair)) {
              float* p = a.state + ((size_t)slot * a.heads + head_of(wk.pair, h)) * kP * N;
#pragma unroll
              for (int i = 0; i < 32; ++i) *elem(p, 0, i) = s[h][i];
            }
      }
      if (it + 1 < count) {
        wk.next(a.pk);
        if (WHOLE && wk.chunk > 0) {
          if (!ch_wait_w(&br.cs_done, ph, dead)) break;
          put_s();
        }
      }
    }
    if (!WHOLE && count > 0 && own) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 32; ++i) *elem(a.local + (size_t)cta * 2 * kP * N, h, i) = s[h][i];
    }
  } else if (warp < 16) {
    // ------------------------------------------------------------------ y
    if (WHOLE) {
      const int q = warp & 3;
      uint8_t* stage = smem + Sm::kY + q * 2048;
      for (int it = 0; it < count; ++it) {
        const uint32_t ph = it & 1;
        bool ok = true;
        for (int h = 0; h < 2; ++h) {
          if (!ch_wait_w(&br.px_done[h], ph, dead)) {
            ok = false;
            break;
          }
          tc_after();
          uint32_t o[32];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            tm_ld32(tmem + ((uint32_t)(32 * q) << 16) + kTmY + 64 * h + 32 * c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              o[16 * c + i] = pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
          }
          if (h == 1) {
            tc_before();
            ch_arrive_w(&br.y_free);
          }
          if (h == 1 && !two(wk.pair)) continue;
          const int left = wk.valid() - 32 * q;  // rows of this warp inside the sequence
          __nv_bfloat16* y = a.y + (size_t)(wk.row0() + 32 * q) * a.y_stride + (size_t)head_of(wk.pair, h) * kP;
          // 16 rows at a time through shared memory: eight lanes store one row's 128 bytes
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            __syncwarp();
            if ((lane >> 4) == g) {
#pragma unroll
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(stage + (lane & 15) * 128 + ((c ^ (lane & 7)) << 4)) =
                    make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = 4 * k + (lane >> 3), c = lane & 7;
              const uint4 val = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
              if (16 * g + r < left)
                *reinterpret_cast<uint4*>(y + (size_t)(16 * g + r) * a.y_stride + 8 * c) = val;
            }
          }
        }
        if (!ok) break;
        if (it + 1 < count) wk.next(a.pk);
      }
    }
  } else if (warp == 16) {
    // ---------------------------------------------------------------- TMA
    if (lane == 0) {
      int it = 0;
      for (; it < count; ++it) {
        const uint32_t ph = it & 1;
        const int grp = wk.pair / a.ppg, row = wk.row0();
        if (WHOLE) {
          if (!ch_wait(&br.cs_done, ph ^ 1, dead)) break;
          mbar_arrive_expect_tx(&br.raw_c, Sm::kTile);
          for (int i = 0; i < N / 64; ++i)
            ch_tma(smem + Sm::kC + i * kPanel, &c_map, grp * N + 64 * i, row, &br.raw_c);
        }
        if (!ch_wait(&br.ds_done, ph ^ 1, dead)) break;
        mbar_arrive_expect_tx(&br.raw_b, Sm::kTile);
        for (int i = 0; i < N / 64; ++i)
          ch_tma(smem + Sm::kB + i * kPanel, &b_map, grp * N + 64 * i, row, &br.raw_b);
        if (WHOLE && !ch_wait(&br.px_done[1], ph ^ 1, dead)) break;
        if (!ch_wait(&br.x_read, ph ^ 1, dead)) break;
        mbar_arrive_expect_tx(&br.raw_x, 2 * kPanel);
        for (int h = 0; h < 2; ++h)
          ch_tma(smem + Sm::kX + h * kPanel, &x_map, head_of(wk.pair, h) * kP, row, &br.raw_x);
        if (it + 1 < count) wk.next(a.pk);
      }
      // no copy is left in flight: wait for every one that was started (a
      // dead CTA's waits return at once, so these go by the clock alone)
      if (*dead) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {
        }
      } else if (count > 0) {
        const uint32_t ph = (count - 1) & 1;
        if (WHOLE) ch_wait(&br.raw_c, ph, dead);
        ch_wait(&br.raw_b, ph, dead);
        ch_wait(&br.raw_x, ph, dead);
      }
    }
  } else if (warp == 17) {
    // --------------------------------------------------------------- MMAs
    if (lane == 0) {
      const uint32_t base = smem_u32(smem);
      constexpr uint32_t id_cb = ch_idesc(128, false, false), id_cs = ch_idesc(128, false, true),
                         id_px = ch_idesc(64, false, true), id_ds = ch_idesc(128, true, true);
      for (int it = 0; it < count; ++it) {
        const uint32_t ph = it & 1;
        if (!ch_wait(&br.rdy_b, ph, dead)) break;
        if (WHOLE) {
          if (!ch_wait(&br.raw_c, ph, dead)) break;
          if (!ch_wait(&br.cb_free, ph ^ 1, dead)) break;
          tc_after();
#pragma unroll
          for (int k = 0; k < N / 16; ++k) {
            const uint32_t o = (k >> 2) * kPanel + (k & 3) * 32;
            mma_ss(tmem + kTmCB, sw_desc(base + Sm::kC + o, 16), sw_desc(base + Sm::kB + o, 16), id_cb, k > 0);
          }
          ch_commit(&br.cb_full);
          if (!ch_wait(&br.s_full, ph, dead)) break;
          if (!ch_wait(&br.y_free, ph ^ 1, dead)) break;
          tc_after();
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < N / 16; ++k)
              mma_ss(tmem + kTmY, sw_desc(base + Sm::kC + (k >> 2) * kPanel + (k & 3) * 32, 16),
                     sw_desc(base + Sm::kS + part * 2 * Sm::kSPanel + k * 2048, Sm::kSPanel), id_cs, part + k > 0);
          ch_commit(&br.cs_done);
          if (!ch_wait(&br.rdy_x, ph, dead)) break;
          if (!ch_wait(&br.p_full, 0, dead)) break;  // phases 2 it, 2 it + 1
          tc_after();
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma_ts(tmem + kTmY, tmem + kTmP + 64 * part + 8 * k, sw_desc(base + Sm::kX + k * 2048, 16), id_px);
          ch_commit(&br.px_done[0]);
        }
        if (!ch_wait(&br.ds_free, ph ^ 1, dead)) break;
        bool ok = true;
        for (int hf = 0; hf < 2 && ok; ++hf)
          for (int part = 0; part < 3; ++part) {
            if (!ch_wait(&br.w_full[part], hf, dead)) {
              ok = false;
              break;
            }
            tc_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)
              // fewer than 128 state columns: the rows behind them repeat the first (panel stride 0)
              mma_ss(tmem + kTmS, sw_desc(base + Sm::kB + (64 * hf + 16 * k) * 128, N == 128 ? kPanel : 0),
                     sw_desc(base + Sm::kW + part * 2 * kHalfPanel + k * 2048, kHalfPanel), id_ds,
                     hf + part + k > 0);
            ch_commit(&br.w_free[part]);
          }
        if (!ok) break;
        ch_commit(&br.ds_done);
        if (WHOLE) {
          if (!ch_wait(&br.p_full, 1, dead)) break;
          tc_after();
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma_ts(tmem + kTmY + 64, tmem + kTmP + 64 * part + 8 * k,
                     sw_desc(base + Sm::kX + kPanel + k * 2048, 16), id_px);
          ch_commit(&br.px_done[1]);
        }
      }
      // every MMA is complete before tensor memory is freed
      ch_commit(&br.mma_done);
      mbar_wait(&br.mma_done, 0, 2000000000LL);
    }
  } else {
    // -------------------------------------------------------------- steps
    const float log2e = 1.4426950408889634f;
    float sum[2] = {0.0f, 0.0f};  // pass 1: exponent of the whole part
    for (int it = 0; it < count; ++it) {
      const uint32_t ph = it & 1;
      const int valid = wk.valid(), row = wk.row0();
      float d[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int head = head_of(wk.pair, h);
        const float bias = a.dt_bias ? a.dt_bias[head] : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 4 * lane + i;
          d[h][i] = t < valid
                        ? softplus(__bfloat162float(a.dt[(size_t)(row + t) * a.dt_stride + head]) + bias)
                        : 0.0f;
        }
      }
      if (!ch_wait_w(&br.sc_free[ph], ((it >> 1) & 1) ^ 1, dead)) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        Steps& st = steps[2 * ph + h];
        const float A2 = a.A[head_of(wk.pair, h)] * log2e;
        float e[4], suf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = d[h][i] * A2;
        const float own = (e[0] + e[1]) + (e[2] + e[3]);
        // over the eight lanes of a block of 32 tokens
        float pre = own, post = own;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
          const float u = __shfl_up_sync(0xffffffffu, pre, o), v = __shfl_down_sync(0xffffffffu, post, o);
          if ((lane & 7) >= o) pre += u;
          if ((lane & 7) + o < 8) post += v;
        }
        float ex = __shfl_up_sync(0xffffffffu, pre, 1), sx = __shfl_down_sync(0xffffffffu, post, 1);
        if ((lane & 7) == 0) ex = 0.0f;
        if ((lane & 7) == 7) sx = 0.0f;
        const float b0 = __shfl_sync(0xffffffffu, pre, 7), b1 = __shfl_sync(0xffffffffu, pre, 15),
                    b2 = __shfl_sync(0xffffffffu, pre, 23), b3 = __shfl_sync(0xffffffffu, pre, 31);
        const int blk = lane >> 3;
        const float after = blk == 0 ? b1 + b2 + b3 : blk == 1 ? b2 + b3 : blk == 2 ? b3 : 0.0f;
        suf[3] = sx;
        suf[2] = suf[3] + e[3];
        suf[1] = suf[2] + e[2];
        suf[0] = suf[1] + e[1];
        float run = ex;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 4 * lane + i;
          run += e[i];
          st.lp[t] = run;
          st.d[t] = d[h][i];
          st.v[t] = d[h][i] * ex2(suf[i]);
          st.w[t] = d[h][i] * ex2(suf[i] + after);
        }
        const float all = (b0 + b1) + (b2 + b3);
        sum[h] += all;
        if (lane == 0) {
          st.blk[0] = b0;
          st.blk[1] = b1;
          st.blk[2] = b2;
          st.blk[3] = b3;
          st.all = ex2(all);
        }
      }
      ch_arrive_w(&br.sc_full[ph]);
      if (!ch_wait_w(&br.raw_b, ph, dead)) break;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      if (valid < kQ) {
        for (int i = lane; i < (kQ - valid) * 8; i += 32)
#pragma unroll
          for (int p = 0; p < N / 64; ++p)
            *reinterpret_cast<uint4*>(smem + Sm::kB + p * kPanel + valid * 128 + i * 16) = zero;
        to_async();
      }
      ch_arrive_w(&br.rdy_b);
      if (!ch_wait_w(&br.raw_x, ph, dead)) break;
      if (valid < kQ) {
        for (int i = lane; i < (kQ - valid) * 8; i += 32)
#pragma unroll
          for (int p = 0; p < 2; ++p)
            *reinterpret_cast<uint4*>(smem + Sm::kX + p * kPanel + valid * 128 + i * 16) = zero;
        to_async();
      }
      ch_arrive_w(&br.rdy_x);
      if (it + 1 < count) wk.next(a.pk);
    }
    if (!WHOLE && count > 0 && lane < 2) a.decay[2 * cta + lane] = ex2(lane ? sum[1] : sum[0]);
  }
  tc_before();
  __syncthreads();
  if (warp == 17)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Pass 2: along each head pair's pieces, in order, state after piece c =
// its own + its decay times the state after piece c - 1 of the same sequence.
// Also gives empty sequences without a carried state their zero state.
constexpr int kJoinThreads = 256;

__global__ void __launch_bounds__(kJoinThreads) scan_join_kernel(ChunkArgs a, int ctas) {
  __shared__ int s_total;
  if (threadIdx.x < 32) {
    int seq, nth, total = 0;
    find_tile(a.pk, -1, kQ, 0, seq, nth, total);
    if (threadIdx.x == 0) s_total = total;
  }
  __syncthreads();
  const int total = s_total, size = 2 * kP * a.n, pair = blockIdx.y;
  const int e = blockIdx.x * kJoinThreads + threadIdx.x;
  if (total > 0 && e < size) {
    const long long all = (long long)total * a.pairs, lo = (long long)pair * total, hi = lo + total;
    const int h = e / (kP * a.n);
    int c = (int)(lo * ctas / all);
    while (c > 0 && cut(all, c, ctas) > lo) --c;
    float carry = 0.0f;
    // pieces that end inside this pair's steps
    for (; c < ctas; ++c) {
      const long long f1 = cut(all, c + 1, ctas);
      if (f1 <= lo) continue;
      if (f1 > hi || cut(all, c, ctas) >= hi) break;
      const int m = a.meta[c];
      if (m == 0) continue;
      float* p = a.local + (size_t)c * size + e;
      carry = m == 2 ? fmaf(a.decay[2 * c + h], carry, *p) : *p;
      *p = carry;
    }
  }
  if (a.state && a.pk.seqs) {
    const size_t per = (size_t)a.heads * kP * a.n;
    const int blocks = gridDim.x * gridDim.y, b = blockIdx.y * gridDim.x + blockIdx.x;
    for (int i = b; i < a.pk.seqs; i += blocks) {
      int begin, len;
      seq_range(a.pk, i, begin, len);
      const int slot = seq_slot(a.pk, i);
      if (len > 0 || slot < 0 || (a.pk.has && a.pk.has[i])) continue;
      for (size_t j = threadIdx.x; j < per; j += kJoinThreads) a.state[slot * per + j] = 0.0f;
    }
  }
}

// ------------------------------------------------------------------- host

typedef CUresult (*ChEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

ChEncodeFn ch_encode_fn() {
  static ChEncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (ChEncodeFn) nullptr;
    return reinterpret_cast<ChEncodeFn>(p);
  }();
  return fn;
}

// bf16 [rows][cols], rows `stride` elements apart, boxes of 128 rows x 64 columns.
int ch_map(CUtensorMap* map, const void* p, int rows, int cols, long long stride) {
  ChEncodeFn enc = ch_encode_fn();
  if (!enc) return kErrLaunch;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t box[2] = {64, kQ};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? kOk
             : kErrArg;
}

bool rows16(const void* p, long long stride) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0;
}

// The chunked form takes bf16, head_dim 64 and 64 or 128 state columns; and
// enough tokens: below, the token-by-token kernel's time (0.55 us a token)
// is less than three launches and a chunk's latency.
bool chunk_sizes(int type, int tokens, int head_dim, int d_state) {
  return type == kTypeBF16 && head_dim == kP && (d_state == 64 || d_state == 128) && tokens > 32;
}

template <int N>
int launch_chunks(const ScanArgs& s, cudaStream_t stream) {
  ChunkArgs a{};
  a.pk = s.pk;
  a.dt = static_cast<const __nv_bfloat16*>(s.dt);
  a.A = s.A;
  a.D = s.D;
  a.dt_bias = s.dt_bias;
  a.state = s.state;
  a.y = static_cast<__nv_bfloat16*>(s.y);
  a.dt_stride = s.dt_stride;
  a.y_stride = s.y_stride;
  a.heads = s.heads;
  a.hpg = s.heads / s.groups;
  a.ppg = (a.hpg + 1) / 2;
  a.pairs = a.ppg * s.groups;
  a.n = N;
  const size_t part = (size_t)kMaxCtas * 2 * kP * N;
  a.local = static_cast<float*>(s.scratch);
  a.init = a.local + part;
  a.decay = a.init + part;
  a.meta = reinterpret_cast<int*>(a.decay + 2 * kMaxCtas);
  CUtensorMap xm, bm, cm;
  if (int e = ch_map(&xm, s.x, s.pk.tokens, s.heads * kP, s.x_stride)) return e;
  if (int e = ch_map(&bm, s.B, s.pk.tokens, s.groups * N, s.b_stride)) return e;
  if (int e = ch_map(&cm, s.C, s.pk.tokens, s.groups * N, s.c_stride)) return e;
  auto pass1 = scan_chunk_kernel<N, false>;
  auto pass3 = scan_chunk_kernel<N, true>;
  constexpr int smem = ChunkSmem<N>::kBytes;
  if (cudaFuncSetAttribute(pass1, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaFuncSetAttribute(pass3, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return kErrLaunch;
  const long long most = ((long long)s.pk.tokens / kQ + s.pk.seqs) * a.pairs;  // steps, at most
  int ctas = device_sm_count();
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  if (most < ctas) ctas = (int)most;
  pass1<<<ctas, kChThreads, smem, stream>>>(xm, bm, cm, a);
  scan_join_kernel<<<dim3((2 * kP * N + kJoinThreads - 1) / kJoinThreads, a.pairs), kJoinThreads, 0, stream>>>(a, ctas);
  pass3<<<ctas, kChThreads, smem, stream>>>(xm, bm, cm, a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace

size_t ssm_prompt_scratch_bytes(int type, int tokens, int, int, int head_dim, int, int d_state) {
  if (!chunk_sizes(type, tokens, head_dim, d_state)) return 0;
  return (size_t)kMaxCtas * (4 * kP * d_state * 4 + 16);
}

int launch_ssm_prompt(const ScanArgs& a, cudaStream_t stream) {
  if (chunk_sizes(a.type, a.pk.tokens, a.head_dim, a.d_state) && rows16(a.x, a.x_stride) && rows16(a.B, a.b_stride) &&
      rows16(a.C, a.c_stride) && rows16(a.y, a.y_stride))
    return a.d_state == 128 ? launch_chunks<128>(a, stream) : launch_chunks<64>(a, stream);
  return launch_scan_tokens(a, stream);
}

int read_scan_device_error(bool clear) { return read_unit_error(clear); }

}  // namespace ervf
