// ssm_chunk.cu -- the selective scan of bf16 prompts on the sm_100a tensor
// cores, in chunks of Q = 128 tokens:
//
//   P[t][s] = (C_t . B_s) exp(c_t - c_s) d_s  for s <= t
//   y_t     = sum_s P[t][s] x_s + exp(c_t) S C_t + D x_t
//   S'      = exp(c_Q) S + sum_s exp(c_Q - c_s) d_s x_s B_s^T
//
// with c the running sum of d A inside the chunk and S the state before it.
// One CTA per SM walks a list of (head pair, sequence, chunk) steps and carries
// the two heads' state in registers; C B^T is shared by the pair.  The list
// is cut into equal pieces, one per CTA, wherever the cuts fall:
//   pass 0  softplus, running sums and weights of every (head, chunk); each
//           CTA's piece
//   pass 1  (WHOLE = false) a CTA whose piece ends inside a sequence computes
//           the state that its own part of that sequence adds, and its decay;
//   pass 2  joins these along each sequence, in order;
//   pass 3  (WHOLE = true) every CTA runs its piece from its true start state.
// Exponents are sums of numbers of one sign (distances within blocks of 32
// tokens plus whole blocks), so no difference of two long sums is taken but
// inside a block.  Products meet the tensor cores in bf16: B, C and x are bf16
// already.  The in-chunk weights P are rounded to bf16 once (2^-8 of each term
// at most, as the output's own rounding; a second part would take the tensor
// memory that keeps both heads' P in work at once); D x is added in f32.  S is
// split into two bf16 numbers for S C (2^-16), the state's new terms into
// three (2^-24: states stay f32).
//
// Warps (a warpgroup's register share in brackets), and what bounds them at
// 128 state columns (clocks per step of two heads, measured tcgen05 rates):
//   0..7   P and y [80]: C B^T from tensor memory, weighted, back to tensor
//          memory as an A operand, both heads; their products with x take the
//          columns of C B^T; then exp(c_t) S C + P x + D x -> bf16
//   8..15  states [96]: the f32 state, 64 registers a thread, split for S C
//   16..23 W [48]: x scaled to the chunk's end and split into three, 32 tokens
//          at a time, as the B operand of the state's new terms
//   24     TMA of the steps and of the B and C tiles
//   25     MMAs C B^T 8 x 65 and P x 16 x 68; TMA of the x tiles
//   26     MMAs of the state's new terms 24 x 69 and S C 16 x 69
//   27     clears rows behind a sequence's end, so that a neighbour's NaN meets
//          no zero weight
// The MMAs take 4370 clocks.  Both operands of a 128-column MMA in shared
// memory take its whole bandwidth (128 bytes a clock); with W, the split state
// and the tiles a step moves 740 KB there, 5800 clocks; its warps issue 5100
// instructions a scheduler.  Measured: 11000 clocks, of which P takes 3500, P x
// 1300 and y 3600 one after the other (64 heads, 8192 tokens: 151 to 156 us in
// all, 27 of them pass 1, which spills 116 bytes at 128 states).  Waits are short
// and loops little unrolled on purpose: seven roles' code has to share the
// instruction cache (waits that watched the clock and unrolled MMA loops: 97 KB,
// 179 us).  Tried without gain: y of the second head by the W warps, S C ahead of
// the state's new terms, W pieces of 16 tokens, C B^T pieces loaded once for both
// heads.
// In pass 1 warps 0..7 do W's work too.  y's test for sums that a NaN or an
// infinity behind their token has spoiled costs 1% (causal_rows).
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
constexpr int kWRows = 32, kPieces = kQ / kWRows, kWPanel = kWRows * 128;  // tokens of a W buffer, one part of one head of it
constexpr int kChWarps = 28, kChThreads = kChWarps * 32;
// registers a thread at launch, and each warpgroup's after its split: the
// shares must not exceed what the block was launched with
constexpr int kRegs = 72, kRegP = 80, kRegS = 96, kRegW = 48, kRegMisc = 56;
static_assert(2 * kRegP + 2 * kRegS + 2 * kRegW + kRegMisc <= 7 * kRegs, "register shares");
constexpr int kMaxCtas = 148;
// tensor-memory columns
constexpr int kTmCB = 0, kTmP = 128, kTmY = 256, kTmS = 384;  // P: 64 columns a head

// Per-token numbers of one head in one chunk, base-2 exponents.
struct alignas(16) Steps {
  float lp[kQ];  // running sum inside the token's block of 32, inclusive
  float d[kQ];   // softplus step, 0 behind the end
  float v[kQ];   // d exp2(distance to the end of the token's block)
  float w[kQ];   // d exp2(distance to the end of the chunk)
  float blk[4];  // sums of the blocks
  float all;     // exp2(sum of the chunk)
  float sum;     // sum of the chunk
  float D;
  float pad;
};
static_assert(sizeof(Steps) % 16 == 0, "bulk copies");

// A CTA's piece of the list: its first step (pair, sequence, chunk), the place
// of that chunk among all sequences', the number of steps, and the piece before
// (pieces may be empty).
struct alignas(16) Plan {
  int pair, seq, chunk, nth, count, before, total, pad;
};

struct ChunkArgs {
  Packing pk;
  const __nv_bfloat16* dt;
  const float *A, *D, *dt_bias;
  float* state;
  __nv_bfloat16* y;
  long long dt_stride, y_stride;
  int heads, hpg, ppg, pairs;  // heads, heads and pairs per group, pairs in all
  int n;                       // d_state
  Steps* steps;                // [pair][chunk][2]
  float* local;                // [ctas][2][kP][n]: pass 1's states, joined in place by pass 2
  float* init;                 // [ctas][2][kP][n]: carried states of sequences that are cut
  float* decay;                // [ctas][2]
  Plan* plan;                  // [pass 1, pass 3][ctas]
  int* meta;                   // [ctas]: 0 no cut, else pair * 4 + (1 from a sequence's start, 2 continued)
};

// kStages tiles of B and x: pass 1 has the room of C and S.  Two teams scale
// x, each into a W buffer of its own (a team may run a step ahead of the
// other: buffers taken in turns would need more than a parity to tell their
// rounds apart).  Pieces of 16 tokens and two buffers a team were slower: the
// issuing thread's waits cost more than the overlap gave.
template <bool WHOLE>
struct Depth {
  static constexpr int kStages = WHOLE ? 1 : 2, kWBufs = 2, kTeam = WHOLE ? 128 : 256;
};

struct Barriers {
  uint64_t raw_b[2], raw_c, raw_x[2];  // TMA bytes landed
  uint64_t rdy_b[2], rdy_x[2];         // and rows behind the end cleared
  uint64_t sc_full[2], sc_free[2];
  uint64_t cb_full, cs_done, p_full, px_done, y_free;
  uint64_t w_full[2], w_free[2], ds_done, ds_free, b_free[2], s_full, x_read[2], mma_done;
};

template <int N, bool WHOLE>
struct ChunkSmem {
  using Dp = Depth<WHOLE>;
  static constexpr int kTile = N / 64 * kPanel;    // B or C
  static constexpr int kB = 0, kX = kB + Dp::kStages * kTile;
  static constexpr int kW = kX + Dp::kStages * 2 * kPanel;  // [buffer][part][head][rows]
  static constexpr int kC = kW + Dp::kWBufs * 6 * kWPanel;
  static constexpr int kS = kC + (WHOLE ? kTile : 0);       // [hi, lo][head][N rows]
  static constexpr int kSPanel = N * 128;
  static constexpr int kY = kS + (WHOLE ? 4 * kSPanel : 0);   // 8 warps x 1 KB
  static constexpr int kSteps = kY + (WHOLE ? 8 * 1024 : 0);  // [2 buffers][2 heads]
  static constexpr int kBar = kSteps + 4 * (int)sizeof(Steps);
  static constexpr int kBytes = 1024 + kBar + 512;
};
static_assert(ChunkSmem<128, true>::kBytes <= 232448 && ChunkSmem<128, false>::kBytes <= 232448, "shared memory");

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
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(db), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void ch_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
               ::"r"(smem_u32(bar)) : "memory");
}
// 16 columns each of two places.
__device__ __forceinline__ void tm_ld16x2(uint32_t t, uint32_t t2, uint32_t (&v)[16], uint32_t (&w)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]),
        "=r"(w[8]), "=r"(w[9]), "=r"(w[10]), "=r"(w[11]), "=r"(w[12]), "=r"(w[13]), "=r"(w[14]), "=r"(w[15])
      : "r"(t), "r"(t2) : "memory");
}
// The wait in the same statement: nothing may use the registers before it.
__device__ __forceinline__ void tm_ld16(uint32_t t, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(t) : "memory");
}
__device__ __forceinline__ void tm_st8(uint32_t t, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
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

// The box into L2 ahead of its load.
__device__ __forceinline__ void ch_prefetch(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

// Bounded wait of one thread: 100,000 tries, each of which the hardware may
// suspend for up to 20 us; gives up too when another role died.  A wait that
// runs out marks the CTA dead (2; its last act tells the host).  Short on
// purpose: the kernel waits in some forty places, and its warps, each in a loop
// of its own, wait for instructions as soon as those loops outgrow the cache.
__device__ __forceinline__ bool ch_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .u32 n, d;\n"
      " mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n mov.u32 n, 100000;\n"
      "AGAIN:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n @p bra DONE;\n"
      " ld.volatile.shared.u32 d, [%3];\n setp.ne.u32 q, d, 0;\n @q bra DONE;\n"
      " sub.u32 n, n, 1;\n setp.ne.u32 q, n, 0;\n @q bra AGAIN;\n"
      " st.volatile.shared.u32 [%3], 2;\n"
      "DONE:\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(smem_u32(const_cast<int*>(dead))), "r"(20000u)
      : "memory");
  return ok != 0;
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

// The passes are launched with programmatic serialisation: each lets the next
// one start as its own CTAs leave, and waits for the one before (and so for all
// before that) ahead of its first read.
__device__ __forceinline__ void pass_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pass_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Heads of a pair; an odd group's last pair has its head twice.
struct Heads {
  int grp, h[2];
  int of = -1;  // the pair they are of
  __device__ void at(const ChunkArgs& a, int pair) {
    if (pair == of) return;
    of = pair;
    grp = pair / a.ppg;
    const int k = (pair - grp * a.ppg) * 2;
    h[0] = grp * a.hpg + k;
    h[1] = k + 1 < a.hpg ? h[0] + 1 : h[0];
  }
};

// First and one-past-last step of CTA c out of g.
__device__ __forceinline__ long long cut(long long steps, int c, int g) { return steps * c / g; }

// Two f32 to their bf16 rounding and to the bf16 rounding of what it leaves.
__device__ __forceinline__ void split2(float e, float o, uint32_t& hi, uint32_t& lo) {
  hi = pack2(e, o);
  lo = pack2(e - lo_f(hi), o - hi_f(hi));
}

// A NaN or an infinity in x meets the zero weights of the tokens before it in
// the tensor cores.  Where that spoiled sums of a warp's 32 tokens (16 columns
// of one head from piece `piece` of x's rows), their lanes form them anew here,
// token by token up to their own, from the weights in tensor memory, and store
// their outputs over the first ones (out: a lane's, or null).  Sums that the
// state before the chunk has spoiled as well stay as they are.
__device__ __forceinline__ void causal_rows(uint32_t p_at, uint32_t y_at, uint32_t px_at, const uint8_t* x, int t,
                                            int piece, float D, float e, __nv_bfloat16* out) {
  uint32_t u[16], v[16];
  tm_ld16x2(y_at, px_at, u, v);
  bool spoiled = false;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    spoiled = spoiled || (!isfinite(__uint_as_float(v[i])) && isfinite(e * __uint_as_float(u[i])));
  if (!__any_sync(0xffffffffu, spoiled)) return;
  float f[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = 0.0f;
#pragma unroll 1
  for (int s = 0; s <= (t | 31); ++s) {
    uint32_t w;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;"
                 : "=r"(w) : "r"(p_at + (s >> 1)) : "memory");
    if (s <= t) {
      const float p = s & 1 ? hi_f(w) : lo_f(w);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 xv = *reinterpret_cast<const uint4*>(x + s * 128 + (((piece + k) ^ (s & 7)) << 4));
        const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[8 * k + 2 * i] = fmaf(p, lo_f(xs[i]), f[8 * k + 2 * i]);
          f[8 * k + 2 * i + 1] = fmaf(p, hi_f(xs[i]), f[8 * k + 2 * i + 1]);
        }
      }
    }
    __syncwarp();
  }
  if (!spoiled || !out) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint4 xv = *reinterpret_cast<const uint4*>(x + t * 128 + (((piece + k) ^ (t & 7)) << 4));
    const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = 8 * k + 2 * i;
      o[i] = pack2(fmaf(D, lo_f(xs[i]), fmaf(e, __uint_as_float(u[m]), f[m])),
                   fmaf(D, hi_f(xs[i]), fmaf(e, __uint_as_float(u[m + 1]), f[m + 1])));
    }
    reinterpret_cast<uint4*>(out)[k] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// W: a team scales x of step `it` to the chunk's end and splits it into three,
// kWRows tokens of both heads at a time: every second such piece of the chunk.
template <int N, bool WHOLE>
__device__ __forceinline__ bool scale_x(uint8_t* smem, Barriers& br, int team, int it, volatile int* dead) {
  using Sm = ChunkSmem<N, WHOLE>;
  constexpr int STG = Depth<WHOLE>::kStages, NT = Depth<WHOLE>::kTeam;
  const Steps* st = reinterpret_cast<const Steps*>(smem + Sm::kSteps) + 2 * (it & 1);
  const int stg = it % STG, wt = threadIdx.x & (NT - 1), ch = wt & 7;
  if (!ch_wait_w(&br.sc_full[it & 1], (it >> 1) & 1, dead)) return false;
  if (!ch_wait_w(&br.rdy_x[stg], (it / STG) & 1, dead)) return false;
  const uint8_t* xt = smem + Sm::kX + stg * 2 * kPanel;
  uint8_t* wb = smem + Sm::kW + team * 6 * kWPanel;
#pragma unroll 1
  for (int i = 0; i < kPieces / 2; ++i) {
    const int row0 = kWRows * (2 * i + team);
    // the buffer's rounds 2 it, 2 it + 1
    if (!ch_wait_w(&br.w_free[team], i ^ 1, dead)) return false;
#pragma unroll 2
    for (int k = 0; k < 512 / NT; ++k) {
      const int h = (k * NT + wt) >> 8, r = ((k * NT + wt) >> 3) & 31;
      const uint32_t off = (uint32_t)(r * 128 + ((ch ^ (r & 7)) << 4));
      const float w = st[h].w[row0 + r];
      const uint4 xv = *reinterpret_cast<const uint4*>(xt + h * kPanel + row0 * 128 + off);
      const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
      uint32_t p0[4], p1[4], p2[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 e = mul2(make_float2(lo_f(xs[j]), hi_f(xs[j])), make_float2(w, w));
        p0[j] = pack2(e.x, e.y);
        e = add2(e, make_float2(-lo_f(p0[j]), -hi_f(p0[j])));
        p1[j] = pack2(e.x, e.y);
        e = add2(e, make_float2(-lo_f(p1[j]), -hi_f(p1[j])));
        p2[j] = pack2(e.x, e.y);
      }
      uint8_t* dst = wb + h * kWPanel + off;
      *reinterpret_cast<uint4*>(dst) = make_uint4(p0[0], p0[1], p0[2], p0[3]);
      *reinterpret_cast<uint4*>(dst + 2 * kWPanel) = make_uint4(p1[0], p1[1], p1[2], p1[3]);
      *reinterpret_cast<uint4*>(dst + 4 * kWPanel) = make_uint4(p2[0], p2[1], p2[2], p2[3]);
    }
    to_async();
    ch_arrive_w(&br.w_full[team]);
  }
  ch_arrive_w(&br.x_read[stg]);
  ch_arrive_w(&br.sc_free[it & 1]);
  return true;
}

// A warpgroup's share: inc below the launch's count, or dec above it, is an
// illegal instruction.
template <int R>
__device__ __forceinline__ void regs_to() {
  static_assert(R % 8 == 0 && R >= 24, "setmaxnreg");
  if constexpr (R > kRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
  if constexpr (R < kRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

template <int N, bool WHOLE>
__global__ void __launch_bounds__(kChThreads, 1)
    scan_chunk_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap b_map,
                      const __grid_constant__ CUtensorMap c_map, ChunkArgs a) {
  using Sm = ChunkSmem<N, WHOLE>;
  constexpr int STG = Depth<WHOLE>::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  Barriers& br = *reinterpret_cast<Barriers*>(smem + Sm::kBar);
  static_assert(sizeof(Barriers) <= 400, "barrier block");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Sm::kBar + 400);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + Sm::kBar + 404);
  Plan* first = reinterpret_cast<Plan*>(smem + Sm::kBar + 416);
  Steps* steps = reinterpret_cast<Steps*>(smem + Sm::kSteps);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;

  if (!WHOLE) pass_next();  // what follows pass 3 is not ours
  pass_wait();
  if (warp == 0) {
    if (lane == 0) {
      const int4* pl = reinterpret_cast<const int4*>(a.plan + (WHOLE ? kMaxCtas : 0) + cta);
      reinterpret_cast<int4*>(first)[0] = pl[0];
      reinterpret_cast<int4*>(first)[1] = pl[1];
      // warps that scale x, and that read the steps
      const int scalers = WHOLE ? 8 : 16, cons = 8 + scalers + (WHOLE ? 8 : 0);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&br.raw_b[i], 1);
        mbar_init(&br.raw_x[i], 1);
        mbar_init(&br.rdy_b[i], 1);
        mbar_init(&br.rdy_x[i], 1);
        mbar_init(&br.sc_full[i], 1);
        mbar_init(&br.sc_free[i], cons);
        mbar_init(&br.b_free[i], 1);
        mbar_init(&br.x_read[i], 16);  // scalers, and whole: y's readers
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&br.w_full[i], Depth<WHOLE>::kTeam / 32);
        mbar_init(&br.w_free[i], 1);
      }
      mbar_init(&br.raw_c, 1);
      mbar_init(&br.cb_full, 1);
      mbar_init(&br.cs_done, 1);
      mbar_init(&br.p_full, 8);
      mbar_init(&br.px_done, 1);
      mbar_init(&br.y_free, 8);
      mbar_init(&br.ds_done, 1);
      mbar_init(&br.ds_free, 8);
      mbar_init(&br.s_full, 8);
      mbar_init(&br.mma_done, 2);
      *dead = 0;
      fence_mbar_init();
    }
  }
  if (warp == 25) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_slot;
  const int count = first->count;
  Walk wk;
  if (count > 0) wk.at(a.pk, first->pair, first->seq, first->chunk);
  const int q = warp & 3;  // tensor-memory lanes 32 q ..
  const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);

  if (warp < 8) {
    // ------------------------------------------------------------------ P
    // Lanes are tokens t; the two warps of a lane quarter share its blocks of
    // 32 tokens s: q, q - 2 for the first, q - 1, q - 3 for the second (of two
    // below the diagonal, the second takes both).
    regs_to<kRegP>();
    if (!WHOLE) {
      for (int it = 0; it < count; ++it)
        if (!scale_x<N, WHOLE>(smem, br, 0, it, dead)) break;
    } else if (count > 0) {
      const int side = warp >> 2, t = 32 * q + lane;
      Heads hd;
      if (side == 1) {
        // columns behind the diagonal block stay zero
        const uint32_t z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int c = 16 * (q + 1); c < 64; c += 8) {
          tm_st8(lanes + kTmP + c, z);
          tm_st8(lanes + kTmP + 64 + c, z);
        }
        tm_wait_st();
      }
      for (int it = 0; it < count; ++it) {
        const uint32_t ph = it & 1;
        if (!ch_wait_w(&br.sc_full[ph], (it >> 1) & 1, dead)) break;
        if (!ch_wait_w(&br.cb_full, ph, dead)) break;
        tc_after();
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const Steps& st = steps[2 * ph + h];
          const float lp = st.lp[t], b1 = st.blk[1], b2 = st.blk[2];
#pragma unroll 1
          for (int j = q - side; j >= 0; j -= (q == 2 && side == 1) ? 1 : 2) {
            if (q == 2 && j == 0 && side == 0) break;
            // from the end of block j to t: whole blocks between, then t's own part
            const float u = ex2(lp + (j + 1 < q ? (j == 0 ? b1 : b2) : 0.0f) + (j + 2 < q ? b2 : 0.0f));
#pragma unroll 1
            for (int c = 0; c < 32; c += 16) {
              uint32_t v[16], o[8];
              tm_ld16(lanes + kTmCB + 32 * j + c, v);
              if (j == q) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                  const float4 ls = *reinterpret_cast<const float4*>(&st.lp[32 * j + c + i]);
                  const float4 ds = *reinterpret_cast<const float4*>(&st.d[32 * j + c + i]);
                  const float lv[4] = {ls.x, ls.y, ls.z, ls.w}, dv[4] = {ds.x, ds.y, ds.z, ds.w};
                  float p[4];
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    p[k] = __uint_as_float(v[i + k]) * (dv[k] * ex2(lp - lv[k]));
                    if (c + i + k > lane) p[k] = 0.0f;
                  }
                  o[i / 2] = pack2(p[0], p[1]);
                  o[i / 2 + 1] = pack2(p[2], p[3]);
                }
              } else {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                  const float4 w = *reinterpret_cast<const float4*>(&st.v[32 * j + c + i]);
                  const float2 e = mul2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])),
                                        mul2(make_float2(w.x, w.y), make_float2(u, u)));
                  const float2 f = mul2(make_float2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])),
                                        mul2(make_float2(w.z, w.w), make_float2(u, u)));
                  o[i / 2] = pack2(e.x, e.y);
                  o[i / 2 + 1] = pack2(f.x, f.y);
                }
              }
              tm_st8(lanes + kTmP + 64 * h + 16 * j + c / 2, o);
            }
          }
        }
        tm_wait_st();
        tc_before();
        ch_arrive_w(&br.p_full);
        // y: exp(c_t) S C + P x + D x, half of each head's columns
        if (!ch_wait_w(&br.cs_done, ph, dead)) break;
        if (!ch_wait_w(&br.px_done, ph, dead)) break;
        tc_after();
        hd.at(a, wk.pair);
        const int left = wk.valid() - 32 * q;  // rows of this warp inside the sequence
        __nv_bfloat16* rows = a.y + (size_t)(wk.row0() + 32 * q) * a.y_stride + 32 * side;
        uint8_t* stage = smem + Sm::kY + warp * 1024;
        uint32_t odd = 0;  // not 0 once an output is no finite number
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const Steps& st = steps[2 * ph + h];
          const float D = st.D, e = ex2(st.lp[t] + (q > 0 ? st.blk[0] : 0.0f) + (q > 1 ? st.blk[1] : 0.0f) +
                                        (q > 2 ? st.blk[2] : 0.0f));
          __nv_bfloat16* y = rows + (size_t)(h ? hd.h[1] : hd.h[0]) * kP;
          const bool put = h == 0 || hd.h[1] != hd.h[0];
          const uint8_t* xr = smem + Sm::kX + h * kPanel + t * 128;
#pragma unroll 1
          for (int c = 0; c < 4; c += 2) {
            uint32_t u[16], v[16];
            tm_ld16x2(lanes + kTmY + 64 * h + 32 * side + 8 * c, lanes + kTmCB + 64 * h + 32 * side + 8 * c, u, v);
            // 32 rows of 32 bytes through shared memory: two lanes store one row's
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint4 xv = *reinterpret_cast<const uint4*>(xr + (((4 * side + c + k) ^ (t & 7)) << 4));
              const uint32_t xs[4] = {xv.x, xv.y, xv.z, xv.w};
              uint32_t o[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int m = 8 * k + 2 * i;
                o[i] = pack2(fmaf(D, lo_f(xs[i]), fmaf(e, __uint_as_float(u[m]), __uint_as_float(v[m]))),
                             fmaf(D, hi_f(xs[i]), fmaf(e, __uint_as_float(u[m + 1]), __uint_as_float(v[m + 1]))));
              }
              *reinterpret_cast<uint4*>(stage + lane * 32 + ((k ^ ((lane >> 2) & 1)) << 4)) =
                  make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
              for (int i = 0; i < 4; ++i) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(odd) : "r"(o[i]), "r"(0));
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int r = 16 * k + (lane >> 1), i = lane & 1;
              const uint4 val = *reinterpret_cast<const uint4*>(stage + r * 32 + ((i ^ ((r >> 2) & 1)) << 4));
              if (put && r < left) *reinterpret_cast<uint4*>(y + (size_t)r * a.y_stride + 8 * (c + i)) = val;
            }
            __syncwarp();
          }
        }
        if (__any_sync(0xffffffffu, (odd & 0x7FFF7FFFu) != 0)) {
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            const int h = i >> 1, c = 2 * (i & 1), col = 64 * h + 32 * side + 8 * c;
            const Steps& st = steps[2 * ph + h];
            const float e = ex2(st.lp[t] + (q > 0 ? st.blk[0] : 0.0f) + (q > 1 ? st.blk[1] : 0.0f) +
                                (q > 2 ? st.blk[2] : 0.0f));
            const bool put = lane < left && (h == 0 || hd.h[1] != hd.h[0]);
            causal_rows(lanes + kTmP + 64 * h, lanes + kTmY + col, lanes + kTmCB + col, smem + Sm::kX + h * kPanel, t,
                        4 * side + c, st.D, e,
                        put ? rows + (size_t)(h ? hd.h[1] : hd.h[0]) * kP + (size_t)lane * a.y_stride + 8 * c : nullptr);
          }
        }
        tc_before();
        ch_arrive_w(&br.y_free);
        ch_arrive_w(&br.x_read[0]);
        ch_arrive_w(&br.sc_free[ph]);
        if (it + 1 < count) wk.next(a.pk);
      }
    }
  } else if (warp < 16) {
    // ------------------------------------------------------------- states
    regs_to<kRegS>();
    const int half = (warp - 8) >> 2;  // state rows 32 q .., columns 32 half ..
    const int n = 32 * q + lane;
    const bool own = n < N;
    float s[2][32];
    float sum0 = 0.0f, sum1 = 0.0f;  // pass 1: exponent of the whole part
    Heads hd;
    // offset of this thread's element i of a head's [kP][N] state
    auto at = [&](int i) { return (size_t)(32 * half + i) * N + n; };
    for (int it = 0; it < count; ++it) {
      const uint32_t ph = it & 1;
      if (wk.chunk == 0 || it == 0) {
        // where the state before this chunk comes from
        const int slot = a.state ? seq_slot(a.pk, wk.seq) : -1;
        hd.at(a, wk.pair);
        const float* src = nullptr;
        bool slots = false;
        if (wk.chunk > 0) {
          if (WHOLE) src = a.local + (size_t)first->before * 2 * kP * N;
        } else if (slot >= 0 && a.pk.has && a.pk.has[wk.seq]) {
          // a sequence that another CTA finishes may already have its new state in the slot
          if (WHOLE && wk.nch > count - it) src = a.init + (size_t)cta * 2 * kP * N;
          else slots = true;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* p = slots ? a.state + ((size_t)slot * a.heads + hd.h[h]) * kP * N
                                 : src ? src + (size_t)h * kP * N : nullptr;
          if (p && own) {
#pragma unroll
            for (int i = 0; i < 32; ++i) s[h][i] = p[at(i)];
            if (!WHOLE) {
              float* o = a.init + ((size_t)cta * 2 + h) * kP * N;
#pragma unroll
              for (int i = 0; i < 32; ++i) o[at(i)] = s[h][i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) s[h][i] = 0.0f;
          }
        }
      }
      if (WHOLE) {
        // both parts of both heads' state as the B operand of S C
        if (!ch_wait_w(&br.cs_done, ph ^ 1, dead)) break;
        if (own) {
          uint8_t* row = smem + Sm::kS + n * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) split2(s[h][8 * c + 2 * i], s[h][8 * c + 2 * i + 1], hi[i], lo[i]);
              uint8_t* p = row + h * Sm::kSPanel + (((4 * half + c) ^ (n & 7)) << 4);
              *reinterpret_cast<uint4*>(p) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              *reinterpret_cast<uint4*>(p + 2 * Sm::kSPanel) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        to_async();
        ch_arrive_w(&br.s_full);
      }
      if (!ch_wait_w(&br.sc_full[ph], (it >> 1) & 1, dead)) break;
      const float d0 = steps[2 * ph].all, d1 = steps[2 * ph + 1].all;
      if (!WHOLE) {
        sum0 += steps[2 * ph].sum;
        sum1 += steps[2 * ph + 1].sum;
      }
      ch_arrive_w(&br.sc_free[ph]);
      if (!ch_wait_w(&br.ds_done, ph, dead)) break;
      tc_after();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[16];
          tm_ld16(lanes + kTmS + 64 * h + 32 * half + 16 * c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[h][16 * c + i] = fmaf(h ? d1 : d0, s[h][16 * c + i], __uint_as_float(v[i]));
        }
      tc_before();
      ch_arrive_w(&br.ds_free);
      if (WHOLE && wk.chunk == wk.nch - 1) {
        const int slot = a.state ? seq_slot(a.pk, wk.seq) : -1;
        if (slot >= 0 && own)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (h == 0 || hd.h[1] != hd.h[0]) {
              float* o = a.state + ((size_t)slot * a.heads + hd.h[h]) * kP * N;
#pragma unroll
              for (int i = 0; i < 32; ++i) o[at(i)] = s[h][i];
            }
      }
      if (it + 1 < count) wk.next(a.pk);
    }
    if (!WHOLE && count > 0 && tid == 256) {
      a.decay[2 * cta] = ex2(sum0);
      a.decay[2 * cta + 1] = ex2(sum1);
    }
    if (!WHOLE && count > 0 && own) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* o = a.local + ((size_t)cta * 2 + h) * kP * N;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[at(i)] = s[h][i];
      }
    }
  } else if (warp < 24) {
    // ------------------------------------------------------------------ W
    regs_to<kRegW>();
    const int team = WHOLE ? (warp - 16) >> 2 : 1;
    for (int it = 0; it < count; ++it)
      if (!scale_x<N, WHOLE>(smem, br, team, it, dead)) break;
  } else {
    regs_to<kRegMisc>();
    if (warp == 24) {
      // --------------------------------------------- TMA of steps, C and B
      if (lane == 0) {
        // the list walks the chunks pair after pair, as the steps lie
        const Steps* src = a.steps + 2 * ((size_t)first->pair * first->total + first->nth);
        Heads hd;
        for (int it = 0; it < count; ++it) {
          const uint32_t ph = it & 1, sph = (it / STG) & 1;
          hd.at(a, wk.pair);
          const int grp = hd.grp, row = wk.row0(), stg = it % STG;
          if (!ch_wait(&br.sc_free[ph], ((it >> 1) & 1) ^ 1, dead)) break;
          mbar_arrive_expect_tx(&br.sc_full[ph], 2 * sizeof(Steps));
          bulk_g2s(steps + 2 * ph, src, 2 * sizeof(Steps), &br.sc_full[ph]);
          src += 2;
          if (WHOLE) {
            // C B^T and S C of the last step are done
            if (!ch_wait(&br.cb_full, ph ^ 1, dead)) break;
            if (!ch_wait(&br.cs_done, ph ^ 1, dead)) break;
            mbar_arrive_expect_tx(&br.raw_c, Sm::kTile);
#pragma unroll
            for (int i = 0; i < N / 64; ++i)
              ch_tma(smem + Sm::kC + i * kPanel, &c_map, grp * N + 64 * i, row, &br.raw_c);
          }
          if (!ch_wait(&br.b_free[stg], sph ^ 1, dead)) break;
          mbar_arrive_expect_tx(&br.raw_b[stg], Sm::kTile);
#pragma unroll
          for (int i = 0; i < N / 64; ++i)
            ch_tma(smem + Sm::kB + stg * Sm::kTile + i * kPanel, &b_map, grp * N + 64 * i, row, &br.raw_b[stg]);
          if (it + 1 < count) wk.next(a.pk);
        }
        // no copy is left in flight: wait for the last ones (a dead CTA's
        // waits return at once, so there a millisecond by the clock)
        if (*dead) {
          const long long t0 = clock64();
          while (clock64() - t0 < 2000000) {
          }
        } else {
          for (int it = count > STG ? count - STG : 0; it < count; ++it) {
            if (WHOLE) ch_wait(&br.raw_c, it & 1, dead);
            ch_wait(&br.raw_b[it % STG], (it / STG) & 1, dead);
            ch_wait(&br.raw_x[it % STG], (it / STG) & 1, dead);
            ch_wait(&br.sc_full[it & 1], (it >> 1) & 1, dead);
          }
        }
      }
    } else if (warp == 25) {
      // --------------------------------- TMA of x, MMAs of C B^T and P x
      if (lane == 0) {
        const uint32_t base = smem_u32(smem);
        constexpr uint32_t id_cb = ch_idesc(128, false, false), id_px = ch_idesc(64, false, true);
        Heads hd;
        const uint64_t dc = sw_desc(base + Sm::kC, 16), db = sw_desc(base + Sm::kB, 16), dx = sw_desc(base + Sm::kX, 16);
        for (int it = 0; it < count; ++it) {
          const uint32_t ph = it & 1;
          const int stg = it % STG;
          if (WHOLE) {
            if (!ch_wait(&br.rdy_b[0], ph, dead)) break;
            if (!ch_wait(&br.raw_c, ph, dead)) break;
            if (!ch_wait(&br.y_free, ph ^ 1, dead)) break;  // the columns' last P x is read
            tc_after();
#pragma unroll
            for (int k = 0; k < N / 16; ++k) {
              const int o = ((k >> 2) * kPanel + (k & 3) * 32) >> 4;
              mma_ss(tmem + kTmCB, dc + o, db + o, id_cb, k > 0);
            }
            ch_commit(&br.cb_full);
          }
          // the x tile's last readers, y's among them, are done with it
          if (!ch_wait(&br.x_read[stg], ((it / STG) & 1) ^ 1, dead)) break;
          hd.at(a, wk.pair);
          mbar_arrive_expect_tx(&br.raw_x[stg], 2 * kPanel);
          ch_tma(smem + Sm::kX + 2 * stg * kPanel, &x_map, hd.h[0] * kP, wk.row0(), &br.raw_x[stg]);
          ch_tma(smem + Sm::kX + (2 * stg + 1) * kPanel, &x_map, hd.h[1] * kP, wk.row0(), &br.raw_x[stg]);
          if (it + 1 < count) wk.next(a.pk);
          if (!WHOLE) continue;
          if (!ch_wait(&br.rdy_x[0], ph, dead)) break;
          if (!ch_wait(&br.p_full, ph, dead)) break;  // P written, C B^T read
          tc_after();
#pragma unroll 4
          for (int k = 0; k < 16; ++k)  // eight of each head; x's panels lie behind each other
            mma_ts(tmem + kTmCB + 64 * (k >> 3), tmem + kTmP + 8 * k, dx + k * (2048 >> 4), id_px, (k & 7) > 0);
          ch_commit(&br.px_done);
        }
        // every MMA is complete before tensor memory is freed
        ch_commit(&br.mma_done);
        mbar_wait(&br.mma_done, 0, 2000000000LL);
      }
    } else if (warp == 26) {
      // --------------------------- MMAs of the state's new terms and S C
      if (lane == 0) {
        const uint32_t base = smem_u32(smem);
        const uint64_t dc = sw_desc(base + Sm::kC, 16), ds = sw_desc(base + Sm::kS, Sm::kSPanel);
        constexpr uint32_t id_ds = ch_idesc(128, true, true), id_cs = ch_idesc(128, false, true);
        for (int it = 0; it < count; ++it) {
          const uint32_t ph = it & 1;
          const int stg = it % STG;
          if (!ch_wait(&br.rdy_b[stg], (it / STG) & 1, dead)) break;
          if (!ch_wait(&br.ds_free, ph ^ 1, dead)) break;
          bool ok = true;
#pragma unroll 1
          for (int pc = 0; pc < kPieces; ++pc) {
            if (WHOLE && pc == kPieces / 2) {
              // S C, half way: the split state is ready by then, and W need not wait for it
              ok = ch_wait(&br.s_full, ph, dead) && ch_wait(&br.raw_c, ph, dead) &&
                   ch_wait(&br.y_free, ph ^ 1, dead);
              if (!ok) break;
              tc_after();
#pragma unroll 4
              for (int i = 0; i < N / 8; ++i) {
                const int part = i / (N / 16), k = i % (N / 16);
                mma_ss(tmem + kTmY, dc + (((k >> 2) * kPanel + (k & 3) * 32) >> 4),
                       ds + ((part * 2 * Sm::kSPanel + k * 2048) >> 4), id_cs, i > 0);
              }
              ch_commit(&br.cs_done);
            }
            const int buf = pc & 1;
            ok = ch_wait(&br.w_full[buf], pc >> 1, dead);
            if (!ok) break;
            tc_after();
            // fewer than 128 state columns: the rows behind them repeat the first (panel stride 0)
            const uint64_t da = sw_desc(base + Sm::kB + stg * Sm::kTile + kWRows * pc * 128, N == 128 ? kPanel : 0);
            const uint64_t db = sw_desc(base + Sm::kW + 6 * buf * kWPanel, kWPanel);
#pragma unroll
            for (int part = 0; part < 3; ++part)
#pragma unroll
              for (int k = 0; k < kWRows / 16; ++k)
                mma_ss(tmem + kTmS, da + k * (2048 >> 4), db + (2 * part * kWPanel + k * 2048 >> 4), id_ds,
                       pc + part + k > 0);
            ch_commit(&br.w_free[buf]);
          }
          if (!ok) break;
          ch_commit(&br.b_free[stg]);
          ch_commit(&br.ds_done);
        }
        ch_commit(&br.mma_done);
        mbar_wait(&br.mma_done, 0, 2000000000LL);
      }
    } else {
      // ------------------------------------------- rows behind an end
      const uint4 zero = make_uint4(0, 0, 0, 0);
      Heads hd;
      for (int it = 0; it < count; ++it) {
        const uint32_t sph = (it / STG) & 1;
        const int valid = wk.valid(), stg = it % STG;
        if (!ch_wait_w(&br.raw_b[stg], sph, dead)) break;
        if (valid < kQ) {
          for (int i = lane; i < (kQ - valid) * 8; i += 32)
#pragma unroll
            for (int p = 0; p < N / 64; ++p)
              *reinterpret_cast<uint4*>(smem + Sm::kB + stg * Sm::kTile + p * kPanel + valid * 128 + i * 16) = zero;
          to_async();
        }
        ch_arrive_w(&br.rdy_b[stg]);
        if (!ch_wait_w(&br.raw_x[stg], sph, dead)) break;
        if (valid < kQ) {
          for (int i = lane; i < (kQ - valid) * 8; i += 32)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              *reinterpret_cast<uint4*>(smem + Sm::kX + (2 * stg + p) * kPanel + valid * 128 + i * 16) = zero;
          to_async();
        }
        ch_arrive_w(&br.rdy_x[stg]);
        if (it + 1 < count) {
          wk.next(a.pk);
          hd.at(a, wk.pair);
          if (lane < N / 64) {
            if (WHOLE) ch_prefetch(&c_map, hd.grp * N + 64 * lane, wk.row0());
            ch_prefetch(&b_map, hd.grp * N + 64 * lane, wk.row0());
          } else if (lane < N / 64 + 2) {
            ch_prefetch(&x_map, (lane == N / 64 ? hd.h[0] : hd.h[1]) * kP, wk.row0());
          }
          __syncwarp();
        }
      }
    }
  }
  tc_before();
  __syncthreads();
  if (tid == 0 && *dead) atomicExch(&g_device_error, kErrTimeout);
  if (warp == 25)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Pass 0: one warp computes the steps of one head of a pair in one chunk; a
// lane holds four tokens, eight lanes a block of 32.
constexpr int kStepThreads = 256;

// A warp finds the pieces of CTA c for both passes.
__device__ __noinline__ void scan_plan(const ChunkArgs& a, int c, int ctas) {
  int seq = 0, nth = 0, total = 0;
  find_tile(a.pk, -1, kQ, seq, nth, total);
  total = min(total, most_chunks(a.pk, kQ));
  const long long all = (long long)total * a.pairs;
  const long long f0 = cut(all, c, ctas), f1 = cut(all, c + 1, ctas);
  const int n = (int)(f1 - f0);
  Plan p3{}, p1{};
  if (n > 0) {
    int before = c - 1, t;
    while (before > 0 && cut(all, before, ctas) == f0) --before;
    p3.pair = (int)(f0 / total);
    p3.nth = (int)(f0 - (long long)p3.pair * total);
    find_tile(a.pk, p3.nth, kQ, p3.seq, p3.chunk, t);
    p3.count = n;
    p3.before = before;
    p3.total = total;
    // pass 1: its part of the sequence that its piece ends in, if that goes on
    p1.pair = (int)((f1 - 1) / total);
    const int last = (int)(f1 - 1 - (long long)p1.pair * total);
    find_tile(a.pk, last, kQ, p1.seq, p1.chunk, t);
    int b, len;
    seq_range(a.pk, p1.seq, b, len);
    if (p1.chunk < chunks_of(len) - 1) {
      p1.count = min(p1.chunk + 1, n);
      p1.chunk += 1 - p1.count;
      p1.nth = last + 1 - p1.count;
      p1.total = total;
    }
  }
  if ((threadIdx.x & 31) == 0) {
    a.plan[c] = p1;
    a.plan[kMaxCtas + c] = p3;
    a.meta[c] = p1.count == 0 ? 0 : (p1.pair << 2) + (p1.chunk == 0 ? 1 : 2);
  }
}

__global__ void __launch_bounds__(kStepThreads) scan_steps_kernel(ChunkArgs a, int ctas) {
  const int lane = threadIdx.x & 31, chunk = blockIdx.x;
  pass_next();
  if (blockIdx.y == gridDim.y - 1) {  // the last row of blocks: pieces
    const int c = blockIdx.x * (kStepThreads / 32) + (threadIdx.x >> 5);
    if (c < ctas) scan_plan(a, c, ctas);
    return;
  }
  const int ph = blockIdx.y * (kStepThreads / 32) + (threadIdx.x >> 5);  // pair and head
  int seq = 0, nth = 0, total = 0;
  if (!find_tile(a.pk, chunk, kQ, seq, nth, total) || ph >= 2 * a.pairs) return;
  if (a.pk.seqs > 1) {
    int s, n;
    find_tile(a.pk, -1, kQ, s, n, total);
  } else {
    int b, len;
    seq_range(a.pk, 0, b, len);
    total = chunks_of(len);
  }
  total = min(total, most_chunks(a.pk, kQ));
  const long long entry = step_entry(ph, chunk, total);
  if (entry < 0) return;
  Walk wk;
  wk.at(a.pk, ph >> 1, seq, nth);
  Heads hd;
  hd.at(a, ph >> 1);
  const int head = hd.h[ph & 1], valid = wk.valid(), row = wk.row0();
  const float bias = a.dt_bias ? a.dt_bias[head] : 0.0f, A2 = a.A[head] * 1.4426950408889634f;
  float d[4], e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * lane + i;
    d[i] = t < valid ? softplus(__bfloat162float(a.dt[(size_t)(row + t) * a.dt_stride + head]) + bias) : 0.0f;
    // exp2(-150) is 0 as every power below it; sums that held a longer step
    // would lose the distances between the tokens behind it (a NaN stays one)
    e[i] = d[i] * A2 < -150.0f ? -150.0f : d[i] * A2;
  }
  const float own = (e[0] + e[1]) + (e[2] + e[3]);
  float pre = own, post = own;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const float u = __shfl_up_sync(0xffffffffu, pre, o), v = __shfl_down_sync(0xffffffffu, post, o);
    if ((lane & 7) >= o) pre += u;
    if ((lane & 7) + o < 8) post += v;
  }
  float run = __shfl_up_sync(0xffffffffu, pre, 1), suf = __shfl_down_sync(0xffffffffu, post, 1);
  if ((lane & 7) == 0) run = 0.0f;
  if ((lane & 7) == 7) suf = 0.0f;
  const float b0 = __shfl_sync(0xffffffffu, pre, 7), b1 = __shfl_sync(0xffffffffu, pre, 15),
              b2 = __shfl_sync(0xffffffffu, pre, 23), b3 = __shfl_sync(0xffffffffu, pre, 31);
  const int blk = lane >> 3;
  const float after = blk == 0 ? b1 + b2 + b3 : blk == 1 ? b2 + b3 : blk == 2 ? b3 : 0.0f;
  float lp[4], v[4], w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    run += e[i];
    lp[i] = run;
  }
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    v[i] = d[i] * ex2(suf);
    w[i] = d[i] * ex2(suf + after);
    suf += e[i];
  }
  Steps& st = a.steps[entry];
  *reinterpret_cast<float4*>(&st.lp[4 * lane]) = make_float4(lp[0], lp[1], lp[2], lp[3]);
  *reinterpret_cast<float4*>(&st.d[4 * lane]) = make_float4(d[0], d[1], d[2], d[3]);
  *reinterpret_cast<float4*>(&st.v[4 * lane]) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(&st.w[4 * lane]) = make_float4(w[0], w[1], w[2], w[3]);
  if (lane == 0) {
    const float all = (b0 + b1) + (b2 + b3);
    *reinterpret_cast<float4*>(st.blk) = make_float4(b0, b1, b2, b3);
    st.all = ex2(all);
    st.sum = all;
    st.D = a.D ? a.D[head] : 0.0f;
  }
}

// Pass 2: along each head pair's pieces, in order, state after piece c =
// its own + its decay times the state after piece c - 1 of the same sequence.
// Also gives empty sequences without a carried state their zero state.
constexpr int kJoinThreads = 256;

__global__ void __launch_bounds__(kJoinThreads) scan_join_kernel(ChunkArgs a, int ctas) {
  __shared__ int list[kMaxCtas], count[kJoinThreads / 32];
  const int pair = blockIdx.y, tid = threadIdx.x, size = 2 * kP * a.n;
  pass_next();
  pass_wait();
  // this pair's pieces, in order
  const int m = tid < ctas ? a.meta[tid] : 0;
  const bool mine = (m & 3) && (m >> 2) == pair;
  const unsigned votes = __ballot_sync(0xffffffffu, mine);
  if ((tid & 31) == 0) count[tid >> 5] = __popc(votes);
  __syncthreads();
  int at = 0, total = 0;
  for (int i = 0; i < kJoinThreads / 32; ++i) {
    if (i < (tid >> 5)) at += count[i];
    total += count[i];
  }
  if (mine) list[at + __popc(votes & ((1u << (tid & 31)) - 1))] = tid * 4 + (m & 3);
  __syncthreads();
  const int e = (blockIdx.x * kJoinThreads + tid) * 4;
  if (e < size) {
    const int h = e / (kP * a.n);
    float4 carry = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int i = 0; i < total; ++i) {
      const int c = list[i] >> 2;
      float4* p = reinterpret_cast<float4*>(a.local + (size_t)c * size + e);
      float4 v = *p;
      if ((list[i] & 3) == 2) {
        const float d = a.decay[2 * c + h];
        v.x = fmaf(d, carry.x, v.x);
        v.y = fmaf(d, carry.y, v.y);
        v.z = fmaf(d, carry.z, v.z);
        v.w = fmaf(d, carry.w, v.w);
      }
      carry = v;
      *p = v;
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
// enough tokens: below, the token-by-token kernel's time (0.4 us a token of one
// sequence) is less than four launches and a chunk's latency.  One sequence of 33
// tokens takes 18 us in chunks and 17 token by token, of 64 tokens 18 and 28 (64
// heads, 128 states).  The rule looks at the tokens of the whole call, while a
// sequence costs a chunk's step however short it is: 8 sequences of 5 take 27 us
// in chunks and 18 token by token, 32 of 8 63 and 66, 96 of 2 161 and 122, 256
// of 16 421 and 752.  And no more than
// kMaxChunkSeqs sequences: pass 0 walks all offsets for every chunk, and every
// role of passes 1 and 3 steps through empty sequences one by one while the
// others' waits, which are bounded, run.
constexpr int kMaxChunkSeqs = 16384;
bool chunk_sizes(int type, int tokens, int seqs, int head_dim, int d_state) {
  return type == kTypeBF16 && head_dim == kP && (d_state == 64 || d_state == 128) && tokens > 32 &&
         seqs <= kMaxChunkSeqs;
}

// The register shares need every register that the block is launched with: a
// build that gave the kernel fewer must not run, its warps would wait for ever.
bool chunk_kernel_ok(const void* fn, int smem) {
  cudaFuncAttributes at;
  return cudaFuncGetAttributes(&at, fn) == cudaSuccess && at.numRegs >= kRegs &&
         cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess;
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
  const long long chunks = most_chunks(s.pk, kQ);
  a.steps = static_cast<Steps*>(s.scratch);
  a.local = reinterpret_cast<float*>(a.steps + 2 * chunks * a.pairs);
  a.init = a.local + part;
  a.decay = a.init + part;
  a.meta = reinterpret_cast<int*>(a.decay + 2 * kMaxCtas);
  a.plan = reinterpret_cast<Plan*>(a.meta + 2 * kMaxCtas);
  CUtensorMap xm, bm, cm;
  if (int e = ch_map(&xm, s.x, s.pk.tokens, s.heads * kP, s.x_stride)) return e;
  if (int e = ch_map(&bm, s.B, s.pk.tokens, s.groups * N, s.b_stride)) return e;
  if (int e = ch_map(&cm, s.C, s.pk.tokens, s.groups * N, s.c_stride)) return e;
  auto pass1 = scan_chunk_kernel<N, false>;
  auto pass3 = scan_chunk_kernel<N, true>;
  constexpr int smem1 = ChunkSmem<N, false>::kBytes, smem3 = ChunkSmem<N, true>::kBytes;
  if (!chunk_kernel_ok((const void*)pass1, smem1) || !chunk_kernel_ok((const void*)pass3, smem3)) return kErrLaunch;
  const long long most = chunks * a.pairs;
  int ctas = device_sm_count();
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  if (most < ctas) ctas = (int)most;
  // one warp a (chunk, head) and, in a last row of blocks, one a CTA's piece
  const unsigned plans = (ctas + kStepThreads / 32 - 1) / (kStepThreads / 32);
  scan_steps_kernel<<<dim3(chunks > plans ? (unsigned)chunks : plans,
                           (2 * a.pairs + kStepThreads / 32 - 1) / (kStepThreads / 32) + 1),
                      kStepThreads, 0, stream>>>(a, ctas);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t chunk{}, join{};
  chunk.gridDim = dim3((unsigned)ctas);
  chunk.blockDim = dim3(kChThreads);
  chunk.dynamicSmemBytes = smem1;
  join.gridDim = dim3((2 * kP * N / 4 + kJoinThreads - 1) / kJoinThreads, a.pairs);
  join.blockDim = dim3(kJoinThreads);
  chunk.stream = join.stream = stream;
  chunk.attrs = join.attrs = &attr;
  chunk.numAttrs = join.numAttrs = 1;
  if (cudaLaunchKernelEx(&chunk, pass1, xm, bm, cm, a) != cudaSuccess ||
      cudaLaunchKernelEx(&join, scan_join_kernel, a, ctas) != cudaSuccess)
    return kErrLaunch;
  chunk.dynamicSmemBytes = smem3;
  if (cudaLaunchKernelEx(&chunk, pass3, xm, bm, cm, a) != cudaSuccess) return kErrLaunch;
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace

size_t ssm_prompt_scratch_bytes(int type, int tokens, int seqs, int heads, int head_dim, int groups, int d_state) {
  if (!chunk_sizes(type, tokens, seqs, head_dim, d_state)) return 0;
  const size_t pairs = (size_t)(heads / groups + 1) / 2 * groups;
  return ((size_t)tokens / kQ + seqs) * pairs * 2 * sizeof(Steps) + (size_t)kMaxCtas * (4 * kP * d_state * 4 + 16 + 2 * sizeof(Plan));
}

int launch_ssm_prompt(const ScanArgs& a, cudaStream_t stream) {
  if (chunk_sizes(a.type, a.pk.tokens, a.pk.seqs, a.head_dim, a.d_state) && rows16(a.x, a.x_stride) &&
      rows16(a.B, a.b_stride) && rows16(a.C, a.c_stride) && rows16(a.y, a.y_stride))
    return a.d_state == 128 ? launch_chunks<128>(a, stream) : launch_chunks<64>(a, stream);
  return launch_scan_tokens(a, stream);
}

int read_scan_device_error(bool clear) { return read_unit_error(clear); }

}  // namespace ervf
