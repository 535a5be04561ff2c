// ssm.cu -- the state-space layer of the hybrid next to its routed experts:
// causal convolution, selective scan (token by token), one-token step and
// gated norm.  The reference runs these one token at a time (conv1d, ssm,
// softplus, gated_rmsnorm: gpu_kernels.py:77-1515); here prompts are packed
// sequences, and a decode step is one launch.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "kernels.h"
#include "ssm.h"
#include "ssm_dev.cuh"

namespace cg = cooperative_groups;

namespace ervf {

namespace {

// ------------------------------------------------------------ small helpers

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements as they lie in memory, V = 1 or V elements one load's
// width (8 or 16 bytes) apart.
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * (int)sizeof(T), kWords = kBytes < 4 ? 1 : kBytes / 4;
  static_assert(V == 1 || kBytes == 8 || kBytes == 16, "one load");
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (kBytes == 8) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      w[0] = q.x; w[1] = q.y;
    } else {
      const uint4 q = *reinterpret_cast<const uint4*>(p);
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float((i & 1) ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  }
  __device__ __forceinline__ void set(const float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (V == 1) {
      w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 2) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(v[i + 1]), "f"(v[i]));
    }
  }
};

// ------------------------------------------------------------- convolution

// y_t = act(bias + sum_j w[j] x[t - width + 1 + j]) for each channel.  A
// thread owns V channels of one tile of a sequence, keeps the window in
// registers and the next tokens' loads in flight while it works on as many
// (eight of bf16: 8192 tokens of 6144 channels in 45 us, 4.5 TB/s; four of
// f32, which at eight ran short of registers).
// Bound by HBM and, near it, by the two special-function operations of each
// silu: every input is read once (and `width - 1` rows again per tile, from
// L2), every output written once.  The thread of a sequence's first tile is
// the only one that touches the carried state: it reads the old inputs, and
// writes the sequence's last `width - 1` ones.
constexpr int kConvThreads = 128;

template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads, sizeof(T) == 2 ? 5 : 6) conv_prompt_kernel(ConvArgs a) {
  const int ch = (blockIdx.y * kConvThreads + threadIdx.x) * V;
  int seq, nth, begin, len;
  if (!find_place(a.pk, blockIdx.x, a.shift, seq, nth, begin, len)) return;
  const int tile = 1 << a.shift;
  // an empty sequence's first tile carries its state on
  if (ch >= a.channels || (nth > 0 && (long long)nth * tile >= len)) return;
  const int t0 = nth * tile, t1 = min(t0 + tile, len);
  const T* x = static_cast<const T*>(a.x) + (size_t)(begin + t0) * a.x_stride + ch;
  T* out = static_cast<T*>(a.out) + (size_t)(begin + t0) * a.out_stride + ch;
  int left = t1 - t0;
  constexpr int kConvAhead = sizeof(T) == 2 ? 8 : 4;
  Raw<T, V> next[kConvAhead];
  auto ahead = [&](const T* p, int n) {
#pragma unroll
    for (int u = 0; u < kConvAhead; ++u)
      if (u < n) next[u].load(p + (size_t)u * a.x_stride);
  };
  ahead(x, left);
  Raw<T, V> old[W - 1];  // the W - 1 inputs before the tile, oldest first
  const int slot = nth == 0 && a.state ? seq_slot(a.pk, seq) : -1;
  T* state = slot < 0 ? nullptr : static_cast<T*>(a.state) + (size_t)slot * (W - 1) * a.channels + ch;
  const bool carried = state && a.pk.has && a.pk.has[seq];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int back = W - 1 - j;
    if (t0 >= back) old[j].load(x - (size_t)back * a.x_stride);
    else if (carried) old[j].load(state + (size_t)j * a.channels);
    else old[j].clear();
  }
  if (state) {
    // last W - 1 inputs of [carried state, sequence]
    Raw<T, V> last[W - 1];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const int t = len - (W - 1) + j;
      if (t >= 0) {
        last[j].load(x + (size_t)t * a.x_stride);
      } else {
        last[j].clear();
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
          if (t + (W - 1) == k) last[j] = old[k];
      }
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) last[j].store(state + (size_t)j * a.channels);
  }
  float w[V][W], bias[V], win[W - 1][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = a.bias ? a.bias[ch + v] : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[v][j] = a.w[(size_t)(ch + v) * W + j];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) win[j][v] = old[j].get(v);
  }
  auto token = [&](const Raw<T, V>& c, T* o) {
    float y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float e = c.get(v);
      float sum = bias[v];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) sum = fmaf(w[v][j], win[j][v], sum);
      sum = fmaf(w[v][W - 1], e, sum);
      y[v] = a.silu ? silu(sum) : sum;
#pragma unroll
      for (int j = 0; j + 1 < W - 1; ++j) win[j][v] = win[j + 1][v];
      win[W - 2][v] = e;
    }
    Raw<T, V> q;
    q.set(y);
    q.store(o);
  };
  while (left > 0) {
    Raw<T, V> cur[kConvAhead];
#pragma unroll
    for (int u = 0; u < kConvAhead; ++u) cur[u] = next[u];
    x += (size_t)kConvAhead * a.x_stride;
    ahead(x, left - kConvAhead);
    if (left >= kConvAhead) {
#pragma unroll
      for (int u = 0; u < kConvAhead; ++u) token(cur[u], out + (size_t)u * a.out_stride);
    } else {
#pragma unroll
      for (int u = 0; u < kConvAhead - 1; ++u)
        if (u < left) token(cur[u], out + (size_t)u * a.out_stride);
    }
    out += (size_t)kConvAhead * a.out_stride;
    left -= kConvAhead;
  }
}

template <typename T, int V>
int launch_conv(ConvArgs a, cudaStream_t stream) {
  // 64 tokens a tile spread the weights' loads further; 32 where that would
  // leave the SMs short of CTAs
  const long long cols = (a.channels + kConvThreads * V - 1) / (kConvThreads * V);
  a.shift = (a.pk.tokens / 64 + a.pk.seqs) * cols >= 12LL * device_sm_count() ? 6 : 5;
  const dim3 grid((unsigned)((a.pk.tokens >> a.shift) + a.pk.seqs), (unsigned)cols);
  if (a.width == 2) conv_prompt_kernel<T, 2, V><<<grid, kConvThreads, 0, stream>>>(a);
  else if (a.width == 3) conv_prompt_kernel<T, 3, V><<<grid, kConvThreads, 0, stream>>>(a);
  else conv_prompt_kernel<T, 4, V><<<grid, kConvThreads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

// Vectors of `bytes` fit a row-strided array.
bool vec_ok(const void* p, long long stride, size_t elem, unsigned bytes = 16) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && ((unsigned long long)stride * elem & (bytes - 1)) == 0;
}

// --------------------------------------------------- scan, token by token

// The recurrence as it stands: S = exp(d A) S + d x B^T, y = S C + D x, with
// d = softplus(dt + bias).  Four neighbouring lanes share one row p of one
// head's state, NL columns each (columns n with (n / 4) % 4 == lane part), in
// registers; B, C, x and the steps of kSeqTile tokens at a time lie in shared
// memory.  Serves every type and size; its time is the length of a sequence
// times the latency of one step: 8192 tokens of 64 heads of 64 with 128 states
// take 3.7 ms in f32 and 4.7 in bf16, where HBM would need 0.05 and 0.03.
// PAD: fewer state columns than 4 NL; those behind them take no part in a step,
// whose x may be infinite (0 times it is NaN).
constexpr int kSeqRows = 32, kSeqThreads = 4 * kSeqRows, kSeqTile = 16;

template <typename T, int NL, bool PAD>
__global__ void __launch_bounds__(kSeqThreads) scan_seq_kernel(ScanArgs a) {
  constexpr int N = 4 * NL;
  __shared__ __align__(16) float sB[kSeqTile][N], sC[kSeqTile][N];
  __shared__ float sx[kSeqTile][kSeqRows], sd[kSeqTile], sa[kSeqTile];
  const int seq = blockIdx.x, head = blockIdx.y, p0 = blockIdx.z * kSeqRows;
  const int tid = threadIdx.x, part = tid & 3, row = tid >> 2, p = p0 + row;
  const int n_real = a.d_state, grp = head / (a.heads / a.groups);
  int begin, len;
  seq_range(a.pk, seq, begin, len);
  const int slot = a.state ? seq_slot(a.pk, seq) : -1;
  const bool live = p < a.head_dim;
  float* state = slot < 0 || !live ? nullptr
      : a.state + (((size_t)slot * a.heads + head) * a.head_dim + p) * n_real;
  const bool has = state && a.pk.has && a.pk.has[seq];
  float s[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int n = (i >> 2) * 16 + part * 4 + (i & 3);
    s[i] = has && n < n_real ? state[n] : 0.0f;
  }
  const float A = a.A[head], D = a.D ? a.D[head] : 0.0f, bias = a.dt_bias ? a.dt_bias[head] : 0.0f;
  const T* gx = static_cast<const T*>(a.x) + (size_t)begin * a.x_stride + (size_t)head * a.head_dim + p0;
  const T* gd = static_cast<const T*>(a.dt) + (size_t)begin * a.dt_stride + head;
  const T* gb = static_cast<const T*>(a.B) + (size_t)begin * a.b_stride + (size_t)grp * n_real;
  const T* gc = static_cast<const T*>(a.C) + (size_t)begin * a.c_stride + (size_t)grp * n_real;
  T* gy = static_cast<T*>(a.y) + (size_t)begin * a.y_stride + (size_t)head * a.head_dim + p;
  for (int t0 = 0; t0 < len; t0 += kSeqTile) {
    const int m = min(kSeqTile, len - t0);
    __syncthreads();
    for (int i = tid; i < m * N; i += kSeqThreads) {
      const int t = i / N, n = i - t * N;
      sB[t][n] = n < n_real ? to_f32(gb[(size_t)(t0 + t) * a.b_stride + n]) : 0.0f;
      sC[t][n] = n < n_real ? to_f32(gc[(size_t)(t0 + t) * a.c_stride + n]) : 0.0f;
    }
    for (int i = tid; i < m * kSeqRows; i += kSeqThreads) {
      const int t = i / kSeqRows, r = i - t * kSeqRows;
      sx[t][r] = p0 + r < a.head_dim ? to_f32(gx[(size_t)(t0 + t) * a.x_stride + r]) : 0.0f;
    }
    if (tid < m) {
      const float d = softplus(to_f32(gd[(size_t)(t0 + tid) * a.dt_stride]) + bias);
      sd[tid] = d;
      sa[tid] = expf(d * A);
    }
    __syncthreads();
    for (int t = 0; t < m; ++t) {
      const float x = sx[t][row], dx = sd[t] * x, da = sa[t];
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NL; i += 4) {
        const float4 b = *reinterpret_cast<const float4*>(&sB[t][i * 4 + part * 4]);
        const float4 c = *reinterpret_cast<const float4*>(&sC[t][i * 4 + part * 4]);
        const int left = n_real - (i * 4 + part * 4);  // real columns from here on
        s[i] = fmaf(!PAD || left > 0 ? dx : 0.0f, b.x, da * s[i]);
        s[i + 1] = fmaf(!PAD || left > 1 ? dx : 0.0f, b.y, da * s[i + 1]);
        s[i + 2] = fmaf(!PAD || left > 2 ? dx : 0.0f, b.z, da * s[i + 2]);
        s[i + 3] = fmaf(!PAD || left > 3 ? dx : 0.0f, b.w, da * s[i + 3]);
        y[0] = fmaf(s[i], c.x, y[0]);
        y[1] = fmaf(s[i + 1], c.y, y[1]);
        y[2] = fmaf(s[i + 2], c.z, y[2]);
        y[3] = fmaf(s[i + 3], c.w, y[3]);
      }
      float v = (y[0] + y[1]) + (y[2] + y[3]);
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (part == 0 && live) gy[(size_t)(t0 + t) * a.y_stride] = from_f32<T>(fmaf(D, x, v));
    }
  }
  if (state) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int n = (i >> 2) * 16 + part * 4 + (i & 3);
      if (n < n_real) state[n] = s[i];
    }
  }
}

template <typename T, int NL>
void scan_seq(const ScanArgs& a, cudaStream_t stream) {
  const dim3 grid(a.pk.seqs, a.heads, (a.head_dim + kSeqRows - 1) / kSeqRows);
  if (a.d_state == 4 * NL) scan_seq_kernel<T, NL, false><<<grid, kSeqThreads, 0, stream>>>(a);
  else scan_seq_kernel<T, NL, true><<<grid, kSeqThreads, 0, stream>>>(a);
}

template <typename T>
int launch_scan_seq(const ScanArgs& a, cudaStream_t stream) {
  if (a.d_state <= 16) scan_seq<T, 4>(a, stream);
  else if (a.d_state <= 64) scan_seq<T, 16>(a, stream);
  else if (a.d_state <= 128) scan_seq<T, 32>(a, stream);
  else scan_seq<T, 64>(a, stream);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

// --------------------------------------------------------- one-token step

// One token of each sequence: convolution, scan step and gated norm in one
// launch.  A cluster of CTAs owns one (sequence, group): CTA r takes heads
// r, r + c, ... of the group.  The heads' states are read and written once,
// which is what the launch costs for a batch (2 x 4 bytes per state element,
// HBM bound); for one sequence it is latency: one round of loads, the
// cluster's two barriers, one round of stores.
//  0. the first rows of the first head's state start on their way;
//  1. every CTA convolves its heads' x channels and, for itself, the group's
//     B and C channels (2 d_state of them: recomputing is cheaper than
//     sending them on), and arrives at the cluster's barrier;
//  2. the states' update and y: L lanes share a row of d_state, a lane works
//     on kRows rows while the next ones are on their way;
//  3. behind the barrier (every CTA has read the carried B / C inputs) CTA 0
//     stores those inputs moved on by one token, and every CTA its sum of
//     squares into each other's shared memory;
//  4. behind a second one the sums are added in rank order: norm and output.
constexpr int kTokThreads = 256;

// What a channel's convolution reads: oldest input first, the new one last.
template <typename T>
struct Taps {
  T v[kMaxConvWidth];
  float w[kMaxConvWidth], bias;
  // all loads before any use; fewer taps than the most leave the first ones zero
  __device__ __forceinline__ void load(const TokenArgs& a, const T* xin, const T* cs, size_t channels, int ch) {
    const int gap = kMaxConvWidth - a.width;
#pragma unroll
    for (int j = 0; j < kMaxConvWidth; ++j) {
      w[j] = j >= gap ? a.conv_w[(size_t)ch * a.width + j - gap] : 0.0f;
      if (j == kMaxConvWidth - 1) v[j] = xin[ch];
      else v[j] = j >= gap && cs ? cs[(size_t)(j - gap) * channels + ch] : from_f32<T>(0.0f);
    }
    bias = a.conv_bias ? a.conv_bias[ch] : 0.0f;
  }
  __device__ __forceinline__ float value() const {
    float s = bias;
#pragma unroll
    for (int j = 0; j < kMaxConvWidth; ++j) s = fmaf(w[j], to_f32(v[j]), s);
    return silu(s);
  }
};

// L lanes of four columns each share a row, NV times over.
template <typename T, int L, int NV>
__global__ void __launch_bounds__(kTokThreads, 4) ssm_token_kernel(TokenArgs a) {
  constexpr int kRows = 4 / NV;                                   // rows of a lane at a time
  constexpr int kStep = kTokThreads / L, kBatch = kRows * kStep;  // rows of the CTA
  constexpr int kWarps = kTokThreads / 32, kOld = kMaxConvWidth - 1;
  extern __shared__ __align__(16) float sm[];
  cg::cluster_group cl = cg::this_cluster();
  const int c = (int)cl.num_blocks(), r = (int)cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x / c, seq = unit / a.groups, grp = unit - seq * a.groups;
  const int hpg = a.heads / a.groups, P = a.head_dim, N = a.d_state;
  const int mine = (hpg - r + c - 1) / c, most = (hpg + c - 1) / c;  // heads of this CTA: r, r + c, ...
  float* sBC = sm;                  // B then C of the group
  float* sy = sBC + 2 * N;          // [mine][P]: x, then the gated output
  float* sz = sy + most * P;        // [mine][P]: silu(z)
  float* sh = sz + most * P;        // [mine]: d, exp(d A), D
  float* red = sh + 3 * most;       // per-warp sums, then the ranks'
  T* old = reinterpret_cast<T*>(red + kWarps + 16);  // rank 0: the B / C inputs to carry on
  const int s0 = a.slots ? a.slots[seq] : seq;
  const int slot = s0 >= 0 && s0 < a.n_slots ? s0 : -1;
  const size_t channels = (size_t)a.heads * P + 2 * (size_t)a.groups * N;
  const T* xin = static_cast<const T*>(a.xbc) + (size_t)seq * a.xbc_stride;
  T* cs = slot < 0 ? nullptr : static_cast<T*>(a.conv_state) + (size_t)slot * (a.width - 1) * channels;
  const int sub = tid / L, n0 = (tid % L) * 4;
  const int batches = (P + kBatch - 1) / kBatch, rounds = mine * batches;
  float4 next[kRows][NV];
  // this lane's first element of head k's state from row p0, where there is a slot
  auto state_at = [&](int k, int p0) {
    return a.state + (((size_t)max(slot, 0) * a.heads + grp * hpg + r + k * c) * P + p0 + sub) * N + n0;
  };
  // rows p0 + sub, p0 + sub + kStep, ...
  auto load = [&](const float* st, int p0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < NV; ++j)
        next[i][j] = slot >= 0 && p0 + i * kStep + sub < P && n0 + j * 4 * L < N
                         ? *reinterpret_cast<const float4*>(st + i * kStep * N + j * 4 * L)
                         : make_float4(0, 0, 0, 0);
  };
  load(state_at(0, 0), 0);
  if (tid >= kTokThreads - 32)
    for (int k = lane; k < mine; k += 32) {
      const int head = grp * hpg + r + k * c;
      const float d = softplus(to_f32(static_cast<const T*>(a.dt)[(size_t)seq * a.dt_stride + head]) +
                               (a.dt_bias ? a.dt_bias[head] : 0.0f));
      sh[3 * k] = d;
      sh[3 * k + 1] = expf(d * a.A[head]);
      sh[3 * k + 2] = a.D ? a.D[head] : 0.0f;
    }
  for (int i = tid; i < 2 * N + mine * P; i += kTokThreads) {
    Taps<T> t;
    if (i < 2 * N) {
      const int ch = a.heads * P + (i < N ? grp * N + i : (a.groups + grp) * N + i - N);
      t.load(a, xin, cs, channels, ch);
      sBC[i] = t.value();
      if (r == 0)
#pragma unroll
        for (int j = 0; j < kOld; ++j) old[j * 2 * N + i] = t.v[j + 1];
    } else {
      const int e = i - 2 * N, k = e / P, ch = (grp * hpg + r + k * c) * P + e - k * P;
      t.load(a, xin, cs, channels, ch);
      const float z = a.z ? to_f32(static_cast<const T*>(a.z)[(size_t)seq * a.z_stride + ch]) : 0.0f;
      sy[e] = t.value();
      sz[e] = a.z ? silu(z) : 1.0f;
      if (cs)
#pragma unroll
        for (int j = 0; j < kOld; ++j)
          if (j >= kMaxConvWidth - a.width) cs[(size_t)(j - kMaxConvWidth + a.width) * channels + ch] = t.v[j + 1];
    }
  }
  cl.barrier_arrive();
  __syncthreads();
  float4 b[NV], cc[NV];  // this lane's columns of B and C
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = n0 + j * 4 * L;
    b[j] = n < N ? *reinterpret_cast<const float4*>(sBC + n) : make_float4(0, 0, 0, 0);
    cc[j] = n < N ? *reinterpret_cast<const float4*>(sBC + N + n) : make_float4(0, 0, 0, 0);
  }
  float ss = 0.0f;
  int k = 0, p0 = 0;
  float* st = state_at(0, 0);
  for (int i = 0; i < rounds; ++i) {
    float4 v[kRows][NV];
#pragma unroll
    for (int q = 0; q < kRows; ++q)
#pragma unroll
      for (int j = 0; j < NV; ++j) v[q][j] = next[q][j];
    int k1 = k, p1 = p0 + kBatch;
    float* st1 = st + kBatch * N;
    if (p1 >= P) {
      ++k1;
      p1 = 0;
      st1 = state_at(k1, 0);
    }
    if (i + 1 < rounds) load(st1, p1);
    const float d = sh[3 * k], da = sh[3 * k + 1], D = sh[3 * k + 2];
    float x[kRows], y[kRows];
#pragma unroll
    for (int q = 0; q < kRows; ++q) {
      const int p = p0 + q * kStep + sub;
      x[q] = p < P ? sy[k * P + p] : 0.0f;
      const float dx = d * x[q];
      y[q] = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float4 e = v[q][j];
        e.x = fmaf(dx, b[j].x, da * e.x);
        e.y = fmaf(dx, b[j].y, da * e.y);
        e.z = fmaf(dx, b[j].z, da * e.z);
        e.w = fmaf(dx, b[j].w, da * e.w);
        const bool real = n0 + j * 4 * L < N;  // the others' 0 times an infinite x is NaN
        if (slot >= 0 && p < P && real) *reinterpret_cast<float4*>(st + q * kStep * N + j * 4 * L) = e;
        const float sum = fmaf(e.x, cc[j].x, fmaf(e.y, cc[j].y, fmaf(e.z, cc[j].z, fmaf(e.w, cc[j].w, y[q]))));
        y[q] = real ? sum : y[q];
      }
    }
    // the rows' sums over their L lanes: each halving step leaves a lane half
    // of the rows, until it has one
    int off = L / 2, mine_q = 0;
#pragma unroll
    for (int rows = kRows; rows > 1; rows >>= 1, off >>= 1) {
      const bool up = tid & off;
#pragma unroll
      for (int q = 0; q < rows / 2; ++q) {
        const float keep = up ? y[q + rows / 2] : y[q], give = up ? y[q] : y[q + rows / 2];
        y[q] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        x[q] = up ? x[q + rows / 2] : x[q];
      }
      mine_q += up ? rows / 2 : 0;
    }
    for (; off; off >>= 1) y[0] += __shfl_xor_sync(0xffffffffu, y[0], off);
    const int p = p0 + mine_q * kStep + sub;
    __syncwarp();  // every x of these rows is read
    if ((tid & (L / kRows - 1)) == 0 && p < P) {
      const float g = fmaf(D, x[0], y[0]) * sz[k * P + p];
      ss = fmaf(g, g, ss);
      sy[k * P + p] = g;
    }
    __syncwarp();
    k = k1;
    p0 = p1;
    st = st1;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  cl.barrier_wait();
  if (r == 0 && cs)
    for (int i = tid; i < 2 * N; i += kTokThreads) {
      const int ch = a.heads * P + (i < N ? grp * N + i : (a.groups + grp) * N + i - N);
#pragma unroll
      for (int j = 0; j < kOld; ++j)
        if (j >= kMaxConvWidth - a.width)
          cs[(size_t)(j - kMaxConvWidth + a.width) * channels + ch] = old[j * 2 * N + i];
    }
  float scale = 1.0f;
  if (a.norm_w) {
    if (tid < c) {
      float t = 0.0f;
      for (int i = 0; i < kWarps; ++i) t += red[i];
      *cl.map_shared_rank(red + kWarps + r, tid) = t;
    }
    cl.sync();
    float t = 0.0f;
    for (int i = 0; i < c; ++i) t += red[kWarps + i];
    scale = rsqrtf(t / (float)(hpg * P) + a.eps);
  }
  T* out = static_cast<T*>(a.out) + (size_t)seq * a.out_stride;
  for (int i = tid; i < mine * P; i += kTokThreads) {
    const int k = i / P, ch = (grp * hpg + r + k * c) * P + i - k * P;
    const float v = sy[i] * scale;
    out[ch] = from_f32<T>(a.norm_w ? v * a.norm_w[ch] : v);
  }
}

template <typename T>
const void* token_kernel(int d_state) {
  if (d_state <= 32) return (const void*)ssm_token_kernel<T, 8, 1>;
  if (d_state <= 64) return (const void*)ssm_token_kernel<T, 16, 1>;
  if (d_state <= 128) return (const void*)ssm_token_kernel<T, 32, 1>;
  return (const void*)ssm_token_kernel<T, 32, 2>;
}

// -------------------------------------------------------------- gated norm

// g = y silu(z), out = w g / sqrt(mean(g^2) + eps) per group of channels.
// Bound by HBM.  A warp holds one group's row in registers (NV vectors of 16
// bytes a lane) and its weights for all the tokens that it walks.
constexpr int kNormThreads = 128;

template <typename T, int NV>
__global__ void __launch_bounds__(kNormThreads, NV <= 2 ? 8 : 4) gated_norm_warp_kernel(NormArgs a) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, grp = blockIdx.y;
  const size_t off = (size_t)grp * a.group_size;
  const T* y = static_cast<const T*>(a.y) + off;
  const T* z = a.z ? static_cast<const T*>(a.z) + off : nullptr;
  T* out = static_cast<T*>(a.out) + off;
  float w[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const int i = (k * 32 + lane) * V + j;
      const float4 q = i < a.group_size ? make_float4(a.w[off + i], a.w[off + i + 1], a.w[off + i + 2], a.w[off + i + 3])
                                        : make_float4(0, 0, 0, 0);
      w[k][j] = q.x; w[k][j + 1] = q.y; w[k][j + 2] = q.z; w[k][j + 3] = q.w;
    }
  const long long step = (long long)gridDim.x * (kNormThreads / 32);
  for (long long t = (long long)blockIdx.x * (kNormThreads / 32) + (threadIdx.x >> 5); t < a.tokens; t += step) {
    Raw<T, V> ry[NV], rz[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * 32 + lane) * V;
      if (i < a.group_size) {
        ry[k].load(y + (size_t)t * a.y_stride + i);
        if (z) rz[k].load(z + (size_t)t * a.z_stride + i);
      }
    }
    float g[NV][V], ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if ((k * 32 + lane) * V < a.group_size) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          g[k][j] = z ? ry[k].get(j) * silu(rz[k].get(j)) : ry[k].get(j);
          ss = fmaf(g[k][j], g[k][j], ss);
        }
      }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float scale = rsqrtf(ss / (float)a.group_size + a.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * 32 + lane) * V;
      if (i < a.group_size) {
#pragma unroll
        for (int j = 0; j < V; ++j) g[k][j] *= scale * w[k][j];
        ry[k].set(g[k]);
        ry[k].store(out + (size_t)t * a.out_stride + i);
      }
    }
  }
}

// Any size and alignment: one CTA per (token, group), two passes over a row.
// 8192 x 4096 in bf16: 77 us off 16-byte rows in groups of 512, 72 as one group (a
// warp per group: 37), f32 as one group 108 (63).
template <typename T>
__global__ void __launch_bounds__(kNormThreads) gated_norm_kernel(NormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const long long unit = blockIdx.x;
  const long long t = unit / a.groups;
  const int grp = (int)(unit - t * a.groups), tid = threadIdx.x;
  const size_t off = (size_t)grp * a.group_size;
  const T* y = static_cast<const T*>(a.y) + (size_t)t * a.y_stride + off;
  const T* z = a.z ? static_cast<const T*>(a.z) + (size_t)t * a.z_stride + off : nullptr;
  T* out = static_cast<T*>(a.out) + (size_t)t * a.out_stride + off;
  float ss = 0.0f;
  for (int i = tid; i < a.group_size; i += kNormThreads) {
    const float g = to_f32(y[i]) * (z ? silu(to_f32(z[i])) : 1.0f);
    ss = fmaf(g, g, ss);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if ((tid & 31) == 0) red[tid >> 5] = ss;
  __syncthreads();
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kNormThreads / 32; ++i) ss += red[i];
  const float scale = rsqrtf(ss / (float)a.group_size + a.eps);
  for (int i = tid; i < a.group_size; i += kNormThreads) {
    const float g = to_f32(y[i]) * (z ? silu(to_f32(z[i])) : 1.0f);
    out[i] = from_f32<T>(g * (scale * a.w[off + i]));
  }
}

template <typename T>
int launch_norm(const NormArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int nv = (a.group_size + 32 * V - 1) / (32 * V);
  // a row of up to four vectors a lane stays in registers
  if (a.group_size % V == 0 && nv <= 4 && a.groups <= 65535 && vec_ok(a.y, a.y_stride, sizeof(T)) &&
      vec_ok(a.z, a.z ? a.z_stride : 0, sizeof(T)) && vec_ok(a.out, a.out_stride, sizeof(T))) {
    const long long rows = ((long long)a.tokens + kNormThreads / 32 - 1) / (kNormThreads / 32);
    const long long most = ((nv <= 2 ? 8LL : 4LL) * device_sm_count() + a.groups - 1) / a.groups;  // one wave, walking
    const dim3 grid((unsigned)(rows < most ? rows : most), a.groups);
    if (nv == 1) gated_norm_warp_kernel<T, 1><<<grid, kNormThreads, 0, stream>>>(a);
    else if (nv == 2) gated_norm_warp_kernel<T, 2><<<grid, kNormThreads, 0, stream>>>(a);
    else if (nv == 3) gated_norm_warp_kernel<T, 3><<<grid, kNormThreads, 0, stream>>>(a);
    else gated_norm_warp_kernel<T, 4><<<grid, kNormThreads, 0, stream>>>(a);
  } else {
    gated_norm_kernel<T><<<(unsigned)((long long)a.tokens * a.groups), kNormThreads, 0, stream>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace

int launch_conv1d_prompt(const ConvArgs& a, cudaStream_t stream) {
  const unsigned e = a.type == kTypeBF16 ? 2 : 4;
  const bool vec = a.channels % 4 == 0 && vec_ok(a.x, a.x_stride, e, 4 * e) && vec_ok(a.out, a.out_stride, e, 4 * e) &&
                   vec_ok(a.state, a.channels, e, 4 * e);
  if (a.type == kTypeBF16)
    return vec ? launch_conv<__nv_bfloat16, 4>(a, stream) : launch_conv<__nv_bfloat16, 1>(a, stream);
  return vec ? launch_conv<float, 4>(a, stream) : launch_conv<float, 1>(a, stream);
}

int launch_scan_tokens(const ScanArgs& a, cudaStream_t stream) {
  return a.type == kTypeBF16 ? launch_scan_seq<__nv_bfloat16>(a, stream) : launch_scan_seq<float>(a, stream);
}

int launch_ssm_token(const TokenArgs& a, cudaStream_t stream) {
  const int hpg = a.heads / a.groups;
  // as many CTAs a group as its heads, but no more than three waves of them: a
  // batch of 96 with eight groups took 117 us with eight CTAs a group, 93 with
  // four, 86 with two and 97 with one (each convolves B and C for itself; two take
  // 79 since the rows' sums go by halves); one sequence's latency is least with
  // eight
  const size_t elem = a.type == kTypeBF16 ? 2 : 4;
  auto smem_of = [&](int ctas) {
    const size_t most = (hpg + ctas - 1) / ctas;
    return (2 * (size_t)a.d_state + 2 * most * a.head_dim + 3 * most + kTokThreads / 32 + 16) * 4 +
           (kMaxConvWidth - 1) * 2 * a.d_state * elem;
  };
  constexpr size_t kMost = 48 * 1024;  // fewer CTAs a group, as long as each needs no more than this
  int c = hpg < 8 ? hpg : 8;
  while (c > 1 && (long long)a.seqs * a.groups * c > 12LL * device_sm_count() && smem_of((c + 1) / 2) <= kMost)
    c = (c + 1) / 2;
  const size_t smem = smem_of(c);
  const void* fn = a.type == kTypeBF16 ? token_kernel<__nv_bfloat16>(a.d_state) : token_kernel<float>(a.d_state);
  // eight CTAs of the widest group of one-channel heads take 90 KB
  static_assert((2 * kMaxDState + 5 * (kMaxGroupChannels / 8) + kTokThreads / 32 + 16 +
                 (kMaxConvWidth - 1) * 2 * kMaxDState) * 4 <= 227 * 1024, "any group fits");
  if (smem > kMost &&
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return kErrLaunch;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.seqs * a.groups * c));
  cfg.blockDim = dim3(kTokThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = c;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TokenArgs copy = a;
  void* args[] = {&copy};
  return cudaLaunchKernelExC(&cfg, fn, args) == cudaSuccess ? kOk : kErrLaunch;
}

int launch_gated_norm(const NormArgs& a, cudaStream_t stream) {
  return a.type == kTypeBF16 ? launch_norm<__nv_bfloat16>(a, stream) : launch_norm<float>(a, stream);
}

}  // namespace ervf
