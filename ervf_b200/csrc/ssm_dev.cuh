// ssm_dev.cuh -- device helpers shared by the state-space kernels: packed
// sequences and the scalar functions of the scan.
#pragma once

#include "common.cuh"
#include "ssm.h"

namespace ervf {

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// v / (1 + exp(-v)) with the approximate exponential and reciprocal: off by a
// few units of 2^-24 |v| (the exponential's error grows with |v|, but weighs
// sigmoid' there).  The exact forms cost four times the instructions, and the
// convolution and the norm were bound by them.
__device__ __forceinline__ float silu(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(v * -1.4426950408889634f)));
  return v * r;
}
// log(1 + exp(v)); above 20 the 1 is below half a unit in the last place
__device__ __forceinline__ float softplus(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

// Tokens [begin, begin + len) of sequence i, kept inside the token array
// whatever the offsets say.
__host__ __device__ __forceinline__ void seq_range(const Packing& p, int i, int& begin, int& len) {
  if (!p.cu) {
    begin = 0;
    len = p.tokens;
    return;
  }
  const int b = min(max(p.cu[i], 0), p.tokens), e = min(max(p.cu[i + 1], 0), p.tokens);
  begin = b;
  len = max(e - b, 0);
}

// State slot of sequence i, or -1 for none.
__device__ __forceinline__ int seq_slot(const Packing& p, int i) {
  const int s = p.slots ? p.slots[i] : i;
  return s >= 0 && s < p.n_slots ? s : -1;
}

// Tile `tile` of the packed sequences, each cut into tiles of `size` tokens
// from its own first token: which sequence, and the tile's place in it.  One
// warp; false past the last tile, with `total` the number of tiles.  Walks the
// offsets: for few sequences.
__device__ __forceinline__ bool find_tile(const Packing& p, int tile, int size, int& seq, int& nth, int& total) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int i0 = 0; i0 < p.seqs; i0 += 32) {
    int n = 0;
    if (i0 + lane < p.seqs) {
      int b, len;
      seq_range(p, i0 + lane, b, len);
      n = (len - 1) / size + (len > 0);
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const int sum = __shfl_sync(0xffffffffu, inc, 31);
    if (tile >= 0 && tile < base + sum) {
      const unsigned m = __ballot_sync(0xffffffffu, tile < base + inc);
      const int l = __ffs(m) - 1;
      seq = i0 + l;
      nth = tile - base - __shfl_sync(0xffffffffu, inc - n, l);
      return true;
    }
    base += sum;
  }
  total = base;
  return false;
}

// Tiles of 2^shift tokens in places of their own, with gaps: sequence i owns the
// places from cu[i] >> shift, plus i, up to the next one's first.  These are
// at least its tiles and never none, and all of them at most (tokens >> shift) +
// seqs; so a tile is found by a search in the offsets instead of their running
// sum.
__host__ __device__ __forceinline__ int first_place(int begin, int i, int shift) { return (begin >> shift) + i; }
// Which sequence owns a place (for falling offsets: some sequence), and its
// tokens; one warp, 32 offsets at a time.  False before the first sequence's.
__device__ __forceinline__ bool find_place(const Packing& p, int place, int shift, int& seq, int& nth, int& begin,
                                           int& len) {
  const int lane = threadIdx.x & 31;
  seq = 0;
  for (int n = p.seqs;;) {
    const int step = (n + 31) / 32, i = lane * step;
    int b = 0, l = 0;
    if (i < n) seq_range(p, seq + i, b, l);
    const unsigned m = __ballot_sync(0xffffffffu, i < n && first_place(b, seq + i, shift) <= place);
    if (!m) return false;
    const int at = 31 - __clz(m);
    seq += at * step;
    n = min(step, n - at * step);
    if (step > 1) continue;
    begin = __shfl_sync(0xffffffffu, b, at);
    len = __shfl_sync(0xffffffffu, l, at);
    nth = place - first_place(begin, seq, shift);
    return true;
  }
}

// The chunked scan's table of steps: pairs of entries (a pair's two heads) for
// each head pair and each chunk of `total`, pair after pair.  It holds
// most_chunks chunks a pair, whatever the offsets say (decreasing ones could
// name a token twice); entry of head k = 2 pair + (0 or 1), or -1 for a chunk
// behind the last.
__host__ __device__ __forceinline__ int most_chunks(const Packing& p, int size) { return p.tokens / size + p.seqs; }
__host__ __device__ __forceinline__ long long step_entry(int k, int chunk, int total) {
  return chunk < total ? 2 * ((long long)(k >> 1) * total + chunk) + (k & 1) : -1;
}

}  // namespace ervf
