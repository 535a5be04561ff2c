// ssm.h -- launchers of the state-space operators (ssm.cu, ssm_chunk.cu) and
// of the dense projection with an epilogue (linear.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ervf {

enum : int { kTypeF32 = 0, kTypeBF16 = 1 };
enum : int { kActNone = 0, kActRelu2 = 1, kActSilu = 2, kActGelu = 3 };

struct LinearArgs {
  const uint16_t* W;  // bf16 [rows][cols]
  const uint16_t* x;  // bf16 [tokens], x_stride elements apart
  const float* bias;  // [rows] or NULL
  const void* resid;  // out_type [tokens], resid_stride apart, or NULL
  void* out;          // out_type [tokens], out_stride apart
  long long x_stride, resid_stride, out_stride;
  int rows, cols, tokens;
  int out_type, act;
};
int launch_linear(const LinearArgs& a, cudaStream_t stream);

// Packed sequences: sequence i holds tokens [cu[i], cu[i + 1]) (cu NULL: one
// sequence of all tokens); its carried state is slot slots[i] (slots NULL: i)
// and is read where has[i] is not zero.  A slot outside [0, n_slots) is no
// state: the sequence starts from zero and nothing is stored.
struct Packing {
  const int* cu;
  const int* slots;
  const uint8_t* has;
  int seqs, tokens, n_slots;
};

struct ConvArgs {
  Packing pk;
  const void* x;
  void* out;
  const float* w;     // [channels][width]
  const float* bias;  // [channels] or NULL
  void* state;        // [n_slots][width - 1][channels], oldest input first, or NULL
  long long x_stride, out_stride;
  int type, channels, width, silu;
  int shift;  // set by the launcher: tokens of a CTA, 2^shift
};
int launch_conv1d_prompt(const ConvArgs& a, cudaStream_t stream);

struct ScanArgs {
  Packing pk;
  const void *x, *dt, *B, *C;
  void* y;
  const float *A, *D, *dt_bias;  // [heads]; D, dt_bias may be NULL
  float* state;                  // [n_slots][heads][head_dim][d_state] or NULL
  long long x_stride, dt_stride, b_stride, c_stride, y_stride;
  int type, heads, head_dim, groups, d_state;
  void* scratch;
  size_t scratch_bytes;
};
size_t ssm_prompt_scratch_bytes(int type, int tokens, int seqs, int heads, int head_dim, int groups, int d_state);
int launch_ssm_prompt(const ScanArgs& a, cudaStream_t stream);
int launch_scan_tokens(const ScanArgs& a, cudaStream_t stream);  // token by token, any type and size

struct TokenArgs {
  const void *xbc, *dt, *z;
  void* out;
  const float *conv_w, *conv_bias;
  void* conv_state;
  const float *A, *D, *dt_bias, *norm_w;
  float* state;
  const int* slots;
  long long xbc_stride, dt_stride, z_stride, out_stride;
  float eps;
  int type, seqs, n_slots, heads, head_dim, groups, d_state, width;
};
int launch_ssm_token(const TokenArgs& a, cudaStream_t stream);

struct NormArgs {
  const void *y, *z;
  void* out;
  const float* w;
  long long y_stride, z_stride, out_stride;
  float eps;
  int type, tokens, groups, group_size;
};
int launch_gated_norm(const NormArgs& a, cudaStream_t stream);

// Limits of the scan and convolution kernels.
constexpr int kMaxHeadDim = 256, kMaxDState = 256, kMaxConvWidth = 4, kMaxGroupChannels = 32768;
constexpr int kMaxConvChannels = 65535 * 128;  // a grid's second dimension, a thread a channel
constexpr int kMaxSeqs = 1 << 26;              // with the most tokens' chunks, a grid's first

}  // namespace ervf
