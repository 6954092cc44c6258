// Launchers of the operators around the matrix products of a language-model
// training step: LayerNorm of any width (layernorm.hip), log probabilities of
// given tokens (token_logprobs.hip) and AdamW over many tensors
// (multi_adamw.hip).  All pointers are device pointers; the binding
// (bindings/lm_binding.cpp) has checked types, shapes and strides.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mfl {

enum ElemType : int { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };

// ---- LayerNorm -----------------------------------------------------------------
struct LayerNormFwd {
  const void* x;       // [M] rows of H, ldx elements apart
  const void* gamma;   // [H] or null
  const void* beta;    // [H] or null
  void* y;             // [M][H]
  float* mean;         // [M]
  float* rstd;         // [M]
  int64_t ldx;
  int M, H;
  float eps;
  int type, param_type;
};
struct LayerNormBwd {
  const void* dy;      // [M] rows of H, lddy apart
  const void* x;       // [M] rows of H, ldx apart
  const void* gamma;   // [H] or null
  const float* mean;
  const float* rstd;
  void* dx;            // [M][H]
  void* dgamma;        // [H] or null (no weight gradient wanted)
  void* dbeta;         // [H] or null
  float* part;         // layer_norm_bwd_parts() * 2 * H floats, when dgamma is wanted (null for none)
  int64_t ldx, lddy;
  int M, H;
  int type, param_type;
};
void launch_layer_norm_fwd(const LayerNormFwd& a, hipStream_t s);
void launch_layer_norm_bwd(const LayerNormBwd& a, hipStream_t s);
int layer_norm_bwd_parts(int M, int H, int type);

// ---- token log probabilities -----------------------------------------------------
constexpr int kTopMax = 32;
struct TokenLogprobs {
  const void* x;            // [N] rows of V logits, ldx apart
  const int64_t* target64;  // [N], or null with target32
  const int32_t* target32;
  float* logp;              // [N]
  float* entropy;           // [N]
  float* stats;             // [N][3]: maximum, sum of exp(x - maximum), entropy
  float* top_logp;          // [N][K]
  int64_t* top_ids;         // [N][K]
  void* work;               // token_logprobs_workspace() bytes
  int64_t ldx;
  int N, V, K, type;
};
struct TokenLogprobsBwd {
  const void* x;
  const int64_t* target64;
  const int32_t* target32;
  const float* stats;       // [N][3]
  const float* d_logp;      // [N] or null
  const float* d_entropy;   // [N] or null
  const float* d_top;       // [N][K] or null
  const int64_t* top_ids;   // [N][K], with d_top
  void* dx;                 // [N][C], columns V..C-1 zero
  int64_t ldx;
  int N, V, C, K, type;
};
size_t token_logprobs_workspace(int N, int V, int K, int type);
void launch_token_logprobs(const TokenLogprobs& a, hipStream_t s);
void launch_token_logprobs_bwd(const TokenLogprobsBwd& a, hipStream_t s);

// ---- AdamW over many tensors ---------------------------------------------------------
constexpr int kAdamBlock = 128;    // elements that share a scale of the 8-bit states
constexpr int kAdamChunk = 2048;   // elements of a workgroup: 8 to each of 256 threads
constexpr int kAdamGrads = 384;    // gradient pointers of a launch (kernel arguments hold 4 KB)
struct AdamTensor {                // one parameter, as the device table holds it
  void* p;
  uint16_t* mirror;                // bf16 copy or null
  int64_t offset;                  // of its states in the flat state buffers, a multiple of kAdamBlock
  int64_t numel;
  int decays;                      // takes the step's weight decay
  int param_type;
};
struct AdamChunk {
  int tensor;
  int chunk;
};
struct AdamScalars {               // written by the step's first launch
  float c1, c2;                    // 1 / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
  float lr;
  uint32_t key;
};
struct AdamStep {
  const AdamTensor* tensors;
  const AdamChunk* chunks;
  AdamScalars* scalars;
  int* arrived;                    // zero between steps
  int* step;
  const float* lr_scale;           // or null
  void* m;
  void* v;
  float* m_scale;                  // 8-bit states
  float* v_scale;
  double beta1, beta2;
  float eps, lr, wd;
  uint32_t seed;
  int state_bits;
};
struct AdamGrads {                 // gradients of tensors first .. first + count - 1
  const void* g[kAdamGrads];
  uint8_t type[kAdamGrads];
};
void launch_adam_begin(const AdamStep& a, hipStream_t s);
// whole: these are all of the step's chunks, at most kAdamWhole, and the launch
// does what launch_adam_begin would
constexpr int kAdamWhole = 512;
void launch_adam_chunks(const AdamStep& a, const AdamGrads& g, int first_tensor, int64_t first_chunk, int64_t chunks,
                        bool whole, hipStream_t s);

}  // namespace mfl
