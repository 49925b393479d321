// Host entry points of the kernels around the policy transformer. Pointers
// are device pointers, sizes have been checked by the caller, and every call
// only enqueues work on `stream`.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace blk {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// ---- layer_norm.hip
struct LayerNormFwd {
  const void *x, *residual, *weight, *bias;   // residual, weight, bias: or null
  void *y, *s;                                // s: or null without a residual
  float *mean, *rstd;                         // or null
  int64_t rows, x_stride, r_stride;           // strides in elements
  int width;
  float eps;
};
struct LayerNormBwd {
  const void *dy, *ds, *s, *weight;           // ds, weight: or null
  const float *mean, *rstd;
  void *dx, *dweight, *dbias;                 // dweight, dbias: both or none
  float *partial;                             // [blocks][2][width]
  int64_t rows, dy_stride, ds_stride, s_stride;
  int width, blocks;
};
int layer_norm_bwd_blocks(int64_t rows, int width, int dtype);
void layer_norm_fwd(const LayerNormFwd&, int dtype, int wdtype, hipStream_t);
void layer_norm_bwd(const LayerNormBwd&, int dtype, int wdtype, hipStream_t);

// ---- token_logprobs.hip
struct LogProbs {
  const void *logits;
  const int64_t *tokens;
  const uint8_t *mask;                        // or null; 1: allowed
  float *logprob, *entropy;
  float *stats;                               // [rows][4] or null
  float *top_logprobs;                        // or null, [rows][top_k]
  int64_t *top_tokens;
  int64_t rows, stride, mask_stride, ignore_index;
  int width, top_k;
  float inv_temperature;
};
struct LogProbsBwd {
  const void *logits;
  const uint8_t *mask;
  const float *stats;                         // the forward pass's
  const float *dlogprob, *dentropy;           // or null
  void *dlogits;                              // contiguous
  int64_t rows, stride, mask_stride;
  int width;
  float inv_temperature;
};
void token_logprobs_fwd(const LogProbs&, int dtype, hipStream_t);
void token_logprobs_bwd(const LogProbsBwd&, int dtype, hipStream_t);

// ---- grad_norm.hip
struct GradTensor {
  const void *in;
  void *out;                                  // where the clipped values go
  int64_t numel;
  int in_dtype, out_dtype;
};
int64_t grad_norm_blocks(const GradTensor*, int count, int64_t* chunk);
void grad_norm(const GradTensor*, int count, int64_t chunk, int order,
               double* partial, int64_t blocks, float* norm, float* coef,
               float max_norm, float eps, hipStream_t);
void grad_scale(const GradTensor*, int count, const float* coef, hipStream_t);

// ---- linear_act.hip
enum Act : int { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };
// out[i][j] = epilogue(sum over r of P[i][r] Q[j][r]), where an operand lies
// with r contiguous (P[i][r] at p + i stride + r) or, `_t`, with its other
// index contiguous (at p + r stride + i).
struct Product {
  const void *p, *q;
  int64_t p_stride, q_stride;
  int64_t p_cols, q_cols;                     // a row's elements, 8 at least: those
                                              // behind r are zero
  int64_t i, j, r;
  bool p_t, q_t;
  void *out;                                  // [i][j], contiguous
  int out_f32;                                // float32 instead of the type
  const void *bias;                           // [j] or null
  int bias_f32;
  const void *residual;                       // or null
  int64_t residual_stride;
  void *z;                                    // what goes into act, or null: float32,
                                              // in the type for a relu
  int act;
  int splits;                                 // parts of r ...
  float *partial;                             // ... [splits][i][partial_cols],
  int64_t partial_cols;                       // j up to a multiple of 8; or null
};
struct ActBwd {
  const void *dy, *z;                         // z: Product's, or null without act
  void *dz;                                   // or null without act
  float *partial;                             // [blocks][n], or null
  void *dbias;
  int dbias_f32;
  int64_t rows, n, dy_stride;
  int act, blocks;
};
int product_splits(const Product&);
void product(const Product&, int dtype, hipStream_t);
int act_bwd_blocks(int64_t rows, int64_t n);
void act_bwd(const ActBwd&, int dtype, hipStream_t);

}  // namespace blk
